// Tile products of the vocabulary cross entropy, element type f32.
#define VG_DT LVAE_F32
#define VG_NAME lvae_vg_launch_f32
#define VG_NAME_BOTH lvae_vg_launch_both_f32
#include "vocab_tiles.h"
