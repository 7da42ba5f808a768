// Tile products of the vocabulary cross entropy, element type f16.
#define VG_DT LVAE_F16
#define VG_NAME lvae_vg_launch_f16
#define VG_NAME_BOTH lvae_vg_launch_both_f16
#include "vocab_tiles.h"
