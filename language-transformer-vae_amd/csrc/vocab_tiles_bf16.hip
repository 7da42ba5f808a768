// Tile products of the vocabulary cross entropy, element type bf16.
#define VG_DT LVAE_BF16
#define VG_NAME lvae_vg_launch_bf16
#define VG_NAME_BOTH lvae_vg_launch_both_bf16
#include "vocab_tiles.h"
