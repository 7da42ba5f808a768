// Launchers of the tile products of one element type; each vocab_tiles_*.hip defines VG_DT, VG_NAME and VG_NAME_BOTH and includes this.
#include "vocab_gemm.h"


template <int DT, bool TRA, bool TRB, int EPI, int WM, int WN, int NJ, int NA>
static int vg_start(const VgArgs& p, hipStream_t st) {
    const int64_t blocks = lvae_round_up((int64_t)p.tiles_m * p.tiles_n * p.splits, 8);
    if (blocks >= 1ll << 31) return lvae_set_error(LVAE_ERR_UNSUPPORTED, "too many tiles: %lld", (long long)blocks);
    vg_kernel<DT, TRA, TRB, EPI, WM, WN, NJ, NA><<<dim3((unsigned)blocks), dim3(64 * WM * WN), 0, st>>>(p);
    LVAE_LAUNCH_CHECK();
    return LVAE_OK;
}

#define VG_WIDE 2, 4, 4, 3
#define VG_NARROW 2, 2, 2, 2

int VG_NAME(int mode, int narrow, const VgArgs& p, hipStream_t st) {
    switch (mode) {
        case VG_LOGITS_LSE:
            return narrow ? vg_start<VG_DT, false, false, VG_LSE, VG_NARROW>(p, st) : vg_start<VG_DT, false, false, VG_LSE, VG_WIDE>(p, st);
        case VG_LOGITS_GRAD:
            return narrow ? vg_start<VG_DT, false, false, VG_GRAD, VG_NARROW>(p, st) : vg_start<VG_DT, false, false, VG_GRAD, VG_WIDE>(p, st);
        case VG_DHIDDEN: return vg_start<VG_DT, true, false, VG_SLAB, VG_WIDE>(p, st);
        case VG_DWEIGHT_SLAB: return vg_start<VG_DT, true, true, VG_SLAB, VG_WIDE>(p, st);
        default: return vg_start<VG_DT, true, true, VG_OUT, VG_WIDE>(p, st);
    }
}

int VG_NAME_BOTH(int mode_w, const VgArgs& h, const VgArgs& w, int h_first, hipStream_t st) {
    const int64_t bh = lvae_round_up((int64_t)h.tiles_m * h.tiles_n * h.splits, 8), bw = lvae_round_up((int64_t)w.tiles_m * w.tiles_n * w.splits, 8);
    if (bh + bw >= 1ll << 31) return lvae_set_error(LVAE_ERR_UNSUPPORTED, "too many tiles: %lld", (long long)(bh + bw));
    const dim3 grid((unsigned)(bh + bw));
    if (mode_w == VG_DWEIGHT_SLAB) vg_both_kernel<VG_DT, VG_SLAB, VG_WIDE><<<grid, 512, 0, st>>>(h, w, (unsigned)bh, (unsigned)bw, h_first);
    else vg_both_kernel<VG_DT, VG_OUT, VG_WIDE><<<grid, 512, 0, st>>>(h, w, (unsigned)bh, (unsigned)bw, h_first);
    LVAE_LAUNCH_CHECK();
    return LVAE_OK;
}
