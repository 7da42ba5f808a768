// Tile products of the vocabulary cross entropy on the bf16 / fp16 matrix cores (gfx950), shared by its three products:
//
//   logits  l[v,t]  = sum_h W[v,h] H[t,h]      both operands hold the summed index contiguously
//   dHidden d[h,t]  = sum_v W[v,h] G[t,v]      W is read ACROSS its rows (transposing LDS read), G along them
//   dWeight d[h,v]  = sum_t H[t,h] G[t,v]      both read across their rows
//
// One workgroup owns a tile of TM x TN outputs and walks the summed index 64 at a time: the two operand slices
// (TM x 64 and TN x 64, 16-bit) go from memory straight into LDS (global_load_lds, 16 bytes a lane), three slices of a and
// two of b deep, 160 KiB.  Nothing is ever transposed in memory: an operand stored [k][m] is staged as it lies and read
// with ds_read_b64_tr_b16, which hands each lane four k values of its own column.
//
// What bounds it, at 16,384 tokens, width 1,024, 50,265 words, bf16 (1.69 TFLOP a product): power.  By the counters
// (SQ_VALU_MFMA_BUSY_CYCLES over 1,024 SIMDs, GRBM_GUI_ACTIVE) the matrix cores are busy for 53 % of the cycles in the logits,
// 45 % in G and 55 % in dHidden and dWeight together, at 1.93-1.97 GHz where 2.4 is the card's; matrix instructions alone, on
// random data in registers, reach 1,925 TFLOP/s (2,447 on zeros), this loop without its loads 1,620 and with everything
// 1,080-1,210; the library's product of 8,192^3 1,253.  Logits 1.45 ms, G 1.68 ms, dHidden and dWeight together 2.79 ms.
// Measured there and not kept: 256 x 128 tiles, two workgroups a CU (64-byte rows: L2 delivers 26 of 55 bytes a clock and
// CU), wave groups taking turns at LDS and matrix cores, a workgroup streaming through several tiles (no gain; not measured
// with tiles of few slices, where power does not bind), four waves of 128 x 128 (registers spill), non-temporal stores of G
// (1.6 times the time).
//
// float32 operands are two fp16 limbs, x 2^e = x1 + 2^-11 x2 with x1 and x2 rounded to 11 bits each, and e such that the
// tensor's largest magnitude is just below 2^15: good to 2^-22 of every element down to 2^-29 of the largest, and to an
// absolute 2^-51 of that below (subnormals).  Three products on the same code by walking the summed index three times:
// x1 y2 + x2 y1 first, then the sums times 2^-11, then x1 y1; x2 y2, below 2^-22 of |x||y|, is left out.  With the upper
// limb's own scale the lower one keeps its bits where a plain fp16 remainder would be subnormal (softmax values of
// unlikely words).  Against three bf16 limbs and six products: half the matrix instructions and two thirds of the bytes
// (log-likelihood of 64 sentences of up to 64 tokens, width 768, 50,265 words: 1,317 us so, 689 us with two limbs).
//
// Row order.  A lane of the 16x16x32 instruction ends up with rows 4g..4g+3 (g = lane / 16) of each of its eight row
// tiles.  The rows of W that feed row tile i are chosen as m = 32 g + 4 i + r, so that a lane's 8 x 4 results are 32
// CONSECUTIVE m of one column: the epilogues store 64 (16-bit) or 128 (float32) contiguous bytes a lane, and the
// reduction over the vocabulary is 32 values in registers plus two cross-lane steps.
//
// LDS.  Both layouts XOR the 16-byte piece index with bits of the row, chosen so that the 16 lanes that one LDS cycle
// serves fall on different banks for this row order; the direct-to-LDS load writes linearly, so the XOR is applied to
// the global address instead.
#pragma once
#include "lvae_common.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// in memory, aligned to their elements alone (the compiler emits unaligned 16-byte accesses)
typedef f32x4 __attribute__((aligned(4))) f32x4_u;
typedef s16x4 __attribute__((aligned(2))) s16x4_u;
typedef s16x8 __attribute__((aligned(2))) s16x8_u;

#define VG_BK 64               // a slice of the summed index: rows of 128 bytes, whole cache lines (64-byte rows load at half the rate)

// what one launch computes; pointers in elements of 16 bits unless named otherwise
struct VgArgs {
    const uint16_t* a;          // first row of the tile range (W at its first vocabulary row of the piece, or H)
    int64_t lda, plane_a;       // row pitch, distance between limb planes
    const uint16_t* b;
    int64_t ldb, plane_b;
    int64_t M;                  // valid outputs along m (rows of W, or columns h)
    int64_t a_cols;             // valid columns of an operand read across its rows
    int64_t N;                  // outputs along n: upper bound; the kept tokens are min(N, *n_rows) where n is tokens
    int64_t K;                  // summed index: vocabulary rows of the piece, padded H, or tokens (bound by *n_rows)
    const int* n_rows;          // kept tokens (device)
    int tiles_m, tiles_n, splits;
    // epilogues
    const float* bias;          // [>= M rounded up to 256] float32 of the piece, -inf behind the vocabulary
    const int* tgt;             // target of each kept token
    const float* lse;           // LSE of each kept token
    const float* gy;            // (scaled) upstream gradient of each kept token
    int64_t v0;                 // first vocabulary row of the piece
    float2* part;               // [tiles_m][ldp] running maximum and sum of each token over the tile
    int64_t ldp;
    float* picked;              // logit of the target
    uint16_t* g;                // [planes][rows][ldg] gradient of the logits
    int64_t ldg, plane_g;
    float* dbias;               // [tiles_n * waves along n][ld_dbias] partial column sums, or NULL
    int64_t ld_dbias;
    float* slab;                // [splits][slab_rows][ld_slab] float32 partial products
    int64_t ld_slab, slab_stride;
    int slab_add;               // add to what the slab holds
    void* out;                  // direct output [N][ld_out] of the operand type (float32 for limbs)
    int64_t ld_out;
    const float* unscale;       // device factor of the outputs, or NULL
    const int* exponents;       // limbs: e of the hidden states and of the weights; an output (dWeight) carries the first
};

enum { VG_LSE = 0, VG_GRAD = 1, VG_SLAB = 2, VG_OUT = 3 };
// the products as launched
enum { VG_LOGITS_LSE = 0, VG_LOGITS_GRAD = 1, VG_DHIDDEN = 2, VG_DWEIGHT_SLAB = 3, VG_DWEIGHT = 4 };
// element types: LVAE_F32 (two fp16 limbs), LVAE_BF16, LVAE_F16

template <int DT> __device__ __forceinline__ f32x4 vg_mma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (DT != LVAE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// round to nearest even (the compiler's conversions: v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <int DT> __device__ __forceinline__ uint16_t vg_round(float x) {
    if constexpr (DT == LVAE_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
    else return __builtin_bit_cast(uint16_t, (__bf16)x);
}
__device__ __forceinline__ float vg_bf16(uint16_t x) { return __uint_as_float((unsigned)x << 16); }

// x as two fp16 limbs, the lower one times 2^11; an infinity or NaN stays in the upper one
__device__ __forceinline__ void vg_limbs(float x, uint16_t l[2]) {
    const _Float16 hi = (_Float16)x;
    float r = (x - (float)hi) * 2048.f;
    if (!(fabsf((float)hi) < INFINITY)) r = 0.f;
    l[0] = __builtin_bit_cast(uint16_t, hi);
    l[1] = vg_round<LVAE_F16>(r);
}

// 16 bytes a lane from base + off (bytes) to LDS at the wave-uniform byte address lds (+ 16 lane).  As inline assembly:
// with the builtin the compiler waits for every load in flight before each transposing LDS read.  It has no output
// register; the waits are vg_wait_loads().
__device__ __forceinline__ const void* vg_uniform(const void* p) {
    const uint64_t a = (uint64_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    return (const void*)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ void vg_load_lds(unsigned lds, unsigned off, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(off), "s"(base) : "memory");
}
// until at most N of this wave's loads are in flight (they complete in order)
template <int N> __device__ __forceinline__ void vg_wait_loads() {
    static_assert(N < 64, "six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x70 | 0xF00);      // vmcnt alone
    asm volatile("" ::: "memory");
}

// until at most N of this wave's LDS reads are under way (they complete in order)
template <int N> __device__ __forceinline__ void vg_wait_lds() {
    static_assert(N < 16, "four bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F | N << 8);                               // lgkmcnt alone
    asm volatile("" ::: "memory");
}
// a barrier that nothing is scheduled across, the matrix instructions included
__device__ __forceinline__ void vg_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Which 16-byte piece of an LDS row holds piece 0 of its slice (XOR), for an operand stored along the summed index.  One
// LDS cycle serves 16 lanes of a 16-byte read, and not neighbours: rows 0-3 and 12-15 of one piece go together with rows
// 4-11 of the next.  With either reading (neighbours, or this) every set of 16 falls on different banks; measured without
// conflicts.  a: rows 32 q + 4 i + r in the row order above, 4 q + r counting for 16; b: 16 consecutive rows.
__device__ __forceinline__ int vg_swizzle(int row16) { return row16 >> 1; }
__device__ __forceinline__ int vg_swizzle_a(int row) { return vg_swizzle(((row >> 5) & 3) * 4 + (row & 3)); }
__device__ __forceinline__ int vg_swizzle_b(int row) { return vg_swizzle(row & 15); }

// sum over the 16 lanes of a row, by DPP (every lane gets it)
__device__ __forceinline__ float vg_row_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));    // quad_perm 1,0,3,2
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));    // quad_perm 2,3,0,1
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));   // half-row mirror
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));   // row mirror
    return v;
}

// TRA / TRB: the operand is stored [k][m] / [k][n].  WM x WN waves, each 128 x (16 NJ); NA slices of a and
// two of b in LDS at a time.
template <int WM, int WN, int NJ, int NA> constexpr int vg_lds_bytes() { return (NA * 128 * WM + 2 * 16 * NJ * WN) * VG_BK * 2; }

template <int DT, bool TRA, bool TRB, int EPI, int WM, int WN, int NJ, int NA>
__device__ __forceinline__ void vg_tile(const VgArgs& p, int tm, int tn, int64_t n0, int split, int n_kept, char* lds) {
    constexpr int W = WM * WN, MI = 8, TM = 128 * WM, TN = 16 * NJ * WN, BK = VG_BK;
    constexpr int A_BYTES = TM * BK * 2, B_BYTES = TN * BK * 2;
    constexpr int QA = A_BYTES / 1024 / W, QB = B_BYTES / 1024 / W;
    static_assert(QA * W * 1024 == A_BYTES && QB * W * 1024 == B_BYTES, "whole loads");

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    const int64_t m0 = (int64_t)tm * TM;
    constexpr bool N_TOKENS = !TRB;                     // n counts tokens unless G is read across its rows
    const int64_t n_lim = N_TOKENS ? (int64_t)n_kept : p.N;
    const int64_t k_lim = TRB ? (int64_t)n_kept : p.K;

    constexpr int NP = DT == LVAE_F32 ? 3 : 1;
    const int ks_all = (int)((k_lim + BK - 1) / BK);
    const int ks_per = (ks_all + p.splits - 1) / p.splits;
    const int ks0 = min(split * ks_per, ks_all), ks = min(ks_per, ks_all - ks0);
    const int steps = ks * NP;

    // ---- per-lane byte offsets of the loads, relative to the tile's (scalar) base
    unsigned offa[QA], offa_last[QA], offb[QB];
    const uint16_t* abase;
    const uint16_t* bbase;
    constexpr int SK = BK / 8, SA = TM / 8, SB = TN / 8;    // 16-byte pieces of a row stored along / across
    if constexpr (!TRA) {
        abase = p.a + m0 * p.lda;
#pragma unroll
        for (int q = 0; q < QA; ++q) {
            const int r = (q * W + wave) * (64 / SK) + lane / SK;
            const int64_t rc = min((int64_t)r, p.M - 1 - m0);
            offa[q] = (unsigned)(rc * p.lda * 2 + (((lane % SK) ^ vg_swizzle_a(r)) << 4));
            offa_last[q] = offa[q];
        }
    } else {
        abase = p.a + m0;
        const int64_t last = (int64_t)(ks_all - 1) * BK;
        const int64_t rows = TRB ? (int64_t)BK : max((int64_t)1, k_lim - last);     // H is padded to whole slices
#pragma unroll
        for (int q = 0; q < QA; ++q) {
            const int r = (q * W + wave) * (64 / SA) + lane / SA;
            const int64_t piece = min((int64_t)((lane % SA) ^ (r & 3)), (p.a_cols - m0) / 8 - 1);
            offa[q] = (unsigned)(r * p.lda * 2 + piece * 16);
            offa_last[q] = (unsigned)(min((int64_t)r, rows - 1) * p.lda * 2 + piece * 16);
        }
    }
    if constexpr (!TRB) {
        bbase = p.b + n0 * p.ldb;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            const int r = (q * W + wave) * (64 / SK) + lane / SK;
            offb[q] = (unsigned)(r * p.ldb * 2 + (((lane % SK) ^ vg_swizzle_b(r)) << 4));
        }
    } else {
        bbase = p.b + n0;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            const int r = (q * W + wave) * (64 / SB) + lane / SB;
            offb[q] = (unsigned)(r * p.ldb * 2 + (((lane % SB) ^ ((r & 3) << 1)) << 4));
        }
    }

    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds;
    // the next slice to load, of each operand: limb pair, slice, ring slot
    struct Next { int pair, k, slot; };
    Next na = {0, 0, 0}, nb_ = {0, 0, 0};
    const void *l_a = nullptr, *l_b = nullptr;
    unsigned l_dst_a = 0, l_dst_b = 0;
    bool l_last = false;
    // limb planes of the three products: (0,1) (1,0) (0,0)
    auto next_a = [&]() {
        const int limb = na.pair == 1;
        const int64_t kk = (int64_t)(ks0 + na.k) * BK;
        l_a = vg_uniform(abase + limb * p.plane_a + (TRA ? kk * p.lda : kk));
        l_last = TRA && !TRB && (ks0 + na.k == ks_all - 1);
        l_dst_a = __builtin_amdgcn_readfirstlane(lds0 + na.slot * A_BYTES + wave * 1024);
        if (++na.k == ks) { na.k = 0; ++na.pair; }
        na.slot = na.slot + 1 == NA ? 0 : na.slot + 1;
    };
    auto next_b = [&]() {
        const int limb = DT == LVAE_F32 && nb_.pair == 0;
        const int64_t kk = (int64_t)(ks0 + nb_.k) * BK;
        l_b = vg_uniform(bbase + limb * p.plane_b + (TRB ? kk * p.ldb : kk));
        l_dst_b = __builtin_amdgcn_readfirstlane(lds0 + NA * A_BYTES + nb_.slot * B_BYTES + wave * 1024);
        if (++nb_.k == ks) { nb_.k = 0; ++nb_.pair; }
        nb_.slot ^= 1;
    };
    auto load_a = [&](int q) { vg_load_lds(l_dst_a + q * W * 1024, (TRA && !TRB) ? (l_last ? offa_last[q] : offa[q]) : offa[q], l_a); };
    auto load_b = [&](int q) { vg_load_lds(l_dst_b + q * W * 1024, offb[q], l_b); };
    auto load_slice_a = [&]() {
        next_a();
#pragma unroll
        for (int q = 0; q < QA; ++q) load_a(q);
    };
    auto load_slice_b = [&]() {
        next_b();
#pragma unroll
        for (int q = 0; q < QB; ++q) load_b(q);
    };
    if (steps > 0) { load_slice_a(); load_slice_b(); }
    if (steps > 1) { load_slice_a(); load_slice_b(); }
    if (NA == 3 && steps > 2) load_slice_a();

    const int mp = lane & 15, g4 = lane >> 4;
    // this lane holds, for column n = n0 + 16 (NJ wn + j) + mp, the rows m = mb + 4 i + r
    const int64_t mb = m0 + wm * 128 + g4 * 32;
    const int nb = wn * 16 * NJ + mp;

    f32x4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if constexpr (DT != LVAE_F32 && (EPI == VG_LSE || EPI == VG_GRAD)) x = *(const f32x4*)(p.bias + mb + 4 * i);
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = x;
    }

    // lane constants of the LDS reads
    const int row_a = wm * 128 + (mp >> 2) * 32 + (mp & 3), row_b = wn * 16 * NJ + mp;
    int a_n[2], b_n[2];                    // along rows, for the two halves of a slice
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
        a_n[kk] = row_a * (BK * 2) + (((kk * 4 + g4) ^ vg_swizzle_a(row_a)) << 4);
        b_n[kk] = row_b * (BK * 2) + (((kk * 4 + g4) ^ vg_swizzle_b(row_b)) << 4);
    }
    const int kr = g4 * 8 + (mp >> 2);     // across rows: the k row this lane addresses (+ 32 kk, + 4 for the upper half)

    // Operands of half a slice in registers: a row tile's are replaced by the next half's as soon as its products are
    // issued; the column tiles', which all row tiles use, have a second set.
    s16x8 af[MI], bf[NJ], bn[NJ];
    auto read_a = [&](int i, const char* la, int kk) {
        if constexpr (!TRA) {
            af[i] = *(const s16x8*)(la + a_n[kk] + i * 4 * BK * 2);
        } else {
            const int piece = (wm * 16 + (mp & 3) * 4 + (i >> 1)) ^ (mp >> 2);
            const int at = (kk * 32 + kr) * (TM * 2) + piece * 16 + (i & 1) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(la + at));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(la + at + 4 * TM * 2));
            af[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    auto read_b = [&](int j, const char* lb, int kk) {
        if constexpr (!TRB) {
            bn[j] = *(const s16x8*)(lb + b_n[kk] + j * 16 * BK * 2);
        } else {
            const int piece = (wn * 2 * NJ + j * 2 + ((mp & 3) >> 1)) ^ ((mp >> 2) << 1);
            const int at = (kk * 32 + kr) * (TN * 2) + piece * 16 + (mp & 1) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lb + at));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lb + at + 4 * TN * 2));
            bn[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };

    if (steps > 0) {
        const char *la = lds, *lb = lds + NA * A_BYTES;
        // the first half slice's operands
        vg_wait_loads<0>();
        vg_barrier();
#pragma unroll
        for (int j = 0; j < NJ; ++j) read_b(j, lb, 0);
#pragma unroll
        for (int i = 0; i < MI; ++i) read_a(i, la, 0);
        int slot_a = 0, slot_b = 0;
        for (int s = 0; s < steps; ++s) {
            if (DT == LVAE_F32 && s == 2 * ks) {            // the mixed products are complete
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] *= 1.f / 2048;
            }
            // Half a slice is multiplied from registers while the next half is read from LDS and later slices' loads are
            // started, each BETWEEN the matrix instructions, a few cycles behind every NJ of them: the loads of a slice
            // in one go would hold up the wave until the address unit has taken them all.
            //
            // First half: reads the second half of slice s; starts the loads of a's slice s+2 (NA = 3), whose slot held
            // slice s-1: all its readers have used it before the barrier.
#pragma unroll
            for (int j = 0; j < NJ; ++j) bf[j] = bn[j];
            vg_barrier();
            const bool more_a = NA == 3 && s > 0 && s + 2 < steps;
            if (more_a) next_a();
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = vg_mma<DT>(af[i], bf[j], acc[i][j]);
                if (i < NJ) read_b(i, lb, 1);
                read_a(i, la, 1);
                if (more_a) {
#pragma unroll
                    for (int q = 0; q < QA; ++q)
                        if (q * MI / QA == i) load_a(q);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // Second half: reads the first half of slice s+1, for which every wave has waited for its own loads before the
            // barrier; starts the loads of b's slice s+2 (and a's, NA = 2) into the slots of slice s.  b's last reads of
            // slice s are waited for before the barrier; a's are used by products issued below, so with NA = 2 its
            // loads go behind them and a second barrier.
            __builtin_amdgcn_sched_barrier(0);
            vg_wait_lds<(MI - NJ) * (TRA ? 2 : 1)>();   // b's reads come before the last MI - NJ of a's
#pragma unroll
            for (int j = 0; j < NJ; ++j) bf[j] = bn[j];
            if (more_a) vg_wait_loads<QA>();
            else vg_wait_loads<0>();
            vg_barrier();
            const bool more = s + 2 < steps;
            if (more) next_b();
            slot_a = slot_a + 1 == NA ? 0 : slot_a + 1;
            slot_b ^= 1;
            la = lds + slot_a * A_BYTES;                // behind the last slice a slot is read that nothing needs
            lb = lds + NA * A_BYTES + slot_b * B_BYTES;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = vg_mma<DT>(af[i], bf[j], acc[i][j]);
                if (i < NJ) read_b(i, lb, 0);
                read_a(i, la, 0);
                if (more) {
#pragma unroll
                    for (int q = 0; q < QB; ++q)
                        if (q * MI / QB == i) load_b(q);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (NA == 2 && more) {
                vg_barrier();
                load_slice_a();
            }
        }
    }
    __syncthreads();

    // ---- epilogues
    if constexpr (DT == LVAE_F32 && (EPI == VG_LSE || EPI == VG_GRAD)) {
        const int e = -(p.exponents[0] + p.exponents[1]);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const f32x4 b = *(const f32x4*)(p.bias + mb + 4 * i);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = ldexpf(acc[i][j][r], e) + b[r];
        }
    }
    if constexpr (EPI == VG_LSE) {
        float2* red = (float2*)lds;                     // [WM][TN]; the last barrier has passed
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int64_t n = n0 + nb + j * 16;
            const int64_t rel = n < n_lim ? (int64_t)p.tgt[n] - p.v0 - mb : -1;
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float ref = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += lvae_exp2((acc[i][j][r] - ref) * LVAE_LOG2E);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (__any(rel >= 0 && rel < 32)) {          // few tiles hold a target of theirs
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (rel == 4 * i + r) p.picked[n] = acc[i][j][r];
            }
            if (g4 == 0) red[wm * TN + nb + j * 16] = make_float2(top, sum);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < TN; c += 64 * W) {
            if (n0 + c >= n_lim) continue;
            float2 x = red[c];
#pragma unroll
            for (int w = 1; w < WM; ++w) {
                const float2 y = red[w * TN + c];
                const float top = fmaxf(x.x, y.x), ref = top == -INFINITY ? 0.f : top;
                x.y = x.y * lvae_exp2((x.x - ref) * LVAE_LOG2E) + y.y * lvae_exp2((y.x - ref) * LVAE_LOG2E);
                x.x = top;
            }
            p.part[(int64_t)tm * p.ldp + n0 + c] = x;
        }
    } else if constexpr (EPI == VG_GRAD) {
        // 16 columns of G at a time go through this wave's own part of LDS, so that a store writes 256 bytes of a row at once
        // instead of 16 bytes of 64 places; two parts in turn.  A wave's LDS accesses complete in order.
        constexpr int PLANES = DT == LVAE_F32 ? 2 : 1, ROW = 256 + 16;
        static_assert(2 * W * PLANES * 16 * ROW <= vg_lds_bytes<WM, WN, WN == 4 ? 4 : NJ, NA>(), "LDS of the kernel");
        f32x4 colsum[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) colsum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int64_t n = n0 + nb + j * 16;
            const bool there = n < n_lim;               // rows behind the last kept token are written as zeros
            const int64_t rel = there ? (int64_t)p.tgt[n] - p.v0 - mb : -1;
            const float lse = there ? p.lse[n] : 0.f, gy = there ? p.gy[n] : 0.f;
            const bool all = n0 + (wn + 1) * 16 * NJ <= n_lim;
            const bool hit = __any(rel >= 0 && rel < 32);
            char* stage = lds + (wave * 2 + (j & 1)) * PLANES * 16 * ROW;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = lvae_exp2((acc[i][j][r] - lse) * LVAE_LOG2E);
            }
            if (hit) {
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] -= rel == 4 * i + r ? 1.f : 0.f;
            }
#pragma unroll
            for (int i = 0; i < MI; i += 2) {
                s16x8 o[2];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int ii = i + (e >> 2), r = e & 3;
                    float x = acc[ii][j][r] * gy;
                    if (!all) x = there ? x : 0.f;
                    colsum[ii][r] += x;
                    if constexpr (DT == LVAE_F32) {
                        uint16_t l[2];
                        vg_limbs(x, l);
                        o[0][e] = l[0]; o[1][e] = l[1];
                    } else {
                        // G is rounded once to the operand type, half a step of each element: the products need a
                        // 16-bit operand, and the gradients are rounded to the same type themselves
                        o[0][e] = vg_round<DT>(x);
                    }
                }
#pragma unroll
                for (int l = 0; l < PLANES; ++l) *(s16x8*)(stage + l * 16 * ROW + mp * ROW + g4 * 64 + i * 8) = o[l];
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int l = 0; l < PLANES; ++l)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = q * 4 + g4;
                    *(s16x8*)(p.g + l * p.plane_g + (n0 + wn * 16 * NJ + j * 16 + r) * p.ldg + m0 + wm * 128 + mp * 8) =
                        *(const s16x8*)(stage + l * 16 * ROW + r * ROW + mp * 16);
                }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
        if (p.dbias) {
            float* d = p.dbias + ((int64_t)tn * WN + wn) * p.ld_dbias + mb;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = vg_row_sum(colsum[i][r]);
                if (mp == 0) *(f32x4*)(d + 4 * i) = v;
            }
        }
    } else {
        // float32 slabs, or the output: 16 columns at a time through LDS as above, 256 or 512 bytes of a row at once
        constexpr bool F32 = EPI == VG_SLAB || DT == LVAE_F32;
        constexpr int ROW = (F32 ? 512 : 256) + 16, LANES = F32 ? 32 : 16, E = 128 / LANES;     // lanes a row, elements a lane
        static_assert(2 * W * 16 * ROW <= vg_lds_bytes<WM, WN, WN == 4 ? 4 : NJ, NA>(), "LDS of the kernel");
        const float f = EPI == VG_OUT && p.unscale ? p.unscale[0] : 1.f;
        const int e = EPI == VG_OUT && DT == LVAE_F32 ? -p.exponents[0] : 0;
        const int64_t m = m0 + wm * 128 + (lane % LANES) * E;
        const bool whole = m + E <= p.M;                // rows of any alignment: the stores need that of an element alone
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            char* stage = lds + (wave * 2 + (j & 1)) * 16 * ROW;
#pragma unroll
            for (int i = 0; i < MI; i += 2) {
                if constexpr (F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        f32x4 o = acc[i + h][j];
                        if constexpr (EPI == VG_OUT)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[r] = ldexpf(o[r] * f, e);
                        *(f32x4*)(stage + mp * ROW + g4 * 128 + (i + h) * 16) = o;
                    }
                } else {
                    s16x8 o;
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[k] = vg_round<DT>(acc[i + (k >> 2)][j][k & 3] * f);
                    *(s16x8*)(stage + mp * ROW + g4 * 64 + i * 8) = o;
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int q = 0; q < LANES / 4; ++q) {
                const int r = q * (64 / LANES) + lane / LANES;
                const int64_t n = n0 + wn * 16 * NJ + j * 16 + r;
                const char* from = stage + r * ROW + (lane % LANES) * 16;
                if (n >= n_lim) continue;
                if constexpr (EPI == VG_SLAB) {
                    float* to = p.slab + split * p.slab_stride + n * p.ld_slab + m;
                    if (m >= p.ld_slab) continue;       // the pitch is a multiple of 64
                    f32x4 v = *(const f32x4*)from;
                    if (p.slab_add) v += *(const f32x4*)to;
                    *(f32x4*)to = v;
                } else if constexpr (F32) {
                    float* to = (float*)p.out + n * p.ld_out + m;
                    const f32x4 v = *(const f32x4*)from;
                    if (whole) *(f32x4_u*)to = v;
                    else
                        for (int k = 0; k < 4; ++k)
                            if (m + k < p.M) to[k] = v[k];
                } else {
                    uint16_t* to = (uint16_t*)p.out + n * p.ld_out + m;
                    const s16x8 v = *(const s16x8*)from;
                    if (whole) *(s16x8_u*)to = v;
                    else
                        for (int k = 0; k < 8; ++k)
                            if (m + k < p.M) to[k] = v[k];
                }
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
    }
}

// The tile of a workgroup.  Workgroups go round the 8 XCDs; each XCD walks a contiguous range of tiles, four row tiles wide,
// so that the operand slices it shares stay in its own L2.  How many tokens count is known on the device alone: a last
// column of tiles with at most half its tokens is multiplied at half the width, and after all others, so that its tiles
// fill the last round (565 float32 tokens, width 768, 50,265 words, forward and backward: 905 us with whole tiles, 804 us
// so; 1,300 bfloat16 tokens: 514 and 496 us).
template <int DT, bool TRA, bool TRB, int EPI, int WM, int WN, int NJ, int NA>
__device__ __forceinline__ void vg_run(const VgArgs& p, unsigned block, char* lds) {
    constexpr int TN = 16 * NJ * WN;
    const int n_kept = __builtin_amdgcn_readfirstlane(p.n_rows[0]);
    int n_whole = p.tiles_n, n_half = 0;
    if constexpr (!TRB) {
        n_whole = (n_kept + TN - 1) / TN;
        if (TN == 256 && n_kept > 0 && n_kept - (n_whole - 1) * TN <= TN / 2) {
            --n_whole;
            n_half = 1;
        }
    }
    // whole tiles and half ones: the remainder of each goes to XCDs of its own, so that no XCD has more than its share
    const int per = p.tiles_m * n_whole, total = per * p.splits, total_h = n_half * p.tiles_m * p.splits;
    const int each = total / 8, rest = total % 8, each_h = total_h / 8, rest_h = total_h % 8;
    const int x = block & 7, x_h = (x - rest) & 7, mine = each + (x < rest ? 1 : 0);
    int l = block >> 3;
    if (l < mine) {
        int id = x * each + min(x, rest) + l;
        const int split = id / per;
        id -= split * per;
        const int group = 4 * n_whole, g = id / group, first = g * 4, wide = min(4, p.tiles_m - first);
        const int tm = first + (id - g * group) % wide, tn = (id - g * group) / wide;
        vg_tile<DT, TRA, TRB, EPI, WM, WN, NJ, NA>(p, tm, tn, (int64_t)tn * TN, split, n_kept, lds);
    } else if constexpr (!TRB && TN == 256) {
        l -= mine;
        if (l >= each_h + (x_h < rest_h ? 1 : 0)) return;
        const int id = x_h * each_h + min(x_h, rest_h) + l, split = id / p.tiles_m;
        vg_tile<DT, TRA, TRB, EPI, WM, WN, NJ / 2, NA>(p, id - split * p.tiles_m, n_whole, (int64_t)n_whole * TN, split, n_kept, lds);
    }
}

template <int DT, bool TRA, bool TRB, int EPI, int WM, int WN, int NJ, int NA>
__global__ __launch_bounds__(64 * WM * WN, 2) void vg_kernel(VgArgs p) {
    __shared__ __align__(1024) char lds[vg_lds_bytes<WM, WN, NJ, NA>()];
    vg_run<DT, TRA, TRB, EPI, WM, WN, NJ, NA>(p, blockIdx.x, lds);
}

// Both products of a piece's G in one launch, so that the tiles of one fill the CUs that the last round of the other
// leaves idle; the longer tiles come first.
template <int DT, int EPI_W, int WM, int WN, int NJ, int NA>
__global__ __launch_bounds__(64 * WM * WN, 2) void vg_both_kernel(VgArgs h, VgArgs w, unsigned blocks_h, unsigned blocks_w, int h_first) {
    __shared__ __align__(1024) char lds[vg_lds_bytes<WM, WN, NJ, NA>()];
    const unsigned b = blockIdx.x;
    if (h_first ? b < blocks_h : b >= blocks_w)
        vg_run<DT, true, false, VG_SLAB, WM, WN, NJ, NA>(h, h_first ? b : b - blocks_w, lds);
    else
        vg_run<DT, true, true, EPI_W, WM, WN, NJ, NA>(w, h_first ? b - blocks_h : b, lds);
}
