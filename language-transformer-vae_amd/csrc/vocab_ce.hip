// Log-likelihood of tokens under the softmax over the vocabulary, from hidden states, with its gradient: the host side
// of the tile products (vocab_gemm.h) and the kernels around them.
//
//   forward   rows -> pack -> tiles (running maximum and sum of each token over 256 words) -> finish
//   backward  rows -> pack -> per piece of the vocabulary: logits again -> G (16 bits, workspace) -> dHidden += G W,
//             dWeight = G^T H -> finish
//   few       up to 64 tokens: every wave streams 16 rows of W past all tokens -> finish
//
// `rows` lists the tokens that count, in order, with the place of their hidden state: padding costs nothing in the
// products, and what a hidden state of padding holds (NaN) meets nothing.
#include "vocab_gemm.h"

int lvae_vg_launch_bf16(int mode, int narrow, const VgArgs& p, hipStream_t st);
int lvae_vg_launch_f16(int mode, int narrow, const VgArgs& p, hipStream_t st);
int lvae_vg_launch_f32(int mode, int narrow, const VgArgs& p, hipStream_t st);
int lvae_vg_launch_both_bf16(int mode_w, const VgArgs& h, const VgArgs& w, int h_first, hipStream_t st);
int lvae_vg_launch_both_f16(int mode_w, const VgArgs& h, const VgArgs& w, int h_first, hipStream_t st);
int lvae_vg_launch_both_f32(int mode_w, const VgArgs& h, const VgArgs& w, int h_first, hipStream_t st);

namespace {

// G in 16 bits is kept relative to the largest upstream gradient: the -1 of a target is then exact (with the 1 / n of a
// mean inside, all targets would share one rounding error), and fp16, with the largest at 2^14, holds what is 2^-28 of it
constexpr float F16_G_SCALE = 16384.f;       // also of the limbs of float32
constexpr int64_t KEPT_HEAD = 256;
constexpr int MAX_PARTS = 512;              // workgroups that look for the largest magnitude of W, and of H
// workgroups that copy W, 1,024 threads each: with those that list tokens (512) and those of the bias (V / 1,024 < 2^16) a
// launch stays below 2^32 threads for every V; up to 2^25 words each copies its 16 rows and is done
constexpr int64_t MAX_COPIERS = 1 << 21;

struct Axes {
    int64_t size[3], stride[3];
};
__device__ __forceinline__ int64_t at_axes(const Axes& a, int64_t t) {
    // there are fewer than 2^31 tokens: 32-bit divisions
    const unsigned u = (unsigned)t, s2 = (unsigned)a.size[2], s1 = (unsigned)a.size[1], r = u / s2, q = r / s1;
    return q * a.stride[0] + (r - q * s1) * a.stride[1] + (u - r * s2) * a.stride[2];
}

template <int DT> __device__ __forceinline__ float load_as_float(const void* p, int64_t i) {
    if constexpr (DT == LVAE_F32) return ((const float*)p)[i];
    else if constexpr (DT == LVAE_BF16) return vg_bf16(((const uint16_t*)p)[i]);
    else return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dt) {
    return dt == LVAE_F32 ? load_as_float<LVAE_F32>(p, i)
         : dt == LVAE_BF16 ? load_as_float<LVAE_BF16>(p, i) : load_as_float<LVAE_F16>(p, i);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, float x, int dt) {
    if (dt == LVAE_F32) ((float*)p)[i] = x;
    else ((uint16_t*)p)[i] = dt == LVAE_BF16 ? vg_round<LVAE_BF16>(x) : vg_round<LVAE_F16>(x);
}

__device__ __forceinline__ int block_sum_int(int v, int* red) {          // 1024 threads
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < 16; ++w) s += red[w];
    return s;
}

struct RowsArgs {
    Axes hid, tgt, g;
    const int64_t* targets;
    const float* lse;           // backward: LSE of every token
    const float* gy;            // backward: upstream gradient
    const float* g_scale;
    int64_t T, V, ignore;
    float g_scale_to;           // what the largest |g| becomes
    int *tok, *tgt_of, *inv;    // of each kept token its number and its target; and back (-1: not kept)
    float *lse_of, *gy_of, *unscale;
    float *ll, *lse_out;        // forward: zeros for tokens that do not count
    int* n_rows;                // [2]: kept tokens; a counter, set to 0
    int64_t tokens;             // of a workgroup, a multiple of 16
    uint16_t* hpack;            // their hidden states
    int64_t hplane;
    // the other workgroups of the launch
    int row_blocks, bias_blocks;
    const void* bias;
    float* bias_out;
    int bias_dtype;
    int64_t Vpad;
    const void* weight;         // copied where the tiles cannot read it as it lies, or NULL
    uint16_t* wpack;
    int64_t wstride;
    const void* hidden;
    int H, Kp;
    float* largest;             // limbs: [2][MAX_PARTS] largest magnitudes, of H and of W
    int h_blocks, w_blocks;
    int* exponents;             // found from these, or with no blocks already there
};

// A row of hidden or of W as the tile products read it: Kp columns, zero behind H; float32 as two limb planes of x 2^e.  One wave per row.
template <int DT> __device__ __forceinline__ void pack_row(const void* src, int64_t base, bool there, int H, int Kp, int e, uint16_t* o, int64_t plane) {
    for (int k = (threadIdx.x & 63) * 8; k < Kp; k += 512) {
        if constexpr (DT == LVAE_F32) {
            const float* q = (const float*)src + base + k;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
            if (there && k + 8 <= H) {
                // past the caches: what is read next are the limbs (step of 565 tokens 770 us without, 761 with)
                const f32x4 a = __builtin_nontemporal_load((const f32x4_u*)q), b = __builtin_nontemporal_load((const f32x4_u*)(q + 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
            } else if (there) {
                for (int i = 0; i < 8; ++i) if (k + i < H) x[i] = q[i];
            }
            s16x8 w[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint16_t l[2];
                vg_limbs(ldexpf(x[i], e), l);
                w[0][i] = l[0]; w[1][i] = l[1];
            }
            *(s16x8*)(o + k) = w[0];
            *(s16x8*)(o + plane + k) = w[1];
        } else {
            const uint16_t* q = (const uint16_t*)src + base + k;
            s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
            if (there && k + 8 <= H) v = *(const s16x8_u*)q;
            else if (there) {
                for (int i = 0; i < 8; ++i) if (k + i < H) v[i] = q[i];
            }
            *(s16x8*)(o + k) = v;
        }
    }
}

// largest finite magnitude of a float32 row; one wave
__device__ __forceinline__ float row_largest(const float* row, int H, float top) {
    const int lane = threadIdx.x & 63;
    auto take = [&](float x) { const float a = fabsf(x); if (a > top && a < INFINITY) top = a; };
    int k = lane * 4;
    for (; k + 4 <= H; k += 256) {
        const f32x4 v = *(const f32x4_u*)(row + k);
#pragma unroll
        for (int i = 0; i < 4; ++i) take(v[i]);
    }
    for (; k < H; ++k) take(row[k]);
    return top;
}
__device__ __forceinline__ void store_largest(float top, float* to) {        // of 1024 threads
    __shared__ float red[16];
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) top = fmaxf(top, red[w]);
        to[0] = top;
    }
}
// e with 2^14 <= largest 2^e < 2^15, from the parts; every thread of a wave gets it
__device__ __forceinline__ int exponent_for(const float* parts, int n) {
    float top = 0.f;
    for (int i = threadIdx.x & 63; i < n; i += 64) top = fmaxf(top, parts[i]);
    top = wave_max(top);
    return top > 0.f ? 14 - ilogbf(top) : 0;
}

// For float32: the largest magnitudes of W and of the hidden states that count, from which the exponents follow.
__global__ __launch_bounds__(1024) void largest_kernel(RowsArgs p) {
    int b = blockIdx.x;
    const int wave = threadIdx.x >> 6;
    float top = 0.f;
    if (b < p.h_blocks) {
        for (int64_t t = (int64_t)b * 16 + wave; t < p.T; t += (int64_t)p.h_blocks * 16)
            if (p.targets[at_axes(p.tgt, t)] != p.ignore) top = row_largest((const float*)p.hidden + at_axes(p.hid, t), p.H, top);
        store_largest(top, p.largest + b);
    } else {
        b -= p.h_blocks;
        for (int64_t v = (int64_t)b * 16 + wave; v < p.V; v += (int64_t)p.w_blocks * 16)
            top = row_largest((const float*)p.weight + v * p.wstride, p.H, top);
        store_largest(top, p.largest + MAX_PARTS + b);
    }
}

// The tokens [first, end) of one workgroup: those that count go into the list, in order, and their hidden states into the
// operand.  How many count before `first` every workgroup finds by itself (8 bytes a token, from L2; at most 512
// workgroups do so) instead of in a launch of its own.
template <int DT> __device__ __forceinline__ void list_rows(const RowsArgs& p, int e) {
    __shared__ int red[16];
    __shared__ float redf[16];
    __shared__ int row_of[1024];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * p.tokens, end = min(first + p.tokens, p.T);
    int count = 0;
    for (int64_t u = threadIdx.x; u < first; u += 1024) count += p.targets[at_axes(p.tgt, u)] != p.ignore;
    int base = block_sum_int(count, red);
    float factor = 1.f, norm = 1.f;
    if (p.gy_of) {
        if (p.g_scale) factor = p.g_scale[0];
        // the largest finite upstream gradient, the same in every workgroup: an infinite one spoils its own token alone
        float top = 0.f;
        if ((p.g.stride[0] | p.g.stride[1] | p.g.stride[2]) == 0) {
            const float a = fabsf(p.gy[0] * factor);
            top = a < INFINITY ? a : 0.f;
        } else {
            for (int64_t u = threadIdx.x; u < p.T; u += 1024)
                if (p.targets[at_axes(p.tgt, u)] != p.ignore) {
                    const float a = fabsf(p.gy[at_axes(p.g, u)] * factor);
                    top = a > top && a < INFINITY ? a : top;
                }
        }
        top = wave_max(top);
        __syncthreads();
        if (lane == 0) redf[wave] = top;
        __syncthreads();
        norm = redf[0];
        for (int w = 1; w < 16; ++w) norm = fmaxf(norm, redf[w]);
        if (!(norm > 0.f)) norm = p.g_scale_to;             // nothing to keep in range: a factor of 1
        if (blockIdx.x == 0 && threadIdx.x == 0) p.unscale[0] = norm / p.g_scale_to;
    }
    for (int64_t c = first; c < end; c += 1024) {
        const int64_t t = c + threadIdx.x;
        const int64_t y = t < end ? p.targets[at_axes(p.tgt, t)] : p.ignore;
        const bool keep = t < end && y != p.ignore;
        const unsigned long long mask = __ballot(keep);
        __syncthreads();
        if (lane == 0) red[wave] = __popcll(mask);
        __syncthreads();
        int j = base + __popcll(mask & ((1ull << lane) - 1));
        for (int w = 0; w < 16; ++w) {
            if (w < wave) j += red[w];
            base += red[w];
        }
        row_of[threadIdx.x] = keep ? j : -1;
        if (t < end) {
            if (p.inv) p.inv[t] = keep ? j : -1;
            if (keep) {
                p.tok[j] = (int)t;
                p.tgt_of[j] = y >= 0 && y < p.V ? (int)y : -2;
                if (p.lse_of) {
                    p.lse_of[j] = p.lse[t];
                    const float g = -(p.gy[at_axes(p.g, t)] * factor);     // on the negative log-likelihood: G = (softmax - onehot) g
                    p.gy_of[j] = (g / norm) * p.g_scale_to;
                }
            } else {
                if (p.ll) p.ll[t] = 0.f;
                if (p.lse_out) p.lse_out[t] = 0.f;
            }
        }
        __syncthreads();
        const int here = (int)min((int64_t)1024, end - c);
        for (int i = wave; i < here; i += 16)
            if (row_of[i] >= 0)
                pack_row<DT>(p.hidden, at_axes(p.hid, c + i), true, p.H, p.Kp, e, p.hpack + (int64_t)row_of[i] * p.Kp, p.hplane);
    }
    if ((int)blockIdx.x == p.row_blocks - 1) {
        // the product of dWeight reads whole slices of tokens: zeros behind the last
        for (int64_t r = base + wave; r < (base + VG_BK - 1) / VG_BK * VG_BK; r += 16)
            pack_row<DT>(p.hidden, 0, false, p.H, p.Kp, e, p.hpack + r * p.Kp, p.hplane);
        if (threadIdx.x == 0) {
            p.n_rows[0] = base;
            p.n_rows[1] = 0;                    // the counter of finish_kernel
        }
    }
}

// All operands of the products in one launch: the list of tokens and their hidden states, the bias in float32 with -inf
// behind the vocabulary (no word beyond the last can count), and a padded copy of W where its rows do not serve as they
// lie.  With float32, two workgroups a CU, so that those that list tokens do not keep W waiting: 64 sentences of 64 tokens,
// width 768, 50,265 words: 83 us with one, 71 us with two; the list alone, 16 bits, gains nothing.
template <int DT> __global__ __launch_bounds__(1024, DT == LVAE_F32 ? 8 : 4) void prepare_kernel(RowsArgs p) {
    int b = blockIdx.x, e_h = 0, e_w = 0;
    if (DT == LVAE_F32) {
        if (p.w_blocks) {
            e_h = exponent_for(p.largest, p.h_blocks);
            e_w = exponent_for(p.largest + MAX_PARTS, p.w_blocks);
            if (b == 0 && threadIdx.x == 0) {
                p.exponents[0] = e_h;
                p.exponents[1] = e_w;
            }
        } else {
            e_h = p.exponents[0];
            e_w = p.exponents[1];
        }
    }
    if (b < p.row_blocks) {
        list_rows<DT>(p, e_h);
        return;
    }
    b -= p.row_blocks;
    if (b < p.bias_blocks) {
        const int64_t v = (int64_t)b * 1024 + threadIdx.x;
        if (v < p.Vpad) p.bias_out[v] = v >= p.V ? -INFINITY : p.bias ? load_any(p.bias, v, p.bias_dtype) : 0.f;
        return;
    }
    b -= p.bias_blocks;
    const int64_t step = (int64_t)(gridDim.x - p.row_blocks - p.bias_blocks) * 16;
    for (int64_t r = (int64_t)b * 16 + (threadIdx.x >> 6); r < p.V; r += step)
        pack_row<DT>(p.weight, r * p.wstride, true, p.H, p.Kp, e_w, p.wpack + r * p.Kp, p.V * p.Kp);
}

__device__ __forceinline__ float2 merge_lse(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x), ref = top == -INFINITY ? 0.f : top;
    return make_float2(top, a.y * lvae_exp2((a.x - ref) * LVAE_LOG2E) + b.y * lvae_exp2((b.x - ref) * LVAE_LOG2E));
}

struct FinishArgs {
    const float2* part;         // [tiles][ldp]
    int tiles;
    int64_t ldp;
    const float* picked;
    const int *tok, *tgt;
    int* n_rows;                // [2]: kept tokens; workgroups that are done
    float *ll, *lse;
    float *loss, *each;         // -sum of ll (over the kept tokens with `mean`) and the factor of each in it, or NULL
    double* sums;               // [workgroups]
    int mean;
};
// LSE of each kept token from its partials; 16 tokens of a workgroup at a time, 16 threads a token.  The loss, where one is asked for:
// every workgroup leaves the sum of its tokens, and the last one to be done adds them up in order.
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs p) {
    __shared__ float2 red[16][16];
    __shared__ double redd[4];
    __shared__ int last;
    const int g = threadIdx.x >> 4;
    const int64_t n = p.n_rows[0];
    double mine = 0.0;
    for (int64_t j0 = (int64_t)blockIdx.x * 16; j0 < n; j0 += (int64_t)gridDim.x * 16) {
        const int64_t j = j0 + (threadIdx.x & 15);
        float2 x = make_float2(-INFINITY, 0.f);
        if (j < n)
            for (int i = g; i < p.tiles; i += 64) {
                float2 y[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    y[u] = i + 16 * u < p.tiles ? p.part[(int64_t)(i + 16 * u) * p.ldp + j] : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int u = 0; u < 4; ++u) x = merge_lse(x, y[u]);
            }
        __syncthreads();
        red[g][threadIdx.x & 15] = x;
        __syncthreads();
        if (g == 0 && j < n) {
            for (int i = 1; i < 16; ++i) x = merge_lse(x, red[i][threadIdx.x]);
            float l = x.x + logf(x.y);
            const bool bad = p.tgt[j] < 0;
            if (bad) l = NAN;
            const float v = bad ? NAN : p.picked[j] - l;
            p.ll[p.tok[j]] = v;
            if (p.lse) p.lse[p.tok[j]] = l;
            mine += v;
        }
    }
    if (!p.loss) return;
    if (threadIdx.x < 64) {
        mine = wave_sum_d(mine);
        if (threadIdx.x == 0) {
            __hip_atomic_store(p.sums + blockIdx.x, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = __hip_atomic_fetch_add(p.n_rows + 1, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    double s = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256)
        s += __hip_atomic_load(p.sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) redd[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double f = -1.0 / (p.mean ? (double)max((int64_t)1, n) : 1.0);
        p.loss[0] = (float)((redd[0] + redd[1] + redd[2] + redd[3]) * f);
        p.each[0] = (float)f;
    }
}

// ---- few tokens: W streamed once -------------------------------------------------------------------------------
// A wave owns 16 words, whose rows come from memory into registers as they lie in the instruction's operand (a lane reads
// 32 consecutive bytes of its word's row: 128 bytes a row and step), a round of steps ahead of their use.  The tokens' rows
// go through LDS a round at a time, shared by eight waves.  The order of the summed index inside a step is the lanes' own,
// the same on both sides.  Bound by the read of W (width 768, 50,265 words, one token: 4.1 TB/s, with the launch that joins
// the parts 22 us in bfloat16, 42 in float32); beyond 32 float32 tokens by the float32 matrix instructions.  Measured, a
// call: 24 float32 tokens with the tokens read from memory by every wave 66 us, through LDS shared by four waves 51, by
// eight 47, by sixteen 47; 64 bfloat16 tokens by four 34, by eight 30.  Rounds of two steps serve more than 16 float32
// tokens and more than 32 others (24 float32: 47 us, 49 with four steps; 64: 69 and 72; 64 bfloat16: 30 both, without
// spilling), of four everything else (one bfloat16 token: 22.4 us, 22.7 with two); loads two rounds ahead gain nothing.
constexpr int FEW_WAVES = 8;
template <int DT> struct FewStep {
    static constexpr int K = DT == LVAE_F32 ? 32 : 64, LANE = K / 4;       // elements a step, and a lane's share
};
// a lane's share of a row at k, zeros behind H
template <int DT, bool ALIGNED> __device__ __forceinline__ void few_load(const void* row, int k, int H, f32x4 out[2]) {
    constexpr int SZ = DT == LVAE_F32 ? 4 : 2, E = 16 / SZ;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = k + h * E;
        out[h] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (ALIGNED) {
            // behind H the row's last piece is read again and dropped: no branch, so that loads go out together and the
            // compiler knows how many are in flight
            const f32x4 v = *(const f32x4*)((const char*)row + min(at, H - E) * SZ);
            out[h] = at < H ? v : out[h];
        } else if constexpr (DT == LVAE_F32) {
            if (at + 4 <= H) out[h] = *(const f32x4_u*)((const float*)row + at);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) if (at + e < H) out[h][e] = ((const float*)row)[at + e];
        } else {
            s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
            if (at + 8 <= H) v = *(const s16x8_u*)((const uint16_t*)row + at);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) if (at + e < H) v[e] = ((const uint16_t*)row)[at + e];
            out[h] = __builtin_bit_cast(f32x4, v);
        }
    }
}
template <int DT> __device__ __forceinline__ f32x4 few_mma(const f32x4 a[2], const f32x4 b[2], f32x4 c) {
    if constexpr (DT == LVAE_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[h][e], b[h][e], c, 0, 0, 0);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) c = vg_mma<DT>(__builtin_bit_cast(s16x8, a[h]), __builtin_bit_cast(s16x8, b[h]), c);
    }
    return c;
}

struct FewArgs {
    const void *hidden, *weight, *bias;
    const int64_t* targets;
    Axes hid, tgt;
    int64_t V, wstride;
    int T, H, bias_dtype, blocks;
    float2* part;               // [T][blocks]
    float* picked;              // [T]
};

template <int DT, int NT, bool ALIGNED> __global__ __launch_bounds__(64 * FEW_WAVES, 4) void few_kernel(FewArgs p) {
    constexpr int SZ = DT == LVAE_F32 ? 4 : 2, KS = FewStep<DT>::K, KL = FewStep<DT>::LANE;
    constexpr int U = NT * SZ > 4 ? 2 : 4, R = U * KS;       // steps and elements a round
    constexpr int PITCH = U * 128 + 16;                 // a token's bytes of a round in LDS
    constexpr int PER = U * 4, ROWS = 64 * FEW_WAVES / PER, PASSES = (NT * 16 + ROWS - 1) / ROWS;      // threads a token
    __shared__ float2 red[FEW_WAVES][NT * 16];
    __shared__ __align__(16) char tok[2][NT * 16 * PITCH];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mp = lane & 15, g4 = lane >> 4;
    const int64_t vw = ((int64_t)blockIdx.x * FEW_WAVES + wave) * 16;
    const char* wrow = (const char*)p.weight + min(vw + mp, p.V - 1) * p.wstride * SZ;
    const int t_row = threadIdx.x / PER, t_at = threadIdx.x % PER;
    const char* trow[PASSES];               // rows that this thread brings into LDS: 32 bytes of each a round
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
        trow[i] = (const char*)p.hidden + at_axes(p.hid, min(i * ROWS + t_row, p.T - 1)) * SZ;
    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};

    f32x4 w[2][U][2], bt[PASSES][2];          // this round's and the next one's
    auto load_w = [&](f32x4 (&to)[U][2], int k0) {
#pragma unroll
        for (int u = 0; u < U; ++u) few_load<DT, ALIGNED>(wrow, k0 + u * KS + g4 * KL, p.H, to[u]);
    };
    auto load_t = [&](int k0) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) few_load<DT, ALIGNED>(trow[i], k0 + t_at * KL, p.H, bt[i]);
    };
    auto store_t = [&](int to) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (NT * 16 < ROWS && t_row >= NT * 16) continue;
            char* q = tok[to] + (i * ROWS + t_row) * PITCH + t_at * 32;
            *(f32x4*)q = bt[i][0];
            *(f32x4*)(q + 16) = bt[i][1];
        }
    };
    load_t(0);
    load_w(w[0], 0);
    store_t(0);
    for (int k0 = 0;; k0 += 2 * R) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int k = k0 + d * R;
            if (k >= p.H) goto done;
            __syncthreads();
            load_t(k + R);
            load_w(w[d ^ 1], k + R);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const char* q = tok[d] + (n * 16 + mp) * PITCH + u * 128 + g4 * 32;
                    const f32x4 b[2] = {*(const f32x4*)q, *(const f32x4*)(q + 16)};
                    acc[n] = few_mma<DT>(w[d][u], b, acc[n]);
                }
            store_t(d ^ 1);                 // the other buffer: its readers have passed the barrier above
        }
    }
done:
    const int64_t v0 = vw + g4 * 4;
    float bias[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[r] = v0 + r < p.V && p.bias ? load_any(p.bias, v0 + r, p.bias_dtype) : 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int t = n * 16 + mp;
        const int64_t y = t < p.T ? p.targets[at_axes(p.tgt, t)] : -1;
        float x[4], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = v0 + r < p.V ? acc[n][r] + bias[r] : -INFINITY;
            if (y == v0 + r && v0 + r < p.V) p.picked[t] = x[r];
            top = fmaxf(top, x[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += lvae_exp2((x[r] - ref) * LVAE_LOG2E);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g4 == 0) red[wave][t] = make_float2(top, sum);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < p.T; t += 64 * FEW_WAVES) {
        float2 x = red[0][t];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) x = merge_lse(x, red[w][t]);
        p.part[(int64_t)t * p.blocks + blockIdx.x] = x;
    }
}

__global__ __launch_bounds__(256) void few_finish_kernel(const float2* part, int blocks, const float* picked,
                                                         const int64_t* targets, Axes tgt, int64_t V, int64_t ignore,
                                                         float* ll, float* lse) {
    __shared__ float2 red[4];
    const int t = blockIdx.x;
    const int64_t y = targets[at_axes(tgt, t)];
    if (y == ignore) {
        if (threadIdx.x == 0) {
            ll[t] = 0.f;
            if (lse) lse[t] = 0.f;
        }
        return;
    }
    float2 x = make_float2(-INFINITY, 0.f);
    for (int i = threadIdx.x; i < blocks; i += 256) x = merge_lse(x, part[(int64_t)t * blocks + i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = merge_lse(x, make_float2(__shfl_xor(x.x, o, 64), __shfl_xor(x.y, o, 64)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) x = merge_lse(x, red[w]);
        float l = x.x + logf(x.y);
        const bool bad = y < 0 || y >= V;
        if (bad) l = NAN;
        ll[t] = bad ? NAN : picked[t] - l;
        if (lse) lse[t] = l;
    }
}

// ---- backward: sums of the partial products ----------------------------------------------------------------------
struct FinalArgs {
    const float* slab;          // d_hidden: the slabs of a token's row, in order; zeros where the token does not count
    int64_t slab_stride, ld, T;
    const int* inv;
    int splits, H, dt, hidden_blocks;
    void* d_hidden;
    const float* part;          // d_bias: the partial column sums of the tiles that hold kept tokens
    int64_t ld_part, V;
    int per_tile, tile_rows, bias_dt;
    void* d_bias;
    const int* n_rows;
    const float* unscale;
    const int* exponents;       // d_hidden of limbs carries that of W
};
__global__ __launch_bounds__(256) void final_kernel(FinalArgs p) {
    __shared__ double red[8][32];
    if ((int)blockIdx.x < p.hidden_blocks) {
        const unsigned per = (p.H + 3) / 4;
        const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (i >= p.T * per) return;
        const int64_t t = i / per;
        const int h = (int)(i - t * per) * 4, j = p.inv[t];
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        if (j >= 0) {
            const float* q = p.slab + j * p.ld + h;
            for (int s = 0; s < p.splits; s += 4) {         // four loads in flight
                f32x4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = *(const f32x4*)(q + min(s + k, p.splits - 1) * p.slab_stride);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (s + k < p.splits) x += v[k];
            }
            x *= p.unscale[0];
            if (p.dt == LVAE_F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ldexpf(x[e], -p.exponents[1]);
            }
        }
        const int64_t o = t * p.H + h;
        if (h + 4 > p.H) {
            for (int e = 0; e < 4; ++e) if (h + e < p.H) store_any(p.d_hidden, o + e, x[e], p.dt);
        } else if (p.dt == LVAE_F32) {
            *(f32x4_u*)((float*)p.d_hidden + o) = x;
        } else {
            s16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = p.dt == LVAE_BF16 ? vg_round<LVAE_BF16>(x[e]) : vg_round<LVAE_F16>(x[e]);
            *(s16x4_u*)((uint16_t*)p.d_hidden + o) = v;
        }
        return;
    }
    const int64_t v = (int64_t)(blockIdx.x - p.hidden_blocks) * 32 + (threadIdx.x & 31);
    const int g = threadIdx.x >> 5;
    const int n = (p.n_rows[0] + p.tile_rows - 1) / p.tile_rows * p.per_tile;
    double x = 0.0;
    if (v < p.V)
        for (int i = g; i < n; i += 8) x += p.part[(int64_t)i * p.ld_part + v];
    red[g][threadIdx.x & 31] = x;
    __syncthreads();
    if (g || v >= p.V) return;
    for (int i = 1; i < 8; ++i) x += red[i][threadIdx.x];
    const float f = (float)x;
    store_any(p.d_bias, v, f * p.unscale[0], p.bias_dt);
}

// rows [0, rows) of the split weight gradient
__global__ __launch_bounds__(256) void dweight_kernel(const float* slab, int splits, int64_t slab_stride, int64_t ld,
                                                      int64_t rows, int H, const float* unscale, const int* exponents, void* out, int dt) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * H) return;
    const int64_t v = i / H;
    const int h = (int)(i - v * H);
    float x = 0.f;
    for (int s = 0; s < splits; ++s) x += slab[s * slab_stride + v * ld + h];
    x *= unscale[0];
    store_any(out, i, dt == LVAE_F32 ? ldexpf(x, -exponents[0]) : x, dt);
}

__global__ __launch_bounds__(256) void segment_sum_kernel(const float* x, int64_t n, int64_t len, float* out) {
    for (int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); s < n; s += (int64_t)gridDim.x * 4) {
        double a = 0.0;
        for (int64_t i = threadIdx.x & 63; i < len; i += 64) a += x[s * len + i];
        a = wave_sum_d(a);
        if ((threadIdx.x & 63) == 0) out[s] = (float)a;
    }
}

// the loss of few tokens
__global__ __launch_bounds__(64) void few_loss_kernel(const int64_t* targets, Axes tgt, int T, int64_t ignore, const float* ll,
                                                      int mean, float* loss, float* each) {
    const int t = threadIdx.x;                  // at most LVAE_VOCAB_FEW tokens
    static_assert(LVAE_VOCAB_FEW <= 64, "one wave");
    const double s = wave_sum_d(t < T ? (double)ll[t] : 0.0);
    const int n = __popcll(__ballot(t < T && targets[at_axes(tgt, t < T ? t : 0)] != ignore));
    if (t == 0) {
        const double f = -1.0 / (mean ? (double)max(1, n) : 1.0);
        loss[0] = (float)(s * f);
        each[0] = (float)f;
    }
}

// ---- the plan ------------------------------------------------------------------------------------------------------
struct Plan {
    int64_t T, Tpad, V, Vpad, H, Kp;
    int planes;
    bool few, direct_w;
    int narrow, tile_n;         // of the logits
    int64_t piece;              // words of the vocabulary a time (backward)
    int splits_h, splits_w;
    // offsets into the workspace, bytes
    int64_t tok, tgt, inv, lse, gy, head, largest, bias, hpack, wpack, part, picked, sums, g, slab, slab_w, dbias, bytes;
    int64_t kept, planes_bytes; // what a forward of float32 leaves for its backward: exponents, and W as limbs from KEPT_HEAD on
    int64_t few_blocks, ld_dbias;
};

int check_problem(const lvae_vocab_problem* q, Plan* pl) {
    LVAE_CHECK_ARG(q, "problem must be non-NULL");
    LVAE_CHECK_ARG(q->dtype >= LVAE_F32 && q->dtype <= LVAE_F16, "unknown dtype %d", q->dtype);
    LVAE_CHECK_ARG(q->bias_dtype >= LVAE_F32 && q->bias_dtype <= LVAE_F16, "unknown bias_dtype %d", q->bias_dtype);
    // the limits keep every launch below 2^32 threads
    LVAE_CHECK_ARG(q->V >= 1 && q->V < 1ll << 26 && q->H >= 1 && q->H <= 65536,
                   "bad shape: V=%lld H=%d (1 <= V < 2^26, 1 <= H <= 65536)", (long long)q->V, q->H);
    int64_t T = 1;
    for (int i = 0; i < 3; ++i) {
        LVAE_CHECK_ARG(q->size[i] >= 1 && q->size[i] < (1ll << 31), "bad shape: size[%d]=%lld", i, (long long)q->size[i]);
        T *= q->size[i];
        LVAE_CHECK_ARG(T < 1ll << 27, "too many tokens: 2^27 or more in one call");
    }
    LVAE_CHECK_ARG(T * q->H < 1ll << 33 && T * q->V < 1ll << 38, "too many tokens: %lld of them x H=%d >= 2^33, or x V=%lld >= 2^38",
                   (long long)T, q->H, (long long)q->V);
    LVAE_CHECK_ARG(q->weight_stride >= q->H, "weight_stride %lld < H %d", (long long)q->weight_stride, q->H);
    pl->T = T;
    pl->Tpad = lvae_round_up(T, 256);
    pl->V = q->V;
    pl->Vpad = lvae_round_up(q->V, 256);
    pl->H = q->H;
    pl->Kp = lvae_round_up(q->H, VG_BK);
    pl->planes = q->dtype == LVAE_F32 ? 2 : 1;
    // the tiles read W where it lies if its rows are whole 128-byte slices on 16-byte boundaries; else a padded copy
    pl->direct_w = q->dtype != LVAE_F32 && q->H % VG_BK == 0 && q->weight_stride % 8 == 0 &&
                   q->weight_stride < (1 << 22) && ((uintptr_t)q->weight & 15) == 0;
    pl->planes_bytes = lvae_round_up(pl->planes * pl->V * pl->Kp * 2, 256);
    pl->kept = q->dtype == LVAE_F32 && T > LVAE_VOCAB_FEW ? KEPT_HEAD + pl->planes_bytes : 0;
    // Tiles of 64 tokens, two workgroups a CU, where tiles of 256 would be mostly empty; for the logits also where these are
    // at most 128, so that the small ones take one round of the 256 CUs.  Step of 1,024 bfloat16 tokens, 4,900 words, width
    // 768 (80 tiles): 101 us narrow, 113 wide; 2,000 tokens, 3,800 words, width 640 (120): 133 and 144; 2,528 tokens, 3,697
    // words, width 640 (150): 157 and 150.
    pl->narrow = T <= 128 || pl->Vpad / 256 * lvae_ceil_div(T, 256) <= 128;
    pl->tile_n = pl->narrow ? 64 : 256;
    return LVAE_OK;
}

int64_t take(int64_t& at, int64_t bytes) {
    const int64_t o = at;
    at += lvae_round_up(bytes, 256);
    return o;
}

void plan_common(Plan* pl) {
    int64_t at = 0;
    pl->head = take(at, 256);                            // n_rows, unscale, exponents
    pl->largest = take(at, 2 * MAX_PARTS * 4);
    pl->tok = take(at, pl->Tpad * 4);
    pl->tgt = take(at, pl->Tpad * 4);
    pl->bias = take(at, pl->Vpad * 4);
    pl->hpack = take(at, pl->planes * pl->Tpad * pl->Kp * 2);
    pl->bytes = at;
}
// the last of the workspace, and not in it with `kept`
void plan_weight(Plan* pl) {
    int64_t at = pl->bytes;
    pl->wpack = pl->direct_w ? 0 : take(at, pl->planes_bytes);
    pl->bytes = at;
}

void plan_forward(Plan* pl) {
    pl->few = pl->T <= LVAE_VOCAB_FEW;
    if (pl->few) {
        int64_t at = 0;
        pl->few_blocks = lvae_ceil_div(pl->V, 16 * FEW_WAVES);
        pl->part = take(at, pl->T * pl->few_blocks * 8);
        pl->picked = take(at, pl->T * 4);
        pl->bytes = at;
        return;
    }
    plan_common(pl);
    int64_t at = pl->bytes;
    pl->part = take(at, pl->Vpad / 256 * pl->Tpad * 8);
    pl->picked = take(at, pl->Tpad * 4);
    pl->sums = take(at, pl->Tpad / 16 * 8);
    pl->bytes = at;
    plan_weight(pl);
}

void plan_backward(Plan* pl, bool want_h, bool want_w, bool want_b) {
    plan_common(pl);
    int64_t at = pl->bytes;
    pl->inv = take(at, pl->T * 4);
    pl->lse = take(at, pl->Tpad * 4);
    pl->gy = take(at, pl->Tpad * 4);
    // pieces of the vocabulary: G of one piece takes at most 512 MiB, and every piece is as large as the others.  Fewer
    // pieces mean fewer rounds of tiles that do not fill the GPU, and fewer additions to the slabs of dHidden (16,384
    // tokens, width 1,024, 50,265 words, bf16: 6.69 / 6.40 / 6.38 / 6.60 ms at 256 / 512 / 1,024 / 2,048 MiB)
    const int64_t per_word = pl->Tpad * pl->planes * 2;
    int64_t piece = (512ll << 20) / per_word / 256 * 256;
    if (piece < 1024) piece = 1024;
    if (piece > 1 << 20) piece = 1 << 20;
    const int64_t pieces = lvae_ceil_div(pl->Vpad, piece);
    pl->piece = lvae_round_up(lvae_ceil_div(pl->V, pieces), 256);
    pl->g = take(at, pl->planes * pl->Tpad * pl->piece * 2);
    const int64_t th = lvae_ceil_div(pl->H, 256);
    // the sum of d_hidden runs over the whole piece: it is split so that no tile takes more than 0.6 of a CU's share of the
    // launch that holds both products
    const int64_t tiles_h = th * lvae_ceil_div(pl->T, 256), tiles_w = th * lvae_ceil_div(pl->piece, 256);
    const int64_t ks_h = lvae_ceil_div(pl->piece, VG_BK), ks_w = lvae_ceil_div(pl->T, VG_BK);
    const int64_t share = (tiles_h * ks_h + tiles_w * ks_w) / 256 + 1;      // slices a CU, both products
    int64_t most = share * 6 / 10;
    if (most < 8) most = 8;
    pl->splits_h = (int)lvae_ceil_div(ks_h, most);
    if (pl->splits_h > 32) pl->splits_h = 32;
    // The weight gradient's sum is split where its tiles, unsplit, would outlast the rest of the launch by more than its
    // slabs take to write and to add up: at about 1.5 us a slice and product of limbs against 4 TB/s and a launch.  2,528
    // float32 tokens, width 640, 3,697 words: both products 188 us unsplit, 114 us and 11 for the sum in three parts.
    pl->splits_w = 1;
    const int64_t most_w = share < 8 ? 8 : share;
    if (ks_w > most_w) {
        const int64_t n = lvae_ceil_div(ks_w, most_w) < 32 ? lvae_ceil_div(ks_w, most_w) : 32;
        const double saved = 1.5 * (pl->planes == 2 ? 3 : 1) * (double)(ks_w - lvae_ceil_div(ks_w, n));
        if (saved > 6.0 + (double)(n * pl->piece * pl->Kp) * 8 / 4e6) pl->splits_w = (int)n;
    }
    pl->slab = want_h ? take(at, pl->splits_h * pl->Tpad * pl->Kp * 4) : 0;
    pl->slab_w = want_w && pl->splits_w > 1 ? take(at, pl->splits_w * pl->piece * pl->Kp * 4) : 0;
    // column sums of all pieces for one reduction at the end, or of one piece where that would take over 256 MiB
    const int64_t parts = pl->Tpad / pl->tile_n * (pl->narrow ? 2 : 4);
    pl->ld_dbias = parts * pl->Vpad * 4 <= 256ll << 20 ? pl->Vpad : pl->piece;
    pl->dbias = want_b ? take(at, parts * pl->ld_dbias * 4) : 0;
    pl->bytes = at;
    plan_weight(pl);
}

Axes axes_of(const lvae_vocab_problem* q, const int64_t* stride) {
    Axes a;
    for (int i = 0; i < 3; ++i) {
        a.size[i] = q->size[i];
        a.stride[i] = stride[i];
    }
    return a;
}

int check_ws(Plan& pl, const void* kept, void* ws, int64_t ws_bytes) {
    LVAE_CHECK_ARG(!kept || pl.kept, "nothing is kept of this problem: kept must be NULL");
    LVAE_CHECK_ARG(((uintptr_t)kept & 255) == 0, "kept must be 256-byte aligned");
    if (kept) pl.bytes -= pl.planes_bytes;
    if (!ws) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace is NULL (%lld bytes needed)", (long long)pl.bytes);
    if ((uintptr_t)ws & 255) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    if (ws_bytes < pl.bytes)
        return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace too small: %lld < %lld bytes", (long long)ws_bytes, (long long)pl.bytes);
    return LVAE_OK;
}

int check_data(const lvae_vocab_problem* q) {
    LVAE_CHECK_ARG(q->hidden && q->weight && q->targets, "hidden, weight and targets must be non-NULL");
    return LVAE_OK;
}

int launch_tiles(int dtype, int mode, int narrow, const VgArgs& a, hipStream_t st) {
    return dtype == LVAE_F32 ? lvae_vg_launch_f32(mode, narrow, a, st)
         : dtype == LVAE_BF16 ? lvae_vg_launch_bf16(mode, narrow, a, st) : lvae_vg_launch_f16(mode, narrow, a, st);
}

#define RUN(call)                    \
    do {                             \
        const int rc__ = (call);     \
        if (rc__ != LVAE_OK) return rc__; \
    } while (0)

int launch_both(int dtype, int mode_w, const VgArgs& h, const VgArgs& w, int h_first, hipStream_t st) {
    return dtype == LVAE_F32 ? lvae_vg_launch_both_f32(mode_w, h, w, h_first, st)
         : dtype == LVAE_BF16 ? lvae_vg_launch_both_bf16(mode_w, h, w, h_first, st) : lvae_vg_launch_both_f16(mode_w, h, w, h_first, st);
}

// rows, bias, W and hidden as the products read them; fills the operands of the logits' product
int launch_operands(const lvae_vocab_problem* q, const Plan& pl, RowsArgs& rows, char* kept, char* ws, VgArgs* a, hipStream_t st) {
    uint16_t* hp = (uint16_t*)(ws + pl.hpack);
    uint16_t* wp = pl.direct_w ? nullptr : (uint16_t*)(kept ? kept + KEPT_HEAD : ws + pl.wpack);
    float* bias = (float*)(ws + pl.bias);
    rows.tokens = lvae_round_up(lvae_ceil_div(pl.T, 512), 16);
    rows.hpack = hp;
    rows.hplane = pl.Tpad * pl.Kp;
    rows.row_blocks = (int)lvae_ceil_div(pl.T, rows.tokens);
    rows.bias_blocks = (int)lvae_ceil_div(pl.Vpad, 1024);
    rows.bias = q->bias;
    rows.bias_out = bias;
    rows.bias_dtype = q->bias_dtype;
    rows.Vpad = pl.Vpad;
    rows.weight = q->weight;
    rows.wpack = wp;
    rows.wstride = q->weight_stride;
    rows.H = q->H;
    rows.Kp = (int)pl.Kp;
    rows.hidden = q->hidden;
    rows.largest = (float*)(ws + pl.largest);
    const bool known = kept && rows.lse_of;                  // a backward that got what its forward has left
    rows.exponents = (int*)(kept ? kept : ws + pl.head + 128);
    if (q->dtype == LVAE_F32 && !known) {
        rows.h_blocks = (int)lvae_ceil_div(pl.T, 16);
        rows.w_blocks = (int)lvae_ceil_div(pl.V, 16);
        if (rows.h_blocks > MAX_PARTS) rows.h_blocks = MAX_PARTS;
        if (rows.w_blocks > MAX_PARTS) rows.w_blocks = MAX_PARTS;
        largest_kernel<<<dim3((unsigned)(rows.h_blocks + rows.w_blocks)), 1024, 0, st>>>(rows);
        LVAE_LAUNCH_CHECK();
    }
    const int64_t copiers = wp && !known ? lvae_ceil_div(pl.V, 16) : 0;
    const dim3 grid((unsigned)(rows.row_blocks + rows.bias_blocks + (copiers < MAX_COPIERS ? copiers : MAX_COPIERS)));
    if (q->dtype == LVAE_F32) prepare_kernel<LVAE_F32><<<grid, 1024, 0, st>>>(rows);
    else prepare_kernel<LVAE_BF16><<<grid, 1024, 0, st>>>(rows);       // 16 bits are 16 bits
    LVAE_LAUNCH_CHECK();
    *a = VgArgs{};
    a->a = (const uint16_t*)q->weight;
    a->lda = q->weight_stride;
    a->a_cols = pl.H;
    if (wp) {
        a->a = wp;
        a->lda = a->a_cols = pl.Kp;
        a->plane_a = pl.V * pl.Kp;
    }
    a->b = hp;
    a->ldb = pl.Kp;
    a->plane_b = pl.Tpad * pl.Kp;
    a->N = pl.T;
    a->K = pl.Kp;
    a->n_rows = rows.n_rows;
    a->tiles_n = (int)lvae_ceil_div(pl.T, pl.tile_n);
    a->splits = 1;
    a->bias = bias;
    a->tgt = rows.tgt_of;
    a->exponents = rows.exponents;
    return LVAE_OK;
}

RowsArgs rows_args(const lvae_vocab_problem* q, const Plan& pl, char* ws) {
    RowsArgs r = {};
    r.hid = axes_of(q, q->hidden_stride);
    r.tgt = axes_of(q, q->target_stride);
    r.targets = q->targets;
    r.T = pl.T;
    r.V = pl.V;
    r.ignore = q->ignore_index;
    r.tok = (int*)(ws + pl.tok);
    r.tgt_of = (int*)(ws + pl.tgt);
    r.n_rows = (int*)(ws + pl.head);
    r.unscale = (float*)(ws + pl.head + 64);
    return r;
}

template <int DT, int NT> void start_few(const FewArgs& f, bool aligned, hipStream_t st) {
    if (aligned) few_kernel<DT, NT, true><<<dim3((unsigned)f.blocks), 64 * FEW_WAVES, 0, st>>>(f);
    else few_kernel<DT, NT, false><<<dim3((unsigned)f.blocks), 64 * FEW_WAVES, 0, st>>>(f);
}
template <int DT> void start_few_n(const FewArgs& f, bool aligned, hipStream_t st) {
    if (f.T <= 16) start_few<DT, 1>(f, aligned, st);
    else if (f.T <= 32) start_few<DT, 2>(f, aligned, st);
    else start_few<DT, 4>(f, aligned, st);
}

}  // namespace

extern "C" int lvae_vocab_ll_workspace_bytes(const lvae_vocab_problem* q, int64_t* out_bytes) {
    Plan pl = {};
    LVAE_CHECK_ARG(out_bytes, "out_bytes must be non-NULL");
    RUN(check_problem(q, &pl));
    plan_forward(&pl);
    *out_bytes = pl.bytes;
    return LVAE_OK;
}

extern "C" int lvae_vocab_ll_kept_bytes(const lvae_vocab_problem* q, int64_t* out_bytes) {
    Plan pl = {};
    LVAE_CHECK_ARG(out_bytes, "out_bytes must be non-NULL");
    RUN(check_problem(q, &pl));
    *out_bytes = pl.kept;
    return LVAE_OK;
}

extern "C" int lvae_vocab_ll(const lvae_vocab_problem* q, float* ll, float* lse, void* kept, float* loss, float* each,
                             int mean, void* wsv, int64_t ws_bytes, void* stream) {
    Plan pl = {};
    RUN(check_problem(q, &pl));
    RUN(check_data(q));
    LVAE_CHECK_ARG(ll, "ll must be non-NULL");
    LVAE_CHECK_ARG(!loss == !each, "loss and each go together");
    plan_forward(&pl);
    RUN(check_ws(pl, kept, wsv, ws_bytes));
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)wsv;
    float2* part = (float2*)(ws + pl.part);
    float* picked = (float*)(ws + pl.picked);
    if (pl.few) {
        FewArgs f = {};
        f.hidden = q->hidden;
        f.weight = q->weight;
        f.bias = q->bias;
        f.targets = q->targets;
        f.hid = axes_of(q, q->hidden_stride);
        f.tgt = axes_of(q, q->target_stride);
        f.V = pl.V;
        f.wstride = q->weight_stride;
        f.T = (int)pl.T;
        f.H = q->H;
        f.bias_dtype = q->bias_dtype;
        f.blocks = (int)pl.few_blocks;
        f.part = part;
        f.picked = picked;
        const int per16 = q->dtype == LVAE_F32 ? 4 : 8;          // elements of 16 bytes
        bool aligned = (((uintptr_t)q->hidden | (uintptr_t)q->weight) & 15) == 0 && q->H % per16 == 0 && q->weight_stride % per16 == 0;
        for (int i = 0; i < 3; ++i) aligned = aligned && q->hidden_stride[i] % per16 == 0;
        if (q->dtype == LVAE_F32) start_few_n<LVAE_F32>(f, aligned, st);
        else if (q->dtype == LVAE_BF16) start_few_n<LVAE_BF16>(f, aligned, st);
        else start_few_n<LVAE_F16>(f, aligned, st);
        LVAE_LAUNCH_CHECK();
        few_finish_kernel<<<dim3((unsigned)pl.T), 256, 0, st>>>(part, f.blocks, picked, q->targets, f.tgt, pl.V, q->ignore_index, ll, lse);
        LVAE_LAUNCH_CHECK();
        if (loss) {
            few_loss_kernel<<<1, 64, 0, st>>>(q->targets, f.tgt, f.T, q->ignore_index, ll, mean, loss, each);
            LVAE_LAUNCH_CHECK();
        }
        return LVAE_OK;
    }
    RowsArgs rows = rows_args(q, pl, ws);
    rows.ll = ll;
    rows.lse_out = lse;
    VgArgs a;
    RUN(launch_operands(q, pl, rows, (char*)kept, ws, &a, st));
    a.M = pl.V;
    a.tiles_m = (int)(pl.Vpad / 256);
    a.part = part;
    a.ldp = pl.Tpad;
    a.picked = picked;
    RUN(launch_tiles(q->dtype, VG_LOGITS_LSE, pl.narrow, a, st));
    FinishArgs f = {};
    f.part = part;
    f.tiles = a.tiles_m;
    f.ldp = pl.Tpad;
    f.picked = picked;
    f.tok = rows.tok;
    f.tgt = rows.tgt_of;
    f.n_rows = rows.n_rows;
    f.ll = ll;
    f.lse = lse;
    f.loss = loss;
    f.each = each;
    f.sums = (double*)(ws + pl.sums);
    f.mean = mean;
    // with a loss at most one workgroup a CU: they leave through one counter (16,384 tokens: 30 us with 1,024, 20 us so)
    const int64_t groups = lvae_ceil_div(pl.T, 16);
    finish_kernel<<<dim3((unsigned)(loss && groups > 256 ? 256 : groups)), 256, 0, st>>>(f);
    LVAE_LAUNCH_CHECK();
    return LVAE_OK;
}

extern "C" int lvae_vocab_ll_bwd_workspace_bytes(const lvae_vocab_problem* q, int want_hidden, int want_weight, int want_bias,
                                                 int64_t* out_bytes) {
    Plan pl = {};
    LVAE_CHECK_ARG(out_bytes, "out_bytes must be non-NULL");
    RUN(check_problem(q, &pl));
    plan_backward(&pl, want_hidden != 0, want_weight != 0, want_bias != 0);
    *out_bytes = pl.bytes;
    return LVAE_OK;
}

extern "C" int lvae_vocab_ll_bwd(const lvae_vocab_problem* q, const float* lse, const float* g, const int64_t* g_stride,
                                 const float* g_scale, const void* kept, void* d_hidden, void* d_weight,
                                 void* d_bias, void* wsv, int64_t ws_bytes, void* stream) {
    Plan pl = {};
    RUN(check_problem(q, &pl));
    RUN(check_data(q));
    LVAE_CHECK_ARG(lse && g && g_stride, "lse, g and g_stride must be non-NULL");
    LVAE_CHECK_ARG(d_hidden || d_weight || d_bias, "no gradient asked for");
    plan_backward(&pl, d_hidden != nullptr, d_weight != nullptr, d_bias != nullptr);
    RUN(check_ws(pl, kept, wsv, ws_bytes));
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)wsv;
    RowsArgs rows = rows_args(q, pl, ws);
    rows.g = axes_of(q, g_stride);
    rows.lse = lse;
    rows.gy = g;
    rows.g_scale = g_scale;
    rows.g_scale_to = q->dtype == LVAE_BF16 ? 1.f : F16_G_SCALE;
    rows.inv = (int*)(ws + pl.inv);
    rows.lse_of = (float*)(ws + pl.lse);
    rows.gy_of = (float*)(ws + pl.gy);
    VgArgs a;
    RUN(launch_operands(q, pl, rows, (char*)const_cast<void*>(kept), ws, &a, st)       /* read only there */);
    const float* unscale = rows.unscale;
    const int64_t esz = q->dtype == LVAE_F32 ? 4 : 2;
    const int th = (int)lvae_ceil_div(pl.H, 256), waves_n = pl.narrow ? 2 : 4;
    uint16_t* gbuf = (uint16_t*)(ws + pl.g);
    VgArgs dl = a;                                       // the gradient of the logits
    dl.lse = rows.lse_of;
    dl.gy = rows.gy_of;
    dl.g = gbuf;
    dl.ldg = pl.piece;
    dl.plane_g = pl.Tpad * pl.piece;
    dl.ld_dbias = pl.ld_dbias;
    const bool bias_whole = pl.ld_dbias >= pl.Vpad;
    VgArgs h = {};                                       // dHidden
    h.lda = a.lda;
    h.plane_a = a.plane_a;
    h.a_cols = a.a_cols;
    h.b = gbuf;
    h.ldb = pl.piece;
    h.plane_b = dl.plane_g;
    h.M = pl.H;
    h.N = pl.T;
    h.n_rows = rows.n_rows;
    h.tiles_m = th;
    h.tiles_n = (int)lvae_ceil_div(pl.T, 256);
    h.splits = pl.splits_h;
    h.slab = (float*)(ws + pl.slab);
    h.ld_slab = pl.Kp;
    h.slab_stride = pl.Tpad * pl.Kp;
    VgArgs w = {};                                       // dWeight
    w.a = a.b;
    w.lda = pl.Kp;
    w.plane_a = a.plane_b;
    w.a_cols = pl.Kp;
    w.b = gbuf;
    w.ldb = pl.piece;
    w.plane_b = dl.plane_g;
    w.M = pl.H;
    w.n_rows = rows.n_rows;
    w.tiles_m = th;
    w.splits = pl.splits_w;
    w.slab = (float*)(ws + pl.slab_w);
    w.ld_slab = pl.Kp;
    w.slab_stride = pl.piece * pl.Kp;
    w.ld_out = pl.H;
    w.exponents = a.exponents;                           // dWeight carries that of H
    w.unscale = unscale;
    const int mode_w = pl.splits_w > 1 ? VG_DWEIGHT_SLAB : VG_DWEIGHT;
    FinalArgs f = {};
    f.part = (float*)(ws + pl.dbias);
    f.ld_part = pl.ld_dbias;
    f.V = d_bias ? pl.V : 0;
    f.per_tile = waves_n;
    f.tile_rows = pl.tile_n;
    f.bias_dt = q->bias_dtype;
    f.d_bias = d_bias;
    f.n_rows = rows.n_rows;
    f.unscale = unscale;
    f.exponents = a.exponents;
    for (int64_t v0 = 0; v0 < pl.V; v0 += pl.piece) {
        const int64_t words = pl.V - v0 < pl.piece ? pl.V - v0 : pl.piece;
        dl.a = a.a + v0 * a.lda;
        dl.M = words;
        dl.tiles_m = (int)lvae_ceil_div(words, 256);
        dl.bias = a.bias + v0;
        dl.v0 = v0;
        dl.dbias = d_bias ? (float*)(ws + pl.dbias) + (bias_whole ? v0 : 0) : nullptr;
        RUN(launch_tiles(q->dtype, VG_LOGITS_GRAD, pl.narrow, dl, st));
        if (d_bias && !bias_whole) {
            FinalArgs b = f;
            b.V = words;
            b.d_bias = (char*)d_bias + v0 * (q->bias_dtype == LVAE_F32 ? 4 : 2);
            final_kernel<<<dim3((unsigned)lvae_ceil_div(words, 32)), 256, 0, st>>>(b);
            LVAE_LAUNCH_CHECK();
        }
        h.a = dl.a;
        h.K = words;
        h.slab_add = v0 > 0;
        w.N = words;
        w.tiles_n = dl.tiles_m;
        w.out = (char*)d_weight + v0 * pl.H * esz;
        if (d_hidden && d_weight) {
            const int64_t ks_h = lvae_ceil_div(words, VG_BK) / pl.splits_h, ks_w = lvae_ceil_div(pl.T, VG_BK) / pl.splits_w;
            RUN(launch_both(q->dtype, mode_w, h, w, ks_h >= ks_w, st));
        } else {
            if (d_hidden) RUN(launch_tiles(q->dtype, VG_DHIDDEN, 0, h, st));
            if (d_weight) RUN(launch_tiles(q->dtype, mode_w, 0, w, st));
        }
        if (d_weight && pl.splits_w > 1) {
            dweight_kernel<<<dim3((unsigned)lvae_ceil_div(words * pl.H, 256)), 256, 0, st>>>(
                w.slab, pl.splits_w, w.slab_stride, w.ld_slab, words, (int)pl.H, unscale, a.exponents, w.out, q->dtype);
            LVAE_LAUNCH_CHECK();
        }
    }
    f.slab = h.slab;
    f.slab_stride = h.slab_stride;
    f.ld = h.ld_slab;
    f.T = pl.T;
    f.inv = rows.inv;
    f.splits = pl.splits_h;
    f.H = q->H;
    f.dt = q->dtype;
    f.hidden_blocks = d_hidden ? (int)lvae_ceil_div(pl.T * ((pl.H + 3) / 4), 256) : 0;
    f.d_hidden = d_hidden;
    if (!bias_whole) f.V = 0;
    const int64_t blocks = f.hidden_blocks + lvae_ceil_div(f.V, 32);
    if (blocks) {
        final_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(f);
        LVAE_LAUNCH_CHECK();
    }
    return LVAE_OK;
}

extern "C" int lvae_segment_sum_f32(const float* x, int64_t n, int64_t len, float* out, void* stream) {
    LVAE_CHECK_ARG(n >= 1 && n < (1ll << 26) && len >= 0, "bad shape: n=%lld len=%lld", (long long)n, (long long)len);
    LVAE_CHECK_ARG(out && (x || len == 0), "x and out must be non-NULL");
    const int64_t blocks = lvae_ceil_div(n, 4), most = 1 << 23;              // 2^24 workgroups would be 2^32 threads
    segment_sum_kernel<<<dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, (hipStream_t)stream>>>(x, n, len, out);
    LVAE_LAUNCH_CHECK();
    return LVAE_OK;
}
