// Norm of many tensors together, and clipping by it, in two launches per list (of up to 112 tensors a launch).
//
//   1. norm_kernel: every workgroup takes a contiguous run of 8,192-element chunks of the list and leaves one partial
//      (sum of squares in float64: no overflow or underflow of any float32 gradient, and an order of its own that never
//      changes; or the largest magnitude).
//   2. scale_kernel: every workgroup adds up all partials itself, in one order, so that no third launch or atomic is
//      needed; where the factor is 1 nothing is read or written in place.
//
// Bound by memory: one read of all gradients for the norm, one read and write more where they are scaled.  The tensor
// table travels as a kernel argument: no copy to the device, nothing to keep alive, and a captured graph holds it.
#include <stdlib.h>

#include "vocab_gemm.h"

namespace {

constexpr int MAX_TENSORS = 112;            // 36 bytes each: below 4 KiB of kernel arguments
constexpr int CHUNK = 8192;
constexpr int BLOCKS = 2048;                // workgroups (and partials) over all launches of a list, or a few more
constexpr int MIN_BLOCKS = 32;

struct Table {
    const void* src[MAX_TENSORS];
    void* dst[MAX_TENSORS];
    int64_t n[MAX_TENSORS];
    uint32_t first[MAX_TENSORS];            // first chunk
    uint8_t type[MAX_TENSORS];              // source type | destination type << 4
    int32_t count;
    uint32_t chunks;
};
static_assert(sizeof(Table) <= 4032, "kernel arguments");

// eight elements from any element-aligned address (the compiler emits unaligned 16-byte accesses)
typedef f32x4 __attribute__((aligned(4))) f32x4_u;
typedef s16x8 __attribute__((aligned(2))) s16x8_u;

__device__ __forceinline__ void load8(const void* p, int64_t i, int dt, float x[8]) {
    if (dt == LVAE_F32) {
        const f32x4_u* q = (const f32x4_u*)((const float*)p + i);
        const f32x4 a = q[0], b = q[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
    } else {
        const s16x8 v = *(const s16x8_u*)((const uint16_t*)p + i);
        if (dt == LVAE_BF16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = vg_bf16((uint16_t)v[e]);
        } else {
            const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
        }
    }
}
__device__ __forceinline__ void store8(void* p, int64_t i, int dt, const float x[8]) {
    if (dt == LVAE_F32) {
        f32x4_u* q = (f32x4_u*)((float*)p + i);
        q[0] = f32x4{x[0], x[1], x[2], x[3]};
        q[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        s16x8 v;
        if (dt == LVAE_BF16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = vg_round<LVAE_BF16>(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = vg_round<LVAE_F16>(x[e]);
        }
        *(s16x8_u*)((uint16_t*)p + i) = v;
    }
}
__device__ __forceinline__ float load1(const void* p, int64_t i, int dt) {
    return dt == LVAE_F32 ? ((const float*)p)[i] : dt == LVAE_BF16 ? vg_bf16(((const uint16_t*)p)[i]) : (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store1(void* p, int64_t i, int dt, float x) {
    if (dt == LVAE_F32) ((float*)p)[i] = x;
    else ((uint16_t*)p)[i] = dt == LVAE_BF16 ? vg_round<LVAE_BF16>(x) : vg_round<LVAE_F16>(x);
}

// the larger, or NaN where there is one
__device__ __forceinline__ double nan_max(double m, double a) { return (a > m || a != a) ? a : m; }

template <bool INF> __device__ __forceinline__ double join(double a, double b) { return INF ? nan_max(a, b) : a + b; }

template <bool INF> __device__ __forceinline__ double block_join(double v, double* red) {       // 256 threads; all get it
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = join<INF>(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return join<INF>(join<INF>(red[0], red[1]), join<INF>(red[2], red[3]));
}

// the tensor that chunk c belongs to
__device__ __forceinline__ int find(const Table& t, uint32_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// this workgroup's chunks, the same share for each
__device__ __forceinline__ void my_chunks(const Table& t, uint32_t& c0, uint32_t& c1) {
    const uint32_t each = t.chunks / gridDim.x, rest = t.chunks % gridDim.x, b = blockIdx.x;
    c0 = b * each + min(b, rest);
    c1 = c0 + each + (b < rest ? 1 : 0);
}

template <bool INF> __global__ __launch_bounds__(256) void norm_kernel(Table t, double* part) {
    __shared__ double red[4];
    uint32_t c, c1;
    my_chunks(t, c, c1);
    double acc[2] = {0.0, 0.0};
    if (c < c1) {
        int e = find(t, c);
        for (; c < c1; ++c) {
            while (e + 1 < t.count && t.first[e + 1] <= c) ++e;
            const void* src = t.src[e];
            const int dt = t.type[e] & 15;
            const int64_t i0 = (int64_t)(c - t.first[e]) * CHUNK, n = t.n[e];
            if (i0 + CHUNK <= n) {
#pragma unroll
                for (int u = 0; u < CHUNK / 2048; ++u) {
                    float x[8];
                    load8(src, i0 + u * 2048 + threadIdx.x * 8, dt, x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if constexpr (INF) acc[k & 1] = nan_max(acc[k & 1], (double)fabsf(x[k]));
                        else acc[k & 1] = fma((double)x[k], (double)x[k], acc[k & 1]);
                    }
                }
            } else {
                for (int64_t i = i0 + threadIdx.x; i < n; i += 256) {
                    const double x = fabs((double)load1(src, i, dt));
                    acc[0] = INF ? nan_max(acc[0], x) : fma(x, x, acc[0]);
                }
            }
        }
    }
    const double v = block_join<INF>(join<INF>(acc[0], acc[1]), red);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <bool INF> __device__ __forceinline__ float total(const double* part, int parts, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) v = join<INF>(v, part[i]);
    v = block_join<INF>(v, red);
    return (float)(INF ? v : sqrt(v));
}

template <bool INF> __global__ __launch_bounds__(256) void total_kernel(const double* part, int parts, float* norm) {
    __shared__ double red[4];
    const float n = total<INF>(part, parts, red);
    if (threadIdx.x == 0) norm[0] = n;
}

template <bool INF> __global__ __launch_bounds__(256) void scale_kernel(Table t, const double* part, int parts, float max_norm,
                                                                        float* norm) {
    __shared__ double red[4];
    const float n_all = total<INF>(part, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = n_all;
    float f = max_norm / (n_all + 1e-6f);
    f = f > 1.f ? 1.f : f;                   // NaN stays
    uint32_t c, c1;
    my_chunks(t, c, c1);
    if (c >= c1) return;
    int e = find(t, c);
    for (; c < c1; ++c) {
        while (e + 1 < t.count && t.first[e + 1] <= c) ++e;
        const void* src = t.src[e];
        void* dst = t.dst[e];
        if (f == 1.f && dst == src) continue;
        const int dt = t.type[e] & 15, ot = t.type[e] >> 4;
        const int64_t i0 = (int64_t)(c - t.first[e]) * CHUNK, n = t.n[e];
        if (i0 + CHUNK <= n) {
#pragma unroll
            for (int u = 0; u < CHUNK / 2048; ++u) {
                const int64_t i = i0 + u * 2048 + threadIdx.x * 8;
                float x[8];
                load8(src, i, dt, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] *= f;
                store8(dst, i, ot, x);
            }
        } else {
            for (int64_t i = i0 + threadIdx.x; i < n; i += 256) store1(dst, i, ot, load1(src, i, dt) * f);
        }
    }
}

int64_t batches_of(int64_t count) { return count > 0 ? lvae_ceil_div(count, MAX_TENSORS) : 1; }
int64_t blocks_of(int64_t count) {
    const int64_t b = BLOCKS / batches_of(count);
    return b < MIN_BLOCKS ? MIN_BLOCKS : b;
}

struct Span {
    uintptr_t a, b;
    int64_t entry;
    int writes;
};
int by_start(const void* x, const void* y) {
    const Span *p = (const Span*)x, *q = (const Span*)y;
    return p->a < q->a ? -1 : p->a > q->a;
}

int64_t size_of(int dt) { return dt == LVAE_F32 ? 4 : 2; }

// no element that is written may belong to a second entry
int check_overlap(const lvae_grad_entry* list, int64_t count, int scale) {
    if (!scale) return LVAE_OK;
    Span* s = (Span*)malloc((size_t)(2 * count + 1) * sizeof(Span));
    if (!s) return lvae_set_error(LVAE_ERR_INVALID, "out of host memory for %lld tensors", (long long)count);
    int64_t m = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (list[i].n == 0) continue;
        const bool in_place = !list[i].dst || list[i].dst == list[i].src;
        const uintptr_t p = (uintptr_t)list[i].src, d = (uintptr_t)list[i].dst;
        s[m++] = Span{p, p + (uintptr_t)(list[i].n * size_of(list[i].dtype)), i, in_place};
        if (!in_place) s[m++] = Span{d, d + (uintptr_t)(list[i].n * size_of(list[i].out_dtype)), i, 1};
    }
    qsort(s, (size_t)m, sizeof(Span), by_start);
    int64_t a = -1, b = -1;
    uintptr_t end = 0, end_w = 0;                          // of what lies before: anything, what is written
    int64_t who = -1, who_w = -1;
    for (int64_t i = 0; i < m && a < 0; ++i) {
        if (s[i].writes && end > s[i].a) { a = who; b = s[i].entry; }
        else if (end_w > s[i].a) { a = who_w; b = s[i].entry; }
        if (s[i].b > end) { end = s[i].b; who = s[i].entry; }
        if (s[i].writes && s[i].b > end_w) { end_w = s[i].b; who_w = s[i].entry; }
    }
    free(s);
    if (a >= 0) return lvae_set_error(LVAE_ERR_INVALID, "tensors %lld and %lld share memory that is written", (long long)a, (long long)b);
    return LVAE_OK;
}

// the table of entries [i0, ...) that fit one launch; returns the next entry
int64_t fill(const lvae_grad_entry* list, int64_t count, int64_t i0, Table* t) {
    t->count = 0;
    t->chunks = 0;
    int64_t i = i0;
    for (; i < count && t->count < MAX_TENSORS; ++i) {
        const lvae_grad_entry& x = list[i];
        if (x.n == 0) continue;
        const int64_t chunks = lvae_ceil_div(x.n, CHUNK);
        if (t->count && (int64_t)t->chunks + chunks > 0x7FFFFFFF) break;
        const int k = t->count++;
        t->src[k] = x.src;
        t->dst[k] = x.dst ? x.dst : (void*)x.src;
        t->n[k] = x.n;
        t->first[k] = t->chunks;
        t->type[k] = (uint8_t)(x.dtype | (x.dst ? x.out_dtype : x.dtype) << 4);
        t->chunks += (uint32_t)chunks;
    }
    return i;
}

}  // namespace

extern "C" int lvae_clip_workspace_bytes(int64_t count, int64_t* out_bytes) {
    LVAE_CHECK_ARG(out_bytes && count >= 0, "bad arguments: count=%lld", (long long)count);
    // one launch more than the count says, should a table end early at its chunk limit
    *out_bytes = lvae_round_up((batches_of(count) * 2 + 1) * blocks_of(count) * 8, 256);
    return LVAE_OK;
}

extern "C" int lvae_clip_grads(const lvae_grad_entry* list, int64_t count, int inf_norm, int scale, double max_norm,
                               float* norm, void* ws, int64_t ws_bytes, void* stream) {
    int64_t need = 0;
    const int rc = lvae_clip_workspace_bytes(count, &need);
    if (rc != LVAE_OK) return rc;
    LVAE_CHECK_ARG(count == 0 || list, "list must be non-NULL");
    LVAE_CHECK_ARG(norm, "norm must be non-NULL");
    LVAE_CHECK_ARG(!scale || max_norm >= 0.0, "max_norm must not be negative or NaN");
    for (int64_t i = 0; i < count; ++i) {
        const lvae_grad_entry& x = list[i];
        LVAE_CHECK_ARG(x.n >= 0 && x.n < (1ll << 43), "tensor %lld: bad size %lld", (long long)i, (long long)x.n);
        LVAE_CHECK_ARG(x.n == 0 || x.src, "tensor %lld: NULL", (long long)i);
        LVAE_CHECK_ARG(x.dtype >= LVAE_F32 && x.dtype <= LVAE_F16 && (!x.dst || (x.out_dtype >= LVAE_F32 && x.out_dtype <= LVAE_F16)),
                       "tensor %lld: unknown dtype", (long long)i);
        LVAE_CHECK_ARG(x.dst != x.src || x.out_dtype == x.dtype, "tensor %lld: in place in another type", (long long)i);
        LVAE_CHECK_ARG(((uintptr_t)x.src % size_of(x.dtype)) == 0 && (!x.dst || ((uintptr_t)x.dst % size_of(x.out_dtype)) == 0),
                       "tensor %lld: not aligned to its elements", (long long)i);
    }
    const int rc2 = check_overlap(list, count, scale);
    if (rc2 != LVAE_OK) return rc2;
    if (!ws) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace is NULL (%lld bytes needed)", (long long)need);
    if ((uintptr_t)ws & 255) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    if (ws_bytes < need) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace too small: %lld < %lld bytes", (long long)ws_bytes, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    double* part = (double*)ws;
    const int64_t blocks = blocks_of(count), room = need / 8;
    int64_t parts = 0;
    Table t;
    for (int64_t i = 0; i < count;) {
        i = fill(list, count, i, &t);
        if (t.count == 0) continue;
        const int64_t g = t.chunks < blocks ? t.chunks : blocks;
        if (parts + g > room) return lvae_set_error(LVAE_ERR_UNSUPPORTED, "more than 2^31 chunks of gradients in one list");
        if (inf_norm) norm_kernel<true><<<dim3((unsigned)g), 256, 0, st>>>(t, part + parts);
        else norm_kernel<false><<<dim3((unsigned)g), 256, 0, st>>>(t, part + parts);
        LVAE_LAUNCH_CHECK();
        parts += g;
    }
    bool said = false;
    if (scale)
        for (int64_t i = 0; i < count;) {
            i = fill(list, count, i, &t);
            if (t.count == 0) continue;
            const int64_t g = t.chunks < blocks ? t.chunks : blocks;
            float* out = said ? nullptr : norm;
            said = true;
            if (inf_norm) scale_kernel<true><<<dim3((unsigned)g), 256, 0, st>>>(t, part, (int)parts, (float)max_norm, out);
            else scale_kernel<false><<<dim3((unsigned)g), 256, 0, st>>>(t, part, (int)parts, (float)max_norm, out);
            LVAE_LAUNCH_CHECK();
        }
    if (!said) {
        if (inf_norm) total_kernel<true><<<1, 256, 0, st>>>(part, (int)parts, norm);
        else total_kernel<false><<<1, 256, 0, st>>>(part, (int)parts, norm);
        LVAE_LAUNCH_CHECK();
    }
    return LVAE_OK;
}
