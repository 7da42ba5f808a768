// Norm of many tensors together, and clipping by it, in two launches.
//
//   1. norm_kernel: every workgroup takes a contiguous run of 2,048-element chunks of the list and leaves one partial
//      (sum of squares in float64: no overflow or underflow of any float32 gradient, and an order of its own that never
//      changes; or the largest magnitude).
//   2. scale_kernel: every workgroup adds up all partials itself, in one order, so that no third launch or atomic is
//      needed; where the factor is 1 nothing is read or written in place.
//
// Bound by memory: one read of all gradients for the norm, one read and write more where they are scaled.  The tensor
// table travels as kernel arguments, so that nothing is copied from host memory and a captured graph holds it: up to 112
// tensors in the arguments of the two kernels themselves; longer lists are first written to the workspace by launches
// that only do that (2 us each), because one full launch over all tensors beats several of a part of the GPU each
// (260 tensors, 60 M bfloat16 elements into float32: 156 us with a launch for each 112, 130 us so; 389 float32 tensors,
// 253 M elements, 715 and 606 us; with scaling past the caches, below, 96 and 560 us).
// The norm reads 5.2-5.8 TB/s (253 M float32), scaling moves 5.4 TB/s (a large copy: 4.8).
#include <stdlib.h>

#include "vocab_gemm.h"

namespace {

constexpr int MAX_TENSORS = 112;            // 33 bytes each: below 4 KiB of kernel arguments
constexpr int CHUNK = 2048;                 // 8 elements a thread
constexpr int BLOCKS = 2048;                // workgroups, and partials: 8 a CU

struct Table {
    const void* src[MAX_TENSORS];
    void* dst[MAX_TENSORS];
    int64_t n[MAX_TENSORS];
    uint32_t first[MAX_TENSORS];            // first chunk
    uint8_t type[MAX_TENSORS];              // source type | destination type << 4
    int32_t count;
    uint32_t chunks;
    int32_t out;                // whether some tensor goes elsewhere
};
static_assert(sizeof(Table) <= 4032, "kernel arguments");

// the same in the workspace
struct LongTable {
    const void** src;
    void** dst;
    int64_t* n;
    uint32_t* first;
    uint8_t* type;
    int32_t count;
    uint32_t chunks;
    int32_t out;                // whether some tensor goes elsewhere
};

__global__ __launch_bounds__(128) void table_kernel(Table t, LongTable l, int at) {
    const int i = threadIdx.x;
    if (i >= t.count) return;
    l.src[at + i] = t.src[i];
    l.dst[at + i] = t.dst[i];
    l.n[at + i] = t.n[i];
    l.first[at + i] = t.first[i];
    l.type[at + i] = t.type[i];
}

// Eight elements of a full chunk: this thread's four of either half, so that the lanes of an access are neighbours in
// float32 (16 bytes a lane) and in 16 bits (8 bytes).  Any element-aligned address (the compiler emits unaligned accesses).
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <bool STREAM> __device__ __forceinline__ void load8(const void* p, int64_t i0, int dt, float x[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t i = i0 + h * (CHUNK / 2) + threadIdx.x * 4;
        if (dt == LVAE_F32) {
            const f32x4_u* q = (const f32x4_u*)((const float*)p + i);
            const f32x4 a = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * h + e] = a[e];
        } else {
            const s16x4_u* q = (const s16x4_u*)((const uint16_t*)p + i);
            const s16x4 v = STREAM ? __builtin_nontemporal_load(q) : *q;
            const f16x4 f = __builtin_bit_cast(f16x4, v);      // the vector: a bit cast of its element reads element 0
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * h + e] = dt == LVAE_BF16 ? vg_bf16((uint16_t)v[e]) : (float)f[e];
        }
    }
}
template <bool STREAM> __device__ __forceinline__ void store8(void* p, int64_t i0, int dt, const float x[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t i = i0 + h * (CHUNK / 2) + threadIdx.x * 4;
        if (dt == LVAE_F32) {
            // the pointer's own type has to reach the store: through a deduced parameter it would lose its alignment
            f32x4_u* q = (f32x4_u*)((float*)p + i);
            const f32x4 v = {x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
            if (STREAM) __builtin_nontemporal_store(v, q);
            else *q = v;
        } else {
            s16x4_u* q = (s16x4_u*)((uint16_t*)p + i);
            s16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = (short)(dt == LVAE_BF16 ? vg_round<LVAE_BF16>(x[4 * h + e]) : vg_round<LVAE_F16>(x[4 * h + e]));
            if (STREAM) __builtin_nontemporal_store(v, q);
            else *q = v;
        }
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
template <class T> __device__ __forceinline__ int find(const T& t, uint32_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// this workgroup's chunks, the same share for each
template <class T> __device__ __forceinline__ void my_chunks(const T& t, uint32_t& c0, uint32_t& c1) {
    const uint32_t each = t.chunks / gridDim.x, rest = t.chunks % gridDim.x, b = blockIdx.x;
    c0 = b * each + min(b, rest);
    c1 = c0 + each + (b < rest ? 1 : 0);
}

template <bool INF, class T> __global__ __launch_bounds__(256) void norm_kernel(T t, double* part) {
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
                float x[8];
                load8<false>(src, i0, dt, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if constexpr (INF) acc[k & 1] = nan_max(acc[k & 1], (double)fabsf(x[k]));
                    else acc[k & 1] = fma((double)x[k], (double)x[k], acc[k & 1]);
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

template <bool INF> __device__ __forceinline__ double total(const double* part, int parts, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) v = join<INF>(v, part[i]);
    v = block_join<INF>(v, red);
    return INF ? v : sqrt(v);
}

template <bool INF> __global__ __launch_bounds__(256) void total_kernel(const double* part, int parts, float* norm) {
    __shared__ double red[4];
    const double n = total<INF>(part, parts, red);
    if (threadIdx.x == 0) norm[0] = (float)n;
}

// STREAM: past the caches, for lists that pass through them anyway and would only push out what others need.  In 16 bits into
// float32, 60 M elements: a call 136 us without, 102 us with (loads alone 127, stores alone 119); 253 M float32: 614 and 571 us.
// The norm gains nothing: where the list fits the memory-side cache it is read from there (60 M: 41 us, streamed 51).
template <bool INF, bool STREAM, class T>
__global__ __launch_bounds__(256) void scale_kernel(T t, const double* part, int parts, double max_norm, float* norm) {
    __shared__ double red[4];
    const double n_all = total<INF>(part, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)n_all;
    // all elements share the factor's error: it is rounded once
    const double factor = max_norm / (n_all + 1e-6);
    const float f = factor > 1.0 ? 1.f : (float)factor;         // NaN stays
    uint32_t c, c1;
    my_chunks(t, c, c1);
    if (c >= c1 || (f == 1.f && !t.out)) return;
    // backwards: what the norm has read last is still in the memory-side cache
    int e = find(t, c1 - 1);
    for (uint32_t k = c1; k > c;) {
        --k;
        while (t.first[e] > k) --e;
        const void* src = t.src[e];
        void* dst = t.dst[e];
        if (f == 1.f && dst == src) continue;
        const int dt = t.type[e] & 15, ot = t.type[e] >> 4;
        const int64_t i0 = (int64_t)(k - t.first[e]) * CHUNK, n = t.n[e];
        if (i0 + CHUNK <= n) {
            float x[8];
            load8<STREAM>(src, i0, dt, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= f;
            store8<STREAM>(dst, i0, ot, x);
        } else {
            for (int64_t i = i0 + threadIdx.x; i < n; i += 256) store1(dst, i, ot, load1(src, i, dt) * f);
        }
    }
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

void sort_spans(Span* s, int64_t n) {
    for (int64_t i = 1; i < n; ++i)
        if (s[i].a < s[i - 1].a) {
            qsort(s, (size_t)n, sizeof(Span), by_start);
            return;
        }
}

int64_t size_of(int dt) { return dt == LVAE_F32 ? 4 : 2; }

// no element that is written may belong to a second entry
int check_overlap(const lvae_grad_entry* list, int64_t count, int scale) {
    if (!scale) return LVAE_OK;
    // sources and destinations apart: either list is mostly in order already (views of one buffer), and needs no sorting
    Span* buf = (Span*)malloc((size_t)(2 * count + 1) * sizeof(Span));
    if (!buf) return lvae_set_error(LVAE_ERR_INVALID, "out of host memory for %lld tensors", (long long)count);
    Span *s = buf, *d = buf + count;
    int64_t ns = 0, nd = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (list[i].n == 0) continue;
        const bool in_place = !list[i].dst || list[i].dst == list[i].src;
        const uintptr_t p = (uintptr_t)list[i].src, q = (uintptr_t)list[i].dst;
        s[ns++] = Span{p, p + (uintptr_t)(list[i].n * size_of(list[i].dtype)), i, in_place};
        if (!in_place) d[nd++] = Span{q, q + (uintptr_t)(list[i].n * size_of(list[i].out_dtype)), i, 1};
    }
    sort_spans(s, ns);
    sort_spans(d, nd);
    int64_t a = -1, b = -1;
    uintptr_t end = 0, end_w = 0;                          // of what lies before: anything, what is written
    int64_t who = -1, who_w = -1;
    for (int64_t i = 0, j = 0; i + j < ns + nd && a < 0;) {
        const Span& x = j >= nd || (i < ns && s[i].a <= d[j].a) ? s[i++] : d[j++];
        if (x.writes && end > x.a) { a = who; b = x.entry; }
        else if (end_w > x.a) { a = who_w; b = x.entry; }
        if (x.b > end) { end = x.b; who = x.entry; }
        if (x.writes && x.b > end_w) { end_w = x.b; who_w = x.entry; }
    }
    free(buf);
    if (a >= 0) return lvae_set_error(LVAE_ERR_INVALID, "tensors %lld and %lld share memory that is written", (long long)a, (long long)b);
    return LVAE_OK;
}

// the next entries from i0 on, at most MAX_TENSORS; chunks are counted over the whole list.  Returns the next entry.
int64_t fill(const lvae_grad_entry* list, int64_t count, int64_t i0, uint32_t* chunks, Table* t) {
    t->count = 0;
    int64_t i = i0;
    for (; i < count && t->count < MAX_TENSORS; ++i) {
        const lvae_grad_entry& x = list[i];
        if (x.n == 0) continue;
        const int k = t->count++;
        t->src[k] = x.src;
        t->dst[k] = x.dst ? x.dst : (void*)x.src;
        t->n[k] = x.n;
        t->first[k] = *chunks;
        t->type[k] = (uint8_t)(x.dtype | (x.dst ? x.out_dtype : x.dtype) << 4);
        *chunks += (uint32_t)lvae_ceil_div(x.n, CHUNK);
    }
    t->chunks = *chunks;
    t->out = 0;
    for (int k = 0; k < t->count; ++k) t->out |= t->dst[k] != t->src[k];
    return i;
}

constexpr int64_t PART_BYTES = BLOCKS * 8;
int64_t long_bytes(int64_t count) { return lvae_round_up(count * (8 + 8 + 8 + 4 + 1) + 256, 256); }

// bytes that scaling moves from which on it goes past the caches: half of the memory-side cache
constexpr int64_t STREAM_BYTES = 128ll << 20;

template <bool INF, class T>
int launch(const T& t, int scale, int64_t bytes, double max_norm, double* part, float* norm, hipStream_t st) {
    const int g = (int)(t.chunks < BLOCKS ? t.chunks : BLOCKS);
    norm_kernel<INF, T><<<dim3((unsigned)g), 256, 0, st>>>(t, part);
    LVAE_LAUNCH_CHECK();
    if (scale && bytes >= STREAM_BYTES) scale_kernel<INF, true, T><<<dim3((unsigned)g), 256, 0, st>>>(t, part, g, max_norm, norm);
    else if (scale) scale_kernel<INF, false, T><<<dim3((unsigned)g), 256, 0, st>>>(t, part, g, max_norm, norm);
    else total_kernel<INF><<<1, 256, 0, st>>>(part, g, norm);
    LVAE_LAUNCH_CHECK();
    return LVAE_OK;
}

}  // namespace

extern "C" int lvae_clip_workspace_bytes(int64_t count, int64_t* out_bytes) {
    LVAE_CHECK_ARG(out_bytes && count >= 0 && count <= (1 << 24), "bad arguments: count=%lld", (long long)count);
    *out_bytes = PART_BYTES + (count > MAX_TENSORS ? long_bytes(count) : 0);
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
    int64_t chunks = 0, bytes = 0;
    for (int64_t i = 0; i < count; ++i) {
        const lvae_grad_entry& x = list[i];
        LVAE_CHECK_ARG(x.n >= 0 && x.n < (1ll << 43), "tensor %lld: bad size %lld", (long long)i, (long long)x.n);
        LVAE_CHECK_ARG(x.n == 0 || x.src, "tensor %lld: NULL", (long long)i);
        LVAE_CHECK_ARG(x.dtype >= LVAE_F32 && x.dtype <= LVAE_F16 && (!x.dst || (x.out_dtype >= LVAE_F32 && x.out_dtype <= LVAE_F16)),
                       "tensor %lld: unknown dtype", (long long)i);
        LVAE_CHECK_ARG(x.dst != x.src || x.out_dtype == x.dtype, "tensor %lld: in place in another type", (long long)i);
        LVAE_CHECK_ARG(((uintptr_t)x.src % size_of(x.dtype)) == 0 && (!x.dst || ((uintptr_t)x.dst % size_of(x.out_dtype)) == 0),
                       "tensor %lld: not aligned to its elements", (long long)i);
        chunks += lvae_ceil_div(x.n, CHUNK);
        bytes += x.n * (size_of(x.dtype) + size_of(x.dst ? x.out_dtype : x.dtype));
    }
    LVAE_CHECK_ARG(chunks < (1ll << 31), "too many elements");
    const int rc2 = check_overlap(list, count, scale);
    if (rc2 != LVAE_OK) return rc2;
    if (!ws) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace is NULL (%lld bytes needed)", (long long)need);
    if ((uintptr_t)ws & 255) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    if (ws_bytes < need) return lvae_set_error(LVAE_ERR_WORKSPACE, "workspace too small: %lld < %lld bytes", (long long)ws_bytes, (long long)need);
    hipStream_t st = (hipStream_t)stream;
    double* part = (double*)ws;
    Table t;
    uint32_t at = 0;
    int64_t i = fill(list, count, 0, &at, &t);
    if (t.count == 0) {                                    // nothing but empty tensors
        total_kernel<false><<<1, 256, 0, st>>>(part, 0, norm);
        LVAE_LAUNCH_CHECK();
        return LVAE_OK;
    }
    if (i == count)
        return inf_norm ? launch<true>(t, scale, bytes, max_norm, part, norm, st) : launch<false>(t, scale, bytes, max_norm, part, norm, st);
    char* p = (char*)ws + PART_BYTES;
    LongTable l;
    l.src = (const void**)p;
    l.dst = (void**)(p + count * 8);
    l.n = (int64_t*)(p + count * 16);
    l.first = (uint32_t*)(p + count * 24);
    l.type = (uint8_t*)(p + count * 28);
    l.count = l.out = 0;
    for (;;) {
        if (t.count) {
            table_kernel<<<1, 128, 0, st>>>(t, l, l.count);
            LVAE_LAUNCH_CHECK();
            l.count += t.count;
            l.out |= t.out;
        }
        if (i == count) break;
        i = fill(list, count, i, &at, &t);
    }
    l.chunks = at;
    return inf_norm ? launch<true>(l, scale, bytes, max_norm, part, norm, st) : launch<false>(l, scale, bytes, max_norm, part, norm, st);
}
