// Gradient norm, clipping and the Adam step over many tensors (include/cista_optim.h).
//
// All of them stream: 1 to 12 operations per 4 to 28 bytes, so they are bound by HBM for large
// models and by launches for small ones.  The tensors' table travels in the kernel argument
// (at most 4 KB), so nothing is uploaded or kept between calls; the work is cut into chunks, and a
// wave finds a chunk's tensor by one comparison per lane and a ballot.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>
#include <vector>

#include "../../include/cista_lstc.h"
#include "../../include/cista_optim.h"

namespace cista_optim {

constexpr int THREADS = 256;
constexpr int NORM_TENSORS = 192;        // 20 B each in the kernel argument
constexpr int NORM_BLOCKS = 1024;        // partial sums of one launch: see norm_partials
constexpr int NORM_UNROLL = 4;           // 16-byte loads in flight per thread
constexpr int NORM_CHUNK = THREADS * 16 * NORM_UNROLL;                   // bytes
constexpr int LINE = 128;                // bytes of a cache line
constexpr int ADAM_TENSORS = 64;         // 52 B each
constexpr int STEP_TENSORS = 448;        // 8 B each
constexpr int ADAM_CHUNK = THREADS * 4;  // elements: 4 of a thread
constexpr int JOIN_ALL = 512;            // partial values that every block of the next launch joins
constexpr long long CACHE = 256ll << 20; // bytes of the last-level cache
constexpr int FIVE = 32000;              // bytes of LDS with which 5 blocks run on a CU

// chunk c belongs to the last tensor whose first chunk is <= c (unused entries: ~0u; an empty
// tensor's first chunk is the next one's, which is found in its place)
template <int N> struct NormTable {
    void *data[N];
    uint64_t info[N];                    // numel | type << 56
    uint32_t first[N];
    uint32_t chunks, pad;
};

struct AdamTable {
    void *param[ADAM_TENSORS];
    const void *grad[ADAM_TENSORS];
    float *exp_avg[ADAM_TENSORS], *exp_avg_sq[ADAM_TENSORS], *master[ADAM_TENSORS];
    uint64_t info[ADAM_TENSORS];
    uint32_t first[ADAM_TENSORS];
    uint32_t chunks, pad;
};

template <int N> struct StepTable {
    float *step[N];
};

// what a tensor's update takes from its step count: lr / (1 - b1^t), 1 / sqrt(1 - b2^t), and for
// decoupled decay lr wd where that is below 1/2 (keep is 1), else 1 - lr wd (decay is 0): float32 holds
// either to 2^-24 of itself, but 1 - lr wd near 1 only to multiples of 2^-24
struct Rates {
    float size, inv_root, keep, decay;
};

struct AdamArgs {
    double lr, log_beta1, log_beta2, weight_decay, max_norm;
    const float *lr_device;
    float rate1, rate2, eps;                 // 1 - b1, 1 - b2
    float beta1, beta2;
    float decay;                             // in the gradient; 0 where it is decoupled
    int decoupled, maximize;
};

__device__ inline float to_f32(float x) { return x; }
__device__ inline float to_f32(__bf16 x) { return (float)x; }
__device__ inline float to_f32(_Float16 x) { return (float)x; }

// V elements at p, which is aligned to T only (global memory takes vector accesses at any address).
// STREAM: with the non-temporal hint, for data that will have left the caches before it is used again.
template <typename T, int V> struct Pack {
    T e[V];
};
template <int BYTES> struct Words {
    typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(2)));
};
#define GLOBAL __attribute__((address_space(1)))
template <bool STREAM, int V, typename T> __device__ inline Pack<T, V> load(const T *p) {
    using W = typename Words<sizeof(T) * V>::type;
    const GLOBAL W *q = (const GLOBAL W *)p;
    const W w = STREAM ? __builtin_nontemporal_load(q) : *q;
    Pack<T, V> r;
    __builtin_memcpy(&r, &w, sizeof(r));
    return r;
}
template <bool STREAM, typename T, int V> __device__ inline void store(T *p, const Pack<T, V> &r) {
    using W = typename Words<sizeof(T) * V>::type;
    W w;
    __builtin_memcpy(&w, &r, sizeof(w));
    GLOBAL W *q = (GLOBAL W *)p;
    if (STREAM) __builtin_nontemporal_store(w, q);
    else *q = w;
}

// the 16-bit value of a float32 result as it is stored: an opaque register keeps the compiler from
// rounding the last fma or product to 16 bits at once (v_fma_mixlo_f16), which is another value near
// a tie, and which it does in some loops and not in others
template <typename T> __device__ inline T rounded(float x) {
    asm("" : "+v"(x));
    return (T)x;
}

template <int N> struct Finder {
    static_assert(N % 64 == 0, "every lane reads an entry");
    uint32_t first[(N + 63) / 64];
    __device__ explicit Finder(const uint32_t *table) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < (N + 63) / 64; ++k) first[k] = table[lane + 64 * k];
    }
    __device__ int operator()(uint32_t chunk) const {
        int n = 0;
#pragma unroll
        for (int k = 0; k < (N + 63) / 64; ++k) n += __popcll(__ballot(first[k] <= chunk));
        return n - 1;
    }
};

// t <- t + 1, and what the update takes from it
__device__ inline void advance(float *step, const AdamArgs &a, Rates *rates) {
    const float t = *step + 1.0f;
    *step = t;
    const double lr = a.lr_device ? (double)*a.lr_device : a.lr;
    // 1 - b^t without the cancellation of small t; log(0) = -inf gives 1
    Rates r;
    r.size = (float)(lr / -expm1((double)t * a.log_beta1));
    r.inv_root = (float)(1.0 / sqrt(-expm1((double)t * a.log_beta2)));
    const double decay = a.decoupled ? lr * a.weight_decay : 0.0;
    r.keep = decay < 0.5 ? 1.0f : (float)(1.0 - decay);
    r.decay = decay < 0.5 ? (float)decay : 0.0f;
    *rates = r;
}

template <int N> __global__ void adam_advance_kernel(StepTable<N> s, int n, AdamArgs a, Rates *rates) {
    const int i = threadIdx.x;
    if (i < n) advance(s.step[i], a, rates + i);
}

// ---------------------------------------------------------------------------------- norm
// A running value of a norm: a float64 sum, or the largest magnitude as float bits (they order
// like the magnitudes, and a NaN's lie above infinity's).
template <int KIND> struct Running {
    double sum = 0.0;
    __device__ void add(float x) {
        if (KIND == CISTA_NORM_2) sum = __builtin_fma((double)x, (double)x, sum);
        else sum += (double)__builtin_fabsf(x);
    }
    __device__ void join(const Running &o) { sum += o.sum; }
    __device__ double bits() const { return sum; }
    __device__ static Running of(double b) {
        Running r;
        r.sum = b;
        return r;
    }
    __device__ Running from(int lane) const { return of(__shfl_xor(sum, lane)); }
    __device__ float value() const { return (float)(KIND == CISTA_NORM_2 ? __builtin_sqrt(sum) : sum); }
};
template <> struct Running<CISTA_NORM_MAX> {
    uint32_t most = 0;
    __device__ void add(float x) { most = max(most, __float_as_uint(x) & 0x7fffffffu); }
    __device__ void join(const Running &o) { most = max(most, o.most); }
    __device__ double bits() const { return __longlong_as_double((long long)most); }
    __device__ static Running of(double b) {
        Running r;
        r.most = (uint32_t)__double_as_longlong(b);
        return r;
    }
    __device__ Running from(int lane) const {
        Running r;
        r.most = __shfl_xor(most, lane);
        return r;
    }
    __device__ float value() const { return __uint_as_float(most); }
};

// the block's value, in every thread
template <int KIND> __device__ Running<KIND> block_join(Running<KIND> r) {
    __shared__ double part[THREADS / 64];
#pragma unroll
    for (int l = 32; l; l >>= 1) r.join(r.from(l));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r.bits();
    __syncthreads();
    r = Running<KIND>::of(part[0]);
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) r.join(Running<KIND>::of(part[w]));
    return r;
}

// A chunk of a tensor for norm and scale: NORM_CHUNK bytes from a cache line's begin, which for the
// first one may lie before the tensor's.  base: the chunk's first element; [lo, hi): its elements
// that are the tensor's.  Cut at the tensor's begin instead, a bf16 tensor at an odd 2-byte place is
// read at 5.2 TB/s, one at an odd 16 bytes at 6.7; cut so, at 6.9 wherever it begins (1.2 GB).
template <typename T> struct Chunk {
    static constexpr int V = 16 / sizeof(T), STRIDE = THREADS * V, SIZE = NORM_UNROLL * STRIDE;
    T *base;
    int64_t lo, hi;
    __device__ Chunk(void *data, uint64_t numel, uint32_t chunk) {
        const uintptr_t at = (uintptr_t)data;
        const int64_t begin = (int64_t)(at % LINE / sizeof(T)) - (int64_t)chunk * SIZE;
        base = (T *)data - begin;
        lo = begin;
        hi = begin + (int64_t)numel;
    }
    __device__ bool full() const { return lo <= 0 && hi >= SIZE; }
    // a thread's vector u, and whether all of it is the tensor's
    __device__ int64_t at(int u) const { return threadIdx.x * V + u * STRIDE; }
    __device__ bool inside(int u) const { return at(u) >= lo && at(u) + V <= hi; }
    // the thread's vectors; zeros for those that are not inside.  All loads are under way at once,
    // also at a tensor's ends: a small tensor is nothing else.
    template <bool STREAM> __device__ void read(Pack<T, V> (&x)[NORM_UNROLL]) const {
        if (full()) {
#pragma unroll
            for (int u = 0; u < NORM_UNROLL; ++u) x[u] = load<STREAM, V>(base + at(u));
        } else {
#pragma unroll
            for (int u = 0; u < NORM_UNROLL; ++u) x[u] = inside(u) ? load<STREAM, V>(base + at(u)) : Pack<T, V>{};
        }
    }
    // f(element) for the tensor's elements in the thread's other vectors
    template <typename F> __device__ void ends(F f) const {
        if (full()) return;
        for (int u = 0; u < NORM_UNROLL; ++u)
            if (!inside(u))
                for (int64_t e = at(u) < lo ? lo : at(u); e < at(u) + V && e < hi; ++e) f(*((GLOBAL T *)base + e));
    }
};

template <int KIND, bool STREAM, typename T>
__device__ void norm_chunk(Running<KIND> (&acc)[NORM_UNROLL], const Chunk<T> &c) {
    Pack<T, Chunk<T>::V> x[NORM_UNROLL];
    c.template read<STREAM>(x);
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u)
#pragma unroll
        for (int e = 0; e < c.V; ++e) acc[u].add(to_f32(x[u].e[e]));
    c.ends([&](GLOBAL T &g) { acc[0].add(to_f32(g)); });
}

// Bound by HBM reads (600 M bf16: 186 us, 6.5 TB/s), or for few elements by the latency of a launch and
// its join.  A block steps through the chunks; 2048 blocks take 189 us and leave twice as many values to
// join (clip of 22 M float32 54.8 -> 55.4 us, Adam of 22 M with clipping 118.7 -> 119.5), but behind a copy
// the clip of 150 M bf16 takes 283 us with them instead of 289.
template <int KIND, bool STREAM, int N>
__device__ void norm_partials(const NormTable<N> &t, double *partials, uint32_t blocks) {
    const Finder<N> find(t.first);
    Running<KIND> acc[NORM_UNROLL];
    for (uint32_t c = blockIdx.x; c < t.chunks; c += blocks) {
        const int i = find(c);
        const uint64_t numel = t.info[i] & ((1ull << 56) - 1);
        const uint32_t k = c - t.first[i];
        switch (t.info[i] >> 56) {
        case CISTA_F32: norm_chunk<KIND, STREAM>(acc, Chunk<float>(t.data[i], numel, k)); break;
        case CISTA_BF16: norm_chunk<KIND, STREAM>(acc, Chunk<__bf16>(t.data[i], numel, k)); break;
        default: norm_chunk<KIND, STREAM>(acc, Chunk<_Float16>(t.data[i], numel, k)); break;
        }
    }
#pragma unroll
    for (int u = 1; u < NORM_UNROLL; ++u) acc[0].join(acc[u]);
    const Running<KIND> r = block_join(acc[0]);
    if (threadIdx.x == 0) partials[blockIdx.x] = r.bits();
}

template <int KIND, bool STREAM>
__global__ __launch_bounds__(THREADS) void norm_partials_kernel(NormTable<NORM_TENSORS> t, double *partials) {
    norm_partials<KIND, STREAM>(t, partials, gridDim.x);
}

// The same for the step's gradients, and in one more block the advance of their step counts: the
// update that follows finds the rates ready, without a launch of their own.
template <int KIND, bool STREAM>
__global__ __launch_bounds__(THREADS) void norm_advance_kernel(NormTable<ADAM_TENSORS> t, double *partials,
                                                               StepTable<ADAM_TENSORS> s, int n, AdamArgs a,
                                                               Rates *rates) {
    if (blockIdx.x + 1 == gridDim.x) {
        const int i = threadIdx.x;
        if (i < n) advance(s.step[i], a, rates + i);
        return;
    }
    norm_partials<KIND, STREAM>(t, partials, gridDim.x - 1);
}

template <int KIND> __device__ float norm_of(const double *partials, int n) {
    constexpr int AT_ONCE = 4;               // loads in flight
    Running<KIND> r;
    for (int i = threadIdx.x; i < n; i += AT_ONCE * THREADS) {
        double x[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) x[k] = i + k * THREADS < n ? partials[i + k * THREADS] : 0.0;
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) r.join(Running<KIND>::of(x[k]));
    }
    return block_join(r).value();
}

// the norm that n partial values make, in every thread of every block that asks
__device__ inline float norm_of(int kind, const double *partials, int n) {
    return kind == CISTA_NORM_1   ? norm_of<CISTA_NORM_1>(partials, n)
           : kind == CISTA_NORM_2 ? norm_of<CISTA_NORM_2>(partials, n)
                                  : norm_of<CISTA_NORM_MAX>(partials, n);
}

// Where a kernel takes its norm from: *given, or (given == nullptr) the partial values of the
// launches before it.  Every block then joins them for itself, in the same order and so to the same
// bits, and block 0 writes the norm down.  For few partial values and one consumer that is cheaper
// than a launch that does it once (network of 1.4 M parameters, 358 values: 27.5 -> 21.6 us for the
// step), but 22 M parameters with 1024 values take 118.7 us with the join of its own and 120.1 without
// (clip: 54.8 and 55.8), 200 M bf16 in 5 launches (of up to 2048 values then) 1435 and 1452 us: see
// JOIN_ALL.
struct NormSource {
    const float *given;
    const double *partials;
    float *norm;
    int n, kind;                         // kind 0: no norm
};

__device__ inline float take_norm(const NormSource &s) {
    if (s.given) return *s.given;
    const float v = norm_of(s.kind, s.partials, s.n);
    if (blockIdx.x == 0 && threadIdx.x == 0) *s.norm = v;
    return v;
}

template <int KIND> __global__ __launch_bounds__(THREADS) void norm_join_kernel(const double *partials, int n, float *norm) {
    const float v = norm_of<KIND>(partials, n);
    if (threadIdx.x == 0) *norm = v;
}

// ---------------------------------------------------------------------------------- scale
__device__ inline float clip_scale(float norm, double max_norm) {
    if (max_norm == __builtin_inf()) return 1.0f;
    const double c = max_norm / ((double)norm + 1e-6);
    return c >= 1.0 ? 1.0f : (float)c;       // a NaN stays one
}

template <typename T> __device__ void scale_chunk(const Chunk<T> &k, float c) {
    Pack<T, Chunk<T>::V> x[NORM_UNROLL];
    k.template read<false>(x);
#pragma unroll
    for (int u = 0; u < NORM_UNROLL; ++u) {
#pragma unroll
        for (int e = 0; e < k.V; ++e) x[u].e[e] = rounded<T>(to_f32(x[u].e[e]) * c);
        if (k.full() || k.inside(u)) store<false>(k.base + k.at(u), x[u]);
    }
    k.ends([&](GLOBAL T &g) { g = rounded<T>(to_f32(g) * c); });
}

// One block per chunk, each rounding once to the gradient's type, of a float32 product.  The chunks
// run backwards: the norm has read them forwards, so what the last-level cache still holds of them
// is met before it is evicted (300 MB of bf16, norm and scale: 170 -> 165 us).  They do so by eights,
// so that a chunk stays on the XCD (block mod 8) whose L2 the norm has brought it to.
__global__ __launch_bounds__(THREADS) void scale_kernel(NormTable<NORM_TENSORS> t, double max_norm, NormSource norm) {
    const float c = clip_scale(take_norm(norm), max_norm);
    if (c == 1.0f) return;                   // x * 1 is x for every x: nothing to read or write
    const Finder<NORM_TENSORS> find(t.first);
    const uint32_t b = blockIdx.x, eights = t.chunks & ~7u;
    const uint32_t k = b < eights ? eights - 8 - (b & ~7u) + (b & 7) : b;
    const int i = find(k);
    const uint64_t numel = t.info[i] & ((1ull << 56) - 1);
    const uint32_t q = k - t.first[i];
    switch (t.info[i] >> 56) {
    case CISTA_F32: scale_chunk(Chunk<float>(t.data[i], numel, q), c); break;
    case CISTA_BF16: scale_chunk(Chunk<__bf16>(t.data[i], numel, q), c); break;
    default: scale_chunk(Chunk<_Float16>(t.data[i], numel, q), c); break;
    }
}

// ---------------------------------------------------------------------------------- Adam
// b1 m + (1 - b1) g.  Near 1 as m + (1 - b1)(g - m), since float32 holds 1 - b1 to 2^-24 of itself, b1
// only to 2^-24 of 1; below 1/2 the roundings of m in g - m would count in full where m itself counts
// with b1 (b1 = 0, m = 1, g = 1e-9: 0 instead of g).  One branch for the whole launch.
__device__ inline float moment1(float m, float g, const AdamArgs &a) {
    return a.rate1 > 0.5f ? fmaf(a.beta1, m, a.rate1 * g) : fmaf(a.rate1, g - m, m);
}

// b2 v + (1 - b2) g^2, with b2 v as v - (1 - b2) v: b2 itself, rounded, would move the average of a long
// run by 2^-24 / (1 - b2).  Below 1/2 it is the other way round (b2 = 1e-9: 1 - b2 is 1, and nothing
// of v would be left).  An average that has overflowed stays infinite, whatever b2 is.
__device__ inline float moment2(float v, float g, const AdamArgs &a) {
    const float kept = a.rate2 > 0.5f ? a.beta2 * v : fmaf(-a.rate2, v, v);
    return fmaf(a.rate2 * g, g, v < __builtin_inff() ? kept : v);
}

__device__ inline void adam_element(float &p, float g, float &m, float &v, const AdamArgs &a, const Rates &r, float c) {
    g *= c;
    g = a.maximize ? -g : g;
    if (a.decay != 0.0f) g = fmaf(a.decay, p, g);
    m = moment1(m, g, a);
    v = moment2(v, g, a);
    const float q = m / fmaf(sqrtf(v), r.inv_root, a.eps);
    // decay and update leave the weight in one subtraction: a decay of less than half a step of float32
    // would not move it by itself, and one rounded to whole steps would be off at every step alike.  An
    // infinite weight, from which its own decay cannot be subtracted, goes the other way and stays.
    const bool together = r.decay != 0.0f && fabsf(p) < __builtin_inff();
    p = together ? p - fmaf(r.decay, p, r.size * q) : fmaf(-r.size, q, p * r.keep);
}

// Elements [chunk * ADAM_CHUNK - shift, + ADAM_CHUNK) of a tensor, 4 to a thread.  The shift puts the
// float32 accesses on whole cache lines where the tensor itself begins within one, and the 16-bit
// ones too if they begin at the same element of a line (AdamW with clipping of 268 M float32 in 147
// tensors end to end 1515 -> 1428 us, of 200 M bf16 in 301 tensors 1115 -> 1005 us).
__host__ __device__ inline int64_t adam_shift(const float *m) { return (uintptr_t)m / 4 % (LINE / 2); }

template <bool STREAM, typename T>
__device__ void adam_chunk(T *p, const T *g, float *m, float *v, float *w, int64_t numel, uint32_t chunk,
                           const AdamArgs &a, const Rates &r, float c) {
    constexpr int V = 4;
    const int64_t i = (int64_t)chunk * ADAM_CHUNK - adam_shift(m) + threadIdx.x * V;
    if (i >= 0 && i + V <= numel) {
        const Pack<T, V> gx = load<STREAM, V>(g + i);
        Pack<float, V> wx = load<STREAM, V>(w + i), mx = load<STREAM, V>(m + i), vx = load<STREAM, V>(v + i);
#pragma unroll
        for (int e = 0; e < V; ++e) adam_element(wx.e[e], to_f32(gx.e[e]), mx.e[e], vx.e[e], a, r, c);
        store<STREAM>(m + i, mx);
        store<STREAM>(v + i, vx);
        store<STREAM>(w + i, wx);
        if (sizeof(T) != 4) {
            Pack<T, V> px;
#pragma unroll
            for (int e = 0; e < V; ++e) px.e[e] = rounded<T>(wx.e[e]);
            store<STREAM>(p + i, px);
        }
    } else {
        for (int64_t e = i < 0 ? 0 : i; e < i + V && e < numel; ++e) {
            adam_element(w[e], to_f32(g[e]), m[e], v[e], a, r, c);
            if (sizeof(T) != 4) p[e] = rounded<T>(w[e]);
        }
    }
}

// Seven streams over HBM, 28 bytes and some 40 operations an element: bound by HBM (268 M float32:
// 1201 us, 6.25 TB/s, where a 4 GiB copy reaches 4.9), or by launches where it is small.  One block
// per chunk, dispatched in the order of the addresses: 2048 blocks that step through the chunks drift
// apart and lose the DRAM's pages (1632 us against 1404, before the lines and STREAM).  Where all of it
// fits the last-level cache STREAM costs (1.4 M parameters: 8.5 -> 9.5 us; 268 M: 1404 -> 1358), so
// it goes by the bytes, and so does FIVE: with 5 blocks on a CU instead of 8 the blocks stay closer
// together (the step of 268 M with clipping 1422 -> 1363 us, 3 blocks 1379; of 200 M bf16 998 -> 981 and 1004;
// of 22 M 120.8 -> 118.5 and 121.2; 1.4 M parameters: update 9.0 -> 9.3).  The blocks of an
// XCD (block mod 8) take the chunks whose gradients its L2 has from the norm: 4 of them to a chunk of
// the norm's.
template <bool STREAM>
__global__ __launch_bounds__(THREADS) void adam_kernel(AdamTable t, AdamArgs a, const Rates *rates, NormSource norm) {
    const Finder<ADAM_TENSORS> find(t.first);
    const float c = norm.kind ? clip_scale(take_norm(norm), a.max_norm) : 1.0f;
    const uint32_t b = blockIdx.x, c32 = b < (t.chunks & ~31u) ? (b & ~31u) + (b & 7) * 4 + (b >> 3 & 3) : b;
    const int i = find(c32);
    const uint32_t k = c32 - t.first[i];
    const int64_t numel = (int64_t)(t.info[i] & ((1ull << 56) - 1));
    const Rates r = rates[i];
    void *p = t.param[i];
    const void *g = t.grad[i];
    float *m = t.exp_avg[i], *v = t.exp_avg_sq[i], *w = t.master[i];
    switch (t.info[i] >> 56) {
    case CISTA_F32: adam_chunk<STREAM>((float *)p, (const float *)g, m, v, (float *)p, numel, k, a, r, c); break;
    case CISTA_BF16: adam_chunk<STREAM>((__bf16 *)p, (const __bf16 *)g, m, v, w, numel, k, a, r, c); break;
    default: adam_chunk<STREAM>((_Float16 *)p, (const _Float16 *)g, m, v, w, numel, k, a, r, c); break;
    }
}

// ---------------------------------------------------------------------------------- host
inline int size_of(long long type) { return type == CISTA_F32 ? 4 : 2; }
inline int hip_ok() { return hipGetLastError() == hipSuccess ? CISTA_OK : CISTA_ERR_HIP; }
inline int launches(int n, int per) { return n <= 0 ? 1 : (n + per - 1) / per; }

// A launch has less than 2^32 threads, so a kernel with a block for each chunk takes less than 2^24
// chunks (the last partly filled ones of a table are within the 2^10 that the limits leave); the
// norm's blocks step through theirs, of which 2^31 can be counted.
constexpr long long MOST_NORM = 1ll << 40, MOST_SCALE = ((1ll << 24) - (1 << 10)) * NORM_CHUNK / 4,
                    MOST_ADAM = ((1ll << 24) - (1 << 10)) * ADAM_CHUNK;       // elements of one call

bool bad_tensor(const void *data, long long numel, long long type) {
    if (numel < 0 || type < CISTA_F32 || type > CISTA_F16) return true;
    return numel > 0 && (!data || (uintptr_t)data % size_of(type));
}

// how a float is aligned, and what the partial values and rates need
bool misplaced(const float *x) { return (uintptr_t)x % sizeof(float); }
bool misplaced(const void *workspace) { return (uintptr_t)workspace % 16; }

struct Range {
    uintptr_t begin, end;
};

// Do the n ranges of get(i) overlap?  Tensors that lie in their list's order, as views of one
// buffer do, need no sorting.
template <typename Get> int overlap(int n, Get get) {
    uintptr_t end = 0;
    int i = 0;
    for (; i < n; ++i) {
        const Range r = get(i);
        if (r.begin == r.end) continue;
        if (r.begin < end) break;
        end = r.end;
    }
    if (i == n) return CISTA_OK;
    try {
        std::vector<Range> all;
        all.reserve(n);
        for (i = 0; i < n; ++i)
            if (get(i).begin != get(i).end) all.push_back(get(i));
        std::sort(all.begin(), all.end(), [](const Range &x, const Range &y) { return x.begin < y.begin; });
        for (size_t k = 1; k < all.size(); ++k)
            if (all[k].begin < all[k - 1].end) return CISTA_ERR_ALIAS;
    } catch (...) {
        return CISTA_ERR_HIP;
    }
    return CISTA_OK;
}

Range range_of(const void *data, long long numel, long long type) {
    return {(uintptr_t)data, (uintptr_t)data + (uintptr_t)numel * size_of(type)};
}

// is the float x within the tensor?  A norm is read, or written, by some workgroups while others write theirs
bool holds(const float *x, const void *data, long long numel, long long type) {
    const Range r = range_of(data, numel, type);
    return numel && (uintptr_t)x < r.end && (uintptr_t)x + sizeof(float) > r.begin;
}

bool holds(const float *x, const cista_tensor *t, int n) {
    for (int i = 0; i < n; ++i)
        if (holds(x, t[i].data, t[i].numel, t[i].type)) return true;
    return false;
}

bool holds(const float *x, const cista_adam_tensor &t) {
    return holds(x, t.param, t.numel, t.type) || holds(x, t.grad, t.numel, t.type) ||
           holds(x, t.exp_avg, t.numel, CISTA_F32) || holds(x, t.exp_avg_sq, t.numel, CISTA_F32) ||
           (t.type != CISTA_F32 && holds(x, t.master, t.numel, CISTA_F32)) || holds(x, t.step, 1, CISTA_F32);
}

int check(const cista_tensor *t, int n, bool written) {
    if (n < 0 || (n && !t)) return CISTA_ERR_INVALID;
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        if (bad_tensor(t[i].data, t[i].numel, t[i].type)) return CISTA_ERR_INVALID;
        const long long most = written ? MOST_SCALE : MOST_NORM;
        if (t[i].numel > most || (total += t[i].numel) > most) return CISTA_ERR_UNSUPPORTED;
    }
    if (!written) return CISTA_OK;
    return overlap(n, [&](int i) { return range_of(t[i].data, t[i].numel, t[i].type); });
}

static_assert(sizeof(NormTable<NORM_TENSORS>) + sizeof(NormSource) + 16 <= 4096, "kernel arguments");
static_assert(sizeof(AdamTable) + sizeof(AdamArgs) + sizeof(NormSource) + 16 <= 4096, "kernel arguments");
static_assert(sizeof(NormTable<ADAM_TENSORS>) + sizeof(StepTable<ADAM_TENSORS>) + sizeof(AdamArgs) + 32 <= 4096,
              "kernel arguments");
static_assert(sizeof(StepTable<STEP_TENSORS>) + sizeof(AdamArgs) + 16 <= 4096, "kernel arguments");

// The next table of at most N of the n tensors get(i), from i on; i becomes the first one left.
template <int N, typename Get> NormTable<N> table_of(int &i, int n, Get get) {
    NormTable<N> t;
    int k = 0;
    uint64_t chunks = 0;
    for (; i < n && k < N; ++i) {
        const cista_tensor x = get(i);
        if (!x.numel) continue;
        t.data[k] = x.data;
        t.info[k] = (uint64_t)x.numel | (uint64_t)x.type << 56;
        t.first[k++] = (uint32_t)chunks;
        chunks += ((uint64_t)x.numel * size_of(x.type) + (uintptr_t)x.data % LINE + NORM_CHUNK - 1) / NORM_CHUNK;
    }
    for (; k < N; ++k) t.data[k] = nullptr, t.info[k] = 0, t.first[k] = ~0u;
    t.chunks = (uint32_t)chunks;
    t.pad = 0;
    return t;
}

int blocks_of(uint32_t chunks, int most) { return (int)std::min<uint32_t>(chunks, most); }

// f(kind as a constant)
template <typename F> int with_kind(int kind, F f) {
    switch (kind) {
    case CISTA_NORM_1: f(std::integral_constant<int, CISTA_NORM_1>()); return CISTA_OK;
    case CISTA_NORM_2: f(std::integral_constant<int, CISTA_NORM_2>()); return CISTA_OK;
    case CISTA_NORM_MAX: f(std::integral_constant<int, CISTA_NORM_MAX>()); return CISTA_OK;
    }
    return CISTA_ERR_INVALID;
}

// launches the partial values of all tensors; returns where a norm comes from
template <typename Get>
NormSource partials_of(int kind, bool stream, int n, Get get, float *norm, double *partials, hipStream_t s) {
    int used = 0;
    for (int i = 0; i < n;) {
        const auto t = table_of<NORM_TENSORS>(i, n, get);
        const int blocks = blocks_of(t.chunks, NORM_BLOCKS);
        if (!blocks) continue;
        with_kind(kind, [&](auto k) {
            const auto f = stream ? norm_partials_kernel<k.value, true> : norm_partials_kernel<k.value, false>;
            f<<<blocks, THREADS, 0, s>>>(t, partials + used);
        });
        used += blocks;
    }
    return {nullptr, partials, norm, used, kind};
}

NormSource join(const NormSource &q, hipStream_t s) {
    with_kind(q.kind, [&](auto k) { norm_join_kernel<k.value><<<1, THREADS, 0, s>>>(q.partials, q.n, q.norm); });
    return {q.norm, nullptr, nullptr, 0, q.kind};
}

int scale(const cista_tensor *grads, int n, double max_norm, NormSource norm, hipStream_t s) {
    for (int last = (launches(n, NORM_TENSORS) - 1) * NORM_TENSORS; last >= 0; last -= NORM_TENSORS) {
        int i = last;
        const auto t = table_of<NORM_TENSORS>(i, std::min(n, last + NORM_TENSORS), [&](int j) { return grads[j]; });
        if (t.chunks) scale_kernel<<<t.chunks, THREADS, 0, s>>>(t, max_norm, norm);
    }
    return hip_ok();
}

AdamArgs args_of(const cista_adam_group &q, double max_norm) {
    AdamArgs a;
    a.lr = q.lr;
    a.log_beta1 = std::log(q.beta1);
    a.log_beta2 = std::log(q.beta2);
    a.weight_decay = q.weight_decay;
    a.max_norm = max_norm;
    a.lr_device = q.lr_device;
    a.rate1 = (float)(1.0 - q.beta1);
    a.rate2 = (float)(1.0 - q.beta2);
    a.beta1 = (float)q.beta1;
    a.beta2 = (float)q.beta2;
    a.eps = (float)q.eps;
    a.decay = q.decoupled ? 0.0f : (float)q.weight_decay;
    a.decoupled = q.decoupled;
    a.maximize = q.maximize;
    return a;
}

// Launches with N step counts each.  A launch costs the host 2.7 us with 64 bytes of arguments, 3.2 us
// with 512 and 3.9 us from 1 KB to 4 KB, so few steps get a table of their own.
template <int N> void advance_all(const cista_adam_tensor *x, int n, const AdamArgs &a, Rates *rates, hipStream_t s) {
    for (int i = 0; i < n; i += N) {
        StepTable<N> steps = {};
        const int now = std::min(N, n - i);
        for (int j = 0; j < now; ++j) steps.step[j] = x[i + j].step;
        adam_advance_kernel<N><<<1, (now + 63) / 64 * 64, 0, s>>>(steps, now, a, rates + i);
    }
}

size_t partial_bytes(int n) { return (size_t)launches(n, NORM_TENSORS) * NORM_BLOCKS * sizeof(double); }

}  // namespace cista_optim

using namespace cista_optim;

extern "C" {

size_t cista_optim_workspace_bytes(int n) {
    return n < 0 ? 0 : partial_bytes(n) + (size_t)std::max(n, 1) * sizeof(Rates);
}

int cista_grad_norm(const cista_tensor *grads, int n, int norm_kind, float *norm, void *workspace,
                    size_t workspace_bytes, void *stream) {
    const int st = check(grads, n, false);
    if (st != CISTA_OK) return st;
    if (!norm || !workspace || norm_kind < CISTA_NORM_1 || norm_kind > CISTA_NORM_MAX || misplaced(norm) ||
        misplaced(workspace))
        return CISTA_ERR_INVALID;
    if (workspace_bytes < cista_optim_workspace_bytes(n)) return CISTA_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    // past the cache's size nobody finds the gradients there anyway (1.2 GB of bf16: 212 -> 199 us)
    long long bytes = 0;
    for (int i = 0; i < n; ++i) bytes += grads[i].numel * size_of(grads[i].type);
    join(partials_of(norm_kind, bytes > CACHE, n, [&](int i) { return grads[i]; }, norm, (double *)workspace, s), s);
    return hip_ok();
}

int cista_scale_grads(const cista_tensor *grads, int n, double max_norm, const float *norm, void *stream) {
    const int st = check(grads, n, true);
    if (st != CISTA_OK) return st;
    if (!norm || misplaced(norm) || !(max_norm >= 0.0)) return CISTA_ERR_INVALID;
    if (holds(norm, grads, n)) return CISTA_ERR_ALIAS;
    return scale(grads, n, max_norm, {norm, nullptr, nullptr, 0, 0}, (hipStream_t)stream);
}

int cista_clip_grads(const cista_tensor *grads, int n, int norm_kind, double max_norm, float *norm, void *workspace,
                     size_t workspace_bytes, void *stream) {
    const int st = check(grads, n, true);
    if (st != CISTA_OK) return st;
    if (!norm || !workspace || norm_kind < CISTA_NORM_1 || norm_kind > CISTA_NORM_MAX || !(max_norm >= 0.0) ||
        misplaced(norm) || misplaced(workspace))
        return CISTA_ERR_INVALID;
    if (workspace_bytes < cista_optim_workspace_bytes(n)) return CISTA_ERR_WORKSPACE;
    if (holds(norm, grads, n)) return CISTA_ERR_ALIAS;
    hipStream_t s = (hipStream_t)stream;
    NormSource q = partials_of(norm_kind, false, n, [&](int i) { return grads[i]; }, norm, (double *)workspace, s);
    // without partial values (nothing but empty tensors) no other launch would write the norm
    if (!q.n || q.n > JOIN_ALL || n > NORM_TENSORS) q = join(q, s);
    return scale(grads, n, max_norm, q, s);
}

int cista_adam_step(const cista_adam_tensor *table, const cista_adam_group *groups, int n_groups, int norm_kind,
                    double max_norm, float *norm, void *workspace, size_t workspace_bytes, void *stream) {
    if (n_groups < 0 || (n_groups && !groups) || norm_kind < 0 || norm_kind > CISTA_NORM_MAX) return CISTA_ERR_INVALID;
    if (norm_kind && (!norm || misplaced(norm) || !(max_norm >= 0.0))) return CISTA_ERR_INVALID;
    int n = 0;
    for (int k = 0; k < n_groups; ++k) {
        const cista_adam_group &q = groups[k];
        if (q.n < 0 || !(q.beta1 >= 0.0 && q.beta1 < 1.0 && q.beta2 >= 0.0 && q.beta2 < 1.0) ||
            misplaced(q.lr_device))
            return CISTA_ERR_INVALID;
        n += q.n;
    }
    if (n && !table) return CISTA_ERR_INVALID;
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        const cista_adam_tensor &x = table[i];
        if (bad_tensor(x.param, x.numel, x.type) || bad_tensor(x.grad, x.numel, x.type) || !x.step || misplaced(x.step) ||
            bad_tensor(x.exp_avg, x.numel, CISTA_F32) || bad_tensor(x.exp_avg_sq, x.numel, CISTA_F32) ||
            (x.type != CISTA_F32 && bad_tensor(x.master, x.numel, CISTA_F32)))
            return CISTA_ERR_INVALID;
        if (x.numel > MOST_ADAM || (total += x.numel) > MOST_ADAM) return CISTA_ERR_UNSUPPORTED;
        if (norm_kind && holds(norm, x)) return CISTA_ERR_ALIAS;
    }
    int apart = overlap(n, [&](int i) { return range_of(table[i].param, table[i].numel, table[i].type); });
    for (auto which : {&cista_adam_tensor::exp_avg, &cista_adam_tensor::exp_avg_sq, &cista_adam_tensor::master,
                       &cista_adam_tensor::step}) {
        if (apart != CISTA_OK) return apart;
        apart = overlap(n, [&](int i) {
            const cista_adam_tensor &x = table[i];
            const bool none = which == &cista_adam_tensor::master && x.type == CISTA_F32;
            return range_of(x.*which, which == &cista_adam_tensor::step ? 1 : none ? 0 : x.numel, CISTA_F32);
        });
    }
    if (apart != CISTA_OK) return apart;
    if (!workspace || misplaced(workspace)) return CISTA_ERR_INVALID;
    if (workspace_bytes < cista_optim_workspace_bytes(n)) return CISTA_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    Rates *rates = (Rates *)((char *)workspace + partial_bytes(n));
    double *partials = (double *)workspace;
    const auto grad = [&](int i) { return cista_tensor{(void *)table[i].grad, table[i].numel, table[i].type}; };
    const bool stream_all = total * 28 > CACHE;
    const bool fused = norm_kind && n_groups == 1 && n <= ADAM_TENSORS;
    NormSource q = {nullptr, nullptr, nullptr, 0, 0};
    if (fused) {
        const AdamArgs a = args_of(groups[0], max_norm);
        int i = 0;
        const auto t = table_of<ADAM_TENSORS>(i, n, grad);
        StepTable<ADAM_TENSORS> steps = {};
        for (int j = 0; j < n; ++j) steps.step[j] = table[j].step;
        const int blocks = blocks_of(t.chunks, NORM_BLOCKS);
        with_kind(norm_kind, [&](auto k) {
            const auto f = stream_all ? norm_advance_kernel<k.value, true> : norm_advance_kernel<k.value, false>;
            f<<<blocks + 1, THREADS, 0, s>>>(t, partials, steps, n, a, rates);
        });
        q = {nullptr, partials, norm, blocks, norm_kind};
    } else if (norm_kind) {
        q = partials_of(norm_kind, stream_all, n, grad, norm, partials, s);
    }
    if (norm_kind && (!q.n || q.n > JOIN_ALL || !fused)) q = join(q, s);
    const cista_adam_tensor *x = table;
    for (int k = 0; k < n_groups; ++k) {
        const AdamArgs a = args_of(groups[k], max_norm);
        if (!fused && groups[k].n <= ADAM_TENSORS) {
            advance_all<ADAM_TENSORS>(x, groups[k].n, a, rates, s);
        } else if (!fused) {
            advance_all<STEP_TENSORS>(x, groups[k].n, a, rates, s);
        }
        for (int i = 0; i < groups[k].n; i += ADAM_TENSORS) {
            AdamTable t = {};
            const int now = std::min(ADAM_TENSORS, groups[k].n - i);
            uint64_t chunks = 0;
            for (int j = 0; j < ADAM_TENSORS; ++j) t.first[j] = ~0u;
            for (int j = 0; j < now; ++j, ++x) {
                t.param[j] = x->param, t.grad[j] = x->grad, t.master[j] = x->master;
                t.exp_avg[j] = x->exp_avg, t.exp_avg_sq[j] = x->exp_avg_sq;
                t.info[j] = (uint64_t)x->numel | (uint64_t)x->type << 56;
                t.first[j] = (uint32_t)chunks;
                if (x->numel) chunks += ((uint64_t)x->numel + adam_shift(x->exp_avg) + ADAM_CHUNK - 1) / ADAM_CHUNK;
            }
            t.chunks = (uint32_t)chunks;
            const auto f = stream_all ? adam_kernel<true> : adam_kernel<false>;
            if (chunks) f<<<t.chunks, THREADS, stream_all ? FIVE : 0, s>>>(t, a, rates, q);
            rates += now;
        }
    }
    return hip_ok();
}

}  // extern "C"
