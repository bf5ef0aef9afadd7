// K9: the optimiser over lists of tensors - gradient norm with clip coefficient and verdict, AdamW with moments in 32 or 8 bits.
//
// Mathematics (all in f32 unless said otherwise; every product and sum rounded by itself, this file is compiled without contraction):
//   norm    N = |grad_scale| sqrt(sum g^2), squares and sums in f64 (a square of an f32 is exact there: no overflow, no order to care
//           about); coef = min(1, max_norm / (N + 1e-6)); N inf or NaN, or the range guard's verdict: the step is skipped
//   AdamW   h = g * grad_scale * coef;  m += (h - m)(1 - b1);  v = v b2 + h^2 (1 - b2);
//           p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//   8 bits  blocks of 128 consecutive elements of a tensor: x = q s, q in e4m3, s = 2^(max(E, -100) - 7), E = floor(log2 max |x|): a
//           power of two scales without rounding and leaves the grid where it is while the block's largest value stays in its binade -
//           an unchanged x keeps its code.  The state of v is its root u = sqrt(v): the 2^17 that a block spans are 2^34 in v.
//           Rounding is stochastic, q = step floor(|x| / (s step) + r): at b2 = 0.999 v moves by 0.1 % a step and an e4m3 step is
//           6-12 %, rounding to nearest would keep a stored v where it is for good.  u > 0 never becomes 0 (at least 2^-9 s): the
//           next update must not be divided by eps alone.  r = 16 bits of Philox(seed; group of four elements, t): the same on every
//           rank of a data-parallel run.
// Both are streams (28 and 16.1 bytes an element in f32): HBM bound where the list is long, launch and latency bound where it is short.
#include "common.h"
#include <math.h>
#include <string.h>

namespace {

constexpr int THREADS = 256;
constexpr int BLOCK = BENERF_ADAMW_BLOCK;
constexpr uint32_t PLAN_MAGIC = 0x41445731u;
static_assert(BLOCK == 128, "a block is half a wavefront of four elements a lane");

// The plan: what a launch needs to find its way through the list, filled on the host, uploaded once.
struct Entry {
    void* param;
    void* m;
    void* v;
    float* ms;
    float* vs;
    float* master;
    int64_t n;
    int64_t first_block;      // number of the tensor's first block of 128 in the list: the generator's counter
    int64_t first_chunk;
};
struct PlanHead {
    uint32_t magic;
    int32_t n_tensors;
    int32_t param_type, state_bits, has_master;
    int32_t unroll;           // a chunk is THREADS * 4 * unroll elements: one workgroup
    int64_t n_chunks;
    int64_t map_at;           // byte offset of int32 map[n_chunks]: the tensor of every chunk
    int64_t bytes;
};
constexpr size_t HEAD_BYTES = 64;
static_assert(sizeof(PlanHead) <= HEAD_BYTES, "plan header");

__host__ __device__ inline const Entry* plan_entries(const void* plan) { return reinterpret_cast<const Entry*>(static_cast<const char*>(plan) + HEAD_BYTES); }

// Gradients change from step to step while the rest of the list stays: their addresses travel in the launch itself, so that a captured
// launch keeps its own and nothing on the device has to be rewritten.  4 KiB is what a launch may carry.
constexpr int PTRS_SMALL = 64, PTRS_LARGE = 480;
template <int N>
struct Ptrs {
    const void* p[N];
};

struct Hyper {
    float gs, decay, step_size, omb1, b2, omb2, eps, inv_bc2;
};
struct AdamwArgs {
    const Entry* entries;
    const int32_t* map;
    int64_t chunk0;            // first chunk of this launch
    int32_t tensor0;           // first tensor of this launch
    int32_t unroll;
    Hyper h;                   // for t = step, lr from the host
    const float* norm;         // [4] of the norm operator, or null
    const uint32_t* status;    // range guard words, or null
    const float* step_dev;     // or null: t = step - skipped
    const float* lr_dev;       // or null
    double lr, beta1, beta2, decay_rate;
    int64_t step;
    uint64_t seed;
};

__device__ __forceinline__ bool guard_says_skip(const uint32_t* st) {
    return st && (st[BENERF_ST_SKIP] != 0u || st[BENERF_ST_ACT] >= 0x477fe000u || st[BENERF_ST_GRAD] >= 0x477fe000u);
}

__host__ __device__ inline double int_power(double b, int64_t t) {
    double r = 1.0;
    for (; t > 0; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// Scalars of this step; false: skipped.  What the host could not know (a counter or a learning rate on the device, steps skipped so
// far) is worked out again here, in f64: 40 multiplications for t < 2^20, once per wave, uniform.
__device__ __forceinline__ bool step_scalars(const AdamwArgs& a, Hyper& h, int64_t& t) {
    if (guard_says_skip(a.status)) return false;
    h = a.h;
    t = a.step;
    float skipped = 0.f;
    if (a.norm) {
        if (a.norm[2] != 0.f) return false;
        h.gs = h.gs * a.norm[1];
        skipped = a.norm[3];
    }
    const uint32_t gated = a.status ? a.status[BENERF_ST_SKIPPED_TOTAL] : 0u;
    if (a.step_dev || a.lr_dev || skipped != 0.f || gated != 0u) {
        t = a.step_dev ? (int64_t)a.step_dev[0] : a.step - (int64_t)skipped - (int64_t)gated;
        if (t < 1) t = 1;
        const double lr = a.lr_dev ? (double)a.lr_dev[0] : a.lr;
        h.decay = (float)(1.0 - lr * a.decay_rate);
        h.step_size = (float)(lr / (1.0 - int_power(a.beta1, t)));
        h.inv_bc2 = (float)(1.0 / sqrt(1.0 - int_power(a.beta2, t)));
    }
    return true;
}

// ---- four consecutive elements, at any element-aligned address -------------------------------------------------------------
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short ushort4v __attribute__((ext_vector_type(4)));
typedef unsigned short ushort4u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32u __attribute__((aligned(1)));

struct F32 {
    typedef float4v raw;
    static constexpr bool NARROW = false;
    __device__ static raw load(const void* p, int64_t i) { return *reinterpret_cast<const float4u*>(static_cast<const float*>(p) + i); }
    __device__ static raw load_part(const void* p, int64_t i, int k) {
        raw r = 0.f;
        for (int j = 0; j < 4; ++j)
            if (j < k) r[j] = static_cast<const float*>(p)[i + j];
        return r;
    }
    __device__ static float4v widen(raw r) { return r; }
    __device__ static raw narrow(float4v x) { return x; }
    __device__ static void store(void* p, int64_t i, raw r) { *reinterpret_cast<float4u*>(static_cast<float*>(p) + i) = r; }
    __device__ static void store_part(void* p, int64_t i, int k, raw r) {
        for (int j = 0; j < 4; ++j)
            if (j < k) static_cast<float*>(p)[i + j] = r[j];
    }
};
template <typename V>
struct Half16 {       // bf16 and f16: rounded to nearest even, once
    typedef ushort4v raw;
    static constexpr bool NARROW = true;
    __device__ static raw load(const void* p, int64_t i) { return *reinterpret_cast<const ushort4u*>(static_cast<const unsigned short*>(p) + i); }
    __device__ static raw load_part(const void* p, int64_t i, int k) {
        raw r = 0;
        for (int j = 0; j < 4; ++j)
            if (j < k) r[j] = static_cast<const unsigned short*>(p)[i + j];
        return r;
    }
    __device__ static float4v widen(raw r) { return __builtin_convertvector(__builtin_bit_cast(V, r), float4v); }
    __device__ static raw narrow(float4v x) { return __builtin_bit_cast(raw, __builtin_convertvector(x, V)); }
    __device__ static void store(void* p, int64_t i, raw r) { *reinterpret_cast<ushort4u*>(static_cast<unsigned short*>(p) + i) = r; }
    __device__ static void store_part(void* p, int64_t i, int k, raw r) {
        for (int j = 0; j < 4; ++j)
            if (j < k) static_cast<unsigned short*>(p)[i + j] = r[j];
    }
};
typedef Half16<bf4v> BF16;
typedef Half16<half4v> F16;

// the update of four elements; v: v itself (32 bits) or, rooted, computed from u by the caller.  Returns the root of the new v.
__device__ __forceinline__ void update(float4v& p, float4v g, float4v& m, float4v& v, float4v& root, const Hyper& h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = g[j] * h.gs;
        m[j] = m[j] + (x - m[j]) * h.omb1;
        v[j] = v[j] * h.b2 + (x * x) * h.omb2;
        root[j] = sqrtf(v[j]);
        p[j] = p[j] * h.decay - h.step_size * (m[j] / (root[j] * h.inv_bc2 + h.eps));
    }
}

template <class PT, class GT, bool MASTER>
__device__ __forceinline__ void four32(const Entry& e, const void* gp, int64_t i, int k, const Hyper& h) {
    const bool full = k >= 4;
    float4v p = MASTER ? (full ? F32::load(e.master, i) : F32::load_part(e.master, i, k))
                       : PT::widen(full ? PT::load(e.param, i) : PT::load_part(e.param, i, k));
    const float4v g = GT::widen(full ? GT::load(gp, i) : GT::load_part(gp, i, k));
    float4v m = full ? F32::load(e.m, i) : F32::load_part(e.m, i, k);
    float4v v = full ? F32::load(e.v, i) : F32::load_part(e.v, i, k);
    float4v root;
    update(p, g, m, v, root, h);
    if (full) {
        if (MASTER) F32::store(e.master, i, p);
        PT::store(e.param, i, PT::narrow(p));
        F32::store(e.m, i, m);
        F32::store(e.v, i, v);
    } else {
        if (MASTER) F32::store_part(e.master, i, k, p);
        PT::store_part(e.param, i, k, PT::narrow(p));
        F32::store_part(e.m, i, k, m);
        F32::store_part(e.v, i, k, v);
    }
}

// ---- 8-bit moments ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float4v decode4(uint32_t w, float s) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return float4v{a[0] * s, a[1] * s, b[0] * s, b[1] * s};
}
// high 16 bits of |x|, 0 for inf and NaN: they must not take the block's other values along
__device__ __forceinline__ uint32_t top16(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// maximum of both 16-bit halves over the 32 lanes of a block
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    for (int d = 1; d < 32; d <<= 1) x = pk_max(x, (uint32_t)__shfl_xor((int)x, d, 32));
    return x;
}
// x scaled by inv, rounded to the e4m3 grid with the draw h16; keep: a value that is not 0 stays so
__device__ __forceinline__ float to_grid(float x, float inv, uint32_t h16, bool keep) {
    const float y = fabsf(x) * inv;
    const uint32_t b = __float_as_uint(y);
    if (!(b < 0x7f800000u)) return __uint_as_float(0x7fc00000u);
    float q;
    if (b >= 0x3c800000u) {               // from 2^-6 on: three bits behind the leading one
        q = __uint_as_float((b + (h16 << 4)) & 0xfff00000u);
    } else {                              // below: steps of 2^-9
        float k = floorf(y * 512.f + (float)h16 * (1.f / 65536.f));
        if (keep && y > 0.f) k = fmaxf(k, 1.f);
        q = k * (1.f / 512.f);
    }
    return copysignf(q, x);
}
__device__ __forceinline__ uint32_t encode4(float4v x, float inv, const uint32_t (&h16)[4], bool keep) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(to_grid(x[0], inv, h16[0], keep), to_grid(x[1], inv, h16[1], keep), w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(to_grid(x[2], inv, h16[2], keep), to_grid(x[3], inv, h16[3], keep), w, true);
    return (uint32_t)w;
}
__device__ __forceinline__ uint32_t load_codes(const void* p, int64_t i, int k) {
    if (k >= 4) return *reinterpret_cast<const u32u*>(static_cast<const uint8_t*>(p) + i);
    uint32_t w = 0;
    for (int j = 0; j < 3; ++j)
        if (j < k) w |= (uint32_t) static_cast<const uint8_t*>(p)[i + j] << (8 * j);
    return w;
}
__device__ __forceinline__ void store_codes(void* p, int64_t i, int k, uint32_t w) {
    if (k >= 4) {
        *reinterpret_cast<u32u*>(static_cast<uint8_t*>(p) + i) = w;
        return;
    }
    for (int j = 0; j < 3; ++j)
        if (j < k) static_cast<uint8_t*>(p)[i + j] = (uint8_t)(w >> (8 * j));
}

// Called by whole wavefronts: a lane behind the tensor's end (k <= 0) takes part in the block's maximum with zeros.
template <class PT, class GT, bool MASTER>
__device__ __forceinline__ void four8(const Entry& e, const void* gp, int64_t i, int k, const Hyper& h, int64_t t, uint64_t seed) {
    const bool live = k > 0, full = k >= 4;
    float4v p = 0.f, g = 0.f, m = 0.f, v = 0.f, root = 0.f;
    const int64_t blk = i >> 7;
    if (live) {
        p = MASTER ? (full ? F32::load(e.master, i) : F32::load_part(e.master, i, k)) : PT::widen(full ? PT::load(e.param, i) : PT::load_part(e.param, i, k));
        g = GT::widen(full ? GT::load(gp, i) : GT::load_part(gp, i, k));
        m = decode4(load_codes(e.m, i, k), e.ms[blk]);
        const float4v u = decode4(load_codes(e.v, i, k), e.vs[blk]);
        v = u * u;
        update(p, g, m, v, root, h);
    }
    uint32_t mx = 0, ux = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mx = max(mx, top16(m[j]));
        ux = max(ux, top16(root[j]));
    }
    const uint32_t top = block_max((mx & 0xffff0000u) | (ux >> 16));
    if (!live) return;
    const uint32_t em = max(top >> 23, 27u), eu = max((top & 0xffffu) >> 7, 27u);
    const int64_t c = (e.first_block * BLOCK + i) >> 2;
    const uint4 r = philox4x32_10(make_uint4((uint32_t)c, (uint32_t)(c >> 32), (uint32_t)t, 0x40000000u), make_uint2((uint32_t)seed, (uint32_t)(seed >> 32)));
    const uint32_t lo[4] = {r.x & 0xffffu, r.y & 0xffffu, r.z & 0xffffu, r.w & 0xffffu}, hi[4] = {r.x >> 16, r.y >> 16, r.z >> 16, r.w >> 16};
    store_codes(e.m, i, k, encode4(m, __uint_as_float((261u - em) << 23), lo, false));
    store_codes(e.v, i, k, encode4(root, __uint_as_float((261u - eu) << 23), hi, true));
    if ((i & (BLOCK - 1)) == 0) {
        e.ms[blk] = __uint_as_float((em - 7u) << 23);
        e.vs[blk] = __uint_as_float((eu - 7u) << 23);
    }
    if (full) {
        if (MASTER) F32::store(e.master, i, p);
        PT::store(e.param, i, PT::narrow(p));
    } else {
        if (MASTER) F32::store_part(e.master, i, k, p);
        PT::store_part(e.param, i, k, PT::narrow(p));
    }
}

// One workgroup per chunk.
template <class PT, class GT, int BITS, bool MASTER, int N>
__global__ __launch_bounds__(THREADS) void adamw_kernel(AdamwArgs a, Ptrs<N> grads) {
    const int64_t chunk = a.chunk0 + blockIdx.x;
    const int tensor = a.map[chunk];
    const void* gp = grads.p[tensor - a.tensor0];
    if (!gp) return;
    Hyper h;
    int64_t t;
    if (!step_scalars(a, h, t)) return;
    const Entry e = a.entries[tensor];
    const int64_t base = (chunk - e.first_chunk) * ((int64_t)THREADS * 4 * a.unroll);
    for (int s = 0; s < a.unroll; ++s) {
        const int64_t i = base + (int64_t)(s * THREADS + threadIdx.x) * 4;
        const int64_t left = e.n - i;
        const int k = left >= 4 ? 4 : (int)left;
        if (BITS == 8) {
            four8<PT, GT, MASTER>(e, gp, i, k, h, t, a.seed);
        } else if (k > 0) {
            four32<PT, GT, MASTER>(e, gp, i, k, h);
        }
    }
}

__global__ void adamw_count_kernel(float* step, const float* norm, const uint32_t* status) {
    if (guard_says_skip(status) || (norm && norm[2] != 0.f)) return;
    step[0] += 1.f;
}

// ---- norm ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_sum(double x) {
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ double group_sum(double x) {       // over the workgroup, in thread 0
    __shared__ double part[THREADS / 64];
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < THREADS / 64; ++w) s += part[w];
    return s;
}

struct NormArgs {
    const Entry* entries;
    const int32_t* map;
    int64_t chunk0, chunk1;
    int32_t tensor0;
    int32_t unroll;
    double* partials;        // one per workgroup
};
template <class GT, int N>
__global__ __launch_bounds__(THREADS) void grad_norm_kernel(NormArgs a, Ptrs<N> grads) {
    double acc = 0.0;
    for (int64_t chunk = a.chunk0 + blockIdx.x; chunk < a.chunk1; chunk += gridDim.x) {
        const int tensor = a.map[chunk];
        const void* gp = grads.p[tensor - a.tensor0];
        if (!gp) continue;
        const int64_t n = a.entries[tensor].n;
        const int64_t base = (chunk - a.entries[tensor].first_chunk) * ((int64_t)THREADS * 4 * a.unroll);
        for (int s = 0; s < a.unroll; ++s) {
            const int64_t i = base + (int64_t)(s * THREADS + threadIdx.x) * 4;
            const int64_t left = n - i;
            if (left <= 0) break;
            const float4v g = GT::widen(left >= 4 ? GT::load(gp, i) : GT::load_part(gp, i, (int)left));
            for (int j = 0; j < 4; ++j) acc += (double)g[j] * (double)g[j];
        }
    }
    const double s = group_sum(acc);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = s;
}

constexpr int MAX_COUNTERS = 64;
struct Counters {
    float* p[MAX_COUNTERS];
    int n;
};
// words: [norm, coef, skip, skipped so far]; accumulate: the last one goes on counting
__global__ __launch_bounds__(THREADS) void grad_norm_finish_kernel(const double* partials, int n, double max_norm, double grad_scale, float* words, int accumulate,
                                                                   const uint32_t* status, Counters counters) {
    double acc = 0.0;
    for (int k = threadIdx.x; k < n; k += THREADS) acc += partials[k];
    const double s = group_sum(acc);
    if (threadIdx.x != 0) return;
    const float norm = (float)(fabs(grad_scale) * sqrt(s));
    const bool finite = norm < INFINITY;       // false for NaN too
    const bool skip = !finite || guard_says_skip(status);
    words[0] = norm;
    words[1] = finite ? (float)fmin(1.0, max_norm / (fabs(grad_scale) * sqrt(s) + 1e-6)) : 0.f;
    words[2] = skip ? 1.f : 0.f;
    words[3] = (accumulate ? words[3] : 0.f) + (skip ? 1.f : 0.f);
    if (!skip)
        for (int k = 0; k < counters.n; ++k) counters.p[k][0] += 1.f;
}

// ---- host ------------------------------------------------------------------------------------------------------------------
bool plan_ok(const PlanHead* p) { return p && p->magic == PLAN_MAGIC && p->n_tensors > 0; }

// tensors per launch, and one launch per run of tensors that holds a gradient
template <class F>
int for_launches(const void* plan_host, const void* const* grads_host, F&& launch) {
    const PlanHead* h = static_cast<const PlanHead*>(plan_host);
    const Entry* e = plan_entries(plan_host);
    const int per = h->n_tensors <= PTRS_SMALL ? PTRS_SMALL : PTRS_LARGE;
    for (int t0 = 0; t0 < h->n_tensors; t0 += per) {
        int lo = t0, hi = t0 + per < h->n_tensors ? t0 + per : h->n_tensors;
        while (lo < hi && (!grads_host[lo] || e[lo].n == 0)) ++lo;
        while (hi > lo && (!grads_host[hi - 1] || e[hi - 1].n == 0)) --hi;
        if (lo == hi) continue;
        const int64_t c0 = e[lo].first_chunk, c1 = hi < h->n_tensors ? e[hi].first_chunk : h->n_chunks;
        const int rc = launch(lo, hi - lo, c0, c1);
        if (rc != BENERF_OK) return rc;
    }
    return BENERF_OK;
}

template <class PT, class GT, int BITS, bool MASTER, int N>
void launch_adamw(const AdamwArgs& a, int64_t chunks, const void* const* grads, int count, hipStream_t s) {
    Ptrs<N> p;
    for (int k = 0; k < N; ++k) p.p[k] = k < count ? grads[k] : nullptr;
    hipLaunchKernelGGL((adamw_kernel<PT, GT, BITS, MASTER, N>), dim3((unsigned)chunks), dim3(THREADS), 0, s, a, p);
}
typedef void (*AdamwLaunch)(const AdamwArgs&, int64_t, const void* const*, int, hipStream_t);
template <class PT, class GT, int BITS, bool MASTER>
AdamwLaunch by_count(bool small) {
    return small ? launch_adamw<PT, GT, BITS, MASTER, PTRS_SMALL> : launch_adamw<PT, GT, BITS, MASTER, PTRS_LARGE>;
}
template <class PT, class GT>
AdamwLaunch by_state(int bits, bool master, bool small) {
    if constexpr (!PT::NARROW) return bits == 8 ? by_count<PT, GT, 8, false>(small) : by_count<PT, GT, 32, false>(small);      // f32 is its own master
    else if (bits == 8) return master ? by_count<PT, GT, 8, true>(small) : by_count<PT, GT, 8, false>(small);
    else return master ? by_count<PT, GT, 32, true>(small) : by_count<PT, GT, 32, false>(small);
}
template <class PT>
AdamwLaunch by_grad(int grad_type, int bits, bool master, bool small) {
    switch (grad_type) {
        case BENERF_F32: return by_state<PT, F32>(bits, master, small);
        case BENERF_BF16: return by_state<PT, BF16>(bits, master, small);
        default: return by_state<PT, F16>(bits, master, small);
    }
}

template <class GT, int N>
void launch_norm(const NormArgs& a, int blocks, const void* const* grads, int count, hipStream_t s) {
    Ptrs<N> p;
    for (int k = 0; k < N; ++k) p.p[k] = k < count ? grads[k] : nullptr;
    hipLaunchKernelGGL((grad_norm_kernel<GT, N>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a, p);
}

int type_bytes(int type) { return type == BENERF_F32 ? 4 : 2; }
int norm_blocks(int64_t chunks) { return (int)(chunks < 1024 ? chunks : 1024); }

}  // namespace

// A chunk of 4096 elements keeps four independent loads of every array in flight; lists too short to give every CU two of them are cut
// into chunks of 1024.
static int plan_unroll(const BenerfAdamwTensor* t, int n) {
    int64_t chunks = 0;
    for (int k = 0; k < n; ++k) chunks += (t[k].n + 4 * 4 * THREADS - 1) / (4 * 4 * THREADS);
    return chunks >= 512 ? 4 : 1;
}
static int64_t plan_chunks(const BenerfAdamwTensor* t, int n, int unroll) {
    const int64_t size = (int64_t)THREADS * 4 * unroll;
    int64_t chunks = 0;
    for (int k = 0; k < n; ++k) chunks += (t[k].n + size - 1) / size;
    return chunks;
}

extern "C" size_t benerf_adamw_plan_bytes(const BenerfAdamwTensor* tensors_host, int n_tensors) {
    if (!tensors_host || n_tensors <= 0) return 0;
    for (int k = 0; k < n_tensors; ++k)
        if (tensors_host[k].n < 0 || tensors_host[k].n > (1ll << 40)) return 0;
    return HEAD_BYTES + sizeof(Entry) * (size_t)n_tensors + 4 * (size_t)plan_chunks(tensors_host, n_tensors, plan_unroll(tensors_host, n_tensors));
}

extern "C" int benerf_adamw_plan_fill(const BenerfAdamwTensor* tensors_host, int n_tensors, int param_type, int state_bits, void* plan_host, size_t plan_bytes) {
    BENERF_REQUIRE(tensors_host && plan_host && n_tensors > 0, "adamw_plan_fill: null pointer or empty list");
    BENERF_REQUIRE(param_type >= BENERF_F32 && param_type <= BENERF_F16, "adamw_plan_fill: unknown parameter type %d", param_type);
    BENERF_REQUIRE(state_bits == 0 || state_bits == 8 || state_bits == 32, "adamw_plan_fill: moments have 8 or 32 bits (0: gradients only), not %d", state_bits);
    const size_t need = benerf_adamw_plan_bytes(tensors_host, n_tensors);
    BENERF_REQUIRE(need != 0, "adamw_plan_fill: a tensor's size is negative or beyond 2^40");
    if (plan_bytes < need) {
        benerf_set_error("adamw_plan_fill: %zu bytes, %zu needed", plan_bytes, need);
        return BENERF_EWORKSPACE;
    }
    const bool master = tensors_host[0].master != nullptr;
    BENERF_REQUIRE(!master || param_type != BENERF_F32, "adamw_plan_fill: a float32 parameter is its own master copy");
    for (int k = 0; k < n_tensors; ++k) {
        const BenerfAdamwTensor& t = tensors_host[k];
        if (state_bits == 0 || t.n == 0) continue;
        BENERF_REQUIRE(t.param && t.exp_avg && t.exp_avg_sq, "adamw_plan_fill: tensor %d has a null pointer", k);
        BENERF_REQUIRE(state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale), "adamw_plan_fill: tensor %d: 8-bit moments need their scales", k);
        BENERF_REQUIRE((t.master != nullptr) == master, "adamw_plan_fill: master copies for all tensors of a plan or for none");
        BENERF_REQUIRE(t.first_block >= 0, "adamw_plan_fill: tensor %d: negative block number", k);
        BENERF_REQUIRE(((uintptr_t)t.param & (uintptr_t)(type_bytes(param_type) - 1)) == 0 && ((uintptr_t)t.master & 3) == 0 &&
                           (state_bits == 8 || ((((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3) == 0)) &&
                           (((uintptr_t)t.exp_avg_scale | (uintptr_t)t.exp_avg_sq_scale) & 3) == 0,
                       "adamw_plan_fill: tensor %d is not aligned to its elements", k);
    }
    memset(plan_host, 0, need);
    PlanHead* h = static_cast<PlanHead*>(plan_host);
    h->magic = PLAN_MAGIC;
    h->n_tensors = n_tensors;
    h->param_type = param_type;
    h->state_bits = state_bits;
    h->has_master = master;
    h->unroll = plan_unroll(tensors_host, n_tensors);
    h->n_chunks = plan_chunks(tensors_host, n_tensors, h->unroll);
    h->map_at = (int64_t)(HEAD_BYTES + sizeof(Entry) * (size_t)n_tensors);
    h->bytes = (int64_t)need;
    BENERF_REQUIRE(h->n_chunks < (1ll << 24), "adamw_plan_fill: more than 2^24 chunks of 4096 elements");      // a grid holds 2^32 threads
    Entry* e = reinterpret_cast<Entry*>(static_cast<char*>(plan_host) + HEAD_BYTES);
    int32_t* map = reinterpret_cast<int32_t*>(static_cast<char*>(plan_host) + h->map_at);
    const int64_t size = (int64_t)THREADS * 4 * h->unroll;
    int64_t chunk = 0;
    for (int k = 0; k < n_tensors; ++k) {
        const BenerfAdamwTensor& t = tensors_host[k];
        e[k] = Entry{t.param, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.master, t.n, t.first_block, chunk};
        for (int64_t c = (t.n + size - 1) / size; c > 0; --c) map[chunk++] = k;
    }
    return BENERF_OK;
}

extern "C" int benerf_adamw_step(const void* plan_host, const void* plan_dev, const void* const* grads_host, int grad_type, const BenerfAdamwCfg* cfg,
                                 const float* norm_words, const uint32_t* skip_if_range, benerf_stream_t stream) {
    const PlanHead* ph = static_cast<const PlanHead*>(plan_host);
    BENERF_REQUIRE(plan_ok(ph) && plan_dev && grads_host && cfg, "adamw_step: null pointer, or no plan");
    BENERF_REQUIRE(ph->state_bits != 0, "adamw_step: the plan was made for gradients only");
    BENERF_REQUIRE(grad_type >= BENERF_F32 && grad_type <= BENERF_F16, "adamw_step: unknown gradient type %d", grad_type);
    BENERF_REQUIRE(cfg->step_dev || cfg->step >= 1, "adamw_step: steps count from 1");
    BENERF_REQUIRE(cfg->beta1 >= 0.0 && cfg->beta1 < 1.0 && cfg->beta2 >= 0.0 && cfg->beta2 < 1.0 && cfg->eps >= 0.0 && cfg->weight_decay >= 0.0,
                   "adamw_step: beta1, beta2 in [0, 1), eps and weight_decay >= 0");
    for (int k = 0; k < ph->n_tensors; ++k)
        BENERF_REQUIRE(((uintptr_t)grads_host[k] & (uintptr_t)(type_bytes(grad_type) - 1)) == 0, "adamw_step: gradient %d is not aligned to its elements", k);
    AdamwArgs a;
    memset(&a, 0, sizeof(a));
    a.entries = plan_entries(plan_dev);
    a.map = reinterpret_cast<const int32_t*>(static_cast<const char*>(plan_dev) + ph->map_at);
    a.unroll = ph->unroll;
    a.norm = norm_words;
    a.status = skip_if_range;
    a.step_dev = cfg->step_dev;
    a.lr_dev = cfg->lr_dev;
    a.lr = cfg->lr;
    a.beta1 = cfg->beta1;
    a.beta2 = cfg->beta2;
    a.decay_rate = cfg->weight_decay;
    a.step = cfg->step;
    a.seed = cfg->seed;
    a.h.gs = (float)cfg->grad_scale;
    a.h.omb1 = (float)(1.0 - cfg->beta1);
    a.h.b2 = (float)cfg->beta2;
    a.h.omb2 = (float)(1.0 - cfg->beta2);
    a.h.eps = (float)cfg->eps;
    const int64_t t = cfg->step < 1 ? 1 : cfg->step;
    a.h.decay = (float)(1.0 - cfg->lr * cfg->weight_decay);
    a.h.step_size = (float)(cfg->lr / (1.0 - int_power(cfg->beta1, t)));
    a.h.inv_bc2 = (float)(1.0 / sqrt(1.0 - int_power(cfg->beta2, t)));
    const bool small = ph->n_tensors <= PTRS_SMALL;
    AdamwLaunch f = ph->param_type == BENERF_F32 ? by_grad<F32>(grad_type, ph->state_bits, ph->has_master, small)
                    : ph->param_type == BENERF_BF16 ? by_grad<BF16>(grad_type, ph->state_bits, ph->has_master, small)
                                                    : by_grad<F16>(grad_type, ph->state_bits, ph->has_master, small);
    return for_launches(plan_host, grads_host, [&](int lo, int count, int64_t c0, int64_t c1) -> int {
        a.chunk0 = c0;
        a.tensor0 = lo;
        f(a, c1 - c0, grads_host + lo, count, as_stream(stream));
        BENERF_LAUNCH_CHECK("adamw_step");
        return BENERF_OK;
    });
}

extern "C" int benerf_adamw_count(float* step_dev, const float* norm_words, const uint32_t* skip_if_range, benerf_stream_t stream) {
    BENERF_REQUIRE(step_dev, "adamw_count: null pointer");
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(1), 0, as_stream(stream), step_dev, norm_words, skip_if_range);
    BENERF_LAUNCH_CHECK("adamw_count");
    return BENERF_OK;
}

extern "C" size_t benerf_grad_norm_partials(const void* plan_host) {
    const PlanHead* ph = static_cast<const PlanHead*>(plan_host);
    if (!plan_ok(ph)) return 0;
    const int per = ph->n_tensors <= PTRS_SMALL ? PTRS_SMALL : PTRS_LARGE;
    return (size_t)norm_blocks(ph->n_chunks < 1 ? 1 : ph->n_chunks) * (size_t)((ph->n_tensors + per - 1) / per);
}

extern "C" int benerf_grad_norm_partial(const void* plan_host, const void* plan_dev, const void* const* grads_host, int grad_type, double* partials, size_t n_partials,
                                        int64_t* used_host, benerf_stream_t stream) {
    const PlanHead* ph = static_cast<const PlanHead*>(plan_host);
    BENERF_REQUIRE(plan_ok(ph) && plan_dev && grads_host && partials && used_host, "grad_norm_partial: null pointer, or no plan");
    BENERF_REQUIRE(grad_type >= BENERF_F32 && grad_type <= BENERF_F16, "grad_norm_partial: unknown gradient type %d", grad_type);
    for (int k = 0; k < ph->n_tensors; ++k)
        BENERF_REQUIRE(((uintptr_t)grads_host[k] & (uintptr_t)(type_bytes(grad_type) - 1)) == 0, "grad_norm_partial: gradient %d is not aligned to its elements", k);
    NormArgs a;
    a.entries = plan_entries(plan_dev);
    a.map = reinterpret_cast<const int32_t*>(static_cast<const char*>(plan_dev) + ph->map_at);
    a.unroll = ph->unroll;
    const bool small = ph->n_tensors <= PTRS_SMALL;
    int64_t used = 0;
    const int rc = for_launches(plan_host, grads_host, [&](int lo, int count, int64_t c0, int64_t c1) -> int {
        const int blocks = norm_blocks(c1 - c0);
        if ((size_t)(used + blocks) > n_partials) {
            benerf_set_error("grad_norm_partial: room for %zu partial sums, benerf_grad_norm_partials says how many", n_partials);
            return BENERF_EWORKSPACE;
        }
        a.chunk0 = c0;
        a.chunk1 = c1;
        a.tensor0 = lo;
        a.partials = partials + used;
        used += blocks;
        const void* const* g = grads_host + lo;
        hipStream_t s = as_stream(stream);
        if (grad_type == BENERF_F32) small ? launch_norm<F32, PTRS_SMALL>(a, blocks, g, count, s) : launch_norm<F32, PTRS_LARGE>(a, blocks, g, count, s);
        else if (grad_type == BENERF_BF16) small ? launch_norm<BF16, PTRS_SMALL>(a, blocks, g, count, s) : launch_norm<BF16, PTRS_LARGE>(a, blocks, g, count, s);
        else small ? launch_norm<F16, PTRS_SMALL>(a, blocks, g, count, s) : launch_norm<F16, PTRS_LARGE>(a, blocks, g, count, s);
        BENERF_LAUNCH_CHECK("grad_norm_partial");
        return BENERF_OK;
    });
    *used_host = used;
    return rc;
}

extern "C" int benerf_grad_norm_finish(const double* partials, int64_t n_partials, double max_norm, double grad_scale, float* words, int accumulate,
                                       const uint32_t* skip_if_range, float* const* counters_host, int n_counters, benerf_stream_t stream) {
    BENERF_REQUIRE(words && (partials || n_partials == 0) && n_partials >= 0 && n_partials < (1ll << 31), "grad_norm_finish: bad args");
    BENERF_REQUIRE(max_norm > 0.0, "grad_norm_finish: max_norm must be positive (infinity: no clipping)");
    BENERF_REQUIRE(n_counters >= 0 && n_counters <= MAX_COUNTERS && (counters_host || n_counters == 0), "grad_norm_finish: at most %d counters", MAX_COUNTERS);
    Counters c;
    memset(&c, 0, sizeof(c));
    c.n = n_counters;
    for (int k = 0; k < n_counters; ++k) {
        BENERF_REQUIRE(counters_host[k], "grad_norm_finish: null counter");
        c.p[k] = counters_host[k];
    }
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(THREADS), 0, as_stream(stream), partials, (int)n_partials, max_norm, grad_scale, words, accumulate,
                       skip_if_range, c);
    BENERF_LAUNCH_CHECK("grad_norm_finish");
    return BENERF_OK;
}
