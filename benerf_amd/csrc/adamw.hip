// K9: the optimiser over lists of tensors - gradient norm with clip coefficient and verdict, AdamW with moments in 32 or 8 bits.
//
// Mathematics (all in f32 unless said otherwise; products and sums of the moments and of the 32-bit update rounded one by one, this file is
// compiled without contraction):
//   norm    N = |grad_scale| sqrt(sum g^2), squares and sums in f64 (a square of an f32 is exact there: no overflow, no order to care
//           about); coef = min(1, max_norm / (N + 1e-6)); N inf or NaN, or the range guard's verdict: the step is skipped
//   AdamW   h = g * grad_scale * coef;  m += (h - m)(1 - b1);  v = v b2 + h^2 (1 - b2);
//           p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)      (the root times a rounded 1 / sqrt(1 - b2^t))
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
#include <type_traits>

namespace {

constexpr int THREADS = 128;
constexpr int BLOCK = BENERF_ADAMW_BLOCK;
constexpr int CHUNK = THREADS * 4;           // elements a workgroup of the step takes: four a thread
constexpr int64_t PAST_BYTES = 320ll << 20;  // see Shape
constexpr int64_t MAX_CHUNKS = 1ll << 24;    // of a list: a grid holds 2^32 threads
constexpr uint32_t PLAN_MAGIC = 0x41445731u;
static_assert(BLOCK == 128, "a block is half a wavefront of four elements a lane");

// The plan: what a launch needs to find its way through the list, filled on the host, uploaded once.  A workgroup takes a chunk and reads
// everything about it in one record - its data's addresses are one load away, not three.
struct Entry {                // one per tensor, for the host
    int64_t n;
    int64_t first_chunk;
};
struct Chunk {
    void* param;              // of the chunk's first element
    void* m;
    void* v;
    float* ms;
    float* vs;
    float* master;
    int64_t block;            // number of its first block of 128 in the list: the generator's counter
    int32_t tensor;
    int32_t index;            // of the chunk in its tensor
    int32_t count;            // elements
    int32_t pad[3];
};
static_assert(sizeof(Chunk) == 80, "a multiple of 16 bytes");
static_assert(sizeof(Chunk) >= BENERF_ST_WORDS * 4, "a record can be read in place of the guard's words");
struct PlanHead {
    uint32_t magic;
    int32_t n_tensors;
    int32_t param_type, state_bits, has_master;
    int32_t shape;            // SHORT ..: how it is launched and read
    int32_t pad;
    int64_t n_chunks;
    int64_t chunks_at;        // byte offset of the chunks' records
    int64_t bytes;
};
constexpr size_t HEAD_BYTES = 64;
static_assert(sizeof(PlanHead) <= HEAD_BYTES, "plan header");

inline const Entry* plan_entries(const void* plan) { return reinterpret_cast<const Entry*>(static_cast<const char*>(plan) + HEAD_BYTES); }
inline const Chunk* plan_chunks_dev(const void* plan_dev, const PlanHead* h) { return reinterpret_cast<const Chunk*>(static_cast<const char*>(plan_dev) + h->chunks_at); }

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
    const Chunk* chunks;       // of this launch
    int64_t tensor0;           // first tensor of this launch
    Hyper h;                   // for t = step, lr from the host
    const float* norm;         // [4] of the norm operator, or null
    const uint32_t* status;    // range guard words, or null
    const float* step_dev;     // or null: t = step - skipped
    const float* lr_dev;       // or null
    double lr, beta1, beta2, decay_rate;
    int64_t step;
    uint64_t seed;
};
static_assert(sizeof(AdamwArgs) + sizeof(Ptrs<PTRS_LARGE>) <= 4096, "a launch's arguments");

constexpr uint32_t GUARD_LIMIT = 0x477fe000u;       // 65504
__device__ __forceinline__ bool guard_says_skip(const uint32_t* st) {
    if (!st) return false;
    const uint32_t skip = st[BENERF_ST_SKIP], act = st[BENERF_ST_ACT], grad = st[BENERF_ST_GRAD];
    return (skip != 0u) | (act >= GUARD_LIMIT) | (grad >= GUARD_LIMIT);         // no word waits for another
}

__host__ __device__ inline double int_power(double b, int64_t t) {
    double r = 1.0;
    for (; t > 0; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

// 1 / x and 1 / sqrt(x) in f64 from the instructions' estimates (2^-14 at worst) and two steps of Newton's method: as good as f32 needs it
// several times over, at a tenth of a division's latency
__device__ __forceinline__ double reciprocal(double x) {
    double r = __builtin_amdgcn_rcp(x);
    r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
}
__device__ __forceinline__ double reciprocal_root(double x) {
    double r = __builtin_amdgcn_rsq(x);
    r = __builtin_fma(__builtin_fma(-x * r, r, 1.0), 0.5 * r, r);
    return __builtin_fma(__builtin_fma(-x * r, r, 1.0), 0.5 * r, r);
}

// Scalars of this step; false: skipped.  What the host could not know (a counter or a learning rate on the device, steps skipped so
// far) is worked out again here, in f64: 40 multiplications for t < 2^20, once per wave, uniform.
__device__ __forceinline__ bool step_scalars(const AdamwArgs& a, Hyper& h, int64_t& t) {
    // Every word that may matter is asked for at once, with the chunk's record, and before any is looked at; where there is none, the plan's
    // records are read for it.  One word after the other: 30 values 3.9 us against 3.4, two networks 6.5 / 6.1, 4.8 M weights with 8-bit moments
    // 18.8 / 17.8.
    auto word = [&](const void* p, int i) { return static_cast<const uint32_t*>(p ? p : static_cast<const void*>(a.chunks))[i]; };
    const uint32_t skip = word(a.status, BENERF_ST_SKIP), act = word(a.status, BENERF_ST_ACT), grad = word(a.status, BENERF_ST_GRAD), total = word(a.status, BENERF_ST_SKIPPED_TOTAL);
    const uint32_t n1 = word(a.norm, 1), n2 = word(a.norm, 2), n3 = word(a.norm, 3), counter = word(a.step_dev, 0), rate_word = word(a.lr_dev, 0);
    const bool guard = (a.status != nullptr) & ((skip != 0u) | (act >= GUARD_LIMIT) | (grad >= GUARD_LIMIT));
    const uint32_t gated = a.status && !a.norm ? total : 0u;      // the norm's count holds them
    const float coef = a.norm ? __uint_as_float(n1) : 1.f, verdict = a.norm ? __uint_as_float(n2) : 0.f, skipped = a.norm ? __uint_as_float(n3) : 0.f;
    const float counted = __uint_as_float(counter), rate = __uint_as_float(rate_word);
    if (guard | (verdict != 0.f)) return false;
    h = a.h;
    h.gs = h.gs * coef;
    t = a.step;
    if (a.step_dev || a.lr_dev || skipped != 0.f || gated != 0u) {
        t = a.step_dev ? (int64_t)counted : a.step - (int64_t)skipped - (int64_t)gated;
        if (t < 1) t = 1;
        const double lr = a.lr_dev ? (double)rate : a.lr;
        h.decay = (float)(1.0 - lr * a.decay_rate);
        h.step_size = (float)(lr * reciprocal(1.0 - int_power(a.beta1, t)));
        h.inv_bc2 = (float)reciprocal_root(1.0 - int_power(a.beta2, t));
    }
    return true;
}

// ---- four consecutive elements, at any element-aligned address -------------------------------------------------------------
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32u __attribute__((aligned(1)));
// addresses come out of the plan: say that they are global memory's, or every access becomes a flat one
// PAST: past the caches, for lists that no cache holds until the next step
template <typename T, bool PAST = false>
__device__ __forceinline__ T get(const void* p, int64_t i) {
    typedef const __attribute__((address_space(1))) T* at;
    const T* q = static_cast<const T*>(p) + i;
    if constexpr (PAST) return __builtin_nontemporal_load((at)q);
    else return *(at)q;
}
template <typename T, bool PAST = false>
__device__ __forceinline__ void put(void* p, int64_t i, T x) {
    typedef __attribute__((address_space(1))) T* at;
    T* q = static_cast<T*>(p) + i;
    if constexpr (PAST) __builtin_nontemporal_store(x, (at)q);
    else *(at)q = x;
}

// V: a vector of four; raw: its bits in memory.  k of the four elements from i on are there.
template <typename E, typename V>
struct Four {
    typedef E raw __attribute__((ext_vector_type(4)));
    typedef E unaligned __attribute__((ext_vector_type(4), aligned(sizeof(E))));
    static constexpr bool NARROW = sizeof(E) < 4;       // rounded to nearest even, once, when stored
    static constexpr int BYTES = sizeof(E);
    template <bool PAST>
    __device__ static raw load(const void* p, int i, int k) {
        if (k >= 4) return get<unaligned, PAST>(static_cast<const E*>(p) + i, 0);
        raw r = 0;
        for (int j = 0; j < 3; ++j)
            if (j < k) r[j] = get<E>(p, i + j);
        return r;
    }
    template <bool PAST>
    __device__ static void store(void* p, int i, int k, raw r) {
        if (k >= 4) return put<unaligned, PAST>(static_cast<E*>(p) + i, 0, r);
        for (int j = 0; j < 3; ++j)
            if (j < k) put<E>(p, i + j, r[j]);
    }
    __device__ static float4v widen(raw r) { return __builtin_convertvector(__builtin_bit_cast(V, r), float4v); }
    __device__ static raw narrow(float4v x) { return __builtin_bit_cast(raw, __builtin_convertvector(x, V)); }
};
typedef Four<float, float4v> F32;
typedef Four<unsigned short, bf4v> BF16;
typedef Four<unsigned short, half4v> F16;

// ---- moments in 32 bits --------------------------------------------------------------------------------------------------------
// Four elements from i on, k of them there; loads and arithmetic apart, so that a chunk's loads can all be on their way first.
template <class PT, class GT, bool MASTER, bool PAST>
struct Four32 {
    typename PT::raw p;
    typename GT::raw g;
    float4v w, m, v;

    __device__ __forceinline__ void load(const Chunk& c, const void* gp, int i, int k) {
        if (MASTER) w = F32::load<PAST>(c.master, i, k);
        else p = PT::template load<PAST>(c.param, i, k);
        g = GT::template load<PAST>(gp, i, k);
        m = F32::load<PAST>(c.m, i, k);
        v = F32::load<PAST>(c.v, i, k);
    }
    // root and quotient correctly rounded: 100 of the 180 vector instructions that a wavefront takes for its 256 elements, in the time that
    // the memory takes for them
    __device__ __forceinline__ void update(const Hyper& h) {
        if (!MASTER) w = PT::widen(p);
        const float4v x = GT::widen(g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gj = x[j] * h.gs;
            m[j] = m[j] + (gj - m[j]) * h.omb1;
            v[j] = v[j] * h.b2 + (gj * gj) * h.omb2;
            w[j] = w[j] * h.decay - h.step_size * (m[j] / (sqrtf(v[j]) * h.inv_bc2 + h.eps));
        }
    }
    __device__ __forceinline__ void store(const Chunk& c, int i, int k) const {
        if (MASTER) F32::store<PAST>(c.master, i, k, w);
        PT::template store<PAST>(c.param, i, k, PT::narrow(w));
        F32::store<PAST>(c.m, i, k, m);
        F32::store<PAST>(c.v, i, k, v);
    }
};

// ---- moments in 8 bits -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float4v decode4(uint32_t w, float s) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true);
    return float4v{a[0], a[1], b[0], b[1]};
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// maximum of both 16-bit halves over the 32 lanes of a block: four steps inside a row of 16, one between two rows
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
    x = pk_max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true));       // lane ^ 1
    x = pk_max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true));       // lane ^ 2
    x = pk_max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, true));      // a quad on
    x = pk_max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true));      // half a row on
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return pk_max(r[0], r[1]);
}
// Four codes: x / scale on the e4m3 grid (steps of 2^(E - 3), 2^-9 from below 2^-6 on), down after the draw h / 2^16 of a step is added.  The
// instruction puts the draw's 20 highest bits behind the grid's three and cuts them off, below 2^-6 too (compared with the formula in f64 for
// 4 M values from 2^-24 to 2^8: no difference); inf becomes NaN.  213 vector instructions a wavefront against 277 without it: 4.3 M weights 13.6 -> 12.8 us.
__device__ __forceinline__ uint32_t codes4(float4v x, float scale, const uint32_t (&h)[4]) {
    int w = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(0, x[0], h[0], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(w, x[1], h[1], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_sr_fp8_f32(w, x[2], h[2], scale, 2);
    return (uint32_t)__builtin_amdgcn_cvt_scalef32_sr_fp8_f32(w, x[3], h[3], scale, 3);
}
template <bool PAST>
__device__ __forceinline__ uint32_t load_codes(const void* p, int i, int k) {
    if (k >= 4) return get<u32u, PAST>(static_cast<const uint8_t*>(p) + i, 0);
    uint32_t w = 0;
    for (int j = 0; j < 3; ++j)
        if (j < k) w |= (uint32_t)get<uint8_t>(p, i + j) << (8 * j);
    return w;
}
template <bool PAST>
__device__ __forceinline__ void store_codes(void* p, int i, int k, uint32_t w) {
    if (k >= 4) {
        put<u32u, PAST>(static_cast<uint8_t*>(p) + i, 0, w);
        return;
    }
    for (int j = 0; j < 3; ++j)
        if (j < k) put<uint8_t>(p, i + j, (uint8_t)(w >> (8 * j)));
}
__device__ __forceinline__ uint32_t pack_tops(uint32_t m, uint32_t u) { return __builtin_amdgcn_perm(m, u, 0x07060302u); }
// bits of |x|: the highest of four, and where only finite ones count
__device__ __forceinline__ uint32_t top_bits(float4v x) {
    return max(max(__float_as_uint(x[0]), __float_as_uint(x[1])), max(__float_as_uint(x[2]), __float_as_uint(x[3])));
}
__device__ __forceinline__ uint32_t finite_top(float4v x) {
    uint32_t top = 0;
    for (int j = 0; j < 4; ++j) top = fabsf(x[j]) < INFINITY ? max(top, __float_as_uint(fabsf(x[j]))) : top;
    return top;
}
// Philox4x32-10 as in common.h, its products as 32 x 32 -> 64 bits and its sums of three as one instruction each: the step is bound by
// vector instructions, and this is the longest part of them
__device__ __forceinline__ uint4 draws4(int64_t group, uint32_t t, uint2 key) {
    uint32_t x = (uint32_t)group, y = (uint32_t)(group >> 32), z = t, w = 0x40000000u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)x * 0xD2511F53u, b = (uint64_t)z * 0xCD9E8D57u;
        x = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), y, key.x, 0x96);
        z = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), w, key.y, 0x96);
        y = (uint32_t)b;
        w = (uint32_t)a;
        key.x += 0x9E3779B9u;
        key.y += 0xBB67AE85u;
    }
    return make_uint4(x, y, z, w);
}

// Called by whole wavefronts: a lane behind the end takes part in its block's maximum with zeros.
template <class PT, class GT, bool MASTER, bool PAST>
struct Four8 {
    typename PT::raw p;
    typename GT::raw g;
    float4v w;
    uint32_t mw, uw;          // codes, before and after the update
    float ms, us;             // scales, likewise

    __device__ __forceinline__ void load(const Chunk& c, const void* gp, int i, int k) {
        if (MASTER) w = F32::load<PAST>(c.master, i, k);
        else p = PT::template load<PAST>(c.param, i, k);
        g = GT::template load<PAST>(gp, i, k);
        mw = load_codes<PAST>(c.m, i, k);
        uw = load_codes<PAST>(c.v, i, k);
        ms = k > 0 ? get<float>(c.ms, i >> 7) : 0.f;
        us = k > 0 ? get<float>(c.vs, i >> 7) : 0.f;
    }
    __device__ __forceinline__ void update(const Hyper& h, int64_t group, uint32_t t, uint2 key) {
        if (!MASTER) w = PT::widen(p);
        const float4v x = GT::widen(g);
        float4v m = decode4(mw, ms), v, root;
        const float4v u = decode4(uw, us);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gj = x[j] * h.gs;
            m[j] = m[j] + (gj - m[j]) * h.omb1;
            v[j] = (u[j] * u[j]) * h.b2 + (gj * gj) * h.omb2;
            root[j] = __builtin_amdgcn_sqrtf(v[j]);              // to 1 ulp: the code has 4 bits
        }
        uint32_t top = block_max(pack_tops(__float_as_uint(fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3])))), top_bits(root)));
        // The instruction takes denormal numbers for 0: their roots (below 2^-63) count where nothing else in the block does, or with an eps
        // that they are not lost in.  The maximum found again is that of the finite ones, so the next branch is not taken behind this one: inf and NaN
        // of any payload are left to the conversion, which makes them NaN (nine patterns, eight draws each).
        if (h.eps < 1e-11f || __any((top & 0xffffu) == 0u)) {
            for (int j = 0; j < 4; ++j) root[j] = sqrtf(v[j]);
            top = block_max(pack_tops(finite_top(m), finite_top(root)));
        }
        // inf or NaN (NaN in m comes with one in v): it must not take the block's other values along
        if (__any((top & 0x7f80u) == 0x7f80u || (top & 0x7f800000u) == 0x7f800000u)) {
            top = block_max(pack_tops(finite_top(m), finite_top(root)));
            for (int j = 0; j < 4; ++j) {
                m[j] = m[j] == m[j] ? m[j] : __uint_as_float(0x7fc00000u);
                root[j] = root[j] == root[j] ? root[j] : __uint_as_float(0x7fc00000u);
            }
        }
        // to a few ulp of the update: the moments behind it have four bits
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = __builtin_fmaf(-h.step_size, m[j] * __builtin_amdgcn_rcpf(__builtin_fmaf(root[j], h.inv_bc2, h.eps)), w[j] * h.decay);
        const uint32_t em = max(top >> 23, 27u), eu = max(top >> 7 & 0xffu, 27u);
        ms = __uint_as_float((em - 7u) << 23);
        us = __uint_as_float((eu - 7u) << 23);
        const float least = __uint_as_float((eu - 16u) << 23);
        const uint4 r = draws4(group, t, key);
        // one step is the least that a root above 0 may become: lifted to it, it stays there whatever the draw
#pragma unroll
        for (int j = 0; j < 4; ++j) root[j] = root[j] < least ? (v[j] > 0.f ? least : 0.f) : root[j];
        mw = codes4(m, ms, {r.x << 16, r.y << 16, r.z << 16, r.w << 16});
        uw = codes4(root, us, {r.x & 0xffff0000u, r.y & 0xffff0000u, r.z & 0xffff0000u, r.w & 0xffff0000u});
    }
    __device__ __forceinline__ void store(const Chunk& c, int i, int k) const {
        if (MASTER) F32::store<PAST>(c.master, i, k, w);
        PT::template store<PAST>(c.param, i, k, PT::narrow(w));
        store_codes<PAST>(c.m, i, k, mw);
        store_codes<PAST>(c.v, i, k, uw);
        if (k > 0 && (i & (BLOCK - 1)) == 0) {
            put<float>(c.ms, i >> 7, ms);
            put<float>(c.vs, i >> 7, us);
        }
    }
};

// Workgroups go to the eight XCDs in turn, each with an L2 of its own; eight chunks share the lines of their scales, two those of their records,
// so RUN chunks in a row stay on one XCD (an incomplete last group stays as it is).  235 M weights with 8-bit moments: 600 us in turn, 616 with
// runs of 8, 578 of 32, 572 of 64, 573 of 128; 126 M bfloat16 with master copies 587 / 590 / 582 / 573 / 584; lists of 48 MB 16.5 / - / 15.3 / 15.2
// / 15.1.
__device__ __forceinline__ uint32_t chunk_of(uint32_t b, uint32_t n) {
    constexpr uint32_t XCDS = 8, RUN = 64, GROUP = XCDS * RUN;
    const uint32_t g = b / GROUP, r = b % GROUP;
    return (g + 1) * GROUP <= n ? g * GROUP + (r % XCDS) * RUN + r / XCDS : b;
}

// One workgroup per chunk, four elements a thread: wide loads, 38 registers, all 32 wavefronts a CU.  Long lists are bound by HBM - 126 M bfloat16
// with master copies 570 us (6.2 TB/s), 235 M with 8-bit moments 577 (6.6) -, short ones by the launch and the way to the data, kernel
// arguments, then record and words, then the gradient's address: 3.4 us for 30 values, 6.1 for two networks of 1.2 M (5.5 TB/s).  Four and eight chunks
// in a row to a workgroup: 639 / 667, 654 / 664 and 9.9 / 13.6 us; workgroups and chunks half and twice as large: 585 / 581, 592 / 599, 6.1 / 6.2.
template <class PT, class GT, int BITS, bool MASTER, int N, bool PAST>
__global__ __launch_bounds__(THREADS) void adamw_kernel(AdamwArgs a, Ptrs<N> grads) {
    const Chunk c = a.chunks[chunk_of(blockIdx.x, gridDim.x)];
    Hyper h;
    int64_t t;
    const bool go = step_scalars(a, h, t);
    const char* gp = static_cast<const char*>(grads.p[c.tensor - a.tensor0]);
    if (!gp || !go) return;
    gp += (int64_t)c.index * CHUNK * GT::BYTES;
    const int i = threadIdx.x * 4;
    typename std::conditional<BITS == 8, Four8<PT, GT, MASTER, PAST>, Four32<PT, GT, MASTER, PAST>>::type f;
    auto chunk = [&](int here) {              // elements there from i on
        f.load(c, gp, i, here);
        if constexpr (BITS == 8) f.update(h, c.block * (BLOCK / 4) + threadIdx.x, (uint32_t)t, make_uint2((uint32_t)a.seed, (uint32_t)(a.seed >> 32)));
        else f.update(h);
        f.store(c, i, here);
    };
    if (c.count == CHUNK) chunk(4);           // no lane looks for an end
    else chunk(c.count - i);
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
// Chunks that a workgroup reads at a time, and most workgroups.  Two networks of 1.2 M weights: 4.1 us with 8, 4.9 with 16; 262 M bfloat16
// gradients, past the caches: 85 us with 8 and 2048 workgroups, 80 us (6.6 TB/s) with 16 and 1024.
constexpr int NORM_THREADS = 256;
constexpr int norm_batch(bool past) { return past ? 16 : 8; }
constexpr int norm_most(bool past) { return past ? 1024 : 2048; }
__device__ __forceinline__ double group_sum(double x) {       // over the workgroup, in thread 0
    __shared__ double part[NORM_THREADS / 64];
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < NORM_THREADS / 64; ++w) s += part[w];
    return s;
}

struct NormArgs {
    const Chunk* chunks;
    int64_t n_chunks;
    int64_t tensor0;
    double* partials;        // one per workgroup
};
// Squares of a workgroup's share, summed: in thread 0.  It takes BATCH chunks at a time.  Where they are one piece of one tensor - nearly always
// in a long list - their first record says all, and FOURS loads of every thread are on their way together.
template <class GT, int N, bool PAST>
__device__ __forceinline__ double share_sum(const NormArgs& a, const Ptrs<N>& grads) {
    constexpr int BATCH = norm_batch(PAST), FOURS = BATCH * CHUNK / 4 / NORM_THREADS;
    auto address = [&](const Chunk& c) {
        const char* gp = static_cast<const char*>(grads.p[c.tensor - a.tensor0]);
        return gp ? gp + (int64_t)c.index * CHUNK * GT::BYTES : nullptr;
    };
    double acc = 0.0;
    auto add = [&](typename GT::raw g) {
        const float4v x = GT::widen(g);
        for (int j = 0; j < 4; ++j) acc = __builtin_fma((double)x[j], (double)x[j], acc);
    };
    for (int64_t k = (int64_t)blockIdx.x * BATCH; k < a.n_chunks; k += (int64_t)gridDim.x * BATCH) {
        const int here = a.n_chunks - k < BATCH ? (int)(a.n_chunks - k) : BATCH;
        const Chunk &c = a.chunks[k], &d = a.chunks[k + here - 1];
        if (here == BATCH && c.tensor == d.tensor && d.count == CHUNK) {
            const char* gp = address(c);
            if (!gp) continue;
            typename GT::raw g[FOURS];
#pragma unroll
            for (int s = 0; s < FOURS; ++s) g[s] = GT::template load<PAST>(gp, (s * NORM_THREADS + threadIdx.x) * 4, 4);
#pragma unroll
            for (int s = 0; s < FOURS; ++s) add(g[s]);
        } else {
            constexpr int SIDE = NORM_THREADS / THREADS;             // chunks side by side in the workgroup, whole wavefronts each
            const int mine = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS), i = (threadIdx.x % THREADS) * 4;
            typename GT::raw g[BATCH / SIDE];
#pragma unroll
            for (int b = 0; b < BATCH / SIDE; ++b) {
                g[b] = 0;
                if (b * SIDE + mine >= here) continue;
                const Chunk& e = a.chunks[k + b * SIDE + mine];
                const char* gp = address(e);
                if (gp) g[b] = GT::template load<PAST>(gp, i, e.count - i);
            }
#pragma unroll
            for (int b = 0; b < BATCH / SIDE; ++b) add(g[b]);
        }
    }
    return group_sum(acc);
}
template <class GT, int N, bool PAST>
__global__ __launch_bounds__(NORM_THREADS) void grad_norm_kernel(NormArgs a, Ptrs<N> grads) {
    const double s = share_sum<GT, N, PAST>(a, grads);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = s;
}

constexpr int MAX_COUNTERS = 64;
// words: [norm, coef, skip, skipped so far]; accumulate: the last one goes on counting
struct Finish {
    double max_norm, grad_scale;
    float* words;
    const uint32_t* status;
    int accumulate;
    int n_counters;
    float* counters[MAX_COUNTERS];
};
__device__ __forceinline__ void finish(const Finish& f, double s) {
    const float norm = (float)(fabs(f.grad_scale) * sqrt(s));
    const bool finite = norm < INFINITY;       // false for NaN too
    const bool skip = !finite || guard_says_skip(f.status);
    f.words[0] = norm;
    f.words[1] = finite ? (float)fmin(1.0, f.max_norm / (fabs(f.grad_scale) * sqrt(s) + 1e-6)) : 0.f;
    f.words[2] = skip ? 1.f : 0.f;
    f.words[3] = (f.accumulate ? f.words[3] : 0.f) + (skip ? 1.f : 0.f);
    if (!skip)
        for (int k = 0; k < f.n_counters; ++k) f.counters[k][0] += 1.f;
}
// One workgroup over at most a few thousand sums, 2.2 us: a launch and two dependent reads.
__global__ __launch_bounds__(NORM_THREADS) void grad_norm_finish_kernel(const double* partials, int n, Finish f) {
    double acc = 0.0;
#pragma unroll 4
    for (int k = threadIdx.x; k < n; k += NORM_THREADS) acc += partials[k];
    const double s = group_sum(acc);
    if (threadIdx.x == 0) finish(f, s);
}
// A list of at most ONE_CHUNKS chunks: one workgroup, one launch.  12 numbers: 9.0 -> 6.7 us a call, 4.3 -> 2.9 us of them on the device; 16 Ki
// 4.6 -> 4.2 on the device, 32 Ki 4.6 -> 6.2.
constexpr int ONE_CHUNKS = 32;
template <class GT>
__global__ __launch_bounds__(NORM_THREADS) void grad_norm_one_kernel(NormArgs a, Ptrs<PTRS_SMALL> grads, Finish f) {
    const double s = share_sum<GT, PTRS_SMALL, false>(a, grads);
    if (threadIdx.x == 0) finish(f, s);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// of a list: SHORT, or MANY where a launch of the small kind cannot carry its addresses; PAST: more than the memory-side cache (256 MB) keeps
// from one step to the next, so it is read and written past the caches.  32-bit step over parameters, gradients and moments of 192 MB: 52 us
// through them, 57 past them; 256 MB 70 / 75; 320 MB 93 / 94; 384 MB 131 / 111; 2 GB 739 / 600 (6.3 TB/s); 8 bits alike.
enum Shape { SHORT, MANY, PAST };
int type_bytes(int type) { return type == BENERF_F32 ? 4 : 2; }
int per_launch(int shape) { return shape == SHORT ? PTRS_SMALL : PTRS_LARGE; }
int64_t count_chunks(const BenerfAdamwTensor* t, int n) {
    int64_t chunks = 0;
    for (int k = 0; k < n; ++k) chunks += (t[k].n + CHUNK - 1) / CHUNK;
    return chunks;
}
// the first tensor with elements says whether the list has masters: an empty one has no memory
bool list_has_master(const BenerfAdamwTensor* t, int n, int state_bits) {
    for (int k = 0; k < n && state_bits != 0; ++k)
        if (t[k].n > 0) return t[k].master != nullptr;
    return false;
}
int plan_shape(const BenerfAdamwTensor* t, int n, int param_type, int state_bits, bool master) {
    int64_t total = 0;
    for (int k = 0; k < n; ++k) total += t[k].n;
    const int width = type_bytes(param_type);
    const int64_t bytes = total * (state_bits == 0 ? width : 2 * width + (state_bits == 8 ? 2 : 8) + (master ? 4 : 0));
    return bytes > PAST_BYTES ? PAST : n <= PTRS_SMALL ? SHORT : MANY;
}

bool plan_ok(const PlanHead* p) { return p && p->magic == PLAN_MAGIC && p->n_tensors > 0; }

// tensors per launch, and one launch per run of tensors that holds a gradient
template <class F>
int for_launches(const void* plan_host, const void* const* grads_host, F&& launch) {
    const PlanHead* h = static_cast<const PlanHead*>(plan_host);
    const Entry* e = plan_entries(plan_host);
    const int per = per_launch(h->shape);
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

template <int N>
Ptrs<N> pack(const void* const* grads, int count) {
    Ptrs<N> p;
    for (int k = 0; k < N; ++k) p.p[k] = k < count ? grads[k] : nullptr;
    return p;
}
typedef void (*AdamwLaunch)(const AdamwArgs&, int64_t, const void* const*, int, hipStream_t);
template <class PT, class GT, int BITS, bool MASTER, int N, bool PAST>
void launch_adamw(const AdamwArgs& a, int64_t chunks, const void* const* grads, int count, hipStream_t s) {
    hipLaunchKernelGGL((adamw_kernel<PT, GT, BITS, MASTER, N, PAST>), dim3((unsigned)chunks), dim3(THREADS), 0, s, a, pack<N>(grads, count));
}
template <class PT, class GT, int BITS, bool MASTER>
AdamwLaunch by_shape(int shape) {
    switch (shape) {
        case SHORT: return launch_adamw<PT, GT, BITS, MASTER, PTRS_SMALL, false>;
        case MANY: return launch_adamw<PT, GT, BITS, MASTER, PTRS_LARGE, false>;
        default: return launch_adamw<PT, GT, BITS, MASTER, PTRS_LARGE, true>;
    }
}
template <class PT, class GT>
AdamwLaunch by_state(int bits, bool master, int shape) {
    if constexpr (!PT::NARROW) return bits == 8 ? by_shape<PT, GT, 8, false>(shape) : by_shape<PT, GT, 32, false>(shape);      // f32 is its own master
    else if (bits == 8) return master ? by_shape<PT, GT, 8, true>(shape) : by_shape<PT, GT, 8, false>(shape);
    else return master ? by_shape<PT, GT, 32, true>(shape) : by_shape<PT, GT, 32, false>(shape);
}
template <class PT>
AdamwLaunch by_grad(int grad_type, int bits, bool master, int shape) {
    switch (grad_type) {
        case BENERF_F32: return by_state<PT, F32>(bits, master, shape);
        case BENERF_BF16: return by_state<PT, BF16>(bits, master, shape);
        default: return by_state<PT, F16>(bits, master, shape);
    }
}

typedef void (*NormLaunch)(const NormArgs&, int, const void* const*, int, hipStream_t);
template <class GT, int N, bool PAST>
void launch_norm(const NormArgs& a, int blocks, const void* const* grads, int count, hipStream_t s) {
    hipLaunchKernelGGL((grad_norm_kernel<GT, N, PAST>), dim3((unsigned)blocks), dim3(NORM_THREADS), 0, s, a, pack<N>(grads, count));
}
template <class GT>
void launch_norm_one(const NormArgs& a, const void* const* grads, int count, const Finish& f, hipStream_t s) {
    hipLaunchKernelGGL((grad_norm_one_kernel<GT>), dim3(1), dim3(NORM_THREADS), 0, s, a, pack<PTRS_SMALL>(grads, count), f);
}
template <class GT>
NormLaunch norm_by_shape(int shape) {
    switch (shape) {
        case SHORT: return launch_norm<GT, PTRS_SMALL, false>;
        case MANY: return launch_norm<GT, PTRS_LARGE, false>;
        default: return launch_norm<GT, PTRS_LARGE, true>;
    }
}

int norm_blocks(int64_t chunks, int shape) {
    const int64_t batch = norm_batch(shape == PAST), most = norm_most(shape == PAST), blocks = (chunks + batch - 1) / batch;
    return (int)(blocks < most ? blocks : most);
}

}  // namespace

extern "C" size_t benerf_adamw_plan_bytes(const BenerfAdamwTensor* tensors_host, int n_tensors) {
    if (!tensors_host || n_tensors <= 0) return 0;
    for (int k = 0; k < n_tensors; ++k)
        if (tensors_host[k].n < 0 || tensors_host[k].n > (1ll << 40)) return 0;
    const int64_t chunks = count_chunks(tensors_host, n_tensors);
    return chunks < MAX_CHUNKS ? HEAD_BYTES + sizeof(Entry) * (size_t)n_tensors + sizeof(Chunk) * (size_t)chunks : 0;
}

extern "C" int benerf_adamw_plan_fill(const BenerfAdamwTensor* tensors_host, int n_tensors, int param_type, int state_bits, void* plan_host, size_t plan_bytes) {
    BENERF_REQUIRE(tensors_host && plan_host && n_tensors > 0, "adamw_plan_fill: null pointer or empty list");
    BENERF_REQUIRE(param_type >= BENERF_F32 && param_type <= BENERF_F16, "adamw_plan_fill: unknown parameter type %d", param_type);
    BENERF_REQUIRE(state_bits == 0 || state_bits == 8 || state_bits == 32, "adamw_plan_fill: moments have 8 or 32 bits (0: gradients only), not %d", state_bits);
    const size_t need = benerf_adamw_plan_bytes(tensors_host, n_tensors);
    BENERF_REQUIRE(need != 0, "adamw_plan_fill: a tensor's size is negative, or the list has 2^24 chunks of 512 elements or more");
    if (plan_bytes < need) {
        benerf_set_error("adamw_plan_fill: %zu bytes, %zu needed", plan_bytes, need);
        return BENERF_EWORKSPACE;
    }
    const bool master = list_has_master(tensors_host, n_tensors, state_bits);
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
    memset(plan_host, 0, HEAD_BYTES);
    PlanHead* h = static_cast<PlanHead*>(plan_host);
    h->magic = PLAN_MAGIC;
    h->n_tensors = n_tensors;
    h->param_type = param_type;
    h->state_bits = state_bits;
    h->has_master = master;
    h->shape = plan_shape(tensors_host, n_tensors, param_type, state_bits, master);
    h->n_chunks = count_chunks(tensors_host, n_tensors);
    h->chunks_at = (int64_t)(HEAD_BYTES + sizeof(Entry) * (size_t)n_tensors);
    h->bytes = (int64_t)need;
    Entry* e = reinterpret_cast<Entry*>(static_cast<char*>(plan_host) + HEAD_BYTES);
    Chunk* chunk = reinterpret_cast<Chunk*>(static_cast<char*>(plan_host) + h->chunks_at);
    int64_t at = 0;
    auto on = [](void* p, int64_t bytes) { return p ? static_cast<char*>(p) + bytes : nullptr; };
    for (int k = 0; k < n_tensors; ++k) {
        const BenerfAdamwTensor& t = tensors_host[k];
        e[k] = Entry{t.n, at};
        for (int64_t i = 0; i < t.n; i += CHUNK, ++at, ++chunk) {
            const int64_t w = state_bits == 8 ? 1 : 4;
            memset(chunk, 0, sizeof(Chunk));
            chunk->param = on(t.param, i * type_bytes(param_type));
            chunk->m = on(t.exp_avg, i * w);
            chunk->v = on(t.exp_avg_sq, i * w);
            if (state_bits == 8) {
                chunk->ms = t.exp_avg_scale + i / BLOCK;
                chunk->vs = t.exp_avg_sq_scale + i / BLOCK;
            }
            chunk->master = t.master ? t.master + i : nullptr;
            chunk->block = t.first_block + i / BLOCK;
            chunk->tensor = k;
            chunk->index = (int32_t)(i / CHUNK);
            chunk->count = (int32_t)(t.n - i < CHUNK ? t.n - i : CHUNK);
        }
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
    AdamwLaunch f = ph->param_type == BENERF_F32 ? by_grad<F32>(grad_type, ph->state_bits, ph->has_master, ph->shape)
                    : ph->param_type == BENERF_BF16 ? by_grad<BF16>(grad_type, ph->state_bits, ph->has_master, ph->shape)
                                                    : by_grad<F16>(grad_type, ph->state_bits, ph->has_master, ph->shape);
    return for_launches(plan_host, grads_host, [&](int lo, int count, int64_t c0, int64_t c1) -> int {
        a.chunks = plan_chunks_dev(plan_dev, ph) + c0;
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
    const int per = per_launch(ph->shape);
    return (size_t)norm_blocks(ph->n_chunks < 1 ? 1 : ph->n_chunks, ph->shape) * (size_t)((ph->n_tensors + per - 1) / per);
}

extern "C" int benerf_grad_norm(const BenerfGradList* lists_host, int n_lists, double* partials, size_t n_partials, double max_norm, double grad_scale, float* words,
                                int accumulate, const uint32_t* skip_if_range, float* const* counters_host, int n_counters, benerf_stream_t stream) {
    BENERF_REQUIRE((lists_host || n_lists == 0) && n_lists >= 0 && words, "grad_norm: null pointer");
    BENERF_REQUIRE(max_norm > 0.0, "grad_norm: max_norm must be positive (infinity: no clipping)");
    BENERF_REQUIRE(n_counters >= 0 && n_counters <= MAX_COUNTERS && (counters_host || n_counters == 0), "grad_norm: at most %d counters", MAX_COUNTERS);
    Finish f;
    memset(&f, 0, sizeof(f));
    f.max_norm = max_norm;
    f.grad_scale = grad_scale;
    f.words = words;
    f.status = skip_if_range;
    f.accumulate = accumulate;
    f.n_counters = n_counters;
    for (int k = 0; k < n_counters; ++k) {
        BENERF_REQUIRE(counters_host[k], "grad_norm: null counter");
        f.counters[k] = counters_host[k];
    }
    size_t room = 0;
    for (int l = 0; l < n_lists; ++l) {
        const BenerfGradList& g = lists_host[l];
        const PlanHead* ph = static_cast<const PlanHead*>(g.plan_host);
        BENERF_REQUIRE(plan_ok(ph) && g.plan_dev && g.grads_host, "grad_norm: list %d: null pointer, or no plan", l);
        BENERF_REQUIRE(g.grad_type >= BENERF_F32 && g.grad_type <= BENERF_F16, "grad_norm: list %d: unknown gradient type %d", l, g.grad_type);
        for (int k = 0; k < ph->n_tensors; ++k)
            BENERF_REQUIRE(((uintptr_t)g.grads_host[k] & (uintptr_t)(type_bytes(g.grad_type) - 1)) == 0, "grad_norm: gradient %d is not aligned to its elements", k);
        room += benerf_grad_norm_partials(g.plan_host);
    }
    BENERF_REQUIRE(room < (1ull << 31) && (partials || room == 0), "grad_norm: null pointer");
    if (n_partials < room) {
        benerf_set_error("grad_norm: room for %zu partial sums, %zu needed (benerf_grad_norm_partials of every list)", n_partials, room);
        return BENERF_EWORKSPACE;
    }
    hipStream_t s = as_stream(stream);
    bool finished = false;
    int used = 0;
    for (int l = 0; l < n_lists; ++l) {
        const BenerfGradList& g = lists_host[l];
        const PlanHead* ph = static_cast<const PlanHead*>(g.plan_host);
        const NormLaunch share = g.grad_type == BENERF_F32 ? norm_by_shape<F32>(ph->shape) : g.grad_type == BENERF_BF16 ? norm_by_shape<BF16>(ph->shape) : norm_by_shape<F16>(ph->shape);
        const int rc = for_launches(g.plan_host, g.grads_host, [&](int lo, int count, int64_t c0, int64_t c1) -> int {
            const int blocks = norm_blocks(c1 - c0, ph->shape);
            const NormArgs a = {plan_chunks_dev(g.plan_dev, ph) + c0, c1 - c0, lo, partials + used};
            if (n_lists == 1 && ph->shape == SHORT && c1 - c0 <= ONE_CHUNKS) {      // the list's only launch
                (g.grad_type == BENERF_F32 ? launch_norm_one<F32> : g.grad_type == BENERF_BF16 ? launch_norm_one<BF16> : launch_norm_one<F16>)(a, g.grads_host + lo, count, f, s);
                finished = true;
            } else {
                used += blocks;
                share(a, blocks, g.grads_host + lo, count, s);
            }
            BENERF_LAUNCH_CHECK("grad_norm");
            return BENERF_OK;
        });
        if (rc != BENERF_OK) return rc;
    }
    if (finished) return BENERF_OK;
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(NORM_THREADS), 0, s, partials, used, f);
    BENERF_LAUNCH_CHECK("grad_norm");
    return BENERF_OK;
}
