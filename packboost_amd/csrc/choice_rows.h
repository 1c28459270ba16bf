// Ragged sets of candidate rows as wavefronts read, reduce and write them: what the kernels on choices share.
//
// Set g holds rows [off[g], off[g + 1]). Row i's logit is score_i + table[bucket(position_i)], -inf where its mask
// is 0. Rows go by runs of 8 a lane, in accesses of 16 bytes where the addresses allow it.
#pragma once

#include "pb_internal.h"

namespace pb {
namespace {

constexpr int kWaves = kBlock / kWave;
constexpr float kInf = __builtin_huge_valf();
// The maximum of no row: below every logit but -inf, whose exponential over it is 0, and finite.
constexpr float kLowest = -3.402823466e38f;
constexpr int kRun = 8;                                     // consecutive rows of a lane
constexpr int kWideRuns = kSetWideRows / (kRun * kBlock);   // runs of a thread of a longer set
constexpr int kTileRounds = kSetTileSets / kWave;           // sets of a tile per lane
constexpr int kBins = 256;     // LDS words of the table's gradient per wave: buckets x copies
constexpr int kLookup = 2048;  // bytes of the position lookup kept in LDS
static_assert(kSetTileRows == kRun * kWave, "a lane holds one run of a tile");

// e^x of a difference to a set's maximum or lse: 2^(x log2(e)) in two instructions. The product's rounding
// and log2(e)'s own move the result by at most |x| 2^-24 of itself and a unit, 64 2^-24 at x = -87. Sums of
// exponentials take it, in which a term of size e^x weighs so much; gradients rounded to 16 bits, too. Results
// below 2^-126 are 0; e^-inf is 0 and NaN stays NaN.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269502162933349609375f); }

// The same within 2 2^-24 beside the instruction's own error, for gradients in float32: e = 2^t, t the rounded
// product, and e (x - t log 2) for what the rounding took (four instructions a row: for bfloat16 scores 3 us of the
// 103 of the policy loss of 40M rows).
__device__ __forceinline__ float close_exp(float x) {
    const float d = __builtin_elementwise_maximum(x, -200.0f);  // a NaN is the larger one
    const float t = d * 1.44269502162933349609375f, e = __builtin_amdgcn_exp2f(t);
    const float rest = __builtin_fmaf(t, 1.904654299957e-9f, __builtin_fmaf(t, -0.693147182464599609375f, d));
    return __builtin_fmaf(e, rest, e);
}

// log x for x = 0 or above 1/2: 0 gives -inf, NaN stays NaN.
__device__ __forceinline__ float log_of(float x) { return __builtin_amdgcn_logf(x) * 0.69314718055994530942f; }

// What a step of a policy has once is taken to below float32's rounding: its loss terms cancel (advantages of
// both signs, e^d - d - 1 of a small d), and its ratio is held against bounds. All in double it took half as
// long again (tiles of 480k sets, before the table's bins had units of their own: 32 us, 24 so, 22.7 in float32
// alone).
//
// log x within 2^-30 for finite x above 1/2 (else as log_of): x = 2^k m, m in [2/3, 4/3), and
// log m = 2 (f + f^3 / 3 + ... + f^11 / 11), f = (m - 1) / (m + 1) with the quotient's remainder, |f| <= 1/5.
__device__ __forceinline__ double fine_log(float x) {
    if (!(x > 0.5f && x < kInf)) return (double)log_of(x);
    const float half = __builtin_amdgcn_frexp_mantf(x);  // [1/2, 1)
    const bool low = half < 0.666666687f;
    const float m = low ? 2.0f * half : half;
    const int k = __builtin_amdgcn_frexp_expf(x) - (low ? 1 : 0);
    const float n = m - 1.0f, s = m + 1.0f, rest = m - (s - 1.0f);  // n, s + rest exact
    const float inv = __builtin_amdgcn_rcpf(s), f = n * inv, q = f * f;
    float p = 1.0f / 11;
    p = __builtin_fmaf(p, q, 1.0f / 9);
    p = __builtin_fmaf(p, q, 1.0f / 7);
    p = __builtin_fmaf(p, q, 1.0f / 5);
    p = __builtin_fmaf(p, q, 1.0f / 3);
    const float small = __builtin_fmaf(p * q, f, (__builtin_fmaf(-f, s, n) - f * rest) * inv);
    return __builtin_fma((double)k, 0.69314718055994531, 2.0 * ((double)f + (double)small));
}

// e^x, e^x - 1 and e^x - 1 - x, within 1, 1 and 4 units in the last place: x = k log 2 + r, |r| <= log(2) / 2, and
// eight terms of r's series (r^2 / 2 + ... + r^8 / 40320 in float32, what is joined with 1, 2^k and x in double).
// From |x| of 200 on, infinities and NaN as of e^x.
struct FineExp {
    float all, less_one, less_line;
    __device__ __forceinline__ explicit FineExp(double x) {
        const float hi = (float)x, k = __builtin_rintf(hi * 1.44269504f);
        const double rest = __builtin_fma((double)k, -0.69314718055994531, x);
        const float r = (float)rest;
        float p = 1.0f / 40320;
        p = __builtin_fmaf(p, r, 1.0f / 5040);
        p = __builtin_fmaf(p, r, 1.0f / 720);
        p = __builtin_fmaf(p, r, 1.0f / 120);
        p = __builtin_fmaf(p, r, 1.0f / 24);
        p = __builtin_fmaf(p, r, 1.0f / 6);
        p = __builtin_fmaf(p, r, 0.5f);
        p *= r * r;
        const bool near = __builtin_fabsf(hi) < 200.0f;
        const int n = near ? (int)k : 0;
        const double unit = ldexp(1.0, n), one = n == 0 ? rest + (double)p : __builtin_fma(unit, rest + (double)p, unit - 1.0);
        all = near ? __builtin_amdgcn_ldexpf(1.0f + (r + p), n) : exp_of(hi);
        less_one = near ? (float)one : all - 1.0f;
        less_line = !near ? (hi > 0.0f ? all : (all - 1.0f) - hi) : n == 0 ? p : (float)(one - x);
    }
};

// Maxima that pass a NaN over (fmaxf first quiets operands that the compiler cannot see through).
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ float bf16_value(uint32_t b) { return __uint_as_float(b << 16); }

__device__ __forceinline__ float f16_value(uint32_t b) {
    const uint16_t u = (uint16_t)b;
    _Float16 h;
    __builtin_memcpy(&h, &u, 2);
    return (float)h;
}

template <int TYPE>
__device__ __forceinline__ float half_value(uint32_t b) {
    return TYPE == PB_BF16 ? bf16_value(b) : f16_value(b);
}

// Two values rounded to nearest, ties to even, as the halves of a word.
template <int TYPE>
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    uint32_t w;
    if (TYPE == PB_BF16) {
        const __bf16 h[2] = {(__bf16)lo, (__bf16)hi};
        __builtin_memcpy(&w, h, 4);
    } else {
        const _Float16 h[2] = {(_Float16)lo, (_Float16)hi};
        __builtin_memcpy(&w, h, 4);
    }
    return w;
}

template <int TYPE>
__device__ __forceinline__ float load_score(const void* p, int64_t i) {
    if (TYPE == PB_F32) return static_cast<const float*>(p)[i];
    return half_value<TYPE>(static_cast<const uint16_t*>(p)[i]);
}

template <int TYPE>
__device__ __forceinline__ void store_score(void* p, int64_t i, float v) {
    if (TYPE == PB_F32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<uint16_t*>(p)[i] = (uint16_t)half_pair<TYPE>(v, 0.0f);
}

// The rows of an item as its lanes count them: from row q0, a multiple of kRun, on; [lo, hi) are the
// item's, and all below `end` lie in the table.
struct Span {
    int64_t q0;
    int lo, hi, end;
};

__device__ __forceinline__ Span span_of(const ChoiceArgs& a, const SetItem& im) {
    Span s;
    s.q0 = im.row0 & ~(int64_t)(kRun - 1);
    s.lo = (int)(im.row0 - s.q0);
    s.hi = s.lo + im.rows;
    s.end = (int)min(a.rows - s.q0, (int64_t)1 << 30);
    return s;
}

// The rows of a lane's run from row i on that lie outside [lo, hi), a bit each.
__device__ __forceinline__ uint32_t outside(const Span& s, int i) {
    uint32_t b = 0;
    if (i < s.lo) b |= (1u << min(s.lo - i, kRun)) - 1u;
    if (i + kRun > s.hi) b |= 0xffu << max(s.hi - i, 0);
    return b & 0xffu;
}

// Whether a run goes in accesses of 16 bytes: the addresses are aligned (a.vec) and all its rows lie in the
// table. Else it goes row by row, in a rolled loop, within [lo, hi). That is what a table whose rows start off a
// 16-byte boundary, or whose scores have a stride, costs the whole call (us, aligned / one row off / stride 2: steps of
// 100k sets 28 / 44 / 52; policy of 480k sets 28 / 38 / 40; 4096 sets of 32000 bfloat16 scores 154 / 509 / 707; with a
// teacher of 8, 100k sets of 24 27 / 33 / 34 and the 4096 sets 112 / 404 / 433; their report without lists 57 / 203 / 297).
__device__ __forceinline__ bool whole_run(const ChoiceArgs& a, const Span& s, int i) { return a.vec && i + kRun <= s.end; }

__device__ __forceinline__ void put_row(float (&x)[kRun], int k, float v) {
#pragma unroll
    for (int j = 0; j < kRun; ++j) x[j] = j == k ? v : x[j];
}

// A run of the rows' gradients, 0 where `off` has a bit.
__device__ __forceinline__ void load_floats(const ChoiceArgs& a, const Span& s, int i, const float* p, uint32_t off,
                                            float (&x)[kRun]) {
    if (whole_run(a, s, i)) {
        const float4* v = reinterpret_cast<const float4*>(p + s.q0 + i);
        const float4 t = v[0], u = v[1];
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
        x[4] = u.x, x[5] = u.y, x[6] = u.z, x[7] = u.w;
    } else {
        const uint32_t out = outside(s, i);
#pragma unroll 1
        for (int k = 0; k < kRun; ++k)
            if (!(out >> k & 1u)) put_row(x, k, p[s.q0 + i + k]);
    }
    if (off) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) x[k] = off >> k & 1u ? 0.0f : x[k];
    }
}

// A run's values out, those in [lo, hi) alone.
template <int TYPE>
__device__ __forceinline__ void store_run(const ChoiceArgs& a, const Span& s, int i, void* p, const float (&x)[kRun]) {
    const uint32_t out = outside(s, i);
    if (a.vec && out == 0) {
        if (TYPE == PB_F32) {
            float4* v = reinterpret_cast<float4*>(static_cast<float*>(p) + s.q0 + i);
            v[0] = make_float4(x[0], x[1], x[2], x[3]);
            v[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + s.q0 + i) =
                make_uint4(half_pair<TYPE>(x[0], x[1]), half_pair<TYPE>(x[2], x[3]), half_pair<TYPE>(x[4], x[5]),
                           half_pair<TYPE>(x[6], x[7]));
        }
    } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
            if (!(out >> k & 1u)) store_score<TYPE>(p, s.q0 + i + k, x[k]);
    }
}

// The position bias in LDS: the table, and the lookup of its buckets where that is short.
struct BiasShared {
    float table[kMaxBuckets];
    uint8_t lookup[kLookup];
};

__device__ __forceinline__ uint32_t bucket_of(const ChoiceArgs& a, const BiasShared& b, int32_t q) {
    const uint32_t d = q < 0 ? 0u - (uint32_t)q : (uint32_t)q;
    const uint32_t i = min(d, (uint32_t)a.reach) + (q > 0 ? (uint32_t)a.reach + 1u : 0u);
    return a.reach < kLookup / 2 ? b.lookup[i] : min((uint32_t)a.buckets[i], (uint32_t)a.num_buckets - 1u);
}

__device__ __forceinline__ void stage_bias(const ChoiceArgs& a, BiasShared& b) {
    for (int i = (int)threadIdx.x; i < a.num_buckets; i += kBlock) b.table[i] = a.table[i];
    if (a.reach < kLookup / 2)
        for (int i = (int)threadIdx.x; i < 2 * (a.reach + 1); i += kBlock) b.lookup[i] = (uint8_t)min((int)a.buckets[i], a.num_buckets - 1);
    __syncthreads();
}

// Buckets of a run's rows, a byte each.
struct Buckets {
    uint32_t w[2];
    __device__ __forceinline__ int at(int k) const { return (int)(w[k >> 2] >> (8 * (k & 3)) & 0xffu); }
};

// A run as it lies in memory, asked for but not waited for; nothing where it goes row by row.
template <int TYPE, bool MASK, bool BIAS>
struct RawRun {
    uint4 score[TYPE == PB_F32 ? 2 : 1];
    uint2 mask;
    int4 pos[2];

    __device__ __forceinline__ void load(const ChoiceArgs& a, const Span& s, int i) {
        if (!whole_run(a, s, i)) return;
        if (TYPE == PB_F32) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(a.scores) + s.q0 + i);
            score[0] = p[0];
            score[TYPE == PB_F32 ? 1 : 0] = p[1];
        } else {
            score[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.scores) + s.q0 + i);
        }
        if (MASK) mask = *reinterpret_cast<const uint2*>(a.mask + s.q0 + i);
        if (BIAS) {
            const int4* p = reinterpret_cast<const int4*>(a.positions + s.q0 + i);
            pos[0] = p[0];
            pos[1] = p[1];
        }
    }

    // the logits: -inf where `off` has a bit, outside [lo, hi) and where masked
    __device__ __forceinline__ void logits(const ChoiceArgs& a, const BiasShared* bias, const Span& s, int i,
                                           float (&x)[kRun], uint32_t& off, Buckets& buckets) const {
        off = outside(s, i);
        buckets.w[0] = buckets.w[1] = 0;
        if (whole_run(a, s, i)) {
            const uint32_t w[8] = {score[0].x, score[0].y, score[0].z, score[0].w, score[TYPE == PB_F32 ? 1 : 0].x,
                                   score[TYPE == PB_F32 ? 1 : 0].y, score[TYPE == PB_F32 ? 1 : 0].z,
                                   score[TYPE == PB_F32 ? 1 : 0].w};
#pragma unroll
            for (int k = 0; k < kRun; ++k)
                x[k] = TYPE == PB_F32 ? __uint_as_float(w[k]) : half_value<TYPE>(k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu);
            if (MASK) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    off |= (mask.x >> (8 * k) & 0xffu) == 0 ? 1u << k : 0u;
                    off |= (mask.y >> (8 * k) & 0xffu) == 0 ? 16u << k : 0u;
                }
            }
            if (BIAS) {
                const int32_t q[kRun] = {pos[0].x, pos[0].y, pos[0].z, pos[0].w, pos[1].x, pos[1].y, pos[1].z, pos[1].w};
#pragma unroll
                for (int k = 0; k < kRun; ++k) {
                    const uint32_t b = bucket_of(a, *bias, q[k]);
                    buckets.w[k >> 2] |= b << (8 * (k & 3));
                    x[k] += bias->table[b];
                }
            }
        } else {
            const uint32_t out = off;
#pragma unroll 1
            for (int k = 0; k < kRun; ++k) {
                if (out >> k & 1u) continue;
                const int64_t row = s.q0 + i + k;
                float v = load_score<TYPE>(a.scores, row * a.stride);
                if (BIAS) {
                    const uint32_t b = bucket_of(a, *bias, a.positions[row]);
                    if (k < 4)
                        buckets.w[0] |= b << (8 * k);
                    else
                        buckets.w[1] |= b << (8 * (k - 4));
                    v += bias->table[b];
                }
                if (MASK && !a.mask[row]) off |= 1u << k;
                put_row(x, k, v);
            }
        }
        if (off) {
#pragma unroll
            for (int k = 0; k < kRun; ++k) x[k] = off >> k & 1u ? -kInf : x[k];
        }
    }
};

template <int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ void load_logits(const ChoiceArgs& a, const BiasShared* bias, const Span& s, int i,
                                            float (&x)[kRun], uint32_t& off, Buckets& buckets) {
    RawRun<TYPE, MASK, BIAS> raw;
    raw.load(a, s, i);
    raw.logits(a, bias, s, i, x, off, buckets);
}

// One logit.
template <int TYPE, bool BIAS>
__device__ __forceinline__ float one_logit(const ChoiceArgs& a, const BiasShared* bias, int64_t row) {
    float x = load_score<TYPE>(a.scores, row * a.stride);
    if (BIAS) x += bias->table[bucket_of(a, *bias, a.positions[row])];
    return x;
}

// LDS written by lanes of this wave is read by others of it: the wave's LDS accesses keep their order,
// the compiler must too.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {  // lanes without a source keep their own
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}

struct TakeMax {
    static constexpr float kNone = kLowest;
    static __device__ __forceinline__ float of(float a, float b) { return max2(a, b); }
};
struct TakeSum {
    static constexpr float kNone = 0.0f;
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};

// One step of a reduction by moves between lanes (CTRL of the rows in ROWS; the others take nothing).
template <class OP, int CTRL, int ROWS>
__device__ __forceinline__ float reduce_step(float v) {
    return OP::of(__int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(OP::kNone), __float_as_int(v), CTRL, ROWS, 0xf, false)), v);
}

// A wave's lanes, the result in all of them: within rows of 16 lanes, then between rows.
template <class OP>
__device__ __forceinline__ float wave_reduce(float v) {
    v = reduce_step<OP, 0x111, 0xf>(v);  // row_shr:1
    v = reduce_step<OP, 0x112, 0xf>(v);  // row_shr:2
    v = reduce_step<OP, 0x114, 0xf>(v);  // row_shr:4
    v = reduce_step<OP, 0x118, 0xf>(v);  // row_shr:8
    v = reduce_step<OP, 0x142, 0xa>(v);  // row_bcast:15
    v = reduce_step<OP, 0x143, 0xc>(v);  // row_bcast:31
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}

__device__ __forceinline__ float wave_max(float v) { return wave_reduce<TakeMax>(v); }
__device__ __forceinline__ float wave_sum(float v) { return wave_reduce<TakeSum>(v); }

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// v of another lane; CTRL as in lane_move
template <int CTRL>
__device__ __forceinline__ double lane_move(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp((int)b, (int)b, CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp((int)(b >> 32), (int)(b >> 32), CTRL, 0xf, 0xf, false);
    return __longlong_as_double((long long)hi << 32 | (uint32_t)lo);
}

template <class F>
__device__ F block_sum(F v, F* sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    F t = sh[0];
    for (int w = 1; w < kWaves; ++w) t += sh[w];
    return t;
}

// (maximum, sum of exponentials) of a set from those of its parts. A part without probability has sum 0
// and the lowest maximum.
struct Soft {
    float top, sum;
};

// The workgroup's from its waves' (every lane of a wave holds the wave's).
__device__ __forceinline__ Soft block_soft(Soft w, Soft* sh) {
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = w;
    __syncthreads();
    Soft t = sh[0];
    for (int i = 1; i < kWaves; ++i) t.top = fmaxf(t.top, sh[i].top);
    t.sum = 0.0f;
    for (int i = 0; i < kWaves; ++i) t.sum += sh[i].sum * exp_of(sh[i].top - t.top);
    return t;
}

// A wave's from its lanes' (one part each, or none).
__device__ __forceinline__ Soft wave_soft(Soft l) {
    Soft w;
    w.top = wave_max(l.top);
    w.sum = wave_sum(l.sum * exp_of(l.top - w.top));
    return w;
}

// A lane's from parts first, first + step, ... of a set.
__device__ __forceinline__ Soft join_parts(const float2* parts, int n, int first, int step) {
    Soft l{kLowest, 0.0f};
    for (int j = first; j < n; j += step) {
        const float2 p = parts[j];
        const float top = fmaxf(l.top, p.x);
        l.sum = l.sum * exp_of(l.top - top) + p.y * exp_of(p.x - top);
        l.top = top;
    }
    return l;
}

// Sums and maxima over runs of rows that may start and end in any lane of a wave: a bit in `heads` where
// a row starts a set, in `tails` where it ends one. A lane's value since its last head is carried on by a
// scan of the lanes that stops at heads: 4 steps in rows of 16 lanes, 2 between them.
struct Segments {
    uint32_t heads, tails;
    uint32_t steps;  // a bit for each step of the scan that stays within the lane's set

    // raw: the sets that start at the lane's rows, 0 for none. A set ends where the next one starts: rows
    // between them that are of no set hold what changes neither a maximum nor a sum.
    __device__ __forceinline__ void start(const int (&raw)[kRun], int lane) {
        heads = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) heads |= raw[k] ? 1u << k : 0u;
        const unsigned long long m = __ballot(heads != 0);
        const unsigned long long next = __ballot((heads & 1u) != 0) >> 1 | 1ull << (kWave - 1);
        tails = heads >> 1 | (uint32_t)(next >> lane & 1ull) << (kRun - 1);
        const unsigned long long below = m & (~0ull >> (kWave - 1 - lane));
        const int at = below ? kWave - 1 - __clzll((long long)below) : 0;  // the last lane up to this one with a head
        const int room = min(lane - at, lane & 15);  // lanes down to it, in the row of 16
        steps = (room >= 1 ? 1u : 0u) | (room >= 2 ? 2u : 0u) | (room >= 4 ? 4u : 0u) | (room >= 8 ? 8u : 0u) |
                ((lane & 16) != 0 && (lane & ~15) - 1 >= at ? 16u : 0u) | (lane >= 32 && 31 >= at ? 32u : 0u);
    }
};

// out[id[k] - 1] = the reduction of x over the set that row k ends. The lane's rows before its first head
// are of a set that began in a lane below. 24 vector instructions for the scan, 6 a row.
template <class OP>
__device__ __forceinline__ void segment_reduce(const Segments& seg, const float (&x)[kRun], const int (&id)[kRun],
                                               int lane, float* out) {
    float v = OP::of(OP::kNone, x[0]);
#pragma unroll
    for (int k = 1; k < kRun; ++k) v = OP::of(seg.heads >> k & 1u ? OP::kNone : v, x[k]);
    float t;
    t = lane_move<0x111>(v), v = (seg.steps & 1u) ? OP::of(t, v) : v;    // row_shr:1
    t = lane_move<0x112>(v), v = (seg.steps & 2u) ? OP::of(t, v) : v;    // row_shr:2
    t = lane_move<0x114>(v), v = (seg.steps & 4u) ? OP::of(t, v) : v;    // row_shr:4
    t = lane_move<0x118>(v), v = (seg.steps & 8u) ? OP::of(t, v) : v;    // row_shr:8
    t = lane_move<0x142>(v), v = (seg.steps & 16u) ? OP::of(t, v) : v;   // row_bcast:15
    t = lane_move<0x143>(v), v = (seg.steps & 32u) ? OP::of(t, v) : v;   // row_bcast:31
    t = __shfl_up(v, 1);
    v = lane > 0 ? t : OP::kNone;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        v = OP::of(seg.heads >> k & 1u ? OP::kNone : v, x[k]);
        if (seg.tails >> k & 1u) out[id[k] - 1] = v;
    }
}

// The table's gradient as a wave gathers it: bins of whole numbers, bin i's in units of 2^-shift[i], so that
// their sums do not depend on the order of the atomics. A bucket has copies of its bin, which keep lanes that
// meet in it apart. Each bin's own gradients set its unit, so that what other buckets hold takes no bits from
// it: a first one, and each one of 2^38 units or more, makes room for 16 times itself, and the bin is brought to
// the larger unit, to the nearest. A gradient is so rounded to 2^-34 or less of the largest in its bin (one unit
// for the whole wave lost a bucket's sum where another held gradients of 2^31 times its own; it took 27.2 us a call
// where this takes 28.2, for the policy loss of 480k sets). A wave's rows, at most about 2^24, stay below 2^62 units.
struct TableSum {
    static constexpr int kUnset = 300;             // above every unit's exponent: any gradient but 0 is too large
    static constexpr float kMost = 274877906944.0f;  // 2^38
    unsigned long long* bins;  // [kBins] of this wave: bucket b's from b << copy_bits on
    int* shift;                // [kBins]
    int* bad;                  // [num_buckets]: a gradient that is not finite
    int copy_bits;
    bool fresh;  // no gradient yet

    __device__ __forceinline__ void start(const ChoiceArgs& a, unsigned long long* b, int* shifts, int* flags) {
        bins = b;
        shift = shifts;
        bad = flags;
        fresh = true;
        copy_bits = 0;
        while ((a.num_buckets << (copy_bits + 1)) <= kBins && copy_bits < 5) ++copy_bits;
        for (int i = (int)threadIdx.x & (kWave - 1); i < kBins; i += kWave) {
            bins[i] = 0;
            shift[i] = kUnset;
        }
        wave_sync();
    }

    __device__ __forceinline__ int bin_of(int b) const {
        return (b << copy_bits) + ((int)threadIdx.x & ((1 << copy_bits) - 1));
    }

    // larger units for the bins of the rows in `over`; the whole wave. Which rows these are was decided with the
    // units before, so that the new ones are the same in any order.
    __device__ __forceinline__ void make_room(const float (&g)[kRun], const Buckets& buckets, uint32_t over) {
        const int lane = (int)threadIdx.x & (kWave - 1);
        int was[kBins / kWave];
        if (!fresh) {
#pragma unroll
            for (int j = 0; j < kBins / kWave; ++j) was[j] = shift[j * kWave + lane];
            wave_sync();
        }
        bool finite = true;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const bool in = fabsf(g[k]) < kInf;
            finite = finite && in;
            atomicMin(&shift[bin_of(buckets.at(k))], in && (over >> k & 1u) ? 34 - __builtin_amdgcn_frexp_expf(g[k]) : kUnset);
        }
        if (!finite) {
#pragma unroll
            for (int k = 0; k < kRun; ++k)
                if (!(fabsf(g[k]) < kInf)) bad[buckets.at(k)] = 1;
        }
        wave_sync();
        if (!fresh) {
#pragma unroll
            for (int j = 0; j < kBins / kWave; ++j) {
                const int i = j * kWave + lane, by = was[j] == kUnset ? 0 : was[j] - shift[i];
                if (by > 0) {
                    const long long t = (long long)bins[i];
                    bins[i] = by > 62 ? 0ull : (unsigned long long)((t + (1ll << (by - 1))) >> by);
                }
            }
            wave_sync();
        }
        fresh = false;
    }

    // ALL: zeros are added, too, without a branch a row. The policy's tiles take that (28.5 us a call for 480k sets, 28.7
    // else); the backward passes' keep the registers of five waves a SIMD without it (steps of 100k sets 48.2 us from
    // call to result, 50.8 else).
    template <bool ALL>
    __device__ __forceinline__ void add(const float (&g)[kRun], const Buckets& buckets) {
        float t[kRun];
        uint32_t over = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            t[k] = __builtin_amdgcn_ldexpf(g[k], fresh ? kUnset : shift[bin_of(buckets.at(k))]);
            over |= fabsf(t[k]) < kMost ? 0u : 1u << k;
        }
        if (__any(over != 0)) {
            make_room(g, buckets, over);
#pragma unroll
            for (int k = 0; k < kRun; ++k)
                t[k] = fabsf(g[k]) < kInf ? __builtin_amdgcn_ldexpf(g[k], shift[bin_of(buckets.at(k))]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            if (!ALL && t[k] == 0.0f) continue;
            // the nearest whole number: the low bits of t + 1.5 2^52
            const long long n = __double_as_longlong((double)t[k] + 6755399441055744.0) - 0x4338000000000000ll;
            atomicAdd(&bins[bin_of(buckets.at(k))], (unsigned long long)n);
        }
    }

    // The buckets' sums in the place of the bins, a double each; the whole wave. A bucket's slot lies at or before
    // its bins, all of which have been read.
    __device__ __forceinline__ void finish() {
        const int lane = (int)threadIdx.x & (kWave - 1);
        double v[kBins / kWave];
        wave_sync();
#pragma unroll
        for (int j = 0; j < kBins / kWave; ++j) {
            const int i = j * kWave + lane;
            v[j] = ldexp((double)(long long)bins[i], -shift[i]);
        }
        wave_sync();
#pragma unroll
        for (int j = 0; j < kBins / kWave; ++j) {  // lanes of one bucket, which hold the same after each step
            if (copy_bits > 0) v[j] += lane_move<0xb1>(v[j]);   // quad_perm:[1,0,3,2]
            if (copy_bits > 1) v[j] += lane_move<0x4e>(v[j]);   // quad_perm:[2,3,0,1]
            if (copy_bits > 2) v[j] += lane_move<0x141>(v[j]);  // row_half_mirror
            if (copy_bits > 3) v[j] += lane_move<0x140>(v[j]);  // row_mirror
            if (copy_bits > 4) v[j] += __shfl_xor(v[j], 16);
        }
        if ((lane & ((1 << copy_bits) - 1)) == 0)
#pragma unroll
            for (int j = 0; j < kBins / kWave; ++j)
                reinterpret_cast<double*>(bins)[(j * kWave + lane) >> copy_bits] = v[j];
        wave_sync();
    }
};

__device__ __forceinline__ void write_run(float* p, const float (&x)[kRun]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ void read_run(const float* p, float (&x)[kRun]) {
    const float4 t = reinterpret_cast<const float4*>(p)[0], u = reinterpret_cast<const float4*>(p)[1];
    x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    x[4] = u.x, x[5] = u.y, x[6] = u.z, x[7] = u.w;
}

// What a workgroup leaves behind of a loss's HEAD sums and the table's gradient: in its row of a.sums
// (workgroup `block` of the call's), or as the result where it is the only one.
template <int HEAD, bool TABLE>
__device__ __forceinline__ void leave_sums(const ChoiceArgs& a, int block, double (&tally)[3], TableSum& table,
                                           unsigned long long (*bins)[kBins], const int* bad, double* shd) {
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int cols = HEAD + (TABLE ? a.num_buckets : 0);
    double* mine = a.sums + (int64_t)block * cols;
    if (HEAD > 0) {
#pragma unroll
        for (int m = kWave / 2; m >= 1; m >>= 1)
#pragma unroll
            for (int j = 0; j < HEAD; ++j) tally[j] += __shfl_xor(tally[j], m);
        if (lane == 0)
#pragma unroll
            for (int j = 0; j < HEAD; ++j) shd[wave * HEAD + j] = tally[j];
        __syncthreads();
        if (tid < HEAD) {
            double t = shd[tid];
            for (int w = 1; w < kWaves; ++w) t += shd[w * HEAD + tid];
            if (a.blocks == 1)
                a.stats[tid] = (float)t;
            else
                mine[tid] = t;
        }
    }
    if (TABLE) {
        table.finish();
        __syncthreads();
        for (int b = tid; b < a.num_buckets; b += kBlock) {
            double t = 0.0;
            for (int w = 0; w < kWaves; ++w) t += reinterpret_cast<const double*>(bins[w])[b];
            if (bad[b]) t = __longlong_as_double(0x7ff8000000000000ll);
            if (a.blocks == 1)
                a.grad_table[b] = (float)t;
            else
                mine[HEAD + b] = t;
        }
    }
}

// ---- probabilities at a temperature T: p_i = exp((z_i - m) / T) / s
// log2(e) / T as the sum of two floats, and the distance to the maximum from which on exponentials are 0.
struct Heat {
    float hi, lo, low;
};

// exp(d / T) of d = z - m, within 2 units. -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float heat_exp(float distance, const Heat& h) {
    const float d = __builtin_elementwise_maximum(distance, h.low);  // a NaN is the larger one
    const float t = d * h.hi, e = __builtin_amdgcn_exp2f(t);
    const float rest = __builtin_fmaf(d, h.lo, __builtin_fmaf(d, h.hi, -t));
    return __builtin_fmaf(e * 0.693147182464599609375f, rest, e);
}

// The same for rows that share a maximum m, with less care (EXACT false): 2 to z hi - c, c = m hi rounded, in one operation
// whose rounding moves the result by at most |d / T| 2^-24 of itself in either direction, and T counts as rounded to 2^-25.
// What c's rounding adds to every exponent (`shift`, at most 2^-25 |m hi|) is taken back from the sums.
// Where |m hi| is 2^31 and more, the next lower logit is 2^7 below m in the exponent and counts as nothing: there a power of
// two in hi's place, which takes m to 2^63 or 2^64, leaves m's rows 0 and takes all others far below.
template <bool EXACT>
struct HeatRows {
    float m, hi, c, shift;
    __device__ __forceinline__ HeatRows(float top, const Heat& h) : m(top), hi(h.hi), c(0.0f), shift(0.0f) {
        if (EXACT) return;
        const bool far = !(__builtin_fabsf(top * h.hi) < 0x1p31f);
        if (far) hi = __builtin_amdgcn_ldexpf(1.0f, 64 - __builtin_amdgcn_frexp_expf(top));
        c = top * hi;
        shift = far ? 0.0f : __builtin_fmaf(top, hi, -c);
    }
    // (z - m) / T in units of its own: bounded below, so that a product with the exponential is 0 where that is
    __device__ __forceinline__ float distance(float z, const Heat& h) const {
        return EXACT ? __builtin_elementwise_maximum(z - m, h.low)
                     : __builtin_elementwise_maximum(__builtin_fmaf(z, hi, -c), -200.0f);
    }
    __device__ __forceinline__ float exp(float distance, const Heat& h) const {
        return EXACT ? heat_exp(distance, h) : __builtin_amdgcn_exp2f(distance);
    }
    // what exponentials are multiplied by, and (the distances less the shift) to be in units of z
    __device__ __forceinline__ float scale() const { return EXACT ? 1.0f : __builtin_amdgcn_exp2f(-shift); }
    static __device__ __forceinline__ double unit(const Heat& h) { return EXACT ? 1.0 : 1.0 / (double)h.hi; }
};

// e^x in double within 2^-34 of itself: x = k log 2 + r, |r| <= log(2) / 2, and ten terms of r's series, those from
// r^4 / 24 on in float. -inf gives 0, NaN and infinity give NaN.
__device__ __forceinline__ double exp_near(double x) {
    x = x < -800.0 ? -800.0 : x;
    const float k = __builtin_rintf((float)x * 1.44269504f);
    const double r = __builtin_fma((double)k, -0.69314718055994531, x);
    const float f = (float)r;
    float p = 1.0f / 3628800;
    p = __builtin_fmaf(p, f, 1.0f / 362880);
    p = __builtin_fmaf(p, f, 1.0f / 40320);
    p = __builtin_fmaf(p, f, 1.0f / 5040);
    p = __builtin_fmaf(p, f, 1.0f / 720);
    p = __builtin_fmaf(p, f, 1.0f / 120);
    p = __builtin_fmaf(p, f, 1.0f / 24);
    double d = __builtin_fma((double)p, r, 1.0 / 6);
    d = __builtin_fma(d, r, 0.5);
    d = __builtin_fma(d, r, 1.0);
    return ldexp(__builtin_fma(d, r, 1.0), (int)k);
}

// log x in double within 2^-31 beside its rounding, and as close relative to itself near 1: x = 2^k m, m in [2/3, 4/3),
// log m = 2 (f + f^3 / 3 + ... + f^13 / 13), f = (m - 1) / (m + 1), the terms after the first in float. 0 gives -inf.
__device__ __forceinline__ double log_near(double x) {
    if (!(x > 0.0 && x < (double)kInf)) return (double)log_of((float)x);
    const double half = __builtin_amdgcn_frexp_mant(x);  // [1/2, 1)
    const bool low = (float)half < 0.6666667f;
    const double m = low ? 2.0 * half : half;
    const int k = __builtin_amdgcn_frexp_exp(x) - (low ? 1 : 0);
    const double n = m - 1.0, s = m + 1.0, inv = (double)__builtin_amdgcn_rcpf((float)s);
    const double f0 = n * inv, f = __builtin_fma(__builtin_fma(-f0, s, n), inv, f0);
    const float g = (float)f, q = g * g;
    float p = 1.0f / 13;
    p = __builtin_fmaf(p, q, 1.0f / 11);
    p = __builtin_fmaf(p, q, 1.0f / 9);
    p = __builtin_fmaf(p, q, 1.0f / 7);
    p = __builtin_fmaf(p, q, 1.0f / 5);
    p = __builtin_fmaf(p, q, 1.0f / 3);
    return __builtin_fma((double)k, 0.69314718055994531, 2.0 * (f + (double)(p * q * g)));
}

// Reductions over teams of 1 << bits neighbouring lanes of a wave, the result in all of them. Lanes that mirror each
// other hold the same after the steps before.
template <class F>
__device__ __forceinline__ double team_reduce(double v, int bits, F f) {
    if (bits > 0) v = f(v, lane_move<0xb1>(v));   // quad_perm:[1,0,3,2]
    if (bits > 1) v = f(v, lane_move<0x4e>(v));   // quad_perm:[2,3,0,1]
    if (bits > 2) v = f(v, lane_move<0x141>(v));  // row_half_mirror
    if (bits > 3) v = f(v, lane_move<0x140>(v));  // row_mirror
    if (bits > 4) v = f(v, __shfl_xor(v, 16));
    if (bits > 5) v = f(v, __shfl_xor(v, 32));
    return v;
}

__device__ __forceinline__ double team_sum(double v, int bits) {
    return team_reduce(v, bits, [](double a, double b) { return a + b; });
}

__device__ __forceinline__ double team_max(double v, int bits) {
    return team_reduce(v, bits, [](double a, double b) { return fmax(a, b); });
}

// What a wave reads of a tile of short sets, asked for before anything is waited for: a lane's run, and where the lane's
// sets lie.
template <int TYPE, bool MASK, bool BIAS>
struct TileRows {
    Span sp;  // of the lane's run alone
    int sets;
    RawRun<TYPE, MASK, BIAS> raw;
    int32_t set[kTileRounds], begin[kTileRounds], end[kTileRounds];  // begin, end: rows of the tile

    __device__ __forceinline__ void load(const ChoiceArgs& a, const SetItem& im, int lane) {
        int64_t row0 = im.row0, rows = im.rows;
        int lane0 = 0;
        int64_t base[kTileRounds];
        sets = im.sets;
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            set[r] = im.set0 + r * kWave + lane;
            base[r] = row0 & ~(int64_t)(kRun - 1);
        }
        for (int e = 0; e < im.parts; ++e) {  // the tile's further segments
            const TileSegment seg = a.segments[im.part + e];
            if (lane >= seg.lane0) {
                row0 = seg.row0;
                rows = seg.rows;
                lane0 = seg.lane0;
            }
#pragma unroll
            for (int r = 0; r < kTileRounds; ++r)
                if (r * kWave + lane >= seg.first) {
                    set[r] = seg.set0 + r * kWave + lane - seg.first;
                    base[r] = (seg.row0 & ~(int64_t)(kRun - 1)) - kRun * seg.lane0;
                }
        }
        sp.q0 = (row0 & ~(int64_t)(kRun - 1)) + kRun * (lane - lane0);
        sp.lo = (int)max(row0 - sp.q0, (int64_t)0);  // below kRun
        sp.hi = (int)min(row0 + rows - sp.q0, (int64_t)kRun);
        sp.end = (int)min(a.rows - sp.q0, (int64_t)kRun);
        if (sp.hi > 0) raw.load(a, sp, 0);
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            begin[r] = end[r] = 0;
            if (r * kWave + lane < sets) {
                begin[r] = (int)(a.off[set[r]] - base[r]);
                end[r] = (int)(a.off[set[r] + 1] - base[r]);
            }
        }
    }
};

// The sets of a tile's rows, and how they are reduced. `head` has the set that starts at a row, from 1, 0 for none.
struct TileSets {
    int id[kRun];  // the row's set, from 1; a slot of none before the first
    Segments seg;

    __device__ __forceinline__ void find(const uint16_t* head, int lane) {
        const uint4 w = *reinterpret_cast<const uint4*>(&head[kRun * lane]);
        const int raw[kRun] = {(int)(w.x & 0xffffu), (int)(w.x >> 16), (int)(w.y & 0xffffu), (int)(w.y >> 16),
                               (int)(w.z & 0xffffu), (int)(w.z >> 16), (int)(w.w & 0xffffu), (int)(w.w >> 16)};
        int last = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) last = raw[k] ? raw[k] : last;
        // the set that the rows before the lane's first head are of: the last head's below
        const unsigned long long below = __ballot(last != 0) & ((1ull << lane) - 1ull);
        const int from = below ? kWave - 1 - __clzll((long long)below) : lane;
        const int carried = __shfl(last, from);
        int now = below ? carried : kSetTileSets + 1;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            now = raw[k] ? raw[k] : now;
            id[k] = now;
        }
        seg.start(raw, lane);
    }
};

}  // namespace
}  // namespace pb
