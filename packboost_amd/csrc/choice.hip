// Learning from choices over ragged sets of candidate rows: grouped log-probabilities with a learned
// position bias, their backward, the clipped policy loss, and the sums of the preference loss.
//
// Set g holds rows [off[g], off[g + 1]). Row i's logit is x_i = score_i + table[bucket(position_i)],
// -inf where its mask is 0. With m = max x (0 where that is -inf) and s = sum exp(x - m) over the set,
// lse = m + log s and log p_i = (x_i - m) - log s; a set without probability (empty, all masked) has
// s = 0 and lse = -inf. The gradient of a step's log p_c is [i = c] - p_i, of all rows' d_i - p_i sum d.
//
// Work is laid out once per table of sets (set_items): a workgroup takes an item at a time, either a
// tile of consecutive short sets, staged in LDS and reduced by teams of lanes, or one long set or a
// part of it, kept in registers. Parts of a set are reduced by an extra pass (part_kernel) before.
// Every sum has a fixed order (teams, workgroups, then items), so results do not change from run to
// run. Maxima, sums of exponentials and log-probabilities are float32; losses and the table's gradient
// are joined in double, each rounded once when it is written.
#include "pb_internal.h"

namespace pb {
namespace {

constexpr int kPer = kSetTileRows / kBlock;  // rows per thread
constexpr int kWaves = kBlock / kWave;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kBins = 1024;  // LDS words of the table's gradient: buckets x copies

__device__ __forceinline__ float bf16_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

__device__ __forceinline__ uint16_t bf16_bits(float f) {  // to nearest, ties to even; NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

template <int TYPE>
__device__ __forceinline__ float load_score(const void* p, int64_t i) {
    if (TYPE == PB_BF16) return bf16_value(static_cast<const uint16_t*>(p)[i]);
    if (TYPE == PB_F16) return (float)static_cast<const _Float16*>(p)[i];
    return static_cast<const float*>(p)[i];
}

template <int TYPE>
__device__ __forceinline__ void store_score(void* p, int64_t i, float v) {
    if (TYPE == PB_BF16)
        static_cast<uint16_t*>(p)[i] = bf16_bits(v);
    else if (TYPE == PB_F16)
        static_cast<_Float16*>(p)[i] = (_Float16)v;
    else
        static_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ int bucket_of(const ChoiceArgs& a, int64_t row) {
    const int32_t q = a.positions[row];
    const uint32_t d = q < 0 ? 0u - (uint32_t)q : (uint32_t)q;
    return a.buckets[min(d, (uint32_t)a.reach) + (q > 0 ? (uint32_t)a.reach + 1u : 0u)];
}

template <int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ float load_logit(const ChoiceArgs& a, int64_t row) {
    float x = load_score<TYPE>(a.scores, row * a.stride);
    if (BIAS) x += a.table[bucket_of(a, row)];
    if (MASK && !a.mask[row]) x = kNegInf;
    return x;
}

__device__ __forceinline__ float nan_max(float a, float b) { return b > a ? b : a; }  // a NaN b is passed over

__device__ float block_max(float v, float* sh) {
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) v = nan_max(v, __shfl_xor(v, m));
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    float t = sh[0];
    for (int w = 1; w < kWaves; ++w) t = nan_max(t, sh[w]);
    return t;
}

template <class F>
__device__ F block_sum(F v, F* sh) {
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    F t = sh[0];
    for (int w = 1; w < kWaves; ++w) t += sh[w];
    return t;
}

// What a step's log-probability gives and takes.
struct Step {
    bool counts;  // the chosen row lies in the set, is on offer, and the set has probability
    float lp;
    float coef;   // gradient of the loss with respect to lp
};

// Where the step's choice lies: the row in the set, or -1 for a step that is left out.
template <bool MASK>
__device__ __forceinline__ int64_t chosen_row(const ChoiceArgs& a, int64_t g, int64_t r0, int64_t size) {
    const int32_t c = a.chosen[g];
    if (c < 0 || c >= size) return -1;
    if (MASK && !a.mask[r0 + c]) return -1;
    return c;
}

// The clipped loss of a step and its slope: surrogate min(rA, clip(r) A) with r = exp(lp - old), and
// kl = e^d - d - 1 with d = ref - lp. A NaN ratio takes no bound, so it stays visible.
__device__ __forceinline__ void policy_step(const ChoiceArgs& a, int64_t g, Step& st, bool tally, double (&sum)[3]) {
    const float w = (a.weights ? a.weights[g] : 1.0f) * a.scale;
    const float adv = a.advantages[g];
    const float ratio = expf(st.lp - a.old[g]);
    const float free = ratio * adv;
    const float held = fminf(fmaxf(ratio, a.ratio_min), a.ratio_max) * adv;
    const bool clipped = free > held;
    float kl = 0.0f, slope = clipped ? 0.0f : -free;
    if (a.ref) {
        const float d = a.ref[g] - st.lp;
        const float e = expf(d);
        kl = e - d - 1.0f;
        slope += a.kl_weight * (1.0f - e);
    }
    st.coef = w * slope;
    if (tally) {
        sum[0] += (double)(w * (a.kl_weight * kl - (clipped ? held : free)));
        sum[1] += (double)(w * kl);
        sum[2] += clipped ? (double)w : 0.0;
    }
}

// The maximum and the sum of exponentials of a part of a set, or (listwise backward) the sum of its
// rows' gradients.
template <int MODE, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void part_kernel(ChoiceArgs a, const int32_t* __restrict__ list) {
    __shared__ float sh[kWaves];
    const int32_t it = list[blockIdx.x];
    const SetItem im = a.items[it];
    float v[kPer], top = kNegInf, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = k * kBlock + (int)threadIdx.x;
        const int64_t row = im.row0 + i;
        if (MODE == kRowsBack) {
            if (i < im.rows && (!MASK || a.mask[row])) sum += a.grad[row];
        } else {
            v[k] = i < im.rows ? load_logit<TYPE, MASK, BIAS>(a, row) : kNegInf;
            top = nan_max(top, v[k]);
        }
    }
    if (MODE != kRowsBack) {
        top = block_max(top, sh);
        if (top == kNegInf) top = 0.0f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) sum += expf(v[k] - top);
    }
    sum = block_sum(sum, sh);
    if (threadIdx.x == 0) a.parts[it] = make_float2(top, sum);
}

// One item at a time per workgroup; see the head of the file.
template <int MODE, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void choice_kernel(ChoiceArgs a) {
    constexpr bool GRAD = MODE == kRowsBack || MODE == kStepsBack || MODE == kPolicy;
    constexpr bool STEPS = MODE != kRows && MODE != kRowsBack;
    constexpr bool TABLE = BIAS && GRAD;
    __shared__ float xs[kSetTileRows];
    __shared__ float dsum[MODE == kRowsBack ? kSetTileRows : 1];
    __shared__ float shf[kWaves];
    __shared__ double shd[kWaves];
    __shared__ unsigned long long bins[TABLE ? kBins : 1];
    __shared__ double table_sum[TABLE ? kMaxBuckets : 1];
    __shared__ int table_nan[TABLE ? kMaxBuckets : 1];
    const int tid = (int)threadIdx.x;
    // copies of the table's bins, so that lanes that meet in a bucket rarely meet in a word
    int copies = 1;
    if (TABLE) {
        while (copies < 32 && copies * 2 * a.num_buckets <= kBins) copies *= 2;
        for (int i = tid; i < copies * a.num_buckets; i += kBlock) bins[i] = 0;
        for (int b = tid; b < a.num_buckets; b += kBlock) {
            table_sum[b] = 0.0;
            table_nan[b] = 0;
        }
    }
    double tally[3] = {0.0, 0.0, 0.0};
    for (int it = (int)blockIdx.x; it < a.num_items; it += (int)gridDim.x) {
        const SetItem im = a.items[it];
        float v[kPer];
        uint32_t hidden = 0;
        int bucket[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int i = k * kBlock + tid;
            v[k] = kNegInf;
            bucket[k] = 0;
            if (i < im.rows) {
                const int64_t row = im.row0 + i;
                float x = load_score<TYPE>(a.scores, row * a.stride);
                if (BIAS) {
                    bucket[k] = bucket_of(a, row);
                    x += a.table[bucket[k]];
                }
                if (MASK && !a.mask[row]) {
                    x = kNegInf;
                    hidden |= 1u << k;
                }
                v[k] = x;
            }
        }
        if (im.parts == 0) {
            __syncthreads();  // the last item's tile has been read
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                if (i < im.rows) {
                    xs[i] = v[k];
                    if (MODE == kRowsBack) dsum[i] = (hidden >> k) & 1u ? 0.0f : a.grad[im.row0 + i];
                }
            }
            __syncthreads();
            const int L = 1 << im.team, lane = tid & (L - 1);
            for (int s = tid >> im.team; s < im.sets; s += kBlock >> im.team) {
                const int64_t g = (int64_t)im.set0 + s;
                const int64_t r0 = a.off[g];
                const int b = (int)(r0 - im.row0), e = (int)(a.off[g + 1] - im.row0);
                float top = 0.0f, sum = 0.0f, lse = 0.0f;
                if (MODE == kRows || MODE == kSteps || MODE == kPolicy) {
                    top = kNegInf;
                    for (int i = b + lane; i < e; i += L) top = nan_max(top, xs[i]);
                    for (int m = 1; m < L; m <<= 1) top = nan_max(top, __shfl_xor(top, m));
                    if (top == kNegInf) top = 0.0f;
                    for (int i = b + lane; i < e; i += L) sum += expf(xs[i] - top);
                    for (int m = 1; m < L; m <<= 1) sum += __shfl_xor(sum, m);
                    lse = top + logf(sum);
                    if (lane == 0 && MODE != kPolicy) a.lse_out[g] = lse;
                } else {
                    lse = a.lse[g];
                }
                if (MODE == kRows) {
                    const float ls = logf(sum);
                    for (int i = b + lane; i < e; i += L) xs[i] = xs[i] == kNegInf ? kNegInf : (xs[i] - top) - ls;
                }
                if (MODE == kRowsBack) {
                    float d = 0.0f;
                    for (int i = b + lane; i < e; i += L) d += dsum[i];
                    for (int m = 1; m < L; m <<= 1) d += __shfl_xor(d, m);
                    for (int i = b + lane; i < e; i += L)
                        xs[i] = dsum[i] - (xs[i] == kNegInf ? 0.0f : expf(xs[i] - lse) * d);
                }
                if (STEPS) {
                    const int64_t c = chosen_row<MASK>(a, g, r0, e - b);
                    Step st;
                    st.counts = c >= 0 && (MODE == kStepsBack ? lse != kNegInf : sum != 0.0f);
                    st.lp = st.counts && MODE != kStepsBack ? (xs[b + c] - top) - logf(sum) : 0.0f;
                    st.coef = 0.0f;
                    if (MODE == kStepsBack && st.counts) st.coef = a.grad[g];
                    if (MODE == kPolicy && st.counts) policy_step(a, g, st, lane == 0, tally);
                    if (MODE != kStepsBack && lane == 0) a.log_probs[g] = st.lp;
                    if (GRAD) {
                        const float shift = MODE == kStepsBack ? lse : top;
                        const float f = MODE == kStepsBack ? st.coef : st.coef / sum;
                        for (int i = b + lane; i < e; i += L) {
                            const float p = xs[i] == kNegInf ? 0.0f : expf(xs[i] - shift);
                            xs[i] = st.counts ? (i - b == c ? st.coef : 0.0f) - f * p : 0.0f;
                        }
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                if (i < im.rows) v[k] = xs[i];
            }
        } else {
            const int64_t g = im.set0;
            const int64_t r0 = a.off[g], size = a.off[g + 1] - r0;
            float top = 0.0f, sum = 0.0f, lse = 0.0f, d = 0.0f, dv[kPer];
            if (MODE == kRowsBack) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const int i = k * kBlock + tid;
                    dv[k] = i < im.rows && !((hidden >> k) & 1u) ? a.grad[im.row0 + i] : 0.0f;
                }
            }
            if (MODE == kStepsBack) {
                lse = a.lse[g];
            } else if (im.parts > 1) {
                const float2* parts = a.parts + (it - im.part);
                top = kNegInf;
                for (int j = tid; j < im.parts; j += kBlock) top = nan_max(top, parts[j].y != 0.0f ? parts[j].x : kNegInf);
                top = block_max(top, shf);
                if (top == kNegInf) top = 0.0f;
                for (int j = tid; j < im.parts; j += kBlock)
                    sum += MODE == kRowsBack ? parts[j].y : parts[j].y != 0.0f ? parts[j].y * expf(parts[j].x - top) : 0.0f;
                sum = block_sum(sum, shf);
                if (MODE == kRowsBack) d = sum;
            } else if (MODE == kRowsBack) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) d += dv[k];
                d = block_sum(d, shf);
            } else {
                top = kNegInf;
#pragma unroll
                for (int k = 0; k < kPer; ++k) top = nan_max(top, v[k]);
                top = block_max(top, shf);
                if (top == kNegInf) top = 0.0f;
#pragma unroll
                for (int k = 0; k < kPer; ++k) sum += expf(v[k] - top);
                sum = block_sum(sum, shf);
            }
            const bool first = im.part == 0 && tid == 0;
            if (MODE == kRowsBack) {
                lse = a.lse[g];
#pragma unroll
                for (int k = 0; k < kPer; ++k) v[k] = dv[k] - (v[k] == kNegInf ? 0.0f : expf(v[k] - lse) * d);
            }
            const float ls = logf(sum);
            if ((MODE == kRows || MODE == kSteps) && first) a.lse_out[g] = top + ls;
            if (MODE == kRows) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) v[k] = v[k] == kNegInf ? kNegInf : (v[k] - top) - ls;
            }
            if (STEPS) {
                const int64_t c = chosen_row<MASK>(a, g, r0, size);
                Step st;
                st.counts = c >= 0 && (MODE == kStepsBack ? lse != kNegInf : sum != 0.0f);
                st.lp = st.counts && MODE != kStepsBack ? (load_logit<TYPE, MASK, BIAS>(a, r0 + c) - top) - ls : 0.0f;
                st.coef = 0.0f;
                if (MODE == kStepsBack && st.counts) st.coef = a.grad[g];
                if (MODE == kPolicy && st.counts) policy_step(a, g, st, first, tally);
                if (MODE != kStepsBack && first) a.log_probs[g] = st.lp;
                if (GRAD) {
                    const float shift = MODE == kStepsBack ? lse : top;
                    const float f = MODE == kStepsBack ? st.coef : st.coef / sum;
                    const int64_t at = r0 + c - im.row0;  // the chosen row, as this part counts
#pragma unroll
                    for (int k = 0; k < kPer; ++k) {
                        const float p = v[k] == kNegInf ? 0.0f : expf(v[k] - shift);
                        v[k] = st.counts ? (k * kBlock + tid == at ? st.coef : 0.0f) - f * p : 0.0f;
                    }
                }
            }
        }
        if (MODE == kRows) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                if (i < im.rows) a.log_probs[im.row0 + i] = v[k];
            }
        }
        if (GRAD) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                if ((hidden >> k) & 1u) v[k] = 0.0f;
                if (i < im.rows) store_score<TYPE>(a.grad_scores, im.row0 + i, v[k]);
            }
        }
        if (TABLE) {
            // The item's gradients as whole numbers of 2^(e - 30), 2^e above the largest of them: their
            // sums do not depend on the order of the atomics, and what the rounding takes is below
            // 2^-31 of the largest a row. Gradients that are not finite make their bucket NaN.
            float big = 0.0f;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                const float m = fabsf(v[k]);
                if (i < im.rows && m < __builtin_huge_valf()) big = fmaxf(big, m);
            }
            big = block_max(big, shf);
            int e = 0;
            (void)frexpf(big, &e);
            const int own_copy = tid & (copies - 1);
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = k * kBlock + tid;
                if (i < im.rows && v[k] != 0.0f) {
                    if (fabsf(v[k]) < __builtin_huge_valf())
                        atomicAdd(&bins[bucket[k] * copies + own_copy],
                                  (unsigned long long)(long long)__float2int_rn(ldexpf(v[k], 30 - e)));
                    else
                        table_nan[bucket[k]] = 1;
                }
            }
            __syncthreads();
            for (int b = tid; b < a.num_buckets; b += kBlock) {
                long long t = 0;
                for (int c = 0; c < copies; ++c) {
                    t += (long long)bins[b * copies + c];
                    bins[b * copies + c] = 0;
                }
                table_sum[b] += ldexp((double)t, e - 30);
            }
            __syncthreads();
        }
    }
    const int cols = (MODE == kPolicy ? 3 : 0) + (TABLE ? a.num_buckets : 0);
    double* mine = a.sums + (int64_t)blockIdx.x * cols;
    if (MODE == kPolicy) {
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const double t = block_sum(tally[j], shd);
            if (tid == 0) {
                if (gridDim.x == 1)
                    a.stats[j] = (float)t;
                else
                    mine[j] = t;
            }
        }
    }
    if (TABLE) {
        for (int b = tid; b < a.num_buckets; b += kBlock) {
            const double t = table_nan[b] ? __longlong_as_double(0x7ff8000000000000ll) : table_sum[b];
            if (gridDim.x == 1)
                a.grad_table[b] = (float)t;
            else
                mine[(MODE == kPolicy ? 3 : 0) + b] = t;
        }
    }
}

// out[j] = sum over the workgroups' sums [n][cols] of column j, in a fixed order; the first `head`
// columns go to stats, the others to the table's gradient.
__global__ __launch_bounds__(kBlock) void join_kernel(const double* __restrict__ sums, int32_t n, int32_t cols,
                                                      int32_t head, float* __restrict__ stats,
                                                      float* __restrict__ table) {
    __shared__ double sh[kWaves];
    const int j = (int)blockIdx.x;
    double t = 0.0;
    for (int i = (int)threadIdx.x; i < n; i += kBlock) t += sums[(int64_t)i * cols + j];
    t = block_sum(t, sh);
    if (threadIdx.x == 0) (j < head ? stats[j] : table[j - head]) = (float)t;
}

// ------------------------------------------------------------------------------ preferences
// Sums over sets in double: of (value - ref) over a sequence's steps, or of the signed slopes of the
// pairs that a value is in (list entry: pair * 2 + (1 where it is the loser)).
struct SumArgs {
    const int64_t* off;
    const SetItem* items;
    int32_t num_items;
    const float* values;
    const float* ref;
    const int32_t* entries;
    const float* slopes;
    float* out;
    double* parts;
};

template <bool PAIRS>
__device__ __forceinline__ double sum_term(const SumArgs& a, int64_t i) {
    if (PAIRS) {
        const int32_t e = a.entries[i];
        const float c = a.slopes[e >> 1];
        return (double)(e & 1 ? -c : c);
    }
    return (double)a.values[i] - (a.ref ? (double)a.ref[i] : 0.0);
}

template <bool PAIRS>
__global__ __launch_bounds__(kBlock) void set_sum_kernel(SumArgs a) {
    __shared__ double xs[kSetTileRows];
    __shared__ double sh[kWaves];
    const int tid = (int)threadIdx.x;
    const SetItem im = a.items[blockIdx.x];
    if (im.parts == 0) {
        for (int i = tid; i < im.rows; i += kBlock) xs[i] = sum_term<PAIRS>(a, im.row0 + i);
        __syncthreads();
        const int L = 1 << im.team, lane = tid & (L - 1);
        for (int s = tid >> im.team; s < im.sets; s += kBlock >> im.team) {
            const int64_t g = (int64_t)im.set0 + s;
            const int b = (int)(a.off[g] - im.row0), e = (int)(a.off[g + 1] - im.row0);
            double t = 0.0;
            for (int i = b + lane; i < e; i += L) t += xs[i];
            for (int m = 1; m < L; m <<= 1) t += __shfl_xor(t, m);
            if (lane == 0) a.out[g] = (float)t;
        }
    } else {
        double t = 0.0;
        for (int i = tid; i < im.rows; i += kBlock) t += sum_term<PAIRS>(a, im.row0 + i);
        t = block_sum(t, sh);
        if (tid == 0) {
            if (im.parts == 1)
                a.out[im.set0] = (float)t;
            else
                a.parts[blockIdx.x] = t;
        }
    }
}

// The sets that were summed in parts.
__global__ __launch_bounds__(kBlock) void set_join_kernel(SumArgs a, const int32_t* __restrict__ list, int32_t n) {
    __shared__ double sh[kWaves];
    const int32_t it = list[blockIdx.x];
    const SetItem im = a.items[it];
    if (im.part != 0) return;  // the whole workgroup
    double t = 0.0;
    for (int j = (int)threadIdx.x; j < im.parts; j += kBlock) t += a.parts[it + j];
    t = block_sum(t, sh);
    if (threadIdx.x == 0) a.out[im.set0] = (float)t;
}

// z = beta (a_w - a_l); the loss w [(1 - e) softplus(-z) + e softplus(z)] and its slope
// beta w (sigmoid(z) - (1 - e)). Sequences' values come from their sums, others' as value - ref, the
// differences taken in double: both can be large where z is small.
__global__ __launch_bounds__(kBlock) void pair_kernel(PairArgs a) {
    __shared__ double sh[kWaves];
    double sum = 0.0;
    for (int64_t p = (int64_t)blockIdx.x * kBlock + threadIdx.x; p < a.num_pairs; p += (int64_t)gridDim.x * kBlock) {
        const int32_t w = a.winners[p], l = a.losers[p];
        double d = (double)a.values[w] - (double)a.values[l];
        if (a.ref) d -= (double)a.ref[w] - (double)a.ref[l];
        const float z = (float)((double)a.beta * d);
        const float weight = (a.weights ? a.weights[p] : 1.0f) * a.scale;
        const float t = expf(-fabsf(z)), soft = log1pf(t);
        const float e = a.smoothing;
        const float up = z > 0.0f ? 1.0f / (1.0f + t) : t / (1.0f + t);    // sigmoid(z)
        const float down = z > 0.0f ? t / (1.0f + t) : 1.0f / (1.0f + t);  // sigmoid(-z)
        a.margins[p] = z;
        a.slopes[p] = a.beta * weight * (e * up - (1.0f - e) * down);
        sum += (double)(weight * ((1.0f - e) * (soft + fmaxf(-z, 0.0f)) + e * (soft + fmaxf(z, 0.0f))));
    }
    sum = block_sum(sum, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            a.loss[0] = (float)sum;
        else
            a.sums[blockIdx.x] = sum;
    }
}

// out[i] = per_set[set of i]
__global__ __launch_bounds__(kBlock) void spread_kernel(const int64_t* __restrict__ off, const SetItem* __restrict__ items,
                                                        const float* __restrict__ per_set, float* __restrict__ out) {
    const int tid = (int)threadIdx.x;
    const SetItem im = items[blockIdx.x];
    if (im.parts == 0) {
        const int L = 1 << im.team, lane = tid & (L - 1);
        for (int s = tid >> im.team; s < im.sets; s += kBlock >> im.team) {
            const int64_t g = (int64_t)im.set0 + s;
            const float v = per_set[g];
            for (int64_t i = off[g] + lane; i < off[g + 1]; i += L) out[i] = v;
        }
    } else {
        const float v = per_set[im.set0];
        for (int i = tid; i < im.rows; i += kBlock) out[im.row0 + i] = v;
    }
}

template <int MODE, int TYPE, bool MASK, bool BIAS>
hipError_t launch_choice_as(const SetLayout& s, const ChoiceArgs& a, int32_t grid, hipStream_t stream) {
    if (MODE != kStepsBack && s.num_split > 0) {
        hipLaunchKernelGGL((part_kernel<MODE, TYPE, MASK, BIAS>), dim3(s.num_split), dim3(kBlock), 0, stream, a, s.split);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((choice_kernel<MODE, TYPE, MASK, BIAS>), dim3(grid), dim3(kBlock), 0, stream, a);
    return hipGetLastError();
}

template <int MODE, int TYPE>
hipError_t launch_choice_typed(const SetLayout& s, const ChoiceArgs& a, int32_t grid, hipStream_t stream) {
    if (a.mask)
        return a.table ? launch_choice_as<MODE, TYPE, true, true>(s, a, grid, stream)
                       : launch_choice_as<MODE, TYPE, true, false>(s, a, grid, stream);
    return a.table ? launch_choice_as<MODE, TYPE, false, true>(s, a, grid, stream)
                   : launch_choice_as<MODE, TYPE, false, false>(s, a, grid, stream);
}

template <int MODE>
hipError_t launch_choice_mode(const SetLayout& s, const ChoiceArgs& a, int32_t type, int32_t grid, hipStream_t stream) {
    if (type == PB_BF16) return launch_choice_typed<MODE, PB_BF16>(s, a, grid, stream);
    if (type == PB_F16) return launch_choice_typed<MODE, PB_F16>(s, a, grid, stream);
    return launch_choice_typed<MODE, PB_F32>(s, a, grid, stream);
}

template <bool PAIRS>
hipError_t launch_set_sum(const SetLayout& s, SumArgs a, hipStream_t stream) {
    if (s.num_items == 0) return hipSuccess;
    a.off = s.off;
    a.items = s.items;
    a.num_items = s.num_items;
    hipLaunchKernelGGL(set_sum_kernel<PAIRS>, dim3(s.num_items), dim3(kBlock), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || s.num_split == 0) return e;
    hipLaunchKernelGGL(set_join_kernel, dim3(s.num_split), dim3(kBlock), 0, stream, a, s.split, s.num_split);
    return hipGetLastError();
}

__global__ __launch_bounds__(kBlock) void zero_kernel(float* __restrict__ out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) out[i] = 0.0f;
}

}  // namespace

hipError_t launch_zero(float* out, int64_t n, hipStream_t stream) {
    if (n <= 0) return hipSuccess;
    const int64_t want = (n + kBlock - 1) / kBlock;
    hipLaunchKernelGGL(zero_kernel, dim3((unsigned)(want < kPairGrid ? want : kPairGrid)), dim3(kBlock), 0, stream, out, n);
    return hipGetLastError();
}

int32_t choice_grid(const SetLayout& s) { return s.num_items < kChoiceGrid ? s.num_items : kChoiceGrid; }

hipError_t launch_choice(int mode, const SetLayout& s, ChoiceArgs a, int32_t type, hipStream_t stream) {
    a.off = s.off;
    a.items = s.items;
    a.num_items = s.num_items;
    const int32_t grid = choice_grid(s);
    hipError_t e = hipSuccess;
    if (mode == kRows) e = launch_choice_mode<kRows>(s, a, type, grid, stream);
    if (mode == kSteps) e = launch_choice_mode<kSteps>(s, a, type, grid, stream);
    if (mode == kRowsBack) e = launch_choice_mode<kRowsBack>(s, a, type, grid, stream);
    if (mode == kStepsBack) e = launch_choice_mode<kStepsBack>(s, a, type, grid, stream);
    if (mode == kPolicy) e = launch_choice_mode<kPolicy>(s, a, type, grid, stream);
    const int32_t head = mode == kPolicy ? 3 : 0;
    const int32_t cols = head + (a.table && mode != kRows && mode != kSteps ? a.num_buckets : 0);
    if (e != hipSuccess || cols == 0 || grid == 1) return e;
    hipLaunchKernelGGL(join_kernel, dim3(cols), dim3(kBlock), 0, stream, a.sums, grid, cols, head, a.stats, a.grad_table);
    return hipGetLastError();
}

hipError_t launch_preference(const PairLayout& p, PairArgs a, const float* values, const float* ref, float* grad,
                             char* work, hipStream_t stream) {
    a.winners = p.winners;
    a.losers = p.losers;
    a.num_pairs = p.num_pairs;
    a.sums = reinterpret_cast<double*>(work);
    double* parts = a.sums + kPairGrid;
    a.slopes = reinterpret_cast<float*>(parts + p.lists.num_items + p.seqs.num_items);
    float* seq_sum = a.slopes + p.num_pairs;
    float* seq_grad = seq_sum + p.seqs.num_sets;
    const bool seqs = p.has_seqs;
    hipError_t e = hipSuccess;
    SumArgs sa{};
    sa.parts = parts;
    if (seqs) {
        sa.values = values;
        sa.ref = ref;
        sa.out = seq_sum;
        if ((e = launch_set_sum<false>(p.seqs, sa, stream)) != hipSuccess) return e;
        a.values = seq_sum;
        a.ref = nullptr;
    } else {
        a.values = values;
        a.ref = ref;
    }
    const int64_t want = (p.num_pairs + kBlock - 1) / kBlock;
    const int grid = (int)(want < 1 ? 1 : want > kPairGrid ? kPairGrid : want);
    hipLaunchKernelGGL(pair_kernel, dim3(grid), dim3(kBlock), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (grid > 1) {
        hipLaunchKernelGGL(join_kernel, dim3(1), dim3(kBlock), 0, stream, a.sums, grid, 1, 1, a.loss, nullptr);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    sa.parts = parts + p.seqs.num_items;
    sa.entries = p.entries;
    sa.slopes = a.slopes;
    sa.out = seqs ? seq_grad : grad;
    if ((e = launch_set_sum<true>(p.lists, sa, stream)) != hipSuccess) return e;
    if (seqs && p.seqs.num_items > 0) {
        hipLaunchKernelGGL(spread_kernel, dim3(p.seqs.num_items), dim3(kBlock), 0, stream, p.seqs.off, p.seqs.items,
                           seq_grad, grad);
        e = hipGetLastError();
    }
    return e;
}

int64_t preference_work_bytes(const PairLayout& p) {
    return 8 * ((int64_t)kPairGrid + p.lists.num_items + p.seqs.num_items) + 4 * (p.num_pairs + 2 * p.seqs.num_sets);
}

}  // namespace pb
