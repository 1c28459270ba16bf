// Gradients of losses that see a set's whole distribution: of the chosen rows' log-probabilities and the entropies, and of
// the divergence from a teacher of which each set's best rows are known. Logits z, temperature T, p_i and the other
// names as in report.hip.
//
// Entropies: with a the gradient of the chosen row's log-probability (0 where left out) and h that of the entropy H,
// dz_i = [a ([i = chosen] - p_i) - h p_i (log p_i + H)] / T, where log p_i + H = (z_i - m) / T - u / (T s).
//
// Distillation: entry j of a set's list names a row and has the teacher's value t_j. Those count that name a row of the
// set that is not masked, the first of those that name one row. q_j = exp(t_j / T) over their sum, or (tail) exp(t_j), and
// what these leave of 1 (rho) stands against the rows not listed, the rest: pi = their sum of p. Where there is no rest, or
// the q_j sum to 1 or more, they are divided by their sum and rho = 0. kl = sum q (log q - log p) + rho (log rho - log pi), and
// loss = scale T^2 sum w kl. Its gradient is scale w T (p_j - q_j) for the listed rows and scale w T r_i (pi - rho) for
// the others, r the softmax over the rest. The rest is reduced by itself, so that pi is no difference. Sets in which the
// teacher's entries or the student have no probability are left out.
//
// A workgroup to a set, whose rows are read three times.
#include <algorithm>

#include "choice_rows.h"

namespace pb {
namespace {

constexpr int kSoftGrid = 2048;

// f(span, row of the span, logits, masked rows, buckets) for every run of rows [r0, r1); whole waves.
template <int TYPE, bool MASK, bool BIAS, class F>
__device__ __forceinline__ void each_run(const ReportArgs& a, const BiasShared* bias, int64_t r0, int64_t r1, F f) {
    constexpr int64_t kPiece = 1 << 20;
    const int lane = (int)threadIdx.x & (kWave - 1), wave0 = (int)threadIdx.x - lane;
    for (int64_t p0 = r0; p0 < r1; p0 += kPiece) {
        Span s;
        s.q0 = p0 & ~(int64_t)(kRun - 1);
        s.lo = (int)(p0 - s.q0);
        s.hi = s.lo + (int)min(kPiece, r1 - p0);
        s.end = (int)min(a.rows - s.q0, (int64_t)1 << 30);
        for (int i0 = kRun * wave0; i0 < s.hi; i0 += kRun * kBlock) {
            const int i = i0 + kRun * lane;
            float z[kRun];
            uint32_t off = 0xffu;
            Buckets buckets{{0, 0}};
#pragma unroll
            for (int k = 0; k < kRun; ++k) z[k] = -kInf;
            if (i < s.hi) load_logits<TYPE, MASK, BIAS>(a, bias, s, i, z, off, buckets);
            f(s, i, z, off, buckets);
        }
    }
}

__device__ __forceinline__ float block_max(float v, float* sh) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) v = max2(v, sh[w]);
    return v;
}

__device__ __forceinline__ float entry_logit(const ReportArgs& a, int64_t i) {
    if (a.entry_type == PB_F32) return load_score<PB_F32>(a.entry_logits, i);
    return a.entry_type == PB_BF16 ? load_score<PB_BF16>(a.entry_logits, i) : load_score<PB_F16>(a.entry_logits, i);
}

// One set's divergence and slopes, a lane to an entry: z the student's logit (-inf where the entry does not count), t
// the teacher's value, top and sum the rest's maximum and sum of exponentials. All sums in double: what they leave is
// small where student and teacher are close.
struct Divergence {
    double kl;
    float own;   // gradient of the lane's listed row
    float rest;  // what the rest's exponentials are multiplied by
};

__device__ __forceinline__ Divergence diverge(const ReportArgs& a, bool on, float z, float t, float rest_top, double rest_sum,
                                              float weight, int bits) {
    const bool has_rest = rest_sum != 0.0;
    const double top = fmax(team_max((double)z, bits), has_rest ? (double)rest_top : (double)kLowest);
    const double x = ((double)z - top) * a.inv_temp, e = on ? exp(x) : 0.0;
    const double rest_x = ((double)rest_top - top) * a.inv_temp, rest = has_rest ? exp(rest_x) * rest_sum : 0.0;
    const double total = team_sum(e, bits) + rest;
    const double given = on ? (a.tail ? (double)t : (double)t * a.inv_temp) : -(double)kInf;
    double given_top = a.tail ? 0.0 : team_max(given, bits);
    if (given_top == -(double)kInf) given_top = 0.0;
    const double part = on ? exp(given - given_top) : 0.0, mass = team_sum(part, bits);
    const bool use = mass != 0.0 && total != 0.0;
    const bool open = a.tail && has_rest && mass < 1.0;
    const double q = open ? part : part / mass, rho = open ? 1.0 - mass : 0.0;
    const double log_q = given - given_top - (open ? 0.0 : log(mass)), log_total = log(total);
    double kl = team_sum(!on || q == 0.0 ? 0.0 : q * (log_q - (x - log_total)), bits);
    if (rho != 0.0) kl += rho * (log(rho) - (rest_x + log(rest_sum) - log_total));
    const double w = use && weight != 0.0f ? (double)weight * (double)a.temp : 0.0;
    Divergence d;
    d.kl = use ? kl : 0.0;
    d.own = w == 0.0 || !on ? 0.0f : (float)(w * (e / total - q));
    d.rest = w == 0.0 || !has_rest ? 0.0f : (float)(w * (rest / total - rho) / rest_sum);
    return d;
}

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void soft_grads_kernel(ReportArgs a, int64_t num_sets) {
    __shared__ BiasShared bias;
    __shared__ unsigned long long bins[BIAS ? kWaves : 1][kBins];
    __shared__ int shifts[BIAS ? kWaves : 1][kBins];
    __shared__ int bad[kMaxBuckets];
    __shared__ float shf[kWaves];
    __shared__ double shd[kWaves * 3];
    __shared__ int64_t listed[kMaxTop];  // rows of the entries that count, -1 for none
    __shared__ float own[kMaxTop];
    __shared__ float factor;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    TableSum table;
    if (BIAS) {
        for (int b = tid; b < kMaxBuckets; b += kBlock) bad[b] = 0;
        table.start(a, bins[wave], shifts[wave], bad);
        stage_bias(a, bias);
    }
    double tally[3] = {0.0, 0.0, 0.0};
    for (int64_t g = blockIdx.x; g < num_sets; g += gridDim.x) {
        const int64_t r0 = a.off[g], r1 = a.off[g + 1];
        int32_t entry = -1;
        bool on = false;
        float z = -kInf;
        __syncthreads();  // the last set's list has been read
        if (DISTILL) {
            if (lane < a.top) entry = a.entry_index[g * a.top + lane];
            on = entry >= 0 && entry < r1 - r0;
            if (MASK && on) on = a.mask[r0 + entry] != 0;
            for (int j = 0; j + 1 < a.top; ++j) {
                const int32_t before = __shfl(entry, j);
                if (j < lane && before == entry) on = false;
            }
            if (on) z = one_logit<TYPE, BIAS>(a, &bias, r0 + entry);
            if (wave == 0) listed[lane] = on ? r0 + entry : -1;
            __syncthreads();
        }
        const auto in_list = [&](int64_t row) {
            uint32_t b = 0;
            for (int j = 0; j < a.top; ++j) {
                const int64_t d = listed[j] - row;
                if (d >= 0 && d < kRun) b |= 1u << d;
            }
            return b;
        };
        float top = kLowest;
        each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](const Span& s, int i, float(&x)[kRun], uint32_t, const Buckets&) {
            const uint32_t out = DISTILL ? in_list(s.q0 + i) : 0;
#pragma unroll
            for (int k = 0; k < kRun; ++k) top = max2(top, out >> k & 1u ? -kInf : x[k]);
        });
        top = block_max(top, shf);
        double sum = 0.0, along = 0.0;
        each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](const Span& s, int i, float(&x)[kRun], uint32_t, const Buckets&) {
            const uint32_t out = DISTILL ? in_list(s.q0 + i) : 0;
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const float e = out >> k & 1u ? 0.0f : heat_exp<true>(x[k] - top, heat);
                sum += (double)e;
                if (!DISTILL) along += e == 0.0f ? 0.0 : (double)e * (double)(x[k] - top);
            }
        });
        sum = block_sum(sum, shd);
        if (!DISTILL) along = block_sum(along, shd);
        int64_t chosen = -1;
        float first = 0.0f, slope = 0.0f;  // a row's gradient: e (first + slope (z - m))
        float extra = 0.0f;
        if (DISTILL) {
            const float w = (a.weights ? a.weights[g] : 1.0f) * a.scale;
            if (wave == 0) {
                const Divergence d = diverge(a, on, z, lane < a.top ? entry_logit(a, g * a.top + lane) : 0.0f, top, sum, w, 6);
                own[lane] = d.own;
                if (lane == 0) {
                    a.kl[g] = (float)d.kl;
                    factor = d.rest;
                    if (w != 0.0f) tally[0] += (double)w * (double)a.temp * (double)a.temp * d.kl;
                }
            }
            __syncthreads();
            first = factor;
        } else if (sum != 0.0) {
            float coef = 0.0f;
            if (a.chosen && a.grad) {
                const int32_t c = a.chosen[g];
                bool counts = c >= 0 && c < r1 - r0;
                if (MASK && counts) counts = a.mask[r0 + c] != 0;
                if (counts) {
                    chosen = r0 + c;
                    coef = a.grad[g];
                }
            }
            const double h = a.grad_entropy ? (double)a.grad_entropy[g] : 0.0, scale = a.inv_temp / sum;
            extra = (float)((double)coef * a.inv_temp);
            first = (float)(scale * (h * (along * a.inv_temp / sum) - (double)coef));
            slope = (float)(-scale * a.inv_temp * h);
        }
        each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](const Span& s, int i, float(&x)[kRun], uint32_t off, const Buckets& buckets) {
            const uint32_t out = DISTILL ? in_list(s.q0 + i) : 0;
            float v[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const float e = heat_exp<true>(x[k] - top, heat);
                const float f = DISTILL ? first : e == 0.0f ? 0.0f : __builtin_fmaf(slope, x[k] - top, first);
                v[k] = f == 0.0f || (out >> k & 1u) ? 0.0f : f * e;
                if (!DISTILL && chosen == s.q0 + i + k) v[k] += extra;
            }
            if (out)
                for (int j = 0; j < a.top; ++j) {
                    const int64_t d = listed[j] - (s.q0 + i);
#pragma unroll
                    for (int k = 0; k < kRun; ++k)
                        if (d == k) v[k] = own[j];
                }
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] = off >> k & 1u ? 0.0f : v[k];
            if (i < s.hi) store_run<TYPE>(a, s, i, a.grad_scores, v);
            if (BIAS) table.add<false>(v, buckets);
        });
    }
    leave_sums<DISTILL ? 1 : 0, BIAS>(a, (int)blockIdx.x, tally, table, bins, bad, shd);
}

int grid_of(const SetLayout& s) { return (int)std::min<int64_t>(s.num_sets, kSoftGrid); }

template <bool DISTILL, int TYPE>
void launch_typed(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    const dim3 grid(a.blocks), block(kBlock);
    if (a.mask && a.table)
        hipLaunchKernelGGL((soft_grads_kernel<DISTILL, TYPE, true, true>), grid, block, 0, stream, a, s.num_sets);
    else if (a.mask)
        hipLaunchKernelGGL((soft_grads_kernel<DISTILL, TYPE, true, false>), grid, block, 0, stream, a, s.num_sets);
    else if (a.table)
        hipLaunchKernelGGL((soft_grads_kernel<DISTILL, TYPE, false, true>), grid, block, 0, stream, a, s.num_sets);
    else
        hipLaunchKernelGGL((soft_grads_kernel<DISTILL, TYPE, false, false>), grid, block, 0, stream, a, s.num_sets);
}

template <bool DISTILL>
void launch_as(const SetLayout& s, const ReportArgs& a, int32_t type, hipStream_t stream) {
    if (type == PB_BF16) return launch_typed<DISTILL, PB_BF16>(s, a, stream);
    if (type == PB_F16) return launch_typed<DISTILL, PB_F16>(s, a, stream);
    launch_typed<DISTILL, PB_F32>(s, a, stream);
}

}  // namespace

int64_t soft_grads_work_bytes(const SetLayout& s, bool distill, int32_t num_buckets) {
    return grid_of(s) <= 1 ? 0 : 8 * (int64_t)grid_of(s) * ((distill ? 1 : 0) + num_buckets);
}

hipError_t launch_soft_grads(bool distill, const SetLayout& s, ReportArgs a, int32_t type, char* work, hipStream_t stream) {
    a.off = s.off;
    a.rows = s.rows;
    a.blocks = grid_of(s);
    a.sums = reinterpret_cast<double*>(work);
    const auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    a.vec = a.stride == 1 && at(a.scores, 16) && at(a.grad_scores, 16) && at(a.mask, 8) && at(a.positions, 16);
    if (distill)
        launch_as<true>(s, a, type, stream);
    else
        launch_as<false>(s, a, type, stream);
    const hipError_t e = hipGetLastError();
    const int32_t cols = (distill ? 1 : 0) + a.num_buckets;
    if (e != hipSuccess || cols == 0 || a.blocks == 1) return e;
    return launch_join_sums(a.sums, a.blocks, cols, distill ? 1 : 0, a.stats, a.grad_table, stream);
}

}  // namespace pb
