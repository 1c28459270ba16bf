// Reports on choices over ragged sets of candidate rows: of each set the chosen row's log-probability, the entropy, and the
// rows of largest probability with theirs, at a temperature T.
//
// With z the logits, m their maximum (0 where that is -inf), e_i = exp((z_i - m) / T), s = sum e and u = sum e (z - m):
// lse = m / T + log s, log p_i = (z_i - m) / T - log s, and the entropy -sum p log p = log s - u / (T s). A set without
// probability has s = 0, lse -inf and entropy 0. Rows are ranked by z, equal ones by index, NaN above all; rows of z = -inf
// are not ranked.
//
// A workgroup to a set: its rows are read once for the maximum, once for the sums, and once for each entry of its list.
#include <algorithm>

#include "choice_rows.h"
#include "report.h"

namespace pb {
namespace {

constexpr int kReportGrid = 4096;

// What orders the rows of a set: larger logits first (-0 as 0, NaN above all), then smaller indices; 0 for none.
__device__ __forceinline__ unsigned long long rank_key(float z, uint32_t index) {
    const uint32_t b = z != z ? 0x7fc00000u : __float_as_uint(z + 0.0f);
    return (unsigned long long)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | (uint32_t)~index;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* sh) {
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) {
        const unsigned long long t = __shfl_xor(v, m);
        v = t > v ? t : v;
    }
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) v = sh[w] > v ? sh[w] : v;
    return v;
}

// f(rows from the set's first, logits) for every run of rows [r0, r1), a thread a run.
template <int TYPE, bool MASK, bool BIAS, class F>
__device__ __forceinline__ void each_run(const ReportArgs& a, const BiasShared* bias, int64_t r0, int64_t r1, F f) {
    constexpr int64_t kPiece = 1 << 20;
    for (int64_t p0 = r0; p0 < r1; p0 += kPiece) {
        Span s;
        s.q0 = p0 & ~(int64_t)(kRun - 1);
        s.lo = (int)(p0 - s.q0);
        s.hi = s.lo + (int)min(kPiece, r1 - p0);
        s.end = (int)min(a.rows - s.q0, (int64_t)1 << 30);
        for (int i = kRun * (int)threadIdx.x; i < s.hi; i += kRun * kBlock) {
            float z[kRun];
            uint32_t off;
            Buckets buckets;
            load_logits<TYPE, MASK, BIAS>(a, bias, s, i, z, off, buckets);
            f(s.q0 + i - r0, z);
        }
    }
}

template <int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void report_kernel(ReportArgs a, int64_t num_sets) {
    __shared__ BiasShared bias;
    __shared__ float shf[kWaves];
    __shared__ double shd[kWaves];
    __shared__ unsigned long long shk[kWaves];
    if (BIAS) stage_bias(a, bias);
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    for (int64_t g = blockIdx.x; g < num_sets; g += gridDim.x) {
        const int64_t r0 = a.off[g], r1 = a.off[g + 1];
        float top = kLowest;
        each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](int64_t, const float(&z)[kRun]) {
#pragma unroll
            for (int k = 0; k < kRun; ++k) top = max2(top, z[k]);
        });
        top = wave_max(top);
        __syncthreads();
        if ((threadIdx.x & (kWave - 1)) == 0) shf[threadIdx.x / kWave] = top;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) top = max2(top, shf[w]);
        double sum = 0.0, along = 0.0;
        each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](int64_t, const float(&z)[kRun]) {
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const float e = heat_exp<true>(z[k] - top, heat);
                sum += (double)e;
                along += e == 0.0f ? 0.0 : (double)e * (double)(z[k] - top);
            }
        });
        sum = block_sum(sum, shd);
        along = block_sum(along, shd);
        const bool none = sum == 0.0;
        const double log_sum = log(sum);
        if (threadIdx.x == 0) {
            const double m = none ? 0.0 : (double)top;
            a.lse_out[g] = (float)(m * a.inv_temp + log_sum);
            a.entropy[g] = none ? 0.0f : (float)(log_sum - along * a.inv_temp / sum);
            if (a.chosen) {
                const int32_t c = a.chosen[g];
                bool counts = c >= 0 && c < r1 - r0 && !none;
                if (MASK && counts) counts = a.mask[r0 + c] != 0;
                a.log_probs[g] = counts ? (float)(((double)one_logit<TYPE, BIAS>(a, &bias, r0 + c) - m) * a.inv_temp - log_sum) : 0.0f;
            }
        }
        unsigned long long last = ~0ull;
        for (int j = 0; j < a.top; ++j) {
            unsigned long long best = 0;
            if (last != 0)
                each_run<TYPE, MASK, BIAS>(a, &bias, r0, r1, [&](int64_t i, const float(&z)[kRun]) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k) {
                        const unsigned long long key = z[k] == -kInf ? 0ull : rank_key(z[k], (uint32_t)(i + k));
                        best = key < last && key > best ? key : best;
                    }
                });
            last = block_max(best, shk);
            if (threadIdx.x == 0) {
                const uint32_t i = ~(uint32_t)last;
                a.top_index[g * a.top + j] = last ? (int32_t)i : -1;
                a.top_log_probs[g * a.top + j] =
                    last ? (float)(((double)one_logit<TYPE, BIAS>(a, &bias, r0 + i) - (double)top) * a.inv_temp - log_sum) : -kInf;
            }
        }
    }
}

template <int TYPE>
hipError_t launch_report_typed(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)std::min<int64_t>(s.num_sets, kReportGrid)), block(kBlock);
    if (a.mask && a.table)
        hipLaunchKernelGGL((report_kernel<TYPE, true, true>), grid, block, 0, stream, a, s.num_sets);
    else if (a.mask)
        hipLaunchKernelGGL((report_kernel<TYPE, true, false>), grid, block, 0, stream, a, s.num_sets);
    else if (a.table)
        hipLaunchKernelGGL((report_kernel<TYPE, false, true>), grid, block, 0, stream, a, s.num_sets);
    else
        hipLaunchKernelGGL((report_kernel<TYPE, false, false>), grid, block, 0, stream, a, s.num_sets);
    return hipGetLastError();
}

}  // namespace

int64_t report_work_bytes(const SetLayout&, int32_t) { return 0; }

hipError_t launch_report(const SetLayout& s, ReportArgs a, int32_t type, char*, hipStream_t stream) {
    a.off = s.off;
    a.rows = s.rows;
    const auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    a.vec = a.stride == 1 && at(a.scores, 16) && at(a.mask, 8) && at(a.positions, 16);
    if (type == PB_BF16) return launch_report_typed<PB_BF16>(s, a, stream);
    if (type == PB_F16) return launch_report_typed<PB_F16>(s, a, stream);
    return launch_report_typed<PB_F32>(s, a, stream);
}

}  // namespace pb
