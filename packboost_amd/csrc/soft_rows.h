// Sums over sets at a temperature, as the kernels of reports and of their gradients join them.
#pragma once

#include "choice_rows.h"
#include "report.h"

namespace pb {
namespace {

// The exponentials of what is rounded to 16 bits round their exponents once.
template <int TYPE, bool BIAS>
constexpr bool kExact = TYPE == PB_F32 || BIAS;

// What a wave takes: the mid sets, then the few short ones. (Six short sets beside 300 longer ones, with a teacher, in a
// launch of tiles of their own cost 11 us of 54.)
__device__ __forceinline__ SetItem wave_item(const ReportArgs& a, int i) { return i < a.num_mid ? a.wide[i] : a.shorts[i - a.num_mid]; }

// What a group's waves leave of their rows.
template <int WAVES>
struct GroupSums {
    float top[WAVES];
    double sum[WAVES], along[WAVES];
};

// A group's sums from those of its waves (each relative to the wave's own maximum), the same in every lane.
template <bool ALONG, int WAVES>
__device__ __forceinline__ SoftSums join_waves(const ReportArgs& a, const SoftSums& own, GroupSums<WAVES>& sh) {
    if (WAVES == 1) return own;
    constexpr int kBits = WAVES == 4 ? 2 : WAVES == 8 ? 3 : 4;
    static_assert(WAVES == 1 || WAVES == 1 << kBits, "4, 8 or 16 waves");
    const int lane = (int)threadIdx.x & (kWave - 1), wave = (int)threadIdx.x / kWave, w = lane & (WAVES - 1);
    if (lane == 0) {
        sh.top[wave] = own.top;
        sh.sum[wave] = own.sum;
        if (ALONG) sh.along[wave] = own.along;
    }
    __syncthreads();
    SoftSums t{sh.top[w], sh.sum[w], ALONG ? sh.along[w] : 0.0};
    const float top = wave_max(t.top);
    const double gap = (double)t.top - (double)top, f = exp_near(gap * a.inv_temp);
    if (ALONG) t.along = team_sum(f == 0.0 ? 0.0 : f * (t.along + t.sum * gap), kBits);
    t.sum = team_sum(t.sum * f, kBits);
    t.top = top;
    return t;
}

// A set's sums from those of its parts.
template <bool ALONG, int WAVES>
__device__ __forceinline__ SoftSums join_set(const ReportArgs& a, const SoftSums* parts, int n, GroupSums<WAVES>& sh) {
    SoftSums t{kLowest, 0.0, 0.0};
    for (int j = (int)threadIdx.x; j < n; j += WAVES * kWave) t.top = max2(t.top, parts[j].top);
    t.top = wave_max(t.top);
    for (int j = (int)threadIdx.x; j < n; j += WAVES * kWave) {
        const SoftSums p = parts[j];
        const double gap = (double)p.top - (double)t.top, f = exp_near(gap * a.inv_temp);
        t.sum += p.sum * f;
        if (ALONG) t.along += f == 0.0 ? 0.0 : f * (p.along + p.sum * gap);
    }
    t.sum = team_sum(t.sum, 6);
    if (ALONG) t.along = team_sum(t.along, 6);
    return join_waves<ALONG>(a, t, sh);
}

}  // namespace
}  // namespace pb
