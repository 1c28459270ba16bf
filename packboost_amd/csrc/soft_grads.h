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
// Rows are laid out, read and written as choice.hip has them: tiles of short sets by a wave, longer sets by a wave or a
// workgroup that holds them in registers, what is longer still in parts that are read twice. A set's list is taken by as many
// lanes as it has entries, rounded up to a power of 2; a byte a row in LDS says which entry names it.
#pragma once

#include <algorithm>

#include "choice_rows.h"
#include "report.h"

namespace pb {
namespace {

// The exponentials of gradients that are rounded to 16 bits, each rounding its exponent once.
template <int TYPE, bool BIAS>
constexpr bool kExact = TYPE == PB_F32 || BIAS;

__device__ __forceinline__ float entry_logit(const ReportArgs& a, int64_t i) {
    if (a.entry_type == PB_F32) return load_score<PB_F32>(a.entry_logits, i);
    return a.entry_type == PB_BF16 ? load_score<PB_BF16>(a.entry_logits, i) : load_score<PB_F16>(a.entry_logits, i);
}

__device__ __forceinline__ double inverse(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// One set's divergence and slopes, a lane of its team to an entry: z the student's logit (-inf where the entry does not
// count), t the teacher's value, top and sum the rest's maximum and sum of exponentials. In double: a divergence is what
// large terms leave where student and teacher are close, and rho is a difference.
struct Divergence {
    double kl;
    float own;   // gradient of the lane's listed row
    float rest;  // what the rest's exponentials are multiplied by
};

__device__ __forceinline__ Divergence diverge(const ReportArgs& a, bool on, float z, float t, float rest_top, double rest_sum,
                                              float weight, int bits) {
    const bool has_rest = rest_sum != 0.0;
    const double top = fmax(team_max((double)z, bits), has_rest ? (double)rest_top : (double)kLowest);
    const double x = ((double)z - top) * a.inv_temp, e = exp_near(x);  // 0 where the entry does not count
    const double rest_x = ((double)rest_top - top) * a.inv_temp, rest_e = has_rest ? exp_near(rest_x) : 0.0;
    const double total = team_sum(e, bits) + (has_rest ? rest_e * rest_sum : 0.0);
    double given = on ? (a.tail ? (double)t : (double)t * a.inv_temp) : -(double)kInf;
    if (!a.tail) {
        const double most = team_max(given, bits);
        if (most > -(double)kInf) given -= most;
    }
    const double part = exp_near(given), mass = team_sum(part, bits);
    const double lost = team_sum(part == 0.0 ? 0.0 : part * (given - x), bits);
    const bool use = mass != 0.0 && total != 0.0;
    const bool open = a.tail && has_rest && mass < 1.0;
    const double rho = open ? 1.0 - mass : 0.0, per_mass = open ? 1.0 : inverse(mass);
    const double log_total = log_near(total), log_left = log_near(open ? rho : mass);
    Divergence d;
    d.kl = lost * per_mass;
    double away = 0.0;  // rho over the rest's sum
    if (open) {
        d.kl += mass * log_total + rho * (log_left - (rest_x + log_near(rest_sum) - log_total));
        away = rho * inverse(rest_sum);
    } else {
        d.kl += log_total - log_left;
    }
    if (!use) d.kl = 0.0;
    const double w = use && weight != 0.0f ? (double)weight * (double)a.temp : 0.0, per_total = inverse(total);
    d.own = w == 0.0 || !on ? 0.0f : (float)(w * (e * per_total - part * per_mass));
    d.rest = w == 0.0 || !has_rest ? 0.0f : (float)(w * (rest_e * per_total - away));
    return d;
}

// A row's gradient is its exponential times (first + slope (z - m)), from a set's sums.
struct Slopes {
    float first, slope;
};

__device__ __forceinline__ Slopes slopes_of(const ReportArgs& a, double sum, double along, float coef, float h) {
    const double per = sum != 0.0 ? inverse(sum) : 0.0, scale = a.inv_temp * per;
    return Slopes{(float)(scale * ((double)h * (along * a.inv_temp * per) - (double)coef)), (float)(-scale * a.inv_temp * (double)h)};
}

// ------------------------------------------------------------------------------------ tiles
struct SoftTile {
    float x[kSetTileRows];        // logits, then what listed and chosen rows have of their own
    float top[kSetTileSets + 4];  // per set: maximum
    union {
        uint16_t head[kSetTileRows];    // the set that starts at a row, from 1; 0: none
        float first[kSetTileSets + 4];  // later: sum of exponentials, then what they are multiplied by
    };
    union {
        uint8_t slot[kSetTileRows];     // distillation: the entry that names a row, from 1; 0: none
        float slope[kSetTileSets + 4];  // entropies: sum of exponentials times distances, then slopes
    };
};

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
struct SoftTileIn {
    TileRows<TYPE, MASK, BIAS> rows;
    int32_t chosen[kTileRounds];
    float coef[kTileRounds], h[kTileRounds];

    __device__ __forceinline__ void load(const ReportArgs& a, const SetItem& im, int lane) {
        rows.load(a, im, lane);
        if (DISTILL) return;
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            chosen[r] = -1;
            coef[r] = h[r] = 0.0f;
            if (r * kWave + lane < rows.sets) {
                const int64_t g = rows.set[r];
                if (a.grad) {
                    chosen[r] = a.chosen[g];
                    coef[r] = a.grad[g];
                }
                if (a.grad_entropy) h[r] = a.grad_entropy[g];
            }
        }
    }
};

// The entries of a tile's lists, 64 at a time: which set's a lane has, and where that set lies.
struct EntryLane {
    int s, j, begin, size;
    int64_t g;
    bool there;

    template <class ROWS>
    __device__ __forceinline__ EntryLane(const ReportArgs& a, const ROWS& in, int it, int lane) {
        const int bits = a.team_bits, first = it << (6 - bits), r = first / kWave;
        s = first + (lane >> bits);
        j = lane & ((1 << bits) - 1);
        const int from = s & (kWave - 1);
        begin = __shfl(r ? in.begin[1] : in.begin[0], from);
        size = __shfl(r ? in.end[1] : in.end[0], from) - begin;
        g = __shfl(r ? in.set[1] : in.set[0], from);
        there = s < in.sets && j < a.top;
    }
};
static_assert(kTileRounds == 2, "a lane has two sets of a tile");

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ void soft_tile(const ReportArgs& a, SoftTileIn<DISTILL, TYPE, MASK, BIAS>& all, SoftTile& sh,
                                          const BiasShared* bias, TableSum& table, double (&tally)[3]) {
    const TileRows<TYPE, MASK, BIAS>& in = all.rows;
    const int lane = (int)threadIdx.x & (kWave - 1), i0 = kRun * lane;
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    const Span sp = in.sp;
    const bool alone = in.sets == 1;
    float x[kRun];
    uint32_t off = 0xffu;
    Buckets buckets{{0, 0}};
#pragma unroll
    for (int k = 0; k < kRun; ++k) x[k] = -kInf;
    if (sp.hi > 0) in.raw.logits(a, bias, sp, 0, x, off, buckets);
    wave_sync();  // the last tile's values have been read
    *reinterpret_cast<uint4*>(&sh.head[i0]) = make_uint4(0, 0, 0, 0);
    if (DISTILL) *reinterpret_cast<uint2*>(&sh.slot[i0]) = make_uint2(0, 0);
    write_run(&sh.x[i0], x);
    wave_sync();
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        if (s < in.sets) {
            if (in.end[r] > in.begin[r]) sh.head[in.begin[r]] = (uint16_t)(s + 1);
            if (!DISTILL) {
                if (all.chosen[r] >= in.end[r] - in.begin[r]) all.chosen[r] = -1;
                // a masked row's logit is -inf, as one of that score is: the mask says which
                if (MASK && all.chosen[r] >= 0 && sh.x[in.begin[r] + all.chosen[r]] == -kInf &&
                    !a.mask[a.off[in.set[r]] + all.chosen[r]])
                    all.chosen[r] = -1;
            }
        }
    }
    const int rounds = DISTILL ? ((in.sets << a.team_bits) + kWave - 1) / kWave : 0;
    if (DISTILL) {
        for (int it = 0; it < rounds; ++it) {
            const EntryLane l(a, in, it, lane);
            const int32_t c = l.there ? a.entry_index[l.g * a.top + l.j] : -1;
            bool on = c >= 0 && c < l.size;
            if (MASK && on && sh.x[l.begin + c] == -kInf) on = a.mask[a.off[l.g] + c] != 0;
            if (on) sh.slot[l.begin + c] = (uint8_t)(l.j + 1);
            wave_sync();
            if (__any(on && sh.slot[l.begin + c] != l.j + 1)) {  // rows named twice: the first entry counts
                const int named = on ? c : -1;
                for (int d = 1; d < 1 << a.team_bits; ++d) {
                    const int before = __shfl(named, lane >= d ? lane - d : lane);
                    if (d <= l.j && before == named) on = false;
                }
                wave_sync();
                if (on) sh.slot[l.begin + c] = (uint8_t)(l.j + 1);
            }
        }
    }
    wave_sync();
    uint2 slots = make_uint2(0, 0);
    if (DISTILL) {
        slots = *reinterpret_cast<const uint2*>(&sh.slot[i0]);
        if (slots.x | slots.y) {
#pragma unroll
            for (int k = 0; k < kRun; ++k) x[k] = ((k < 4 ? slots.x : slots.y) >> (8 * (k & 3)) & 0xffu) ? -kInf : x[k];
        }
    }
    TileSets sets;
    if (alone) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) sets.id[k] = 1;
    } else {
        sets.find(sh.head, lane);
    }
    wave_sync();  // the heads have been read
    float v[kRun], d[kRun];
    if (alone) {
        float top = kLowest, sum = 0.0f, along = 0.0f;
#pragma unroll
        for (int k = 0; k < kRun; k += 2) top = max3(top, x[k], x[k + 1]);
        top = wave_max(top);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            d[k] = __builtin_elementwise_maximum(x[k] - top, heat.low);
            sum += v[k] = heat_exp<kExact<TYPE, BIAS>>(d[k], heat);
            along += v[k] * d[k];
        }
        sum = wave_sum(sum);
        if (!DISTILL) along = wave_sum(along);
        if (lane == 0) {
            sh.top[0] = top;
            sh.first[0] = sum;
            if (!DISTILL) sh.slope[0] = along;
        }
        wave_sync();
    } else {
        segment_reduce<TakeMax>(sets.seg, x, sets.id, lane, sh.top);
        wave_sync();
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            d[k] = __builtin_elementwise_maximum(x[k] - sh.top[sets.id[k] - 1], heat.low);
            v[k] = heat_exp<kExact<TYPE, BIAS>>(d[k], heat);
        }
        segment_reduce<TakeSum>(sets.seg, v, sets.id, lane, sh.first);
        if (!DISTILL) {
            float w[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k) w[k] = v[k] * d[k];
            segment_reduce<TakeSum>(sets.seg, w, sets.id, lane, sh.slope);
        }
        wave_sync();
    }
    if (DISTILL) {
        for (int it = 0; it < rounds; ++it) {
            const EntryLane l(a, in, it, lane);
            const int32_t c = l.there ? a.entry_index[l.g * a.top + l.j] : -1;
            const bool on = c >= 0 && c < l.size && sh.slot[l.begin + c] == l.j + 1;
            const float t = on ? entry_logit(a, l.g * a.top + l.j) : 0.0f;
            const float w = l.there ? (a.weights ? a.weights[l.g] : 1.0f) * a.scale : 0.0f;
            const Divergence r = diverge(a, on, on ? sh.x[l.begin + c] : -kInf, t, sh.top[l.s], l.size > 0 ? (double)sh.first[l.s] : 0.0,
                                         w, a.team_bits);
            wave_sync();
            if (on) sh.x[l.begin + c] = r.own;
            if (l.there && l.j == 0) {
                sh.first[l.s] = r.rest;
                a.kl[l.g] = (float)r.kl;
                if (w != 0.0f) tally[0] += (double)w * (double)a.temp * (double)a.temp * r.kl;
            }
        }
        wave_sync();
        float own[kRun];
        read_run(&sh.x[i0], own);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float f = sh.first[sets.id[k] - 1];
            v[k] = ((k < 4 ? slots.x : slots.y) >> (8 * (k & 3)) & 0xffu) ? own[k] : f == 0.0f ? 0.0f : f * v[k];
        }
    } else {
        Slopes f[kTileRounds];
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            const int s = r * kWave + lane;
            if (s < in.sets) {
                const float sum = in.end[r] > in.begin[r] ? sh.first[s] : 0.0f;
                if (sum == 0.0f) all.chosen[r] = -1;
                if (all.chosen[r] < 0) all.coef[r] = 0.0f;
                f[r] = slopes_of(a, (double)sum, sum != 0.0f ? (double)sh.slope[s] : 0.0, all.coef[r], all.h[r]);
                sh.first[s] = f[r].first;
                sh.slope[s] = f[r].slope;
            }
        }
        const float none[kRun] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        write_run(&sh.x[i0], none);
        wave_sync();
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r)
            if (r * kWave + lane < in.sets && all.chosen[r] >= 0)
                sh.x[in.begin[r] + all.chosen[r]] = (float)((double)all.coef[r] * a.inv_temp);
        wave_sync();
        float own[kRun];
        read_run(&sh.x[i0], own);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float f0 = sh.first[sets.id[k] - 1], f1 = sh.slope[sets.id[k] - 1];
            v[k] = v[k] * __builtin_fmaf(f1, d[k], f0) + own[k];
        }
    }
    if (off) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[k] = off >> k & 1u ? 0.0f : v[k];
    }
    if (sp.hi > 0) store_run<TYPE>(a, sp, 0, a.grad_scores, v);
    if (BIAS) table.add<false>(v, buckets);
}

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, DISTILL ? 3 : 4) void soft_tile_kernel(ReportArgs a) {
    __shared__ SoftTile tiles[kWaves];
    __shared__ BiasShared bias;
    __shared__ unsigned long long bins[BIAS ? kWaves : 1][kBins];
    __shared__ int shifts[BIAS ? kWaves : 1][kBins];
    __shared__ int bad[kMaxBuckets];
    __shared__ double shd[kWaves * 3];
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    TableSum table;
    if (BIAS) {
        for (int b = tid; b < kMaxBuckets; b += kBlock) bad[b] = 0;
        table.start(a, bins[wave], shifts[wave], bad);
        stage_bias(a, bias);
    }
    double tally[3] = {0.0, 0.0, 0.0};
    const int step = (int)gridDim.x * kWaves;
    int it = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + wave);
    SetItem next = a.tiles[min(it, a.num_tiles - 1)];
    SoftTileIn<DISTILL, TYPE, MASK, BIAS> in;
    while (it < a.num_tiles) {
        in.load(a, next, lane);
        next = a.tiles[min(it + step, a.num_tiles - 1)];
        soft_tile<DISTILL, TYPE, MASK, BIAS>(a, in, tiles[wave], &bias, table, tally);
        it += step;
    }
    leave_sums<DISTILL ? 1 : 0, BIAS>(a, (int)blockIdx.x, tally, table, bins, bad, shd);
}

// ------------------------------------------------------------------------------------ longer sets
// What a group of lanes (a wave, or a workgroup) shares of its set.
template <int THREADS, int RUNS>
struct SoftGroup {
    static constexpr int kGroupWaves = THREADS / kWave;
    uint8_t slot[THREADS * RUNS * kRun];  // the entry that names a row, from 1; 0: none
    float own[kMaxTop];
    float factor;
    float top[kGroupWaves];
    double sum[kGroupWaves], along[kGroupWaves];
};

template <int THREADS>
__device__ __forceinline__ void group_sync() {
    if (THREADS == kWave)
        wave_sync();
    else
        __syncthreads();
}

// A set's sums from those of the lanes (each wave's relative to its own maximum), the same in every lane.
template <bool ALONG, int THREADS, int RUNS>
__device__ __forceinline__ SoftSums join_waves(const ReportArgs& a, SoftSums t, SoftGroup<THREADS, RUNS>& sh) {
    if (THREADS == kWave) return t;
    const int tid = (int)threadIdx.x;
    if ((tid & (kWave - 1)) == 0) {
        sh.top[tid / kWave] = t.top;
        sh.sum[tid / kWave] = t.sum;
        if (ALONG) sh.along[tid / kWave] = t.along;
    }
    __syncthreads();
    SoftSums j{sh.top[0], 0.0, 0.0};
    for (int w = 1; w < THREADS / kWave; ++w) j.top = max2(j.top, sh.top[w]);
    for (int w = 0; w < THREADS / kWave; ++w) {
        const double gap = (double)sh.top[w] - (double)j.top, f = exp_near(gap * a.inv_temp);
        j.sum += sh.sum[w] * f;
        if (ALONG) j.along += f == 0.0 ? 0.0 : f * (sh.along[w] + sh.sum[w] * gap);
    }
    return j;
}

// A set's sums from those of its parts.
template <bool ALONG, int THREADS, int RUNS>
__device__ __forceinline__ SoftSums join_set(const ReportArgs& a, const SoftSums* parts, int n, SoftGroup<THREADS, RUNS>& sh) {
    SoftSums t{kLowest, 0.0, 0.0};
    for (int j = (int)threadIdx.x; j < n; j += THREADS) t.top = max2(t.top, parts[j].top);
    t.top = wave_max(t.top);
    for (int j = (int)threadIdx.x; j < n; j += THREADS) {
        const double gap = (double)parts[j].top - (double)t.top, f = exp_near(gap * a.inv_temp);
        t.sum += parts[j].sum * f;
        if (ALONG) t.along += f == 0.0 ? 0.0 : f * (parts[j].along + parts[j].sum * gap);
    }
    t.sum = team_sum(t.sum, 6);
    if (ALONG) t.along = team_sum(t.along, 6);
    return join_waves<ALONG>(a, t, sh);
}

enum SoftPhase { kWholeSet, kPartSums, kPartGrads };

// One set of more than kSetShort rows, or a part of one, by a group of THREADS lanes with RUNS runs each, in registers
// from the load to the store.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS, int THREADS, int RUNS, SoftPhase PHASE>
__device__ __forceinline__ void soft_pass(const ReportArgs& a, const SetItem& im, int32_t index, SoftGroup<THREADS, RUNS>& sh,
                                          const BiasShared* bias, TableSum& table, double (&tally)[3]) {
    constexpr bool EXACT = kExact<TYPE, BIAS>;
    const int tid = (int)threadIdx.x & (THREADS - 1), lane = tid & (kWave - 1);
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~(kWave - 1));  // the wave's first thread
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    const Span sp = span_of(a, im);
    const int64_t g = im.set0, r0 = a.off[g], size = a.off[g + 1] - r0;
    int32_t c = -1;
    if (DISTILL && wave0 == 0 && lane < a.top) c = a.entry_index[g * a.top + lane];
    RawRun<TYPE, MASK, BIAS> raw[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = kRun * (j * THREADS + tid);
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) raw[j].load(a, sp, i);
    }
    bool on = false;
    float z = -kInf, t = 0.0f, w = 0.0f;
    if (DISTILL) {
        group_sync<THREADS>();  // the last set's slots have been read
#pragma unroll
        for (int j = 0; j < RUNS; ++j) *reinterpret_cast<uint2*>(&sh.slot[kRun * (j * THREADS + tid)]) = make_uint2(0, 0);
        if (wave0 == 0) {
            on = c >= 0 && c < size;
            if (PHASE != kPartSums) {
                if (lane < a.top) t = entry_logit(a, g * a.top + lane);
                w = (a.weights ? a.weights[g] : 1.0f) * a.scale;
            }
            if (MASK && on) on = a.mask[r0 + c] != 0;
            if (PHASE != kPartSums) {
                if (on) z = one_logit<TYPE, BIAS>(a, bias, r0 + c);
                for (int j = 0; j + 1 < a.top; ++j) {  // rows named twice: the first entry counts
                    const int before = __builtin_amdgcn_readlane(c, j);
                    if (j < lane && before == c) on = false;
                }
                if (!on) z = -kInf;
            }
        }
        group_sync<THREADS>();
        const int64_t row = r0 + c - sp.q0;
        if (wave0 == 0 && on && row >= sp.lo && row < sp.hi) sh.slot[row] = (uint8_t)(lane + 1);
        group_sync<THREADS>();
    }
    float v[RUNS][kRun];
    uint32_t off[RUNS];
    Buckets buckets[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = kRun * (j * THREADS + tid);
        off[j] = 0xffu;
        buckets[j].w[0] = buckets[j].w[1] = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[j][k] = -kInf;
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) {
            raw[j].logits(a, bias, sp, i, v[j], off[j], buckets[j]);
            if (DISTILL) {
                const uint2 s = *reinterpret_cast<const uint2*>(&sh.slot[i]);
                if (s.x | s.y) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k) v[j][k] = ((k < 4 ? s.x : s.y) >> (8 * (k & 3)) & 0xffu) ? -kInf : v[j][k];
                }
            }
        }
    }
    const int live = sp.hi <= kRun * wave0 ? 0 : (sp.hi - kRun * wave0 + kRun * THREADS - 1) / (kRun * THREADS);  // the wave's runs
    SoftSums own{kLowest, 0.0, 0.0}, sums;
    if (PHASE == kPartGrads) {
        sums = join_set<!DISTILL>(a, a.part_sums + (index - im.part), im.parts, sh);
        own.top = sums.top;
    } else {
#pragma unroll
        for (int j = 0; j < RUNS; ++j)
            if (j < live)
#pragma unroll
                for (int k = 0; k < kRun; k += 2) own.top = max3(own.top, v[j][k], v[j][k + 1]);
        own.top = wave_max(own.top);
    }
    float sum = 0.0f, along = 0.0f;
#pragma unroll
    for (int j = 0; j < RUNS; ++j)
        if (j < live)
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const float d = __builtin_elementwise_maximum(v[j][k] - own.top, heat.low), e = heat_exp<EXACT>(d, heat);
                if (PHASE != kPartGrads) sum += e;
                if (!DISTILL && PHASE != kPartGrads) along = __builtin_fmaf(e, d, along);
                if (DISTILL && PHASE != kPartSums) v[j][k] = e;
            }
    if (PHASE != kPartGrads) {
        own.sum = team_sum((double)sum, 6);
        if (!DISTILL) own.along = team_sum((double)along, 6);
        sums = join_waves<!DISTILL>(a, own, sh);
    }
    if (PHASE == kPartSums) {
        if (tid == 0) a.part_sums[index] = sums;
        return;
    }
    // what the wave's exponentials are multiplied by: they are relative to its own maximum
    const double gap = (double)own.top - (double)sums.top;
    float first, slope = 0.0f, extra = 0.0f;
    int at = -kRun;  // the chosen row, as the span counts
    if (DISTILL) {
        if (wave0 == 0) {
            const Divergence r = diverge(a, on, z, t, sums.top, sums.sum, w, 6);
            sh.own[lane] = r.own;
            if (lane == 0) {
                sh.factor = r.rest;
                if (im.part == 0) {
                    a.kl[g] = (float)r.kl;
                    if (w != 0.0f) tally[0] += (double)w * (double)a.temp * (double)a.temp * r.kl;
                }
            }
        }
        group_sync<THREADS>();
        first = sh.factor == 0.0f ? 0.0f : (float)((double)sh.factor * exp_near(gap * a.inv_temp));
    } else {
        float coef = 0.0f;
        if (a.grad && sums.sum != 0.0) {
            const int32_t chosen = a.chosen[g];
            bool counts = chosen >= 0 && chosen < size;
            if (MASK && counts) counts = a.mask[r0 + chosen] != 0;
            if (counts) {
                coef = a.grad[g];
                extra = (float)((double)coef * a.inv_temp);
                const int64_t row = r0 + chosen - sp.q0;
                if (row >= sp.lo && row < sp.hi) at = (int)row;
            }
        }
        const Slopes f = slopes_of(a, sums.sum, sums.along, coef, a.grad_entropy ? a.grad_entropy[g] : 0.0f);
        const double near = exp_near(gap * a.inv_temp);
        slope = (float)((double)f.slope * near);
        first = near == 0.0 ? 0.0f : (float)(near * ((double)f.first + (double)f.slope * gap));
    }
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        if (j < live) {
            const int i = kRun * (j * THREADS + tid);
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                if (DISTILL) {
                    v[j][k] = first == 0.0f ? 0.0f : first * v[j][k];
                } else {
                    const float d = __builtin_elementwise_maximum(v[j][k] - own.top, heat.low);
                    v[j][k] = heat_exp<EXACT>(d, heat) * __builtin_fmaf(slope, d, first);
                }
            }
            if (DISTILL && i < sp.hi) {
                const uint2 s = *reinterpret_cast<const uint2*>(&sh.slot[i]);
                if (s.x | s.y) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k) {
                        const uint32_t b = (k < 4 ? s.x : s.y) >> (8 * (k & 3)) & 0xffu;
                        if (b) v[j][k] = sh.own[b - 1];
                    }
                }
            }
            if (!DISTILL && at >= i && at < i + kRun) {
#pragma unroll
                for (int k = 0; k < kRun; ++k)
                    if (at - i == k) v[j][k] += extra;
            }
            if ((MASK || BIAS) && off[j]) {
#pragma unroll
                for (int k = 0; k < kRun; ++k) v[j][k] = off[j] >> k & 1u ? 0.0f : v[j][k];
            }
            if (i < sp.hi) store_run<TYPE>(a, sp, i, a.grad_scores, v[j]);
            if (BIAS) table.add<false>(v[j], buckets[j]);
        }
    }
    if (THREADS != kWave) __syncthreads();  // the group's sums have been read
}

// The sums of the sets' parts.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void soft_part_kernel(ReportArgs a, int first, const int32_t* __restrict__ list) {
    __shared__ SoftGroup<kBlock, kWideRuns> sh;
    __shared__ BiasShared bias;
    const int it = list ? list[blockIdx.x] : first + (int)blockIdx.x;
    if (BIAS) stage_bias(a, bias);
    TableSum table;
    double tally[3];
    soft_pass<DISTILL, TYPE, MASK, BIAS, kBlock, kWideRuns, kPartSums>(a, a.wide[it], it, sh, &bias, table, tally);
}

// The longer sets: workgroups [0, mid_blocks) take those for a wave, the others those for a workgroup, then the parts (all
// from num_mid + num_whole on, or those in `list`), one at a time.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void soft_wide_kernel(ReportArgs a, int mid_blocks, int num_parts, const int32_t* __restrict__ list,
                                                           int first_block) {
    __shared__ union {
        SoftGroup<kWave, kWideRuns> mid[kWaves];
        SoftGroup<kBlock, kWideRuns> whole;
    } sh;
    __shared__ BiasShared bias;
    __shared__ unsigned long long bins[BIAS ? kWaves : 1][kBins];
    __shared__ int shifts[BIAS ? kWaves : 1][kBins];
    __shared__ int bad[kMaxBuckets];
    __shared__ double shd[kWaves * 3];
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    TableSum table;
    if (BIAS) {
        for (int b = tid; b < kMaxBuckets; b += kBlock) bad[b] = 0;
        table.start(a, bins[wave], shifts[wave], bad);
        stage_bias(a, bias);
    }
    double tally[3] = {0.0, 0.0, 0.0};
    if ((int)blockIdx.x < mid_blocks) {
        const int step = mid_blocks * kWaves;
        for (int it = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + wave); it < a.num_mid; it += step)
            soft_pass<DISTILL, TYPE, MASK, BIAS, kWave, kWideRuns, kWholeSet>(a, a.wide[it], it, sh.mid[wave], &bias, table, tally);
    } else {
        const int n = a.num_whole + num_parts;
        for (int k = (int)blockIdx.x - mid_blocks; k < n; k += (int)gridDim.x - mid_blocks) {
            if (k < a.num_whole) {
                soft_pass<DISTILL, TYPE, MASK, BIAS, kBlock, kWideRuns, kWholeSet>(a, a.wide[a.num_mid + k], 0, sh.whole, &bias, table, tally);
            } else {
                const int it = list ? list[k - a.num_whole] : a.num_mid + k;
                soft_pass<DISTILL, TYPE, MASK, BIAS, kBlock, kWideRuns, kPartGrads>(a, a.wide[it], it, sh.whole, &bias, table, tally);
            }
        }
    }
    leave_sums<DISTILL ? 1 : 0, BIAS>(a, first_block + (int)blockIdx.x, tally, table, bins, bad, shd);
}

int tile_blocks(const SetLayout& s) { return std::min((s.num_tiles + kWaves - 1) / kWaves, kChoiceGrid); }

int mid_blocks(const SetLayout& s) { return std::min((s.num_mid + kWaves - 1) / kWaves, kChoiceGrid); }

int group_blocks(const SetLayout& s) { return std::min(s.num_wide, kChoiceGrid); }

int num_parts(const SetLayout& s) { return s.num_wide - s.num_whole; }

int soft_blocks(const SetLayout& s) { return tile_blocks(s) + mid_blocks(s) + group_blocks(s); }

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
hipError_t launch_as(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    const int parts = num_parts(s), first = s.num_mid + s.num_whole;
    if (parts > 0) {
        hipLaunchKernelGGL((soft_part_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(parts), dim3(kBlock), 0, stream, a, first, nullptr);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (s.num_tiles > 0) {
        hipLaunchKernelGGL((soft_tile_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(tile_blocks(s)), dim3(kBlock), 0, stream, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int wide = mid_blocks(s) + group_blocks(s);
    if (wide > 0) {
        hipLaunchKernelGGL((soft_wide_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(wide), dim3(kBlock), 0, stream, a, mid_blocks(s), parts,
                           nullptr, tile_blocks(s));
        e = hipGetLastError();
    }
    return e;
}

template <bool DISTILL, int TYPE>
hipError_t launch_typed(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    if (a.mask)
        return a.table ? launch_as<DISTILL, TYPE, true, true>(s, a, stream) : launch_as<DISTILL, TYPE, true, false>(s, a, stream);
    return a.table ? launch_as<DISTILL, TYPE, false, true>(s, a, stream) : launch_as<DISTILL, TYPE, false, false>(s, a, stream);
}

template <bool DISTILL>
hipError_t launch_mode(const SetLayout& s, const ReportArgs& a, int32_t type, hipStream_t stream) {
    if (type == PB_BF16) return launch_typed<DISTILL, PB_BF16>(s, a, stream);
    if (type == PB_F16) return launch_typed<DISTILL, PB_F16>(s, a, stream);
    return launch_typed<DISTILL, PB_F32>(s, a, stream);
}

}  // namespace
}  // namespace pb
