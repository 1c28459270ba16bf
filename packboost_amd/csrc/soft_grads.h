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
// workgroup that holds them in registers (of up to 65536 rows where that pays, see kBigSets), what is longer still in parts
// that are read twice. A set's list is taken by as many
// lanes as it has entries, rounded up to a power of 2; a byte a row in LDS says which entry names it.
#pragma once

#include <algorithm>
#include <type_traits>

#include "soft_rows.h"

namespace pb {
namespace {

// A teacher's value as it lies in memory, asked for but not waited for, and what it stands for.
__device__ __forceinline__ uint32_t entry_bits(const ReportArgs& a, int64_t i) {
    return a.entry_type == PB_F32 ? static_cast<const uint32_t*>(a.entry_logits)[i] : (uint32_t)static_cast<const uint16_t*>(a.entry_logits)[i];
}

__device__ __forceinline__ float entry_value(const ReportArgs& a, uint32_t bits) {
    return a.entry_type == PB_F32 ? __uint_as_float(bits) : a.entry_type == PB_BF16 ? bf16_value(bits) : f16_value(bits);
}

__device__ __forceinline__ double inverse(double d) {
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// What a set's list says without the rows that are not listed: zmax the largest listed logit, e the sum of the listed rows'
// exp((z - zmax) / T), most the teacher's largest value (0 where that is -inf), mass the sum of the terms exp(t - most) (over
// T without tail), lost that of the terms times ((t - most) - (z - zmax) / T), and left, with tail, the sum of exp(t) itself, as far
// as it matters (see list_share), else mass. Terms over the largest are neither too small nor too large for what is divided by
// their sum, wherever the values lie. mass and lost are sums, in double, of the same terms, so that a term's rounding moves a
// divergence by its share of log (q / p) alone. In tiles the terms of e, and the sums over the rest, are float32, and
// the teacher's terms have a float32's digits.
struct ListSide {
    float zmax, most;
    double e, mass, left, lost;
};

// exp(t) of a log-probability. From 1 on the list leaves nothing to the rest, by however much.
__device__ __forceinline__ double list_share(double t) { return exp_near(t > 1.0 ? 1.0 : t); }

// e^x as a float's digits with a double's exponent: a term that is nothing beside the others counts where the student is as
// far off. Within 2^-22 of itself; -inf gives 0, NaN stays NaN.
__device__ __forceinline__ double list_exp(double x) {
    const double t = (x < -800.0 ? -800.0 : x) * 1.4426950408889634, k = __builtin_rint(t);
    return ldexp((double)__builtin_amdgcn_exp2f((float)(t - k)), (int)k);
}

// An entry's terms; z is -inf and t -inf where it does not count.
struct ListTerms {
    double e, part, lost;
    __device__ __forceinline__ ListTerms(const ReportArgs& a, float z, double t, float zmax) {
        const double x = ((double)z - (double)zmax) * a.inv_temp;
        e = exp_near(x);
        part = exp_near(t);
        lost = part == 0.0 ? 0.0 : part * (t - x);
    }
};

// The teacher's value as the terms take it.
__device__ __forceinline__ double entry_term(const ReportArgs& a, float t, float most) {
    return ((double)t - (double)most) * (a.tail ? 1.0 : a.inv_temp);
}

// What the rows' terms are multiplied by: a listed row's gradient is student e - teacher part, another's rest times its
// exponential over the rest's maximum. And the set's divergence, where it is asked for.
struct ListFactors {
    float student, teacher, rest;
    double kl;
};

// From the list's side and the rest's maximum and sum of exponentials; w is the set's weight times scale.
template <bool KL>
__device__ __forceinline__ ListFactors list_factors(const ReportArgs& a, const ListSide& l, float rest_top, double rest_sum, float w) {
    const bool has_rest = rest_sum != 0.0;
    const double gap = has_rest ? ((double)rest_top - (double)l.zmax) * a.inv_temp : -(double)kInf, up = fmax(gap, 0.0);
    const double less = exp_near(up == 0.0 ? gap : -up);  // of the two sides' exponentials one is 1
    const double ours = up == 0.0 ? 1.0 : less, theirs = up == 0.0 ? less : 1.0;
    const double total = l.e * ours + (has_rest ? rest_sum * theirs : 0.0);
    if (l.left == 0.0 || total == 0.0) return ListFactors{0.0f, 0.0f, 0.0f, 0.0};
    const bool open = a.tail && has_rest && l.left < 1.0;
    const double wt = (double)w * (double)a.temp, per_total = inverse(total), per = inverse(l.mass);
    const double share = open ? l.left : 1.0, rho = 1.0 - l.left;  // the list's sum of q; the rest's, where it is open
    ListFactors f{(float)(wt * ours * per_total), (float)(wt * share * per),
                  has_rest ? (float)(wt * (theirs * per_total - (open ? rho * inverse(rest_sum) : 0.0))) : 0.0f, 0.0};
    if (w == 0.0f) f.student = f.teacher = f.rest = 0.0f;
    if (KL) {  // one logarithm after the other: beside each other they take the registers of the rows
        __builtin_amdgcn_sched_barrier(0);
        const double log_total = log_near(total) + up;  // over the largest listed logit
        __builtin_amdgcn_sched_barrier(0);
        const double log_left = log_near(open ? rho : l.mass);
        __builtin_amdgcn_sched_barrier(0);
        f.kl = share * (l.lost * per + (open ? (double)l.most : -log_left) + log_total);
        if (open) f.kl += rho * (log_left - (gap + log_near(rest_sum) - log_total));
    }
    return f;
}

// A listed row's gradient. A set that counts for nothing has factors of 0, whatever its terms.
__device__ __forceinline__ float listed_grad(float student, float teacher, float e, float part) {
    return student == 0.0f && teacher == 0.0f ? 0.0f : student * e - teacher * part;
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
struct alignas(16) SoftTile {
    float x[kSetTileRows];        // logits, then what listed and chosen rows have of their own
    float top[kSetTileSets + 4];  // per set: maximum
    union {
        uint16_t head[kSetTileRows];    // the set that starts at a row, from 1; 0: none
        float first[kSetTileSets + 4];  // later: sum of exponentials, then what they are multiplied by
    };
    float slope[kSetTileSets + 4];  // entropies: sum of exponentials times distances, then slopes
};

struct alignas(16) ListTile : SoftTile {
    float part[kSetTileRows];    // of listed rows: the teacher's terms
    double left[kSetTileSets];   // with tail: the lists' sums of exp(t)
    uint8_t slot[kSetTileRows];  // the entry that names a row, from 1; 0: none
    float other[kSetTileSets + 4];  // slope and other: the list's largest logit and teacher's value, then factors
};

// How a wave takes the lists of a tile: a team of 1 << bits lanes to a set, as many as there are (64 sets at a time), each lane
// entry after entry, kGroup at a time. So the exponentials of 20 lists of 8 take one group and a reduction over 2 lanes.
constexpr int kGroup = 4;
struct ListWalk {
    int bits, rounds, groups;  // groups: of a round

    __device__ __forceinline__ ListWalk(const ReportArgs& a, int num_sets) {
        bits = num_sets > 32 ? 0 : num_sets > 1 ? __clz(num_sets - 1) - 26 : 6;
        bits = min(bits, a.team_bits);
        rounds = num_sets > kWave ? 2 : 1;
        groups = (((a.top + (1 << bits) - 1) >> bits) + kGroup - 1) / kGroup;
    }
    // entry u of a lane's group
    __device__ __forceinline__ int entry(int group, int u, int lane) const {
        return ((group * kGroup + u) << bits) + (lane & ((1 << bits) - 1));
    }
};
static_assert(kTileRounds == 2, "a lane has two sets of a tile");

// A lane's entries of a group, counted over the rounds.
struct EntryGroup {
    int32_t c[kGroup];
    uint32_t t[kGroup];

    __device__ __forceinline__ void load(const ReportArgs& a, const ListWalk& walk, int num_sets, const int32_t (&set)[kTileRounds],
                                         int index, int lane) {
        const bool upper = index >= walk.groups;
        const int team = lane >> walk.bits, group = upper ? index - walk.groups : index;
        const int64_t list = (int64_t)__shfl(upper ? set[1] : set[0], team) * a.top;
        const bool there = index < walk.rounds * walk.groups && (upper ? kWave : 0) + team < num_sets;
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            const int j = walk.entry(group, u, lane);
            c[u] = -1;
            t[u] = 0;
            if (there && j < a.top) {
                c[u] = a.entry_index[list + j];
                t[u] = entry_bits(a, list + j);
            }
        }
    }
};

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
struct SoftTileIn {
    TileRows<TYPE, MASK, BIAS> rows;
    int32_t chosen[kTileRounds];
    float coef[kTileRounds], h[kTileRounds], weight[kTileRounds];
    EntryGroup ahead[2];  // the first two groups

    __device__ __forceinline__ void load(const ReportArgs& a, const SetItem& im, int lane) {
        rows.load(a, im, lane);
        if (DISTILL) {
            const ListWalk walk(a, rows.sets);
            ahead[0].load(a, walk, rows.sets, rows.set, 0, lane);
            ahead[1].load(a, walk, rows.sets, rows.set, 1, lane);
        }
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            chosen[r] = -1;
            coef[r] = h[r] = 0.0f;
            weight[r] = 1.0f;
            if (r * kWave + lane < rows.sets) {
                const int64_t g = rows.set[r];
                if (DISTILL && a.weights) weight[r] = a.weights[g];
                if (!DISTILL && a.grad) {
                    chosen[r] = a.chosen[g];
                    coef[r] = a.grad[g];
                }
                if (!DISTILL && a.grad_entropy) h[r] = a.grad_entropy[g];
            }
        }
    }
};

// Where a round's set of the lane's team lies.
struct RoundSet {
    int s, begin, size, g, place;
    bool first;  // the team's first lane, of a set that is there

    template <class IN>
    __device__ __forceinline__ RoundSet(const ListWalk& walk, const IN& in, int round, int lane) {
        const int team = lane >> walk.bits;
        s = round * kWave + team;
        begin = __shfl(round ? in.begin[1] : in.begin[0], team);
        size = __shfl(round ? in.end[1] : in.end[0], team) - begin;
        g = __shfl(round ? in.set[1] : in.set[0], team);
        place = lane & ((1 << walk.bits) - 1);
        first = place == 0 && s < in.sets;
    }
};

// Marks the rows that a tile's lists name, and leaves each list's largest logit and teacher's value. With tail also its sum
// of exp(t), in double: 1 less that may be small. (All sums here or all in weigh_listed, where the rows' exponentials
// lie in registers, would take one wave a SIMD.)
template <bool MASK, class IN>
__device__ __forceinline__ void mark_listed(const ReportArgs& a, const ListWalk& walk, IN& all, ListTile& sh, int lane) {
    const auto& in = all.rows;
#pragma unroll 1
    for (int round = 0; round < walk.rounds; ++round) {
        const RoundSet r(walk, in, round, lane);
        float zmax = kLowest, tmax = -kInf;
        double left = 0.0;
#pragma unroll 1
        for (int group = 0; group < walk.groups; ++group) {
            const int index = round * walk.groups + group;
            EntryGroup e = index & 1 ? all.ahead[1] : all.ahead[0];
            if (index > 1) e.load(a, walk, in.sets, in.set, index, lane);
            bool on[kGroup];
            float z[kGroup];
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                on[u] = e.c[u] >= 0 && e.c[u] < r.size;
                const int row = on[u] ? r.begin + e.c[u] : 0;
                z[u] = sh.x[row];
                on[u] = on[u] && sh.slot[row] == 0;  // of entries that name one row the first counts
            }
            if (MASK) {
#pragma unroll
                for (int u = 0; u < kGroup; ++u)
                    if (on[u] && z[u] == -kInf) on[u] = a.mask[a.off[r.g] + e.c[u]] != 0;
            }
#pragma unroll
            for (int u = 0; u < kGroup; ++u)
                if (on[u]) sh.slot[r.begin + e.c[u]] = (uint8_t)(walk.entry(group, u, lane) + 1);
            wave_sync();
            bool lost = false;
#pragma unroll
            for (int u = 0; u < kGroup; ++u) lost = lost || (on[u] && sh.slot[r.begin + e.c[u]] != walk.entry(group, u, lane) + 1);
            if (__any(lost)) {  // entries of this group name one row: one after the other
#pragma unroll
                for (int u = 0; u < kGroup; ++u)
                    if (on[u]) sh.slot[r.begin + e.c[u]] = 0;
                wave_sync();
#pragma unroll
                for (int u = 0; u < kGroup; ++u) {
                    if (on[u]) on[u] = sh.slot[r.begin + e.c[u]] == 0;
                    const int named = on[u] ? e.c[u] : -1;
                    for (int d = 1; d < 1 << walk.bits; ++d) {
                        const int before = __shfl(named, lane >= d ? lane - d : lane);
                        if (d <= r.place && before == named) on[u] = false;
                    }
                    if (on[u]) sh.slot[r.begin + e.c[u]] = (uint8_t)(walk.entry(group, u, lane) + 1);
                    wave_sync();
                }
            }
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                zmax = on[u] ? fmaxf(zmax, z[u]) : zmax;
                tmax = on[u] ? fmaxf(tmax, entry_value(a, e.t[u])) : tmax;
            }
            if (a.tail) {
#pragma unroll
                for (int u = 0; u < kGroup; ++u) left += on[u] ? list_share((double)entry_value(a, e.t[u])) : 0.0;
            }
        }
        zmax = (float)team_max((double)zmax, walk.bits);
        tmax = (float)team_max((double)tmax, walk.bits);
        if (a.tail) left = team_sum(left, walk.bits);
        if (r.first) {
            sh.slope[r.s] = zmax;
            sh.other[r.s] = tmax;
            sh.left[r.s] = left;
        }
    }
}

// The terms of the listed rows, and the sets' factors and divergences.
template <class IN>
__device__ __forceinline__ void weigh_listed(const ReportArgs& a, const ListWalk& walk, IN& all, ListTile& sh, int lane,
                                             double (&tally)[3]) {
    const auto& in = all.rows;
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
#pragma unroll 1
    for (int round = 0; round < walk.rounds; ++round) {
        const RoundSet r(walk, in, round, lane);
        const float w = __shfl(round ? all.weight[1] : all.weight[0], lane >> walk.bits) * a.scale, tmax = sh.other[r.s];
        const float most = tmax > -kInf ? tmax : 0.0f;
        ListSide l{sh.slope[r.s], most, 0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
        for (int group = 0; group < walk.groups; ++group) {
            const int index = round * walk.groups + group;
            EntryGroup e = index & 1 ? all.ahead[1] : all.ahead[0];
            if (index > 1) e.load(a, walk, in.sets, in.set, index, lane);
#pragma unroll
            for (int u = 0; u < kGroup; ++u) {
                bool on = e.c[u] >= 0 && e.c[u] < r.size;
                const int row = on ? r.begin + e.c[u] : 0;
                on = on && sh.slot[row] == walk.entry(group, u, lane) + 1;
                const float z = on ? sh.x[row] : -kInf, t = on ? entry_value(a, e.t[u]) : -kInf;
                const float student = heat_exp(z - l.zmax, heat);
                const double term = entry_term(a, t, most), part = list_exp(term);
                if (on) {
                    sh.x[row] = student;
                    sh.part[row] = (float)part;
                }
                const double x = ((double)z - (double)l.zmax) * a.inv_temp;
                l.e += (double)student;
                l.mass += part;
                l.lost += part == 0.0 ? 0.0 : part * (term - x);
            }
        }
        l.e = team_sum(l.e, walk.bits);
        l.mass = team_sum(l.mass, walk.bits);
        l.lost = team_sum(l.lost, walk.bits);
        l.left = a.tail ? sh.left[min(r.s, kSetTileSets - 1)] : l.mass;
        const ListFactors f = list_factors<true>(a, l, r.size > 0 ? sh.top[r.s] : kLowest, r.size > 0 ? (double)sh.first[r.s] : 0.0, w);
        wave_sync();
        if (r.first) {
            sh.first[r.s] = f.rest;
            sh.slope[r.s] = f.student;
            sh.other[r.s] = f.teacher;
            a.kl[r.g] = (float)f.kl;
            if (w != 0.0f) tally[0] += (double)w * (double)a.temp * (double)a.temp * f.kl;
        }
    }
}

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ void soft_tile(const ReportArgs& a, SoftTileIn<DISTILL, TYPE, MASK, BIAS>& all,
                                          std::conditional_t<DISTILL, ListTile, SoftTile>& sh,
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
    if constexpr (DISTILL) *reinterpret_cast<uint2*>(&sh.slot[i0]) = make_uint2(0, 0);
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
    const ListWalk walk(a, DISTILL ? in.sets : 1);
    if constexpr (DISTILL) mark_listed<MASK>(a, walk, all, sh, lane);
    wave_sync();
    uint2 slots = make_uint2(0, 0);
    if constexpr (DISTILL) {
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
            sum += v[k] = heat_exp(d[k], heat);
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
            v[k] = heat_exp(d[k], heat);
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
    if constexpr (DISTILL) {
        weigh_listed(a, walk, all, sh, lane, tally);
        wave_sync();
        float e[kRun], part[kRun];
        slots = *reinterpret_cast<const uint2*>(&sh.slot[i0]);  // again: two registers less meanwhile
        const bool any = (slots.x | slots.y) != 0;
        if (any) {
            read_run(&sh.x[i0], e);
            read_run(&sh.part[i0], part);
        }
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const int s = sets.id[k] - 1;
            const float f = sh.first[s];
            v[k] = f == 0.0f ? 0.0f : f * v[k];
            if (any && ((k < 4 ? slots.x : slots.y) >> (8 * (k & 3)) & 0xffu)) v[k] = listed_grad(sh.slope[s], sh.other[s], e[k], part[k]);
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

// The tiles, one a wave at a time. Bound by instructions and by a tile's chain of loads, scans and sums at 3 or 4 waves a SIMD:
// 100 thousand masked sets of 24 rows with a bias 20 us (1175 vector instructions a tile, issued in 70 % of the time that
// four waves give them), with a teacher's lists of 8 39 us (2125, a third of them the lists' doubles).
template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, DISTILL ? 3 : 4) void soft_tile_kernel(ReportArgs a) {
    __shared__ std::conditional_t<DISTILL, ListTile, SoftTile> tiles[kWaves];
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
// What a group of lanes (a wave, or a workgroup) shares of its set. ROWS: 0 without lists.
template <int THREADS, int ROWS>
struct SoftGroup {
    uint8_t slot[ROWS ? ROWS : 8];  // the entry that names a row, from 1; 0: none
    float e[kMaxTop], part[kMaxTop];
    ListSide list;
    float weight;
    GroupSums<THREADS / kWave> sums;
};

template <int THREADS>
__device__ __forceinline__ void group_sync() {
    if (THREADS == kWave)
        wave_sync();
    else
        __syncthreads();
}

enum SoftPhase { kWholeSet, kPartSums, kPartGrads };

template <bool DISTILL, int THREADS, int RUNS>
constexpr int kListRows = DISTILL ? THREADS * RUNS * kRun : 0;

// One set of more than kSetShort rows, or a part of one, by a group of THREADS lanes with RUNS runs each, in registers
// from the load to the store. The first wave takes the list beside its rows; what the rest's sums add is little, and every
// lane forms it for itself, so that a set waits for its slots and for its sums alone.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS, int THREADS, int RUNS, SoftPhase PHASE>
__device__ __forceinline__ void soft_pass(const ReportArgs& a, const SetItem& im, int32_t index,
                                          SoftGroup<THREADS, kListRows<DISTILL, THREADS, RUNS>>& sh, const BiasShared* bias,
                                          TableSum& table, double (&tally)[3]) {
    constexpr bool EXACT = kExact<TYPE, BIAS>;
    const int tid = (int)threadIdx.x & (THREADS - 1), lane = tid & (kWave - 1);
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~(kWave - 1));  // the wave's first thread
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    const Span sp = span_of(a, im);
    const int64_t g = im.set0;
    int32_t c = -1;
    uint32_t bits = 0;
    float w = 1.0f;
    if (DISTILL && wave0 == 0 && lane < a.top) {
        c = a.entry_index[g * a.top + lane];
        if (PHASE != kPartSums) bits = entry_bits(a, g * a.top + lane);
    }
    if (DISTILL && wave0 == 0 && PHASE != kPartSums && a.weights) w = a.weights[g];
    const int64_t r0 = a.off[g], size = a.off[g + 1] - r0;
    RawRun<TYPE, MASK, BIAS> raw[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = kRun * (j * THREADS + tid);
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) raw[j].load(a, sp, i);
    }
    if (DISTILL) {
#pragma unroll
        for (int j = 0; j < RUNS; ++j) *reinterpret_cast<uint2*>(&sh.slot[kRun * (j * THREADS + tid)]) = make_uint2(0, 0);
        bool on = c >= 0 && c < size;
        float z = -kInf;
        if (wave0 == 0) {
            if (MASK && on) on = a.mask[r0 + c] != 0;
            if (PHASE != kPartSums && on) z = one_logit<TYPE, BIAS>(a, bias, r0 + c);
        }
        group_sync<THREADS>();
        if (wave0 == 0) {
            const int64_t row = r0 + c - sp.q0;
            const bool here = on && row >= sp.lo && row < sp.hi;
            if (here) sh.slot[row] = (uint8_t)(lane + 1);
            wave_sync();
            // rows named twice: the first entry counts. Of other parts' rows the slots do not tell.
            if (PHASE != kPartSums && (PHASE == kPartGrads || __any(here && sh.slot[row] != lane + 1))) {
                for (int j = 0; j + 1 < a.top; ++j) {
                    const int before = __builtin_amdgcn_readlane(c, j);
                    if (j < lane && before == c) on = false;
                }
                wave_sync();
                if (here && on) sh.slot[row] = (uint8_t)(lane + 1);
            }
        }
        group_sync<THREADS>();
        if (wave0 == 0 && PHASE != kPartSums) {
            if (!on) z = -kInf;
            const float t = on ? entry_value(a, bits) : -kInf;
            ListSide l;
            l.zmax = (float)team_max((double)(on ? fmaxf(kLowest, z) : kLowest), 6);
            const float tmax = (float)team_max((double)t, 6);
            l.most = tmax > -kInf ? tmax : 0.0f;
            const ListTerms terms(a, z, entry_term(a, t, l.most), l.zmax);
            l.e = team_sum(terms.e, 6);
            l.mass = team_sum(terms.part, 6);
            l.left = a.tail ? l.mass * list_share((double)l.most) : l.mass;
            l.lost = team_sum(terms.lost, 6);
            sh.e[lane] = (float)terms.e;
            sh.part[lane] = (float)terms.part;
            if (lane == 0) {
                sh.list = l;
                sh.weight = w * a.scale;
            }
        }
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
        sums = join_set<!DISTILL>(a, a.part_sums + (index - im.part), im.parts, sh.sums);
        own.top = sums.top;
    } else {
#pragma unroll
        for (int j = 0; j < RUNS; ++j)
            if (j < live)
#pragma unroll
                for (int k = 0; k < kRun; k += 2) own.top = max3(own.top, v[j][k], v[j][k + 1]);
        own.top = wave_max(own.top);
    }
    const HeatRows<EXACT> rows(own.top, heat);
    float sum = 0.0f, along = 0.0f;
#pragma unroll
    for (int j = 0; j < RUNS; ++j)
        if (j < live)
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                if (!DISTILL && PHASE == kPartGrads) continue;
                // without the sum along, -inf needs no bound
                const float d = DISTILL && !EXACT ? __builtin_fmaf(v[j][k], rows.hi, -rows.c) : rows.distance(v[j][k], heat);
                const float e = rows.exp(d, heat);
                if (PHASE != kPartGrads) sum += e;
                if (!DISTILL) along = __builtin_fmaf(e, d, along);
                if (DISTILL && PHASE != kPartSums) v[j][k] = e;
            }
    if (PHASE != kPartGrads) {
        const double all = team_sum((double)sum, 6), scale = (double)rows.scale();
        own.sum = all * scale;
        if (!DISTILL) own.along = (team_sum((double)along, 6) - all * (double)rows.shift) * (scale * rows.unit(heat));
        sums = join_waves<!DISTILL>(a, own, sh.sums);
    }
    if (PHASE == kPartSums) {
        if (tid == 0) a.part_sums[index] = sums;
        return;
    }
    // what the wave's exponentials are multiplied by: they are relative to its own maximum
    const double gap = (double)own.top - (double)sums.top;
    float first, slope = 0.0f, extra = 0.0f;
    ListFactors f{0.0f, 0.0f, 0.0f, 0.0};
    int at = -kRun;  // the chosen row, as the span counts
    if (DISTILL) {
        if (THREADS == kWave) wave_sync();
        f = list_factors<false>(a, sh.list, sums.top, sums.sum, sh.weight);
        first = f.rest == 0.0f ? 0.0f : (float)((double)f.rest * exp_near(gap * a.inv_temp) * (double)rows.scale());
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
        const Slopes t = slopes_of(a, sums.sum, sums.along, coef, a.grad_entropy ? a.grad_entropy[g] : 0.0f);
        const double near = exp_near(gap * a.inv_temp) * (double)rows.scale();
        const double step = rows.unit(heat);
        slope = (float)((double)t.slope * near * step);
        first = near == 0.0 ? 0.0f : (float)(near * ((double)t.first + (double)t.slope * (gap - (double)rows.shift * step)));
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
                    const float d = rows.distance(v[j][k], heat);
                    v[j][k] = rows.exp(d, heat) * __builtin_fmaf(slope, d, first);
                }
            }
            if (DISTILL && i < sp.hi) {
                const uint2 s = *reinterpret_cast<const uint2*>(&sh.slot[i]);
                if (s.x | s.y) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k) {
                        const uint32_t b = (k < 4 ? s.x : s.y) >> (8 * (k & 3)) & 0xffu;
                        if (b) v[j][k] = listed_grad(f.student, f.teacher, sh.e[b - 1], sh.part[b - 1]);
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
    if (DISTILL && tid == 0 && im.part == 0) {
        const double kl = list_factors<true>(a, sh.list, sums.top, sums.sum, sh.weight).kl;
        a.kl[g] = (float)kl;
        if (sh.weight != 0.0f) tally[0] += (double)sh.weight * (double)a.temp * (double)a.temp * kl;
    }
    group_sync<THREADS>();  // the group's sums and slots have been read
}

// The sums of the sets' parts: all from `first` on, or those in `list`. 40 MB of 10 million rows in 11 us, 3.6 TB/s: too short
// to reach a copy's rate.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void soft_part_kernel(ReportArgs a, int first, const int32_t* __restrict__ list) {
    __shared__ SoftGroup<kBlock, kListRows<DISTILL, kBlock, kWideRuns>> sh;
    __shared__ BiasShared bias;
    const int it = list ? list[blockIdx.x] : first + (int)blockIdx.x;
    if (BIAS) stage_bias(a, bias);
    TableSum table;
    double tally[3];
    soft_pass<DISTILL, TYPE, MASK, BIAS, kBlock, kWideRuns, kPartSums>(a, a.wide[it], it, sh, &bias, table, tally);
}

// The longer sets: workgroups [0, mid_blocks) take those for a wave, the others those for a workgroup, then the parts (all
// from num_mid + num_whole on, or those in `list`), one at a time. 30M bfloat16 rows of 17 thousand sets 45 us, by instructions
// (1118 a wave, 70 % of the time). The parts of 10 million rows of 300 sets with a teacher of 64 31 us, by the chain of a
// part, which takes its set's list and joins its parts' sums before it can write, in two rounds of workgroups. The waves a
// SIMD are those that registers allow without spills.
template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, BIAS ? 2 : MASK ? 3 : DISTILL || TYPE != PB_F32 ? 4 : 5) void soft_wide_kernel(ReportArgs a, int mid_blocks, int num_parts, const int32_t* __restrict__ list,
                                                           int first_block) {
    __shared__ union {
        SoftGroup<kWave, kListRows<DISTILL, kWave, kWideRuns>> mid[kWaves];
        SoftGroup<kBlock, kListRows<DISTILL, kBlock, kWideRuns>> whole;
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
        for (int it = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + wave); it < a.num_mid + a.num_shorts; it += step)
            soft_pass<DISTILL, TYPE, MASK, BIAS, kWave, kWideRuns, kWholeSet>(a, wave_item(a, it), it, sh.mid[wave], &bias, table, tally);
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

// Sets of up to THREADS * 64 rows, a workgroup each: rows that would be read twice in parts are read once. 4096 sets of 32
// thousand bfloat16 rows and a teacher of 16 in 110 us: 4.8 TB/s read and written, a large copy's rate.
template <bool DISTILL, int TYPE, bool MASK, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void soft_big_kernel(ReportArgs a, const SetItem* __restrict__ items, int first_block) {
    constexpr int kBigRuns = kSetBig / (1024 * kRun);
    __shared__ SoftGroup<THREADS, kListRows<DISTILL, THREADS, kBigRuns>> sh;
    TableSum table;
    double tally[3] = {0.0, 0.0, 0.0};
    soft_pass<DISTILL, TYPE, MASK, false, THREADS, kBigRuns, kWholeSet>(a, items[blockIdx.x], 0, sh, nullptr, table, tally);
    if (DISTILL && threadIdx.x == 0) {
        if (a.blocks == 1)
            a.stats[0] = (float)tally[0];
        else
            a.sums[first_block + (int)blockIdx.x] = tally[0];
    }
}

// Long sets have a workgroup each where nothing else is there for the kernels of parts (bfloat16 sets of 30 thousand rows,
// with a teacher / without: 16 sets 10.7 / 8.2 us, in parts 14.3 / 8.9; 256 14 / 11 and 22 / 17; 2048 58 / 55 and 100 / 80),
// and beside others from so many on: 512 take 21 / 18 us, and add 28 / 23 in parts; 256 add about as much as they take.
constexpr int kBigSets = 512;
constexpr int kOneLaunch = 256;  // as many of mixed lengths as fit beside each other go in one launch

bool takes_big(const SetLayout& s, bool bias) {
    const bool alone = s.num_mid + s.num_shorts + s.num_whole + s.num_giant == 0;
    return !bias && s.num_big > 0 && (alone || s.num_big >= kBigSets);
}

int tile_blocks(const SetLayout& s) { return s.num_shorts > 0 ? 0 : std::min((s.num_tiles + kWaves - 1) / kWaves, kChoiceGrid); }

int mid_blocks(const SetLayout& s) { return std::min((s.num_mid + s.num_shorts + kWaves - 1) / kWaves, kChoiceGrid); }

int num_parts(const SetLayout& s, bool bias) { return takes_big(s, bias) ? s.num_giant : s.num_wide - s.num_whole; }

int group_blocks(const SetLayout& s, bool bias) { return std::min(s.num_whole + num_parts(s, bias), kChoiceGrid); }

int soft_blocks(const SetLayout& s, bool bias) {
    return tile_blocks(s) + mid_blocks(s) + group_blocks(s, bias) + (takes_big(s, bias) ? s.num_big : 0);
}

template <bool DISTILL, int TYPE, bool MASK, bool BIAS>
hipError_t launch_as(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    const bool big = takes_big(s, BIAS);
    const int parts = num_parts(s, BIAS), first = s.num_mid + s.num_whole;
    const int32_t* list = big ? s.giant : nullptr;
    if (parts > 0) {
        hipLaunchKernelGGL((soft_part_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(parts), dim3(kBlock), 0, stream, a, first, list);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if constexpr (!BIAS) {
        const int half = s.num_half < s.num_big && s.num_big <= kOneLaunch ? 0 : s.num_half, first_block = a.blocks - s.num_big;
        if (big && s.num_big > half) {
            hipLaunchKernelGGL((soft_big_kernel<DISTILL, TYPE, MASK, 1024>), dim3(s.num_big - half), dim3(1024), 0, stream, a, s.big + half,
                               first_block + half);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        if (big && half > 0) {
            hipLaunchKernelGGL((soft_big_kernel<DISTILL, TYPE, MASK, 512>), dim3(half), dim3(512), 0, stream, a, s.big, first_block);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    if (tile_blocks(s) > 0) {
        hipLaunchKernelGGL((soft_tile_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(tile_blocks(s)), dim3(kBlock), 0, stream, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int wide = mid_blocks(s) + group_blocks(s, BIAS);
    if (wide > 0) {
        hipLaunchKernelGGL((soft_wide_kernel<DISTILL, TYPE, MASK, BIAS>), dim3(wide), dim3(kBlock), 0, stream, a, mid_blocks(s), parts,
                           list, tile_blocks(s));
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
