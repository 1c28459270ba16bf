// Learning from choices over ragged sets of candidate rows: grouped log-probabilities with a learned
// position bias, their backward, the clipped policy loss, and the sums of the preference loss.
//
// Set g holds rows [off[g], off[g + 1]). Row i's logit is x_i = score_i + table[bucket(position_i)],
// -inf where its mask is 0. With m = max x (0 where that is -inf) and s = sum exp(x - m) over the set,
// lse = m + log s and log p_i = (x_i - m) - log s; a set without probability (empty, all masked) has
// s = 0 and lse = -inf. The gradient of a step's log p_c is [i = c] - p_i, of all rows' d_i - p_i sum d.
//
// Work is laid out once per table of sets. A wavefront takes a tile of short sets, 8 rows a lane, and
// reduces them by a segmented scan over the lanes, whose cost does not depend on how the rows fall into
// sets; a wave or a workgroup takes one longer set, or a part of it, in registers. Parts of a set are
// reduced by a pass before (part_kernel). All of it is bound by memory at best: a row has 8 to 20 bytes and
// some 20 operations, so every row is read once, in 16-byte accesses, and scores, masks, positions and what
// the sets have are asked for before anything is waited for (teams of lanes that walked each set's rows in
// LDS took 15 us for tiles that take 5 to 7 us so). Every sum has a fixed order (lanes, waves, workgroups), so
// results do not change from run to run. Maxima, sums of exponentials and log-probabilities are float32;
// losses, the table's gradient and sequences' sums are joined in double, each rounded once when it is written.
#include <algorithm>

#include "choice_rows.h"

namespace pb {
namespace {

// Values are laid beside their references first where both are many: the two arrays pass an XCD's 4 MB of
// L2, and a pair's four reads become two (us a call, so / without: 1M values, 4M pairs 207 / 259; 512k, 512k
// 39 / 42; 128k, 512k 35 / 37; with fewer pairs the launch costs more: 256k, 256k 25 / 22; 128k, 128k 21 / 18).
constexpr int64_t kBothValues = 1 << 17, kBothPairs = 1 << 19;
constexpr int kJoin = 8;
constexpr int kPairs = 4;  // pairs a thread has in flight

template <int MODE, int TYPE, bool BIAS>
__device__ __forceinline__ float row_exp(float x) {
    constexpr bool GRAD = MODE == kRowsBack || MODE == kStepsBack || MODE == kPolicy;
    return GRAD && (TYPE == PB_F32 || BIAS) ? close_exp(x) : exp_of(x);
}

// Backward passes take a set's probabilities as exp(x - lse), from an lse that is rounded: all of them are off
// by up to |lse| 2^-24 of themselves, 2^-20 at kFarLse (where a set of ordinary scores stays below). A common
// offset of the scores, which a softmax does not see, must not grow that. So beyond kFarLse the exponentials of
// the set are summed anew and divided by their sum, which costs sets in parts another reading of them.
constexpr float kFarLse = 16.0f;
__device__ __forceinline__ bool far_lse(float lse) { return __builtin_fabsf(lse) >= kFarLse && __builtin_fabsf(lse) < kInf; }

// The clipped loss of a step and its slope: surrogate min(rA, clip(r) A) with r = exp(lp - old), and
// kl = e^d - d - 1 with d = ref - lp. A NaN ratio takes no bound, so it stays visible.
struct PolicyIn {
    float adv, old, ref, w;
};

__device__ __forceinline__ PolicyIn load_policy(const ChoiceArgs& a, int64_t g) {
    return PolicyIn{a.advantages[g], a.old[g], a.ref ? a.ref[g] : 0.0f, a.weights ? a.weights[g] : 1.0f};
}

// A step's gradient with respect to its log-probability lp, and its part of the sums. Ratio and KL term may
// overflow: where their weight, kl_weight or advantage is 0 they count for nothing all the same.
__device__ __forceinline__ float policy_step(const ChoiceArgs& a, const PolicyIn& in, double lp, bool tally, double (&sum)[3]) {
    const float w = in.w * a.scale;
    const float ratio = FineExp(lp - (double)in.old).all;
    const float free = in.adv == 0.0f && ratio == kInf ? 0.0f : ratio * in.adv;
    const float held = fminf(fmaxf(ratio, a.ratio_min), a.ratio_max) * in.adv;
    const bool clipped = free > held;
    float kl = 0.0f, term = 0.0f, slope = clipped ? 0.0f : -free;
    if (a.ref) {
        const FineExp e((double)in.ref - lp);
        kl = e.less_line;
        if (a.kl_weight != 0.0f) {
            term = a.kl_weight * kl;
            slope -= a.kl_weight * e.less_one;
        }
    }
    if (tally) {
        sum[0] += w == 0.0f ? 0.0 : (double)(w * (term - (clipped ? held : free)));
        sum[1] += w == 0.0f ? 0.0 : (double)(w * kl);
        sum[2] += clipped ? (double)w : 0.0;
    }
    return w == 0.0f ? 0.0f : w * slope;
}

// The maximum and the sum of exponentials of a part of a set. 11 vector instructions a row and one barrier: bound
// by reading the rows (4096 sets of 32000 bfloat16 scores, 262 MB: 60 us, 4.4 TB/s).
template <int MODE, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void part_kernel(ChoiceArgs a, int first) {
    __shared__ Soft sh[kWaves];
    __shared__ BiasShared bias;
    const int it = first + (int)blockIdx.x;
    const Span s = span_of(a, a.wide[it]);
    if (BIAS) stage_bias(a, bias);
    float v[kWideRuns][kRun];
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j) {
        const int i = kRun * (j * kBlock + (int)threadIdx.x);
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[j][k] = -kInf;
        if (i < s.hi) {
            uint32_t off;
            Buckets buckets;
            load_logits<TYPE, MASK, BIAS>(a, &bias, s, i, v[j], off, buckets);
        }
    }
    float top = kLowest, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j)
#pragma unroll
        for (int k = 0; k < kRun; k += 2) top = max3(top, v[j][k], v[j][k + 1]);
    top = wave_max(top);
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j)
#pragma unroll
        for (int k = 0; k < kRun; ++k) sum += exp_of(v[j][k] - top);
    const Soft t = block_soft(Soft{top, wave_sum(sum)}, sh);
    if (threadIdx.x == 0) a.parts[it] = make_float2(t.top, t.sum);
}

// The sum of a part's rows' gradients.
template <bool MASK>
__global__ __launch_bounds__(kBlock) void part_grads_kernel(ChoiceArgs a, int first) {
    __shared__ float shf[kWaves];
    const int it = first + (int)blockIdx.x;
    const Span s = span_of(a, a.wide[it]);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j) {
        const int i = kRun * (j * kBlock + (int)threadIdx.x);
        float v[kRun] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (i < s.hi) {
            uint32_t off = outside(s, i);
            if (MASK) {
                const uint32_t out = off;
                for (int k = 0; k < kRun; ++k)
                    if (!(out >> k & 1u) && !a.mask[s.q0 + i + k]) off |= 1u << k;
            }
            load_floats(a, s, i, a.grad, off, v);
        }
#pragma unroll
        for (int k = 0; k < kRun; ++k) sum += v[k];
    }
    sum = block_sum(sum, shf);
    if (threadIdx.x == 0) a.parts[it].y = sum;
}

// The sum of exp(x - lse) of the parts [first, first + n) whose set's lse is far (far_lse). A workgroup looks at
// 64 of its parts at a time, a lane each, so that a table without such sets costs a launch (16384 parts: 4.7 us, and
// 42 more where all are: 4096 sets of 32000 in bfloat16).
template <int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void part_far_kernel(ChoiceArgs a, int first, int n) {
    __shared__ float shf[kWaves];
    __shared__ BiasShared bias;
    const int lane = (int)threadIdx.x & (kWave - 1), step = (int)gridDim.x;
    bool staged = false;
    for (int64_t i0 = blockIdx.x; i0 < n; i0 += (int64_t)step * kWave) {
        const int64_t mine = i0 + (int64_t)step * lane;
        unsigned long long far = __ballot(mine < n && far_lse(a.lse[a.wide[first + (mine < n ? mine : 0)].set0]));
        for (; far; far &= far - 1) {  // the same in all waves
            const int it = first + (int)(i0 + (int64_t)step * (__ffsll((long long)far) - 1));
            const SetItem im = a.wide[it];
            const Span s = span_of(a, im);
            const float lse = a.lse[im.set0];
            if (BIAS && !staged) stage_bias(a, bias);
            staged = true;
            float sum = 0.0f;
#pragma unroll 1
            for (int j = 0; j < kWideRuns; ++j) {
                const int i = kRun * (j * kBlock + (int)threadIdx.x);
                if (i < s.hi) {
                    float v[kRun];
                    uint32_t off;
                    Buckets buckets;
                    load_logits<TYPE, MASK, BIAS>(a, &bias, s, i, v, off, buckets);
#pragma unroll
                    for (int k = 0; k < kRun; ++k) sum += exp_of(v[k] - lse);
                }
            }
            sum = block_sum(sum, shf);
            if (threadIdx.x == 0) a.parts[it].x = sum;
        }
    }
}

// What a wave keeps of its tile in LDS.
struct TileShared {
    float x[kSetTileRows];          // logits, then what the chosen rows' gradients are more than the others'
    float shift[kSetTileSets + 4];  // per set: maximum, or lse
    union {
        uint16_t head[kSetTileRows];  // the set that starts at a row, from 1; 0: none
        float factor[kSetTileSets + 4];  // later: sum of exponentials, then what the rows' are multiplied by
    };
};

// What a tile reads, asked for before anything is waited for: a lane's run, and the lane's sets. (The rows' given
// gradients, of the rows' backward, are asked for when the logits have come.)
template <int MODE, int TYPE, bool MASK, bool BIAS>
struct TileIn {
    Span sp;   // of the lane's run alone
    int sets;
    RawRun<TYPE, MASK, BIAS> raw;
    int32_t set[kTileRounds], begin[kTileRounds], end[kTileRounds], chosen[kTileRounds];  // begin, end: rows of the tile
    float given[kTileRounds], lse[kTileRounds];
    PolicyIn pol[kTileRounds];

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
            const int64_t g = set[r];
            chosen[r] = -1;
            given[r] = lse[r] = 0.0f;
            if (r * kWave + lane < sets) {
                begin[r] = (int)(a.off[g] - base[r]);
                end[r] = (int)(a.off[g + 1] - base[r]);
                if (MODE != kRows && MODE != kRowsBack) chosen[r] = a.chosen[g];
                if (MODE == kStepsBack) given[r] = a.grad[g];
                if (MODE == kStepsBack || MODE == kRowsBack) lse[r] = a.lse[g];
                if (MODE == kPolicy) pol[r] = load_policy(a, g);
            }
        }
    }
};

// One tile of short sets by one wave: the maximum and the sum of exponentials by two segmented scans, which
// leave them in LDS by set; a lane to a set then forms log-probabilities, losses and slopes, 64 sets at a
// time; the rows take their set's factor from LDS. A tile of one set has no need of the scans (policy steps
// of 30000 sets of 300 rows: 37 us, 44 with them; 68 and 76 for steps in float32 with their backward). With mask and
// bias a tile of 512 rows takes 504 vector instructions for the steps, 814 for their backward and 1465 for the
// policy; a SIMD issues in 45 to 47 % of the time, and waves wait for half of theirs. So what bounds a few
// thousand tiles is the chain from the loads to the stores, of one tile a wave, and how many waves are resident:
// four a SIMD in the policy's, whose last workgroups run a second round. 2.4M rows of 100k sets: steps 9.1 us, their
// backward with the table's gradient 14.0 us; the policy loss of 480k sets 25.4 us. Tens of thousands of tiles
// issue in 69 % (40M rows in bfloat16: 43.5 us).
template <int MODE, int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ void tile_pass(const ChoiceArgs& a, TileIn<MODE, TYPE, MASK, BIAS>& in, TileShared& sh,
                                          const BiasShared* bias, TableSum& table, double (&tally)[3]) {
    constexpr bool GRAD = MODE == kRowsBack || MODE == kStepsBack || MODE == kPolicy;
    constexpr bool STEPS = MODE != kRows && MODE != kRowsBack;
    constexpr bool SOFT = MODE == kRows || MODE == kSteps || MODE == kPolicy;
    const int lane = (int)threadIdx.x & (kWave - 1);
    const Span sp = in.sp;
    const int i0 = kRun * lane;
    const bool alone = in.sets == 1;
    float x[kRun], d[kRun];
    uint32_t off = 0xffu;
    Buckets buckets{{0, 0}};
#pragma unroll
    for (int k = 0; k < kRun; ++k) x[k] = -kInf, d[k] = 0.0f;
    if (sp.hi > 0) {
        in.raw.logits(a, bias, sp, 0, x, off, buckets);
        if (MODE == kRowsBack) load_floats(a, sp, 0, a.grad, off, d);
    }
    const int32_t (&begin)[kTileRounds] = in.begin;
    const int32_t (&end)[kTileRounds] = in.end;
    int32_t (&chosen)[kTileRounds] = in.chosen;
    wave_sync();  // the last tile's values have been read
    if (!alone) *reinterpret_cast<uint4*>(&sh.head[i0]) = make_uint4(0, 0, 0, 0);
    if (STEPS) write_run(&sh.x[i0], x);
    if (!SOFT) {
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r)
            if (r * kWave + lane < in.sets) sh.shift[r * kWave + lane] = in.lse[r];
    }
    wave_sync();
    // which set each row is of, and the chosen rows' logits (a choice outside its set or masked is none)
    float picked[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        if (s < in.sets) {
            if (!alone && end[r] > begin[r]) sh.head[begin[r]] = (uint16_t)(s + 1);
            if (STEPS) {
                if (chosen[r] >= end[r] - begin[r]) chosen[r] = -1;
                picked[r] = chosen[r] >= 0 ? sh.x[begin[r] + chosen[r]] : -kInf;
                // a masked row's logit is -inf, as one of that score is: the mask says which
                if (MASK && chosen[r] >= 0 && picked[r] == -kInf && !a.mask[a.off[in.set[r]] + chosen[r]]) chosen[r] = -1;
            }
        }
    }
    wave_sync();
    // What a set's exponentials over a far lse sum to, 1 where that is not asked for: every gradient is divided by it.
    // (With the division under a branch on whether the tile has such a set, the compiler dropped the other
    // branch's sign.) Lanes walk the sets' logits: scans would take registers from tables without such sets.
    float anew[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) anew[r] = 1.0f;
    if (!SOFT) {
        bool far = false;
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) far = far || (r * kWave + lane < in.sets && far_lse(in.lse[r]));
        if (__any(far)) {
            if (!STEPS) {
                write_run(&sh.x[i0], x);
                wave_sync();
            }
            // as many lanes to a set as there are (8M rows in sets of 30 to 400: 21 to 23 us, 18 to 19 without far sets; by
            // a lane to a set 26 to 133)
            if (in.sets <= kWave / 2) {
                const int bits = in.sets > 1 ? __clz(in.sets - 1) - 26 : 6, team = lane >> bits, from = min(team, in.sets - 1);
                const int e = __shfl(end[0], from);
                const float lse = __shfl(in.lse[0], from);
                double t = 0.0;
                for (int i = __shfl(begin[0], from) + (lane & ((1 << bits) - 1)); i < e; i += 1 << bits) t += (double)exp_of(sh.x[i] - lse);
                for (int m = 1; m < 1 << bits; m *= 2) t += __shfl_xor(t, m);
                t = __shfl(t, (lane << bits) & (kWave - 1));
                if (lane < in.sets && far_lse(in.lse[0])) anew[0] = (float)t;
            } else {
#pragma unroll
                for (int r = 0; r < kTileRounds; ++r)
                    if (r * kWave + lane < in.sets && far_lse(in.lse[r])) {
                        double t = 0.0;
                        for (int i = begin[r]; i < end[r]; ++i) t += (double)exp_of(sh.x[i] - in.lse[r]);
                        anew[r] = (float)t;
                    }
            }
            wave_sync();
        }
    }
    int id[kRun];
    float v[kRun];
    if (alone) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) id[k] = 1;
        if (SOFT) {
            float top = TakeMax::kNone, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kRun; k += 2) top = max3(top, x[k], x[k + 1]);
            top = wave_max(top);
#pragma unroll
            for (int k = 0; k < kRun; ++k) sum += v[k] = row_exp<MODE, TYPE, BIAS>(x[k] - top);
            sum = wave_sum(sum);
            if (lane == 0) {
                sh.shift[0] = top;
                sh.factor[0] = sum;
            }
        }
        if (MODE == kRowsBack) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kRun; ++k) sum += d[k];
            sum = wave_sum(sum);
            if (lane == 0) sh.factor[0] = sum;
        }
        wave_sync();
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(&sh.head[i0]);
        const int raw[kRun] = {(int)(w.x & 0xffffu), (int)(w.x >> 16), (int)(w.y & 0xffffu), (int)(w.y >> 16),
                               (int)(w.z & 0xffffu), (int)(w.z >> 16), (int)(w.w & 0xffffu), (int)(w.w >> 16)};
        int last = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) last = raw[k] ? raw[k] : last;
        // the set that the rows before the lane's first head are of: the last head's below
        const unsigned long long below = __ballot(last != 0) & ((1ull << lane) - 1ull);
        const int from = below ? kWave - 1 - __clzll((long long)below) : lane;
        const int carried = __shfl(last, from);
        int now = below ? carried : kSetTileSets + 1;  // before the first set: a slot of none
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            now = raw[k] ? raw[k] : now;
            id[k] = now;
        }
        Segments seg;
        if (SOFT || MODE == kRowsBack) seg.start(raw, lane);
        if (SOFT) {
            segment_reduce<TakeMax>(seg, x, id, lane, sh.shift);
            wave_sync();
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] = row_exp<MODE, TYPE, BIAS>(x[k] - sh.shift[id[k] - 1]);
            segment_reduce<TakeSum>(seg, v, id, lane, sh.factor);
            wave_sync();
        }
        if (MODE == kRowsBack) {
            segment_reduce<TakeSum>(seg, d, id, lane, sh.factor);
            wave_sync();
        }
    }
    // a lane to a set: log-probabilities, losses, slopes
    float coef[kTileRounds];
    if (SOFT || STEPS) {
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) {
            const int s = r * kWave + lane;
            coef[r] = 0.0f;
            if (s < in.sets) {
                const int64_t g = in.set[r];
                const bool empty = end[r] == begin[r];
                const float top = SOFT ? (empty ? 0.0f : sh.shift[s]) : in.lse[r];
                const float sum = SOFT && !empty ? sh.factor[s] : 0.0f;
                const float ls = SOFT ? log_of(sum) : 0.0f;
                if (MODE == kRows || MODE == kSteps) a.lse_out[g] = top + ls;
                if (MODE == kRows) {
                    sh.shift[s] = top;
                    sh.factor[s] = ls;
                }
                if (STEPS) {
                    // left out: a choice outside the set or masked, a set without probability
                    const bool counts = chosen[r] >= 0 && (SOFT ? sum != 0.0f : top != -kInf);
                    float lp = SOFT && counts ? (picked[r] - top) - ls : 0.0f;
                    if (MODE == kStepsBack && counts) coef[r] = in.given[r];
                    if (MODE == kPolicy && counts) {
                        const double fine = ((double)picked[r] - (double)top) - fine_log(sum);
                        lp = (float)fine;
                        coef[r] = policy_step(a, in.pol[r], fine, true, tally);
                    }
                    if (SOFT) a.log_probs[g] = lp;
                    if (GRAD) sh.factor[s] = counts ? (SOFT ? -coef[r] * __builtin_amdgcn_rcpf(sum) : -coef[r] / anew[r]) : 0.0f;
                    if (!counts) chosen[r] = -1;
                }
            }
        }
    }
    if (MODE == kSteps) return;
    if (MODE == kRowsBack) {
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r)
            if (r * kWave + lane < in.sets && end[r] > begin[r]) sh.factor[r * kWave + lane] /= anew[r];
    }
    if (STEPS) {  // the chosen rows' own part
        const float none[kRun] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        write_run(&sh.x[i0], none);
        wave_sync();
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r)
            if (r * kWave + lane < in.sets && chosen[r] >= 0) sh.x[begin[r] + chosen[r]] = coef[r];
    }
    wave_sync();
    if (MODE == kRows) {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
            v[k] = x[k] == -kInf ? -kInf : (x[k] - sh.shift[id[k] - 1]) - sh.factor[id[k] - 1];
    }
    if (MODE == kRowsBack) {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
            v[k] = d[k] - (x[k] == -kInf ? 0.0f : row_exp<MODE, TYPE, BIAS>(x[k] - sh.shift[id[k] - 1]) * sh.factor[id[k] - 1]);
    }
    if (STEPS) {
        float own[kRun];
        read_run(&sh.x[i0], own);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float f = sh.factor[id[k] - 1];
            const float e = SOFT ? v[k] : row_exp<MODE, TYPE, BIAS>(x[k] - sh.shift[id[k] - 1]);
            v[k] = (f == 0.0f ? 0.0f : f * e) + own[k];
        }
    }
    if (GRAD && off) {
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[k] = off >> k & 1u ? 0.0f : v[k];
    }
    if (sp.hi > 0) {
        if (MODE == kRows)
            store_run<PB_F32>(a, sp, 0, a.log_probs, v);
        else
            store_run<TYPE>(a, sp, 0, a.grad_scores, v);
    }
    if (BIAS && GRAD) table.add<MODE == kPolicy>(v, buckets);
}

// One set of more than kSetShort rows by a wave (THREADS 64), or a longer one or a part of it by a
// workgroup. A wave passes over runs beyond its rows. The rows stay in registers from the load to the
// store, one exponential each, so that a set of up to kSetWideRows rows is read once; a longer one's parts are
// read a second time. Bound by memory for sets of thousands of rows (backward of 4096 sets of 32000
// bfloat16 scores, 524 MB: 87.5 us, 6.0 TB/s), by the instructions a set takes beside its rows (about 250)
// for hundreds (100k policy steps, 29M of their 40M rows here: 42.4 us, 2.7 TB/s).
template <int MODE, int TYPE, bool MASK, bool BIAS, int THREADS>
__device__ __forceinline__ void wide_pass(const ChoiceArgs& a, const SetItem& im, int32_t index, Soft* shs, float* shf,
                                          const BiasShared* bias, TableSum& table, double (&tally)[3]) {
    constexpr bool GRAD = MODE == kRowsBack || MODE == kStepsBack || MODE == kPolicy;
    constexpr bool STEPS = MODE != kRows && MODE != kRowsBack;
    constexpr bool SOFT = MODE == kRows || MODE == kSteps || MODE == kPolicy;
    constexpr bool ALONE = THREADS == kWave;
    const int tid = (int)threadIdx.x & (THREADS - 1);
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~(kWave - 1));  // the wave's first thread
    const Span sp = span_of(a, im);
    const int64_t g = im.set0;
    const bool first = im.part == 0 && tid == 0;
    // the parts' sums first, then the rows: the ones are joined while the others are on their way
    Soft joined{kLowest, 0.0f};
    if (SOFT && !ALONE && im.parts > 1) joined = join_parts(a.parts + (index - im.part), im.parts, tid, THREADS);
    RawRun<TYPE, MASK, BIAS> raw[kWideRuns];
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j) {
        const int i = kRun * (j * THREADS + tid);
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) raw[j].load(a, sp, i);
    }
    // what the set has beside its rows, asked for with them
    const float lse = SOFT ? 0.0f : a.lse[g];
    const int64_t r0 = STEPS ? a.off[g] : 0, size = STEPS ? a.off[g + 1] - r0 : 0;
    const int32_t c = STEPS ? a.chosen[g] : -1;
    const float given = MODE == kStepsBack ? a.grad[g] : 0.0f;
    PolicyIn pol{0.0f, 0.0f, 0.0f, 0.0f};
    if (MODE == kPolicy) pol = load_policy(a, g);
    bool counts = STEPS && c >= 0 && c < size;
    float xc = 0.0f;
    if (STEPS && counts) {
        if (MASK) counts = a.mask[r0 + c] != 0;
        if (SOFT) xc = one_logit<TYPE, BIAS>(a, bias, r0 + c);
    }
    Soft t{0.0f, 0.0f};
    if (SOFT && !ALONE && im.parts > 1) t = block_soft(wave_soft(joined), shs);
    float v[kWideRuns][kRun], d[kWideRuns][kRun];
    uint32_t off[kWideRuns];
    Buckets buckets[kWideRuns];
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j) {
        const int i = kRun * (j * THREADS + tid);
        off[j] = 0xffu;
        buckets[j].w[0] = buckets[j].w[1] = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[j][k] = -kInf, d[j][k] = 0.0f;
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) {
            raw[j].logits(a, bias, sp, i, v[j], off[j], buckets[j]);
            if (MODE == kRowsBack) load_floats(a, sp, i, a.grad, off[j], d[j]);
        }
    }
    const int live = sp.hi <= kRun * wave0 ? 0 : (sp.hi - kRun * wave0 + kRun * THREADS - 1) / (kRun * THREADS);  // the wave's runs
    float own = 1.0f;  // what the wave's exponentials are relative to, over the set's maximum
    if (SOFT) {
        Soft w;
        if (!ALONE && im.parts > 1) {
            w.top = t.top;
        } else {
            w.top = kLowest;
#pragma unroll
            for (int j = 0; j < kWideRuns; ++j)
                if (j < live)
#pragma unroll
                    for (int k = 0; k < kRun; k += 2) w.top = max3(w.top, v[j][k], v[j][k + 1]);
            w.top = wave_max(w.top);
        }
        w.sum = 0.0f;
        if (ALONE || im.parts == 1 || GRAD) {
#pragma unroll
            for (int j = 0; j < kWideRuns; ++j)
                if (j < live)
#pragma unroll
                    for (int k = 0; k < kRun; ++k) {
                        const float e = row_exp<MODE, TYPE, BIAS>(v[j][k] - w.top);
                        w.sum += e;
                        if (GRAD) v[j][k] = e;
                    }
        }
        if (ALONE || im.parts == 1) {
            w.sum = wave_sum(w.sum);
            t = ALONE ? w : block_soft(w, shs);
            if (GRAD && !ALONE) own = row_exp<MODE, TYPE, BIAS>(w.top - t.top);
        }
    }
    const float ls = SOFT ? log_of(t.sum) : 0.0f;
    if ((MODE == kRows || MODE == kSteps) && first) a.lse_out[g] = t.top + ls;
    if (MODE == kRows) {
#pragma unroll
        for (int j = 0; j < kWideRuns; ++j)
            if (j < live)
#pragma unroll
                for (int k = 0; k < kRun; ++k) v[j][k] = v[j][k] == -kInf ? -kInf : (v[j][k] - t.top) - ls;
    }
    float anew = 1.0f;  // what the exponentials over a far lse sum to
    if (!SOFT && far_lse(lse)) {
        anew = 0.0f;
        if (!ALONE && im.parts > 1) {
            const float2* parts = a.parts + (index - im.part);
            for (int j = tid; j < im.parts; j += THREADS) anew += parts[j].x;
        } else {
#pragma unroll
            for (int j = 0; j < kWideRuns; ++j)
                if (j < live)
#pragma unroll
                    for (int k = 0; k < kRun; ++k) anew += row_exp<MODE, TYPE, BIAS>(v[j][k] - lse);
        }
        anew = ALONE ? wave_sum(anew) : block_sum(anew, shf);
    }
    if (MODE == kRowsBack) {
        float total = 0.0f;
        if (!ALONE && im.parts > 1) {
            const float2* parts = a.parts + (index - im.part);
            for (int j = tid; j < im.parts; j += THREADS) total += parts[j].y;
        } else {
#pragma unroll
            for (int j = 0; j < kWideRuns; ++j)
#pragma unroll
                for (int k = 0; k < kRun; ++k) total += d[j][k];
        }
        total = (ALONE ? wave_sum(total) : block_sum(total, shf)) / anew;
#pragma unroll
        for (int j = 0; j < kWideRuns; ++j)
            if (j < live)
#pragma unroll
                for (int k = 0; k < kRun; ++k)
                    v[j][k] = d[j][k] - (v[j][k] == -kInf ? 0.0f : row_exp<MODE, TYPE, BIAS>(v[j][k] - lse) * total);
    }
    int at = -kRun;  // the chosen row, as the span counts
    float extra = 0.0f;
    if (STEPS) {
        counts = counts && (SOFT ? t.sum != 0.0f : lse != -kInf);
        const double fine = MODE == kPolicy && counts ? ((double)xc - (double)t.top) - fine_log(t.sum) : 0.0;
        const float lp = MODE == kPolicy ? (float)fine : SOFT && counts ? (xc - t.top) - ls : 0.0f;
        if (SOFT && first) a.log_probs[g] = lp;
        if (GRAD) {
            float coef = 0.0f;
            if (MODE == kStepsBack && counts) coef = given;
            if (MODE == kPolicy && counts) coef = policy_step(a, pol, fine, first, tally);
            const float f = counts ? (SOFT ? -coef * __builtin_amdgcn_rcpf(t.sum) : -coef / anew) : 0.0f;
            const float fw = f * own;
            const int64_t row = r0 + c - sp.q0;
            if (counts && row >= sp.lo && row < sp.hi) {
                at = (int)row;
                extra = coef;
            }
#pragma unroll
            for (int j = 0; j < kWideRuns; ++j)
                if (j < live)
#pragma unroll
                    for (int k = 0; k < kRun; ++k) {
                        const float e = SOFT ? v[j][k] : row_exp<MODE, TYPE, BIAS>(v[j][k] - lse);
                        v[j][k] = f == 0.0f ? 0.0f : fw * e;
                    }
        }
    }
    if (MODE == kSteps) return;
#pragma unroll
    for (int j = 0; j < kWideRuns; ++j) {
        if (j < live) {
            const int i = kRun * (j * THREADS + tid);
            if (MODE == kRows) {
                if (i < sp.hi) store_run<PB_F32>(a, sp, i, a.log_probs, v[j]);
            } else {
                if (off[j]) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k) v[j][k] = off[j] >> k & 1u ? 0.0f : v[j][k];
                }
                if (STEPS && at >= i && at < i + kRun) {
#pragma unroll
                    for (int k = 0; k < kRun; ++k)
                        if (at - i == k) v[j][k] += extra;
                }
                if (i < sp.hi) store_run<TYPE>(a, sp, i, a.grad_scores, v[j]);
                if (BIAS) table.add<MODE == kPolicy>(v[j], buckets[j]);
            }
        }
    }
}

// The steps of the sets in parts, from the parts' maxima and sums: a wave to a set (4096 sets: 5 us).
template <int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void split_steps_kernel(ChoiceArgs a, const int32_t* __restrict__ firsts, int n) {
    __shared__ BiasShared bias;
    if (BIAS) stage_bias(a, bias);
    const int lane = (int)threadIdx.x & (kWave - 1), k = (int)blockIdx.x * kWaves + (int)threadIdx.x / kWave;
    if (k >= n) return;
    const SetItem im = a.wide[firsts[k]];
    const int64_t g = im.set0, r0 = a.off[g], size = a.off[g + 1] - r0;
    const int32_t c = a.chosen[g];
    const Soft t = wave_soft(join_parts(a.parts + firsts[k], im.parts, lane, kWave));
    bool counts = c >= 0 && c < size && t.sum != 0.0f;
    if (MASK && counts) counts = a.mask[r0 + c] != 0;
    const float ls = log_of(t.sum);
    if (lane == 0) {
        a.lse_out[g] = t.top + ls;
        a.log_probs[g] = counts ? (one_logit<TYPE, BIAS>(a, &bias, r0 + c) - t.top) - ls : 0.0f;
    }
}

template <int MODE, bool BIAS>
constexpr bool kTable = BIAS && (MODE == kRowsBack || MODE == kStepsBack || MODE == kPolicy);

// The tiles, one a wave at a time.
template <int MODE, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, 4) void tile_kernel(ChoiceArgs a) {
    constexpr bool TABLE = kTable<MODE, BIAS>;
    __shared__ TileShared tiles[kWaves];
    __shared__ BiasShared bias;
    __shared__ unsigned long long bins[TABLE ? kWaves : 1][kBins];
    __shared__ int shifts[TABLE ? kWaves : 1][kBins];
    __shared__ int bad[kMaxBuckets];
    __shared__ double shd[kWaves * 3];
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    TableSum table;
    if (TABLE) {
        for (int b = tid; b < kMaxBuckets; b += kBlock) bad[b] = 0;
        table.start(a, bins[wave], shifts[wave], bad);
    }
    double tally[3] = {0.0, 0.0, 0.0};
    const int lane = tid & (kWave - 1), step = (int)gridDim.x * kWaves;
    int it = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + wave);
    SetItem next = a.tiles[min(it, a.num_tiles - 1)];
    TileIn<MODE, TYPE, MASK, BIAS> in;
    // The first tile is asked for before the bias is staged (a wave beyond the tiles asks for the last one
    // and leaves it), which with the table's gradient costs more registers than it gains.
    if (!TABLE) in.load(a, next, lane);
    if (BIAS) stage_bias(a, bias);
    while (it < a.num_tiles) {
        if (TABLE) in.load(a, next, lane);
        next = a.tiles[min(it + step, a.num_tiles - 1)];
        tile_pass<MODE, TYPE, MASK, BIAS>(a, in, tiles[wave], &bias, table, tally);
        it += step;
        if (!TABLE && it < a.num_tiles) in.load(a, next, lane);
    }
    leave_sums<MODE == kPolicy ? 3 : 0, TABLE>(a, (int)blockIdx.x, tally, table, bins, bad, shd);
}

// The longer sets: workgroups [0, mid_blocks) take those for a wave, the others those for a workgroup and
// the parts, one at a time.
template <int MODE, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void wide_kernel(ChoiceArgs a, int mid_blocks) {
    constexpr bool TABLE = kTable<MODE, BIAS>;
    __shared__ BiasShared bias;
    __shared__ unsigned long long bins[TABLE ? kWaves : 1][kBins];
    __shared__ int shifts[TABLE ? kWaves : 1][kBins];
    __shared__ int bad[kMaxBuckets];
    __shared__ Soft shs[kWaves];
    __shared__ float shf[kWaves];
    __shared__ double shd[kWaves * 3];
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    TableSum table;
    if (TABLE) {
        for (int b = tid; b < kMaxBuckets; b += kBlock) bad[b] = 0;
        table.start(a, bins[wave], shifts[wave], bad);
    }
    if (BIAS) stage_bias(a, bias);
    double tally[3] = {0.0, 0.0, 0.0};
    if ((int)blockIdx.x < mid_blocks) {
        const int step = mid_blocks * kWaves;
        int it = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kWaves + wave);
        SetItem next = a.wide[min(it, a.num_mid - 1)];
        for (; it < a.num_mid; it += step) {
            const SetItem im = next;
            next = a.wide[min(it + step, a.num_mid - 1)];
            wide_pass<MODE, TYPE, MASK, BIAS, kWave>(a, im, it, shs, shf, &bias, table, tally);
        }
    } else {
        const int n = a.num_mid + (MODE == kSteps ? a.num_whole : a.num_wide);
        for (int it = a.num_mid + (int)blockIdx.x - mid_blocks; it < n; it += (int)gridDim.x - mid_blocks)
            wide_pass<MODE, TYPE, MASK, BIAS, kBlock>(a, a.wide[it], it, shs, shf, &bias, table, tally);
    }
    leave_sums<MODE == kPolicy ? 3 : 0, TABLE>(a, a.blocks - (int)gridDim.x + (int)blockIdx.x, tally, table, bins, bad, shd);
}

// out[j] = sum over the workgroups' sums [n][cols] of column j, in a fixed order; the first `head`
// columns go to stats, the others to the table's gradient. A launch of its own (3 to 5 us, most of it
// latency): joining in the last workgroup to finish would have every workgroup write back its L2 first.
__global__ __launch_bounds__(kBlock) void join_kernel(const double* __restrict__ sums, int32_t n, int32_t cols,
                                                      int32_t head, float* __restrict__ stats,
                                                      float* __restrict__ table) {
    __shared__ double sh[kWaves];
    const int j = (int)blockIdx.x;
    double t = 0.0;
    for (int i0 = 0; i0 < n; i0 += kBlock * kJoin) {  // kJoin loads in flight
        double v[kJoin];
#pragma unroll
        for (int k = 0; k < kJoin; ++k) {
            const int i = i0 + k * kBlock + (int)threadIdx.x;
            v[k] = i < n ? sums[(int64_t)i * cols + j] : 0.0;
        }
#pragma unroll
        for (int k = 0; k < kJoin; ++k) t += v[k];
    }
    t = block_sum(t, sh);
    if (threadIdx.x == 0) (j < head ? stats[j] : table[j - head]) = (float)t;
}

// ------------------------------------------------------------------------------ preferences
// Sums over sets in double: of (value - ref) over a sequence's steps, or of the signed slopes of the
// pairs that a value is in (list entry: pair * 2 + (1 where it is the loser)). A pair's slope is computed once
// and gathered twice, in the lists' order: no atomics, so hubs (values in thousands of pairs) cost
// what their entries cost and sums keep their order. Bound by the gathers, which find little of 20 MB of
// slopes in an XCD's 4 MB of L2: 10M entries of 1M lists 149 to 152 us, 3.6 TB/s of 64-byte lines. They
// are taken in the caller's order of the pairs; an order in which neighbouring entries share lines is not tried.
struct SumArgs {
    const int64_t* off;
    const SetItem* tiles;
    const SetItem* wide;
    int32_t num_tiles;
    int32_t num_wide;
    const float* values;
    const float* ref;
    const int32_t* entries;
    const float* slopes;
    float* out;
    double* totals;      // in the place of `out`, for sequences: their sums nearly cancel in pairs
    double* parts;
    const double* sums;  // the pairs' workgroups' losses [num_sums], joined by a workgroup more
    int32_t num_sums;
    float* loss;
};

// loss[0] = the sum of the workgroups' sums, in a fixed order.
__device__ void join_loss(const SumArgs& a, double* sh) {
    double t = 0.0;
    for (int i = (int)threadIdx.x; i < a.num_sums; i += kBlock) t += a.sums[i];
    t = block_sum(t, sh);
    if (threadIdx.x == 0) a.loss[0] = (float)t;
}

template <bool PAIRS>
__device__ __forceinline__ double sum_term(const SumArgs& a, int64_t i) {
    if (PAIRS) {
        const int32_t e = __builtin_nontemporal_load(a.entries + i);
        const float c = a.slopes[e >> 1];
        return (double)(e & 1 ? -c : c);
    }
    return (double)a.values[i] - (a.ref ? (double)a.ref[i] : 0.0);
}

template <bool PAIRS>
__device__ __forceinline__ void put_sum(const SumArgs& a, int64_t g, double t) {
    if (PAIRS)
        a.out[g] = (float)t;
    else
        a.totals[g] = t;
}

template <bool PAIRS>
__global__ __launch_bounds__(kBlock) void set_sum_kernel(SumArgs a) {
    constexpr int kPer = kSetTileRows / kWave;
    __shared__ double xs[kWaves][kSetTileRows];
    __shared__ double sh[kWaves];
    const int tid = (int)threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    if ((int)blockIdx.x < a.num_wide) {
        const SetItem im = a.wide[blockIdx.x];
        double t = 0.0;
        for (int i = tid; i < im.rows; i += kBlock) t += sum_term<PAIRS>(a, im.row0 + i);
        t = block_sum(t, sh);
        if (tid == 0) {
            if (im.parts == 1)
                put_sum<PAIRS>(a, im.set0, t);
            else
                a.parts[blockIdx.x] = t;
        }
        return;
    }
    const int it = ((int)blockIdx.x - a.num_wide) * kWaves + wave;
    if (it - wave >= a.num_tiles) {
        if (PAIRS) join_loss(a, sh);
        return;
    }
    if (it >= a.num_tiles) return;
    const SetItem im = a.tiles[it];
    double v[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = k * kWave + lane;
        v[k] = i < im.rows ? sum_term<PAIRS>(a, im.row0 + i) : 0.0;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) xs[wave][k * kWave + lane] = v[k];
    wave_sync();
    const int L = 1 << im.team, sub = lane & (L - 1);
    for (int s = lane >> im.team; s < im.sets; s += kWave >> im.team) {
        const int64_t g = (int64_t)im.set0 + s;
        const int b = (int)(a.off[g] - im.row0), e = (int)(a.off[g + 1] - im.row0);
        double t = 0.0;
        for (int i = b + sub; i < e; i += L) t += xs[wave][i];
        for (int m = 1; m < L; m <<= 1) t += __shfl_xor(t, m);
        if (sub == 0) put_sum<PAIRS>(a, g, t);
    }
}

// The sets that were summed in parts.
template <bool PAIRS>
__global__ __launch_bounds__(kBlock) void set_join_kernel(SumArgs a, const int32_t* __restrict__ list) {
    __shared__ double sh[kWaves];
    const int32_t it = list[blockIdx.x];
    const SetItem im = a.wide[it];
    double t = 0.0;
    for (int j = (int)threadIdx.x; j < im.parts; j += kBlock) t += a.parts[it + j];
    t = block_sum(t, sh);
    if (threadIdx.x == 0) put_sum<PAIRS>(a, im.set0, t);
}

// z = beta (a_w - a_l); the loss w [(1 - e) softplus(-z) + e softplus(z)] and its slope
// beta w (sigmoid(z) - (1 - e)). Sequences' values come from their sums in double, others' as value
// - ref, the differences taken in double: both can be large where z is small. Bound by the gathers of the values: 5M
// pairs of 1M values, values and references side by side, 93 us (160 us in arrays of their own). Four
// pairs are in flight a thread.
__global__ __launch_bounds__(kBlock) void pair_kernel(PairArgs a) {
    __shared__ double sh[kWaves];
    double sum = 0.0;
    const int64_t stride = (int64_t)gridDim.x * kBlock;
    for (int64_t p0 = (int64_t)blockIdx.x * kBlock + threadIdx.x; p0 < a.num_pairs; p0 += stride * kPairs) {
        int32_t w[kPairs], l[kPairs];
        float weight[kPairs];
        double d[kPairs];
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {  // past the end: the last pair again, unused
            const int64_t p = min(p0 + k * stride, a.num_pairs - 1);
            w[k] = __builtin_nontemporal_load(a.winners + p);
            l[k] = __builtin_nontemporal_load(a.losers + p);
            weight[k] = a.weights ? __builtin_nontemporal_load(a.weights + p) : 1.0f;
        }
        if (a.totals) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) d[k] = a.totals[w[k]] - a.totals[l[k]];
        } else if (a.both) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float2 t = a.both[w[k]], u = a.both[l[k]];
                d[k] = ((double)t.x - (double)u.x) - ((double)t.y - (double)u.y);
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                d[k] = (double)a.values[w[k]] - (double)a.values[l[k]];
                if (a.ref) d[k] -= (double)a.ref[w[k]] - (double)a.ref[l[k]];
            }
        }
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const int64_t p = p0 + k * stride;
            if (p >= a.num_pairs) break;
            const float z = (float)((double)a.beta * d[k]);
            const float ws = weight[k] * a.scale;
            const float t = expf(-fabsf(z)), soft = log1pf(t);
            const float e = a.smoothing, h = 1.0f - e;
            const float up = z > 0.0f ? 1.0f / (1.0f + t) : t / (1.0f + t);    // sigmoid(z)
            const float down = z > 0.0f ? t / (1.0f + t) : 1.0f / (1.0f + t);  // sigmoid(-z)
            __builtin_nontemporal_store(z, a.margins + p);
            a.slopes[p] = ws == 0.0f ? 0.0f : a.beta * ws * (e * up - h * down);
            // a term of factor 0 counts for nothing, whatever its margin
            const float lost = (h == 0.0f ? 0.0f : h * (soft + fmaxf(-z, 0.0f))) + (e == 0.0f ? 0.0f : e * (soft + fmaxf(z, 0.0f)));
            if (ws != 0.0f) sum += (double)(ws * lost);
        }
    }
    sum = block_sum(sum, sh);
    if (threadIdx.x == 0) {
        if (gridDim.x == 1)
            a.loss[0] = (float)sum;
        else
            a.sums[blockIdx.x] = sum;
    }
}

// Values beside their references, so that a pair finds both in one access (1M: 5 us).
__global__ __launch_bounds__(kBlock) void both_kernel(const float* __restrict__ values, const float* __restrict__ ref,
                                                      int64_t n, float2* __restrict__ both) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i < n) both[i] = make_float2(values[i], ref[i]);
}

// The pairs' slopes summed over a sequence's list (a team of L lanes, this one `sub`).
__device__ __forceinline__ float list_slope(const SumArgs& a, const int64_t* list_off, int64_t g, int sub, int L) {
    double t = 0.0;
    const int64_t e = list_off[g + 1];
    for (int64_t i0 = list_off[g] + sub; i0 < e; i0 += 4 * L) {  // four in flight; past the end none
        double v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = i0 + (int64_t)k * L;
            v[k] = sum_term<true>(a, min(i, e - 1));
            if (i >= e) v[k] = 0.0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) t += v[k];
    }
    for (int m = 1; m < L; m <<= 1) t += __shfl_xor(t, m);
    return (float)t;
}

// out[i] = the slope of step i's sequence: per_set[sequence], or (per_set NULL) the sum over the sequence's
// list of pairs, where no list is long (300k steps of 4001 sequences in 6000 pairs: 9 us, against 8 + 4 in
// two launches and what they cost the host).
__global__ __launch_bounds__(kBlock) void spread_kernel(SumArgs a, const float* __restrict__ per_set,
                                                        const int64_t* __restrict__ list_off) {
    __shared__ double sh[kWaves];
    const int tid = (int)threadIdx.x, lane = tid & (kWave - 1);
    if ((int)blockIdx.x < a.num_wide) {
        const SetItem im = a.wide[blockIdx.x];
        const float v = per_set ? per_set[im.set0] : list_slope(a, list_off, im.set0, lane, kWave);
        for (int i = tid; i < im.rows; i += kBlock) a.out[im.row0 + i] = v;
        return;
    }
    const int first = ((int)blockIdx.x - a.num_wide) * kWaves, it = first + tid / kWave;
    if (first >= a.num_tiles) {
        join_loss(a, sh);
        return;
    }
    if (it >= a.num_tiles) return;
    const SetItem im = a.tiles[it];
    const int L = 1 << im.team, sub = lane & (L - 1);
    for (int s = lane >> im.team; s < im.sets; s += kWave >> im.team) {
        const int64_t g = (int64_t)im.set0 + s;
        const float v = per_set ? per_set[g] : list_slope(a, list_off, g, sub, L);
        const int64_t e = a.off[g + 1];
        for (int64_t i = a.off[g] + sub; i < e; i += L) a.out[i] = v;
    }
}

int tile_groups(const SetLayout& s) { return (s.num_tiles + kWaves - 1) / kWaves; }

int tile_blocks(const SetLayout& s) { return std::min(tile_groups(s), kChoiceGrid); }

int mid_blocks(const SetLayout& s) { return std::min((s.num_mid + kWaves - 1) / kWaves, kChoiceGrid); }

int wide_blocks(int wide) { return std::min(wide, kChoiceGrid); }

template <int MODE, int TYPE, bool MASK, bool BIAS>
hipError_t launch_choice_as(const SetLayout& s, const ChoiceArgs& a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    const int parts = s.num_wide - s.num_whole;
    if (parts > 0) {
        const int first = s.num_mid + s.num_whole;
        if constexpr (MODE == kRowsBack || MODE == kStepsBack) {
            if (MODE == kRowsBack) {
                hipLaunchKernelGGL(part_grads_kernel<MASK>, dim3(parts), dim3(kBlock), 0, stream, a, first);
                if ((e = hipGetLastError()) != hipSuccess) return e;
            }
            hipLaunchKernelGGL((part_far_kernel<TYPE, MASK, BIAS>), dim3(std::min(parts, kChoiceGrid)), dim3(kBlock), 0, stream,
                               a, first, parts);
        } else {
            hipLaunchKernelGGL((part_kernel<MODE, TYPE, MASK, BIAS>), dim3(parts), dim3(kBlock), 0, stream, a, first);
        }
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (s.num_tiles > 0) {
        hipLaunchKernelGGL((tile_kernel<MODE, TYPE, MASK, BIAS>), dim3(tile_blocks(s)), dim3(kBlock), 0, stream, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int wide = mid_blocks(s) + wide_blocks(MODE == kSteps ? s.num_whole : s.num_wide);
    if (wide > 0) {
        hipLaunchKernelGGL((wide_kernel<MODE, TYPE, MASK, BIAS>), dim3(wide), dim3(kBlock), 0, stream, a, mid_blocks(s));
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (MODE == kSteps && s.num_split > 0) {
        hipLaunchKernelGGL((split_steps_kernel<TYPE, MASK, BIAS>), dim3((s.num_split + kWaves - 1) / kWaves), dim3(kBlock), 0,
                           stream, a, s.split, s.num_split);
        e = hipGetLastError();
    }
    return e;
}

template <int MODE, int TYPE>
hipError_t launch_choice_typed(const SetLayout& s, const ChoiceArgs& a, hipStream_t stream) {
    if (a.mask)
        return a.table ? launch_choice_as<MODE, TYPE, true, true>(s, a, stream)
                       : launch_choice_as<MODE, TYPE, true, false>(s, a, stream);
    return a.table ? launch_choice_as<MODE, TYPE, false, true>(s, a, stream)
                   : launch_choice_as<MODE, TYPE, false, false>(s, a, stream);
}

template <int MODE>
hipError_t launch_choice_mode(const SetLayout& s, const ChoiceArgs& a, int32_t type, hipStream_t stream) {
    if (type == PB_BF16) return launch_choice_typed<MODE, PB_BF16>(s, a, stream);
    if (type == PB_F16) return launch_choice_typed<MODE, PB_F16>(s, a, stream);
    return launch_choice_typed<MODE, PB_F32>(s, a, stream);
}

// Items a workgroup each of the sums
int long_items(const SetLayout& s) { return s.num_mid + s.num_wide; }

SumArgs sum_args(const SetLayout& s) {
    SumArgs a{};
    a.off = s.off;
    a.tiles = s.tiles;
    a.wide = s.wide;
    a.num_tiles = s.num_tiles;
    a.num_wide = s.num_mid + s.num_wide;
    return a;
}

bool side_by_side(const PairLayout& p) {
    return !p.has_seqs && p.lists.num_sets >= kBothValues && p.num_pairs >= kBothPairs;
}

template <bool PAIRS>
hipError_t launch_set_sum(const SetLayout& s, const SumArgs& a, hipStream_t stream) {
    const int grid = long_items(s) + tile_groups(s) + (PAIRS && a.num_sums > 0 ? 1 : 0);
    if (grid == 0) return hipSuccess;
    hipLaunchKernelGGL(set_sum_kernel<PAIRS>, dim3(grid), dim3(kBlock), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || s.num_split == 0) return e;
    hipLaunchKernelGGL(set_join_kernel<PAIRS>, dim3(s.num_split), dim3(kBlock), 0, stream, a, s.split);
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

int32_t choice_grid(const SetLayout& s) { return tile_blocks(s) + mid_blocks(s) + wide_blocks(s.num_wide); }

hipError_t launch_choice(int mode, const SetLayout& s, ChoiceArgs a, int32_t type, hipStream_t stream) {
    a.off = s.off;
    a.tiles = s.tiles;
    a.wide = s.wide;
    a.segments = s.segments;
    a.num_tiles = s.num_tiles;
    a.num_wide = s.num_wide;
    a.num_mid = s.num_mid;
    a.num_whole = s.num_whole;
    a.blocks = choice_grid(s);
    a.rows = s.rows;
    // runs of eight rows in accesses of 16 bytes, 8 of the mask
    const auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    a.vec = a.stride == 1 && at(a.scores, 16) && at(a.grad_scores, 16) && at(a.mask, 8) && at(a.positions, 16) &&
            (mode != kRows || at(a.log_probs, 16)) && (mode != kRowsBack || at(a.grad, 16));
    hipError_t e = hipSuccess;
    if (mode == kRows) e = launch_choice_mode<kRows>(s, a, type, stream);
    if (mode == kSteps) e = launch_choice_mode<kSteps>(s, a, type, stream);
    if (mode == kRowsBack) e = launch_choice_mode<kRowsBack>(s, a, type, stream);
    if (mode == kStepsBack) e = launch_choice_mode<kStepsBack>(s, a, type, stream);
    if (mode == kPolicy) e = launch_choice_mode<kPolicy>(s, a, type, stream);
    const int32_t head = mode == kPolicy ? 3 : 0;
    const int32_t cols = head + (a.table && mode != kRows && mode != kSteps ? a.num_buckets : 0);
    if (e != hipSuccess || cols == 0 || a.blocks == 1) return e;
    return launch_join_sums(a.sums, a.blocks, cols, head, a.stats, a.grad_table, stream);
}

hipError_t launch_join_sums(const double* sums, int32_t n, int32_t cols, int32_t head, float* stats, float* table,
                            hipStream_t stream) {
    hipLaunchKernelGGL(join_kernel, dim3(cols), dim3(kBlock), 0, stream, sums, n, cols, head, stats, table);
    return hipGetLastError();
}

hipError_t launch_preference(const PairLayout& p, PairArgs a, const float* values, const float* ref, float* grad,
                             char* work, hipStream_t stream) {
    a.winners = p.winners;
    a.losers = p.losers;
    a.num_pairs = p.num_pairs;
    a.sums = reinterpret_cast<double*>(work);
    double* parts = a.sums + kPairGrid;
    double* totals = parts + long_items(p.lists) + long_items(p.seqs);
    a.slopes = reinterpret_cast<float*>(totals + p.seqs.num_sets);
    float* seq_grad = a.slopes + p.num_pairs;
    const bool seqs = p.has_seqs;
    hipError_t e = hipSuccess;
    if (seqs) {
        SumArgs sa = sum_args(p.seqs);
        sa.parts = parts;
        sa.values = values;
        sa.ref = ref;
        sa.totals = totals;
        if ((e = launch_set_sum<false>(p.seqs, sa, stream)) != hipSuccess) return e;
        a.totals = totals;
    } else {
        a.values = values;
        a.ref = ref;
        if (ref && side_by_side(p)) {
            float2* both = reinterpret_cast<float2*>(parts + long_items(p.lists));
            a.slopes = reinterpret_cast<float*>(both + p.lists.num_sets);
            a.both = both;
            hipLaunchKernelGGL(both_kernel, dim3((unsigned)((p.lists.num_sets + kBlock - 1) / kBlock)), dim3(kBlock), 0, stream,
                               values, ref, p.lists.num_sets, both);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    const int64_t want = (p.num_pairs + kBlock - 1) / kBlock;
    const int grid = (int)(want < 1 ? 1 : want > kPairGrid ? kPairGrid : want);
    hipLaunchKernelGGL(pair_kernel, dim3(grid), dim3(kBlock), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    // the losses of several workgroups are joined by the next launch
    const int num_sums = grid > 1 ? grid : 0;
    SumArgs sa = sum_args(p.lists);
    sa.parts = parts + long_items(p.seqs);
    sa.entries = p.entries;
    sa.slopes = a.slopes;
    sa.out = seqs ? seq_grad : grad;
    sa.sums = a.sums;
    sa.num_sums = num_sums;
    sa.loss = a.loss;
    // Sequences whose lists are all short are summed where their steps are written
    const bool direct = seqs && long_items(p.lists) == 0;
    if (!direct && (e = launch_set_sum<true>(p.lists, sa, stream)) != hipSuccess) return e;
    if (!seqs) return e;
    SumArgs sp = sum_args(p.seqs);
    sp.entries = p.entries;
    sp.slopes = a.slopes;
    sp.out = grad;
    sp.sums = a.sums;
    sp.num_sums = num_sums;
    sp.loss = a.loss;
    const int steps = long_items(p.seqs) + tile_groups(p.seqs) + (direct && num_sums > 0 ? 1 : 0);
    if (steps > 0) {
        hipLaunchKernelGGL(spread_kernel, dim3(steps), dim3(kBlock), 0, stream, sp, direct ? nullptr : seq_grad, p.lists.off);
        e = hipGetLastError();
    }
    return e;
}

int64_t preference_work_bytes(const PairLayout& p) {
    return 8 * ((int64_t)kPairGrid + long_items(p.lists) + long_items(p.seqs) + p.seqs.num_sets) + 4 * (p.num_pairs + p.seqs.num_sets) +
           (side_by_side(p) ? 8 * p.lists.num_sets : 0);
}

}  // namespace pb
