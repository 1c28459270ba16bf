// Reports on choices over ragged sets of candidate rows: of each set the chosen row's log-probability, the entropy, and the
// rows of largest probability with theirs, at a temperature T.
//
// With z the logits, m their maximum (0 where that is -inf), e_i = exp((z_i - m) / T), s = sum e and u = sum e (z - m):
// lse = m / T + log s, log p_i = (z_i - m) / T - log s, and the entropy -sum p log p = log s - u / (T s). A set without
// probability has s = 0, lse -inf and entropy 0. Rows are ranked by z, equal ones by index, NaN above all; rows of z = -inf
// are not ranked.
//
// Rows are laid out and read as choice.hip has them, each once: tiles of short sets by a wave, longer sets by a wave or a
// workgroup that holds them in registers (of up to 65536 rows where that pays, see kBigSets), what is longer still in parts
// that a second kernel joins. In a tile, a row of
// a short set counts the rows that rank above it. Of longer sets a bound is found first that at least as many rows reach as
// are listed, from the maxima of the lanes; the rows that reach it, few where they lie in no order, are gathered and
// ranked by counting.
#include <algorithm>
#include <utility>

#include "soft_rows.h"

namespace pb {
namespace {

// Rows of a tile's set whose rows count what ranks above them; of a longer one the wave finds a bound. 1M rows in sets of
// one size, counted / by a bound: 40 rows 20 / 52 us, 64 20 / 27, 80 27 / 23, 96 30 / 20, 192 37 / 12, 384 58 / 9. With sizes
// about 12.5 on average, where the few longer ones hold up their tiles, 64 costs 11 us and 192 costs 10.
constexpr int kCountRows = 80;
constexpr int kWaveList = 256;   // rows that reach the bound: room for a wave's
constexpr int kGroupList = 512;  // and a workgroup's
constexpr int kJoinList = kMaxTop * kMaxTop;
// Up to so many tiles have a workgroup each, whose waves share the lists, else a wave each: 64 tiles of 21 sets 7 / 11 us,
// 512 7.8 / 11.4, 1024 13.7 / 11.7, 4096 38 / 25.
constexpr int kSharedTiles = 512;
// Long sets have a workgroup each where nothing else is there for the kernel of parts (4 sets of 30 thousand 16-bit rows
// 9 us, in parts 12; 256 sets 11 and 15; 2048 sets 45 and 68), and beside others from so many on: parts add 27 us to what
// that kernel takes for 1024 sets, as much as a launch of their own.
constexpr int kBigSets = 1024;
constexpr int kOneLaunch = 256;  // as many of mixed lengths as fit beside each other go in one launch
// Parts whose bound is found by counting, not bit by bit: 256 parts 20 / 48 us, 1024 85 / 87, 2048 276 / 140.
constexpr int kBoundParts = 1024;

// Orders logits as whole numbers: larger first, -0 as 0, NaN above all; 0 for what is not ranked.
__device__ __forceinline__ uint32_t rank_of(float z) {
    if (z == -kInf) return 0;
    const uint32_t b = z != z ? 0x7fc00000u : __float_as_uint(z + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float rank_value(uint32_t r) { return __uint_as_float(r & 0x80000000u ? r ^ 0x80000000u : ~r); }

// A row of a list is held as a key: its rank, 32 bits up, and the complement of its index. 0 for none.
__device__ __forceinline__ float list_log_prob(const ReportArgs& a, float z, float top, double log_sum) {
    return (float)(((double)z - (double)top) * a.inv_temp - log_sum);
}

// What a set's sums say, by one lane.
__device__ __forceinline__ void put_report(const ReportArgs& a, int64_t g, const SoftSums& t, double log_sum, bool counts, float z) {
    const bool none = t.sum == 0.0;
    const double m = none ? 0.0 : (double)t.top;
    a.lse_out[g] = (float)(m * a.inv_temp + log_sum);
    const double h = log_sum - t.along * a.inv_temp / t.sum;
    a.entropy[g] = none || h < 0.0 ? 0.0f : (float)h;  // roundings may leave less than 0; NaN is kept
    if (a.chosen) a.log_probs[g] = counts && !none ? (float)(((double)z - m) * a.inv_temp - log_sum) : 0.0f;
}

__device__ __forceinline__ void put_entry(const ReportArgs& a, int64_t at, int32_t index, float log_prob) {
    a.top_index[at] = index;
    a.top_log_probs[at] = log_prob;
}

// ------------------------------------------------------------------------------------ lists of longer sets
template <int THREADS, int LIST>
struct RankGroup {
    static constexpr int kGroupWaves = THREADS / kWave;
    unsigned long long list[LIST];
    uint32_t bound[kGroupWaves], count[2][kGroupWaves];
    uint32_t size;
};

// The number of a group's lanes' v, the same in every lane; `turn` is 0 and 1 in turn.
template <int THREADS, int LIST>
__device__ __forceinline__ uint32_t group_count(uint32_t wave_count, RankGroup<THREADS, LIST>& sh, int& turn) {
    if (THREADS == kWave) return wave_count;
    turn ^= 1;
    if ((threadIdx.x & (kWave - 1)) == 0) sh.count[turn][threadIdx.x / kWave] = wave_count;
    __syncthreads();
    uint32_t n = 0;
    for (int w = 0; w < THREADS / kWave; ++w) n += sh.count[turn][w];
    return n;
}

// The largest bound, in steps of 2^16 of the ranks, that at least n of the wave's COUNT x 64 maxima reach; 0 if there are
// fewer. So many rows reach it at least.
template <int COUNT>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t (&most)[COUNT], uint32_t n) {
    uint32_t t = 0;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
        uint32_t c = 0;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) c += (uint32_t)__popcll(__ballot(most[j] >= (t | bit)));
        if (c >= n) t |= bit;
    }
    return t;
}

// f of 0 .. N - 1 as constants: loops within f keep the compiler from unrolling one over the runs, which lie in registers.
template <class F, int... J>
__device__ __forceinline__ void each_run(F f, std::integer_sequence<int, J...>) {
    (f(std::integral_constant<int, J>{}), ...);
}

// The largest of a run, NaN left aside.
__device__ __forceinline__ float run_max(const float (&x)[kRun]) {
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max2(x[6], x[7]));
}

// The rows of a group's logits v (run j, row k: row kRun (j THREADS + tid) + k of the group's, from index0 on within the set)
// that rank highest, at least a.top of them where there are so many, as keys in sh.list; returns their number. tops: the
// largest of the runs; `odd`: there may be NaN, which those leave aside. again(j, x): run j once more, for the rare case that
// more rows reach the bound than there is room for.
template <int THREADS, int LIST, int RUNS, class AGAIN>
__device__ __forceinline__ int gather_best(const ReportArgs& a, const float (&v)[RUNS][kRun], const float (&tops)[RUNS], int live,
                                           bool odd, int64_t index0, RankGroup<THREADS, LIST>& sh, AGAIN again) {
    const int tid = (int)threadIdx.x & (THREADS - 1), lane = tid & (kWave - 1);
    const uint32_t n = (uint32_t)a.top;
    uint32_t most[RUNS], all[1] = {0};
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        most[j] = j < live ? rank_of(tops[j]) : 0;
        all[0] = max(all[0], most[j]);
    }
    uint32_t bound;
    if (THREADS == kWave) {
        // where the lanes' largest would let many rows through, the runs' have a say, or each row
        if (n <= 16) {
            bound = wave_bound<1>(all, n);
        } else if (RUNS > 1) {
            bound = wave_bound<RUNS>(most, n);
        } else {
            uint32_t each[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k) each[k] = rank_of(v[0][k]);
            bound = wave_bound<kRun>(each, n);
        }
    } else {
        // of each wave's rows a share; a wave that has too few leaves it to the others
        const uint32_t waves = THREADS / kWave;
        const uint32_t mine = wave_bound<1>(all, (n + waves - 1) / waves);
        if (lane == 0) sh.bound[tid / kWave] = mine;
        if (tid == 0) sh.size = 0;
        __syncthreads();
        bound = ~0u;
        for (uint32_t w = 0; w < waves; ++w) bound = min(bound, sh.bound[w]);
        if (bound == 0) {
            const uint32_t whole = wave_bound<RUNS>(most, n);
            __syncthreads();
            if (lane == 0) sh.bound[tid / kWave] = whole;
            __syncthreads();
            for (uint32_t w = 0; w < waves; ++w) bound = max(bound, sh.bound[w]);
        }
    }
    // the lane's rows of run j with a bit in `in`, one of each lane at a time
    const auto add = [&](const float (&row)[kRun], int j, uint32_t in, uint32_t& count) {
        for (unsigned long long m = __ballot(in != 0); m; m = __ballot(in != 0)) {
            uint32_t at = count;
            if (THREADS == kWave) {
                count += (uint32_t)__popcll(m);
            } else {
                if (lane == 0) at = atomicAdd(&sh.size, (uint32_t)__popcll(m));
                at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
            }
            at += (uint32_t)__popcll(m & ((1ull << lane) - 1ull));
            if (in != 0 && at < (uint32_t)LIST) {
                const int k = __ffs((int)in) - 1;
                uint32_t x = 0;  // row[k]; a choice between the rows' places would put them in memory
#pragma unroll
                for (int l = 0; l < kRun; ++l) x |= __float_as_uint(row[l]) & (0u - (uint32_t)(l == k));
                sh.list[at] = (unsigned long long)rank_of(__uint_as_float(x)) << 32 | (uint32_t)~(uint32_t)(index0 + kRun * (j * THREADS + tid) + k);
            }
            in &= in - 1;
        }
    };
    const float least = bound < 0x00800000u ? kLowest : rank_value(bound);
    uint32_t count = 0;
    wave_sync();
    each_run([&](auto at) {
        constexpr int j = decltype(at)::value;
        if (j < live && (odd || __any(tops[j] >= least))) {
            uint32_t in = 0;
#pragma unroll
            for (int k = 0; k < kRun; ++k) in |= v[j][k] < least ? 0u : 1u << k;
            add(v[j], j, in, count);
        }
    }, std::make_integer_sequence<int, RUNS>{});
    if (THREADS != kWave) {
        __syncthreads();
        count = sh.size;
    }
    wave_sync();
    if (count <= (uint32_t)LIST) return (int)count;
    // Too many rows reach the bound, where many are of one value, or rise or fall along a workgroup's set, where the wave at
    // the lower end gives a low bound: the least rank that a.top rows reach, and of those that have it the first. The rows are read
    // anew for each bit: held in registers, they would cost the usual path a third of its waves. 4096 sets of 32 thousand
    // bfloat16 rows with lists of 8 take 2520 us here, 87 in any order (2000 sets of 6000 float32 rows 218 and 18).
    int turn = 0;
    const auto rows = [&](auto holds) {
        uint32_t c = 0;
#pragma unroll 1
        for (int j = 0; j < live; ++j) {
            float x[kRun];
            again(j, x);
#pragma unroll
            for (int k = 0; k < kRun; ++k) c += holds(rank_of(x[k]), kRun * (j * THREADS + tid) + k) ? 1u : 0u;
        }
        return group_count((uint32_t)wave_sum((float)c), sh, turn);
    };
    // mostly the bound's high half is the rank's, too
    const bool near = bound != 0 && rows([&](uint32_t r, int) { return r > (bound | 0xffffu); }) < n;
    uint32_t t = near ? bound : 0;
#pragma unroll 1
    for (uint32_t bit = near ? 1u << 15 : 1u << 31; bit != 0; bit >>= 1)
        if (rows([&](uint32_t r, int) { return r >= (t | bit); }) >= n) t |= bit;
    const uint32_t above = rows([&](uint32_t r, int) { return r > t; });
    int last = RUNS * THREADS * kRun - 1;
#pragma unroll 1
    for (int bit = RUNS * THREADS * kRun / 2; bit != 0; bit >>= 1)
        if (above + rows([&](uint32_t r, int i) { return r == t && i <= last - bit; }) >= n) last -= bit;
    if (THREADS != kWave) {
        if (tid == 0) sh.size = 0;
        __syncthreads();
    }
    count = 0;
#pragma unroll 1
    for (int j = 0; j < live; ++j) {
        float x[kRun];
        again(j, x);
        uint32_t in = 0;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const uint32_t r = rank_of(x[k]);
            in |= r > t || (r == t && t != 0 && kRun * (j * THREADS + tid) + k <= last) ? 1u << k : 0u;
        }
        add(x, j, in, count);
    }
    if (THREADS != kWave) {
        __syncthreads();
        count = sh.size;
    }
    wave_sync();
    return (int)count;
}

// How many of n keys are larger, eight asked for at a time.
__device__ __forceinline__ int keys_above(const unsigned long long* list, int n, unsigned long long key) {
    constexpr int kAhead = 8;
    int place = 0, i = 0;
    for (; i + kAhead <= n; i += kAhead) {
        unsigned long long o[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) o[u] = list[i + u];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) place += o[u] > key ? 1 : 0;
    }
    if (i < n) {
        unsigned long long o[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) o[u] = list[min(i + u, n - 1)];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) place += i + u < n && o[u] > key ? 1 : 0;
    }
    return place;
}

// f(place, key) of the first a.top of n keys, and of none (key 0) behind the last.
template <int THREADS, class F>
__device__ __forceinline__ void rank_list(const ReportArgs& a, const unsigned long long* list, int n, F f) {
    const int tid = (int)threadIdx.x & (THREADS - 1);
    for (int c = tid; c < n; c += THREADS) {
        const unsigned long long key = list[c];
        const int place = keys_above(list, n, key);
        if (place < a.top) f(place, key);
    }
    for (int c = n + tid; c < a.top; c += THREADS) f(c, 0ull);
}

// ------------------------------------------------------------------------------------ tiles
struct alignas(16) SumTile {
    float x[kSetTileRows];        // logits
    float top[kSetTileSets + 4];  // per set: maximum
    union {
        uint16_t head[kSetTileRows];  // the set that starts at a row, from 1; 0: none
        float sum[kSetTileSets + 4];  // later: sum of exponentials, then its logarithm
    };
    float along[kSetTileSets + 4];  // sum of exponentials times distances
};

struct alignas(16) ReportTile : SumTile {
    unsigned long long key[kSetTileRows];  // the rows' ranks and the complements of their places, 0 for none
    uint32_t range[kSetTileSets + 4];      // first row and, 16 bits up, the row behind the last
    int32_t set[kSetTileSets + 4];
    int32_t ranked[kSetTileSets + 4];  // rows that are ranked
    uint8_t id[kSetTileRows];          // a row's set, from 1
    int32_t behind, sets;              // the row behind the last set's
};

// What the lists of a tile are made of, by the tile's wave: the rows' keys, and where the sets lie.
template <class ROWS>
__device__ __forceinline__ void prepare_lists(const ROWS& in, const float (&x)[kRun], const int (&id)[kRun], ReportTile& sh) {
    const int lane = (int)threadIdx.x & (kWave - 1), i0 = kRun * lane;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        const uint32_t r = rank_of(x[k]);
        sh.key[i0 + k] = r ? (unsigned long long)r << 32 | (uint32_t)~(uint32_t)(i0 + k) : 0ull;
    }
    *reinterpret_cast<uint2*>(&sh.id[i0]) =
        make_uint2((uint32_t)id[0] | (uint32_t)id[1] << 8 | (uint32_t)id[2] << 16 | (uint32_t)id[3] << 24,
                   (uint32_t)id[4] | (uint32_t)id[5] << 8 | (uint32_t)id[6] << 16 | (uint32_t)id[7] << 24);
    int behind = 0;
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        sh.range[s] = (uint32_t)in.begin[r] | (uint32_t)in.end[r] << 16;
        sh.set[s] = in.set[r];
        sh.ranked[s] = 0;
        // an empty set behind a longer one may lie past the tile's rows
        behind = max(behind, in.end[r] > in.begin[r] ? in.end[r] : 0);
    }
    if (lane < 4) sh.range[kSetTileSets + lane] = 0;
    behind = (int)wave_max((float)behind);
    if (lane == 0) {
        sh.behind = behind;
        sh.sets = in.sets;
    }
}

// The lists of a tile, by wave `part` of `parts`. A lane takes a row and counts the larger keys of its set, 64 rows at a
// time, and a wave waits for its longest set; sets of more than kCountRows rows are taken by a whole wave each. (A lane with
// eight neighbouring rows took 11 us for 37 rows, where this takes 5.5 us.)
__device__ __forceinline__ void take_lists(const ReportArgs& a, ReportTile& sh, RankGroup<kWave, kWaveList>& group, int part, int parts) {
    const int lane = (int)threadIdx.x & (kWave - 1), num_sets = sh.sets;
#pragma unroll 1
    for (int p = part * kWave; p < sh.behind; p += parts * kWave) {
        const int i = p + lane, s = (int)sh.id[i] - 1;
        const unsigned long long key = sh.key[i];
        const uint32_t range = sh.range[s];
        const int b = (int)(range & 0xffffu), n = (int)(range >> 16) - b;
        if (key != 0 && n <= kCountRows) {
            atomicAdd(&sh.ranked[s], 1);
            const int place = keys_above(&sh.key[b], n, key);
            if (place < a.top)
                put_entry(a, (int64_t)sh.set[s] * a.top + place, i - b,
                          list_log_prob(a, rank_value((uint32_t)(key >> 32)), sh.top[s], (double)sh.sum[s]));
        }
    }
    if (parts > 1)
        __syncthreads();
    else
        wave_sync();
    // behind the last: lists with fewer ranked rows than entries
    bool gaps = false;
    unsigned long long longer[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        const uint32_t range = sh.range[s];
        const bool counted = (int)(range >> 16) - (int)(range & 0xffffu) <= kCountRows;
        gaps = gaps || (s < num_sets && counted && sh.ranked[s] < a.top);
        longer[r] = __ballot(!counted);
    }
    if (__any(gaps)) {
        const int bits = a.team_bits, entries = num_sets << bits, j = lane & ((1 << bits) - 1);
#pragma unroll 4
        for (int e = part * kWave + lane; e < entries; e += parts * kWave) {
            const int s = e >> bits;
            const uint32_t range = sh.range[s];
            if (j < a.top && j >= sh.ranked[s] && (int)(range >> 16) - (int)(range & 0xffffu) <= kCountRows)
                put_entry(a, (int64_t)sh.set[s] * a.top + j, -1, -kInf);
        }
    }
    int turn = 0;
    for (int r = 0; r < kTileRounds; ++r)
        for (unsigned long long m = r ? longer[1] : longer[0]; m; m &= m - 1, ++turn) {
            if (parts > 1 && turn % parts != part) continue;
            const int s = r * kWave + __ffsll((long long)m) - 1;
            const uint32_t range = sh.range[s];
            const int b = (int)(range & 0xffffu) + kRun * lane, e = (int)(range >> 16);
            const auto read = [&](int, float(&x)[kRun]) {
#pragma unroll
                for (int k = 0; k < kRun; ++k) {
                    const unsigned long long o = b + k < e ? sh.key[b + k] : 0ull;
                    x[k] = o ? rank_value((uint32_t)(o >> 32)) : -kInf;
                }
            };
            float v[1][kRun];
            read(0, v[0]);
            const float tops[1] = {run_max(v[0])};
            const int n = gather_best(a, v, tops, 1, true, 0, group, read);
            rank_list<kWave>(a, group.list, n, [&](int place, unsigned long long key) {
                const bool there = key != 0;
                put_entry(a, (int64_t)sh.set[s] * a.top + place, there ? (int32_t)~(uint32_t)key : -1,
                          there ? list_log_prob(a, rank_value((uint32_t)(key >> 32)), sh.top[s], (double)sh.sum[s]) : -kInf);
            });
            wave_sync();
        }
}

template <bool LISTS, int TYPE, bool MASK, bool BIAS>
__device__ __forceinline__ void report_tile(const ReportArgs& a, const TileRows<TYPE, MASK, BIAS>& in,
                                            int32_t (&chosen)[kTileRounds], std::conditional_t<LISTS, ReportTile, SumTile>& sh,
                                            const BiasShared* bias) {
    const int lane = (int)threadIdx.x & (kWave - 1), i0 = kRun * lane;
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    const bool alone = in.sets == 1;
    float x[kRun];
    uint32_t off;
    Buckets buckets;
#pragma unroll
    for (int k = 0; k < kRun; ++k) x[k] = -kInf;
    if (in.sp.hi > 0) in.raw.logits(a, bias, in.sp, 0, x, off, buckets);
    wave_sync();  // the last tile's values have been read
    *reinterpret_cast<uint4*>(&sh.head[i0]) = make_uint4(0, 0, 0, 0);
    write_run(&sh.x[i0], x);
    wave_sync();
    float picked[kTileRounds];
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        picked[r] = -kInf;
        if (s < in.sets) {
            if (in.end[r] > in.begin[r]) sh.head[in.begin[r]] = (uint16_t)(s + 1);
            if (chosen[r] >= in.end[r] - in.begin[r]) chosen[r] = -1;
            if (chosen[r] >= 0) picked[r] = sh.x[in.begin[r] + chosen[r]];
            // a masked row's logit is -inf, as one of that score is: the mask says which
            if (MASK && chosen[r] >= 0 && picked[r] == -kInf && !a.mask[a.off[in.set[r]] + chosen[r]]) chosen[r] = -1;
        }
    }
    wave_sync();
    TileSets sets;
    float v[kRun], w[kRun];
    if (alone) {
        float top = kLowest, sum = 0.0f, along = 0.0f;
#pragma unroll
        for (int k = 0; k < kRun; ++k) sets.id[k] = 1;
#pragma unroll
        for (int k = 0; k < kRun; k += 2) top = max3(top, x[k], x[k + 1]);
        top = wave_max(top);
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float d = __builtin_elementwise_maximum(x[k] - top, heat.low), e = heat_exp(d, heat);
            sum += e;
            along += e * d;
        }
        sum = wave_sum(sum);
        along = wave_sum(along);
        wave_sync();
        if (lane == 0) {
            sh.top[0] = top;
            sh.sum[0] = sum;
            sh.along[0] = along;
        }
    } else {
        sets.find(sh.head, lane);
        wave_sync();  // the heads have been read
        segment_reduce<TakeMax>(sets.seg, x, sets.id, lane, sh.top);
        wave_sync();
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            const float d = __builtin_elementwise_maximum(x[k] - sh.top[sets.id[k] - 1], heat.low);
            v[k] = heat_exp(d, heat);
            w[k] = v[k] * d;
        }
        segment_reduce<TakeSum>(sets.seg, v, sets.id, lane, sh.sum);
        segment_reduce<TakeSum>(sets.seg, w, sets.id, lane, sh.along);
    }
    wave_sync();
#pragma unroll
    for (int r = 0; r < kTileRounds; ++r) {
        const int s = r * kWave + lane;
        if (s < in.sets) {
            const bool empty = in.end[r] == in.begin[r];
            const SoftSums t{empty ? kLowest : sh.top[s], empty ? 0.0 : (double)sh.sum[s], empty ? 0.0 : (double)sh.along[s]};
            const double log_sum = log_near(t.sum);
            put_report(a, in.set[r], t, log_sum, chosen[r] >= 0, picked[r]);
            sh.sum[s] = (float)log_sum;
        }
    }
    if constexpr (LISTS) {
        wave_sync();
        prepare_lists(in, x, sets.id, sh);
        wave_sync();
    }
}

template <int TYPE, bool MASK, bool BIAS>
struct ReportTileIn {
    TileRows<TYPE, MASK, BIAS> rows;
    int32_t chosen[kTileRounds];

    __device__ __forceinline__ void load(const ReportArgs& a, const SetItem& im, int lane) {
        rows.load(a, im, lane);
#pragma unroll
        for (int r = 0; r < kTileRounds; ++r) chosen[r] = a.chosen && r * kWave + lane < rows.sets ? a.chosen[rows.set[r]] : -1;
    }
};

// The tiles, one a wave at a time, the first asked for before the bias is staged; or (`share`) one a workgroup, whose waves
// share its lists. Bound by the chain of a tile (loads, scans, lists) and by instructions: 100 thousand masked sets of 24
// rows with a bias 10.3 us (683 vector instructions a wave; 12.1 at 4 waves a SIMD), 16 thousand of 12 with lists of 8 12.3,
// one of 37 rows 6.
template <bool LISTS, int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, LISTS ? 3 : 5) void report_tile_kernel(ReportArgs a, bool share) {
    __shared__ std::conditional_t<LISTS, ReportTile, SumTile> tiles[kWaves];
    __shared__ RankGroup<kWave, LISTS ? kWaveList : 1> groups[kWaves];
    __shared__ BiasShared bias;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const bool one = LISTS && share;
    const int step = (int)gridDim.x * (one ? 1 : kWaves);
    auto& sh = tiles[one ? 0 : wave];
    int it = __builtin_amdgcn_readfirstlane(one ? (int)blockIdx.x : (int)blockIdx.x * kWaves + wave);
    ReportTileIn<TYPE, MASK, BIAS> in;
    in.load(a, a.tiles[min(it, a.num_tiles - 1)], lane);
    if (BIAS) stage_bias(a, bias);
    while (it < a.num_tiles) {
        if (!one || wave == 0) report_tile<LISTS, TYPE, MASK, BIAS>(a, in.rows, in.chosen, sh, &bias);
        if constexpr (LISTS) {
            if (one) {
                __syncthreads();
                take_lists(a, sh, groups[wave], wave, kWaves);
                __syncthreads();  // the lists have been taken
            } else {
                take_lists(a, sh, groups[wave], 0, 1);
            }
        }
        it += step;
        if (it < a.num_tiles) in.load(a, a.tiles[it], lane);
    }
}

// ------------------------------------------------------------------------------------ longer sets
template <int THREADS, int LIST>
struct ReportGroup {
    RankGroup<THREADS, LIST> rank;
    GroupSums<THREADS / kWave> sums;
};

// One set of more than kSetShort rows by a wave (THREADS 64), or a longer one or a part of it by a workgroup, its rows in
// registers.
template <int TYPE, bool MASK, bool BIAS, int THREADS, int RUNS, int LIST>
__device__ __forceinline__ void report_pass(const ReportArgs& a, const SetItem& im, int32_t index, ReportGroup<THREADS, LIST>& sh,
                                            const BiasShared* bias) {
    const int tid = (int)threadIdx.x & (THREADS - 1);
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~(kWave - 1));  // the wave's first thread
    const Heat heat{a.heat_hi, a.heat_lo, a.heat_low};
    const Span sp = span_of(a, im);
    const int64_t g = im.set0;
    RawRun<TYPE, MASK, BIAS> raw[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = kRun * (j * THREADS + tid);
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) raw[j].load(a, sp, i);
    }
    const int64_t r0 = a.off[g], size = a.off[g + 1] - r0;
    bool counts = false;
    float z = 0.0f;
    if (a.chosen && im.parts == 1 && wave0 == 0) {
        const int32_t c = a.chosen[g];
        counts = c >= 0 && c < size;
        if (MASK && counts) counts = a.mask[r0 + c] != 0;
        if (counts) z = one_logit<TYPE, BIAS>(a, bias, r0 + c);
    }
    float v[RUNS][kRun], tops[RUNS];
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        const int i = kRun * (j * THREADS + tid);
#pragma unroll
        for (int k = 0; k < kRun; ++k) v[j][k] = -kInf;
        if (kRun * (j * THREADS + wave0) < sp.hi && i < sp.hi) {
            uint32_t off;
            Buckets buckets;
            raw[j].logits(a, bias, sp, i, v[j], off, buckets);
        }
    }
    const int live = sp.hi <= kRun * wave0 ? 0 : (sp.hi - kRun * wave0 + kRun * THREADS - 1) / (kRun * THREADS);  // the wave's runs
    SoftSums t{kLowest, 0.0, 0.0};
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
        tops[j] = -kInf;
        if (j < live) t.top = max2(t.top, tops[j] = run_max(v[j]));
    }
    t.top = wave_max(t.top);
    // sums alone: roundings of single rows in either direction leave them as they are
    const HeatRows<false> rows(t.top, heat);
    float sum = 0.0f, along = 0.0f;
#pragma unroll
    for (int j = 0; j < RUNS; ++j)
        if (j < live)
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                const float d = rows.distance(v[j][k], heat), e = rows.exp(d, heat);
                sum += e;
                along = __builtin_fmaf(e, d, along);
            }
    const double all = team_sum((double)sum, 6), scale = (double)rows.scale();
    t.sum = all * scale;
    t.along = (team_sum((double)along, 6) - all * (double)rows.shift) * (scale * rows.unit(heat));
    t = join_waves<true>(a, t, sh.sums);
    const double log_sum = log_near(t.sum);
    if (tid == 0) {
        if (im.parts == 1)
            put_report(a, g, t, log_sum, counts, z);
        else
            a.part_sums[index] = t;
    }
    if (a.top > 0) {
        const int n = gather_best(a, v, tops, live, !(t.sum == t.sum), sp.q0 - r0, sh.rank, [&](int j, float(&x)[kRun]) {
            const int i = kRun * (j * THREADS + tid);
            uint32_t off;
            Buckets buckets;
#pragma unroll
            for (int k = 0; k < kRun; ++k) x[k] = -kInf;
            if (i < sp.hi) load_logits<TYPE, MASK, BIAS>(a, bias, sp, i, x, off, buckets);
        });
        if (im.parts == 1)
            rank_list<THREADS>(a, sh.rank.list, n, [&](int place, unsigned long long key) {
                const bool there = key != 0;
                put_entry(a, g * a.top + place, there ? (int32_t)~(uint32_t)key : -1,
                          there ? list_log_prob(a, rank_value((uint32_t)(key >> 32)), t.top, log_sum) : -kInf);
            });
        else
            rank_list<THREADS>(a, sh.rank.list, n,
                               [&](int place, unsigned long long key) { a.part_keys[(int64_t)index * a.top + place] = key; });
    }
    if (THREADS != kWave)
        __syncthreads();  // the list and the sums have been read
    else
        wave_sync();
}

// Workgroups [0, mid_blocks) take the sets for a wave, the others those for a workgroup, then the parts (all from num_mid +
// num_whole on, or those in `list`), one at a time. 30M bfloat16 rows of 17 thousand sets in 30 us (33 at 4 waves a SIMD, which
// is what masks, a bias and float16 have registers for): vector instructions are issued in two thirds of the time. Parts
// with lists of 64 12 us for 20 MB, a chain of a workgroup: rows, sums, bound, list.
template <int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock, BIAS ? 3 : MASK || TYPE == PB_F16 ? 4 : 5) void report_wide_kernel(ReportArgs a, int mid_blocks, int num_parts,
                                                             const int32_t* __restrict__ list) {
    __shared__ union {
        ReportGroup<kWave, kWaveList> mid[kWaves];
        ReportGroup<kBlock, kGroupList> whole;
    } sh;
    __shared__ BiasShared bias;
    if (BIAS) stage_bias(a, bias);
    if ((int)blockIdx.x < mid_blocks) {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), step = mid_blocks * kWaves;
        for (int it = (int)blockIdx.x * kWaves + wave; it < a.num_mid + a.num_shorts; it += step)
            report_pass<TYPE, MASK, BIAS, kWave, kWideRuns, kWaveList>(a, wave_item(a, it), it, sh.mid[wave], &bias);
    } else {
        const int n = a.num_whole + num_parts;
        for (int k = (int)blockIdx.x - mid_blocks; k < n; k += (int)gridDim.x - mid_blocks) {
            const int it = list && k >= a.num_whole ? list[k - a.num_whole] : a.num_mid + k;
            report_pass<TYPE, MASK, BIAS, kBlock, kWideRuns, kGroupList>(a, a.wide[it], it, sh.whole, &bias);
        }
    }
}

// Sets of up to THREADS * RUNS * 8 rows, a workgroup each. Bound by instructions: 4096 sets of 32 thousand bfloat16 rows with
// lists of 8 in 88 us (3.0 TB/s), 1156 vector instructions a wave of 64 rows a lane, 78 % of the time. One such set: 10.8 us
// (11.2 with 1024 lanes).
template <int TYPE, bool MASK, int THREADS, int RUNS>
__global__ __launch_bounds__(THREADS, 4) void report_big_kernel(ReportArgs a, const SetItem* __restrict__ items) {
    __shared__ ReportGroup<THREADS, kGroupList> sh;
    report_pass<TYPE, MASK, false, THREADS, RUNS, kGroupList>(a, items[blockIdx.x], 0, sh, nullptr);
}

__device__ __forceinline__ uint32_t block_count(uint32_t v, uint32_t* sh) {
    for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) sh[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kWaves; ++w) v += sh[w];
    return v;
}

// The sets in parts, a workgroup each: sums and lists from those of the parts. With d = top / parts, rounded up, entry d of
// a part says that d of its rows rank as high: the bound is the (top / d)-th largest of these, which at most top / d parts
// reach with all of their entries and the others with fewer than d of them, 64 x 64 at most. A chain of loads and counts:
// 22 sets in 600 parts with lists of 64 take 10 us (13 with the entries asked for after the bound), without lists 4.5.
template <int TYPE, bool MASK, bool BIAS>
__global__ __launch_bounds__(kBlock) void report_join_kernel(ReportArgs a, const int32_t* __restrict__ firsts) {
    constexpr int kAhead = 8, kHeld = 8;
    __shared__ unsigned long long list[kJoinList], bound;
    __shared__ uint32_t shc[kWaves], size;
    __shared__ GroupSums<kWaves> sums;
    __shared__ BiasShared bias;
    const int tid = (int)threadIdx.x;
    const int32_t first = firsts[blockIdx.x];
    const SetItem im = a.wide[first];
    const int64_t g = im.set0, r0 = a.off[g];
    const int n = im.parts;
    if (BIAS) stage_bias(a, bias);
    const unsigned long long* keys = a.part_keys + (int64_t)first * a.top;
    const int d = (a.top + n - 1) / n, want = d > 0 ? (a.top + d - 1) / d : 0;
    const bool bounded = (int64_t)n * a.top > kBlock, few = n <= kBoundParts;
    // up to 2048 entries are all asked for at once, before it is known which of them count
    const bool held = (int64_t)n * a.top <= kHeld * kBlock;
    unsigned long long own[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) own[u] = held && u * kBlock + tid < n * a.top ? keys[u * kBlock + tid] : 0ull;
    if (bounded && few)
        for (int j = tid; j < n; j += kBlock) list[j] = keys[(int64_t)j * a.top + d - 1];
    if (tid == 0) {
        size = 0;
        bound = 0;
    }
    bool counts = false;
    float z = 0.0f;
    if (tid == 0 && a.chosen) {
        const int32_t c = a.chosen[g];
        counts = c >= 0 && c < a.off[g + 1] - r0;
        if (MASK && counts) counts = a.mask[r0 + c] != 0;
        if (!BIAS && counts) z = one_logit<TYPE, BIAS>(a, &bias, r0 + c);
    }
    const SoftSums t = join_set<true>(a, a.part_sums + first, n, sums);  // a barrier within
    const double log_sum = log_near(t.sum);
    if (tid == 0) {
        if (BIAS && counts) z = one_logit<TYPE, BIAS>(a, &bias, r0 + (int64_t)a.chosen[g]);
        put_report(a, g, t, log_sum, counts, z);
    }
    if (a.top == 0) return;
    if (bounded) {
        if (few) {
            for (int j = tid; j < n; j += kBlock) {
                const unsigned long long key = list[j];
                if (keys_above(list, n, key) == want - 1 && key != 0) bound = key;  // keys other than 0 differ
            }
        } else {
            unsigned long long least = 0;
            for (int bit = 63; bit >= 0; --bit) {
                const unsigned long long trial = least | 1ull << bit;
                uint32_t c = 0;
                for (int j = tid; j < n; j += kBlock) c += keys[(int64_t)j * a.top + d - 1] >= trial ? 1u : 0u;
                if (block_count(c, shc) >= (uint32_t)want) least = trial;
            }
            if (tid == 0) bound = least;
        }
        __syncthreads();
    }
    // a part's entries down to the bound, kAhead asked for at a time
    const unsigned long long least = bound;
    __syncthreads();
    if (held)
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (own[u] != 0 && own[u] >= least) list[atomicAdd(&size, 1u)] = own[u];
    for (int j = held ? n : tid; j < n; j += kBlock) {
        const unsigned long long* mine = keys + (int64_t)j * a.top;
        bool more = true;
        for (int e = 0; more && e < a.top; e += kAhead) {
            unsigned long long key[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) key[u] = e + u < a.top ? mine[e + u] : 0ull;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                more = more && key[u] != 0 && key[u] >= least;
                if (more) list[atomicAdd(&size, 1u)] = key[u];
            }
        }
    }
    __syncthreads();
    int c = (int)size;
    if (c > kGroupList) {  // the a.top-th key itself, then what reaches it
        unsigned long long nth = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = nth | 1ull << bit;
            uint32_t m = 0;
            for (int i = tid; i < c; i += kBlock) m += list[i] >= trial ? 1u : 0u;
            if (block_count(m, shc) >= (uint32_t)a.top) nth = trial;
        }
        unsigned long long mine[kJoinList / kBlock];
#pragma unroll
        for (int i = 0; i < kJoinList / kBlock; ++i) mine[i] = i * kBlock + tid < c ? list[i * kBlock + tid] : 0ull;
        __syncthreads();
        if (tid == 0) size = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kJoinList / kBlock; ++i)
            if (mine[i] >= nth && mine[i] != 0) list[atomicAdd(&size, 1u)] = mine[i];
        __syncthreads();
        c = (int)size;
    }
    rank_list<kBlock>(a, list, c, [&](int place, unsigned long long key) {
        const bool there = key != 0;
        put_entry(a, g * a.top + place, there ? (int32_t)~(uint32_t)key : -1,
                  there ? list_log_prob(a, rank_value((uint32_t)(key >> 32)), t.top, log_sum) : -kInf);
    });
}

int tile_blocks(const SetLayout& s) { return s.num_shorts > 0 ? 0 : std::min((s.num_tiles + kWaves - 1) / kWaves, kChoiceGrid); }

int mid_blocks(const SetLayout& s) { return std::min((s.num_mid + s.num_shorts + kWaves - 1) / kWaves, kChoiceGrid); }

bool takes_big(const SetLayout& s, bool bias) {
    const bool alone = s.num_mid + s.num_shorts + s.num_whole + s.num_giant == 0;
    return !bias && s.num_big > 0 && (alone || s.num_big >= kBigSets);
}

int num_parts(const SetLayout& s, bool bias) { return takes_big(s, bias) ? s.num_giant : s.num_wide - s.num_whole; }

template <int TYPE, bool MASK, bool BIAS>
hipError_t launch_as(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    hipError_t e = hipSuccess;
    const bool big = takes_big(s, BIAS);
    const int parts = num_parts(s, BIAS);
    if constexpr (!BIAS) {
        const int half = s.num_half < s.num_big && s.num_big <= kOneLaunch ? 0 : s.num_half;
        if (big && s.num_big > half) {
            hipLaunchKernelGGL((report_big_kernel<TYPE, MASK, 1024, 8>), dim3(s.num_big - half), dim3(1024), 0, stream, a, s.big + half);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        if (big && half > 0) {
            hipLaunchKernelGGL((report_big_kernel<TYPE, MASK, 512, 8>), dim3(half), dim3(512), 0, stream, a, s.big);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    const int wide = mid_blocks(s) + std::min(s.num_whole + parts, kChoiceGrid);
    if (wide > 0) {
        hipLaunchKernelGGL((report_wide_kernel<TYPE, MASK, BIAS>), dim3(wide), dim3(kBlock), 0, stream, a, mid_blocks(s), parts,
                           big ? s.giant : nullptr);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (tile_blocks(s) > 0) {
        const bool share = a.top > 0 && s.num_tiles <= kSharedTiles;
        const dim3 grid(share ? s.num_tiles : tile_blocks(s));
        if (a.top > 0)
            hipLaunchKernelGGL((report_tile_kernel<true, TYPE, MASK, BIAS>), grid, dim3(kBlock), 0, stream, a, share);
        else
            hipLaunchKernelGGL((report_tile_kernel<false, TYPE, MASK, BIAS>), grid, dim3(kBlock), 0, stream, a, false);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    const int joins = big ? s.num_split - s.num_big : s.num_split;
    if (joins > 0) {
        hipLaunchKernelGGL((report_join_kernel<TYPE, MASK, BIAS>), dim3(joins), dim3(kBlock), 0, stream, a, big ? s.giant_split : s.split);
        e = hipGetLastError();
    }
    return e;
}

template <int TYPE>
hipError_t launch_typed(const SetLayout& s, const ReportArgs& a, hipStream_t stream) {
    if (a.mask) return a.table ? launch_as<TYPE, true, true>(s, a, stream) : launch_as<TYPE, true, false>(s, a, stream);
    return a.table ? launch_as<TYPE, false, true>(s, a, stream) : launch_as<TYPE, false, false>(s, a, stream);
}

int64_t part_items(const SetLayout& s, bool bias) { return num_parts(s, bias) > 0 ? s.num_mid + s.num_wide : 0; }

}  // namespace

int64_t report_work_bytes(const SetLayout& s, int32_t top, bool bias) {
    return part_items(s, bias) * ((int64_t)sizeof(SoftSums) + 8 * top);
}

hipError_t launch_report(const SetLayout& s, ReportArgs a, int32_t type, char* work, hipStream_t stream) {
    a.off = s.off;
    a.tiles = s.tiles;
    a.wide = s.wide;
    a.segments = s.segments;
    a.num_tiles = s.num_tiles;
    a.shorts = s.shorts;
    a.num_shorts = s.num_shorts;
    a.num_wide = s.num_wide;
    a.num_mid = s.num_mid;
    a.num_whole = s.num_whole;
    a.rows = s.rows;
    a.part_sums = reinterpret_cast<SoftSums*>(work);
    a.part_keys = reinterpret_cast<unsigned long long*>(work + sizeof(SoftSums) * part_items(s, a.num_buckets > 0));
    a.team_bits = 0;
    while (1 << a.team_bits < a.top) ++a.team_bits;
    const auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    a.vec = a.stride == 1 && at(a.scores, 16) && at(a.mask, 8) && at(a.positions, 16);
    if (type == PB_BF16) return launch_typed<PB_BF16>(s, a, stream);
    if (type == PB_F16) return launch_typed<PB_F16>(s, a, stream);
    return launch_typed<PB_F32>(s, a, stream);
}

}  // namespace pb
