// Laying out pairs of values: each value's entries (pair * 2 + (1 where it is the loser)), in the order of
// its pairs. Entry i is of pair i / 2, so a stable sort of the entries by their values is that layout: a radix
// sort, 8 bits of the value a pass. A pass counts each workgroup's digits, sums the counts over the
// workgroups before it and writes its entries behind theirs; within a wave an entry's place is the number of
// lanes below that hold its digit, so equal digits keep their order and the layout has one result only.
//
// A pass reads an entry twice and writes it once (4 + 8 + 8 bytes) at places that are scattered over 256
// runs, and is bound by those writes: for 10M entries of 1M values 16 to 27 us to count and 87 to 226 us to
// write, three passes of them, 0.65 ms in all. What a caller waits for is the device memory taken for the
// call and the list starts that go to the host, whose lists' work is laid out there (4.4 ms).
#include "pb_internal.h"

namespace pb {
namespace {

constexpr int kWaves = kBlock / kWave;
constexpr int kDigitBits = 8;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortRun = 1024;  // consecutive entries of a wave
constexpr int kSortChunk = kSortRun * kWaves;
static_assert(kDigits == kBlock, "a thread to a digit");

struct SortPass {
    const int32_t* winners;  // first pass: entry i's value is winners[i / 2] or losers[i / 2]
    const int32_t* losers;
    const uint32_t* keys;    // later ones
    const int32_t* entries;
    uint32_t* keys_out;
    int32_t* entries_out;
    uint32_t* counts;  // [kDigits][blocks]: a workgroup's entries of a digit, then those of the ones before it
    uint32_t* totals;  // [kDigits]
    int64_t n;
    int32_t blocks;
    int32_t shift;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t key_of(const SortPass& a, int64_t i) {
    if (!FIRST) return a.keys[i];
    return (uint32_t)(i & 1 ? a.losers[i >> 1] : a.winners[i >> 1]);
}

__device__ __forceinline__ uint32_t digit_of(const SortPass& a, uint32_t key) { return key >> a.shift & (kDigits - 1); }

// LDS written by lanes of this wave is read by others of it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The sum of v over the threads before this one; `total`: over all of them.
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t* sh, uint32_t& total) {
    const int lane = (int)threadIdx.x & (kWave - 1), wave = (int)threadIdx.x / kWave;
    uint32_t upto = v;
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const uint32_t t = __shfl_up(upto, m);
        if (lane >= m) upto += t;
    }
    __syncthreads();
    if (lane == kWave - 1) sh[wave] = upto;
    __syncthreads();
    uint32_t before = upto - v;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sh[w];
        total += sh[w];
    }
    return before;
}

template <bool FIRST>
__global__ __launch_bounds__(kBlock) void digit_count_kernel(SortPass a) {
    __shared__ uint32_t count[kDigits];
    const int tid = (int)threadIdx.x;
    const int64_t i0 = (int64_t)blockIdx.x * kSortChunk, end = min(i0 + kSortChunk, a.n);
    count[tid] = 0;
    __syncthreads();
    for (int64_t i = i0 + tid; i < end; i += kBlock) atomicAdd(&count[digit_of(a, key_of<FIRST>(a, i))], 1u);
    __syncthreads();
    a.counts[(int64_t)tid * a.blocks + blockIdx.x] = count[tid];
}

// A workgroup to a digit: its counts become those of the workgroups before.
__global__ __launch_bounds__(kBlock) void digit_scan_kernel(SortPass a) {
    __shared__ uint32_t sh[kWaves];
    uint32_t* row = a.counts + (int64_t)blockIdx.x * a.blocks;
    uint32_t carry = 0;
    for (int b0 = 0; b0 < a.blocks; b0 += kBlock) {
        const int b = b0 + (int)threadIdx.x;
        uint32_t total;
        const uint32_t before = block_before(b < a.blocks ? row[b] : 0, sh, total);
        if (b < a.blocks) row[b] = carry + before;
        carry += total;
    }
    if (threadIdx.x == 0) a.totals[blockIdx.x] = carry;
}

template <bool FIRST>
__global__ __launch_bounds__(kBlock) void digit_scatter_kernel(SortPass a) {
    __shared__ uint32_t at[kWaves][kDigits];  // a wave's entries of a digit, then where the next one goes
    __shared__ uint32_t sh[kWaves];
    const int tid = (int)threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
    const int64_t i0 = (int64_t)blockIdx.x * kSortChunk + (int64_t)wave * kSortRun, end = min(i0 + kSortRun, a.n);
    for (int w = 0; w < kWaves; ++w) at[w][tid] = 0;
    __syncthreads();
    for (int64_t i = i0 + lane; i < end; i += kWave) atomicAdd(&at[wave][digit_of(a, key_of<FIRST>(a, i))], 1u);
    uint32_t all;
    uint32_t next = block_before(a.totals[tid], sh, all) + a.counts[(int64_t)tid * a.blocks + blockIdx.x];
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t t = at[w][tid];
        at[w][tid] = next;
        next += t;
    }
    __syncthreads();
    for (int64_t j0 = i0; j0 < end; j0 += kWave) {
        const int64_t i = j0 + lane;
        const bool live = i < end;
        const uint32_t key = live ? key_of<FIRST>(a, i) : 0;
        const uint32_t digit = digit_of(a, key);
        unsigned long long same = __ballot(live);  // the lanes that hold the digit
#pragma unroll
        for (int bit = 0; bit < kDigitBits; ++bit) {
            const bool one = digit >> bit & 1u;
            const unsigned long long ones = __ballot(one);
            same &= one ? ones : ~ones;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        const uint32_t first = at[wave][digit];
        wave_sync();
        if (live && rank == 0) at[wave][digit] = first + (uint32_t)__popcll(same);
        wave_sync();
        if (live) {
            a.keys_out[first + rank] = key;
            a.entries_out[first + rank] = FIRST ? (int32_t)i : a.entries[i];
        }
    }
}

// off[v]: the first entry of a value of at least v.
__global__ __launch_bounds__(kBlock) void list_start_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                            int64_t num_values, int64_t* __restrict__ off) {
    const int64_t v = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (v > num_values) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = lo + (hi - lo) / 2;
        if ((int64_t)keys[mid] < v)
            lo = mid + 1;
        else
            hi = mid;
    }
    off[v] = lo;
}

__global__ __launch_bounds__(kBlock) void narrow_kernel(const int64_t* __restrict__ winners,
                                                        const int64_t* __restrict__ losers, int64_t num_pairs,
                                                        int64_t num_values, int32_t* __restrict__ out,
                                                        int32_t* __restrict__ bad) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= 2 * num_pairs) return;
    const int64_t v = i < num_pairs ? winners[i] : losers[i - num_pairs];
    const bool in = v >= 0 && v < num_values;
    if (!in) *bad = 1;
    out[i] = in ? (int32_t)v : 0;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int64_t sort_blocks(int64_t n) { return (n + kSortChunk - 1) / kSortChunk; }

unsigned int blocks_of(int64_t n) { return (unsigned int)((n + kBlock - 1) / kBlock); }

}  // namespace

size_t pair_layout_bytes(int64_t num_pairs, int64_t num_values) {
    const int64_t n = 2 * num_pairs;
    return round256((size_t)(num_values + 1) * 8) + 3 * round256((size_t)n * 4) +
           round256((size_t)(sort_blocks(n) * kDigits + kDigits) * 4);
}

hipError_t launch_narrow_pairs(const int64_t* winners, const int64_t* losers, int64_t num_pairs, int64_t num_values,
                               int32_t* out, int32_t* bad, hipStream_t stream) {
    hipLaunchKernelGGL(narrow_kernel, dim3(blocks_of(2 * num_pairs)), dim3(kBlock), 0, stream, winners, losers, num_pairs,
                       num_values, out, bad);
    return hipGetLastError();
}

hipError_t launch_pair_layout(int32_t* pairs, int64_t num_pairs, int64_t num_values, void* work, hipStream_t stream) {
    const int64_t n = 2 * num_pairs;
    char* p = static_cast<char*>(work);
    int64_t* off = reinterpret_cast<int64_t*>(p);
    p += round256((size_t)(num_values + 1) * 8);
    uint32_t* keys[2];
    for (uint32_t*& k : keys) {
        k = reinterpret_cast<uint32_t*>(p);
        p += round256((size_t)n * 4);
    }
    int32_t* lists[2] = {reinterpret_cast<int32_t*>(p), pairs + n};
    p += round256((size_t)n * 4);
    int passes = 1;
    while (passes < 4 && (num_values - 1) >> (kDigitBits * passes) != 0) ++passes;
    SortPass a{};
    a.winners = pairs;
    a.losers = pairs + num_pairs;
    a.totals = reinterpret_cast<uint32_t*>(p);
    a.counts = a.totals + kDigits;
    a.n = n;
    a.blocks = (int32_t)sort_blocks(n);
    int to = passes & 1;  // so that the last pass writes the lists in their place
    for (int i = 0; i < passes; ++i, to ^= 1) {
        a.keys_out = keys[to];
        a.entries_out = lists[to];
        a.keys = keys[to ^ 1];
        a.entries = lists[to ^ 1];
        a.shift = kDigitBits * i;
        const dim3 grid((unsigned int)a.blocks);
        if (i == 0)
            hipLaunchKernelGGL(digit_count_kernel<true>, grid, dim3(kBlock), 0, stream, a);
        else
            hipLaunchKernelGGL(digit_count_kernel<false>, grid, dim3(kBlock), 0, stream, a);
        hipLaunchKernelGGL(digit_scan_kernel, dim3(kDigits), dim3(kBlock), 0, stream, a);
        if (i == 0)
            hipLaunchKernelGGL(digit_scatter_kernel<true>, grid, dim3(kBlock), 0, stream, a);
        else
            hipLaunchKernelGGL(digit_scatter_kernel<false>, grid, dim3(kBlock), 0, stream, a);
    }
    hipLaunchKernelGGL(list_start_kernel, dim3(blocks_of(num_values + 1)), dim3(kBlock), 0, stream, a.keys_out, n, num_values,
                       off);
    return hipGetLastError();
}

}  // namespace pb
