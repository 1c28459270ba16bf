// Gradients of the chosen rows' log-probabilities and of the entropies, and what they share with the loss of distillation;
// see soft_grads.h.
#include "soft_grads.h"

namespace pb {
namespace {

int64_t sum_cols(const SetLayout& s, bool distill, int32_t num_buckets) {
    return soft_blocks(s, num_buckets > 0) <= 1 ? 0 : (distill ? 1 : 0) + num_buckets;
}

}  // namespace

int64_t soft_grads_work_bytes(const SetLayout& s, bool distill, int32_t num_buckets) {
    return 8 * sum_cols(s, distill, num_buckets) * soft_blocks(s, num_buckets > 0) +
           (num_parts(s, num_buckets > 0) > 0 ? (int64_t)sizeof(SoftSums) * (s.num_mid + s.num_wide) : 0);
}

hipError_t launch_soft_grads(bool distill, const SetLayout& s, ReportArgs a, int32_t type, char* work, hipStream_t stream) {
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
    a.blocks = soft_blocks(s, a.num_buckets > 0);
    a.rows = s.rows;
    a.sums = reinterpret_cast<double*>(work);
    a.part_sums = reinterpret_cast<SoftSums*>(a.sums + sum_cols(s, distill, a.num_buckets) * a.blocks);
    a.team_bits = 0;
    while (1 << a.team_bits < a.top) ++a.team_bits;
    const auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    a.vec = a.stride == 1 && at(a.scores, 16) && at(a.grad_scores, 16) && at(a.mask, 8) && at(a.positions, 16);
    const hipError_t e = distill ? launch_distill(s, a, type, stream) : launch_mode<false>(s, a, type, stream);
    const int32_t cols = (distill ? 1 : 0) + a.num_buckets;
    if (e != hipSuccess || cols == 0 || a.blocks == 1) return e;
    return launch_join_sums(a.sums, a.blocks, cols, distill ? 1 : 0, a.stats, a.grad_table, stream);
}

}  // namespace pb
