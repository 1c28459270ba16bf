// Reports on choices and distillation (report.hip, report_grads.hip, distill.hip): their arguments and entry points.
#pragma once

#include "pb_internal.h"

namespace pb {

constexpr int kMaxTop = 64;  // entries of a set's list, a lane each
// A set's, or a part's, logits: their maximum, the sum of exponentials over it, and the sum of these times the distance
// to it. Nothing: the lowest maximum, 0, 0.
struct SoftSums {
    float top;
    double sum, along;
};
struct ReportArgs : ChoiceArgs {
    double inv_temp;
    float temp;
    float heat_hi, heat_lo, heat_low;  // log2(e) / T in two parts; see Heat
    int32_t top;                       // entries of each set's list
    int32_t num_shorts;                // sets that waves take behind the mid ones, instead of tiles
    const SetItem* shorts;
    int32_t team_bits;                 // 1 << team_bits lanes take it
    SoftSums* part_sums;               // of the parts of split sets, by wide item
    unsigned long long* part_keys;     // [top] of each, best first
    float* entropy;
    int32_t* top_index;
    float* top_log_probs;
    const float* grad_entropy;
    // the teacher's
    const int32_t* entry_index;
    const void* entry_logits;
    int32_t entry_type;
    bool tail;
    float* kl;
};
int64_t report_work_bytes(const SetLayout& s, int32_t top, bool bias);
hipError_t launch_report(const SetLayout& s, ReportArgs a, int32_t type, char* work, hipStream_t stream);
// distill: the loss's gradient, else that of the log-probabilities and entropies; `sums` are in the workspace
int64_t soft_grads_work_bytes(const SetLayout& s, bool distill, int32_t num_buckets);
hipError_t launch_distill(const SetLayout& s, const ReportArgs& a, int32_t type, hipStream_t stream);
hipError_t launch_soft_grads(bool distill, const SetLayout& s, ReportArgs a, int32_t type, char* work, hipStream_t stream);

}  // namespace pb
