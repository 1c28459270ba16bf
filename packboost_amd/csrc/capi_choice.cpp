// C-ABI host layer of the choice and preference operators: their layouts (built on the host, kept on
// the device), argument checks, workspaces.
#include <algorithm>
#include <memory>
#include <exception>
#include <string>
#include <vector>

#include "pb_internal.h"
#include "report.h"

struct pb_sets {
    pb::SetLayout s;
    int32_t device;
    char* arena;  // offsets, items and split list
    int64_t largest;
};

struct pb_pairs {
    pb::PairLayout p;
    int32_t device;
    pb_sets* lists;
    pb_sets* seqs;
    int32_t* arena;  // winners, losers, entries
};

namespace {

using pb::SetItem;

void free_sets(pb_sets* s) {
    if (!s) return;
    if (s->arena) (void)hipFree(s->arena);
    delete s;
}

void free_pairs(pb_pairs* p) {
    if (!p) return;
    free_sets(p->lists);
    free_sets(p->seqs);
    if (p->arena) (void)hipFree(p->arena);
    delete p;
}

// Lanes to a set of a tile: about 4 rows a lane on average and at most 32 in the tile's largest set,
// whose lanes the others' would wait for.
int32_t team_of(int64_t rows, int64_t sets, int64_t largest) {
    int32_t t = 0;
    while (t < 6 && (((int64_t)4 << t) * sets < rows || ((int64_t)32 << t) < largest)) ++t;
    return t;
}

struct Layout {
    std::vector<SetItem> tiles, mid, whole, parts, half, big, shorts;
    std::vector<pb::TileSegment> segments;
    std::vector<int32_t> split;  // the first part of each split set, within `parts`
    std::vector<int32_t> giant;  // the parts of sets that are not in `half` or `big`, too, and the first of each
    std::vector<int32_t> giant_split;
};

// The tile that is being filled.
class TileFill {
  public:
    TileFill(Layout& out, bool segments) : out_(out), most_segments_(segments ? pb::kTileSegments : 1) {}

    // a longer set lies between the sets before and those after
    void interrupt() { broken_ = tile_.sets > 0; }

    void add(int64_t row0, int64_t size, int64_t set) {
        if (tile_.sets > 0 && !fits(row0, size)) flush();
        if (tile_.sets == 0) {
            tile_.row0 = row0;
            tile_.set0 = (int32_t)set;
            row0_ = row0;
            rows_ = lane0_ = 0;
        } else if (broken_) {
            if (tile_.parts == 0) tile_.part = (int32_t)out_.segments.size();
            lane0_ = lanes();
            row0_ = row0;
            rows_ = 0;
            out_.segments.push_back({row0, 0, (int32_t)set, (int32_t)lane0_, tile_.sets});
            ++tile_.parts;
        }
        broken_ = false;
        rows_ += size;
        (tile_.parts == 0 ? tile_.rows : out_.segments.back().rows) = (int32_t)rows_;
        total_ += size;
        ++tile_.sets;
        largest_ = std::max(largest_, size);
    }

    void flush() {
        broken_ = false;
        if (tile_.sets == 0) return;
        tile_.team = team_of(total_, tile_.sets, largest_);
        out_.tiles.push_back(tile_);
        tile_ = SetItem{};
        total_ = largest_ = 0;
    }

  private:
    static int64_t lanes_of(int64_t row0, int64_t rows) { return rows == 0 ? 0 : ((row0 & 7) + rows + 7) / 8; }
    int64_t lanes() const { return lane0_ + lanes_of(row0_, rows_); }
    bool fits(int64_t row0, int64_t size) const {
        if (tile_.sets == pb::kSetTileSets) return false;
        if (!broken_) return lane0_ + lanes_of(row0_, rows_ + size) <= pb::kWave;
        return tile_.parts + 1 < most_segments_ && lanes() + lanes_of(row0, size) <= pb::kWave;
    }

    Layout& out_;
    const int most_segments_;
    SetItem tile_{};
    bool broken_ = false;
    int64_t row0_ = 0, rows_ = 0, lane0_ = 0;  // of the last segment
    int64_t total_ = 0, largest_ = 0;
};

SetItem whole_set(const int64_t* off, int64_t g) {
    SetItem im{};
    im.row0 = off[g];
    im.rows = (int32_t)std::min<int64_t>(off[g + 1] - off[g], pb::kSetWideRows);
    im.set0 = (int32_t)g;
    im.sets = im.parts = 1;
    return im;
}

void lay_out(const int64_t* off, int64_t num_sets, bool segments, Layout& out) {
    TileFill tiles(out, segments);
    for (int64_t g = 0; g < num_sets; ++g) {
        const int64_t size = off[g + 1] - off[g];
        if (size <= pb::kSetShort) {
            tiles.add(off[g], size, g);
            if ((int)out.shorts.size() <= pb::kSetFewShorts) out.shorts.push_back(whole_set(off, g));
            continue;
        }
        tiles.interrupt();
        SetItem im = whole_set(off, g);
        if ((off[g] & 7) + size <= pb::kSetMidRows) {
            out.mid.push_back(im);
        } else if ((off[g] & 7) + size <= pb::kSetWideRows) {
            out.whole.push_back(im);
        } else {
            const int64_t most = pb::kSetWideRows - 8;
            const int64_t want = (size + most - 1) / most;
            const int64_t each = ((size + want - 1) / want + 7) / 8 * 8;  // at most `most`, itself a multiple of 8
            const int64_t span = (off[g] & 7) + size;
            if (span <= pb::kSetBig) {
                im.rows = (int32_t)size;
                (span <= pb::kSetHalfBig ? out.half : out.big).push_back(im);
            }
            im.parts = (int32_t)((size + each - 1) / each);
            out.split.push_back((int32_t)out.parts.size());
            for (im.part = 0; im.part < im.parts; ++im.part) {
                if (span > pb::kSetBig) out.giant.push_back((int32_t)out.parts.size());
                if (span > pb::kSetBig && im.part == 0) out.giant_split.push_back((int32_t)out.parts.size());
                im.row0 = off[g] + im.part * each;
                im.rows = (int32_t)std::min(each, off[g + 1] - im.row0);
                out.parts.push_back(im);
            }
        }
    }
    tiles.flush();
    if ((int)out.shorts.size() > pb::kSetFewShorts || out.mid.size() + out.whole.size() + out.parts.size() == 0) out.shorts.clear();
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// segments: tiles may hold sets from either side of longer ones (not where sums are laid out).
int sets_create(const int64_t* off, int64_t num_sets, bool segments, pb_sets** out) {
    if (num_sets < 0 || num_sets >= INT32_MAX) return pb::api_fail(PB_ERR_UNSUPPORTED, "pb_sets_create: num_sets must lie in [0, 2^31 - 1)");
    if (off[0] != 0) return pb::api_fail(PB_ERR_INVALID, "pb_sets_create: offsets must start at 0");
    for (int64_t g = 0; g < num_sets; ++g)
        if (off[g + 1] < off[g]) return pb::api_fail(PB_ERR_INVALID, "pb_sets_create: offsets must not decrease");
    if (off[num_sets] > ((int64_t)1 << 37))  // what the sums of the bias table's gradient hold
        return pb::api_fail(PB_ERR_UNSUPPORTED, "pb_sets_create: more than 2^37 rows");
    Layout lay;
    lay_out(off, num_sets, segments, lay);
    const size_t tiles = lay.tiles.size(), mid = lay.mid.size(), whole = lay.whole.size();
    std::vector<SetItem>& items = lay.tiles;  // the tiles, the wide items
    items.insert(items.end(), lay.mid.begin(), lay.mid.end());
    items.insert(items.end(), lay.whole.begin(), lay.whole.end());
    items.insert(items.end(), lay.parts.begin(), lay.parts.end());
    const size_t wide_end = items.size(), half = lay.half.size();
    items.insert(items.end(), lay.half.begin(), lay.half.end());
    items.insert(items.end(), lay.big.begin(), lay.big.end());
    const size_t big_end = items.size();
    items.insert(items.end(), lay.shorts.begin(), lay.shorts.end());
    for (int32_t& first : lay.split) first += (int32_t)(mid + whole);
    for (int32_t& part : lay.giant) part += (int32_t)(mid + whole);
    for (int32_t& part : lay.giant_split) part += (int32_t)(mid + whole);
    std::vector<int32_t>& split = lay.split;  // and `giant`, `giant_split` behind it
    const size_t num_split = split.size();
    split.insert(split.end(), lay.giant.begin(), lay.giant.end());
    split.insert(split.end(), lay.giant_split.begin(), lay.giant_split.end());
    const size_t b_off = round256(sizeof(int64_t) * (size_t)(num_sets + 1));
    const size_t b_items = round256(sizeof(SetItem) * items.size());
    const size_t b_split = round256(sizeof(int32_t) * split.size());
    const size_t b_segments = round256(sizeof(pb::TileSegment) * lay.segments.size());
    std::vector<char> host(b_off + b_items + b_split + b_segments);
    std::copy_n(off, num_sets + 1, reinterpret_cast<int64_t*>(host.data()));
    std::copy(items.begin(), items.end(), reinterpret_cast<SetItem*>(host.data() + b_off));
    std::copy(split.begin(), split.end(), reinterpret_cast<int32_t*>(host.data() + b_off + b_items));
    std::copy(lay.segments.begin(), lay.segments.end(),
              reinterpret_cast<pb::TileSegment*>(host.data() + b_off + b_items + b_split));
    pb_sets* h = new pb_sets();
    hipError_t e = hipGetDevice(&h->device);
    if (e == hipSuccess) e = hipMalloc(&h->arena, host.size());
    if (e == hipSuccess) e = hipMemcpy(h->arena, host.data(), host.size(), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        free_sets(h);
        return pb::api_hip_fail(e, "pb_sets_create");
    }
    h->s.off = reinterpret_cast<int64_t*>(h->arena);
    h->s.tiles = reinterpret_cast<SetItem*>(h->arena + b_off);
    h->s.wide = h->s.tiles + tiles;
    h->s.split = reinterpret_cast<int32_t*>(h->arena + b_off + b_items);
    h->s.segments = reinterpret_cast<pb::TileSegment*>(h->arena + b_off + b_items + b_split);
    h->s.num_tiles = (int32_t)tiles;
    h->s.num_mid = (int32_t)mid;
    h->s.num_wide = (int32_t)(wide_end - tiles - mid);
    h->s.num_whole = (int32_t)whole;
    h->s.num_split = (int32_t)num_split;
    h->s.big = h->s.tiles + wide_end;
    h->s.num_big = (int32_t)(big_end - wide_end);
    h->s.shorts = h->s.tiles + big_end;
    h->s.num_shorts = (int32_t)lay.shorts.size();
    h->s.num_half = (int32_t)half;
    h->s.giant = h->s.split + num_split;
    h->s.num_giant = (int32_t)lay.giant.size();
    h->s.giant_split = h->s.giant + lay.giant.size();
    h->s.num_sets = num_sets;
    h->s.rows = off[num_sets];
    for (int64_t g = 0; g < num_sets; ++g) h->largest = std::max(h->largest, off[g + 1] - off[g]);
    *out = h;
    return PB_OK;
}

// Device memory for the time of a call.
struct DeviceScratch {
    void* at = nullptr;
    ~DeviceScratch() {
        if (at) (void)hipFree(at);
    }
};

// The pairs by index: on the host, or (from_device) on the device, where `stream` has written them.
int pairs_create(const char* who, const int64_t* winners, const int64_t* losers, int64_t num_pairs, int64_t num_values,
                 const int64_t* seq_off, bool from_device, hipStream_t stream, pb_pairs** out) {
    const auto bad = [&](int code, const char* what) {
        return pb::api_fail(code, (std::string(who) + ": " + what).c_str());
    };
    if (num_values >= INT32_MAX || num_pairs >= ((int64_t)1 << 30))
        return bad(PB_ERR_UNSUPPORTED, "at most 2^30 pairs and 2^31 - 2 values");
    const char* range = "a pair names a value out of range";
    std::vector<int32_t> host;  // winners, losers
    if (!from_device && num_pairs > 0) {
        host.resize((size_t)num_pairs * 2);
        for (int64_t i = 0; i < 2 * num_pairs; ++i) {
            const int64_t v = i < num_pairs ? winners[i] : losers[i - num_pairs];
            if (v < 0 || v >= num_values) return bad(PB_ERR_RANGE, range);
            host[(size_t)i] = (int32_t)v;
        }
    }
    std::unique_ptr<pb_pairs, void (*)(pb_pairs*)> h(new pb_pairs(), free_pairs);
    std::vector<int64_t> off((size_t)num_values + 1, 0);
    hipError_t e = hipGetDevice(&h->device);
    if (e == hipSuccess) e = hipMalloc(&h->arena, std::max<size_t>(256, (size_t)num_pairs * 16));
    if (e == hipSuccess && num_pairs > 0) {
        DeviceScratch work;
        int32_t wrong = 0;
        e = hipMalloc(&work.at, pb::pair_layout_bytes(num_pairs, num_values));
        int32_t* flag = static_cast<int32_t*>(work.at);
        if (e == hipSuccess && from_device) {
            if ((e = hipMemcpyAsync(flag, &wrong, sizeof(wrong), hipMemcpyHostToDevice, stream)) == hipSuccess &&
                (e = pb::launch_narrow_pairs(winners, losers, num_pairs, num_values, h->arena, flag, stream)) == hipSuccess &&
                (e = hipMemcpyAsync(&wrong, flag, sizeof(wrong), hipMemcpyDeviceToHost, stream)) == hipSuccess)
                e = hipStreamSynchronize(stream);
            if (e == hipSuccess && wrong) return bad(PB_ERR_RANGE, range);
        } else if (e == hipSuccess) {
            e = hipMemcpy(h->arena, host.data(), host.size() * sizeof(int32_t), hipMemcpyHostToDevice);
        }
        if (e == hipSuccess) e = pb::launch_pair_layout(h->arena, num_pairs, num_values, work.at, stream);
        if (e == hipSuccess)
            e = hipMemcpyAsync(off.data(), work.at, off.size() * sizeof(int64_t), hipMemcpyDeviceToHost, stream);
        const hipError_t waited = hipStreamSynchronize(stream);  // whatever was enqueued uses `work` and `off`
        if (e == hipSuccess) e = waited;
    }
    if (e != hipSuccess) return pb::api_hip_fail(e, who);
    int rc = sets_create(off.data(), num_values, false, &h->lists);
    if (rc == PB_OK && seq_off) rc = sets_create(seq_off, num_values, false, &h->seqs);
    if (rc != PB_OK) return rc;
    h->p.winners = h->arena;
    h->p.losers = h->arena + num_pairs;
    h->p.entries = h->arena + 2 * num_pairs;
    h->p.num_pairs = num_pairs;
    h->p.lists = h->lists->s;
    h->p.has_seqs = h->seqs != nullptr;
    if (h->seqs) h->p.seqs = h->seqs->s;
    *out = h.release();
    return PB_OK;
}

int pairs_entry(const char* who, const int64_t* winners, const int64_t* losers, int64_t num_pairs, int64_t num_values,
                const int64_t* seq_off, bool from_device, hipStream_t stream, pb_pairs** out) {
    const auto bad = [&](int code, const char* what) {
        return pb::api_fail(code, (std::string(who) + ": " + what).c_str());
    };
    try {
        if (!out) return bad(PB_ERR_INVALID, "null output");
        *out = nullptr;
        if (num_pairs < 0 || num_values < 0 || (num_pairs > 0 && (!winners || !losers)))
            return bad(PB_ERR_INVALID, "bad shape or null pairs");
        return pairs_create(who, winners, losers, num_pairs, num_values, seq_off, from_device, stream, out);
    } catch (const std::exception&) {
        return pb::api_fail(PB_ERR_NOMEM, "pairs: out of host memory");
    }
}

// Sums that a workgroup leaves (none where there is one workgroup, which writes the results itself).
int64_t sum_cols(const pb_sets* s, int32_t op, int32_t num_buckets) {
    if (op == PB_LOG_PROBS || pb::choice_grid(s->s) <= 1) return 0;
    return (op == PB_POLICY ? 3 : 0) + num_buckets;
}

int64_t work_need(const pb_sets* s, int32_t op, int32_t num_buckets) {
    const int64_t parts = s->s.num_wide > s->s.num_whole ? s->s.num_mid + s->s.num_wide : 0;
    return 8 * (sum_cols(s, op, num_buckets) * pb::choice_grid(s->s) + parts);
}

// Checks what every choice call takes (its workspace of `need` bytes among it) and fills the arguments it shares.
int scores_args(const char* who, const pb_sets* s, const pb_choice_scores* in, const void* work, int64_t work_bytes,
                int64_t need, pb::ChoiceArgs& a) {
    const auto bad = [&](int code, const char* what) {
        return pb::api_fail(code, (std::string(who) + ": " + what).c_str());
    };
    if (s->s.rows > 0 && !in->scores_dev) return bad(PB_ERR_INVALID, "null scores");
    if (in->score_type != PB_F32 && in->score_type != PB_BF16 && in->score_type != PB_F16)
        return bad(PB_ERR_UNSUPPORTED, "scores must be float32, bfloat16 or float16");
    if (in->num_buckets > 0 && (!in->table_dev || !in->buckets_dev || (s->s.rows > 0 && !in->positions_dev)))
        return bad(PB_ERR_INVALID, "a position bias needs its table, buckets and positions");
    if (in->num_buckets > 0 && in->reach < 0) return bad(PB_ERR_INVALID, "reach must not be negative");
    if (need > 0 && (!work || work_bytes < need)) return bad(PB_ERR_INVALID, "workspace too small");
    if (reinterpret_cast<uintptr_t>(work) & 15) return bad(PB_ERR_INVALID, "workspace must be 16-byte aligned");
    a.num_buckets = in->num_buckets;
    a.scores = in->scores_dev;
    a.stride = in->score_stride;
    a.mask = in->mask_dev;
    a.positions = in->positions_dev;
    a.table = in->num_buckets > 0 ? in->table_dev : nullptr;
    a.buckets = in->buckets_dev;
    a.reach = in->reach;
    return PB_OK;
}

// What comes before anything that reads the handle or asks for a number of buckets.
int check_scores(const char* who, const pb_sets* s, const pb_choice_scores* in) {
    if (!s || !in) return pb::api_fail(PB_ERR_INVALID, (std::string(who) + ": null argument").c_str());
    if (in->num_buckets < 0 || in->num_buckets > pb::kMaxBuckets)
        return pb::api_fail(PB_ERR_UNSUPPORTED, (std::string(who) + ": at most 256 position buckets").c_str());
    return PB_OK;
}

int choice_args(const char* who, int32_t op, const pb_sets* s, const pb_choice_scores* in, void* work,
                int64_t work_bytes, pb::ChoiceArgs& a) {
    int rc = check_scores(who, s, in);
    if (rc == PB_OK) rc = scores_args(who, s, in, work, work_bytes, work_need(s, op, in->num_buckets), a);
    if (rc != PB_OK) return rc;
    a.sums = static_cast<double*>(work);
    a.parts = reinterpret_cast<float2*>(a.sums + sum_cols(s, op, in->num_buckets) * pb::choice_grid(s->s));
    return PB_OK;
}

// The temperature's part of a report's arguments, and the length of the lists.
int report_args(const char* who, float temperature, int32_t top, pb::ReportArgs& a) {
    const auto bad = [&](int code, const char* what) {
        return pb::api_fail(code, (std::string(who) + ": " + what).c_str());
    };
    if (!(temperature >= 0x1p-20f && temperature <= 0x1p20f)) return bad(PB_ERR_INVALID, "the temperature must lie in [2^-20, 2^20]");
    if (top > pb::kMaxTop) return bad(PB_ERR_UNSUPPORTED, "at most 64 entries to a list");
    a.temp = temperature;
    a.inv_temp = 1.0 / (double)temperature;
    const double heat = 1.4426950408889634 * a.inv_temp;
    a.heat_hi = (float)heat;
    a.heat_lo = (float)(heat - (double)a.heat_hi);
    a.heat_low = (float)(-200.0 / heat);  // 2^-200 is 0
    a.top = top;
    return PB_OK;
}

int launch(const char* who, int mode, const pb_sets* s, const pb::ChoiceArgs& a, int32_t type, void* stream) {
    const hipError_t e = pb::launch_choice(mode, s->s, a, type, (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, who);
}

// A table of sets without any set has no work to launch: its sums are zeros.
int clear(const char* who, float* out, int64_t n, void* stream) {
    const hipError_t e = pb::launch_zero(out, n, (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, who);
}

}  // namespace

extern "C" {

int pb_sets_create(const int64_t* offsets_host, int64_t num_sets, pb_sets** out) {
    if (!out) return pb::api_fail(PB_ERR_INVALID, "pb_sets_create: null output");
    *out = nullptr;
    if (!offsets_host) return pb::api_fail(PB_ERR_INVALID, "pb_sets_create: null offsets");
    try {
        return sets_create(offsets_host, num_sets, true, out);
    } catch (const std::exception&) {
        return pb::api_fail(PB_ERR_NOMEM, "pb_sets_create: out of host memory");
    }
}

int pb_sets_destroy(pb_sets* sets) {
    free_sets(sets);
    return PB_OK;
}

int64_t pb_choice_work_bytes(const pb_sets* s, int32_t op, int32_t num_buckets) {
    if (!s || op < PB_LOG_PROBS || op > PB_DISTILL || num_buckets < 0 || num_buckets > pb::kMaxBuckets) return -1;
    if (op >= PB_REPORT_BACKWARD) return pb::soft_grads_work_bytes(s->s, op == PB_DISTILL, num_buckets);
    return work_need(s, op, num_buckets);
}

int64_t pb_choice_report_work_bytes(const pb_sets* s, int32_t top, int32_t num_buckets) {
    if (!s || top < 0 || top > pb::kMaxTop || num_buckets < 0 || num_buckets > pb::kMaxBuckets) return -1;
    return pb::report_work_bytes(s->s, top, num_buckets > 0);
}

int pb_choice_log_probs(const pb_sets* s, const pb_choice_scores* in, const int32_t* chosen_dev, float* log_probs_dev,
                        float* lse_dev, void* work_dev, int64_t work_bytes, void* stream) {
    pb::ChoiceArgs a{};
    const int rc = choice_args("pb_choice_log_probs", PB_LOG_PROBS, s, in, work_dev, work_bytes, a);
    if (rc != PB_OK) return rc;
    if (s->s.num_sets == 0) return PB_OK;
    if (!lse_dev || ((chosen_dev || s->s.rows > 0) && !log_probs_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_choice_log_probs: null output");
    a.chosen = chosen_dev;
    a.log_probs = log_probs_dev;
    a.lse_out = lse_dev;
    return launch("pb_choice_log_probs", chosen_dev ? pb::kSteps : pb::kRows, s, a, in->score_type, stream);
}

int pb_choice_log_probs_backward(const pb_sets* s, const pb_choice_scores* in, const int32_t* chosen_dev,
                                 const float* grad_dev, const float* lse_dev, void* grad_scores_dev,
                                 float* grad_table_dev, void* work_dev, int64_t work_bytes, void* stream) {
    pb::ChoiceArgs a{};
    const int rc = choice_args("pb_choice_log_probs_backward", PB_BACKWARD, s, in, work_dev, work_bytes, a);
    if (rc != PB_OK) return rc;
    if (in->num_buckets > 0 && !grad_table_dev)
        return pb::api_fail(PB_ERR_INVALID, "pb_choice_log_probs_backward: null table gradient");
    if (s->s.num_sets == 0) return clear("pb_choice_log_probs_backward", grad_table_dev, in->num_buckets, stream);
    if (!lse_dev || ((chosen_dev || s->s.rows > 0) && !grad_dev) || (s->s.rows > 0 && !grad_scores_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_choice_log_probs_backward: null argument");
    a.chosen = chosen_dev;
    a.grad = grad_dev;
    a.lse = lse_dev;
    a.grad_scores = grad_scores_dev;
    a.grad_table = grad_table_dev;
    return launch("pb_choice_log_probs_backward", chosen_dev ? pb::kStepsBack : pb::kRowsBack, s, a, in->score_type, stream);
}

int pb_policy_loss(const pb_sets* s, const pb_choice_scores* in, const pb_policy_terms* t, const int32_t* chosen_dev,
                   float* stats_dev, float* log_probs_dev, void* grad_scores_dev, float* grad_table_dev, void* work_dev,
                   int64_t work_bytes, void* stream) {
    pb::ChoiceArgs a{};
    const int rc = choice_args("pb_policy_loss", PB_POLICY, s, in, work_dev, work_bytes, a);
    if (rc != PB_OK) return rc;
    if (!t || !stats_dev || (in->num_buckets > 0 && !grad_table_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_policy_loss: null argument");
    if (s->s.num_sets == 0) {
        const int rz = clear("pb_policy_loss", stats_dev, 3, stream);
        return rz != PB_OK ? rz : clear("pb_policy_loss", grad_table_dev, in->num_buckets, stream);
    }
    if (!chosen_dev || !log_probs_dev || !t->advantages_dev || !t->old_log_probs_dev || (s->s.rows > 0 && !grad_scores_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_policy_loss: null argument");
    a.chosen = chosen_dev;
    a.advantages = t->advantages_dev;
    a.old = t->old_log_probs_dev;
    a.ref = t->ref_log_probs_dev;
    a.weights = t->weights_dev;
    a.ratio_min = t->ratio_min;
    a.ratio_max = t->ratio_max;
    a.kl_weight = t->kl_weight;
    a.scale = t->scale;
    a.stats = stats_dev;
    a.log_probs = log_probs_dev;
    a.grad_scores = grad_scores_dev;
    a.grad_table = grad_table_dev;
    return launch("pb_policy_loss", pb::kPolicy, s, a, in->score_type, stream);
}

int pb_choice_report(const pb_sets* s, const pb_choice_scores* in, const int32_t* chosen_dev, float temperature, int32_t top,
                     float* log_probs_dev, float* entropy_dev, float* lse_dev, int32_t* top_index_dev,
                     float* top_log_probs_dev, void* work_dev, int64_t work_bytes, void* stream) {
    const char* who = "pb_choice_report";
    pb::ReportArgs a{};
    int rc = check_scores(who, s, in);
    if (rc == PB_OK && top < 0) rc = pb::api_fail(PB_ERR_INVALID, "pb_choice_report: a list has at least 0 entries");
    if (rc == PB_OK) rc = report_args(who, temperature, top, a);
    if (rc == PB_OK && top > 0 && s->largest > INT32_MAX)
        rc = pb::api_fail(PB_ERR_UNSUPPORTED, "pb_choice_report: lists name rows of sets of at most 2^31 - 1 rows");
    if (rc == PB_OK) rc = scores_args(who, s, in, work_dev, work_bytes, pb::report_work_bytes(s->s, top, in->num_buckets > 0), a);
    if (rc != PB_OK || s->s.num_sets == 0) return rc;
    if (!entropy_dev || !lse_dev || (chosen_dev && !log_probs_dev) || (top > 0 && (!top_index_dev || !top_log_probs_dev)))
        return pb::api_fail(PB_ERR_INVALID, "pb_choice_report: null output");
    a.chosen = chosen_dev;
    a.log_probs = log_probs_dev;
    a.entropy = entropy_dev;
    a.lse_out = lse_dev;
    a.top_index = top_index_dev;
    a.top_log_probs = top_log_probs_dev;
    const hipError_t e = pb::launch_report(s->s, a, in->score_type, static_cast<char*>(work_dev), (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, who);
}

int pb_choice_report_backward(const pb_sets* s, const pb_choice_scores* in, const int32_t* chosen_dev, float temperature,
                              const float* grad_log_probs_dev, const float* grad_entropy_dev, void* grad_scores_dev,
                              float* grad_table_dev, void* work_dev, int64_t work_bytes, void* stream) {
    const char* who = "pb_choice_report_backward";
    pb::ReportArgs a{};
    int rc = check_scores(who, s, in);
    if (rc == PB_OK) rc = report_args(who, temperature, 0, a);
    if (rc == PB_OK)
        rc = scores_args(who, s, in, work_dev, work_bytes, pb::soft_grads_work_bytes(s->s, false, in->num_buckets), a);
    if (rc != PB_OK) return rc;
    if (in->num_buckets > 0 && !grad_table_dev) return pb::api_fail(PB_ERR_INVALID, "pb_choice_report_backward: null table gradient");
    if (s->s.num_sets == 0) return clear(who, grad_table_dev, in->num_buckets, stream);
    if ((grad_log_probs_dev && !chosen_dev) || (s->s.rows > 0 && !grad_scores_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_choice_report_backward: null argument");
    a.chosen = chosen_dev;
    a.grad = grad_log_probs_dev;
    a.grad_entropy = grad_entropy_dev;
    a.grad_scores = grad_scores_dev;
    a.grad_table = grad_table_dev;
    const hipError_t e = pb::launch_soft_grads(false, s->s, a, in->score_type, static_cast<char*>(work_dev), (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, who);
}

int pb_distillation_loss(const pb_sets* s, const pb_choice_scores* in, const pb_teacher* t, float* loss_dev, float* kl_dev,
                         void* grad_scores_dev, float* grad_table_dev, void* work_dev, int64_t work_bytes, void* stream) {
    const char* who = "pb_distillation_loss";
    pb::ReportArgs a{};
    int rc = check_scores(who, s, in);
    if (rc == PB_OK && !t) rc = pb::api_fail(PB_ERR_INVALID, "pb_distillation_loss: null argument");
    if (rc == PB_OK && t->entries < 1) rc = pb::api_fail(PB_ERR_INVALID, "pb_distillation_loss: a list has at least 1 entry");
    if (rc == PB_OK) rc = report_args(who, t->temperature, t->entries, a);
    if (rc == PB_OK && t->logit_type != PB_F32 && t->logit_type != PB_BF16 && t->logit_type != PB_F16)
        rc = pb::api_fail(PB_ERR_UNSUPPORTED, "pb_distillation_loss: the teacher's logits must be float32, bfloat16 or float16");
    if (rc == PB_OK)
        rc = scores_args(who, s, in, work_dev, work_bytes, pb::soft_grads_work_bytes(s->s, true, in->num_buckets), a);
    if (rc != PB_OK) return rc;
    if (!loss_dev || (in->num_buckets > 0 && !grad_table_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_distillation_loss: null argument");
    if (s->s.num_sets == 0) {
        rc = clear(who, loss_dev, 1, stream);
        return rc != PB_OK ? rc : clear(who, grad_table_dev, in->num_buckets, stream);
    }
    if (!t->index_dev || !t->logits_dev || !kl_dev || (s->s.rows > 0 && !grad_scores_dev))
        return pb::api_fail(PB_ERR_INVALID, "pb_distillation_loss: null argument");
    a.entry_index = t->index_dev;
    a.entry_logits = t->logits_dev;
    a.entry_type = t->logit_type;
    a.tail = t->tail != 0;
    a.weights = t->weights_dev;
    a.scale = t->scale;
    a.stats = loss_dev;
    a.kl = kl_dev;
    a.grad_scores = grad_scores_dev;
    a.grad_table = grad_table_dev;
    const hipError_t e = pb::launch_soft_grads(true, s->s, a, in->score_type, static_cast<char*>(work_dev), (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, who);
}

int pb_pairs_create(const int64_t* winners_host, const int64_t* losers_host, int64_t num_pairs, int64_t num_values,
                    const int64_t* seq_offsets_host, pb_pairs** out) {
    return pairs_entry("pb_pairs_create", winners_host, losers_host, num_pairs, num_values, seq_offsets_host, false,
                       nullptr, out);
}

int pb_pairs_create_from_device(const int64_t* winners_dev, const int64_t* losers_dev, int64_t num_pairs,
                                int64_t num_values, const int64_t* seq_offsets_host, void* stream, pb_pairs** out) {
    return pairs_entry("pb_pairs_create_from_device", winners_dev, losers_dev, num_pairs, num_values, seq_offsets_host,
                       true, (hipStream_t)stream, out);
}

int pb_pairs_destroy(pb_pairs* pairs) {
    free_pairs(pairs);
    return PB_OK;
}

int64_t pb_preference_work_bytes(const pb_pairs* p) { return p ? pb::preference_work_bytes(p->p) : -1; }

int pb_preference_loss(const pb_pairs* p, const float* values_dev, const float* ref_dev, const float* weights_dev,
                       float beta, float label_smoothing, float scale, float* loss_dev, float* grad_dev,
                       float* margins_dev, void* work_dev, int64_t work_bytes, void* stream) {
    if (!p || !loss_dev) return pb::api_fail(PB_ERR_INVALID, "pb_preference_loss: null argument");
    const int64_t n = p->p.has_seqs ? p->p.seqs.rows : p->p.lists.num_sets;
    if (n > 0 && (!values_dev || !grad_dev)) return pb::api_fail(PB_ERR_INVALID, "pb_preference_loss: null argument");
    if (p->p.num_pairs > 0 && !margins_dev) return pb::api_fail(PB_ERR_INVALID, "pb_preference_loss: null margins");
    if (!work_dev || work_bytes < pb::preference_work_bytes(p->p))
        return pb::api_fail(PB_ERR_INVALID, "pb_preference_loss: workspace too small");
    if (reinterpret_cast<uintptr_t>(work_dev) & 15)
        return pb::api_fail(PB_ERR_INVALID, "pb_preference_loss: workspace must be 16-byte aligned");
    pb::PairArgs a{};
    a.weights = weights_dev;
    a.beta = beta;
    a.smoothing = label_smoothing;
    a.scale = scale;
    a.margins = margins_dev;
    a.loss = loss_dev;
    const hipError_t e = pb::launch_preference(p->p, a, values_dev, ref_dev, grad_dev, static_cast<char*>(work_dev),
                                               (hipStream_t)stream);
    return e == hipSuccess ? PB_OK : pb::api_hip_fail(e, "pb_preference_loss");
}

}  // extern "C"
