// Decoding steps over a paged key/value cache: the C entry points, the checks of their arguments and
// the host plan (which pages a step's tokens write and read) that one upload hands to the kernels of
// every layer.
#include "decode.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstring>
#include <exception>
#include <mutex>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../include/ripvec_b200.h"
#include "tmap.h"

namespace {

struct DeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(int d) {
    cudaGetDevice(&prev);
    if (prev != d) ok = cudaSetDevice(d) == cudaSuccess;
    else prev = -1;
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Pinned staging of a small plan's upload; reused once its copy has left it.
struct Staging {
  char* p = nullptr;
  cudaEvent_t done = nullptr;
};

constexpr size_t kSmallPlan = 64 * 1024;          // bytes of records that go through pinned memory
constexpr size_t kFirstRecords = 1024 * 1024;     // bytes of records that a new step has room for
constexpr size_t kCounterBytes = 128;             // the two counters, at the head of a plan's records
constexpr int64_t kMaxTokens = int64_t(1) << 24;  // of one step
constexpr int64_t kMaxKeys = int64_t(1) << 30;    // of one sequence or prefix

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What one sequence's queries see: its tokens tok0 .. tok0 + n - 1, prefix keys [0, len_a) in the pages from
// pg[pg_a] and own keys [0, len_b) in those from pg[pg_b], of which token i sees those below diag + i + 1.
struct StepSeq {
  int tok0, n, pg_a, len_a, pg_b, len_b, diag;
};
// diag of a sequence that is not causal.  A causal one's is its keys less its tokens: smaller where there are two
// tokens and more.
constexpr int kSeesAll = kMaxKeys - 1;

// The attention work of a plan.
struct Schedule {
  std::vector<rv::StepItem> row_items, tile_items;
  std::vector<rv::StepParts> parts;  // by token
  std::vector<int> joined;
  int64_t n_parts = 0;
  int tile_sms = 0;  // CTAs of the tensor-core kernel
};

}  // namespace

struct rv_step {
  int device = 0;
  int q_heads = 0, kv_heads = 0, head_dim = 0, page_size = 0;
  std::mutex mu;
  std::string err;
  // the plan
  bool planned = false, can_append = false;
  int n_tokens = 0;
  int64_t num_pages = 0;
  int last_pos = -1;  // largest position of a new token
  char* meta = nullptr;
  size_t meta_cap = 0;
  bool own_meta = false;
  int fold = 1;  // query heads of a key/value head that share a row tile: the largest divisor up to kRowTile
  const rv::StepToken* tokens = nullptr;
  const rv::StepParts* parts = nullptr;
  const rv::StepItem *row_items = nullptr, *tile_items = nullptr;
  const int *joined = nullptr, *pages = nullptr;
  int n_row_items = 0, n_tile_items = 0, n_joined = 0;
  float* work = nullptr;  // partial results
  size_t work_cap = 0;    // floats
  int64_t n_parts = 0;
  char* base_host = nullptr;         // pinned: the error word and the staging
  char* base_dev = nullptr;          // records until a plan needs more
  unsigned int* err_host = nullptr;  // error word in mapped host memory: kernels write it, calls look at it
  unsigned int* err_dev = nullptr;
  int* counter = nullptr;
  Staging staging[2];
  int turn = 0;
  // host side of the plan, kept for its memory
  std::vector<char> host;
  std::vector<rv::StepToken> tok;
  std::vector<StepSeq> seq;
  std::vector<int> group_first, pg;
  std::vector<int> written;  // pages that new tokens go to
  std::vector<uint64_t> written_bits;
  Schedule sched;
  // Calls on different streams wait for one another: plan, append and attend share the plan's device
  // records and the workspace.
  cudaEvent_t last = nullptr;
  unsigned long long last_stream = 0;  // its id: a handle may stand for one stream a thread, or for a later stream
  bool used = false;
};

namespace {

int fail(rv_step* s, int code, const std::string& why) {
  s->err = why;
  return code;
}

int cuda_fail(rv_step* s, const char* what, cudaError_t e) {
  return fail(s, e == cudaErrorMemoryAllocation ? RV_E_NOMEM : RV_E_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// A record's double as f32; what is beyond its range becomes an infinity.
float to_float(double v) {
  return std::fabs(v) > double(FLT_MAX) ? float(std::copysign(HUGE_VAL, v)) : float(v);
}

// An error that an earlier call's kernels reported (without waiting for those still queued).
bool device_error(rv_step* s) {
  volatile unsigned int* w = s->err_host;
  if (!*w) return false;
  *w = 0;
  s->err = "a kernel of an earlier call gave up waiting: its outputs are not valid";
  return true;
}

bool capturing(cudaStream_t st) {
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  return cudaStreamIsCapturing(st, &cs) == cudaSuccess && cs != cudaStreamCaptureStatusNone;
}

// Makes st wait for this step's earlier work on another stream.  Under stream capture the order is the
// caller's: an event of uncaptured work cannot be waited for there.
cudaError_t enter(rv_step* s, cudaStream_t st) {
  if (!s->used || capturing(st)) return cudaSuccess;
  unsigned long long id = 0;
  const cudaError_t e = cudaStreamGetId(st, &id);
  if (e != cudaSuccess) return e;
  return id == s->last_stream ? cudaSuccess : cudaStreamWaitEvent(st, s->last, 0);
}
cudaError_t leave(rv_step* s, cudaStream_t st) {
  if (capturing(st)) return cudaSuccess;
  const cudaError_t e = cudaStreamGetId(st, &s->last_stream);
  if (e != cudaSuccess) return e;
  s->used = true;
  return cudaEventRecord(s->last, st);
}

// The pools as the kernels take them, checked against the step; an empty string, or what is wrong.
std::string take_pool(const rv_step* s, const rv_kv_cache* c, rv::KvPool* out, rv::Act* act) {
  if (!c || !c->k || !c->v) return "null cache";
  if (c->dtype != RV_DTYPE_BF16 && c->dtype != RV_DTYPE_F16) return "the cache's dtype is neither bf16 nor f16";
  if (c->kv_heads != s->kv_heads || c->head_dim != s->head_dim || c->page_size != s->page_size)
    return "the cache's kv_heads, head_dim or page_size are not the step's";
  if (c->num_pages < s->num_pages) return "the cache has fewer pages than the plan was made for";
  if (!aligned16(c->k) || !aligned16(c->v) || (c->num_pages > 1 && c->page_stride % 8) || (s->kv_heads > 1 && c->head_stride % 8) ||
      c->slot_stride % 8)
    return "the cache's pools and strides must be multiples of 16 bytes";
  // The stride of an axis of one entry has no meaning (and may be anything).
  const int64_t page_stride = c->num_pages > 1 ? c->page_stride : s->head_dim;
  const int64_t head_stride = s->kv_heads > 1 ? c->head_stride : s->head_dim;
  if (page_stride <= 0 || head_stride <= 0 || c->slot_stride < s->head_dim)
    return "the cache's strides must be positive, the slot stride at least head_dim";
  out->k = c->k;
  out->v = c->v;
  out->page_stride = page_stride;
  out->head_stride = head_stride;
  out->slot_stride = c->slot_stride;
  out->page_size = c->page_size;
  *act = c->dtype == RV_DTYPE_BF16 ? rv::Act::kBf16 : rv::Act::kF16;
  return "";
}

bool rows_aligned(const void* p, int64_t ts, int64_t hs) { return aligned16(p) && ts % 8 == 0 && hs % 8 == 0; }

// ---------------------------------------------------------------- attention schedule
// Attention work before its keys are split.
struct Job {
  rv::StepItem it;
  bool packed;  // rows of several sequences against their prefix
};

int tiles_of(const rv::StepItem& it, int keys) {
  return (it.a1 - it.a0 + keys - 1) / keys + (it.b1 - it.b0 + keys - 1) / keys;
}

// So many tiles of 64 keys are one part of the few-row kernel whatever there is to do: with 8 rows of 128 values,
// 4 tiles whole take 8.3 us and 8 take 11.3, in parts with their join 8.4.
constexpr int kWhole = 4;

// Cuts an item's key tiles into parts of at most `most` tiles of about equal length.
template <class F>
void cut(const rv::StepItem& it, int keys, int most, F&& emit) {
  const int na = (it.a1 - it.a0 + keys - 1) / keys, n = tiles_of(it, keys);
  const int parts = keys == rv::kRowKeys && n <= kWhole ? 1 : std::max(1, (n + most - 1) / most);
  for (int k = 0; k < parts; ++k) {
    const int lo = int(int64_t(n) * k / parts), hi = int(int64_t(n) * (k + 1) / parts);
    rv::StepItem x = it;
    x.a0 = std::min(it.a1, it.a0 + std::min(lo, na) * keys);
    x.a1 = std::min(it.a1, it.a0 + std::min(hi, na) * keys);
    x.b0 = std::min(it.b1, it.b0 + std::max(0, lo - na) * keys);
    x.b1 = std::min(it.b1, it.b0 + std::max(0, hi - na) * keys);
    x.part = k;
    emit(x, parts);
  }
}

// Time of a part of `tiles` key tiles in the tensor-core kernel, in key tiles of two row tiles: a lone row
// tile leaves the tensor cores waiting for its softmax; starting and writing a part takes about two tiles.
double tile_cost(const rv::StepItem& it, int tiles, int per) { return (it.n > per ? 1.0 : 0.7) * tiles + 2.0; }

// The longest time of any CTA, and all CTAs' together, when parts of at most `most` tiles are dealt out to `ctas`,
// longest first, forwards and backwards in turn, as the kernel walks them.
struct Span {
  double longest, all;
};
Span makespan(const std::vector<Job>& jobs, int most, int per, int groups, int ctas) {
  std::vector<double> cost;  // by part, for one of `groups`
  for (const Job& j : jobs)
    cut(j.it, rv::kTileKeys, most, [&](const rv::StepItem& x, int parts) {
      cost.push_back(tile_cost(x, tiles_of(x, rv::kTileKeys), per) + (parts > 1 ? 1.0 : 0.0));
    });
  std::sort(cost.begin(), cost.end(), [](double a, double b) { return a > b; });
  std::vector<double> load(size_t(ctas), 0.0);
  int64_t w = 0;
  double all = 0;
  for (const double c : cost)
    for (int k = 0; k < groups; ++k, ++w) {
      const int64_t round = w / ctas, at = w % ctas;
      load[size_t(round & 1 ? ctas - 1 - at : at)] += c;
      all += c;
    }
  return {*std::max_element(load.begin(), load.end()), all};
}

// How the tensor-core kernel's jobs are cut (longest part, in key tiles) and how many CTAs it gets.  Cutting keys
// costs a partial result and its join, so it is done only where it shortens the step: with few jobs that each walk
// many keys.  `rows` is the few-row kernel's time, summed over SMs, in the same unit; it runs on the SMs that are
// left, so the step takes as long as the longest CTA here, or as all the work spread over all SMs.
struct TileCut {
  int most, ctas;
};
TileCut choose_tile_cut(const std::vector<Job>& jobs, int per, int groups, double rows, int sms) {
  int64_t total = 0;
  int longest = 1;
  for (const Job& j : jobs) {
    const int n = tiles_of(j.it, rv::kTileKeys);
    total += n;
    longest = std::max(longest, n);
  }
  total *= groups;
  // Enough work for every SM many times over, none of it long against an SM's share: leave it whole.
  if (int64_t(longest) * sms * 4 <= total) return {longest, sms};
  TileCut best{longest, sms};
  double best_time = 1e300;
  for (int k = 1; k <= 64; k += k < 12 ? 1 : k / 4) {
    const int u = (longest + k - 1) / k;
    int64_t parts = 0;
    for (const Job& j : jobs) parts += (tiles_of(j.it, rv::kTileKeys) + u - 1) / u;
    parts *= groups;
    if (k > 1 && parts > int64_t(sms) * 16) break;
    // As many CTAs as parts, or as a half or a third of them, which leave SMs for the other kernel.
    for (int d = 1; d <= (rows > 0 ? 3 : 1); ++d) {
      const int ctas = int(std::min<int64_t>(sms, (parts + d - 1) / d));
      const Span m = makespan(jobs, u, per, groups, ctas);
      const double t = std::max(m.longest, (m.all + rows) / sms);
      if (t < 0.97 * best_time) {
        best_time = t;
        best = {u, ctas};
      }
    }
    if (u == 1) break;
  }
  return best;
}

// Longest part, in 64-key tiles, for the few-row kernel's jobs: where there is much work, about three parts for each
// of two CTAs an SM, which take them as they come; where there is little, short parts, so that all SMs have one.
int choose_row_cut(const std::vector<Job>& jobs, int groups, int sms) {
  int64_t total = 0;
  for (const Job& j : jobs) total += tiles_of(j.it, rv::kRowKeys);
  total *= groups;
  return int(std::max<int64_t>(2, (total + 6 * sms - 1) / (6 * sms)));
}

// Sequences of half a row tile and more pack up to so many rows, and while two partial results of all their rows take no
// more than so many bytes of workspace.
constexpr int kPackRows = 4 * rv::kTileRows;
constexpr int64_t kPackBytes = int64_t(1) << 30;

// What is saved, in key tiles of two row tiles, where a sequence of `rows` rows shares the walk of its prefix of `keys`
// keys with its neighbours.  By itself it walks the prefix once for every two row tiles, 0.7 as long for a last one
// alone, however few rows that holds; packed with others for its share of them, at the cost of partial results: three
// tiles of time for every two row tiles, one for its own keys, and 0.022 a row to write and join them.
double packing_saves(int64_t rows, int keys) {
  constexpr int kPair = 2 * rv::kTileRows;
  const int rest = int(rows % kPair);
  const double alone = double(rows / kPair) + (rest == 0 ? 0.0 : rest <= rv::kTileRows ? 0.7 : 1.0);
  const double share = double(rows) / kPair;
  return double(keys) / rv::kTileKeys * (alone - share) - 1.0 - 3.0 * share - 0.022 * double(rows);
}

// Divides a step's attention into items.  Sequences that pack share the prefix: the rows of all of them are packed
// into row tiles that read each prefix key once, and their own keys are separate items.  The others walk the prefix
// and their own keys in one item, without partial results.  Sequences of less than half a row tile pack; those of
// more, up to kPackRows, do where it saves time, all of a group's or none, so that runs stay whole.  32 query and
// 8 key/value heads of 128, packed against not: 64 sequences of 20 tokens over 32768 keys 714 and 1333 us, 16 of 30 to
// 60 over 8000 121 and 135, 32 of 20 to 120 over 8000 334 and 368, 32 of 16 to 24 over 2000 57 and 63; over 1000 45 and
// 42, where they walk alone.  (Those constants are this one layout's.  Below half a row tile nothing is weighed: for 17
// to 63 rows behind some hundred prefix keys the same formula would have each walk alone.)
void schedule(const std::vector<StepSeq>& seqs, const std::vector<int>& group_first, int n_tokens, int fold,
              int groups, int head_dim,
              int sms, Schedule* out) {
  const int per = rv::kTileRows / fold;
  std::vector<Job> rows, tiles;
  auto add = [&](bool to_rows, int tok0, int n, const StepSeq& s, bool prefix, bool own, int diag, bool packed) {
    rv::StepItem it{};
    it.tok0 = tok0;
    it.n = n;
    it.pg_a = s.pg_a;
    it.a1 = prefix ? s.len_a : 0;
    it.pg_b = s.pg_b;
    it.b1 = own ? int(std::max<int64_t>(0, std::min<int64_t>(s.len_b, int64_t(diag) + n))) : 0;
    it.diag = diag;
    if (it.a1 == 0 && it.b1 == 0) return;
    (to_rows ? rows : tiles).push_back({it, packed});
  };
  // A sequence's keys, or its own ones only.
  auto whole = [&](const StepSeq& s, bool prefix) {
    if (s.n * fold <= rv::kRowTile) return add(true, s.tok0, s.n, s, prefix, true, s.diag, false);
    for (int t = 0; t < s.n; t += 2 * per)
      add(false, s.tok0 + t, std::min(2 * per, s.n - t), s, prefix, true, s.diag == kSeesAll ? kSeesAll : s.diag + t,
          false);
  };
  for (size_t g = 0; g + 1 < group_first.size(); ++g) {
    int b = group_first[g];
    const int end = group_first[g + 1];
    double vote = 0;
    int64_t middle = 0;  // rows of a key/value head that it is about
    for (int k = b; k < end; ++k) {
      const int64_t r = int64_t(seqs[k].n) * fold;
      if (r < rv::kTileRows / 2 || r >= kPackRows) continue;
      vote += packing_saves(r, seqs[k].len_a);
      middle += r;
    }
    if (middle * groups * head_dim * 8 > kPackBytes) vote = 0;
    auto packs = [&](const StepSeq& q) {
      const int64_t r = int64_t(q.n) * fold;
      return r < rv::kTileRows / 2 || (r < kPackRows && vote > 0);
    };
    while (b < end) {
      // A run of sequences that pack.
      int e = b, live = 0, n = 0, longest = 0;
      while (e < end && packs(seqs[e])) {
        live += seqs[e].n > 0;
        n += seqs[e].n;
        if (seqs[e].n > 0) longest = std::max(longest, (seqs[e].len_b + rv::kRowKeys - 1) / rv::kRowKeys);
        ++e;
      }
      // Each by itself where there is nothing to share, and where prefix and own keys together are so few that an
      // item takes them in one part: no join then (prefix 128, 40 own keys: 7.3 us against 8 to 11 for 2 to 64
      // sequences).
      const int shared = (seqs[b].len_a + rv::kRowKeys - 1) / rv::kRowKeys;
      if (live == 1 || (live > 1 && (shared == 0 || shared + longest <= kWhole))) {
        for (; b < e; ++b)
          if (seqs[b].n > 0) whole(seqs[b], true);
        continue;
      }
      if (live > 1) {
        const int t0 = seqs[b].tok0;
        // One kernel for all of a run, so that all its tokens get as many partials of the prefix.
        if (n * fold <= rv::kRowTile) add(true, t0, n, seqs[b], true, false, 0, true);
        else
          for (int t = 0; t < n; t += 2 * per) add(false, t0 + t, std::min(2 * per, n - t), seqs[b], true, false, 0, true);
        for (; b < e; ++b)
          if (seqs[b].n > 0) whole(seqs[b], false);
        continue;
      }
      // A sequence that does not (or a run without any rows).
      if (seqs[b].n > 0) whole(seqs[b], true);
      b = std::max(e, b + 1);
    }
  }
  // Parts: a token's partials are numbered through its items in order.
  out->parts.assign(size_t(n_tokens), {0, 0});
  const int row_cut = rows.empty() ? 1 : choose_row_cut(rows, groups, sms);
  TileCut tile_cut{1, 0};
  if (!tiles.empty()) {
    // The few-row kernel's time: its bytes at an SM's share of the memory bandwidth, 43 GB/s, against the 2.2 us (1.6
    // at head dim 64) that 128 keys of two row tiles take.
    double row_time = 0;
    for (const Job& j : rows) row_time += tiles_of(j.it, rv::kRowKeys) * double(rv::kRowKeys * head_dim * 4) / 43e3;
    tile_cut = choose_tile_cut(tiles, per, groups, row_time * groups / (head_dim == 64 ? 1.6 : 2.2), sms);
  }
  out->tile_sms = tile_cut.ctas;
  auto emit = [&](const std::vector<Job>& jobs, bool packed, int keys, int most, std::vector<rv::StepItem>* items) {
    for (const Job& j : jobs) {
      if (j.packed != packed) continue;
      const int base = out->parts[size_t(j.it.tok0)].count;
      int count = 0;
      cut(j.it, keys, most, [&](rv::StepItem x, int parts) {
        count = parts;
        x.part += base;
        items->push_back(x);
      });
      for (int t = j.it.tok0; t < j.it.tok0 + j.it.n; ++t) out->parts[size_t(t)].count += count;
    }
  };
  // Prefixes first: their items cut through sequences, and a sequence's tokens must agree in what came before
  // the item of its own keys.
  for (const bool packed : {true, false}) {
    emit(tiles, packed, rv::kTileKeys, tile_cut.most, &out->tile_items);
    emit(rows, packed, rv::kRowKeys, row_cut, &out->row_items);
  }
  std::stable_sort(out->tile_items.begin(), out->tile_items.end(), [&](const rv::StepItem& a, const rv::StepItem& b) {
    return tile_cost(a, tiles_of(a, rv::kTileKeys), per) > tile_cost(b, tiles_of(b, rv::kTileKeys), per);
  });
  std::stable_sort(out->row_items.begin(), out->row_items.end(), [](const rv::StepItem& a, const rv::StepItem& b) {
    return tiles_of(a, rv::kRowKeys) > tiles_of(b, rv::kRowKeys);
  });
  for (int t = 0; t < n_tokens; ++t) {
    rv::StepParts& pt = out->parts[size_t(t)];
    pt.first = int(out->n_parts);
    if (pt.count == 1) continue;
    out->joined.push_back(t);
    out->n_parts += pt.count;
  }
}

int plan(rv_step* s, int32_t n_seqs, const int32_t* q_lens, const int32_t* own_lens, const int32_t* own_pages,
         int32_t n_groups, const int32_t* group_sizes, const int32_t* prefix_lens, const int32_t* prefix_pages,
         int64_t num_pages, int32_t causal, cudaStream_t st) {
  s->planned = false;
  if (device_error(s)) return RV_E_DEVICE;
  if (n_seqs < 0 || n_groups < 0 || num_pages < 0 || num_pages > INT_MAX || (n_seqs > 0 && (!q_lens || !own_lens)) ||
      (n_groups > 0 && (!group_sizes || !prefix_lens)))
    return fail(s, RV_E_INVALID, "null or negative argument");
  if (capturing(st)) return fail(s, RV_E_INVALID, "a plan cannot be made on a capturing stream");
  const int ps = s->page_size;
  auto count = [ps](int64_t keys) { return (keys + ps - 1) / ps; };
  int64_t in_groups = 0, n_prefix_pages = 0, n_own_pages = 0, tokens = 0;
  for (int g = 0; g < n_groups; ++g) {
    if (group_sizes[g] < 0 || prefix_lens[g] < 0 || prefix_lens[g] > kMaxKeys)
      return fail(s, RV_E_INVALID, "group sizes and prefix lengths must be from 0 to 2^30");
    in_groups += group_sizes[g];
    n_prefix_pages += count(prefix_lens[g]);
  }
  if (in_groups != n_seqs) return fail(s, RV_E_INVALID, "the group sizes do not add up to the sequences");
  bool can_append = true;
  for (int b = 0; b < n_seqs; ++b) {
    if (q_lens[b] < 0 || own_lens[b] < 0 || own_lens[b] > kMaxKeys)
      return fail(s, RV_E_INVALID, "lengths must be from 0 to 2^30");
    tokens += q_lens[b];
    n_own_pages += count(own_lens[b]);
    can_append = can_append && own_lens[b] >= q_lens[b];
  }
  if (tokens > kMaxTokens) return fail(s, RV_E_INVALID, "more than 2^24 tokens in one step");
  if (n_prefix_pages + n_own_pages > INT_MAX / 8) return fail(s, RV_E_INVALID, "too many pages in one step");
  if ((n_prefix_pages > 0 && !prefix_pages) || (n_own_pages > 0 && !own_pages))
    return fail(s, RV_E_INVALID, "null page list");
  for (int64_t i = 0; i < n_prefix_pages; ++i)
    if (prefix_pages[i] < 0 || prefix_pages[i] >= num_pages) return fail(s, RV_E_INVALID, "prefix page out of range");
  for (int64_t i = 0; i < n_own_pages; ++i)
    if (own_pages[i] < 0 || own_pages[i] >= num_pages) return fail(s, RV_E_INVALID, "page out of range");

  s->tok.resize(size_t(tokens));
  s->seq.resize(size_t(n_seqs));
  s->group_first.assign(1, 0);
  auto* tk = s->tok.data();
  auto* sq = s->seq.data();
  std::vector<int>& pg = s->pg;
  pg.assign(prefix_pages, prefix_pages + n_prefix_pages);
  pg.insert(pg.end(), own_pages, own_pages + n_own_pages);
  std::vector<int>& written = s->written;
  written.clear();
  int t = 0, b = 0, last_pos = -1;
  int64_t pa = 0, pb = n_prefix_pages;
  for (int g = 0; g < n_groups; ++g) {
    for (int k = 0; k < group_sizes[g]; ++k, ++b) {
      const int n = q_lens[b], own = own_lens[b];
      sq[b] = {t, n, int(pa), prefix_lens[g], int(pb), own, causal ? own - n : kSeesAll};
      for (int i = 0; i < n; ++i) {
        const int place = own - n + i;  // negative only when nothing can be appended
        const int page = place >= 0 ? pg[size_t(pb + place / ps)] : 0;
        tk[t++] = {page, place >= 0 ? place % ps : 0, prefix_lens[g] + place, b};
        if (place < 0) continue;
        if (i == 0 || place % ps == 0) written.push_back(page);
        if (prefix_lens[g] + place > last_pos) last_pos = prefix_lens[g] + place;
      }
      pb += count(own);
    }
    pa += count(prefix_lens[g]);
    s->group_first.push_back(b);
  }
  // A page that new tokens go to is none that this step reads through another entry of its lists: another sequence's
  // new tokens', a prefix's, or an earlier page of any sequence with queries.  (A sequence's new tokens take consecutive
  // places, and all its entries before theirs are full of earlier keys.)  A table of 2^16 bits, by the low bits of the
  // page, spares most entries the search.
  std::sort(written.begin(), written.end());
  if (std::adjacent_find(written.begin(), written.end()) != written.end()) can_append = false;
  if (can_append && !written.empty()) {
    std::vector<uint64_t>& bits = s->written_bits;
    bits.assign(1024, 0);
    for (const int page : written) bits[page >> 6 & 1023] |= uint64_t(1) << (page & 63);
    auto is_written = [&](int page) {
      return (bits[page >> 6 & 1023] >> (page & 63) & 1) && std::binary_search(written.begin(), written.end(), page);
    };
    for (int64_t i = 0; i < n_prefix_pages && can_append; ++i) can_append = !is_written(prefix_pages[i]);
    const int* list = own_pages;
    for (b = 0; b < n_seqs && can_append; list += count(own_lens[b++]))
      for (int i = 0; q_lens[b] > 0 && i < (own_lens[b] - q_lens[b]) / ps && can_append; ++i) can_append = !is_written(list[i]);
  }

  Schedule& sc = s->sched;
  sc.row_items.clear();
  sc.tile_items.clear();
  sc.joined.clear();
  sc.n_parts = 0;
  schedule(s->seq, s->group_first, int(tokens), s->fold, s->q_heads / s->fold, s->head_dim, rv::device_sm_count(), &sc);
  if (sc.n_parts > INT_MAX || int64_t(sc.joined.size()) * s->q_heads > INT_MAX ||
      (int64_t(sc.row_items.size()) + int64_t(sc.tile_items.size())) * (s->q_heads / s->fold) > INT_MAX)
    return fail(s, RV_E_INVALID, "the step is too large");

  // The records, one after the other, each on 16 bytes.
  size_t bytes = 0;
  auto place_of = [&bytes](size_t n) {
    const size_t at = bytes;
    bytes += (n + 15) / 16 * 16;
    return at;
  };
  // The few-row kernel's counters come first, as zeros, on a cache line of their own: uploaded with the plan, they are
  // in the order of streams that every call on the plan is in.
  place_of(kCounterBytes);
  const size_t o_tokens = place_of(s->tok.size() * sizeof(rv::StepToken));
  // (Where every token is one item's, nothing is looked up by token.)
  const size_t n_parts = sc.joined.empty() ? 0 : sc.parts.size();
  const size_t o_parts = place_of(n_parts * sizeof(rv::StepParts));
  const size_t o_rows = place_of(sc.row_items.size() * sizeof(rv::StepItem));
  const size_t o_tiles = place_of(sc.tile_items.size() * sizeof(rv::StepItem));
  const size_t o_joined = place_of(sc.joined.size() * sizeof(int));
  const size_t o_pages = place_of(pg.size() * sizeof(int));
  const size_t floats = size_t(sc.n_parts) * size_t(s->q_heads) * size_t(s->head_dim + 2);

  // Small plans, those of decoding steps, are copied from pinned memory and leave the host at once.  The records of
  // long prompts come from pageable memory, which the copy takes over before it returns: pinned memory for them takes
  // milliseconds to get.
  Staging& sg = s->staging[s->turn];
  const bool small = bytes <= kSmallPlan;
  char* from = sg.p;
  cudaError_t e = cudaSuccess;
  if (small) {
    s->turn ^= 1;
    e = cudaEventSynchronize(sg.done);  // the copy before last has left this buffer
    if (e != cudaSuccess) return cuda_fail(s, "waiting for an earlier plan", e);
  } else {
    s->host.resize(bytes);
    from = s->host.data();
  }
  if (s->meta_cap < bytes) {
    if (s->own_meta) cudaFree(s->meta);  // waits for the kernels that still read it
    s->meta = nullptr;
    s->meta_cap = 0;
    s->own_meta = true;
    const size_t want = bytes + bytes / 2 + 4096;
    if ((e = cudaMalloc(reinterpret_cast<void**>(&s->meta), want)) != cudaSuccess)
      return cuda_fail(s, "plan records", e);
    s->meta_cap = want;
  }
  auto put = [from](size_t at, const void* p, size_t n) {
    if (n) std::memcpy(from + at, p, n);
  };
  std::memset(from, 0, kCounterBytes);
  put(o_tokens, s->tok.data(), s->tok.size() * sizeof(rv::StepToken));
  put(o_parts, sc.parts.data(), n_parts * sizeof(rv::StepParts));
  put(o_rows, sc.row_items.data(), sc.row_items.size() * sizeof(rv::StepItem));
  put(o_tiles, sc.tile_items.data(), sc.tile_items.size() * sizeof(rv::StepItem));
  put(o_joined, sc.joined.data(), sc.joined.size() * sizeof(int));
  put(o_pages, pg.data(), pg.size() * sizeof(int));
  if (s->work_cap < floats) {
    if (s->work) cudaFree(s->work);
    s->work = nullptr;
    s->work_cap = 0;
    const size_t want = floats + floats / 4;
    if ((e = cudaMalloc(reinterpret_cast<void**>(&s->work), want * sizeof(float))) != cudaSuccess)
      return cuda_fail(s, "partial results", e);
    s->work_cap = want;
  }
  if ((e = enter(s, st)) != cudaSuccess) return cuda_fail(s, "ordering streams", e);
  if ((e = cudaMemcpyAsync(s->meta, from, bytes, cudaMemcpyHostToDevice, st)) != cudaSuccess)
    return cuda_fail(s, "plan upload", e);
  if (small && (e = cudaEventRecord(sg.done, st)) != cudaSuccess) return cuda_fail(s, "plan upload", e);
  if ((e = leave(s, st)) != cudaSuccess) return cuda_fail(s, "ordering streams", e);
  s->counter = reinterpret_cast<int*>(s->meta);
  s->tokens = reinterpret_cast<rv::StepToken*>(s->meta + o_tokens);
  s->parts = n_parts ? reinterpret_cast<rv::StepParts*>(s->meta + o_parts) : nullptr;
  s->row_items = reinterpret_cast<rv::StepItem*>(s->meta + o_rows);
  s->tile_items = reinterpret_cast<rv::StepItem*>(s->meta + o_tiles);
  s->joined = reinterpret_cast<int*>(s->meta + o_joined);
  s->pages = reinterpret_cast<int*>(s->meta + o_pages);
  s->n_row_items = int(sc.row_items.size());
  s->n_tile_items = int(sc.tile_items.size());
  s->n_joined = int(sc.joined.size());
  s->n_parts = sc.n_parts;
  s->n_tokens = int(tokens);
  s->num_pages = num_pages;
  s->last_pos = last_pos;
  s->can_append = can_append;
  s->planned = true;
  return RV_OK;
}

}  // namespace

extern "C" {

int rv_step_create(int device, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t page_size, rv_step** out) {
  if (!out) return RV_E_INVALID;
  *out = nullptr;
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads > 1024 || (head_dim != 64 && head_dim != 128) ||
      (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256))
    return RV_E_INVALID;
  rv_step* s = new (std::nothrow) rv_step;
  if (!s) return RV_E_NOMEM;
  s->device = device;
  s->q_heads = q_heads;
  s->kv_heads = kv_heads;
  s->head_dim = head_dim;
  s->page_size = page_size;
  for (int f = 1; f <= rv::kRowTile; ++f)
    if (q_heads / kv_heads % f == 0) s->fold = f;
  DeviceGuard g(device);
  bool ok = g.ok && cudaEventCreateWithFlags(&s->last, cudaEventDisableTiming) == cudaSuccess;
  for (auto& sg : s->staging) ok = ok && cudaEventCreateWithFlags(&sg.done, cudaEventDisableTiming) == cudaSuccess;
  // Allocations of pinned memory take most of the time that making a step takes, so one serves its small needs.
  ok = ok && cudaHostAlloc(reinterpret_cast<void**>(&s->base_host), 2 * kSmallPlan + 256, cudaHostAllocMapped) == cudaSuccess;
  ok = ok && cudaMalloc(reinterpret_cast<void**>(&s->base_dev), kFirstRecords) == cudaSuccess;
  if (ok) {
    s->err_host = reinterpret_cast<unsigned int*>(s->base_host);
    *s->err_host = 0;
    ok = cudaHostGetDevicePointer(reinterpret_cast<void**>(&s->err_dev), s->err_host, 0) == cudaSuccess;
    for (int i = 0; i < 2; ++i) {
      s->staging[i].p = s->base_host + 256 + i * kSmallPlan;
    }
    s->meta = s->base_dev;
    s->meta_cap = kFirstRecords;
  }
  if (!ok) {
    cudaGetLastError();
    rv_step_destroy(s);
    return RV_E_CUDA;
  }
  *out = s;
  return RV_OK;
}

void rv_step_destroy(rv_step* s) {
  if (!s) return;
  {
    DeviceGuard g(s->device);
    if (s->used) cudaEventSynchronize(s->last);
    for (auto& sg : s->staging) {
      if (sg.done) {
        cudaEventSynchronize(sg.done);
        cudaEventDestroy(sg.done);
      }
    }
    if (s->own_meta) cudaFree(s->meta);
    if (s->work) cudaFree(s->work);
    if (s->base_dev) cudaFree(s->base_dev);
    if (s->base_host) cudaFreeHost(s->base_host);
    if (s->last) cudaEventDestroy(s->last);
  }
  delete s;
}

const char* rv_step_last_error(const rv_step* s) { return s ? s->err.c_str() : "null step"; }

int rv_step_tokens(const rv_step* s) { return s && s->planned ? s->n_tokens : 0; }

int rv_step_plan(rv_step* s, int32_t n_seqs, const int32_t* q_lens, const int32_t* own_lens, const int32_t* own_pages,
                 int32_t n_groups, const int32_t* group_sizes, const int32_t* prefix_lens, const int32_t* prefix_pages,
                 int64_t num_pages, int32_t causal, void* stream) {
  if (!s) return RV_E_INVALID;
  std::lock_guard<std::mutex> lk(s->mu);
  DeviceGuard g(s->device);
  if (!g.ok) return fail(s, RV_E_CUDA, "cudaSetDevice failed");
  try {
    return plan(s, n_seqs, q_lens, own_lens, own_pages, n_groups, group_sizes, prefix_lens, prefix_pages, num_pages,
                causal, static_cast<cudaStream_t>(stream));
  } catch (const std::exception& e) {
    s->planned = false;
    return fail(s, RV_E_NOMEM, e.what());
  }
}

int rv_step_append(rv_step* s, const rv_kv_cache* cache, const void* q, int64_t q_token, int64_t q_head, const void* k,
                   int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head, void* q_out,
                   int64_t q_out_token, int64_t q_out_head, const float* cos, const float* sin, int64_t positions,
                   int32_t rot, int32_t interleaved, void* stream) {
  if (!s) return RV_E_INVALID;
  std::lock_guard<std::mutex> lk(s->mu);
  try {
    if (device_error(s)) return RV_E_DEVICE;
    if (!s->planned) return fail(s, RV_E_NOT_READY, "no plan");
    if (!s->can_append)
      return fail(s, RV_E_INVALID, "the plan cannot append: own_lens below q_lens, or a page that new tokens go to is "
                                   "a prefix's, another sequence's or listed twice");
    rv::AppendArgs a{};
    rv::Act act;
    const std::string why = take_pool(s, cache, &a.pool, &act);
    if (!why.empty()) return fail(s, RV_E_INVALID, why);
    if (rot < 0 || rot > s->head_dim || rot % 2) return fail(s, RV_E_INVALID, "rot must be even, from 0 to head_dim");
    if (s->n_tokens == 0) return RV_OK;
    if (!k || !v || !q != !q_out) return fail(s, RV_E_INVALID, "null keys or values, or queries without their output");
    if (q && ((s->n_tokens > 1 && q_out_token == 0) || (s->q_heads > 1 && q_out_head == 0)))
      return fail(s, RV_E_INVALID, "the rotated queries of several tokens or heads would go to one place");
    if (rot > 0 && (!cos || !sin || s->last_pos >= positions))
      return fail(s, RV_E_INVALID, "the rotation table is missing or shorter than the step's positions");
    a.tokens = s->tokens;
    a.n_tokens = s->n_tokens;
    a.q_heads = s->q_heads;
    a.kv_heads = s->kv_heads;
    a.head_dim = s->head_dim;
    a.q = {q, q_token, q_head};
    a.k = {k, k_token, k_head};
    a.v = {v, v_token, v_head};
    a.q_out = q_out;
    a.q_out_token = q_out_token;
    a.q_out_head = q_out_head;
    a.cos = cos;
    a.sin = sin;
    a.rot = rot;
    a.interleaved = interleaved != 0;
    a.vec = rows_aligned(q, q_token, q_head) && rows_aligned(k, k_token, k_head) && rows_aligned(v, v_token, v_head) &&
            rows_aligned(q_out, q_out_token, q_out_head) && aligned16(cos) && aligned16(sin) && rot % 16 == 0;
    DeviceGuard g(s->device);
    if (!g.ok) return fail(s, RV_E_CUDA, "cudaSetDevice failed");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = enter(s, st);
    if (e == cudaSuccess) e = rv::kv_append(act, a, st);
    if (e == cudaSuccess) e = leave(s, st);
    return e == cudaSuccess ? RV_OK : cuda_fail(s, "rv_step_append", e);
  } catch (const std::exception& e) {
    return fail(s, RV_E_NOMEM, e.what());
  }
}

int rv_step_attend(rv_step* s, const rv_kv_cache* cache, const void* q, int64_t q_token, int64_t q_head, void* out,
                   int64_t out_token, int64_t out_head, float* lse, float scale, void* stream) {
  if (!s) return RV_E_INVALID;
  std::lock_guard<std::mutex> lk(s->mu);
  try {
    if (device_error(s)) return RV_E_DEVICE;
    if (!s->planned) return fail(s, RV_E_NOT_READY, "no plan");
    rv::AttendArgs a{};
    rv::Act act;
    const std::string why = take_pool(s, cache, &a.pool, &act);
    if (!why.empty()) return fail(s, RV_E_INVALID, why);
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail(s, RV_E_INVALID, "scale must be positive and finite");
    if (s->n_tokens == 0) return RV_OK;
    if (!q || !out) return fail(s, RV_E_INVALID, "null queries or output");
    if (s->q_heads == 1) q_head = out_head = s->head_dim;
    if (s->n_tokens == 1) {
      q_token = q_head * s->q_heads;
      out_token = out_head * s->q_heads;
    }
    if (!rows_aligned(q, q_token, q_head) || !rows_aligned(out, out_token, out_head))
      return fail(s, RV_E_INVALID, "queries and output must start on 16 bytes and have strides of 16 bytes");
    if (q_token <= 0 || q_head <= 0 || out_token <= 0 || out_head <= 0)
      return fail(s, RV_E_INVALID, "the strides of queries and output must be positive");
    a.row_items = s->row_items;
    a.tile_items = s->tile_items;
    a.parts = s->parts;
    a.joined = s->joined;
    a.pages = s->pages;
    a.n_row_items = s->n_row_items;
    a.n_tile_items = s->n_tile_items;
    a.n_joined = s->n_joined;
    a.tile_sms = s->sched.tile_sms;
    a.n_tokens = s->n_tokens;
    a.fold = s->fold;
    a.part_o = s->work;
    a.part_ml = reinterpret_cast<float2*>(s->work + s->n_parts * s->q_heads * s->head_dim);
    a.num_pages = cache->num_pages;
    a.err = s->err_dev;
    a.counter = s->counter;
    a.q_heads = s->q_heads;
    a.kv_heads = s->kv_heads;
    a.head_dim = s->head_dim;
    a.q = {q, q_token, q_head};
    a.out = out;
    a.out_token = out_token;
    a.out_head = out_head;
    a.lse = lse;
    a.scale = scale;
    DeviceGuard g(s->device);
    if (!g.ok) return fail(s, RV_E_CUDA, "cudaSetDevice failed");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = enter(s, st);
    if (e == cudaSuccess) e = rv::step_attend(act, a, st);
    if (e == cudaSuccess) e = leave(s, st);
    return e == cudaSuccess ? RV_OK : cuda_fail(s, "rv_step_attend", e);
  } catch (const std::exception& e) {
    return fail(s, RV_E_NOMEM, e.what());
  }
}

int rv_rms_norm(int32_t act_dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                const float* weight, void* residual_out, int64_t residual_out_stride, void* out, int64_t out_stride,
                int32_t out_dtype, float* scales, int32_t group, int64_t rows, int32_t hidden, float eps,
                void* stream) {
  if (act_dtype != RV_DTYPE_BF16 && act_dtype != RV_DTYPE_F16) return RV_E_INVALID;
  if (out_dtype != act_dtype && out_dtype != RV_DTYPE_E4M3) return RV_E_INVALID;
  const bool out8 = out_dtype == RV_DTYPE_E4M3;
  if (rows < 0 || hidden <= 0 || hidden > 65536 || !(eps >= 0.f) || !std::isfinite(eps)) return RV_E_INVALID;
  if (group != 0 && (!out8 || (group != 32 && group != 64 && group != 128 && group != 256) || hidden % group))
    return RV_E_INVALID;
  if (rows == 0) return RV_OK;
  if (!x || !weight || !out || (out8 != (scales != nullptr))) return RV_E_INVALID;
  // Input rows may repeat (stride 0); output rows may not overlap.
  if (x_stride < 0 || (residual && residual_stride < 0) ||
      (rows > 1 && (out_stride < hidden || (residual_out && residual_out_stride < hidden))))
    return RV_E_INVALID;
  rv::NormArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.rows = rows;
  a.hidden = hidden;
  a.x_stride = x_stride;
  a.residual_stride = residual_stride;
  a.residual_out_stride = residual_out_stride;
  a.out_stride = out_stride;
  a.residual_out = residual_out;
  a.out = out;
  a.scales = scales;
  a.group = group ? group : hidden;
  a.eps = eps;
  auto on16 = [](const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; };
  a.vec = hidden % 8 == 0 && on16(x, x_stride) && on16(residual, residual_stride) &&
          on16(residual_out, residual_out_stride) &&
          (out8 ? reinterpret_cast<uintptr_t>(out) % 8 == 0 && out_stride % 8 == 0 : on16(out, out_stride));
  const cudaError_t e =
      rv::rms_norm(act_dtype == RV_DTYPE_BF16 ? rv::Act::kBf16 : rv::Act::kF16, a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? RV_OK : RV_E_CUDA;
}

int rv_step_append_record(rv_step* s, const rv_step_append_args* a) {
  if (!a) return RV_E_INVALID;
  return rv_step_append(s, a->cache, a->q, a->q_token_stride, a->q_head_stride, a->k, a->k_token_stride,
                        a->k_head_stride, a->v, a->v_token_stride, a->v_head_stride, a->q_out, a->q_out_token_stride,
                        a->q_out_head_stride, a->cos, a->sin, a->positions, a->rot, a->interleaved, a->stream);
}

int rv_step_attend_record(rv_step* s, const rv_step_attend_args* a) {
  if (!a) return RV_E_INVALID;
  return rv_step_attend(s, a->cache, a->q, a->q_token_stride, a->q_head_stride, a->out, a->out_token_stride,
                        a->out_head_stride, a->lse, to_float(a->scale), a->stream);
}

int rv_rms_norm_record(const rv_rms_norm_args* a) {
  if (!a) return RV_E_INVALID;
  auto go = [a] {
    return rv_rms_norm(a->act_dtype, a->x, a->x_stride, a->residual, a->residual_stride, a->weight, a->residual_out,
                       a->residual_out_stride, a->out, a->out_stride, a->out_dtype, a->scales, a->group, a->rows,
                       a->hidden, to_float(a->eps), a->stream);
  };
  if (a->device < 0) return go();
  DeviceGuard g(a->device);
  return g.ok ? go() : RV_E_CUDA;
}

}  // extern "C"
