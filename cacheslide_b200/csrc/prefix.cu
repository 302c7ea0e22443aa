// Attention of a batch behind shared prefixes (cs_prefix_plan,
// cs_prefix_attn): the host's plan of the batch and the CUDA-core kernel.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <functional>
#include <type_traits>
#include <vector>

#include "prefix.cuh"

namespace cs {
namespace {

constexpr int kRowWarps = 4;
constexpr int kMaxDim = 512;
constexpr int kLaneElems = kMaxDim / 32;

struct RowArgs {
  const char* q;
  int64_t qt, qh;  // byte strides
  PagedView pv;
  const int64_t* prefix_slots;
  const int64_t* suffix_slots;
  const int4* tokens;
  int hq, group, dim;
  float scale;
  char* out;
  int64_t ot, oh;
  float* lse;
  int32_t* status;
};

// One block per (token, query head): warp w takes keys w, w + 4, ... of the
// token's prefix and own range with its own running maximum and sum, lanes
// holding the head's elements; the warps join in shared memory.  A key whose
// score is -inf adds nothing (as exp(-inf) = 0), also where it comes first.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) prefix_rows_kernel(RowArgs a) {
  __shared__ float acc_s[kRowWarps][kMaxDim];
  __shared__ float ml_s[kRowWarps][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x / a.hq;
  const int h = (int)(blockIdx.x - t * a.hq);
  const int kvh = h / a.group;
  const int4 tok = a.tokens[t];
  const T* q = reinterpret_cast<const T*>(a.q + t * a.qt + h * a.qh);
  float qr[kLaneElems], acc[kLaneElems];
#pragma unroll
  for (int m = 0; m < kLaneElems; ++m) {
    const int e = lane + 32 * m;
    qr[m] = e < a.dim ? Elem<T>::to_f(q[e]) * a.scale : 0.f;
    acc[m] = 0.f;
  }
  float mx = -INFINITY, sum = 0.f;
  const int np = tok.y - tok.x, n = np + (tok.w - tok.z);
  for (int j = warp; j < n; j += kRowWarps) {
    const int64_t s = j < np ? a.prefix_slots[tok.x + j] : a.suffix_slots[tok.z + (j - np)];
    const bool ok = a.pv.valid(s);
    if (!ok && lane == 0) report(a.status, CS_ST_SLOT_RANGE);
    float dot = 0.f;
#pragma unroll
    for (int m = 0; m < kLaneElems; ++m) {
      const int e = lane + 32 * m;
      if (e < a.dim && ok)
        dot += qr[m] * Elem<T>::to_f(*reinterpret_cast<const T*>(a.pv.addr(s, kvh, e)));
    }
    dot = warp_sum(dot);
    if (dot == -INFINITY) continue;
    const float top = fmaxf(mx, dot);
    const float keep = mx == -INFINITY ? 0.f : expf(mx - top), p = expf(dot - top);
    // a NaN score keeps p NaN (fmaxf drops it, the subtraction does not)
    mx = top;
    sum = sum * keep + p;
#pragma unroll
    for (int m = 0; m < kLaneElems; ++m) {
      const int e = lane + 32 * m;
      if (e < a.dim)
        acc[m] = acc[m] * keep +
                 (ok ? p * Elem<T>::to_f(*reinterpret_cast<const T*>(a.pv.addr(s, kvh, a.dim + e)))
                     : 0.f);
    }
  }
#pragma unroll
  for (int m = 0; m < kLaneElems; ++m) {
    const int e = lane + 32 * m;
    if (e < a.dim) acc_s[warp][e] = acc[m];
  }
  if (lane == 0) {
    ml_s[warp][0] = mx;
    ml_s[warp][1] = sum;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f, f[kRowWarps];
  for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, ml_s[w][0]);
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) {
    f[w] = ml_s[w][0] == -INFINITY ? 0.f : expf(ml_s[w][0] - top);
    // a warp that saw nothing has sum 0; one that saw only NaN has sum NaN
    total += ml_s[w][1] == 0.f ? 0.f : (f[w] == 0.f && ml_s[w][1] != ml_s[w][1] ? ml_s[w][1]
                                                                                : f[w] * ml_s[w][1]);
  }
  T* out = reinterpret_cast<T*>(a.out + t * a.ot + h * a.oh);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int e = threadIdx.x; e < a.dim; e += blockDim.x) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w)
      if (ml_s[w][1] != 0.f) o += f[w] * acc_s[w][e];
    out[e] = Elem<T>::from_f(total == total ? o * inv : total);
  }
  if (a.lse && threadIdx.x == 0) a.lse[t * a.hq + h] = total == 0.f ? -INFINITY : top + logf(total);
}

}  // namespace
}  // namespace cs

namespace cs {
namespace {

// A unit of work before it is cut: tokens x prefix keys, then own keys.
struct Unit {
  int64_t tok0, ntok, a0, a1, b0, b1;
  int64_t steps() const { return tiles(a1 - a0) + tiles(b1 - b0); }
  static int64_t tiles(int64_t n) { return (n + kPrefixTile - 1) / kPrefixTile; }
};

struct Layout {
  const int32_t* tok;  // the plan's token rows
  int64_t tokens;
  int group;           // query heads a KV head
  int kv_heads, q_heads, head_dim;
  std::vector<int64_t> group_tok;   // first token of each group, and the end
  std::vector<int64_t> req_tok;     // first token of each request, and the end
  int64_t lo(int64_t t) const { return tok[4 * t + 2]; }
  int64_t hi(int64_t t) const { return tok[4 * t + 3]; }
};

// Row tiles of `rows` query rows with all their keys: the prefix, then every
// own key that one of the tile's tokens sees.
std::vector<Unit> whole_units(const Layout& l, int rows) {
  std::vector<Unit> out;
  const int64_t per = (int64_t)(kPrefixTile / l.group) * (rows / kPrefixTile);
  for (size_t g = 0; g + 1 < l.group_tok.size(); ++g)
    for (int64_t t = l.group_tok[g]; t < l.group_tok[g + 1]; t += per) {
      const int64_t n = std::min(per, l.group_tok[g + 1] - t);
      out.push_back({t, n, l.tok[4 * t], l.tok[4 * t + 1], l.lo(t), l.hi(t + n - 1)});
    }
  return out;
}

// The prefix apart from the own keys: row tiles over the prefix alone, and
// runs of whole requests (at most a row tile of tokens, about `keys` keys)
// over their own keys, so that few rows meet keys that they do not see.
std::vector<Unit> split_units(const Layout& l, int64_t keys) {
  std::vector<Unit> out;
  const int64_t per = kPrefixTile / l.group;
  for (size_t g = 0; g + 1 < l.group_tok.size(); ++g)
    for (int64_t t = l.group_tok[g]; t < l.group_tok[g + 1]; t += per)
      out.push_back({t, std::min(per, l.group_tok[g + 1] - t), l.tok[4 * t], l.tok[4 * t + 1], 0,
                     0});
  int64_t first = 0, count = 0, b0 = 0, b1 = 0;
  auto flush = [&] {
    if (count > 0) out.push_back({first, count, 0, 0, b0, b1});
    count = 0;
  };
  for (size_t r = 0; r + 1 < l.req_tok.size(); ++r) {
    const int64_t t0 = l.req_tok[r], n = l.req_tok[r + 1] - t0;
    if (n == 0 || l.hi(t0 + n - 1) == l.lo(t0)) continue;  // no query, or no own key seen
    if (n > per) {
      flush();
      for (int64_t t = t0; t < t0 + n; t += per) {
        const int64_t m = std::min(per, t0 + n - t);
        out.push_back({t, m, 0, 0, l.lo(t), l.hi(t + m - 1)});
      }
      continue;
    }
    const int64_t k0 = l.lo(t0), k1 = l.hi(t0 + n - 1);
    if (count > 0 && (t0 + n - first > per || k1 - b0 > keys)) flush();
    if (count == 0) {
      first = t0;
      b0 = k0;
    }
    count = t0 + n - first;
    b1 = k1;
  }
  flush();
  return out;
}

// Every unit from `whole` on cut into equal runs of at most `most` key tiles
// (those before it stay whole), of a part's tokens only those that see its keys.
std::vector<PrefixItem> cut(const Layout& l, const std::vector<Unit>& units, int64_t most,
                            size_t whole) {
  std::vector<PrefixItem> out;
  for (size_t x = 0; x < units.size(); ++x) {
    const Unit& u = units[x];
    const int64_t steps = u.steps(), na = Unit::tiles(u.a1 - u.a0);
    if (steps == 0) continue;
    const int64_t parts = x < whole ? 1 : (steps + most - 1) / most;
    for (int64_t p = 0; p < parts; ++p) {
      const int64_t s0 = steps * p / parts, s1 = steps * (p + 1) / parts;
      Unit v = u;
      v.a0 = std::min(u.a1, u.a0 + std::min(s0, na) * kPrefixTile);
      v.a1 = std::min(u.a1, u.a0 + std::min(s1, na) * kPrefixTile);
      v.b0 = std::min(u.b1, u.b0 + std::max<int64_t>(s0 - na, 0) * kPrefixTile);
      v.b1 = std::min(u.b1, u.b0 + std::max<int64_t>(s1 - na, 0) * kPrefixTile);
      if (v.a0 == v.a1) {
        while (v.ntok > 0 && l.hi(v.tok0) <= v.b0) ++v.tok0, --v.ntok;
        while (v.ntok > 0 && l.lo(v.tok0 + v.ntok - 1) >= v.b1) --v.ntok;
        if (v.ntok == 0) continue;
      }
      out.push_back({(int32_t)v.tok0, (int32_t)v.ntok, (int32_t)v.a0, (int32_t)v.a1,
                     (int32_t)v.b0, (int32_t)v.b1, -1, 0});
    }
  }
  return out;
}

// What a block costs, in microseconds: a tile of prefix keys, and its start and
// end.  A tile of own keys costs more: masks, and rows that lie apart.
struct Cost {
  int slots;
  double step, fixed;
  double of(const PrefixItem& i) const {
    return step * (Unit::tiles(i.a1 - i.a0) + 1.3 * Unit::tiles(i.b1 - i.b0)) + fixed;
  }
};

// Estimated time of a launch: the blocks dealt out in order to the slot that
// is free first (their sum and half the longest where they are many), joined
// with the way of their records to the SMs by a soft maximum; then the partial
// results to memory and back and the launch that joins them.
class Estimate {
 public:
  Estimate(const Layout& l, const std::vector<PrefixItem>& items, const Cost& c)
      : heads_(l.kv_heads), c_(c) {
    if (items.empty()) return;
    double tiles = 0, sum = 0, longest = 0;
    const PrefixItem* first = &items[0];  // of those with the most key tiles
    std::vector<int32_t> cover(l.tokens + 1, 0);  // items that begin less those that end
    for (const PrefixItem& i : items) {
      tiles += i.steps();
      sum += c.of(i);
      longest = std::max(longest, c.of(i));
      if (i.steps() > first->steps()) first = &i;
      ++cover[i.tok0];
      --cover[i.tok0 + i.ntok];
    }
    double parts = 0;  // of the tokens in several items
    for (int64_t t = 0, n = 0; t < l.tokens; ++t) {
      n += cover[t];
      if (n > 1) parts += n;
    }
    const double bytes = tiles * l.kv_heads * kPrefixTile * 4.0 * l.head_dim;
    read_ = std::pow(bytes / 6.0e6 + c.fixed, 3);
    joined_ = parts > 0 ? 4.0 + parts * l.q_heads * l.head_dim * 8.0 / 4.0e6 : 0.0;
    const double even = sum * heads_ / c.slots;
    many_ = (int64_t)items.size() * heads_ > 4ll * c.slots;
    bound = total(many_ ? even + 0.5 * c.of(*first) : std::max(longest, even));
  }
  // of the items as the blocks are dealt out, long ones first
  double of(const std::vector<PrefixItem>& items) const {
    if (items.empty() || many_) return bound;
    double end = 0;
    std::vector<double> busy(c_.slots, 0.0);  // a heap, the first to be free in front
    for (const PrefixItem& i : items)
      for (int h = 0; h < heads_; ++h) {
        std::pop_heap(busy.begin(), busy.end(), std::greater<double>());
        busy.back() += c_.of(i);
        end = std::max(end, busy.back());
        std::push_heap(busy.begin(), busy.end(), std::greater<double>());
      }
    return total(end);
  }
  double bound = 0;  // what it is not below

 private:
  double total(double end) const { return std::cbrt(end * end * end + read_) + joined_; }
  int heads_;
  Cost c_;
  double read_ = 0, joined_ = 0;
  bool many_ = false;
};

// The cut of least estimated time, if that is below `least` (or that is
// negative): candidates are numbers of key tiles a part, and with them numbers
// of units that stay whole (what full rounds of the slots take; the rest, cut,
// fills the last one).  They are tried by their bounds, the lowest first, until
// no other can be better.
template <typename Make>
double best_cut(const Layout& l, const Cost& c, Make units_for, double least,
                std::vector<PrefixItem>& best) {
  struct Candidate {
    double bound;
    int64_t most;
    size_t whole;
  };
  std::vector<Candidate> candidates;
  int64_t longest = 1, tiles = 0;
  for (const Unit& u : units_for(1)) tiles += u.steps();
  // from what gives at most eight blocks a slot
  const int64_t from = std::max<int64_t>(1, tiles * l.kv_heads / (8ll * c.slots));
  for (int64_t most = from; most <= std::max(from, 2 * longest);
       most += most < 6 ? 1 : most / 4) {
    const std::vector<Unit> units = units_for(most);
    for (const Unit& u : units) longest = std::max(longest, u.steps());
    const size_t rounds = units.size() * l.kv_heads / c.slots;
    for (size_t whole : {(size_t)0, rounds * c.slots / l.kv_heads}) {
      if (whole > 0 && most >= longest) continue;
      const Estimate e(l, cut(l, units, most, whole), c);
      if (least < 0 || e.bound < least) candidates.push_back({e.bound, most, whole});
      if (rounds == 0) break;
    }
  }
  std::stable_sort(candidates.begin(), candidates.end(),
                   [](const Candidate& x, const Candidate& y) { return x.bound < y.bound; });
  for (const Candidate& x : candidates) {
    if (least >= 0 && x.bound >= least) break;
    std::vector<PrefixItem> items = cut(l, units_for(x.most), x.most, x.whole);
    std::stable_sort(items.begin(), items.end(), [](const PrefixItem& a, const PrefixItem& b) {
      return a.steps() > b.steps();
    });
    const double e = Estimate(l, items, c).of(items);
    if (least < 0 || e < least) {
      least = e;
      best = std::move(items);
    }
  }
  return least;
}

// partial results: an output row and its sum, float32
int64_t part_bytes(int64_t part_tokens, int64_t q_heads, int64_t head_dim) {
  return part_tokens * q_heads * (head_dim + 1) * (int64_t)sizeof(float);
}

int make_plan(const cs_prefix_shape* s, cs_prefix_plan_info* info, int32_t* words,
              int64_t capacity) {
  int64_t tokens = 0, n_suffix = 0, n_prefix = 0, members = 0;
  // each length is bounded before it is added, so that no sum wraps
  for (int b = 0; b < s->requests; ++b) {
    CS_HOST_CHECK(s->query_lens[b] >= 0 && s->suffix_lens[b] >= 0);
    if (s->query_lens[b] > INT32_MAX || s->suffix_lens[b] > INT32_MAX) return CS_ERR_UNSUPPORTED;
    tokens += s->query_lens[b];
    n_suffix += s->suffix_lens[b];
    if (tokens > INT32_MAX / 8 || n_suffix > INT32_MAX / 2) return CS_ERR_UNSUPPORTED;
  }
  for (int g = 0; g < s->groups; ++g) {
    CS_HOST_CHECK(s->group_sizes[g] >= 0 && s->prefix_lens[g] >= 0);
    CS_HOST_CHECK(s->group_sizes[g] <= s->requests - members);
    members += s->group_sizes[g];
    if (s->prefix_lens[g] > INT32_MAX) return CS_ERR_UNSUPPORTED;
    n_prefix += s->prefix_lens[g];
    if (n_prefix > INT32_MAX / 2) return CS_ERR_UNSUPPORTED;
  }
  CS_HOST_CHECK(members == s->requests);
  std::memset(info, 0, sizeof(*info));
  info->group = s->q_heads / s->kv_heads;
  info->tokens = tokens;
  info->n_prefix = n_prefix;
  info->n_suffix = n_suffix;

  std::vector<int32_t> rows(tokens * 4);
  Layout l{rows.data(), tokens, s->q_heads / s->kv_heads, s->kv_heads, s->q_heads, s->head_dim,
           {0}, {0}};
  int32_t* w = rows.data();
  int64_t b = 0, p0 = 0, k0 = 0, t = 0;
  for (int g = 0; g < s->groups; ++g) {
    for (int64_t m = 0; m < s->group_sizes[g]; ++m, ++b) {
      const int64_t n = s->query_lens[b], keys = s->suffix_lens[b];
      for (int64_t i = 0; i < n; ++i, w += 4) {
        const int64_t seen = keys - n + i + 1;
        w[0] = (int32_t)p0;
        w[1] = (int32_t)(p0 + s->prefix_lens[g]);
        w[2] = (int32_t)k0;
        w[3] = (int32_t)(k0 + (seen > 0 ? seen : 0));
      }
      k0 += keys;
      t += n;
      l.req_tok.push_back(t);
    }
    p0 += s->prefix_lens[g];
    l.group_tok.push_back(t);
  }

  std::vector<PrefixItem> items;
  std::vector<int32_t> join, list;
  const bool tc = (s->dtype == CS_F16 || s->dtype == CS_BF16) &&
                  (s->head_dim == 64 || s->head_dim == 128) && l.group <= kPrefixTile;
  if (tc && tokens > 0) {
    info->variant = 1;
    const int sms = num_sms();
    // two blocks of 128 rows an SM, which read their keys for each row tile,
    // or one of 256 rows; both costs as measured with 32/8 heads of 128 (of 64 a
    // step costs less, which only the byte terms know)
    const double narrow = best_cut(
        l, Cost{2 * sms, 1.75, 5.0},
        [&](int64_t most) { return split_units(l, most * kPrefixTile); }, -1, items);
    std::vector<PrefixItem> wide;
    if (best_cut(l, Cost{sms, 2.1, 6.0},
                 [&](int64_t) { return whole_units(l, 2 * kPrefixTile); }, narrow, wide) < narrow) {
      info->variant = 2;
      items = std::move(wide);
    }
    // a token in one item alone gets its output from it, if that holds for
    // all of the item's tokens; the others are joined from partials
    std::vector<int32_t> in(tokens + 1, 0);
    for (const PrefixItem& i : items)
      for (int32_t k = 0; k < i.ntok; ++k) ++in[i.tok0 + k];
    std::vector<char> alone(items.size(), 1);
    std::vector<int32_t> parts(tokens + 1, 0);
    for (size_t x = 0; x < items.size(); ++x) {
      PrefixItem& i = items[x];
      for (int32_t k = 0; k < i.ntok; ++k)
        if (in[i.tok0 + k] != 1) alone[x] = 0;
      if (alone[x]) continue;
      if (info->part_tokens > INT32_MAX / 2) return CS_ERR_UNSUPPORTED;
      i.part = (int32_t)info->part_tokens;
      info->part_tokens += i.ntok;
      for (int32_t k = 0; k < i.ntok; ++k) ++parts[i.tok0 + k];
    }
    std::vector<int32_t> at(tokens + 1, 0);
    int32_t entries = 0;
    for (int64_t x = 0; x < tokens; ++x) {
      at[x] = entries;
      if (parts[x] == 0 && in[x] != 0) continue;  // written by its item
      join.insert(join.end(), {(int32_t)x, entries, parts[x], 0});
      entries += parts[x];
    }
    list.resize(entries);
    for (const PrefixItem& i : items)
      for (int32_t k = 0; i.part >= 0 && k < i.ntok; ++k) list[at[i.tok0 + k]++] = i.part + k;
  }
  const int64_t iw = (int64_t)items.size() * (sizeof(PrefixItem) / 4);
  info->n_items = (int64_t)items.size();
  info->n_join = (int64_t)join.size() / 4;
  info->item_off = tokens * 4;
  info->join_off = info->item_off + iw;
  info->list_off = info->join_off + (int64_t)join.size();
  info->words = info->list_off + (int64_t)list.size();
  info->workspace = part_bytes(info->part_tokens, s->q_heads, s->head_dim);
  if (words == nullptr || capacity < info->words) return CS_ERR_TOO_LARGE;
  std::copy(rows.begin(), rows.end(), words);
  if (iw) std::memcpy(words + info->item_off, items.data(), iw * 4);
  std::copy(join.begin(), join.end(), words + info->join_off);
  std::copy(list.begin(), list.end(), words + info->list_off);
  return CS_OK;
}

}  // namespace
}  // namespace cs

extern "C" int cs_prefix_plan(const cs_prefix_shape* s, cs_prefix_plan_info* info, int32_t* words,
                              int64_t capacity) {
  using namespace cs;
  CS_HOST_CHECK(s != nullptr && info != nullptr && capacity >= 0);
  CS_HOST_CHECK(s->q_heads > 0 && s->kv_heads > 0 && s->q_heads % s->kv_heads == 0);
  CS_HOST_CHECK(s->head_dim > 0 && s->groups >= 0 && s->requests >= 0);
  CS_HOST_CHECK(s->groups == 0 || (s->prefix_lens && s->group_sizes));
  CS_HOST_CHECK(s->requests == 0 || (s->query_lens && s->suffix_lens));
  if (s->dtype != CS_F32 && s->dtype != CS_F16 && s->dtype != CS_BF16) return CS_ERR_UNSUPPORTED;
  if (s->head_dim > kMaxDim) return CS_ERR_UNSUPPORTED;
  try {
    return make_plan(s, info, words, capacity);
  } catch (...) {  // no memory: nothing may leave a C entry but a status
    return CS_ERR_TOO_LARGE;
  }
}

extern "C" int cs_prefix_attn(const cs_prefix_params* p, const cs_prefix_plan_info* info,
                              const int32_t* plan, void* workspace, void* stream) {
  using namespace cs;
  CS_HOST_CHECK(p != nullptr && info != nullptr);
  const cs_paged_kv& kv = p->paged;
  CS_HOST_CHECK(kv.cache != nullptr && kv.block_size > 0 && kv.kv_heads > 0 && kv.head_dim > 0);
  CS_HOST_CHECK(p->q_heads > 0 && p->q_heads % kv.kv_heads == 0);
  CS_HOST_CHECK(std::isfinite((float)p->scale));  // as the kernels use it
  if (kv.dtype != CS_F32 && kv.dtype != CS_F16 && kv.dtype != CS_BF16) return CS_ERR_UNSUPPORTED;
  if (kv.head_dim > kMaxDim) return CS_ERR_UNSUPPORTED;
  // a plan's row tiles, partials and workspace belong to its heads and type
  CS_HOST_CHECK(info->group == p->q_heads / kv.kv_heads);
  if (info->variant > 0)
    CS_HOST_CHECK((kv.dtype == CS_F16 || kv.dtype == CS_BF16) &&
                  (kv.head_dim == 64 || kv.head_dim == 128) &&
                  info->workspace == part_bytes(info->part_tokens, p->q_heads, kv.head_dim));
  if (info->tokens == 0) return CS_OK;
  CS_HOST_CHECK(p->q && p->out && plan && (info->workspace == 0 || workspace));
  CS_HOST_CHECK((info->n_prefix == 0 || p->prefix_slots) &&
                (info->n_suffix == 0 || p->suffix_slots));
  if (info->variant > 0) {
    const int rc = prefix_attn_sm100(*p, *info, plan, workspace, as_stream(stream));
    if (rc != CS_ERR_UNSUPPORTED) return rc;
  }
  const int64_t es = dtype_size(kv.dtype);
  RowArgs a{static_cast<const char*>(p->q), p->q_stride_tok * es, p->q_stride_head * es,
            PagedView::make(kv), p->prefix_slots, p->suffix_slots,
            reinterpret_cast<const int4*>(plan), p->q_heads, (int)(p->q_heads / kv.kv_heads),
            (int)kv.head_dim, (float)p->scale, static_cast<char*>(p->out), p->o_stride_tok * es,
            p->o_stride_head * es, p->lse, p->status};
  if (info->tokens * p->q_heads > INT32_MAX) return CS_ERR_UNSUPPORTED;
  const unsigned blocks = (unsigned)(info->tokens * p->q_heads);
  if (kv.dtype == CS_F32)
    prefix_rows_kernel<float><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  else if (kv.dtype == CS_F16)
    prefix_rows_kernel<__half><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  else
    prefix_rows_kernel<__nv_bfloat16><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  CS_LAUNCH_CHECK();
  return CS_OK;
}
