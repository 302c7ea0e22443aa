// Block tables and slot maps of a step, from request lengths on the device.
//
// Three lists are filled: the new tokens' rows, the slots of every key, and the
// blocks taken from the free ones.  Where an element of a list belongs follows
// from sums over the requests before its own, so every block sums up all
// requests for itself (8 bytes each, from L2) instead of waiting for a first
// launch to do it, and then searches the sums of its 256 threads' shares: one
// launch, and no block waits for another.  A block taken from the free ones is
// read from their stack by whoever needs it, never from the tables that another
// thread writes meanwhile.
//
// Bound by latency: 32 decodes take 4 us, of which the launch and the sums of the
// requests are most; 500 requests with 2M key slots (16 MB, which stay in L2) 17.
#include "common.cuh"

namespace cs {
namespace {

constexpr int kMapThreads = 256, kKeysEach = 8;

struct Sums {
  int64_t tok, key, need;
};

struct Located {
  int request, local;  // local: place among the request's own elements
  int64_t need;        // blocks that the requests before it take
};

__device__ __forceinline__ int64_t blocks_of(int64_t n, int bs) { return (n + bs - 1) / bs; }

struct Request {
  int len, fresh;  // tokens after the step, of which new
  int had, want;   // blocks before and after (had = want without a free stack)
};

__device__ __forceinline__ Request request_of(const cs_step_maps_params& p, int r) {
  Request q;
  q.len = p.lengths[r];
  q.fresh = p.new_tokens[r];
  q.want = (int)blocks_of(q.len, p.block_size);
  q.had = p.free_blocks ? (int)blocks_of(q.len - q.fresh, p.block_size) : q.want;
  return q;
}

__global__ void __launch_bounds__(kMapThreads) step_maps_kernel(const cs_step_maps_params p) {
  __shared__ Sums before[kMapThreads + 1];  // sums before a thread's share; the totals
  __shared__ Sums warps[kMapThreads / 32];
  __shared__ int failed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = (p.requests + kMapThreads - 1) / kMapThreads;
  const int r0 = min(p.requests, tid * share), r1 = min(p.requests, r0 + share);
  if (tid == 0) failed = 0;
  __syncthreads();
  Sums own{0, 0, 0};
  bool bad = false;
  for (int r = r0; r < r1; ++r) {
    const int len = p.lengths[r], fresh = p.new_tokens[r];
    bad |= len < 0 || fresh < 0 || fresh > len || blocks_of(len, p.block_size) > p.table_width;
    if (bad) break;
    const Request q = request_of(p, r);
    own.tok += q.fresh;
    own.key += q.len;
    own.need += q.want - q.had;
  }
  Sums run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(~0u, run.tok, o), b = __shfl_up_sync(~0u, run.key, o),
                  c = __shfl_up_sync(~0u, run.need, o);
    if (lane >= o) run.tok += a, run.key += b, run.need += c;
  }
  if (lane == 31) warps[warp] = run;
  if (bad) failed = 1;
  __syncthreads();
  for (int w = 0; w < warp; ++w)
    run.tok += warps[w].tok, run.key += warps[w].key, run.need += warps[w].need;
  before[tid] = Sums{run.tok - own.tok, run.key - own.key, run.need - own.need};
  if (tid == kMapThreads - 1) before[kMapThreads] = run;
  __syncthreads();
  const Sums all = before[kMapThreads];
  const int have = p.free_blocks ? *p.free_count : 0;
  const bool fail = failed || all.tok > p.tokens || (p.key_slots && all.key > p.keys) ||
                    all.need > have || have < 0 || (p.free_blocks && have > p.free_size);
  const int64_t step = (int64_t)gridDim.x * kMapThreads;
  const int64_t first = (int64_t)blockIdx.x * kMapThreads + tid;

  if (blockIdx.x == 0) {
    Sums at = before[tid];
    for (int r = r0; r < r1; ++r) {
      p.starts[r] = fail ? 0 : (int32_t)at.tok;
      if (p.key_starts) p.key_starts[r] = fail ? 0 : at.key;
      if (fail) continue;
      at.tok += p.new_tokens[r];
      at.key += p.lengths[r];
    }
    if (tid == 0) {
      p.starts[p.requests] = fail ? 0 : (int32_t)all.tok;
      if (p.key_starts) p.key_starts[p.requests] = fail ? 0 : all.key;
      if (p.free_left) *p.free_left = have - (fail ? 0 : (int32_t)all.need);
      if (fail) report(p.status, CS_ST_CAPACITY);
    }
  }

  // the request that holds element v of the list whose sums `sum` reads, and
  // whose requests have `count` elements each
  auto locate = [&](int64_t v, auto sum, auto count) {
    int lo = 0, hi = kMapThreads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sum(before[mid]) <= v) lo = mid;
      else hi = mid - 1;
    }
    Located l;
    l.request = lo * share;
    l.need = before[lo].need;
    int64_t at = sum(before[lo]);
    while (true) {
      const Request q = request_of(p, l.request);
      const int64_t n = count(q);
      if (v < at + n) break;
      at += n;
      l.need += q.want - q.had;
      ++l.request;
    }
    l.local = (int)(v - at);
    return l;
  };
  auto block_id = [&](const Located& l, const Request& q, int j) {
    return j >= q.had ? p.free_blocks[have - 1 - (l.need + j - q.had)]
                      : p.tables[l.request * p.table_stride + j];
  };
  auto slot_of = [&](int64_t id, int offset) {
    if (id < 0 || id >= p.num_blocks) {
      report(p.status, CS_ST_SLOT_RANGE);
      return (int64_t)-1;
    }
    return id * p.block_size + offset;
  };

  for (int64_t i = first; i < p.tokens; i += step) {
    int64_t position = 0, slot = -1;
    if (!fail && i < all.tok) {
      const Located l = locate(i, [](const Sums& s) { return s.tok; },
                               [](const Request& q) { return (int64_t)q.fresh; });
      const Request q = request_of(p, l.request);
      const int at = q.len - q.fresh + l.local, j = at / p.block_size;
      position = (int64_t)at + p.position_offset;
      slot = slot_of(block_id(l, q, j), at - j * p.block_size);
    }
    p.positions[i] = position;
    p.slots[i] = slot;
  }
  if (p.key_slots) {
    // kKeysEach keys a thread: one search, and mostly one block
    for (int64_t i = kKeysEach * first; i < p.keys; i += kKeysEach * step) {
      int64_t out[kKeysEach], base = -1;  // base: slot of the block's first key
      Located l{0, 0, 0};
      Request q{0, 0, 0, 0};
      int block = 0, offset = 0;
#pragma unroll
      for (int k = 0; k < kKeysEach; ++k) {
        out[k] = -1;
        if (fail || i + k >= all.key) continue;
        const bool search = l.local >= q.len;  // the first one, or the next request's
        if (search) {
          l = locate(i + k, [](const Sums& s) { return s.key; },
                     [](const Request& r) { return (int64_t)r.len; });
          q = request_of(p, l.request);
          block = l.local / p.block_size;
          offset = l.local - block * p.block_size;
        } else if (offset == p.block_size) {
          ++block;
          offset = 0;
        }
        if (search || offset == 0) base = slot_of(block_id(l, q, block), 0);
        out[k] = base < 0 ? -1 : base + offset;
        ++l.local;
        ++offset;
      }
      if (i + kKeysEach <= p.keys && reinterpret_cast<uintptr_t>(p.key_slots) % 16 == 0) {
        longlong2* to = reinterpret_cast<longlong2*>(p.key_slots + i);
#pragma unroll
        for (int k = 0; k < kKeysEach / 2; ++k) to[k] = make_longlong2(out[2 * k], out[2 * k + 1]);
      } else {
        for (int k = 0; k < kKeysEach && i + k < p.keys; ++k) p.key_slots[i + k] = out[k];
      }
    }
  }
  if (!fail) {
    for (int64_t i = first; i < all.need; i += step) {
      const Located l = locate(i, [](const Sums& s) { return s.need; },
                               [](const Request& q) { return (int64_t)(q.want - q.had); });
      const int j = request_of(p, l.request).had + l.local;
      p.tables[l.request * p.table_stride + j] = p.free_blocks[have - 1 - i];
    }
  }
}

}  // namespace
}  // namespace cs

extern "C" int cs_step_maps(const cs_step_maps_params* p, void* stream) {
  using namespace cs;
  CS_HOST_CHECK(p != nullptr && p->requests >= 0 && p->block_size > 0 && p->num_blocks >= 0);
  CS_HOST_CHECK(p->table_width >= 0 && p->tokens >= 0 && p->tokens < INT32_MAX && p->keys >= 0);
  CS_HOST_CHECK(p->starts != nullptr && (p->tokens == 0 || (p->positions && p->slots)));
  CS_HOST_CHECK(p->requests == 0 || (p->lengths && p->new_tokens));
  CS_HOST_CHECK(p->requests == 0 || p->table_width == 0 || p->tables);
  CS_HOST_CHECK(p->requests <= 1 || p->table_stride >= p->table_width);
  CS_HOST_CHECK(!p->free_blocks ||
                (p->free_count && p->free_left && p->free_left != p->free_count));
  CS_HOST_CHECK(p->key_slots != nullptr || p->keys == 0);
  // blocks that fit the machine at once: each sums up every request (500 requests
  // with 2M keys in all take 41 us with one an SM, 23 with four)
  const int64_t work = p->tokens + (p->key_slots ? (p->keys + kKeysEach - 1) / kKeysEach : 0);
  const int64_t blocks = (work + kMapThreads - 1) / kMapThreads;
  const int64_t most = 4ll * num_sms();
  step_maps_kernel<<<(unsigned)(blocks < 1 ? 1 : blocks > most ? most : blocks), kMapThreads, 0,
                     as_stream(stream)>>>(*p);
  CS_LAUNCH_CHECK();
  return CS_OK;
}
