// The paged pool held in 4 bits: its layout, and how its attention kernels
// divide a batch among their blocks.
//
// A unit is 16 tokens of one head, contiguous: one bulk copy fetches all that
// 16 keys of a head need.  The order of the codes in a row is the tensor
// unit's: a lane's 16 bytes of a key row (8 of a value row) are its part of the
// operand fragments of every product over that row, two codes of a pair four
// (for values: two) apart, so that one AND leaves a pair of 16-bit numbers.
#pragma once

#include "common.cuh"

namespace cs {

constexpr int kUnit = 16;  // tokens of a unit

template <int D, int NG>  // head dim, groups of a head
struct Unit4 {
  static constexpr int W = D / 32;
  static constexpr int kRow = D / 2;  // bytes of a token's key (or value) codes
  static constexpr int oV = kUnit * kRow, oKp = 2 * oV, oVp = oKp + kUnit * NG * 4;
  static constexpr int kBytes = oVp + kUnit * NG * 4;
  static_assert(kBytes % 128 == 0, "units are whole lines");
};

// a slot's unit and its token there
struct Place4 {
  int64_t block;
  int unit, row;
};

struct Pool4 {
  char* base;
  int64_t num_blocks;
  int hkv, bs, units, unit_bytes;
  int shift;  // log2(bs), -1 when it is no power of two

  __host__ static Pool4 make(const cs_kv4_pool& p) {
    Pool4 v;
    v.base = static_cast<char*>(p.storage);
    v.num_blocks = p.num_blocks;
    v.hkv = p.kv_heads;
    v.bs = p.block_size;
    v.units = p.block_size / kUnit;
    v.shift = -1;
    for (int s = 0; s < 31; ++s)
      if (1 << s == p.block_size) v.shift = s;
    v.unit_bytes = kUnit * p.head_dim + 8 * kUnit * (p.head_dim / p.group);
    return v;
  }
  __device__ __forceinline__ char* unit(int64_t block, int head, int u) const {
    return base + ((block * hkv + head) * units + u) * unit_bytes;
  }
  __device__ __forceinline__ bool valid(int64_t slot) const {
    return slot >= 0 && slot < num_blocks * bs;
  }
  __device__ __forceinline__ Place4 place(int64_t slot) const {
    Place4 p;
    if (shift >= 0) {
      p.block = slot >> shift;
      p.row = (int)slot & (bs - 1);
    } else if (slot < (1ll << 32)) {  // a 64-bit division is about 100 instructions
      const uint32_t b = (uint32_t)slot / (uint32_t)bs;
      p.block = b;
      p.row = (int)((uint32_t)slot - b * (uint32_t)bs);
    } else {
      p.block = slot / bs;
      p.row = (int)(slot - p.block * bs);
    }
    p.unit = p.row / kUnit;
    p.row %= kUnit;
    return p;
  }
};

// what the host checks of a pool
inline int check_pool4(const cs_kv4_pool& p) {
  CS_HOST_CHECK(p.storage != nullptr || p.num_blocks == 0);
  CS_HOST_CHECK(p.num_blocks >= 0 && p.kv_heads > 0 && p.block_size > 0);
  if (p.head_dim != 64 && p.head_dim != 128) return CS_ERR_UNSUPPORTED;
  if (p.group != 32 && p.group != 64 && p.group != 128) return CS_ERR_UNSUPPORTED;
  if (p.group > p.head_dim || p.block_size % kUnit) return CS_ERR_UNSUPPORTED;
  if (p.dtype != CS_F16 && p.dtype != CS_BF16) return CS_ERR_UNSUPPORTED;
  CS_HOST_CHECK(reinterpret_cast<uintptr_t>(p.storage) % 16 == 0);
  return CS_OK;
}

// f(type, dim, groups) with the three as types
template <typename F>
int by_pool4(const cs_kv4_pool& p, F f) {
  auto dims = [&](auto* t) {
    const int ng = p.head_dim / p.group;
    auto go = [&](auto d, auto n) { return f(t, d, n); };
    using std::integral_constant;
    if (p.head_dim == 128) {
      if (ng == 4) return go(integral_constant<int, 128>(), integral_constant<int, 4>());
      if (ng == 2) return go(integral_constant<int, 128>(), integral_constant<int, 2>());
      return go(integral_constant<int, 128>(), integral_constant<int, 1>());
    }
    if (ng == 2) return go(integral_constant<int, 64>(), integral_constant<int, 2>());
    return go(integral_constant<int, 64>(), integral_constant<int, 1>());
  };
  return p.dtype == CS_F16 ? dims(static_cast<__half*>(nullptr))
                           : dims(static_cast<__nv_bfloat16*>(nullptr));
}

// a pair of 16-bit numbers as floats
template <typename T> __device__ __forceinline__ float2 pair_of(uint32_t x);
template <> __device__ __forceinline__ float2 pair_of<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<__half2*>(&x));
}
template <> __device__ __forceinline__ float2 pair_of<__nv_bfloat16>(uint32_t x) {
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// ... and as such a pair
template <typename T> struct Pair16;
template <> struct Pair16<__half> {
  using type = __half2;
};
template <> struct Pair16<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <typename T> using pair16 = typename Pair16<T>::type;
template <typename T> __device__ __forceinline__ pair16<T> as_pair(uint32_t x) {
  return *reinterpret_cast<pair16<T>*>(&x);
}
template <typename P> __device__ __forceinline__ uint32_t pair_bits(P x) {
  return *reinterpret_cast<uint32_t*>(&x);
}

// ------------------------------------------------------------- attention
struct Attn4 {
  Pool4 pool;
  const char* q;
  int64_t qt, qh;  // byte strides
  char* out;
  int64_t ot, oh;
  float* lse;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* starts;
  int32_t* status;
  float* part_o;    // [2 * workers][rows][dim]: normalised
  float* part_lse;  // [2 * workers][rows]: log2 of the softmax denominator
  int4* joins;      // [workers]: request, row tile, head, last worker; request -1: none
  int64_t tokens, longest;  // longest: what a row of the tables holds
  int requests, hq, G;
  int vec_q, vec_out;  // 16-byte loads, 8-byte stores fit
  int zero_rest;
  uint32_t flip;  // the scale is negative: the queries' signs
  float scale2;   // |scale| * log2 e
};

struct Request4 {
  int len, n, start;
};

// `floor`: the largest start before its own (0 at least), below which its rows
// belong to another request
__device__ __forceinline__ Request4 request4(const Attn4& a, int b, int floor) {
  Request4 r;
  r.len = a.lengths[b];
  r.start = a.starts ? a.starts[b] : b;
  const int end = a.starts ? a.starts[b + 1] : b + 1;
  const bool rows = r.start >= floor && end >= r.start && end <= a.tokens;
  if (!rows || r.len > a.longest) report(a.status, CS_ST_CAPACITY);
  r.n = rows ? end - r.start : 0;
  r.len = r.len < 0 ? 0 : r.len > a.longest ? (int)a.longest : r.len;
  return r;
}

// The rows of a (request, KV head) are its tokens' G heads each, token after
// token, in tiles of RT; the keys of a row tile go in steps of KT.  A tile's
// steps are those its last token sees, one at least (its rows are written).
template <int RT, int KT>
struct Share4 {
  int request, tile, head, step;  // where the worker begins
  int64_t todo, per;              // steps it takes, and every one takes at most
  Request4 r;

  static __device__ __forceinline__ int tiles(const Request4& r, int G) {
    return (r.n * G + RT - 1) / RT;  // (31 bits hold any row count and a tile more)
  }
  static __device__ __forceinline__ int last_token(const Request4& r, int G, int tile) {
    const int i = (tile * RT + RT - 1) / G;
    return i < r.n ? i : r.n - 1;
  }
  static __device__ __forceinline__ int steps(const Request4& r, int G, int tile) {
    const int keys = r.len - r.n + last_token(r, G, tile) + 1;
    return keys > 0 ? (keys + KT - 1) / KT : 1;
  }
  static __device__ __forceinline__ int64_t cost(const Attn4& a, const Request4& r) {
    int64_t s = 0;
    const int n = tiles(r, a.G);
    for (int t = 0; t < n; ++t) s += steps(r, a.G, t);
    return s * a.pool.hkv;
  }

  // Every worker (block) sums up all requests for itself and takes an equal
  // range of all steps, `least` of them at least; the thread whose requests hold
  // the range's first step says where that is.  `Scratch` is shared memory; the
  // first THREADS threads sum, all threads of the block call.  Returns whether the
  // starts are in order; where they are not, the sums are made once more with each
  // thread's largest start before its own.
  template <int THREADS>
  struct Scratch {
    int64_t warps[THREADS / 32];
    int floors[THREADS / 32];
    Share4 found;
  };
  template <int THREADS>
  __device__ __forceinline__ bool find(const Attn4& a, int worker, int workers, int least,
                                       Scratch<THREADS>& s) {
    constexpr int kWarps = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int share = (a.requests + THREADS - 1) / THREADS;
    const int b0 = min(a.requests, tid * share), b1 = min(a.requests, b0 + share);
    Request4 mine{0, 0, 0};
    int64_t own = 0, run = 0;
    int floor = 0;  // before this thread's first request
    bool ordered;
    for (int pass = 0;; ++pass) {
      bool falls = false;
      if (tid < THREADS) {
        own = 0;
        int low = floor;
        for (int b = b0; b < b1; ++b) {
          mine = request4(a, b, low);
          if (a.starts) {
            falls |= a.starts[b + 1] < a.starts[b];
            low = max(low, a.starts[b]);
          }
          own += cost(a, mine);
        }
        run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(~0u, run, o);
          if (lane >= o) run += x;
        }
        if (lane == 31) s.warps[warp] = run;
      }
      ordered = !__syncthreads_or(falls);
      if (ordered || pass) break;
      if (tid < THREADS) {
        for (int b = b0; b < b1; ++b) floor = max(floor, a.starts[b]);
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(~0u, floor, o);
          if (lane >= o) floor = max(floor, x);
        }
        if (lane == 31) s.floors[warp] = floor;
        floor = __shfl_up_sync(~0u, floor, 1);
        if (lane == 0) floor = 0;
      }
      __syncthreads();
      if (tid < THREADS)
        for (int w = 0; w < warp; ++w) floor = max(floor, s.floors[w]);
    }
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) run += all;
      all += s.warps[w];
    }
    per = max((all + workers - 1) / workers, (int64_t)least);
    const int64_t from = worker * per;
    todo = max((int64_t)0, min(per, all - from));
    if (todo > 0 && tid < THREADS && from >= run - own && from < run) {
      int64_t at = run - own;
      Share4 f;
      for (f.request = b0;; ++f.request) {  // one of this thread's requests has it
        f.r = share == 1 ? mine : request4(a, f.request, floor);
        const int64_t c = cost(a, f.r);
        if (from < at + c) break;
        at += c;
        if (a.starts) floor = max(floor, a.starts[f.request]);
      }
      for (f.tile = 0;; ++f.tile) {
        const int64_t c = (int64_t)steps(f.r, a.G, f.tile) * a.pool.hkv;
        if (from < at + c) break;
        at += c;
      }
      const int n = steps(f.r, a.G, f.tile);
      f.head = (int)((from - at) / n);
      f.step = (int)(from - at - (int64_t)f.head * n);
      s.found = f;
    }
    __syncthreads();
    request = s.found.request, tile = s.found.tile, head = s.found.head, step = s.found.step;
    r = s.found.r;
    return ordered;
  }

  // to the first step of the next (head, tile, request) that has rows
  __device__ __forceinline__ void next(const Attn4& a) {
    step = 0;
    if (++head < a.pool.hkv) return;
    head = 0;
    if (++tile < tiles(r, a.G)) return;
    tile = 0;
    int floor = r.start + r.n;  // the largest start so far: its rows were in order
    do {
      r = request4(a, ++request, floor);  // there is one: the worker has steps to do
      floor = max(floor, r.start);
    } while (r.n == 0);
  }
};

}  // namespace cs
