// Head norms and position rotation (cs_qk_norm_rope and its gradient), and
// their append form into the paged pool (cs_kv_append_rotated).
//
// For one head x of a token, with r = (mean x^2 + eps)^-1/2, n = x r:
//   forward   y  = R(pos) (n w)
//   backward  g  = R(pos)^T dy,  dx = r (w g - n mean(w g n)),  dw += g n
// R turns pairs of elements, so a lane that owns whole pairs needs nothing
// from its neighbours but the sum over the row.  Sums and products are
// float32; the result is rounded once, to the output's type.
//
// Bound: HBM.  Each element is read once and written once (16-bit: 4 bytes
// an element and direction); the arithmetic is about ten operations an
// element.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace cs {
namespace {

constexpr int kMaxDim = 512;
constexpr int kMaxPairs = kMaxDim / 2 / 32;  // pairs a lane of a warp-per-row kernel
constexpr int kStreamBlocks = 296;           // 148 SMs x 2: the fixed partition of the gradient
// A token's angles, in row groups of the streamed gradient.  With none, the
// blocks of the kind with fewer heads ended last; 32/8 heads of 128, 64/4 of
// 128, 32/8 of 64 took 178, 367, 214 us at 0; 165, 283, 184 at 0.5; 162, 270,
// 172 at 1; 168, 273, 178 at 1.5.
constexpr double kAngleCost = 1.0;
constexpr int kRowWarps = 8;

struct Rows {
  const char* x;
  const char* dy;  // gradient only
  char* y;
  const void* w;
  int64_t xt, xh, yt, yh;  // byte strides
  int heads;
};

struct RotArgs {
  Rows q, k;
  const float* cos;
  const float* sin;
  int64_t table_rows, table_stride;
  const int64_t* positions;
  int64_t tokens;
  int dim, rot, interleaved, wdtype;
  float eps, inv_dim;
  int32_t* status;
};

__device__ __forceinline__ float load_weight(const void* w, int dtype, int i) {
  if (dtype == CS_F32) return static_cast<const float*>(w)[i];
  if (dtype == CS_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// the two elements of pair p: rotated ones first, then the rest in halves
__device__ __forceinline__ void pair_elems(const RotArgs& a, int p, int& i, int& j) {
  const int half = a.rot >> 1;
  if (p < half) {
    i = a.interleaved ? 2 * p : p;
    j = a.interleaved ? 2 * p + 1 : p + half;
  } else {
    i = a.rot + (p - half);
    j = i + ((a.dim - a.rot) >> 1);
  }
}

// of a pair that turns (p < rot / 2)
__device__ __forceinline__ void angle(const RotArgs& a, int64_t pos, int p, float& c, float& s) {
  const bool ok = pos >= 0 && pos < a.table_rows;
  c = ok ? a.cos[pos * a.table_stride + p] : __int_as_float(0x7fc00000);
  s = ok ? a.sin[pos * a.table_stride + p] : __int_as_float(0x7fc00000);
}

// one pair turned; the products' order is fixed, so that every kernel here
// rounds alike
__device__ __forceinline__ float turned0(float a, float b, float c, float s) {
  return fmaf(a, c, -__fmul_rn(b, s));
}
__device__ __forceinline__ float turned1(float a, float b, float c, float s) {
  return fmaf(b, c, __fmul_rn(a, s));
}

// One warp per row (token, head): lane l owns pairs l, l + 32, ...; at(i) is
// the place of output element i.  The whole row is read before any of it is
// written, so the output may be the input.
template <typename T, typename At>
__device__ __forceinline__ void norm_turn_row(const RotArgs& a, const T* x, At at, const void* w,
                                              int64_t pos, int lane) {
  float u[kMaxPairs], v[kMaxPairs], ss = 0.f;
  const int pairs = a.dim >> 1;
#pragma unroll
  for (int m = 0; m < kMaxPairs; ++m) {
    const int p = lane + 32 * m;
    u[m] = v[m] = 0.f;
    if (p < pairs) {
      int i, j;
      pair_elems(a, p, i, j);
      u[m] = Elem<T>::to_f(x[i]);
      v[m] = Elem<T>::to_f(x[j]);
      ss += u[m] * u[m] + v[m] * v[m];
    }
  }
  const float r = w ? rsqrtf(warp_sum(ss) * a.inv_dim + a.eps) : 1.f;
#pragma unroll
  for (int m = 0; m < kMaxPairs; ++m) {
    const int p = lane + 32 * m;
    if (p < pairs) {
      int i, j;
      pair_elems(a, p, i, j);
      float p0 = u[m], p1 = v[m];
      if (w) {
        p0 *= r * load_weight(w, a.wdtype, i);
        p1 *= r * load_weight(w, a.wdtype, j);
      }
      // elements past rot are not turned by a zero angle: 0 x inf is NaN
      if (p < (a.rot >> 1)) {
        float c, s;
        angle(a, pos, p, c, s);
        const float t = turned0(p0, p1, c, s);
        p1 = turned1(p0, p1, c, s);
        p0 = t;
      }
      *at(i) = Elem<T>::from_f(p0);
      *at(j) = Elem<T>::from_f(p1);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32)
    norm_rope_rows_kernel(const __grid_constant__ RotArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.q.heads + a.k.heads;
  const int64_t total = a.tokens * heads;
  for (int64_t row = blockIdx.x * (int64_t)kRowWarps + (threadIdx.x >> 5); row < total;
       row += (int64_t)gridDim.x * kRowWarps) {
    const int64_t t = row / heads;
    int h = (int)(row - t * heads);
    const bool isq = h < a.q.heads;
    const Rows& rw = isq ? a.q : a.k;
    if (!isq) h -= a.q.heads;
    const int64_t pos = a.positions[t];
    if (lane == 0 && (pos < 0 || pos >= a.table_rows)) report(a.status, CS_ST_POS_RANGE);
    T* y = reinterpret_cast<T*>(rw.y + t * rw.yt + h * rw.yh);
    norm_turn_row<T>(a, reinterpret_cast<const T*>(rw.x + t * rw.xt + h * rw.xh),
                     [&](int i) { return y + i; }, rw.w, pos, lane);
  }
}

// Append: rows of q (dense out), k (rotated into the record's K half) and v
// (copied into its V half).  These one-warp-a-row kernels serve the heads,
// strides and pools that vectors do not fit (latency bound, about 0.8 TB/s).
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32)
    append_rows_kernel(RotArgs a, PagedView pv, const int64_t* __restrict__ slots, Rows v) {
  const int lane = threadIdx.x & 31;
  const int heads = a.q.heads + 2 * a.k.heads;
  const int64_t total = a.tokens * heads;
  for (int64_t row = blockIdx.x * (int64_t)kRowWarps + (threadIdx.x >> 5); row < total;
       row += (int64_t)gridDim.x * kRowWarps) {
    const int64_t t = row / heads;
    int h = (int)(row - t * heads);
    const int64_t pos = a.positions[t];
    const bool pos_ok = pos >= 0 && pos < a.table_rows;
    if (lane == 0 && !pos_ok) report(a.status, CS_ST_POS_RANGE);
    if (h < a.q.heads) {
      T* y = reinterpret_cast<T*>(a.q.y + t * a.q.yt + h * a.q.yh);
      norm_turn_row<T>(a, reinterpret_cast<const T*>(a.q.x + t * a.q.xt + h * a.q.xh),
                       [&](int i) { return y + i; }, a.q.w, pos, lane);
      continue;
    }
    h -= a.q.heads;
    const bool isv = h >= a.k.heads;
    if (isv) h -= a.k.heads;
    const int64_t slot = slots[t];
    if (!pv.valid(slot)) {
      if (lane == 0 && slot != -1) report(a.status, CS_ST_SLOT_RANGE);
      continue;
    }
    if (!pos_ok) continue;
    if (isv) {
      const T* x = reinterpret_cast<const T*>(v.x + t * v.xt + h * v.xh);
      for (int e = lane; e < a.dim; e += 32)
        *reinterpret_cast<T*>(pv.addr(slot, h, a.dim + e)) = x[e];
      continue;
    }
    norm_turn_row<T>(a, reinterpret_cast<const T*>(a.k.x + t * a.k.xt + h * a.k.xh),
                     [&](int i) { return reinterpret_cast<T*>(pv.addr(slot, h, i)); }, a.k.w, pos,
                     lane);
  }
}

// Gradient, one warp per row; blocks below nq take rows of q, the rest rows
// of k.  Each warp keeps dw of its rows in registers, the block adds its warps
// in order, and its partial goes to part[block * dim].
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32)
    norm_rope_grad_rows_kernel(RotArgs a, int nq, float* __restrict__ part) {
  __shared__ float acc[kRowWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool isk = (int)blockIdx.x >= nq;
  const Rows& rw = isk ? a.k : a.q;
  const int b = isk ? blockIdx.x - nq : blockIdx.x, blocks = isk ? gridDim.x - nq : nq;
  const int pairs = a.dim >> 1;
  float d0[kMaxPairs], d1[kMaxPairs];
#pragma unroll
  for (int m = 0; m < kMaxPairs; ++m) d0[m] = d1[m] = 0.f;
  const int64_t total = a.tokens * rw.heads;
  for (int64_t row = b * (int64_t)kRowWarps + warp; row < total;
       row += (int64_t)blocks * kRowWarps) {
    const int64_t t = row / rw.heads;
    const int h = (int)(row - t * rw.heads);
    const int64_t pos = a.positions[t];
    const T* x = reinterpret_cast<const T*>(rw.x + t * rw.xt + h * rw.xh);
    const T* dy = reinterpret_cast<const T*>(rw.dy + t * rw.yt + h * rw.yh);
    T* dx = reinterpret_cast<T*>(rw.y + t * rw.yt + h * rw.yh);
    if (lane == 0 && (pos < 0 || pos >= a.table_rows)) report(a.status, CS_ST_POS_RANGE);
    float n0[kMaxPairs], n1[kMaxPairs], g0[kMaxPairs], g1[kMaxPairs], ss = 0.f, dot = 0.f;
#pragma unroll
    for (int m = 0; m < kMaxPairs; ++m) {
      const int p = lane + 32 * m;
      n0[m] = n1[m] = g0[m] = g1[m] = 0.f;
      if (p < pairs) {
        int i, j;
        pair_elems(a, p, i, j);
        g0[m] = Elem<T>::to_f(dy[i]);
        g1[m] = Elem<T>::to_f(dy[j]);
        if (p < (a.rot >> 1)) {
          float c, s;
          angle(a, pos, p, c, s);
          const float t = turned0(g0[m], g1[m], c, -s);
          g1[m] = turned1(g0[m], g1[m], c, -s);
          g0[m] = t;
        }
        if (rw.w) {
          n0[m] = Elem<T>::to_f(x[i]);
          n1[m] = Elem<T>::to_f(x[j]);
          ss += n0[m] * n0[m] + n1[m] * n1[m];
          dot += load_weight(rw.w, a.wdtype, i) * g0[m] * n0[m] +
                 load_weight(rw.w, a.wdtype, j) * g1[m] * n1[m];
        }
      }
    }
    float r = 1.f, mean = 0.f;
    if (rw.w) {
      r = rsqrtf(warp_sum(ss) * a.inv_dim + a.eps);
      mean = warp_sum(dot) * r * a.inv_dim;  // mean(w g n)
    }
#pragma unroll
    for (int m = 0; m < kMaxPairs; ++m) {
      const int p = lane + 32 * m;
      if (p < pairs) {
        int i, j;
        pair_elems(a, p, i, j);
        if (rw.w) {
          const float u = n0[m] * r, v = n1[m] * r;
          d0[m] += g0[m] * u;
          d1[m] += g1[m] * v;
          g0[m] = r * (load_weight(rw.w, a.wdtype, i) * g0[m] - u * mean);
          g1[m] = r * (load_weight(rw.w, a.wdtype, j) * g1[m] - v * mean);
        }
        dx[i] = Elem<T>::from_f(g0[m]);
        dx[j] = Elem<T>::from_f(g1[m]);
      }
    }
  }
  if (!rw.w) return;
#pragma unroll
  for (int m = 0; m < kMaxPairs; ++m) {
    const int p = lane + 32 * m;
    if (p < pairs) {
      int i, j;
      pair_elems(a, p, i, j);
      acc[warp][i] = d0[m];
      acc[warp][j] = d1[m];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.dim; e += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < kRowWarps; ++w) s += acc[w][e];
    part[(int64_t)blockIdx.x * a.dim + e] = s;
  }
}

// ------------------------------------------------------------ vector kernels
// LPR lanes own a row, each 4 pairs of it as two vectors of 4 elements:
// half-split pairs take one vector of either half, interleaved pairs lie
// inside the vectors.  A warp takes a task: up to kGroups groups of 32 / LPR
// heads of one token and one kind (q, k or v), whose angles and weights it
// loads once, all rows' loads before the first arithmetic.  Vectors of 4
// keep a lane's share small (8 elements of a row): with 8 pairs a lane the
// kernels held 98 (forward) and 118 (gradient) registers, a quarter of the
// SM's warps, and 2.9 TB/s.
//
// Forward, 32768 tokens of 32/8 heads of 128, bf16: 115 us, 5.8 TB/s (113 with
// the row sums' shuffles left out: the rest is HBM and the warps' starts);
// append of 65536 tokens of 64/8 heads without norms, fp16: 400 us, 6.8 TB/s, in
// a short run, 428 us, 6.35 TB/s, sustained (a plain copy: 6.46): HBM.  Two
// groups a task: 143 and 497 us; eight: 144 and 412 us; two warps a block: 117
// and 400 us; eight: 122 and 434 us.  Registers for nine blocks an SM against
// the 60 that the compiler takes (32768 tokens of 32/8 heads of 128): forward
// 114 to 117 us in bf16, 118 to 129 interleaved, 113 to 118 in fp16; append 139
// to 146, 139 to 148, 133 to 141; the 56 registers that this leaves cost most
// bf16 forms 4 to 24 bytes of spills, which these times include.  For ten
// blocks the forward was 15 us worse; in float32 (103 us for 16384 tokens)
// nine are 2 us worse.
constexpr int kP = 4;        // pairs a lane
constexpr int kGroups = 4;   // row groups a task
constexpr int kVecWarps = 4;
template <typename T> constexpr int kVecBlocks = sizeof(T) == 2 ? 9 : 1;

template <typename T> struct Vec4 { using type = uint2; };
template <> struct Vec4<float> { using type = uint4; };

template <typename T>
__device__ __forceinline__ void unpack(const typename Vec4<T>::type& v, float* f) {
  if constexpr (std::is_same<T, float>::value) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  } else if constexpr (std::is_same<T, __half>::value) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
  } else {
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ typename Vec4<T>::type pack(const float* f) {
  if constexpr (std::is_same<T, float>::value)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  else
    return make_uint2(Pack2<T>::pack(f[0], f[1]), Pack2<T>::pack(f[2], f[3]));
}

// A lane's P pairs, two at a time for the packed float32 instructions: a[i]
// holds the first elements of pairs 2i and 2i + 1, b[i] the second.
template <int P>
struct Pairs {
  float2 a[P / 2], b[P / 2];
};

// two vectors' elements <-> pairs
template <int P, bool INTER>
__device__ __forceinline__ void to_pairs(const float* u, const float* v, Pairs<P>& p) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    if constexpr (INTER) {
      const float* x = i < P / 4 ? u + 4 * i : v + 4 * i - P;
      p.a[i] = make_float2(x[0], x[2]);
      p.b[i] = make_float2(x[1], x[3]);
    } else {
      p.a[i] = make_float2(u[2 * i], u[2 * i + 1]);
      p.b[i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
  }
}
template <int P, bool INTER>
__device__ __forceinline__ void from_pairs(const Pairs<P>& p, float* u, float* v) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    if constexpr (INTER) {
      float* x = i < P / 4 ? u + 4 * i : v + 4 * i - P;
      x[0] = p.a[i].x, x[2] = p.a[i].y;
      x[1] = p.b[i].x, x[3] = p.b[i].y;
    } else {
      u[2 * i] = p.a[i].x, u[2 * i + 1] = p.a[i].y;
      v[2 * i] = p.b[i].x, v[2 * i + 1] = p.b[i].y;
    }
  }
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg(float2 x) { return make_float2(-x.x, -x.y); }

// 4 weights from element e of a head on, as float32
__device__ __forceinline__ void weights_at(const void* w, int dtype, int e, float* f) {
  if (dtype == CS_F32) {
    unpack<float>(__ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + e)), f);
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + e));
    if (dtype == CS_F16) unpack<__half>(v, f);
    else unpack<__nv_bfloat16>(v, f);
  }
}

// which elements a lane owns: vectors at e0 and e1; pairs p0 .. p0 + 3 when
// they turn
struct Lane {
  int p0, e0, e1;
  bool turns;
};
template <bool INTER>
__device__ __forceinline__ Lane lane_of(const RotArgs& a, int l) {
  Lane n;
  n.p0 = l * kP;
  const int half = a.rot >> 1;
  n.turns = n.p0 < half;
  if (n.turns) {
    n.e0 = INTER ? 2 * n.p0 : n.p0;
    n.e1 = INTER ? n.e0 + kP : n.p0 + half;
  } else {
    n.e0 = a.rot + (n.p0 - half);
    n.e1 = n.e0 + ((a.dim - a.rot) >> 1);
  }
  return n;
}

__device__ __forceinline__ void angles(const RotArgs& a, int64_t pos, int p0, float* c, float* s) {
  if (pos >= 0 && pos < a.table_rows) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(a.cos + pos * a.table_stride + p0));
    const float4 y = __ldg(reinterpret_cast<const float4*>(a.sin + pos * a.table_stride + p0));
    c[0] = x.x, c[1] = x.y, c[2] = x.z, c[3] = x.w;
    s[0] = y.x, s[1] = y.y, s[2] = y.z, s[3] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < kP; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

struct AppendArgs {
  PagedView pv;
  const int64_t* slots;  // NULL: dense outputs only
  Rows v;
  int bs_shift;
};

// tasks that cover `heads` rows of a token
__host__ __device__ inline int tasks_of(int heads, int lanes) {
  const int per = 32 / lanes * kGroups;
  return (heads + per - 1) / per;
}

// Forward and append: tasks of q, then k, then (append) v of each token.
template <typename T, int LPR, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kVecWarps * 32, kVecBlocks<T>)
    norm_rope_vec_kernel(const __grid_constant__ RotArgs a, const __grid_constant__ AppendArgs ap,
                         unsigned tasks) {
  using V = typename Vec4<T>::type;
  constexpr int S = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const unsigned task = blockIdx.x * kVecWarps + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const int nq = tasks_of(a.q.heads, LPR), nk = tasks_of(a.k.heads, LPR);
  const unsigned per = nq + (APPEND ? 2 : 1) * nk;
  const unsigned t = task / per;
  int part = task - t * per;
  int kind = 0;  // 0: q, 1: k, 2: v
  if (part >= nq) part -= nq, kind = 1;
  if (APPEND && kind == 1 && part >= nk) part -= nk, kind = 2;
  const Rows& rw = kind == 0 ? a.q : (kind == 1 ? a.k : ap.v);
  const int heads = rw.heads;
  const int h0 = part * (S * kGroups) + lane / LPR;
  const Lane ln = lane_of<INTER>(a, lane % LPR);
  const char* x = rw.x + t * rw.xt + h0 * rw.xh;
  V x0[kGroups], x1[kGroups];
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    if (h0 + u * S < heads) {
      const T* row = reinterpret_cast<const T*>(x + u * S * rw.xh);
      x0[u] = *reinterpret_cast<const V*>(row + ln.e0);
      x1[u] = *reinterpret_cast<const V*>(row + ln.e1);
    } else {
      x0[u] = x1[u] = V{};
    }
  }
  const int64_t pos = a.positions[t];
  const bool pos_ok = pos >= 0 && pos < a.table_rows;
  if (!pos_ok && lane == 0) report(a.status, CS_ST_POS_RANGE);
  char* y = rw.y + t * rw.yt + h0 * rw.yh;
  int64_t yh = rw.yh;
  if (APPEND && kind > 0) {
    const int64_t slot = ap.slots[t];
    if (!ap.pv.valid(slot)) {
      if (slot != -1 && lane == 0) report(a.status, CS_ST_SLOT_RANGE);
      return;
    }
    if (!pos_ok) return;
    if (slot < ap.pv.native_total) {
      const int64_t b = ap.bs_shift >= 0 ? slot >> ap.bs_shift : slot / ap.pv.bs;
      const int64_t o = slot - (ap.bs_shift >= 0 ? b << ap.bs_shift : b * ap.pv.bs);
      yh = ap.pv.sh;
      y = ap.pv.cache + b * ap.pv.sb + o * ap.pv.so + h0 * yh +
          (kind == 2 ? a.dim * (int)sizeof(T) : 0);
    } else {
      yh = ap.pv.ssh;
      y = (kind == 2 ? ap.pv.side_v : ap.pv.side_k) + (slot - ap.pv.native_total) * ap.pv.ssr +
          h0 * yh;
    }
  }
  if (!APPEND || kind < 2) {
    float c[kP], s[kP];
    if (ln.turns) angles(a, pos, ln.p0, c, s);
    Pairs<kP> w;
    if (rw.w) {
      float w0[kP], w1[kP];
      weights_at(rw.w, a.wdtype, ln.e0, w0);
      weights_at(rw.w, a.wdtype, ln.e1, w1);
      to_pairs<kP, INTER>(w0, w1, w);
    }
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      float f0[kP], f1[kP];
      unpack<T>(x0[u], f0);
      unpack<T>(x1[u], f1);
      Pairs<kP> n;
      to_pairs<kP, INTER>(f0, f1, n);
      if (rw.w) {
        float2 ss = both(0.f);
#pragma unroll
        for (int i = 0; i < kP / 2; ++i)
          ss = __ffma2_rn(n.a[i], n.a[i], __ffma2_rn(n.b[i], n.b[i], ss));
        const float2 r = both(rsqrtf(row_sum<LPR>(ss.x + ss.y) * a.inv_dim + a.eps));
#pragma unroll
        for (int i = 0; i < kP / 2; ++i) {
          n.a[i] = __fmul2_rn(n.a[i], __fmul2_rn(r, w.a[i]));
          n.b[i] = __fmul2_rn(n.b[i], __fmul2_rn(r, w.b[i]));
        }
      }
      if (ln.turns) {
#pragma unroll
        for (int i = 0; i < kP / 2; ++i) {
          const float2 ci = make_float2(c[2 * i], c[2 * i + 1]);
          const float2 si = make_float2(s[2 * i], s[2 * i + 1]);
          const float2 t = __ffma2_rn(n.a[i], ci, neg(__fmul2_rn(n.b[i], si)));
          n.b[i] = __ffma2_rn(n.b[i], ci, __fmul2_rn(n.a[i], si));
          n.a[i] = t;
        }
      }
      from_pairs<kP, INTER>(n, f0, f1);
      x0[u] = pack<T>(f0);
      x1[u] = pack<T>(f1);
    }
  }
#pragma unroll
  for (int u = 0; u < kGroups; ++u) {
    if (h0 + u * S < heads) {
      T* row = reinterpret_cast<T*>(y + u * S * yh);
      *reinterpret_cast<V*>(row + ln.e0) = x0[u];
      *reinterpret_cast<V*>(row + ln.e1) = x1[u];
    }
  }
}

// ----------------------------------------------------------- streamed kernel
// For many rows: 16-byte vectors (P = 8 pairs a lane, 4 in float32), each warp
// streaming its rows through a ring of row groups in shared memory by
// cp.async, every lane its own vectors (so no barrier): bytes in flight cost
// no registers, and a lane's longer share halves the instructions a row.
template <typename T> constexpr int kPairs = 16 / (int)sizeof(T);

template <typename T, int P>
__device__ __forceinline__ void unpack16(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (P == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = x.x, f[2 * i + 1] = x.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T, int P>
__device__ __forceinline__ uint4 pack16(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (P == 4) w[i] = __float_as_uint(f[i]);
    else w[i] = Pack2<T>::pack(f[2 * i], f[2 * i + 1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, int P, bool INTER>
__device__ __forceinline__ void load_pairs(const uint4& x, const uint4& y, Pairs<P>& p) {
  float u[P], v[P];
  unpack16<T, P>(x, u);
  unpack16<T, P>(y, v);
  to_pairs<P, INTER>(u, v, p);
}
template <typename T, int P, bool INTER>
__device__ __forceinline__ void store_pairs(const Pairs<P>& p, uint4& x, uint4& y) {
  float u[P], v[P];
  from_pairs<P, INTER>(p, u, v);
  x = pack16<T, P>(u);
  y = pack16<T, P>(v);
}
// which elements a lane owns: vectors at e0 and e1; its pairs are pa on (the
// first half of them) and pb on, each half turning or not.  Interleaved pairs
// lie inside a vector, and a row's vectors go to its lanes in two rounds, so
// that an instruction copies neighbouring vectors (adjacent vectors a lane
// left half of every sector to a second copy: 240 us against 180).
struct Lane16 {
  int e0, e1, pa, pb;
  bool ta, tb;
};
template <int P, int LPR, bool INTER>
__device__ __forceinline__ Lane16 lane_of16(const RotArgs& a, int l) {
  Lane16 n;
  const int half = a.rot >> 1;
  if constexpr (INTER) {
    n.e0 = l * P;
    n.e1 = (l + LPR) * P;
    n.pa = n.e0 / 2;
    n.pb = n.e1 / 2;
  } else {
    n.pa = l * P;
    n.pb = n.pa + P / 2;
    n.e0 = n.pa < half ? n.pa : a.rot + (n.pa - half);
    n.e1 = n.e0 + (n.pa < half ? half : (a.dim - a.rot) >> 1);
  }
  n.ta = n.pa < half;
  n.tb = n.pb < half;
  return n;
}

// P floats of shared memory, 16-byte aligned
template <int P>
__device__ __forceinline__ void load_floats(const float* src, float* f) {
  if constexpr (P == 2) {
    const float2 v = *reinterpret_cast<const float2*>(src);
    f[0] = v.x, f[1] = v.y;
  }
#pragma unroll
  for (int i = 0; i < P / 4; ++i) {
    const float4 v = reinterpret_cast<const float4*>(src)[i];
    f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
  }
}
template <int P, bool INTER>
__device__ __forceinline__ void shared_weights(const float* w, const Lane16& ln, Pairs<P>& p) {
  float u[P], v[P];
  load_floats<P>(w + ln.e0, u);
  load_floats<P>(w + ln.e1, v);
  to_pairs<P, INTER>(u, v, p);
}

// a warp's place in its share: row group u of a part of token t
struct Place {
  unsigned task, t;
  int u, end;
  __device__ __forceinline__ void start(unsigned total, unsigned parts, int groups) {
    if (task >= total) return;
    t = task / parts;
    const int q = (int)(task - t * parts);
    u = groups * q / (int)parts;
    end = groups * (q + 1) / (int)parts;
  }
};

// Gradient: blocks below nq take tokens of q, the rest tokens of k, each warp
// every W-th (token, part of its heads), a fixed share; dw of a lane's
// elements stays in its registers, then lanes, warps and (in
// grad_weight_kernel) blocks are added in order.  Angles come with the rows
// of a token's first group, weights lie in shared memory.
//
// 32768 tokens of 32/8 heads of 128, bf16: 162 us, 6.2 TB/s (interleaved pairs
// as fast); float32, half the tokens: 177 us.  Tried: plain loads of 4 pairs a
// lane, two row groups in flight, three blocks an SM (286 us); this ring with
// 80 registers and three blocks (325 us: spills); a ring of 4 groups (166 us).
constexpr int kStreamWarps = 8;
constexpr int kRing = 3;  // row groups a warp has in flight, one being read

template <typename T, int LPR>
struct Stream {
  static constexpr int P = kPairs<T>, kDim = 2 * P * LPR;
  static constexpr int kVecs = 4;  // x0, x1, dy0, dy1
  // 16-byte units: rows [ring][vector][lane], angles [ring][cos, sin][dim / 2],
  // a warp each; then the weights, a block
  static constexpr int kRows = kRing * kVecs * 32, kAngles = kRing * (kDim / 4);
  static constexpr int kWarp = kRows + kAngles;
  static constexpr int kUnits = kStreamWarps * kWarp + kDim / 4;
  static_assert(kStreamWarps * kDim <= kStreamWarps * kWarp * 4, "dw sums alias the ring");
};

template <typename T, int LPR, bool INTER>
__global__ void __launch_bounds__(kStreamWarps * 32, 2)
    norm_rope_grad_kernel(const __grid_constant__ RotArgs a, int nq, int most_parts,
                          float* __restrict__ part) {
  using St = Stream<T, LPR>;
  constexpr int P = St::P, S = 32 / LPR, D = St::kDim;
  extern __shared__ uint4 smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* ring = smem + warp * St::kWarp + lane;
  const uint32_t ring_at = smem_u32(ring);
  float* ang = reinterpret_cast<float*>(smem + warp * St::kWarp + St::kRows);
  const uint32_t ang_at = smem_u32(ang);
  float* wsm = reinterpret_cast<float*>(smem + kStreamWarps * St::kWarp);
  const bool isk = (int)blockIdx.x >= nq;
  const Rows& rw = isk ? a.k : a.q;
  const int first = isk ? nq : 0;
  const unsigned step = (isk ? gridDim.x - nq : nq) * kStreamWarps;
  const Lane16 ln = lane_of16<P, LPR, INTER>(a, lane % LPR);
  const bool norm = rw.w != nullptr;
  const int half = a.rot >> 1;
  for (int e = threadIdx.x; e < D; e += blockDim.x)
    wsm[e] = norm ? load_weight(rw.w, a.wdtype, e) : 1.f;
  __syncthreads();

  Pairs<P> d;
#pragma unroll
  for (int i = 0; i < P / 2; ++i) d.a[i] = d.b[i] = both(0.f);
  const int groups = (rw.heads + S - 1) / S;
  // no part is empty: q and k have different numbers of groups
  const unsigned parts = most_parts < groups ? most_parts : groups;
  const unsigned total = (unsigned)a.tokens * parts;
  Place in{(unsigned)(blockIdx.x - first) * kStreamWarps + warp, 0, 0, 0};
  in.start(total, parts, groups);
  Place at = in;
  // the position of the token that `in` comes to next, read a task ahead
  int64_t pos = in.task < total ? a.positions[in.t] : 0;
  bool fresh = true;  // `in` is at a task's first group
  int in_slot = 0, in_ang = 0;
  auto copy = [&](uint32_t dst, const T* src) { cp_async16(dst, src, true); };
  auto issue = [&]() {
    if (in.task < total) {
      if (fresh) {
        const bool ok = pos >= 0 && pos < a.table_rows;
        if (!ok && lane == 0 && in.u == 0) report(a.status, CS_ST_POS_RANGE);
        for (int i = lane; i < half / 2; i += 32) {
          // units of 4 angles: half / 4 of cos, as many of sin
          const bool sn = i >= half / 4;
          const int e = 4 * (sn ? i - half / 4 : i), to = in_ang * D + (sn ? D / 2 : 0) + e;
          if (ok)
            cp_async16(ang_at + to * 4, (sn ? a.sin : a.cos) + pos * a.table_stride + e, true);
          else
            *reinterpret_cast<float4*>(ang + to) = make_float4(NAN, NAN, NAN, NAN);
        }
        const unsigned ahead = in.task + step;
        if (ahead < total) pos = a.positions[ahead / parts];
        in_ang = in_ang == kRing - 1 ? 0 : in_ang + 1;
        fresh = false;
      }
      const int h = in.u * S + lane / LPR;
      if (h < rw.heads) {
        const uint32_t to = ring_at + in_slot * (St::kVecs * 512);
        if (norm) {
          const T* x = reinterpret_cast<const T*>(rw.x + in.t * rw.xt + h * rw.xh);
          copy(to, x + ln.e0);
          copy(to + 512, x + ln.e1);
        }
        const T* dy = reinterpret_cast<const T*>(rw.dy + in.t * rw.yt + h * rw.yh);
        copy(to + 1024, dy + ln.e0);
        copy(to + 1536, dy + ln.e1);
      }
      if (++in.u == in.end) {
        in.task += step;
        in.start(total, parts, groups);
        fresh = true;
      }
    }
    cp_async_commit();
    in_slot = in_slot == kRing - 1 ? 0 : in_slot + 1;
  };
#pragma unroll
  for (int r = 0; r < kRing - 1; ++r) issue();

  int slot = 0, aslot = 0;
  while (at.task < total) {
    const float* cs = ang + aslot * D;
    aslot = aslot == kRing - 1 ? 0 : aslot + 1;
    for (; at.u < at.end; ++at.u) {
      cp_async_wait<kRing - 2>();
      __syncwarp();  // the angles are the warp's
      const uint4* mine = ring + slot * (St::kVecs * 32);
      slot = slot == kRing - 1 ? 0 : slot + 1;
      const int h = at.u * S + lane / LPR;
      const bool live = h < rw.heads;
      Pairs<P> g, n, w;
      load_pairs<T, P, INTER>(mine[64], mine[96], g);
      if (norm) load_pairs<T, P, INTER>(mine[0], mine[32], n);
      float cv[P], sv[P];
      auto turn_back = [&](int i, const float* cp, const float* sp) {
        const float2 c = make_float2(cp[2 * i], cp[2 * i + 1]);
        const float2 s = make_float2(sp[2 * i], sp[2 * i + 1]);
        const float2 t = __ffma2_rn(g.a[i], c, __fmul2_rn(g.b[i], s));
        g.b[i] = __ffma2_rn(g.b[i], c, neg(__fmul2_rn(g.a[i], s)));
        g.a[i] = t;
      };
      if constexpr (!INTER) {
        if (ln.ta) {
          load_floats<P>(cs + ln.pa, cv);
          load_floats<P>(cs + D / 2 + ln.pa, sv);
#pragma unroll
          for (int i = 0; i < P / 2; ++i) turn_back(i, cv, sv);
        }
      } else {
        if (ln.ta) {
          load_floats<P / 2>(cs + ln.pa, cv);
          load_floats<P / 2>(cs + D / 2 + ln.pa, sv);
#pragma unroll
          for (int i = 0; i < P / 4; ++i) turn_back(i, cv, sv);
        }
        if (ln.tb) {
          load_floats<P / 2>(cs + ln.pb, cv + P / 2);
          load_floats<P / 2>(cs + D / 2 + ln.pb, sv + P / 2);
#pragma unroll
          for (int i = P / 4; i < P / 2; ++i) turn_back(i, cv, sv);
        }
      }
      issue();  // into the slot read in the last round
      if (norm) {
        float2 ss = both(0.f), dot = both(0.f);
        shared_weights<P, INTER>(wsm, ln, w);
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
          w.a[i] = __fmul2_rn(w.a[i], g.a[i]);
          w.b[i] = __fmul2_rn(w.b[i], g.b[i]);
          ss = __ffma2_rn(n.a[i], n.a[i], ss);
          ss = __ffma2_rn(n.b[i], n.b[i], ss);
          dot = __ffma2_rn(w.a[i], n.a[i], dot);
          dot = __ffma2_rn(w.b[i], n.b[i], dot);
        }
        const float r = rsqrtf(row_sum<LPR>(ss.x + ss.y) * a.inv_dim + a.eps);
        // n is x r: dx = r (w g) - n (r mean(w g n))
        const float m = row_sum<LPR>(dot.x + dot.y) * r * a.inv_dim * r;
        const float2 rr = both(r), mm = both(-m);
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
          n.a[i] = __fmul2_rn(n.a[i], rr);
          n.b[i] = __fmul2_rn(n.b[i], rr);
          if (live) {
            d.a[i] = __ffma2_rn(g.a[i], n.a[i], d.a[i]);
            d.b[i] = __ffma2_rn(g.b[i], n.b[i], d.b[i]);
          }
          g.a[i] = __ffma2_rn(n.a[i], mm, __fmul2_rn(w.a[i], rr));
          g.b[i] = __ffma2_rn(n.b[i], mm, __fmul2_rn(w.b[i], rr));
        }
      }
      if (live) {
        uint4 y0, y1;
        store_pairs<T, P, INTER>(g, y0, y1);
        T* row = reinterpret_cast<T*>(rw.y + at.t * rw.yt + h * rw.yh);
        *reinterpret_cast<uint4*>(row + ln.e0) = y0;
        *reinterpret_cast<uint4*>(row + ln.e1) = y1;
      }
    }
    at.task += step;
    at.start(total, parts, groups);
  }
  cp_async_wait<0>();
  if (!norm) return;
  __syncthreads();  // the ring becomes the place of the block's sums
  float* acc = reinterpret_cast<float*>(smem);
  float d0[P], d1[P];
  from_pairs<P, INTER>(d, d0, d1);
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      d0[i] += __shfl_xor_sync(0xffffffffu, d0[i], o);
      d1[i] += __shfl_xor_sync(0xffffffffu, d1[i], o);
    }
    if (lane < LPR) {
      acc[warp * D + ln.e0 + i] = d0[i];
      acc[warp * D + ln.e1 + i] = d1[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kStreamWarps; ++w) s += acc[w * D + e];
    part[(int64_t)blockIdx.x * D + e] = s;
  }
}

__device__ __forceinline__ void store_weight(void* w, int dtype, int i, float x) {
  if (dtype == CS_F32) static_cast<float*>(w)[i] = x;
  else if (dtype == CS_F16) static_cast<__half*>(w)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(x);
}

// dw of 32 elements per block: 32 x 32 threads add the partials of blocks
// [0, nq) (q) or [nq, n) (k), each thread every 32nd, in a fixed order
__global__ void __launch_bounds__(1024)
    grad_weight_kernel(const float* __restrict__ part, int nq, int n, int dim, int wdtype,
                       void* qdw, void* kdw) {
  __shared__ float s[32][33];
  void* dw = blockIdx.y ? kdw : qdw;
  if (dw == nullptr) return;
  const int e = blockIdx.x * 32 + threadIdx.x;
  const int b1 = blockIdx.y ? n : nq;
  float x = 0.f;
  if (e < dim)
    for (int b = (blockIdx.y ? nq : 0) + threadIdx.y; b < b1; b += 32)
      x += part[(int64_t)b * dim + e];
  s[threadIdx.y][threadIdx.x] = x;
  __syncthreads();
  x = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int e2 = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && e2 < dim) store_weight(dw, wdtype, e2, x);
}

bool weight_ok(const cs_rotary_params* p) {
  if (!p->q_weight && !p->k_weight) return true;
  return p->weight_dtype == CS_F32 || p->weight_dtype == CS_F16 || p->weight_dtype == CS_BF16;
}

int make_args(const cs_rotary_params* p, RotArgs& a, bool need_k_out) {
  CS_HOST_CHECK(p != nullptr && p->tokens >= 0 && p->q_heads >= 0 && p->k_heads >= 0);
  CS_HOST_CHECK(p->head_dim > 0 && p->head_dim % 2 == 0 && p->rot >= 0 && p->rot % 2 == 0 &&
                p->rot <= p->head_dim && p->table_rows >= 0);
  CS_HOST_CHECK(p->eps >= 0.0 && weight_ok(p));
  if (p->head_dim > kMaxDim) return CS_ERR_UNSUPPORTED;
  if (p->dtype != CS_F32 && p->dtype != CS_F16 && p->dtype != CS_BF16) return CS_ERR_UNSUPPORTED;
  if (p->tokens > 0) {
    CS_HOST_CHECK(p->positions != nullptr && (p->rot == 0 || (p->cos && p->sin)));
    CS_HOST_CHECK(p->q_heads == 0 || (p->q && p->q_out));
    CS_HOST_CHECK(p->k_heads == 0 || (p->k && (p->k_out || !need_k_out)));
  }
  const int64_t es = dtype_size(p->dtype);
  a.q = Rows{static_cast<const char*>(p->q), nullptr, static_cast<char*>(p->q_out), p->q_weight,
             p->q_stride_tok * es, p->q_stride_head * es, p->qo_stride_tok * es,
             p->qo_stride_head * es, p->q_heads};
  a.k = Rows{static_cast<const char*>(p->k), nullptr, static_cast<char*>(p->k_out), p->k_weight,
             p->k_stride_tok * es, p->k_stride_head * es, p->ko_stride_tok * es,
             p->ko_stride_head * es, p->k_heads};
  a.cos = p->cos;
  a.sin = p->sin;
  a.table_rows = p->rot ? p->table_rows : INT64_MAX;
  a.table_stride = p->table_stride;
  a.positions = p->positions;
  a.tokens = p->tokens;
  a.dim = p->head_dim;
  a.rot = p->rot;
  a.interleaved = p->interleaved;
  a.wdtype = p->weight_dtype;
  a.eps = (float)p->eps;
  a.inv_dim = 1.f / (float)p->head_dim;
  a.status = p->status;
  return CS_OK;
}

// blocks of kRowWarps warp-rows, at most 16 an SM (the kernels loop)
unsigned row_blocks(int64_t rows) {
  const int64_t want = (rows + kRowWarps - 1) / kRowWarps, cap = (int64_t)num_sms() * 16;
  return (unsigned)(want < cap ? want : cap);
}

// Lanes a row for `pairs` pairs a lane, 0 where that does not fit: whole
// vectors of `pairs` elements in every part of a head, rows, tables and
// weights aligned to them, and fewer than 2^31 tasks.
int vec_lanes(const RotArgs& a, int dtype, int pairs, bool grad) {
  const int half = a.dim / 2, lanes = half / pairs;
  if (half % pairs || (a.rot / 2) % pairs || lanes > 32 || (lanes & (lanes - 1))) return 0;
  const int64_t unit = pairs * dtype_size(dtype);
  auto al = [](const void* x, int64_t t, int64_t h, int64_t unit) {
    return reinterpret_cast<uintptr_t>(x) % unit == 0 && t % unit == 0 && h % unit == 0;
  };
  for (const Rows* r : {&a.q, &a.k}) {
    if (r->heads == 0) continue;
    if (!al(r->x, r->xt, r->xh, unit) || !al(r->y, r->yt, r->yh, unit) || !al(r->w, 0, 0, 16))
      return 0;
    if (grad && !al(r->dy, r->yt, r->yh, unit)) return 0;
  }
  if (a.rot > 0 && (!al(a.cos, a.table_stride * 4, 0, 16) || !al(a.sin, 0, 0, 16))) return 0;
  const int64_t most = 2ll * (a.q.heads + a.k.heads) + 3;
  if (a.tokens > INT32_MAX / most) return 0;
  return lanes;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == CS_F32) f((float*)nullptr);
  else if (dtype == CS_F16) f((__half*)nullptr);
  else f((__nv_bfloat16*)nullptr);
  CS_LAUNCH_CHECK();
  return CS_OK;
}

template <typename F>
void by_lanes(int lanes, F f) {
  switch (lanes) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    case 4: return f(std::integral_constant<int, 4>());
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    default: return f(std::integral_constant<int, 32>());
  }
}

// The streamed kernel's blocks: in proportion to the kinds' row groups a token,
// with what a token's angles cost, no more than the rows fill; where the
// tokens alone do not fill them, a token's row groups go to several warps.
struct Shares {
  int nq, n, parts;
};
Shares shares(const RotArgs& a, int lanes) {
  auto groups = [&](int h) { return (h * lanes + 31) / 32; };
  const int gq = groups(a.q.heads), gk = groups(a.k.heads);
  const int64_t fill = (int64_t)kStreamBlocks * kStreamWarps;
  Shares s;
  s.parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::max(gq, gk), fill / a.tokens));
  const int64_t want = (a.tokens * s.parts + kStreamWarps - 1) / kStreamWarps;
  auto cost = [&](int g) { return g + kAngleCost * std::min(g, s.parts); };
  auto blocks = [&](int g) {
    if (g == 0) return 0;
    const double share = kStreamBlocks * cost(g) / (cost(gq) + cost(gk));
    return (int)std::min<int64_t>(std::max<int64_t>(1, (int64_t)share), want);
  };
  s.nq = blocks(gq);
  s.n = s.nq + blocks(gk);
  return s;
}

int launch_vec(const RotArgs& a, const AppendArgs* ap, int dtype, int lanes, cudaStream_t stream) {
  const int64_t tasks = a.tokens * (tasks_of(a.q.heads, lanes) +
                                    (ap ? 2 : 1) * tasks_of(a.k.heads, lanes));
  const unsigned blocks = (unsigned)((tasks + kVecWarps - 1) / kVecWarps);
  return by_type(dtype, [&](auto* ty) {
    using T = std::remove_pointer_t<decltype(ty)>;
    by_lanes(lanes, [&](auto l) {
      constexpr int L = decltype(l)::value;
      auto go = [&](auto inter, auto append) {
        norm_rope_vec_kernel<T, L, decltype(inter)::value, decltype(append)::value>
            <<<blocks, kVecWarps * 32, 0, stream>>>(a, ap ? *ap : AppendArgs{}, (unsigned)tasks);
      };
      if (a.interleaved && ap) go(std::true_type(), std::true_type());
      else if (a.interleaved) go(std::true_type(), std::false_type());
      else if (ap) go(std::false_type(), std::true_type());
      else go(std::false_type(), std::false_type());
    });
  });
}

}  // namespace
}  // namespace cs

extern "C" int cs_qk_norm_rope(const cs_rotary_params* p, void* stream) {
  using namespace cs;
  RotArgs a;
  if (int rc = make_args(p, a, true)) return rc;
  const int64_t rows = p->tokens * (p->q_heads + p->k_heads);
  if (rows == 0) return CS_OK;
  if (const int lanes = vec_lanes(a, p->dtype, kP, false))
    return launch_vec(a, nullptr, p->dtype, lanes, as_stream(stream));
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    norm_rope_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a);
  });
}

extern "C" int64_t cs_qk_norm_rope_grad_workspace(const cs_rotary_params* p) {
  if (p == nullptr || p->head_dim <= 0 || p->head_dim > cs::kMaxDim) return 0;
  return (int64_t)cs::kStreamBlocks * p->head_dim * (int64_t)sizeof(float);
}

extern "C" int cs_qk_norm_rope_grad(const cs_rotary_params* p, const void* q_dy, const void* k_dy,
                                    void* q_dw, void* k_dw, void* workspace, void* stream) {
  using namespace cs;
  RotArgs a;
  if (int rc = make_args(p, a, true)) return rc;
  const bool qw = p->q_weight != nullptr, kw = p->k_weight != nullptr;
  CS_HOST_CHECK((!qw || q_dw) && (!kw || k_dw) && ((!qw && !kw) || workspace));
  CS_HOST_CHECK(p->tokens == 0 || ((p->q_heads == 0 || q_dy) && (p->k_heads == 0 || k_dy)));
  a.q.dy = static_cast<const char*>(q_dy);
  a.k.dy = static_cast<const char*>(k_dy);
  if (p->tokens == 0) {  // no rows: the sums are empty
    if (qw || kw)
      grad_weight_kernel<<<dim3((p->head_dim + 31) / 32, 2), dim3(32, 32), 0, as_stream(stream)>>>(
          static_cast<const float*>(workspace), 0, 0, p->head_dim, p->weight_dtype,
          qw ? q_dw : nullptr, kw ? k_dw : nullptr);
    CS_LAUNCH_CHECK();
    return CS_OK;
  }
  float* part = static_cast<float*>(workspace);
  const int lanes = vec_lanes(a, p->dtype, 16 / dtype_size(p->dtype), true);
  int nq, n, rc;
  if (lanes) {
    const Shares s = shares(a, lanes);
    bool ready = true;
    nq = s.nq, n = s.n;
    rc = n == 0 ? CS_OK : by_type(p->dtype, [&](auto* ty) {
      using T = std::remove_pointer_t<decltype(ty)>;
      by_lanes(lanes, [&](auto l) {
        auto go = [&](auto inter) {
          constexpr int L = decltype(l)::value;
          constexpr auto kernel = norm_rope_grad_kernel<T, L, decltype(inter)::value>;
          constexpr int kBytes = Stream<T, L>::kUnits * 16;
          if (!allow_smem<kernel>(kBytes)) {
            ready = false;
            return;
          }
          kernel<<<s.n, kStreamWarps * 32, kBytes, as_stream(stream)>>>(a, s.nq, s.parts, part);
        };
        if (a.interleaved) go(std::true_type());
        else go(std::false_type());
      });
    });
    if (!ready) return CS_ERR_CUDA;
  } else {
    const int hq = p->q_heads, heads = hq + p->k_heads;
    auto share = [&](int h) {
      return h == 0 ? 0
                    : (int)std::min<int64_t>(std::max(1, (int)((int64_t)kStreamBlocks * h / heads)),
                                             (p->tokens * h + kRowWarps - 1) / kRowWarps);
    };
    nq = share(hq), n = nq + share(p->k_heads);
    rc = n == 0 ? CS_OK : by_type(p->dtype, [&](auto* ty) {
      using T = std::remove_pointer_t<decltype(ty)>;
      norm_rope_grad_rows_kernel<T><<<n, kRowWarps * 32, 0, as_stream(stream)>>>(a, nq, part);
    });
  }
  if (rc != CS_OK || (!qw && !kw)) return rc;
  grad_weight_kernel<<<dim3((p->head_dim + 31) / 32, 2), dim3(32, 32), 0, as_stream(stream)>>>(
      static_cast<const float*>(workspace), nq, n, p->head_dim, p->weight_dtype,
      qw ? q_dw : nullptr, kw ? k_dw : nullptr);
  CS_LAUNCH_CHECK();
  return CS_OK;
}

extern "C" int cs_kv_append_rotated(const cs_rotary_params* p, const cs_paged_kv* kv,
                                    const int64_t* slots, const void* v, int64_t v_stride_tok,
                                    int64_t v_stride_head, void* stream) {
  using namespace cs;
  RotArgs a;
  if (int rc = make_args(p, a, false)) return rc;
  CS_HOST_CHECK(kv != nullptr && kv->cache != nullptr && kv->dtype == p->dtype);
  CS_HOST_CHECK(kv->kv_heads == p->k_heads && kv->head_dim == p->head_dim && kv->block_size > 0);
  const int64_t rows = p->tokens * (p->q_heads + 2 * p->k_heads);
  if (rows == 0) return CS_OK;
  CS_HOST_CHECK(slots != nullptr && v != nullptr);
  const int64_t es = dtype_size(p->dtype);
  const Rows vr{static_cast<const char*>(v), nullptr, nullptr, nullptr, v_stride_tok * es,
                v_stride_head * es, 0, 0, p->k_heads};
  const PagedView pv = PagedView::make(*kv);
  if (pv.vec16() && reinterpret_cast<uintptr_t>(v) % (4 * es) == 0 && vr.xt % (4 * es) == 0 &&
      vr.xh % (4 * es) == 0) {
    RotArgs d = a;  // k has no dense output
    d.k.y = nullptr;
    d.k.yt = d.k.yh = 0;
    if (const int lanes = vec_lanes(d, p->dtype, kP, false)) {
      int shift = -1;
      for (int s = 0; s < 31; ++s)
        if ((int64_t)1 << s == kv->block_size) shift = s;
      const AppendArgs ap{pv, slots, vr, shift};
      return launch_vec(d, &ap, p->dtype, lanes, as_stream(stream));
    }
  }
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    append_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a, pv, slots,
                                                                                    vr);
  });
}
