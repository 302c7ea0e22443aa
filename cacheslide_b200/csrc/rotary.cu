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
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace cs {
namespace {

constexpr int kMaxDim = 512;
constexpr int kMaxPairs = kMaxDim / 2 / 32;  // pairs a lane of a warp-per-row kernel
constexpr int kGradBlocks = 740;             // 148 SMs x 5: the fixed partition of dw
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

__device__ __forceinline__ void angle(const RotArgs& a, int64_t pos, int p, float& c, float& s) {
  c = 1.f;
  s = 0.f;
  if (p < (a.rot >> 1)) {
    const bool ok = pos >= 0 && pos < a.table_rows;
    c = ok ? a.cos[pos * a.table_stride + p] : __int_as_float(0x7fc00000);
    s = ok ? a.sin[pos * a.table_stride + p] : __int_as_float(0x7fc00000);
  }
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
      float c, s;
      pair_elems(a, p, i, j);
      angle(a, pos, p, c, s);
      float p0 = u[m], p1 = v[m];
      if (w) {
        p0 *= r * load_weight(w, a.wdtype, i);
        p1 *= r * load_weight(w, a.wdtype, j);
      }
      *at(i) = Elem<T>::from_f(turned0(p0, p1, c, s));
      *at(j) = Elem<T>::from_f(turned1(p0, p1, c, s));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) norm_rope_rows_kernel(RotArgs a) {
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
// (copied into its V half).
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
        float c, s;
        pair_elems(a, p, i, j);
        angle(a, pos, p, c, s);
        const float y0 = Elem<T>::to_f(dy[i]), y1 = Elem<T>::to_f(dy[j]);
        g0[m] = turned0(y0, y1, c, -s);
        g1[m] = turned1(y0, y1, c, -s);
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
// LPR lanes own a row, each two 16-byte vectors of it (P pairs of elements):
// half-split pairs take one vector of either half, interleaved pairs lie
// inside the vectors.  A warp takes 32 / LPR rows at once and U such groups
// back to back, all loads before the first arithmetic, so that a thread has
// 2 U vectors in flight; rows are flattened over (token, head).
template <typename T> constexpr int kVecPairs = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) w[i] = __float_as_uint(f[i]);
    else w[i] = Pack2<T>::pack(f[2 * i], f[2 * i + 1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// the P weights at element e of a head (16-byte aligned), as float32
template <typename T, int P>
__device__ __forceinline__ void weights_at(const void* w, int dtype, int e, float* f) {
  if (dtype == CS_F32) {
#pragma unroll
    for (int i = 0; i < P / 4; ++i)
      unpack<float>(__ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + e) + i),
                    f + 4 * i);
  } else if constexpr (P == 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + e));
    if (dtype == CS_F16) unpack<__half>(v, f);
    else unpack<__nv_bfloat16>(v, f);
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + e));
    float g[8];
    if (dtype == CS_F16) unpack<__half>(make_uint4(v.x, v.y, 0u, 0u), g);
    else unpack<__nv_bfloat16>(make_uint4(v.x, v.y, 0u, 0u), g);
#pragma unroll
    for (int i = 0; i < P; ++i) f[i] = g[i];
  }
}

// which elements a lane owns: vectors at e0 and e1; pairs p0 .. p0 + P - 1
// when they turn
struct Lane {
  int p0, e0, e1;
  bool turns;
};
template <int P>
__device__ __forceinline__ Lane lane_of(const RotArgs& a, int l) {
  Lane n;
  n.p0 = l * P;
  const int half = a.rot >> 1;
  n.turns = n.p0 < half;
  if (n.turns) {
    n.e0 = a.interleaved ? 2 * n.p0 : n.p0;
    n.e1 = a.interleaved ? n.e0 + P : n.p0 + half;
  } else {
    n.e0 = a.rot + (n.p0 - half);
    n.e1 = n.e0 + ((a.dim - a.rot) >> 1);
  }
  return n;
}

template <int P>
__device__ __forceinline__ void angles(const RotArgs& a, int64_t pos, int p0, float* c, float* s) {
  if (pos >= 0 && pos < a.table_rows) {
    const float4* cr = reinterpret_cast<const float4*>(a.cos + pos * a.table_stride + p0);
    const float4* sr = reinterpret_cast<const float4*>(a.sin + pos * a.table_stride + p0);
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      const float4 x = __ldg(cr + i), y = __ldg(sr + i);
      c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
      s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
  }
}

// (x0, x1): a lane's two vectors, turned by +angle (sign 1) or -angle (-1)
template <int P>
__device__ __forceinline__ void turn(float* x0, float* x1, const float* c, const float* s,
                                     bool interleaved, float sign) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      float a = x0[2 * i], b = x0[2 * i + 1], t = sign * s[i];
      x0[2 * i] = turned0(a, b, c[i], t);
      x0[2 * i + 1] = turned1(a, b, c[i], t);
      a = x1[2 * i], b = x1[2 * i + 1], t = sign * s[P / 2 + i];
      x1[2 * i] = turned0(a, b, c[P / 2 + i], t);
      x1[2 * i + 1] = turned1(a, b, c[P / 2 + i], t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float a = x0[i], b = x1[i], t = sign * s[i];
      x0[i] = turned0(a, b, c[i], t);
      x1[i] = turned1(a, b, c[i], t);
    }
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

// Forward and append: rows of q, then k, then (append) v of each token.
template <typename T, int LPR, int U>
__global__ void __launch_bounds__(256)
    norm_rope_vec_kernel(const RotArgs a, const AppendArgs ap) {
  constexpr int P = kVecPairs<T>, S = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int heads = a.q.heads + a.k.heads + (ap.slots ? a.k.heads : 0);
  const int64_t total = a.tokens * heads;
  const int64_t base = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * (S * U) + lane / LPR;
  if (base - lane / LPR >= total) return;
  const Lane ln = lane_of<P>(a, lane % LPR);
  int64_t t = base / heads;
  int h = (int)(base - t * heads);
  uint4 x0[U], x1[U];
  char* dst[U];
  int kind[U];  // 0: no row, 1: norm and turn, 2: copy
  int64_t pos[U];
  const void* wp[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    kind[u] = 0;
    wp[u] = nullptr;
    if (base + u * S < total) {
      int hh = h;
      const Rows* rw = &a.q;
      kind[u] = 1;
      if (hh >= a.q.heads) {
        hh -= a.q.heads;
        rw = &a.k;
        if (hh >= a.k.heads) {
          hh -= a.k.heads;
          rw = &ap.v;
          kind[u] = 2;
        }
      }
      const T* x = reinterpret_cast<const T*>(rw->x + t * rw->xt + hh * rw->xh);
      x0[u] = *reinterpret_cast<const uint4*>(x + ln.e0);
      x1[u] = *reinterpret_cast<const uint4*>(x + ln.e1);
      wp[u] = rw->w;
      pos[u] = a.positions[t];
      dst[u] = rw->y + t * rw->yt + hh * rw->yh;
      const bool pos_ok = pos[u] >= 0 && pos[u] < a.table_rows;
      if (!pos_ok && lane % LPR == 0) report(a.status, CS_ST_POS_RANGE);
      if (ap.slots && h >= a.q.heads) {
        const int64_t slot = ap.slots[t];
        if (!ap.pv.valid(slot) || !pos_ok) {
          if (slot != -1 && !ap.pv.valid(slot) && lane % LPR == 0)
            report(a.status, CS_ST_SLOT_RANGE);
          dst[u] = nullptr;
        } else if (slot < ap.pv.native_total && ap.bs_shift >= 0) {
          const int64_t b = slot >> ap.bs_shift, o = slot - (b << ap.bs_shift);
          dst[u] = ap.pv.cache + b * ap.pv.sb + hh * ap.pv.sh + o * ap.pv.so +
                   (kind[u] == 2 ? a.dim * (int)sizeof(T) : 0);
        } else {
          dst[u] = ap.pv.addr(slot, hh, kind[u] == 2 ? a.dim : 0);
        }
      }
    }
    h += S;
    while (h >= heads) {
      h -= heads;
      ++t;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // every lane takes part in the row sums
    float f0[P], f1[P];
    float ss = 0.f;
    if (kind[u] == 1) {
      unpack<T>(x0[u], f0);
      unpack<T>(x1[u], f1);
#pragma unroll
      for (int i = 0; i < P; ++i) ss += f0[i] * f0[i] + f1[i] * f1[i];
    }
    ss = row_sum<LPR>(ss);
    if (kind[u] == 0) continue;
    if (kind[u] == 1) {
      if (wp[u]) {
        const float r = rsqrtf(ss * a.inv_dim + a.eps);
        float w[P];
        weights_at<T, P>(wp[u], a.wdtype, ln.e0, w);
#pragma unroll
        for (int i = 0; i < P; ++i) f0[i] *= r * w[i];
        weights_at<T, P>(wp[u], a.wdtype, ln.e1, w);
#pragma unroll
        for (int i = 0; i < P; ++i) f1[i] *= r * w[i];
      }
      if (ln.turns) {
        float c[P], s[P];
        angles<P>(a, pos[u], ln.p0, c, s);
        turn<P>(f0, f1, c, s, a.interleaved, 1.f);
      }
      x0[u] = pack<T>(f0);
      x1[u] = pack<T>(f1);
    }
    if (dst[u] == nullptr) continue;
    T* y = reinterpret_cast<T*>(dst[u]);
    *reinterpret_cast<uint4*>(y + ln.e0) = x0[u];
    *reinterpret_cast<uint4*>(y + ln.e1) = x1[u];
  }
}

// Gradient: blocks below nq take rows of q, the rest rows of k, each a fixed
// share whatever the count; dw of a lane's elements stays in its registers,
// then lanes, warps and (in grad_weight_kernel) blocks are added in order.
template <typename T, int LPR>
__global__ void __launch_bounds__(256)
    norm_rope_grad_vec_kernel(const RotArgs a, int nq, float* __restrict__ part) {
  constexpr int P = kVecPairs<T>, S = 32 / LPR;
  __shared__ float acc[8][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool isk = (int)blockIdx.x >= nq;
  const Rows& rw = isk ? a.k : a.q;
  const int b = isk ? blockIdx.x - nq : blockIdx.x;
  const int blocks = isk ? gridDim.x - nq : nq;
  const Lane ln = lane_of<P>(a, lane % LPR);
  float w0[P], w1[P], d0[P], d1[P];
#pragma unroll
  for (int i = 0; i < P; ++i) w0[i] = w1[i] = d0[i] = d1[i] = 0.f;
  if (rw.w) {
    weights_at<T, P>(rw.w, a.wdtype, ln.e0, w0);
    weights_at<T, P>(rw.w, a.wdtype, ln.e1, w1);
  }
  const int64_t total = a.tokens * rw.heads;
  const int64_t step = (int64_t)blocks * 8 * S;
  for (int64_t first = ((int64_t)b * 8 + warp) * S; first < total; first += step) {
    const int64_t row = first + lane / LPR;
    const bool live = row < total;
    float g0[P], g1[P], n0[P], n1[P];
    float ss = 0.f, dot = 0.f;
    T* dx = nullptr;
    if (live) {
      const int64_t t = row / rw.heads;
      const int h = (int)(row - t * rw.heads);
      const int64_t pos = a.positions[t];
      const T* dy = reinterpret_cast<const T*>(rw.dy + t * rw.yt + h * rw.yh);
      dx = reinterpret_cast<T*>(rw.y + t * rw.yt + h * rw.yh);
      const uint4 y0 = *reinterpret_cast<const uint4*>(dy + ln.e0);
      const uint4 y1 = *reinterpret_cast<const uint4*>(dy + ln.e1);
      uint4 x0, x1;
      if (rw.w) {
        const T* x = reinterpret_cast<const T*>(rw.x + t * rw.xt + h * rw.xh);
        x0 = *reinterpret_cast<const uint4*>(x + ln.e0);
        x1 = *reinterpret_cast<const uint4*>(x + ln.e1);
      }
      if (lane % LPR == 0 && (pos < 0 || pos >= a.table_rows)) report(a.status, CS_ST_POS_RANGE);
      unpack<T>(y0, g0);
      unpack<T>(y1, g1);
      if (ln.turns) {
        float c[P], s[P];
        angles<P>(a, pos, ln.p0, c, s);
        turn<P>(g0, g1, c, s, a.interleaved, -1.f);
      }
      if (rw.w) {
        unpack<T>(x0, n0);
        unpack<T>(x1, n1);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          ss += n0[i] * n0[i] + n1[i] * n1[i];
          dot += w0[i] * g0[i] * n0[i] + w1[i] * g1[i] * n1[i];
        }
      }
    }
    if (rw.w) {
      ss = row_sum<LPR>(ss);
      dot = row_sum<LPR>(dot);
      if (live) {
        const float r = rsqrtf(ss * a.inv_dim + a.eps);
        const float mean = dot * r * a.inv_dim;  // mean(w g n)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float u = n0[i] * r, v = n1[i] * r;
          d0[i] += g0[i] * u;
          d1[i] += g1[i] * v;
          g0[i] = r * (w0[i] * g0[i] - u * mean);
          g1[i] = r * (w1[i] * g1[i] - v * mean);
        }
      }
    }
    if (live) {
      *reinterpret_cast<uint4*>(dx + ln.e0) = pack<T>(g0);
      *reinterpret_cast<uint4*>(dx + ln.e1) = pack<T>(g1);
    }
  }
  if (!rw.w) return;
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      d0[i] += __shfl_xor_sync(0xffffffffu, d0[i], o);
      d1[i] += __shfl_xor_sync(0xffffffffu, d1[i], o);
    }
    if (lane < LPR) {
      acc[warp][ln.e0 + i] = d0[i];
      acc[warp][ln.e1 + i] = d1[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.dim; e += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += acc[w][e];
    part[(int64_t)blockIdx.x * a.dim + e] = s;
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

// Lanes a row of the vector kernels, 0 where they do not fit: whole vectors
// in every part of a head, and 16-byte aligned rows, tables and weights.
int vec_lanes(const RotArgs& a, int dtype, bool grad) {
  const int P = 16 / dtype_size(dtype), half = a.dim / 2;
  const int lanes = half / P;
  if (half % P || (a.rot / 2) % P || lanes > 32 || (lanes & (lanes - 1))) return 0;
  auto al = [](const void* x, int64_t t, int64_t h) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && t % 16 == 0 && h % 16 == 0;
  };
  for (const Rows* r : {&a.q, &a.k}) {
    if (r->heads == 0) continue;
    if (!al(r->x, r->xt, r->xh) || !al(r->y, r->yt, r->yh) || !al(r->w, 0, 0)) return 0;
    if (grad && !al(r->dy, r->yt, r->yh)) return 0;
  }
  if (a.rot > 0 && (!al(a.cos, a.table_stride * 4, 0) || !al(a.sin, 0, 0))) return 0;
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

int launch_vec(const RotArgs& a, const AppendArgs& ap, int64_t rows, int dtype, int lanes,
               cudaStream_t stream) {
  return by_type(dtype, [&](auto* ty) {
    using T = std::remove_pointer_t<decltype(ty)>;
    by_lanes(lanes, [&](auto l) {
      constexpr int LPR = decltype(l)::value;
      // one group of rows a warp while that leaves SMs idle, four when not
      const int64_t per = 8 * (32 / LPR);
      const int64_t one = (rows + per - 1) / per;
      if (one <= 4ll * num_sms())
        norm_rope_vec_kernel<T, LPR, 1><<<(unsigned)one, 256, 0, stream>>>(a, ap);
      else
        norm_rope_vec_kernel<T, LPR, 4>
            <<<(unsigned)((rows + 4 * per - 1) / (4 * per)), 256, 0, stream>>>(a, ap);
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
  if (const int lanes = vec_lanes(a, p->dtype, false))
    return launch_vec(a, AppendArgs{}, rows, p->dtype, lanes, as_stream(stream));
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    norm_rope_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a);
  });
}

extern "C" int64_t cs_qk_norm_rope_grad_workspace(const cs_rotary_params* p) {
  if (p == nullptr || p->head_dim <= 0 || p->head_dim > cs::kMaxDim) return 0;
  return (cs::kGradBlocks + 1ll) * p->head_dim * (int64_t)sizeof(float);
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
  // blocks in proportion to the heads, no more than the rows fill
  const int heads = p->q_heads + p->k_heads;
  const int lanes = vec_lanes(a, p->dtype, true);
  const int64_t per = lanes ? 8 * (32 / lanes) : kRowWarps;
  auto share = [&](int h) {
    const int64_t most = heads ? ((int64_t)kGradBlocks * h + heads - 1) / heads : 0;
    const int64_t want = (p->tokens * h + per - 1) / per;
    return (int)std::max<int64_t>(1, std::min(most, want));
  };
  const int nq = share(p->q_heads), n = nq + share(p->k_heads);
  const int rc = by_type(p->dtype, [&](auto* ty) {
    using T = std::remove_pointer_t<decltype(ty)>;
    float* part = static_cast<float*>(workspace);
    if (lanes)
      by_lanes(lanes, [&](auto l) {
        norm_rope_grad_vec_kernel<T, decltype(l)::value>
            <<<n, 256, 0, as_stream(stream)>>>(a, nq, part);
      });
    else
      norm_rope_grad_rows_kernel<T><<<n, kRowWarps * 32, 0, as_stream(stream)>>>(a, nq, part);
  });
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
  if (pv.vec16() && reinterpret_cast<uintptr_t>(v) % 16 == 0 && vr.xt % 16 == 0 &&
      vr.xh % 16 == 0) {
    RotArgs d = a;  // k has no dense output
    d.k.y = nullptr;
    d.k.yt = d.k.yh = 0;
    if (const int lanes = vec_lanes(d, p->dtype, false)) {
      int shift = -1;
      for (int s = 0; s < 31; ++s)
        if ((int64_t)1 << s == kv->block_size) shift = s;
      return launch_vec(d, AppendArgs{pv, slots, vr, shift}, rows, p->dtype, lanes,
                        as_stream(stream));
    }
  }
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    append_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a, pv, slots,
                                                                                    vr);
  });
}
