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
#include "common.cuh"

namespace cs {
namespace {

constexpr int kMaxDim = 512;
constexpr int kMaxPairs = kMaxDim / 2 / 32;  // pairs a lane of a warp-per-row kernel
constexpr int kGradBlocks = 592;             // 148 SMs x 4: the fixed partition of dw
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
      *at(i) = Elem<T>::from_f(p0 * c - p1 * s);
      *at(j) = Elem<T>::from_f(p1 * c + p0 * s);
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

// Gradient, one warp per row; blockIdx.y picks q or k.  Each warp keeps dw of
// its rows in registers, the block adds its warps in order, and the partial
// of block b goes to part[(y * kGradBlocks + b) * dim].
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32)
    norm_rope_grad_rows_kernel(RotArgs a, float* __restrict__ part) {
  __shared__ float acc[kRowWarps][kMaxDim];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Rows& rw = blockIdx.y ? a.k : a.q;
  const int pairs = a.dim >> 1;
  float d0[kMaxPairs], d1[kMaxPairs];
#pragma unroll
  for (int m = 0; m < kMaxPairs; ++m) d0[m] = d1[m] = 0.f;
  const int64_t total = a.tokens * rw.heads;
  for (int64_t row = blockIdx.x * (int64_t)kRowWarps + warp; row < total;
       row += (int64_t)gridDim.x * kRowWarps) {
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
        g0[m] = y0 * c + y1 * s;
        g1[m] = y1 * c - y0 * s;
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
    part[((int64_t)blockIdx.y * kGradBlocks + blockIdx.x) * a.dim + e] = s;
  }
}

__device__ __forceinline__ void store_weight(void* w, int dtype, int i, float x) {
  if (dtype == CS_F32) static_cast<float*>(w)[i] = x;
  else if (dtype == CS_F16) static_cast<__half*>(w)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(x);
}

// dw of one element per block, the partials added in a fixed order
__global__ void __launch_bounds__(256)
    grad_weight_kernel(const float* __restrict__ part, int blocks, int dim, int wdtype, void* qdw,
                       void* kdw) {
  __shared__ float s[8];
  void* dw = blockIdx.y ? kdw : qdw;
  if (dw == nullptr) return;
  const float* p = part + (int64_t)blockIdx.y * kGradBlocks * dim + blockIdx.x;
  float x = 0.f;
  for (int b = threadIdx.x; b < blocks; b += 256) x += p[(int64_t)b * dim];
  x = warp_sum(x);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) x += s[w];
    store_weight(dw, wdtype, blockIdx.x, x);
  }
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

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == CS_F32) f((float*)nullptr);
  else if (dtype == CS_F16) f((__half*)nullptr);
  else f((__nv_bfloat16*)nullptr);
  CS_LAUNCH_CHECK();
  return CS_OK;
}

}  // namespace
}  // namespace cs

extern "C" int cs_qk_norm_rope(const cs_rotary_params* p, void* stream) {
  using namespace cs;
  RotArgs a;
  if (int rc = make_args(p, a, true)) return rc;
  const int64_t rows = p->tokens * (p->q_heads + p->k_heads);
  if (rows == 0) return CS_OK;
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    norm_rope_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a);
  });
}

extern "C" int64_t cs_qk_norm_rope_grad_workspace(const cs_rotary_params* p) {
  if (p == nullptr || p->head_dim <= 0 || p->head_dim > cs::kMaxDim) return 0;
  return 2ll * cs::kGradBlocks * p->head_dim * (int64_t)sizeof(float);
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
  const int64_t rows = p->tokens * (p->q_heads > p->k_heads ? p->q_heads : p->k_heads);
  const int64_t want = (rows + kRowWarps - 1) / kRowWarps;
  const unsigned blocks = (unsigned)(want < kGradBlocks ? (want > 0 ? want : 1) : kGradBlocks);
  const int rc = by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    norm_rope_grad_rows_kernel<T><<<dim3(blocks, 2), kRowWarps * 32, 0, as_stream(stream)>>>(
        a, static_cast<float*>(workspace));
  });
  if (rc != CS_OK || (!qw && !kw)) return rc;
  grad_weight_kernel<<<dim3(p->head_dim, 2), 256, 0, as_stream(stream)>>>(
      static_cast<const float*>(workspace), (int)blocks, p->head_dim, p->weight_dtype,
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
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    append_rows_kernel<T><<<row_blocks(rows), kRowWarps * 32, 0, as_stream(stream)>>>(a, pv, slots,
                                                                                    vr);
  });
}
