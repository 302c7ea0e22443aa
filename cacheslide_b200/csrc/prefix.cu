// Attention of a batch behind shared prefixes (cs_prefix_plan,
// cs_prefix_attn): the host's plan of the batch and the CUDA-core kernel.
//
// Plan, int32 words:
//   tokens   [tokens][4]  prefix keys [p0, p1) and own keys [lo, hi) that the
//                         token sees, as places in the two slot arrays
#include <cstring>
#include <type_traits>

#include "common.cuh"

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
  int64_t tokens = 0, n_suffix = 0, n_prefix = 0, members = 0;
  for (int b = 0; b < s->requests; ++b) {
    CS_HOST_CHECK(s->query_lens[b] >= 0 && s->suffix_lens[b] >= 0);
    tokens += s->query_lens[b];
    n_suffix += s->suffix_lens[b];
    if (tokens > INT32_MAX / 8 || n_suffix > INT32_MAX / 2) return CS_ERR_UNSUPPORTED;
  }
  for (int g = 0; g < s->groups; ++g) {
    CS_HOST_CHECK(s->group_sizes[g] >= 0 && s->prefix_lens[g] >= 0);
    members += s->group_sizes[g];
    n_prefix += s->prefix_lens[g];
    if (n_prefix > INT32_MAX / 2 || members > s->requests) break;
  }
  if (n_prefix > INT32_MAX / 2) return CS_ERR_UNSUPPORTED;
  CS_HOST_CHECK(members == s->requests);
  std::memset(info, 0, sizeof(*info));
  info->tokens = tokens;
  info->n_prefix = n_prefix;
  info->n_suffix = n_suffix;
  info->words = tokens * 4;
  if (words == nullptr || capacity < info->words) return CS_ERR_TOO_LARGE;
  int32_t* w = words;
  int64_t b = 0, p0 = 0, k0 = 0;
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
    }
    p0 += s->prefix_lens[g];
  }
  return CS_OK;
}

extern "C" int cs_prefix_attn(const cs_prefix_params* p, const cs_prefix_plan_info* info,
                              const int32_t* plan, void* workspace, void* stream) {
  using namespace cs;
  CS_HOST_CHECK(p != nullptr && info != nullptr);
  const cs_paged_kv& kv = p->paged;
  CS_HOST_CHECK(kv.cache != nullptr && kv.block_size > 0 && kv.kv_heads > 0 && kv.head_dim > 0);
  CS_HOST_CHECK(p->q_heads > 0 && p->q_heads % kv.kv_heads == 0);
  if (kv.dtype != CS_F32 && kv.dtype != CS_F16 && kv.dtype != CS_BF16) return CS_ERR_UNSUPPORTED;
  if (kv.head_dim > kMaxDim) return CS_ERR_UNSUPPORTED;
  if (info->tokens == 0) return CS_OK;
  CS_HOST_CHECK(p->q && p->out && plan && (info->workspace == 0 || workspace));
  CS_HOST_CHECK((info->n_prefix == 0 || p->prefix_slots) &&
                (info->n_suffix == 0 || p->suffix_slots));
  const int64_t es = dtype_size(kv.dtype);
  RowArgs a{static_cast<const char*>(p->q), p->q_stride_tok * es, p->q_stride_head * es,
            PagedView::make(kv), p->prefix_slots, p->suffix_slots,
            reinterpret_cast<const int4*>(plan), p->q_heads, (int)(p->q_heads / kv.kv_heads),
            (int)kv.head_dim, (float)p->scale, static_cast<char*>(p->out), p->o_stride_tok * es,
            p->o_stride_head * es, p->lse, p->status};
  const unsigned blocks = (unsigned)(info->tokens * p->q_heads);
  if (info->tokens * p->q_heads > INT32_MAX) return CS_ERR_UNSUPPORTED;
  if (kv.dtype == CS_F32)
    prefix_rows_kernel<float><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  else if (kv.dtype == CS_F16)
    prefix_rows_kernel<__half><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  else
    prefix_rows_kernel<__nv_bfloat16><<<blocks, kRowWarps * 32, 0, as_stream(stream)>>>(a);
  CS_LAUNCH_CHECK();
  return CS_OK;
}
