// Rows into the 4-bit pool and back.
//
//   scale = (max x - min x) / 15,  code = (x - min x) / scale to the nearest
//
// A lane holds 8 neighbouring elements of a row (one 16-byte load), a row is 16
// or 8 lanes, and a group's extremes are two to four shuffles of packed pairs.
// Its codes are one 32-bit word of the key row, or two half-words of the value
// row, which lanes of neighbouring half-words trade so that each stores one
// word.  Rows of D = 128 in groups of 64 move 512 + 144 bytes a (token, head);
// both are bound by their instructions before HBM: 65536 tokens of 8 heads in
// groups of 128 (52 us at HBM's rate each way) take 108 us in, at 85 % of the
// issue slots (139 with a second look at doubtful codes and two rows a warp), and
// 74 us out.
//
// A code is decided by the quotient, in infinite precision, of the float32
// difference x - min x: that is either half way between two codes or 2^-16 of
// itself from there (scales have 11 bits).  The difference of two numbers of the
// type is mostly exact in float32; one that is not can lie on a half way that the
// exact one misses (-832 and 2^-24 at a scale of 128: 6, not 7).
#include <math.h>

#include <type_traits>

#include "kv4.cuh"
#include "kv4_attn.cuh"
#include "sm100.cuh"

namespace cs {
namespace {

constexpr int kRowThreads = 256;

struct Rows4 {
  char* x;
  int64_t st, sh;  // byte strides of tokens and heads
};

// A block takes a head of 16 (D = 64: 32) neighbouring tokens, whose records are
// mostly neighbours too: their stores then fill whole lines.  (Blocks of two
// tokens' eight heads took 139 us for 65536 tokens of 8 heads of 128.)
struct Row4 {
  int64_t token;
  int head;
};
template <int L>
__device__ __forceinline__ Row4 row_of(int hkv) {
  const unsigned group = blockIdx.x / (unsigned)hkv;
  return Row4{(int64_t)group * (kRowThreads / L) + threadIdx.x / L,
              (int)(blockIdx.x - group * (unsigned)hkv)};
}

template <typename T> __device__ __forceinline__ float overflow_of();  // rounds to infinity
template <> __device__ __forceinline__ float overflow_of<__half>() { return 65520.f; }
template <> __device__ __forceinline__ float overflow_of<__nv_bfloat16>() {
  return __uint_as_float(0x7f7f8000u);
}
template <typename T> __device__ __forceinline__ uint32_t bits_of(float x) {
  const T y = Elem<T>::from_f(x);
  return *reinterpret_cast<const uint16_t*>(&y);
}
template <typename T> __device__ __forceinline__ float of_bits(uint32_t b) {
  return pair_of<T>(b & 0xffffu).x;
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// eight elements' codes (element i in bits 4 i ..) and their group's (scale, low)
template <typename T, int LANES>
__device__ __forceinline__ uint32_t encode(const uint32_t (&x)[4], uint32_t& pair) {
  // the extremes as a pair (least, -most), NaN if any element is
  uint32_t least, most;
  {
    const auto a = __hmin2_nan(__hmin2_nan(as_pair<T>(x[0]), as_pair<T>(x[1])),
                               __hmin2_nan(as_pair<T>(x[2]), as_pair<T>(x[3])));
    const auto b = __hmax2_nan(__hmax2_nan(as_pair<T>(x[0]), as_pair<T>(x[1])),
                               __hmax2_nan(as_pair<T>(x[2]), as_pair<T>(x[3])));
    least = pair_bits(a), most = pair_bits(b) ^ 0x80008000u;
  }
  uint32_t ends = pair_bits(__hmin2_nan(as_pair<T>(__byte_perm(least, most, 0x5410u)),
                                        as_pair<T>(__byte_perm(least, most, 0x7632u))));
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1)
    ends = pair_bits(__hmin2_nan(as_pair<T>(ends), as_pair<T>(__shfl_xor_sync(~0u, ends, o))));
  const float2 end = pair_of<T>(ends ^ 0x80000000u);
  const float lo = end.x, hi = end.y;
  // a sixteenth of the range, which cannot overflow
  const float range = fabsf(hi * 0.0625f - lo * 0.0625f);  // (no zero with a sign)
  if (!(range < INFINITY)) {
    pair = 0x7fff7fffu;  // NaN in both types
    return 0u;
  }
  // range / 0.9375, rounded to nearest: the product with the rounded reciprocal,
  // corrected once by its exact remainder (Markstein 1990)
  constexpr float kRecip = 16.f / 15.f;
  const float near = range * kRecip;
  uint32_t sb = bits_of<T>(fmaf(fmaf(-0.9375f, near, range), kRecip, near));
  float s = of_bits<T>(sb);
  if (!(fmaf(15.f, s, lo) < overflow_of<T>())) s = of_bits<T>(--sb);
  pair = sb | (lo == 0.f ? 0u : ends << 16);  // (a zero without a sign)
  if (sb == 0) return 0u;
  // both scaled by a power of two, so that 1 / s and the differences are finite
  const float up = s < 0x1p-60f ? 0x1p60f : 0x1p-4f;
  const float su = s * up, lu = lo * up, inv = rcp_approx(su);
  // Quotients, corrected once by their exact remainders: a quotient that lies
  // half way between two codes then comes out exactly (and goes to the even one),
  // and none other is as near to a half way as its error.  Four codes become one
  // number of 16 bits.
  constexpr float kWhole = 0x1.8p23f;
  const bool over = (hi * up - lu) * inv > 15.4f;  // a scale of few bits: codes over 15
  float2 c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 d = __ffma2_rn(pair_of<T>(x[i]), both(up), both(-lu));
    const float2 f = __fmul2_rn(d, both(inv));
    c[i] = __ffma2_rn(__ffma2_rn(f, both(-su), d), both(inv), f);
    if (over) c[i] = make_float2(fminf(c[i].x, 15.f), fminf(c[i].y, 15.f));
    c[i] = __fadd2_rn(__fadd2_rn(c[i], both(kWhole)), both(-kWhole));
  }
  const float low4 = fmaf(c[1].y, 4096.f, fmaf(c[1].x, 256.f, fmaf(c[0].y, 16.f, c[0].x)));
  const float high4 = fmaf(c[3].y, 4096.f, fmaf(c[3].x, 256.f, fmaf(c[2].y, 16.f, c[2].x)));
  return __byte_perm(__float_as_uint(low4 + kWhole), __float_as_uint(high4 + kWhole), 0x5410u);
}

// a pair of codes, in bits 0 .. 3 and 16 .. 19, as numbers (exact)
template <typename T> __device__ __forceinline__ pair16<T> whole_pair(uint32_t x);
template <> __device__ __forceinline__ __half2 whole_pair<__half>(uint32_t x) {
  return __hsub2(as_pair<__half>(x | 0x64006400u), as_pair<__half>(0x64006400u));  // 1024
}
template <> __device__ __forceinline__ __nv_bfloat162 whole_pair<__nv_bfloat16>(uint32_t x) {
  return __hsub2(as_pair<__nv_bfloat16>(x | 0x43004300u),
                 as_pair<__nv_bfloat16>(0x43004300u));  // 128
}

// eight codes as low + scale code, rounded once
template <typename T>
__device__ __forceinline__ uint4 decode(uint32_t code, uint32_t pair) {
  const pair16<T> scale = as_pair<T>(__byte_perm(pair, 0u, 0x1010u)),
                  low = as_pair<T>(__byte_perm(pair, 0u, 0x3232u));
  uint32_t y[4];  // elements (i, i + 4)
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = pair_bits(__hfma2(whole_pair<T>(code >> (4 * i) & 0x000f000fu), scale, low));
  return make_uint4(__byte_perm(y[0], y[1], 0x5410u), __byte_perm(y[2], y[3], 0x5410u),
                    __byte_perm(y[0], y[1], 0x7632u), __byte_perm(y[2], y[3], 0x7632u));
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kRowThreads)
    kv4_append_kernel(const Pool4 pool, const int64_t* slots, int64_t n, const Rows4 k,
                      const Rows4 v, int vec, int32_t* status) {
  using U = Unit4<D, NG>;
  constexpr int L = D / 8, LG = L / NG, W = U::W;  // lanes a row and a group
  const Row4 w4 = row_of<L>(pool.hkv);
  const int64_t token = w4.token;
  const int head = w4.head, lane = threadIdx.x % L;
  const bool in = token < n;
  const int64_t slot = in ? slots[token] : -1;
  const bool live = pool.valid(slot);
  if (in && !live && slot != -1 && lane == 0 && head == 0) report(status, CS_ST_SLOT_RANGE);
  uint32_t x[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const Rows4& r = h ? v : k;
    const char* p = r.x + token * r.st + head * r.sh + lane * 16;
    if (!live) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[h][i] = 0u;
    } else if (vec) {
      const uint4 y = *reinterpret_cast<const uint4*>(p);
      x[h][0] = y.x, x[h][1] = y.y, x[h][2] = y.z, x[h][3] = y.w;
    } else {
      const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[h][i] = e[2 * i] | (uint32_t)e[2 * i + 1] << 16;
    }
  }
  uint32_t kp, vp;
  const uint32_t kw = encode<T, LG>(x[0], kp);
  const uint32_t vw = encode<T, LG>(x[1], vp);
  // half-words g W + w: this lane has g = 2 (lane % 4) and the next, of
  // w = lane / 4; lanes of neighbouring w trade one each
  const int w = lane / 4, g = 2 * (lane % 4);
  const uint32_t got = __shfl_xor_sync(~0u, (w & 1) ? vw & 0xffffu : vw >> 16, 4);
  if (!live) return;
  const Place4 pl = pool.place(slot);
  char* unit = pool.unit(pl.block, head, pl.unit);
  *reinterpret_cast<uint32_t*>(unit + pl.row * U::kRow + 4 * ((lane % 4) * W + w)) = kw;
  const int half = (w & 1) ? (g + 1) * W + w - 1 : g * W + w;
  *reinterpret_cast<uint32_t*>(unit + U::oV + pl.row * U::kRow + 2 * half) =
      (w & 1) ? got | (vw & 0xffff0000u) : (vw & 0xffffu) | got << 16;
  if (lane % LG == 0) {
    const int pair = 4 * (pl.row * NG + lane / LG);
    *reinterpret_cast<uint32_t*>(unit + U::oKp + pair) = kp;
    *reinterpret_cast<uint32_t*>(unit + U::oVp + pair) = vp;
  }
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(kRowThreads)
    kv4_gather_kernel(const Pool4 pool, const int64_t* slots, int64_t n, const Rows4 k,
                      const Rows4 v, int vec, int32_t* status) {
  using U = Unit4<D, NG>;
  constexpr int L = D / 8, LG = L / NG, W = U::W;
  const Row4 w4 = row_of<L>(pool.hkv);
  const int64_t token = w4.token;
  const int head = w4.head, lane = threadIdx.x % L;
  if (token >= n) return;
  const int64_t slot = slots[token];
  const bool live = pool.valid(slot);
  if (!live && slot != -1 && lane == 0 && head == 0) report(status, CS_ST_SLOT_RANGE);
  uint32_t code[2] = {0u, 0u}, pair[2] = {0u, 0u};
  if (live) {
    const Place4 pl = pool.place(slot);
    const char* unit = pool.unit(pl.block, head, pl.unit);
    const int w = lane / 4, g = 2 * (lane % 4), at = 4 * (pl.row * NG + lane / LG);
    code[0] = *reinterpret_cast<const uint32_t*>(unit + pl.row * U::kRow +
                                                 4 * ((lane % 4) * W + w));
    const uint16_t* vc = reinterpret_cast<const uint16_t*>(unit + U::oV + pl.row * U::kRow);
    code[1] = vc[g * W + w] | (uint32_t)vc[(g + 1) * W + w] << 16;
    pair[0] = *reinterpret_cast<const uint32_t*>(unit + U::oKp + at);
    pair[1] = *reinterpret_cast<const uint32_t*>(unit + U::oVp + at);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const Rows4& r = h ? v : k;
    const uint4 y = decode<T>(code[h], pair[h]);
    char* p = r.x + token * r.st + head * r.sh + lane * 16;
    if (vec) {
      *reinterpret_cast<uint4*>(p) = y;
    } else {
      uint16_t* e = reinterpret_cast<uint16_t*>(p);
      const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) e[2 * i] = (uint16_t)z[i], e[2 * i + 1] = (uint16_t)(z[i] >> 16);
    }
  }
}

bool vec_rows(const Rows4& r) {
  return reinterpret_cast<uintptr_t>(r.x) % 16 == 0 && r.st % 16 == 0 && r.sh % 16 == 0;
}

int rows_call(bool append, const cs_kv4_pool* pool, const int64_t* slots, int64_t n, const void* k,
              int64_t kst, int64_t ksh, const void* v, int64_t vst, int64_t vsh, int32_t* status,
              void* stream) {
  CS_HOST_CHECK(pool != nullptr && n >= 0);
  if (const int rc = check_pool4(*pool)) return rc;
  if (n == 0) return CS_OK;
  CS_HOST_CHECK(slots != nullptr && k != nullptr && v != nullptr);
  const Rows4 kr{static_cast<char*>(const_cast<void*>(k)), 2 * kst, 2 * ksh};
  const Rows4 vr{static_cast<char*>(const_cast<void*>(v)), 2 * vst, 2 * vsh};
  const int64_t per = kRowThreads / (pool->head_dim / 8);
  const int64_t blocks = (n + per - 1) / per * pool->kv_heads;
  if (blocks > INT32_MAX) return CS_ERR_TOO_LARGE;
  const Pool4 p = Pool4::make(*pool);
  const int vec = vec_rows(kr) && vec_rows(vr);
  return by_pool4(*pool, [&](auto* t, auto d, auto g) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    if (append)
      kv4_append_kernel<T, D, NG><<<(unsigned)blocks, kRowThreads, 0, as_stream(stream)>>>(
          p, slots, n, kr, vr, vec, status);
    else
      kv4_gather_kernel<T, D, NG><<<(unsigned)blocks, kRowThreads, 0, as_stream(stream)>>>(
          p, slots, n, kr, vr, vec, status);
    CS_LAUNCH_CHECK();
    return CS_OK;
  });
}

}  // namespace
}  // namespace cs

extern "C" int cs_kv4_append(const cs_kv4_pool* pool, const int64_t* slots, int64_t n,
                             const void* k, int64_t k_stride_tok, int64_t k_stride_head,
                             const void* v, int64_t v_stride_tok, int64_t v_stride_head,
                             int32_t* status, void* stream) {
  return cs::rows_call(true, pool, slots, n, k, k_stride_tok, k_stride_head, v, v_stride_tok,
                       v_stride_head, status, stream);
}

extern "C" int cs_kv4_gather(const cs_kv4_pool* pool, const int64_t* slots, int64_t n, void* k,
                             int64_t k_stride_tok, int64_t k_stride_head, void* v,
                             int64_t v_stride_tok, int64_t v_stride_head, int32_t* status,
                             void* stream) {
  return cs::rows_call(false, pool, slots, n, k, k_stride_tok, k_stride_head, v, v_stride_tok,
                       v_stride_head, status, stream);
}

// ------------------------------------------------------------- attention
namespace cs {

Plan4 plan4(const cs_kv4_attn_params& p) {
  Plan4 plan;
  const int64_t g = p.q_heads / p.pool.kv_heads;
  // Query rows of a KV head an average request has.  Up to 32 go to the kernel
  // for few, in tiles of 16 that each read the keys: 16 requests behind 4096 keys
  // take 82 us with 24 or 28 rows and 98 in the wide kernel; 117 with 48 rows and
  // 100 there, 205 with 96 and 102.  (The wide kernel in blocks of 128 rows was no
  // faster with any of these, and slower with less work.)  One kernel takes the
  // whole batch: 63 decodes of up to 16K keys beside a chunk of 512 tokens take 756
  // us in the wide one, in two calls 174 and 86.
  const int64_t rows = p.requests > 0 ? p.tokens * g / p.requests : 0;
  plan.wide = rows > 32;
  plan.rows = plan.wide ? kWideRows : rows <= 8 ? 8 : 16;
  plan.workers = num_sms() * (plan.wide ? 1 : kv4_decode_blocks(plan.rows, p.pool.head_dim,
                                                                p.pool.group));
  return plan;
}

namespace {

int check_attn4(const cs_kv4_attn_params* p) {
  CS_HOST_CHECK(p != nullptr && p->tokens >= 0 && p->tokens < INT32_MAX && p->requests >= 0);
  if (const int rc = check_pool4(p->pool)) return rc;
  CS_HOST_CHECK(p->q_heads > 0 && p->q_heads % p->pool.kv_heads == 0);
  CS_HOST_CHECK(p->tokens * (p->q_heads / p->pool.kv_heads) < INT32_MAX - kWideRows);
  CS_HOST_CHECK(p->starts != nullptr || p->tokens == p->requests);
  CS_HOST_CHECK(p->requests == 0 || (p->lengths && (p->tables || p->table_width == 0)));
  CS_HOST_CHECK(p->table_width >= 0 && (p->requests <= 1 || p->table_stride >= p->table_width));
  CS_HOST_CHECK(p->tokens == 0 || (p->q && p->out));
  CS_HOST_CHECK(isfinite((float)p->scale));
  return CS_OK;
}

}  // namespace
}  // namespace cs

extern "C" int64_t cs_kv4_attn_workspace(const cs_kv4_attn_params* p) {
  using namespace cs;
  if (check_attn4(p) != CS_OK) return 0;
  const Plan4 plan = plan4(*p);
  return (int64_t)plan.workers * (16 + 2 * plan.rows * (p->pool.head_dim + 1) * 4);
}

extern "C" int cs_kv4_attn(const cs_kv4_attn_params* p, void* workspace, void* stream) {
  using namespace cs;
  if (const int rc = check_attn4(p)) return rc;
  if (p->tokens == 0) return CS_OK;
  CS_HOST_CHECK(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0);
  const Plan4 plan = plan4(*p);
  Attn4 a;
  a.pool = Pool4::make(p->pool);
  a.q = static_cast<const char*>(p->q);
  a.qt = 2 * p->q_stride_tok;
  a.qh = 2 * p->q_stride_head;
  a.out = static_cast<char*>(p->out);
  a.ot = 2 * p->o_stride_tok;
  a.oh = 2 * p->o_stride_head;
  a.lse = p->lse;
  a.tables = p->tables;
  a.table_stride = p->table_stride;
  a.lengths = p->lengths;
  a.starts = p->starts;
  a.status = p->status;
  a.joins = static_cast<int4*>(workspace);
  a.part_o = reinterpret_cast<float*>(a.joins + plan.workers);
  a.part_lse = a.part_o + 2ll * plan.workers * plan.rows * p->pool.head_dim;
  a.tokens = p->tokens;
  const int64_t longest = (int64_t)p->table_width * p->pool.block_size;
  a.longest = longest < INT32_MAX - 256 ? longest : INT32_MAX - 256;
  a.requests = p->requests;
  a.hq = p->q_heads;
  a.G = p->q_heads / p->pool.kv_heads;
  auto aligned = [](const void* x, int64_t t, int64_t h, int64_t to) {
    return reinterpret_cast<uintptr_t>(x) % to == 0 && t % to == 0 && h % to == 0;
  };
  a.vec_q = aligned(p->q, a.qt, a.qh, 16);
  a.vec_out = aligned(p->out, a.ot, a.oh, 8);
  a.zero_rest = p->zero_rest;
  a.flip = p->scale < 0.0 ? 0x80008000u : 0u;
  a.scale2 = fabsf((float)p->scale) * 1.4426950408889634f;
  return plan.wide ? kv4_wide(a, p->pool, plan.workers, as_stream(stream))
                   : kv4_decode(a, p->pool, plan.rows, plan.workers, as_stream(stream));
}
