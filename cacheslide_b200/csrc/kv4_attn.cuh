// What the two attention kernels of the 4-bit pool share: how a row's result is
// written, and the join of partial results.
#pragma once

#include "kv4.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace cs {

// the kernel for few query rows a KV head (kv4_decode.cu) and the one for many
// (kv4_sm100.cu), for `workers` blocks
int kv4_decode_blocks(int rows, int dim, int group);  // an SM's, with so many rows a block
int kv4_decode(const Attn4& a, const cs_kv4_pool& pool, int rows, int workers,
               cudaStream_t stream);
constexpr int kWideRows = 256;  // query rows a block of the wide kernel
int kv4_wide(const Attn4& a, const cs_kv4_pool& pool, int workers, cudaStream_t stream);
// workers and query rows a block for a call: the workspace's shape
struct Plan4 {
  int workers, rows;
  bool wide;
};
Plan4 plan4(const cs_kv4_attn_params& p);

// rows of a joining block: one a warp, four where a tile has many
template <int RT> constexpr int kJoinRows = RT > 16 ? 16 : 4;
constexpr float kLn2 = 0.6931471805599453f;

// A mean of the type's numbers is none past its largest: what the weights'
// rounding (2^-11 of it at most) carried there comes back.  Bfloat16's own half
// step is wider than that.
template <typename T> __device__ __forceinline__ float mean_of(float x) { return x; }
template <> __device__ __forceinline__ float mean_of<__half>(float x) {
  return fabsf(x) < 65600.f ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
}
// two of them as a pair of the type, none of which is an infinity of its own
template <typename T> __device__ __forceinline__ uint32_t mean_pair(float x, float y) {
  return Pack2<T>::pack(x, y);
}
template <> __device__ __forceinline__ uint32_t mean_pair<__half>(float x, float y) {
  const uint32_t z = Pack2<__half>::pack(x, y);
  return pair_bits(__hmin2_nan(__hmax2_nan(as_pair<__half>(z), as_pair<__half>(0xfbfffbffu)),
                               as_pair<__half>(0x7bff7bffu)));
}

// four neighbouring elements from `c` on of row `row` of a (request, KV head)
template <typename T>
__device__ __forceinline__ void write4(const Attn4& a, int start, int row, int h, int c, float4 y) {
  const int tok = row / a.G;
  char* to = a.out + (int64_t)(start + tok) * a.ot +
             (int64_t)(h * a.G + (row - tok * a.G)) * a.oh + 2 * c;
  const uint32_t lo = Pack2<T>::pack(mean_of<T>(y.x), mean_of<T>(y.y)),
                 hi = Pack2<T>::pack(mean_of<T>(y.z), mean_of<T>(y.w));
  if (a.vec_out) {
    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
  } else {
    uint16_t* e = reinterpret_cast<uint16_t*>(to);
    e[0] = (uint16_t)lo, e[1] = (uint16_t)(lo >> 16);
    e[2] = (uint16_t)hi, e[3] = (uint16_t)(hi >> 16);
  }
}
__device__ __forceinline__ void write_lse(const Attn4& a, int start, int row, int h, float lse2) {
  if (a.lse == nullptr) return;
  const int tok = row / a.G;
  a.lse[(int64_t)(start + tok) * a.hq + h * a.G + (row - tok * a.G)] = lse2 * kLn2;
}

// rows outside every request, when they are to be zeros (`ordered`: the starts
// are)
template <typename T, int D>
__device__ __forceinline__ void zero_rest(const Attn4& a, bool ordered) {
  if (!a.zero_rest || a.starts == nullptr) return;
  const int64_t first = a.starts[0], end = a.starts[a.requests];
  const bool plain = ordered && first >= 0 && end <= a.tokens;
  if (plain && first == 0 && end == a.tokens) return;
  // Requests that were left out leave rows in between.  A row belongs to the
  // newest of the starts up to it that lies below none before.
  auto owned = [&](int64_t row) {
    for (int b = 0, floor = 0; b < a.requests; ++b) {
      const int lo = a.starts[b], hi = a.starts[b + 1];
      if (lo >= floor && lo <= row && row < hi && hi <= a.tokens) return true;
      floor = max(floor, lo);
    }
    return false;
  };
  const int64_t n = a.tokens * a.hq * (D / 4);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t token = i / (a.hq * (D / 4));
    if (plain ? token >= first && token < end : owned(token)) continue;
    const int at = (int)(i - token * (a.hq * (D / 4)));
    const int head = at / (D / 4), c = 4 * (at % (D / 4));
    uint16_t* to = reinterpret_cast<uint16_t*>(a.out + token * a.ot + head * a.oh) + c;
    to[0] = to[1] = to[2] = to[3] = 0;
    if (a.lse && c == 0) a.lse[token * a.hq + head] = -INFINITY;
  }
}

// o = sum_c w_c o_c / sum_c w_c with w_c = 2^(lse_c - max) over the blocks that
// shared a row tile, in their order; a block kJoinRows rows of a tile that was
// cut, a warp a row, 32 weights at once and eight partial rows in flight.
template <typename T, int D, int RT>
__global__ void __launch_bounds__(128) kv4_join_kernel(const __grid_constant__ Attn4 a) {
  constexpr int E = D / 32;
  using V = typename std::conditional<E == 4, float4, float2>::type;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 j = a.joins[blockIdx.x];
  if (j.x < 0) return;
  const int lane = threadIdx.x & 31, first = blockIdx.x, parts = j.w - first + 1;
  const Request4 r = request4(a, j.x, 0);  // (its blocks have seen to its starts)
  const int row0 = j.y * RT, h = j.z >> 1;
  const int rows = min(min(RT, r.n * a.G - row0), (int)(blockIdx.y + 1) * kJoinRows<RT>);
  auto place = [&](int i) { return i == 0 ? 2ll * first + (j.z & 1) : 2ll * (first + i); };
  // the weights are down by a power of two that keeps their sum below 1, and so
  // that of the parts within float32
  const float back = __int_as_float((127 + 32 - __clz(parts)) << 23), down = 1.f / back;
  for (int row = blockIdx.y * kJoinRows<RT> + (threadIdx.x >> 5); row < rows; row += 4) {
    float top = -INFINITY, sum = 0.f, o[E];
    for (int i = lane; i < parts; i += 32)
      top = fmaxf(top, a.part_lse[place(i) * RT + row]);
    top = warp_max(top);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const float l = i0 + lane < parts ? a.part_lse[place(i0 + lane) * RT + row] : -INFINITY;
      // one below 2^-126 of the largest is that, not 0: what is not finite stays
      const float f = l == -INFINITY ? 0.f : down * max_nan(ex2(l - top), 0x1p-126f);
      sum += warp_sum(f);
      const int m = min(32, parts - i0);
#pragma unroll 1
      for (int c = 0; c < m; c += 8) {
        V x[8];
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          w[k] = __shfl_sync(~0u, f, (c + k) & 31);
          if (c + k >= m) w[k] = 0.f;
          if (w[k] != 0.f)
            x[k] = reinterpret_cast<const V*>(a.part_o + (place(i0 + c + k) * RT + row) * D)[lane];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (w[k] == 0.f) continue;
          const float* v = reinterpret_cast<const float*>(&x[k]);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = fmaf(w[k], v[e], o[e]);
        }
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tok = (row0 + row) / a.G, head = h * a.G + (row0 + row - tok * a.G);
    T* out = reinterpret_cast<T*>(a.out + (int64_t)(r.start + tok) * a.ot + (int64_t)head * a.oh);
#pragma unroll
    for (int e = 0; e < E; ++e) out[lane * E + e] = Elem<T>::from_f(mean_of<T>(o[e] * inv));
    if (lane == 0)
      write_lse(a, r.start, row0 + row, h, sum == 0.f ? -INFINITY : top + log2f(sum * back));
  }
}

template <typename T, int D, int RT>
int launch_join(const Attn4& a, int workers, cudaStream_t stream) {
  return launch_dependent(kv4_join_kernel<T, D, RT>,
                          dim3(workers, RT / kJoinRows<RT>), 128, 0, stream, a);
}

}  // namespace cs
