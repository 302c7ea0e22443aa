// Attention over the 4-bit pool for few query rows a KV head (decodes, drafted
// tokens), and the join of its partial results.
//
// Per unit of 16 keys a warp forms
//   S^T = K Q^T  (16 keys x 8 rows),  P = 2^(S c - m),  O^T += V^T P^T
// on mma.sync.  The codes go into the products as they are: a 4-bit code in the
// low bits of a 16-bit number is that number of the smallest fp16 subnormals,
// exactly (and 16 times that, four bits up), so a word of eight codes becomes
// four operand registers with a shift and four ANDs, with no bias to take off
// and no rounding.  Scale and lowest value of a group enter in float32,
//   q.k = scale (q.c) + low sum(q),   p v = (p scale) c + p low,
// where p scale is rounded to fp16 for the product, and low is the middle of the
// group's values: their codes lose 8 (one subtraction a pair, exact), so that the
// long sums in the tensor unit stay as small as their results.  With codes 0 ..
// 15 even weights over 30,000 keys gave float16 outputs 0.00043 off, 0.0002 of
// which is the output's own rounding.  Queries are fp16 too, each row scaled by a power
// of two so that its largest element lies in [2^13, 2^14): 16-bit inputs of
// either type keep every bit down to 2^-27 of that.
//
// HBM (136 to 160 bytes a key and head) is the floor; what bounds it is the issue
// of about 255 instructions a unit, half of them on the ALU, at 0.55 a clock with
// four warps a scheduler.  8 decodes of 65K keys (64/8 heads, groups of 128) take
// 135 us, 4.2 TB/s; 32 of up to 16K (32/8, groups of 64) 87 us, 3.5 TB/s (85 with a
// reference by the scales alone, which constant values overflow); four drafts each
// (16 rows, groups of 32) 171 us.  The products are far too small for
// tcgen05, whose operands would have to be written to shared memory
// in 16 bits first, four times the bytes that come in -- at full bandwidth 87
// bytes a clock and SM written and as many read again, of 128.  Here the codes
// go from a ring of raw units (one bulk copy each) to registers.
#include <math.h>

#include <type_traits>

#include "kv4.cuh"
#include "kv4_attn.cuh"
#include "sm100.cuh"

namespace cs {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kLeast = 1;              // steps a block takes at least
constexpr float kUp = 6.f;  // a new largest p scale is 2^6: fp16's normal numbers reach 2^-20 of it
constexpr float kTooLarge = 0x1p14f;  // it may grow to 2^14 before O is rescaled
constexpr float kLowest = -3e38f;     // below every score, and finite
// What a key may add goes by its largest scale, 2^-40 of its largest lowest value
// (constant groups have no scale: p low then stays below 2^54) and at least
// 2^-100; the sums of p, which are kept 2^-24 of theirs, then stay below 2^121 over
// 2^31 keys of zeros.  Above 2^116 the reference stops rising: p scale is at most
// 2^16 there, and p at least 2^-110 for a row's largest score, 2^-16 of which
// float32 still holds.
constexpr float kLowCounts = 0x1p-40f, kLeastMost = 0x1p-100f, kMostLog = 116.f;
constexpr float kSumDown = 0x1p-24f;

// Blocks an SM holds, as the registers allow without spilling in the loop over
// the keys: 32 decodes of up to 16K keys in four groups take 102 us with three
// and 129 with four, in two groups 92 and 90; four drafts each (16 rows) in four
// groups 183 with two and 251 with three, in two groups 159 and 161.
constexpr int decode_blocks(int tiles, int dim, int groups) {
  return tiles == 1 ? (dim == 128 && groups == 4 ? 3 : 4) : (dim == 128 ? 2 : 3);
}

template <int D, int NG, int NT>
struct Ring {
  static constexpr int RT = 8 * NT;  // query rows of a block
  // units a warp takes at once: two have twice the independent work and one
  // wait, copy and vote between them
  static constexpr int E = NT == 1 ? 2 : 1;
  static constexpr int kStep = kUnit * kWarps * E;  // keys of a block's step
  static constexpr int kStages = 4 / E;             // of E units
  static constexpr int kBlocks = decode_blocks(NT, D, NG);  // an SM's
  static constexpr int oBars = kWarps * kStages * E * Unit4<D, NG>::kBytes;
  static constexpr int oSums = oBars + kWarps * kStages * 8;
  static constexpr int oMax = oSums + 96;
  static constexpr int oOut = (oMax + 2 * kWarps * RT * 4 + 15) / 16 * 16;
  // the queries' operand registers, for 16 rows (those of 8 stay in registers)
  static constexpr int oQuery = oOut + kWarps * RT * D * 4;
  static constexpr int kBytes = oQuery + (NT > 1 ? NT * (D / 32) * 512 : 0);
};

// D += A B, 16 x 8 x 16 in fp16 with float32 sums
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D = A B
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the largest that is a number
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// a pair of codes (of 16 times codes: 128) less 8, as numbers of 2^-24
__device__ __forceinline__ uint32_t less_middle(uint32_t x, uint32_t by) {
  const uint32_t m = by * 0x10001u;
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x),
                            *reinterpret_cast<const __half2*>(&m));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
template <int N> struct Words;
template <> struct Words<4> {
  static __device__ __forceinline__ void load(uint32_t (&w)[4], const char* p) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  }
};
template <> struct Words<2> {
  static __device__ __forceinline__ void load(uint32_t (&w)[2], const char* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  }
};
template <> struct Words<1> {
  static __device__ __forceinline__ void load(uint32_t (&w)[1], const char* p) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
};

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;

template <typename T, int D, int NG, int NT>
__global__ void __launch_bounds__(kThreads, Ring<D, NG, NT>::kBlocks)
    kv4_decode_kernel(const __grid_constant__ Attn4 a) {
  using U = Unit4<D, NG>;
  using R = Ring<D, NG, NT>;
  using Share = Share4<R::RT, R::kStep>;
  constexpr int W = U::W, RT = R::RT, S = R::kStages, E = R::E, WG = W / NG;  // words a group
  constexpr int kStage = E * U::kBytes;
  extern __shared__ __align__(128) char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  char* ring = smem + warp * S * kStage;
  const uint32_t bars = smem_u32(smem + R::oBars) + warp * S * 8;
  float* maxima = reinterpret_cast<float*>(smem + R::oMax);       // [warp][row]
  float* sums = maxima + kWarps * RT;                             // [warp][row]
  float* outs = reinterpret_cast<float*>(smem + R::oOut);         // [warp][row][dim]
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(bars + 8 * s, E);
    mbar_init_fence();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Share work;
  using Scratch = typename Share::template Scratch<kThreads>;
  static_assert(sizeof(Scratch) <= R::oMax - R::oSums, "its place");
  const bool ordered = work.template find<kThreads>(a, blockIdx.x, gridDim.x, kLeast,
                                                    *reinterpret_cast<Scratch*>(smem + R::oSums));
  zero_rest<T, D>(a, ordered);
  int issued = 0, taken = 0;  // units of this warp's ring
  bool late = false, bad_block = false;
  int which = 0;  // of this block's partial results
  int4 join = make_int4(-1, 0, 0, 0);

  while (work.todo > 0) {
    const Request4 r = work.r;
    const int all_steps = Share::steps(r, a.G, work.tile);
    const int s0 = work.step;
    const int s1 = (int)min((int64_t)all_steps, s0 + work.todo);
    const int row0 = work.tile * RT, rows = r.n * a.G;
    const int h = work.head;
    // ------------------------------------------------------------ keys ahead
    // this warp's pass i takes units unit_of(i, 0 .. E - 1); beyond the tile's
    // last key none is fetched
    const int seen = max(0, r.len - r.n + Share::last_token(r, a.G, work.tile) + 1);
    const int units = (seen + kUnit - 1) / kUnit;
    auto unit_of = [&](int i, int e) { return ((s0 + i) * kWarps + warp) * E + e; };
    int count = s1 - s0;  // passes
    if (count > 0 && unit_of(count - 1, 0) >= units) --count;
    const int32_t* table = a.tables + work.request * a.table_stride;
    // this lane's unit of passes batch .. batch + 32 / E - 1: -1 none, 0 no block
    int64_t from = -1;
    int batch = 0, sent = 0;
    auto find_units = [&] {
      batch = sent;
      const int u = unit_of(sent + lane / E, lane % E), j = u / a.pool.units;
      from = -1;
      if (u < units) {
        const int id = table[j];
        from = id >= 0 && id < a.pool.num_blocks
                   ? reinterpret_cast<int64_t>(a.pool.unit(id, h, u - j * a.pool.units))
                   : 0;
        bad_block |= from == 0;
      }
    };
    auto send = [&] {  // the whole warp
      if (sent - batch == 32 / E) find_units();
      if (lane / E == sent - batch) {
        const int st = issued % S;
        const uint32_t bar = bars + 8 * st;
        char* to = ring + st * kStage + (lane % E) * U::kBytes;
        if (from > 0) {
          mbar_arrive_expect(bar, U::kBytes);
          bulk_copy(smem_u32(to), reinterpret_cast<const void*>(from), U::kBytes, bar);
        } else {
          if (from == 0) {  // zero codes, scales and lows: zero keys and values
            for (int i = 0; i < U::kBytes / 16; ++i)
              *reinterpret_cast<uint4*>(to + 16 * i) = make_uint4(0, 0, 0, 0);
            fence_async_smem();  // before a later copy into this place
          }
          mbar_arrive(bar);
        }
      }
      ++issued;
      ++sent;
    };
    find_units();
    for (int i = 0; i < S && i < count; ++i) send();

    // --------------------------------------------------------------- queries
    uint4 qf[NT == 1 ? W : 1];      // operand registers: word w's lower half, then its upper
    uint4* query = reinterpret_cast<uint4*>(smem + R::oQuery) + lane;  // [nt][w], 32 lanes each
    float2 qs[NT][NG];              // sum(q) of rows 2t, 2t + 1, as the products have it
    float2 qm[NT];                  // from there to log2 of the weights
    int limit[NT][2];               // the newest key these rows see
    int low_limit = INT32_MAX;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + 8 * nt + g;
      const bool ok = row < rows;
      const int tok = ok ? row / a.G : 0;
      const char* p = a.q + (int64_t)(r.start + tok) * a.qt +
                      (int64_t)(h * a.G + (ok ? row - tok * a.G : 0)) * a.qh;
      float f[W][8];
      float top = 0.f, sum[NG];
#pragma unroll
      for (int k = 0; k < NG; ++k) sum[k] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t x[4];
        const char* e = p + 2 * (32 * w + 8 * t);
        if (!ok) {
          x[0] = x[1] = x[2] = x[3] = 0u;
        } else if (a.vec_q) {
          Words<4>::load(x, e);
        } else {
          const uint16_t* u = reinterpret_cast<const uint16_t*>(e);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 y = pair_of<T>(x[i] ^ a.flip);
          f[w][2 * i] = y.x, f[w][2 * i + 1] = y.y;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          top = fmaxf(top, fabsf(f[w][i]));
          sum[w / WG] += f[w][i];
        }
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(~0u, sum[k], 1);
        sum[k] += __shfl_xor_sync(~0u, sum[k], 2);
      }
      // (2^-124 and 2^124 below: queries of up to 2^116)
      const int e = min(113, max(-100, (int)(__float_as_uint(top) >> 23) - 127));
      const float up = pow2(13 - e);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // elements 2k, 2k + 4 and (sixteenths) 2k + 1, 2k + 5
        const float less = up * 0.0625f;
        const uint4 y = make_uint4(Pack2<__half>::pack(f[w][0] * up, f[w][4] * up),
                                   Pack2<__half>::pack(f[w][1] * less, f[w][5] * less),
                                   Pack2<__half>::pack(f[w][2] * up, f[w][6] * up),
                                   Pack2<__half>::pack(f[w][3] * less, f[w][7] * less));
        if constexpr (NT == 1) qf[w] = y;
        else if (warp == 0) query[32 * (W * nt + w)] = y;
      }
      // the codes are 2^-24 of theirs, the queries `up` of theirs; masked scores
      // are -inf before they are scaled, so the factor is never 0
      const float back = fmaxf(pow2(11 + e) * a.scale2, 1e-30f);
#pragma unroll
      for (int w = 0; w < NG; ++w) sum[w] *= pow2(-11 - e);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int from_lane = 4 * (2 * t + k), m = row0 + 8 * nt + 2 * t + k;
        (k ? qm[nt].y : qm[nt].x) = __shfl_sync(~0u, back, from_lane);
#pragma unroll
        for (int w = 0; w < NG; ++w)
          (k ? qs[nt][w].y : qs[nt][w].x) = __shfl_sync(~0u, sum[w], from_lane);
        // (no row: what lies behind the last key is not to move the others' reference)
        limit[nt][k] = m < rows ? r.len - r.n + m / a.G : seen - 1;
        low_limit = min(low_limit, limit[nt][k]);
      }
    }
    low_limit = __reduce_min_sync(~0u, low_limit);
    if constexpr (NT > 1) __syncthreads();

    // ------------------------------------------------------------------ keys
    float o[NT][2 * W][4];
    // log2 of the largest p scale so far, less kUp; and float32 sums of two rows
    float2 ref[NT], lsum[NT], lows[NT][NG];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.f;
      }
      ref[nt] = make_float2(kLowest, kLowest);
      lsum[nt] = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NG; ++w) lows[nt][w] = make_float2(0.f, 0.f);
    }
    for (int i = 0; i < count; ++i) {
      const int st = taken % S;
      if (!mbar_try(bars + 8 * st, (taken / S) & 1) && !late) {
        const long long begin = clock64();
        while (!late && !mbar_try(bars + 8 * st, (taken / S) & 1))
          late = clock64() - begin > kWaitCycles;
      }
      __syncwarp();
      const char* stage = ring + st * kStage;
      ++taken;
      float2 x[E][NT][2];  // rows 2t and 2t + 1 at key g, and at key g + 8
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const char* unit = stage + e * U::kBytes;
        uint32_t ka[W], kb[W];
        Words<W>::load(ka, unit + g * U::kRow + 4 * W * t);
        Words<W>::load(kb, unit + (g + 8) * U::kRow + 4 * W * t);
        uint32_t pa[NG], pb[NG];
        Words<NG>::load(pa, unit + U::oKp + 4 * NG * g);
        Words<NG>::load(pb, unit + U::oKp + 4 * NG * (g + 8));
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const float2 fa = pair_of<T>(pa[k]), fb = pair_of<T>(pb[k]);
          float acc[NT][4];
#pragma unroll
          for (int w = k * WG; w < (k + 1) * WG; ++w) {
            const uint32_t ya = ka[w] >> 8, yb = kb[w] >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint4 q;
              if constexpr (NT == 1) q = qf[w];
              else q = query[32 * (W * nt + w)];
              if (w == k * WG)
                mma16_first(acc[nt], ka[w] & kLow, kb[w] & kLow, ka[w] & kHigh, kb[w] & kHigh, q.x,
                            q.y);
              else
                mma16(acc[nt], ka[w] & kLow, kb[w] & kLow, ka[w] & kHigh, kb[w] & kHigh, q.x, q.y);
              mma16(acc[nt], ya & kLow, yb & kLow, ya & kHigh, yb & kHigh, q.z, q.w);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 sa = make_float2(acc[nt][0], acc[nt][1]),
                         sb = make_float2(acc[nt][2], acc[nt][3]);
            const float2 la = __fmul2_rn(both(fa.y), qs[nt][k]),
                         lb = __fmul2_rn(both(fb.y), qs[nt][k]);
            x[e][nt][0] = __ffma2_rn(both(fa.x), sa, k ? __fadd2_rn(x[e][nt][0], la) : la);
            x[e][nt][1] = __ffma2_rn(both(fb.x), sb, k ? __fadd2_rn(x[e][nt][1], lb) : lb);
          }
        }
      }
      const int key0 = kUnit * unit_of(i, 0);
      uint32_t shown = ~0u;  // bit 4 (NT e + nt) + c: the row sees the key
      const bool some_hidden = key0 + E * kUnit - 1 > low_limit;
      if (some_hidden) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (key0 + kUnit * e + g + 8 * (c / 2) <= limit[nt][c & 1]) continue;
              (c & 1 ? x[e][nt][c / 2].y : x[e][nt][c / 2].x) = -INFINITY;
              shown &= ~(1u << (4 * (NT * e + nt) + c));
            }
          }
        }
      }
      // ------------------------------------------------------------- weights
      // p scale has to fit fp16 (and p float32): where it would not, the
      // reference moves up and what was summed goes down
      float2 p[E][NT][2];
      float most[E][2], top = 0.f;
      // a scale or low that is not finite (or whatever lies behind the last key),
      // and a key hidden from a row
      bool careful = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t v[NG];
          Words<NG>::load(v, stage + e * U::kBytes + U::oVp + 4 * NG * (g + 8 * c));
          // |scale| and |low|, the largest of the groups' (NaN: the others')
          pair16<T> ends = __habs2(as_pair<T>(v[0]));
#pragma unroll
          for (int k = 1; k < NG; ++k) ends = __hmax2(ends, __habs2(as_pair<T>(v[k])));
          const float2 end = pair_of<T>(pair_bits(ends));
          most[e][c] = max3(end.x, end.y * kLowCounts, kLeastMost);
          if (some_hidden) {
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              const float2 y = pair_of<T>(v[k]);
              careful |= !(8.f * fabsf(y.x) + fabsf(y.y) < INFINITY);
            }
          }
        }
      }
      auto weights = [&] {
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float2 y = __ffma2_rn(x[e][nt][c], qm[nt], make_float2(-ref[nt].x, -ref[nt].y));
              p[e][nt][c] = make_float2(ex2(y.x), ex2(y.y));
            }
          }
        }
      };
      weights();
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float y = fmaxf(p[e][0][c].x, p[e][0][c].y);
#pragma unroll
          for (int nt = 1; nt < NT; ++nt) y = fmaxf(y, fmaxf(p[e][nt][c].x, p[e][nt][c].y));
          top = fmaxf(top, y * most[e][c]);
        }
      }
      if (__any_sync(~0u, top > kTooLarge)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
          for (int e = 0; e < E; ++e) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float l = fminf(lg2(most[e][c]), kMostLog) - kUp;
              ma = fmaxf(ma, fmaf(x[e][nt][c].x, qm[nt].x, l));
              mb = fmaxf(mb, fmaf(x[e][nt][c].y, qm[nt].y, l));
            }
          }
          auto raise = [&](float& old, float m) {
            m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
            m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
            m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
            m = fmaxf(m, old);
            const float f = m == old ? 1.f : ex2(0.5f * (old - m));
            old = m;
            return f;
          };
          // The root, since the reference may rise by more than float32's range
          // (zero values, then large ones); the sums of p, which were as much
          // larger, keep theirs.
          const float2 half = make_float2(raise(ref[nt].x, ma), raise(ref[nt].y, mb));
          const float2 down = __fmul2_rn(half, half);
          lsum[nt] = __fmul2_rn(__fmul2_rn(lsum[nt], half), half);
#pragma unroll
          for (int w = 0; w < NG; ++w) lows[nt][w] = __fmul2_rn(lows[nt][w], down);
#pragma unroll
          for (int w = 0; w < 2 * W; ++w) {
            o[nt][w][0] *= down.x, o[nt][w][1] *= down.y;
            o[nt][w][2] *= down.x, o[nt][w][3] *= down.y;
          }
        }
        weights();
      }
      auto finish = [&](auto hidden) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const char* unit = stage + e * U::kBytes;
          uint32_t v[4][(W + 1) / 2], va[NG], vb[NG];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            Words<W / 2>::load(v[k], unit + U::oV + (2 * t + (k & 1) + 4 * (k & 2)) * U::kRow +
                                         2 * W * g);
          Words<NG>::load(va, unit + U::oVp + 4 * NG * g);
          Words<NG>::load(vb, unit + U::oVp + 4 * NG * (g + 8));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            lsum[nt] = __ffma2_rn(__fadd2_rn(p[e][nt][0], p[e][nt][1]), both(kSumDown), lsum[nt]);
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            uint32_t pf[NT][2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float2 s = pair_of<T>(c ? vb[k] : va[k]);
              s.y = fmaf(8.f, s.x, s.y);  // the middle of the group's values
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float2 w = __fmul2_rn(p[e][nt][c], both(s.x));
                if constexpr (decltype(hidden)::value) {
                  // a scale that is not finite reaches no row that does not see its key
                  const int bit = 4 * (NT * e + nt) + 2 * c;
                  const bool sx = shown >> bit & 1u, sy = shown >> (bit + 1) & 1u;
                  w = make_float2(sx ? w.x : 0.f, sy ? w.y : 0.f);
                  const float2 low = make_float2(sx ? s.y : 0.f, sy ? s.y : 0.f);
                  lows[nt][k] = __ffma2_rn(p[e][nt][c], low, lows[nt][k]);
                } else {
                  lows[nt][k] = __ffma2_rn(p[e][nt][c], both(s.y), lows[nt][k]);
                }
                pf[nt][c] = transposed(Pack2<__half>::pack(w.x, w.y));
              }
            }
#pragma unroll
            for (int w = k * WG; w < (k + 1) * WG; ++w) {
              const uint32_t sel = w & 1 ? 0x7632u : 0x5410u;
              const uint32_t xa = __byte_perm(v[0][w / 2], v[1][w / 2], sel);
              const uint32_t xb = __byte_perm(v[2][w / 2], v[3][w / 2], sel);
              const uint32_t ya = xa >> 8, yb = xb >> 8;
              const uint32_t v0 = less_middle(xa & kLow, 8), v1 = less_middle(xa & kHigh, 128),
                             v2 = less_middle(xb & kLow, 8), v3 = less_middle(xb & kHigh, 128),
                             v4 = less_middle(ya & kLow, 8), v5 = less_middle(ya & kHigh, 128),
                             v6 = less_middle(yb & kLow, 8), v7 = less_middle(yb & kHigh, 128);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16(o[nt][2 * w], v0, v1, v2, v3, pf[nt][0], pf[nt][1]);
                mma16(o[nt][2 * w + 1], v4, v5, v6, v7, pf[nt][0], pf[nt][1]);
              }
            }
          }
        }
      };
      if (__any_sync(~0u, careful)) finish(std::true_type());
      else finish(std::false_type());
      __syncwarp();  // the units have been read
      if (sent < count) send();
    }

    // --------------------------------------------------- the warps' results
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) {
        auto add = [&](float2& y) {
          y = __fadd2_rn(y, make_float2(__shfl_xor_sync(~0u, y.x, s),
                                        __shfl_xor_sync(~0u, y.y, s)));
        };
        add(lsum[nt]);
#pragma unroll
        for (int w = 0; w < NG; ++w) add(lows[nt][w]);
      }
      if (g == 0) {
        *reinterpret_cast<float2*>(maxima + warp * RT + 8 * nt + 2 * t) = ref[nt];
        *reinterpret_cast<float2*>(sums + warp * RT + 8 * nt + 2 * t) = lsum[nt];
      }
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = 8 * nt + 2 * t + k;
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, maxima[w * RT + row]);
        const float mine = k ? ref[nt].y : ref[nt].x;
        const float f = mine == top ? 1.f : ex2(mine - top);
        float* to = outs + (warp * RT + row) * D + 4 * g;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float z = k ? lows[nt][w / WG].y : lows[nt][w / WG].x;
          float4 y;
          y.x = fmaf(o[nt][2 * w][k], 0x1p24f, z) * f;
          y.y = fmaf(o[nt][2 * w][k + 2], 0x1p20f, z) * f;
          y.z = fmaf(o[nt][2 * w + 1][k], 0x1p24f, z) * f;
          y.w = fmaf(o[nt][2 * w + 1][k + 2], 0x1p20f, z) * f;
          *reinterpret_cast<float4*>(to + 32 * w) = y;
        }
      }
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == all_steps;
    const int64_t part = 2ll * blockIdx.x + which;
    for (int i = tid; i < RT * (D / 4); i += kThreads) {
      const int row = i / (D / 4), c = 4 * (i % (D / 4));
      if (row0 + row >= rows) break;
      float top = kLowest, l = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, maxima[w * RT + row]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float m = maxima[w * RT + row];
        const float half = m == top ? 1.f : ex2(0.5f * (m - top));
        l += sums[w * RT + row] * half * half;
        const float4 z = *reinterpret_cast<const float4*>(outs + (w * RT + row) * D + c);
        y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
      }
      // (l from 2^-134 to 2^121: its reciprocal in float32's range)
      const float up = l < 0x1p-60f ? 0x1p64f : 1.f, down = up * kSumDown;
      const float inv = l == 0.f ? 0.f : 1.f / (l * up);
      const float lse2 = l == 0.f ? -INFINITY : top + (log2f(l) + 24.f);
      y.x = y.x * down * inv, y.y = y.y * down * inv;
      y.z = y.z * down * inv, y.w = y.w * down * inv;
      if (whole) {
        write4<T>(a, r.start, row0 + row, h, c, y);
        if (c == 0) write_lse(a, r.start, row0 + row, h, lse2);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (part * RT + row) * D + c) = y;
        if (c == 0) a.part_lse[part * RT + row] = lse2;
      }
    }
    if (!whole) {
      if (s0 == 0)  // the first of the tile's blocks has them joined
        join = make_int4(work.request, work.tile, 2 * h + which,
                         blockIdx.x + (int)((all_steps - s1 + work.per - 1) / work.per));
      which = 1;
    }
    __syncthreads();  // the results have been read
    work.todo -= s1 - s0;
    if (work.todo > 0) work.next(a);
  }
  if (tid == 0) a.joins[blockIdx.x] = join;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (bad_block) report(a.status, CS_ST_SLOT_RANGE);
  // (any lane's wait: another may have seen the phase end just after)
  if (__any_sync(~0u, late)) {  // copies of this block are to have landed before it ends
    for (int s = taken - S < 0 ? 0 : taken - S; s < taken; ++s) {
      const long long begin = clock64();
      while (!mbar_try(bars + 8 * (s % S), (s / S) & 1) && clock64() - begin < kWaitCycles) {
      }
    }
    if (lane == 0) report(a.status, CS_ST_TIMEOUT);
  }
}

template <typename T, int D, int NG, int NT>
int launch_decode(const Attn4& a, int workers, cudaStream_t stream) {
  constexpr auto kernel = kv4_decode_kernel<T, D, NG, NT>;
  constexpr int kBytes = Ring<D, NG, NT>::kBytes;
  if (!allow_smem<kernel>(kBytes)) return CS_ERR_CUDA;
  if (const int rc = launch_dependent(kernel, dim3(workers), kThreads, kBytes, stream, a))
    return rc;
  return launch_join<T, D, 8 * NT>(a, workers, stream);
}

}  // namespace

int kv4_decode_blocks(int rows, int dim, int group) {
  return decode_blocks(rows <= 8 ? 1 : 2, dim, dim / group);
}

int kv4_decode(const Attn4& a, const cs_kv4_pool& pool, int rows, int workers,
               cudaStream_t stream) {
  return by_pool4(pool, [&](auto* t, auto d, auto g) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    return rows <= 8 ? launch_decode<T, D, NG, 1>(a, workers, stream)
                     : launch_decode<T, D, NG, 2>(a, workers, stream);
  });
}

}  // namespace cs
