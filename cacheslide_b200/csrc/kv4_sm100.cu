// Tensor-core attention over the 4-bit pool for many query rows a KV head
// (questions, prompt chunks): tcgen05, TMEM.
//
// One block takes a range of the steps of all row tiles (Share4): up to two
// tiles of 128 query rows of a (request, KV head) and the keys that they see,
// 64 a step.  Per step
//   S = Q K^T (tcgen05, TMEM),  P = 2^(S c - m),  O += P V (P from TMEM)
// with the running maximum m and sum of each row in float32 registers.
//
// Two warps turn the step's key codes into the operand tile and two the value
// codes: a word of eight codes, fetched a step ahead, becomes four pairs of
// fp16 numbers with five bit operations (1024 + code has the code in its low
// bits), four subtractions and four multiply-adds with scale and lowest value;
// that is shared by all rows of the block, up to 256.  Operands are fp16
// whatever the pool's type: queries are scaled by a power of two a row, bfloat16
// keys and values by one for 32 of a step (of what their scales and lowest values
// can reach), so they keep fp16's 11 bits, where bfloat16 operands would keep 8:
// queries up to 2^127, keys from 2^-126 and values from 2^-118 on, and down to
// 2^-27 of the largest of the 32 (whether a row sees that one or not; 2^-38 of it
// is 0).  P carries the values' power of two, the rows' sums do not.  Float16
// outputs would show the rounding of such keys and values (0.00047 to 0.00054 off
// with both, 0.00033 with the values', 0.00021 of which is the output's own), so
// those of float16 pools are two operands each, scale (code - zero) and what is
// left.
//
// Bound by the softmax warps: 2600 clocks a step of 64 keys of two row tiles, of
// which the exponentials take 1024.  8 chunks of 512 tokens over 4096 keys (32/8
// heads of 128, bfloat16) take 393 us, 655 TFLOP/s (406 us sustained, under the
// power limit; 583 with codes fetched from global memory by the warps that decode
// them), 490 in float16, 13 questions of 3 to 150 tokens 70 us.
//
// Pairs lie in the tiles as the codes come, elements (0, 4), (1, 5), (2, 6), (3,
// 7) of eight: the queries are written in the same order, and the output's
// columns are put back as they are written.
#include <math.h>

#include <type_traits>

#include "kv4.cuh"
#include "kv4_attn.cuh"
#include "sm100.cuh"

namespace cs {
namespace {

constexpr int kKeys = 64;         // keys of a step
constexpr int kTileRows = 128, NT = 2;  // query rows of a tile, row tiles of a block
static_assert(kTileRows * NT == kWideRows, "the workspace's rows");
constexpr int kLeastSteps = 4;    // steps a block takes at least
constexpr float kLazy = 8.f;      // O is rescaled when the maximum grew by more than 2^8
constexpr float kUp = 7.f;        // P is stored up by 2^7: fp16's normal numbers reach 2^-21
constexpr float kSumDown = 0x1p-24f;  // the sums of weights are kept this much smaller
// A thread's weights (which carry the values' power of two) that all lie below
// 2^-100 of the reference are summed without that power, which may be as far down.
constexpr float kFaint = 100.f;
constexpr int kInfo = 8;          // steps whose scales are kept
constexpr int kSegments = 4;      // segments the loader may be ahead

// TERMS 2: key and value tiles in two parts (float16 pools)
template <int D, int NG, int TERMS>
struct Shape4 {
  // threads a row in the softmax: two, as in the wide blocks of the shared-prefix
  // kernel (chunks of 512 tokens over 4096: 403 us against 431 with one)
  static constexpr int TPR = 2;
  static constexpr int kTile = kTileRows * TPR;  // softmax threads of a row tile
  // the softmax warps, then a warpgroup of 2 K and 2 V warps, and one of the
  // loader and NT MMA warps
  static constexpr int kSoft = 4 * NT * TPR;
  static constexpr int kThreads = 32 * (kSoft + 8);
  // registers: the launch's share, then the softmax's, the producers', the rest's
  static constexpr int kLaunchRegs = 80, kSoftRegs = 88, kMakeRegs = 72, kRestRegs = 56;
  static_assert(kSoft * kSoftRegs + 4 * (kMakeRegs + kRestRegs) <= (kSoft + 8) * kLaunchRegs,
                "more registers than the block is launched with");
  static constexpr uint32_t TB = kKeys * D * 2;  // (a part of) a K or V tile
  static constexpr uint32_t RB = (kKeys / kUnit) * Unit4<D, NG>::kBytes;  // a step's raw units
  // stages of K and V tiles, and of raw units
  static constexpr int KS = 2, VS = 2, RS = TERMS == 2 ? 2 : 3;
  // a query tile's place also takes its output rows, 2 D bytes each and 16 more
  static constexpr uint32_t QB = kTileRows * D * 2 + kTileRows * 16;
  static constexpr uint32_t oQ = 0, oK = NT * QB, oV = oK + KS * TERMS * TB,
                            oR = oV + VS * TERMS * TB, oMeta = oR + RS * RB;
  // barriers: a row tile's queries, and their place free; a stage's K and V; a
  // score buffer's S, P and PV of a row tile; a row's maxima; raw units there, and
  // read; a segment said, and read
  static constexpr uint32_t bQ = 0, bFree = bQ + 8 * NT, bK = bFree + 8 * NT, bV = bK + 16,
                            bS = bV + 16, bP = bS + 16 * NT, bPV = bP + 16 * NT,
                            bMax = bPV + 16 * NT, bR = bMax + 32 * NT, bRead = bR + 8 * RS,
                            bSeg = bRead + 8 * RS,
                            bSegRead = bSeg + 8 * kSegments, oTmem = bSegRead + 8 * kSegments,
                            oAbort = oTmem + 4, oWalked = oAbort + 4, oFlag = oWalked + 4,
                            oScale = oFlag + 4 * kInfo, oPower = oScale + 8 * kInfo,
                            oBad = oPower + 8 * kInfo, oRow = oBad + kInfo * kKeys,
                            oMax = oRow + NT * kTileRows * 4,
                            oSeg = oMax + NT * 2 * 2 * 128 * 4,
                            oSums = (oSeg + 48 * kSegments + 7) / 8 * 8,
                            kMeta = oSums + 96;
  static_assert(oR % 1024 == 0 && RB % 128 == 0 && oTmem % 4 == 0 && oRow % 4 == 0, "alignment");
  static constexpr uint32_t kSmem = oMeta + kMeta + 1024;  // the base is rounded up to 1024
  static_assert(kSmem <= 232448, "shared memory");
  static constexpr uint32_t kCols = 256 * NT;
  // two score buffers of 64 columns at 128 i for row tile i, O at cO + D i
  static constexpr uint32_t cS = 0, cO = 128 * NT;
};

struct Segment {  // of a row tile's steps, for a block
  int start;                // its first token's row
  int g, row0, rows, tiles; // KV head, first row, rows and row tiles
  int s0, steps;            // steps -1: no more segments
  int seen, first_limit;    // keys its last token sees; the newest key of token 0
  int part;                 // place of its partial results; -1: writes the output
};

template <int R> __device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R> __device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }

// eight codes as low + scale code, pairs (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ uint4 decode8(uint32_t w, __half2 scale, __half2 low) {
  const uint32_t magic = 0x64006400u;  // 1024; codes in bits 0 .. 3, or 4 .. 7 (16 times them)
  const __half2 k1024 = as_half2(magic), sixteenth = as_half2(0x2c002c00u),
                k64 = as_half2(0xd400d400u);  // -64
  const uint32_t y = w >> 8;
  const __half2 a = __hsub2(as_half2((w & 0x000f000fu) | magic), k1024);
  const __half2 b = __hfma2(as_half2((w & 0x00f000f0u) | magic), sixteenth, k64);
  const __half2 c = __hsub2(as_half2((y & 0x000f000fu) | magic), k1024);
  const __half2 d = __hfma2(as_half2((y & 0x00f000f0u) | magic), sixteenth, k64);
  return make_uint4(as_u32(__hfma2(a, scale, low)), as_u32(__hfma2(b, scale, low)),
                    as_u32(__hfma2(c, scale, low)), as_u32(__hfma2(d, scale, low)));
}
// where element d of eight lies in that order
__host__ __device__ constexpr int place8(int d) { return 2 * (d & 3) + (d >> 2 & 1); }

// the same in two parts: scale (code - zero), for a scale of 7 significant bits
// exact, and low + more (code - zero); `zero` is 1024 + the code nearest to zero
__device__ __forceinline__ void decode8(uint32_t w, __half2 scale, __half2 more, __half2 low,
                                        __half2 zero, uint4& main, uint4& rest) {
  const uint32_t magic = 0x64006400u;
  const __half2 sixteenth = as_half2(0x2c002c00u), k960 = as_half2(0x63806380u);
  const __half2 zero16 = __hsub2(k960, zero);  // -(64 + the code)
  const uint32_t y = w >> 8;
  const __half2 a = __hsub2(as_half2((w & 0x000f000fu) | magic), zero);
  const __half2 b = __hfma2(as_half2((w & 0x00f000f0u) | magic), sixteenth, zero16);
  const __half2 c = __hsub2(as_half2((y & 0x000f000fu) | magic), zero);
  const __half2 d = __hfma2(as_half2((y & 0x00f000f0u) | magic), sixteenth, zero16);
  main = make_uint4(as_u32(__hmul2(a, scale)), as_u32(__hmul2(b, scale)), as_u32(__hmul2(c, scale)),
                    as_u32(__hmul2(d, scale)));
  rest = make_uint4(as_u32(__hfma2(a, more, low)), as_u32(__hfma2(b, more, low)),
                    as_u32(__hfma2(c, more, low)), as_u32(__hfma2(d, more, low)));
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const char* p) {
  if constexpr (N == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(Shape4<D, NG, std::is_same<T, __half>::value ? 2 : 1>::kThreads,
                                  1)
    kv4_sm100_kernel(const __grid_constant__ Attn4 a) {
  constexpr int TERMS = std::is_same<T, __half>::value ? 2 : 1;
  using Sh = Shape4<D, NG, TERMS>;
  using U = Unit4<D, NG>;
  constexpr int RT = kWideRows, W = U::W, WG = W / NG, KS = Sh::KS, RS = Sh::RS;
  using Share = Share4<RT, kKeys>;
  extern __shared__ char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  char* smem = smem_raw + (sbase - raw);
  const uint32_t mb = sbase + Sh::oMeta;
  char* meta = smem + Sh::oMeta;
  volatile int* abort = reinterpret_cast<volatile int*>(meta + Sh::oAbort);
  volatile int* walked = reinterpret_cast<volatile int*>(meta + Sh::oWalked);
  volatile int* flag = reinterpret_cast<volatile int*>(meta + Sh::oFlag);  // step + 1: bad values
  // 2^E of 32 keys, and E of 32 values: [step % kInfo][half]
  volatile float* key_scale = reinterpret_cast<volatile float*>(meta + Sh::oScale);
  volatile float* val_power = reinterpret_cast<volatile float*>(meta + Sh::oPower);
  uint8_t* bad = reinterpret_cast<uint8_t*>(meta + Sh::oBad);  // [step % kInfo][key]: groups
  float* row_scale = reinterpret_cast<float*>(meta + Sh::oRow);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == Sh::kSoft + 5) tmem_alloc(mb + Sh::oTmem, Sh::kCols);
  if (tid == 0) {
    for (int k = 0; k < NT; ++k) {
      mbar_init(mb + Sh::bQ + 8 * k, Sh::kTile);
      mbar_init(mb + Sh::bFree + 8 * k, Sh::kTile / 32);
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(mb + Sh::bK + 8 * k, 64);
      mbar_init(mb + Sh::bV + 8 * k, 64);
    }
    for (int k = 0; k < 2 * NT; ++k) {
      mbar_init(mb + Sh::bS + 8 * k, 1);
      mbar_init(mb + Sh::bP + 8 * k, Sh::kTile);
      mbar_init(mb + Sh::bPV + 8 * k, 1);
    }
    for (int k = 0; k < 4 * NT; ++k) mbar_init(mb + Sh::bMax + 8 * k, 2);
    for (int k = 0; k < RS; ++k) {
      mbar_init(mb + Sh::bR + 8 * k, kKeys / kUnit);
      mbar_init(mb + Sh::bRead + 8 * k, 4);
    }
    for (int k = 0; k < kSegments; ++k) {
      mbar_init(mb + Sh::bSeg + 8 * k, 1);
      mbar_init(mb + Sh::bSegRead + 8 * k, Sh::kSoft + 4 + NT);
    }
    mbar_init_fence();
    for (int k = 0; k < kInfo; ++k) flag[k] = -1;
    *abort = 0;
    *walked = 0;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Share work;
  using Scratch = typename Share::template Scratch<128>;
  static_assert(sizeof(Scratch) <= Sh::kMeta - Sh::oSums, "its place");
  const bool ordered = work.template find<128>(a, blockIdx.x, gridDim.x, kLeastSteps,
                                               *reinterpret_cast<Scratch*>(meta + Sh::oSums));
  zero_rest<T, D>(a, ordered);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(meta + Sh::oTmem);

  // Steps are counted over the whole block, those of the second row tile (which
  // not every segment has) apart; step n uses score buffer n & 1 of its row tile.
  auto at = [&](uint32_t bar, int qt, int n) { return mb + bar + 8 * (2 * qt + (n & 1)); };
  // The loader says what the block's segments are; every other role walks them
  // for itself.  What keeps them apart are the barriers of the steps and the
  // order within a role: the next segment's keys are on their way, and their
  // first tiles made, while this one's rows are written.
  const Segment* segs = reinterpret_cast<const Segment*>(meta + Sh::oSeg);
  auto segments = [&](auto role) {
    for (int n = 0;; ++n) {
      const int k = n % kSegments;
      if (!warp_wait(mb + Sh::bSeg + 8 * k, (n / kSegments) & 1, abort)) break;
      if (segs[k].steps < 0) break;
      if (!role(segs[k])) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(mb + Sh::bSegRead + 8 * k);
    }
  };

  // The second row tile's MMA warp, having left out segments, must not look at a
  // step's K and V barriers before the steps in between are over (a parity tells
  // no phase from the last but one): the first tile's MMA warp, which walks every
  // step, says how many have their tiles.
  auto caught_up = [&](int qt, int n) {
    if (qt == 0 || *walked >= n) return true;
    const long long t0 = clock64();
    while (*walked < n) {
      if (*abort) return false;
      if (clock64() - t0 > kWaitCycles) {
        *abort = 1;
        return false;
      }
    }
    return true;
  };

  if (warp >= Sh::kSoft && warp < Sh::kSoft + 4) {
    // ============================================= producers: K, then V pair
    regs_down<Sh::kMakeRegs>();
    const bool isv = warp >= Sh::kSoft + 2;
    // a warp makes 32 keys' rows, with a power of two of their own; this thread's
    // part of every eight is the W words from word W c on of row r
    const int half = warp & 1, r = lane & 7, c = lane >> 3;
    int n = 0, n1 = 0;           // steps, and those of the second row tile
    int second[2] = {-1, -1};    // its step in the last two, if it had one
    segments([&](const Segment& seg) {
      const int steps = seg.steps, seen = seg.seen, first_key = seg.s0 * kKeys + 32 * half + r;
      const bool two = seg.tiles == 2;
      for (int t = 0; t < steps; ++t, ++n) {
        uint32_t code[4][W], pair[4][NG], values[4][NG];
        if (!warp_wait(mb + Sh::bR + 8 * (n % RS), (n / RS) & 1, abort)) return false;
        const char* units = smem + Sh::oR + (n % RS) * Sh::RB;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const char* p = units + (2 * half + j / 2) * U::kBytes;
          const int token = 8 * (j & 1) + r;
          load_words(code[j], p + (isv ? U::oV : 0) + token * U::kRow + 4 * W * c);
          load_words(pair[j], p + (isv ? U::oVp : U::oKp) + 4 * NG * token);
          if (!isv) load_words(values[j], p + U::oVp + 4 * NG * token);
        }
        // The stage may be filled again once these loads have come back, which an
        // arrival does not wait for by itself: it is made by a lane that a vote
        // over the loaded words names (any of two will do).
        uint32_t words = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int w = 0; w < W; ++w) words |= code[j][w];
#pragma unroll
          for (int k = 0; k < NG; ++k) words |= isv ? pair[j][k] : pair[j][k] | values[j][k];
        }
        if (lane == (__any_sync(~0u, words == 0x9e3779b9u) ? 1 : 0))
          mbar_arrive(mb + Sh::bRead + 8 * (n % RS));
        // ------------------------------- the powers of two, bad values
        // (the K warps look at the values' pairs too, and say with the key tile
        // what the softmax has to know of them)
        const int key0 = first_key + t * kKeys;
        auto reach_of = [&](uint32_t (&pairs)[4][NG], int least, uint32_t& wrong) {
          float reach = 0.f;
          wrong = 0u;  // bit NG j + k
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              if (key0 + 8 * j >= seen) pairs[j][k] = 0u;  // zeros: P is zero there too
              const float2 f = pair_of<T>(pairs[j][k]);
              const float m = fmaxf(fabsf(f.y), fabsf(fmaf(15.f, f.x, f.y)));
              if (m < INFINITY && f.x == f.x) reach = fmaxf(reach, m);
              else wrong |= 1u << (NG * j + k);
            }
          }
          // scale (code - zero), scale rounded to 7 bits, reaches 1.08 of this at
          // most, so two parts hold any number below 2^15; the keys (values) of a
          // warp that have larger ones are halved
          if constexpr (TERMS == 2) return __any_sync(~0u, reach >= 0x1p15f) ? 1 : 0;
          const uint32_t m = __reduce_max_sync(~0u, __float_as_uint(reach));
          return m == 0u ? 0 : min(114, max(least, (int)(m >> 23) - 127 - 13));
        };
        uint32_t wrong, wrong_values = 0u;
        // (the rows' sums, which are 2^-24 of theirs, take the values' power off again:
        // 2^104 times 2^15 of 2^31 keys)
        constexpr int kLeastKeys = -114, kLeastValues = -104;
        const int e = reach_of(pair, isv ? kLeastValues : kLeastKeys, wrong);
        const int ev = isv ? 0 : reach_of(values, kLeastValues, wrong_values);
        if (isv && wrong) {  // a bad value becomes 0 and marks the rows that see it
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int k = 0; k < NG; ++k)
              if (wrong >> (NG * j + k) & 1u) pair[j][k] = 0u;
          }
        }
        const float down = pow2(-e);
        if constexpr (TERMS == 2) {
          if (e) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
              for (int k = 0; k < NG; ++k)
                pair[j][k] = as_u32(__hmul2(as_half2(pair[j][k]), __float2half2_rn(0.5f)));
            }
          }
        }
        // --------------------------------------------------- a free stage
        const int stages = isv ? Sh::VS : KS;
        if (n >= stages) {
          const int u = n - stages, u1 = second[u & 1];
          const uint32_t bar = isv ? Sh::bPV : Sh::bS;
          if (!warp_wait(at(bar, 0, u), (u >> 1) & 1, abort) ||
              (u1 >= 0 && !warp_wait(at(bar, 1, u1), (u1 >> 1) & 1, abort)))
            return false;
        }
        second[n & 1] = two ? n1++ : -1;
        if (!isv) {
          const int info = n % kInfo;
          if (lane == 0) {
            key_scale[2 * info + half] = pow2(e);
            val_power[2 * info + half] = (float)ev;
          }
          if (c == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              bad[info * kKeys + 32 * half + 8 * j + r] =
                  (uint8_t)(wrong_values >> (NG * j) & ((1u << NG) - 1u));
          }
          if (wrong_values) flag[info] = n;
        }
        const uint32_t tile =
            sbase + (isv ? Sh::oV + (n % Sh::VS) * TERMS * Sh::TB
                         : Sh::oK + (n % KS) * TERMS * Sh::TB);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t to = tile + sw128(32 * half + 8 * j + r, 4 * w + c, kKeys);
            const uint32_t x = isv ? __byte_perm(code[j][w / 2], code[j][W / 2 + w / 2],
                                                 w & 1 ? 0x7632u : 0x5410u)
                                   : code[j][w];
            const float2 y = pair_of<T>(pair[j][w / WG]);
            if constexpr (TERMS == 1) {
              st_shared16(to, decode8(x, __float2half2_rn(y.x * down),
                                      __float2half2_rn(y.y * down)));
            } else {
              const uint32_t main = (pair[j][w / WG] + 8u) & 0xfff0u;  // 7 significant bits
              const float zero = fminf(fmaxf(rintf(-y.y * rcp_approx(y.x)), 0.f), 15.f);
              uint4 first, rest;
              decode8(x, as_half2(main * 0x10001u), __float2half2_rn(y.x - pair_of<T>(main).x),
                      __float2half2_rn(fmaf(zero, y.x, y.y)), __float2half2_rn(1024.f + zero),
                      first, rest);
              st_shared16(to, first);
              st_shared16(to + Sh::TB, rest);
            }
          }
        }
        fence_async_smem();
        mbar_arrive(mb + (isv ? Sh::bV + 8 * (n % Sh::VS) : Sh::bK + 8 * (n % KS)));
      }
      return true;
    });

  } else if (warp >= Sh::kSoft + 4) {
    // a warpgroup's warps give up registers at one instruction, before their roles part
    regs_down<Sh::kRestRegs>();
    if (warp == Sh::kSoft + 4) {
      // ============================================================ the loader
      bool bad_block = false;
      int which = 0;  // of this block's partial results
      int4 join = make_int4(-1, 0, 0, 0);
      int n = 0;  // steps
      for (int k = 0;; ++k) {
        Segment& s = reinterpret_cast<Segment*>(meta + Sh::oSeg)[k % kSegments];
        const uint32_t said = mb + Sh::bSeg + 8 * (k % kSegments);
        if (k >= kSegments && !warp_wait(mb + Sh::bSegRead + 8 * (k % kSegments),
                                         (k / kSegments - 1) & 1, abort))
          break;
        if (work.todo <= 0) {
          if (lane == 0) {
            s.steps = -1;
            mbar_arrive(said);
          }
          break;
        }
        const int all_steps = Share::steps(work.r, a.G, work.tile);
        const int s0 = work.step, s1 = (int)min((int64_t)all_steps, s0 + work.todo), g = work.head;
        const bool whole = s0 == 0 && s1 == all_steps;
        const int first_limit = work.r.len - work.r.n;
        const int seen = max(0, first_limit + Share::last_token(work.r, a.G, work.tile) + 1);
        const int steps = max(0, min(s1, (seen + kKeys - 1) / kKeys) - s0);
        if (lane == 0) {
          s.start = work.r.start;
          s.g = g;
          s.s0 = s0;
          s.row0 = work.tile * RT;
          s.rows = min(RT, work.r.n * a.G - s.row0);
          s.tiles = s.rows > kTileRows ? 2 : 1;
          s.first_limit = first_limit;
          s.seen = seen;
          s.steps = steps;
          s.part = whole ? -1 : 2 * (int)blockIdx.x + which;
          mbar_arrive(said);
        }
        if (!whole) {
          if (s0 == 0)  // the first of the tile's blocks has them joined
            join = make_int4(work.request, work.tile, 2 * g + which,
                             blockIdx.x + (int)((all_steps - s1 + work.per - 1) / work.per));
          which = 1;
        }
        const int32_t* table = a.tables + work.request * a.table_stride;
        const int units = (seen + kUnit - 1) / kUnit;
        int64_t from = -1;  // this lane's unit of eight steps: -1 none, 0 no block
        bool ok = true;
        for (int t = 0; ok && t < steps; ++t, ++n) {
          if (t % 8 == 0) {
            const int u = (s0 + t) * (kKeys / kUnit) + lane, j = u / a.pool.units;
            from = -1;
            if (u < units) {
              const int id = table[j];
              from = id >= 0 && id < a.pool.num_blocks
                         ? reinterpret_cast<int64_t>(a.pool.unit(id, g, u - j * a.pool.units))
                         : 0;
              bad_block |= from == 0;
            }
          }
          if (n >= RS) {
            ok = warp_wait(mb + Sh::bRead + 8 * (n % RS), (n / RS - 1) & 1, abort);
            if (!ok) break;
          }
          if (lane / 4 == t % 8) {
            const uint32_t bar = mb + Sh::bR + 8 * (n % RS);
            const uint32_t to = Sh::oR + (n % RS) * Sh::RB + (lane % 4) * U::kBytes;
            if (from > 0) {
              mbar_arrive_expect(bar, U::kBytes);
              bulk_copy(sbase + to, reinterpret_cast<const void*>(from), U::kBytes, bar);
            } else {
              if (from == 0) {  // zero codes, scales and lows: zero keys and values
                for (int m = 0; m < U::kBytes / 16; ++m)
                  st_shared16(sbase + to + 16 * m, make_uint4(0, 0, 0, 0));
                fence_async_smem();  // before a later copy into this place
              }
              mbar_arrive(bar);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        work.todo -= s1 - s0;
        if (work.todo > 0) work.next(a);
      }
      // nothing of this block's copies is in flight when it ends
      for (int u = n - RS < 0 ? 0 : n - RS; u < n; ++u) {
        const long long t0 = clock64();
        while (!mbar_try(mb + Sh::bR + 8 * (u % RS), (u / RS) & 1) &&
               clock64() - t0 < kWaitCycles) {
        }
      }
      if (lane == 0) a.joins[blockIdx.x] = join;
      if (bad_block) report(a.status, CS_ST_SLOT_RANGE);

    } else {
      // ==================================================== MMA, one warp a tile
      const int qt = __shfl_sync(~0u, warp, 0) - (Sh::kSoft + 5);
      const bool leader = elect_one();
      const uint32_t id_s = umma_idesc(128, kKeys, 0, 0, 0);
      const uint32_t id_o = umma_idesc(128, D, 0, 0, 1);  // V is MN-major
      const uint64_t dq = umma_desc(sbase + Sh::oQ + qt * Sh::QB, 16, 1024);
      const uint64_t dk0 = umma_desc(sbase + Sh::oK, 16, 1024);
      const uint64_t dv0 = umma_desc(sbase + Sh::oV, kKeys * 128, 1024);
      const uint32_t tm = __shfl_sync(~0u, tmem, 0);
      const uint32_t sc = tm + Sh::cS + 128 * qt, oc = tm + Sh::cO + D * qt;
      int n = 0, m = 0, queries = 0;  // steps of the block and of the row tile; its segments
      uint32_t last = 0, lastph = 0;  // the newest group issued
      auto drained = [&] {
        const long long t0 = clock64();
        while (last && !mbar_try(last, lastph) && clock64() - t0 < kWaitCycles) {
        }
        last = 0;
      };
      if (qt < NT) segments([&](const Segment& seg) {
        const int steps = seg.steps;
        if (qt < seg.tiles) {
          if (!warp_wait(mb + Sh::bQ + 8 * qt, queries++ & 1, abort) ||
              !__all_sync(~0u, caught_up(qt, n)))
            return false;
          auto arrived = [&](uint32_t bar, int u, int stages) {
            return warp_wait(mb + bar + 8 * (u % stages), (u / stages) & 1, abort);
          };
          auto scores = [&](int t) {
            if (!arrived(Sh::bK, n + t, KS)) return false;
            tc_fence_after();
            const uint64_t dk = dk0 + (uint64_t)(((n + t) % KS) * TERMS * (Sh::TB >> 4));
            const uint32_t sb = sc + kKeys * ((m + t) & 1);
            last = at(Sh::bS, qt, m + t);
            lastph = ((m + t) >> 1) & 1;
            if (leader) {
  #pragma unroll
              for (int term = 0; term < TERMS; ++term) {
  #pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)  // offsets in 16-byte units
                  tc_mma(sb, dq + (kk >> 2) * 1024 + (kk & 3) * 2,
                         dk + term * (Sh::TB >> 4) + (kk >> 2) * (kKeys * 8) + (kk & 3) * 2, id_s,
                         term + kk ? 1u : 0u);
              }
              tc_commit(last);
            }
            __syncwarp();
            return true;
          };
          for (int t = 0; t < 2 && t < steps; ++t)
            if (!scores(t)) return false;
          for (int t = 0; t < steps; ++t) {
            const uint32_t ph = ((m + t) >> 1) & 1;
            if (!arrived(Sh::bV, n + t, Sh::VS) || !warp_wait(at(Sh::bP, qt, m + t), ph, abort))
              return false;
            if (qt == 0 && lane == 0) *walked = n + t + 1;
            tc_fence_after();
            const uint64_t dv = dv0 + (uint64_t)(((n + t) % Sh::VS) * TERMS * (Sh::TB >> 4));
            const uint32_t p = sc + kKeys * ((m + t) & 1);
            last = at(Sh::bPV, qt, m + t);
            lastph = ph;
            if (leader) {
  #pragma unroll
              for (int term = 0; term < TERMS; ++term) {
  #pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk)
                  tc_mma_ts(oc, p + kk * 8, dv + term * (Sh::TB >> 4) + kk * 128, id_o,
                            (t | kk | term) ? 1u : 0u);
              }
              tc_commit(last);
            }
            __syncwarp();
            // the next scores but one take the buffer that P lies in
            if (t + 2 < steps &&
                (!warp_wait(at(Sh::bPV, qt, m + t), ph, abort) || !scores(t + 2)))
              return false;
          }
          drained();  // (the next segment's scores take both buffers)
          m += steps;
        }
        n += steps;
        return true;
      });
      drained();
      __syncwarp();
    }

  } else {
    // ================================================================= softmax
    regs_up<Sh::kSoftRegs>();
    int n = 0, m = 0, queries = 0;  // steps of the block and of the row tile; its segments
    int exchanges = 0;  // of maxima with the row's other thread
    segments([&](const Segment& seg) {
      const int row0 = seg.row0, steps = seg.steps, s0 = seg.s0;
      constexpr int TPR = Sh::TPR, VC = kKeys / TPR;  // scores of a step a thread holds
      static_assert(VC == 32, "the keys of one power of two");
      const int qt = warp / (4 * TPR), part2 = (warp >> 2) % TPR;
      if (qt >= seg.tiles) {
        n += steps;
        return true;
      }
      // all rows of the last segment are written: their places may take queries
      if (queries > 0 && !warp_wait(mb + Sh::bFree + 8 * qt, (queries - 1) & 1, abort))
        return false;
      const int r = (warp & 3) * 32 + lane;  // TMEM lane
      const int row = qt * kTileRows + r;    // of the block's
      const bool row_ok = row < seg.rows;
      {
        // queries into the swizzled operand layout, a power of two a row
        constexpr int C = D / 8;
        const int c = tid % C;
        const uint32_t qs = sbase + Sh::oQ + qt * Sh::QB;
        constexpr int kRows = kTileRows * C / Sh::kTile;  // a thread's, all fetched at once
        uint32_t x[kRows][4];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          const int q = qt * kTileRows + (tid % Sh::kTile) / C + k * (Sh::kTile / C);
          const bool ok = q < seg.rows;
          const int tk = ok ? (row0 + q) / a.G : 0;
          const char* p = a.q + (int64_t)(seg.start + tk) * a.qt +
                          (int64_t)(seg.g * a.G + (ok ? row0 + q - tk * a.G : 0)) * a.qh + 16 * c;
          if (ok && a.vec_q) {
            load_words(x[k], p);
          } else if (ok) {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int w = 0; w < 4; ++w) x[k][w] = u[2 * w] | (uint32_t)u[2 * w + 1] << 16;
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) x[k][w] = 0u;
          }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          const int q = (tid % Sh::kTile) / C + k * (Sh::kTile / C);
          float f[8], top = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 y = pair_of<T>(x[k][w] ^ a.flip);
            f[2 * w] = y.x, f[2 * w + 1] = y.y;
            top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));
          }
#pragma unroll
          for (int o = 1; o < C; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
          const int e = min(114, max(-100, (int)(__float_as_uint(top) >> 23) - 127 - 13));
          const float up = pow2(-e);
          if (c == 0) row_scale[qt * kTileRows + q] = pow2(e);
          uint32_t y[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) y[w] = Pack2<__half>::pack(f[w] * up, f[w + 4] * up);
          st_shared16(qs + sw128(q, c, kTileRows), make_uint4(y[0], y[1], y[2], y[3]));
        }
        fence_async_smem();
        mbar_arrive(mb + Sh::bQ + 8 * qt);
      }
      bool ok = warp_wait(mb + Sh::bQ + 8 * qt, queries++ & 1, abort);
      const float row_factor = row_scale[qt * kTileRows + r] * a.scale2;
      // the newest key this row sees; no row: of no matter
      const int limit = row_ok ? seg.first_limit + (row0 + row) / a.G : INT32_MAX;
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t sc0 = tmem + lane_base + Sh::cS + 128 * qt;
      const uint32_t oc = tmem + lane_base + Sh::cO + D * qt;
      float mref = -INFINITY, lsum = 0.f;  // log2 domain; P = 2^(x + E - mref + up)
      uint32_t poison = 0u;  // groups of values that are not finite and that the row sees
      const uint32_t pair = mb + Sh::bMax + 8 * (4 * qt + (warp & 3));
      float* row_max = reinterpret_cast<float*>(meta + Sh::oMax) + qt * 512;
      const bool any_row = __any_sync(~0u, row_ok);
      auto wait_pv = [&](int t) {
        ok = warp_wait(at(Sh::bPV, qt, m + t), ((m + t) >> 1) & 1, abort);
        tc_fence_after();
        return ok;
      };

      for (int t = 0; ok && t < steps; ++t) {
        const int base = (s0 + t) * kKeys;
        const int vhi = limit - base >= kKeys ? kKeys : limit - base + 1;  // keys seen
        const uint32_t sc = sc0 + kKeys * ((m + t) & 1);
        const int info = (n + t) % kInfo;
        ok = warp_wait(at(Sh::bS, qt, m + t), ((m + t) >> 1) & 1, abort);
        if (!ok) break;  // a wait expired
        tc_fence_after();
        uint32_t v[VC];
        // both threads of a row leave this way together
        if (!any_row || __all_sync(~0u, vhi <= 0)) {  // nothing to see for these 32 rows
#pragma unroll
          for (int c = 0; c < 16; ++c) v[c] = 0u;
          CS_TMEM_ST16(sc + 16 * part2, v);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(at(Sh::bP, qt, m + t));
          continue;
        }
        CS_TMEM_LD32(sc + 32 * part2, v);
        float power = val_power[2 * info + part2];
        const float factor = fmaxf(row_factor * key_scale[2 * info + part2], 1e-30f);
        tmem_wait_ld();
        if (!__all_sync(~0u, vhi >= kKeys)) {
          const uint32_t bits = col_bits(0, vhi, 32 * part2);
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = (bits >> c) & 1u ? v[c] : 0xff800000u;  // -inf
        }
        if (flag[info] == n + t) {
          for (int c = 0; c < VC; ++c) {
            const int key = 32 * part2 + c;
            if (key < vhi) poison |= bad[info * kKeys + key];
          }
        }
        float top;  // of log2 of the weights, with the values' power
        {
          float m4[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            m4[k] = max_nan(__uint_as_float(v[k]), __uint_as_float(v[k + 4]));
#pragma unroll
          for (int c = 8; c < 32; c += 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              m4[k] = max3_nan(m4[k], __uint_as_float(v[c + k]), __uint_as_float(v[c + k + 4]));
          }
          top = fmaf(max_nan(max3_nan(m4[0], m4[1], m4[2]), m4[3]), factor, power);
        }
        // the row's maximum from both its threads; past this barrier both have
        // read their scores, so P may take their columns
        float* mx = row_max + (exchanges & 1) * 256;
        mx[part2 * 128 + r] = top;
        const float own = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        ok = warp_wait(pair, exchanges & 1, abort);
        if (!ok) break;
        ++exchanges;
        top = max_nan(top, mx[(1 - part2) * 128 + r]);
        if (!(top < INFINITY)) {  // a NaN or +inf score makes the row NaN
          lsum = __int_as_float(0x7fffffff);
          top = -INFINITY;
        }
        const bool grow = top > mref + kLazy || mref == -INFINITY;
        const bool rescale = grow && mref > -INFINITY && top > mref;
        // weights that leave float32 beside larger values' (own: not the masked -inf)
        const bool faint = own < (grow ? top : mref) - kFaint && own > -INFINITY;
        if (__any_sync(~0u, rescale || faint)) {
          if (__any_sync(~0u, rescale)) {  // t > 0: a row has a finite maximum
            if (!wait_pv(t - 1)) break;
            // the root, since the reference may rise by more than float32's range;
            // the sums of weights without the values' powers keep theirs
            const float h = rescale ? ex2(0.5f * (mref - top)) : 1.f, f = h * h;
            lsum = lsum * h * h;
            uint32_t o[16];
#pragma unroll 1
            for (int cc = 0; cc < D / 16 / TPR; ++cc) {
              const uint32_t col = oc + part2 * (D / 2) + 16 * cc;
              CS_TMEM_LD16(col, o);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              CS_TMEM_ST16(col, o);
            }
            tmem_wait_st();
          }
          if (faint) {  // these weights count in the sum alone, and are zeros below
            const float off = kUp - (grow ? top : mref);
#pragma unroll
            for (int c = 0; c < VC; ++c)
              lsum = fmaf(ex2(fmaf(__uint_as_float(v[c]), factor, off)), kSumDown, lsum);
            power -= 126.f - kFaint + kUp;
          }
        }
        if (grow) mref = top;
        const float less = power - ((mref > -INFINITY ? mref : 0.f) - kUp);
        const float2 scale = make_float2(factor, factor), off = make_float2(less, less);
        float2 p0 = make_float2(0.f, 0.f), p1 = p0;
#pragma unroll
        for (int c = 0; c < VC; c += 2) {
          const float2 x = __ffma2_rn(
              make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale, off);
          v[c] = __float_as_uint(x.x);
          v[c + 1] = __float_as_uint(x.y);
        }
#pragma unroll
        for (int c = 0; c < VC; ++c) v[c] = __float_as_uint(ex2(__uint_as_float(v[c])));
#pragma unroll
        for (int c = 0; c < VC; c += 4) {
          p0 = __fadd2_rn(p0, make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])));
          p1 = __fadd2_rn(p1, make_float2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])));
        }
        // (in two steps: the power goes from -137 to 114)
        lsum = fmaf(((p0.x + p0.y) + (p1.x + p1.y)) * 0x1p-12f, ex2(-12.f - power), lsum);
#pragma unroll
        for (int c = 0; c < VC / 2; ++c)
          v[c] = Pack2<__half>::pack(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]));
        CS_TMEM_ST16(sc + 16 * part2, v);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(at(Sh::bP, qt, m + t));
      }

      // -------------------------------------------------------------- output
      if (ok && steps > 0) wait_pv(steps - 1);
      // the row's sum and bad groups from both its threads
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        float* both = row_max + (exchanges & 1) * 256;
        both[part2 * 128 + r] = turn ? __uint_as_float(poison) : lsum;
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        ok = ok && warp_wait(pair, exchanges & 1, abort);
        ++exchanges;
        const float other = both[(1 - part2) * 128 + r];
        if (turn) poison |= __float_as_uint(other);
        else lsum += other;
      }
      // (the sum from 2^-131 to 2^126: its reciprocal in float32's range)
      const float up = lsum < 0x1p-60f ? 0x1p64f : 1.f, down = up * kSumDown;
      const float inv = lsum == 0.f ? 0.f : 1.f / (lsum * up);
      const float lse2 = lsum == 0.f ? -INFINITY
                                     : (mref > -INFINITY ? mref : 0.f) - kUp + (log2f(lsum) + 24.f);
      const int tok = (row0 + row) / a.G, h = seg.g * a.G + (row0 + row - tok * a.G);
      const bool whole = seg.part < 0;
      const int64_t prow = (int64_t)seg.part * RT + row;
      char* orow = whole ? a.out + (int64_t)(seg.start + tok) * a.ot + (int64_t)h * a.oh
                         : reinterpret_cast<char*>(a.part_o + prow * D);
      const bool have = ok && steps > 0 && lsum != 0.f;
      const bool write = ok && row_ok;
      // element d of this thread's columns, which are loaded from column c0 on
      auto final = [&](const uint32_t* v, int c0, int d) {
        const float x = __uint_as_float(v[(d & ~7) + place8(d & 7)]);
        const int group = (part2 * (D / 2) + c0 + d) / 32 / WG;
        return poison >> group & 1u ? __int_as_float(0x7fffffff) : have ? x * down * inv : 0.f;
      };
      if (!whole || a.vec_out) {
        // each thread stages its row where the queries were, and the warp
        // writes whole rows: 32-bit partials in two halves
        constexpr int B = 2 * D / TPR;  // bytes of a row a thread stages at once
        constexpr int L = B / 16;       // lanes that write them
        constexpr int WR = 2 * D + 16;
        const uint32_t stage = sbase + Sh::oQ + qt * Sh::QB + (r - lane) * WR + part2 * B;
        const uint32_t buf = stage + lane * WR;
        const uint64_t to = write ? reinterpret_cast<uint64_t>(orow) : 0;
#pragma unroll 1
        for (int round = 0; round < (whole ? 1 : 2); ++round) {
          uint32_t v[32];
          const uint32_t col = oc + part2 * (D / 2);
          if (!whole) {
#pragma unroll
            for (int cc = 0; cc < B / 64; ++cc) {
              const int c0 = round * (B / 4) + 16 * cc;
              CS_TMEM_LD16(col + c0, v);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 16; d += 4)
                st_shared16(buf + 64 * cc + 4 * d,
                            make_uint4(__float_as_uint(final(v, c0, d)),
                                       __float_as_uint(final(v, c0, d + 1)),
                                       __float_as_uint(final(v, c0, d + 2)),
                                       __float_as_uint(final(v, c0, d + 3))));
            }
          } else {
#pragma unroll
            for (int cc = 0; cc < B / 64; ++cc) {
              CS_TMEM_LD32(col + 32 * cc, v);
              tmem_wait_ld();
#pragma unroll
              for (int d = 0; d < 32; d += 8) {
                uint32_t y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  y[k] = mean_pair<T>(final(v, 32 * cc, d + 2 * k),
                                      final(v, 32 * cc, d + 2 * k + 1));
                st_shared16(buf + 64 * cc + 2 * d, make_uint4(y[0], y[1], y[2], y[3]));
              }
            }
          }
          __syncwarp();
          // a partial's thread has two rounds, an output's one
          const int64_t at0 = whole ? part2 * B : (part2 * 2 + round) * B;
#pragma unroll
          for (int n0 = 0; n0 < L; n0 += 4) {
            uint4 x[4];
            uint64_t dst[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int rw = (n0 + n) * (32 / L) + lane / L;
              dst[n] = __shfl_sync(~0u, to, rw);
              x[n] = ld_shared16(stage + rw * WR + 16 * (lane % L));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              if (!dst[n]) continue;
              uint2* y = reinterpret_cast<uint2*>(dst[n] + at0 + 16 * (lane % L));
              y[0] = make_uint2(x[n].x, x[n].y);
              y[1] = make_uint2(x[n].z, x[n].w);
            }
          }
          __syncwarp();
        }
      } else {
#pragma unroll 1
        for (int cc = 0; cc < D / 32 / TPR; ++cc) {
          uint32_t v[32];
          const int col = part2 * (D / 2) + 32 * cc;
          CS_TMEM_LD32(oc + col, v);
          tmem_wait_ld();
          if (!write) continue;
#pragma unroll
          for (int d = 0; d < 32; ++d)
            reinterpret_cast<T*>(orow)[col + d] = Elem<T>::from_f(mean_of<T>(final(v, 32 * cc, d)));
        }
      }
      if (write && part2 == 0) {
        if (whole) write_lse(a, seg.start, row0 + row, seg.g, lse2);
        else a.part_lse[prow] = lse2;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(mb + Sh::bFree + 8 * qt);
      n += steps;
      m += steps;
      return ok;
    });
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort) report(a.status, CS_ST_TIMEOUT);
  if (warp == Sh::kSoft + 5) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kCols);
  }
}

// The register split inside the kernel is made for a launch at this many a
// thread: with another number a warpgroup could wait for registers for ever.
template <auto Kernel>
bool launched_with(int regs) {
  static const int have = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, Kernel) == cudaSuccess ? f.numRegs : -1;
  }();
  return have == regs;
}

template <typename T, int D, int NG>
int launch_wide(const Attn4& a, int workers, cudaStream_t stream) {
  using Sh = Shape4<D, NG, std::is_same<T, __half>::value ? 2 : 1>;
  constexpr auto kernel = kv4_sm100_kernel<T, D, NG>;
  if (!allow_smem<kernel>(Sh::kSmem) || !launched_with<kernel>(Sh::kLaunchRegs))
    return CS_ERR_CUDA;
  if (const int rc = launch_dependent(kernel, dim3(workers), Sh::kThreads, Sh::kSmem, stream, a))
    return rc;
  return launch_join<T, D, kWideRows>(a, workers, stream);
}

}  // namespace

int kv4_wide(const Attn4& a, const cs_kv4_pool& pool, int workers, cudaStream_t stream) {
  return by_pool4(pool, [&](auto* t, auto d, auto g) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_wide<T, decltype(d)::value, decltype(g)::value>(a, workers, stream);
  });
}

}  // namespace cs
