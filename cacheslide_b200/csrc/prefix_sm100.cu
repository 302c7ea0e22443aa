// Tensor-core attention behind shared prefixes for sm_100a (tcgen05, TMEM,
// TMA), and the join of its partial results.
//
// One block takes one work item of the plan for one KV head: up to NT tiles
// of 128 query rows (128 / G tokens x the G query heads of the KV head) and
// the item's keys, first its range of the prefix, then its range of the own
// keys, in steps of 64.  Per step
//   S = Q K^T (tcgen05, TMEM),  P = 2^(S c - m),  O += P V (P from TMEM)
// with the running maximum m and sum of each row in float32 registers; P is
// rounded to the inputs' type, as the tensor unit takes it, and the sum is
// taken before that: outputs lie 2.3e-3 (bf16) and 2.9e-4 (fp16) from float64,
// 1.7e-3 and 2.1e-4 of which their own rounding is; the rest of P as a second
// 16-bit operand would be another product as large as P V.  Every row sees the whole prefix range; of the own keys
// it sees [lo, hi) of its token, which covers the causal limit, requests of
// other lengths in the same tile and padding alike.
//
// Warps: softmax (one thread a row, two in the wide block), a K and a V
// producer, NT MMA issuers.  Scores have two buffers a row tile, so that the
// next step's product runs beside this step's softmax.  Keys come through the
// slot arrays: TMA boxes of 64 x 16 for runs of 16 keys in consecutive rows
// of the pool, 16-byte cp.async row by row for the rest (scattered slots, the
// sidecar, range ends, which are filled with zeros, and pools no tensor map
// describes).
//
// Measured with 32/8 heads of 128, bf16 (64/8 and fp16 where said), twelve
// calls in a row:
//   64 questions of 64 tokens behind 5120 keys: 336 us, 1.03 PFLOP/s (368 us,
//     0.94 PFLOP/s, sustained, under the power limit); bound by the softmax
//     warps: 64 keys of two row tiles take 1950 clocks, of which the
//     exponentials, at 8 clocks a warp instruction, take 1024;
//   8 decodes behind 65536 keys (64/8): 54 us, 5.0 TB/s;
//   32 sessions of 4 drafts, own keys up to 16K (fp16): 216 us, 5.1 TB/s (245
//     us sustained: the power limit takes the clock to 1.55 GHz);
//   64 decodes behind 5120 keys: 24 us, of which 9 are the block's eight
//     steps of 1500 clocks and 5 the join: latency.
#include <cuda.h>
#include <math.h>

#include <numeric>
#include <type_traits>

#include "prefix.cuh"
#include "sm100.cuh"
#include "tma_rows.cuh"

namespace cs {
namespace {

constexpr int kKeys = 64;  // keys of a step: one K and V tile, scores, softmax, P V
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kKinds = 3;  // of values that are not finite: NaN, +inf, -inf

struct PArgs {
  CUtensorMap tm;  // the pool's rows in boxes of 64 x 16
  PagedView pv;
  const char* q;
  int64_t qt, qh;  // byte strides
  char* out;
  int64_t ot, oh;
  float* lse;
  const int64_t* prefix_slots;
  const int64_t* suffix_slots;
  const int4* tokens;
  const PrefixItem* items;
  float* part_o;    // [part token][query head][dim], normalised
  float* part_lse;  // [part token][query head], log2 of the softmax denominator
  int32_t* status;
  int64_t nrb, nrh, nro;  // block, head, offset -> map row
  int hq, hkv, G, R;  // R: tokens a row tile
  int bs_shift;       // log2(block size), -1 when it is no power of two
  int tma;            // 1: tensor maps describe the pool
  int vec_q, vec_out; // 16-byte loads / stores fit
  int neg;            // the scale is negative: the queries are negated
  float scale2;       // |scale| * log2 e
};

template <typename T> constexpr int umma_format() { return std::is_same<T, __half>::value ? 0 : 1; }
// P is stored as 2^(x - m + kUp): fp16's normal numbers then reach 2^-21 of the
// row's largest weight, and 2^(kUp + kLazy) stays below its maximum
template <typename T> constexpr float p_up() { return std::is_same<T, __half>::value ? 7.f : 0.f; }
constexpr float kLazy = 8.f;  // O is rescaled when the maximum grew by more than 2^8

template <int D, int NT>
struct Shape {
  // key tiles in flight; two blocks of one row tile share an SM
  static constexpr int KS = NT == 2 ? 4 : 2, VS = KS;
  // A stage of two is free with the product before last, whose barrier cannot
  // move on before the stage is filled again; deeper rings have barriers of
  // their own for "read".
  static constexpr bool kDirect = KS == 2;
  // threads a row in the softmax: two where one block has the SM (64 questions
  // of 64 tokens behind 5120 keys: 357 us against 367 with one), one where two
  // blocks share it (32 sessions of 4 drafts: 208 us against 224 with two).
  // Making the row tiles' exponentials take turns, or start half a step apart,
  // cost more than it gave (364 and 366 us).
  static constexpr int TPR = NT;
  static constexpr int kTile = 128 * TPR;  // softmax threads of a row tile
  // the softmax warps, then K, V and NT MMA warps, to a whole warpgroup
  static constexpr int kSoft = 4 * NT * TPR;
  static constexpr int kThreads = kTile * NT + 128;
  static constexpr uint32_t TB = kKeys * D * 2;  // a K or V tile
  // a query tile's place also takes its output rows, 2 D bytes each and 16 more
  static constexpr uint32_t QB = kPrefixTile * D * 2 + 128 * 16;
  static constexpr uint32_t oQ = 0, oK = NT * QB, oV = oK + KS * TB, oMeta = oV + VS * TB;
  // barriers, 8 bytes each; S, P and PV a score buffer of a row tile, K / V and
  // their "read" barriers a stage
  static constexpr uint32_t bQ = 0, bK = 8, bV = bK + 8 * KS, bKr = bV + 8 * VS,
                            bVr = bKr + 8 * KS, bS = bVr + 8 * VS, bP = bS + 16 * NT,
                            bPV = bP + 16 * NT, bMax = bPV + 16 * NT, oTmem = bMax + 32 * NT,
                            oAbort = oTmem + 4,
                            oAgain = oAbort + 4, bClean = oAgain + 8, oFound = bClean + 8,
                            oRows = (oFound + 8 + 15) / 16 * 16,
                            oMax = oRows + 2 * kKeys * 8, oBad = oMax + NT * 2 * 2 * 128 * 4,
                            kMeta = oBad + 2 * kKinds * kKeys * (D / 8);
  static_assert(oMeta % 1024 == 0 && oRows % 16 == 0 && oTmem % 4 == 0 && bClean % 8 == 0 &&
                    oBad % 16 == 0,
                "alignment of the shared-memory places");
  static constexpr uint32_t kSmem = oMeta + kMeta + 1024;  // the base is rounded up to 1024
  static constexpr uint32_t kCols = 256 * NT;
  // two score buffers of 64 columns at 128 i for row tile i, O at cO + D i
  static constexpr uint32_t cS = 0, cO = 128 * NT;
};

struct Step {
  int base, n, own;  // first key, keys, 1: own keys
};
__device__ __forceinline__ Step step_of(const PrefixItem& it, int na, int t) {
  Step s;
  s.own = t >= na;
  s.base = s.own ? it.b0 + (t - na) * kKeys : it.a0 + t * kKeys;
  const int end = s.own ? it.b1 : it.a1;
  s.n = end - s.base < kKeys ? end - s.base : kKeys;
  return s;
}

// where the keys of one lane (2 consecutive keys of a tile) come from
struct Src {
  uint64_t at[2];  // the K or V half of the record; 0: none (beyond the range, or no valid slot)
  int row;         // row of the tensor map of the first key
  bool run;        // the two lie in consecutive rows of the pool's map
};

// bits of the elements of a 16-bit pair that are not finite (0, 1), and the pair
// without them
template <typename T>
__device__ __forceinline__ uint32_t take_out(uint32_t& x) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const bool lo = (x & e) == e, hi = (x & (e << 16)) == (e << 16);
  if (lo) x &= 0xffff0000u;
  if (hi) x &= 0x0000ffffu;
  return (lo ? 1u : 0u) | (hi ? 2u : 0u);
}
// of those, the NaN ones (mantissa not 0), given the pair as it was
template <typename T>
__device__ __forceinline__ uint32_t nan_bits(uint32_t x, uint32_t bad) {
  constexpr uint32_t m = std::is_same<T, __half>::value ? 0x03ffu : 0x007fu;
  return bad & ((x & m ? 1u : 0u) | (x & (m << 16) ? 2u : 0u));
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, NT == 1 ? 2 : 1)
    prefix_sm100_kernel(const __grid_constant__ PArgs a) {
  using Sh = Shape<D, NT>;
  extern __shared__ char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  char* smem = smem_raw + (sbase - raw);
  const uint32_t mb = sbase + Sh::oMeta;
  volatile int* abort = reinterpret_cast<volatile int*>(smem + Sh::oMeta + Sh::oAbort);
  volatile int* again = reinterpret_cast<volatile int*>(smem + Sh::oMeta + Sh::oAgain);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = blockIdx.x % a.hkv;
  const PrefixItem it = a.items[blockIdx.x / a.hkv];
  const int na = (it.a1 - it.a0 + kKeys - 1) / kKeys;
  const int steps = na + (it.b1 - it.b0 + kKeys - 1) / kKeys;
  const int tiles = NT == 2 && it.ntok > a.R ? 2 : 1;

  // (producers) the slots of a key tile are read three tiles ahead: beside the
  // streams of K and V such a read takes 2500 clocks
  bool slot_bad = false;
  const bool isv = warp != Sh::kSoft;
  struct Slots {
    int64_t s[2];
  };
  auto load_slots = [&](int t) {
    Slots r{{-1, -1}};
    if (t < steps) {
      const Step st = step_of(it, na, t);
      const int64_t* slots = (st.own ? a.suffix_slots : a.prefix_slots) + st.base;
#pragma unroll
      for (int m = 0; m < 2; ++m)
        if (2 * lane + m < st.n) r.s[m] = slots[2 * lane + m];
    }
    return r;
  };
  // rows of the pool's map, for two keys in one block (32-bit arithmetic: a map
  // has fewer than 2^31 rows, and there is none for larger pools)
  auto resolve = [&](const Slots& in, Src& s) {
    const uint32_t s0 = (uint32_t)in.s[0];
    s.run = a.tma != 0 && in.s[0] >= 0 && in.s[1] == in.s[0] + 1 && in.s[1] < a.pv.native_total;
    const uint32_t b = s.run ? (a.bs_shift >= 0 ? s0 >> a.bs_shift : s0 / (uint32_t)a.pv.bs) : 0u;
    const uint32_t o = s0 - b * (uint32_t)a.pv.bs;
    s.run = s.run && o + 1 < (uint32_t)a.pv.bs;
    s.row = (int)(b * (uint32_t)a.nrb + g * (uint32_t)a.nrh + o);
  };
  auto addresses = [&](int t, const Slots& in, Src& s) {
    const Step st = step_of(it, na, t);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s.at[m] = 0;
      const int64_t sl = in.s[m];
      if (a.pv.valid(sl)) {
        if (sl < a.pv.native_total) {
          const int64_t b = a.bs_shift >= 0 ? sl >> a.bs_shift : sl / a.pv.bs;
          const int64_t o = sl - (a.bs_shift >= 0 ? b << a.bs_shift : b * a.pv.bs);
          s.at[m] = reinterpret_cast<uint64_t>(a.pv.cache) + b * a.pv.sb + g * a.pv.sh +
                    o * a.pv.so + (isv ? 2 * D : 0);
        } else {
          s.at[m] = reinterpret_cast<uint64_t>(isv ? a.pv.side_v : a.pv.side_k) +
                    (sl - a.pv.native_total) * a.pv.ssr + g * a.pv.ssh;
        }
      } else if (2 * lane + m < st.n) {
        slot_bad = true;
      }
    }
  };
  auto init_barriers = [&] {
    mbar_init(mb + Sh::bQ, Sh::kTile * tiles);
    for (int s = 0; s < Sh::KS; ++s) mbar_init(mb + Sh::bK + 8 * s, 32);
    for (int s = 0; s < Sh::VS; ++s) mbar_init(mb + Sh::bV + 8 * s, 32);
    for (int s = 0; s < Sh::KS; ++s) mbar_init(mb + Sh::bKr + 8 * s, tiles);
    for (int s = 0; s < Sh::VS; ++s) mbar_init(mb + Sh::bVr + 8 * s, tiles);
    for (int s = 0; s < 2 * NT; ++s) {
      mbar_init(mb + Sh::bS + 8 * s, 1);
      mbar_init(mb + Sh::bP + 8 * s, Sh::kTile);
      mbar_init(mb + Sh::bPV + 8 * s, 1);
    }
    for (int s = 0; s < 4 * NT; ++s) mbar_init(mb + Sh::bMax + 8 * s, 2);
    mbar_init_fence();
  };
  if (tid == 0) {
    init_barriers();
    *abort = 0;
    *again = 0;
    if (a.tma)
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.tm)) : "memory");
  }
  if (warp == Sh::kSoft + 2) tmem_alloc(mb + Sh::oTmem, Sh::kCols);
  // everything above touches only this block and the plan, which no kernel
  // writes; from here on the preceding grids' results are read
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Slots ahead[3];
  if (warp == Sh::kSoft || warp == Sh::kSoft + 1) {
#pragma unroll
    for (int k = 0; k < 3; ++k) ahead[k] = load_slots(k);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Sh::oMeta + Sh::oTmem);
  // step t uses score buffer t & 1 of its row tile
  auto at = [&](uint32_t bar, int qt, int t) { return mb + bar + 8 * (2 * qt + (t & 1)); };

  bool bad_row = false;  // (softmax) this thread's columns of its row came out not finite

  // One pass of the block over its keys.  The careful one follows where a value
  // that is not finite got into a row's sums: it takes such values out of the V
  // tiles and writes again the columns that were not finite.  With one such
  // value in a prefix of 5120 keys, 64 questions of 64 tokens take 1.0 ms and 64
  // decodes 57 us, against 0.34 ms and 30 us (a block's rows walked one by one,
  // key after key, took 1.5 s and 42 ms).
  auto pass = [&](auto careful) {
  constexpr bool kCareful = decltype(careful)::value;
  if (warp == Sh::kSoft || warp == Sh::kSoft + 1) {
    // ============================================== producers: K, then V warp
    const int ST = isv ? Sh::VS : Sh::KS;
    if constexpr (kCareful) {
#pragma unroll
      for (int k = 0; k < 3; ++k) ahead[k] = load_slots(k);
    }
    int issued = 0;
    auto produce = [&](int t, Slots& mine) {
      Src cur;
      resolve(mine, cur);
      const int r16 = __shfl_sync(~0u, cur.row, lane & ~7);
      const uint32_t sq = __ballot_sync(~0u, cur.run && cur.row == r16 + 2 * (lane & 7));
      const bool in_run = ((sq >> (lane & ~7)) & 0xFFu) == 0xFFu;
      const uint32_t leads = __ballot_sync(~0u, in_run) & 0x01010101u;
      if (leads != 0x01010101u) addresses(t, mine, cur);
      mine = load_slots(t + 3);
      // the stage is free once every row tile is done with its last use
      if (t >= ST) {
        bool ok = true;
        if constexpr (Sh::kDirect) {
          for (int qt = 0; qt < tiles; ++qt)
            ok = ok && warp_wait(at(isv ? Sh::bPV : Sh::bS, qt, t), (t / 2 - 1) & 1, abort);
        } else {
          ok = warp_wait(mb + (isv ? Sh::bVr : Sh::bKr) + 8 * (t % ST), (t / ST - 1) & 1, abort);
        }
        if (!ok) return false;
      }
      const uint32_t bar = mb + (isv ? Sh::bV : Sh::bK) + 8 * (t % ST);
      const uint32_t dst = sbase + (isv ? Sh::oV : Sh::oK) + (t % ST) * Sh::TB;
      // 16 keys (8 lanes) in consecutive rows: one TMA box an operand half;
      // the others row by row with cp.async, whole rows an instruction, the
      // addresses through shared memory.  (tile::gather4 is issued lane by
      // lane, about 100 clocks each: 6400 for a tile of scattered rows.)
      const uint32_t tab_at = Sh::oRows + (isv ? kKeys * 8 : 0);
      if (leads != 0x01010101u)
        st_shared16(mb + tab_at + 16 * lane,
                    make_uint4((uint32_t)cur.at[0], (uint32_t)(cur.at[0] >> 32),
                               (uint32_t)cur.at[1], (uint32_t)(cur.at[1] >> 32)));
      if (lane == 0) mbar_expect_tx(bar, __popc(leads) * 16 * D * 2);
      __syncwarp();
      if (in_run && (lane & 7) < D / 64) {
        const int c = lane & 7;  // 64 columns each
        tma_tile2d(dst + c * (kKeys * 128) + 2 * (lane & ~7) * 128, &a.tm, (isv ? D : 0) + 64 * c,
                   r16, bar);
      }
      if (leads != 0x01010101u) {
        constexpr int C = D / 8, RI = 32 / C;  // 16-byte pieces a row, rows an instruction
        const uint64_t* tab = reinterpret_cast<const uint64_t*>(smem + Sh::oMeta + tab_at);
        for (int q = 0; q < kKeys / 16; ++q) {
          if ((leads >> (8 * q)) & 1u) continue;
          uint64_t src[16 / RI];
#pragma unroll
          for (int i = 0; i < 16 / RI; ++i) src[i] = tab[16 * q + i * RI + lane / C];
#pragma unroll
          for (int i = 0; i < 16 / RI; ++i) {
            const int j = 16 * q + i * RI + lane / C;
            const uint64_t p =
                src[i] ? src[i] + 16 * (lane % C) : reinterpret_cast<uint64_t>(a.pv.cache);
            cp_async16(dst + sw128(j, lane % C, kKeys), reinterpret_cast<const void*>(p),
                       src[i] != 0);
          }
        }
        __syncwarp();
      }
      cp_async_arrive_noinc(bar);
      issued = t + 1;
      return true;
    };
    // three at a time: a slot moved between registers would have to arrive first
    for (int t = 0; t < steps; t += 3) {
      if (!produce(t, ahead[0])) break;
      if (t + 1 < steps && !produce(t + 1, ahead[1])) break;
      if (t + 2 < steps && !produce(t + 2, ahead[2])) break;
    }
    // nothing of this block's copies is in flight when it ends
    for (int t = issued - ST < 0 ? 0 : issued - ST; t < issued; ++t) {
      const uint32_t bar = mb + (isv ? Sh::bV : Sh::bK) + 8 * (t % ST);
      const long long t0 = clock64();
      while (!mbar_try(bar, (t / ST) & 1) && clock64() - t0 < kWaitCycles) {
      }
    }
    if (slot_bad) report(a.status, CS_ST_SLOT_RANGE);

  } else if (warp >= Sh::kSoft + 2) {
    // ==================================================== MMA, one warp a tile
    // The whole warp walks the steps, so that descriptors stay in uniform
    // registers; one elected lane issues.  (One lane alone, with descriptors
    // built for each product, took 90 clocks a product of 64.)
    const int qt = __shfl_sync(~0u, warp, 0) - (Sh::kSoft + 2);
    if (qt < tiles) {
      const bool leader = elect_one();
      const uint32_t id_s = umma_idesc(128, kKeys, umma_format<T>(), 0, 0);
      const uint32_t id_o = umma_idesc(128, D, umma_format<T>(), 0, 1);  // V is MN-major
      const uint64_t dq = umma_desc(sbase + Sh::oQ + qt * Sh::QB, 16, 1024);
      const uint64_t dk0 = umma_desc(sbase + Sh::oK, 16, 1024);
      const uint64_t dv0 = umma_desc(sbase + Sh::oV, kKeys * 128, 1024);
      const uint32_t tm = __shfl_sync(~0u, tmem, 0);
      const uint32_t sc = tm + Sh::cS + 128 * qt, oc = tm + Sh::cO + D * qt;
      bool ok = warp_wait(mb + Sh::bQ, 0, abort);
      uint32_t last = 0, lastph = 0;  // the newest group issued
      // a key tile that has arrived (and, for rows copied by cp.async, may be
      // read by the tensor unit); waited for ahead of what comes later
      auto arrived = [&](uint32_t bar, int t, int stages) {
        ok = ok && warp_wait(mb + bar + 8 * (t % stages), (t / stages) & 1, abort);
        fence_async_smem();
        return ok;
      };
      auto scores = [&](int t) {
        tc_fence_after();
        const uint64_t dk = dk0 + (uint64_t)((t % Sh::KS) * (Sh::TB >> 4));
        const uint32_t s = sc + kKeys * (t & 1);
        last = at(Sh::bS, qt, t);
        lastph = (t >> 1) & 1;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)  // offsets in 16-byte units
            tc_mma(s, dq + (kk >> 2) * 1024 + (kk & 3) * 2,
                   dk + (kk >> 2) * (kKeys * 8) + (kk & 3) * 2, id_s, kk ? 1u : 0u);
          tc_commit(last);
        }
        __syncwarp();
      };
      if (steps > 0 && arrived(Sh::bK, 0, Sh::KS)) scores(0);
      if (steps > 1 && arrived(Sh::bK, 1, Sh::KS)) scores(1);
      for (int t = 0; ok && t < steps; ++t) {
        const uint32_t ph = (t >> 1) & 1;
        if (!arrived(Sh::bV, t, Sh::VS)) break;
        if (!(ok = warp_wait(at(Sh::bP, qt, t), ph, abort))) break;
        tc_fence_after();
        const uint64_t dv = dv0 + (uint64_t)((t % Sh::VS) * (Sh::TB >> 4));
        const uint32_t p = sc + kKeys * (t & 1);
        last = at(Sh::bPV, qt, t);
        lastph = ph;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            tc_mma_ts(oc, p + kk * 8, dv + kk * 128, id_o, (t | kk) ? 1u : 0u);
          tc_commit(last);
        }
        __syncwarp();
        // the next scores but one take the buffer that P lies in, and a later
        // V tile the stage just read
        const bool refill = !Sh::kDirect && t + Sh::VS < steps;
        if (t + 2 < steps || refill) {
          if (t + 2 < steps && Sh::kDirect && !arrived(Sh::bK, t + 2, Sh::KS)) break;
          if (!(ok = warp_wait(at(Sh::bPV, qt, t), ph, abort))) break;
          if (refill && leader) mbar_arrive(mb + Sh::bVr + 8 * (t % Sh::VS));
          if (t + 2 < steps && (Sh::kDirect || arrived(Sh::bK, t + 2, Sh::KS))) scores(t + 2);
        }
      }
      if (last) {
        const long long t0 = clock64();
        while (!mbar_try(last, lastph) && clock64() - t0 < kWaitCycles) {
        }
      }
    }
    __syncwarp();

  } else {
    constexpr int TPR = Sh::TPR, VC = kKeys / TPR;  // scores of a step a thread holds
    if (warp / (4 * TPR) < tiles) {
    // ================================================================= softmax
    const int qt = warp / (4 * TPR), part2 = (warp >> 2) % TPR;
    const int r = (warp & 3) * 32 + lane;  // TMEM lane
    const int tok = qt * a.R + r / a.G, h = g * a.G + r % a.G;
    const bool row_ok = r < a.R * a.G && tok < it.ntok;
    {
      // queries into the swizzled operand layout, 16 bytes a step
      constexpr int C = D / 8;
      const int left = it.ntok - qt * a.R;
      const int rows = (left < a.R ? left : a.R) * a.G;
      const uint32_t qs = sbase + Sh::oQ + qt * Sh::QB;
      const char* base = a.q + (int64_t)(it.tok0 + qt * a.R) * a.qt + (int64_t)(g * a.G) * a.qh;
      const int c = tid % C;
      auto from = [&](int row) {
        const int tk = row / a.G;
        return base + tk * a.qt + (row - tk * a.G) * a.qh + 16 * c;
      };
      if (a.vec_q && !a.neg) {
        // rows without a query are zeros: their scores then are zeros too, which
        // is what P should hold for them, and multiplying zeros draws less of
        // the power that decodes are held back by
#pragma unroll 4
        for (int row = (tid % Sh::kTile) / C; row < kPrefixTile; row += Sh::kTile / C)
          cp_async16(qs + sw128(row, c, kPrefixTile), row < rows ? from(row) : a.q, row < rows);
        cp_async_wait_all();
      } else {
        for (int row = (tid % Sh::kTile) / C; row < kPrefixTile; row += Sh::kTile / C) {
          uint16_t e[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            e[k] = row < rows ? reinterpret_cast<const uint16_t*>(from(row))[k] ^
                                    (a.neg ? 0x8000 : 0)
                              : 0;
          st_shared16(qs + sw128(row, c, kPrefixTile),
                      make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
                                 e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16));
        }
      }
      fence_async_smem();
      mbar_arrive(mb + Sh::bQ);
    }
    const int4 tk = row_ok ? a.tokens[it.tok0 + tok] : make_int4(0, 0, 0, 0);
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t sc0 = tmem + lane_base + Sh::cS + 128 * qt;
    const uint32_t oc = tmem + lane_base + Sh::cO + D * qt;
    float mref = -INFINITY, lsum = 0.f;  // log2 domain; P = 2^(x - mref + up)
    bool ok = true;
    [[maybe_unused]] int exchanges = 0;  // of maxima with the row's other thread
    [[maybe_unused]] const uint32_t pair = mb + Sh::bMax + 8 * (4 * qt + (warp & 3));
    [[maybe_unused]] float* row_max =
        reinterpret_cast<float*>(smem + Sh::oMeta + Sh::oMax) + qt * 512;
    const bool any_row = __any_sync(~0u, row_ok);
    // (careful) which columns of the row keys that it sees make not finite: a
    // bit a column, NaN, +inf and -inf
    uint32_t poison[kCareful ? kKinds : 1][D / 32];
    if constexpr (kCareful) {
#pragma unroll
      for (int k = 0; k < kKinds; ++k) {
#pragma unroll
        for (int w = 0; w < D / 32; ++w) poison[k][w] = 0u;
      }
    }
    auto wait_pv = [&](int t) {
      ok = warp_wait(at(Sh::bPV, qt, t), (t >> 1) & 1, abort);
      tc_fence_after();
      return ok;
    };

    // (careful) takes the values that are not finite out of step t's V tile,
    // all softmax threads an equal share of its 16-byte pieces, and notes which
    // they were: a byte of column bits a piece and kind, for two steps in turn
    const int softs = Sh::kTile * tiles;
    volatile int* found = reinterpret_cast<volatile int*>(smem + Sh::oMeta + Sh::oFound);
    auto clean = [&](int t) {
      if (!warp_wait(mb + Sh::bV + 8 * (t % Sh::VS), (t / Sh::VS) & 1, abort)) return false;
      constexpr int C = D / 8;
      const uint32_t tile = sbase + Sh::oV + (t % Sh::VS) * Sh::TB;
      uint8_t* notes = reinterpret_cast<uint8_t*>(smem + Sh::oMeta + Sh::oBad) +
                       (t & 1) * kKinds * kKeys * C;
      for (int i = tid; i < kKeys * C; i += softs) {
        const uint32_t at = tile + sw128(i / C, i % C, kKeys);
        const uint4 was = ld_shared16(at);
        const uint32_t x[4] = {was.x, was.y, was.z, was.w};
        uint32_t y[4], bad = 0u, nan = 0u, minus = 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[k] = x[k];
          const uint32_t b = take_out<T>(y[k]);
          bad |= b << (2 * k);
          nan |= nan_bits<T>(x[k], b) << (2 * k);
          minus |= ((x[k] >> 15 & 1u) | (x[k] >> 30 & 2u)) << (2 * k);
        }
        notes[i] = (uint8_t)nan;
        notes[kKeys * C + i] = (uint8_t)(bad & ~nan & ~minus);
        notes[2 * kKeys * C + i] = (uint8_t)(bad & ~nan & minus);
        if (bad) {
          st_shared16(at, make_uint4(y[0], y[1], y[2], y[3]));
          found[t & 1] = t + 1;
        }
      }
      fence_async_smem();
      mbar_arrive(mb + Sh::bClean);
      return warp_wait(mb + Sh::bClean, t & 1, abort);
    };

    for (int t = 0; t < steps; ++t) {
      const Step st = step_of(it, na, t);
      int vlo = 0, vhi = 0;
      if (row_ok) {
        vlo = st.own ? (tk.z > st.base ? tk.z - st.base : 0) : 0;
        vhi = st.own ? (tk.w - st.base < st.n ? tk.w - st.base : st.n) : st.n;
      }
      const uint32_t sc = sc0 + kKeys * (t & 1);
      ok = warp_wait(at(Sh::bS, qt, t), (t >> 1) & 1, abort);
      if (!ok) break;  // a wait expired
      if (!Sh::kDirect && tid % Sh::kTile == 0) mbar_arrive(mb + Sh::bKr + 8 * (t % Sh::KS));
      tc_fence_after();
      if constexpr (kCareful) {
        ok = clean(t);
        if (!ok) break;
      }
      if (!any_row) {  // no query in these 32 rows: their P is zero already
        mbar_arrive(at(Sh::bP, qt, t));
        continue;
      }
      uint32_t v[VC];
      // both threads of a row leave this way together
      if (__all_sync(~0u, vhi <= vlo)) {  // nothing to see for these 32 rows
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c] = 0u;
#pragma unroll
        for (int cc = 0; cc < VC / 32; ++cc) CS_TMEM_ST16(sc + 16 * (part2 + cc), v);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(at(Sh::bP, qt, t));
        continue;
      }
      CS_TMEM_LD32(sc + 32 * part2, v);
      if constexpr (TPR == 1) CS_TMEM_LD32(sc + 32, (v + 32));
      tmem_wait_ld();
      if (!__all_sync(~0u, vlo <= 0 && vhi >= kKeys)) {
#pragma unroll
        for (int cc = 0; cc < VC / 32; ++cc) {
          const uint32_t bits = col_bits(vlo, vhi, 32 * (part2 + cc));
#pragma unroll
          for (int c = 0; c < 32; ++c)
            v[32 * cc + c] = (bits >> c) & 1u ? v[32 * cc + c] : 0xff800000u;  // -inf
        }
      }
      if constexpr (kCareful) {
        if (found[t & 1] == t + 1) {
          // keys that the row sees, but for scores of -inf, which weigh nothing
          uint32_t seen[VC / 32];
#pragma unroll
          for (int cc = 0; cc < VC / 32; ++cc) {
            seen[cc] = 0u;
#pragma unroll
            for (int c = 0; c < 32; ++c)
              seen[cc] |= v[32 * cc + c] != 0xff800000u ? 1u << c : 0u;
          }
          const uint32_t* notes = reinterpret_cast<const uint32_t*>(smem + Sh::oMeta + Sh::oBad) +
                                  (t & 1) * kKinds * kKeys * (D / 32);
#pragma unroll
          for (int cc = 0; cc < VC / 32; ++cc) {
#pragma unroll 1
            for (int c = 0; c < 32; ++c) {
              if (!(seen[cc] >> c & 1u)) continue;
#pragma unroll
              for (int k = 0; k < kKinds; ++k) {
#pragma unroll
                for (int w = 0; w < D / 32; ++w)
                  poison[k][w] |=
                      notes[(k * kKeys + 32 * (part2 + cc) + c) * (D / 32) + w];
              }
            }
          }
        }
      }
      float top;
      {
        float m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          m[k] = max_nan(__uint_as_float(v[k]), __uint_as_float(v[k + 4]));
#pragma unroll
        for (int c = 8; c < VC; c += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            m[k] = max3_nan(m[k], __uint_as_float(v[c + k]), __uint_as_float(v[c + k + 4]));
        }
        top = max_nan(max3_nan(m[0], m[1], m[2]), m[3]);
      }
      // the row's maximum from both its threads; past this barrier both have
      // read their scores, so P may take their columns
      if constexpr (TPR == 2) {
        float* mx = row_max + (exchanges & 1) * 256;
        mx[part2 * 128 + r] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(pair);
        ok = warp_wait(pair, exchanges & 1, abort);
        if (!ok) break;
        ++exchanges;
        top = max_nan(top, mx[(1 - part2) * 128 + r]);
      }
      if (!(top < INFINITY)) {  // a NaN or +inf score makes the row NaN
        lsum = __int_as_float(0x7fffffff);
        top = -INFINITY;
      }
      const float top2 = top == -INFINITY ? -INFINITY : top * a.scale2;
      const bool grow = top2 > mref + kLazy || mref == -INFINITY;
      const bool rescale = grow && mref > -INFINITY && top2 > mref;
      if (__any_sync(~0u, rescale)) {  // t > 0: a row has a finite maximum
        if (!wait_pv(t - 1)) break;
        const float f = rescale ? ex2(mref - top2) : 1.f;
        lsum *= f;
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
      if (grow) mref = top2;
      // the largest weight so far is 2^up, or up to 2^kLazy more
      const float sub = (mref > -INFINITY ? mref : 0.f) - p_up<T>();
      const float2 scale = make_float2(a.scale2, a.scale2), off = make_float2(-sub, -sub);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
      // in passes over the scores, so that no instruction waits for the one
      // before it
#pragma unroll
      for (int c = 0; c < VC; c += 2) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])),
                                    scale, off);
        v[c] = __float_as_uint(x.x);
        v[c + 1] = __float_as_uint(x.y);
      }
#pragma unroll
      for (int c = 0; c < VC; ++c) v[c] = __float_as_uint(ex2(__uint_as_float(v[c])));
#pragma unroll
      for (int c = 0; c < VC; c += 4) {
        s0 = __fadd2_rn(s0, make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])));
        s1 = __fadd2_rn(s1, make_float2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])));
      }
#pragma unroll
      for (int c = 0; c < VC / 2; ++c)
        v[c] = Pack2<T>::pack(__uint_as_float(v[2 * c]), __uint_as_float(v[2 * c + 1]));
#pragma unroll
      for (int cc = 0; cc < VC / 32; ++cc) CS_TMEM_ST16(sc + 16 * (part2 + cc), (v + 16 * cc));
      lsum += (s0.x + s0.y) + (s1.x + s1.y);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(at(Sh::bP, qt, t));
    }

    // ---------------------------------------------------------------- output
    if (ok && steps > 0) wait_pv(steps - 1);
    if constexpr (TPR == 2) {  // the row's sum from both its threads
      float* sum = row_max + (exchanges & 1) * 256;
      sum[part2 * 128 + r] = lsum;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      ok = ok && warp_wait(pair, exchanges & 1, abort);
      lsum += sum[(1 - part2) * 128 + r];
      if constexpr (kCareful) {
        // each thread looked at half the step's keys: both halves' findings,
        // through the place of the queries (read by no product any more)
        ++exchanges;
        constexpr int kWords = kKinds * (D / 32);
        static_assert(2 * kWords * 4 <= 2 * D + 16, "within the row's place of the staging below");
        uint32_t* row = reinterpret_cast<uint32_t*>(smem + Sh::oQ + qt * Sh::QB + r * (2 * D + 16));
        uint32_t *mine = row + part2 * kWords, *theirs = row + (1 - part2) * kWords;
#pragma unroll
        for (int k = 0; k < kKinds; ++k) {
#pragma unroll
          for (int w = 0; w < D / 32; ++w) mine[k * (D / 32) + w] = poison[k][w];
        }
        for (int turn = 0; turn < 2; ++turn) {  // written, then read
          __syncwarp();
          if (lane == 0) mbar_arrive(pair);
          ok = ok && warp_wait(pair, exchanges & 1, abort);
          ++exchanges;
          if (turn == 0) {
#pragma unroll
            for (int k = 0; k < kKinds; ++k) {
#pragma unroll
              for (int w = 0; w < D / 32; ++w) poison[k][w] |= theirs[k * (D / 32) + w];
            }
          }
        }
      }
    }
    const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
    const float lse2 = lsum == 0.f ? -INFINITY
                                   : (mref > -INFINITY ? mref : 0.f) - p_up<T>() + log2f(lsum);
    const int64_t token = it.tok0 + tok;
    const int64_t prow = ((int64_t)it.part + tok) * a.hq + h;
    char* orow = a.out + token * a.ot + (int64_t)h * a.oh;
    const bool part = it.part >= 0;
    if (part) orow = reinterpret_cast<char*>(a.part_o + prow * D);
    const bool have = ok && steps > 0 && lsum != 0.f;
    // An infinite or NaN value of a key that this row does not see reaches its
    // sums as 0 x inf = NaN.  So where a row (a thread's columns of it) is not
    // finite, the block passes over its keys once more, with such values taken
    // out of the V tiles, and the columns that they belong to are set for the
    // rows that see them.  (A NaN sum of weights makes the row NaN as it is.)
    float worst = 0.f;
    uint32_t set_to[kKinds][D / 32 / TPR];  // of this thread's columns
    if constexpr (kCareful) {
#pragma unroll
      for (int k = 0; k < kKinds; ++k) {
#pragma unroll
        for (int w = 0; w < D / 32 / TPR; ++w) {
          const uint32_t low = poison[k][w], high = poison[k][w + D / 32 - D / 32 / TPR];
          set_to[k][w] = part2 == 0 ? low : high;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32 / TPR; ++w) set_to[0][w] |= set_to[1][w] & set_to[2][w];
    }
    // element c of this thread's columns as it is written
    auto final = [&](float x, int c) {
      if constexpr (kCareful) {
        const int w = c / 32, b = c % 32;
        if (set_to[2][w] >> b & 1u) x = -INFINITY;
        if (set_to[1][w] >> b & 1u) x = INFINITY;
        if (set_to[0][w] >> b & 1u) x = __int_as_float(0x7fffffff);
      } else {
        worst = max_nan(worst, fabsf(x));
      }
      return x;
    };
    const bool write = ok && (kCareful ? bad_row : row_ok);
    if (part || a.vec_out) {
      // each thread stages its row (32-bit partials in two halves) where the
      // queries were, and the warp writes whole rows: stores straight from the
      // registers touch 32 rows an instruction, and a bulk copy a row is
      // issued lane by lane (5300 clocks a tile, either way)
      constexpr int B = 2 * D / TPR;  // bytes of a row a thread stages at once
      constexpr int L = B / 16;       // lanes that write them
      constexpr int W = 2 * D + 16;
      const uint32_t stage = sbase + Sh::oQ + qt * Sh::QB + (r - lane) * W + part2 * B;
      const uint32_t buf = stage + lane * W;
      const uint64_t to = write ? reinterpret_cast<uint64_t>(orow) : 0;
#pragma unroll(kCareful ? 2 : 1)
      for (int round = 0; round < (part ? 2 : 1); ++round) {
        uint32_t v[32];
        const uint32_t col = oc + part2 * (D / 2);
        if (part) {
#pragma unroll
          for (int cc = 0; cc < B / 64; ++cc) {
            CS_TMEM_LD16(col + round * (B / 4) + 16 * cc, v);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c)
              v[c] = __float_as_uint(final(have ? __uint_as_float(v[c]) * inv : 0.f,
                                           round * (B / 4) + 16 * cc + c));
#pragma unroll
            for (int c = 0; c < 4; ++c)
              st_shared16(buf + 64 * cc + 16 * c,
                          make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]));
          }
        } else {
#pragma unroll
          for (int cc = 0; cc < B / 64; ++cc) {
            CS_TMEM_LD32(col + 32 * cc, v);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float x = have ? __uint_as_float(v[2 * c]) * inv : 0.f;
              const float y = have ? __uint_as_float(v[2 * c + 1]) * inv : 0.f;
              v[c] = Pack2<T>::pack(final(x, 32 * cc + 2 * c), final(y, 32 * cc + 2 * c + 1));
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
              st_shared16(buf + 64 * cc + 16 * c,
                          make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]));
          }
        }
        __syncwarp();
        // a partial's thread has two rounds, an output's one
        const int64_t first = part ? (part2 * 2 + round) * B : part2 * B;
#pragma unroll
        for (int n0 = 0; n0 < L; n0 += 4) {
          uint4 x[4];
          uint64_t dst[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int row = (n0 + n) * (32 / L) + lane / L;
            dst[n] = __shfl_sync(~0u, to, row);
            x[n] = ld_shared16(stage + row * W + 16 * (lane % L));
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (dst[n]) *reinterpret_cast<uint4*>(dst[n] + first + 16 * (lane % L)) = x[n];
        }
        __syncwarp();
      }
    } else {
#pragma unroll(kCareful ? D / 32 / TPR : 1)
      for (int cc = 0; cc < D / 32 / TPR; ++cc) {
        uint32_t v[32];
        const int col = part2 * (D / 2) + 32 * cc;
        CS_TMEM_LD32(oc + col, v);
        tmem_wait_ld();
        if (!write) continue;
#pragma unroll
        for (int c = 0; c < 32; ++c)
          reinterpret_cast<T*>(orow)[col + c] = Elem<T>::from_f(
              final(have ? __uint_as_float(v[c]) * inv : 0.f, 32 * cc + c));
      }
    }
    if constexpr (!kCareful) {
      bad_row = write && have && lsum == lsum && !(worst < INFINITY);
      if (bad_row) *again = 1;
    }
    if (!kCareful && write && part2 == 0) {
      if (it.part >= 0) a.part_lse[prow] = lse2;
      else if (a.lse) a.lse[token * a.hq + h] = lse2 * kLn2;
    }
    }
  }
  };
  pass(std::false_type());

  // the joining grid starts while the last blocks write (told earlier, its
  // blocks wait beside these and cost 8 decodes behind 65536 keys 5 us)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (*again && !*abort) {  // nothing of the first pass is in flight
    tc_fence_after();
    if (tid == 0) {
      for (uint32_t b = Sh::bQ; b < Sh::oTmem; b += 8) mbar_inval(mb + b);
      init_barriers();
      mbar_init(mb + Sh::bClean, Sh::kTile * tiles);
      mbar_init_fence();
      volatile int* found = reinterpret_cast<volatile int*>(smem + Sh::oMeta + Sh::oFound);
      found[0] = found[1] = 0;
    }
    __syncthreads();
    pass(std::true_type());
    tc_fence_before();
    __syncthreads();
  }
  if (tid == 0 && *abort) report(a.status, CS_ST_TIMEOUT);
  if (warp == Sh::kSoft + 2) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kCols);
  }
}

// WPR warps per (join token, head): o = sum_c w_c o_c / sum_c w_c with
// w_c = 2^(lse_c - max), warp i taking partials i, i + WPR, ... of the plan's
// order, the warps' sums added in order.  Four warps where tokens have more
// than 16 partials: 8 decodes behind 65536 keys (36 a token) take 53 us with
// four and 59 with one, 64 decodes behind 5120 (11 a token) 26.7 and 23.5.
template <typename T, int D, int WPR>
__global__ void __launch_bounds__(128) prefix_join_kernel(const PArgs a, const int4* join,
                                                          const int32_t* list, int n) {
  constexpr int E = D / 32;
  using V = typename std::conditional<E == 4, float4, float2>::type;
  __shared__ V part_sum[WPR][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, wi = (threadIdx.x >> 5) % WPR;
  const int64_t w = blockIdx.x * (4ll / WPR) + (threadIdx.x >> 5) / WPR;
  const bool live = w < (int64_t)n * a.hq;
  const int4 j = live ? join[w / a.hq] : make_int4(0, 0, 0, 0);
  const int h = (int)(w % a.hq);
  int32_t first = lane < j.z ? list[j.y + lane] : 0;
  // the plan may be read before the preceding grid is done, its results not
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float l0 = lane < j.z ? a.part_lse[(int64_t)first * a.hq + h] : -INFINITY;
  float top = l0;
  for (int c = 32 + lane; c < j.z; c += 32)
    top = fmaxf(top, a.part_lse[(int64_t)list[j.y + c] * a.hq + h]);
  top = warp_max(top);
  float o[E], sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int c0 = 0; c0 < j.z; c0 += 32) {
    // a lane's partial of these 32: its place and weight (NaN stays NaN; one
    // below 2^-126 of the largest is that, not 0, so that what is not finite
    // in it is not lost)
    float l = l0;
    if (c0 > 0) {
      first = c0 + lane < j.z ? list[j.y + c0 + lane] : 0;
      l = c0 + lane < j.z ? a.part_lse[(int64_t)first * a.hq + h] : -INFINITY;
    }
    const float f = l == -INFINITY ? 0.f : max_nan(ex2(l - top), 0x1p-126f);
    sum += warp_sum(f);
    const int m = j.z - c0 < 32 ? j.z - c0 : 32;
#pragma unroll 1
    for (int c = wi; c < m; c += 8 * WPR) {
      V x[8];
      float wk[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int q = c + k * WPR;
        const int64_t place = __shfl_sync(~0u, first, q & 31);
        const float fk = __shfl_sync(~0u, f, q & 31);
        wk[k] = q < m ? fk : 0.f;
        if (wk[k] != 0.f)
          x[k] = reinterpret_cast<const V*>(a.part_o + (place * a.hq + h) * D)[lane];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (wk[k] != 0.f) {
          const float* v = reinterpret_cast<const float*>(&x[k]);
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = fmaf(wk[k], v[e], o[e]);
        }
    }
  }
  if constexpr (WPR > 1) {
    V mine;
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<float*>(&mine)[e] = o[e];
    part_sum[wi][lane] = mine;
    __syncthreads();
    if (wi > 0) return;
#pragma unroll
    for (int k = 1; k < WPR; ++k) {
      const V x = part_sum[k][lane];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += reinterpret_cast<const float*>(&x)[e];
    }
  }
  if (!live) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* out = reinterpret_cast<T*>(a.out + (int64_t)j.x * a.ot + (int64_t)h * a.oh) + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = Elem<T>::from_f(o[e] * inv);
  if (a.lse && lane == 0)
    a.lse[(int64_t)j.x * a.hq + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

bool setup_maps(PArgs& a, const cs_paged_kv& kv) {
  const PagedView& pv = a.pv;
  const bool bf16 = kv.dtype == CS_BF16;
  const int64_t D = pv.head_dim;
  if (pv.sb < 0 || pv.sh < 0 || pv.so < 0) return false;
  const int64_t unit = std::gcd(std::gcd(pv.sb, pv.sh), pv.so);
  if (unit <= 0) return false;
  const int64_t rows = ((kv.num_blocks - 1) * pv.sb + (pv.kv_heads - 1) * pv.sh +
                        (pv.bs - 1) * pv.so) / unit + 1;
  if (!encode_rows(&a.tm, pv.cache, bf16, 2 * D, rows, unit, 16)) return false;
  a.nrb = pv.sb / unit;
  a.nrh = pv.sh / unit;
  a.nro = pv.so / unit;
  return true;
}

template <typename T, int D, int NT>
int launch_main(const PArgs& a, int64_t blocks, cudaStream_t stream) {
  constexpr auto kernel = prefix_sm100_kernel<T, D, NT>;
  if (!allow_smem<kernel>(Shape<D, NT>::kSmem)) return CS_ERR_CUDA;
  return launch_dependent(kernel, dim3((unsigned)blocks), Shape<D, NT>::kThreads,
                          Shape<D, NT>::kSmem, stream, a);
}

template <typename T, int D>
int launch_all(const PArgs& a, const cs_prefix_plan_info& info, const int32_t* plan,
               cudaStream_t stream) {
  if (info.n_items > 0) {
    const int64_t blocks = info.n_items * a.hkv;
    const int rc = info.variant == 2 ? launch_main<T, D, 2>(a, blocks, stream)
                                     : launch_main<T, D, 1>(a, blocks, stream);
    if (rc != CS_OK) return rc;
  }
  if (info.n_join > 0) {
    const int4* join = reinterpret_cast<const int4*>(plan + info.join_off);
    const int32_t* list = plan + info.list_off;
    const int64_t rows = info.n_join * a.hq, entries = info.words - info.list_off;
    if (entries > 16 * info.n_join)
      return launch_dependent(prefix_join_kernel<T, D, 4>, dim3((unsigned)rows), 128, 0, stream, a,
                              join, list, (int)info.n_join);
    return launch_dependent(prefix_join_kernel<T, D, 1>, dim3((unsigned)((rows + 3) / 4)), 128, 0,
                            stream, a, join, list, (int)info.n_join);
  }
  return CS_OK;
}

}  // namespace

int prefix_attn_sm100(const cs_prefix_params& p, const cs_prefix_plan_info& info,
                      const int32_t* plan, void* workspace, cudaStream_t stream) {
  const cs_paged_kv& kv = p.paged;
  PArgs a;
  a.pv = PagedView::make(kv);
  if (!a.pv.vec16()) return CS_ERR_UNSUPPORTED;
  a.q = static_cast<const char*>(p.q);
  a.qt = p.q_stride_tok * 2;
  a.qh = p.q_stride_head * 2;
  a.out = static_cast<char*>(p.out);
  a.ot = p.o_stride_tok * 2;
  a.oh = p.o_stride_head * 2;
  auto al = [](const void* x, int64_t t, int64_t h) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && t % 16 == 0 && h % 16 == 0;
  };
  a.vec_q = al(p.q, a.qt, a.qh);
  a.vec_out = al(p.out, a.ot, a.oh);
  a.lse = p.lse;
  a.prefix_slots = p.prefix_slots;
  a.suffix_slots = p.suffix_slots;
  a.tokens = reinterpret_cast<const int4*>(plan);
  a.items = reinterpret_cast<const PrefixItem*>(plan + info.item_off);
  a.part_o = static_cast<float*>(workspace);
  a.part_lse = a.part_o + info.part_tokens * p.q_heads * kv.head_dim;
  a.status = p.status;
  a.hq = p.q_heads;
  a.hkv = (int)kv.kv_heads;
  a.G = a.hq / a.hkv;
  a.R = kPrefixTile / a.G;
  a.bs_shift = -1;
  for (int s = 0; s < 31; ++s)
    if ((int64_t)1 << s == kv.block_size) a.bs_shift = s;
  a.neg = p.scale < 0.0;
  // masked scores are -inf before they are scaled, so the factor is never 0
  a.scale2 = fmaxf(fabsf((float)p.scale) * kLog2e, 1e-30f);
  a.nrb = a.nrh = a.nro = 0;
  // runs are found where a block's offsets are consecutive rows
  a.tma = setup_maps(a, kv) && a.nro == 1 ? 1 : 0;
  const bool half = kv.dtype == CS_F16;
  if (kv.head_dim == 128)
    return half ? launch_all<__half, 128>(a, info, plan, stream)
                : launch_all<__nv_bfloat16, 128>(a, info, plan, stream);
  return half ? launch_all<__half, 64>(a, info, plan, stream)
              : launch_all<__nv_bfloat16, 64>(a, info, plan, stream);
}

}  // namespace cs
