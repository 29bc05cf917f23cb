// Attention of many query tokens over packed or paged sequences with grouped heads: prompts and chunks.  The formulas are in
// fmha_grouped_sm100.cuh.
//
//   unit     = one key head and two neighbouring tiles A, B of 128 query rows of one sequence.  A row is (token, head of the group), so a tile is
//              128 / G tokens, all G heads that share the keys; both tiles share every key tile that is brought in.
//   persistent: one CTA per SM walks units; the longest ones come first.
//   warps 0-3, 4-7   softmax of tile A, of tile B: one thread per row, the 128 scores of a key tile in registers
//   warps 8-11       turn V from int8 into fp16, once for both tiles
//   warp 12          TMA loads: Q once per unit (two buffers), rings of K and V
//   warp 13          issues S = Q K^T (kind::i8, exact)
//   warp 15          issues O += P V (kind::f16, P from tensor memory)
//   warp 14          turns unit numbers into sequences, tiles and key ranges, ahead of the others
//
// The output stays in tensor memory for a whole unit: a row's exponentials are taken relative to a reference that follows the running
// maximum only when that has grown by more than 2^8 in p, and then the output is rescaled in place.  That is rare behind a row's first keys.  P is 2^7 at the
// reference: fp16 holds 2^15, and its smallest step, 2^-24, is 2^-31 of that, so that many keys far below one are not lost.
// Tensor memory (512 columns): S of A, of B (128 columns each; P as fp16 over the first 64), O of A, of B (128 each).
//
// What bounds it: a tile's chain scores - softmax - P.V - scores.  A step of both tiles takes 3300 cycles: 220 from the scores' barrier to registers, 350 for the maximum, 1900 for 128
// exponentials and their conversion (in halves, P.V of the first beside the second), 770 for P.V and the next scores.  The tiles run half a step apart, so that one's
// exponentials hide the other's products; a third would need tensor memory that there is not.  A unit's end takes 3700 cycles: the output is read, scaled and stored while the tensor
// cores have only the other tile.  Tensor pipe 45 % of the cycles, issue 45 %, HBM 9 %.
//   1 x 16384 tokens, 32 heads on 8 of 128, causal, some values eight times as large   1767 us, 1.25 PFLOP/s (1.34 without those values: references that move)
//   8 x 2048 tokens                                                                     247 us, 1.11 PFLOP/s; among other calls, at the power limit, 1840 and 266
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace chunk {

using namespace grouped;

constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128;
constexpr int kSoftmaxRegs = 200, kConvertRegs = 56, kOtherRegs = 56;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kOtherRegs <= 4 * kLaunchRegs, "setmaxnreg targets exceed the CTA's register allocation: the kernel would hang");
constexpr int kWarpConvert = 8, kWarpLoad = 12, kWarpScore = 13, kWarpWalk = 14, kWarpOutput = 15;
// A warp may wait for a whole unit of another's, and gives up after about 1.5 s: 2^26 keys are 0.9 s.  Where a sequence has more, whatever bound the
// call was given, its units are not walked.
constexpr int kMostKeys = 1 << 26;
constexpr int kInfos = 4;
constexpr int kInfoConsumers = 8 + 4 + 1 + 2;      // softmax warps, converters, loader, issuers
constexpr uint32_t kTmemCols = 512;
// Scores come as the bits of the float kMagic + score (see issue_scores), which order like integers.
constexpr int kLowest = static_cast<int>(kMagicBits) - (1 << 22);        // below every score (127 * 127 * 128 < 2^21)
constexpr float kLift = 7.f;                                             // P is 2^kLift at the reference, and 2^kGrowth more at most
constexpr uint32_t kMasked = 0xFF000000u;                                // -2^127: below that, and its exponential is zero

template <int D> struct Cfg {
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kStagesK = 3, kStagesV = 2, kStagesH = 2;          // K, V as int8, V as fp16
  static constexpr int kHalfBytes = 2 * kTileBytes;                      // a tile of V as fp16
  static constexpr int kQ = 0, kK = 4 * kTileBytes, kV = kK + kStagesK * kTileBytes, kH = kV + kStagesV * kTileBytes;
  static constexpr int kBias = kH + kStagesH * kHalfBytes;              // constant operands, 128 and 64 rows of 32 bytes
  static constexpr int kBytes = kBias + (kTile + kTile / 2) * 32;
};
// What all roles need to know of a unit, and what the loader and the softmax warps do.
struct Steps {
  int valid;
  int n[2];             // key tiles of A, of B
  __device__ __forceinline__ int all() const { return max(n[0], n[1]); }
};
struct Unit : Steps {
  Seq seq;
  int b, head;
  int token0;           // first token of tile A; tile B begins tq later
  int end;              // keys that the last token of the unit sees
  int first;            // key tile at which this CTA begins (0 unless the unit is split)
};
template <int D> struct Ctl {
  using C = Cfg<D>;
  uint64_t info_full[kInfos], info_empty[kInfos];
  uint64_t q_full[2], q_empty[2], k_full[C::kStagesK], k_empty[C::kStagesK], v_full[C::kStagesV], v_empty[C::kStagesV], h_full[C::kStagesH], h_empty[C::kStagesH];
  uint64_t s_full[2], s_read[2];                     // per tile: the scores of a step are there, and in registers
  uint64_t p_ready[2][2];                            // per tile: either half of P
  uint64_t o_full[2], o_free[2];                     // per tile: the unit's output is complete, and has been read
  uint32_t tmem_base;
  int abort;
  Unit unit[kInfos];
  float2 part[2][kTile];                             // split units: a row's reference and sum in this CTA
};
// Split units: where a CTA leaves its rows for the others once its tiles are no longer needed, four floats further apart than they are long.
template <int D> constexpr int kPitch = D + 4;
static_assert(2 * kTile * kPitch<128> * 4 <= Cfg<128>::kBias - Cfg<128>::kK && 2 * kTile * kPitch<64> * 4 <= Cfg<64>::kBias - Cfg<64>::kK, "the partial rows do not fit");
template <int D> constexpr size_t smem_bytes() { return 1024 + Cfg<D>::kBytes + sizeof(Ctl<D>); }

// Reads units in order, one slot of the ring after the other.
template <int D> struct UnitReader {
  Ctl<D>* ctl;
  uint32_t n = 0;
  __device__ __forceinline__ bool next(Unit& u) {
    if (!wait()) return false;
    u = here();
    release();
    return true;
  }
  // For those who need no more.  They see the numbers as uniform values (see uniform()).
  __device__ __forceinline__ bool next(Steps& u) {
    if (!wait()) return false;
    const Unit& x = here();
    u.valid = uniform(x.valid);
    u.n[0] = uniform(x.n[0]);
    u.n[1] = uniform(x.n[1]);
    release();
    return true;
  }
  // The same in two steps, for those who leave it where it is: here() until release().
  __device__ __forceinline__ bool wait() { return warp_wait(smem_u32(&ctl->info_full[n % kInfos]), (n / kInfos) & 1u, &ctl->abort); }
  __device__ __forceinline__ const Unit& here() const { return ctl->unit[n % kInfos]; }
  __device__ __forceinline__ void release() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl->info_empty[n % kInfos]));
    ++n;
  }
};

struct Failure {
  const Params& p;
  int* abort;
  // by one lane or all of a warp
  __device__ __forceinline__ void operator()(unsigned code, unsigned at) const {
    *reinterpret_cast<volatile int*>(abort) = 1;
    if ((threadIdx.x & 31) == 0) report(p.status, p.host_word, code, threadIdx.x >> 5, at);
  }
};

// ------------------------------------------------------------------------------------------------ units
// The pairs of tiles of all sequences, the last of each sequence first, then the ones before those, and so on: with causal masks the ones with most keys
// come first.  Every pair is one unit per key head.  CTA c takes units c, 2 grid - 1 - c, 2 grid + c, ...: a round in one direction, the next in the other.
// The sequences are gone through in lots of 32, for the pairs of a level once, whatever number of units a CTA finds there: from the first one for every unit, 4096 prompts of 60 tokens (12 heads on
// 4 of 64) took 1898 us instead of 468, 1024 of 100 328 instead of 208.  Sequences without a pair of a level have none of the next, so that the lots of a level lie between the first and the
// last one with a pair of the level before.  All lots on every level: a chunk of 8192 tokens among 4096 sequences 5.7 ms instead of 1.0.  (A bit for every lot, which would help
// where long sequences stand at both ends too, changes how the compiler arranges the softmax warps: 4 to 7 % of every prompt.)
template <int D, bool kSplit> __device__ __forceinline__ void walk_role(const Params& p, Ctl<D>* ctl) {
  const int lane = threadIdx.x & 31;
  const Failure fail{p, &ctl->abort};
  int level = -1, before = 0, here = 0;             // pairs of earlier levels, and of this one
  int first_lot = 0, last_lot = p.B;                // sequences between which the pairs of this level lie
  int from = 0, passed = 0;                         // pairs of a CTA come in order: where the last one of this level was found, and how many lie before that
  bool checked = blockIdx.x != 0;
  auto pairs_of = [&](int b) {
    if (b >= p.B) return 0;
    const Seq s = load_seq(p, b);
    const bool ours = s.nq * p.G > p.few_rows, too_long = ours && s.nk > kMostKeys;
    if (!checked && (s.bad || too_long)) report_index(p.status, 0u, b);
    return ours && !too_long ? (s.nq + 2 * p.tq - 1) / (2 * p.tq) : 0;
  };
  const int few = p.B <= 32 ? pairs_of(lane) : 0;   // up to 32 sequences: kept in registers
  for (uint32_t n = 0;; ++n) {
    const long long round = n, ctas = gridDim.x;
    const long long u = kSplit ? static_cast<long long>(blockIdx.x / cluster_ctas()) : p.first_unit + round * ctas + ((n & 1u) ? ctas - 1 - blockIdx.x : blockIdx.x);
    const int head = static_cast<int>(u % p.Hkv);
    const long long pair = u / p.Hkv;
    bool more = !kSplit || n == 0;
    while (more && (level < 0 || pair >= static_cast<long long>(before) + here)) {
      before += here;
      ++level;
      here = passed = 0;
      if (p.B <= 32) here = __popc(__ballot_sync(0xFFFFFFFFu, few > level));
      else
      {
        const int end = last_lot;
        int at = first_lot;
        first_lot = -1;
        for (; at < end; at += 32) {
          const int count = __popc(__ballot_sync(0xFFFFFFFFu, pairs_of(at + lane) > level));
          here += count;
          if (count > 0) {
            if (first_lot < 0) first_lot = at;
            last_lot = at + 32;
          }
        }
      }
      from = first_lot;
      checked = true;
      if (here == 0) { more = false; break; }
    }
    Unit unit{};
    if (more) {
      int b = 0, pairs = 0;
      for (int at = static_cast<int>(pair - before);; from += 32) {
        const int mine = p.B <= 32 ? few : pairs_of(from + lane);
        const uint32_t with = __ballot_sync(0xFFFFFFFFu, mine > level);
        const int count = __popc(with);
        if (at < passed + count) {
          const int src = __fns(with, 0u, at - passed + 1);
          b = from + src;
          pairs = __shfl_sync(0xFFFFFFFFu, mine, src);
          break;
        }
        passed += count;
      }
      unit.valid = 1;
      unit.b = b;
      unit.head = head;
      unit.seq = load_seq(p, b);
      unit.token0 = (pairs - 1 - level) * 2 * p.tq;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int first = unit.token0 + t * p.tq, last = min(first + p.tq, unit.seq.nq) - 1;
        const int keys = first < unit.seq.nq ? visible(p, unit.seq, last) : 0;
        unit.n[t] = (keys + kTile - 1) / kTile;
        unit.end = max(unit.end, keys);
      }
      if constexpr (kSplit) {
        const int all = unit.all(), parts = static_cast<int>(cluster_ctas()), rank = static_cast<int>(cluster_rank());
        unit.first = static_cast<int>(static_cast<long long>(all) * rank / parts);
        const int last = static_cast<int>(static_cast<long long>(all) * (rank + 1) / parts);
#pragma unroll
        for (int t = 0; t < 2; ++t) unit.n[t] = max(min(unit.n[t], last) - unit.first, 0);
      }
    }
    const uint32_t slot = n % kInfos;
    if (n >= kInfos && !warp_wait(smem_u32(&ctl->info_empty[slot]), ((n / kInfos) - 1) & 1u, &ctl->abort)) { fail(FMHA_I8_DEV_WAIT_INFO, n); return; }
    if (lane == 0) {
      ctl->unit[slot] = unit;
      mbar_arrive(smem_u32(&ctl->info_full[slot]));
    }
    __syncwarp();
    if (!more) return;
  }
}

// ------------------------------------------------------------------------------------------------ loads
template <int D> __device__ __forceinline__ void load_role(const Params& p, Ctl<D>* ctl, const CUtensorMap* map_q, const CUtensorMap* map_k, const CUtensorMap* map_v, uint32_t smem) {
  using C = Cfg<D>;
  const int lane = threadIdx.x & 31;
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  UnitReader<D> units{ctl};
  Unit u;
  uint32_t g = 0, nq = 0;                            // key tiles and units with keys so far
  while (true) {
    if (!units.next(u)) return fail(FMHA_I8_DEV_WAIT_INFO, g);
    if (!u.valid) return;
    const int n = u.all();
    if (n == 0) continue;
    bool bad_page = false;
    const uint32_t buf = nq & 1u;
    if (nq >= 2 && !warp_wait(smem_u32(&ctl->q_empty[buf]), ((nq >> 1) - 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_Q_LOAD, nq);
    if (lane == 0) {
      const uint32_t bar = smem_u32(&ctl->q_full[buf]), bytes = static_cast<uint32_t>(p.G * p.tq * D);
      mbar_arrive_expect_tx(bar, bytes * ((u.n[0] > 0) + (u.n[1] > 0)));
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (u.n[t] > 0) tma_load_3d(smem + C::kQ + (2 * buf + t) * C::kTileBytes, map_q, bar, 0, u.head * p.G, u.seq.q0 + u.token0 + t * p.tq);
    }
    __syncwarp();
    ++nq;
    int page = page_of(p, u.b, u.first * kTile, u.end, lane);
    for (int j = 0; j < n; ++j, ++g) {
      const int key0 = (u.first + j) * kTile, copies = copies_of(p, key0, u.end);
      const uint32_t bytes = static_cast<uint32_t>((copies << p.box_shift) * D);
      if (page < 0 || page >= p.num_pages) { page = p.num_pages; bad_page |= lane < copies; }      // reads zeros
      const int next_page = page_of(p, u.b, key0 + kTile, u.end, lane);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t stages = kv ? C::kStagesV : C::kStagesK, st = g % stages;
        const uint32_t full = smem_u32(kv ? &ctl->v_full[st] : &ctl->k_full[st]), empty = smem_u32(kv ? &ctl->v_empty[st] : &ctl->k_empty[st]);
        if (g >= stages && !warp_wait(empty, ((g / stages) - 1) & 1u, abort_flag)) return fail(kv ? FMHA_I8_DEV_WAIT_V_FREE : FMHA_I8_DEV_WAIT_K_FREE, g);
        if (lane == 0) mbar_arrive_expect_tx(full, bytes);
        __syncwarp();
        if (lane < copies) issue_copy<D>(p, kv ? map_v : map_k, smem + (kv ? C::kV : C::kK) + st * C::kTileBytes, full, u.seq, u.head, key0, lane, page);
        __syncwarp();
      }
      page = next_page;
    }
    if (bad_page) report_index(p.status, 1u, u.b);
    __syncwarp();
  }
}

// ------------------------------------------------------------------------------------------------ V from int8 to fp16
// A key's D values become one row of 128 bytes (D = 64) or one in each of two slabs of 64 columns (D = 128), swizzled as the tensor core wants
// them.  A thread turns 16 bytes at a time; the two 16-byte pieces that these make are written in an order that keeps eight lanes on eight
// different columns of banks.
template <int D> __device__ __forceinline__ void convert_role(const Params& p, Ctl<D>* ctl, uint8_t* tiles) {
  using C = Cfg<D>;
  constexpr int kChunks = D / 16;
  const int lane = threadIdx.x & 31, at = static_cast<int>(threadIdx.x) - kWarpConvert * 32;
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  const int c = at % kChunks, key0 = at / kChunks;
  UnitReader<D> units{ctl};
  Steps u;
  uint32_t g = 0;
  while (true) {
    if (!units.next(u)) return fail(FMHA_I8_DEV_WAIT_INFO, g);
    if (!u.valid) return;
    const int n = u.all();
    for (int j = 0; j < n; ++j, ++g) {
      const uint32_t st = g % C::kStagesV, sh = g % C::kStagesH;
      if (!warp_wait(smem_u32(&ctl->v_full[st]), (g / C::kStagesV) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_V_LOAD, g);
      if (g >= C::kStagesH && !warp_wait(smem_u32(&ctl->h_empty[sh]), ((g / C::kStagesH) - 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_V_FREE, g);
      const uint8_t* src = tiles + C::kV + st * C::kTileBytes;
      uint8_t* dst = tiles + C::kH + sh * C::kHalfBytes;
#pragma unroll 4
      for (int i = 0; i < kTile * kChunks / 128; ++i) {
        const int key = key0 + i * (128 / kChunks);
        const uint4 w = D == 128 ? *reinterpret_cast<const uint4*>(src + key * 128 + ((c ^ (key & 7)) << 4))
                                 : *reinterpret_cast<const uint4*>(src + key * 64 + ((c ^ ((key >> 1) & 3)) << 4));
        uint4 lo, hi;
        unpack4(w.x, lo.x, lo.y);
        unpack4(w.y, lo.z, lo.w);
        unpack4(w.z, hi.x, hi.y);
        unpack4(w.w, hi.z, hi.w);
        uint8_t* row = dst + (D == 128 ? (c >> 2) * (C::kHalfBytes / 2) : 0) + key * 128;
        const int first = 2 * (c & 3);
        const bool swap = D == 128 && (c >> 2) != 0;
        *reinterpret_cast<uint4*>(row + (((first + (swap ? 1 : 0)) ^ (key & 7)) << 4)) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(row + (((first + (swap ? 0 : 1)) ^ (key & 7)) << 4)) = swap ? lo : hi;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&ctl->h_full[sh]));
        mbar_arrive(smem_u32(&ctl->v_empty[st]));
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ MMAs
// Two warps issue them, each going through the steps of both tiles in turn.  Their code is kept small and is not unrolled over tiles: it runs
// once per step between others' code, and what it took was above all the fetching of its instructions (one warp for both products, unrolled: 1425
// cycles for a step of one tile, of which the tensor core is busy 450).
// P of a step takes the first half of the columns of its scores.  The scores of the next step's last 64 keys therefore follow as soon as these are in
// registers (one warp), those of the first 64 behind the P.V that reads P (the other: MMAs of one thread execute in order).
// S of 64 keys.  The accumulator is first set to 2048 * 6144 = kMagic by a product of constants (16 bits, one step); the integer products then add to the
// bits of that float, which reads as kMagic + score without a conversion: 128 integer additions of a thread less, 8 % of a long prompt.
template <int D> __device__ __forceinline__ void issue_scores(uint32_t dst, uint64_t dq, uint64_t dk, uint32_t bias) {
  constexpr uint32_t kIdescS = make_idesc_i8(kTile / 2, false);
  mma_f16_ss(dst, make_smem_desc_noswizzle(bias, 128, 256), make_smem_desc_noswizzle(bias + kTile * 32, 128, 256), make_idesc_bf16(kTile / 2), 0);
#pragma unroll
  for (int y = 0; y < D / 32; ++y) mma_i8_ss(dst, desc_advance(dq, 32 * y), desc_advance(dk, 32 * y), kIdescS, 1);
}
template <int D> __device__ __forceinline__ void score_role(const Params& p, Ctl<D>* ctl, uint32_t smem, uint32_t tmem) {
  using C = Cfg<D>;
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  UnitReader<D> units{ctl};
  Steps u;
  uint32_t st = 0, k_phase = 0, nq = 0;              // K stage and its phase, units with keys
  uint32_t count_a = 0, count_b = 0;                 // steps issued for A, for B
  while (true) {
    if (!units.next(u)) return fail(FMHA_I8_DEV_WAIT_INFO, count_a);
    if (!u.valid) return;
    const int all = u.all();
    if (all == 0) continue;
    const uint32_t q = nq & 1u;
    if (!warp_wait(smem_u32(&ctl->q_full[q]), (nq >> 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_Q_LOAD, nq);
    ++nq;
#pragma unroll 1
    for (int i = 0; i < all; ++i) {
      if (!warp_wait(smem_u32(&ctl->k_full[st]), k_phase, abort_flag)) return fail(FMHA_I8_DEV_WAIT_K_LOAD, i);
      const uint64_t dk = make_smem_desc(smem + C::kK + st * C::kTileBytes + C::kTileBytes / 2, D);
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        if (i >= (t ? u.n[1] : u.n[0])) continue;
        const uint32_t c = t ? count_b++ : count_a++;
        if (c > 0 && !warp_wait(smem_u32(&ctl->s_read[t]), (c - 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_S_FREE, c);
        tc_fence_after();
        if (elect_one()) {
          issue_scores<D>(tmem + t * kTile + kTile / 2, make_smem_desc(smem + C::kQ + (2 * q + t) * C::kTileBytes, D), dk, smem + C::kBias);
          mma_commit(smem_u32(&ctl->s_full[t]));
        }
        __syncwarp();
      }
      if (elect_one()) mma_commit(smem_u32(&ctl->k_empty[st]));
      __syncwarp();
      if (++st == C::kStagesK) { st = 0; k_phase ^= 1u; }
    }
    if (elect_one()) mma_commit(smem_u32(&ctl->q_empty[q]));
    __syncwarp();
  }
}

template <int D> __device__ __forceinline__ void output_role(const Params& p, Ctl<D>* ctl, uint32_t smem, uint32_t tmem) {
  using C = Cfg<D>;
  constexpr uint32_t kIdescO = make_idesc_f16_b_mn(D);
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  UnitReader<D> units{ctl};
  Steps u;
  uint32_t st = 0, k_phase = 0, sh = 0, h_phase = 0, nq = 0;
  uint32_t count_a = 0, count_b = 0, outs_a = 0, outs_b = 0;      // steps issued and units begun for A, for B
  while (true) {
    if (!units.next(u)) return fail(FMHA_I8_DEV_WAIT_INFO, count_a);
    if (!u.valid) return;
    const int all = u.all();
    if (all == 0) continue;
    const uint32_t q = nq & 1u;
    if (!warp_wait(smem_u32(&ctl->q_full[q]), (nq >> 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_Q_LOAD, nq);
    ++nq;
    // Step i: P.V of key tile i (none for i = -1), then the scores of the first 64 keys of tile i + 1.
#pragma unroll 1
    for (int i = -1; i < all; ++i) {
      if (i >= 0 && !warp_wait(smem_u32(&ctl->h_full[sh]), h_phase, abort_flag)) return fail(FMHA_I8_DEV_WAIT_V_LOAD, i);
      if (i + 1 < all && !warp_wait(smem_u32(&ctl->k_full[st]), k_phase, abort_flag)) return fail(FMHA_I8_DEV_WAIT_K_LOAD, i);
      const uint64_t dv0 = make_smem_desc_slabs(smem + C::kH + sh * C::kHalfBytes, C::kHalfBytes / 2);
      const uint64_t dk = make_smem_desc(smem + C::kK + st * C::kTileBytes, D);
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const int n = t ? u.n[1] : u.n[0];
        if (i >= n) continue;
        if (i >= 0) {
          const uint32_t c = t ? count_b++ : count_a++;
          if (i == 0) {
            const uint32_t outs = t ? outs_b++ : outs_a++;
            if (outs > 0 && !warp_wait(smem_u32(&ctl->o_free[t]), (outs - 1) & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_O_FREE, outs);
          }
#pragma unroll 1
          for (int upper = 0; upper < 2; ++upper) {
            if (!warp_wait(smem_u32(&ctl->p_ready[t][upper]), c & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_P_READY, c);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int y = 0; y < kTile / 32; ++y)
                mma_f16_ts(tmem + 2 * kTile + t * kTile, tmem + t * kTile + upper * (kTile / 4) + 8 * y, desc_advance(dv0, upper * (kTile / 2 * 128) + 16 * 128 * y), kIdescO,
                           i > 0 || upper > 0 || y > 0);
              if (upper && i == n - 1) mma_commit(smem_u32(&ctl->o_full[t]));
            }
            __syncwarp();
          }
        }
        if (i + 1 < n) {
          tc_fence_after();
          if (elect_one()) {
            issue_scores<D>(tmem + t * kTile, make_smem_desc(smem + C::kQ + (2 * q + t) * C::kTileBytes, D), dk, smem + C::kBias);
            mma_commit(smem_u32(&ctl->s_full[t]));
          }
          __syncwarp();
        }
      }
      if (i >= 0) {
        if (elect_one()) mma_commit(smem_u32(&ctl->h_empty[sh]));    // both tiles have read this V tile
        __syncwarp();
        if (++sh == C::kStagesH) { sh = 0; h_phase ^= 1u; }
      }
      if (i + 1 < all) {
        if (elect_one()) mma_commit(smem_u32(&ctl->k_empty[st]));
        __syncwarp();
        if (++st == C::kStagesK) { st = 0; k_phase ^= 1u; }
      }
    }
    if (elect_one()) mma_commit(smem_u32(&ctl->q_empty[q]));
    __syncwarp();
  }
}

// ------------------------------------------------------------------------------------------------ softmax
__device__ __forceinline__ int max3(int a, int b, int c) { return __vimax3_s32(a, b, c); }

template <int D, bool kWide, bool kSplit> __device__ __forceinline__ void softmax_role(const Params& p, Ctl<D>* ctl, uint32_t tmem) {
  const int warp = warp_index(), t = warp >> 2, quad = warp & 3, lane = threadIdx.x & 31;
  const int row = quad * 32 + lane;
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
  const uint32_t tS = tmem + lanes + t * kTile, tO = tmem + lanes + 2 * kTile + t * kTile;
  const int my_token = row / p.G;
  const float2 c2 = make_float2(p.c2, p.c2);
  UnitReader<D> units{ctl};
  uint32_t steps = 0, outs = 0;
  while (true) {
    if (!units.wait()) return fail(FMHA_I8_DEV_WAIT_INFO, steps);
    const Unit& u = units.here();
    if (!u.valid) return;
    const int n = uniform(u.n[t]);
    bool real;
    int limit;
    {
      const int token = u.token0 + t * p.tq + my_token;
      real = my_token < p.tq && token < u.seq.nq;
      limit = (real ? visible(p, u.seq, token) : 0) - (kSplit ? u.first * kTile : 0);      // (of this CTA's keys)
    }
    const bool any = __any_sync(0xFFFFFFFFu, limit > 0);            // a warp without a row that sees a key leaves its part of P as it is
    const int least = __reduce_min_sync(0xFFFFFFFFu, real ? limit : 0x7FFFFFFF);      // keys that all rows see
    // p = 2^((x - ref) c2), x and ref as the floats kMagic + score.  Exponents are x c2 - hi with hi = ref c2 rounded, the same for a row as long as its
    // reference is, and rounded once.  (kLift is in hi.)  Where c2 is large the difference is taken first: hi would be off by as much as 16.
    int ref = 0;
    float hi = 0.f;
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
    for (int i = 0; i < n; ++i, ++steps) {
      if (!warp_wait(smem_u32(&ctl->s_full[t]), steps & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_S_READY, steps);
      uint32_t r[8][16];
      bool grew = false;
      float factor = 1.f;
      if (any) {
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 8; ++x) tmem_ld16_issue(tS + 16 * x, r[x]);
#pragma unroll
        for (int x = 0; x < 8; ++x) tmem_ld_fence(r[x]);
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->s_read[t]));
      if (any) {
        if (i * kTile + kTile > least) {
          const int open = limit - i * kTile;
#pragma unroll
          for (int x = 0; x < kTile; ++x)
            if (x >= open) r[x >> 4][x & 15] = kMasked;
        }
        int m0 = kLowest, m1 = kLowest;
#pragma unroll
        for (int x = 0; x < kTile; x += 4) {
          m0 = max3(m0, static_cast<int>(r[x >> 4][x & 15]), static_cast<int>(r[x >> 4][(x & 15) + 1]));
          m1 = max3(m1, static_cast<int>(r[x >> 4][(x & 15) + 2]), static_cast<int>(r[x >> 4][(x & 15) + 3]));
        }
        const int m = max(m0, m1);
        if (i == 0) {
          ref = m;
          hi = fmaf(__int_as_float(m), p.c2, -kLift);
        } else {
          const bool grown = m - ref > p.growth;
          if (__any_sync(0xFFFFFFFFu, grown)) {
            grew = true;
            const float next = grown ? fmaf(__int_as_float(m), p.c2, -kLift) : hi;
            factor = !grown ? 1.f : kWide ? ex2((__int_as_float(ref) - __int_as_float(m)) * p.c2) : ex2(hi - next);
            if (grown) ref = m;
            hi = next;
            sum[0].x *= factor; sum[0].y *= factor; sum[1].x *= factor; sum[1].y *= factor;
          }
        }
      }
      if (any) {
        const float2 less = make_float2(-hi, -hi), from = make_float2(-__int_as_float(ref), -__int_as_float(ref));
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          if (h == 4 && grew) {
            // The reference has moved: what has been summed so far is rescaled before more is added.  (The scores of this step were formed behind P.V of the one
            // before.)  Here, where half of the scores have become powers, there are registers for 16 columns.
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
              uint32_t o[16];
              tmem_ld16_issue(tO + x, o);
              tmem_ld_fence(o);
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * factor);
              tmem_st16(tO + x, o);
            }
          }
          uint32_t packed[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float2 v = make_float2(__uint_as_float(r[h][2 * x]), __uint_as_float(r[h][2 * x + 1]));
            const float2 a = kWide ? __ffma2_rn(__fadd2_rn(v, from), c2, make_float2(kLift, kLift)) : __ffma2_rn(v, c2, less);
            const float2 e = make_float2(ex2(a.x), ex2(a.y));
            sum[x & 1] = __fadd2_rn(sum[x & 1], e);
            const __half2 q = __floats2half2_rn(e.x, e.y);
            packed[x] = *reinterpret_cast<const uint32_t*>(&q);
          }
          if (h == 4) {                              // the first half of P; the latency of its stores lies behind the powers of this lot
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->p_ready[t][0]));
          }
          tmem_st8(tS + 8 * h, packed);
        }
        tmem_wait_st();
      } else if (lane == 0) {
        mbar_arrive(smem_u32(&ctl->p_ready[t][0]));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->p_ready[t][1]));
    }
    if constexpr (kSplit) {                          // the rows are put together behind all roles
      if (n > 0 && !warp_wait(smem_u32(&ctl->o_full[t]), outs & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_O_READY, steps);
      if (n > 0) ++outs;
      const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      ctl->part[t][row] = make_float2(__int_as_float(ref), n > 0 && limit > 0 ? l : 0.f);
      units.release();
      continue;
    }
    // ---- the row's output
    const long long at = (u.seq.q0 + u.token0 + t * p.tq + my_token) * p.o_stride + static_cast<long long>((u.head - my_token) * p.G + row) * D;
    units.release();
    float scale = 0.f;
    if (n > 0) {
      if (!warp_wait(smem_u32(&ctl->o_full[t]), outs & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_O_READY, steps);
      tc_fence_after();
      ++outs;
      const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      scale = l > 0.f ? p.out_scale / l : 0.f;
    }
    if (limit <= 0) scale = 0.f;
#pragma unroll 1
    for (int i = 0; i < D; i += 32) {
      uint32_t o[32];
      if (n > 0 && any) tmem_ld32(tO + i, o);
      if (real) {
        if (limit <= 0) {                            // (what stands in its place may be no number)
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0u;
        }
        if (p.out_down != 1.f) {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * p.out_down);
        }
        store32(p.o, p.o_type, p.o_wide != 0, at + i, o, scale);
      }
      __syncwarp();
    }
    if (n > 0) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->o_free[t]));
    }
  }
}

// The parts of a split unit: every CTA leaves its rows, references and sums in shared memory, and puts together its share of them.  By all threads.
template <int D> __device__ __forceinline__ void join_parts(const Params& p, Ctl<D>* ctl, uint8_t* tiles, uint32_t tmem) {
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int parts = static_cast<int>(cluster_ctas()), rank = static_cast<int>(cluster_rank());
  const Unit& u = ctl->unit[0];
  float* rows = reinterpret_cast<float*>(tiles + Cfg<D>::kK);
  if (warp < kWarpConvert && u.valid) {
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tO = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + 2 * kTile + t * kTile;
    const bool some = ctl->part[t][row].y > 0.f;
    if (__any_sync(0xFFFFFFFFu, some)) {
#pragma unroll 1
      for (int i = 0; i < D; i += 16) {
        uint32_t o[16];
        tmem_ld16_issue(tO + i, o);
        tmem_ld_fence(o);
        float4* to = reinterpret_cast<float4*>(rows + (t * kTile + row) * kPitch<D> + i);
#pragma unroll
        for (int y = 0; y < 4; ++y) to[y] = make_float4(__uint_as_float(o[4 * y]), __uint_as_float(o[4 * y + 1]), __uint_as_float(o[4 * y + 2]), __uint_as_float(o[4 * y + 3]));
      }
    }
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (u.valid) {
    constexpr int kQuads = D / 4;
    const uint32_t rows_at = smem_u32(rows), part_at = smem_u32(ctl->part);
    const int from = 2 * kTile * rank / parts, to = 2 * kTile * (rank + 1) / parts;
    for (int i = from * kQuads + static_cast<int>(threadIdx.x); i < to * kQuads; i += kThreads) {
      const int r = i / kQuads, c = i - r * kQuads, t = r / kTile, in_tile = r - t * kTile, my_token = in_tile / p.G;
      const int token = u.token0 + t * p.tq + my_token;
      if (my_token >= p.tq || token >= u.seq.nq) continue;
      float m = 0.f, l = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};           // (references are floats above 2^22)
      for (int y = 0; y < parts; ++y) {
        const float2 st = ld_cluster_v2(map_to_rank(part_at + 8 * r, y));
        if (st.y > 0.f) m = fmaxf(m, st.x);
      }
      for (int y = 0; y < parts; ++y) {
        const float2 st = ld_cluster_v2(map_to_rank(part_at + 8 * r, y));
        if (!(st.y > 0.f)) continue;
        const float e = ex2((st.x - m) * p.c2);
        const float4 v = ld_cluster_v4(map_to_rank(rows_at + static_cast<uint32_t>((r * kPitch<D> + 4 * c) * 4), y));
        l = fmaf(e, st.y, l);
        a[0] = fmaf(e, v.x, a[0]); a[1] = fmaf(e, v.y, a[1]); a[2] = fmaf(e, v.z, a[2]); a[3] = fmaf(e, v.w, a[3]);
      }
      const float scale = l > 0.f ? p.out_scale / l : 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) a[y] = a[y] * scale * p.out_down;
      store4(p.o, p.o_type, (u.seq.q0 + token) * p.o_stride + static_cast<long long>(u.head * p.G + in_tile - my_token * p.G) * D + 4 * c, a);
    }
  }
  __syncwarp();
  cluster_arrive();                                  // nobody leaves while another still reads its rows
  cluster_wait();
}

// kWide: the factor from scores to exponents is large (see softmax_role).  kSplit: one unit per cluster, whose CTAs share its key tiles: for calls of few
// tokens against many keys, whose units would leave most SMs idle.
template <int D, bool kWide, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Ctl<D>* ctl = reinterpret_cast<Ctl<D>*>(tiles + C::kBytes);
  const int warp = warp_index();
  if (threadIdx.x == 0) {
    ctl->abort = 0;
    for (int i = 0; i < kInfos; ++i) { mbar_init(smem_u32(&ctl->info_full[i]), 1); mbar_init(smem_u32(&ctl->info_empty[i]), kInfoConsumers); }
    for (int i = 0; i < C::kStagesK; ++i) { mbar_init(smem_u32(&ctl->k_full[i]), 1); mbar_init(smem_u32(&ctl->k_empty[i]), 2); }
    for (int i = 0; i < C::kStagesV; ++i) { mbar_init(smem_u32(&ctl->v_full[i]), 1); mbar_init(smem_u32(&ctl->v_empty[i]), 4); }
    for (int i = 0; i < C::kStagesH; ++i) { mbar_init(smem_u32(&ctl->h_full[i]), 4); mbar_init(smem_u32(&ctl->h_empty[i]), 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->q_full[i]), 1);
      mbar_init(smem_u32(&ctl->q_empty[i]), 2);
      mbar_init(smem_u32(&ctl->s_full[i]), 2);
      mbar_init(smem_u32(&ctl->s_read[i]), 4);
      mbar_init(smem_u32(&ctl->p_ready[i][0]), 4);
      mbar_init(smem_u32(&ctl->p_ready[i][1]), 4);
      mbar_init(smem_u32(&ctl->o_full[i]), 1);
      mbar_init(smem_u32(&ctl->o_free[i]), 4);
    }
    mbar_init_fence();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  for (int i = threadIdx.x; i < (kTile + kTile / 2) * 2; i += kThreads)      // unswizzled: 8 rows of 16 bytes, the other half of their K behind them
    reinterpret_cast<uint4*>(tiles + C::kBias)[i] = make_uint4((i & 8) ? 0u : i < kTile * 2 ? 0x4500u : 0x45C0u, 0u, 0u, 0u);      // 2048 and 6144 in bf16
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base));
  follow_previous_kernel();

  if (warp < kWarpConvert) {
    setmaxnreg_inc<kSoftmaxRegs>();
    softmax_role<D, kWide, kSplit>(p, ctl, tmem);
  } else if (warp < kWarpLoad) {
    setmaxnreg_dec<kConvertRegs>();
    convert_role<D>(p, ctl, tiles);
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == kWarpLoad) load_role<D>(p, ctl, &map_q, &map_k, &map_v, smem_u32(tiles));
    else if (warp == kWarpScore) score_role<D>(p, ctl, smem_u32(tiles), tmem);
    else if (warp == kWarpOutput) output_role<D>(p, ctl, smem_u32(tiles), tmem);
    else walk_role<D, kSplit>(p, ctl);
  }
  __syncwarp();
  if (ctl->abort) {                                  // copies still in flight land before their memory is used again
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kSplit) {
    // (the registers as they were at launch again)
    if (warp < kWarpConvert) setmaxnreg_dec<kLaunchRegs>();
    else setmaxnreg_inc<kLaunchRegs>();
    tc_fence_after();
    join_parts<D>(p, ctl, tiles, tmem);
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace chunk
}  // namespace fmha
