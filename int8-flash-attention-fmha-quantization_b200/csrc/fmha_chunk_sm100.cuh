// Attention of many query tokens over packed or paged sequences with grouped heads: prompts and chunks.  The formulas are in
// fmha_grouped_sm100.cuh.
//
//   unit     = one key head and two neighbouring tiles A, B of 128 query rows of one sequence.  A row is (token, head of the group), so a tile is
//              128 / G tokens, all G heads that share the keys; both tiles share every key tile that is brought in.
//   persistent: one CTA per SM walks units; the longest ones come first.
//   warps 0-3, 4-7   softmax of tile A, of tile B: one thread per row, its 128 scores in registers
//   warps 8-11       turn V from int8 into fp16, once for both tiles
//   warp 12          TMA loads: Q once per unit (two buffers), rings of K and V
//   warp 13          issues all MMAs:  S = Q K^T (kind::i8, exact),  O += P V (kind::f16, P from tensor memory)
//   warp 14          turns unit numbers into sequences, tiles and key ranges, ahead of the others
//
// Per tile S(j+1) is issued behind P.V(j), into the columns that P(j) occupied; while one tile's softmax runs, the other's products do.
// The output stays in tensor memory for a whole unit: a row's exponentials are taken relative to a reference that follows the running
// maximum only when that has grown by more than 2^8, which fp16 holds easily, and then the output is rescaled in place.  That is rare
// behind a row's first keys.
// Tensor memory (512 columns): S of A, S of B (128 each; P as fp16 over the first 64), O of A, O of B (128 each).
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace chunk {

using namespace grouped;

constexpr int kThreads = 512;
constexpr int kLaunchRegs = 128;
constexpr int kSoftmaxRegs = 184, kConvertRegs = 80, kOtherRegs = 64;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kOtherRegs <= 4 * kLaunchRegs, "setmaxnreg targets exceed the CTA's register allocation: the kernel would hang");
constexpr int kWarpConvert = 8, kWarpLoad = 12, kWarpMma = 13, kWarpWalk = 14;
constexpr int kInfos = 4;
constexpr int kInfoConsumers = 8 + 4 + 1 + 1;      // softmax warps, converters, loader, issuer
constexpr uint32_t kTmemCols = 512;
constexpr int kMasked = static_cast<int>(0xFF800000u - kMagicBits);      // a score that reads as minus infinity once kMagicBits are added
constexpr int kLowest = -(1 << 22);                                      // below every score

template <int D> struct Cfg {
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kStagesK = 3, kStagesV = 2, kStagesH = 2;          // K, V as int8, V as fp16
  static constexpr int kHalfBytes = 2 * kTileBytes;                      // a tile of V as fp16
  static constexpr int kQ = 0, kK = 4 * kTileBytes, kV = kK + kStagesK * kTileBytes, kH = kV + kStagesV * kTileBytes;
  static constexpr int kBytes = kH + kStagesH * kHalfBytes;
};
// What all roles need to know of a unit, and what the loader and the softmax warps do.
struct Steps {
  int valid;
  int n[2];             // key tiles of A, of B
};
struct Unit : Steps {
  Seq seq;
  int b, head;
  int token0;           // first token of tile A; tile B begins tq later
  int end;              // keys that the last token of the unit sees
};
template <int D> struct Ctl {
  using C = Cfg<D>;
  uint64_t info_full[kInfos], info_empty[kInfos];
  uint64_t q_full[2], q_empty[2], k_full[C::kStagesK], k_empty[C::kStagesK], v_full[C::kStagesV], v_empty[C::kStagesV], h_full[C::kStagesH], h_empty[C::kStagesH];
  uint64_t s_full[2], p_ready[2], o_full[2], o_free[2];      // per tile
  uint32_t tmem_base;
  int abort;
  Unit unit[kInfos];
};
template <int D> constexpr size_t smem_bytes() { return 1024 + Cfg<D>::kBytes + sizeof(Ctl<D>); }

// Reads units in order, one slot of the ring after the other.
template <int D> struct UnitReader {
  Ctl<D>* ctl;
  uint32_t n = 0;
  template <typename T> __device__ __forceinline__ bool next(T& u) {       // a Unit or its Steps
    const uint32_t slot = n % kInfos;
    if (!warp_wait(smem_u32(&ctl->info_full[slot]), (n / kInfos) & 1u, &ctl->abort)) return false;
    u = static_cast<const T&>(ctl->unit[slot]);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&ctl->info_empty[slot]));
    ++n;
    return true;
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
template <int D> __device__ __forceinline__ void walk_role(const Params& p, Ctl<D>* ctl) {
  const int lane = threadIdx.x & 31;
  const Failure fail{p, &ctl->abort};
  int level = -1, before = 0, here = 0;             // pairs of earlier levels, and of this one
  bool checked = blockIdx.x != 0;
  auto pairs_of = [&](int b) {
    if (b >= p.B) return 0;
    const Seq s = load_seq(p, b);
    if (!checked && (s.bad)) report(p.status, p.host_word, FMHA_I8_DEV_BAD_INDEX, 0u, b);
    return (s.nq + 2 * p.tq - 1) / (2 * p.tq);
  };
  const int few = p.B <= 32 ? pairs_of(lane) : 0;   // up to 32 sequences: kept in registers
  for (uint32_t n = 0;; ++n) {
    const long long round = n, ctas = gridDim.x;
    const long long u = round * ctas + ((n & 1u) ? ctas - 1 - blockIdx.x : blockIdx.x);
    const int head = static_cast<int>(u % p.Hkv);
    const long long pair = u / p.Hkv;
    bool more = true;
    while (level < 0 || pair >= static_cast<long long>(before) + here) {
      before += here;
      ++level;
      here = 0;
      if (p.B <= 32) here = __popc(__ballot_sync(0xFFFFFFFFu, few > level));
      else
        for (int b0 = 0; b0 < p.B; b0 += 32) here += __popc(__ballot_sync(0xFFFFFFFFu, pairs_of(b0 + lane) > level));
      checked = true;
      if (here == 0) { more = false; break; }
    }
    Unit unit{};
    if (more) {
      int at = static_cast<int>(pair - before), b = 0, pairs = 0;
      for (int b0 = 0;; b0 += 32) {
        const int mine = p.B <= 32 ? few : pairs_of(b0 + lane);
        const uint32_t with = __ballot_sync(0xFFFFFFFFu, mine > level);
        const int count = __popc(with);
        if (at < count) {
          const int src = __fns(with, 0u, at + 1);
          b = b0 + src;
          pairs = __shfl_sync(0xFFFFFFFFu, mine, src);
          break;
        }
        at -= count;
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
    const int n = max(u.n[0], u.n[1]);
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
    int page = page_of(p, u.b, 0, u.end, lane);
    for (int j = 0; j < n; ++j, ++g) {
      const int copies = copies_of(p, j * kTile, u.end);
      const uint32_t bytes = static_cast<uint32_t>((copies << p.box_shift) * D);
      if (page < 0 || page >= p.num_pages) { page = p.num_pages; bad_page |= lane < copies; }      // reads zeros
      const int next_page = page_of(p, u.b, (j + 1) * kTile, u.end, lane);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t stages = kv ? C::kStagesV : C::kStagesK, st = g % stages;
        const uint32_t full = smem_u32(kv ? &ctl->v_full[st] : &ctl->k_full[st]), empty = smem_u32(kv ? &ctl->v_empty[st] : &ctl->k_empty[st]);
        if (g >= stages && !warp_wait(empty, ((g / stages) - 1) & 1u, abort_flag)) return fail(kv ? FMHA_I8_DEV_WAIT_V_FREE : FMHA_I8_DEV_WAIT_K_FREE, g);
        if (lane == 0) mbar_arrive_expect_tx(full, bytes);
        __syncwarp();
        if (lane < copies) issue_copy<D>(p, kv ? map_v : map_k, smem + (kv ? C::kV : C::kK) + st * C::kTileBytes, full, u.seq, u.head, j * kTile, lane, page);
        __syncwarp();
      }
      page = next_page;
    }
    if (bad_page) report(p.status, p.host_word, FMHA_I8_DEV_BAD_INDEX, 1u, u.b);
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
    const int n = max(u.n[0], u.n[1]);
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
template <int D> __device__ __forceinline__ void mma_role(const Params& p, Ctl<D>* ctl, uint32_t smem, uint32_t tmem) {
  using C = Cfg<D>;
  constexpr uint32_t kIdescS = make_idesc_i8(kTile, false), kIdescO = make_idesc_f16_b_mn(D);
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  UnitReader<D> units{ctl};
  Steps cur, next;
  uint32_t g = 0, nq = 0;                            // key tiles and units with keys before the present unit
  uint32_t steps[2] = {0, 0}, outs[2] = {0, 0};      // P.V issued, units begun, per tile
  // S of tile t, step j of a unit whose first key tile is g0 and which is the n-th with keys
  auto issue_s = [&](const Steps& u, int t, int j, uint32_t g0, uint32_t n) -> bool {
    const uint32_t gj = g0 + static_cast<uint32_t>(j), st = gj % C::kStagesK, buf = n & 1u;
    if (j == 0 && !warp_wait(smem_u32(&ctl->q_full[buf]), (n >> 1) & 1u, abort_flag)) { fail(FMHA_I8_DEV_WAIT_Q_LOAD, n); return false; }
    if (!warp_wait(smem_u32(&ctl->k_full[st]), (gj / C::kStagesK) & 1u, abort_flag)) { fail(FMHA_I8_DEV_WAIT_K_LOAD, gj); return false; }
    tc_fence_after();
    const uint64_t dq = make_smem_desc(smem + C::kQ + (2 * buf + t) * C::kTileBytes, D), dk = make_smem_desc(smem + C::kK + st * C::kTileBytes, D);
    const int all = max(u.n[0], u.n[1]);
    if (elect_one()) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) mma_i8_ss(tmem + t * kTile, desc_advance(dq, 32 * i), desc_advance(dk, 32 * i), kIdescS, i > 0);
      mma_commit(smem_u32(&ctl->s_full[t]));
      if (t == (j < u.n[1] ? 1 : 0)) {               // the last one to read this K tile
        mma_commit(smem_u32(&ctl->k_empty[st]));
        if (j == all - 1) mma_commit(smem_u32(&ctl->q_empty[buf]));
      }
    }
    __syncwarp();
    return true;
  };
  if (!units.next(cur)) return fail(FMHA_I8_DEV_WAIT_INFO, 0);
  if (!cur.valid) return;
  bool ok = true;
#pragma unroll
  for (int t = 0; t < 2; ++t)
    if (ok && cur.n[t] > 0) ok = issue_s(cur, t, 0, g, nq);
  while (ok) {
    if (!units.next(next)) return fail(FMHA_I8_DEV_WAIT_INFO, g);
    const int all = max(cur.n[0], cur.n[1]);
    const uint32_t g_next = g + static_cast<uint32_t>(all), nq_next = nq + (all > 0);
    for (int j = 0; j < max(all, 1) && ok; ++j) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok) break;
        if (j < cur.n[t]) {
          const uint32_t gj = g + static_cast<uint32_t>(j), sh = gj % C::kStagesH;
          if (j == 0 && outs[t] > 0 && !warp_wait(smem_u32(&ctl->o_free[t]), (outs[t] - 1) & 1u, abort_flag)) { fail(FMHA_I8_DEV_WAIT_O_FREE, gj); return; }
          if (!warp_wait(smem_u32(&ctl->h_full[sh]), (gj / C::kStagesH) & 1u, abort_flag)) { fail(FMHA_I8_DEV_WAIT_V_LOAD, gj); return; }
          if (!warp_wait(smem_u32(&ctl->p_ready[t]), steps[t] & 1u, abort_flag)) { fail(FMHA_I8_DEV_WAIT_P_READY, gj); return; }
          tc_fence_after();
          const uint64_t dv = make_smem_desc_slabs(smem + C::kH + sh * C::kHalfBytes, C::kHalfBytes / 2);
          if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i)
              mma_f16_ts(tmem + 2 * kTile + t * kTile, tmem + t * kTile + 8 * i, desc_advance(dv, 16 * 128 * i), kIdescO, j > 0 || i > 0);
            if (t == (j < cur.n[1] ? 1 : 0)) mma_commit(smem_u32(&ctl->h_empty[sh]));
            if (j == cur.n[t] - 1) mma_commit(smem_u32(&ctl->o_full[t]));
          }
          __syncwarp();
          ++steps[t];
          if (j == 0) ++outs[t];
        }
        if (j + 1 < cur.n[t]) ok = issue_s(cur, t, j + 1, g, nq);
        else if (j == max(all, 1) - 1 && next.valid && next.n[t] > 0) ok = issue_s(next, t, 0, g_next, nq_next);
      }
    }
    if (!next.valid) return;
    cur = next;
    g = g_next;
    nq = nq_next;
  }
}

// ------------------------------------------------------------------------------------------------ softmax
__device__ __forceinline__ int max3(int a, int b, int c) { return __vimax3_s32(a, b, c); }

template <int D> __device__ __forceinline__ void softmax_role(const Params& p, Ctl<D>* ctl, uint32_t tmem) {
  const int warp = warp_index(), t = warp >> 2, lane = threadIdx.x & 31;
  const int row = (warp & 3) * 32 + lane;
  const Failure fail{p, &ctl->abort};
  volatile int* abort_flag = &ctl->abort;
  const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + lanes + t * kTile, tO = tmem + lanes + 2 * kTile + t * kTile;
  const int my_token = row / p.G, my_head = row - my_token * p.G;
  const float2 c2 = make_float2(p.c2, p.c2);
  UnitReader<D> units{ctl};
  Unit u;
  uint32_t steps = 0, outs = 0;
  while (true) {
    if (!units.next(u)) return fail(FMHA_I8_DEV_WAIT_INFO, steps);
    if (!u.valid) return;
    const int token = u.token0 + t * p.tq + my_token;
    const bool real = my_token < p.tq && token < u.seq.nq;
    const int n = u.n[t];
    const int limit = real ? visible(p, u.seq, token) : 0;
    const bool any = __any_sync(0xFFFFFFFFu, limit > 0);            // a warp without a row that sees a key leaves its part of P as it is
    const int least = __reduce_min_sync(0xFFFFFFFFu, real ? limit : 0x7FFFFFFF);
    float ref = kMagic, hi = 0.f;                                  // a reference score, as the float kMagic + score, and its exponent
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
    for (int j = 0; j < n; ++j, ++steps) {
      if (!warp_wait(smem_u32(&ctl->s_full[t]), steps & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_S_READY, steps);
      tc_fence_after();
      if (any) {
        uint32_t r[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32_issue(tS + 32 * i, r[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_fence(r[i]);
        if (j * kTile + kTile > least) {
          const int open = limit - j * kTile;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= open) r[i >> 5][i & 31] = static_cast<uint32_t>(kMasked);
        }
        int m0 = kLowest, m1 = kLowest;
#pragma unroll
        for (int i = 0; i < 128; i += 4) {
          m0 = max3(m0, static_cast<int>(r[i >> 5][i & 31]), static_cast<int>(r[i >> 5][(i & 31) + 1]));
          m1 = max3(m1, static_cast<int>(r[i >> 5][(i & 31) + 2]), static_cast<int>(r[i >> 5][(i & 31) + 3]));
        }
        const float m = __int_as_float(max(m0, m1) + static_cast<int>(kMagicBits));
        if (j == 0) {
          ref = m;
          hi = m * p.c2;
        } else {
          const bool grown = (m - ref) * p.c2 > 8.f;
          if (__any_sync(0xFFFFFFFFu, grown)) {
            const float next = grown ? m * p.c2 : hi, factor = grown ? ex2(hi - next) : 1.f;
            if (grown) ref = m;
            hi = next;
            sum[0].x *= factor; sum[0].y *= factor; sum[1].x *= factor; sum[1].y *= factor;
            // (the last P.V of this tile was issued before the S that has just been waited for, and is complete with it)
#pragma unroll 1
            for (int i = 0; i < D; i += 16) {
              uint32_t o[16];
              tmem_ld16_issue(tO + i, o);
              tmem_ld_fence(o);
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * factor);
              tmem_st8(tO + i, reinterpret_cast<uint32_t(&)[8]>(o[0]));
              tmem_st8(tO + i + 8, reinterpret_cast<uint32_t(&)[8]>(o[8]));
            }
          }
        }
        const float2 neg = make_float2(-hi, -hi);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t packed[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const int at = 64 * i + 2 * x;
            const float2 s = make_float2(__uint_as_float(r[at >> 5][at & 31] + kMagicBits), __uint_as_float(r[at >> 5][(at & 31) + 1] + kMagicBits));
            const float2 a = __ffma2_rn(s, c2, neg);
            const float2 e = make_float2(ex2(a.x), ex2(a.y));
            sum[x & 1] = __fadd2_rn(sum[x & 1], e);
            const __half2 h = __floats2half2_rn(e.x, e.y);
            packed[x] = *reinterpret_cast<const uint32_t*>(&h);
          }
          tmem_st32(tS + 32 * i, packed);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->p_ready[t]));
    }
    // ---- the row's output
    const long long at = (u.seq.q0 + token) * p.o_stride + static_cast<long long>(u.head * p.G + my_head) * D;
    float scale = 0.f;
    if (n > 0) {
      if (!warp_wait(smem_u32(&ctl->o_full[t]), outs & 1u, abort_flag)) return fail(FMHA_I8_DEV_WAIT_O_READY, steps);
      tc_fence_after();
      ++outs;
      const float l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      scale = l > 0.f ? p.out_scale / l : 0.f;
    }
    const bool some = limit > 0;
#pragma unroll 1
    for (int i = 0; i < D; i += 32) {
      uint32_t o[32];
      if (n > 0 && any) tmem_ld32(tO + i, o);
      if (real) {
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
          float v[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) v[y] = some ? __uint_as_float(o[x + y]) * scale : 0.f;
          store4(p.o, p.o_type, at + i + x, v);
        }
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

template <int D>
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
    for (int i = 0; i < C::kStagesK; ++i) { mbar_init(smem_u32(&ctl->k_full[i]), 1); mbar_init(smem_u32(&ctl->k_empty[i]), 1); }
    for (int i = 0; i < C::kStagesV; ++i) { mbar_init(smem_u32(&ctl->v_full[i]), 1); mbar_init(smem_u32(&ctl->v_empty[i]), 4); }
    for (int i = 0; i < C::kStagesH; ++i) { mbar_init(smem_u32(&ctl->h_full[i]), 4); mbar_init(smem_u32(&ctl->h_empty[i]), 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->q_full[i]), 1);
      mbar_init(smem_u32(&ctl->q_empty[i]), 1);
      mbar_init(smem_u32(&ctl->s_full[i]), 1);
      mbar_init(smem_u32(&ctl->p_ready[i]), 4);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&ctl->tmem_base);
  follow_previous_kernel();

  if (warp < kWarpConvert) {
    setmaxnreg_inc<kSoftmaxRegs>();
    softmax_role<D>(p, ctl, tmem);
  } else if (warp < kWarpLoad) {
    setmaxnreg_dec<kConvertRegs>();
    convert_role<D>(p, ctl, tiles);
  } else {
    setmaxnreg_dec<kOtherRegs>();
    if (warp == kWarpLoad) load_role<D>(p, ctl, &map_q, &map_k, &map_v, smem_u32(tiles));
    else if (warp == kWarpMma) mma_role<D>(p, ctl, smem_u32(tiles), tmem);
    else if (warp == kWarpWalk) walk_role<D>(p, ctl);
  }
  __syncwarp();
  if (ctl->abort) {                                  // copies still in flight land before their memory is used again
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace chunk
}  // namespace fmha
