// Attention of a few query rows per key head over packed or paged sequences with grouped heads: single new tokens against a cache.
// The formulas are in fmha_grouped_sm100.cuh.
//
// The G heads of a group and the new tokens of a sequence make the rows: row r is token r / G, head r % G of the group, four, eight or sixteen at a time.
// What bounds it: K and V of a key head are read once for all of a group's rows, so HBM does, 2 D bytes per key.  A tensor-core tile of
// tcgen05.mma has 128 rows; here eight or sixteen are enough, so the products are warp-level ones, and
//   * a warp owns whole tiles of 128 keys, with its running maximum, sum and output rows in registers; it asks for its next K
//     when it has formed the scores of this one, and for the next V behind P.V;
//   * scores are products of bytes (m16n8k32) on top of the bits of the float kMagic, so that they read as kMagic + score;
//   * up to eight rows (one token of a model with up to eight query heads to a key head), P is a whole number, its bytes the rows of a product of bytes with V:
//     nothing is converted, no row is idle, and the products of a tile are exact.  It is 65535 e with e relative to the largest score of the tile.
//     Up to four rows have four bytes each: 65535 e rounded down, and as many bits of what that leaves.  Up to eight have two, rn(65535 e), off by 2^-17 of the
//     tile's largest e for every key however small its own is; where that may count, in a tile in which few keys have most of a row's weight, they have four too and
//     there are two products (1190 instructions a tile of four rows, 1280 of eight with one).  (With 16 bits relative to the running maximum 131,072 keys behind one that lies 12.5 nats above them lost a third of their weight.);
//   * up to sixteen rows P is fp16, 2^15 where p is 1, and V becomes fp16 in registers (integers up to 2048 are exact there), m16n8k16;
//   * which key, column or row a lane's element belongs to is free as long as both operands agree, and is chosen so that each lane reads 16 bytes at a time
//     without bank conflicts from the swizzled tiles, and so that the scores' registers are P's operand as they are;
//   * the keys of a sequence are split over the warps of a cluster of CTAs, whose partial rows meet through distributed shared memory.
//
// 64 sequences of 1 to 8192 keys, 32 heads on 8 of 128: 105 us, 5.8 TB/s, 88 % of a copy's rate; 172 with P as fp16 (issue: 53 M instructions of six warps to an SM).  64 heads, eight
// rows: 108, and 117 with two products in every tile.
// One sequence of 1025 keys: 7.2 us, latencies in a row.  Two of 125,000 keys on 4 key heads, seven rows: 64 us on the 64 SMs that eight clusters
// of eight have, 3.9 TB/s; 77 with scores of a deviation of 3, most of whose tiles need two products.
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace rows {

using namespace grouped;

constexpr int kMaxCluster = 16;
constexpr float kLevels = 65535.f;                   // of P in 16 bits
constexpr uint32_t kCap = 2047u;                     // 2^-5 of them
// Sixteen rows: P, sums and outputs are 2^15 times as large, so that the largest p still is an fp16 and the smallest step of one, 2^-24, is 2^-39 of it.
constexpr float kHalfLift = 15.f;
// 64 KB of tiles per CTA and three CTAs to an SM, or one CTA with three times as many warps
template <int D> struct Cfg {
  static constexpr int kWarps = (D == 128) ? 2 : 4;
  static constexpr int kWarpsWide = 3 * kWarps;
  static constexpr int kTileBytes = kTile * D;
};
template <int D, int W, int kRows> struct Smem {
  alignas(1024) uint8_t ring[2 * W * kTile * D];     // per warp: one K tile, one V tile; at the end its partial rows
  float2 stat[W][kRows];                             // reference exponent and sum of each partial row
  float2 together[kRows];                            // the same of the CTA's rows
  uint64_t k_full[W], v_full[W];
  int abort;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A unsigned; kFirst: on top of the bits of kMagic in all places instead of c.
template <bool kFirst>
__device__ __forceinline__ void mma16832_u(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kFirst) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(kMagicBits));
  } else {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// Four neighbouring columns of four keys, from a word per key to a word per column.
__device__ __forceinline__ void turn4(uint32_t k0, uint32_t k1, uint32_t k2, uint32_t k3, uint32_t (&columns)[4]) {
  const uint32_t t0 = __byte_perm(k0, k1, 0x5140), t1 = __byte_perm(k2, k3, 0x5140), t2 = __byte_perm(k0, k1, 0x7362), t3 = __byte_perm(k2, k3, 0x7362);
  columns[0] = __byte_perm(t0, t1, 0x5410); columns[1] = __byte_perm(t0, t1, 0x7632);
  columns[2] = __byte_perm(t2, t3, 0x5410); columns[3] = __byte_perm(t2, t3, 0x7632);
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
// Byte offset of 16-byte chunk c of row r in a tile as the copy engine writes it: chunks of a row of 128 bytes change places with the row
// modulo 8, of 64 bytes with half the row modulo 4.
template <int D> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return D == 128 ? static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)) : static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// grid: clusters of c CTAs, one per (sequence, key head, group of kRows rows).  kRows: 4, 8 or 16.
template <int D, int W, int kRows>
__global__ void __launch_bounds__(W * 32, W <= 4 ? 3 : 1)
rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  constexpr bool kWhole = kRows <= 8;                // P in whole numbers
  constexpr int kHalves = kWhole ? 1 : 2;            // rows of a lane
  constexpr int kWords = D / 16;                     // words that a lane holds of a row of Q or K
  constexpr int kOut = D / 8;                        // 8-column tiles of the output
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<D, W, kRows>& sm = *reinterpret_cast<Smem<D, W, kRows>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = warp_index();
  const int ctas = static_cast<int>(cluster_ctas()), rank = static_cast<int>(cluster_rank());
  if (threadIdx.x == 0) sm.abort = 0;
  if (lane == 0) {
    mbar_init(smem_u32(&sm.k_full[warp]), 1);
    mbar_init(smem_u32(&sm.v_full[warp]), 1);
    mbar_init_fence();
    if (warp == 0) { tma_prefetch_desc(&map_k); tma_prefetch_desc(&map_v); }
  }
  __syncthreads();
  follow_previous_kernel();

  int unit = static_cast<int>(blockIdx.x) / ctas;
  const int group = unit % p.row_groups;
  unit /= p.row_groups;
  const int head = unit % p.Hkv, b = unit / p.Hkv;
  const Seq s = load_seq(p, b);
  // (of a mixed batch the chunk kernel computes sequences longer than the bound in full)
  if (threadIdx.x == 0 && rank == 0 && group == 0 && head == 0 && (s.bad || (s.nq > p.max_q && p.few_rows == 0))) report_index(p.status, 0u, b);
  const int n_rows = s.nq * p.G, row0 = group * kRows;
  if (row0 >= n_rows || (p.few_rows != 0 && n_rows > p.few_rows)) return;      // the whole cluster
  const int end = visible(p, s, min(row0 + kRows - 1, n_rows - 1) / p.G);      // the last token of the group sees most
  const int n_tiles = (end + kTile - 1) / kTile;
  const int first = static_cast<int>(static_cast<long long>(n_tiles) * rank / ctas), last = static_cast<int>(static_cast<long long>(n_tiles) * (rank + 1) / ctas);

  const int g = lane >> 2, t4 = lane & 3, mine = kRows == 4 ? g & 3 : g;      // my row: g, one more of sixteen: g + 8, the same as lane - 16 of four
  uint32_t qa[kHalves][kWords];
  int limit[kHalves], least = 0x7FFFFFFF;            // keys that my rows see, that all rows see (a row that there is not is not stored)
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const int row = row0 + mine + 8 * h, token = row / p.G;
    const bool real = row < n_rows;
    limit[h] = real ? visible(p, s, token) : 0;
    least = min(least, real ? limit[h] : 0x7FFFFFFF);
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (s.q0 + token) * p.q_stride + (head * p.G + row - token * p.G) * D + t4 * (D / 4));
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = real ? src[c] : make_uint4(0u, 0u, 0u, 0u);
      qa[h][4 * c] = w.x; qa[h][4 * c + 1] = w.y; qa[h][4 * c + 2] = w.z; qa[h][4 * c + 3] = w.w;
    }
  }
  least = __reduce_min_sync(0xFFFFFFFFu, least);

  const uint32_t k_tile = smem_u32(sm.ring) + static_cast<uint32_t>(warp * 2 * C::kTileBytes), v_tile = k_tile + C::kTileBytes;
  const uint32_t bar_k = smem_u32(&sm.k_full[warp]), bar_v = smem_u32(&sm.v_full[warp]);
  volatile int* abort_flag = &sm.abort;
  bool bad_page = false;
  auto fetch = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int tile, int page) {
    const int n = copies_of(p, tile * kTile, end);
    if (page < 0 || page >= p.num_pages) { page = p.num_pages; bad_page |= lane < n; }      // reads zeros
    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>((n << p.box_shift) * D));
    __syncwarp();
    if (lane < n) issue_copy<D>(p, map, dst, bar, s, head, tile * kTile, lane, page);
  };

  // Outputs: rows g (and g + 8) times columns n = 2 t4 and 2 t4 + 1 of kOut tiles.
  float o[kHalves][kOut][2], ref[kHalves], sum[kHalves];      // p = 2^((x - ref) c2)
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    ref[h] = -INFINITY;
    sum[h] = 0.f;
#pragma unroll
    for (int j = 0; j < kOut; ++j) o[h][j][0] = o[h][j][1] = 0.f;
  }
  // Eight rows: products of the bytes of P and V, upper bytes of a row in c[0], c[1] and lower ones in c[2], c[3], on top of the bits of kMagic (of 128 keys at most
  // 128 * 255 * 128 < 2^22), go to two columns.
  auto add_products = [&](float (&to)[2], const int (&c)[4], float factor) {
    const float2 less = make_float2(-kMagic, -kMagic);
    const float2 upper = __fadd2_rn(make_float2(__int_as_float(c[0]), __int_as_float(c[1])), less), lower = __fadd2_rn(make_float2(__int_as_float(c[2]), __int_as_float(c[3])), less);
    const float2 sum2 = __ffma2_rn(upper, make_float2(256.f * factor, 256.f * factor), __ffma2_rn(lower, make_float2(factor, factor), make_float2(to[0], to[1])));
    to[0] = sum2.x;
    to[1] = sum2.y;
  };

  bool ok = true;
  unsigned waited = FMHA_I8_DEV_WAIT_K_LOAD;         // what for, if not ok
  auto arrived = [&](bool v) {                       // V has, for all lanes
    ok = __all_sync(0xFFFFFFFFu, v);
    if (!ok) waited = FMHA_I8_DEV_WAIT_V_LOAD;
    return ok;
  };
  uint32_t n = 0;
  int page = 0, next_page = 0;
  if (first + warp < last) {
    page = page_of(p, b, (first + warp) * kTile, end, lane);
    fetch(&map_k, k_tile, bar_k, first + warp, page);
    fetch(&map_v, v_tile, bar_v, first + warp, page);
  }
  for (int tile = first + warp; tile < last; tile += W, ++n) {
    const bool more = tile + W < last;
    if (more) next_page = page_of(p, b, (tile + W) * kTile, end, lane);
    // ---- scores: column n of product j is key 8 j + n; my columns of K are the D / 4 from t4 * D / 4 on
    if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait_timed(bar_k, n & 1u, abort_flag)))) break;
    float x[kHalves][16][2];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      int c[4] = {static_cast<int>(kMagicBits), static_cast<int>(kMagicBits), static_cast<int>(kMagicBits), static_cast<int>(kMagicBits)};
#pragma unroll
      for (int y = 0; y < D / 64; ++y) {
        const uint4 w = lds16(k_tile + chunk_at<D>(8 * j + g, t4 * (D / 64) + y));
        mma16832(c, qa[0][4 * y], kWhole ? 0u : qa[kHalves - 1][4 * y], qa[0][4 * y + 1], kWhole ? 0u : qa[kHalves - 1][4 * y + 1], w.x, w.y);
        mma16832(c, qa[0][4 * y + 2], kWhole ? 0u : qa[kHalves - 1][4 * y + 2], qa[0][4 * y + 3], kWhole ? 0u : qa[kHalves - 1][4 * y + 3], w.z, w.w);
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        x[h][j][0] = __int_as_float(c[2 * h]);
        x[h][j][1] = __int_as_float(c[2 * h + 1]);
      }
    }
    __syncwarp();
    if (more) fetch(&map_k, k_tile, bar_k, tile + W, next_page);

    if (tile * kTile + kTile > least) {
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (tile * kTile + 8 * j + 2 * t4 + i >= limit[h]) x[h][j][i] = -INFINITY;
    }
    // ---- softmax of the tile; lanes with the same g share rows
    float most[kHalves], shrink[kHalves];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = fmaxf(m, fmaxf(x[h][j][0], x[h][j][1]));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      most[h] = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      const float next = fmaxf(ref[h], most[h]);
      moved |= next != ref[h];
      shrink[h] = next == ref[h] ? 1.f : ex2((ref[h] - next) * p.c2);
      ref[h] = next;
    }
    if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          o[h][j][0] *= shrink[h];
          o[h][j][1] *= shrink[h];
        }
    }
    // P as operands: of sixteen rows two fp16 a tile of eight keys, else the whole numbers of two keys, 16 bits each
    uint32_t pa[kHalves][16];
    const float2 c2 = make_float2(p.c2, p.c2), levels = make_float2(kLevels, kLevels), magic = make_float2(8388608.f, 8388608.f);
    float ratio = 1.f;                               // p = ratio * e
    uint32_t mine = 0u;                              // of my keys: sums of their 16-bit numbers, none counted with more than kCap, two in a word
    if constexpr (kWhole) ratio = most[0] == ref[0] ? 1.f : ex2((most[0] - ref[0]) * p.c2);
    auto power = [&](int h, int j) {
      const float to = kWhole ? most[h] : ref[h], base = to == -INFINITY ? 0.f : to;      // a row that sees no key: all e are zero
      const float2 from_base = __fadd2_rn(make_float2(x[h][j][0], x[h][j][1]), make_float2(-base, -base));
      const float2 a = kWhole ? __fmul2_rn(from_base, c2) : __ffma2_rn(from_base, c2, make_float2(kHalfLift, kHalfLift));
      return make_float2(ex2(a.x), ex2(a.y));
    };
    auto pack = [&](const float2& y) { return __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x5410); };
    // 65535 e: 2^23 + its whole part, and 2^23 + rn(65535 times what that leaves)
    auto split = [&](const float2& e, uint32_t& first, uint32_t& second) {
      const float2 y = __ffma2_rd(e, levels, magic), left = __ffma2_rn(e, levels, __fadd2_rn(magic, make_float2(-y.x, -y.y)));
      first = pack(y);
      second = pack(__ffma2_rn(left, levels, magic));
    };
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float2 part = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 e = power(h, j);
        part = __fadd2_rn(part, e);
        if constexpr (kRows == 4) {
          uint32_t first, second;
          split(e, first, second);
          pa[0][j] = lane < 16 ? first : second;
        } else if constexpr (kRows == 8) {
          pa[0][j] = pack(__ffma2_rn(e, levels, magic));
          mine += __vminu2(pa[0][j], kCap * 0x10001u);
        } else {
          const __half2 packed = __floats2half2_rn(e.x, e.y);
          pa[h][j] = *reinterpret_cast<const uint32_t*>(&packed);
        }
      }
      sum[h] = fmaf(sum[h], shrink[h], (part.x + part.y) * ratio);
    }

    // ---- P.V: column n of output tile j is column n * D / 8 + j of V
    const bool here = mbar_wait_timed(bar_v, n & 1u, abort_flag);
    auto load_v = [&](uint32_t (&v)[D / 32], int key) {              // my D / 8 columns of a key
      if constexpr (D == 128) {
        const uint4 w = lds16(v_tile + chunk_at<D>(key, g));
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
      } else {
        const uint2 w = lds8(v_tile + chunk_at<D>(key, g >> 1) + 8 * (g & 1));
        v[0] = w.x; v[1] = w.y;
      }
    };
    // V times whole numbers, one or two of 16 bits for a key; two go over half of the columns at a time where the accumulators of all would be too many.
    auto products = [&](const auto& words) {
      constexpr int kWords = sizeof(words) / sizeof(words[0]), kParts = kWords == 2 && D == 128 ? 2 : 1, kTiles = kOut / kParts;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        int whole[kWords][kTiles][4];
        // 32 keys at a time: bytes 0-3 of a word of P are keys 2 t4, 2 t4 + 1, 8 + 2 t4 and 9 + 2 t4, of the second word 16 more
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          uint32_t a[kWords][4];                     // upper bytes, lower bytes of the first and of the second half of the keys
#pragma unroll
          for (int i = 0; i < kWords; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              a[i][2 * y] = __byte_perm(words[i][4 * kb + 2 * y], words[i][4 * kb + 2 * y + 1], 0x7531);
              a[i][2 * y + 1] = __byte_perm(words[i][4 * kb + 2 * y], words[i][4 * kb + 2 * y + 1], 0x6420);
            }
          uint32_t v[8][D / 32];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int key = 32 * kb + 2 * t4 + (r & 1) + 8 * (r >> 1);
            if constexpr (kParts == 1) {
              load_v(v[r], key);
            } else {
              const uint2 w = lds8(v_tile + chunk_at<D>(key, g) + 8 * part);
              v[r][0] = w.x; v[r][1] = w.y;
            }
          }
#pragma unroll
          for (int w = 0; w < D / 32 / kParts; ++w) {
            uint32_t bytes[2][4];                    // bytes[y][i]: column 4 w + i of the four keys of half y
#pragma unroll
            for (int y = 0; y < 2; ++y) turn4(v[4 * y][w], v[4 * y + 1][w], v[4 * y + 2][w], v[4 * y + 3][w], bytes[y]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int z = 0; z < kWords; ++z) {
                if (kb == 0) mma16832_u<true>(whole[z][4 * w + i], a[z], bytes[0][i], bytes[1][i]);
                else mma16832_u<false>(whole[z][4 * w + i], a[z], bytes[0][i], bytes[1][i]);
              }
          }
        }
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int z = 0; z < kWords; ++z) add_products(o[0][part * kTiles + j], whole[z][j], z == 0 && (kRows == 8 || lane < 16) ? ratio : ratio / kLevels);
      }
    };
    if constexpr (kRows == 4) {
      if (!arrived(here)) break;
      products(pa);
    } else if constexpr (kRows == 8) {
      // Are 16 bits enough?  Not where few keys of the tile have most of a row's weight and the others so little that 2^-17 for each counts: where e, none counted with more
      // than 2^-5, is less than 2^-7 on average over the keys that the row sees.  Elsewhere they are off by 2^-10 of that sum, and by 2^-11 of the tile's weight, at most.
      // (Where each of a row's four lanes has a quarter of it there is nothing to add up.  The question goes with the wait for V.)
      const int least_sum = 511 * min(limit[0] - tile * kTile, kTile);
      int all = static_cast<int>((mine & 0xFFFFu) + (mine >> 16));
      bool thin = false;
      if (!__all_sync(0xFFFFFFFFu, here && 4 * all >= least_sum)) {
        if (!arrived(here)) break;
        all += __shfl_xor_sync(0xFFFFFFFFu, all, 1);
        all += __shfl_xor_sync(0xFFFFFFFFu, all, 2);
        thin = __any_sync(0xFFFFFFFFu, all < least_sum);
      }
      if (thin) {
        uint32_t both[2][16];
#pragma unroll
        for (int j = 0; j < 16; ++j) split(power(0, j), both[0][j], both[1][j]);
        products(both);
      } else {
        products(pa);
      }
    } else {
      if (!arrived(here)) break;
      // sixteen keys at a time
#pragma unroll
      for (int kb = 0; kb < 8; ++kb) {
        uint32_t v[4][D / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) load_v(v[r], 16 * kb + 2 * t4 + (r & 1) + 8 * (r >> 1));
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          const uint32_t a = v[0][w] ^ 0x80808080u, b2 = v[1][w] ^ 0x80808080u, c = v[2][w] ^ 0x80808080u, d = v[3][w] ^ 0x80808080u, e = 0x64646464u;
          const uint32_t ab[2] = {__byte_perm(a, b2, 0x5140), __byte_perm(a, b2, 0x7362)}, cd[2] = {__byte_perm(c, d, 0x5140), __byte_perm(c, d, 0x7362)};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t pick = (i & 1) ? 0x4342 : 0x4140;
            float acc[4] = {o[0][4 * w + i][0], o[0][4 * w + i][1], o[kHalves - 1][4 * w + i][0], o[kHalves - 1][4 * w + i][1]};
            mma16816(acc, pa[0][2 * kb], pa[kHalves - 1][2 * kb], pa[0][2 * kb + 1], pa[kHalves - 1][2 * kb + 1], sub1152(__byte_perm(ab[i >> 1], e, pick)),
                     sub1152(__byte_perm(cd[i >> 1], e, pick)));
            o[0][4 * w + i][0] = acc[0]; o[0][4 * w + i][1] = acc[1];
            o[kHalves - 1][4 * w + i][0] = acc[2]; o[kHalves - 1][4 * w + i][1] = acc[3];
          }
        }
      }
    }
    __syncwarp();
    if (more) fetch(&map_v, v_tile, bar_v, tile + W, next_page);
  }
  if (!ok) {
    if (lane == 0) {
      *abort_flag = 1;
      report(p.status, p.host_word, waited, warp, n);
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { /* copies still in flight land before their memory is used again */ }
    }
    __syncwarp();
  }
  if (bad_page) report_index(p.status, 1u, b);

  // ---- the warp's partial rows go over its own tiles, which it has done with
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 2);
    if (t4 == 0 && g < kRows) sm.stat[warp][g + 8 * h] = make_float2(ref[h], sum[h]);
    float* dst = reinterpret_cast<float*>(sm.ring + warp * 2 * C::kTileBytes) + (g + 8 * h) * D + t4 * (D / 4);
#pragma unroll
    for (int y = 0; y < 2; ++y)                      // columns n = 2 t4 + y: D / 8 neighbours
#pragma unroll
      for (int j = 0; j < kOut; j += 4)
        *reinterpret_cast<float4*>(dst + y * (D / 8) + j) = make_float4(o[h][j][y], o[h][j + 1][y], o[h][j + 2][y], o[h][j + 3][y]);
  }
  __syncthreads();

  // ---- the CTA puts its warps' rows together, then the cluster its CTAs': one thread, four outputs
  constexpr int kQuads = D / 4;
  auto store = [&](int r, int c, float l, float (&a)[4]) {
    const int row = row0 + r, token = row / p.G;
    if (row >= n_rows) return;
    const float scale = l > 0.f ? p.out_scale / (kWhole ? l * kLevels : l) : 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) a[y] = a[y] * scale * p.out_down;
    store4(p.o, p.o_type, (s.q0 + token) * p.o_stride + static_cast<long long>(head * p.G + row - token * p.G) * D + 4 * c, a);
  };
  float* together = reinterpret_cast<float*>(sm.ring + C::kTileBytes);      // behind the first warp's rows
  for (int i = threadIdx.x; i < kRows * kQuads; i += W * 32) {
    const int r = i / kQuads, c = i % kQuads;
    float m = -INFINITY, l = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < W; ++y) m = fmaxf(m, sm.stat[y][r].x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int y = 0; y < W; ++y) {
      const float2 st = sm.stat[y][r];
      const float e = ex2((st.x - base) * p.c2);
      const uint8_t* from = sm.ring + y * 2 * C::kTileBytes + (r * D + 4 * c) * 4;
      float4 v = *reinterpret_cast<const float4*>(from);
      if constexpr (kRows == 4) {                    // what the lower 16 bits of P gave
        const float4 more = *reinterpret_cast<const float4*>(from + 4 * D * 4);
        v = make_float4(v.x + more.x, v.y + more.y, v.z + more.z, v.w + more.w);
      }
      l = fmaf(e, st.y, l);
      a[0] = fmaf(e, v.x, a[0]); a[1] = fmaf(e, v.y, a[1]); a[2] = fmaf(e, v.z, a[2]); a[3] = fmaf(e, v.w, a[3]);
    }
    if (ctas == 1) {
      store(r, c, l, a);
    } else {
      *reinterpret_cast<float4*>(together + r * D + 4 * c) = make_float4(a[0], a[1], a[2], a[3]);
      if (c == 0) sm.together[r] = make_float2(m, l);
    }
  }
  if (ctas == 1) return;
  cluster_arrive();
  cluster_wait();
  const uint32_t rows_at = smem_u32(together), stat_at = smem_u32(sm.together);
  for (int i = rank * W * 32 + threadIdx.x; i < kRows * kQuads; i += ctas * W * 32) {
    const int r = i / kQuads, c = i % kQuads;
    float m = -INFINITY, l = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int y = 0; y < ctas; ++y) m = fmaxf(m, ld_cluster_v2(map_to_rank(stat_at + 8 * r, y)).x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int y = 0; y < ctas; ++y) {
      const float2 st = ld_cluster_v2(map_to_rank(stat_at + 8 * r, y));
      const float4 v = ld_cluster_v4(map_to_rank(rows_at + static_cast<uint32_t>((r * D + 4 * c) * 4), y));
      const float e = ex2((st.x - base) * p.c2);
      l = fmaf(e, st.y, l);
      a[0] = fmaf(e, v.x, a[0]); a[1] = fmaf(e, v.y, a[1]); a[2] = fmaf(e, v.z, a[2]); a[3] = fmaf(e, v.w, a[3]);
    }
    store(r, c, l, a);
  }
  cluster_arrive();                                  // nobody leaves while another still reads its rows
  cluster_wait();
}

}  // namespace rows
}  // namespace fmha
