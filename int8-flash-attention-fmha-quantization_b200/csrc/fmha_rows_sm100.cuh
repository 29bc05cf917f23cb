// Attention of a few query rows per key head over packed or paged sequences with grouped heads: single new tokens against a cache.
// The formulas are in fmha_grouped_sm100.cuh.
//
// The G heads of a group and the new tokens of a sequence make the rows: row r is token r / G, head r % G of the group, sixteen at a time.
// What bounds it: K and V of a key head are read once for all of a group's rows, so HBM does, 2 D bytes per key.  A tensor-core tile of
// tcgen05.mma has 128 rows; here sixteen are enough, so the products are warp-level ones (m16n8k16, fp16 in, fp32 out), and
//   * a warp owns whole tiles of 128 keys, with its running maximum, sum and output rows in registers; it asks for its next K
//     when it has formed the scores of this one, and for the next V behind P.V;
//   * int8 becomes fp16 in registers on its way from shared memory into the product: integers up to 2048 are exact there, and the
//     scores are exact in fp32 (at most 127 * 127 * 128 < 2^24).  Which key, column or row a lane's element belongs to is free as
//     long as both operands agree, and is chosen so that each lane reads 16 bytes at a time without bank conflicts from the swizzled
//     tiles, and so that the scores' registers are P's operand as they are;
//   * the keys of a sequence are split over the warps of a cluster of CTAs, whose partial rows meet through distributed shared memory.
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace rows {

using namespace grouped;

constexpr int kRows = 16;
constexpr int kMaxCluster = 16;
// 64 KB of tiles per CTA and three CTAs to an SM, or one CTA with three times as many warps
template <int D> struct Cfg {
  static constexpr int kWarps = (D == 128) ? 2 : 4;
  static constexpr int kWarpsWide = 3 * kWarps;
  static constexpr int kTileBytes = kTile * D;
};
template <int D, int W> struct Smem {
  alignas(1024) uint8_t ring[2 * W * kTile * D];     // per warp: one K tile, one V tile; at the end its partial rows
  float2 stat[W][kRows];                             // reference exponent and sum of each partial row
  float weight[kMaxCluster * W][kRows];              // what each partial row counts in the whole
  uint64_t k_full[W], v_full[W];
  int abort;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// grid: clusters of c CTAs, one per (sequence, key head, group of rows).
template <int D, int W>
__global__ void __launch_bounds__(W * 32, W <= 4 ? 3 : 1)
rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  constexpr int kSteps = D / 16;                     // products of 16 columns in a score; 8-column tiles of the output are D / 8
  constexpr int kOut = D / 8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<D, W>& sm = *reinterpret_cast<Smem<D, W>*>(smem_raw);
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
  if (threadIdx.x == 0 && rank == 0 && group == 0 && head == 0 && (s.bad || s.nq > p.max_q)) report(p.status, p.host_word, FMHA_I8_DEV_BAD_INDEX, 0u, b);
  const int n_rows = s.nq * p.G, row0 = group * kRows;
  if (row0 >= n_rows) return;                        // the whole cluster
  const int end = visible(p, s, min(row0 + kRows - 1, n_rows - 1) / p.G);      // the last token of the group sees most
  const int n_tiles = (end + kTile - 1) / kTile;
  const int first = n_tiles * rank / ctas, last = n_tiles * (rank + 1) / ctas; // this CTA's share

  const int g = lane >> 2, t4 = lane & 3;            // my rows: g and g + 8
  uint32_t qa[kSteps][4];
  int limit[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + g + 8 * h, token = row / p.G;
    const bool real = row < n_rows;
    limit[h] = real ? visible(p, s, token) : 0;
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (s.q0 + token) * p.q_stride + (head * p.G + row - token * p.G) * D + t4 * (D / 4));
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const uint4 w = real ? src[c] : make_uint4(0u, 0u, 0u, 0u);
      unpack4(w.x, qa[4 * c][h], qa[4 * c][2 + h]);
      unpack4(w.y, qa[4 * c + 1][h], qa[4 * c + 1][2 + h]);
      unpack4(w.z, qa[4 * c + 2][h], qa[4 * c + 2][2 + h]);
      unpack4(w.w, qa[4 * c + 3][h], qa[4 * c + 3][2 + h]);
    }
  }
  const int least = __reduce_min_sync(0xFFFFFFFFu, min(limit[0], limit[1]));   // keys that all rows see

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

  float o[kOut][4], ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};      // p = 2^(s c2 - ref)
#pragma unroll
  for (int j = 0; j < kOut; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;

  bool ok = true;
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
    float sc[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[j][i] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint4 w = lds16(k_tile + chunk_at<D>(8 * j + g, t4 * (D / 64) + c));
        uint32_t lo, hi;
        unpack4(w.x, lo, hi);
        mma16816(sc[j], qa[4 * c][0], qa[4 * c][1], qa[4 * c][2], qa[4 * c][3], lo, hi);
        unpack4(w.y, lo, hi);
        mma16816(sc[j], qa[4 * c + 1][0], qa[4 * c + 1][1], qa[4 * c + 1][2], qa[4 * c + 1][3], lo, hi);
        unpack4(w.z, lo, hi);
        mma16816(sc[j], qa[4 * c + 2][0], qa[4 * c + 2][1], qa[4 * c + 2][2], qa[4 * c + 2][3], lo, hi);
        unpack4(w.w, lo, hi);
        mma16816(sc[j], qa[4 * c + 3][0], qa[4 * c + 3][1], qa[4 * c + 3][2], qa[4 * c + 3][3], lo, hi);
      }
    }
    __syncwarp();
    if (more) fetch(&map_k, k_tile, bar_k, tile + W, next_page);

    if (tile * kTile + kTile > least) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (tile * kTile + 8 * j + 2 * t4 + (i & 1) >= limit[i >> 1]) sc[j][i] = -INFINITY;
    }
    // ---- softmax of the tile; lanes with the same g share rows
    uint32_t pa[16][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = fmaxf(m, fmaxf(sc[j][2 * h], sc[j][2 * h + 1]));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      const float next = fmaxf(ref[h], m * p.c2);                    // the same float in every lane of the row
      const float base = next == -INFINITY ? 0.f : next;             // a row that has seen no key yet: all p are zero
      const float shrink = ex2(ref[h] - base);
      ref[h] = next;
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p0 = ex2(fmaf(sc[j][2 * h], p.c2, -base)), p1 = ex2(fmaf(sc[j][2 * h + 1], p.c2, -base));
        part += p0 + p1;
        const __half2 packed = __floats2half2_rn(p0, p1);
        pa[j][h] = *reinterpret_cast<const uint32_t*>(&packed);
      }
      sum[h] = fmaf(sum[h], shrink, part);
#pragma unroll
      for (int j = 0; j < kOut; ++j) {
        o[j][2 * h] *= shrink;
        o[j][2 * h + 1] *= shrink;
      }
    }

    // ---- P.V: sixteen keys at a time; column n of output tile j is column n * D / 8 + j of V
    if (!(ok = __all_sync(0xFFFFFFFFu, mbar_wait_timed(bar_v, n & 1u, abort_flag)))) break;
#pragma unroll
    for (int kb = 0; kb < 8; ++kb) {
      uint32_t v[4][D / 32];                         // my D / 8 columns of four keys
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 16 * kb + 2 * t4 + (r & 1) + 8 * (r >> 1);
        if constexpr (D == 128) {
          const uint4 w = lds16(v_tile + chunk_at<D>(key, g));
          v[r][0] = w.x; v[r][1] = w.y; v[r][2] = w.z; v[r][3] = w.w;
        } else {
          const uint2 w = lds8(v_tile + chunk_at<D>(key, g >> 1) + 8 * (g & 1));
          v[r][0] = w.x; v[r][1] = w.y;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t a = v[0][w] ^ 0x80808080u, b2 = v[1][w] ^ 0x80808080u, c = v[2][w] ^ 0x80808080u, d = v[3][w] ^ 0x80808080u;
        const uint32_t ab01 = __byte_perm(a, b2, 0x5140), ab23 = __byte_perm(a, b2, 0x7362), cd01 = __byte_perm(c, d, 0x5140), cd23 = __byte_perm(c, d, 0x7362);
        const uint32_t e = 0x64646464u;
        mma16816(o[4 * w], pa[2 * kb][0], pa[2 * kb][1], pa[2 * kb + 1][0], pa[2 * kb + 1][1], sub1152(__byte_perm(ab01, e, 0x4140)), sub1152(__byte_perm(cd01, e, 0x4140)));
        mma16816(o[4 * w + 1], pa[2 * kb][0], pa[2 * kb][1], pa[2 * kb + 1][0], pa[2 * kb + 1][1], sub1152(__byte_perm(ab01, e, 0x4342)), sub1152(__byte_perm(cd01, e, 0x4342)));
        mma16816(o[4 * w + 2], pa[2 * kb][0], pa[2 * kb][1], pa[2 * kb + 1][0], pa[2 * kb + 1][1], sub1152(__byte_perm(ab23, e, 0x4140)), sub1152(__byte_perm(cd23, e, 0x4140)));
        mma16816(o[4 * w + 3], pa[2 * kb][0], pa[2 * kb][1], pa[2 * kb + 1][0], pa[2 * kb + 1][1], sub1152(__byte_perm(ab23, e, 0x4342)), sub1152(__byte_perm(cd23, e, 0x4342)));
      }
    }
    __syncwarp();
    if (more) fetch(&map_v, v_tile, bar_v, tile + W, next_page);
  }
  if (!ok) {
    if (lane == 0) {
      *abort_flag = 1;
      report(p.status, p.host_word, FMHA_I8_DEV_WAIT_K_LOAD, warp, n);
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { /* copies still in flight land before their memory is used again */ }
    }
    __syncwarp();
  }
  if (bad_page) report(p.status, p.host_word, FMHA_I8_DEV_BAD_INDEX, 1u, b);

  // ---- the warp's partial rows go over its own tiles, which it has done with
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xFFFFFFFFu, sum[h], 2);
    if (t4 == 0) sm.stat[warp][g + 8 * h] = make_float2(ref[h], sum[h]);
    float* dst = reinterpret_cast<float*>(sm.ring + warp * 2 * C::kTileBytes) + (g + 8 * h) * D + t4 * (D / 4);
#pragma unroll
    for (int x = 0; x < 2; ++x)                      // columns n = 2 t4 + x: D / 8 neighbours
#pragma unroll
      for (int j = 0; j < kOut; j += 4)
        *reinterpret_cast<float4*>(dst + x * (D / 8) + j) = make_float4(o[j][2 * h + x], o[j + 1][2 * h + x], o[j + 2][2 * h + x], o[j + 3][2 * h + x]);
  }
  cluster_arrive();
  cluster_wait();

  // ---- every CTA of the cluster puts together its part of the outputs
  const int parts = ctas * W;
  for (int i = threadIdx.x; i < kRows; i += W * 32) {
    float m = -INFINITY, l = 0.f;
    for (int x = 0; x < parts; ++x) m = fmaxf(m, ld_cluster_v2(map_to_rank(smem_u32(&sm.stat[x % W][i]), x / W)).x);
    const float base = m == -INFINITY ? 0.f : m;
    for (int x = 0; x < parts; ++x) {
      const float2 st = ld_cluster_v2(map_to_rank(smem_u32(&sm.stat[x % W][i]), x / W));
      const float e = ex2(st.x - base);
      l = fmaf(e, st.y, l);
      sm.weight[x][i] = e;
    }
    const float inv = l > 0.f ? p.out_scale / l : 0.f;
    for (int x = 0; x < parts; ++x) sm.weight[x][i] *= inv;
  }
  __syncthreads();
  constexpr int kQuads = D / 4;
  for (int i = rank * W * 32 + threadIdx.x; i < kRows * kQuads; i += ctas * W * 32) {
    const int r = i / kQuads, c = i % kQuads, row = row0 + r;
    if (row >= n_rows) break;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < parts; ++x) {
      const float e = sm.weight[x][r];
      if (e == 0.f) continue;                        // a warp without keys for this row
      const float4 v = ld_cluster_v4(map_to_rank(smem_u32(sm.ring + (x % W) * 2 * C::kTileBytes) + static_cast<uint32_t>((r * D + 4 * c) * 4), x / W));
      a[0] = fmaf(e, v.x, a[0]); a[1] = fmaf(e, v.y, a[1]); a[2] = fmaf(e, v.z, a[2]); a[3] = fmaf(e, v.w, a[3]);
    }
    const int token = row / p.G;
    store4(p.o, p.o_type, (s.q0 + token) * p.o_stride + static_cast<long long>(head * p.G + row - token * p.G) * D + 4 * c, a);
  }
  cluster_arrive();                                  // nobody leaves while another still reads its rows
  cluster_wait();
}

}  // namespace rows
}  // namespace fmha
