// What the kernels of attention with grouped heads over packed or paged sequences share (fmha_rows_sm100.cuh,
// fmha_chunk_sm100.cuh): parameters, the geometry of a sequence, where its keys lie.
//
// For every token i of a sequence with n_q query tokens and n_k keys, and every head h with key head h / G:
//   o_i = sum_j softmax_j(c q_i . k_j) v_j,   c = q_amax k_amax / (127^2 sqrt(D)),   j < n_k and, causal, j <= i + n_k - n_q
// (the last query token sees all keys).  A token that sees no key gives zeros.  The scores are exact integers, the probabilities
// p = 2^(c log2(e) (s - m)) are rounded to fp16 for P.V (11 bits: half a step is 2^-11 of a p that is not subnormal, at most), whose other operand, the int8 values, fp16
// holds exactly; up to eight rows, to whole numbers of 32 bits, or of 16 where these add up to errors of 2^-11 of a tile's weight at most (fmha_rows_sm100.cuh).  Products
// are summed in fp32 (those of whole numbers exactly, in 32 bits, before that), and so is the row sum, of the unrounded p.  (8 bits for P, as in the padded calls of this library,
// would be 2^-8 of the largest p for every key: 3 % of the output of a row that spreads over 4096 keys.)
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cstdint>
#include "ptx.cuh"
#include "../../include/fmha_i8_c.h"

namespace fmha {
namespace grouped {

constexpr int kTile = 128;             // keys per tile
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kGrowth = 8.f;
constexpr uint32_t kMagicBits = 0x4B400000u;

struct Params {
  const int8_t* q;
  void* o;
  long long q_stride, o_stride;        // elements from one token to the next
  const int* cu_q;                     // [B + 1]
  const int* cu_k;                     // [B + 1], packed keys
  const int* lens_k;                   // [B], paged keys
  const int* page_table;               // [B, table_width], nullptr: packed keys
  long long table_stride;              // entries from one sequence to the next
  int table_width, page_shift, num_pages;
  int box_shift;                       // log2 of the keys that one copy brings: a page, or a tile where that is less
  int B, H, Hkv, G;
  int total_q, total_k, max_q;
  int o_type, causal;
  int o_wide;                          // rows of o are 32-byte aligned
  int row_groups;                      // rows kernel: groups of 4, 8 or 16 rows per sequence and key head
  int tq;                              // chunk kernel: tokens per tile of 128 rows
  int few_rows;                        // 0, or: sequences with up to this many rows to a key head are the rows kernel's, the others the chunk kernel's
  long long first_unit;                // chunk kernel, units not split: those before this one are another launch's
  float c2;                            // from a difference of scores to an exponent of 2
  int growth;                          // chunk kernel: a reference is kept while the maximum exceeds it by no more than this, 2^kGrowth in p
  float out_scale, out_down;           // from sum p v / sum p, v in codes, to the output's unit: their product (where it is tiny, out_scale over a sum would be none of fp32)
  unsigned* status;                    // eight device status words
  unsigned* host_word;                 // the host-visible failure word
};

// Records which wait ran out first: words {code, block, detail0, detail1}, and tells the host.
__device__ __noinline__ void report(unsigned* status, unsigned* host_word, unsigned code, unsigned detail0, unsigned detail1) {
  if (atomicCAS(&status[0], 0u, code) == 0u) {
    status[1] = blockIdx.x;
    status[2] = detail0;
    status[3] = detail1;
    if (host_word != nullptr) {
      *reinterpret_cast<volatile unsigned*>(host_word) = 1u;
      __threadfence_system();
    }
  }
}

// Records an index that points outside its tensor, in the words behind: that is one caller's data, the output of others is right, so it hides no failure and the host is not told.
__device__ __noinline__ void report_index(unsigned* status, unsigned detail0, unsigned detail1) {
  if (atomicCAS(&status[4], 0u, static_cast<unsigned>(FMHA_I8_DEV_BAD_INDEX)) == 0u) {
    status[5] = blockIdx.x;
    status[6] = detail0;
    status[7] = detail1;
  }
}

// Blocks until the kernels before this one in the stream have finished, and lets the next one start.
__device__ __forceinline__ void follow_previous_kernel() {
  grid_launch_dependents();
  grid_dependency_wait();
}

// One sequence.  What the tables say is cut to what the tensors hold, so that no access leaves them; `bad`: something had to be cut.
struct Seq {
  int q0, nq, k0, nk;
  bool bad;
};
__device__ __forceinline__ Seq load_seq(const Params& p, int b) {
  Seq s;
  const int a0 = p.cu_q[b], a1 = p.cu_q[b + 1];
  s.q0 = min(max(a0, 0), p.total_q);
  const int q1 = min(max(a1, s.q0), p.total_q);
  s.nq = q1 - s.q0;
  s.bad = s.q0 != a0 || q1 != a1;
  if (p.page_table != nullptr) {
    const int n = p.lens_k[b];
    s.k0 = 0;
    s.nk = static_cast<int>(min(static_cast<long long>(max(n, 0)), static_cast<long long>(p.table_width) << p.page_shift));
    s.bad |= s.nk != n;
  } else {
    const int b0 = p.cu_k[b], b1 = p.cu_k[b + 1];
    s.k0 = min(max(b0, 0), p.total_k);
    const int k1 = min(max(b1, s.k0), p.total_k);
    s.nk = k1 - s.k0;
    s.bad |= s.k0 != b0 || k1 != b1;
  }
  return s;
}
// Keys that token t of the sequence sees: the first visible(...) of them.
__device__ __forceinline__ int visible(const Params& p, const Seq& s, int t) {
  return p.causal ? min(max(t + 1 - s.nq + s.nk, 0), s.nk) : s.nk;
}

// The copies that bring keys [key0, key0 + 128) of sequence b: copy i (lane i of the warp that calls this) brings 2^box_shift of them.  `page`
// is what page_of() said for that copy.  Rows past the sequence are of another one, of the rest of a page or zeros: their scores are
// masked, and an int8 value is finite whatever it is.
__device__ __forceinline__ int page_of(const Params& p, int b, int key0, int end, int i) {
  const int key = key0 + (i << p.box_shift);
  if (p.page_table == nullptr || i >= (kTile >> p.box_shift) || key >= end) return 0;
  return p.page_table[b * p.table_stride + (key >> p.page_shift)];
}
__device__ __forceinline__ int copies_of(const Params& p, int key0, int end) {      // copies of this tile that hold a key below `end`
  const int keys = min(kTile, end - key0);
  return (keys + (1 << p.box_shift) - 1) >> p.box_shift;
}
template <int D>
__device__ __forceinline__ void issue_copy(const Params& p, const CUtensorMap* map, uint32_t dst, uint32_t bar, const Seq& s, int head, int key0, int i, int page) {
  const int key = key0 + (i << p.box_shift);
  const bool paged = p.page_table != nullptr;
  tma_load_4d(dst + static_cast<uint32_t>((i << p.box_shift) * D), map, bar, 0, paged ? key & ((1 << p.page_shift) - 1) : s.k0 + key, head, paged ? page : 0);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four int8 as fp16: with the sign bit turned a byte is v + 128, which under the bits 0x6400 reads as 1024 + v + 128; both steps are exact.
__device__ __forceinline__ uint32_t sub1152(uint32_t h) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ void unpack4(uint32_t word, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = word ^ 0x80808080u;
  lo = sub1152(__byte_perm(u, 0x64646464u, 0x4140));
  hi = sub1152(__byte_perm(u, 0x64646464u, 0x4342));
}

// N neighbouring outputs, in units of the output's type before rounding, to its memory; N = 4 (o is 16-byte aligned, and so are its rows).
__device__ __forceinline__ void store4(void* o, int type, long long at, const float (&v)[4]) {
  if (type == FMHA_I8_TYPE_I8) {
    uint32_t word = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= (__float_as_uint(fminf(fmaxf(v[i], -127.f), 127.f) + kMagic) & 0xFFu) << (8 * i);
    *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(o) + at) = word;
  } else if (type == FMHA_I8_TYPE_BF16) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(o) + at) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  } else {
    __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(static_cast<__half*>(o) + at) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
}

// Thirty-two neighbouring outputs x * scale, x as the bits of floats.  A warp's threads write rows of their own, so that every store instruction touches 32 lines
// whatever its width; `wide`: rows are 32-byte aligned, and fewer and wider stores will do.
__device__ __forceinline__ void store32(void* o, int type, bool wide, long long at, const uint32_t (&x)[32], float scale) {
  uint32_t w[16];
  auto value = [&](int i) { return __uint_as_float(x[i]) * scale; };
  if (type == FMHA_I8_TYPE_I8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) v[y] = fminf(fmaxf(value(4 * i + y), -127.f), 127.f) + kMagic;
      w[i] = __byte_perm(__byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x0040), __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x0040), 0x5410);
    }
  } else if (type == FMHA_I8_TYPE_BF16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(value(2 * i), value(2 * i + 1));
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __half2 h = __floats2half2_rn(value(2 * i), value(2 * i + 1));
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  uint8_t* to = static_cast<uint8_t*>(o) + at * (type == FMHA_I8_TYPE_I8 ? 1 : 2);
  const int words = type == FMHA_I8_TYPE_I8 ? 8 : 16;
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    if (i >= words) break;
    if (wide) {
      st_global_v8(to + 4 * i, reinterpret_cast<const uint32_t(&)[8]>(w[i]));
    } else {
      *reinterpret_cast<uint4*>(to + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      *reinterpret_cast<uint4*>(to + 4 * i + 16) = make_uint4(w[i + 4], w[i + 5], w[i + 6], w[i + 7]);
    }
  }
}

}  // namespace grouped
}  // namespace fmha
