// Rotary positions, quantisation to int8 and the write into the cache, in one pass over the outputs of a projection.
//
//   y = rotate(x, position),  code = clamp(floor(y * (127 / amax) + 1/2), -127, 127)
//
// Every element is read once (2 bytes, or 4) and leaves one byte; the rotation is two multiplications an element.  The codes are
// those of 64-bit arithmetic, so that they depend on nothing but their inputs: they are computed in 32 bits, with a bound of the error, and a
// thread one of whose values lies closer to a border between two codes than that looks for it and computes the pair again in 64 bits, with the table's second
// plane.  With normal values and ranges of 3 to 5 that is one thread in 600 to 1100 where they are rotated, and one in 30 to 120 where bf16 values are not: their products
// with the scale reach exact halves.
//
// 8192 tokens of 48 heads of 128, bf16: 42 us, 3.7 TB/s, 57 % of a copy's rate (neighbouring pairs 41, fp16 40, fp32 49).  No unit is full: issue 58 % of the cycles, 245
// instructions of a warp for 512 elements, DRAM 37 %; 4.4 warps to a scheduler, with one head's loads ahead each, do not hide them all.  Pairs of values in one instruction, the next head's loads ahead and the search of the one pair made 76 us 42.  A range of v whose halves are not reached
// (3.93 for 4.25) takes 40.6; the division 127 / range taken out of the 64-bit path changes nothing.
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace rope {

using grouped::kMagic;
using grouped::report_index;

constexpr int kThreads = 128;

struct Params {
  const void *q, *k, *v;
  int8_t *q_out, *k_out, *v_out;
  const int* positions;
  const float* table;                  // [2][in_table][rot / 2][2]
  const long long* slots;              // nullptr: packed outputs
  long long in_table;
  long long q_stride, k_stride, v_stride;      // elements from one token to the next
  long long page_stride, num_slots;
  int page_shift;
  int tokens, H, Hkv, rot;
  int rounds;                          // a warp goes over rounds * (heads that it takes at once) heads of a token
  int parts;                           // warps per token
  float amax[3], scale[3];             // ranges of q, k, v, and 127 / range
  unsigned* status;
};

// Eight neighbouring elements as they are in memory, and as four pairs of floats.
template <typename T> struct Eight { uint4 w; };
template <> struct Eight<float> { float4 w[2]; };
template <typename T> __device__ __forceinline__ void load8(const T* at, Eight<T>& e) {
  if constexpr (sizeof(T) == 4) {
    e.w[0] = reinterpret_cast<const float4*>(at)[0];
    e.w[1] = reinterpret_cast<const float4*>(at)[1];
  } else {
    e.w = *reinterpret_cast<const uint4*>(at);
  }
}
__device__ __forceinline__ float2 pair_of(uint32_t u, __nv_bfloat16) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
__device__ __forceinline__ float2 pair_of(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <typename T> __device__ __forceinline__ void floats(const Eight<T>& e, float2 (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    x[0] = make_float2(e.w[0].x, e.w[0].y); x[1] = make_float2(e.w[0].z, e.w[0].w);
    x[2] = make_float2(e.w[1].x, e.w[1].y); x[3] = make_float2(e.w[1].z, e.w[1].w);
  } else {
    x[0] = pair_of(e.w.x, T()); x[1] = pair_of(e.w.y, T()); x[2] = pair_of(e.w.z, T()); x[3] = pair_of(e.w.w, T());
  }
}

// The code of y in 64 bits: the definition.
__device__ __forceinline__ float code_exact(double y, double scale) {
  const double z = floor(__dadd_rn(__dmul_rn(y, scale), 0.5));
  return z == z ? static_cast<float>(fmin(fmax(z, -127.0), 127.0)) : 0.f;
}
__device__ __forceinline__ uint2 pack8(const float2 (&c)[4]) {
  auto word = [&](const float2& a, const float2& b) {
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
  };
  return make_uint2(word(c[0], c[1]), word(c[2], c[3]));
}
__device__ __forceinline__ float max_abs(float m, const float2 (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max3_abs_nan(m, x[i].x, x[i].y);
  return m;
}

// What a thread knows of the rotations of its eight pairs.
struct Turn {
  float2 c[4], s[4];                   // cosines and sines of pairs 2 i and 2 i + 1
  float most;                          // the largest of them
  const float* low;                    // second plane of the table
};
__device__ __forceinline__ float at(const float2 (&x)[4], int i) { return (i & 1) ? x[i >> 1].y : x[i >> 1].x; }

// Sixteen elements, a and b.  With kTurn they are eight pairs -- (a[i], b[i]), or interleaved neighbours in a and then in b -- and are turned.
template <bool kTurn, bool kInterleaved>
__device__ __forceinline__ void quantise16(float2 (&a)[4], float2 (&b)[4], const Turn& turn, float amax, float scale, uint2& first, uint2& second) {
  const float most = max_abs(max_abs(0.f, a), b);
  float2 y[2][4];
  if constexpr (kTurn && !kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __fmul2_rn(b[i], turn.s[i]);
      y[0][i] = __ffma2_rn(a[i], turn.c[i], make_float2(-t.x, -t.y));
      y[1][i] = __ffma2_rn(b[i], turn.c[i], __fmul2_rn(a[i], turn.s[i]));
    }
  } else if constexpr (kTurn) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = i < 4 ? a[i] : b[i - 4];
      const float c = at(turn.c, i), s = at(turn.s, i);
      y[i >> 2][i & 3] = make_float2(fmaf(v.x, c, -__fmul_rn(v.y, s)), fmaf(v.y, c, __fmul_rn(v.x, s)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { y[0][i] = a[i]; y[1][i] = b[i]; }
  }
  // With m the largest |x| and c the largest |cos|, |sin| here, a product is at most m c.  Half a step (2^-24) of each of table, product, and sum
  // of two: 2^-24 (2 + 1 + 2) m c; times the scale, itself half a step off (2^-24 of at most 2 m c); and half a step of the result, at most 2^-18 below
  // 128.  Together 7 * 2^-24 m c scale + 2^-18 codes; taken: 2^-21 m c scale + 2^-17.
  const float error = fmaf(most * (kTurn ? turn.most : 1.f) * scale, 0x1p-21f, 0x1p-17f);
  // z and the whole number next to it, as kMagic + n: rounded to nearest, which is floor(z + 1/2) unless z lies half way between two.
  const float2 scale2 = make_float2(scale, scale), magic = make_float2(kMagic, kMagic), less = make_float2(-kMagic, -kMagic);
  float2 code[2][4];
  float off = 0.f, largest = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 z = __fmul2_rn(y[h][i], scale2);
      code[h][i] = __fadd2_rn(z, magic);
      const float2 n = __fadd2_rn(code[h][i], less), d = __fadd2_rn(z, make_float2(-n.x, -n.y));
      off = max3_abs_nan(off, d.x, d.y);
      largest = max3_abs_nan(largest, z.x, z.y);
    }
  if (!(largest < 127.25f)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        code[h][i].x = fminf(fmaxf(code[h][i].x, kMagic - 127.f), kMagic + 127.f);
        code[h][i].y = fminf(fmaxf(code[h][i].y, kMagic - 127.f), kMagic + 127.f);
      }
  }
  // (beyond 2^22 a float next to kMagic has no room for n; d is then as large as z or not a number)
  if (!(off < 0.5f - error)) {
    const double scale64 = 127.0 / static_cast<double>(amax);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = i < 4 ? a[i & 3] : b[i & 3];
      const float x1 = kTurn && kInterleaved ? v.x : at(a, i), x2 = kTurn && kInterleaved ? v.y : at(b, i);
      const float c = kTurn ? at(turn.c, i) : 1.f, s = kTurn ? at(turn.s, i) : 0.f;
      // which of the pairs it is: the same as above, within the error
      const float z1 = fmaf(x1, c, -(x2 * s)) * scale, z2 = fmaf(x2, c, x1 * s) * scale;
      const float d = fmaxf(fabsf(z1 - rintf(z1)), fabsf(z2 - rintf(z2)));
      if (d < 0.5f - 2.f * error) continue;
      double c64 = 1.0, s64 = 0.0;
      if (kTurn) {
        c64 = static_cast<double>(c) + static_cast<double>(turn.low[2 * i]);
        s64 = static_cast<double>(s) + static_cast<double>(turn.low[2 * i + 1]);
      }
      const double u1 = x1, u2 = x2;
      const float y1 = kMagic + code_exact(kTurn ? __dadd_rn(__dmul_rn(u1, c64), -__dmul_rn(u2, s64)) : u1, scale64);
      const float y2 = kMagic + code_exact(kTurn ? __dadd_rn(__dmul_rn(u2, c64), __dmul_rn(u1, s64)) : u2, scale64);
      if (kTurn && kInterleaved) {
        code[i >> 2][i & 3] = make_float2(y1, y2);
      } else if (i & 1) {
        code[0][i >> 1].y = y1; code[1][i >> 1].y = y2;
      } else {
        code[0][i >> 1].x = y1; code[1][i >> 1].x = y2;
      }
    }
  }
  first = pack8(code[0]);
  second = pack8(code[1]);
}

// A warp takes some heads of one token, 512 / D at a time; thread l of the D / 16 that share a head has pairs 8 l .. 8 l + 7 of it where it is
// rotated, elements 16 l .. 16 l + 15 otherwise.  The next head's elements are asked for before this one's are quantised.
template <int D, typename T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 5) append_kernel(const Params p) {
  constexpr int kLanes = D / 16, kHeads = 32 / kLanes;
  grouped::follow_previous_kernel();
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int token = static_cast<int>(w / p.parts), part = static_cast<int>(w - static_cast<long long>(token) * p.parts);
  if (token >= p.tokens) return;
  const int position = p.positions[token];
  long long slot = p.slots != nullptr ? p.slots[token] : 0;
  const bool turned = 16 * l < p.rot;
  const int half = p.rot / 2;
  const int heads = p.H + 2 * p.Hkv;
  const int head0 = part * p.rounds * kHeads + lane / kLanes, stop = min(heads, head0 + p.rounds * kHeads);
  Eight<T> a, b, next_a, next_b;
  auto load = [&](int head, Eight<T>& x, Eight<T>& y) {
    const int kind = head < p.H ? 0 : head < p.H + p.Hkv ? 1 : 2;
    const T* in = kind == 0 ? static_cast<const T*>(p.q) + token * p.q_stride + head * D
                  : kind == 1 ? static_cast<const T*>(p.k) + token * p.k_stride + (head - p.H) * D : static_cast<const T*>(p.v) + token * p.v_stride + (head - p.H - p.Hkv) * D;
    const bool apart = !kInterleaved && turned && kind != 2;      // halves of the rotated part
    load8(in + (apart ? 8 * l : 16 * l), x);
    load8(in + (apart ? half + 8 * l : 16 * l + 8), y);
  };
  if (head0 < stop) load(head0, a, b);
  const bool no_position = p.rot > 0 && (position < 0 || position >= p.in_table), no_slot = p.slots != nullptr && slot >= p.num_slots;
  if ((no_position || no_slot) && lane == 0 && part == 0) report_index(p.status, 2u, token);
  if (no_position) return;
  if (no_slot) slot = -1;
  Turn turn;
  turn.most = 0.f;
  turn.low = nullptr;
  if (turned) {
    const float* row = p.table + (static_cast<long long>(position) * half + 8 * l) * 2;
    turn.low = row + p.in_table * p.rot;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(row)[i];
      turn.c[i] = make_float2(t.x, t.z);
      turn.s[i] = make_float2(t.y, t.w);
      turn.most = max3_abs(max3_abs(turn.most, t.x, t.y), t.z, t.w);
    }
  }
#pragma unroll 1
  for (int head = head0; head < stop; head += kHeads) {
    if (head + kHeads < stop) load(head + kHeads, next_a, next_b);
    const int kind = head < p.H ? 0 : head < p.H + p.Hkv ? 1 : 2;
    const int h = kind == 0 ? head : kind == 1 ? head - p.H : head - p.H - p.Hkv;
    int8_t* out = kind == 0 ? p.q_out + (static_cast<long long>(token) * p.H + h) * D : kind == 1 ? p.k_out : p.v_out;
    if (kind != 0)
      out += p.slots == nullptr ? (static_cast<long long>(token) * p.Hkv + h) * D
                                : (slot >> p.page_shift) * p.page_stride + ((static_cast<long long>(h) << p.page_shift) + (slot & ((1 << p.page_shift) - 1))) * D;
    if (kind == 0 || slot >= 0) {
      float2 x[4], y[4];
      floats<T>(a, x);
      floats<T>(b, y);
      uint2 first, second;
      if (turned && kind != 2) quantise16<true, kInterleaved>(x, y, turn, p.amax[kind], p.scale[kind], first, second);
      else quantise16<false, false>(x, y, turn, p.amax[kind], p.scale[kind], first, second);
      if (!kInterleaved && turned && kind != 2) {
        *reinterpret_cast<uint2*>(out + 8 * l) = first;
        *reinterpret_cast<uint2*>(out + half + 8 * l) = second;
      } else {
        *reinterpret_cast<uint4*>(out + 16 * l) = make_uint4(first.x, first.y, second.x, second.y);
      }
    }
    a = next_a;
    b = next_b;
  }
}

// One thread per position and pair.
__global__ void __launch_bounds__(256) rope_table_kernel(const double* inv_freq, int pairs, long long positions, double magnitude, float* table) {
  const long long n = positions * pairs;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    const long long position = i / pairs;
    double s, c;
    sincos(static_cast<double>(position) * inv_freq[i - position * pairs], &s, &c);
    c *= magnitude;
    s *= magnitude;
    const float ch = static_cast<float>(c), sh = static_cast<float>(s);
    reinterpret_cast<float2*>(table)[i] = make_float2(ch, sh);
    reinterpret_cast<float2*>(table)[n + i] = make_float2(static_cast<float>(c - ch), static_cast<float>(s - sh));
  }
}

}  // namespace rope
}  // namespace fmha
