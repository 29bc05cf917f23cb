// Rotary positions, quantisation to int8 and the write into the cache, in one pass over the outputs of a projection.
//
//   y = rotate(x, position),  code = clamp(floor(y * (127 / amax) + 1/2), -127, 127)
//
// Bound by memory: every element is read once (2 bytes, or 4) and leaves one byte; the rotation is two multiplications an element.  The codes are
// those of 64-bit arithmetic, so that they depend on nothing but their inputs: they are computed in 32 bits, with a bound of the error, and a
// thread one of whose values lies closer to a border between two codes than that computes its values again in 64 bits, with the table's second
// plane.  With normal values that is one thread in 600.
#pragma once
#include "fmha_grouped_sm100.cuh"

namespace fmha {
namespace rope {

using grouped::kMagic;
using grouped::report;

constexpr int kThreads = 256;

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
  int tokens, H, Hkv, rot, interleaved;
  int rounds;                          // a warp goes over rounds * (heads that it takes at once) heads of a token
  int parts;                           // warps per token
  float amax[3], scale[3];             // ranges of q, k, v, and 127 / range
  unsigned* status;
  unsigned* host_word;
};

// Sixteen elements of one head: eight and eight.
template <typename T> struct Load;
template <> struct Load<float> {
  static __device__ __forceinline__ void eight(const float* at, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
};
template <> struct Load<__nv_bfloat16> {
  static __device__ __forceinline__ void eight(const __nv_bfloat16* at, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u); }
  }
};
template <> struct Load<__half> {
  static __device__ __forceinline__ void eight(const __half* at, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
};

// The code of y in 64 bits: the definition.
__device__ __forceinline__ float code_exact(double y, double scale) {
  const double z = floor(__dadd_rn(__dmul_rn(y, scale), 0.5));
  return z == z ? static_cast<float>(fmin(fmax(z, -127.0), 127.0)) : 0.f;
}
// Codes of eight values y (as floats plus kMagic), whose errors are at most `error` in codes.  False if one of them may be another.
__device__ __forceinline__ bool codes_fast(const float (&y)[8], float scale, float error, float (&code)[8]) {
  float least = 1.f, most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // between -127 and -126, and from 127 on, the code is the same; the clamped values lie in the middle of those
    const float z = fminf(fmaxf(fmaf(y[i], scale, 0.5f), -126.5f), 127.5f);
    code[i] = __fadd_rd(z, kMagic);
    const float part = z - (code[i] - kMagic);         // exact
    least = fminf(least, part);
    most = fmaxf(most, part);
  }
  return least > error && most < 1.f - error;
}
__device__ __forceinline__ uint2 pack8(const float (&c)[8]) {
  auto word = [&](int i) {
    return __byte_perm(__byte_perm(__float_as_uint(c[i]), __float_as_uint(c[i + 1]), 0x0040),
                       __byte_perm(__float_as_uint(c[i + 2]), __float_as_uint(c[i + 3]), 0x0040), 0x5410);
  };
  return make_uint2(word(0), word(4));
}

// Sixteen elements, a and b: with kRotate pairs -- (a[i], b[i]), or interleaved neighbours in a and then in b -- are turned by cs; otherwise
// they are quantised as they are.  `low`: second plane of the table for these pairs.
template <bool kRotate>
__device__ __forceinline__ void quantise16(const float (&a)[8], const float (&b)[8], const float2 (&cs)[8], float most_cs, const float* low, bool interleaved, float amax, float scale,
                                           uint2& first, uint2& second) {
  float ya[8], yb[8], most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max3_abs_nan(most, a[i], b[i]);
  if constexpr (kRotate) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x1 = !interleaved ? a[i] : i < 4 ? a[2 * i] : b[2 * i - 8], x2 = !interleaved ? b[i] : i < 4 ? a[2 * i + 1] : b[2 * i - 7];
      const float y1 = fmaf(x1, cs[i].x, -__fmul_rn(x2, cs[i].y)), y2 = fmaf(x2, cs[i].x, __fmul_rn(x1, cs[i].y));
      if (!interleaved) { ya[i] = y1; yb[i] = y2; }
      else if (i < 4) { ya[2 * i] = y1; ya[2 * i + 1] = y2; }
      else { yb[2 * i - 8] = y1; yb[2 * i - 7] = y2; }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) { ya[i] = a[i]; yb[i] = b[i]; }
  }
  // With m the largest |x| and c the largest |cos|, |sin| here, a product is at most m c.  y1: half a step (2^-24) of each of table, product, and sum
  // of two: 2^-24 (2 + 1 + 2) m c; times the scale, itself half a step off (2^-24 of at most 2 m c); and half a step of the result, which counts only
  // below 128 (2^-17).  Together 7 * 2^-24 m c scale + 2^-17 / 2 codes; taken: 2^-21 m c scale + 2^-17.
  const float error = fmaf(most * most_cs * scale, 0x1p-21f, 0x1p-17f);
  float ca[8], cb[8];
  const bool sure_a = codes_fast(ya, scale, error, ca), sure_b = codes_fast(yb, scale, error, cb);
  if (!(sure_a && sure_b)) {
    const double scale64 = 127.0 / static_cast<double>(amax);
    if constexpr (kRotate) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double c = static_cast<double>(cs[i].x) + static_cast<double>(low[2 * i]), s = static_cast<double>(cs[i].y) + static_cast<double>(low[2 * i + 1]);
        const double x1 = !interleaved ? a[i] : i < 4 ? a[2 * i] : b[2 * i - 8], x2 = !interleaved ? b[i] : i < 4 ? a[2 * i + 1] : b[2 * i - 7];
        const float y1 = kMagic + code_exact(__dadd_rn(__dmul_rn(x1, c), -__dmul_rn(x2, s)), scale64);
        const float y2 = kMagic + code_exact(__dadd_rn(__dmul_rn(x2, c), __dmul_rn(x1, s)), scale64);
        if (!interleaved) { ca[i] = y1; cb[i] = y2; }
        else if (i < 4) { ca[2 * i] = y1; ca[2 * i + 1] = y2; }
        else { cb[2 * i - 8] = y1; cb[2 * i - 7] = y2; }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) { ca[i] = kMagic + code_exact(a[i], scale64); cb[i] = kMagic + code_exact(b[i], scale64); }
    }
  }
  first = pack8(ca);
  second = pack8(cb);
}

// A warp takes some heads of one token, 512 / D at a time; thread l of the D / 16 that share a head has pairs 8 l .. 8 l + 7 of it where it is
// rotated, elements 16 l .. 16 l + 15 otherwise.
template <int D, typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const Params p) {
  constexpr int kLanes = D / 16, kHeads = 32 / kLanes;
  grouped::follow_previous_kernel();
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int token = static_cast<int>(w / p.parts), part = static_cast<int>(w - static_cast<long long>(token) * p.parts);
  if (token >= p.tokens) return;
  const int position = p.positions[token];
  long long slot = p.slots != nullptr ? p.slots[token] : 0;
  const bool no_position = position < 0 || position >= p.in_table, no_slot = p.slots != nullptr && slot >= p.num_slots;
  if ((no_position || no_slot) && lane == 0 && part == 0) report(p.status, p.host_word, FMHA_I8_DEV_BAD_INDEX, 2u, token);
  if (no_position) return;
  if (no_slot) slot = -1;
  const bool turned = 16 * l < p.rot;
  const int half = p.rot / 2;
  // elements a = [at_a, at_a + 8) and b = [at_b, at_b + 8)
  const int at_a = turned && !p.interleaved ? 8 * l : 16 * l, at_b = turned && !p.interleaved ? half + 8 * l : 16 * l + 8;
  float2 cs[8];
  float most_cs = 1.f;
  const float* low = nullptr;
  if (turned) {
    const float* row = p.table + (static_cast<long long>(position) * half + 8 * l) * 2;
    low = row + p.in_table * p.rot;
    most_cs = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(row)[i];
      cs[2 * i] = make_float2(t.x, t.y);
      cs[2 * i + 1] = make_float2(t.z, t.w);
      most_cs = max3_abs(max3_abs(most_cs, t.x, t.y), t.z, t.w);
    }
  }
  const int heads = p.H + 2 * p.Hkv;
  const int head0 = part * p.rounds * kHeads + lane / kLanes;
#pragma unroll 1
  for (int r = 0; r < p.rounds; ++r) {
    const int head = head0 + r * kHeads;
    if (head >= heads) break;
    const int kind = head < p.H ? 0 : head < p.H + p.Hkv ? 1 : 2;
    const int h = kind == 0 ? head : kind == 1 ? head - p.H : head - p.H - p.Hkv;
    int8_t* out;
    if (kind == 0) {
      out = p.q_out + (static_cast<long long>(token) * p.H + h) * D;
    } else {
      out = kind == 1 ? p.k_out : p.v_out;
      if (p.slots == nullptr) out += (static_cast<long long>(token) * p.Hkv + h) * D;
      else if (slot >= 0) out += (slot >> p.page_shift) * p.page_stride + ((static_cast<long long>(h) << p.page_shift) + (slot & ((1 << p.page_shift) - 1))) * D;
      else continue;
    }
    const T* in = static_cast<const T*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + token * (kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride) + h * D;
    const float amax = p.amax[kind], scale = p.scale[kind];
    float a[8], b[8];
    uint2 first, second;
    if (turned && kind != 2) {
      Load<T>::eight(in + at_a, a);
      Load<T>::eight(in + at_b, b);
      quantise16<true>(a, b, cs, most_cs, low, p.interleaved != 0, amax, scale, first, second);
      *reinterpret_cast<uint2*>(out + at_a) = first;
      *reinterpret_cast<uint2*>(out + at_b) = second;
    } else {
      Load<T>::eight(in + 16 * l, a);
      Load<T>::eight(in + 16 * l + 8, b);
      quantise16<false>(a, b, cs, 1.f, nullptr, false, amax, scale, first, second);
      *reinterpret_cast<uint4*>(out + 16 * l) = make_uint4(first.x, first.y, second.x, second.y);
    }
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
