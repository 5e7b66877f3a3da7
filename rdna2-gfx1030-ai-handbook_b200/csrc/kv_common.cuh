// Device helpers shared by the rotary, cache-append and cached-attention
// kernels: the rotation of one pair of vectors, 8-bit codes, and the mapping
// from a call's tokens to sequences, positions and pages.
#pragma once

#include "b2_common.cuh"

namespace b2 {

enum RotaryLayout : int { kRotaryHalf = 0, kRotaryInterleaved = 1 };
enum CodeType : int { kCodeInt8 = 0, kCodeE4M3 = 1 };

// Scale of a block whose tokens are all zero: small enough that any later
// token sets the block's scale, large enough that its reciprocal and its
// logarithm are ordinary numbers.
constexpr float kScaleFloor = 7.888609052210118e-31f;  // 2^-100

constexpr int kWarp = 32;
constexpr unsigned kFullMask = 0xffffffffu;

// a / b of non-negative numbers, in 32 bits where they fit: a 64-bit division
// is a hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

inline __host__ __device__ int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------ 16-byte vectors
// Vec<T>::kN elements of T in 16 bytes, widened to fp32 and rounded back.
template <typename T>
struct Vec;

template <>
struct Vec<float> {
  static constexpr int kN = 4;
  __device__ static void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  __device__ static uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  __device__ static void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ uint4 ldg_v4(const void* p) { return __ldg(static_cast<const uint4*>(p)); }

// ------------------------------------------------------------------- rotation
// Two fp32 numbers in a register pair.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// (a, b) -> (a cos - b sin, b cos + a sin), products and sums each rounded to
// fp32, so the result is the same as elementwise torch.  The intrinsics are
// never contracted; a packed mul.rn.f32x2 and the add after it were.
__device__ __forceinline__ void rotate_pair(float& a, float& b, float cos, float sin) {
  const float x = __fsub_rn(__fmul_rn(a, cos), __fmul_rn(b, sin));
  const float y = __fadd_rn(__fmul_rn(b, cos), __fmul_rn(a, sin));
  a = x;
  b = y;
}

// A head is handled in units of two vectors of V elements, so that a unit
// holds whole pairs in either layout: "half" pairs element i with element
// i + rot/2, "interleaved" pairs neighbours.  Unit u covers elements
// [o0, o0 + V) and [o1, o1 + V) and, where it is rotated, the angles
// [pair, pair + V).  rot and dim - rot are multiples of 2V.
struct RotaryUnit {
  int o0, o1, pair;  // pair < 0: not rotated
};

template <int V>
__device__ __forceinline__ RotaryUnit rotary_unit(int u, int rot, bool interleaved) {
  RotaryUnit r;
  const int rotated = rot / (2 * V);
  if (u >= rotated || interleaved) {
    r.o0 = 2 * V * u;
    r.o1 = r.o0 + V;
  } else {
    r.o0 = V * u;
    r.o1 = V * u + rot / 2;
  }
  r.pair = u < rotated ? V * u : -1;
  return r;
}

template <int V>
__device__ __forceinline__ void rotate_unit(float (&a)[V], float (&b)[V], const float (&cos)[V], const float (&sin)[V],
                                            bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      rotate_pair(a[2 * i], a[2 * i + 1], cos[i], sin[i]);
      rotate_pair(b[2 * i], b[2 * i + 1], cos[V / 2 + i], sin[V / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) rotate_pair(a[i], b[i], cos[i], sin[i]);
  }
}

template <int V>
__device__ __forceinline__ void load_angles(const float* row, int rot, float (&cos)[V], float (&sin)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(row + i));
    const float4 y = __ldg(reinterpret_cast<const float4*>(row + rot / 2 + i));
    cos[i] = x.x, cos[i + 1] = x.y, cos[i + 2] = x.z, cos[i + 3] = x.w;
    sin[i] = y.x, sin[i + 1] = y.y, sin[i + 2] = y.z, sin[i + 3] = y.w;
  }
}

// V cosines and sines of one position; NaN for a position outside the table,
// which makes the mistake visible in every value that it reaches.
template <int V>
__device__ __forceinline__ void load_angles(const float* angles, int64_t rows, int rot, int64_t position, int pair,
                                            float (&cos)[V], float (&sin)[V]) {
  if (position < 0 || position >= rows) {
#pragma unroll
    for (int i = 0; i < V; ++i) cos[i] = sin[i] = __int_as_float(0x7fffffff);
    return;
  }
  load_angles<V>(angles + position * rot + pair, rot, cos, sin);
}

// --------------------------------------------------------- tokens of a call
// The new tokens of `batch` sequences, packed: sequence b owns tokens
// [begin(b), begin(b + 1)) and its last one is at position lengths[b] - 1.
struct Tokens {
  const int32_t* lengths;  // [batch], the call's own tokens included
  const int32_t* offsets;  // [batch + 1], or nullptr: `each` tokens a sequence
  int batch, tokens, each;

  // Kept inside [0, tokens] whatever the offsets hold.
  __device__ __forceinline__ int begin(int b) const {
    if (offsets == nullptr) return b * each;
    const int o = __ldg(offsets + b);
    return o < 0 ? 0 : (o > tokens ? tokens : o);
  }
};

// The largest b in [0, batch) with key(b) <= x, for a key that does not
// decrease and has key(0) <= x.  Called by a converged warp: 32 probes a round.
template <typename Key>
__device__ __forceinline__ int warp_search(int batch, int64_t x, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;  // key(lo) <= x, and key(hi) > x or hi == batch
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int b = lo + step * lane;
    const unsigned found = __ballot_sync(kFullMask, b < hi && key(b) <= x);
    const int last = found ? 31 - __clz(found) : 0;
    hi = min(hi, lo + step * (last + 1));
    lo = lo + step * last;
  }
  return lo;
}

// ------------------------------------------------------------------ 8-bit codes
// Four codes of numbers x / scale, round to nearest even.  They are in the
// codes' range but for a rounding, since the scale covers the block (adding
// 1.5 * 2^23 leaves the integer in the low byte; e4m3 saturates).  Where the
// scale is no number the codes are 0: a NaN or an infinity shows by the scale.
template <int CODE>
__device__ __forceinline__ uint32_t pack_codes(const float (&x)[4], float scale) {
  uint32_t w;
  if constexpr (CODE == kCodeInt8) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(__fadd_rn(x[i], 12582912.0f));
    w = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
    w = lo | hi << 16;
  }
  return scale < INFINITY ? w : 0u;
}

// The numbers that four codes stand for, before their scale: an int8 code +
// 128 in the low byte of 2^23 + (c + 128), e4m3 by way of fp16.
template <int CODE>
__device__ __forceinline__ void code_values(uint32_t w, float* f) {
  if constexpr (CODE == kCodeInt8) {
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + j)) - 8388736.0f;
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * j)), __NV_E4M3);
      const float2 v = __half22float2(__half2(h));
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
  }
}

}  // namespace b2
