// Rotary positions: x [tokens, heads, dim] -> each head's first `rot` channels
// rotated pairwise by the token's angles, the others copied.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)
//
// The gradient with respect to x is the same map with -t.  One pass over
// memory, nothing shared between tokens but the table row, which a lane keeps
// in registers for the heads that its warp takes.  Memory bounds it: 65536
// tokens of 32 heads of 128 in bf16 take 180 us, 6.15 TB/s.
#include "../../include/b2_attention.h"
#include "b2_internal.h"
#include "kv_common.cuh"

namespace b2 {
namespace {

struct RotaryParams {
  const void* x;
  void* out;
  int64_t x_token, x_head, out_token, out_head;  // strides in elements
  int64_t tokens;
  int heads, dim, rot, interleaved;
  float sign;
  const float* angles;  // [rows][rot]: cosines, then sines
  int64_t rows;
  const void* positions;
  int positions_64;
};

__device__ __forceinline__ int64_t position_of(const RotaryParams& p, int64_t token) {
  return p.positions_64 ? static_cast<const int64_t*>(p.positions)[token]
                        : static_cast<const int32_t*>(p.positions)[token];
}

// A warp takes `kRotaryUnroll` groups of heads of one token: each lane keeps
// its unit's angles in registers and loads kRotaryUnroll heads before it
// stores the first.
constexpr int kRotaryUnroll = 4;
constexpr int kRotaryThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_vec_kernel(RotaryParams p, int lanes_row, int chunks) {
  constexpr int V = Vec<T>::kN;
  const uint32_t warp = blockIdx.x * (kRotaryThreads / kWarp) + threadIdx.x / kWarp;
  const int lane = threadIdx.x % kWarp;
  const int64_t token = warp / static_cast<uint32_t>(chunks);
  if (token >= p.tokens) return;
  const int rows = kWarp / lanes_row;  // heads at once
  const int u = lane % lanes_row;
  if (u >= p.dim / (2 * V)) return;
  const RotaryUnit unit = rotary_unit<V>(u, p.rot, p.interleaved);
  float cos[V], sin[V];
  if (unit.pair >= 0) {
    load_angles<V>(p.angles, p.rows, p.rot, position_of(p, token), unit.pair, cos, sin);
#pragma unroll
    for (int i = 0; i < V; ++i) sin[i] *= p.sign;
  }
  const int head0 = static_cast<int>(warp - token * chunks) * rows * kRotaryUnroll + lane / lanes_row;
  const T* x = static_cast<const T*>(p.x) + token * p.x_token;
  T* out = static_cast<T*>(p.out) + token * p.out_token;
  uint4 va[kRotaryUnroll], vb[kRotaryUnroll];
#pragma unroll
  for (int i = 0; i < kRotaryUnroll; ++i) {
    const int h = head0 + i * rows;
    if (h < p.heads) {
      const T* row = x + h * p.x_head;
      va[i] = *reinterpret_cast<const uint4*>(row + unit.o0);
      vb[i] = *reinterpret_cast<const uint4*>(row + unit.o1);
    }
  }
#pragma unroll
  for (int i = 0; i < kRotaryUnroll; ++i) {
    const int h = head0 + i * rows;
    if (h < p.heads) {
      if (unit.pair >= 0) {
        float a[V], b[V];
        Vec<T>::unpack(va[i], a);
        Vec<T>::unpack(vb[i], b);
        rotate_unit<V>(a, b, cos, sin, p.interleaved);
        va[i] = Vec<T>::pack(a);
        vb[i] = Vec<T>::pack(b);
      }
      T* row = out + h * p.out_head;
      *reinterpret_cast<uint4*>(row + unit.o0) = va[i];
      *reinterpret_cast<uint4*>(row + unit.o1) = vb[i];
    }
  }
}

// Any dimension, stride and alignment: one thread for each pair of rotated
// channels and for each channel that is copied.
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_any_kernel(RotaryParams p) {
  const int half = p.rot / 2, items = half + p.dim - p.rot;
  const int64_t total = p.tokens * p.heads * items;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kRotaryThreads + threadIdx.x;
  if (i >= total) return;
  const int item = static_cast<int>(i % items);
  const int64_t row = i / items, token = row / p.heads;
  const int h = static_cast<int>(row % p.heads);
  const T* x = static_cast<const T*>(p.x) + token * p.x_token + h * p.x_head;
  T* out = static_cast<T*>(p.out) + token * p.out_token + h * p.out_head;
  if (item >= half) {
    out[item + half] = x[item + half];
    return;
  }
  const int ia = p.interleaved ? 2 * item : item, ib = p.interleaved ? 2 * item + 1 : item + half;
  const int64_t position = position_of(p, token);
  float cos = __int_as_float(0x7fffffff), sin = cos;
  if (position >= 0 && position < p.rows) {
    cos = p.angles[position * p.rot + item];
    sin = p.angles[position * p.rot + half + item] * p.sign;
  }
  float a = static_cast<float>(x[ia]), b = static_cast<float>(x[ib]);
  rotate_pair(a, b, cos, sin);
  out[ia] = static_cast<T>(a);
  out[ib] = static_cast<T>(b);
}

template <typename T>
cudaError_t run_rotary(const RotaryParams& p, cudaStream_t stream) {
  constexpr int V = Vec<T>::kN;
  const auto whole = [](int64_t v) { return v % V == 0; };
  const bool vec = p.rot % (2 * V) == 0 && (p.dim - p.rot) % (2 * V) == 0 && p.dim <= 2 * V * kWarp &&
                   whole(p.x_token) && whole(p.x_head) && whole(p.out_token) && whole(p.out_head) &&
                   reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.angles) % 16 == 0;
  int64_t threads;
  int lanes_row = 1, chunks = 1;
  if (vec) {
    while (lanes_row < p.dim / (2 * V)) lanes_row *= 2;
    chunks = static_cast<int>(ceil_div64(p.heads, kWarp / lanes_row * kRotaryUnroll));
    threads = p.tokens * chunks * kWarp;
  } else {
    threads = p.tokens * p.heads * (p.dim - p.rot / 2);
  }
  const int64_t blocks = ceil_div64(threads, kRotaryThreads);
  if (blocks > INT32_MAX / (kRotaryThreads / kWarp)) return cudaErrorInvalidValue;  // warps are counted in 32 bits
  const dim3 grid(static_cast<unsigned>(blocks));
  if (vec) {
    rotary_vec_kernel<T><<<grid, kRotaryThreads, 0, stream>>>(p, lanes_row, chunks);
  } else {
    rotary_any_kernel<T><<<grid, kRotaryThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace
}  // namespace b2

extern "C" int b2_rotary(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t x_token_stride,
                         int64_t x_head_stride, const float* angles, int64_t angle_rows, int64_t rotary_dim, int layout,
                         int inverse, const void* positions, int positions_64, void* out, int64_t out_token_stride,
                         int64_t out_head_stride, void* stream) {
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (dtype < b2::kF32 || dtype > b2::kBF16 || layout < 0 || layout > 1) return invalid;
  if (tokens < 0 || heads < 0 || dim < 1 || heads > INT32_MAX || dim > 65536) return invalid;
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > dim || angle_rows < 1) return invalid;
  if (x_token_stride < 0 || x_head_stride < 0 || out_token_stride < 0 || out_head_stride < 0) return invalid;
  if (tokens == 0 || heads == 0) return 0;
  if (!x || !angles || !positions || !out) return invalid;
  b2::RotaryParams p{};
  p.x = x;
  p.out = out;
  p.x_token = x_token_stride;
  p.x_head = x_head_stride;
  p.out_token = out_token_stride;
  p.out_head = out_head_stride;
  p.tokens = tokens;
  p.heads = static_cast<int>(heads);
  p.dim = static_cast<int>(dim);
  p.rot = static_cast<int>(rotary_dim);
  p.interleaved = layout == b2::kRotaryInterleaved;
  p.sign = inverse ? -1.0f : 1.0f;
  p.angles = angles;
  p.rows = angle_rows;
  p.positions = positions;
  p.positions_64 = positions_64;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == b2::kF32) return static_cast<int>(b2::run_rotary<float>(p, s));
  if (dtype == b2::kF16) return static_cast<int>(b2::run_rotary<__half>(p, s));
  return static_cast<int>(b2::run_rotary<__nv_bfloat16>(p, s));
}
