// What the two cached-attention kernels share: a call's parameters, which
// cached tokens a row sees, and the arithmetic of the softmax.
#pragma once

#include "kv_common.cuh"

namespace b2 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A softmax goes on with the reference it has while its weights (in the tile
// kernel their sum over a tile) stay below this.
constexpr float kMostWeight = 49152.0f;

// A reference is set this far below the largest weight, so that fp16 holds
// weights down to 2^-(24 + kReferenceLog2) of that one.  Those below half of
// that round to zero, while the sum of the weights, in fp32, counts them: over
// 2^18 tokens up to 2^-13 of the largest weight is lost with 6, and a quarter
// of it would be with a reference 2^5 above the largest.  What lies between
// here and kMostWeight is what later tokens may bring before the reference is
// raised, which the tile kernel pays for with a second pass over a tile: an
// 8192-token prompt takes 695 us with 6, 688, 680 and 677 us with 3, 0 and -5.
constexpr float kReferenceLog2 = 6.0f;

struct AttendParams {
  Tokens tok;
  const void* q;
  int q_bf16;
  int64_t q_token, q_head;
  const int32_t* table;
  int width;
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const float* k_scale;
  const float* v_scale;
  int64_t pages;
  int page_shift, kv_heads, group;
  float scale_log2;  // scale * log2(e)
  int causal;
  int64_t window;    // 0: none
  void* out;
  float* lse;
  int* status;       // the bounded-wait status word
  int* counters;     // [grid], zero between calls
  float* partial;    // [grid][2] slots
};

// One sequence of the call.
struct Sequence {
  int first, count;     // rows of the call
  int64_t start;        // position of the first one
  int lo, hi;           // cached tokens that any row may see: [lo, hi)
};

__device__ __forceinline__ Sequence load_sequence(const AttendParams& p, int b) {
  Sequence s;
  s.first = p.tok.begin(b);
  s.count = max(0, p.tok.begin(b + 1) - s.first);
  const int length = __ldg(p.tok.lengths + b);
  s.start = static_cast<int64_t>(length) - s.count;
  const int64_t held = static_cast<int64_t>(p.width) << p.page_shift;
  s.hi = static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(length), held)));
  int64_t lo = p.window > 0 ? s.start - p.window + 1 : 0;
  s.lo = static_cast<int>(min(max(lo, int64_t(0)), static_cast<int64_t>(s.hi)));
  return s;
}

// Cached tokens [lo, hi) that the row at `position` sees.
__device__ __forceinline__ void row_bounds(const AttendParams& p, const Sequence& s, int64_t position, int& lo,
                                           int& hi) {
  hi = p.causal ? static_cast<int>(min(max(position + 1, int64_t(0)), static_cast<int64_t>(s.hi))) : s.hi;
  lo = p.window > 0 ? static_cast<int>(min(max(position - p.window + 1, int64_t(0)), static_cast<int64_t>(s.hi))) : 0;
}

// Row r of (sequence, kv head) in the output and in lse.
__device__ __forceinline__ int output_row(const AttendParams& p, const Sequence& s, int head, int r) {
  const int token = r / p.group;
  return (s.first + token) * (p.kv_heads * p.group) + head * p.group + (r - token * p.group);
}

// A row's power of two: q * factor is below 2 in magnitude (4 at the very top
// of the range), and q = (q * factor) * gain.
__device__ __forceinline__ void row_power(uint32_t top_bits, float& factor, float& gain) {
  const uint32_t e = min(max(top_bits >> 23, 1u), 253u);
  factor = __uint_as_float((254u - e) << 23);
  gain = __uint_as_float(e << 23);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^x within 2^-22 of itself, and zero below 2^-126, which no weight needs.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes (the bytes of w, in order) as fp16 operands.
//
// e4m3: every code is an fp16 number; the NaN byte is NaN, which append never
// writes (a NaN or infinite token shows by its block's scale).
//
// int8 keys become operands without their sign: u = c + 128 in the low byte
// of a half is the (subnormal) number u 2^-24, and the score is
// q . u - 128 sum(q), a term of the row that the exponent's product takes in.
// The sums do not cancel much: u is at most 255, twice the codes' spread.
//
// int8 values are converted to c itself, since their weighted sums may cancel
// to any degree: u below an exponent that makes it 1024 + u, minus 1152.
template <int CODE, bool KEYS>
__device__ __forceinline__ void to_operand(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == kCodeE4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u, high = KEYS ? 0u : 0x64646464u;
    lo = __byte_perm(u, high, 0x4140);
    hi = __byte_perm(u, high, 0x4342);
    if constexpr (!KEYS) {
      const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
      const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&lo), bias);
      const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&hi), bias);
      lo = *reinterpret_cast<const uint32_t*>(&x);
      hi = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}

// What the products with keys have to be multiplied by for it.
template <int CODE>
__device__ __forceinline__ float key_gain() {
  return CODE == kCodeInt8 ? 16777216.0f : 1.0f;
}

// A block that no token was appended to may hold any scale: one at or below
// zero has no logarithm and reads as the smallest scale.  NaN stays NaN.
__device__ __forceinline__ float value_scale(float s) { return s < kScaleFloor ? kScaleFloor : s; }

// Quiet blocks.  A token's share of l is its p_j divided by its block's value
// scale, which holds while p_j does not underflow where 2^(u_j - n) counts:
// m is at most n + the largest log2 vs met, so a block within 2^-kQuietLog2 of
// that one has its p_j above 2^-70 there.  A block below it is quiet: its share
// of l is summed from exponentials of its own, against a raised n.
constexpr float kQuietLog2 = 64.0f;

// log2 of a block's value scale, and whether the block is quiet beside the
// largest scale that this warp has met.
__device__ __forceinline__ float value_exponent(float scale, float& largest, bool& quiet) {
  const float lv = __log2f(value_scale(scale));
  largest = fmaxf(largest, lv < 256.0f ? lv : largest);  // an infinite scale is a matter of its own block
  quiet = lv < largest - kQuietLog2;
  return lv;
}

// Two running sums are joined relative to the larger maximum; a side that has
// seen nothing has m = -inf and weight 0.
__device__ __forceinline__ float weight_of(float m, float top) {
  return top == -INFINITY ? 0.0f : exp2_approx(m - top);
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device,
// once for each device (`done`, one entry a device).
inline cudaError_t allow_shared(const void* kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (done[dev]) return cudaSuccess;
  const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done[dev] = set == cudaSuccess;
  return set;
}

// Tiles of 128 cached tokens x 256 query rows on the 5th-generation tensor
// cores (kv_tiles.cu): the workspace and the launch of a call with many rows.
size_t tiles_workspace_bytes(int64_t tokens, int64_t batch, int64_t group, int64_t kv_heads, int dim, int64_t width,
                             int page, int64_t window);
cudaError_t run_tiles(const AttendParams& p, int dim, int code, void* workspace, cudaStream_t stream);

}  // namespace b2
