// Appends keys and values to a paged cache held in 8 bits, with the rotary
// positions applied to the keys (and the call's queries) on the way.
//
// Everything is read and written once (rows past a CTA's registers twice, the
// second time from the second-level cache), so memory bounds it: a block of a
// head is one CTA's work, since its scale needs all of it, and the queries'
// CTAs come behind the blocks' in one grid.  Measured: 65536 tokens, 32 query
// and 8 kv heads of 128, bf16 to e4m3: 270 us for 1.49 GB, 5.5 TB/s; one token
// each for 128 sequences 14 us, a warp a block, and 10 us where no block's
// scale grows, so that no earlier codes are brought to a new one.
//
// A page holds `page` tokens of a sequence for every kv head, K and V apart:
// codes [page][dim] and one fp32 scale, so a token's value is code * scale.
// For each (page, head) that receives tokens, with x the new tokens there
// (keys after rotation), top = 127 or 448:
//
//   s   = max(s_old if the page holds earlier tokens, max|x| / top, 2^-100)
//   c   = RNE(c * (s_old / s))            earlier codes, where s grew
//   c   = clamp(RNE(x * fp32(1 / s)))     new codes
//
// A NaN or infinite token makes s NaN or infinite and with it the block.
// Every division is IEEE, every product rounded on its own.
#include "../../include/b2_attention.h"
#include "b2_internal.h"
#include "kv_common.cuh"

namespace b2 {
namespace {

struct AppendParams {
  Tokens tok;
  const void* k;
  const void* v;
  int64_t k_token, k_head, v_token, v_head;
  const int32_t* table;
  int width;
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* k_scale;
  float* v_scale;
  int64_t pages;
  int page, page_shift, kv_heads;
  const float* angles;
  int64_t rows;
  int rot, interleaved;
  const void* q;
  void* q_out;
  int64_t q_token, q_head;
  int q_heads;
  int slots;        // blocks of tokens this call may touch, at most
  int slots_each;   // of every sequence, where all have the same number of tokens, else 0
  int kv_ctas;      // for slots * kv_heads * 2 blocks; the rest of the grid rotates queries
};

constexpr int kAppendThreads = 256;
// Rows of a block that a thread keeps, rotated and in fp32, between finding
// the block's largest value and quantizing.
constexpr int kHold = 2;

// Slot s of the call belongs to the sequence with first_slot(b) <= s; the
// slots of a sequence are enough for the blocks that its tokens touch,
// floor((n - 2) / page) + 2 at most.
__device__ __forceinline__ int first_slot(const Tokens& tok, int b, int page_shift) {
  return (tok.begin(b) >> page_shift) + 2 * b;
}

// The larger one, or NaN where either is (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// One block of one head, keys or values, by THREADS threads: a warp of its
// own where sequences bring a few tokens each, a CTA where they bring pages
// of them.  Rows beyond the kHold that a thread keeps are read, from the
// second-level cache as a rule, and rotated again.
template <typename T, int DIM, int CODE, int THREADS>
__device__ __forceinline__ void append_block(const AppendParams& p, uint32_t item, int tid) {
  constexpr int V = Vec<T>::kN;
  constexpr int kLanes = DIM / (2 * V);  // lanes a token
  constexpr int kRows = THREADS / kLanes;
  const bool is_v = item & 1;
  const int slot = static_cast<int>((item >> 1) / static_cast<uint32_t>(p.kv_heads));
  const int head = static_cast<int>((item >> 1) - slot * static_cast<uint32_t>(p.kv_heads));

  int b, nth;  // block of the sequence's tokens, counted from the first that the call touches
  if (p.slots_each) {
    b = slot / p.slots_each;
    nth = slot - b * p.slots_each;
  } else {
    b = warp_search(p.tok.batch, slot, [&](int i) { return first_slot(p.tok, i, p.page_shift); });
    nth = slot - first_slot(p.tok, b, p.page_shift);
  }
  const int first = p.tok.begin(b);
  const int count = p.tok.begin(b + 1) - first;
  const int64_t start = static_cast<int64_t>(__ldg(p.tok.lengths + b)) - count;  // position of the first new token
  // block index of this slot, and the positions [from, to) that it receives
  const int64_t block = ((start > 0 ? start : 0) >> p.page_shift) + nth;
  int64_t from = block << p.page_shift, to = from + p.page;
  const bool earlier = from < start;
  from = from > start ? from : start;
  from = from > 0 ? from : 0;
  to = to < start + count ? to : start + count;
  if (nth < 0 || from >= to || block >= p.width) return;  // nth < 0: offsets that decrease
  const int64_t page_id = __ldg(p.table + static_cast<int64_t>(b) * p.width + block);

  // this thread's rows of the block's new ones, kRows apart
  const int rows = static_cast<int>(to - from), row0 = tid / kLanes;
  const RotaryUnit unit = rotary_unit<V>(tid % kLanes, is_v ? 0 : p.rot, p.interleaved);
  const int64_t x_token = is_v ? p.v_token : p.k_token;
  const T* x = static_cast<const T*>(is_v ? p.v : p.k) + head * (is_v ? p.v_head : p.k_head) +
               (first + (from - start) + row0) * x_token;
  const float* angles = p.angles + (from + row0) * p.rot + unit.pair;
  const int in_table = to <= p.rows ? rows : static_cast<int>(p.rows > from ? p.rows - from : 0);
  float a[kHold][V], c[kHold][V];
  const auto load = [&](int batch) {
    uint4 va[kHold], vb[kHold];
    float cos[kHold][V], sin[kHold][V];
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int row = (batch * kHold + i) * kRows;
      va[i] = vb[i] = make_uint4(0, 0, 0, 0);
      if (row0 + row < rows) {
        va[i] = ldg_v4(x + row * x_token + unit.o0);
        vb[i] = ldg_v4(x + row * x_token + unit.o1);
      }
    }
    if (unit.pair >= 0) {  // on their way with the rows
#pragma unroll
      for (int i = 0; i < kHold; ++i) {
        const int row = (batch * kHold + i) * kRows;
        if (row0 + row < in_table) {
          load_angles<V>(angles + row * p.rot, p.rot, cos[i], sin[i]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) cos[i][j] = sin[i][j] = __int_as_float(0x7fffffff);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      Vec<T>::unpack(va[i], a[i]);
      Vec<T>::unpack(vb[i], c[i]);
      if (unit.pair >= 0 && row0 + (batch * kHold + i) * kRows < rows)
        rotate_unit<V>(a[i], c[i], cos[i], sin[i], p.interleaved);
    }
  };

  // the largest magnitude; a NaN stays, and rows that are not there are zero
  float most = 0.0f;
  const int batches = (rows + kRows * kHold - 1) / (kRows * kHold);
#pragma unroll 1
  for (int batch = 0; batch < batches; ++batch) {
    load(batch);
#pragma unroll
    for (int i = 0; i < kHold; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) most = max_nan(most, max_nan(fabsf(a[i][j]), fabsf(c[i][j])));
  }
  uint32_t top = __float_as_uint(most) & 0x7fffffffu;  // ordered like the numbers, NaN above them
  if (page_id < 0 || page_id >= p.pages) return;
  uint8_t* codes = (is_v ? p.v_codes : p.k_codes) + (page_id * p.kv_heads + head) * p.page * DIM;
  float* scale = (is_v ? p.v_scale : p.k_scale) + page_id * p.kv_heads + head;
  const int slot0 = static_cast<int>(from - (block << p.page_shift));  // place of the first new row
  const float was = earlier ? *scale : 0.0f;
  top = __reduce_max_sync(kFullMask, top);
  if constexpr (THREADS > kWarp) {
    __shared__ uint32_t tops[THREADS / kWarp];
    if (tid % kWarp == 0) tops[tid / kWarp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / kWarp; ++i) top = max(top, tops[i]);
  } else {
    __syncwarp();  // every lane has read the scale
  }
  float now = __fdiv_rn(__uint_as_float(top), CODE == kCodeInt8 ? 127.0f : 448.0f);
  now = now < kScaleFloor ? kScaleFloor : now;
  now = (was > now || was != was) ? was : now;

  if (earlier && now != was) {
    const float ratio = __fdiv_rn(was, now);
    const int words = slot0 * (DIM / 4);
    uint32_t* row = reinterpret_cast<uint32_t*>(codes);
    for (int i = tid; i < words; i += THREADS) {
      const uint32_t w = row[i];
      float f[4];
      code_values<CODE>(w, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __fmul_rn(f[j], ratio);
      row[i] = pack_codes<CODE>(f, now);
    }
  }
  if (tid == 0) *scale = now;

  const float inv = __fdiv_rn(1.0f, now);
#pragma unroll 1
  for (int batch = batches - 1; batch >= 0; --batch) {
    if (batch != batches - 1) load(batch);
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const int row = row0 + (batch * kHold + i) * kRows;
      if (row >= rows) break;
      uint32_t wa[V / 4], wc[V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        float f[4], g[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[k] = __fmul_rn(a[i][4 * j + k], inv);
          g[k] = __fmul_rn(c[i][4 * j + k], inv);
        }
        wa[j] = pack_codes<CODE>(f, now);
        wc[j] = pack_codes<CODE>(g, now);
      }
      uint8_t* out = codes + (slot0 + row) * DIM;
      if constexpr (V == 8) {
        *reinterpret_cast<uint2*>(out + unit.o0) = make_uint2(wa[0], wa[1]);
        *reinterpret_cast<uint2*>(out + unit.o1) = make_uint2(wc[0], wc[1]);
      } else {
        *reinterpret_cast<uint32_t*>(out + unit.o0) = wa[0];
        *reinterpret_cast<uint32_t*>(out + unit.o1) = wc[0];
      }
    }
  }
}

// Queries: a warp rotates 32 / lanes heads of one token, kQUnroll times.
constexpr int kQUnroll = 4;

template <typename T, int DIM>
__device__ __forceinline__ void rotate_queries(const AppendParams& p, uint32_t warp) {
  constexpr int V = Vec<T>::kN;
  constexpr int kLanes = DIM / (2 * V), kHeads = kWarp / kLanes;
  const uint32_t chunks = (p.q_heads + kHeads * kQUnroll - 1) / (kHeads * kQUnroll);
  const int token = static_cast<int>(warp / chunks);
  if (token >= p.tok.tokens) return;
  const int b = p.tok.offsets == nullptr ? token / p.tok.each
                                         : warp_search(p.tok.batch, token, [&](int i) { return p.tok.begin(i); });
  const int64_t position = static_cast<int64_t>(__ldg(p.tok.lengths + b)) - p.tok.begin(b + 1) + token;
  const int lane = threadIdx.x % kWarp;
  const RotaryUnit unit = rotary_unit<V>(lane % kLanes, p.rot, p.interleaved);
  float cos[V], sin[V];
  if (unit.pair >= 0) load_angles<V>(p.angles, p.rows, p.rot, position, unit.pair, cos, sin);
  const int head0 = static_cast<int>(warp % chunks) * kHeads * kQUnroll + lane / kLanes;
  const T* x = static_cast<const T*>(p.q) + token * p.q_token;
  T* out = static_cast<T*>(p.q_out) + static_cast<int64_t>(token) * p.q_heads * DIM;
  uint4 va[kQUnroll], vb[kQUnroll];
#pragma unroll
  for (int i = 0; i < kQUnroll; ++i) {
    const int h = head0 + i * kHeads;
    if (h < p.q_heads) {
      va[i] = ldg_v4(x + h * p.q_head + unit.o0);
      vb[i] = ldg_v4(x + h * p.q_head + unit.o1);
    }
  }
#pragma unroll
  for (int i = 0; i < kQUnroll; ++i) {
    const int h = head0 + i * kHeads;
    if (h < p.q_heads) {
      if (unit.pair >= 0) {
        float a[V], c[V];
        Vec<T>::unpack(va[i], a);
        Vec<T>::unpack(vb[i], c);
        rotate_unit<V>(a, c, cos, sin, p.interleaved);
        va[i] = Vec<T>::pack(a);
        vb[i] = Vec<T>::pack(c);
      }
      *reinterpret_cast<uint4*>(out + h * DIM + unit.o0) = va[i];
      *reinterpret_cast<uint4*>(out + h * DIM + unit.o1) = vb[i];
    }
  }
}

template <typename T, int DIM, int CODE, int THREADS>
__global__ void __launch_bounds__(kAppendThreads, 3) append_kernel(AppendParams p) {
  const int cta = blockIdx.x;
  if (cta < p.kv_ctas) {
    const uint32_t item = static_cast<uint32_t>(cta) * (kAppendThreads / THREADS) + threadIdx.x / THREADS;
    if (item < static_cast<uint32_t>(p.slots) * p.kv_heads * 2)
      append_block<T, DIM, CODE, THREADS>(p, item, threadIdx.x % THREADS);
  } else {
    constexpr int kWarps = kAppendThreads / kWarp;
    rotate_queries<T, DIM>(p, static_cast<uint32_t>(cta - p.kv_ctas) * kWarps + threadIdx.x / kWarp);
  }
}

// Up to this many tokens a sequence (on the average, where they differ) a
// block is a warp's: most CTAs would idle otherwise.
constexpr int64_t kFewTokens = 4;

template <typename T, int DIM, int CODE>
cudaError_t run_append(AppendParams p, cudaStream_t stream) {
  constexpr int kHeads = kWarp / (DIM / (2 * Vec<T>::kN));
  const bool few = p.tok.tokens <= kFewTokens * p.tok.batch;
  if (p.tok.offsets == nullptr) {
    p.slots_each = p.tok.each == 1 ? 1 : (p.tok.each - 2) / p.page + 2;
    p.slots = p.slots_each * p.tok.batch;  // at most 2 * tokens
  } else {
    p.slots = (p.tok.tokens >> p.page_shift) + 2 * p.tok.batch;
  }
  const int64_t blocks = static_cast<int64_t>(p.slots) * p.kv_heads * 2;
  const int64_t chunks = p.q != nullptr ? ceil_div64(p.q_heads, kHeads * kQUnroll) : 0;
  if (blocks > INT32_MAX || chunks * p.tok.tokens > INT32_MAX) return cudaErrorInvalidValue;
  p.kv_ctas = static_cast<int>(few ? ceil_div64(blocks, kAppendThreads / kWarp) : blocks);
  const int64_t grid = p.kv_ctas + ceil_div64(chunks * p.tok.tokens, kAppendThreads / kWarp);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  if (few) {
    append_kernel<T, DIM, CODE, kWarp><<<static_cast<unsigned>(grid), kAppendThreads, 0, stream>>>(p);
  } else {
    append_kernel<T, DIM, CODE, kAppendThreads><<<static_cast<unsigned>(grid), kAppendThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T, int DIM>
cudaError_t run_append_code(const AppendParams& p, int code, cudaStream_t s) {
  return code == kCodeInt8 ? run_append<T, DIM, kCodeInt8>(p, s) : run_append<T, DIM, kCodeE4M3>(p, s);
}

template <typename T>
cudaError_t run_append_dim(const AppendParams& p, int dim, int code, cudaStream_t s) {
  return dim == 64 ? run_append_code<T, 64>(p, code, s) : run_append_code<T, 128>(p, code, s);
}

// ------------------------------------------------------------------ read back
// Values of whole pages: [n][kv_heads][page][dim], K and V.
constexpr int kReadThreads = 256;

template <typename T, int CODE>
__global__ void __launch_bounds__(kReadThreads)
    read_kernel(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scale, const float* v_scale,
                const int32_t* pages, int64_t n, int64_t num_pages, int kv_heads, int block_bytes, T* k_out, T* v_out,
                float* scales_out) {
  const uint32_t item = blockIdx.x;  // (page, head, K or V)
  const bool is_v = item & 1;
  const int64_t i = (item >> 1) / static_cast<uint32_t>(kv_heads);
  const int head = static_cast<int>((item >> 1) - i * kv_heads);
  const int64_t page = pages[i];
  T* out = (is_v ? v_out : k_out) + (i * kv_heads + head) * block_bytes;
  const bool held = page >= 0 && page < num_pages;
  const float scale = held ? (is_v ? v_scale : k_scale)[page * kv_heads + head] : __int_as_float(0x7fffffff);
  if (scales_out != nullptr && threadIdx.x == 0) scales_out[((is_v ? n : 0) + i) * kv_heads + head] = scale;
  const uint8_t* codes = (is_v ? v_codes : k_codes) + (held ? (page * kv_heads + head) * block_bytes : 0);
  // eight codes a thread: a warp's stores are contiguous (sixteen, in two
  // stores of 16 bytes each, took 65 us where this takes 58)
#pragma unroll 2
  for (int e = threadIdx.x * 8; e < block_bytes; e += kReadThreads * 8) {
    const uint2 w = held ? __ldg(reinterpret_cast<const uint2*>(codes + e)) : make_uint2(0, 0);
    float f[8];
    code_values<CODE>(w.x, f);
    code_values<CODE>(w.y, f + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], scale);
#pragma unroll
    for (int j = 0; j < 8; j += Vec<T>::kN) {
      float part[Vec<T>::kN];
#pragma unroll
      for (int x = 0; x < Vec<T>::kN; ++x) part[x] = f[j + x];
      *reinterpret_cast<uint4*>(out + e + j) = Vec<T>::pack(part);
    }
  }
}

template <typename T>
cudaError_t run_read(const uint8_t* kc, const uint8_t* vc, const float* ks, const float* vs, const int32_t* pages,
                     int64_t n, int64_t num_pages, int kv_heads, int block_bytes, int code, void* k_out, void* v_out,
                     float* scales, cudaStream_t stream) {
  const int64_t grid = n * kv_heads * 2;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  const unsigned g = static_cast<unsigned>(grid);
  T* k = static_cast<T*>(k_out);
  T* v = static_cast<T*>(v_out);
  if (code == kCodeInt8) {
    read_kernel<T, kCodeInt8><<<g, kReadThreads, 0, stream>>>(kc, vc, ks, vs, pages, n, num_pages, kv_heads,
                                                              block_bytes, k, v, scales);
  } else {
    read_kernel<T, kCodeE4M3><<<g, kReadThreads, 0, stream>>>(kc, vc, ks, vs, pages, n, num_pages, kv_heads,
                                                              block_bytes, k, v, scales);
  }
  return cudaGetLastError();
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace b2

extern "C" {

int b2_kv_append(const void* k, const void* v, int dtype, int64_t tokens, int64_t kv_heads, int64_t dim,
                 int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                 const int32_t* lengths, const int32_t* offsets, int64_t batch, const int32_t* table, int64_t width,
                 const void* q, int64_t q_heads, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                 const float* angles, int64_t angle_rows, int64_t rotary_dim, int layout, int code, void* k_codes,
                 void* v_codes, float* k_scale, float* v_scale, int64_t pages, int64_t page, void* stream) {
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (dtype < b2::kF32 || dtype > b2::kBF16 || layout < 0 || layout > 1 || code < 0 || code > 1) return invalid;
  if (tokens < 0 || tokens > INT32_MAX / 2 || batch < 0 || batch > (1 << 20) || width < 0 || width > INT32_MAX)
    return invalid;
  if (kv_heads < 1 || kv_heads > 65536 || (dim != 64 && dim != 128)) return invalid;
  if (page != 16 && page != 32 && page != 64 && page != 128) return invalid;
  if (pages < 0 || pages > INT32_MAX) return invalid;
  if (tokens == 0) return 0;
  if (batch < 1 || (offsets == nullptr && tokens % batch)) return invalid;
  if (!k || !v || !lengths || (!table && width)) return invalid;
  if (pages && (!k_codes || !v_codes || !k_scale || !v_scale)) return invalid;
  const int64_t unit = dtype == b2::kF32 ? 4 : 8;
  const auto rows_ok = [&](const void* x, int64_t ts, int64_t hs) {
    return b2::aligned16(x) && ts >= 0 && hs >= 0 && ts % unit == 0 && hs % unit == 0;
  };
  if (!rows_ok(k, k_token_stride, k_head_stride) || !rows_ok(v, v_token_stride, v_head_stride)) return invalid;
  if (!b2::aligned16(k_codes) || !b2::aligned16(v_codes)) return invalid;
  if (angles) {
    if (!b2::aligned16(angles) || angle_rows < 1 || rotary_dim < 16 || rotary_dim % 16 || rotary_dim > dim)
      return invalid;
  }
  if (q) {
    if (q_heads < 1 || q_heads > 65536 || !angles || !q_out || !b2::aligned16(q_out)) return invalid;
    if (!rows_ok(q, q_token_stride, q_head_stride)) return invalid;
  }
  b2::AppendParams p{};
  p.tok = {lengths, offsets, static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(tokens / batch)};
  p.k = k;
  p.v = v;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.table = table;
  p.width = static_cast<int>(width);
  p.k_codes = static_cast<uint8_t*>(k_codes);
  p.v_codes = static_cast<uint8_t*>(v_codes);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.pages = pages;
  p.page = static_cast<int>(page);
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  p.kv_heads = static_cast<int>(kv_heads);
  p.angles = angles;
  p.rows = angle_rows;
  p.rot = angles ? static_cast<int>(rotary_dim) : 0;
  p.interleaved = layout == b2::kRotaryInterleaved;
  p.q = q;
  p.q_out = q_out;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.q_heads = static_cast<int>(q_heads);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = static_cast<int>(dim);
  if (dtype == b2::kF32) return static_cast<int>(b2::run_append_dim<float>(p, d, code, s));
  if (dtype == b2::kF16) return static_cast<int>(b2::run_append_dim<__half>(p, d, code, s));
  return static_cast<int>(b2::run_append_dim<__nv_bfloat16>(p, d, code, s));
}

int b2_kv_read(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, int code,
               int64_t num_pages, int64_t kv_heads, int64_t page, int64_t dim, const int32_t* pages, int64_t n,
               int dtype, void* k_out, void* v_out, float* scales_out, void* stream) {
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  if (code < 0 || code > 1 || dtype < b2::kF32 || dtype > b2::kBF16) return invalid;
  if (num_pages < 0 || num_pages > INT32_MAX || kv_heads < 1 || kv_heads > 65536 || n < 0 || n > INT32_MAX)
    return invalid;
  if ((dim != 64 && dim != 128) || (page != 16 && page != 32 && page != 64 && page != 128)) return invalid;
  if (n == 0) return 0;
  if (num_pages && (!k_codes || !v_codes || !k_scale || !v_scale)) return invalid;
  if (!pages || !k_out || !v_out) return invalid;
  if (!b2::aligned16(k_codes) || !b2::aligned16(v_codes) || !b2::aligned16(k_out) || !b2::aligned16(v_out))
    return invalid;
  const auto* kc = static_cast<const uint8_t*>(k_codes);
  const auto* vc = static_cast<const uint8_t*>(v_codes);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int heads = static_cast<int>(kv_heads), bytes = static_cast<int>(page * dim);
  const auto run = dtype == b2::kF32 ? b2::run_read<float> : dtype == b2::kF16 ? b2::run_read<__half>
                                                                               : b2::run_read<__nv_bfloat16>;
  return static_cast<int>(run(kc, vc, k_scale, v_scale, pages, n, num_pages, heads, bytes, code, k_out, v_out,
                              scales_out, s));
}

}  // extern "C"
