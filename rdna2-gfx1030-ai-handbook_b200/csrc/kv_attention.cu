// Attention over the paged 8-bit cache.
//
//   s_j = scale * q . (c_j ks_page(j)),   out = sum_j softmax(s)_j c'_j vs_page(j)
//
// The codes go to the matrix unit as they are (every code is an fp16 number)
// and the block scales stay outside the products.  The values' scale is
// folded into the exponent,
//
//   u_j = log2(e) s_j,   n = running max u,   l = sum_j 2^(u_j - n)
//   t_j = u_j + log2 vs_page(j),   m = running max t,   p_j = 2^(t_j - m)
//   out = 2^(m - n) sum_j p_j c'_j / l
//
// so that p_j <= 1 is what the matrix unit multiplies the codes with,
// whatever the blocks' scales are, and rounding p_j to fp16 is relative to
// the largest contribution.  There is one exponential a token: within a block
// 2^(u_j - n) is p_j times a number of the block.  Queries are brought to
// |q| < 2 by a power of two of their own (exact), so fp16 holds bf16 queries
// of any range.  m, n, l and the sums are fp32; l sums the unrounded p_j.
//
// kv_rows_kernel: few query rows.  The rows of one kv head (its query heads
// times the call's tokens) are the N = 8 or 16 columns of mma.sync m16n8k16
// and 16 cached tokens its M: the cache is read once, straight from global
// memory into the operand registers, since a code needs only to be where its
// product is formed, and products may be formed in any order of channels.
#include "../../include/b2_attention.h"
#include "b2_internal.h"
#include "kv_attention.cuh"

namespace b2 {
namespace {

// ----------------------------------------------------------- few query rows
constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = kRowsWarps * kWarp;
constexpr int kRowsTile = 16 * kRowsWarps;  // cached tokens a CTA takes at once
constexpr int kRowsMaxGrid = 1024;

template <int DIM, int NT>
struct RowsShared {
  float sums[kRowsWarps][8 * NT][DIM];
  float m[kRowsWarps][8 * NT], n[kRowsWarps][8 * NT], l[kRowsWarps][8 * NT];
  int64_t scan[kRowsWarps];
  int64_t local;
  int sequence, last;
};

template <int NT>
__device__ __forceinline__ int rows_tiles(const Sequence& s) {
  return max(1, (s.hi + kRowsTile - 1) / kRowsTile - s.lo / kRowsTile);
}

// Row tiles x heads of a sequence, each with rows_tiles() token tiles.
template <int NT>
__device__ __forceinline__ int64_t rows_items(const AttendParams& p, const Sequence& s) {
  return ceil_div64(static_cast<int64_t>(s.count) * p.group, 8 * NT) * p.kv_heads;
}

template <int DIM, int CODE, int NT>
__global__ void __launch_bounds__(kRowsThreads) kv_rows_kernel(AttendParams p) {
  constexpr int kRows = 8 * NT;
  constexpr int kChunks = DIM / 64;  // 16-byte pieces of a key row a lane takes
  constexpr int kVWords = DIM / 32;  // words of a value row a lane takes
  extern __shared__ __align__(16) uint8_t raw[];
  RowsShared<DIM, NT>& sh = *reinterpret_cast<RowsShared<DIM, NT>*>(raw);
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int g = lane / 4, t = lane % 4;
  const int cta = blockIdx.x;

  // ---- this CTA's share of all (item, token tile) pairs, in order
  const auto cost = [&](int b) -> int64_t {
    if (b >= p.tok.batch) return 0;
    const Sequence s = load_sequence(p, b);
    return s.count ? rows_items<NT>(p, s) * rows_tiles<NT>(s) : 0;
  };
  // inclusive sum over the CTA's threads, and the sum of all
  const auto scan = [&](int64_t v, int64_t& all) -> int64_t {
#pragma unroll
    for (int d = 1; d < kWarp; d *= 2) {
      const int64_t o = __shfl_up_sync(kFullMask, v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == kWarp - 1) sh.scan[warp] = v;
    __syncthreads();
    all = 0;
    int64_t before = 0;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      if (w < warp) before += sh.scan[w];
      all += sh.scan[w];
    }
    return v + before;
  };
  int64_t total = 0;
  for (int base = 0; base < p.tok.batch; base += kRowsThreads) {
    int64_t all;
    scan(cost(base + threadIdx.x), all);
    total += all;
  }
  const int64_t parts = min(static_cast<int64_t>(gridDim.x), total);  // CTAs with work: none of them is empty
  if (cta >= parts) return;
  const int64_t begin = cta * total / parts, end = (cta + 1) * total / parts;
  int64_t before = 0;
  for (int base = 0; base < p.tok.batch && before <= begin; base += kRowsThreads) {
    int64_t all;
    const int64_t c = cost(base + threadIdx.x), upto = before + scan(c, all);
    if (upto - c <= begin && begin < upto) {
      sh.sequence = base + threadIdx.x;
      sh.local = begin - (upto - c);
    }
    before += all;
  }
  __syncthreads();
  int b = sh.sequence;
  int64_t local = sh.local;
  Sequence s = load_sequence(p, b);

  for (int64_t at = begin; at < end;) {
    const int tiles = rows_tiles<NT>(s);
    const int64_t row_tiles = ceil_div64(static_cast<int64_t>(s.count) * p.group, kRows);
    const int64_t item = local / tiles;
    const int tile0 = static_cast<int>(local % tiles);
    const int take = static_cast<int>(min(static_cast<int64_t>(tiles - tile0), end - at));
    const int head = static_cast<int>(item / row_tiles);
    const int64_t row0 = item % row_tiles * kRows;
    const int64_t item_begin = at - tile0, item_end = item_begin + tiles;
    const int64_t rows = static_cast<int64_t>(s.count) * p.group;

    // ---- queries: lane (g, t) holds of row g the channels its key chunks hold
    uint32_t qf[NT][kChunks][8];
    float qs[NT][2], m[NT][2], mu[NT][2], l[NT][2], o[NT][kVWords * 2][4];
    float largest = -INFINITY;
    int lo[NT][2], hi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t r = row0 + n * 8 + g;
      uint4 raw_q[kChunks][2];
      uint32_t top = 0;
      float f[kChunks][16];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        raw_q[c][0] = raw_q[c][1] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
          const uint16_t* row = static_cast<const uint16_t*>(p.q) + (s.first + r / p.group) * p.q_token +
                                (head * p.group + r % p.group) * p.q_head + (t + 4 * c) * 16;
          raw_q[c][0] = ldg_v4(row);
          raw_q[c][1] = ldg_v4(row + 8);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float v[8];
          if (p.q_bf16) {
            Vec<__nv_bfloat16>::unpack(raw_q[c][x], v);
          } else {
            Vec<__half>::unpack(raw_q[c][x], v);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[c][8 * x + i] = v[i];
            top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
          }
        }
      }
      top = max(top, __shfl_xor_sync(kFullMask, top, 1));
      top = max(top, __shfl_xor_sync(kFullMask, top, 2));
      float factor, gain;
      row_power(top, factor, gain);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          qf[n][c][i] = pack_half2(f[c][2 * i] * factor, f[c][2 * i + 1] * factor);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        qs[n][j] = __shfl_sync(kFullMask, gain, 8 * t + 4 * j) * p.scale_log2;
        m[n][j] = mu[n][j] = -INFINITY;
        l[n][j] = 0.0f;
        const int64_t rj = row0 + n * 8 + 2 * t + j;
        lo[n][j] = hi[n][j] = 0;
        if (rj < rows) row_bounds(p, s, s.start + rj / p.group, lo[n][j], hi[n][j]);
      }
#pragma unroll
      for (int i = 0; i < kVWords * 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.0f;
    }

    // ---- tokens: each warp its own 16 of every tile
    const int first_tile = s.lo / kRowsTile + tile0;
    for (int i = 0; i < take; ++i) {
      const int base = (first_tile + i) * kRowsTile + warp * 16;
      if (base >= s.hi) break;
      const int64_t page = __ldg(p.table + static_cast<int64_t>(b) * p.width + (base >> p.page_shift));
      if (page < 0 || page >= p.pages) continue;
      const int64_t block = page * p.kv_heads + head;
      const int64_t byte0 = ((block << p.page_shift) + (base & ((1 << p.page_shift) - 1))) * DIM;
      uint4 kw[kChunks][2];
      uint32_t vw[4][kVWords];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint8_t* row = p.k_codes + byte0 + g * DIM + (t + 4 * c) * 16;
        kw[c][0] = ldg_v4(row);
        kw[c][1] = ldg_v4(row + 8 * DIM);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint8_t* row = p.v_codes + byte0 + (2 * t + (x & 1) + 8 * (x >> 1)) * DIM + g * (DIM / 8);
        if constexpr (kVWords == 4) {
          const uint4 w = ldg_v4(row);
          vw[x][0] = w.x, vw[x][1] = w.y, vw[x][2] = w.z, vw[x][3] = w.w;
        } else {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(row));
          vw[x][0] = w.x, vw[x][1] = w.y;
        }
      }
      const float ks = __ldg(p.k_scale + block) * code_gain<CODE>();
      const float lv = value_exponent(__ldg(p.v_scale + block), CODE == kCodeE4M3 ? 8.0f : 0.0f, largest);

      // scores of tokens g and g + 8 (rows) for query rows 2t and 2t + 1
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[n][j] = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint32_t w0[4] = {kw[c][0].x, kw[c][0].y, kw[c][0].z, kw[c][0].w};
        const uint32_t w1[4] = {kw[c][1].x, kw[c][1].y, kw[c][1].z, kw[c][1].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a[4];
          codes_to_half<CODE>(w0[k], a[0], a[2]);
          codes_to_half<CODE>(w1[k], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(sc[n], a, qf[n][c][2 * k], qf[n][c][2 * k + 1]);
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = j & 1, token = base + g + 8 * (j >> 1);
          const bool seen = token >= lo[n][col] && token < hi[n][col];
          sc[n][j] = seen ? fmaf(sc[n][j], qs[n][col] * ks, lv) : -INFINITY;
          top[col] = fmaxf(top[col], sc[n][j]);
        }
#pragma unroll
        for (int col = 0; col < 2; ++col) {
#pragma unroll
          for (int d = 4; d < kWarp; d *= 2) top[col] = fmaxf(top[col], __shfl_xor_sync(kFullMask, top[col], d));
          const float next = fmaxf(m[n][col], top[col]);
          const float alpha = weight_of(m[n][col], next);
          const float ref = next == -INFINITY ? 0.0f : next;
          m[n][col] = next;
          sc[n][col] = exp2_approx(sc[n][col] - ref);
          sc[n][col + 2] = exp2_approx(sc[n][col + 2] - ref);
          const float next_u = fmaxf(mu[n][col], top[col] - lv);
          const float ref_u = next_u == -INFINITY ? 0.0f : next_u;
          l[n][col] = fmaf(l[n][col], weight_of(mu[n][col], next_u),
                           (sc[n][col] + sc[n][col + 2]) * exp2_approx(ref - lv - ref_u));
          mu[n][col] = next_u;
#pragma unroll
          for (int x = 0; x < kVWords * 2; ++x) {
            o[n][x][col] *= alpha;
            o[n][x][col + 2] *= alpha;
          }
        }
        pf[n][0] = transpose_8x8(pack_half2(sc[n][0], sc[n][1]));
        pf[n][1] = transpose_8x8(pack_half2(sc[n][2], sc[n][3]));
      }
      // channels 2x and 2x + 1 of this lane's chunk are output rows g and g + 8
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        const uint32_t l01 = __byte_perm(vw[0][w], vw[1][w], 0x5140), l23 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
        const uint32_t h01 = __byte_perm(vw[2][w], vw[3][w], 0x5140), h23 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
        uint32_t a[4];
        codes_to_half<CODE>(l01, a[0], a[1]);
        codes_to_half<CODE>(h01, a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w], a, pf[n][0], pf[n][1]);
        codes_to_half<CODE>(l23, a[0], a[1]);
        codes_to_half<CODE>(h23, a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w + 1], a, pf[n][0], pf[n][1]);
      }
    }

    // ---- join the warps
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int col = 0; col < 2; ++col) {
        float sum = l[n][col];
#pragma unroll
        for (int d = 4; d < kWarp; d *= 2) sum += __shfl_xor_sync(kFullMask, sum, d);
        if (g == 0) {
          sh.m[warp][n * 8 + 2 * t + col] = m[n][col];
          sh.n[warp][n * 8 + 2 * t + col] = mu[n][col];
          sh.l[warp][n * 8 + 2 * t + col] = sum;
        }
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int col = 0; col < 2; ++col) {
        const int r = n * 8 + 2 * t + col;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, sh.m[w][r]);
        const float weight = weight_of(m[n][col], top);
#pragma unroll
        for (int x = 0; x < kVWords * 2; ++x) {
          sh.sums[warp][r][g * (DIM / 8) + 2 * x] = o[n][x][col] * weight;
          sh.sums[warp][r][g * (DIM / 8) + 2 * x + 1] = o[n][x][col + 2] * weight;
        }
      }
    __syncthreads();

    const bool whole = take == tiles;
    // CTAs that share the item: the one it begins in and those that follow
    const int owner = static_cast<int>(ceil_div64((item_begin + 1) * parts, total) - 1);
    const int sharers = whole ? 1 : static_cast<int>(ceil_div64(item_end * parts, total) - 1) - owner + 1;
    constexpr int kSlot = kRows * (DIM + 3);
    float* slot = p.partial + (static_cast<int64_t>(cta) * 2 + (item_begin >= begin ? 1 : 0)) * kSlot;
    const auto store = [&](int64_t r, int d, float4 v, float top, float top_u, float sum) {
      if (r >= rows) return;
      const float inv = sum == 0.0f ? 0.0f : exp2_approx(top - top_u) / sum;
      const int64_t row = (s.first + r / p.group) * static_cast<int64_t>(p.kv_heads * p.group) + head * p.group +
                          r % p.group;
      uint2 w;
      if (p.q_bf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x * inv, v.y * inv);
        const __nv_bfloat162 c = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
      } else {
        w = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + row * DIM + d) = w;
      if (p.lse != nullptr && d == 0) p.lse[row] = sum == 0.0f ? -INFINITY : (top_u + __log2f(sum)) * kLn2;
    };
    for (int e = threadIdx.x; e < kRows * DIM / 4; e += kRowsThreads) {
      const int r = e / (DIM / 4), d = e % (DIM / 4) * 4;
      float top = -INFINITY, top_u = -INFINITY, sum = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        top = fmaxf(top, sh.m[w][r]);
        top_u = fmaxf(top_u, sh.n[w][r]);
      }
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&sh.sums[w][r][d]);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        sum = fmaf(sh.l[w][r], weight_of(sh.n[w][r], top_u), sum);
      }
      if (sharers == 1) {
        store(row0 + r, d, v, top, top_u, sum);
      } else {
        *reinterpret_cast<float4*>(slot + r * DIM + d) = v;
        if (d == 0) {
          slot[kRows * DIM + r] = top;
          slot[kRows * DIM + kRows + r] = top_u;
          slot[kRows * DIM + 2 * kRows + r] = sum;
        }
      }
    }

    // ---- join the CTAs: the last to arrive adds the parts in their order
    if (sharers > 1) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int arrived = atomicAdd(p.counters + owner, 1);
        sh.last = arrived == sharers - 1;
        if (sh.last) p.counters[owner] = 0;
      }
      __syncthreads();
      if (sh.last) {
        __threadfence();
        for (int e = threadIdx.x; e < kRows * DIM / 4; e += kRowsThreads) {
          const int r = e / (DIM / 4), d = e % (DIM / 4) * 4;
          const auto part = [&](int i) {
            return p.partial + (static_cast<int64_t>(owner + i) * 2 + (i == 0 ? 1 : 0)) * kSlot;
          };
          float top = -INFINITY, top_u = -INFINITY, sum = 0.0f;
          for (int i = 0; i < sharers; ++i) {
            top = fmaxf(top, __ldcg(part(i) + kRows * DIM + r));
            top_u = fmaxf(top_u, __ldcg(part(i) + kRows * DIM + kRows + r));
          }
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int i = 0; i < sharers; ++i) {
            const float weight = weight_of(__ldcg(part(i) + kRows * DIM + r), top);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part(i) + r * DIM + d));
            v.x = fmaf(x.x, weight, v.x), v.y = fmaf(x.y, weight, v.y);
            v.z = fmaf(x.z, weight, v.z), v.w = fmaf(x.w, weight, v.w);
            sum = fmaf(__ldcg(part(i) + kRows * DIM + 2 * kRows + r),
                       weight_of(__ldcg(part(i) + kRows * DIM + kRows + r), top_u), sum);
          }
          store(row0 + r, d, v, top, top_u, sum);
        }
      }
    }
    __syncthreads();

    at += take;
    local += take;
    if (local == row_tiles * p.kv_heads * tiles && at < end) {
      do {
        s = load_sequence(p, ++b);
      } while (s.count == 0);
      local = 0;
    }
  }
}

template <int DIM, int CODE, int NT>
cudaError_t run_rows(const AttendParams& p, int grid, cudaStream_t stream) {
  constexpr int kBytes = sizeof(RowsShared<DIM, NT>);
  static const cudaError_t ready = cudaFuncSetAttribute(
      kv_rows_kernel<DIM, CODE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (ready != cudaSuccess) return ready;
  kv_rows_kernel<DIM, CODE, NT><<<grid, kRowsThreads, kBytes, stream>>>(p);
  return cudaGetLastError();
}

template <int DIM, int CODE>
cudaError_t run_rows_nt(const AttendParams& p, int nt, int grid, cudaStream_t s) {
  return nt == 1 ? run_rows<DIM, CODE, 1>(p, grid, s) : run_rows<DIM, CODE, 2>(p, grid, s);
}

cudaError_t run_rows_any(const AttendParams& p, int dim, int code, int nt, int grid, cudaStream_t s) {
  if (dim == 64)
    return code == kCodeInt8 ? run_rows_nt<64, kCodeInt8>(p, nt, grid, s) : run_rows_nt<64, kCodeE4M3>(p, nt, grid, s);
  return code == kCodeInt8 ? run_rows_nt<128, kCodeInt8>(p, nt, grid, s) : run_rows_nt<128, kCodeE4M3>(p, nt, grid, s);
}

// Most query rows of a (sequence, kv head) that kv_rows_kernel takes; it
// reads the cache once for every 16 of them.
constexpr int64_t kRowsMost = 32;

// How a call is launched: on tensor-core tiles, or with `nt` times 8 columns
// on `grid` CTAs.
struct Plan {
  bool tiles;
  int nt, grid;
  size_t workspace;
};

Plan make_plan(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads, int64_t kv_heads, int64_t dim,
               int64_t width, int64_t page) {
  Plan plan{};
  const int64_t group = q_heads / kv_heads;
  plan.tiles = max_new * group > kRowsMost;
  if (plan.tiles) {
    plan.workspace = kRowsMaxGrid * sizeof(int) + tiles_workspace_bytes(tokens, batch, group, kv_heads,
                                                                        static_cast<int>(dim), width,
                                                                        static_cast<int>(page));
    return plan;
  }
  plan.nt = max_new * group <= 8 ? 1 : 2;
  // no more CTAs than token tiles at the longest that the table can hold
  const int64_t row_tiles = tokens * group / (8 * plan.nt) + batch;
  const int64_t tiles = row_tiles * kv_heads * (ceil_div64(width * page, kRowsTile) + 1);
  const int64_t most = 2 * static_cast<int64_t>(device_sm_count());
  plan.grid = static_cast<int>(tiles < most ? (tiles > 1 ? tiles : 1) : most);
  if (plan.grid > kRowsMaxGrid) plan.grid = kRowsMaxGrid;
  plan.workspace = kRowsMaxGrid * sizeof(int) +
                   static_cast<size_t>(plan.grid) * 2 * (8 * plan.nt) * static_cast<size_t>(dim + 3) * sizeof(float);
  return plan;
}

bool shapes_ok(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads, int64_t kv_heads, int64_t dim,
               int64_t width, int64_t page) {
  if (tokens < 0 || tokens > INT32_MAX / 2 || batch < 0 || batch > (1 << 20) || max_new < 0) return false;
  if (kv_heads < 1 || kv_heads > 65536 || q_heads < kv_heads || q_heads > 65536 || q_heads % kv_heads) return false;
  if ((dim != 64 && dim != 128) || (page != 16 && page != 32 && page != 64 && page != 128)) return false;
  return width >= 0 && width * page <= INT32_MAX / 2;
}

}  // namespace
}  // namespace b2

extern "C" {

size_t b2_kv_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                                       int64_t kv_heads, int64_t dim, int64_t width, int64_t page) {
  if (!b2::shapes_ok(tokens, batch, max_new, q_heads, kv_heads, dim, width, page) || tokens == 0) return 0;
  return b2::make_plan(tokens, batch, max_new, q_heads, kv_heads, dim, width, page).workspace;
}

int b2_kv_attention(const void* q, int dtype, int64_t tokens, int64_t q_heads, int64_t q_token_stride,
                    int64_t q_head_stride, const int32_t* lengths, const int32_t* offsets, int64_t batch,
                    int64_t max_new, const int32_t* table, int64_t width, int code, const void* k_codes,
                    const void* v_codes, const float* k_scale, const float* v_scale, int64_t pages, int64_t kv_heads,
                    int64_t page, int64_t dim, float scale, int causal, int64_t window, void* out, float* lse,
                    void* workspace, size_t workspace_bytes, void* stream) {
  const int invalid = static_cast<int>(cudaErrorInvalidValue);
  const auto aligned = [](const void* x, uintptr_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  if ((dtype != b2::kF16 && dtype != b2::kBF16) || code < 0 || code > 1) return invalid;
  if (!b2::shapes_ok(tokens, batch, max_new, q_heads, kv_heads, dim, width, page)) return invalid;
  if (pages < 0 || pages > INT32_MAX || window < 0 || !(scale > 0.0f) || scale > 3.0e38f) return invalid;
  if (tokens == 0) return 0;
  if (batch < 1 || max_new < 1 || (offsets == nullptr && (tokens % batch || tokens / batch > max_new))) return invalid;
  if (!q || !lengths || (!table && width) || !k_codes || !v_codes || !k_scale || !v_scale || !out) return invalid;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_codes, 16) || !aligned(v_codes, 16)) return invalid;
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return invalid;
  const b2::Plan plan = b2::make_plan(tokens, batch, max_new, q_heads, kv_heads, dim, width, page);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < plan.workspace) return invalid;
  b2::AttendParams p{};
  p.tok = {lengths, offsets, static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(tokens / batch)};
  p.q = q;
  p.q_bf16 = dtype == b2::kBF16;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.table = table;
  p.width = static_cast<int>(width);
  p.k_codes = static_cast<const uint8_t*>(k_codes);
  p.v_codes = static_cast<const uint8_t*>(v_codes);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.pages = pages;
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  p.kv_heads = static_cast<int>(kv_heads);
  p.group = static_cast<int>(q_heads / kv_heads);
  p.scale_log2 = scale * b2::kLog2e;
  p.causal = causal;
  p.window = window;
  p.out = out;
  p.lse = lse;
  p.counters = static_cast<int*>(workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + b2::kRowsMaxGrid * sizeof(int));
  if (plan.tiles)
    return static_cast<int>(
        b2::run_tiles(p, static_cast<int>(dim), code, p.partial, static_cast<cudaStream_t>(stream)));
  return static_cast<int>(
      b2::run_rows_any(p, static_cast<int>(dim), code, plan.nt, plan.grid, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
