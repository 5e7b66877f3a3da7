// Attention over the paged 8-bit cache.
//
//   s_j = scale * q . (c_j ks_page(j)),   out = sum_j softmax(s)_j c'_j vs_page(j)
//
// The codes go to the matrix unit as they are (every code is an fp16 number)
// and the block scales stay outside the products.  The values' scale is
// folded into the exponent,
//
//   u_j = log2(e) s_j,                  l = sum_j 2^(u_j - n)
//   t_j = u_j + log2 vs_page(j),        p_j = 2^(t_j - m)
//   out = 2^(m - n) sum_j p_j c'_j / l
//
// so that p_j is what the matrix unit multiplies the codes with, whatever the
// blocks' scales are.  p_j is rounded to fp16 for it, by 2^-12 of itself or
// 2^-31 of the largest one: products of 32-bit weights would take twice the
// matrix unit's time or more, and outputs of 16 bits would not show them (fp16
// outputs are off by 2.1e-4 to 2.4e-4 from 64 bits, 2.05e-4 with 32-bit
// weights).  m and n are references near the largest t and u: they are
// set from the first tokens and raised, with what was summed so far brought
// down, only where a weight passes kMostWeight, so that the ordinary step
// looks for no maximum.  There is one exponential a token: within a block
// 2^(u_j - n) is p_j times a number of the block.  Queries are brought to
// |q| < 2 by a power of two of their own, so fp16 holds bf16 queries of any
// range: exactly, but for channels below 2^-14 of a row's largest, which may be
// off by 2^-25 of it.  m, n, l and the sums are fp32; l sums the unrounded p_j.
//
// kv_rows_kernel: few query rows.  The rows of one kv head (its query heads
// times the call's tokens) are the N = 8 or 16 columns of mma.sync m16n8k16
// and 16 cached tokens its M, so that the cache is read once and nothing is
// padded to a large tile.  A code needs only to be where its product is
// formed, and products may be formed in any order of channels and tokens: a
// lane takes whole 16-byte pieces of rows, and the order of rows is the one
// that keeps those reads free of bank conflicts.  Every warp has its own ring
// of 16-token stages, filled by TMA, and its own softmax; the warps of a CTA,
// and the CTAs that share a (sequence, kv head), are joined at its end.
//
// Memory should bound it and does not quite: about 420 instructions a warp for
// 16 tokens of K and V, a third of them conversions.  One sequence of 262131
// tokens, 8 kv heads of 128, 4 rows each, e4m3: 111 us for 537 MB, 4.8 TB/s;
// 64 sequences of up to 8192, 8 rows each, int8: 123 us, 4.2 TB/s.
#include "../../include/b2_attention.h"
#include "b2_internal.h"
#include "kv_attention.cuh"

namespace b2 {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder();  // qgemm.cu

namespace {

// ----------------------------------------------------------- few query rows
constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = kRowsWarps * kWarp;
constexpr int kRowsTile = 16 * kRowsWarps;  // cached tokens a CTA takes at once
constexpr int kRowsMaxGrid = 1024;
// What an item costs beside its token tiles, in tiles: the start of its
// pipeline, its queries and its join.  Shares that left it out made the CTAs
// with many short sequences the last to finish.
constexpr int kItemTiles = 4;

// Stages of a warp's ring, 16 tokens of K and V each: two CTAs of an SM with
// two, or one with four.
template <int NT>
constexpr int kStages = NT == 1 ? 2 : 4;

// A run of token tiles (none, if only kItemTiles fall to it) of one item: a sequence, a kv head and 8 * NT rows.
// Kept in shared memory, the registers being short.
struct Segment {
  Sequence s;
  int b, head, tile0, take, tiles;
  int unit0, units;  // its part of the item's kItemTiles + tiles
  int row0, rows;
  int64_t local, at;  // `local` and `at`: its first tile within the sequence's and within all
};

template <int DIM, int NT>
struct __align__(1024) RowsShared {
  uint8_t ring[kRowsWarps][kStages<NT>][2][16 * DIM];
  float sums[kRowsWarps][8 * NT][DIM];
  float m[kRowsWarps][8 * NT], n[kRowsWarps][8 * NT], l[kRowsWarps][8 * NT];
  uint64_t full[kRowsWarps][kStages<NT>];
  int block[kRowsWarps][kStages<NT>];  // of a stage's tokens, or -1
  int64_t scan[kRowsWarps];
  Segment seg[2];
  int last, abort;
};

__device__ __forceinline__ int rows_tiles(const Sequence& s) {
  return max(1, (s.hi + kRowsTile - 1) / kRowsTile - s.lo / kRowsTile);
}

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Where channels d .. d + 3 of row r lie while warps are joined: rows 2t (and
// 2t + 1), which a quarter-warp writes at once, in banks of their own.
template <int DIM>
__device__ __forceinline__ int sum_place(int r, int d) {
  const int t = r >> 1 & 3;
  return d ^ (DIM == 128 ? t : (t & 1) | (t & 2) << 1) << 2;
}

// Row of a stage that holds the i-th token of each half of 8.  Keys are read
// by quarter-warps of two rows (i, i + 1), values by t = 0..3 of rows 2t, then
// of rows 2t + 1; in this order, under the swizzle of the load, neither meets
// a bank twice.
template <int DIM>
__device__ __forceinline__ int stage_row(int i) {
  return (DIM == 128 ? 0x37156240u : 0x65742130u) >> (4 * i) & 7;
}

// Byte `at` of row `row` in a stage as the load swizzles it.
template <int DIM>
__device__ __forceinline__ uint32_t stage_byte(int row, int at) {
  return row * DIM + (DIM == 128 ? at ^ ((row & 7) << 4) : at ^ ((row >> 1 & 3) << 4));
}

template <int NT>
__device__ __forceinline__ Segment segment_at(const AttendParams& p, const Sequence& s, int b, int64_t local,
                                              int64_t at, int64_t end) {
  Segment g;
  g.s = s;
  g.b = b;
  g.local = local;
  g.at = at;
  g.rows = s.count * p.group;
  g.tiles = rows_tiles(s);
  const int row_tiles = (g.rows + 8 * NT - 1) / (8 * NT), all = kItemTiles + g.tiles;
  const int64_t item = quotient(local, all);
  g.unit0 = static_cast<int>(local - item * all);
  g.units = static_cast<int>(min(static_cast<int64_t>(all - g.unit0), end - at));
  g.tile0 = max(0, g.unit0 - kItemTiles);
  g.take = max(0, g.unit0 + g.units - kItemTiles) - g.tile0;
  g.head = static_cast<int>(quotient(item, row_tiles));
  g.row0 = static_cast<int>(item - static_cast<int64_t>(g.head) * row_tiles) * (8 * NT);
  return g;
}

template <int DIM, int CODE, int NT>
__global__ void __launch_bounds__(kRowsThreads, NT == 1 ? 2 : 1)
    kv_rows_kernel(const AttendParams p, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map) {
  constexpr int kRows = 8 * NT, kRing = kStages<NT>;
  constexpr int kChunks = DIM / 64;  // 16-byte pieces of a key row a lane takes
  constexpr int kVWords = DIM / 32;  // words of a value row a lane takes
  extern __shared__ uint8_t raw[];
  RowsShared<DIM, NT>& sh =
      *reinterpret_cast<RowsShared<DIM, NT>*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int g = lane / 4, t = lane % 4;
  const int cta = blockIdx.x;
  if (lane == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(&sh.full[warp][i], 1);
    if (warp == 0) sh.abort = 0;
    fence_mbar_init();
  }

  // ---- this CTA's share of all items' tiles, in order
  const auto cost = [&](int b) -> int64_t {
    if (b >= p.tok.batch) return 0;
    const Sequence s = load_sequence(p, b);
    return static_cast<int64_t>((s.count * p.group + kRows - 1) / kRows) * p.kv_heads * (kItemTiles + rows_tiles(s));
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
  int64_t total = 0, first_cost = 0, first_upto = 0;
  for (int base = 0; base < p.tok.batch; base += kRowsThreads) {
    int64_t all;
    const int64_t c = cost(base + threadIdx.x), upto = scan(c, all);
    if (base == 0) first_cost = c, first_upto = upto;
    total += all;
  }
  const int64_t parts = min(static_cast<int64_t>(gridDim.x), total);  // CTAs with work: none of them is empty
  if (cta >= parts) return;
  const int64_t begin = quotient(cta * total, parts), end = quotient((cta + 1) * total, parts);
  int64_t before = 0;
  for (int base = 0; base < p.tok.batch && before <= begin; base += kRowsThreads) {
    int64_t all = 0, c = first_cost, upto = first_upto;
    if (base > 0 || p.tok.batch > kRowsThreads) {
      c = cost(base + threadIdx.x);
      upto = before + scan(c, all);
    }
    if (upto - c <= begin && begin < upto) {
      const int b = base + threadIdx.x;
      sh.seg[0] = segment_at<NT>(p, load_sequence(p, b), b, begin - (upto - c), begin, end);
    }
    before += all;
  }
  __syncthreads();

  // ---- this warp's ring, and its groups of the segment at hand
  uint32_t issued = 0, used = 0;  // stages, ever
  bool failed = false;            // a wait gave up: no more loads, and no more waits but those for loads in flight
  int groups = 0, base0 = 0;
  int next_block = -1;            // of the group that is issued next
  float next_ks = 0.0f, next_vs = 0.0f;
  const auto block_at = [&](const Segment& seg, int i) -> int {
    if (i >= groups) return -1;
    const int token = base0 + i * kRowsTile;
    const int page = __ldg(p.table + static_cast<int64_t>(seg.b) * p.width + (token >> p.page_shift));
    return page >= 0 && page < p.pages ? page * p.kv_heads + seg.head : -1;
  };
  const auto issue = [&](int i, int block) {
    const int stage = issued % kRing;
    if (elect_one()) {
      sh.block[warp][stage] = block;
      uint64_t* bar = &sh.full[warp][stage];
      if (block >= 0) {
        const int y = (base0 + i * kRowsTile) & ((1 << p.page_shift) - 1);
        mbar_arrive_expect_tx(bar, 2 * 16 * DIM);
        tma_load_3d(&k_map, bar, sh.ring[warp][stage][0], 0, y, block);
        tma_load_3d(&v_map, bar, sh.ring[warp][stage][1], 0, y, block);
      } else {
        mbar_arrive(bar);
      }
    }
    ++issued;
    __syncwarp();
  };
  const auto fetch_scales = [&] {
    const int block = sh.block[warp][used % kRing];
    next_ks = block < 0 ? 0.0f : __ldg(p.k_scale + block);
    next_vs = block < 0 ? 0.0f : __ldg(p.v_scale + block);
  };
  const auto start = [&](const Segment& seg) {
    base0 = (seg.s.lo / kRowsTile + seg.tile0) * kRowsTile + warp * 16;
    groups = base0 < seg.s.hi && !failed ? min(seg.take, (seg.s.hi - base0 + kRowsTile - 1) / kRowsTile) : 0;
    int block[kRing];
#pragma unroll
    for (int i = 0; i < kRing; ++i) block[i] = block_at(seg, i);
#pragma unroll
    for (int i = 0; i < kRing; ++i)
      if (i < groups) issue(i, block[i]);
    next_block = block_at(seg, kRing);
    if (groups > 0) fetch_scales();
  };

  start(sh.seg[0]);
  for (int which = 0;; which ^= 1) {
    const Segment& seg = sh.seg[which];
    const bool more = seg.at + seg.units < end;
    if (more && threadIdx.x == kRowsThreads - 1) {  // seen by the others after the barrier below
      Sequence s = seg.s;
      int b = seg.b;
      int64_t local = seg.local + seg.units;
      if (local == static_cast<int64_t>((seg.rows + kRows - 1) / kRows) * p.kv_heads * (kItemTiles + seg.tiles)) {
        do {
          s = load_sequence(p, ++b);
        } while (s.count == 0);
        local = 0;
      }
      sh.seg[which ^ 1] = segment_at<NT>(p, s, b, local, seg.at + seg.units, end);
    }
    __syncwarp();
    const int row0 = seg.row0, rows = seg.rows;
    // ---- queries: lane (g, t) holds of row g the channels its key chunks hold
    uint32_t qf[NT][kChunks][8];
    float qa[NT][2], qb[NT][2];  // u = product * qa * ks + qb * ks
    float m[NT][2], mu[NT][2], l[NT][2], o[NT][kVWords * 2][4];
    int lo[NT][2], hi[NT][2];
    float largest = -INFINITY;
    int lo_most = 0, hi_least = INT32_MAX;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + n * 8 + g;
      uint4 raw_q[kChunks][2];
      uint32_t top = 0;
      float f[kChunks][16], sum = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        raw_q[c][0] = raw_q[c][1] = make_uint4(0, 0, 0, 0);
        if (r < rows) {
          const uint16_t* row = static_cast<const uint16_t*>(p.q) + (seg.s.first + r / p.group) * p.q_token +
                                (seg.head * p.group + r % p.group) * p.q_head + (t + 4 * c) * 16;
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
        for (int i = 0; i < 8; ++i) {
          qf[n][c][i] = pack_half2(f[c][2 * i] * factor, f[c][2 * i + 1] * factor);
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&qf[n][c][i]));
          sum += h.x + h.y;
        }
      sum += __shfl_xor_sync(kFullMask, sum, 1);
      sum += __shfl_xor_sync(kFullMask, sum, 2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float qs = __shfl_sync(kFullMask, gain, 8 * t + 4 * j) * p.scale_log2;
        qa[n][j] = qs * key_gain<CODE>();
        qb[n][j] = CODE == kCodeInt8 ? -128.0f * __shfl_sync(kFullMask, sum, 8 * t + 4 * j) * qs : 0.0f;
        m[n][j] = mu[n][j] = -INFINITY;
        l[n][j] = 0.0f;
        const int rj = row0 + n * 8 + 2 * t + j;
        lo[n][j] = 0;
        hi[n][j] = INT32_MAX;  // a row that is not one of the sequence's: whatever it sums is not stored
        if (rj < rows) row_bounds(p, seg.s, seg.s.start + rj / p.group, lo[n][j], hi[n][j]);
        lo_most = max(lo_most, lo[n][j]);
        hi_least = min(hi_least, hi[n][j]);
      }
#pragma unroll
      for (int i = 0; i < kVWords * 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.0f;
    }
    lo_most = __reduce_max_sync(kFullMask, lo_most);
    hi_least = __reduce_min_sync(kFullMask, hi_least);

    // ---- tokens: each warp its own 16 of every tile
    const int row_a = stage_row<DIM>(g);                                        // key rows row_a, row_a + 8
    const int row_b = stage_row<DIM>(2 * t), row_c = stage_row<DIM>(2 * t + 1);  // value rows, and those + 8
    const int seg_hi = seg.s.hi;
    for (int i = 0; i < groups; ++i) {
      const int stage = used % kRing, base = base0 + i * kRowsTile;
      if (!__all_sync(kFullMask, mbar_wait(&sh.full[warp][stage], used / kRing & 1, &sh.abort, kSiteProducer,
                                           p.status))) {
        failed = true;
        break;
      }
      ++used;
      const bool here = sh.block[warp][stage] >= 0;
      const float ks = next_ks, vs = next_vs;
      uint4 kw[kChunks][2];
      if (here) {
        const uint32_t k_at = smem_u32(sh.ring[warp][stage][0]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t at = k_at + stage_byte<DIM>(row_a, (t + 4 * c) * 16);
          kw[c][0] = lds_v4(at);
          kw[c][1] = lds_v4(at + 8 * DIM);
        }
      }
      if (i + 1 < groups) fetch_scales();
      const auto refill = [&] {  // the stage has been read
        __syncwarp();
        if (i + kRing < groups) {
          issue(i + kRing, next_block);
          next_block = block_at(seg, i + kRing + 1);
        }
      };
      if (!here) {
        refill();
        continue;
      }
      bool quiet;
      const float lv = value_exponent(vs, largest, quiet);

      // scores of tokens row_a and row_a + 8 (rows) for query rows 2t and
      // 2t + 1, in a chain of products for each piece of the key row
      float sc[NT][4], part[kChunks][NT][4];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[c][n][j] = 0.0f;
        const uint32_t w0[4] = {kw[c][0].x, kw[c][0].y, kw[c][0].z, kw[c][0].w};
        const uint32_t w1[4] = {kw[c][1].x, kw[c][1].y, kw[c][1].z, kw[c][1].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a[4];
          to_operand<CODE, true>(w0[k], a[0], a[2]);
          to_operand<CODE, true>(w1[k], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(part[c][n], a, qf[n][c][2 * k], qf[n][c][2 * k + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[n][j] = kChunks == 1 ? part[0][n][j] : part[0][n][j] + part[kChunks - 1][n][j];
      const bool whole = lo_most <= base && base + 16 <= hi_least;
      // t of the group's tokens, their weights against the references of
      // earlier groups, and whether those have to be raised: a row has none
      // yet, or a weight is above what fp16 should hold, or the block is quiet
      bool raise = quiet;
      float weight[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int col = 0; col < 2; ++col) {
          const float a = qa[n][col] * ks, d = fmaf(qb[n][col], ks, lv);
          float x = fmaf(sc[n][col], a, d), y = fmaf(sc[n][col + 2], a, d);
          if (!whole) {
            const int token = base + row_a;
            x = token >= lo[n][col] && token < hi[n][col] ? x : -INFINITY;
            y = token + 8 >= lo[n][col] && token + 8 < hi[n][col] ? y : -INFINITY;
          }
          sc[n][col] = x;
          sc[n][col + 2] = y;
          const float ref = m[n][col] == -INFINITY ? 0.0f : m[n][col];
          weight[n][col] = exp2_approx(x - ref);
          weight[n][col + 2] = exp2_approx(y - ref);
          raise |= fmaxf(weight[n][col], weight[n][col + 2]) > kMostWeight;
          raise |= m[n][col] == -INFINITY && fmaxf(x, y) > -INFINITY;
        }
      if (__any_sync(kFullMask, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int col = 0; col < 2; ++col) {
            float top = fmaxf(sc[n][col], sc[n][col + 2]);
#pragma unroll
            for (int s = 4; s < kWarp; s *= 2) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, s));
            const float next = fmaxf(m[n][col], top - kReferenceLog2), next_u = fmaxf(mu[n][col], top - lv);
            const float ref = next == -INFINITY ? 0.0f : next, alpha = weight_of(m[n][col], next);
            l[n][col] *= weight_of(mu[n][col], next_u);
            m[n][col] = next;
            mu[n][col] = next_u;
            weight[n][col] = exp2_approx(sc[n][col] - ref);
            weight[n][col + 2] = exp2_approx(sc[n][col + 2] - ref);
#pragma unroll
            for (int v = 0; v < kVWords * 2; ++v) {
              o[n][v][col] *= alpha;
              o[n][v][col + 2] *= alpha;
            }
          }
      }
      uint32_t pf[NT][2];
      // a row that sees a block with a NaN scale has NaN weights; one that does not has zeros, and must not meet it
      const float lw = lv != lv ? 0.0f : lv;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int col = 0; col < 2; ++col) {
          const float ref = m[n][col] == -INFINITY ? 0.0f : m[n][col];
          const float ref_u = mu[n][col] == -INFINITY ? 0.0f : mu[n][col];
          if (quiet) {
            l[n][col] += exp2_approx(sc[n][col] - lv - ref_u) + exp2_approx(sc[n][col + 2] - lv - ref_u);
          } else {
            l[n][col] = fmaf(weight[n][col] + weight[n][col + 2], exp2_approx(ref - lw - ref_u), l[n][col]);
          }
        }
        pf[n][0] = transpose_8x8(pack_half2(weight[n][0], weight[n][1]));
        pf[n][1] = transpose_8x8(pack_half2(weight[n][2], weight[n][3]));
      }
      uint32_t vw[4][kVWords];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = x & 1 ? row_c : row_b;
        const uint32_t at =
            smem_u32(sh.ring[warp][stage][1]) + stage_byte<DIM>(row, g * (DIM / 8)) + (x >> 1) * 8 * DIM;
        if constexpr (kVWords == 4) {
          const uint4 w = lds_v4(at);
          vw[x][0] = w.x, vw[x][1] = w.y, vw[x][2] = w.z, vw[x][3] = w.w;
        } else {
          lds_v2(at, vw[x][0], vw[x][1]);
        }
      }
      if (base + 16 > seg_hi) {  // what lies behind the last token may be no number, and meets weights of zero
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (base + (x & 1 ? row_c : row_b) + 8 * (x >> 1) >= seg_hi)
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vw[x][w] = 0;
      }
      refill();
      // channels 2x and 2x + 1 of this lane's chunk are output rows g and g + 8
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        const uint32_t l01 = __byte_perm(vw[0][w], vw[1][w], 0x5140), l23 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
        const uint32_t h01 = __byte_perm(vw[2][w], vw[3][w], 0x5140), h23 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
        uint32_t a[4];
        to_operand<CODE, false>(l01, a[0], a[1]);
        to_operand<CODE, false>(h01, a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w], a, pf[n][0], pf[n][1]);
        to_operand<CODE, false>(l23, a[0], a[1]);
        to_operand<CODE, false>(h23, a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * w + 1], a, pf[n][0], pf[n][1]);
      }
    }

    // ---- join the warps, with the next segment's first loads on their way
    __syncthreads();
    if (more) start(sh.seg[which ^ 1]);
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
        for (int x = 0; x < kVWords; ++x)
          *reinterpret_cast<float4*>(&sh.sums[warp][r][sum_place<DIM>(r, g * (DIM / 8) + 4 * x)]) =
              make_float4(o[n][2 * x][col] * weight, o[n][2 * x][col + 2] * weight, o[n][2 * x + 1][col] * weight,
                          o[n][2 * x + 1][col + 2] * weight);
      }
    __syncthreads();

    // CTAs that share the item: the one it begins in and those that follow
    const int64_t item_begin = seg.at - seg.unit0, item_end = item_begin + kItemTiles + seg.tiles;
    const int owner = static_cast<int>(quotient((item_begin + 1) * parts + total - 1, total) - 1);
    const int sharers =
        seg.units == kItemTiles + seg.tiles
            ? 1
            : static_cast<int>(quotient(item_end * parts + total - 1, total) - 1) - owner + 1;
    constexpr int kSlot = kRows * (DIM + 3);
    float* slot = p.partial + (static_cast<int64_t>(cta) * 2 + (item_begin >= begin ? 1 : 0)) * kSlot;
    const auto store = [&](int r, int d, float4 v, float top, float top_u, float sum) {
      if (r >= rows) return;
      const float inv = sum == 0.0f ? 0.0f : exp2_approx(top - top_u) / sum;
      const int64_t row = output_row(p, seg.s, seg.head, r);
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
        const float4 x = *reinterpret_cast<const float4*>(&sh.sums[w][r][sum_place<DIM>(r, d)]);
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
    if (!more) break;
    __syncthreads();
  }
  // after a wait that gave up, loads may still be in flight
  for (; used != issued; ++used) {
    volatile int never = 0;
    mbar_wait(&sh.full[warp][used % kRing], used / kRing & 1, &never, kSiteProducer, p.status);
  }
}

// [pages * kv_heads][page][DIM] codes, in boxes of 16 tokens.
template <int DIM>
bool encode_codes(CUtensorMap* map, const void* codes, int64_t blocks, int page) {
  const auto encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {DIM, static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(blocks)};
  const cuuint64_t strides[2] = {DIM, static_cast<cuuint64_t>(page) * DIM};
  const cuuint32_t box[3] = {DIM, 16, 1}, step[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, DIM == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DIM, int CODE, int NT>
cudaError_t run_rows(const AttendParams& p, int grid, cudaStream_t stream) {
  constexpr int kBytes = sizeof(RowsShared<DIM, NT>) + 1024;
  static bool ready[64] = {};
  const cudaError_t e = allow_shared(reinterpret_cast<const void*>(kv_rows_kernel<DIM, CODE, NT>), kBytes, ready);
  if (e != cudaSuccess) return e;
  CUtensorMap k_map{}, v_map{};
  const int64_t blocks = p.pages * p.kv_heads;
  if (blocks > 0 && !(encode_codes<DIM>(&k_map, p.k_codes, blocks, 1 << p.page_shift) &&
                      encode_codes<DIM>(&v_map, p.v_codes, blocks, 1 << p.page_shift)))
    return cudaErrorInvalidValue;
  kv_rows_kernel<DIM, CODE, NT><<<grid, kRowsThreads, kBytes, stream>>>(p, k_map, v_map);
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

// Most query rows of a (sequence, kv head) that kv_rows_kernel takes: what
// one of its passes over the cache serves.  Measured with this kernel and with
// the tiles, 8 kv heads of 128 over 32768 tokens and 16 sequences of 4096:
// 16 rows 72 and 78 us against 73 and 99, 24 rows 82 and 117 against 73 and 99,
// 32 rows 84 and 119 against 69 and 96.
constexpr int64_t kRowsMost = 16;

// How a call is launched: on tensor-core tiles, or with `nt` times 8 columns
// on `grid` CTAs.
struct Plan {
  bool tiles;
  int nt, grid;
  size_t workspace;
};

Plan make_plan(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads, int64_t kv_heads, int64_t dim,
               int64_t width, int64_t page, int64_t window) {
  Plan plan{};
  const int64_t group = q_heads / kv_heads;
  if (max_new > tokens) max_new = tokens;
  plan.tiles = max_new * group > kRowsMost;
  if (plan.tiles) {
    plan.workspace = kRowsMaxGrid * sizeof(int) + tiles_workspace_bytes(tokens, batch, group, kv_heads,
                                                                        static_cast<int>(dim), width,
                                                                        static_cast<int>(page), window);
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

// A window of 2^31 tokens reaches over any sequence.
int64_t held_window(int64_t window) { return window < (int64_t(1) << 31) ? window : int64_t(1) << 31; }

bool shapes_ok(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads, int64_t kv_heads, int64_t dim,
               int64_t width, int64_t page) {
  if (tokens < 0 || tokens > INT32_MAX / 2 || batch < 0 || batch > (1 << 20) || max_new < 0) return false;
  if (kv_heads < 1 || kv_heads > 65536 || q_heads < kv_heads || q_heads > 65536 || q_heads % kv_heads) return false;
  if ((dim != 64 && dim != 128) || (page != 16 && page != 32 && page != 64 && page != 128)) return false;
  // rows of q and tokens of a table are counted in 32 bits
  return tokens * q_heads <= INT32_MAX / 2 && width >= 0 && width <= INT32_MAX / 2 / page;
}

}  // namespace
}  // namespace b2

extern "C" {

size_t b2_kv_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_new, int64_t q_heads,
                                       int64_t kv_heads, int64_t dim, int64_t width, int64_t page, int64_t window) {
  if (!b2::shapes_ok(tokens, batch, max_new, q_heads, kv_heads, dim, width, page) || window < 0 || tokens == 0 ||
      batch == 0)
    return 0;
  return b2::make_plan(tokens, batch, max_new, q_heads, kv_heads, dim, width, page, b2::held_window(window)).workspace;
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
  if (pages < 0 || pages * kv_heads > INT32_MAX || window < 0 || !(scale > 0.0f) || scale > 3.0e38f) return invalid;
  if (tokens == 0) return 0;
  if (batch < 1 || max_new < 1 || (offsets == nullptr && (tokens % batch || tokens / batch > max_new))) return invalid;
  if (!q || !lengths || (!table && width) || !out) return invalid;
  if (pages && (!k_codes || !v_codes || !k_scale || !v_scale)) return invalid;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_codes, 16) || !aligned(v_codes, 16)) return invalid;
  if (q_token_stride < 0 || q_head_stride < 0 || q_token_stride % 8 || q_head_stride % 8) return invalid;
  window = b2::held_window(window);
  const b2::Plan plan = b2::make_plan(tokens, batch, max_new, q_heads, kv_heads, dim, width, page, window);
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
  p.status = b2::status_word_ptr();
  p.counters = static_cast<int*>(workspace);
  p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + b2::kRowsMaxGrid * sizeof(int));
  if (plan.tiles)
    return static_cast<int>(
        b2::run_tiles(p, static_cast<int>(dim), code, p.partial, static_cast<cudaStream_t>(stream)));
  return static_cast<int>(
      b2::run_rows_any(p, static_cast<int>(dim), code, plan.nt, plan.grid, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
