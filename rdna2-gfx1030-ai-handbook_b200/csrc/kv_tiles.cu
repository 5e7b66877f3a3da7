// Attention over the paged 8-bit cache for calls with many query rows, on
// tcgen05 (the arithmetic is stated in kv_attention.cu).
//
// A CTA takes 256 rows of one sequence and kv head -- its tokens times the
// head's query heads -- as two row tiles of 128, and walks the cached tokens
// they see in tiles of 128.  Roles:
//
//   warps 0-7, 8-15 softmax of row tile 0 and 1, two threads a row with 64
//                   tokens each: scores come from tensor memory, weights go
//                   back there as fp16 over the scores' own columns
//   warps 16-23     codes -> fp16 operands in shared memory (128-byte swizzle),
//                   two tiles of K and V each; every operand serves both row
//                   tiles, so a code is converted once for 256 rows
//   warps 24, 25    issue the products of row tile 0 and 1: S_t = Q_t K^T (both
//                   operands in shared memory) and O_t += P_t V (P_t in tensor
//                   memory, V as stored: its channels are contiguous)
//   warp 26         the scales of the next tiles' blocks
//   warp 27         nothing: registers are shared out by groups of four warps
//
// A block of 128 rows or fewer uses row tile 0 alone.
//
// Measured: an 8192-token causal prompt, 32 query and 8 kv heads of 128, int8:
// 696 us, 790 TFLOP/s.  A pair of row tiles x 128 tokens takes about 5500
// cycles, starts, ends and raised references included, 2048 of them of the
// tensor pipe and as many of the exponential unit: the chain scores, weights,
// sums, next scores of a row tile bounds it.
//
// The two row tiles alternate on the tensor cores: while one is in its
// softmax the other multiplies, and they take turns so that it stays that way
// (left alone they fall into step, exponentials and products in turn for
// both).  A softmax is one pass and looks for no
// maximum: weights are taken relative to that of the row's first tile, which
// fp16 allows while they stay below kMostWeight.  Where a tile's weights sum
// to more, and where a row has no reference yet, the tile's maxima are found,
// O_t is rescaled in tensor memory and the tile is gone through once more.
#include "../../include/b2_attention.h"
#include "b2_internal.h"
#include "kv_attention.cuh"

namespace b2 {
namespace {

constexpr int kTileRows = 128;              // rows of one product (UMMA M)
constexpr int kCtaRows = 2 * kTileRows;
constexpr int kTileTokens = 128;
constexpr int kGroups = kTileTokens / 16;   // a group of 16 tokens is in one block, whatever the page
constexpr int kSoftmaxWarps = 16, kConvertWarps = 8;
constexpr int kMmaWarp = kSoftmaxWarps + kConvertWarps, kInfoWarp = kMmaWarp + 2;
constexpr int kTilesThreads = 28 * kWarp;
// Registers a thread: 72 at launch, 4 * 80 + 2 * 64 + 56 = 7 * 72 afterwards.
constexpr int kSoftmaxRegs = 80, kConvertRegs = 64, kOtherRegs = 56;
constexpr int kHalfTokens = kTileTokens / 2;  // of a softmax thread
constexpr uint32_t kMinusInf = 0xff800000u;
constexpr float kMostOffset = 2.59614843e33f;  // 2^111: a row's bias is below 2^17

// One row tile of queries, or one tile of K or V: panels of 64 channels, 128
// rows of 128 bytes each, 128-byte swizzle.
constexpr int kPanel = 128 * 128;

constexpr uint32_t kQuiet = 1u << kGroups;
constexpr int kOddBit = 2 * kGroups;

struct __align__(16) GroupInfo {
  float ks, lv, iv, unused;  // key scale, log2 of the value scale, 2^(top_lv - lv)
};

// Tensor memory, 512 columns: scores of the row tiles at 0 and 128, sums at
// 256, DIM columns each.  Heads of 64 leave 128 columns, so that the weights
// have a place of their own and the next scores are on their way while they
// are multiplied; with heads of 128 the weights overlay the scores.
template <int DIM>
constexpr bool kApart = DIM == 64;

template <int DIM>
struct TilesShared {
  static constexpr int kTile = DIM / 64 * kPanel;
  static constexpr int kOffQ = 0;                     // 2 row tiles
  static constexpr int kOffK = kOffQ + 2 * kTile;     // 2 stages
  static constexpr int kOffV = kOffK + 2 * kTile;     // 2 stages
  static constexpr int kOffCtl = kOffV + 2 * kTile;
};

// A row block and the token tiles that any of its rows sees.
struct Block {
  Sequence s;
  int b;
  int row0, rows;       // its first row, and the rows of the sequence
  int tile0, tiles;
};

// What a CTA works on.  It is kept in shared memory: a softmax thread has no
// registers to spare, and spilled ones would be fetched past the codes that
// stream through the first-level cache.
struct Work {
  Block blk;
  int slot, head, split, parts;
};

struct TilesControl {
  uint64_t q_full[2], k_full[2], k_free[2], v_full[2], v_free[2];
  uint64_t s_full[2], s_read[2], p_full[2], o_done[2], info_full[4], turn[2], last[2];
  GroupInfo info[4][kGroups];
  float top_lv[4];
  // Bit g: group g lies on a page of the cache and has scales that are numbers.
  // Bit kOddBit + g: it has scales that are not.  It is masked then, so that
  // they meet no row that does not see it, and the sum of the weights of the
  // rows that do is NaN.  kQuiet, for each half of the tokens: the tile has a
  // quiet block, its weights are summed apart, and iv is 0 and top_lv infinite.
  uint32_t present[4];
  Work work;
  // what the two threads of a row tell each other: maxima, and the sum of q
  float row[2][2][kCtaRows], sum[2][kCtaRows];
  // a softmax thread's own: what it needs once a tile
  int lo[kSoftmaxWarps * kWarp], hi[kSoftmaxWarps * kWarp];
  float n[kSoftmaxWarps * kWarp], l[kSoftmaxWarps * kWarp], bias[kSoftmaxWarps * kWarp];
  uint32_t tmem;
  int abort, drained;
};

template <int DIM>
constexpr int kTilesBytes = TilesShared<DIM>::kOffCtl + static_cast<int>(sizeof(TilesControl)) + 1024;

struct TilesParams {
  AttendParams a;
  int slots;      // row blocks of all sequences, at most
  int splits;     // parts of the cached tokens that a row block is split into
  float* partial; // [slots][heads][splits][256][DIM] sums, then [..][3][256] m, n, l
  int* status;
};

// m, n and l of the parts, behind their sums.
template <int DIM>
__device__ __forceinline__ float* part_stats(const TilesParams& p) {
  return p.partial + static_cast<int64_t>(p.slots) * p.a.kv_heads * p.splits * kCtaRows * DIM;
}

// Slot s of the call is a row block of the sequence with first_block(b) <= s.
__device__ __forceinline__ int first_block(const AttendParams& p, int b) {
  return p.tok.begin(b) * p.group / kCtaRows + b;
}

__device__ __forceinline__ bool load_block(const AttendParams& p, int slot, Block& k) {
  k.b = warp_search(p.tok.batch, slot, [&](int i) { return first_block(p, i); });
  k.s = load_sequence(p, k.b);
  k.rows = k.s.count * p.group;
  k.row0 = (slot - first_block(p, k.b)) * kCtaRows;
  if (k.row0 < 0 || k.row0 >= k.rows) return false;  // below 0: offsets that decrease
  int lo, hi, unused;
  const int last = min(k.row0 + kCtaRows, k.rows) - 1;
  row_bounds(p, k.s, k.s.start + k.row0 / p.group, lo, unused);
  row_bounds(p, k.s, k.s.start + last / p.group, unused, hi);
  k.tile0 = lo / kTileTokens;
  k.tiles = max(0, (hi + kTileTokens - 1) / kTileTokens - k.tile0);
  return true;
}

// Parts that a block's tiles are split into, and the tiles of one part.
__device__ __forceinline__ int part_tiles(const TilesParams& p, int tiles) { return (tiles + p.splits - 1) / p.splits; }
__device__ __forceinline__ int part_count(const TilesParams& p, int tiles) {
  const int per = part_tiles(p, tiles);
  return per ? (tiles + per - 1) / per : 1;
}

__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Descriptor of V as the K x N operand with N (channels) contiguous: panels
// of 64 channels kPanel apart, groups of 8 tokens 1024 bytes apart.
__device__ __forceinline__ uint64_t channels_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kPanel >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// 32 columns of this thread's row, complete: loading and waiting in one
// statement leaves the registers where the load put them.
__device__ __forceinline__ void tmem_read32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Bits [lo, hi) of a word.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (lo >= hi) return 0u;
  return (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
}

// SEG: tokens of a thread that are taken to lie in one block, which pages of
// SEG and more grant.
template <int DIM, int CODE, int SEG>
__global__ void __launch_bounds__(kTilesThreads, 1) kv_tiles_kernel(TilesParams tp) {
  using Shared = TilesShared<DIM>;
  constexpr int kPanels = DIM / 64;
  const AttendParams& p = tp.a;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  TilesControl& ctl = *reinterpret_cast<TilesControl*>(smem + Shared::kOffCtl);
  const uint32_t base_u32 = smem_u32(smem);
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

  const int unit = blockIdx.x, item = unit / tp.splits, from_last = item / p.kv_heads;
  Work mine;
  mine.split = unit - item * tp.splits;
  mine.head = item - from_last * p.kv_heads;
  mine.slot = tp.slots - 1 - from_last;  // the heaviest blocks of a causal prompt, its last rows, come first
  if (!load_block(p, mine.slot, mine.blk)) return;
  mine.parts = part_count(tp, mine.blk.tiles);
  if (mine.split >= mine.parts) return;
  const int per = part_tiles(tp, mine.blk.tiles), first = mine.split * per;
  const int count = min(per, mine.blk.tiles - first);
  const int token0 = (mine.blk.tile0 + first) * kTileTokens;
  const int used = mine.blk.rows - mine.blk.row0 > kTileRows ? 2 : 1;  // row tiles that hold rows
  if (threadIdx.x == 0) ctl.work = mine;
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(&ctl.q_full[i], kSoftmaxWarps / 2);
        mbar_init(&ctl.k_full[i], kConvertWarps);
        mbar_init(&ctl.v_full[i], kConvertWarps);
        mbar_init(&ctl.k_free[i], used);
        mbar_init(&ctl.v_free[i], used);
        mbar_init(&ctl.s_full[i], 1);
        mbar_init(&ctl.s_read[i], kSoftmaxWarps / 2);
        mbar_init(&ctl.p_full[i], kSoftmaxWarps / 2);
        mbar_init(&ctl.o_done[i], 1);
        mbar_init(&ctl.turn[i], kSoftmaxWarps / 2);
        mbar_init(&ctl.last[i], 1);
      }
      for (int i = 0; i < 4; ++i) mbar_init(&ctl.info_full[i], 1);
      ctl.abort = ctl.drained = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(&ctl.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const Work& work = ctl.work;
  const Block& blk = work.blk;
  const uint32_t tmem = ctl.tmem;
  volatile int* abort_flag = &ctl.abort;
  // called by a whole warp, which leaves with one answer
  const auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
    return __all_sync(kFullMask, mbar_wait(bar, parity, abort_flag, site, tp.status));
  };

  // The block of the cache that holds `token` for this head, or -1.
  const auto block_of = [&](int token) -> int64_t {
    if (token >= blk.s.hi) return -1;
    const int64_t page = __ldg(p.table + static_cast<int64_t>(blk.b) * p.width + (token >> p.page_shift));
    return page >= 0 && page < p.pages ? page * p.kv_heads + work.head : -1;
  };
  if (warp >= kMmaWarp) fewer_registers<kOtherRegs>();
  if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ------------------------------------------------------- products
    constexpr uint32_t kIdescS = make_idesc<kKindF16>(kTileRows, kTileTokens);
    constexpr uint32_t kIdescO = make_idesc<kKindF16>(kTileRows, DIM) | (1u << 16);  // V: N contiguous
    const int t = warp - kMmaWarp;
    const uint32_t weights = tmem + (kApart<DIM> ? 384 + t * 64 : t * 128);
    const auto scores = [&](int stage) {
      if (elect_one()) {
        const uint32_t q = base_u32 + Shared::kOffQ + t * Shared::kTile;
        const uint32_t k = base_u32 + Shared::kOffK + stage * Shared::kTile;
#pragma unroll
        for (int x = 0; x < DIM / 16; ++x) {
          const uint32_t off = x / 4 * kPanel + x % 4 * 32;
          umma<kKindF16>(tmem + t * 128, sw128_desc(q + off), sw128_desc(k + off), kIdescS, x > 0);
        }
        umma_commit(&ctl.s_full[t]);
        umma_commit(&ctl.k_free[stage]);
      }
      __syncwarp();
    };
    const auto output = [&](int stage, bool add) {
      if (elect_one()) {
        const uint32_t v = base_u32 + Shared::kOffV + stage * Shared::kTile;
#pragma unroll
        for (int x = 0; x < kTileTokens / 16; ++x)
          umma_ts_f16(tmem + 256 + t * DIM, weights + 8 * x, channels_desc(v + x * 2048), kIdescO, add || x > 0);
        umma_commit(&ctl.o_done[t]);
        umma_commit(&ctl.v_free[stage]);
      }
      __syncwarp();
    };
    // The scores of a tile wait for its blocks' scales too, although only the
    // softmax reads those: the warp that brings them goes by the parity of
    // k_free, and would miss a phase if a second one could complete meanwhile.
    const int todo = t < used ? count : 0;
    bool ok = todo == 0 || (wait(&ctl.q_full[t], 0, kSiteMma) && wait(&ctl.k_full[0], 0, kSiteMma) &&
                            wait(&ctl.info_full[0], 0, kSiteMma));
    if (ok && todo > 0) {
      tc_fence_after();
      scores(0);
    }
    for (int i = 0; ok && i < todo; ++i) {
      const auto next_scores = [&](uint64_t* before) {
        ok = wait(&ctl.k_full[(i + 1) & 1], ((i + 1) >> 1) & 1, kSiteMma) &&
             wait(&ctl.info_full[(i + 1) & 3], ((i + 1) >> 2) & 1, kSiteMma) && wait(before, i & 1, kSiteMma);
        if (!ok) return;
        tc_fence_after();
        scores((i + 1) & 1);
      };
      if (kApart<DIM> && i + 1 < todo) next_scores(&ctl.s_read[t]);
      ok = ok && wait(&ctl.v_full[i & 1], (i >> 1) & 1, kSiteMma) && wait(&ctl.p_full[t], i & 1, kSiteMma);
      if (!ok) break;
      tc_fence_after();
      output(i & 1, i > 0);
      // the weights lie where the next scores go: they have been read first
      if (!kApart<DIM> && i + 1 < todo) next_scores(&ctl.o_done[t]);
    }
    // nothing is in flight when tensor memory is given back, after a wait
    // that gave up either
    if (elect_one()) umma_commit(&ctl.last[t]);
    __syncwarp();
    mbar_wait(&ctl.last[t], 0, &ctl.drained, kSiteMma, tp.status);
    __syncwarp();
  } else if (warp == kInfoWarp) {
    // ------------------------------------------------------- blocks' scales
    // A lane a group of 16 tokens.  The ring's place for tile i was last read
    // by the softmax of tile i - 4, whose end the scores of tile i - 2 need:
    // they have been formed when k_free completes its phase, and the next phase
    // needs the scores of tile i, which wait for what is written here.
    int64_t block = lane < kGroups ? block_of(token0 + 16 * lane) : -1;
    float ks = 0.0f, vs = 0.0f, largest = -INFINITY;
    const auto load = [&] {
      ks = block < 0 ? 0.0f : __ldg(p.k_scale + block);
      vs = block < 0 ? 0.0f : __ldg(p.v_scale + block);
    };
    load();
    for (int i = 0; i < count; ++i) {
      const bool odd = block >= 0 && !(fabsf(ks) < INFINITY && fabsf(vs) < INFINITY), here = block >= 0 && !odd;
      const float lv = here ? __log2f(value_scale(vs)) : -INFINITY;
      float top = lv;
#pragma unroll
      for (int d = 1; d < kGroups; d *= 2) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
      top = __shfl_sync(kFullMask, top, 0);
      largest = fmaxf(largest, top);
      const bool quiet = __any_sync(kFullMask, here && lv < largest - kQuietLog2);
      const unsigned present = __ballot_sync(kFullMask, here) | (quiet ? kQuiet | kQuiet << kGroups / 2 : 0u) |
                               __ballot_sync(kFullMask, odd) << kOddBit;
      const GroupInfo info = {here ? ks : 0.0f, lv, here && !quiet ? exp2_approx(top - lv) : 0.0f, 0.0f};
      block = lane < kGroups && i + 1 < count ? block_of(token0 + (i + 1) * kTileTokens + 16 * lane) : -1;
      load();
      if (i >= 2 && !wait(&ctl.k_free[i & 1], ((i >> 1) & 1) ^ 1, kSiteTransform)) break;
      if (lane < kGroups) ctl.info[i & 3][lane] = info;
      if (lane == 0) {
        ctl.top_lv[i & 3] = quiet ? INFINITY : top == -INFINITY ? 0.0f : top;
        ctl.present[i & 3] = present;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.info_full[i & 3]);
    }
  } else if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // ------------------------------------------------------- codes to fp16
    // Each operand's codes are loaded as soon as the one before it has left
    // the registers, and the pages of a tile a tile ahead of that.
    fewer_registers<kConvertRegs>();
    constexpr int kRowsEach = 2;
    constexpr int kLoads = kRowsEach * kPanels;  // 16-byte pieces of a tile a thread takes
    const int tid = threadIdx.x - kSoftmaxWarps * kWarp;
    const int chunk = tid % 4;                   // quarter-warps take two rows: no bank conflicts below
    const int page_mask = (1 << p.page_shift) - 1;
    int64_t block[kRowsEach];                    // of this thread's rows in the next tile
    const auto locate = [&](int i) {
#pragma unroll
      for (int j = 0; j < kRowsEach; ++j)
        block[j] = i < count ? block_of(token0 + i * kTileTokens + tid / 4 + 64 * j) : -1;
    };
    // where the rows begin in the codes, or -1
    const auto place = [&](int64_t (&at)[kRowsEach]) {
#pragma unroll
      for (int j = 0; j < kRowsEach; ++j)
        at[j] = block[j] < 0 ? -1 : ((block[j] << p.page_shift) + ((tid / 4 + 64 * j) & page_mask)) * DIM + chunk * 16;
    };
    const auto load = [&](const uint8_t* codes, const int64_t (&at)[kRowsEach], uint4 (&w)[kLoads]) {
#pragma unroll
      for (int j = 0; j < kRowsEach; ++j)
#pragma unroll
        for (int x = 0; x < kPanels; ++x)
          w[j * kPanels + x] = at[j] < 0 ? make_uint4(0, 0, 0, 0) : ldg_v4(codes + at[j] + x * 64);
    };
    const auto store = [&](bool keys, uint8_t* dst, const uint4 (&w)[kLoads]) {
#pragma unroll
      for (int j = 0; j < kRowsEach; ++j)
#pragma unroll
        for (int x = 0; x < kPanels; ++x) {
          const uint4 c = w[j * kPanels + x];
          uint4 a, b;
          if (keys) {
            to_operand<CODE, true>(c.x, a.x, a.y);
            to_operand<CODE, true>(c.y, a.z, a.w);
            to_operand<CODE, true>(c.z, b.x, b.y);
            to_operand<CODE, true>(c.w, b.z, b.w);
          } else {
            to_operand<CODE, false>(c.x, a.x, a.y);
            to_operand<CODE, false>(c.y, a.z, a.w);
            to_operand<CODE, false>(c.z, b.x, b.y);
            to_operand<CODE, false>(c.w, b.z, b.w);
          }
          const int rr = tid / 4 + 64 * j;
          *reinterpret_cast<uint4*>(dst + x * kPanel + swizzled(rr, 2 * chunk)) = a;
          *reinterpret_cast<uint4*>(dst + x * kPanel + swizzled(rr, 2 * chunk + 1)) = b;
        }
    };
    const auto done = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    uint4 kw[kLoads], vw[kLoads];
    int64_t at[kRowsEach];
    locate(0);
    place(at);
    load(p.k_codes, at, kw);
    load(p.v_codes, at, vw);
    locate(1);
    for (int i = 0; i < count; ++i) {
      const int stage = i & 1;
      const uint32_t parity = ((i >> 1) & 1) ^ 1;
      place(at);  // of tile i + 1
      locate(i + 2);
      if (i >= 2 && !wait(&ctl.k_free[stage], parity, kSiteTransform)) break;
      store(true, smem + Shared::kOffK + stage * Shared::kTile, kw);
      done(&ctl.k_full[stage]);
      load(p.k_codes, at, kw);
      if (i >= 2 && !wait(&ctl.v_free[stage], parity, kSiteTransform)) break;
      store(false, smem + Shared::kOffV + stage * Shared::kTile, vw);
      done(&ctl.v_full[stage]);
      load(p.v_codes, at, vw);
    }
  } else if (warp < 8 * used) {
    // ------------------------------------------------------- softmax
    more_registers<kSoftmaxRegs>();
    const int tile = warp / 8, half = warp / 4 % 2, row = threadIdx.x % kTileRows;
    const int cta_row = tile * kTileRows + row, other = half ^ 1;
    const int pair = 1 + tile * 4 + warp % 4;  // named barrier of the two warps that share rows
    // a thread brings half of its row's channels
    float qs;
    {
      constexpr int kChunks = DIM / 16;  // 16-byte pieces of half a row
      const int r = blk.row0 + cta_row;
      const bool valid = r < blk.rows;
      const uint16_t* src = static_cast<const uint16_t*>(p.q) +
                            static_cast<int64_t>(blk.s.first + r / p.group) * p.q_token +
                            (work.head * p.group + r % p.group) * p.q_head + half * (DIM / 2);
      uint4 v[kChunks];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) v[c] = valid ? ldg_v4(src + 8 * c) : make_uint4(0, 0, 0, 0);
      const auto unpack = [&](int c, float (&f)[8]) {
        if (p.q_bf16) {
          Vec<__nv_bfloat16>::unpack(v[c], f);
        } else {
          Vec<__half>::unpack(v[c], f);
        }
      };
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float f[8];
        unpack(c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
      }
      ctl.row[0][half][cta_row] = __uint_as_float(top);
      named_bar_sync(pair, 2 * kWarp);
      float factor, gain, sum = 0.0f;
      row_power(max(top, __float_as_uint(ctl.row[0][other][cta_row])), factor, gain);
      qs = gain * p.scale_log2;
      uint8_t* dst = smem + Shared::kOffQ + tile * Shared::kTile;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        float f[8];
        unpack(c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= factor;
        const uint4 h = Vec<__half>::pack(f);
        if (CODE == kCodeInt8) {
          Vec<__half>::unpack(h, f);
          sum += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        }
        const int chunk = half * kChunks + c;
        *reinterpret_cast<uint4*>(dst + chunk / 8 * kPanel + swizzled(row, chunk % 8)) = h;
      }
      ctl.sum[half][cta_row] = sum;
      fence_proxy_async_smem();
      named_bar_sync(pair, 2 * kWarp);
      if (lane == 0) mbar_arrive(&ctl.q_full[tile]);
    }
    const uint32_t lanes = static_cast<uint32_t>(warp % 4 * 32) << 16;
    const uint32_t s_col = tmem + lanes + tile * 128 + half * kHalfTokens;         // this thread's scores,
    const uint32_t p_col = tmem + lanes + (kApart<DIM> ? 384 + tile * 64 : tile * 128) + half * (kHalfTokens / 2);
    const uint32_t o_col = tmem + lanes + 256 + tile * DIM + half * (DIM / 2);     // weights and channels
    const int me = threadIdx.x;
    // references of t and u; a row that is not one of the sequence needs none
    float m = 0.0f;
    {
      int lo = 0, hi = 0;
      if (blk.row0 + cta_row < blk.rows) {
        row_bounds(p, blk.s, blk.s.start + (blk.row0 + cta_row) / p.group, lo, hi);
        m = -INFINITY;
      }
      ctl.lo[me] = lo;
      ctl.hi[me] = hi;
      ctl.n[me] = m;
      ctl.l[me] = 0.0f;
      // what int8 keys without their sign add to a row's products; those are no
      // numbers where this is none, and masked ones must not become so
      const float sum = ctl.sum[0][cta_row] + ctl.sum[1][cta_row];
      ctl.bias[me] = CODE == kCodeInt8 && fabsf(sum) < INFINITY ? -128.0f * sum : 0.0f;
    }
    bool ok = true;
    for (int i = 0; i < count; ++i) {
      // After a wait that gave up the loop goes on without waiting: the two
      // warps of a row meet at the same barriers whatever either has seen.
      ok = ok && wait(&ctl.info_full[i & 3], (i >> 2) & 1, kSiteEpilogue);
      const GroupInfo* info = ctl.info[i & 3] + half * (kHalfTokens / 16);
      const uint32_t present = ctl.present[i & 3] >> (half * (kHalfTokens / 16));
      const int base = token0 + i * kTileTokens + half * kHalfTokens;
      // every row of this warp sees every one of its tokens
      const bool whole = __all_sync(kFullMask, ctl.lo[me] <= base && base + kHalfTokens <= ctl.hi[me]) &&
                         (present & 0xfu) == 0xfu;
      if (!whole && present >> kOddBit & 0xfu) {
#pragma unroll 1
        for (int g = 0; g < kHalfTokens / 16; ++g)
          if (present >> (kOddBit + g) & 1 && max(ctl.lo[me], base + 16 * g) < min(ctl.hi[me], base + 16 * g + 16))
            ctl.l[me] = __int_as_float(0x7fffffff);
      }

      // 32 scores; -inf where masked
      const auto fetch = [&](int c, uint32_t (&x)[32]) {
        tmem_read32(s_col + 32 * c, x);
        if (whole) return;
        const uint32_t seen = bit_range(ctl.lo[me] - base - 32 * c, ctl.hi[me] - base - 32 * c) &
                              ((present >> (2 * c) & 1 ? 0xffffu : 0u) | (present >> (2 * c) & 2 ? 0xffff0000u : 0u));
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = seen >> j & 1 ? x[j] : kMinusInf;
      };
      // Factor and offset that make u of a product, for one block.  A factor
      // of zero, or an infinite offset, would make NaN of a masked score.
      const auto factor = [&](const GroupInfo& g, float& a, float& d) {
        const float product = qs * g.ks;
        d = ctl.bias[me] * fminf(product, kMostOffset);
        a = product * key_gain<CODE>();
        a = a == 0.0f ? 1.17549435e-38f : a;
      };
      ok = ok && wait(&ctl.s_full[tile], i & 1, kSiteEpilogue);
      if (used == 2 && i + tile > 0) ok = ok && wait(&ctl.turn[tile], (i + tile - 1) & 1, kSiteEpilogue);
      tc_fence_after();
      uint32_t w[kHalfTokens / 2];
      float sum, ref;
      bool raise = i == 0 || present & kQuiet, last = true;  // last: the turn has not been passed on
      for (;;) {
        if (raise) {
          float top_t = -INFINITY, top_u = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < kHalfTokens / 32; ++c) {
            uint32_t sc[32];
            fetch(c, sc);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float top = -INFINITY, a, d;
#pragma unroll
              for (int j = 0; j < 16; ++j) top = fmaxf(top, __uint_as_float(sc[16 * h + j]));
              const GroupInfo g = info[2 * c + h];
              factor(g, a, d);
              const float u = fmaf(top, a, d);
              top_u = fmaxf(top_u, u);
              top_t = fmaxf(top_t, u + g.lv);
            }
          }
          ctl.row[0][half][cta_row] = top_t;
          ctl.row[1][half][cta_row] = top_u;
          named_bar_sync(pair, 2 * kWarp);
          const float next = fmaxf(m, fmaxf(top_t, ctl.row[0][other][cta_row]) - kReferenceLog2);
          const float next_n = fmaxf(ctl.n[me], fmaxf(top_u, ctl.row[1][other][cta_row]));
          const float alpha = weight_of(m, next);
          ctl.l[me] *= weight_of(ctl.n[me], next_n);
          ctl.n[me] = next_n;
          m = next;
          if (i > 0) {
            if (kApart<DIM>) {
              ok = ok && wait(&ctl.o_done[tile], (i - 1) & 1, kSiteEpilogue);
              tc_fence_after();
            }
#pragma unroll 1
            for (int c = 0; c < DIM / 64; ++c) {
              uint32_t o[32];
              tmem_read32(o_col + 32 * c, o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st32(o_col + 32 * c, o);
            }
          }
          if (present & kQuiet) {
            const float from = next_n == -INFINITY ? 0.0f : next_n;
            float all = 0.0f;
#pragma unroll 1
            for (int c = 0; c < kHalfTokens / 32; ++c) {
              uint32_t sc[32];
              fetch(c, sc);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float a, d;
                factor(info[2 * c + h], a, d);
                d -= from;
#pragma unroll
                for (int j = 0; j < 16; ++j) all += exp2_approx(fmaf(__uint_as_float(sc[16 * h + j]), a, d));
              }
            }
            ctl.l[me] += all;
          }
        }
        ref = m == -INFINITY ? 0.0f : m;
        float weights = 0.0f;
        sum = 0.0f;
        uint32_t sc[32];
#pragma unroll
        for (int x = 0; x < kHalfTokens / SEG; ++x) {
          const GroupInfo g = info[x * (SEG / 16)];
          float a, d;
          factor(g, a, d);
          d += g.lv - ref;
          const uint64_t aa = pair_of(a, a), dd = pair_of(d, d);
          uint64_t part = 0;
#pragma unroll
          for (int y = 0; y < SEG; y += 2) {
            const int at = x * SEG + y;
            if (at % 32 == 0) fetch(at / 32, sc);
            // the other row tile's turn, with its first steps under these
            if (at == 32 && last && lane == 0) mbar_arrive(&ctl.turn[tile ^ 1]);
            const uint32_t* two = &sc[at % 32];
            float v0, v1;
            unpair(fma_pair(pair_of(__uint_as_float(two[0]), __uint_as_float(two[1])), aa, dd), v0, v1);
            v0 = exp2_approx(v0);
            v1 = exp2_approx(v1);
            part = add_pair(part, pair_of(v0, v1));
            w[at / 2] = pack_half2(v0, v1);
          }
          float even, odd;
          unpair(part, even, odd);
          weights += even + odd;
          sum = fmaf(even + odd, g.iv, sum);
        }
        // both threads of a row go on, or both raise its reference; weights
        // may lie where the other one's scores were
        tc_fence_before();
        const bool fits = raise || (weights <= kMostWeight && m > -INFINITY) || weights != weights;
        if (bar_and(pair, 2 * kWarp, fits)) break;
        raise = true;
        last = false;
      }
      if (kApart<DIM>) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.s_read[tile]);
        if (i > 0) ok = ok && wait(&ctl.o_done[tile], (i - 1) & 1, kSiteEpilogue);
      }
      tc_fence_after();
      tmem_st32(p_col, w);
      const float n = ctl.n[me];
      ctl.l[me] = fmaf(sum, exp2_approx(ref - ctl.top_lv[i & 3] - (n == -INFINITY ? 0.0f : n)), ctl.l[me]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.p_full[tile]);
    }
    if (ok && count > 0) ok = wait(&ctl.o_done[tile], (count - 1) & 1, kSiteEpilogue);
    ctl.row[0][half][cta_row] = ctl.l[me];
    ok = bar_and(pair, 2 * kWarp, ok);
    if (ok) {
      tc_fence_after();
      const float n = ctl.n[me], l = ctl.row[0][0][cta_row] + ctl.row[0][1][cta_row];
      const float inv = l == 0.0f ? 0.0f : exp2_approx(m - n) / l;
      const int r = blk.row0 + cta_row;
      const bool valid = r < blk.rows;
      const int64_t out_row = output_row(p, blk.s, work.head, r);
      float* sums = nullptr;
      if (work.parts > 1) {
        const int64_t part = static_cast<int64_t>(work.slot * p.kv_heads + work.head) * tp.splits + work.split;
        sums = tp.partial + (part * kCtaRows + cta_row) * DIM + half * (DIM / 2);
        if (half == 0) {
          float* stats = part_stats<DIM>(tp) + part * 3 * kCtaRows + cta_row;
          stats[0] = m;
          stats[kCtaRows] = n;
          stats[2 * kCtaRows] = l;
        }
      } else if (half == 0 && valid && p.lse != nullptr) {
        p.lse[out_row] = l == 0.0f ? -INFINITY : (n + __log2f(l)) * kLn2;
      }
#pragma unroll 1
      for (int c = 0; c < DIM / 64; ++c) {
        uint32_t o[32];
        if (count > 0) {
          tmem_read32(o_col + 32 * c, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0;
        }
        if (sums != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(sums + 32 * c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        } else if (valid) {
          uint16_t* dst = static_cast<uint16_t*>(p.out) + out_row * DIM + half * (DIM / 2) + 32 * c;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(o[j + x]) * inv;
            *reinterpret_cast<uint4*>(dst + j) = p.q_bf16 ? Vec<__nv_bfloat16>::pack(f) : Vec<__half>::pack(f);
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// Joins the parts of row blocks that were split: a thread 4 channels of a row.
constexpr int kJoinThreads = 256;

template <int DIM>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(TilesParams tp) {
  constexpr int kRowsEach = kJoinThreads / (DIM / 4);
  const AttendParams& p = tp.a;
  const int item = blockIdx.x / (kCtaRows / kRowsEach), slot = item / p.kv_heads;
  const int head = item - slot * p.kv_heads;
  Block blk;
  if (!load_block(p, slot, blk)) return;
  const int parts = part_count(tp, blk.tiles);
  const int rr = blockIdx.x % (kCtaRows / kRowsEach) * kRowsEach + threadIdx.x / (DIM / 4);
  const int r = blk.row0 + rr;
  if (parts == 1 || r >= blk.rows) return;
  const int d = threadIdx.x % (DIM / 4) * 4;
  const int64_t part0 = static_cast<int64_t>(item) * tp.splits;
  const float* stats = part_stats<DIM>(tp) + part0 * 3 * kCtaRows + rr;
  float m = -INFINITY, n = -INFINITY, l = 0.0f;
  for (int i = 0; i < parts; ++i) {
    m = fmaxf(m, stats[i * 3 * kCtaRows]);
    n = fmaxf(n, stats[i * 3 * kCtaRows + kCtaRows]);
  }
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int i = 0; i < parts; ++i) {
    const float w = weight_of(stats[i * 3 * kCtaRows], m);
    l = fmaf(stats[i * 3 * kCtaRows + 2 * kCtaRows], weight_of(stats[i * 3 * kCtaRows + kCtaRows], n), l);
    const float4 x = *reinterpret_cast<const float4*>(tp.partial + ((part0 + i) * kCtaRows + rr) * DIM + d);
    v.x = fmaf(x.x, w, v.x), v.y = fmaf(x.y, w, v.y), v.z = fmaf(x.z, w, v.z), v.w = fmaf(x.w, w, v.w);
  }
  const float inv = l == 0.0f ? 0.0f : exp2_approx(m - n) / l;
  const int64_t out_row = output_row(p, blk.s, head, r);
  uint2 w;
  if (p.q_bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x * inv, v.y * inv);
    const __nv_bfloat162 c = __floats2bfloat162_rn(v.z * inv, v.w * inv);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
  } else {
    w = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
  }
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out_row * DIM + d) = w;
  if (p.lse != nullptr && d == 0) p.lse[out_row] = l == 0.0f ? -INFINITY : (n + __log2f(l)) * kLn2;
}

int64_t block_slots(int64_t tokens, int64_t batch, int64_t group) { return tokens * group / kCtaRows + batch; }

// Parts that every row block's tokens are split into: the number that gives
// the least time for CTAs of equal length, one an SM, where a part costs its
// tiles and about kPartTiles more (its start, its end and its share of the
// join).  Lengths are not known here: the longest that the table can hold, or
// the window, stands for them.
constexpr int64_t kPartTiles = 4, kMostParts = 64;

int tile_splits(int64_t tokens, int64_t batch, int64_t group, int64_t kv_heads, int64_t width, int page,
                int64_t window) {
  const int64_t items = block_slots(tokens, batch, group) * kv_heads, sms = device_sm_count();
  int64_t seen = width * page;
  if (window > 0 && window + kCtaRows / group < seen) seen = window + kCtaRows / group;
  const int64_t tiles = ceil_div64(seen, kTileTokens);
  int64_t best = 1, least = ceil_div64(items, sms) * (tiles + kPartTiles);
  for (int64_t s = 2; s <= kMostParts && s <= tiles && items * s <= 4 * sms; ++s) {
    const int64_t time = ceil_div64(items * s, sms) * (ceil_div64(tiles, s) + kPartTiles) + kPartTiles;
    if (time < least) best = s, least = time;
  }
  return static_cast<int>(best);
}

template <int DIM, int CODE, int SEG>
cudaError_t launch_tiles(const TilesParams& tp, cudaStream_t stream) {
  constexpr int kBytes = kTilesBytes<DIM>;
  static_assert(kBytes <= 227 * 1024, "a tile's operands do not fit in shared memory");
  const int64_t items = static_cast<int64_t>(tp.slots) * tp.a.kv_heads;
  if (items * tp.splits > INT32_MAX / 32) return cudaErrorInvalidValue;
  static bool ready[64] = {};
  cudaError_t e = allow_shared(reinterpret_cast<const void*>(kv_tiles_kernel<DIM, CODE, SEG>), kBytes, ready);
  if (e != cudaSuccess) return e;
  kv_tiles_kernel<DIM, CODE, SEG><<<static_cast<unsigned>(items * tp.splits), kTilesThreads, kBytes, stream>>>(tp);
  e = cudaGetLastError();
  if (e != cudaSuccess || tp.splits == 1) return e;
  constexpr int kBlocks = kCtaRows / (kJoinThreads / (DIM / 4));
  kv_join_kernel<DIM><<<static_cast<unsigned>(items * kBlocks), kJoinThreads, 0, stream>>>(tp);
  return cudaGetLastError();
}

template <int DIM, int CODE>
cudaError_t launch_tiles_page(const TilesParams& tp, cudaStream_t stream) {
  if (tp.a.page_shift >= 6) return launch_tiles<DIM, CODE, 64>(tp, stream);
  // pages of 32, an 8192-token prompt of 32 heads of 128: 735 us with their
  // own variant, 847 us with that of 16; heads of 64: 633 and 623 us
  if constexpr (DIM == 128) {
    if (tp.a.page_shift == 5) return launch_tiles<DIM, CODE, 32>(tp, stream);
  }
  return launch_tiles<DIM, CODE, 16>(tp, stream);
}

}  // namespace

size_t tiles_workspace_bytes(int64_t tokens, int64_t batch, int64_t group, int64_t kv_heads, int dim, int64_t width,
                             int page, int64_t window) {
  const int splits = tile_splits(tokens, batch, group, kv_heads, width, page, window);
  if (splits == 1) return 0;
  return static_cast<size_t>(block_slots(tokens, batch, group) * kv_heads * splits) * kCtaRows * (dim + 3) *
         sizeof(float);
}

cudaError_t run_tiles(const AttendParams& p, int dim, int code, void* workspace, cudaStream_t stream) {
  TilesParams tp{};
  tp.a = p;
  tp.slots = static_cast<int>(block_slots(p.tok.tokens, p.tok.batch, p.group));
  tp.splits = tile_splits(p.tok.tokens, p.tok.batch, p.group, p.kv_heads, p.width, 1 << p.page_shift, p.window);
  tp.partial = static_cast<float*>(workspace);
  tp.status = status_word_ptr();
  const bool int8 = code == kCodeInt8;
  if (dim == 64)
    return int8 ? launch_tiles_page<64, kCodeInt8>(tp, stream) : launch_tiles_page<64, kCodeE4M3>(tp, stream);
  return int8 ? launch_tiles_page<128, kCodeInt8>(tp, stream) : launch_tiles_page<128, kCodeE4M3>(tp, stream);
}

}  // namespace b2
