// Products grouped by expert on the Blackwell tensor cores: TMA -> shared memory -> tcgen05.mma -> TMEM -> tcgen05.ld.
//   rows:  C[r, j] = sum_k A[r, k] B[g][k, j]            r in group g; bf16, fp16, or 8 bits with block scales
//   inner: D[g][i, j] = sum over r in group g of L[r, i] R[r, j]   (the gradient of the weights)
//
// The product is formed transposed.  The 128 lanes of an accumulator (M of the MMA) are output columns j, which are adjacent in
// memory, so that a warp's store is one run of them; the accumulator's columns (N of the MMA) are rows of the group, and N is
// chosen tile by tile in steps of 16: a group of 20 rows costs 32, not the 128 that rows on the M side would cost.
//
// Tiles.  Wide: pairs of CTAs (cta_group::2) make 256 output columns x up to 256 rows; each CTA loads its 128 columns of the
// weights and half of the rows, so that an operand byte feeds twice the work that it feeds in one CTA.  Narrow, for groups of few
// rows, whose time is the reading of the weights: one CTA makes 128 columns x up to 64 (16 bits: or 128) rows, and a cluster of up
// to eight CTAs shares the inner axis of a tile where there are few tiles; their sums are added through distributed shared memory,
// in the order of the CTAs' ranks, so that results do not depend on timing and no workspace is needed.
//
// Which tile lies where is worked out on the device from the offsets: every CTA builds the table of the groups' tiles in shared
// memory, and the CTAs (pairs, clusters) walk the tiles in turn.
//
// Operands whose rows do not lie on 16-byte boundaries, which TMA cannot copy, are first copied to rows that do, in memory from the
// context's stream-ordered pool: of the weights those of groups with rows.  (3,001 rows, 7 groups, 1111 x 777: warps that read such
// rows themselves and shift them into place for every tile took 62 us, the copy and the product 21.  Not measured where a group has
// few rows, whose weights the copy moves three times: 512 rows, 64 groups, 2047 x 1536 198 us, 2048 x 1536 69.)
//
// Roles: warp 0 copies, warp 1 issues the MMAs, warp 2 clears the rows behind a group's last (inner form),
// four warps (wide tiles: eight) from warp 4 on read the accumulators, round and store.
//
// The inner form has rows of the result on the lanes, whose results then lie in a row in each lane's registers.  Wide 8-bit tiles
// have their rows on the lanes too, and 256 columns of the weights as accumulator columns: a row's scale is then one
// register of its lane.  (With the columns on the lanes each row's scale must reach all lanes, 128 KB a block through the
// shared memory's 128 bytes a clock, twice the time of the block's products: 8192^3 905 us.)
//
// 8-bit operands: the 128 products of a scale block are one chain of the tensor core in an accumulator of its own; the storing
// warps add it, times the scales of its row and block, to f32 sums in their registers (two sums per fma.f32x2).
//
// What bounds it (one B200; ncu: profiles of these kernels).  Wide, 16 bits, large groups: the tensor pipe, 92 % of whose cycles are
// active (8192 rows, 4 groups, 4096 x 4096, 530 clocks a stage of 512), at the clock that the power limit leaves: 8192^3 707 us =
// 1,555 TFLOP/s alone, some 1,300 over and over at 1.2 GHz.  Ragged groups of some 256 rows do not fill the pipe: 62 % (16,384 rows,
// 64 groups, 2048 x 1536, with HBM at 63 %), since a tile of 128 to 192 rows brings a whole stage of weights for its share of the
// products.  Wide, 8 bits: the round trip of an accumulator (products 512 clocks, their completion some 500, reading 350, the next
// products' issue 250; two accumulators fill TMEM): 8192^3 469 us = 2,340 TFLOP/s alone.  Few rows: HBM, and some 3 us of launch,
// set-up and pipeline fill (narrow: one group of 64 rows, 4096 x 4096 11.6 us for 35 MB; wide, which takes the same time as narrow
// tiles on many groups: 8 rows on 8 of 64, 2048 x 1536 12.1 us for 50 MB, 512 rows on 64 69 us for 406 MB).
//
// Tried: four operand boxes a stage issued by one lane's own code (250 us for 187), scales by way of shared memory (see above), a
// tile's shared sums stored to where they are added instead of fetched (64 rows 7.7 -> 8.8 us, 256 rows 10.2 -> 13.0), storing warps
// that sleep between polls (no change), results of 64 columns on their way while 32 are stored (no change).
//
// Every mbarrier wait is bounded: when one runs out the kernel raises the status word, frees its TMEM columns and returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "grouped_tiles.cuh"
#include "swb_chain.cuh"
#include "swb_index.h"
#include "swb_kernels.h"

namespace swb {
namespace {

constexpr uint32_t WAIT_LIMIT = 1u << 22;  // polls of some 1.5 us each
constexpr int LANES = 128;           // output columns of a CTA's tile
constexpr int ROW_BYTES = 128;       // of a swizzled row of an operand in shared memory
constexpr int BOX_BYTES = 64 * ROW_BYTES;  // a box of 64 inner rows x 64 16-bit elements
constexpr int FIRST_STORE_WARP = 4;
constexpr unsigned FULL = 0xffffffffu;
constexpr int MOST_TILES = 1 << 30;  // of a call

// SHARED (inner form): a group's rows are shared among p.splits parts, whose f32 sums go to p.partials.
template <int CTAS_, int TILE_, bool FP8_, bool MN_, bool INNER_, bool SHARED_ = false>
struct Config {
  static constexpr bool SHARED = SHARED_;
  static constexpr int CTAS = CTAS_, TILE = TILE_;   // TILE: accumulator columns, the rows of a tile
  static constexpr bool FP8 = FP8_, MN = MN_, INNER = INNER_;  // MN: the lanes' operand has its columns contiguous
  static constexpr bool ROWS_ON_LANES = (FP8 && CTAS == 2) || INNER;  // see above
  static constexpr int STEP = FP8 ? 128 : 64;        // inner elements of a stage: 128 bytes
  static constexpr int MMA_STEP = FP8 ? 32 : 16;     // of an MMA
  static constexpr int ROWS_CTA = TILE / CTAS;       // of a tile's rows in one CTA's shared memory
  static constexpr int ROW_BOX = INNER ? 64 : FP8 && CTAS == 2 ? 128 : CTAS == 2 ? 32 : 16;  // rows of a copy
  static constexpr int L_BYTES = LANES * ROW_BYTES, T_BYTES = ROWS_CTA * ROW_BYTES, STAGE = L_BYTES + T_BYTES;
  static constexpr int BUFFERS = 512 / TILE < 4 ? 512 / TILE : 4;
  static constexpr int TMEM_COLS = BUFFERS * TILE;
  static constexpr int STORE_WARPS = CTAS == 2 ? 8 : 4;
  static constexpr int WARP_COLS = TILE / (STORE_WARPS / 4);  // accumulator columns of a storing warp
  static constexpr int THREADS = 32 * (FIRST_STORE_WARP + STORE_WARPS);
  static constexpr bool SPLITS = CTAS == 1 && !INNER;
  static constexpr int PARTIAL = SPLITS ? TILE * LANES * 4 : 0;       // f32 sums of this CTA's share of the inner axis
  static constexpr int SCALES = FP8 && !ROWS_ON_LANES ? STORE_WARPS * 4 * WARP_COLS * 4 : 0;
  static constexpr int STAGED = STORE_WARPS * 32 * 64;                // 32 x 32 results of a warp on their way to rows of C
  static constexpr int TABLE = (int)kMaxGroups * 16 + 16;             // GroupTiles, and first tiles
  static constexpr int STAGES = (232448 - 1024 - 512 - PARTIAL - SCALES - STAGED - TABLE) / STAGE;
  static constexpr int SMEM = 1024 + STAGES * STAGE + PARTIAL + SCALES + STAGED + TABLE;
  static constexpr int MOST_SORTED = CTAS == 2 ? 128 : 1;             // groups
  static constexpr int ROUND = 16 * CTAS;                             // N of an MMA is a multiple of this
};

// Division by a number known beforehand: the product with 2^32 / d, rounded down, gives the quotient or one less.
struct Divisor {
  uint32_t d, inverse;

  __host__ __device__ static Divisor of(uint32_t d) { return {d, d > 1 ? (uint32_t)((1ull << 32) / d) : 0xffffffffu}; }
  __device__ __forceinline__ int divide(int x, int *rest) const {
    uint32_t q = __umulhi((uint32_t)x, inverse), r = (uint32_t)x - q * d;
    if (r >= d) {
      ++q;
      r -= d;
    }
    *rest = (int)r;
    return (int)q;
  }
};

struct Product {
  int rows, inner, cols, groups;  // inner form: `inner` is the size of i, `cols` that of j
  const int32_t *offsets;
  uint16_t *out;
  uint32_t instruction;           // descriptor without N
  bool half_out;
  const float *a_scales, *b_scales;
  bool sorted;                    // groups are taken by the work of a tile, largest first, and the walkers to and fro
  int col_tiles;                  // tiles along the columns
  Divisor per_band;               // tiles of eight row tiles
  Divisor per_group, per_column;  // inner form: tiles of a group, of a column of tiles
  Divisor splits;                 // ... and parts of its rows, whose f32 sums lie in `partials`, rows of `pitch`, where it is above 1
  float *partials;
  int64_t pitch;
  int scale_k, scale_j;
  int64_t scale_group;
  int *status;
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ uint64_t make_desc(uint32_t addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {  // 128-byte swizzle
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ bool elected() {  // one lane of a converged warp
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Copies, MMAs and accumulators are ordered by their own rules, so that a wait needs to see plain stores of its own CTA at most;
// CLUSTER: stores of other CTAs too.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    if constexpr (CLUSTER)
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// `bar` may be another CTA's of the cluster (mapped).  RELEASE: the warp's plain stores before it are visible to who waits.
template <bool RELEASE = false>
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  if constexpr (RELEASE)
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t mapped(uint32_t addr, uint32_t rank) {  // the same place in CTA `rank` of the cluster
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}

template <int CTAS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

template <int CTAS, bool FP8>
__device__ __forceinline__ void issue_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
#define SWB_MMA(group, kind)                                                                                     \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma." group "." kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
               "l"(a), "l"(b), "r"(instruction), "r"(add ? 1u : 0u) : "memory")
  if constexpr (CTAS == 2 && FP8) SWB_MMA("cta_group::2", "kind::f8f6f4");
  else if constexpr (CTAS == 2) SWB_MMA("cta_group::2", "kind::f16");
  else if constexpr (FP8) SWB_MMA("cta_group::1", "kind::f8f6f4");
  else SWB_MMA("cta_group::1", "kind::f16");
#undef SWB_MMA
}
// Arrives on `bar` (of both CTAs of a pair) when the MMAs issued so far have completed.
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 accumulator columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_load(uint32_t (&v)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr) : "memory");
}
// 16 lanes x 32 accumulator columns: register 4 i + 2 a + b of lane l is lane l / 4 + 8 a, column 8 i + 2 (l % 4) + b.
__device__ __forceinline__ void tmem_load_blocks(uint32_t (&v)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A load that stays where it is written: the compiler moves others down to where their value is needed, to save registers.
__device__ __forceinline__ float load_here(const float *p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ uint64_t pack(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ void unpack(uint64_t v, uint32_t &lo, uint32_t &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {  // two f32 each
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint16_t rounded(float v, bool half_out) {  // once, to nearest
  return half_out ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ uint32_t rounded_two(float lo, float hi, bool half_out) {
  uint32_t r;
  if (half_out) {
    const __half2 two = __floats2half2_rn(lo, hi);
    memcpy(&r, &two, 4);
  } else {
    const __nv_bfloat162 two = __floats2bfloat162_rn(lo, hi);
    memcpy(&r, &two, 4);
  }
  return r;
}

__device__ __forceinline__ Divisor up_to_eight(int d) {
  const uint32_t inverse = d == 1 ? 0xffffffffu : d == 2 ? 1u << 31 : d == 3 ? 0x55555555u : d == 4 ? 1u << 30 : d == 5 ? 0x33333333u
                           : d == 6 ? 0x2aaaaaaau : d == 7 ? 0x24924924u : 1u << 29;
  return {(uint32_t)d, inverse};
}

// A group's rows, and its row tiles: as few as the tile size allows, of equal heights (a multiple of 16) but for the last.
struct GroupTiles {
  int begin, end;
  uint32_t packed;

  template <class S>
  __device__ __forceinline__ static GroupTiles of(RowSpan span) {
    const int m = span.end - span.begin, count = (m + S::TILE - 1) / S::TILE;
    const int height = count ? ((m + count - 1) / count + S::ROUND - 1) / S::ROUND * S::ROUND : S::ROUND;
    return {span.begin, span.end, (uint32_t)count << 5 | (uint32_t)(height / 16)};
  }
  __device__ __forceinline__ int count() const { return (int)(packed >> 5); }
  __device__ __forceinline__ int height() const { return (int)(packed & 31u) * 16; }
};

struct Tile {
  int group, row0, valid;     // rows [row0, row0 + valid) (inner form: of axis i)
  int col0;                   // first output column of this CTA (pair)
  int n;                      // accumulator columns that are computed: those of the rows, or (rows on the lanes) of the columns
  int k0, k_blocks, k_valid;  // first stage of the inner axis, stages, elements of the last that exist
};

__device__ __forceinline__ Tile uniform(const Tile &t) {  // the same in all lanes, known to be
  Tile u;
  u.group = __shfl_sync(FULL, t.group, 0);
  u.row0 = __shfl_sync(FULL, t.row0, 0);
  u.valid = __shfl_sync(FULL, t.valid, 0);
  u.n = __shfl_sync(FULL, t.n, 0);
  u.col0 = __shfl_sync(FULL, t.col0, 0);
  u.k0 = __shfl_sync(FULL, t.k0, 0);
  u.k_blocks = __shfl_sync(FULL, t.k_blocks, 0);
  u.k_valid = __shfl_sync(FULL, t.k_valid, 0);
  return u;
}

template <class S>
struct Tiles {
  const GroupTiles *spans;
  const int *first;       // first tile of each group, in the order in which they are taken, and the end
  const uint16_t *order;  // NULL: as they come
  int groups, total, walker, walkers;

  // The tile of this walker (CTA, pair, cluster) in a round; there may be none in the last.
  __device__ __forceinline__ int of_round(int round) const {
    return round * walkers + (order && round % 2 == 1 ? walkers - 1 - walker : walker);
  }
  __device__ __forceinline__ int rounds() const { return (total + walkers - 1) / walkers; }

  __device__ __forceinline__ Tile at(int t, const Product &p, int part, int parts) const {
    Tile tile;
    if constexpr (S::INNER) {
      static_assert(S::TILE == LANES * S::CTAS, "");  // square tiles
      int local, it;
      tile.group = p.per_group.divide(t, &local);
      if (order) tile.group = order[tile.group];
      tile.col0 = p.per_column.divide(local, &it) * (LANES * S::CTAS);
      tile.row0 = it * S::TILE;
      tile.valid = p.inner - tile.row0 < S::TILE ? p.inner - tile.row0 : S::TILE;
      const int n = p.cols - tile.col0 < S::TILE ? p.cols - tile.col0 : S::TILE;
      tile.n = (n + S::ROUND - 1) / S::ROUND * S::ROUND;
      if constexpr (S::SHARED) {  // a part of the group's rows
        int sub, rest;
        const GroupTiles span = spans[p.splits.divide(tile.group, &sub)];
        const int blocks = (span.end - span.begin + S::STEP - 1) / S::STEP;
        const int each = p.splits.divide(blocks + (int)p.splits.d - 1, &rest);
        tile.k0 = span.begin + (each * sub < blocks ? each * sub : blocks) * S::STEP;
        const int left = span.end - tile.k0 > 0 ? span.end - tile.k0 : 0, m = left < each * S::STEP ? left : each * S::STEP;
        tile.k_blocks = (m + S::STEP - 1) / S::STEP;
        tile.k_valid = m - (tile.k_blocks - 1) * S::STEP;
      } else {
        const GroupTiles span = spans[tile.group];
        const int m = span.end - span.begin;
        tile.k0 = span.begin;
        tile.k_blocks = (m + S::STEP - 1) / S::STEP;
        tile.k_valid = m - (tile.k_blocks - 1) * S::STEP;
      }
    } else {
      int lo = 0, hi = groups;  // the last group whose first tile is at most t
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= t) lo = mid; else hi = mid;
      }
      tile.group = order ? order[lo] : lo;
      const GroupTiles span = spans[tile.group];
      // bands of eight row tiles, column tile after column tile within one: what runs at a time shares both operands in L2
      int in_band, in_rows;
      const int band = p.per_band.divide(t - first[lo], &in_band);
      const int left = span.count() - band * 8;
      tile.col0 = up_to_eight(left < 8 ? left : 8).divide(in_band, &in_rows) * (LANES * S::CTAS);
      tile.row0 = span.begin + (band * 8 + in_rows) * span.height();
      tile.valid = span.end - tile.row0 < span.height() ? span.end - tile.row0 : span.height();
      int n = tile.valid;
      if constexpr (S::ROWS_ON_LANES) n = p.cols - tile.col0 < S::TILE ? p.cols - tile.col0 : S::TILE;
      tile.n = (n + S::ROUND - 1) / S::ROUND * S::ROUND;
      const int blocks = (p.inner + S::STEP - 1) / S::STEP;
      tile.k0 = (int)((int64_t)blocks * part / parts);
      tile.k_blocks = (int)((int64_t)blocks * (part + 1) / parts) - tile.k0;
      tile.k_valid = S::STEP;  // copies fill what lies behind the axis with zeros
    }
    return tile;
  }
};

template <class S>
__global__ void __launch_bounds__(S::THREADS, 1) grouped_tcgen05_kernel(const __grid_constant__ CUtensorMap map_l,
                                                                        const __grid_constant__ CUtensorMap map_t, const Product p,
                                                                        const int cluster_parts) {
  const int parts = S::SPLITS ? cluster_parts : 1;  // CTAs that share a tile's inner axis
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[S::STAGES], bar_empty[S::STAGES], bar_landed[S::STAGES];
  __shared__ __align__(8) uint64_t bar_sums[S::BUFFERS], bar_stored[S::BUFFERS], bar_parts, bar_added;
  __shared__ uint16_t order[S::MOST_SORTED];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int tid = threadIdx.x, warp = __shfl_sync(FULL, tid >> 5, 0), lane = tid & 31;
  const uint32_t stage0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *behind = smem_raw + (stage0 - smem_u32(smem_raw)) + S::STAGES * S::STAGE;
  float *partial = reinterpret_cast<float *>(behind);                         // [TILE][LANES]
  float *scales = reinterpret_cast<float *>(behind + S::PARTIAL);             // [warp][4][WARP_COLS]
  uint8_t *staged_all = behind + S::PARTIAL + S::SCALES;
  GroupTiles *spans = reinterpret_cast<GroupTiles *>(staged_all + S::STAGED);
  int *first = reinterpret_cast<int *>(spans + kMaxGroups);
  const int rank = S::CTAS == 2 || S::SPLITS ? (int)(blockIdx.x % (unsigned)(S::CTAS == 2 ? 2 : parts)) : 0;
  const int part = S::CTAS == 2 ? 0 : rank;  // of the inner axis

  if (tid == 0) {
    failed = 0;
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(smem_u32(&bar_full[s]), S::CTAS);
      mbar_init(smem_u32(&bar_empty[s]), 1);
      mbar_init(smem_u32(&bar_landed[s]), 1);
    }
    for (int a = 0; a < S::BUFFERS; ++a) {
      mbar_init(smem_u32(&bar_sums[a]), 1);
      mbar_init(smem_u32(&bar_stored[a]), S::STORE_WARPS * S::CTAS);
    }
    mbar_init(smem_u32(&bar_parts), S::STORE_WARPS * parts);
    mbar_init(smem_u32(&bar_added), S::STORE_WARPS * parts);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_l) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_t) : "memory");
  }
  after_previous_kernel();
  RowSpan own_rows = {};  // on its way while the rest is set up
  if (tid < p.groups) own_rows = group_rows(p.offsets, tid, p.rows);
  if (warp == 1) {
    if constexpr (S::CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                   "r"(S::TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                   "r"(S::TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  __syncwarp();
  const bool in_cluster = S::CTAS == 2 || parts > 1;
  if (in_cluster) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  Tiles<S> tiles;
  tiles.spans = spans;
  tiles.first = first;
  tiles.order = S::CTAS == 2 && p.sorted ? order : nullptr;
  tiles.groups = p.groups;
  tiles.walkers = (int)gridDim.x / (S::CTAS == 2 ? 2 : parts);
  tiles.walker = (int)blockIdx.x / (S::CTAS == 2 ? 2 : parts);
  const bool one_group = S::CTAS == 1 && p.groups == 1;  // (pairs: the case costs the 8-bit form registers that it lacks)
  bool decreasing = own_rows.decreasing;
  for (int g = tid + S::THREADS; g < p.groups; g += S::THREADS) decreasing |= group_rows(p.offsets, g, p.rows).decreasing;
  if (tid == 0) first[0] = 0;
  const bool none = __syncthreads_or(decreasing);  // groups that share rows would make work without bounds: all count as empty
  if (tid < p.groups) spans[tid] = GroupTiles::of<S>(none ? RowSpan{0, 0} : own_rows);
  for (int g = tid + S::THREADS; g < p.groups; g += S::THREADS)
    spans[g] = GroupTiles::of<S>(none ? RowSpan{0, 0} : group_rows(p.offsets, g, p.rows));
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (S::CTAS == 2 && p.sorted) {  // by a tile's stages (inner form) or rows, equal ones as they come
    auto work = [&](int g) { return S::INNER ? spans[g].end - spans[g].begin : spans[g].height(); };
    for (int g = tid; g < p.groups; g += S::THREADS) {
      const int own = work(g);
      int place = 0;
      for (int h = 0; h < p.groups; ++h) {
        const int other = work(h);
        place += other > own || (other == own && h < g);
      }
      order[place] = (uint16_t)g;
    }
    __syncthreads();
  }
  if (!S::INNER && !one_group) {
    if (warp == 0) {
      int before = 0;
      for (int g0 = 0; g0 < p.groups; g0 += 32) {
        int through = 0;
        if (g0 + lane < p.groups) through = spans[tiles.order ? order[g0 + lane] : g0 + lane].count() * p.col_tiles;
        const int own = through;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int v = __shfl_up_sync(FULL, through, d);
          if (lane >= d) through += v;
        }
        if (g0 + lane < p.groups) first[g0 + lane] = before + through - own;
        before += __shfl_sync(FULL, through, 31);
      }
      if (lane == 0) first[p.groups] = before;
    }
    __syncthreads();
  }
  __syncwarp();
  // The barriers of the other CTAs, and the pair's TMEM, are ready too.
  if (in_cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(FULL, tmem_slot, 0);
  if constexpr (S::INNER) tiles.total = p.groups * (int)((S::SHARED ? p.splits.d : 1u) * p.per_group.d);
  else tiles.total = __shfl_sync(FULL, one_group ? spans[0].count() * p.col_tiles : first[p.groups], 0);

  const int rounds = __shfl_sync(FULL, tiles.rounds(), 0);

  auto gave_up = [&] {
    failed = 1;
    atomicExch(p.status, 1);
  };

  // The warps that copy and that issue MMAs walk their loops as whole warps and elect a lane for the instructions alone: what these
  // take then lies in uniform registers (as one lane's own code, four MMAs took their thread 690 clocks whatever their size).
  // The eight storing warps of the wide 8-bit form need more registers than 12 warps can have alike: 128 x 56 + 256 x 224 are the
  // 384 x 168 of the launch.
  if (warp < FIRST_STORE_WARP) {
    if constexpr (S::FP8 && S::CTAS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      int s = 0;
      uint32_t round = 0;
      bool ok = true;
      const bool issues = elected();
      const uint32_t leader_full = S::CTAS == 2 ? mapped(smem_u32(bar_full), 0) : smem_u32(bar_full);
      for (int turn = 0; ok && turn < rounds; ++turn) {
        const int t = tiles.of_round(turn);
        if (t >= tiles.total) continue;
        const Tile tile = uniform(tiles.at(t, p, part, parts));
        const int mine = tile.n / S::CTAS, row = tile.row0 + (S::CTAS == 2 ? rank * mine : 0);
        const int col = tile.col0 + (S::CTAS == 2 ? rank * LANES : 0);
        const int boxes = S::FP8 && S::ROWS_ON_LANES ? 1 : (mine + S::ROW_BOX - 1) / S::ROW_BOX;
        const uint32_t bytes = (uint32_t)(S::L_BYTES + boxes * S::ROW_BOX * ROW_BYTES);
        for (int kb = 0; kb < tile.k_blocks; ++kb) {
          if (round > 0) ok = __all_sync(FULL, mbar_wait(smem_u32(&bar_empty[s]), (round - 1) & 1u));
          if (!ok) {
            if (issues) gave_up();
            break;
          }
          const uint32_t l = stage0 + (uint32_t)(s * S::STAGE), tt = l + S::L_BYTES;
          uint32_t bar = leader_full + (uint32_t)(8 * s);
          if constexpr (S::INNER) {
            if (kb == tile.k_blocks - 1 && tile.k_valid % S::MMA_STEP != 0) bar = smem_u32(&bar_landed[s]);
            const int k = tile.k0 + kb * S::STEP;
            if (issues) {
              const int i = tile.row0 + rank * LANES, j = tile.col0 + rank * mine;
              mbar_arrive_expect(bar, bytes);
              tma_load_2d<S::CTAS>(l, &map_t, i, k, bar);
              tma_load_2d<S::CTAS>(l + BOX_BYTES, &map_t, i + 64, k, bar);
              for (int b = 0; b < boxes; ++b) tma_load_2d<S::CTAS>(tt + (uint32_t)(b * BOX_BYTES), &map_l, j + 64 * b, k, bar);
            }
          } else {
            const int k = (tile.k0 + kb) * S::STEP;
            if (issues) {
              mbar_arrive_expect(bar, bytes);
              if constexpr (S::ROWS_ON_LANES) {  // map_l: the weights, which are the columns' operand here
                const int w = tile.col0 + rank * mine;
                tma_load_2d<S::CTAS>(l, &map_t, k, tile.row0 + rank * LANES, bar);
                if constexpr (S::MN) tma_load_3d<S::CTAS>(tt, &map_l, w, k, tile.group, bar);
                else tma_load_3d<S::CTAS>(tt, &map_l, k, w, tile.group, bar);
              } else {
                if constexpr (!S::MN) {
                  tma_load_3d<S::CTAS>(l, &map_l, k, col, tile.group, bar);
                } else {
                  tma_load_3d<S::CTAS>(l, &map_l, col, k, tile.group, bar);
                  if constexpr (!S::FP8) tma_load_3d<S::CTAS>(l + BOX_BYTES, &map_l, col + 64, k, tile.group, bar);
                }
                for (int b = 0; b < boxes; ++b)
                  tma_load_2d<S::CTAS>(tt + (uint32_t)(b * S::ROW_BOX * ROW_BYTES), &map_t, k, row + b * S::ROW_BOX, bar);
              }
            }
          }
          __syncwarp();
          if (++s == S::STAGES) { s = 0; ++round; }
        }
      }
      // the last arrivals on `empty` before the shared memory goes back
      for (int i = 0; ok && i < S::STAGES; ++i) {
        if (s == 0) {
          if (round == 0) break;
          s = S::STAGES;
          --round;
        }
        --s;
        ok = mbar_wait(smem_u32(&bar_empty[s]), round & 1u);
      }
    } else if (warp == 1) {
      if (S::CTAS == 1 || rank == 0) {
        int s = 0, buffer = 0;
        uint32_t round = 0, made = 0;  // accumulators begun
        bool ok = true;
        const bool issues = elected();
        for (int turn = 0; ok && turn < rounds; ++turn) {
          const int t = tiles.of_round(turn);
          if (t >= tiles.total) continue;
          const Tile tile = uniform(tiles.at(t, p, part, parts));
          const uint32_t instruction = p.instruction | ((uint32_t)(tile.n >> 3) << 17);
          uint32_t sums = 0;
          for (int kb = 0; kb < tile.k_blocks; ++kb) {
            const bool fresh = S::FP8 || kb == 0;
            // (inner form: the rows cleared in a group's last stage are plain stores, of the pair's other CTA too)
            if (S::INNER && kb == tile.k_blocks - 1) ok = mbar_wait<true>(smem_u32(&bar_full[s]), round & 1u);
            else ok = mbar_wait(smem_u32(&bar_full[s]), round & 1u);
            if (fresh) {
              buffer = (int)(made % S::BUFFERS);
              if (made >= S::BUFFERS) ok = ok && mbar_wait(smem_u32(&bar_stored[buffer]), (made / S::BUFFERS - 1) & 1u);
              sums = tmem + (uint32_t)(buffer * S::TILE);
              ++made;
            }
            ok = __all_sync(FULL, ok);
            if (!ok) {
              if (issues) gave_up();
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t l = stage0 + (uint32_t)(s * S::STAGE), tt = l + S::L_BYTES;
            const bool last = kb == tile.k_blocks - 1;
            const int steps = S::INNER && last ? (tile.k_valid + S::MMA_STEP - 1) / S::MMA_STEP : S::STEP / S::MMA_STEP;
            constexpr bool A_MN = S::INNER || (S::MN && !S::ROWS_ON_LANES), B_MN = S::INNER || (S::MN && S::ROWS_ON_LANES);
            constexpr uint64_t A_STEP = A_MN ? S::MMA_STEP * ROW_BYTES / 16 : 2, B_STEP = B_MN ? S::MMA_STEP * ROW_BYTES / 16 : 2;
            const uint64_t a = A_MN ? make_desc(l, BOX_BYTES, 1024u) : make_desc(l, 16u, 1024u);
            const uint64_t b = B_MN ? make_desc(tt, BOX_BYTES, 1024u) : make_desc(tt, 16u, 1024u);
            if (issues) {
#pragma unroll
              for (int k = 0; k < S::STEP / S::MMA_STEP; ++k)
                if (!S::INNER || k < steps)
                  issue_mma<S::CTAS, S::FP8>(sums, a + (uint64_t)k * A_STEP, b + (uint64_t)k * B_STEP, instruction, k > 0 || !fresh);
              mma_commit<S::CTAS>(smem_u32(&bar_empty[s]));
              if (S::FP8 || last) mma_commit<S::CTAS>(smem_u32(&bar_sums[buffer]));
            }
            __syncwarp();
            if (++s == S::STAGES) { s = 0; ++round; }
          }
        }
      }
    } else if (warp == 2) {
      if constexpr (S::INNER) {
        // The last stage of a group also holds rows behind the group's last: those that an MMA would read become zeros in both
        // operands (only one would leave a product of zero and whatever the other rows hold).
        uint32_t used = 0, turns = 0;  // stages copied so far; a bit per stage: parity of its turns here
        bool ok = true;
        const uint32_t leader_full = S::CTAS == 2 ? mapped(smem_u32(bar_full), 0) : smem_u32(bar_full);
        for (int turn = 0; ok && turn < rounds; ++turn) {
          const int t = tiles.of_round(turn);
          if (t >= tiles.total) continue;
          const Tile tile = tiles.at(t, p, part, parts);
          used += (uint32_t)tile.k_blocks;
          if (tile.k_blocks == 0 || tile.k_valid % S::MMA_STEP == 0) continue;
          const int s = (int)((used - 1) % S::STAGES);
          ok = mbar_wait(smem_u32(&bar_landed[s]), (turns >> s) & 1u);
          ok = __all_sync(FULL, ok);
          if (!ok) {
            if (lane == 0) gave_up();
            break;
          }
          turns ^= 1u << s;
          const uint32_t base = stage0 + (uint32_t)(s * S::STAGE);
          const int clear = (tile.k_valid + S::MMA_STEP - 1) / S::MMA_STEP * S::MMA_STEP - tile.k_valid;
          constexpr int BOXES = S::STAGE / BOX_BYTES, PIECES = ROW_BYTES / 16;
          for (int i = lane; i < clear * BOXES * PIECES; i += 32) {
            const int piece = i % PIECES, box = i / PIECES % BOXES, row = tile.k_valid + i / (PIECES * BOXES);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + (uint32_t)(box * BOX_BYTES + row * ROW_BYTES + piece * 16)),
                         "r"(0u) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive<true>(leader_full + (uint32_t)(8 * s));
        }
      }
    }
  } else {
    if constexpr (S::FP8 && S::CTAS == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int store_warp = warp - FIRST_STORE_WARP, quarter = warp & 3;
    const int c0 = store_warp / 4 * S::WARP_COLS;  // first accumulator column of this warp
    const uint32_t lanes_at = (uint32_t)(quarter * 32) << 16;
    uint32_t made = 0, shared_tiles = 0;
    bool ok = true;
    auto wait_sums = [&](int buffer) {
      ok = mbar_wait(smem_u32(&bar_sums[buffer]), (made / S::BUFFERS) & 1u);
      ok = __all_sync(FULL, ok);
      if (!ok && lane == 0) gave_up();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return ok;
    };
    auto release_sums = [&](int buffer) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        const uint32_t bar = smem_u32(&bar_stored[buffer]);
        mbar_arrive(S::CTAS == 2 ? mapped(bar, 0) : bar);
      }
      ++made;
    };
    // 32 x 32 results of the warp go to rows of C by way of shared memory: four lanes store 64 adjacent bytes of a row.
    // Rows of 64 bytes, whose four pieces of 16 change places from row pair to row pair: eight rows' pieces lie in different banks.
    uint8_t *staged = staged_all + store_warp * 32 * 64;
    auto place = [](int row, int piece) { return row * 64 + ((piece ^ (row >> 1 & 3)) * 16); };
    // Bytes on whose boundary every row of C starts, up to 16.
    const uint32_t start = (uint32_t)p.cols * 2u | (uint32_t)reinterpret_cast<uintptr_t>(p.out);
    const int width = start % 16 == 0 ? 16 : start % 8 == 0 ? 8 : 2;
    auto lay_down = [&](const uint32_t (&w)[16]) {  // the lane's row
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4 *>(staged + place(lane, i)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    };
    auto store_block = [&](uint16_t *out, int row0, int rows_end, int col0) {
      __syncwarp();
      if (width == 16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + lane / 4, piece = lane % 4;
          const uint4 v = *reinterpret_cast<const uint4 *>(staged + place(r, piece));
          if (row0 + r < rows_end && col0 + piece * 8 < p.cols)
            *reinterpret_cast<uint4 *>(out + (int64_t)(row0 + r) * p.cols + col0 + piece * 8) = v;
        }
      } else if (width == 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + lane / 8, piece = lane % 8;
          const uint2 v = *reinterpret_cast<const uint2 *>(staged + place(r, piece / 2) + piece % 2 * 8);
          if (row0 + r < rows_end && col0 + piece * 4 < p.cols)
            *reinterpret_cast<uint2 *>(out + (int64_t)(row0 + r) * p.cols + col0 + piece * 4) = v;
        }
      } else if (col0 + lane < p.cols) {
        // Rows on no 8-byte boundary.  (Four bytes at a time where rows allow it: no change.  Eight at a time 23.8 us for 21.6, pairs of columns 32: 3,001 rows, 7 groups, 1111 x 777.)
        const int count = rows_end - row0 < 32 ? rows_end - row0 : 32;
        for (int r = 0; r < count; ++r)
          out[(int64_t)(row0 + r) * p.cols + col0 + lane] = *reinterpret_cast<const uint16_t *>(staged + place(r, lane / 8) + lane % 8 * 2);
      }
    };
    for (int turn = 0; ok && turn < rounds; ++turn) {
      const int t = tiles.of_round(turn);
      if (t >= tiles.total) continue;
      const Tile tile = tiles.at(t, p, part, parts);
      if constexpr (S::INNER) {
        const int buffer = (int)(made % S::BUFFERS);
        const bool empty = tile.k_blocks == 0;  // a group without rows: zeros
        if (!empty && !wait_sums(buffer)) break;
        uint16_t *out = p.out + (int64_t)tile.group * p.inner * p.cols;
        const int c_end = tile.n < c0 + S::WARP_COLS ? tile.n : c0 + S::WARP_COLS;
        if (!empty && c0 >= tile.n) release_sums(buffer);
        for (int c = c0; c < c_end; c += 32) {
          uint32_t v[32], w[16];
          if (!empty) {
            tmem_load(v, tmem + lanes_at + (uint32_t)(buffer * S::TILE + c));
            tmem_wait_loads();
            if (c + 32 >= c_end) release_sums(buffer);
          }
          if constexpr (S::SHARED) {
            const int row = tile.row0 + rank * LANES + quarter * 32 + lane;
            float *to = p.partials + ((int64_t)tile.group * p.inner + row) * p.pitch + tile.col0 + c;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (row < tile.row0 + tile.valid && tile.col0 + c + i < p.pitch)
                *reinterpret_cast<uint4 *>(to + i) = empty ? make_uint4(0, 0, 0, 0) : make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              w[i] = empty ? 0u : rounded_two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), p.half_out);
            lay_down(w);
            store_block(out, tile.row0 + rank * LANES + quarter * 32, tile.row0 + tile.valid, tile.col0 + c);
          }
        }
        continue;
      }
      if constexpr (S::FP8 && S::ROWS_ON_LANES) {
        const int row = tile.row0 + rank * LANES + quarter * 32 + lane, rows_end = tile.row0 + tile.valid;
        const int used = tile.n - c0;  // accumulator columns of this warp that are computed
        uint64_t sum[S::WARP_COLS / 2];
#pragma unroll
        for (int i = 0; i < S::WARP_COLS / 2; ++i) sum[i] = 0;
        // The scales of two blocks at a time, asked for two blocks ahead (four: 1 % slower).  Loads of places that exist, whatever the
        // lane's row: behind a condition each would wait for the one before (eight loads some 7,000 clocks).
        constexpr int AHEAD = 2;
        float scale[AHEAD], next_a[AHEAD], next_b[AHEAD];
        const float *a_scale = p.a_scales + (row < rows_end ? row : tile.row0);
        const float *b_scale = p.b_scales + tile.group * p.scale_group +
                               (int64_t)((tile.col0 + (used > 0 ? c0 : 0)) / 128) * p.scale_j;
        auto fetch = [&](int kb) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const int64_t block = kb + i < tile.k_blocks ? kb + i : tile.k_blocks - 1;
            next_a[i] = load_here(a_scale + block * p.rows);
            next_b[i] = load_here(b_scale + block * p.scale_k);
          }
        };
        fetch(0);
        for (int k0 = 0; ok && k0 < tile.k_blocks; k0 += AHEAD) {
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) scale[i] = next_a[i] * next_b[i];
          fetch(k0 + AHEAD);
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            if (k0 + k >= tile.k_blocks) break;
            const int buffer = (int)(made % S::BUFFERS);
            if (!wait_sums(buffer)) break;
            const uint32_t at = tmem + lanes_at + (uint32_t)(buffer * S::TILE + c0);
            const uint64_t f = pack(__float_as_uint(scale[k]), __float_as_uint(scale[k]));
            uint32_t v[2][32];  // 64 columns are loaded at a time
            if (used > 0) tmem_load(v[0], at);
            if (used > 32) tmem_load(v[1], at + 32u);
#pragma unroll
            for (int c = 0; c < S::WARP_COLS; c += 32) {
              uint32_t (&now)[32] = v[c / 32 % 2];
              if (c % 64 == 0) tmem_wait_loads();
              if (c == 64) release_sums(buffer);
              if (c < used) {
#pragma unroll
                for (int i = 0; i < 32; i += 2) sum[(c + i) / 2] = fma_two(pack(now[i], now[i + 1]), f, sum[(c + i) / 2]);
              }
              if (c < 64 && c + 64 < used) tmem_load(now, at + (uint32_t)(c + 64));
            }
          }
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < S::WARP_COLS; c += 32) {
          if (tile.col0 + c0 + c >= p.cols) break;
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            uint32_t lo, hi;
            unpack(sum[c / 2 + i], lo, hi);
            w[i] = rounded_two(__uint_as_float(lo), __uint_as_float(hi), false);
          }
          lay_down(w);
          store_block(p.out, tile.row0 + rank * LANES + quarter * 32, rows_end, tile.col0 + c0 + c);
        }
        continue;
      }
      const int col = tile.col0 + (S::CTAS == 2 ? rank * LANES : 0) + quarter * 32 + lane;
      const bool stores = col < p.cols;
      uint16_t *out = p.out + (int64_t)tile.row0 * p.cols + col;
      if constexpr (S::ROWS_ON_LANES) {
      } else if constexpr (!S::FP8) {
        const int buffer = (int)(made % S::BUFFERS);
        if (!wait_sums(buffer)) break;
        const bool split = S::SPLITS && parts > 1;
        if (S::SPLITS && split && shared_tiles > 0) {  // the sums of the tile before have been read
          ok = __all_sync(FULL, mbar_wait<true>(smem_u32(&bar_added), (shared_tiles - 1) & 1u));
          if (!ok) {
            if (lane == 0) gave_up();
            break;
          }
        }
        const int c_end = tile.valid < c0 + S::WARP_COLS ? tile.valid : c0 + S::WARP_COLS;
        if (c0 >= tile.valid) release_sums(buffer);
        for (int c = c0; c < c_end; c += 32) {
          const uint32_t at = tmem + lanes_at + (uint32_t)(buffer * S::TILE + c);
          if (split) {
            uint32_t v[32];
            tmem_load(v, at);
            tmem_wait_loads();
            if (c + 32 >= c_end) release_sums(buffer);
#pragma unroll
            for (int i = 0; i < 32; ++i) partial[(c + i) * LANES + quarter * 32 + lane] = __uint_as_float(v[i]);
            continue;
          }
          // 16 lanes x 32 columns each: blocks of 8 lanes (columns of C) x 8 columns (rows of C) as the warp-level MMAs hold them,
          // two rows of C to a register, which stmatrix lays down transposed
          uint32_t v[2][16];
          tmem_load_blocks(v[0], at);
          tmem_load_blocks(v[1], at + (16u << 16));
          tmem_wait_loads();
          if (c + 32 >= c_end) release_sums(buffer);
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              uint32_t w[4];
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const int r = 4 * (i + m / 2) + 2 * (m % 2);
                w[m] = rounded_two(__uint_as_float(v[h][r]), __uint_as_float(v[h][r + 1]), p.half_out);
              }
              const int m = lane / 8;
              const uint32_t to = smem_u32(staged) + (uint32_t)place(8 * (i + m / 2) + lane % 8, h * 2 + m % 2);
              asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[0]), "r"(w[1]),
                           "r"(w[2]), "r"(w[3]) : "memory");
            }
          store_block(p.out, tile.row0 + c, tile.row0 + tile.valid, tile.col0 + (S::CTAS == 2 ? rank * LANES : 0) + quarter * 32);
        }
      } else {
        uint64_t sum[S::WARP_COLS / 2];
#pragma unroll
        for (int i = 0; i < S::WARP_COLS / 2; ++i) sum[i] = 0;
        float *mine = scales + store_warp * 4 * S::WARP_COLS;
        const float *b_scale = p.b_scales + tile.group * p.scale_group +
                               (int64_t)(tile.col0 / 128) * p.scale_j;
        constexpr int PER_LANE = S::WARP_COLS / 32, AHEAD = 4;
        float next_a[AHEAD][PER_LANE], next_b[AHEAD];
        auto fetch = [&](int kb) {  // four blocks' scales, of rows that exist (see above)
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) {
            const int64_t block = tile.k0 + (kb + j < tile.k_blocks ? kb + j : tile.k_blocks - 1);
            next_b[j] = load_here(b_scale + block * p.scale_k);
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
              const int c = c0 + i * 32 + lane;
              next_a[j][i] = load_here(p.a_scales + block * p.rows + tile.row0 + (c < tile.valid ? c : 0));
            }
          }
        };
        if (tile.k_blocks > 0) fetch(0);
        for (int k4 = 0; ok && k4 < tile.k_blocks; k4 += AHEAD) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) mine[j * S::WARP_COLS + i * 32 + lane] = next_a[j][i] * next_b[j];
          __syncwarp();
          fetch(k4 + AHEAD);
          for (int k = 0; k < AHEAD && k4 + k < tile.k_blocks; ++k) {
            const float *here = mine + k * S::WARP_COLS;
            const int buffer = (int)(made % S::BUFFERS);
            if (!wait_sums(buffer)) break;
            // The loads of 32 columns run while those before are added.
            const uint32_t at = tmem + lanes_at + (uint32_t)(buffer * S::TILE + c0);
            uint32_t v[2][32];
            if (c0 < tile.valid) tmem_load(v[0], at);
#pragma unroll
            for (int c = 0; c < S::WARP_COLS; c += 32) {
              uint32_t (&now)[32] = v[c / 32 % 2];
              tmem_wait_loads();
              if (c + 32 < S::WARP_COLS && c0 + c + 32 < tile.valid) tmem_load(v[(c / 32 + 1) % 2], at + (uint32_t)(c + 32));
              if (c + 32 == S::WARP_COLS) release_sums(buffer);
              if (c0 + c < tile.valid) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(here + c + i);
                  sum[(c + i) / 2] = fma_two(pack(now[i], now[i + 1]), f.x, sum[(c + i) / 2]);
                  sum[(c + i) / 2 + 1] = fma_two(pack(now[i + 2], now[i + 3]), f.y, sum[(c + i) / 2 + 1]);
                }
              }
            }
          }
        }
        if (!ok) break;
        if (S::SPLITS && parts > 1) {
          if (shared_tiles > 0) {
            ok = __all_sync(FULL, mbar_wait<true>(smem_u32(&bar_added), (shared_tiles - 1) & 1u));
            if (!ok) {
              if (lane == 0) gave_up();
              break;
            }
          }
#pragma unroll
          for (int i = 0; i < S::WARP_COLS; i += 2) {
            uint32_t lo, hi;
            unpack(sum[i / 2], lo, hi);
            if (c0 + i >= tile.valid) break;
            partial[(c0 + i) * LANES + quarter * 32 + lane] = __uint_as_float(lo);
            partial[(c0 + i + 1) * LANES + quarter * 32 + lane] = __uint_as_float(hi);
          }
        } else if (stores) {
#pragma unroll
          for (int i = 0; i < S::WARP_COLS; i += 2) {
            uint32_t lo, hi;
            unpack(sum[i / 2], lo, hi);
            if (c0 + i < tile.valid) out[(int64_t)(c0 + i) * p.cols] = rounded(__uint_as_float(lo), false);
            if (c0 + i + 1 < tile.valid) out[(int64_t)(c0 + i + 1) * p.cols] = rounded(__uint_as_float(hi), false);
          }
        }
      }
      if constexpr (S::SPLITS) {
        if (parts > 1) {
          // Each CTA's sums lie in its shared memory; the CTAs of the cluster add every `parts`-th row of C, in rank order.
          __syncwarp();
          if (lane < parts) mbar_arrive<true>(mapped(smem_u32(&bar_parts), (uint32_t)lane));
          ok = __all_sync(FULL, mbar_wait<true>(smem_u32(&bar_parts), shared_tiles & 1u));
          if (!ok) {
            if (lane == 0) gave_up();
            break;
          }
          // Four columns of C a lane, so that the loads of a row of C are few and on their way together.
          const int col4 = tile.col0 + lane * 4;
          const bool fours = p.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 7u) == 0;
          for (int c = part + parts * store_warp; c < tile.valid; c += parts * S::STORE_WARPS) {
            const uint32_t at = smem_u32(partial) + (uint32_t)(c * LANES + lane * 4) * 4u;
            float v[8][4], total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (r < parts)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[r][0]), "=f"(v[r][1]), "=f"(v[r][2]), "=f"(v[r][3])
                             : "r"(mapped(at, (uint32_t)r)) : "memory");
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (r < parts)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[i] += v[r][i];
            uint16_t *to = p.out + (int64_t)(tile.row0 + c) * p.cols + col4;
            if (fours) {
              if (col4 < p.cols)
                *reinterpret_cast<uint2 *>(to) = make_uint2(rounded_two(total[0], total[1], p.half_out), rounded_two(total[2], total[3], p.half_out));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (col4 + i < p.cols) to[i] = rounded(total[i], p.half_out);
            }
          }
          __syncwarp();
          if (lane < parts) mbar_arrive<true>(mapped(smem_u32(&bar_added), (uint32_t)lane));
          ++shared_tiles;
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (failed) {
    // A wait gave up with copies or MMAs possibly still in flight: give them a bounded time (1 ms) to land before the shared
    // memory and the TMEM columns go back to the SM.
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (S::CTAS == 2 || parts > 1)  // no CTA leaves while another may use its shared memory, barriers or TMEM
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) {
    if constexpr (S::CTAS == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
  }
}

int64_t element_size(int type) { return type == kBF16 || type == kF16 ? 2 : 1; }

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  return fn;
}

// `stack` matrices of `outer` rows of `inner` contiguous elements (rank 2 without a stack), `pitch` elements apart; boxes of 128
// swizzled bytes x box_rows.
bool make_map(CUtensorMap *map, const void *base, int type, int64_t inner, int64_t outer, int64_t stack, int64_t pitch,
              uint32_t box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t size = element_size(type);
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)stack};
  cuuint64_t strides[2] = {(cuuint64_t)pitch * size, (cuuint64_t)(pitch * outer) * size};
  cuuint32_t box[3] = {(cuuint32_t)(ROW_BYTES / size), box_rows, 1};
  cuuint32_t elem[3] = {1, 1, 1};
  const CUtensorMapDataType data = type == kBF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  return fn(map, data, stack > 0 ? 3 : 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int REALIGN_THREADS = 256, REALIGN_AHEAD = 4;

// Matrices on their way to rows on 16-byte boundaries.
struct Realigned {
  const uint8_t *from;
  uint8_t *to;
  int matrices;          // 0: they stay where they are
  int64_t rows;          // of a matrix; one without a stack goes in slices of `rows`, of which the last may have fewer
  int64_t all_rows;
  int64_t bytes, pitch;  // of a row; of a row of the copy
  bool by_group;         // matrix g is copied only if group g has rows
};

// 16 bytes where `wanted`, else zeros, without a branch: loads behind branches wait for one another.
__device__ __forceinline__ uint4 load_if(const uint8_t *p, bool wanted) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@q ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"(wanted ? 1 : 0));
  return v;
}
// Bytes shift ... shift + 16 of two adjacent vectors.
__device__ __forceinline__ uint4 shifted(const uint4 &low, const uint4 &high, int shift) {
  const uint32_t w[8] = {low.x, low.y, low.z, low.w, high.x, high.y, high.z, high.w};
  uint32_t u[7], v[5];
#pragma unroll
  for (int i = 0; i < 7; ++i) u[i] = shift & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = shift & 8 ? u[i + 2] : u[i];
  const uint32_t bits = (uint32_t)(shift & 3) * 8;
  return make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits), __funnelshift_r(v[2], v[3], bits),
                    __funnelshift_r(v[3], v[4], bits));
}

// The blocks of a y copy a matrix: first those of a, then those of b.  A warp copies a row, 16 bytes of the copy a lane: the aligned
// vectors that hold them, shifted into place.  The first and the last bytes of the matrices, whose vectors reach over them, go byte by
// byte.  What lies behind a row's last byte in the copy is not its own (copies by TMA end there).
__global__ void __launch_bounds__(REALIGN_THREADS) realign_kernel(const Realigned a, const Realigned b, const int32_t *offsets, int rows) {
  after_previous_kernel();
  const Realigned &m = (int)blockIdx.y < a.matrices ? a : b;
  const int matrix = (int)blockIdx.y - ((int)blockIdx.y < a.matrices ? 0 : a.matrices);
  if (m.by_group) {
    const RowSpan span = group_rows(offsets, matrix, rows);
    if (span.begin == span.end) return;
  }
  const int lane = threadIdx.x % 32;
  const uint8_t *begin = m.from, *end = m.from + m.all_rows * m.bytes;
  const int64_t pieces = (m.bytes + 15) / 16, step = (int64_t)gridDim.x * (REALIGN_THREADS / 32);
  for (int64_t r = (int64_t)blockIdx.x * (REALIGN_THREADS / 32) + threadIdx.x / 32; r < m.rows; r += step) {
    const int64_t row = matrix * m.rows + r;
    if (row >= m.all_rows) return;
    const uint8_t *from = m.from + row * m.bytes;
    const int shift = (int)(reinterpret_cast<uintptr_t>(from) & 15u);
    uint4 *to = reinterpret_cast<uint4 *>(m.to + row * m.pitch);
    for (int64_t q0 = lane; q0 < pieces; q0 += 32 * REALIGN_AHEAD) {
      uint4 low[REALIGN_AHEAD], high[REALIGN_AHEAD];
#pragma unroll
      for (int u = 0; u < REALIGN_AHEAD; ++u) {
        const uint8_t *p = from + (q0 + 32 * u) * 16 - shift;
        const bool whole = q0 + 32 * u < pieces && p >= begin && p + 32 <= end;
        low[u] = load_if(p, whole);
        high[u] = load_if(p + 16, whole && shift != 0);
      }
#pragma unroll
      for (int u = 0; u < REALIGN_AHEAD; ++u) {
        const int64_t q = q0 + 32 * u;
        const uint8_t *p = from + q * 16;
        if (q >= pieces) break;
        if (p - shift >= begin && p - shift + 32 <= end) {
          to[q] = shift != 0 ? shifted(low[u], high[u], shift) : low[u];
        } else {
          for (int i = 0; i < 16 && q * 16 + i < m.bytes; ++i) reinterpret_cast<uint8_t *>(to + q)[i] = __ldg(p + i);
        }
      }
    }
  }
}

// Rows of the groups as zeros, for an inner axis without elements.
__global__ void __launch_bounds__(256) zero_rows_kernel(uint16_t *out, const int32_t *offsets, int groups, int rows, int64_t cols) {
  after_previous_kernel();
  bool decreasing = false;
  for (int g = threadIdx.x; g < groups; g += 256) decreasing |= group_rows(offsets, g, rows).decreasing;
  if (__syncthreads_or(decreasing)) return;
  for (int g = 0; g < groups; ++g) {
    const RowSpan span = group_rows(offsets, g, rows);
    for (int64_t i = (int64_t)span.begin * cols + blockIdx.x * 256 + threadIdx.x; i < span.end * cols; i += (int64_t)gridDim.x * 256) out[i] = 0;
  }
}

// Sums of the parts of a group's rows, in the order of the rows, rounded once.
__global__ void __launch_bounds__(256) add_partials_kernel(const float *partials, uint16_t *out, int groups, int splits, int rows, int cols,
                                                           int64_t pitch, bool half_out) {
  after_previous_kernel();
  const int64_t all = (int64_t)groups * rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t line = i / cols, group = line / rows;
    const float *from = partials + ((group * splits) * rows + (line - group * rows)) * pitch + (i - line * cols);
    float sum = 0.0f;
    for (int s = 0; s < splits; ++s) sum += __ldg(from + (int64_t)s * rows * pitch);
    out[i] = rounded(sum, half_out);
  }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Both operands as TMA can copy them: in place, or in memory of the stream-ordered pool that `release` gives back.
struct Operands {
  const void *a, *b;
  int64_t a_pitch, b_pitch;  // elements
  void *memory = nullptr;

  // a: a_rows x a_cols; b: stack matrices of b_rows x b_cols, of which a call uses those of groups with rows (stack 0: one, all of it)
  cudaError_t align(const void *a_, int64_t a_rows, int64_t a_cols, const void *b_, int64_t stack, int64_t b_rows, int64_t b_cols,
                    int64_t size, const int32_t *offsets, int64_t rows, const DeviceInfo &dev, cudaMemPool_t pool, cudaStream_t s,
                    int64_t *launches) {
    a = a_;
    b = b_;
    a_pitch = a_cols;
    b_pitch = b_cols;
    const bool move_a = !aligned16(a) || a_cols * size % 16 != 0, move_b = !aligned16(b) || b_cols * size % 16 != 0;
    if (!move_a && !move_b) return cudaSuccess;
    const int64_t a_row = copy_pitch(a_cols * size), b_row = copy_pitch(b_cols * size);
    auto slices = [](int64_t all) { return (int)ceil_div(all, slice_rows(all)); };
    static_assert(2 * kMostSlices <= kMaxGridY && kMostSlices + kMaxGroups <= kMaxGridY, "");
    const int64_t b_all = (stack > 0 ? stack : 1) * b_rows;
    const int64_t a_bytes = move_a ? ceil_div(a_rows * a_row, 128) * 128 : 0, b_bytes = move_b ? b_all * b_row : 0;
    cudaError_t e = cudaMallocFromPoolAsync(&memory, (size_t)(a_bytes + b_bytes), pool, s);
    if (e != cudaSuccess) return e;
    Realigned ra = {}, rb = {};
    if (move_a) {
      ra = {static_cast<const uint8_t *>(a_), static_cast<uint8_t *>(memory), slices(a_rows), slice_rows(a_rows), a_rows, a_cols * size,
            a_row, false};
      a = ra.to;
      a_pitch = ra.pitch / size;
    }
    if (move_b) {
      rb = {static_cast<const uint8_t *>(b_), static_cast<uint8_t *>(memory) + a_bytes, stack > 0 ? (int)stack : slices(b_rows),
            stack > 0 ? b_rows : slice_rows(b_rows), b_all, b_cols * size, b_row, stack > 0 && offsets};
      b = rb.to;
      b_pitch = rb.pitch / size;
    }
    ++*launches;
    // Blocks for a row a warp, up to 32 per SM in all, but 64 for a matrix in any case: of many groups few may have rows.
    const int matrices = ra.matrices + rb.matrices;
    const int64_t rows_most = ra.rows > rb.rows ? ra.rows : rb.rows, blocks = ceil_div(rows_most, REALIGN_THREADS / 32);
    const int64_t share = 32 * (int64_t)dev.sm_count / matrices, most = share > 64 ? share : 64;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks < most ? blocks : most), (unsigned)matrices);
    cfg.blockDim = dim3(REALIGN_THREADS);
    cfg.stream = s;
    cfg.attrs = attribute;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, realign_kernel, ra, rb, offsets, (int)rows);
  }
  cudaError_t release(cudaStream_t s, cudaError_t e) {
    const cudaError_t freed = memory ? cudaFreeAsync(memory, s) : cudaSuccess;
    return e != cudaSuccess ? e : freed;
  }
};

// Opts a kernel into its shared memory, once per device; racing threads repeat an idempotent call.
template <class S>
cudaError_t configure() {
  static std::atomic<bool> configured[64];
  int device = 0;
  cudaGetDevice(&device);
  if (device >= 0 && device < 64 && configured[device].load(std::memory_order_acquire)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(grouped_tcgen05_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e == cudaSuccess && device >= 0 && device < 64) configured[device].store(true, std::memory_order_release);
  return e;
}

// A launch of `clusters` clusters of `cluster` CTAs, set up while the kernel before it drains.
template <class S>
struct LaunchShape {
  cudaLaunchAttribute attributes[2];
  cudaLaunchConfig_t cfg = {};

  LaunchShape(int64_t clusters, int cluster, cudaStream_t s) {
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned)cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(clusters * cluster));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cfg.attrs = attributes;
    cfg.numAttrs = 2;
  }
};

// Clusters of a size that run at a time (on 148 SMs 74 of two, 33 of four, 15 of eight): asked once per device.
template <class S>
int resident_clusters(int cluster, const DeviceInfo &dev) {
  static std::atomic<int> known[64][9];
  int device = 0, n = 0;
  cudaGetDevice(&device);
  const bool keep = device >= 0 && device < 64 && cluster <= 8;
  if (keep && (n = known[device][cluster].load(std::memory_order_acquire)) > 0) return n;
  if (configure<S>() != cudaSuccess) return 1;  // the launch reports it
  LaunchShape<S> shape(dev.sm_count, cluster, nullptr);
  if (cudaOccupancyMaxActiveClusters(&n, grouped_tcgen05_kernel<S>, &shape.cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return dev.sm_count / cluster > 0 ? dev.sm_count / cluster : 1;
  }
  if (keep) known[device][cluster].store(n, std::memory_order_release);
  return n;
}

template <class S>
cudaError_t launch(const CUtensorMap &map_l, const CUtensorMap &map_t, Product p, int64_t most_tiles, int parts, const DeviceInfo &dev,
                   cudaStream_t s) {
  if (most_tiles == 0) return cudaSuccess;
  if (most_tiles > MOST_TILES) return cudaErrorInvalidConfiguration;
  cudaError_t e = configure<S>();
  if (e != cudaSuccess) return e;
  p.col_tiles = (int)ceil_div(p.cols, LANES * S::CTAS);
  const int64_t inner_tiles = ceil_div(p.inner, S::TILE);
  if (8LL * p.col_tiles > 2147483647LL || (S::INNER && p.col_tiles * inner_tiles > 2147483647LL)) return cudaErrorInvalidConfiguration;
  p.per_band = Divisor::of(8u * (uint32_t)p.col_tiles);
  if (S::INNER) {
    p.per_group = Divisor::of((uint32_t)(p.col_tiles * inner_tiles));
    p.per_column = Divisor::of((uint32_t)inner_tiles);
  }
  const int cluster = S::CTAS == 2 ? 2 : parts;
  const int64_t resident = resident_clusters<S>(cluster, dev);
  // In the order of their work tiles are dealt more evenly (1,999 rows, 12 groups, a third of them empty, 1032 x 520, dA and dB:
  // 24.2 us as they come, 23.1 by work; 16,384 rows, 32 groups of 189 to 2426, 2048 x 1536, dA and dB 220.0 and 219.1; 64 groups
  // forward 127.1 and 126.7).
  // The order costs each CTA some 400 clocks: where walkers take one tile or two it stays as it comes.
  p.sorted = p.groups > 1 && p.groups <= S::MOST_SORTED && most_tiles > 2 * resident && !S::SHARED;
  LaunchShape<S> shape(most_tiles < resident ? most_tiles : resident, cluster, s);
  return cudaLaunchKernelEx(&shape.cfg, grouped_tcgen05_kernel<S>, map_l, map_t, p, parts);
}

// kind::f16 and kind::f8f6f4: f32 sums (bits 4-5), types of A and B (bits 7-9, 10-12), MN-major A and B (bits 15, 16),
// N >> 3 (bits 17-22, per tile), M >> 4 (bits 24-28).
uint32_t instruction_descriptor(int a_type, int b_type, bool a_mn, bool b_mn, int m) {
  auto code = [](int type) { return type == kBF16 || type == kE5M2 ? 1u : 0u; };
  return (1u << 4) | (code(a_type) << 7) | (code(b_type) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(m >> 4) << 24);
}

template <int CTAS, int TILE, bool FP8, bool MN>
cudaError_t launch_rows(const GroupedArgs &a, const Operands &from, Product p, int parts, const DeviceInfo &dev, cudaStream_t s) {
  using S = Config<CTAS, TILE, FP8, MN, false>;
  CUtensorMap map_l, map_t;
  const int b_type = FP8 ? a.b_type : a.type;
  // (rows on the lanes: boxes of 128 rows or columns of either operand)
  const bool made = (MN ? make_map(&map_l, from.b, b_type, a.n, a.inner, a.groups, from.b_pitch, S::STEP)
                        : make_map(&map_l, from.b, b_type, a.inner, a.n, a.groups, from.b_pitch, LANES)) &&
                    make_map(&map_t, from.a, a.type, a.inner, a.rows, 0, from.a_pitch, S::ROW_BOX);
  if (!made) return cudaErrorInvalidValue;
  p.instruction = S::ROWS_ON_LANES ? instruction_descriptor(a.type, b_type, false, MN, LANES * CTAS)
                                   : instruction_descriptor(b_type, a.type, MN, false, LANES * CTAS);
  const int64_t most = (ceil_div(a.rows, TILE) + (a.groups < a.rows ? a.groups : a.rows)) * ceil_div(a.n, LANES * CTAS);
  return launch<S>(map_l, map_t, p, most, parts, dev, s);
}

// Which tiles, and how many CTAs share a tile's inner axis: what the host knows are the sizes, so it takes the rows to be dealt evenly
// to as many groups as can have some, and compares times in us as measured (2048 x 1536, 1 to 64 groups of 8 to 512 rows), each
// rounds x (stages of a CTA x time of one + what a tile costs beside them) + the launch:
//   narrow   a stage 0.23 + 0.0006 per row (8 bits 0.45 + 0.0015), a tile 0.5, shared 1.6 + 0.024 per row, the launch 3.3;
//   wide     a stage 0.095 + 0.00075 per row, at least 0.155 (8 bits 0.48), a tile 1.0, the launch 5.
// us narrow (64 rows), narrow (128) and wide, measured: one group of 8 rows 6.2, -, 9.7; of 96 -, 8.3, 10.4; of 512 39, 26, 14.8;
// 8 groups of 32 12.0, -, 10.6; of 96 20.9, 13.9, 11.9; 64 of 8 69.4, -, 69.8; of 128 100, 87, 80.
struct Plan {
  int tile = 0;  // rows; 256: wide
  int parts = 1;
  double us = 1e30;
};

template <class S>
void consider(Plan *best, const GroupedArgs &a, const DeviceInfo &dev) {
  const int64_t active = a.groups < a.rows ? a.groups : a.rows, mean = ceil_div(a.rows, active);
  const int64_t row_tiles = ceil_div(mean, S::TILE), tiles = active * row_tiles * ceil_div(a.n, LANES * S::CTAS);
  const int64_t stages = ceil_div(a.inner, S::STEP);
  const double rows = (double)mean / (double)row_tiles;
  for (int parts = 1; parts <= (S::SPLITS ? 8 : 1) && parts <= stages; ++parts) {
    const int64_t rounds = ceil_div(tiles, resident_clusters<S>(S::CTAS == 2 ? 2 : parts, dev));
    double stage, tile, launch;
    if (S::CTAS == 2) {
      stage = S::FP8 ? 0.48 : 0.095 + 0.00075 * rows > 0.155 ? 0.095 + 0.00075 * rows : 0.155;
      tile = 1.0;
      launch = 5.0;
    } else {
      stage = S::FP8 ? 0.45 + 0.0015 * rows : 0.23 + 0.0006 * rows;
      tile = parts > 1 ? 1.6 + 0.024 * rows : 0.5;
      launch = 3.3;
    }
    const double us = (double)rounds * ((double)ceil_div(stages, parts) * stage + tile) + launch;
    if (us < best->us) *best = {S::TILE, parts, us};
  }
}

template <bool FP8, bool MN>
cudaError_t launch_best(const GroupedArgs &a, const Operands &from, const Product &p, const DeviceInfo &dev, cudaStream_t s) {
  Plan plan;
  consider<Config<2, 256, FP8, MN, false>>(&plan, a, dev);
  consider<Config<1, 64, FP8, MN, false>>(&plan, a, dev);
  if constexpr (!FP8) consider<Config<1, 128, FP8, MN, false>>(&plan, a, dev);
  if (plan.tile == 256) return launch_rows<2, 256, FP8, MN>(a, from, p, 1, dev, s);
  if constexpr (!FP8)
    if (plan.tile == 128) return launch_rows<1, 128, FP8, MN>(a, from, p, plan.parts, dev, s);
  return launch_rows<1, 64, FP8, MN>(a, from, p, plan.parts, dev, s);
}

}  // namespace

cudaError_t launch_grouped_rows_tcgen05(const GroupedArgs &a, int *status_flag, const DeviceInfo &dev, cudaMemPool_t pool,
                                        cudaStream_t s, int64_t *launches) {
  if (a.rows == 0) return cudaSuccess;
  if (a.inner == 0) {
    ++*launches;
    return launch_chained(zero_rows_kernel, (unsigned)dev.sm_count, 256, 0, s, static_cast<uint16_t *>(a.C), a.offsets, (int)a.groups,
                          (int)a.rows, a.n);
  }
  const bool fp8 = a.a_scales != nullptr;
  Operands from;
  cudaError_t e = from.align(a.A, a.rows, a.inner, a.B, a.groups, a.transpose_b ? a.n : a.inner, a.transpose_b ? a.inner : a.n,
                             fp8 ? 1 : 2, a.offsets, a.rows, dev, pool, s, launches);
  if (e != cudaSuccess) return from.release(s, e);
  ++*launches;
  Product p = {};
  p.rows = (int)a.rows;
  p.inner = (int)a.inner;
  p.cols = (int)a.n;
  p.groups = (int)a.groups;
  p.offsets = a.offsets;
  p.out = static_cast<uint16_t *>(a.C);
  p.half_out = !fp8 && a.type == kF16;
  p.a_scales = a.a_scales;
  p.b_scales = a.b_scales;
  const int64_t kb = ceil_div(a.inner, kScaleBlock), nb = ceil_div(a.n, kScaleBlock);
  p.scale_k = (int)(a.transpose_b ? 1 : nb);
  p.scale_j = (int)(a.transpose_b ? kb : 1);
  p.scale_group = kb * nb;
  p.status = status_flag;
  if (fp8) e = a.transpose_b ? launch_best<true, false>(a, from, p, dev, s) : launch_best<true, true>(a, from, p, dev, s);
  else e = a.transpose_b ? launch_best<false, false>(a, from, p, dev, s) : launch_best<false, true>(a, from, p, dev, s);
  return from.release(s, e);
}

cudaError_t launch_grouped_inner_tcgen05(const GroupedInnerArgs &a, int *status_flag, const DeviceInfo &dev, cudaMemPool_t pool,
                                         cudaStream_t s, int64_t *launches) {
  if (a.rows == 0) return cudaMemsetAsync(a.out, 0, (size_t)(a.groups * a.i_size * a.j_size) * 2, s);
  Operands from;
  cudaError_t e = from.align(a.left, a.rows, a.i_size, a.right, 0, a.rows, a.j_size, 2, nullptr, a.rows, dev, pool, s, launches);
  if (e != cudaSuccess) return from.release(s, e);
  ++*launches;
  using S = Config<2, 256, false, true, true>;
  CUtensorMap map_l, map_t;
  if (!make_map(&map_l, from.b, a.type, a.j_size, a.rows, 0, from.b_pitch, S::STEP) ||
      !make_map(&map_t, from.a, a.type, a.i_size, a.rows, 0, from.a_pitch, S::ROW_BOX))
    return from.release(s, cudaErrorInvalidValue);
  Product p = {};
  p.rows = (int)a.rows;
  p.inner = (int)a.i_size;
  p.cols = (int)a.j_size;
  p.groups = (int)a.groups;
  p.offsets = a.offsets;
  p.out = static_cast<uint16_t *>(a.out);
  p.half_out = a.type == kF16;
  p.status = status_flag;
  p.instruction = instruction_descriptor(a.type, a.type, true, true, LANES * 2);
  int64_t tiles = a.groups * ceil_div(a.i_size, S::TILE) * ceil_div(a.j_size, LANES * 2);
  // Where there are fewer tiles than pairs of CTAs, each group's rows are shared among several, whose f32 sums a second kernel adds:
  // as many as make rounds x (stages x 0.28 us + 1.5) plus 4 us and the sums' way through memory least (25,381 rows,
  // 1408 x 512: 118 us for one, 46 for six).
  const int64_t resident = resident_clusters<S>(2, dev), stages = ceil_div(ceil_div(a.rows, a.groups), S::STEP);
  int splits = 1;
  double best = 1e30;
  for (int n = 1; n <= 32 && n <= stages && (n == 1 || tiles * n <= resident); ++n) {
    const double bytes = n > 1 ? 8.0 * (double)n * (double)(a.groups * a.i_size) * (double)a.j_size : 0.0;
    const double us = (double)ceil_div(tiles * n, resident) * ((double)ceil_div(stages, n) * 0.28 + 1.5) + (n > 1 ? 4.0 + bytes / 5e6 : 0.0);
    if (us < best) {
      best = us;
      splits = n;
    }
  }
  void *partials = nullptr;
  p.splits = Divisor::of((uint32_t)splits);
  p.pitch = ceil_div(a.j_size, 4) * 4;
  if (splits > 1) {
    tiles *= splits;
    e = cudaMallocFromPoolAsync(&partials, (size_t)(a.groups * splits * a.i_size * p.pitch) * 4, pool, s);
    if (e != cudaSuccess) return from.release(s, e);
    p.partials = static_cast<float *>(partials);
  }
  e = splits > 1 ? launch<Config<2, 256, false, true, true, true>>(map_l, map_t, p, tiles, 1, dev, s)
                 : launch<S>(map_l, map_t, p, tiles, 1, dev, s);
  if (splits > 1) {
    if (e == cudaSuccess) {
      ++*launches;
      const int64_t blocks = ceil_div(a.groups * a.i_size * a.j_size, 256), most = 16 * (int64_t)dev.sm_count;
      e = launch_chained(add_partials_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, s, p.partials, p.out, p.groups, splits,
                         p.inner, p.cols, p.pitch, p.half_out);
    }
    const cudaError_t freed = cudaFreeAsync(partials, s);
    if (e == cudaSuccess) e = freed;
  }
  return from.release(s, e);
}

}  // namespace swb
