// Attention of prompt chunks over the 4-bit KV pool, on the 5th-generation tensor cores.
//
// A unit is one row, one kv head and a pair of query tiles; the 128 MMA rows of a tile pack
// (token, query head of the group) pairs, row m = token m / group, head m % group. One CTA
// per SM takes units in turn:
//   warps 0-7   a warpgroup for each query tile, a thread for each row: brings its query to
//               shared memory, then for every 128 keys reads its scores from TMEM, softmax
//               with a lazily moved reference, writes P over them; at the end O / l and LSE;
//   warps 8-11  turn K's codes of 8 blocks into fp16 and store them as the MMA's operand,
//   warps 12-15 V's;
//   warp 16     owns TMEM and issues S(t) = Q(t) K^T and O(t) += P(t) V, tile t's while the
//               other tile's softmax runs;
//   warp 17     copies the pool's rows of the next blocks to shared memory;
//   warp 18     finds the CTA's next units, or pieces of them, and says what they are.
// K is stored by keys, V by dims (V^T): both K-major, and both as the pool has them, so a
// word of 8 codes becomes one 16-byte store (V: of 4 pairs of tokens, 4 such stores).
// Registers are split between the roles (setmaxnreg); none may spill, with shared memory
// taking what would be L1.
//
// In a tile key 16 b + r of block b has place 16 b + (r ^ 4) where r >= 8: V's rows in shared
// memory are then read in an order that meets no bank twice.
//
// Rounding to 16 bits: a query to fp16 after a power of two of its own that puts its largest
// element at 2^14 (exact, see q4_attention.cu; the power is part of the row's scale); K and
// V values once to fp16 (unit 2^-11; clamped to +-65504), which is what a 16-bit pool would
// hold; P to fp16, below 2^15. Scores, O and all sums are fp32. One rounding of K costs a
// score about 2e-4 at unit scores, and LSE that over the root of the keys seen; units whose
// first token sees few keys take K as the sum of two fp16 numbers, one product for each.
//
// Bound: the two softmax warpgroups, 256 x 128 scores for every 128 keys: a maximum, an
// exponential at 16 a clock and SM, a rounding and two passes through TMEM; beside them the MMAs
// take 1.6 us of the 3.0 us that an SM spends on 128 keys of two query tiles (head_dim 128),
// and a unit's start and end, when the MMAs run dry, another 7. 16 rows of 512 tokens that see
// 2560 keys, 32/8 heads of 128, bf16: 462 us, 669 TFLOP/s; 1 row of 512 that sees 32,768: 715 TFLOP/s.
#include "q4_attention.cuh"
#include "seb_softmax.cuh"
#include "seb_tcgen05.cuh"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace seb {
namespace {

constexpr int kKeys = 128;     // keys of a K / V tile
constexpr int kRows = 128;     // rows of a query tile
constexpr int kTiles = 2;      // query tiles of a unit
constexpr int kStages = 2;     // K tiles, and V tiles, in shared memory
constexpr int kRawStages = 3;  // the pool's rows of K(0), V(0), K(1), ... before they are decoded
constexpr int kThreads = 640;  // 5 warpgroups; the last has the MMA warp, the copying one, the one that plans, an idle one
constexpr int kPieces = 4;     // places for what the planning warp says of pieces
constexpr int kTmemCols = 512;
constexpr int kColO = 256;     // S of tile t at 128 t (P over its first 64 columns), O at 256 + t * D
// The reference is put 2^7 below the largest score, and moved when one exceeds it by 2^15: P stays below fp16's
// 65504, and weights down to 2^-21 of the largest are not subnormal.
constexpr float kBelow = 7.f, kLazy = 15.f;
// Keys seen by a unit's first token from which on K is rounded once. 16 chunks of 512 over 2560 keys: LSE is
// off by 1.4e-6 of itself (2.4e-4 at most) in 448 us; with K in two parts for all by 5.7e-8 (1.8e-6 at most) in
// 762 us, and O, in bf16, by as much as before. Below 512 keys one rounding could leave LSE off by 1e-4 and more.
constexpr int kSplitBelow = 512;

template <int D>
struct Smem {
  static constexpr int kPanel = 128 * 128;      // 128 rows of 128 bytes
  static constexpr int kTile = D / 64 * kPanel;  // of Q, K or V^T
  static constexpr int oQ = 0;
  static constexpr int oK = oQ + kTiles * kTile;
  static constexpr int oV = oK + kStages * kTile;
  static constexpr int kRawRow = q4::Layout<D>::kRow + 16;  // 16 more: blocks start in different banks
  static constexpr int kRaw = 8 * kRawRow;                  // K or V rows of a tile's 8 blocks
  static constexpr int oRaw = oV + kStages * kTile;
  static constexpr int oBar = oRaw + kRawStages * kRaw;
  static constexpr int oInfo = oBar + 384;                  // TileInfo [4]
  static constexpr int oPieces = oInfo + 4 * 16;            // Unit [kPieces], 96 bytes each
  static constexpr int oNan = oPieces + kPieces * 96;       // int [kPieces][2]
  static constexpr int oPrefix = oNan + kPieces * 8;        // uint32 [kThreads + 1]
  static constexpr int oLongest = oPrefix + (kThreads + 1) * 4;            // uint32
  static constexpr int oMl = (oLongest + 4 + 7) / 8 * 8;    // float2 [2][kRows]
  static constexpr int kBytes = oMl + 2 * kRows * 8;
};

enum {
  kBarQFull = 0,                      // + tile: its 128 threads stored the unit's queries
  kBarKFull = kBarQFull + kTiles,     // + stage
  kBarKEmpty = kBarKFull + kStages,   // + stage: S of every tile has read K
  kBarVFull = kBarKEmpty + kStages,   // + stage
  kBarVEmpty = kBarVFull + kStages,   // + stage
  kBarSFull = kBarVEmpty + kStages,   // + tile: S(t, j) complete, and every MMA before it
  kBarPFull = kBarSFull + kTiles,     // + tile: P(t, j) stored
  kBarODone = kBarPFull + kTiles,     // + tile: the unit's last PV complete
  // + n % kRawStages for K's rows of tile n, and kRawStages on for V's: rows have come. A place holds K's and V's in
  // turn; whoever waits for one kind alone needs a barrier whose every phase is of that kind.
  kBarRawFull = kBarODone + kTiles,
  kBarRawEmpty = kBarRawFull + 2 * kRawStages,  // + place: the 128 threads that decode K, or V, are done with them
  kBarMerge = kBarRawEmpty + kRawStages,  // both warpgroups have come to this point of a unit that they share
  kBarPieceFull,                            // + place: a piece, or the end, is described there
  kBarPieceEmpty = kBarPieceFull + kPieces,  // + place: the copying, the MMA and the 8 softmax warps are done with it
  kBarFinal = kBarPieceEmpty + kPieces,
  kNumBars = kBarFinal + 1
};
static_assert(kNumBars * 8 + 8 <= 384, "barrier region");

// A unit, or a CTA's piece of it, as every role sees it.
struct Unit {
  int row;             // -1: there are no more
  int kvh, k_len, q_len;
  int64_t token;       // the first of the unit's tokens
  int tok0;            // and its place in the row
  int sees;            // keys that it sees; each later token sees one more (causal)
  int nblk, ntiles;    // blocks that some token sees, and tiles of 128 keys
  int tiles;           // query tiles, 1 or 2
  int j0, n;           // the piece: n key tiles from j0 on
  int tile0;           // key tiles of the CTA's pieces before it
  int slots;           // warpgroups that have some of it
  bool twin;           // one query tile, whose key tiles the two warpgroups take in turn
  bool start;          // the piece is the unit's first
  uint32_t first, last;  // CTAs with key tiles of the unit (0, 0 where units are not cut)
  bool split;          // K in two parts: a tile of keys takes two places of the ring
};

// What the copying warp says of a tile of keys.
struct TileInfo {
  int limit;      // its keys below this exist
  unsigned none;  // bit b: block b has no data
  int kind;       // kSplit, kDiag, or kEnd: no more tiles; and kPlace times its piece's place
  int key0;       // its first key
};
constexpr int kSplit = 1;  // K in two parts
// Some token does not see all of it. There a V that is NaN must not meet a weight of zero: it is taken as 0,
// and a group's first key of this kind is kept for the piece; whoever sees that key gets NaN in the group.
constexpr int kDiag = 2;
constexpr int kEnd = 4;
constexpr int kPlace = 8;

// Units are whole where there are at least as many as CTAs (each takes every so manieth).
// Fewer are laid end to end, kUnitPlaces places for a start and one for each key tile, and
// cut in equal runs, one for each CTA; what is left of a unit that was cut is joined by
// the last of its CTAs to come, in order of the parts' places. Measured, whole and cut (bf16,
// 32/8 heads of 128), with an earlier softmax: 1 row of 512 tokens that sees 32,768 keys 720 and 367 us
// (382 now), 1 of 64 and 131,072 keys 2776 and 221 (225 now); but 4 rows of 512 and 4096 keys (256 units)
// 206 and 227. A start, with a part's join, costs as much as 10 key tiles (48 rows of drafts: 3 places
// 205 us, 6 202, 10 196).
constexpr uint32_t kUnitPlaces = 10;
// Shortest run worth a CTA. One row of 64 tokens that sees 2000 / 4000 / 8000 keys, us: 4: 40.8 / 48.4 / 66.3;
// 8: 49.9 / 53.1 / 60.5; 12: 61.4 / 63.8 / 66.3; 20: 65.5 / 85.7 / 84.3. Where such a run would be as long as the
// longest unit, units stay whole (one row of 200 tokens and 400 keys: 64 us cut, 39 whole).
constexpr uint32_t kMinPlaces = 4;

__device__ __forceinline__ int pairs_of(const Q4Params& p, const Row& w) {
  return (w.q_len + kTiles * p.tile - 1) / (kTiles * p.tile);
}
// Blocks that some token of a row's pair of query tiles sees.
__device__ __forceinline__ int blocks_of(const Q4Params& p, const Row& w, int pair) {
  if (!p.causal) return (w.k_len + 15) >> 4;
  const int64_t past = (int64_t)w.q_pos + min((pair + 1) * kTiles * p.tile, w.q_len);
  return (int)((max(min(past, (int64_t)w.k_len), (int64_t)0) + 15) >> 4);
}
__device__ __forceinline__ uint32_t places_of(int blocks) { return (uint32_t)((blocks + 7) >> 3) + kUnitPlaces; }

// How all rows are shared out.
struct Plan {
  bool cut;            // units are cut
  uint32_t per;        // places of a CTA's run
  uint32_t pos, stop;  // the CTA's next unit or place, and where to stop
};
__device__ __forceinline__ uint32_t length_of(const Q4Params& p, const Row& w, bool cut) {
  const int pairs = pairs_of(p, w);
  if (!cut) return (uint32_t)pairs * p.hkv;
  uint32_t sum = 0;
#pragma unroll 1
  for (int i = 0; i < pairs; ++i) sum += places_of(blocks_of(p, w, i));
  return sum * p.hkv;
}

// The CTA's next unit, or piece of one; false past the last.
__device__ __forceinline__ bool next_piece(const Q4Params& p, const uint32_t* prefix, Plan& plan, Unit& w) {
  if (plan.pos >= plan.stop) return false;
  int lo = 0, hi = kThreads - 1;
#pragma unroll 1
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= plan.pos) lo = mid;
    else hi = mid - 1;
  }
  const int chunk = (p.num_rows + kThreads - 1) / kThreads;
  int r = lo * chunk;
  uint32_t off = plan.pos - prefix[lo], bad = 0;
  Row row = row_of<true>(p, r, &bad);
  uint32_t len = length_of(p, row, plan.cut);
#pragma unroll 1
  while (off >= len && r + 1 < p.num_rows) {
    off -= len;
    row = row_of<true>(p, ++r, &bad);
    len = length_of(p, row, plan.cut);
  }
  if (off >= len) return false;
  int pr = pairs_of(p, row) - 1;  // a row's last tokens first: they see the most keys
  uint32_t place = 0;
  if (plan.cut) {
#pragma unroll 1
    for (;; --pr) {
      len = places_of(blocks_of(p, row, pr));
      if (off < len * p.hkv || pr == 0) break;
      off -= len * p.hkv;
    }
    w.kvh = off / len;
    place = off - w.kvh * len;
  } else {
    pr -= off / p.hkv;
    w.kvh = off % p.hkv;
  }
  w.row = r;
  w.k_len = row.k_len;
  w.q_len = row.q_len;
  w.tok0 = pr * kTiles * p.tile;
  w.token = (int64_t)row.q_start + w.tok0;
  w.sees = p.causal ? (int)min((int64_t)row.q_pos + w.tok0 + 1, (int64_t)(1 << 30)) : row.k_len;
  w.tiles = min(kTiles * p.tile, row.q_len - w.tok0) > p.tile ? 2 : 1;
  w.split = w.sees < kSplitBelow;
  w.nblk = blocks_of(p, row, pr);
  w.ntiles = (w.nblk + 7) >> 3;
  w.start = place == 0;
  w.first = w.last = 0;
  if (plan.cut) {
    const uint32_t n = min(len - place, plan.stop - plan.pos), at = plan.pos - place;
    w.j0 = max((int)(place - kUnitPlaces), 0);
    w.n = max((int)(place + n - kUnitPlaces), 0) - w.j0;
    w.first = (at + kUnitPlaces) / plan.per;
    w.last = (at + len - 1) / plan.per;
    plan.pos += n;
  } else {
    w.j0 = 0;
    w.n = w.ntiles;
    plan.pos += gridDim.x;
  }
  w.twin = w.tiles == 1 && w.n > 1;
  w.slots = w.n == 0 ? 0 : w.twin ? 2 : w.tiles;
  return true;
}

// 8 codes of a word, two of each 16 bits (lowest first), times s plus l.
template <bool CLAMP>
__device__ __forceinline__ void decode8(uint32_t w, __half2 s, __half2 l, uint32_t (&v)[4]) {
  const __half2 k1024 = __half2half2(__ushort_as_half(0x6400));
  const __half2 k16th = __half2half2(__ushort_as_half(0x2c00)), k64 = __half2half2(__ushort_as_half(0xd400));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // 1024 + n and 1024 + 16 n
    const uint32_t a = (w & 0x000f000fu) | 0x64006400u, b = (w & 0x00f000f0u) | 0x64006400u;
    const __half2 na = __hsub2(*reinterpret_cast<const __half2*>(&a), k1024);
    const __half2 nb = __hfma2(*reinterpret_cast<const __half2*>(&b), k16th, k64);
    __half2 x = __hfma2(na, s, l), y = __hfma2(nb, s, l);
    if constexpr (CLAMP) {
      const __half2 top = __half2half2(__ushort_as_half(0x7bff));
      x = __hmax2_nan(__hmin2_nan(x, top), __hneg2(top));
      y = __hmax2_nan(__hmin2_nan(y, top), __hneg2(top));
    }
    v[2 * h] = *reinterpret_cast<const uint32_t*>(&x);
    v[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&y);
    w >>= 8;
  }
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ bool is_nan_pair(uint32_t x) { return (x & 0x7fffu) > 0x7c00u; }  // the scale decides
// Whether a group with this (scale, low), or the elementwise largest of several, may pass 65504.
__device__ __forceinline__ bool may_overflow(__half2 most) {
  return __hgt(__low2half(most), __ushort_as_half(0x6800)) || __hgt(__high2half(most), __ushort_as_half(0x7800));
}

// Registers of the warpgroup's threads.
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// True in one lane of a converged warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}
// Of the 96 that a thread has at the launch. No role spills: 16 bytes of it took 16 chunks of 512 tokens, heads
// of 128, from 453 to 483 us; heads of 64 with the other's split, 8 bytes, 383 instead of 372.
template <int D>
struct Regs {
  static constexpr int kSoftmax = D == 64 ? 128 : 120, kK = D == 64 ? 72 : 80, kV = 80, kMma = D == 64 ? 72 : 80;
  static_assert(2 * kSoftmax + kK + kV + kMma <= 5 * 96, "the roles' registers are those of the launch");
};
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) q4_prefill_kernel(const Q4Params p) {
  using S = Smem<D>;
  using L = q4::Layout<D>;
  constexpr int G = L::kGroups;
  static_assert(L::kPanels == 1, "head_dim 64 or 128");
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  char* sbase = smem_raw + (base - raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar = base + S::oBar;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sbase + S::oBar + 8 * kNumBars);
  TileInfo* info = reinterpret_cast<TileInfo*>(sbase + S::oInfo);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(sbase + S::oPrefix);
  Unit* pieces = reinterpret_cast<Unit*>(sbase + S::oPieces);
  int* nans = reinterpret_cast<int*>(sbase + S::oNan);
  static_assert(sizeof(Unit) <= 96, "room for pieces");

  // ---- the rows' units, and where there are few their places; errors in rows are reported by
  // the kernel for the other rows
  Plan plan;
  uint32_t units = 0;  // of the rows up to this thread's
  uint32_t* longest = reinterpret_cast<uint32_t*>(sbase + S::oLongest);
  if (tid == 0) *longest = 0;
#pragma unroll 1
  for (int cut = 0; cut < 2; ++cut) {
    const int chunk = (p.num_rows + kThreads - 1) / kThreads;
    uint32_t sum = 0, bad = 0;
#pragma unroll 1
    for (int r = tid * chunk; r < min((tid + 1) * chunk, p.num_rows); ++r) {
      const Row row = row_of<true>(p, r, &bad);
      sum += length_of(p, row, cut);
      if (!cut) sum = min(sum, 1u << 22);  // rows whose tokens overlap: 640 such sums still fit 32 bits
      if (cut && row.q_len > 0) atomicMax(longest, places_of(blocks_of(p, row, pairs_of(p, row) - 1)));
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(kFull, sum, off);
      if (lane >= off) sum += o;
    }
    prefix[tid + 1] = sum;
    if (tid == 0) prefix[0] = 0;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll 1
    for (int w = 0; w < warp; ++w) before += prefix[(w + 1) * 32];
    __syncthreads();
    prefix[tid + 1] += before;
    __syncthreads();
    const uint32_t total = prefix[kThreads];
    plan.cut = cut;
    plan.per = cut ? max((total + gridDim.x - 1) / gridDim.x, kMinPlaces) : 1;
    plan.pos = blockIdx.x * plan.per;
    plan.stop = cut ? min(plan.pos + plan.per, total) : total;
    if (cut == 0) {
      units = prefix[tid + 1];
      if (total == 0 || total >= p.cut_below) break;
      __syncthreads();
    } else if (plan.per >= *longest) {  // a CTA for each unit is done sooner
      __syncthreads();
      prefix[tid + 1] = units;
      __syncthreads();
      plan = Plan{false, 1, blockIdx.x, prefix[kThreads]};
    }
  }
  if (plan.pos >= plan.stop) return;

  if (tid == 0) {
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(bar + 8 * (kBarQFull + t), 128);
      mbar_init(bar + 8 * (kBarSFull + t), 1);
      mbar_init(bar + 8 * (kBarPFull + t), 4);
      mbar_init(bar + 8 * (kBarODone + t), 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar + 8 * (kBarKFull + s), 128);
      mbar_init(bar + 8 * (kBarKEmpty + s), 1);
      mbar_init(bar + 8 * (kBarVFull + s), 128);
      mbar_init(bar + 8 * (kBarVEmpty + s), 1);
    }
    for (int s = 0; s < kRawStages; ++s) {
      mbar_init(bar + 8 * (kBarRawFull + s), 1);
      mbar_init(bar + 8 * (kBarRawFull + kRawStages + s), 1);
      mbar_init(bar + 8 * (kBarRawEmpty + s), 128);
    }
    for (int s = 0; s < kPieces; ++s) {
      mbar_init(bar + 8 * (kBarPieceFull + s), 1);
      mbar_init(bar + 8 * (kBarPieceEmpty + s), 10);
    }
    mbar_init(bar + 8 * kBarMerge, 8);
    mbar_init(bar + 8 * kBarFinal, 1);
    fence_mbar_init();
  }
  if (warp == 16) {
    tc::tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  bool failed = false;

  // The CTA's i-th piece, and word that this warp is done with it.
  auto piece = [&](int i) -> const Unit* {
    if (!wait_or_flag(bar + 8 * (kBarPieceFull + i % kPieces), (i / kPieces) & 1, failed)) return nullptr;
    const Unit* w = pieces + i % kPieces;
    return w->row < 0 ? nullptr : w;
  };
  auto piece_done = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar + 8 * (kBarPieceEmpty + i % kPieces));
  };
  // Of place i of the run K(0), V(0), K(1), ...
  auto raw_full_bar = [&](int i) { return bar + 8 * (kBarRawFull + (i & 1) * kRawStages + (i >> 1) % kRawStages); };
  auto raw_full_parity = [&](int i) { return ((i >> 1) / kRawStages) & 1; };
  auto raw_full = [&](int i) { return wait_or_flag(raw_full_bar(i), raw_full_parity(i), failed); };
  if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------ K
    registers_down<Regs<D>::kK>();
    const int th = tid - 256;
    const int kt = th & 3, kr = th >> 2;  // for i < 4 token 32 i + kr of the tile, chunk kt of its dims
    int gk = 0;  // places of the K ring filled
    auto k_place = [&]() -> char* {
      const int s = gk % kStages;
      if (gk >= kStages && !wait_or_flag(bar + 8 * (kBarKEmpty + s), (gk / kStages - 1) & 1, failed)) return nullptr;
      return sbase + S::oK + s * S::kTile;
    };
    auto k_stored = [&]() {
      fence_proxy_async_smem();
      mbar_arrive(bar + 8 * (kBarKFull + gk % kStages));
      ++gk;
    };
    // Where this thread's chunk 2 kt of K's row kr goes, in the stage; chunk 2 kt + 1 is 16 bytes on or
    // back, and row 32 i + kr 4096 i bytes on.
    const int at = kr ^ ((kr >> 1) & 4);
    const int k_at = at * 128 + (((2 * kt) ^ (at & 7)) << 4);
#pragma unroll 1
    for (int n = 0;; ++n) {
      const int ik = 2 * n;  // K's place in the run of rows; V's is the next. Whoever decodes rows gives them back.
      if (!raw_full(ik)) break;
      const TileInfo ti = info[n & 3];
      if (ti.kind & kEnd) break;
      char* tile = k_place();
      if (!tile) break;
      const char* raw_k = sbase + S::oRaw + ik % kRawStages * S::kRaw + (th >> 6) * S::kRawRow;
      const int parts = ti.kind & kSplit ? 2 : 1;
      // K(key, 16 dims of each group): two 16-byte chunks a group, 128-byte swizzled rows of 64 dims
#pragma unroll 1
      for (int part = 0; part < parts; ++part) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int row = 2 * i * S::kRawRow;
          __align__(16) uint32_t kw[2 * G], kp[G];
          const char* words = raw_k + row + (kr & 15) * (L::kWidth / 2) + kt * (8 * G);
          const int pairs = row + L::kCodes + (kr & 15) * 4 * G;
          if constexpr (G == 2) {
            *reinterpret_cast<uint4*>(kw) = *reinterpret_cast<const uint4*>(words);
            *reinterpret_cast<uint2*>(kp) = *reinterpret_cast<const uint2*>(raw_k + pairs);
          } else {
            *reinterpret_cast<uint2*>(kw) = *reinterpret_cast<const uint2*>(words);
            kp[0] = *reinterpret_cast<const uint32_t*>(raw_k + pairs);
          }
          const bool gone = 32 * i + kr >= ti.limit || ((ti.none >> (2 * i + (th >> 6))) & 1);
          __half2 most = as_half2(0);
#pragma unroll
          for (int e = 0; e < G; ++e) {
            if (gone) kp[e] = 0;
            most = __hmax2(most, __habs2(as_half2(kp[e])));
          }
          const bool clamp = __any_sync(kFull, may_overflow(most));
          auto store = [&](int gi, int w, const uint32_t (&v)[4]) {
            *reinterpret_cast<uint4*>(tile + i * 4096 + gi * S::kPanel + (k_at ^ (w << 4))) =
                make_uint4(v[0], v[1], v[2], v[3]);
          };
          auto all = [&](auto limited) {
            constexpr bool kLimited = decltype(limited)::value;
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
              const __half2 pr = as_half2(kp[gi]);
              const float2 prf = __half22float2(pr);
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                uint32_t v[4];
                decode8<kLimited>(kw[2 * gi + w], __low2half2(pr), __high2half2(pr), v);
                if (part == 1) {  // what that rounding left
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 hi = __half22float2(as_half2(v[e]));
                    float x[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 2^23 + code, an integer's float without a conversion
                      const float code = __uint_as_float(q4::k_code(kw[2 * gi + w], 2 * e + h) | 0x4b000000u) - 8388608.f;
                      x[h] = fmaf(code, prf.x, prf.y);
                      if (kLimited) x[h] = q4::max_nan(q4::min_nan(x[h], 65504.f), -65504.f);
                      x[h] -= h ? hi.y : hi.x;
                    }
                    v[e] = Mma<__half>::pack(x[0], x[1]);
                  }
                }
                store(gi, w, v);
              }
            }
          };
          if (clamp) all(std::true_type{});
          else all(std::false_type{});
        }
        k_stored();
        if (part + 1 < parts) {
          tile = k_place();
          if (!tile) break;
        }
      }
      if (!tile) break;
      mbar_arrive(bar + 8 * (kBarRawEmpty + ik % kRawStages));
    }
  } else if (warp >= 12 && warp < 16) {
    // ------------------------------------------------------------ V
    registers_down<Regs<D>::kV>();
    const int th = tid - 384;
    // half block vc (of 16) and dims 8 vg ... of each group
    const int vc = (th & 7) + 8 * (th >> 6), vg = ((th >> 3) & 3) + 4 * ((th >> 5) & 1);
    const int h = vc & 1;
    const int v_at = (vc >> 3) * (D * 128) + vg * 1024 + ((vc & 7) << 4);
#pragma unroll 1
    for (int n = 0;; ++n) {
      const int s = n % kStages, iv = 2 * n + 1;
      if (!raw_full(iv)) break;
      const TileInfo ti = info[n & 3];
      if (ti.kind & kEnd) break;
      const bool diag = ti.kind & kDiag;
      // V of 8 tokens, 8 dims of each group: one 16-byte chunk a dim, rows of 64 keys. The tokens are in the
      // places' order: of a block's second half the last four come first.
      {
        if (n >= kStages && !wait_or_flag(bar + 8 * (kBarVEmpty + s), (n / kStages - 1) & 1, failed)) break;
        const char* raw_v = sbase + S::oRaw + iv % kRawStages * S::kRaw + (vc >> 1) * S::kRawRow;
        char* tile = sbase + S::oV + s * S::kTile;
        const bool none = (ti.none >> (vc >> 1)) & 1;
#pragma unroll 1
        for (int gi = 0; gi < G; ++gi) {
          __align__(8) uint32_t vw[4][2];
          uint32_t vp[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pair = (4 * h + i) ^ (2 * h);
            *reinterpret_cast<uint2*>(vw[i]) =
                *reinterpret_cast<const uint2*>(raw_v + pair * L::kWidth + (vg ^ L::turn(pair)) * (8 * G) + gi * 8);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            vp[i] = *reinterpret_cast<const uint32_t*>(raw_v + L::kCodes + (8 * h + (i ^ (4 * h))) * 4 * G + gi * 4);
          if (ti.limit < kKeys || ti.none != 0 || diag) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (8 * vc + (i ^ (4 * h)) >= ti.limit || none) vp[i] = 0;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) nan |= is_nan_pair(vp[i]);
            if (diag && nan) {
#pragma unroll 1
              for (int i = 7; i >= 0; --i) {  // vp[0] in turn
                if (is_nan_pair(vp[0])) {
                  atomicMin(nans + ti.kind / kPlace * 2 + gi, ti.key0 + 8 * vc + ((7 - i) ^ (4 * h)));
                  vp[0] = 0;
                }
                const uint32_t first = vp[0];
#pragma unroll
                for (int e = 0; e < 7; ++e) vp[e] = vp[e + 1];
                vp[7] = first;
              }
            }
          }
          __half2 most = as_half2(0), sc[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half2 a = as_half2(vp[2 * i]), b = as_half2(vp[2 * i + 1]);
            most = __hmax2(most, __hmax2(__habs2(a), __habs2(b)));
            sc[i] = __lows2half2(a, b);
            lo[i] = __highs2half2(a, b);
          }
          auto all = [&](auto limited) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              uint32_t v[4][4];
#pragma unroll
              for (int i = 0; i < 4; ++i) decode8<decltype(limited)::value>(vw[i][w], sc[i], lo[i], v[i]);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4*>(tile + gi * 8192 + (4 * w + e) * 128 + (v_at ^ ((4 * w + e) << 4))) =
                    make_uint4(v[0][e], v[1][e], v[2][e], v[3][e]);
            }
          };
          if (__any_sync(kFull, may_overflow(most))) all(std::true_type{});
          else all(std::false_type{});
        }
        mbar_arrive(bar + 8 * (kBarRawEmpty + iv % kRawStages));
        fence_proxy_async_smem();
        mbar_arrive(bar + 8 * (kBarVFull + s));
      }
    }
  } else if (warp >= 16) {
    registers_down<Regs<D>::kMma>();
    if (warp > 18) goto done;
    if (warp == 18) {
      // --------------------------------------------------------------- plan
      int tiles = 0, i = 0;
#pragma unroll 1
      for (bool more = true; more && !failed; ++i) {
        const int s = i % kPieces;
        Unit w;
        w.n = 0;
        more = next_piece(p, prefix, plan, w);
        if (!more) w.row = -1;
        w.tile0 = tiles;
        tiles += w.n;
        // its queries on their way to L2 meanwhile
        if (more && w.slots > 0) {
          const int tokens = min(kTiles * p.tile, w.q_len - w.tok0), lines = D / 64;
#pragma unroll 1
          for (int k = lane; k < tokens * p.group * lines; k += 32) {
            const int line = k % lines, at = k / lines, tk = at / p.group;
            const T* q = reinterpret_cast<const T*>(p.q) + (w.token + tk) * p.q_st +
                         (int64_t)(w.kvh * p.group + at - tk * p.group) * p.q_sh + 64 * line;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
          }
        }
        if (i >= kPieces) {  // a piece may take long: as many waits as its tiles
          const uint32_t empty = bar + 8 * (kBarPieceEmpty + s), parity = (i / kPieces - 1) & 1;
          int tries = pieces[s].n + 1;
          while (tries > 0 && !mbar_wait_bounded(empty, parity)) --tries;
          if (tries == 0) failed = true;
          __syncwarp();
        }
        if (lane == 0) {
          pieces[s] = w;
          nans[2 * s] = nans[2 * s + 1] = INT32_MAX;
          mbar_arrive(bar + 8 * (kBarPieceFull + s));
        }
      }
      goto done;
    }
    if (warp == 17) {
      // -------------------------------------------------------------- copies
      int i = 0, n = 0;  // rows of K and V asked for, and tiles
#pragma unroll 1
      for (int ip = 0;; ++ip) {
        const Unit* at = piece(ip);
        if (!at) break;
        const Unit w = *at;
        piece_done(ip);
        const int32_t* table = p.block_table + (int64_t)w.row * p.bt_stride;
        auto fetch = [&](int b) -> int {
          if (b >= w.nblk) return -1;
          const int id = __ldg(table + b);
          if (id >= 0 && id < p.num_blocks) return id;
          atomic_or_err(p.err, SEB_ERRBIT_BLOCK_ID);
          return -1;
        };
        if (w.n == 0) continue;
        int ids = fetch(8 * w.j0 + lane), next = fetch(8 * w.j0 + 32 + lane);  // of 32 blocks, and of the 32 after them
#pragma unroll 1
        for (int k = 0; k < w.n && !failed; ++k, ++n) {
          const int j = w.j0 + k;
          if (k > 0 && (k & 3) == 0) {
            ids = next;
            next = fetch(8 * j + 32 + lane);
          }
          const int id = __shfl_sync(kFull, ids, (k & 3) * 8 + (lane & 7));
          const unsigned have = __ballot_sync(kFull, id >= 0) & 0xffu;
#pragma unroll 1
          for (int is_v = 0; is_v < 2; ++is_v, ++i) {
            const int s = i % kRawStages;
            if (i >= kRawStages && !wait_or_flag(bar + 8 * (kBarRawEmpty + s), (i / kRawStages - 1) & 1, failed)) break;
            if (lane == 0) {
              if (!is_v)
                info[n & 3] = TileInfo{w.k_len - j * kKeys, ~have & 0xffu,
                                       (w.split ? kSplit : 0) |
                                           ((j + 1) * kKeys > min(w.sees, w.k_len) ? kDiag : 0) |
                                           ip % kPieces * kPlace,
                                       j * kKeys};
              mbar_arrive_expect_tx(raw_full_bar(i), __popc(have) * L::kRow);
            }
            __syncwarp();
            if (lane < 8 && id >= 0)
              bulk_g2s(base + S::oRaw + s * S::kRaw + lane * S::kRawRow,
                       (is_v ? p.v_cache : p.k_cache) + ((int64_t)id * p.hkv + w.kvh) * L::kRow, L::kRow,
                       raw_full_bar(i));
          }
        }
      }
      for (int last = i + 2; i < last && !failed; ++i) {  // the end, to K's warps and to V's
        const int s = i % kRawStages;
        if (i >= kRawStages && !wait_or_flag(bar + 8 * (kBarRawEmpty + s), (i / kRawStages - 1) & 1, failed)) break;
        if (lane == 0) {
          info[n & 3].kind = kEnd;
          mbar_arrive(raw_full_bar(i));
        }
        __syncwarp();
      }
      if (failed) {  // whoever would have waited for the copies has given up: leave none in flight
        for (int k = max(0, i - kRawStages); k < i; ++k)
          mbar_wait_bounded(raw_full_bar(k), raw_full_parity(k), 1u << 16);
      }
      goto done;
    }
    // ---------------------------------------------------------------- MMA
    constexpr uint32_t idesc_qk = tc::idesc_f16(false, false, kRows, kKeys);
    constexpr uint32_t idesc_pv = tc::idesc_f16(false, false, kRows, D);
    // Descriptors of the first tile of each operand; others are so many 16-byte units on.
    const uint64_t desc_q = tc::smem_desc_sw128(base + S::oQ, 16, 1024);
    const uint64_t desc_k = tc::smem_desc_sw128(base + S::oK, 16, 1024);
    const uint64_t desc_v = tc::smem_desc_sw128(base + S::oV, 16, 1024);
    // S(t) from the K places g and, where K is in two parts, g + 1.
    auto issue_s = [&](int t, int g, int parts) {
      if (elect_one()) {
        const uint64_t dq = desc_q + t * (S::kTile >> 4);
        uint64_t dk = desc_k + g % kStages * (S::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc::mma_ss(tmem + t * 128, dq + (((kk >> 2) * S::kPanel + (kk & 3) * 32) >> 4),
                     dk + (((kk >> 2) * S::kPanel + (kk & 3) * 32) >> 4), idesc_qk, kk > 0);
        if (parts == 2) {
          dk = desc_k + (g + 1) % kStages * (S::kTile >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            tc::mma_ss(tmem + t * 128, dq + (((kk >> 2) * S::kPanel + (kk & 3) * 32) >> 4),
                       dk + (((kk >> 2) * S::kPanel + (kk & 3) * 32) >> 4), idesc_qk, true);
        }
        tc::commit(bar + 8 * (kBarSFull + t));
      }
      __syncwarp();
    };
    auto wait_k = [&](int g, int parts) {
      for (int part = 0; part < parts; ++part)
        if (!wait_or_flag(bar + 8 * (kBarKFull + (g + part) % kStages), ((g + part) / kStages) & 1, failed)) return false;
      return true;
    };
    auto release_k = [&](int g, int parts) {
      if (elect_one())
        for (int part = 0; part < parts; ++part) tc::commit(bar + 8 * (kBarKEmpty + (g + part) % kStages));
    };
    auto issue_pv = [&](int t, int s, bool first) {
      if (elect_one()) {
        const uint64_t dv = desc_v + s * (S::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          tc::mma_ts(tmem + kColO + t * D, tmem + t * 128 + 8 * kk,
                     dv + (((kk >> 2) * (D * 128) + (kk & 3) * 32) >> 4), idesc_pv, !first || kk > 0);
      }
      __syncwarp();
    };
    // For each K / V tile j and query tile t: PV(t, j), then S(t, j + 1) over the columns that it
    // read P from; one thread issues both, and its MMAs run in order.
    int gk = 0, gv = 0, nu = 0;
    uint32_t pphase = 0;
#pragma unroll 1
    for (int ip = 0;; ++ip) {
      const Unit* at = piece(ip);
      if (!at) break;
      const struct {
        int n, slots;
        bool twin, split;
      } w = {at->n, at->slots, at->twin, at->split};
      piece_done(ip);
      const int parts = w.split ? 2 : 1;
      for (int t = 0; t < w.slots && !failed; ++t) {
        if ((t == 0 || w.twin) && !wait_k(gk, parts)) break;
        if (!wait_or_flag(bar + 8 * (kBarQFull + t), (nu >> t) & 1, failed)) break;
        nu ^= 1 << t;
        tc::fence_after_sync();
        issue_s(t, gk, parts);
        if (w.twin || t + 1 == w.slots) {
          release_k(gk, parts);
          __syncwarp();
          gk += parts;
        }
      }
      if (w.twin) {  // tile j by warpgroup j & 1, with its O
#pragma unroll 1
        for (int j = 0; j < w.n && !failed; ++j, ++gv) {
          const int sv = gv % kStages, t = j & 1;
          if (!wait_or_flag(bar + 8 * (kBarVFull + sv), (gv / kStages) & 1, failed)) break;
          if (!wait_or_flag(bar + 8 * (kBarPFull + t), (pphase >> t) & 1, failed)) break;
          pphase ^= 1u << t;
          tc::fence_after_sync();
          issue_pv(t, sv, j < 2);
          if (elect_one()) {
            tc::commit(bar + 8 * (kBarVEmpty + sv));
            if (j + 2 >= w.n) tc::commit(bar + 8 * (kBarODone + t));
          }
          __syncwarp();
          if (j + 2 >= w.n) continue;
          if (!wait_k(gk, parts)) break;
          tc::fence_after_sync();
          issue_s(t, gk, parts);
          release_k(gk, parts);
          __syncwarp();
          gk += parts;
        }
        continue;
      }
#pragma unroll 1
      for (int j = 0; j < w.n && !failed; ++j) {
        const int sv = gv % kStages;
        if (!wait_or_flag(bar + 8 * (kBarVFull + sv), (gv / kStages) & 1, failed)) break;
        const bool more = j + 1 < w.n;
        for (int t = 0; t < w.slots && !failed; ++t) {
          if (!wait_or_flag(bar + 8 * (kBarPFull + t), (pphase >> t) & 1, failed)) break;
          pphase ^= 1u << t;
          tc::fence_after_sync();
          issue_pv(t, sv, j == 0);
          if (!more) {
            if (elect_one()) tc::commit(bar + 8 * (kBarODone + t));
            __syncwarp();
            continue;
          }
          if (t == 0 && !wait_k(gk, parts)) break;
          tc::fence_after_sync();
          issue_s(t, gk, parts);
        }
        if (elect_one()) tc::commit(bar + 8 * (kBarVEmpty + sv));
        if (more) {
          release_k(gk, parts);
          gk += parts;
        }
        __syncwarp();
        ++gv;
      }
    }
    if (elect_one()) tc::commit(bar + 8 * kBarFinal);  // every MMA is complete before TMEM is released
    __syncwarp();
    mbar_wait_bounded(bar + 8 * kBarFinal, 0, 1u << 20);
  } else {
    // ------------------------------------------------------------ softmax
    registers_up<Regs<D>::kSoftmax>();
    const int qt = warp >> 2;
    const int m = (warp & 3) * 32 + lane;
    const uint32_t taddr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t col_s = qt * 128, col_o = kColO + qt * D;
    const int tk = m / p.group, gh = m - tk * p.group;
    auto tile_of = [&](const Unit& w) { return w.twin ? 0 : qt; };  // the query tile
    auto token_of = [&](const Unit& w) { return tile_of(w) * p.tile + tk; };  // the row's token, of the unit
    int ns = 0, nd = 0;  // tiles of scores and pieces done by this warpgroup
    int nm = 0;          // times that it met the other one
    auto is_live = [&](const Unit& w) { return tk < p.tile && w.tok0 + token_of(w) < w.q_len; };
    // The row's query to shared memory as fp16 after a power of two; returns what brings its scores to log2 units.
    auto store_query = [&](const Unit& w) -> float {
      using T2 = typename Two<T>::type;
      const bool live = is_live(w);
      __align__(16) T2 q[D / 2];
      T2 most = Two<T>::zero();
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (w.token + token_of(w)) * p.q_st +
                                                        (int64_t)(w.kvh * p.group + gh) * p.q_sh);
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        *reinterpret_cast<uint4*>(&q[4 * i]) = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < D / 2; ++i) most = __hmax2_nan(most, __habs2(q[i]));
      const float top = q4::max_nan(Elem<T>::to_float(low_of(most)), Elem<T>::to_float(high_of(most)));
      const int ex = query_exponent(top);
      const float down = power2(-ex);
      char* row = sbase + S::oQ + qt * S::kTile + m * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = Mma<__half>::pack(Elem<T>::to_float(low_of(q[4 * i + e])) * down,
                                   Elem<T>::to_float(high_of(q[4 * i + e])) * down);
        *reinterpret_cast<uint4*>(row + (i >> 3) * S::kPanel + (((i & 7) ^ (m & 7)) << 4)) =
            make_uint4(v[0], v[1], v[2], v[3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(bar + 8 * (kBarQFull + qt));
      return copysignf(fminf(fabsf(p.scale_log2) * power2(ex), FLT_MAX), p.scale_log2);
    };
    // The CTA's first piece from the ip-th on, and before the until-th, that has work for this warpgroup; rows
    // that see nothing are written here.
    auto next_unit = [&](int& ip, int until) -> const Unit* {
#pragma unroll 1
      for (; ip < until; ++ip) {
        const Unit* at = piece(ip);
        if (!at || qt < at->slots) return at;
        const Unit& w = *at;
        if (qt < w.tiles && w.ntiles == 0 && w.start && is_live(w)) {
          const int head = w.kvh * p.group + gh;
          const int64_t token = w.token + token_of(w);
          uint4* op = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + token * p.o_st + (int64_t)head * p.o_sh);
#pragma unroll 1
          for (int d = 0; d < D / 8; ++d) op[d] = make_uint4(0u, 0u, 0u, 0u);
          p.lse[token * p.lse_st + head] = -INFINITY;
        }
        piece_done(ip);
      }
      return nullptr;
    };
    int ip = 0, ip_next = 0;
    const Unit* at = nullptr;
    float c_next = 0.f;
    bool later = true;  // the next unit is still to be looked for
#pragma unroll 1
    for (;;) {
      if (later) {
        at = next_unit(ip_next, INT32_MAX);
        if (at) c_next = store_query(*at);
      }
      if (!at) break;
      const Unit& w = *at;
      ip = ip_next;
      const float c = c_next;
      const bool live = is_live(w);
      const int first_tile = w.tile0 - w.j0;
      const int head = w.kvh * p.group + gh;
      const int64_t token = w.token + token_of(w);
      const int vis = !live ? 0 : p.causal ? min(w.k_len, w.sees + token_of(w)) : w.k_len;
      const int all_see = p.causal ? min(w.k_len, w.sees + tile_of(w) * p.tile) : w.k_len;  // every row of the tile
      const bool twin = w.twin;
      const int nblk = w.nblk;
      float m_ref = -INFINITY, l = 0.f;
      const int j_first = w.j0 + (twin ? qt : 0), j_end = w.j0 + w.n, j_step = twin ? 2 : 1;
#pragma unroll 1
      for (int j = j_first; j < j_end; j += j_step, ++ns) {
        wait_or_flag(bar + 8 * (kBarSFull + qt), ns & 1, failed);  // and PV(t, j - 1): O is stable
        tc::fence_after_sync();
        const unsigned holes = info[(first_tile + j) & 3].none & ((1u << min(8, nblk - 8 * j)) - 1);
        const bool plain = c > 0.f && (j + 1) * kKeys <= all_see && holes == 0;
        const int lim = vis - j * kKeys;
        const float cm = plain ? c : 1.f;
        // The row's scores, 32 at a time, twice: for their maximum, and for P; the next 32 are on
        // their way meanwhile. Held all at once they would not fit beside what else a thread has.
        float xa[32], xb[32];
        auto fetch = [&](float (&x)[32], int ch) { tc::tmem_ld32(taddr + col_s + 32 * (ch & 3), x); };
        auto mask = [&](float (&x)[32], int ch) {  // and into log2 units
          const int rest = lim - 32 * ch;
          const unsigned h0 = (holes >> (2 * ch)) & 1, h1 = (holes >> (2 * ch + 1)) & 1;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const bool seen = (i ^ ((i >> 1) & 4)) < rest && !(i < 16 ? h0 : h1);
            x[i] = seen ? x[i] * c : -INFINITY;
          }
        };
        float top = -INFINITY;
        auto take_max = [&](float (&x)[32], int ch) {
          if (!plain) mask(x, ch);
          float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
          for (int i = 4; i < 28; i += 8) {
            m0 = fmax3(m0, x[i], x[i + 1]);
            m1 = fmax3(m1, x[i + 2], x[i + 3]);
            m2 = fmax3(m2, x[i + 4], x[i + 5]);
            m3 = fmax3(m3, x[i + 6], x[i + 7]);
          }
          m0 = fmax3(m0, x[28], x[29]);
          m1 = fmax3(m1, x[30], x[31]);
          top = fmax3(top, fmaxf(m0, m1), fmaxf(m2, m3));
        };
        fetch(xa, 0);
        tc::tmem_wait_ld();
#pragma unroll 1
        for (int ch = 0; ch < 4; ch += 2) {
          fetch(xb, ch + 1);
          take_max(xa, ch);
          tc::tmem_wait_ld();
          fetch(xa, ch + 2);
          take_max(xb, ch + 1);
          tc::tmem_wait_ld();
        }
        top *= cm;
        const bool move = top > m_ref + kLazy;
        float factor = 1.f;
        if (move) {
          factor = fast_exp2(m_ref - (top - kBelow));
          l *= factor;
          m_ref = top - kBelow;
        }
        const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
        // scores so large that a product's rounding matters: rounded as in the reference
        const bool large = plain && fabsf(m_ref) > 1e6f;
        const float cx = large ? 1.f : cm;
        float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
        auto take_p = [&](float (&x)[32], int ch) {
          if (!plain) mask(x, ch);
          if (large) {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __fmul_rn(x[i], c);
          }
          uint32_t hi[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 d = fma2(make_float2(x[2 * e], x[2 * e + 1]), splat2(cx), splat2(neg));
            const float2 pr = make_float2(fast_exp2(d.x), fast_exp2(d.y));
            if (e & 1) sum1 = add2(sum1, pr);
            else sum0 = add2(sum0, pr);
            hi[e] = Mma<__half>::pack(pr.x, pr.y);
          }
          tc::tmem_st16u(taddr + col_s + 16 * ch, hi);
        };
#pragma unroll 1
        for (int ch = 0; ch < 4; ch += 2) {  // P of 32 keys covers 16 columns, of scores that were read
          fetch(xb, ch + 1);
          take_p(xa, ch);
          tc::tmem_wait_ld();
          if (ch == 0) fetch(xa, 2);
          take_p(xb, ch + 1);
          tc::tmem_wait_ld();
        }
        sum0 = add2(sum0, sum1);
        l += sum0.x + sum0.y;
        if (j > j_first && __any_sync(kFull, move)) {
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            float o[16];
            tc::tmem_ld16(taddr + col_o + 16 * cc, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= factor;
            tc::tmem_st16(taddr + col_o + 16 * cc, o);
          }
        }
        tc::tmem_wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar + 8 * (kBarPFull + qt));
      }
      // ---- the next unit's query, so that its first scores come while this one's O is written
      // A piece that takes this one's place is described only once this one is given back: not waited for here.
      ++ip_next;
      at = __any_sync(kFull, failed) ? nullptr : next_unit(ip_next, ip + kPieces);
      later = ip_next == ip + kPieces;
      if (at) c_next = store_query(*at);
      // ---- O is final
      wait_or_flag(bar + 8 * (kBarODone + qt), nd & 1, failed);
      ++nd;
      tc::fence_after_sync();
      if (__any_sync(kFull, failed)) break;
      // Both warpgroups have a sum: they tell each other of their references, and each takes half of
      // the dims of both.
      float f0 = 1.f, f1 = 0.f;
      auto meet = [&]() {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar + 8 * kBarMerge);
        wait_or_flag(bar + 8 * kBarMerge, nm & 1, failed);
        ++nm;
        tc::fence_after_sync();
      };
      if (twin) {
        float2* ml = reinterpret_cast<float2*>(sbase + S::oMl);
        ml[qt * kRows + m] = make_float2(m_ref, l);
        meet();
        const float2 other = ml[(qt ^ 1) * kRows + m];
        const float top = fmaxf(m_ref, other.x), ref = top == -INFINITY ? 0.f : top;
        f0 = fast_exp2(m_ref - ref);
        f1 = fast_exp2(other.x - ref);
        l = fmaf(other.y, f1, l * f0);
        m_ref = top;
      }
      const int col_mine = col_o, col_other = kColO + (qt ^ 1) * D;
      auto take_o = [&](float (&o)[32], int d) {  // dims d .. d + 31 of the sum
        tc::tmem_ld32(taddr + col_mine + d, o);
        tc::tmem_wait_ld();
        if (twin) {
          float x[32];
          tc::tmem_ld32(taddr + col_other + d, x);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = fmaf(x[i], f1, o[i] * f0);
        }
        if (nans[ip % kPieces * 2 + d / q4::kGroup] < vis) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __int_as_float(0x7fffffff);
        }
      };
      T* op = reinterpret_cast<T*>(p.out) + token * p.o_st + (int64_t)head * p.o_sh;
      auto write_o = [&](const float (&o)[32], int d, float inv) {
#pragma unroll
        for (int v8 = 0; v8 < 4; ++v8) {
          uint32_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = Mma<T>::pack(o[8 * v8 + 2 * e] * inv, o[8 * v8 + 2 * e + 1] * inv);
          *reinterpret_cast<uint4*>(op + d + 8 * v8) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      };
      auto write_lse = [&](float top, float sum) {
        p.lse[token * p.lse_st + head] = sum == 0.f ? -INFINITY : fmaf(top, kLn2, logf(sum));
      };
      const int d0 = twin ? qt * (D / 2) : 0, d1 = twin ? d0 + D / 2 : D;
      const uint32_t first = w.first, last = w.last;
      if (first == last) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int d = d0; d < d1; d += 32) {
          float o[32];
          take_o(o, d);
          if (live) write_o(o, d, inv);
        }
        if (live && d0 == 0) write_lse(m_ref, l);
      } else {
        // A part: of each row its dims in fours, then (m, l). Units of one query tile have two, of
        // half the dims each, so that either warpgroup or both can leave them.
        const bool one = w.tiles == 1;
        const int width = one ? D / 2 : D;
        auto part_of = [&](uint32_t cta, int part) {
          return p.ws + (((int64_t)cta * 2 + (cta == first)) * 2 + part) * (kRows * (D + 2));
        };
        const int part0 = one ? d0 / (D / 2) : qt, parts = (d1 - d0) / width;
#pragma unroll 1
        for (int d = d0; d < d1; d += 32) {
          float o[32];
          take_o(o, d);
          if (live) {
            float4* dst = reinterpret_cast<float4*>(part_of(blockIdx.x, part0 + (d - d0) / width)) + m;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              __stcg(dst + ((d - d0) % width / 4 + i) * kRows, make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
          }
        }
#pragma unroll 1
        for (int part = part0; part < part0 + parts; ++part) {
          if (live) __stcg(reinterpret_cast<float2*>(part_of(blockIdx.x, part) + kRows * D) + m, make_float2(m_ref, l));
          __threadfence();
          __syncwarp();
          int32_t* ctr = p.chunk_arrivals + (first * 2 + part) * 4 + (warp & 3);
          int arrived = 0;
          if (lane == 0) arrived = atomicAdd(ctr, 1);
          arrived = __shfl_sync(kFull, arrived, 0);
          if (arrived != (int)(last - first)) continue;
          // the last to come joins the rows of its warp, in order of the parts' places
          __threadfence();
          if (!live) continue;
          float top = -INFINITY;
#pragma unroll 4
          for (uint32_t c = first; c <= last; ++c)
            top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(part_of(c, part) + kRows * D) + m).x);
          const float ref = top == -INFINITY ? 0.f : top;
          const int from = one ? part * width : 0;
#pragma unroll 1
          for (int d = 0; d < width; d += 32) {
            float o[32], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 1
            for (uint32_t c = first; c <= last; ++c) {
              const float* src = part_of(c, part);
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + kRows * D) + m);
              const float weight = fast_exp2(ml.x - ref);
              sum = fmaf(ml.y, weight, sum);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(src) + (d / 4 + i) * kRows + m);
                o[4 * i] = fmaf(x.x, weight, o[4 * i]);
                o[4 * i + 1] = fmaf(x.y, weight, o[4 * i + 1]);
                o[4 * i + 2] = fmaf(x.z, weight, o[4 * i + 2]);
                o[4 * i + 3] = fmaf(x.w, weight, o[4 * i + 3]);
              }
            }
            write_o(o, from + d, sum == 0.f ? 0.f : 1.f / sum);
            if (from + d == 0) write_lse(top, sum);
          }
        }
      }
      if (twin) meet();  // the other's O has been read
      piece_done(ip);
      tc::fence_before_sync();  // the next unit's first PV overwrites O
    }
  }

done:
  if (failed && lane == 0) atomic_or_err(p.err, SEB_ERRBIT_TIMEOUT);
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 16) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

int ctas_of() { return std::min(num_sms(), kMaxChunkCtas); }

template <typename T, int D>
int launch(Q4Params p, cudaStream_t s) {
  constexpr auto kern = q4_prefill_kernel<T, D>;
  constexpr int smem = Smem<D>::kBytes + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of an SM");
  const int rc = set_smem_limit_once<kern>(smem);
  if (rc != SEB_OK) return rc;
  p.tile = kRows / p.group;
  // no more CTAs than the tokens' units have key tiles; units: at most one for each row and kv head beyond the full ones
  const int64_t units = ((int64_t)p.total_query / (kTiles * p.tile) + p.num_rows) * p.hkv;
  const int64_t places = (p.max_blocks + 7) / 8 + kUnitPlaces;
  const int64_t grid = std::min<int64_t>(ctas_of(), units * places);
  // places are counted in 32 bits
  p.cut_below = (uint32_t)std::min<int64_t>(grid, (int64_t)0x7fffffff / places);
  kern<<<(unsigned)grid, kThreads, smem, s>>>(p);
  return launch_status("q4_prefill_kernel");
}

}  // namespace

int launch_q4_prefill(const Q4Params& p, int head_dim, int dtype, cudaStream_t s) {
  if (dtype == SEB_BF16)
    return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
  return head_dim == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
}

int64_t q4_prefill_workspace(int head_dim) { return ctas_of() * 4ll * kRows * (head_dim + 2) * 4; }

}  // namespace seb
