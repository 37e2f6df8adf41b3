// Paged attention over the 4-bit KV pool.
//
//   O = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = scale * q . k_j,
//   LSE = log(sum_j exp(s_j)),
// over the keys j < k_lens[r] (causal: and j <= the query's position). Rows follow
// seb_paged_decode; a query that sees no key gets O = 0 and LSE = -inf.
//
// With k_j = s n + l for each group G of 64 dims the codes go through the tensor
// cores as they are and the parameters meet the results:
//   s_j = scale * sum_G (sK_jG (q_G . n_jG) + lK_jG sum(q_G)),
//   sum_j p_j v_j = sum_j (p_j sV_jG) n_jG + sum_j p_j lV_jG.
// A code masked out of its word is the fp16 number n * 2^-24 (or n * 2^-20 for the
// upper four bits of a byte), an exact operand: one AND gives two, one shift serves
// four. The powers of two are undone in the queries (scaled by 1/16 where the upper
// codes meet them) and in the results. So a value costs 0.6 instructions before its
// mma.sync, and the pool's bytes, a quarter of a 16-bit pool's, still set the time.
//
// Rounding to 16 bits: q becomes fp16 after a power of two per head that puts its
// largest element at 2^14 (exact for bf16 and fp16 down to 2^-28 of that element);
// p_j sV_jG becomes fp16 (unit 2^-11) after a power of two that keeps it below 2^15.
// Scores, maxima, sums and O are fp32.
//
// Work: a unit is (row, tile of tokens, kv head) and its blocks; the units of all rows
// laid end to end are cut in equal runs of blocks, one per resident warp, whatever
// the rows' lengths. A warp keeps all query heads of the group (and several tokens of
// a row, up to 8 * NT columns) on one tile, so each KV byte is read once per tile.
// Parts of a unit are joined in shared memory, and over CTAs in the workspace by the
// last to arrive, in order of their place, so results do not depend on timing.
#include "q4_format.cuh"

#include <algorithm>
#include <cfloat>

namespace seb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -FLT_MAX;       // no score yet: any score is above it by more than the threshold
constexpr float kThreshold = 8.f;        // scores may exceed the reference by 2^8 before it is moved
constexpr float kScaleThreshold = 64.f;  // p * V scale stays below 2^8 * 2^6

struct Q4Params {
  const char* q;
  int64_t q_st, q_sh;  // elements
  const char* k_cache;
  const char* v_cache;
  int64_t num_blocks;
  const int32_t* block_table;
  int64_t bt_stride;
  int64_t max_blocks;
  const int32_t* q_starts;
  const int32_t* q_lens;
  const int32_t* k_lens;
  const int32_t* q_pos;
  int32_t num_rows;
  int32_t total_query;
  int32_t hq, hkv, group;
  int32_t tile;  // tokens of a tile
  float scale_log2;
  int32_t causal;
  int32_t vec;   // q and out rows are 16-byte aligned
  char* out;
  int64_t o_st, o_sh;  // elements
  float* lse;
  int64_t lse_st;
  int32_t counter_slot;
  float* ws_o;        // [CTA][2][columns][D]
  float* ws_ml;       // [CTA][2][columns][2]
  int32_t* err;
};

// Arrivals at the units that span CTAs, one for each column, at the CTA that a unit
// starts in. Zero when the library is loaded, and again after every call (the last to
// arrive clears it); calls that may overlap use different slots.
constexpr int kMaxCtas = 512;
__device__ int32_t g_q4_counters[SEB_Q4_COUNTER_SLOTS][kMaxCtas * 32];

struct Row {
  int q_len, q_start, q_pos, k_len;
  int nblk;   // blocks of each of its units; at least 1 where it has tokens
  int tiles;
};

__device__ __forceinline__ Row row_of(const Q4Params& p, int r, uint32_t* bad) {
  Row w;
  w.q_len = max(__ldg(p.q_lens + r), 0);
  w.q_start = __ldg(p.q_starts + r);
  w.q_pos = __ldg(p.q_pos + r);
  w.k_len = max(__ldg(p.k_lens + r), 0);
  if (w.q_len > 0 && (w.q_start < 0 || (int64_t)w.q_start + w.q_len > p.total_query)) {
    *bad |= SEB_ERRBIT_META;
    w.q_len = 0;
  }
  if (w.k_len > p.max_blocks * kBlockSize) {
    *bad |= SEB_ERRBIT_KLEN;
    w.k_len = (int)(p.max_blocks * kBlockSize);
  }
  int64_t seen = w.k_len;
  if (p.causal) seen = min(seen, (int64_t)w.q_pos + w.q_len);
  w.nblk = max((int)((seen + 15) >> 4), 1);
  w.tiles = (w.q_len + p.tile - 1) / p.tile;
  return w;
}

__device__ __forceinline__ int64_t blocks_of(const Q4Params& p, const Row& w) {
  return (int64_t)w.tiles * p.hkv * w.nblk;
}

// What a warp leaves of a unit that it did not do alone.
struct Part {
  int64_t unit;  // the unit's first block in the run of all units; -1: no part
  int64_t end;   // and past its last
  int row, tile, kvh, cols;
};

template <int D, int NT, int NW, int STAGES>
struct Smem {
  static constexpr int kCols = 8 * NT;
  static constexpr int kStage = 2 * q4::Layout<D>::kRow;
  static constexpr int kPartBytes = kCols * (D + 2) * 4;
  static constexpr int kRing = STAGES * kStage > kPartBytes ? STAGES * kStage : kPartBytes;
  static constexpr int kWarp = (kRing + kPartBytes + 127) / 128 * 128;
  static constexpr int kParts = 0;                                  // Part[NW][2]
  static constexpr int kPrefix = kParts + NW * 2 * (int)sizeof(Part);  // int64 [NW * 32 + 1]
  static constexpr int kBars = kPrefix + (NW * 32 + 2) * 8;
  static constexpr int kWarps = (kBars + NW * STAGES * 8 + 127) / 128 * 128;
  static constexpr int kBytes = kWarps + NW * kWarp;
};

// Weighted sum of `n` parts of one column; lane l holds dims l * D / 32 and on, so that
// O = o / l with scores against m. part(i) gives part i's O row and its (m, l).
template <int D, bool GLOBAL, typename F>
__device__ __forceinline__ void join(int n, int lane, F part, float (&o)[D / 32], float& m, float& l) {
  constexpr int DL = D / 32;
  m = -INFINITY;
  for (int i = lane; i < n; i += 32) {
    const float2* ml;
    const float* row;
    part(i, row, ml);
    m = fmaxf(m, GLOBAL ? __ldcg(ml).x : ml->x);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, off));
  const float ref = m == -INFINITY ? 0.f : m;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < DL; ++e) o[e] = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    float w = 0.f, li = 0.f;
    if (i0 + lane < n) {
      const float2* ml;
      const float* row;
      part(i0 + lane, row, ml);
      const float2 v = GLOBAL ? __ldcg(ml) : *ml;
      w = exp2f(v.x - ref);
      li = v.y * w;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) li += __shfl_xor_sync(kFull, li, off);
    l += li;
    const int cnt = min(32, n - i0);
#pragma unroll 8
    for (int k = 0; k < cnt; ++k) {
      const float2* ml;
      const float* row;
      part(i0 + k, row, ml);
      const float wk = __shfl_sync(kFull, w, k);
      float v[DL];
      if constexpr (DL == 2) {
        const float2 x = GLOBAL ? __ldcg(reinterpret_cast<const float2*>(row) + lane)
                                : reinterpret_cast<const float2*>(row)[lane];
        v[0] = x.x, v[1] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < DL / 4; ++c) {
          const float4* at = reinterpret_cast<const float4*>(row) + lane * (DL / 4) + c;
          const float4 x = GLOBAL ? __ldcg(at) : *at;
          v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
        }
      }
#pragma unroll
      for (int e = 0; e < DL; ++e) o[e] = fmaf(wk, v[e], o[e]);
    }
  }
}

template <typename T, int D, int NT, int NW, int STAGES, int CTAS>
__global__ void __launch_bounds__(NW * 32, CTAS) q4_attention_kernel(const Q4Params p) {
  using L = q4::Layout<D>;
  using S = Smem<D, NT, NW, STAGES>;
  constexpr int P = L::kPanels, G = L::kGroups;  // panels, groups of a panel
  constexpr int kCols = S::kCols;
  extern __shared__ __align__(128) char smem[];
  Part* parts = reinterpret_cast<Part*>(smem + S::kParts);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + S::kPrefix);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // ---- the units of all rows, and this warp's run of blocks
  const int chunk = (p.num_rows + NW * 32 - 1) / (NW * 32);  // rows that a thread sums up
  {
    int64_t sum = 0;
    uint32_t bad = 0;
    for (int r = tid * chunk; r < min((tid + 1) * chunk, p.num_rows); ++r) sum += blocks_of(p, row_of(p, r, &bad));
    if (bad && blockIdx.x == 0) atomic_or_err(p.err, bad);
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t o = __shfl_up_sync(kFull, sum, off);
      if (lane >= off) sum += o;
    }
    prefix[tid + 1] = sum;
    if (tid == 0) prefix[0] = 0;
    if (lane < 2) parts[warp * 2 + lane].unit = -1;
  }
  __syncthreads();
  int64_t total = 0, before = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) before = total;
    total += prefix[(w + 1) * 32];
  }
  __syncthreads();
  prefix[tid + 1] += before;
  __syncthreads();
  const int64_t warps = (int64_t)gridDim.x * NW;
  const int64_t per = max((total + warps - 1) / warps, (int64_t)4);
  const int64_t cta0 = (int64_t)blockIdx.x * NW * per, cta1 = min(cta0 + NW * per, total);
  if (cta0 >= total) return;
  int64_t pos = cta0 + warp * per;
  const int64_t stop = min(pos + per, total);

  const uint32_t bars = smem_u32(smem + S::kBars) + warp * STAGES * 8;
  char* ring = smem + S::kWarps + warp * S::kWarp;
  const uint32_t ring_a = smem_u32(ring);
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  __syncwarp();

  if (pos < stop) {
    // the row that holds block `pos`, and pos's place in the row
    int lo = 0, hi = NW * 32 - 1;
    while (lo < hi) {  // last chunk that starts at or before pos
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= pos) lo = mid;
      else hi = mid - 1;
    }
    int r = lo * chunk;
    int64_t off = pos - prefix[lo];
    uint32_t bad = 0;
    Row row = row_of(p, r, &bad);
    uint32_t it = 0;  // blocks taken through the ring so far
    bool dead = false;

    while (pos < stop) {
      int64_t len = blocks_of(p, row);
      while (off >= len) {
        off -= len;
        row = row_of(p, ++r, &bad);
        len = blocks_of(p, row);
      }
      const int64_t unit = off / row.nblk;
      const int blk0 = (int)(off - unit * row.nblk);
      const int kvh = (int)(unit % p.hkv), tile = (int)(unit / p.hkv);
      const int n = (int)min((int64_t)(row.nblk - blk0), stop - pos);
      const int tok0 = tile * p.tile;                    // first token of the tile in the row
      const int toks = min(p.tile, row.q_len - tok0);
      const int cols = toks * p.group;
      // keys that the tile's first and last token see
      int64_t seen0 = row.k_len, seen1 = row.k_len;
      if (p.causal) {
        seen0 = min(seen0, max((int64_t)row.q_pos + tok0 + 1, (int64_t)0));
        seen1 = min(seen1, max((int64_t)row.q_pos + tok0 + toks, (int64_t)0));
      }
      const int see_all = (int)seen0, see_any = (int)seen1;
      const int first_sees = (int)min((int64_t)row.q_pos + tok0 + 1, (int64_t)(1 << 30));  // and one more per token
      const int blk1 = min(blk0 + n, (see_any + 15) >> 4);  // blocks from here on hold nothing for this tile

      // ---- block ids, 32 at a time; ring prologue
      const int32_t* table = p.block_table + (int64_t)r * p.bt_stride;
      auto load_id = [&](int b) -> int {
        if (b >= blk1) return -1;
        int id = __ldg(table + b);
        if (id < 0 || id >= p.num_blocks) {
          atomic_or_err(p.err, SEB_ERRBIT_BLOCK_ID);
          id = -1;
        }
        return id;
      };
      int ids = load_id(blk0 + lane), ids_next = load_id(blk0 + 32 + lane);
      uint32_t issued = it;
      auto issue = [&](int b) {  // stage block b (of the row); called for blk0, blk0 + 1, ... in turn
        const int j = b - blk0;
        if (j > 0 && (j & 31) == 0) {
          ids = ids_next;
          ids_next = load_id(b + 32 + lane);
        }
        const int id = __shfl_sync(kFull, ids, j & 31);
        if (lane == 0) {
          const uint32_t s = issued % STAGES;
          const uint32_t bar = bars + 8 * s, dst = ring_a + s * S::kStage;
          if (id >= 0) {
            const int64_t at = ((int64_t)id * p.hkv + kvh) * L::kRow;
            mbar_arrive_expect_tx(bar, S::kStage);
            bulk_g2s(dst, p.k_cache + at, L::kRow, bar);
            bulk_g2s(dst + L::kRow, p.v_cache + at, L::kRow, bar);
          } else {
            mbar_arrive_expect_tx(bar, 0);
          }
        }
        ++issued;
        return id;
      };
      uint32_t unread = 0;  // bit s: the block in ring place s could not be read
      auto stage = [&](int b) {
        const uint32_t s = issued % STAGES;
        unread = (unread & ~(1u << s)) | (issue(b) < 0 ? 1u << s : 0u);
      };
      for (int b = blk0; b < min(blk0 + STAGES, blk1); ++b) stage(b);

      // ---- Q as the B operand: column 8 nt + g, dims 16 t .. 16 t + 15 of every group
      uint32_t qf[P * G][NT][4][2];
      float qs[P * G][NT][2], ch[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int col = nt * 8 + g;
        const bool live = col < cols;
        const int tk = live ? col / p.group : 0, hd = live ? col - tk * p.group : 0;
        const T* src = reinterpret_cast<const T*>(p.q) + ((int64_t)row.q_start + tok0 + tk) * p.q_st +
                       (int64_t)(kvh * p.group + hd) * p.q_sh + 16 * t;
        float top = 0.f;
        uint4 raw[P * G][2];
#pragma unroll
        for (int gr = 0; gr < P * G; ++gr)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            raw[gr][h] = make_uint4(0u, 0u, 0u, 0u);
            if (live) {
              const T* at = src + gr * 64 + 8 * h;
              if (p.vec) {
                raw[gr][h] = *reinterpret_cast<const uint4*>(at);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(&raw[gr][h])[e] = at[e];
              }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              top = q4::max_nan(top, fabsf(Elem<T>::to_float(reinterpret_cast<const T*>(&raw[gr][h])[e])));
          }
        top = q4::max_nan(top, __shfl_xor_sync(kFull, top, 1));
        top = q4::max_nan(top, __shfl_xor_sync(kFull, top, 2));
        // 2^-e with the largest element in [2^14, 2^15) after it
        const int ex = top > 0.f ? min(max((int)((__float_as_uint(top) >> 23) & 255) - 127 - 14, -100), 112) : 0;
        const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int gr = 0; gr < P * G; ++gr) {
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {  // 4 elements: two that meet lower codes, two that meet upper ones
            const T* e = reinterpret_cast<const T*>(&raw[gr][w >> 1]) + (w & 1) * 4;
            const __half2 a = __floats2half2_rn(Elem<T>::to_float(e[0]) * down, Elem<T>::to_float(e[1]) * down);
            const __half2 b = __floats2half2_rn(Elem<T>::to_float(e[2]) * (down * 0.0625f),
                                                Elem<T>::to_float(e[3]) * (down * 0.0625f));
            qf[gr][nt][w][0] = *reinterpret_cast<const uint32_t*>(&a);
            qf[gr][nt][w][1] = *reinterpret_cast<const uint32_t*>(&b);
            sum += __low2float(a) + __high2float(a) + 16.f * (__low2float(b) + __high2float(b));
          }
          sum += __shfl_xor_sync(kFull, sum, 1);
          sum += __shfl_xor_sync(kFull, sum, 2);
          sum *= 5.9604644775390625e-8f;  // 2^-24, as the codes carry it
          qs[gr][nt][0] = __shfl_sync(kFull, sum, 8 * t);
          qs[gr][nt][1] = __shfl_sync(kFull, sum, 8 * t + 4);
        }
        // back: 2^(ex + 24), in two steps where one would leave the range
        const float up = fminf(fabsf(p.scale_log2) * 16777216.f, FLT_MAX) * __uint_as_float((uint32_t)(127 + ex) << 23);
        const float c = copysignf(fminf(up, FLT_MAX), p.scale_log2);
        ch[nt][0] = __shfl_sync(kFull, c, 8 * t);
        ch[nt][1] = __shfl_sync(kFull, c, 8 * t + 4);
      }

      // ---- the blocks
      float m[NT][2], l[NT][2], low[P * G][NT][2], o[P * G][4][NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          m[nt][h] = kNoMax;
          l[nt][h] = 0.f;
#pragma unroll
          for (int gr = 0; gr < P * G; ++gr) low[gr][nt][h] = 0.f;
        }
#pragma unroll
      for (int gr = 0; gr < P * G; ++gr)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[gr][mt][nt][c] = 0.f;
      float v_down = 0.f;  // power of two that V's scales are taken by; 0 until a block sets it

      for (int b = blk0; b < blk1; ++b, ++it) {
        const uint32_t s = it % STAGES;
        if (dead || !mbar_wait_bounded(bars + 8 * s, (it / STAGES) & 1)) {
          if (!dead && lane == 0) atomic_or_err(p.err, SEB_ERRBIT_TIMEOUT);
          dead = true;
          break;
        }
        const char* kb = ring + s * S::kStage;
        const char* vb = kb + L::kRow;
        uint32_t kw[P][2][2 * G], vw[P][2][2 * G];  // words of keys g, g + 8; of key pairs t, t + 4
        float2 kp[P * G][2], vp[P * G][2];          // (scale, low) of keys g, g + 8
#pragma unroll
        for (int pn = 0; pn < P; ++pn)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const char* ka = kb + pn * 8 * L::kWidth + (g + 8 * h) * (L::kWidth / 2) + t * (8 * G);
            const char* va = vb + pn * 8 * L::kWidth + (t + 4 * h) * L::kWidth + (g ^ L::turn(t)) * (8 * G);
            const char* kq = kb + L::kCodes + pn * 64 * G + (g + 8 * h) * 4 * G;
            const char* vq = vb + L::kCodes + pn * 64 * G + (g + 8 * h) * 4 * G;
            __half2 a[G], c[G];
            if constexpr (G == 2) {
              *reinterpret_cast<uint4*>(kw[pn][h]) = *reinterpret_cast<const uint4*>(ka);
              *reinterpret_cast<uint4*>(vw[pn][h]) = *reinterpret_cast<const uint4*>(va);
              *reinterpret_cast<uint2*>(a) = *reinterpret_cast<const uint2*>(kq);
              *reinterpret_cast<uint2*>(c) = *reinterpret_cast<const uint2*>(vq);
            } else {
              *reinterpret_cast<uint2*>(kw[pn][h]) = *reinterpret_cast<const uint2*>(ka);
              *reinterpret_cast<uint2*>(vw[pn][h]) = *reinterpret_cast<const uint2*>(va);
              *reinterpret_cast<uint32_t*>(a) = *reinterpret_cast<const uint32_t*>(kq);
              *reinterpret_cast<uint32_t*>(c) = *reinterpret_cast<const uint32_t*>(vq);
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              kp[pn * G + gr][h] = __half22float2(a[gr]);
              vp[pn * G + gr][h] = __half22float2(c[gr]);
            }
          }
        const bool bad_block = (unread >> s) & 1;
        __syncwarp();  // every lane has its words: the place may be filled again
        if (b + STAGES < blk1) stage(b + STAGES);

        // S^T = K Q^T: 16 keys x 8 NT columns, one sum for each group
        float x[NT][4];
#pragma unroll
        for (int gr = 0; gr < P * G; ++gr) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[nt][c] = 0.f;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t k0 = kw[gr / G][0][gr % G * 2 + w], k1 = kw[gr / G][1][gr % G * 2 + w];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                Mma<__half>::run(acc[nt], k0 & 0x000f000fu, k1 & 0x000f000fu, k0 & 0x00f000f0u, k1 & 0x00f000f0u,
                                 qf[gr][nt][2 * w + h][0], qf[gr][nt][2 * w + h][1]);
              k0 >>= 8, k1 >>= 8;
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float2 pr = kp[gr][c >> 1];
              const float base = gr == 0 ? pr.y * qs[gr][nt][c & 1] : fmaf(pr.y, qs[gr][nt][c & 1], x[nt][c]);
              x[nt][c] = fmaf(pr.x, acc[nt][c], base);
            }
        }
        // masked keys: score -inf, and no parameter of theirs (it may be NaN) meets a zero weight
        const int key = b * 16 + g;
        const bool masked = bad_block || (b + 1) * 16 > see_all;
        bool hide[NT][4];
        if (masked) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int tk = (nt * 8 + 2 * t + (c & 1)) / p.group;
              const int last = p.causal ? min(row.k_len, first_sees + tk) : row.k_len;
              hide[nt][c] = bad_block || key + 8 * (c >> 1) >= last;
            }
        }
        float d[NT][4], far = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            d[nt][c] = fmaf(x[nt][c], ch[nt][c & 1], -m[nt][c & 1]);
            if (masked && hide[nt][c]) d[nt][c] = -INFINITY;
            far = fmaxf(far, d[nt][c]);
          }
        float sv[P * G][2], big = 0.f;
#pragma unroll
        for (int gr = 0; gr < P * G; ++gr)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sv[gr][h] = vp[gr][h].x * v_down;
            big = fmaxf(big, sv[gr][h]);
          }
        if (__any_sync(kFull, far > kThreshold || big > kScaleThreshold || v_down == 0.f)) {
          // move the references: scores' maxima, and the power of two of V's scales
          float vmax = 0.f;
#pragma unroll
          for (int gr = 0; gr < P * G; ++gr)
#pragma unroll
            for (int h = 0; h < 2; ++h) vmax = fmaxf(vmax, key + 8 * h < see_any && !bad_block ? vp[gr][h].x : 0.f);
#pragma unroll
          for (int k = 16; k >= 1; k >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(kFull, vmax, k));
          float v_fix = 1.f;
          if (v_down == 0.f || vmax * v_down > kScaleThreshold) {
            const int ex = min(max((int)((__float_as_uint(vmax) >> 23) & 255) - 127, -24), 16);
            const float now = __uint_as_float((uint32_t)(127 - ex) << 23);
            v_fix = v_down == 0.f ? 1.f : now / v_down;
            v_down = now;
#pragma unroll
            for (int gr = 0; gr < P * G; ++gr)
#pragma unroll
              for (int h = 0; h < 2; ++h) sv[gr][h] = vp[gr][h].x * v_down;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mx = -INFINITY;
#pragma unroll
              for (int c = h; c < 4; c += 2)
                if (!(masked && hide[nt][c])) mx = fmaxf(mx, __fmul_rn(x[nt][c], ch[nt][h]));
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
              const float now = fmaxf(mx, m[nt][h]);
              const float fix = m[nt][h] == kNoMax ? 0.f : exp2f(m[nt][h] - now);
              m[nt][h] = now;
              l[nt][h] *= fix;
#pragma unroll
              for (int gr = 0; gr < P * G; ++gr) {
                low[gr][nt][h] *= fix;
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                  o[gr][mt][nt][h] *= fix * v_fix;
                  o[gr][mt][nt][h + 2] *= fix * v_fix;
                }
              }
#pragma unroll
              for (int c = h; c < 4; c += 2)  // the product rounded as in `now`: the largest score gets 0, however large
                d[nt][c] = masked && hide[nt][c] ? -INFINITY : __fsub_rn(__fmul_rn(x[nt][c], ch[nt][h]), now);
            }
        }
        float pr[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c) pr[nt][c] = exp2f(d[nt][c]);
          l[nt][0] += pr[nt][0] + pr[nt][2];
          l[nt][1] += pr[nt][1] + pr[nt][3];
        }

        // O^T += V^T (P sV)^T, and the lows' share
#pragma unroll
        for (int gr = 0; gr < P * G; ++gr) {
          uint32_t b0[NT], b1[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4], z[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              w[c] = pr[nt][c] * sv[gr][c >> 1];
              z[c] = pr[nt][c] * vp[gr][c >> 1].y;
              if (masked && hide[nt][c]) w[c] = z[c] = 0.f;
            }
            low[gr][nt][0] += z[0] + z[2];
            low[gr][nt][1] += z[1] + z[3];
            b0[nt] = movmatrix_trans(Mma<__half>::pack(w[0], w[1]));
            b1[nt] = movmatrix_trans(Mma<__half>::pack(w[2], w[3]));
          }
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t v0 = vw[gr / G][0][gr % G * 2 + w], v1 = vw[gr / G][1][gr % G * 2 + w];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                Mma<__half>::run(o[gr][2 * w + h][nt], v0 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x000f000fu,
                                 v1 & 0x00f000f0u, b0[nt], b1[nt]);
              v0 >>= 8, v1 >>= 8;
            }
          }
        }
      }
      if (dead)  // leave no copy in flight behind
        for (; it != issued; ++it) mbar_wait_bounded(bars + 8 * (it % STAGES), (it / STAGES) & 1, 1u << 16);

      // ---- the unit's result, or this warp's part of it
      const float v_up = v_down == 0.f ? 0.f : 16777216.f / v_down;
      const bool whole = blk0 == 0 && n == row.nblk;
      const bool last_run = pos + n == stop;
      float* po = reinterpret_cast<float*>(last_run ? ring : ring + S::kRing);
      __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float lt = l[nt][h];
#pragma unroll
          for (int k = 4; k <= 16; k <<= 1) lt += __shfl_xor_sync(kFull, lt, k);
          const int col = nt * 8 + 2 * t + h;
          const float mm = m[nt][h] == kNoMax ? -INFINITY : m[nt][h];
          const float inv = whole ? (lt == 0.f ? 0.f : 1.f / lt) : 1.f;
          const int tk = col / p.group, hd = col - tk * p.group;
          const int64_t tok = (int64_t)row.q_start + tok0 + tk;
#pragma unroll
          for (int gr = 0; gr < P * G; ++gr) {
            float z = low[gr][nt][h];
#pragma unroll
            for (int k = 4; k <= 16; k <<= 1) z += __shfl_xor_sync(kFull, z, k);
            if (col >= cols) continue;
            float v[8];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              v[2 * mt] = fmaf(o[gr][mt][nt][h], v_up, z) * inv;
              v[2 * mt + 1] = fmaf(o[gr][mt][nt][h + 2], v_up * 0.0625f, z) * inv;
            }
            const int dim = gr * 64 + g * 8;
            if (!whole) {
              float4* dst = reinterpret_cast<float4*>(po + col * D + dim);
              dst[0] = make_float4(v[0], v[1], v[2], v[3]);
              dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
              T* dst = reinterpret_cast<T*>(p.out) + tok * p.o_st + (int64_t)(kvh * p.group + hd) * p.o_sh + dim;
              T r8[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) r8[e] = Elem<T>::from_float(v[e]);
              if (p.vec) {
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(r8);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e] = r8[e];
              }
            }
          }
          if (g == 0 && col < cols) {
            if (!whole) {
              po[kCols * D + 2 * col] = mm;
              po[kCols * D + 2 * col + 1] = lt;
            } else {
              p.lse[tok * p.lse_st + kvh * p.group + hd] = lt == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(lt));
            }
          }
        }
      if (!whole && lane == 0) {
        const int64_t first = pos - blk0;
        parts[warp * 2 + (last_run ? 1 : 0)] = Part{first, first + row.nblk, r, tile, kvh, cols};
      }
      pos += n;
      off += n;
    }
  }

  // ---- join the parts. Neighbours of one unit are neighbours in the list; a warp takes a column.
  __syncthreads();
  const float* base = reinterpret_cast<const float*>(smem + S::kWarps);
  auto part_at = [&](int i) { return base + ((i >> 1) * S::kWarp + ((i & 1) ? 0 : S::kRing)) / 4; };
  int job = 0;
  for (int i = 0; i < 2 * NW;) {
    const Part pt = parts[i];
    if (pt.unit < 0) {
      ++i;
      continue;
    }
    int n = 0, j = i;
    unsigned list = 0;  // bit k: entry k is a part of this unit
    for (; j < 2 * NW; ++j) {
      if (parts[j].unit < 0) continue;
      if (parts[j].unit != pt.unit) break;
      list |= 1u << j;
      ++n;
    }
    i = j;
    for (int col = 0; col < pt.cols; ++col, ++job) {
      if (job % NW != warp) continue;
      float o[D / 32], m, l;
      join<D, false>(n, lane, [&](int k, const float*& row, const float2*& ml) {
        const float* at = part_at(__fns(list, 0, k + 1));
        row = at + col * D;
        ml = reinterpret_cast<const float2*>(at + kCols * D) + col;
      }, o, m, l);
      if (pt.unit < cta0 || pt.end > cta1) {  // the unit goes on in other CTAs
        const int64_t span = NW * per;
        const int first = (int)(pt.unit / span), last = (int)((pt.end - 1) / span);
        const int64_t slot = ((int64_t)blockIdx.x * 2 + (pt.unit >= cta0 ? 1 : 0)) * kCols + col;
        float* dst = p.ws_o + slot * D + lane * (D / 32);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) dst[e] = o[e];
        if (lane == 0) reinterpret_cast<float2*>(p.ws_ml)[slot] = make_float2(m, l);
        __threadfence();
        __syncwarp();
        int32_t* ctr = g_q4_counters[p.counter_slot] + first * kCols + col;
        int arrived = 0;
        if (lane == 0) arrived = atomicAdd(ctr, 1);
        arrived = __shfl_sync(kFull, arrived, 0);
        if (arrived != last - first) continue;
        if (lane == 0) *ctr = 0;
        __threadfence();
        join<D, true>(last - first + 1, lane, [&](int k, const float*& row, const float2*& ml) {
          const int64_t at = ((int64_t)(first + k) * 2 + (k == 0 ? 1 : 0)) * kCols + col;
          row = p.ws_o + at * D;
          ml = reinterpret_cast<const float2*>(p.ws_ml) + at;
        }, o, m, l);
      }
      const int tk = col / p.group, hd = col - tk * p.group;
      const int64_t tok = (int64_t)__ldg(p.q_starts + pt.row) + pt.tile * p.tile + tk;
      const int head = pt.kvh * p.group + hd;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* dst = reinterpret_cast<T*>(p.out) + tok * p.o_st + (int64_t)head * p.o_sh + lane * (D / 32);
#pragma unroll
      for (int e = 0; e < D / 32; ++e) dst[e] = Elem<T>::from_float(o[e] * inv);
      if (lane == 0) p.lse[tok * p.lse_st + head] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
    }
  }
}

// Warps of a CTA and CTAs of an SM by the columns of a warp's tile, as registers allow.
template <int D, int NT>
struct Shape {
  static constexpr int kRegs = D / 64 * NT;  // a measure of the tile's accumulators
  static constexpr int kWarps = kRegs <= 2 ? 8 : kRegs <= 4 ? 4 : 6;
  static constexpr int kCtas = kRegs <= 2 ? 2 : kRegs <= 4 ? 3 : 1;
  static constexpr int kStages = D == 256 ? 2 : 4;
};

// Columns (in eights) of a warp's tile: enough for the group, and for the tokens of an average row.
int tiles_of_columns(int group, int head_dim, int rows, int total_query) {
  const int most = head_dim == 256 ? 2 : 4;
  const int64_t tokens = (total_query + (int64_t)rows - 1) / rows;
  const int64_t cols = group * std::max<int64_t>(tokens, 1);
  int nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  if (group > 8 && nt < 2) nt = 2;
  return std::min(nt, most);
}

template <int D, int NT>
int grid_of() {
  return std::min(num_sms() * Shape<D, NT>::kCtas, kMaxCtas);
}

template <int D, int NT>
int64_t workspace_of() {
  return grid_of<D, NT>() * 2ll * 8 * NT * (D + 2) * 4;
}

template <typename T, int D, int NT>
int launch(Q4Params& p, void* workspace, int64_t bytes, cudaStream_t s) {
  using Sh = Shape<D, NT>;
  constexpr auto kern = q4_attention_kernel<T, D, NT, Sh::kWarps, Sh::kStages, Sh::kCtas>;
  constexpr int smem = Smem<D, NT, Sh::kWarps, Sh::kStages>::kBytes;
  static_assert(smem * Sh::kCtas <= 227 * 1024 - Sh::kCtas * 1024, "CTAs do not fit an SM");
  const int64_t need = workspace_of<D, NT>();
  if (workspace == nullptr || bytes < need || !aligned(workspace, 16)) {
    set_error("seb_paged_attention_q4: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)need,
              (long long)bytes);
    return SEB_EWORKSPACE;
  }
  const int ctas = grid_of<D, NT>();
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = p.ws_o + (int64_t)ctas * 2 * 8 * NT * D;
  p.tile = std::max(1, 8 * NT / p.group);
  const int rc = set_smem_limit_once<kern>(smem);
  if (rc != SEB_OK) return rc;
  kern<<<ctas, Sh::kWarps * 32, smem, s>>>(p);
  return launch_status("q4_attention_kernel");
}

template <typename T>
int launch_shape(Q4Params& p, int d, int nt, void* workspace, int64_t bytes, cudaStream_t s) {
  if (d == 64)
    return nt == 1 ? launch<T, 64, 1>(p, workspace, bytes, s)
                   : nt == 2 ? launch<T, 64, 2>(p, workspace, bytes, s) : launch<T, 64, 4>(p, workspace, bytes, s);
  if (d == 128)
    return nt == 1 ? launch<T, 128, 1>(p, workspace, bytes, s)
                   : nt == 2 ? launch<T, 128, 2>(p, workspace, bytes, s) : launch<T, 128, 4>(p, workspace, bytes, s);
  return nt == 1 ? launch<T, 256, 1>(p, workspace, bytes, s) : launch<T, 256, 2>(p, workspace, bytes, s);
}

}  // namespace
}  // namespace seb

extern "C" int64_t seb_paged_attention_q4_workspace_size(int32_t num_rows, int32_t total_query, int32_t num_q_heads,
                                                         int32_t num_kv_heads, int32_t head_dim) {
  using namespace seb;
  if (num_rows <= 0 || total_query <= 0 || num_q_heads <= 0 || num_kv_heads <= 0) return 0;
  const int nt = tiles_of_columns(num_q_heads / num_kv_heads, head_dim, num_rows, total_query);
  if (head_dim == 64) return nt == 1 ? workspace_of<64, 1>() : nt == 2 ? workspace_of<64, 2>() : workspace_of<64, 4>();
  if (head_dim == 128)
    return nt == 1 ? workspace_of<128, 1>() : nt == 2 ? workspace_of<128, 2>() : workspace_of<128, 4>();
  return head_dim == 256 ? (nt == 1 ? workspace_of<256, 1>() : workspace_of<256, 2>()) : 0;
}

extern "C" int seb_paged_attention_q4(const void* q, int64_t q_stride_token, int64_t q_stride_head,
                                      const void* k_cache, const void* v_cache, int64_t num_blocks,
                                      const int32_t* block_table, int64_t block_table_stride, int64_t max_blocks,
                                      const int32_t* q_starts, const int32_t* q_lens, const int32_t* k_lens,
                                      const int32_t* q_pos_offsets, int32_t num_rows, int32_t total_query,
                                      int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                                      float scale, int32_t is_causal, void* out, int64_t out_stride_token,
                                      int64_t out_stride_head, float* lse, int64_t lse_stride_token, void* workspace,
                                      int64_t workspace_bytes, int32_t counter_slot, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(dtype == SEB_BF16 || dtype == SEB_F16, "seb_paged_attention_q4: bf16 or fp16 required (dtype %d)",
                dtype);
  SEB_CHECK_ARG(num_rows >= 0 && total_query >= 0, "seb_paged_attention_q4: negative count");
  SEB_CHECK_ARG(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
                "seb_paged_attention_q4: num_q_heads (%d) must be a positive multiple of num_kv_heads (%d)",
                num_q_heads, num_kv_heads);
  const int group = num_q_heads / num_kv_heads;
  SEB_CHECK_ARG(group <= 16, "seb_paged_attention_q4: GQA group %d > 16 not supported", group);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("seb_paged_attention_q4: head_dim %d not supported (64, 128, 256)", head_dim);
    return SEB_EUNSUPPORTED;
  }
  if (num_rows == 0 || total_query == 0) return SEB_OK;
  SEB_CHECK_ARG(q && k_cache && v_cache && block_table && q_starts && q_lens && k_lens && q_pos_offsets && out && lse,
                "seb_paged_attention_q4: NULL pointer argument");
  SEB_CHECK_ARG(num_blocks > 0 && max_blocks > 0 && block_table_stride >= max_blocks,
                "seb_paged_attention_q4: bad block table shape (num_blocks %lld, max_blocks %lld, stride %lld)",
                (long long)num_blocks, (long long)max_blocks, (long long)block_table_stride);
  SEB_CHECK_ARG(max_blocks <= (1 << 26), "seb_paged_attention_q4: max_blocks %lld too large", (long long)max_blocks);
  SEB_CHECK_ARG(aligned(k_cache, 16) && aligned(v_cache, 16), "seb_paged_attention_q4: the pool must be 16-byte aligned");
  SEB_CHECK_ARG(counter_slot >= 0 && counter_slot < SEB_Q4_COUNTER_SLOTS,
                "seb_paged_attention_q4: counter_slot %d outside [0, %d)", counter_slot, SEB_Q4_COUNTER_SLOTS);
  Q4Params p{};
  p.counter_slot = counter_slot;
  p.q = static_cast<const char*>(q);
  p.q_st = q_stride_token;
  p.q_sh = q_stride_head;
  p.k_cache = static_cast<const char*>(k_cache);
  p.v_cache = static_cast<const char*>(v_cache);
  p.num_blocks = num_blocks;
  p.block_table = block_table;
  p.bt_stride = block_table_stride;
  p.max_blocks = max_blocks;
  p.q_starts = q_starts;
  p.q_lens = q_lens;
  p.k_lens = k_lens;
  p.q_pos = q_pos_offsets;
  p.num_rows = num_rows;
  p.total_query = total_query;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = group;
  p.scale_log2 = scale * kLog2e;
  p.causal = is_causal ? 1 : 0;
  p.vec = aligned(q, 16) && aligned(out, 16) && q_stride_token % 8 == 0 && q_stride_head % 8 == 0 &&
          out_stride_token % 8 == 0 && out_stride_head % 8 == 0;
  p.out = static_cast<char*>(out);
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.lse = lse;
  p.lse_st = lse_stride_token;
  p.err = err;
  const int nt = tiles_of_columns(group, head_dim, num_rows, total_query);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SEB_BF16 ? launch_shape<__nv_bfloat16>(p, head_dim, nt, workspace, workspace_bytes, s)
                           : launch_shape<__half>(p, head_dim, nt, workspace, workspace_bytes, s);
}
