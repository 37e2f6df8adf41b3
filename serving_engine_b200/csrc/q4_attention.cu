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
// p_j sV_jG becomes fp16 (unit 2^-11), p_j counting from a reference that keeps it below 2^15: each column's
// own, from the largest p_j sV_jG of the keys that it sees, so that no other key, and none of no weight,
// costs those that count their bits. Where O is fp16 it is the sum of two such numbers, a product for each:
// with one, O was off by 2.9e-4 and 3.7e-4 (256 rows, heads of 64; 2 of 120,000 keys) where its own rounding
// is 2.1e-4, with two by 2.1e-4 and 2.6e-4, for 48 us instead of 45 and 85 instead of 73. In bf16 its own
// rounding (1.7e-3) hides either. Scores, maxima, sums and O are fp32.
//
// Work: a unit is (row, tile of tokens, kv head) and its blocks, taken in pairs; the units
// of all rows laid end to end are cut in equal runs of pairs, one per resident warp,
// whatever the rows' lengths. A warp keeps all query heads of the group (and several tokens of
// a row, up to 8 * NT columns) on one tile, so each KV byte is read once per tile.
// Parts of a unit are joined in shared memory, and over CTAs in the workspace by the
// last to arrive, in order of their place, so results do not depend on timing.
#include "q4_attention.cuh"
#include "seb_softmax.cuh"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace seb {
namespace {

// Pairs of blocks of the shortest run worth a warp. One row of 75 / 200 / 1500 / 6000 keys, 8 kv heads of
// 128, us: 1: 7.7 / 10.6 / 12.0 / 19.8; 2: 8.9 / 8.6 / 12.9 / 16.0; 4: 15.0 / 16.3 / 15.3 / 16.4.
constexpr uint32_t kMinRun = 2;
// What a unit's start and end cost a warp, in pairs of blocks. 256 rows of 32 to 4352 keys, heads of 64:
// 0: 55.6 us, 1: 49.2, 2: 45.1, 3: 44.8, 4: 44.6, 6: 45.9; 64 rows of 1024 to 8192, heads of 128: 1 84.2, 2 83.6, 3 83.6.
constexpr uint32_t kUnitCost = 2;
// The reference of a column's exponents is where the largest p * scale is 2^8, and moved when one passes 2^15: what
// is 2^-22 of that one is still not subnormal in fp16. (p itself stays below 2^45, in fp32.)
constexpr float kNoMax = -FLT_MAX;  // no key yet: any score passes it
constexpr float kScaleTop = 15.f, kScalePlace = 8.f;

// Arrivals at the units that span CTAs, one for each four columns, at the CTA that a unit
// starts in. Zero when the library is loaded, and again after every call (the last to
// arrive clears it); calls that may overlap use different slots.
constexpr int kMaxCtas = 512;
__device__ int32_t g_q4_counters[SEB_Q4_COUNTER_SLOTS][kMaxCtas * 4];

// What the units of a call may come to, in such places: less than 32 bits hold by what rounding each thread's
// sum down to 2^12 hides (512 threads at most).
constexpr uint32_t kMostWork = 0xffe00000u;

// A unit's length in the run of all units: kUnitCost places that stand for no blocks, then its pairs.
__device__ __forceinline__ uint32_t length_of(const Row& w) { return w.pairs + kUnitCost; }
__device__ __forceinline__ uint32_t pairs_of(const Q4Params& p, const Row& w) { return w.tiles * p.hkv * length_of(w); }

// What a warp leaves of a unit that it did not do alone.
struct Part {
  uint32_t unit;  // the unit's first place in the run of all units
  uint32_t end;   // and past its last; 0: no part
  int64_t token;  // the tile's first
  int kvh, cols;
};

// Shared memory: parts, prefix sums and barriers, then for each warp its ring of pairs
// of blocks and room for the first of its two parts (the last one goes where the ring was).
template <int D, int NT, int NW, int STAGES>
struct Smem {
  static constexpr int kCols = 8 * NT;
  static constexpr int kStage = 4 * q4::Layout<D>::kRow;  // K and V rows of two blocks
  static constexpr int kPartBytes = kCols * (D + 2) * 4;
  static constexpr int kRing = STAGES * kStage > kPartBytes ? STAGES * kStage : kPartBytes;
  static constexpr int kWarp = (kRing + kPartBytes + 127) / 128 * 128;
  static constexpr int kParts = 0;                                     // Part[NW][2]
  static constexpr int kPrefix = kParts + NW * 2 * (int)sizeof(Part);  // uint32 [NW * 32 + 2]
  static constexpr int kMuch = kPrefix + (NW * 32 + 2) * 4;            // uint32 [NW]
  static constexpr int kBars = kMuch + NW * 4;
  static constexpr int kWarps = (kBars + NW * STAGES * 8 + 127) / 128 * 128;
  static constexpr int kBytes = kWarps + NW * kWarp;
};

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The token, of its tile, of a column.
__device__ __forceinline__ int token_of(const Q4Params& p, int col) { return (int)(col * p.by_group >> 16); }

// Lane l's dims l * D / 32 and on of a row of floats.
template <int D, bool GLOBAL>
__device__ __forceinline__ void load_dims(const float* row, int lane, float (&v)[D / 32]) {
  constexpr int DL = D / 32;
  if constexpr (DL == 2) {
    const float2* at = reinterpret_cast<const float2*>(row) + lane;
    const float2 x = GLOBAL ? __ldcg(at) : *at;
    v[0] = x.x, v[1] = x.y;
  } else {
#pragma unroll
    for (int c = 0; c < DL / 4; ++c) {
      const float4* at = reinterpret_cast<const float4*>(row) + lane * (DL / 4) + c;
      const float4 x = GLOBAL ? __ldcg(at) : *at;
      v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
    }
  }
}

// Joins `n` parts of up to four columns. Lane l gets its dims of each column's sum of O, and
// lanes 8 c .. 8 c + 7 have column c's reference m and sum l. part(i) is where part i's O
// rows and, `ml` floats on, (m, l) pairs begin, those of the first of the columns.
template <int D, bool GLOBAL, typename F>
__device__ __forceinline__ void join(int n, int cols, int lane, F part, int ml, float (&o)[4][D / 32], float& m,
                                     float& l) {
  constexpr int DL = D / 32;
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < DL; ++e) o[c][e] = 0.f;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 8) {
    float2 mine = make_float2(-INFINITY, 0.f);
    if (i0 + (lane & 7) < n && (lane >> 3) < cols) {
      const float2* at = reinterpret_cast<const float2*>(part(i0 + (lane & 7)) + ml) + (lane >> 3);
      mine = GLOBAL ? __ldcg(at) : *at;
    }
    float top = fmaxf(m, mine.x);
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
    const float ref = top == -INFINITY ? 0.f : top;
    const float keep = fast_exp2(m - ref), w = fast_exp2(mine.x - ref);
    float sum = mine.y * w;
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
    l = fmaf(l, keep, sum);
    m = top;
    if (i0 > 0) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float k = __shfl_sync(kFull, keep, 8 * c);
#pragma unroll
        for (int e = 0; e < DL; ++e) o[c][e] *= k;
      }
    }
    const int cnt = min(8, n - i0);
#pragma unroll(GLOBAL ? 4 : 2)
    for (int k = 0; k < cnt; ++k) {
      const float* row = part(i0 + k);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float wk = __shfl_sync(kFull, w, 8 * c + k);
        if (c < cols) {
          float v[DL];
          load_dims<D, GLOBAL>(row + c * D, lane, v);
#pragma unroll
          for (int e = 0; e < DL; ++e) o[c][e] = fmaf(wk, v[e], o[c][e]);
        }
      }
    }
  }
}

// One column's result: O / l and LSE, by a warp.
template <typename T, int D>
__device__ __forceinline__ void write_column(const Q4Params& p, int64_t token, int kvh, int col, int lane,
                                             const float (&o)[D / 32], float m, float l) {
  constexpr int DL = D / 32;
  const int tk = token_of(p, col);
  const int64_t tok = token + tk;
  const int head = kvh * p.group + col - tk * p.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* dst = reinterpret_cast<T*>(p.out) + tok * p.o_st + (int64_t)head * p.o_sh + lane * DL;
  T r[DL];
#pragma unroll
  for (int e = 0; e < DL; ++e) r[e] = Elem<T>::from_float(o[e] * inv);
  if constexpr (DL == 2) *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(r);
  else if constexpr (DL == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(r);
  else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(r);
  if (lane == 0) p.lse[tok * p.lse_st + head] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
}

// D = A B on fp16 operands, m16n8k16.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// What a warp keeps of the unit it is on.
template <int D, int NT>
struct Tile {
  static constexpr int GR = D / q4::kGroup;
  uint32_t qf[GR][NT][4][2];  // Q as the B operand: column 8 nt + g, dims 16 t .. 16 t + 15 of every group
  float qs[GR][NT][2];        // sum of q over a group, columns 8 nt + 2 t and the next
  float ch[NT][2];            // what brings a score to log2 units
  float m[NT][2], l[NT][2];   // reference, and this lane's share of the sum
  float low[GR][NT][2];       // this lane's share of sum p (low + 8 scale)
  float one[(GR + 1) / 2][NT][4];  // sum of the rounded p * scale, two groups to a tile
  float o[GR][4][NT][4];      // sum of those and the codes: n of a dim, and 16 n of the next
};

// From the sums over codes, 8 times the sum of what they were taken by, which is then counted
// from here. The tensor cores cut a sum off where they add to it, so that each step costs it up
// to 2^-23 of itself, always towards zero. The codes' sums only grow, and what they stand for is
// the small rest once 8 of each code is taken off: over a long run the cuts would be what is
// left (120,000 keys: 1.1e-2 of O; taken off every 256 keys 2.9e-4, 128 2.8e-4, 64 2.6e-4, where O in fp16
// alone is 2.1e-4; the last costs 0.4 us of 83.4 at 64 decode rows).
constexpr int kCentreBlocks = 4;
template <int D, int NT>
__device__ __forceinline__ void centre(Tile<D, NT>& u) {
#pragma unroll
  for (int gr = 0; gr < D / q4::kGroup; ++gr)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float& one = u.one[gr / 2][nt][(gr & 1) * 2 + h];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          u.o[gr][mt][nt][h] = fmaf(one, -8.f * power2(-24), u.o[gr][mt][nt][h]);
          u.o[gr][mt][nt][h + 2] = fmaf(one, -128.f * power2(-24), u.o[gr][mt][nt][h + 2]);
        }
        one = 0.f;
      }
}

// A lane's share of the columns' queries, as they are.
template <typename T, int D, int NT>
struct Queries {
  typename Two<T>::type raw[NT][D / q4::kGroup][8];
};

template <typename T, int D, int NT>
__device__ __forceinline__ void fetch_queries(const Q4Params& p, Queries<T, D, NT>& q, int64_t token, int kvh, int cols,
                                              int lane) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = nt * 8 + (lane >> 2);
    const bool live = col < cols;
    const int tk = live ? token_of(p, col) : 0, hd = live ? col - tk * p.group : 0;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (token + tk) * p.q_st +
                                                      (int64_t)(kvh * p.group + hd) * p.q_sh + 16 * (lane & 3));
#pragma unroll
    for (int gr = 0; gr < D / q4::kGroup; ++gr)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint4*>(&q.raw[nt][gr][4 * h]) = live ? __ldg(src + gr * 8 + h) : make_uint4(0u, 0u, 0u, 0u);
  }
}

// Scaled by a power of two for each column, so that fp16 holds them, as the B operand.
template <typename T, int D, int NT>
__device__ __forceinline__ void convert_queries(const Q4Params& p, Tile<D, NT>& u, const Queries<T, D, NT>& q, int lane) {
  constexpr int GR = D / q4::kGroup;
  const int t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const auto& raw = q.raw[nt];
    auto most = Two<T>::zero();
#pragma unroll
    for (int gr = 0; gr < GR; ++gr)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = __hmax2_nan(most, __habs2(raw[gr][e]));
    float top = q4::max_nan(Elem<T>::to_float(low_of(most)), Elem<T>::to_float(high_of(most)));
    top = q4::max_nan(top, __shfl_xor_sync(kFull, top, 1));
    top = q4::max_nan(top, __shfl_xor_sync(kFull, top, 2));
    const int ex = query_exponent(top);
    const float down = power2(-ex);
#pragma unroll
    for (int gr = 0; gr < GR; ++gr) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {  // pairs that meet lower codes and pairs that meet upper ones, in turn
        const float a = Elem<T>::to_float(low_of(raw[gr][w])) * down;
        const float b = Elem<T>::to_float(high_of(raw[gr][w])) * down;
        sum += a + b;
        u.qf[gr][nt][w >> 1][w & 1] = w & 1 ? Mma<__half>::pack(a * 0.0625f, b * 0.0625f) : Mma<__half>::pack(a, b);
      }
      sum += __shfl_xor_sync(kFull, sum, 1);
      sum += __shfl_xor_sync(kFull, sum, 2);
      sum *= power2(-24);  // as the codes carry it
      u.qs[gr][nt][0] = __shfl_sync(kFull, sum, 8 * t);
      u.qs[gr][nt][1] = __shfl_sync(kFull, sum, 8 * t + 4);
    }
    const float up = fminf(fminf(fabsf(p.scale_log2) * power2(24), FLT_MAX) * power2(ex), FLT_MAX);
    const float c = copysignf(up, p.scale_log2);
    u.ch[nt][0] = __shfl_sync(kFull, c, 8 * t);
    u.ch[nt][1] = __shfl_sync(kFull, c, 8 * t + 4);
  }
}

// A lane's words of a panel, and its tokens' (scale, low) pairs.
template <int G>
__device__ __forceinline__ void load_words(const char* at, uint32_t (&w)[2 * G]) {
  if constexpr (G == 2) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(at);
  else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(at);
}
template <int G>
__device__ __forceinline__ void load_pairs(const char* at, __half2 (&a)[G]) {
  if constexpr (G == 2) *reinterpret_cast<uint2*>(a) = *reinterpret_cast<const uint2*>(at);
  else *reinterpret_cast<uint32_t*>(a) = *reinterpret_cast<const uint32_t*>(at);
}

// What rounding two numbers to fp16 leaves of them.
__device__ __forceinline__ uint32_t rest(float a, float b) {
  const uint32_t w = Mma<__half>::pack(a, b);
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return Mma<__half>::pack(a - r.x, b - r.y);
}

// KB blocks of 16 keys. `place` holds their rows, K and V of one after the other. MASK: some
// key is not for every column; of keys key0 and on a column then sees those below its
// `end`, and none of block i where bit i of `unread` says that it has no data. FINE: p * scale in two parts.
template <bool FINE, int D, int NT, int KB, bool MASK>
__device__ __forceinline__ void take_blocks(Tile<D, NT>& u, const char* place, int lane, int key0, unsigned unread,
                                            const int (&end)[NT][2]) {
  using L = q4::Layout<D>;
  constexpr int P = L::kPanels, G = L::kGroups, GR = P * G;
  const int g = lane >> 2, t = lane & 3;
  auto hidden = [&](int b, int nt, int c) {
    return MASK && (((unread >> b) & 1) || key0 + 16 * b + g + 8 * (c >> 1) >= end[nt][c & 1]);
  };

  // S^T = K Q^T in log2 units: for each block 16 keys x 8 NT columns, one sum for each group
  float x[KB][NT][4];
#pragma unroll
  for (int b = 0; b < KB; ++b) {
#pragma unroll
    for (int pn = 0; pn < P; ++pn) {
      const char* kb = place + b * 2 * L::kRow;
      uint32_t w[2][2 * G];  // of keys g and g + 8
      __half2 pr[2][G];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_words<G>(kb + pn * 8 * L::kWidth + (g + 8 * h) * (L::kWidth / 2) + t * (8 * G), w[h]);
        load_pairs<G>(kb + L::kCodes + pn * 64 * G + (g + 8 * h) * 4 * G, pr[h]);
      }
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const int gr = pn * G + gi;
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t k0 = w[0][gi * 2 + i], k1 = w[1][gi * 2 + i];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = k0 & 0x000f000fu, a1 = k1 & 0x000f000fu, a2 = k0 & 0x00f000f0u, a3 = k1 & 0x00f000f0u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t(&q)[2] = u.qf[gr][nt][2 * i + h];
              if (i == 0 && h == 0) mma_first(acc[nt], a0, a1, a2, a3, q[0], q[1]);
              else Mma<__half>::run(acc[nt], a0, a1, a2, a3, q[0], q[1]);
            }
            k0 >>= 8, k1 >>= 8;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float scale = __low2float(pr[h][gi]), low = __high2float(pr[h][gi]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 2 * h; c < 2 * h + 2; ++c) {
              const float q = u.qs[gr][nt][c & 1];
              x[b][nt][c] = fmaf(scale, acc[nt][c], gr == 0 ? low * q : fmaf(low, q, x[b][nt][c]));
            }
        }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[b][nt][c] *= u.ch[nt][c & 1];
        if (hidden(b, nt, c)) x[b][nt][c] = -INFINITY;
      }
  }

  // The largest score of each column that this lane has. What p * scale may be is first bounded by it and
  // the largest scale, and worked out key by key only where that bound calls for a move: a column moves
  // for keys that it sees and no others.
  __half2 vp[KB][P][2][G];  // of keys g and g + 8
  float top[NT][2];
  __half2 most[KB][2];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int pn = 0; pn < P; ++pn)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_pairs<G>(place + (b * 2 + 1) * L::kRow + L::kCodes + pn * 64 * G + (g + 8 * h) * 4 * G, vp[b][pn][h]);
#pragma unroll
        for (int gi = 0; gi < G; ++gi)
          most[b][h] = pn + gi == 0 ? vp[b][pn][h][gi] : __hmax2(most[b][h], vp[b][pn][h][gi]);
      }
  auto log2_scale = [](__half2 pair) { return log2_fast(fmaxf(__low2float(pair), power2(-30))); };  // a NaN counts as 0
  __half2 largest = most[0][0];
#pragma unroll
  for (int b = 0; b < KB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (b + h > 0) largest = __hmax2(largest, most[b][h]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 2 * h; c < 2 * h + 2; ++c)
          top[nt][c & 1] = b + h == 0 ? x[b][nt][c] : fmaxf(top[nt][c & 1], x[b][nt][c]);
    }
  const float above = log2_scale(largest) - (kScaleTop - 0.01f);
  bool move = false;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      move |= top[nt][h] - u.m[nt][h] + above > 0.f;
    }
  if (__any_sync(kFull, move)) {
    // move the references of the columns that need it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = top[nt][h];
#pragma unroll
        for (int k = 4; k <= 16; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, k));
        float z = -INFINITY;  // log2 of the largest p * scale, as if the largest score were the reference
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          z = fmaxf(z, x[b][nt][h] - mx + log2_scale(most[b][0]));
          z = fmaxf(z, x[b][nt][h + 2] - mx + log2_scale(most[b][1]));
        }
#pragma unroll
        for (int k = 4; k <= 16; k <<= 1) z = fmaxf(z, __shfl_xor_sync(kFull, z, k));
        float fix = 1.f;
        if (mx - u.m[nt][h] + z > kScaleTop) {
          // at most the largest score, rounded up: scores may be so large that the sum is not exact
          const float now = __fadd_ru(mx, fminf(z - kScalePlace, 0.f));
          fix = fast_exp2(u.m[nt][h] - now);  // from kNoMax: 0
          u.m[nt][h] = now;
        }
        u.l[nt][h] *= fix;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
          u.low[gr][nt][h] *= fix;
          u.one[gr / 2][nt][(gr & 1) * 2 + h] *= fix;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            u.o[gr][mt][nt][h] *= fix;
            u.o[gr][mt][nt][h + 2] *= fix;
          }
        }
      }
  }

  // O^T += V^T (P scale)^T, and the lows' share. The codes count from 8 here: sum p scale n +
  // sum p low = sum p' (n - 8) + sum p (low + 8 scale) with p' = p scale rounded to fp16, so
  // that its rounding meets n - 8 and no more; sum p' is one more row of the product.
  // Keys that a column does not see have p = 0, and none of their parameters is used.
#pragma unroll
  for (int b = 0; b < KB; ++b) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[b][nt][c] = fast_exp2(x[b][nt][c] - u.m[nt][c & 1]);
      u.l[nt][0] += x[b][nt][0] + x[b][nt][2];
      u.l[nt][1] += x[b][nt][1] + x[b][nt][3];
    }
#pragma unroll
    for (int pn = 0; pn < P; ++pn) {
      const char* vb = place + (b * 2 + 1) * L::kRow + pn * 8 * L::kWidth + (g ^ L::turn(t)) * (8 * G);
      uint32_t w[2][2 * G];  // of key pairs t and t + 4
      load_words<G>(vb + t * L::kWidth, w[0]);
      load_words<G>(vb + (t + 4) * L::kWidth, w[1]);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        const int gr = pn * G + gi;
        uint32_t b0[NT], b1[NT], r0[NT], r1[NT];
        float z[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // A group that is NaN is so by its share of the lows alone: in the products it would make the
          // other group of the tile of sums NaN too.
          const float2 pair = __half22float2(vp[b][pn][h][gi]);
          const float scale = fmaxf(pair.x, 0.f), mid = fmaf(8.f, pair.x, pair.y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 2 * h; c < 2 * h + 2; ++c) {
              const bool hide = hidden(b, nt, c);
              z[nt][c] = hide ? 0.f : x[b][nt][c] * scale;
              u.low[gr][nt][c & 1] = fmaf(x[b][nt][c], hide ? 0.f : mid, u.low[gr][nt][c & 1]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          b0[nt] = movmatrix_trans(Mma<__half>::pack(z[nt][0], z[nt][1]));
          b1[nt] = movmatrix_trans(Mma<__half>::pack(z[nt][2], z[nt][3]));
          constexpr uint32_t kOnes = 0x3c003c00u;
          Mma<__half>::run(u.one[gr / 2][nt], gr & 1 ? 0u : kOnes, gr & 1 ? kOnes : 0u, gr & 1 ? 0u : kOnes,
                           gr & 1 ? kOnes : 0u, b0[nt], b1[nt]);
          if constexpr (FINE) {  // and what its rounding left
            r0[nt] = movmatrix_trans(rest(z[nt][0], z[nt][1]));
            r1[nt] = movmatrix_trans(rest(z[nt][2], z[nt][3]));
            Mma<__half>::run(u.one[gr / 2][nt], gr & 1 ? 0u : kOnes, gr & 1 ? kOnes : 0u, gr & 1 ? 0u : kOnes,
                             gr & 1 ? kOnes : 0u, r0[nt], r1[nt]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t v0 = w[0][gi * 2 + i], v1 = w[1][gi * 2 + i];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x0 = h ? v0 >> 8 : v0, x1 = h ? v1 >> 8 : v1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              Mma<__half>::run(u.o[gr][2 * i + h][nt], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu,
                               x1 & 0x00f000f0u, b0[nt], b1[nt]);
              if constexpr (FINE)
                Mma<__half>::run(u.o[gr][2 * i + h][nt], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu,
                                 x1 & 0x00f000f0u, r0[nt], r1[nt]);
            }
          }
        }
      }
    }
  }
}

template <typename T, int D, int NT, int NW, int STAGES, int CTAS>
__global__ void __launch_bounds__(NW * 32, CTAS) q4_attention_kernel(const Q4Params p) {
  using L = q4::Layout<D>;
  using S = Smem<D, NT, NW, STAGES>;
  constexpr int GR = D / q4::kGroup;
  constexpr int kCols = S::kCols;
  constexpr int kPart = kCols * (D + 2);  // floats of a part: O, then (m, l)
  extern __shared__ __align__(128) char smem[];
  Part* parts = reinterpret_cast<Part*>(smem + S::kParts);
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + S::kPrefix);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  if (p.chunk_from > 0)
    for (int i = blockIdx.x * (NW * 32) + tid; i < kChunkArrivals; i += gridDim.x * (NW * 32)) p.chunk_arrivals[i] = 0;

  // ---- the units of all rows, and this warp's run of blocks
  const int chunk = (p.num_rows + NW * 32 - 1) / (NW * 32);  // rows that a thread sums up
  {
    uint32_t bad = 0;
    uint64_t all = 0;
#pragma unroll 1
    for (int r = tid * chunk; r < min((tid + 1) * chunk, p.num_rows); ++r) {
      const Row row = row_of<false>(p, r, &bad);
      all += pairs_of(p, row);
      if (r == 0) prefix[NW * 32 + 1] = length_of(row);
    }
    if (bad && blockIdx.x == 0) atomic_or_err(p.err, bad);
    uint32_t sum = (uint32_t)all;
    const uint32_t much = __reduce_add_sync(kFull, (uint32_t)min(all >> 12, (uint64_t)1 << 22));
    if (lane == 0) reinterpret_cast<uint32_t*>(smem + S::kMuch)[warp] = much;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(kFull, sum, off);
      if (lane >= off) sum += o;
    }
    prefix[tid + 1] = sum;
    if (tid == 0) prefix[0] = 0;
    if (lane < 2) parts[warp * 2 + lane].end = 0;
  }
  __syncthreads();
  uint32_t total = 0, before = 0, much = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) before = total;
    total += prefix[(w + 1) * 32];
    much += reinterpret_cast<const uint32_t*>(smem + S::kMuch)[w];
  }
  if (much > kMostWork >> 12) {  // rows whose tokens overlap: the sums have passed 32 bits
    if (blockIdx.x == 0 && tid == 0) atomic_or_err(p.err, SEB_ERRBIT_META);
    return;
  }
  __syncthreads();
  prefix[tid + 1] += before;
  __syncthreads();
  const uint32_t warps = gridDim.x * NW;
  const uint32_t per = max((total + warps - 1) / warps, kMinRun);
  uint32_t span = NW * per;
  // Where CTAs are left over, those of whole units of the first row's length: no unit of that length is
  // then joined over CTAs (one row of 75 keys, 8 kv heads of 128: 13.0 us with such joins, 9 without).
  const uint32_t unit0 = prefix[NW * 32 + 1], even = span - span % unit0;
  if (per == kMinRun && even > 0 && (uint64_t)even * gridDim.x >= total) span = even;
  const uint32_t cta0 = blockIdx.x * span, cta1 = min(cta0 + span, total);
  if (cta0 >= total) return;
  uint32_t pos = cta0 + warp * per;
  const uint32_t stop = min(pos + per, cta1);

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
    uint32_t off = pos - prefix[lo], bad = 0;
    Row row = row_of<false>(p, r, &bad);
    uint32_t it = 0;  // pairs taken through the ring so far
    bool dead = false;

    while (pos < stop) {
      uint32_t len = pairs_of(p, row);
#pragma unroll 1
      while (off >= len && r + 1 < p.num_rows) {
        off -= len;
        row = row_of<false>(p, ++r, &bad);
        len = pairs_of(p, row);
      }
      if (off >= len) break;
      const uint32_t length = length_of(row);
      const uint32_t unit = off / length;  // tiles of one kv head are neighbours: they read the same blocks
      const uint32_t place = off - unit * length, n = min(length - place, stop - pos);
      const int kvh = (int)(unit / row.tiles), tile = (int)(unit - kvh * row.tiles);
      const int blk0 = 2 * max((int)(place - kUnitCost), 0);
      const int tok0 = tile * p.tile;  // first token of the tile in the row
      const int toks = min(p.tile, row.q_len - tok0);
      const int cols = toks * p.group;
      const int64_t token = (int64_t)row.q_start + tok0;
      // keys that the tile's first and last token see; each token sees one more than the one before it
      const int first_sees =
          p.causal ? (int)min((int64_t)row.q_pos + tok0 + 1, (int64_t)(1 << 30)) : row.k_len;
      const int see_all = min(row.k_len, max(first_sees, 0));
      const int see_any = p.causal ? min(row.k_len, max(first_sees + toks - 1, 0)) : row.k_len;
      const int blk1 = min(2 * (int)(place + n - kUnitCost), (see_any + 15) >> 4);  // blocks from here on hold nothing for this tile

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
      int ids = load_id(blk0 + lane);
      Queries<T, D, NT> queries;
      fetch_queries(p, queries, token, kvh, cols, lane);
      unsigned unread = 0;  // bits 2 s, 2 s + 1: that block of ring place s has no data
      uint32_t issued = it;
      // Stage blocks b and b + 1; called for blk0, blk0 + 2, ... in turn. Lanes 0..3 copy a row each.
      auto stage = [&](int b) {
        const int j = b - blk0;
        if (j > 0 && (j & 31) == 0) ids = load_id(b + lane);
        const int id = __shfl_sync(kFull, ids, (j + ((lane >> 1) & 1)) & 31);
        const unsigned read = __ballot_sync(kFull, id >= 0) & 5u;  // lanes 0 and 2
        const uint32_t s = issued % STAGES;
        const uint32_t bar = bars + 8 * s;
        unread = (unread & ~(3u << (2 * s))) | ((read & 1 ? 0u : 1u) | (read & 4 ? 0u : 2u)) << (2 * s);
        if (lane == 0) mbar_arrive_expect_tx(bar, __popc(read) * 2 * L::kRow);
        __syncwarp();
        if (lane < 4 && id >= 0) {
          const int64_t at = ((int64_t)id * p.hkv + kvh) * L::kRow;
          bulk_g2s(ring_a + s * S::kStage + lane * L::kRow, (lane & 1 ? p.v_cache : p.k_cache) + at, L::kRow, bar);
        }
        ++issued;
      };
      for (int b = blk0; b < min(blk0 + 2 * STAGES, blk1); b += 2) stage(b);

      Tile<D, NT> u;
      convert_queries(p, u, queries, lane);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u.m[nt][h] = kNoMax;
          u.l[nt][h] = 0.f;
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) u.low[gr][nt][h] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            u.one[gr / 2][nt][c] = 0.f;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) u.o[gr][mt][nt][c] = 0.f;
          }
      }
      int end[NT][2];  // keys that the lane's columns see
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          end[nt][h] = p.causal ? min(row.k_len, first_sees + token_of(p, nt * 8 + 2 * t + h)) : row.k_len;

      for (int b = blk0; b < blk1; b += 2, ++it) {
        const uint32_t s = it % STAGES;
        if (dead || !mbar_wait_bounded(bars + 8 * s, (it / STAGES) & 1)) {
          if (!dead && lane == 0) atomic_or_err(p.err, SEB_ERRBIT_TIMEOUT);
          dead = true;
          break;
        }
        const unsigned none = (unread >> (2 * s)) & 3;
        const char* place = ring + s * S::kStage;
        // two blocks at once where the tile leaves registers for it
        constexpr bool kFine = std::is_same<T, __half>::value;
        constexpr int KB = GR * NT <= 2 ? 2 : 1;
        if (none == 0 && (b + 2) * 16 <= see_all) {
#pragma unroll 1
          for (int i = 0; i < 2; i += KB)
            take_blocks<kFine, D, NT, KB, false>(u, place + i * 2 * L::kRow, lane, (b + i) * 16, 0, end);
        } else {
#pragma unroll 1
          for (int i = 0; i < 2; ++i)
            take_blocks<kFine, D, NT, 1, true>(u, place + i * 2 * L::kRow, lane, (b + i) * 16, (none >> i) & 1, end);
        }
        __syncwarp();  // every lane has read the place: it may be filled again
        if (((b - blk0) & (kCentreBlocks - 1)) == kCentreBlocks - 2) centre(u);
        if (b + 2 * STAGES < blk1) stage(b + 2 * STAGES);
      }
      if (dead)  // leave no copy in flight behind
        for (; it != issued; ++it) mbar_wait_bounded(bars + 8 * (it % STAGES), (it / STAGES) & 1, 1u << 16);

      // ---- the result, or this warp's part of it, by way of shared memory. Nothing is in flight to the ring now.
      const bool whole = n == length;
      const bool last_run = pos + n == stop;
      float* po = reinterpret_cast<float*>(whole || last_run ? ring : ring + S::kRing);
      __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = nt * 8 + 2 * t + h;
          constexpr float v_up = 16777216.f;  // 2^24, as the codes carry it
          float lt = u.l[nt][h];
#pragma unroll
          for (int k = 4; k <= 16; k <<= 1) lt += __shfl_xor_sync(kFull, lt, k);
#pragma unroll
          for (int gr = 0; gr < GR; ++gr) {
            float z = u.low[gr][nt][h];
#pragma unroll
            for (int k = 4; k <= 16; k <<= 1) z += __shfl_xor_sync(kFull, z, k);
            const float one = 8.f * power2(-24) * u.one[gr / 2][nt][(gr & 1) * 2 + h];
            float v[8];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              v[2 * mt] = fmaf(u.o[gr][mt][nt][h] - one, v_up, z);
              v[2 * mt + 1] = fmaf(fmaf(u.o[gr][mt][nt][h + 2], 0.0625f, -one), v_up, z);
            }
            if (col < cols) {
              float4* dst = reinterpret_cast<float4*>(po + col * D + gr * 64 + g * 8);
              dst[0] = make_float4(v[0], v[1], v[2], v[3]);
              dst[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
          if (g == 0 && col < cols)
            reinterpret_cast<float2*>(po + kCols * D)[col] =
                make_float2(lt == 0.f ? -INFINITY : u.m[nt][h], lt);
        }
      __syncwarp();
      if (whole) {
#pragma unroll 1
        for (int col = 0; col < cols; ++col) {
          float o[D / 32];
          load_dims<D, false>(po + col * D, lane, o);
          const float2 ml = reinterpret_cast<const float2*>(po + kCols * D)[col];
          write_column<T, D>(p, token, kvh, col, lane, o, ml.x, ml.y);
        }
      } else if (lane == 0) {
        parts[warp * 2 + (last_run ? 1 : 0)] = Part{pos - place, pos - place + length, token, kvh, cols};
      }
      fence_proxy_async_smem();  // the ring is written by copies next
      __syncwarp();
      pos += n;
      off += n;
    }
  }

  // ---- join the parts. A unit's parts are one of each of neighbouring warps, so in the list of
  // 2 NW places neighbours but for empty places; a bit of a mask stands for each place. A warp
  // takes four columns; of units that go on in other CTAs first, so that their arrival is early.
  __syncthreads();
  const float* base = reinterpret_cast<const float*>(smem + S::kWarps);
  uint32_t unit = 0, end = 0;
  if (lane < 2 * NW) {
    unit = parts[lane].unit;
    end = parts[lane].end;
  }
  const unsigned used = __ballot_sync(kFull, end != 0);
  const unsigned below = used & ((1u << lane) - 1);
  const uint32_t before_me = __shfl_sync(kFull, unit, below ? 31 - __clz(below) : 0);
  const unsigned starts = __ballot_sync(kFull, end != 0 && (below == 0 || before_me != unit));
  const unsigned spanning = __ballot_sync(kFull, end != 0 && (unit < cta0 || end > cta1)) & starts;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int job = 0;
#pragma unroll 1
    for (unsigned left = pass == 0 ? spanning : starts & ~spanning; left; left &= left - 1) {
      const int i = __ffs(left) - 1, w0 = i >> 1;
      const unsigned later = starts & ~((2u << i) - 1);  // the next unit's first place and on
      const unsigned list = used & ~((1u << i) - 1) & (later ? (1u << (__ffs(later) - 1)) - 1 : ~0u);
      const Part pt = parts[i];
#pragma unroll 1
      for (int col = 0; col < pt.cols; col += 4, ++job) {
        if (job % NW != warp) continue;
        const int cols = min(4, pt.cols - col);
        float o[4][D / 32], m, l;
        join<D, false>(__popc(list), cols, lane, [&](int k) {
          return base + ((w0 + k) * S::kWarp + (list >> (2 * (w0 + k)) & 1 ? S::kRing : 0)) / 4 + col * D;
        }, kCols * D - col * D + 2 * col, o, m, l);
        if (pass == 0) {
          const int first = pt.unit / span, last = (pt.end - 1) / span;
          const int64_t slot = ((int64_t)blockIdx.x * 2 + (pt.unit >= cta0 ? 1 : 0)) * kPart;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < cols) {
              float* dst = p.ws + slot + (col + c) * D + lane * (D / 32);
#pragma unroll
              for (int e = 0; e < D / 32; ++e) dst[e] = o[c][e];
            }
          if ((lane & 7) == 0 && (lane >> 3) < cols)
            reinterpret_cast<float2*>(p.ws + slot + kCols * D)[col + (lane >> 3)] = make_float2(m, l);
          __threadfence();
          __syncwarp();
          int32_t* ctr = g_q4_counters[p.counter_slot] + (first * kCols + col) / 4;
          int arrived = 0;
          if (lane == 0) arrived = atomicAdd(ctr, 1);
          arrived = __shfl_sync(kFull, arrived, 0);
          if (arrived != last - first) continue;
          if (lane == 0) *ctr = 0;
          __threadfence();
          join<D, true>(last - first + 1, cols, lane, [&](int k) {
            return p.ws + ((int64_t)(first + k) * 2 + (k == 0 ? 1 : 0)) * kPart + col * D;
          }, kCols * D - col * D + 2 * col, o, m, l);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float mc = __shfl_sync(kFull, m, 8 * c), lc = __shfl_sync(kFull, l, 8 * c);
          if (c < cols) write_column<T, D>(p, pt.token, pt.kvh, col + c, lane, o[c], mc, lc);
        }
      }
    }
  }
}

// Warps of a CTA and CTAs of an SM by the columns of a warp's tile, as registers allow: the more
// warps the more hides a warp's waits, until two blocks at once, which do as much, no longer fit. Heads
// of 128, one tile of columns (64 rows of 1024 to 8192 keys; 2 of 120,000 to 131,072; 1 of 75), us, all with
// p * scale in one part:
// 2 x 8 warps, a block at a time 87.5, 77.1, 14.0; 2 x 7 96.3, 83.8, 14.1; 2 x 6 87.3, 76.7, 12.9; 2 x 6, two
// blocks 83.7, 73.7, 13.0; 2 x 5, two blocks 98.1, 85.3, 8.8; 1 x 12, two blocks 83.4, 71.5, 14.3.
// Heads of 64: 2 x 8 44.6 (256 rows), 2 x 7 48.7, 2 x 6 47.8; two tiles of columns of 64 (48 rows of 2
// tokens, 3000 keys): 2 x 6, two blocks 48.7, one 49.4; 2 x 8 51.2. Two tiles of 128: 2 x 4 196 (48 rows of
// drafts, with their chunks), 2 x 5 214. Heads of 256, 2 x 4 with one ring stage: 172 us (the 64 rows, bf16);
// their two tiles of columns (groups above 8) spill some 700 bytes.
template <int D, int NT>
struct Shape {
  static constexpr int kSize = D / 64 * NT;  // a measure of the tile's accumulators
  static constexpr int kWarps = kSize == 1 ? 8 : kSize == 2 ? 6 : kSize <= 4 ? 4 : 6;
  static constexpr int kCtas = kSize <= 2 ? 2 : kSize <= 4 ? 2 : 1;
  static constexpr int kStages = D == 64 ? 4 : D == 128 ? 2 : 1;
};

// (token, query head of a group) pairs from which a row is a chunk. Measured at 48 rows of 1 to 8
// drafted tokens, 64/8 heads of 128, up to 6000 keys: from 16 256 us, 24 240, 32 226, 48 211; no chunks 293.
constexpr int kChunkFrom = 48;
bool may_have_chunks(int head_dim, int rows, int total_query) { return head_dim <= 128 && total_query > rows; }

// Columns (in eights) of a warp's tile: enough for the group, and for more tokens where rows
// have several and the registers hold them.
int column_tiles(int group, int head_dim, int rows, int total_query) {
  return group > 8 || (total_query > rows && head_dim <= 128) ? 2 : 1;
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
  const int64_t need = std::max(workspace_of<D, NT>(), p.chunk_from > 0 ? q4_prefill_workspace(D) + kChunkArrivals * 4 : 0);
  if (workspace == nullptr || bytes < need || !aligned(workspace, 16)) {
    set_error("seb_paged_attention_q4: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)need,
              (long long)bytes);
    return SEB_EWORKSPACE;
  }
  const int ctas = grid_of<D, NT>();
  p.ws = static_cast<float*>(workspace);
  if (p.chunk_from > 0) p.chunk_arrivals = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + q4_prefill_workspace(D));
  p.tile = std::max(1, 8 * NT / p.group);
  p.by_group = (65536 + p.group - 1) / p.group;
  const int rc = set_smem_limit_once<kern>(smem);
  if (rc != SEB_OK) return rc;
  // no more CTAs than the longest rows that the table allows would fill; where there may be chunks, rows that
  // are none have fewer tokens than one
  int64_t tiles = ((int64_t)p.total_query + (int64_t)p.num_rows * (p.tile - 1)) / p.tile;
  if (p.chunk_from > 0)
    tiles = std::min<int64_t>(tiles, (int64_t)p.num_rows * (((p.chunk_from - 1) / p.group + p.tile - 1) / p.tile));
  const int64_t pairs = tiles * p.hkv * ((p.max_blocks + 1) / 2 + kUnitCost);
  if (pairs > (int64_t)kMostWork) {
    set_error("seb_paged_attention_q4: %lld tiles of %lld blocks are too much work for one call", (long long)tiles * p.hkv,
              (long long)p.max_blocks);
    return SEB_EUNSUPPORTED;
  }
  // (a CTA may take little more than half of its warps' shortest runs, see `even`)
  const int64_t most = 2 * pairs / (Sh::kWarps * kMinRun) + 1;
  kern<<<(unsigned)std::min<int64_t>(ctas, most), Sh::kWarps * 32, smem, s>>>(p);
  return launch_status("q4_attention_kernel");
}

template <typename T, int D>
int launch_columns(Q4Params& p, int nt, void* workspace, int64_t bytes, cudaStream_t s) {
  return nt == 1 ? launch<T, D, 1>(p, workspace, bytes, s) : launch<T, D, 2>(p, workspace, bytes, s);
}

template <typename T>
int launch_dim(Q4Params& p, int d, int nt, void* workspace, int64_t bytes, cudaStream_t s) {
  return d == 64 ? launch_columns<T, 64>(p, nt, workspace, bytes, s)
                 : d == 128 ? launch_columns<T, 128>(p, nt, workspace, bytes, s)
                            : launch_columns<T, 256>(p, nt, workspace, bytes, s);
}

}  // namespace
}  // namespace seb

extern "C" int64_t seb_paged_attention_q4_workspace_size(int32_t num_rows, int32_t total_query, int32_t num_q_heads,
                                                         int32_t num_kv_heads, int32_t head_dim) {
  using namespace seb;
  if (num_rows <= 0 || total_query <= 0 || num_q_heads <= 0 || num_kv_heads <= 0) return 0;
  const int nt = column_tiles(num_q_heads / num_kv_heads, head_dim, num_rows, total_query);
  const int64_t chunks = may_have_chunks(head_dim, num_rows, total_query) ? q4_prefill_workspace(head_dim) + kChunkArrivals * 4 : 0;
  if (head_dim == 64) return std::max(chunks, nt == 1 ? workspace_of<64, 1>() : workspace_of<64, 2>());
  if (head_dim == 128) return std::max(chunks, nt == 1 ? workspace_of<128, 1>() : workspace_of<128, 2>());
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
  SEB_CHECK_ARG(aligned(q, 16) && aligned(out, 16) && q_stride_token % 8 == 0 && q_stride_head % 8 == 0 &&
                    out_stride_token % 8 == 0 && out_stride_head % 8 == 0,
                "seb_paged_attention_q4: rows of q and out must be 16-byte aligned");
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
  p.out = static_cast<char*>(out);
  p.o_st = out_stride_token;
  p.o_sh = out_stride_head;
  p.lse = lse;
  p.lse_st = lse_stride_token;
  p.err = err;
  p.chunk_from = may_have_chunks(head_dim, num_rows, total_query) ? kChunkFrom : 0;
  const int nt = column_tiles(group, head_dim, num_rows, total_query);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = dtype == SEB_BF16 ? launch_dim<__nv_bfloat16>(p, head_dim, nt, workspace, workspace_bytes, s)
                                   : launch_dim<__half>(p, head_dim, nt, workspace, workspace_bytes, s);
  if (rc != SEB_OK || p.chunk_from == 0) return rc;
  return launch_q4_prefill(p, head_dim, dtype, s);
}
