// What the two kernels of paged attention over a 4-bit pool share: their arguments and
// the rows. Rows of a few tokens go to q4_attention.cu, chunks to q4_prefill.cu.
#pragma once

#include "q4_format.cuh"

namespace seb {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

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
  int32_t chunk_from;  // rows of this many (token, query head of a group) pairs and more are chunks; 0: none are
  int32_t tile;       // tokens of a tile
  uint32_t by_group;  // col / group == col * by_group >> 16 for the columns of a tile
  float scale_log2;
  int32_t causal;
  char* out;
  int64_t o_st, o_sh;  // elements
  float* lse;
  int64_t lse_st;
  int32_t counter_slot;
  float* ws;           // what CTAs leave of units that others share; each kernel has its own layout
  int32_t* chunk_arrivals;  // [kChunkArrivals], zeroed by the kernel for the other rows, which runs first
  uint32_t cut_below;       // chunks: fewer units than this are cut between CTAs
  int32_t* err;
};

struct Row {
  int q_len, q_start, q_pos, k_len;
  uint32_t pairs;  // pairs of blocks of each of its units; at least 1
  uint32_t tiles;
};

// Row r as the kernel for chunks sees it (CHUNK), or the other one: the other's rows have no tokens.
template <bool CHUNK>
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
  if ((p.chunk_from > 0 && (int64_t)w.q_len * p.group >= p.chunk_from) != CHUNK) w.q_len = 0;
  int64_t seen = w.k_len;
  if (p.causal) seen = min(seen, (int64_t)w.q_pos + w.q_len);
  w.pairs = (uint32_t)max((int)((seen + 31) >> 5), 1);
  w.tiles = (w.q_len + p.tile - 1) / p.tile;
  return w;
}

// 2^e as a float, e in [-126, 127]; and the exponent of a float that is not subnormal
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }

// Pairs of elements of either type.
template <typename T> struct Two;
template <> struct Two<__half> {
  using type = __half2;
  static __device__ __forceinline__ type zero() { return __half2half2(__ushort_as_half(0)); }
};
template <> struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type zero() { return __bfloat162bfloat162(__ushort_as_bfloat16(0)); }
};
__device__ __forceinline__ __half low_of(__half2 x) { return __low2half(x); }
__device__ __forceinline__ __half high_of(__half2 x) { return __high2half(x); }
__device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 x) { return __low2bfloat16(x); }
__device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 x) { return __high2bfloat16(x); }

// The power of two that brings a head's largest element to [2^14, 2^15), and the one back
// to log2 units of a score (without the codes' own factor).
__device__ __forceinline__ int query_exponent(float top) {
  return top > 0.f ? min(max(exponent(top) - 14, -100), 112) : 0;
}

// The kernel for chunks (q4_prefill.cu); p is complete but for its tile and cut_below, and p.ws
// has room for as many bytes as the second says, the arrivals behind them.
constexpr int kMaxChunkCtas = 256;
constexpr int kChunkArrivals = kMaxChunkCtas * 8;
int launch_q4_prefill(const Q4Params& p, int head_dim, int dtype, cudaStream_t s);
int64_t q4_prefill_workspace(int head_dim);

}  // namespace seb
