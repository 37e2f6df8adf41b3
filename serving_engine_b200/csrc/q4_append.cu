// Writing the 4-bit KV pool, reading it back, and the append that norms and rotates.
//
// seb_qk_norm_rope_append: for every token and query or key head x of head_dim values
//   y = x * rsqrt(mean(x^2) + eps) * w          (when norm weights are given)
//   z = (y1 * cos1 - y2 * sin1, y2 * cos2 + y1 * sin2)   (halves 1 and 2: rotate-half)
// in fp32, rounded once to the element type. Query heads go to q_out; key heads, and
// value heads as they are, go to the token's slot of a 16-bit or of a 4-bit pool.
//
// The fp32 operations and their order are fixed (no contraction to FMA; the sum of
// squares over halves, then over neighbours), so that a quantised key does not depend
// on how a compiler arranged it: a last-bit difference would move codes.
//
// Bound: HBM. Every input is read once and every output written once; head_dim / 16
// threads hold a head as two 16-byte vectors each, one from each half, so that the
// rotation needs no exchange and a group's extremes three shuffles. 8192 tokens, 32/8
// heads of 128 into the 4-bit pool: 41 us, 4.4 TB/s (two and four heads to a thread, which
// load the token's cos and sin once, took 56 and 71 us: fewer threads fit an SM).
#include "q4_format.cuh"
#include "seb_vec.cuh"

namespace seb {
namespace {

// 8192 tokens, 32/8 heads of 128: 41.3 us at 128 threads, 44.0 at 256.
constexpr int kAppendThreads = 128;

struct QkvParams {
  const char* qkv;
  int64_t qkv_st;  // elements per token
  const char* cos;
  const char* sin;
  int64_t cs_st;
  const char* wq;  // norm weights, or NULL (no norm of that kind of head)
  const char* wk;
  float eps;
  const int64_t* slots;
  int64_t num_slots;
  char* q_out;
  int64_t q_st;
  char* k_cache;
  char* v_cache;
  uint32_t units;
  int32_t hq, hkv;
  int32_t* err;
};

struct KvParams {
  const char* k_new;
  int64_t k_st, k_sh;  // elements
  const char* v_new;
  int64_t v_st, v_sh;
  const int64_t* slots;
  int64_t num_slots;
  char* k_cache;
  char* v_cache;
  uint32_t units;
  int32_t hkv;
  int32_t* err;
};

// 8 elements at any address (VEC: 16-byte aligned).
template <typename T, bool VEC>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> v;
  if constexpr (VEC) {
    v.raw = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(&v.raw)[e] = p[e];
  }
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& v) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p) = v.raw;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = reinterpret_cast<const T*>(&v.raw)[e];
  }
}

// Quantises one head held by D / 16 lanes (this one: dims [i, i + 8) in a and [D / 2 + i,
// D / 2 + i + 8) in b) into token r of the plane's row. `mask` names the head's lanes.
template <typename T, int D, bool IS_V>
__device__ __forceinline__ void quantise_row(const Vec8<T>& a, const Vec8<T>& b, int i, char* row, int r,
                                             unsigned mask) {
  using L = q4::Layout<D>;
  constexpr int kLanes = D / 16;
  constexpr int kSpan = D == 64 ? 4 : 8;  // lanes that share a group
  float lo[2], hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const Vec8<T>& v = h ? b : a;
    lo[h] = hi[h] = v.get(0);
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo[h] = q4::min_nan(lo[h], v.get(e));
      hi[h] = q4::max_nan(hi[h], v.get(e));
    }
  }
  if constexpr (D == 64) {  // one group: both halves
    lo[0] = q4::min_nan(lo[0], lo[1]);
    hi[0] = q4::max_nan(hi[0], hi[1]);
  }
#pragma unroll
  for (int h = 0; h < (D == 64 ? 1 : 2); ++h) {
#pragma unroll
    for (int off = 1; off < kSpan; off <<= 1) {
      lo[h] = q4::min_nan(lo[h], __shfl_xor_sync(mask, lo[h], off));
      hi[h] = q4::max_nan(hi[h], __shfl_xor_sync(mask, hi[h], off));
    }
  }
  static_assert(kLanes >= kSpan, "a group's lanes are a head's");
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const q4::Params p = q4::params_of(lo[D == 64 ? 0 : h], hi[D == 64 ? 0 : h]);
    const Vec8<T>& v = h ? b : a;
    const int dim = h * (D / 2) + i;
    uint32_t n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = q4::code_of(v.get(e), p);
    if constexpr (IS_V) {
      char* at = row + L::v_half(r, dim);
      *reinterpret_cast<uint16_t*>(at) = (uint16_t)q4::v_pack(n);
      *reinterpret_cast<uint16_t*>(at + 4) = (uint16_t)q4::v_pack(n + 4);
    } else {
      *reinterpret_cast<uint32_t*>(row + L::k_word(r, dim)) = q4::k_pack(n);
    }
    if (dim % q4::kGroup == 0) *reinterpret_cast<uint32_t*>(row + L::pair(r, dim)) = p.bits;
  }
}

// D / 16 lanes per (token, head): heads [0, hq) are queries, [hq, hq + hkv) keys, the rest values.
template <typename T, int D, bool POOL4, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) qk_norm_rope_append_kernel(QkvParams p) {
  constexpr int kLanes = D / 16;
  const uint32_t u = blockIdx.x * (kAppendThreads / kLanes) + threadIdx.x / kLanes;
  if (u >= p.units) return;
  const int sub = threadIdx.x % kLanes;
  const unsigned mask = (unsigned)(((1ull << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes));
  const uint32_t heads = p.hq + 2 * p.hkv, tok = u / heads;
  const int64_t t = tok;
  const int h = (int)(u - tok * heads);
  const int i = 8 * sub;
  const T* src = reinterpret_cast<const T*>(p.qkv) + t * p.qkv_st + (int64_t)h * D;
  Vec8<T> a = load8<T, VEC>(src + i), b = load8<T, VEC>(src + D / 2 + i);
  if (h < p.hq + p.hkv) {
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = a.get(e);
      y[e] = b.get(e);
    }
    const T* w = reinterpret_cast<const T*>(h < p.hq ? p.wq : p.wk);
    if (w) {
      float s[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = __fadd_rn(__fmul_rn(x[e], x[e]), __fmul_rn(y[e], y[e]));
      float sum = __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3])),
                            __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7])));
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) sum = __fadd_rn(sum, __shfl_xor_sync(mask, sum, off));
      const float r = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(sum, 1.f / D), p.eps)));
      const Vec8<T> wa = load8<T, VEC>(w + i), wb = load8<T, VEC>(w + D / 2 + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = __fmul_rn(__fmul_rn(x[e], r), wa.get(e));
        y[e] = __fmul_rn(__fmul_rn(y[e], r), wb.get(e));
      }
    }
    const T* cs = reinterpret_cast<const T*>(p.cos) + t * p.cs_st;
    const T* sn = reinterpret_cast<const T*>(p.sin) + t * p.cs_st;
    const Vec8<T> c1 = load8<T, VEC>(cs + i), c2 = load8<T, VEC>(cs + D / 2 + i);
    const Vec8<T> s1 = load8<T, VEC>(sn + i), s2 = load8<T, VEC>(sn + D / 2 + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a.set(e, __fsub_rn(__fmul_rn(x[e], c1.get(e)), __fmul_rn(y[e], s1.get(e))));
      b.set(e, __fadd_rn(__fmul_rn(y[e], c2.get(e)), __fmul_rn(x[e], s2.get(e))));
    }
  }
  if (h < p.hq) {
    T* dst = reinterpret_cast<T*>(p.q_out) + t * p.q_st + (int64_t)h * D;
    store8<T, VEC>(dst + i, a);
    store8<T, VEC>(dst + D / 2 + i, b);
    return;
  }
  const int64_t slot = __ldg(p.slots + t);
  if (slot < 0 || slot >= p.num_slots) {
    if (slot != -1 && h == p.hq && sub == 0) atomic_or_err(p.err, SEB_ERRBIT_SLOT);
    return;
  }
  const bool is_v = h >= p.hq + p.hkv;
  const int kvh = h - p.hq - (is_v ? p.hkv : 0);
  char* plane = is_v ? p.v_cache : p.k_cache;
  if constexpr (POOL4) {
    char* row = plane + (slot / kBlockSize * p.hkv + kvh) * (int64_t)q4::Layout<D>::kRow;
    const int r = (int)(slot % kBlockSize);
    if (is_v) quantise_row<T, D, true>(a, b, i, row, r, mask);
    else quantise_row<T, D, false>(a, b, i, row, r, mask);
  } else {
    T* dst = reinterpret_cast<T*>(plane) + (slot * p.hkv + kvh) * (int64_t)D;
    store8<T, VEC>(dst + i, a);
    store8<T, VEC>(dst + D / 2 + i, b);
  }
}

// D / 16 lanes per (token, kv head, plane). 8192 tokens, 8 heads of 128: 16.6 us, 2.6 TB/s.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) kv_append_q4_kernel(KvParams p) {
  constexpr int kLanes = D / 16;
  const uint32_t u = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  if (u >= p.units) return;
  const int sub = threadIdx.x % kLanes;
  const unsigned mask = (unsigned)(((1ull << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes));
  const uint32_t tok = u / (2 * p.hkv);
  const int64_t t = tok;
  const int h = (int)(u - tok * 2 * p.hkv);
  const int64_t slot = __ldg(p.slots + t);
  if (slot < 0 || slot >= p.num_slots) {
    if (slot != -1 && h == 0 && sub == 0) atomic_or_err(p.err, SEB_ERRBIT_SLOT);
    return;
  }
  const bool is_v = h >= p.hkv;
  const int kvh = h - (is_v ? p.hkv : 0);
  const T* src = is_v ? reinterpret_cast<const T*>(p.v_new) + t * p.v_st + kvh * p.v_sh
                      : reinterpret_cast<const T*>(p.k_new) + t * p.k_st + kvh * p.k_sh;
  const int i = 8 * sub;
  const Vec8<T> a = load8<T, VEC>(src + i), b = load8<T, VEC>(src + D / 2 + i);
  char* row = (is_v ? p.v_cache : p.k_cache) + (slot / kBlockSize * p.hkv + kvh) * (int64_t)q4::Layout<D>::kRow;
  const int r = (int)(slot % kBlockSize);
  if (is_v) quantise_row<T, D, true>(a, b, i, row, r, mask);
  else quantise_row<T, D, false>(a, b, i, row, r, mask);
}

// The values that the pool's slots stand for: 4 threads per (token, plane, kv head), each with
// 16 dims of every group of a panel, as K's chunks have them (V: two neighbouring chunks).
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_gather_q4_kernel(const char* k_cache, const char* v_cache, int64_t num_slots,
                                                           const int64_t* slots, uint32_t units, int hkv, T* k_out,
                                                           T* v_out, int32_t* err) {
  using L = q4::Layout<D>;
  constexpr int G = L::kGroups;
  const uint32_t u = blockIdx.x * 64 + threadIdx.x / 4;
  if (u >= units) return;
  const int c = threadIdx.x & 3;
  const uint32_t tok = u / (2 * hkv);
  const int64_t t = tok;
  const int h = (int)(u - tok * 2 * hkv);
  const bool is_v = h >= hkv;
  const int kvh = h - (is_v ? hkv : 0);
  T* dst = (is_v ? v_out : k_out) + (t * hkv + kvh) * D + 16 * c;
  const int64_t slot = __ldg(slots + t);
  const bool ok = slot >= 0 && slot < num_slots;
  if (!ok && slot != -1 && h == 0 && c == 0) atomic_or_err(err, SEB_ERRBIT_SLOT);
  const char* row = (is_v ? v_cache : k_cache) + ((ok ? slot : 0) / kBlockSize * hkv + kvh) * (int64_t)L::kRow;
  const int r = (int)(slot & (kBlockSize - 1));
#pragma unroll
  for (int pn = 0; pn < L::kPanels; ++pn) {
    // words: K's [group][8 dims], each dims 0 2 4 6 1 3 5 7; V's [chunk][group][4 dims], both tokens of a pair
    __align__(16) uint32_t w[4 * G];
    __half2 pr[G];
    const char* codes = row + pn * 8 * L::kWidth;
    if (is_v) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const char* at = codes + (r >> 1) * L::kWidth + ((2 * c + k) ^ L::turn(r >> 1)) * (8 * G);
        if constexpr (G == 2) *reinterpret_cast<uint4*>(w + 4 * k) = *reinterpret_cast<const uint4*>(at);
        else *reinterpret_cast<uint2*>(w + 2 * k) = *reinterpret_cast<const uint2*>(at);
      }
    } else {
      const char* at = codes + r * (L::kWidth / 2) + c * (8 * G);
      if constexpr (G == 2) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(at);
      else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(at);
    }
    const char* pairs = row + L::kCodes + pn * 64 * G + r * 4 * G;
    if constexpr (G == 2) *reinterpret_cast<uint2*>(pr) = *reinterpret_cast<const uint2*>(pairs);
    else *reinterpret_cast<uint32_t*>(pr) = *reinterpret_cast<const uint32_t*>(pairs);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float scale = ok ? __low2float(pr[g]) : 0.f, low = ok ? __high2float(pr[g]) : 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {  // 8 dims
        float x[8];
        if (is_v) {
          const uint32_t lo = w[k * 2 * G + 2 * g] >> (16 * (r & 1)), hi = w[k * 2 * G + 2 * g + 1] >> (16 * (r & 1));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = q4::value_of(q4::v_code(e < 4 ? lo : hi, e & 3), scale, low);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = q4::value_of(q4::k_code(w[2 * g + k], e), scale, low);
        }
        T* out = dst + pn * L::kWidth + g * q4::kGroup + 8 * k;
        if constexpr (sizeof(T) == 2) {
          Vec8<T> o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o.set(e, x[e]);
          *reinterpret_cast<uint4*>(out) = o.raw;
        } else {
          *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(out + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
    }
  }
}

unsigned blocks_for(uint32_t units, int per_block) { return (unsigned)(((int64_t)units + per_block - 1) / per_block); }

// Heads of all tokens, which the kernels count in 32 bits; past that, an error.
int units_of(int64_t n_tokens, int64_t heads, const char* what, uint32_t* units) {
  SEB_CHECK_ARG(n_tokens <= (int64_t)0x7fffffff / heads, "%s: too many tokens", what);
  *units = (uint32_t)(n_tokens * heads);
  return SEB_OK;
}

template <typename T, int D>
int launch_qkv(const QkvParams& p, bool pool4, bool vec, cudaStream_t s) {
  const unsigned grid = blocks_for(p.units, kAppendThreads / (D / 16));
  if (pool4 && vec) qk_norm_rope_append_kernel<T, D, true, true><<<grid, kAppendThreads, 0, s>>>(p);
  else if (pool4) qk_norm_rope_append_kernel<T, D, true, false><<<grid, kAppendThreads, 0, s>>>(p);
  else if (vec) qk_norm_rope_append_kernel<T, D, false, true><<<grid, kAppendThreads, 0, s>>>(p);
  else qk_norm_rope_append_kernel<T, D, false, false><<<grid, kAppendThreads, 0, s>>>(p);
  return launch_status("qk_norm_rope_append_kernel");
}

template <typename T>
int launch_qkv_dim(const QkvParams& p, int d, bool pool4, bool vec, cudaStream_t s) {
  return d == 64 ? launch_qkv<T, 64>(p, pool4, vec, s)
                 : d == 128 ? launch_qkv<T, 128>(p, pool4, vec, s) : launch_qkv<T, 256>(p, pool4, vec, s);
}

template <typename T, int D>
int launch_kv(const KvParams& p, bool vec, cudaStream_t s) {
  const unsigned grid = blocks_for(p.units, 256 / (D / 16));
  if (vec) kv_append_q4_kernel<T, D, true><<<grid, 256, 0, s>>>(p);
  else kv_append_q4_kernel<T, D, false><<<grid, 256, 0, s>>>(p);
  return launch_status("kv_append_q4_kernel");
}

template <typename T>
int launch_kv_dim(const KvParams& p, int d, bool vec, cudaStream_t s) {
  return d == 64 ? launch_kv<T, 64>(p, vec, s) : d == 128 ? launch_kv<T, 128>(p, vec, s) : launch_kv<T, 256>(p, vec, s);
}

bool q4_head_dim(int d) { return d == 64 || d == 128 || d == 256; }

}  // namespace
}  // namespace seb

extern "C" int seb_qk_norm_rope_append(const void* qkv, int64_t qkv_stride_token, int64_t n_tokens,
                                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* cos,
                                       const void* sin, int64_t cos_sin_stride_token, const void* q_weight,
                                       const void* k_weight, float eps, const int64_t* slot_mapping, void* q_out,
                                       int64_t q_out_stride_token, void* k_cache, void* v_cache, int64_t num_blocks,
                                       int32_t cache_bits, int32_t dtype, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(dtype == SEB_BF16 || dtype == SEB_F16, "seb_qk_norm_rope_append: bf16 or fp16 required (dtype %d)",
                dtype);
  SEB_CHECK_ARG(cache_bits == 4 || cache_bits == 16, "seb_qk_norm_rope_append: cache_bits must be 4 or 16, got %d",
                cache_bits);
  SEB_CHECK_ARG(n_tokens >= 0, "seb_qk_norm_rope_append: n_tokens < 0");
  SEB_CHECK_ARG(num_q_heads > 0 && num_kv_heads > 0 && num_blocks > 0,
                "seb_qk_norm_rope_append: head counts and num_blocks must be positive");
  if (!q4_head_dim(head_dim)) {
    set_error("seb_qk_norm_rope_append: head_dim %d not supported (64, 128, 256)", head_dim);
    return SEB_EUNSUPPORTED;
  }
  if (n_tokens == 0) return SEB_OK;
  SEB_CHECK_ARG(qkv && cos && sin && slot_mapping && q_out && k_cache && v_cache,
                "seb_qk_norm_rope_append: NULL pointer argument");
  SEB_CHECK_ARG(qkv_stride_token >= (int64_t)(num_q_heads + 2 * num_kv_heads) * head_dim &&
                    q_out_stride_token >= (int64_t)num_q_heads * head_dim && cos_sin_stride_token >= head_dim,
                "seb_qk_norm_rope_append: a token stride is smaller than its row");
  SEB_CHECK_ARG(cache_bits == 16 || (aligned(k_cache, 16) && aligned(v_cache, 16)),
                "seb_qk_norm_rope_append: a 4-bit pool must be 16-byte aligned");
  QkvParams p;
  p.qkv = static_cast<const char*>(qkv);
  p.qkv_st = qkv_stride_token;
  p.cos = static_cast<const char*>(cos);
  p.sin = static_cast<const char*>(sin);
  p.cs_st = cos_sin_stride_token;
  p.wq = static_cast<const char*>(q_weight);
  p.wk = static_cast<const char*>(k_weight);
  p.eps = eps;
  p.slots = slot_mapping;
  p.num_slots = num_blocks * kBlockSize;
  p.q_out = static_cast<char*>(q_out);
  p.q_st = q_out_stride_token;
  p.k_cache = static_cast<char*>(k_cache);
  p.v_cache = static_cast<char*>(v_cache);
  const int rc = units_of(n_tokens, num_q_heads + 2 * (int64_t)num_kv_heads, "seb_qk_norm_rope_append", &p.units);
  if (rc != SEB_OK) return rc;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.err = err;
  const bool vec = aligned(qkv, 16) && aligned(cos, 16) && aligned(sin, 16) && aligned(q_weight, 16) &&
                   aligned(k_weight, 16) && aligned(q_out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                   qkv_stride_token % 8 == 0 && cos_sin_stride_token % 8 == 0 && q_out_stride_token % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SEB_BF16 ? launch_qkv_dim<__nv_bfloat16>(p, head_dim, cache_bits == 4, vec, s)
                           : launch_qkv_dim<__half>(p, head_dim, cache_bits == 4, vec, s);
}

extern "C" int seb_kv_append_q4(const void* k_new, int64_t k_stride_token, int64_t k_stride_head, const void* v_new,
                                int64_t v_stride_token, int64_t v_stride_head, int64_t n_tokens,
                                const int64_t* slot_mapping, void* k_cache, void* v_cache, int64_t num_blocks,
                                int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(dtype == SEB_BF16 || dtype == SEB_F16, "seb_kv_append_q4: bf16 or fp16 required (dtype %d)", dtype);
  SEB_CHECK_ARG(n_tokens >= 0 && num_kv_heads > 0 && num_blocks > 0,
                "seb_kv_append_q4: n_tokens must be non-negative, num_kv_heads and num_blocks positive");
  if (!q4_head_dim(head_dim)) {
    set_error("seb_kv_append_q4: head_dim %d not supported (64, 128, 256)", head_dim);
    return SEB_EUNSUPPORTED;
  }
  if (n_tokens == 0) return SEB_OK;
  SEB_CHECK_ARG(k_new && v_new && slot_mapping && k_cache && v_cache, "seb_kv_append_q4: NULL pointer argument");
  SEB_CHECK_ARG(aligned(k_cache, 16) && aligned(v_cache, 16), "seb_kv_append_q4: the pool must be 16-byte aligned");
  KvParams p;
  p.k_new = static_cast<const char*>(k_new);
  p.k_st = k_stride_token;
  p.k_sh = k_stride_head;
  p.v_new = static_cast<const char*>(v_new);
  p.v_st = v_stride_token;
  p.v_sh = v_stride_head;
  p.slots = slot_mapping;
  p.num_slots = num_blocks * kBlockSize;
  p.k_cache = static_cast<char*>(k_cache);
  p.v_cache = static_cast<char*>(v_cache);
  const int rc = units_of(n_tokens, 2 * (int64_t)num_kv_heads, "seb_kv_append_q4", &p.units);
  if (rc != SEB_OK) return rc;
  p.hkv = num_kv_heads;
  p.err = err;
  const bool vec = aligned(k_new, 16) && aligned(v_new, 16) && k_stride_token % 8 == 0 && k_stride_head % 8 == 0 &&
                   v_stride_token % 8 == 0 && v_stride_head % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SEB_BF16 ? launch_kv_dim<__nv_bfloat16>(p, head_dim, vec, s)
                           : launch_kv_dim<__half>(p, head_dim, vec, s);
}

namespace seb {
namespace {

template <typename T>
int launch_gather(const void* k, const void* v, int64_t num_slots, const int64_t* slots, int64_t n, int hkv, int d,
                  void* k_out, void* v_out, int32_t* err, cudaStream_t s) {
  uint32_t units;
  const int rc = units_of(n, 2 * (int64_t)hkv, "seb_kv_gather_q4", &units);
  if (rc != SEB_OK) return rc;
  const unsigned grid = blocks_for(units, 64);
  const char* kc = static_cast<const char*>(k);
  const char* vc = static_cast<const char*>(v);
  T* ko = static_cast<T*>(k_out);
  T* vo = static_cast<T*>(v_out);
  if (d == 64) kv_gather_q4_kernel<T, 64><<<grid, 256, 0, s>>>(kc, vc, num_slots, slots, units, hkv, ko, vo, err);
  else if (d == 128) kv_gather_q4_kernel<T, 128><<<grid, 256, 0, s>>>(kc, vc, num_slots, slots, units, hkv, ko, vo, err);
  else kv_gather_q4_kernel<T, 256><<<grid, 256, 0, s>>>(kc, vc, num_slots, slots, units, hkv, ko, vo, err);
  return launch_status("kv_gather_q4_kernel");
}

}  // namespace
}  // namespace seb

extern "C" int seb_kv_gather_q4(const void* k_cache, const void* v_cache, int64_t num_blocks, int32_t num_kv_heads,
                                int32_t head_dim, const int64_t* slots, int64_t n_tokens, void* k_out, void* v_out,
                                int32_t dtype, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(elem_size(dtype) > 0, "seb_kv_gather_q4: unknown dtype %d", dtype);
  SEB_CHECK_ARG(n_tokens >= 0 && num_kv_heads > 0 && num_blocks > 0,
                "seb_kv_gather_q4: n_tokens must be non-negative, num_kv_heads and num_blocks positive");
  if (!q4_head_dim(head_dim)) {
    set_error("seb_kv_gather_q4: head_dim %d not supported (64, 128, 256)", head_dim);
    return SEB_EUNSUPPORTED;
  }
  if (n_tokens == 0) return SEB_OK;
  SEB_CHECK_ARG(k_cache && v_cache && slots && k_out && v_out, "seb_kv_gather_q4: NULL pointer argument");
  SEB_CHECK_ARG(aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_out, 16) && aligned(v_out, 16),
                "seb_kv_gather_q4: the pool and the outputs must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t num_slots = num_blocks * kBlockSize;
  switch (dtype) {
    case SEB_BF16:
      return launch_gather<__nv_bfloat16>(k_cache, v_cache, num_slots, slots, n_tokens, num_kv_heads, head_dim, k_out,
                                          v_out, err, s);
    case SEB_F16:
      return launch_gather<__half>(k_cache, v_cache, num_slots, slots, n_tokens, num_kv_heads, head_dim, k_out, v_out,
                                   err, s);
    default:
      return launch_gather<float>(k_cache, v_cache, num_slots, slots, n_tokens, num_kv_heads, head_dim, k_out, v_out,
                                  err, s);
  }
}
