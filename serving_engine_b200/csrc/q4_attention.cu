// Paged attention over the 4-bit KV pool.
//
//   O = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = scale * q . k_j,
//   LSE = log(sum_j exp(s_j)),  k_j = scale_j * n_j + low_j for each group of 64 dims,
// over the keys j < k_lens[r] (causal: and j <= the query's position). Rows follow
// seb_paged_decode; a query that sees no key gets O = 0 and LSE = -inf.
#include "q4_format.cuh"

namespace seb {
namespace {

constexpr unsigned kFull = 0xffffffffu;

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
  float scale;
  int32_t causal;
  char* out;
  int64_t o_st, o_sh;  // elements
  float* lse;
  int64_t lse_st;
  int32_t* err;
};

// One warp per (row, query token, query head); lane l holds dims l * D / 32 and on.
template <typename T, int D>
__global__ void __launch_bounds__(128) q4_attention_kernel(Q4Params p) {
  using L = q4::Layout<D>;
  constexpr int DL = D / 32;
  const int lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int row = blockIdx.x;
  if (h >= p.hq) return;
  const int q_len = max(__ldg(p.q_lens + row), 0), q_start = __ldg(p.q_starts + row);
  const int q_pos = __ldg(p.q_pos + row);
  int k_len = max(__ldg(p.k_lens + row), 0);
  if (q_len == 0) return;
  if (q_start < 0 || (int64_t)q_start + q_len > p.total_query) {
    if (lane == 0 && h == 0) atomic_or_err(p.err, SEB_ERRBIT_META);
    return;
  }
  if (k_len > p.max_blocks * kBlockSize) {
    if (lane == 0 && h == 0) atomic_or_err(p.err, SEB_ERRBIT_KLEN);
    k_len = (int)(p.max_blocks * kBlockSize);
  }
  const int kvh = h / p.group;
  for (int i = blockIdx.z; i < q_len; i += gridDim.z) {
    const int64_t tok = q_start + i;
    const int64_t seen = p.causal ? min((int64_t)k_len, (int64_t)q_pos + i + 1) : k_len;
    float q[DL], o[DL], m = -INFINITY, l = 0.f;
    const T* qp = reinterpret_cast<const T*>(p.q) + tok * p.q_st + (int64_t)h * p.q_sh + lane * DL;
#pragma unroll
    for (int e = 0; e < DL; ++e) {
      q[e] = Elem<T>::to_float(qp[e]) * p.scale;
      o[e] = 0.f;
    }
    for (int64_t j = 0; j < seen; ++j) {
      const int id = __ldg(p.block_table + row * p.bt_stride + (j >> 4));
      if (id < 0 || id >= p.num_blocks) {  // unreadable: as if masked
        if (lane == 0) atomic_or_err(p.err, SEB_ERRBIT_BLOCK_ID);
        continue;
      }
      const int r = (int)(j & 15);
      const int64_t at = ((int64_t)id * p.hkv + kvh) * L::kRow;
      const char* kr = p.k_cache + at;
      const char* vr = p.v_cache + at;
      const __half2 kp = *reinterpret_cast<const __half2*>(kr + L::pair(r, lane * DL));
      const __half2 vp = *reinterpret_cast<const __half2*>(vr + L::pair(r, lane * DL));
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < DL; ++e) {
        const int dim = lane * DL + e;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(kr + L::k_word(r, dim & ~7));
        s = fmaf(q[e], q4::value_of(q4::k_code(w, dim & 7), __low2float(kp), __high2float(kp)), s);
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(kFull, s, off);
      const float m_new = fmaxf(m, s);
      const float keep = m_new == -INFINITY ? 1.f : expf(m - m_new);
      const float pr = m_new == -INFINITY ? 0.f : expf(s - m_new);
      l = l * keep + pr;
#pragma unroll
      for (int e = 0; e < DL; ++e) {
        const int dim = lane * DL + e;
        const uint32_t w = *reinterpret_cast<const uint16_t*>(vr + L::v_half(r, dim & ~3));
        o[e] = o[e] * keep + pr * q4::value_of(q4::v_code(w, dim & 3), __low2float(vp), __high2float(vp));
      }
      m = m_new;
    }
    T* op = reinterpret_cast<T*>(p.out) + tok * p.o_st + (int64_t)h * p.o_sh + lane * DL;
#pragma unroll
    for (int e = 0; e < DL; ++e) op[e] = Elem<T>::from_float(l == 0.f ? 0.f : o[e] / l);
    if (lane == 0) p.lse[tok * p.lse_st + h] = l == 0.f ? -INFINITY : m + logf(l);
  }
}

template <typename T>
int launch(const Q4Params& p, int d, cudaStream_t s) {
  const int z = (p.total_query + p.num_rows - 1) / p.num_rows;
  const dim3 grid(p.num_rows, (p.hq + 3) / 4, z < 1 ? 1 : z > 64 ? 64 : z);
  if (d == 64) q4_attention_kernel<T, 64><<<grid, 128, 0, s>>>(p);
  else if (d == 128) q4_attention_kernel<T, 128><<<grid, 128, 0, s>>>(p);
  else q4_attention_kernel<T, 256><<<grid, 128, 0, s>>>(p);
  return launch_status("q4_attention_kernel");
}

}  // namespace
}  // namespace seb

extern "C" int64_t seb_paged_attention_q4_workspace_size(int32_t num_rows, int32_t total_query, int32_t num_q_heads,
                                                         int32_t num_kv_heads, int32_t head_dim) {
  (void)num_rows, (void)total_query, (void)num_q_heads, (void)num_kv_heads, (void)head_dim;
  return 0;
}

extern "C" int seb_paged_attention_q4(const void* q, int64_t q_stride_token, int64_t q_stride_head,
                                      const void* k_cache, const void* v_cache, int64_t num_blocks,
                                      const int32_t* block_table, int64_t block_table_stride, int64_t max_blocks,
                                      const int32_t* q_starts, const int32_t* q_lens, const int32_t* k_lens,
                                      const int32_t* q_pos_offsets, int32_t num_rows, int32_t total_query,
                                      int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                                      float scale, int32_t is_causal, void* out, int64_t out_stride_token,
                                      int64_t out_stride_head, float* lse, int64_t lse_stride_token, void* workspace,
                                      int64_t workspace_bytes, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(dtype == SEB_BF16 || dtype == SEB_F16, "seb_paged_attention_q4: bf16 or fp16 required (dtype %d)",
                dtype);
  SEB_CHECK_ARG(num_rows >= 0 && total_query >= 0, "seb_paged_attention_q4: negative count");
  SEB_CHECK_ARG(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
                "seb_paged_attention_q4: num_q_heads (%d) must be a positive multiple of num_kv_heads (%d)",
                num_q_heads, num_kv_heads);
  SEB_CHECK_ARG(num_q_heads / num_kv_heads <= 16, "seb_paged_attention_q4: GQA group %d > 16 not supported",
                num_q_heads / num_kv_heads);
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
  SEB_CHECK_ARG(aligned(k_cache, 16) && aligned(v_cache, 16), "seb_paged_attention_q4: the pool must be 16-byte aligned");
  (void)workspace, (void)workspace_bytes;
  Q4Params p{static_cast<const char*>(q), q_stride_token, q_stride_head, static_cast<const char*>(k_cache),
             static_cast<const char*>(v_cache), num_blocks, block_table, block_table_stride, max_blocks, q_starts,
             q_lens, k_lens, q_pos_offsets, num_rows, total_query, num_q_heads, num_kv_heads,
             num_q_heads / num_kv_heads, scale, is_causal ? 1 : 0, static_cast<char*>(out), out_stride_token,
             out_stride_head, lse, lse_stride_token, err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SEB_BF16 ? launch<__nv_bfloat16>(p, head_dim, s) : launch<__half>(p, head_dim, s);
}
