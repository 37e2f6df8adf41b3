// Per-step metadata from request lengths, on the GPU.
//
// Row r holds context_lens[r] tokens and adds q_lens[r]. With sums over the rows before r:
//   q_starts[r] = sum q_lens,  k_lens[r] = context + q,  q_pos_offsets[r] = context,
//   need[r] = ceil(k / 16) - ceil(context / 16) new blocks, the step's blocks number
//   sum need ... of the free list (a ring: block j is free_ids[(head + j) mod capacity]),
// token t of row r is at position context + t - q_starts[r] and goes to slot
// block_table[r][position / 16] * 16 + position mod 16. This is what the engine's host
// code does for every step (serving_engine/block_manager.py:87-111,
// serving_engine/model_runner.py:127-170).
//
// Bound: latency. The rows are few (their arrays stay in L2), so every CTA does the
// whole scan in its own shared memory and then takes its share of the tokens and of
// the new blocks, each found by binary search: one launch and no wait between CTAs.
// 4.9 us for 256 rows of one token, of which 2.3 are an empty launch's; 9.7 us for 4096 rows,
// whose scan, eight rows to a thread, every CTA repeats.
#include "seb_common.cuh"

#include <algorithm>

namespace seb {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxRows = 16384;  // three 4-byte words of shared memory per row

struct TableParams {
  const int32_t* q_lens;
  const int32_t* context_lens;
  int32_t rows;
  int32_t total_query;
  int32_t* block_table;
  int64_t bt_stride;
  int64_t max_blocks;
  const int32_t* free_ids;
  int32_t capacity;
  const int32_t* free_state;  // head, count
  int32_t* q_starts;
  int32_t* k_lens;
  int32_t* q_pos;
  int32_t* item_row;
  int64_t* positions;
  int64_t* slots;
  int32_t* free_next;
  int32_t* err;
};

// First index of ends[0, n) that is above x; n if none.
__device__ __forceinline__ int first_above(const int32_t* ends, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int64_t warp_scan(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}

// A row's lengths as the step takes them: negative ones are 0, k_len ends at INT32_MAX, and
// blocks past the table's width are not taken.
struct StepRow {
  int q, ctx;
  int64_t k, need;
  __device__ __forceinline__ StepRow(const TableParams& p, int r, uint32_t* bad) {
    q = __ldg(p.q_lens + r);
    ctx = __ldg(p.context_lens + r);
    if (q < 0 || ctx < 0) *bad |= SEB_ERRBIT_META;
    q = max(q, 0);
    ctx = max(ctx, 0);
    k = min((int64_t)ctx + q, (int64_t)INT32_MAX);
    if (k > p.max_blocks * kBlockSize) *bad |= SEB_ERRBIT_KLEN;
    need = min((k + 15) >> 4, p.max_blocks) - min(((int64_t)ctx + 15) >> 4, p.max_blocks);
  }
};

__global__ void __launch_bounds__(kThreads) step_tables_kernel(TableParams p) {
  extern __shared__ int32_t rows_smem[];
  int32_t* tok_end = rows_smem;            // tokens up to and with the row
  int32_t* blk_end = tok_end + p.rows;     // new blocks up to and with the row
  int32_t* ctx_of = blk_end + p.rows;
  __shared__ int64_t warp_tok[kThreads / 32], warp_blk[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int capacity = p.capacity;
  const int raw_head = __ldg(p.free_state), raw_count = __ldg(p.free_state + 1);
  const bool state_ok = raw_head >= 0 && raw_head < capacity && raw_count >= 0 && raw_count <= capacity;
  const int head = state_ok ? raw_head : 0;
  const int count = state_ok ? raw_count : 0;
  uint32_t bad = state_ok ? 0u : SEB_ERRBIT_META;

  // A thread takes neighbouring rows: their sums, one scan over the threads, and the sums again.
  const int per = (p.rows + kThreads - 1) / kThreads;
  const int r0 = min(tid * per, p.rows), r1 = min(r0 + per, p.rows);
  int64_t tok = 0, blk = 0;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    const StepRow w(p, r, &bad);
    tok += w.q;
    blk += w.need;
  }
  const int64_t my_tok = tok, my_blk = blk;
  tok = warp_scan(tok, lane);
  blk = warp_scan(blk, lane);
  if (lane == 31) {
    warp_tok[warp] = tok;
    warp_blk[warp] = blk;
  }
  __syncthreads();
  int64_t tok_base = 0, blk_base = 0;  // of all rows, at last
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) {
      tok += tok_base;
      blk += blk_base;
    }
    tok_base += warp_tok[w];
    blk_base += warp_blk[w];
  }
  tok -= my_tok;
  blk -= my_blk;
#pragma unroll 4
  for (int r = r0; r < r1; ++r) {
    const StepRow w(p, r, &bad);
    tok += w.q;
    blk += w.need;
    tok_end[r] = (int)min(tok, (int64_t)INT32_MAX);
    blk_end[r] = (int)min(blk, (int64_t)INT32_MAX);
    ctx_of[r] = w.ctx;
  }
  __syncthreads();
  if (tok_base > p.total_query) bad |= SEB_ERRBIT_META;
  if (blk_base > count) bad |= SEB_ERRBIT_NOBLOCK;
  if (bad && blockIdx.x == 0) atomic_or_err(p.err, bad);
  const int fresh = (int)min(blk_base, (int64_t)count);  // blocks that the free list has
  if (blockIdx.x == 0 && tid == 0) {
    const int64_t next = (int64_t)head + fresh;
    p.free_next[0] = (int)(next >= capacity ? next - capacity : next);
    p.free_next[1] = count - fresh;
  }
  auto free_block = [&](int64_t j) -> int {  // the step's new block j
    if (j >= count) return -1;
    const int64_t at = (int64_t)head + j;
    return __ldg(p.free_ids + (at >= capacity ? at - capacity : at));
  };

  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t first = (int64_t)blockIdx.x * kThreads + tid;
  for (int64_t r = first; r < p.rows; r += step) {
    const StepRow w(p, (int)r, &bad);
    p.q_starts[r] = r ? tok_end[r - 1] : 0;
    p.k_lens[r] = (int)w.k;
    p.q_pos[r] = w.ctx;
  }
  for (int64_t t = first; t < p.total_query; t += step) {
    const int r = first_above(tok_end, p.rows, (int)t);
    int64_t pos = 0, slot = -1;
    if (r < p.rows) {
      const int ctx = ctx_of[r];
      pos = ctx + t - (r ? tok_end[r - 1] : 0);
      const int64_t col = pos >> 4;
      const int64_t had = ((int64_t)ctx + 15) >> 4;
      int id = -1;
      if (col < p.max_blocks)
        id = col < had ? p.block_table[r * p.bt_stride + col] : free_block((r ? blk_end[r - 1] : 0) + col - had);
      if (id >= 0) slot = (int64_t)id * kBlockSize + (pos & 15);
    }
    p.item_row[t] = r < p.rows ? r : -1;
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
  const int64_t new_blocks = min(blk_base, (int64_t)INT32_MAX);
  for (int64_t j = first; j < new_blocks; j += step) {
    const int r = first_above(blk_end, p.rows, (int)j);
    const int64_t had = ((int64_t)ctx_of[r] + 15) >> 4;
    p.block_table[r * p.bt_stride + had + j - (r ? blk_end[r - 1] : 0)] = free_block(j);
  }
}

}  // namespace
}  // namespace seb

extern "C" int seb_step_tables(const int32_t* q_lens, const int32_t* context_lens, int32_t num_rows,
                               int32_t total_query, int32_t* block_table, int64_t block_table_stride,
                               int64_t max_blocks, const int32_t* free_ids, int32_t free_capacity,
                               const int32_t* free_state, int32_t* q_starts, int32_t* k_lens,
                               int32_t* q_pos_offsets, int32_t* item_row, int64_t* positions, int64_t* slot_mapping,
                               int32_t* free_next, int32_t* err, void* stream) {
  using namespace seb;
  clear_error();
  SEB_CHECK_ARG(num_rows >= 0 && total_query >= 0, "seb_step_tables: negative count");
  SEB_CHECK_ARG(num_rows == 0 || (max_blocks > 0 && block_table_stride >= max_blocks),
                "seb_step_tables: bad block table shape (max_blocks %lld, stride %lld)", (long long)max_blocks,
                (long long)block_table_stride);
  SEB_CHECK_ARG(free_capacity > 0, "seb_step_tables: free_capacity must be positive");
  SEB_CHECK_ARG(free_ids && free_state && free_next, "seb_step_tables: free_ids, free_state and free_next are required");
  SEB_CHECK_ARG(num_rows == 0 || (q_lens && context_lens && block_table && q_starts && k_lens && q_pos_offsets),
                "seb_step_tables: NULL row array");
  SEB_CHECK_ARG(total_query == 0 || (item_row && positions && slot_mapping), "seb_step_tables: NULL token array");
  // Every CTA reads what the rows hold while others write already: no output may lie over an input, nor over
  // another output.
  const struct {
    const void* at;
    int64_t bytes;
    const char* name;
  } arrays[] = {{q_lens, 4ll * num_rows, "q_lens"},
                {context_lens, 4ll * num_rows, "context_lens"},
                {free_ids, 4ll * free_capacity, "free_ids"},
                {free_state, 8, "free_state"},
                {block_table, num_rows ? 4 * ((num_rows - 1) * block_table_stride + max_blocks) : 0, "block_table"},
                {q_starts, 4ll * num_rows, "q_starts"},
                {k_lens, 4ll * num_rows, "k_lens"},
                {q_pos_offsets, 4ll * num_rows, "q_pos_offsets"},
                {item_row, 4ll * total_query, "item_row"},
                {positions, 8ll * total_query, "positions"},
                {slot_mapping, 8ll * total_query, "slot_mapping"},
                {free_next, 8, "free_next"}};
  constexpr int kInputs = 4, kArrays = sizeof(arrays) / sizeof(arrays[0]);
  for (int i = kInputs; i < kArrays; ++i)
    for (int j = 0; j < i; ++j) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(arrays[i].at), b = reinterpret_cast<uintptr_t>(arrays[j].at);
      SEB_CHECK_ARG(a + arrays[i].bytes <= b || b + arrays[j].bytes <= a || !arrays[i].bytes || !arrays[j].bytes,
                    "seb_step_tables: %s overlaps %s", arrays[i].name, arrays[j].name);
    }
  if (num_rows > kMaxRows) {
    set_error("seb_step_tables: %d rows above %d", num_rows, kMaxRows);
    return SEB_EUNSUPPORTED;
  }
  TableParams p{q_lens,     context_lens, num_rows,      total_query, block_table, block_table_stride, max_blocks,
                free_ids,   free_capacity, free_state,   q_starts,    k_lens,      q_pos_offsets,      item_row,
                positions,  slot_mapping, free_next,     err};
  const int smem = 12 * std::max(num_rows, 1);
  const int rc = set_smem_limit_once<step_tables_kernel>(12 * kMaxRows);
  if (rc != SEB_OK) return rc;
  // a thread for each token, row and new block; more than one of each per thread past the GPU's SMs
  const int64_t most = std::max<int64_t>(num_rows, total_query);
  const int64_t ctas = std::min<int64_t>(num_sms(), std::max<int64_t>((most + kThreads - 1) / kThreads, 1));
  step_tables_kernel<<<(unsigned)ctas, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("step_tables_kernel");
}
