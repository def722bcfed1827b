// Tables of a step from request lengths: row ranges, lengths, positions, cache slots, last rows, and the cache blocks that
// the new tokens need, handed out of a free list in the order of the requests (contract: ops/tables.py).
//
//   end[b]   = sum_{i <= b} q[i]                                    rows of request b: [end[b - 1], end[b])
//   have[b]  = ceil(ctx[b] / page)      need[b] = ceil((ctx[b] + q[b]) / page)
//   upto[b]  = sum_{i <= b} (need[i] - have[i]) over requests that fit the table's width and the rows
//   request b is served iff it fits and (need[b] == have[b] or upto[b] <= free blocks)
//
// One launch: every block scans the lengths itself (8 bytes a request, from L2 after the first) into shared memory and then
// writes its own share of the token rows, so no block waits for another.  A block of the cache is named by the free list for
// whoever needs it, never read back from the table, and the row of its first token writes it there: a new block begins with
// a token of this step.  Bound by launching and the chain length -> prefix -> entry -> slot: 64 requests that decode 3.2 us, 3000
// requests with 270000 rows 10 us (one B200).
#include "common.cuh"

namespace xllm {

struct StepTablesParams {
  int32_t* block_table;
  int64_t bt_stride;
  int B, width;
  const int32_t* ctx;
  const int32_t* q;
  int page, n_rows;
  const int32_t* free_blocks;
  int n_free;
  int32_t* cu_q;
  int32_t* kv_lens;
  int64_t* positions;
  int32_t* slots;
  int64_t* last_rows;
  int32_t* taken;
};

constexpr int kTablesThreads = 1024;       // at most
constexpr int kTablesMaxRequests = 8192;
constexpr int kTablesStatic = kTablesThreads / 32 * sizeof(long long);

// Exclusive prefix of v over the block and its total; `red` is shared memory for 32 values.  All threads call it.
__device__ __forceinline__ long long block_prefix(long long v, long long* red, long long& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();                                   // `red` of an earlier call has been read
  if (lane == 31) red[wid] = incl;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int w = 0; w < nw; ++w) {
    const long long s = red[w];
    if (w < wid) before += s;
    total += s;
  }
  return before + incl - v;
}

__global__ void __launch_bounds__(kTablesThreads) step_tables_kernel(StepTablesParams p) {
  extern __shared__ int32_t s_mem[];
  __shared__ long long red[kTablesThreads / 32];
  int32_t* s_ctx = s_mem;                            // [B] tokens in the cache
  int32_t* s_end = s_mem + p.B;                      // [B] new tokens, then the request's last row + 1, n_rows at most
  int32_t* s_first = s_mem + 2 * p.B;                // [B] its first new block's place in the free list, -1: refused
  pdl_wait();
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) {
    s_ctx[b] = max(p.ctx[b], 0);
    s_end[b] = max(p.q[b], 0);
  }
  __syncthreads();
  const uint32_t page = p.page;
  const int shift = (page & (page - 1)) == 0 ? 31 - __clz(page) : -1;
  const auto divide = [&](uint32_t n) { return shift >= 0 ? n >> shift : n / page; };
  const auto blocks_of = [&](uint32_t n) { return divide(n + page - 1); };      // n and page below 2^31: the sum fits
  const int per = (p.B + blockDim.x - 1) / blockDim.x;
  const int b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);

  long long sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += s_end[b];
  const long long start = block_prefix(sum, red, total);
  // new blocks of request b, whose rows end at e
  const auto added_of = [&](int b, long long e, bool& fits) {
    const uint32_t c = s_ctx[b], n = c + (uint32_t)s_end[b];
    fits = n <= 0x7fffffffu && e <= p.n_rows;
    if (!fits) return 0u;
    const uint32_t need = blocks_of(n);
    fits = need <= (uint32_t)p.width;
    return fits ? need - blocks_of(c) : 0u;
  };
  long long end = start, blocks = 0;
  for (int b = b0; b < b1; ++b) {
    bool fits;
    end += s_end[b];
    blocks += added_of(b, end, fits);
  }
  long long upto = block_prefix(blocks, red, total), mine = 0;
  end = start;
  for (int b = b0; b < b1; ++b) {
    bool fits;
    end += s_end[b];
    const uint32_t added = added_of(b, end, fits);
    const bool ok = fits && (added == 0 || upto + added <= p.n_free);
    s_end[b] = (int32_t)min(end, (long long)p.n_rows);
    s_first[b] = ok ? (int32_t)min(upto, 0x7fffffffLL) : -1;
    if (ok) mine += added;
    upto += added;
  }
  if (blockIdx.x == 0) {                             // uniform in the block
    block_prefix(mine, red, total);
    if (threadIdx.x == 0) {
      *p.taken = (int32_t)total;
      p.cu_q[0] = 0;
    }
  }
  __syncthreads();

  const int stride = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
  for (int b = first; b < p.B; b += stride) {
    const int e = s_end[b], s = b > 0 ? s_end[b - 1] : 0;
    p.cu_q[b + 1] = e;
    p.kv_lens[b] = s_first[b] < 0 ? 0 : s_ctx[b] + (e - s);
    p.last_rows[b] = max(e - 1, 0);
  }
  const int rows_end = s_end[p.B - 1];
  for (int64_t row = first; row < p.n_rows; row += stride) {
    uint32_t pos = 0;
    int32_t slot = -1;
    if (row < rows_end) {
      int lo = 0, hi = p.B - 1;                      // the first request that ends behind this row
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > row) hi = mid; else lo = mid + 1;
      }
      if (s_first[lo] >= 0) {
        const uint32_t c = s_ctx[lo];
        pos = c + (uint32_t)(row - (lo > 0 ? s_end[lo - 1] : 0));
        const uint32_t column = divide(pos), have = blocks_of(c), off = pos - column * page;
        int32_t* entry = p.block_table + lo * p.bt_stride + column;
        int32_t block;
        if (column < have) {
          block = *entry;
        } else {
          block = p.free_blocks[s_first[lo] + (int64_t)(column - have)];
          if (off == 0) *entry = block;
        }
        const int64_t at = (int64_t)block * page + off;
        if (block >= 0 && at <= 0x7fffffffLL) slot = (int32_t)at;
      }
    }
    p.positions[row] = pos;
    p.slots[row] = slot;
  }
}

}  // namespace xllm

XLLM_API int xllm_step_tables(void* block_table, int64_t bt_stride, int B, int width, const void* ctx, const void* q, int page,
                              int n_rows, const void* free_blocks, int n_free, void* cu_q, void* kv_lens, void* positions,
                              void* slots, void* last_rows, void* taken, void* stream) {
  using namespace xllm;
  if (B < 1 || B > kTablesMaxRequests || width < 1 || page < 1 || n_rows < 0 || n_free < 0 || (n_free > 0 && free_blocks == nullptr))
    return (int)cudaErrorInvalidValue;
  StepTablesParams p{(int32_t*)block_table, bt_stride, B, width, (const int32_t*)ctx, (const int32_t*)q, page, n_rows,
                     (const int32_t*)free_blocks, n_free, (int32_t*)cu_q, (int32_t*)kv_lens, (int64_t*)positions,
                     (int32_t*)slots, (int64_t*)last_rows, (int32_t*)taken};
  const int smem = B * 12;
  if (smem + kTablesStatic > 48 * 1024) {            // what a block gets without asking is for both kinds of shared memory
    const cudaError_t e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTablesMaxRequests * 12);
    if (e != cudaSuccess) return (int)e;
  }
  // the scans take a thread's requests one after the other, the rest is the same whatever the block (8000 requests: 22.2 us with 512
  // threads, 15.8 with 1024; 2000: 6.1 and 8.8; one: 4.2 us with 512, 2.8 with 128)
  const int threads = B <= 128 && n_rows <= 128 ? 128 : B <= 4096 ? 512 : kTablesThreads, blocks = (n_rows + threads - 1) / threads;
  launch_pdl(step_tables_kernel, dim3(blocks < 1 ? 1 : blocks > 148 ? 148 : blocks), dim3(threads), smem, (cudaStream_t)stream, p);
  return XLLM_LAUNCH_CHECK();
}
