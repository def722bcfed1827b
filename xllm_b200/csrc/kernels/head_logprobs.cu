// Log-probabilities and entropies straight from hidden states and the output projection (contract: ops/score.py): the scores
// x = h W^T are tallied where they are computed, in the tensor cores' accumulators, and never stored.
//
//   head_tally_kernel  tiles of 256 rows x up to 256 columns of the vocabulary: the rows' tallies (logprob_math.cuh) of the tile's
//                      columns, and the given token's score from whichever tile holds it
//   head_join_kernel   a row's tallies over all tiles, joined in a fixed order
//
// A tile is a pair of CTAs' (cta_group::2): each loads its 128 rows of h and half of the columns' rows of W by TMA into a ring
// of stages, one thread of the pair's first CTA issues the products into one of two accumulators in tensor memory, and four warps
// of each CTA read the other one back, a thread a row, 32 columns at a time.  Few rows are bound by W's way from HBM, many
// by the tensor cores; the tally (some 6 instructions a score, 2000 cycles a tile) hides behind the next tile's products from a width of 256 on.
//
// Every wait is bounded; on expiry the kernel raises an error word, all roles leave their loops, tensor memory is freed and the
// kernel returns.
#include "logprob_math.cuh"
#include "tc_common.cuh"
#include "vec_io.cuh"

namespace xllm {

using namespace tc;

constexpr int kHeadRows = 128, kHeadCols = 256, kHeadK = 64;        // rows of a CTA, most columns of a tile, a K block
constexpr int kHeadStages = 7, kHeadThreads = 192;
constexpr int kHeadABytes = kHeadRows * kHeadK * 2, kHeadBBytes = kHeadCols / 2 * kHeadK * 2;
constexpr int kHeadStageBytes = kHeadABytes + kHeadBBytes;
constexpr int kHeadBarOff = kHeadStages * kHeadStageBytes;
constexpr int kHeadSmem = kHeadBarOff + (2 * kHeadStages + 4) * 8 + 16 + 1024;
static_assert(kHeadSmem <= 232448, "exceeds the 227 KB of shared memory per CTA");

__device__ int g_head_error = 0;

// workspace: tallies [column tiles][rows] and the given tokens' scores [rows]
struct HeadParams {
  int T, V, K, cols, n_tiles, m_tiles, a_box;
  const int64_t* ids;
  const float* temperature;
  Tally* tallies;
  float* given;
};

// Tile u of the order in which they are worked on: the row tiles of a column tile side by side, so that W is read from HBM once for
// them all, in groups of 16 (4096 rows), whose rows stay in L2.
constexpr int kHeadGroup = 16;
__device__ __forceinline__ void head_tile(const HeadParams& p, int u, int& m, int& n) {
  const int whole = kHeadGroup * p.n_tiles, g = u / whole, r = u - g * whole;
  const int wide = min(kHeadGroup, p.m_tiles - g * kHeadGroup);
  n = r / wide;
  m = g * kHeadGroup + r - n * wide;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kHeadThreads, 1)
head_tally_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, const HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem), bar0 = sbase + kHeadBarOff;
  const auto full_bar = [&](int s) { return bar0 + 8u * s; };
  const auto empty_bar = [&](int s) { return bar0 + 8u * (kHeadStages + s); };
  const auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kHeadStages + a); };
  const auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kHeadStages + 2 + a); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + kHeadBarOff + (2 * kHeadStages + 4) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int units = p.m_tiles * p.n_tiles, k_blocks = (p.K + kHeadK - 1) / kHeadK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kHeadStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 8);                    // four warps in each CTA of the pair
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                     // both CTAs' barriers exist before anything can signal them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_wait();
  pdl_launch_dependents();                            // after the allocation: what starts early may want tensor memory too

  if (warp == 0) {
    // ------------------------------------------------------------------ loads (both CTAs)
    const uint32_t bytes = 2u * (p.a_box + p.cols / 2) * kHeadK * 2;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = pair; u < units && ok; u += n_pairs) {
      int m, n;
      head_tile(p, u, m, n);
      const int m0 = m * 2 * kHeadRows + (int)rank * kHeadRows, n0 = n * p.cols + (int)rank * (p.cols / 2);
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!mbar_wait_cluster_warp(empty_bar(stage), phase ^ 1, abort_flag)) { ok = false; break; }
        const uint32_t dst = sbase + stage * kHeadStageBytes;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(full_bar(stage), bytes);
          tma_load_2d_pair(dst, &map_h, kb * kHeadK, m0, full_bar(stage));
          tma_load_2d_pair(dst + kHeadABytes, &map_w, kb * kHeadK, n0, full_bar(stage));
        }
        __syncwarp();
        if (++stage == kHeadStages) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) {
      const long long t0 = clock64();
      while (clock64() - t0 < 20000000LL) {}          // bounded grace period for copies still in flight
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------------------------------------------------------- products (the pair's first CTA)
      const uint32_t id = idesc_pair(p.cols);
      int stage = 0, t = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = pair; u < units && ok; u += n_pairs, ++t) {
        const int acc = t & 1;
        if (!mbar_wait_cluster_warp(tempty_bar(acc), ((t >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + acc * kHeadCols;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_cluster_warp(full_bar(stage), phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = sbase + stage * kHeadStageBytes;
          if (elect_one()) {
            const uint64_t a = smem_desc(at, 16, 1024), b = smem_desc(at + kHeadABytes, 16, 1024);
#pragma unroll
            for (int k = 0; k < kHeadK / 16; ++k) umma_pair(d, a + 2 * k, b + 2 * k, id, (kb | k) != 0);
            umma_commit_pair(empty_bar(stage));
          }
          __syncwarp();
          if (++stage == kHeadStages) { stage = 0; phase ^= 1; }
        }
        if (ok && elect_one()) umma_commit_pair(tfull_bar(acc));
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------------ tallies (both CTAs), a thread a row
    const int q = warp & 3;
    const uint32_t leader_tempty = in_cta(tempty_bar(0), 0);
    int t = 0;
    for (int u = pair; u < units; u += n_pairs, ++t) {
      int m, n;
      head_tile(p, u, m, n);
      const int row0 = m * 2 * kHeadRows + (int)rank * kHeadRows + q * 32, row = row0 + lane, n0 = n * p.cols, acc = t & 1;
      const float c = row < p.T ? row_scale(p.temperature, row) * kLog2e : 1.f;
      const int64_t want = row < p.T ? p.ids[row] - n0 : -1;
      if (!mbar_wait_cluster_warp(tfull_bar(acc), (t >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + acc * kHeadCols + ((uint32_t)(q * 32) << 16);
      if (row0 < p.T) {
        PairTally run = pair_empty();
        for (int c0 = 0; c0 < p.cols; c0 += 32) {
          uint32_t r[32];
          tmem_ld32(taddr + c0, r);
          tmem_ld_wait();
          const int left = p.V - n0 - c0;
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= left) r[j] = 0xFF800000u;
          }
          float most = __uint_as_float(r[0]);
#pragma unroll
          for (int j = 1; j < 32; ++j) most = fmaxf(most, __uint_as_float(r[j]));
          if (most > run.m) pair_rebase(run, most, c);
#pragma unroll
          for (int j = 0; j < 32; j += 2) pair_add(run, {__uint_as_float(r[j]), __uint_as_float(r[j + 1])}, c);
          const bool here = want >= c0 && want < c0 + 32 && want < p.V - n0;
          if (__any_sync(0xffffffffu, here)) {
            float x = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (want == c0 + j) x = __uint_as_float(r[j]);
            if (here) p.given[row] = x;
          }
        }
        if (row < p.T) p.tallies[(int64_t)n * p.T + row] = pair_sum(run);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(leader_tempty + 8u * acc);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicExch(&g_head_error, 1);
  cluster_sync();                                     // neither CTA leaves while the other may touch its barriers or memory
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base));
  }
}

// A block joins `rows` rows (a power of two, 32 at most), 256 / rows threads each: a thread every so many tiles, then in pairs.
__global__ void __launch_bounds__(256) head_join_kernel(const HeadParams p, int rows, float* out_lp, float* out_entropy) {
  __shared__ Tally part[256];
  pdl_wait();
  const int r = threadIdx.x % rows, slice = threadIdx.x / rows, slices = 256 / rows;
  const int64_t row = (int64_t)blockIdx.x * rows + r;
  Tally a = tally_empty();
  float scale = 1.f, c = kLog2e;
  if (row < p.T) {
    scale = row_scale(p.temperature, row);
    c = scale * kLog2e;
    for (int i = slice; i < p.n_tiles; i += slices) a = tally_join(a, p.tallies[(int64_t)i * p.T + row], c);
  }
  part[threadIdx.x] = a;
  __syncthreads();
  for (int half = slices / 2; half > 0; half /= 2) {
    if (slice < half) part[threadIdx.x] = a = tally_join(a, part[threadIdx.x + half * rows], c);
    __syncthreads();
  }
  if (slice == 0 && row < p.T) {
    const int64_t id = p.ids[row];
    out_lp[row] = id < 0 ? 0.f : id >= p.V ? -INFINITY : tally_logprob(a, p.given[row], scale);
    out_entropy[row] = tally_entropy(a);
  }
}

// Columns of a tile: the width whose rounds over the 74 pairs of SMs cost least, a round as its columns and some 32 for its ends.
static int head_cols(int rows, int vocab) {
  const int64_t m_tiles = (rows + 2 * kHeadRows - 1) / (2 * kHeadRows);
  int64_t best = 0;
  int cols = kHeadCols;
  for (int c = kHeadCols; c >= 128; c -= 32) {
    const int64_t tiles = m_tiles * ((vocab + c - 1) / c), cost = (tiles + 73) / 74 * (c + 32);
    if (best == 0 || cost < best) {
      best = cost;
      cols = c;
    }
  }
  return cols;
}

}  // namespace xllm

// Bytes of workspace of xllm_head_logprobs.
XLLM_API int64_t xllm_head_logprobs_workspace(int rows, int vocab) {
  using namespace xllm;
  const int cols = head_cols(rows, vocab);
  return ((int64_t)((vocab + cols - 1) / cols) * sizeof(Tally) + sizeof(float)) * rows;
}

// Reads and clears the error word: non-zero when a bounded wait expired since the last query.
XLLM_API int xllm_head_logprobs_error_status() {
  using namespace xllm;
  int v = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_head_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_head_error, &zero, sizeof(int));
  return v;
}

// hidden [rows, width] and weight [vocab, width] bf16, row strides ldh and ldw in elements; width, ldh and ldw % 8 == 0, 16-byte
// aligned bases.  ids int64 [rows], temperature fp32 [rows] or null.
XLLM_API int xllm_head_logprobs(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int rows, int vocab, int width,
                                const void* ids, const void* temperature, void* workspace, void* out_lp, void* out_entropy,
                                void* stream) {
  using namespace xllm;
  if (rows == 0) return 0;
  if (rows < 0 || vocab < 1 || width < 1 || width % 8 || ldh % 8 || ldw % 8) return (int)cudaErrorInvalidValue;
  if (((uintptr_t)hidden | (uintptr_t)weight) & 15) return (int)cudaErrorInvalidValue;
  int dev = 0;
  cudaGetDevice(&dev);
  static bool attr_done[64] = {};
  if (!attr_done[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(head_tally_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeadSmem);
    if (e != cudaSuccess) return (int)e;
    attr_done[dev & 63] = true;
  }
  const int cols = head_cols(rows, vocab), n_tiles = (vocab + cols - 1) / cols;
  const int m_tiles = (rows + 2 * kHeadRows - 1) / (2 * kHeadRows), a_box = rows >= kHeadRows ? kHeadRows : (rows + 7) & ~7;
  if ((int64_t)m_tiles * n_tiles > 0x7fffffff) return (int)cudaErrorInvalidValue;
  CUtensorMap map_h, map_w;
  if (!make_map(&map_h, hidden, rows, width, ldh, a_box) || !make_map(&map_w, weight, vocab, width, ldw, cols / 2))
    return (int)cudaErrorInvalidValue;
  Tally* tallies = (Tally*)workspace;
  const HeadParams p{rows, vocab, width, cols, n_tiles, m_tiles, a_box, (const int64_t*)ids, (const float*)temperature, tallies,
                     (float*)(tallies + (int64_t)n_tiles * rows)};
  cudaStream_t s = (cudaStream_t)stream;
  const int pairs = m_tiles * n_tiles < 74 ? m_tiles * n_tiles : 74;
  cudaError_t e = launch_pdl(head_tally_kernel, dim3(2 * pairs), dim3(kHeadThreads), kHeadSmem, s, map_h, map_w, p);
  if (e != cudaSuccess) return (int)e;
  int join = 1;
  while (join < 32 && join < rows) join *= 2;
  e = launch_pdl(head_join_kernel, dim3((rows + join - 1) / join), dim3(256), 0, s, p, join, (float*)out_lp, (float*)out_entropy);
  return e != cudaSuccess ? (int)e : XLLM_LAUNCH_CHECK();
}
