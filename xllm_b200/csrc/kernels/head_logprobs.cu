// Log-probabilities and entropies straight from hidden states and the output projection (contract: ops/score.py): the scores
// x = h W^T are tallied where they are computed, in the tensor cores' accumulators, and never stored.
//
//   head_tally_kernel  tiles of 256 rows x up to 256 columns of the vocabulary: the rows' tallies (logprob_math.cuh) of the tile's
//                      columns, and the given token's score from whichever tile holds it
//   head_join_kernel   a row's tallies over all tiles, joined in a fixed order
//
// Many rows: a tile is a pair of CTAs' (cta_group::2), each loads its 128 rows of h and half of the columns' rows of W by TMA into
// a ring of stages, one thread of the pair's first CTA issues the products into one of two accumulators in tensor memory, and eight
// warps of each CTA read the other one back, two threads a row, 32 columns at a time.  Bound by the tensor cores; the tally (some
// 4500 cycles a tile) hides behind the next tile's products where K is 512 and more.
// Up to 128 rows: a tile is one CTA's and bound by W's way from HBM, and for long by the power that memory and products draw together:
// up to 64 rows are multiplied by instructions of 64 (for seconds 3 % quicker than by those of 128, 45 x 2048 x 151936 and 1 x 4096).  An
// SM's share of the bandwidth depends on its die (of two equal shares one was read in 176 us, the other in 203), so a CTA that is done
// takes over one that has not started.
//
//   one B200             floor   time  for seconds        (us, back to back from a graph; 6536 GB/s, 1670 TFLOP/s)
//   1 x 4096 x 151936      190    192    194    6.5 TB/s
//   45 x 2048 x 151936      95    100    106
//   128 x 4096 x 151936    191    202    227    power, of memory and products
//   200 x 4096 x 151936    191    252    313    the same, of products of 256 rows; 10 more with takeover by pairs, 15 with 256 rows on a single CTA
//   1000 x 4096 x 32768    161    180    213
//   4096 x 512 x 151936    382    450           the tally
//   4096 x 4096 x 151936  3053   3060   3520    the burst rate; for seconds above the sustained one (3626)
//
// The tensor cores cut a sum of products off at each of its K / 16 steps, by 2^-26 of what is there on average (measured against 64 bits:
// scores of dense rows come out smaller by 0.94e-9 K of themselves, those of one large channel in front of all others by twice that).  So
// no more than 1024 products are summed there: longer rows in chunks of up to 896, whose sums are added up in fp32, with rounding, by the
// threads that read the accumulators.  Off against 64 bits, relative, 1000 x 4096 x 32768: log-probabilities 3.2e-7, entropies 2.0e-7 (a
// product in fp32 3.5e-7 and 1.4e-7; unchunked 1.5e-6).  Chunks cost time where power is short: 4096 x 1536 x
// 151936 for seconds 1388 us, 1358 unchunked; 200 x 4096 x 151936 313 and 308; 4096 x 4096 x 151936 nothing, in chunks of 512 4 %.
//
// Every wait is bounded; on expiry the kernel raises an error word and the call's own, all roles leave their loops, tensor memory is
// freed and the kernel returns.  What the call's tiles would have been is then not there: all its results are NaN.
#include "logprob_math.cuh"
#include "tc_common.cuh"
#include "vec_io.cuh"

namespace xllm {

using namespace tc;

constexpr int kHeadRows = 128, kHeadCols = 256, kHeadK = 64;        // rows of a CTA, most columns of a tile, a K block
constexpr int kHeadWarps = 8, kHeadThreads = 64 + 32 * kHeadWarps, kHeadMostStages = 16;
constexpr int kHeadRing = 7 * 32 * 1024;                            // bytes of the ring of stages
constexpr int kHeadBars = 2 * kHeadMostStages + 16;
constexpr int kHeadFixed = 2 * 16 + kHeadBars * 8 + 16;                // behind it: answers, barriers, two words; then tallies of 128 rows
constexpr int kHeadSmem = kHeadRing + kHeadFixed + kHeadRows * sizeof(Tally) + 1024;
static_assert(kHeadSmem <= 232448, "exceeds the 227 KB of shared memory per CTA");

constexpr int kHeadOne = 16, kHeadChunk = 14;                       // most K blocks that are summed in tensor memory: alone, and as a chunk

__device__ int g_head_error = 0;

// workspace: tallies (m, z, s, -) [rows][column tiles], the given tokens' scores [rows], and whether a wait of this call expired
struct HeadParams {
  int T, V, K, cols, n_tiles, m_tiles;
  int a_box, per_stage, stages, chunk;                // rows of h that are loaded, K blocks of a stage, stages, K blocks of a chunk
  int m_rows, zeros;                                  // rows of an instruction of a single CTA, 64 or 128; the others are zeros
  const int64_t* ids;
  const float* temperature;
  float4* tallies;
  float* given;
  int* lost;
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

// adds the first `left` of 32 columns
__device__ __forceinline__ void tally_columns(PairTally& run, float* x, int left, float c) {
  if (left < 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i >= left) x[i] = -INFINITY;
  }
  float most[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    most[k] = x[k];
#pragma unroll
    for (int i = k + 4; i < 32; i += 4) most[k] = fmaxf(most[k], x[i]);
  }
  most[0] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  if (most[0] > run.m) pair_rebase(run, most[0], c);
#pragma unroll
  for (int i = 0; i < 32; i += 2) pair_add(run, {x[i], x[i + 1]}, c);
}
// x += 32 columns of an accumulator, 16 at a time: the threads that do have no registers to spare, and next to no L1 for what is spilled
__device__ __forceinline__ void add_columns(uint32_t taddr, float* x) {
#pragma unroll
  for (int k = 0; k < 32; k += 16) {
    uint32_t r[16];
    tmem_ld16(taddr + k, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) x[k + i] += __uint_as_float(r[i]);
  }
}

// ONE: a row's K blocks are one chunk.
template <bool PAIR, bool ONE>
__global__ void __launch_bounds__(kHeadThreads, 1)
head_tally_kernel(const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_w, const HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem), answer0 = sbase + kHeadRing, bar0 = answer0 + 32;
  const auto full_bar = [&](int s) { return bar0 + 8u * s; };
  const auto empty_bar = [&](int s) { return bar0 + 8u * (kHeadMostStages + s); };
  const auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kHeadMostStages + a); };
  const auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kHeadMostStages + 2 + a); };
  const auto next_bar = [&](int a) { return bar0 + 8u * (2 * kHeadMostStages + 4 + a); };       // an answer has arrived
  const auto read_bar = [&](int a) { return bar0 + 8u * (2 * kHeadMostStages + 6 + a); };       // all warps have read it
  const auto give_bar = [&](int q) { return bar0 + 8u * (2 * kHeadMostStages + 8 + q); };       // one thread's tally of a row lies there
  const auto took_bar = [&](int q) { return bar0 + 8u * (2 * kHeadMostStages + 12 + q); };      // the row's other thread has read it
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + kHeadRing + 32 + kHeadBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0u;
  const int units = p.m_tiles * p.n_tiles, k_blocks = (p.K + kHeadK - 1) / kHeadK;
  const int w_rows = PAIR ? p.cols / 2 : p.cols;                                  // of W that this CTA loads for a tile
  const int a_bytes = (PAIR ? kHeadRows : p.m_rows) * kHeadK * 2;
  const int block_bytes = a_bytes + w_rows * kHeadK * 2, loaded = (p.a_box + w_rows) * kHeadK * 2;       // of a K block
  const int stage_bytes = p.per_stage * block_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), PAIR ? 2 * kHeadWarps : kHeadWarps);
      mbar_init(next_bar(a), 1);
      mbar_init(read_bar(a), 2 + kHeadWarps);
    }
    for (int q = 0; q < 4; ++q) {
      mbar_init(give_bar(q), 1);
      mbar_init(took_bar(q), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Rows of h that are not there are zeros: what else lies in shared memory would be multiplied all the same, and draw power that the
  // memory needs (one row x 4096 x 151936, sustained: 201 us at 1.4 GHz, 214 us at 0.86 GHz without).  Not where a call is too short
  // for that to count, but not for the writing (64 x 512 x 32003: 15.3 us, 14.6 without).
  if (p.zeros) {
    const int vecs = a_bytes / 16 - p.a_box * 8, blocks = p.stages * p.per_stage;
    uint4* at = reinterpret_cast<uint4*>(smem + p.a_box * kHeadK * 2) + threadIdx.x;
    for (int b = 0; b < blocks; ++b, at += block_bytes / 16)
      for (int i = threadIdx.x; i < vecs; i += kHeadThreads) at[i - threadIdx.x] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::%1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_holder)), "n"(PAIR ? 2 : 1)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::%0.sync.aligned;" ::"n"(PAIR ? 2 : 1));
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();                 // both CTAs' barriers exist before anything can signal them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_wait();
  pdl_launch_dependents();                            // after the allocation: what starts early may want tensor memory too

  // The tile behind the t-th one, u, of this CTA or pair, or -1: pairs take turns, a single CTA takes over one that has not started.
  const auto next_unit = [&](int u, int t, bool& ok) {
    if constexpr (PAIR) {
      u += gridDim.x >> 1;
      return u < units ? u : -1;
    } else {
      if (!mbar_wait_warp(next_bar(t & 1), (t >> 1) & 1, abort_flag)) { ok = false; return -1; }
      const int taken = taken_cta(answer0 + 16 * (t & 1));
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // before the place is written again
      __syncwarp();
      if (lane == 0) mbar_arrive(read_bar(t & 1));
      return taken;
    }
  };
  const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x;

  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    int stage = 0, t = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = first; u >= 0 && ok; u = next_unit(u, t, ok), ++t) {
      if constexpr (!PAIR) {
        if (!mbar_wait_warp(read_bar(t & 1), ((t >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
        if (elect_one()) {
          mbar_expect_tx(next_bar(t & 1), 16);
          take_cta(answer0 + 16 * (t & 1), next_bar(t & 1));
        }
        __syncwarp();
      }
      int m, n;
      head_tile(p, u, m, n);
      const int m0 = m * 2 * kHeadRows + (int)rank * kHeadRows, n0 = n * p.cols + (int)rank * w_rows;
      for (int kb = 0; kb < k_blocks; kb += p.per_stage) {
        if (!mbar_wait_warp(empty_bar(stage), phase ^ 1, abort_flag)) { ok = false; break; }
        const int blocks = min(p.per_stage, k_blocks - kb);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(full_bar(stage), (PAIR ? 2u : 1u) * blocks * loaded);
          for (int i = 0; i < blocks; ++i) {
            const uint32_t dst = sbase + stage * stage_bytes + i * block_bytes;
            if constexpr (PAIR) {
              tma_load_2d_pair(dst, &map_h, (kb + i) * kHeadK, m0, full_bar(stage));
              tma_load_2d_pair(dst + a_bytes, &map_w, (kb + i) * kHeadK, n0, full_bar(stage));
            } else {
              tma_load_2d(dst, &map_h, (kb + i) * kHeadK, m0, full_bar(stage));
              tma_load_2d(dst + a_bytes, &map_w, (kb + i) * kHeadK, n0, full_bar(stage));
            }
          }
        }
        __syncwarp();
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------------------------------------------------------- products (a pair's first CTA)
      const uint32_t id = PAIR ? idesc_pair(p.cols) : idesc(false, p.cols, p.m_rows);
      int stage = 0, t = 0, chunks = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = first; u >= 0 && ok; u = next_unit(u, t, ok), ++t) {
        for (int kc = 0; kc < k_blocks && ok; kc += p.chunk, ++chunks) {
          const int acc = chunks & 1, end = min(kc + p.chunk, k_blocks);
          const uint32_t parity = ((chunks >> 1) & 1) ^ 1;
          if (!(PAIR ? mbar_wait_cluster_warp(tempty_bar(acc), parity, abort_flag) : mbar_wait_warp(tempty_bar(acc), parity, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + acc * kHeadCols;
          for (int kb = kc; kb < end; kb += p.per_stage) {
            if (!mbar_wait_warp(full_bar(stage), phase, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const int blocks = min(p.per_stage, end - kb);
            if (elect_one()) {
              for (int i = 0; i < blocks; ++i) {
                const uint32_t at = sbase + stage * stage_bytes + i * block_bytes;
                const uint64_t a = smem_desc(at, 16, 1024), b = smem_desc(at + a_bytes, 16, 1024);
#pragma unroll
                for (int k = 0; k < kHeadK / 16; ++k) {
                  if constexpr (PAIR) umma_pair(d, a + 2 * k, b + 2 * k, id, (kb + i - kc | k) != 0);
                  else umma(d, a + 2 * k, b + 2 * k, id, (kb + i - kc | k) != 0);
                }
              }
              if constexpr (PAIR) umma_commit_pair(empty_bar(stage));
              else umma_commit(empty_bar(stage));
            }
            __syncwarp();
            if (++stage == p.stages) { stage = 0; phase ^= 1; }
          }
          if (ok && elect_one()) {
            if constexpr (PAIR) umma_commit_pair(tfull_bar(acc));
            else umma_commit(tfull_bar(acc));
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ tallies, two threads a row: every other 32 columns
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t leader_tempty = PAIR ? in_cta(tempty_bar(0), 0) : 0u;
    // of an instruction of 64 rows, 16 lie in every 32 lanes of tensor memory
    const bool half_rows = !PAIR && p.m_rows == 64;
    const auto row_of = [&](int m) { return m * 2 * kHeadRows + (int)rank * kHeadRows + q * (half_rows ? 16 : 32); };
    const int lane_row = half_rows && lane >= 16 ? p.T : lane;       // or none
    // a row's token and temperature are fetched a tile ahead
    int64_t id_next = -1;
    float c_next = kLog2e;
    const auto fetch = [&](int m) {
      const int row = row_of(m) + lane_row;
      id_next = row < p.T ? p.ids[row] : -1;
      c_next = (row < p.T ? row_scale(p.temperature, row) : 1.f) * kLog2e;
    };
    int t = 0, chunks = 0, m, n, m_next, n_next, given_over = 0;
    bool ok = true;
    head_tile(p, first, m_next, n_next);
    fetch(m_next);
    for (int u = first; u >= 0 && ok; u = next_unit(u, t, ok), ++t) {
      m = m_next;
      n = PAIR ? n_next : u;
      const int row0 = row_of(m), row = row0 + lane_row, n0 = n * p.cols;
      const float c = c_next;
      const int64_t want = id_next - n0;              // the given token's column, if it is one of this tile's
      if (u == 0 && rank == 0 && threadIdx.x == 64) *p.lost = 0;         // long before a wait can expire
      if (PAIR && u + (int)(gridDim.x >> 1) < units) {
        head_tile(p, u + (gridDim.x >> 1), m_next, n_next);
        if (m_next != m) fetch(m_next);
      }
      const int width = min(p.V - n0, p.cols);
      const bool idle = row0 >= p.T || half * 32 >= width;
      const uint32_t lanes = tmem_base + ((uint32_t)(q * 32) << 16) + half * 32;
      const auto wait = [&] {
        if (!mbar_wait_warp(tfull_bar(chunks & 1), (chunks >> 1) & 1, abort_flag)) ok = false;
        tc_fence_after();
        return ok;
      };
      // the accumulator is free once its columns are in registers
      const auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_remote(leader_tempty + 8u * (chunks & 1));
          else mbar_arrive(tempty_bar(chunks & 1));
        }
      };
      // where the given token is one of 32 columns
      const auto keep_given = [&](const float* x, int c0, int left) {
        const bool here = want >= c0 && want < c0 + left;
        if (!__any_sync(0xffffffffu, here)) return;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (want == c0 + i) v = x[i];
        if (here) p.given[row] = v;
      };
      PairTally run = pair_empty();
      if constexpr (ONE) {
        if (!wait()) break;
        if (idle) {
          release();
        } else {
          const uint32_t taddr = lanes - half * 32 + (chunks & 1) * kHeadCols;
          for (int c0 = half * 32; c0 < width; c0 += 64) {
            float x[32];
            tmem_ld32(taddr + c0, reinterpret_cast<uint32_t*>(x));
            tmem_ld_wait();
            if (c0 + 64 >= width) release();
            const int left = min(32, width - c0);
            tally_columns(run, x, left, c);
            keep_given(x, c0, left);
          }
        }
        ++chunks;
      } else {
        // all of the thread's columns, summed over the chunks
        float x[kHeadCols / 64][32];
        for (int kc = 0; kc < k_blocks; kc += p.chunk, ++chunks) {
          if (!wait()) break;
          const uint32_t taddr = lanes + (chunks & 1) * kHeadCols;
          if (!idle && kc == 0) {
#pragma unroll
            for (int j = 0; j < kHeadCols / 64; ++j)
              if (half * 32 + 64 * j < width) tmem_ld32(taddr + 64 * j, reinterpret_cast<uint32_t*>(x[j]));
            tmem_ld_wait();
          } else if (!idle) {
#pragma unroll
            for (int j = 0; j < kHeadCols / 64; ++j)
              if (half * 32 + 64 * j < width) add_columns(taddr + 64 * j, x[j]);
          }
          release();
        }
        if (!ok) break;
        if (!idle) {
#pragma unroll
          for (int j = 0; j < kHeadCols / 64; ++j) {
            const int c0 = half * 32 + 64 * j, left = min(32, width - c0);
            if (left <= 0) continue;
            tally_columns(run, x[j], left, c);
            keep_given(x[j], c0, left);
          }
        }
      }
      if (row0 < p.T) {
        // One thread of the row gives its tally to the other.  Bounded like every wait: a warp that has left its role is not waited for.
        const Tally a = pair_sum(run);
        Tally* other = reinterpret_cast<Tally*>(smem + kHeadRing + kHeadFixed) + q * 32 + lane;
        const uint32_t parity = given_over++ & 1;
        if (!mbar_wait_warp(half == 1 ? took_bar(q) : give_bar(q), half == 1 ? parity ^ 1 : parity, abort_flag)) break;
        if (half == 1) {
          *other = a;
        } else {
          const Tally both = tally_join(a, *other, c);
          if (row < p.T) p.tallies[(int64_t)row * p.n_tiles + n] = make_float4(both.m, both.z, both.s, 0.f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(half == 1 ? give_bar(q) : took_bar(q));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 20000000LL) {}            // copies, products and answers in flight, whichever role gave up
    if (threadIdx.x == 0) {
      atomicExch(&g_head_error, 1);
      atomicExch(p.lost, 1);
    }
  }
  if constexpr (PAIR) cluster_sync();                 // neither CTA leaves while the other may touch its barriers or memory
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::%1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base), "n"(PAIR ? 2 : 1));
  }
}

// `threads` of a block (a warp, or all of them) join a row: a thread every so many tiles, then in pairs.
__global__ void __launch_bounds__(256) head_join_kernel(const HeadParams p, int threads, float* out_lp, float* out_entropy) {
  __shared__ Tally part[8];
  pdl_wait();
  const int t = threadIdx.x % threads, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * (256 / threads) + threadIdx.x / threads;
  if (row >= p.T) return;                            // whole warps; no block is left by some of the threads of a row
  const float scale = row_scale(p.temperature, row), c = scale * kLog2e;
  const int64_t id = p.ids[row];
  const bool given = id >= 0 && id < p.V, lost = *p.lost != 0;
  const float x = given ? p.given[row] : 0.f;        // on its way while the tallies are joined
  const float4* tallies = p.tallies + row * p.n_tiles;
  Tally a = tally_empty();
  for (int i = t; i < p.n_tiles; i += 4 * threads) {
    Tally b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] = tally_empty();
      if (i + j * threads < p.n_tiles) {
        const float4 v = tallies[i + j * threads];
        b[j] = {v.x, v.y, v.z};
      }
    }
    a = tally_join(a, tally_join(tally_join(b[0], b[1], c), tally_join(b[2], b[3], c), c), c);
  }
  tally_rebase(a, warp_max(a.m), c);
  a.z = warp_sum(a.z);
  a.s = warp_sum(a.s);
  if (threads > 32) {
    if (lane == 0) part[wid] = a;
    __syncthreads();
    a = part[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) a = tally_join(a, part[w], c);
  }
  if (t != 0) return;
  // a given token's score is one of those that the tally is made of: no more than its maximum, so that no log-probability is above 0
  const float lp = given ? tally_logprob(a, x, scale) : id < 0 ? 0.f : -INFINITY;
  out_lp[row] = lost ? NAN : lp;
  out_entropy[row] = lost ? NAN : tally_entropy(a);
}

// Columns of a tile: the width whose rounds over the SMs (or pairs of them) and last tally cost least.  A round costs its columns and
// some 16 (a pair's some 32) for its ends; a tally 16 ns a column, where loading a column takes an SM 0.045 ns K.
static int head_cols(int rows, int vocab, int width) {
  const bool pair = rows > kHeadRows;
  const int64_t m_tiles = (rows + 2 * kHeadRows - 1) / (2 * kHeadRows), slots = pair ? 74 : 148;
  double best = 0;
  int cols = kHeadCols;
  for (int c = kHeadCols; c >= 128; c -= 16) {
    const int64_t tiles = m_tiles * ((vocab + c - 1) / c);
    const double cost = (double)((tiles + slots - 1) / slots) * (c + (pair ? 32 : 16)) + c * 350. / width;
    if (best == 0 || cost < best) {
      best = cost;
      cols = c;
    }
  }
  return cols;
}

template <bool PAIR, bool ONE>
static cudaError_t launch_head_tally(const CUtensorMap& h, const CUtensorMap& w, const HeadParams& p, int ctas, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  static bool attr_done[64] = {};
  if (!attr_done[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(head_tally_kernel<PAIR, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeadSmem);
    if (e != cudaSuccess) return e;
    attr_done[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kHeadThreads);
  cfg.dynamicSmemBytes = kHeadSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, head_tally_kernel<PAIR, ONE>, h, w, p);
}

}  // namespace xllm

// Bytes of workspace of xllm_head_logprobs.
XLLM_API int64_t xllm_head_logprobs_workspace(int rows, int vocab, int width) {
  using namespace xllm;
  const int cols = head_cols(rows, vocab, width);
  return ((int64_t)((vocab + cols - 1) / cols) * sizeof(float4) + sizeof(float)) * rows + sizeof(int);
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
  const bool pair = rows > kHeadRows;
  const int cols = head_cols(rows, vocab, width), n_tiles = (vocab + cols - 1) / cols, w_box = pair ? cols / 2 : cols;
  const int m_tiles = (rows + 2 * kHeadRows - 1) / (2 * kHeadRows), a_box = rows >= kHeadRows ? kHeadRows : (rows + 7) & ~7;
  if ((int64_t)m_tiles * n_tiles > 0x3fffffff) return (int)cudaErrorInvalidValue;
  CUtensorMap map_h, map_w;
  if (!make_map(&map_h, hidden, rows, width, ldh, a_box) || !make_map(&map_w, weight, vocab, width, ldw, w_box))
    return (int)cudaErrorInvalidValue;
  // a stage costs the issuing warps some 370 cycles whatever it holds: two K blocks where they are small (64 x 1024 x 32768: 17.5 us,
  // 19.0 with one; 128 rows in tiles of 208 columns, 4096 x 151936: 211 us, 199 with one)
  const int per_stage = a_box + w_box <= 192 ? 2 : 1;
  const int m_rows = rows <= 64 ? 64 : kHeadRows;
  int stages = kHeadRing / (per_stage * (m_rows + w_box) * kHeadK * 2);
  if (stages > kHeadMostStages) stages = kHeadMostStages;
  // chunks of one length, whole stages each
  const int k_blocks = (width + kHeadK - 1) / kHeadK, n_chunks = k_blocks <= kHeadOne ? 1 : (k_blocks + kHeadChunk - 1) / kHeadChunk;
  const int chunk = ((k_blocks + n_chunks - 1) / n_chunks + 1) & ~1;
  float4* tallies = (float4*)workspace;
  float* given = (float*)(tallies + (int64_t)n_tiles * rows);
  const int zeros = a_box < m_rows && (int64_t)vocab * width > (64 << 20);
  const HeadParams p{rows, vocab, width, cols, n_tiles, m_tiles, a_box, per_stage, stages, chunk, m_rows, zeros,
                     (const int64_t*)ids, (const float*)temperature, tallies, given, (int*)(given + rows)};
  cudaStream_t s = (cudaStream_t)stream;
  const int units = m_tiles * n_tiles;
  const auto launch = n_chunks == 1 ? pair ? launch_head_tally<true, true> : launch_head_tally<false, true>
                                    : pair ? launch_head_tally<true, false> : launch_head_tally<false, false>;
  cudaError_t e = launch(map_h, map_w, p, pair ? 2 * (units < 74 ? units : 74) : units, s);
  if (e != cudaSuccess) return (int)e;
  const int threads = rows <= 296 && n_tiles > 128 ? 256 : 32;       // a block a row while that fills the SMs
  e = launch_pdl(head_join_kernel, dim3((unsigned)(((int64_t)rows * threads + 255) / 256)), dim3(256), 0, s, p, threads, (float*)out_lp,
                 (float*)out_entropy);
  return e != cudaSuccess ? (int)e : XLLM_LAUNCH_CHECK();
}
