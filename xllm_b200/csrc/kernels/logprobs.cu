// Log-probabilities of given tokens with the entropy and the most likely alternatives of their rows (contract: ops/score.py).
//
// A row is read once.  A thread keeps a tally (logprob_math.cuh) of its 16-byte vectors: the maximum of a group of vectors
// first, so that what is summed so far is rebased at most once a group.  Few rows are cut into parts, one block of a cluster
// each, and joined through distributed shared memory in the parts' order.
//
// Alternatives: a thread's maximum is one of the row's scores, so the n-th largest of the threads' (or of groups of threads')
// maxima bounds the n-th largest score from below.  Only the vectors of the threads whose maximum reaches it are read again
// (from L2; about n of a block's threads), the scores that reach it, some 2 n, are listed, and a score's place in the order
// (score, lowest index first) is the number of listed ones in front of it.  A list that overflows (thousands of ties, or
// scores in ascending order) is made by one pass over the part for each place instead.
#include "logprob_math.cuh"
#include "tc_common.cuh"
#include "vec_io.cuh"

namespace xllm {

constexpr int kScoreThreads = 256;
constexpr int kScoreListed = 2048;         // candidates of a part; also 16 parts x 128 alternatives
constexpr int kScoreMaxTop = 128, kScoreMaxSplit = 16;

struct ScoreParams {
  const void* logits;
  int64_t row_stride;
  int V, n_top;
  const int64_t* ids;
  const float* temperature;
  float* out_lp;
  float* out_entropy;
  int32_t* out_ids;
  float* out_lps;
};

// Unique keys in the order (score, lowest index first); 0 is nobody's.  -0 ties with 0.
__device__ __forceinline__ uint64_t score_key(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (uint64_t)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32 | (0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ float key_score(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xFFFFFFFFu - (uint32_t)k); }

// One 16-byte vector of scores.
template <typename T>
struct ScoreVec {
  static constexpr int N = 16 / (int)sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void nothing() {                      // -inf everywhere
    raw.x = raw.y = raw.z = raw.w = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  }
  __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
  __device__ __forceinline__ f32x2 pair(int i) const {             // scores 2 i and 2 i + 1
    if constexpr (sizeof(T) == 2) return {__uint_as_float(word(i) << 16), __uint_as_float(word(i) & 0xFFFF0000u)};
    else return {__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1))};
  }
};
template <int U>
__device__ __forceinline__ float vec_max(const ScoreVec<bf16>* v) {
  bf162 m = *reinterpret_cast<const bf162*>(&v[0].raw.x);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = v[u].word(i);
      m = __hmax2(m, *reinterpret_cast<const bf162*>(&w));         // a NaN loses against a number
    }
  const float2 f = __bfloat1622float2(m);
  return fmaxf(f.x, f.y);
}
template <int U>
__device__ __forceinline__ float vec_max(const ScoreVec<float>* v) {
  float m = __uint_as_float(v[0].raw.x);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(v[u].word(i)));
  return m;
}

__device__ __forceinline__ void tally_add(Tally& a, float x, float c) {
  if (x > a.m) tally_rebase(a, x, c);
  const float t = bounded((x - a.m) * c), e = exp2_fast(t);
  a.z += e;
  a.s = fmaf(e, t, a.s);
}

// The block's tally from its threads', in a fixed order; `red` is shared memory for 8 tallies.
__device__ __forceinline__ Tally block_tally(Tally a, float c, Tally* red) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  tally_rebase(a, warp_max(a.m), c);
  a.z = warp_sum(a.z);
  a.s = warp_sum(a.s);
  if (lane == 0) red[wid] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < kScoreThreads / 32; ++w) a = tally_join(a, red[w], c);
  return a;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float remote_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t remote_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

struct ScoreShared {
  alignas(16) float most[kScoreThreads];    // read four at a time
  Tally red[kScoreThreads / 32];
  Tally part;                               // this block's, for the first block of the cluster
  int chosen[kScoreThreads];
  uint64_t top[kScoreMaxTop];
  uint64_t listed[kScoreListed];
  uint64_t best[kScoreThreads / 32];
  float bound;
  int n_chosen, n_listed;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads, 5) token_logprobs_kernel(ScoreParams p) {
  using Vec = ScoreVec<T>;
  constexpr int U = 4;
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int split = (int)cluster_size(), part = (int)tc::cluster_rank();
  const int row = blockIdx.x / split;
  pdl_wait();
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
  const float scale = row_scale(p.temperature, row), c = scale * kLog2e;
  // aligned vectors between a head and a tail of single scores
  const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int head = off == 0 ? 0 : min(p.V, Vec::N - off);
  const int n_vec = (p.V - head) / Vec::N, tail = head + n_vec * Vec::N;
  const int v0 = (int)((int64_t)n_vec * part / split), v1 = (int)((int64_t)n_vec * (part + 1) / split);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const int single = part == 0 && tid < head ? tid : part == split - 1 && tid >= 32 && tail + tid - 32 < p.V ? tail + tid - 32 : -1;

  PairTally run = pair_empty();
  for (int j = v0 + tid; j < v1; j += kScoreThreads * U) {
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = j + u * kScoreThreads;
      if (at < v1) v[u].raw = __ldg(xv + at);
      else v[u].nothing();
    }
    const float m = vec_max<U>(v);
    if (m > run.m) pair_rebase(run, m, c);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < Vec::N / 2; ++i) pair_add(run, v[u].pair(i), c);
  }
  Tally a = pair_sum(run);
  if (single >= 0) tally_add(a, to_f32(x[single]), c);

  const int n = p.n_top;
  if constexpr (TOP) {
    // groups of 4 threads are enough to bound few alternatives, and 16 times fewer comparisons
    const int width = n <= 32 ? 4 : 1, groups = kScoreThreads / width;
    float most = a.m;
    if (width == 4) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    }
    if (tid % width == 0) sh.most[tid / width] = most;
    if (tid == 0) sh.n_chosen = sh.n_listed = 0;
    __syncthreads();
    if (tid < groups) {
      const float mine = sh.most[tid];
      int above = 0, same = 0;
      for (int i = 0; i < groups; i += 4) {
        const float4 o = *reinterpret_cast<const float4*>(sh.most + i);
        above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
        same += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
      }
      if (above < n && above + same >= n) sh.bound = mine;
    }
    __syncthreads();
    const float bound = sh.bound;
    if (a.m >= bound) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = tid;
    const auto list = [&](float v, int i) {
      if (v >= bound && v > -INFINITY) {
        const int at = atomicAdd(&sh.n_listed, 1);
        if (at < kScoreListed) sh.listed[at] = score_key(v, i);
      }
    };
    if (single >= 0) list(to_f32(x[single]), single);
    __syncthreads();
    const int each = (v1 - v0 + kScoreThreads - 1) / kScoreThreads, items = sh.n_chosen * each;
    for (int i = tid; i < items; i += kScoreThreads) {
      const int at = v0 + sh.chosen[i / each] + i % each * kScoreThreads;
      if (at < v1) {
        Vec v;
        v.raw = __ldg(xv + at);
#pragma unroll
        for (int k = 0; k < Vec::N / 2; ++k) {
          const f32x2 f = v.pair(k);
          list(f.x, head + at * Vec::N + 2 * k);
          list(f.y, head + at * Vec::N + 2 * k + 1);
        }
      }
    }
    if (tid < n) sh.top[tid] = 0;
    __syncthreads();
    const int n_listed = sh.n_listed;
    if (n_listed <= kScoreListed) {
      for (int i = tid; i < n_listed; i += kScoreThreads) {
        const uint64_t mine = sh.listed[i];
        int place = 0;
        for (int k = 0; k < n_listed; ++k) place += sh.listed[k] > mine;
        if (place < n) sh.top[place] = mine;
      }
    } else {
      uint64_t last = ~0ull;
      for (int k = 0; k < n; ++k) {
        uint64_t most_key = 0;
        const auto look = [&](float v, int i) {
          const uint64_t key = v > -INFINITY ? score_key(v, i) : 0;
          if (key < last && key > most_key) most_key = key;
        };
        if (single >= 0) look(to_f32(x[single]), single);
        for (int j = v0 + tid; j < v1; j += kScoreThreads) {
          Vec v;
          v.raw = __ldg(xv + j);
#pragma unroll
          for (int q = 0; q < Vec::N / 2; ++q) {
            const f32x2 f = v.pair(q);
            look(f.x, head + j * Vec::N + 2 * q);
            look(f.y, head + j * Vec::N + 2 * q + 1);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most_key = max(most_key, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)most_key, o));
        if (lane == 0) sh.best[wid] = most_key;
        __syncthreads();
        for (int w = 0; w < kScoreThreads / 32; ++w) most_key = max(most_key, sh.best[w]);
        if (tid == 0) sh.top[k] = most_key;
        last = most_key;
        __syncthreads();
        if (last == 0) break;                        // uniform: nobody is left
      }
    }
  }
  a = block_tally(a, c, sh.red);

  if (split > 1) {
    if (tid == 0) sh.part = a;
    tc::cluster_sync();
    if (part == 0) {
      a = tally_empty();
      for (int r = 0; r < split; ++r) {
        const uint32_t at = tc::in_cta(smem_u32(&sh.part), r);
        a = tally_join(a, {remote_f32(at), remote_f32(at + 4), remote_f32(at + 8)}, c);
      }
      if constexpr (TOP) {
        for (int i = tid; i < split * n; i += kScoreThreads) sh.listed[i] = remote_u64(tc::in_cta(smem_u32(sh.top + i % n), i / n));
        __syncthreads();
        uint64_t mine[kScoreListed / kScoreThreads];
        int place[kScoreListed / kScoreThreads];
#pragma unroll
        for (int q = 0; q < kScoreListed / kScoreThreads; ++q) {
          const int i = tid + q * kScoreThreads;
          mine[q] = 0;
          if (i < split * n) {
            mine[q] = sh.listed[i];
            place[q] = 0;
            for (int k = 0; k < split * n; ++k) place[q] += sh.listed[k] > mine[q];
          }
        }
        tc::cluster_sync();                              // the others' places have been read; every block passes here once
        if (tid < n) sh.top[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < kScoreListed / kScoreThreads; ++q)
          if (mine[q] != 0 && place[q] < n) sh.top[place[q]] = mine[q];
      } else {
        tc::cluster_sync();
      }
    } else {
      tc::cluster_sync();
      return;
    }
  }
  if (tid == 0) {
    const int64_t id = p.ids[row];
    p.out_lp[row] = id < 0 ? 0.f : id >= p.V ? -INFINITY : tally_logprob(a, to_f32(x[id]), scale);
    p.out_entropy[row] = tally_entropy(a);
  }
  if constexpr (TOP) {
    __syncthreads();
    if (tid < n) {
      const uint64_t k = sh.top[tid];
      p.out_ids[(int64_t)row * n + tid] = k == 0 ? -1 : key_index(k);
      p.out_lps[(int64_t)row * n + tid] = k == 0 ? -INFINITY : tally_logprob(a, key_score(k), scale);
    }
  }
}

template <typename T, bool TOP>
static int launch_token_logprobs(const ScoreParams& p, int rows, int split, cudaStream_t s) {
  auto kernel = token_logprobs_kernel<T, TOP>;
  if (split > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return (int)e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * split));
  cfg.blockDim = dim3(kScoreThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e != cudaSuccess ? (int)e : XLLM_LAUNCH_CHECK();
}

static int score_split(int rows, int V) {
  int split = 1;
  while (split < kScoreMaxSplit && rows * split * 2 <= 740 && V / (split * 2) >= 2048) split *= 2;
  return split;
}

}  // namespace xllm

// dtype: 0 = bf16 logits, 1 = fp32 logits; ids int64 [rows], temperature fp32 [rows] or null; out_ids, out_lps [rows, n_top].
XLLM_API int xllm_token_logprobs(const void* logits, int64_t row_stride, int dtype, int rows, int vocab, const void* ids,
                                 const void* temperature, int n_top, void* out_lp, void* out_entropy, void* out_ids,
                                 void* out_lps, void* stream) {
  using namespace xllm;
  if (rows == 0) return 0;
  if (rows < 0 || vocab < 1 || n_top < 0 || n_top > vocab || n_top > kScoreMaxTop || (dtype != 0 && dtype != 1))
    return (int)cudaErrorInvalidValue;
  const ScoreParams p{logits, row_stride, vocab, n_top, (const int64_t*)ids, (const float*)temperature, (float*)out_lp,
                      (float*)out_entropy, (int32_t*)out_ids, (float*)out_lps};
  const int split = score_split(rows, vocab);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == 0) return n_top ? launch_token_logprobs<bf16, true>(p, rows, split, s) : launch_token_logprobs<bf16, false>(p, rows, split, s);
  return n_top ? launch_token_logprobs<float, true>(p, rows, split, s) : launch_token_logprobs<float, false>(p, rows, split, s);
}
