// Log-probabilities of given tokens with the entropy and the most likely alternatives of their rows (contract: ops/score.py).
//
// A row is read once.  A thread keeps a tally (logprob_math.cuh) of its 16-byte vectors: the maximum of a group of vectors
// first, so that what is summed so far is rebased at most once a group.  Few rows are cut into parts, one block of a cluster
// each, and joined through distributed shared memory in the parts' order.
//
// Alternatives: a thread's maximum is one of the row's scores, so the n-th largest of the maxima of 32 groups of threads (of all 256
// threads for many alternatives) bounds the n-th largest score from below.  The maximum of every group of vectors (32 bf16 scores)
// was put aside on the way, so only the some 1.5 n groups that reach the bound are read again, from L2; the scores that reach it, some
// 2 n, are listed, and a score's place in the order (score, lowest index first) is the number of listed ones in front of it.  A list
// that overflows (thousands of ties) is made by one pass over the part for each place instead.
#include "logprob_math.cuh"
#include "tc_common.cuh"
#include "vec_io.cuh"

namespace xllm {

constexpr int kScoreThreads = 256;
constexpr int kScoreListed = 2048;         // candidates of a part; of 8 parts 128 alternatives each
constexpr int kScoreGroups = 20, kScoreChosen = 512;        // groups of a thread; read again of a block's
constexpr int kScoreMaxTop = 128, kScoreMaxSplit = 8;

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

// The 256 threads that score a row (a whole block, or all but the warp that loads).
__device__ __forceinline__ void score_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The row's (or part's) tally from its threads', in a fixed order: the warps' (in front of a barrier), then all of them.
__device__ __forceinline__ void warp_tally(Tally a, float c, Tally* red) {
  tally_rebase(a, warp_max(a.m), c);
  a.z = warp_sum(a.z);
  a.s = warp_sum(a.s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
}
__device__ __forceinline__ Tally block_tally(float c, const Tally* red) {
  const int lane = threadIdx.x & 31;
  Tally a = lane < kScoreThreads / 32 ? red[lane] : tally_empty();
  tally_rebase(a, warp_max(a.m), c);
  a.z = warp_sum(a.z);
  a.s = warp_sum(a.s);
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
  float group[kScoreGroups][kScoreThreads]; // maxima of groups of vectors
  int chosen[kScoreChosen];
  uint64_t top[kScoreMaxTop];
  uint64_t listed[kScoreListed];
  uint64_t best[kScoreThreads / 32];
  float bound;
  int n_chosen, n_listed;
};

// Part `part` of `split` of a row: the aligned vectors [v0, v1) of xv, and a single score for some threads of the first and the last
// part, which have the row's head and tail.
template <typename T>
struct RowPart {
  const T* x;
  const uint4* xv;
  int head, v0, v1, single;
  __device__ __forceinline__ RowPart(const ScoreParams& p, int64_t row, int part, int split) {
    constexpr int N = ScoreVec<T>::N;
    const int tid = threadIdx.x;
    x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
    const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
    head = off == 0 ? 0 : min(p.V, N - off);
    const int n_vec = (p.V - head) / N, tail = head + n_vec * N;
    v0 = (int)((int64_t)n_vec * part / split);
    v1 = (int)((int64_t)n_vec * (part + 1) / split);
    xv = reinterpret_cast<const uint4*>(x + head);
    single = part == 0 && tid < head ? tid : part == split - 1 && tid >= 32 && tail + tid - 32 < p.V ? tail + tid - 32 : -1;
  }
};

template <typename T, int U>
__device__ __forceinline__ float tally_vectors(PairTally& run, const ScoreVec<T>* v, float c) {      // returns their maximum
  const float m = vec_max<U>(v);
  if (m > run.m) pair_rebase(run, m, c);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < ScoreVec<T>::N / 2; ++i) pair_add(run, v[u].pair(i), c);
  return m;
}

constexpr int kScoreFewTop = 24;           // alternatives that the maxima of 32 groups of threads bound well

// The threads' maxima, in front of a barrier.
__device__ __forceinline__ void share_most(float most, int n, ScoreShared& sh) {
  const int tid = threadIdx.x;
  if (n <= kScoreFewTop) {
#pragma unroll
    for (int o = 1; o < 8; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (tid % 8 == 0) sh.most[tid / 8] = most;
  } else {
    sh.most[tid] = most;
  }
  if (tid == 0) sh.n_chosen = sh.n_listed = 0;
}

// Lists the scores of the part that may be among its n largest.  A thread's group g has its vectors v0 + tid + 256 i, i in
// [g << shift, (g + 1) << shift); it has `groups` of them.  False: there are too many.
template <typename T>
__device__ __forceinline__ bool list_alternatives(const RowPart<T>& r, int groups, int shift, int n, ScoreShared& sh) {
  using Vec = ScoreVec<T>;
  const int tid = threadIdx.x, lane = tid & 31;
  float bound;
  if (n <= kScoreFewTop) {
    // the 32 groups of threads' maxima in descending order, in every warp
    float m = sh.most[lane];
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
      for (int j = k / 2; j > 0; j /= 2) {
        const float o = __shfl_xor_sync(0xffffffffu, m, j);
        m = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(m, o) : fminf(m, o);
      }
    bound = __shfl_sync(0xffffffffu, m, n - 1);
  } else {
    const float mine = sh.most[tid];
    int above = 0, same = 0;
    for (int i = 0; i < kScoreThreads; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(sh.most + i);
      above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      same += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
    }
    if (above < n && above + same >= n) sh.bound = mine;
    score_sync();
    bound = sh.bound;
  }
  const auto list = [&](float v, int i) {
    if (v >= bound && v > -INFINITY) {
      const int at = atomicAdd(&sh.n_listed, 1);
      if (at < kScoreListed) sh.listed[at] = score_key(v, i);
    }
  };
  if (r.single >= 0) list(to_f32(r.x[r.single]), r.single);
  for (int g = 0; g < groups; ++g) {
    const float v = sh.group[g][tid];
    if (v >= bound && v > -INFINITY) {
      const int at = atomicAdd(&sh.n_chosen, 1);
      if (at < kScoreChosen) sh.chosen[at] = g * kScoreThreads + tid;
    }
  }
  score_sync();
  const int n_chosen = sh.n_chosen;
  if (n_chosen > kScoreChosen) return false;
  for (int i = tid; i < n_chosen << shift; i += kScoreThreads) {
    const int chosen = sh.chosen[i >> shift], t = chosen % kScoreThreads, g = chosen / kScoreThreads;
    const int at = r.v0 + t + ((g << shift) + (i & ((1 << shift) - 1))) * kScoreThreads;
    if (at < r.v1) {
      Vec v;
      v.raw = __ldg(r.xv + at);
#pragma unroll
      for (int k = 0; k < Vec::N / 2; ++k) {
        const f32x2 f = v.pair(k);
        list(f.x, r.head + at * Vec::N + 2 * k);
        list(f.y, r.head + at * Vec::N + 2 * k + 1);
      }
    }
  }
  score_sync();
  return sh.n_listed <= kScoreListed;
}

// sh.listed: the n largest keys of the part, found by a pass over it for each; returns how many there are.
template <typename T>
__device__ __noinline__ int search_alternatives(const RowPart<T>& r, int n, ScoreShared& sh) {
  using Vec = ScoreVec<T>;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  uint64_t last = ~0ull;
  for (int k = 0; k < n; ++k) {
    uint64_t best = 0;
    const auto look = [&](float v, int i) {
      const uint64_t key = v > -INFINITY ? score_key(v, i) : 0;
      if (key < last && key > best) best = key;
    };
    if (r.single >= 0) look(to_f32(r.x[r.single]), r.single);
    for (int j = r.v0 + tid; j < r.v1; j += kScoreThreads) {
      Vec v;
      v.raw = __ldg(r.xv + j);
#pragma unroll
      for (int q = 0; q < Vec::N / 2; ++q) {
        const f32x2 f = v.pair(q);
        look(f.x, r.head + j * Vec::N + 2 * q);
        look(f.y, r.head + j * Vec::N + 2 * q + 1);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
    score_sync();                                    // the places of the round before have been read
    if (lane == 0) sh.best[wid] = best;
    score_sync();
    for (int w = 0; w < kScoreThreads / 32; ++w) best = max(best, sh.best[w]);
    if (best == 0) return k;                         // uniform: nobody is left
    if (tid == 0) sh.listed[k] = best;
    last = best;
  }
  return n;
}

// write(place, key) for the n largest of the n_listed keys of sh.listed
template <typename F>
__device__ __forceinline__ void place_alternatives(const ScoreShared& sh, int n_listed, int n, F write) {
  for (int i = threadIdx.x; i < n_listed; i += kScoreThreads) {
    const uint64_t mine = sh.listed[i];
    int place = 0;
    for (int k = 0; k < n_listed; ++k) place += sh.listed[k] > mine;
    if (mine != 0 && place < n) write(place, mine);
  }
}

// A row is a cluster's, a part a block's.  Bound by HBM and, over longer stretches, by the power that reading it and some 6 instructions a
// score draw together (4000 x 151936 bf16: 182 us or 6.7 TB/s at 1965 MHz, 205 us where the cap lets 1.6 GHz; a quarter of the
// exponentials as polynomials: 8 % more).  Five blocks an SM, four where alternatives are asked for: 1000 x 151936 with 5 of them
// 60.2 us, 62.1 with five; 4000 x 151936 without 205 us, 208 with four.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads, TOP ? 4 : 5) token_logprobs_kernel(ScoreParams p) {
  using Vec = ScoreVec<T>;
  constexpr int U = 4, shift = 2;                    // vectors of a step
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x;
  const int split = (int)cluster_size(), part = (int)tc::cluster_rank();
  const int row = blockIdx.x / split;
  pdl_wait();
  const float scale = row_scale(p.temperature, row), c = scale * kLog2e;
  const RowPart<T> r(p, row, part, split);
  const int64_t id = tid == 0 ? p.ids[row] : -1;
  PairTally run = pair_empty();
  constexpr int step = kScoreThreads * U;
  // what the next two steps read starts for L2: a block alone on its SM, at the end, has enough on its way too (1000 x 151936: 52.8 us,
  // 56.9 without; 4000: 185.5 and 193.1; four and eight steps ahead 56.8 and 76.4 us)
  const auto prefetch = [&](int v) {
    const int n = min(step, r.v1 - v);
    if (n > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(r.xv + v), "r"(16 * n) : "memory");
  };
  if (tid == 0) prefetch(r.v0 + step);
  // steps of a group of vectors: 1, or more where a thread would have too many groups
  int more = 0, groups = 0;
  if constexpr (TOP)
    while ((r.v1 - r.v0 + step - 1) / step > kScoreGroups << more) ++more;
  float most = -INFINITY;
  const auto take = [&](const Vec* v, int i, bool last) {
    const float m = tally_vectors<T, U>(run, v, c);
    if constexpr (TOP) {
      most = fmaxf(most, m);
      if ((i & ((1 << more) - 1)) == 0 || last) {
        sh.group[groups++][tid] = most;
        most = -INFINITY;
      }
    }
  };
  int at = r.v0, i = 1;                              // the same in all threads
  for (; at + step <= r.v1; at += step, ++i) {
    if (tid == 0) prefetch(at + 2 * step);
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].raw = __ldg(r.xv + at + tid + u * kScoreThreads);
    take(v, i, at + step == r.v1);
  }
  if (at < r.v1) {
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = at + tid + u * kScoreThreads;
      if (j < r.v1) v[u].raw = __ldg(r.xv + j);
      else v[u].nothing();
    }
    take(v, i, true);
  }
  const float given = id >= 0 && id < p.V ? to_f32(r.x[id]) : 0.f;
  Tally a = pair_sum(run);
  if (r.single >= 0) tally_add(a, to_f32(r.x[r.single]), c);
  const int n = TOP ? p.n_top : 0;
  int n_listed = 0;
  if constexpr (TOP) share_most(a.m, n, sh);
  warp_tally(a, c, sh.red);
  score_sync();
  if constexpr (TOP) {
    if (list_alternatives<T>(r, groups, shift + more, n, sh)) {
      n_listed = sh.n_listed;
    } else {
      n_listed = search_alternatives<T>(r, n, sh);
      score_sync();
    }
  }
  a = block_tally(c, sh.red);

  if (split > 1) {
    if constexpr (TOP) {
      if (tid < n) sh.top[tid] = 0;
      score_sync();
      place_alternatives(sh, n_listed, n, [&](int place, uint64_t key) { sh.top[place] = key; });
    }
    if (tid == 0) sh.part = a;
    tc::cluster_sync();
    if (part != 0) {
      tc::cluster_sync();                            // the others' places are being read
      return;
    }
    a = tally_empty();
    for (int q = 0; q < split; ++q) {
      const uint32_t at = tc::in_cta(smem_u32(&sh.part), q);
      a = tally_join(a, {remote_f32(at), remote_f32(at + 4), remote_f32(at + 8)}, c);
    }
    if constexpr (TOP) {
      n_listed = split * n;                          // some of them nobody's, behind all others
      for (int i = tid; i < n_listed; i += kScoreThreads) sh.listed[i] = remote_u64(tc::in_cta(smem_u32(sh.top + i % n), i / n));
    }
    tc::cluster_sync();
  }
  if (tid == 0) {
    p.out_lp[row] = id < 0 ? 0.f : id >= p.V ? -INFINITY : tally_logprob(a, given, scale);
    p.out_entropy[row] = tally_entropy(a);
  }
  if constexpr (TOP) {
    int32_t* ids = p.out_ids + (int64_t)row * n;
    float* lps = p.out_lps + (int64_t)row * n;
    // places behind the last alternative: fewer than n scores of the row are above -inf
    if (tid < n) {
      int some = n_listed;
      if (split > 1) {
        some = 0;
        for (int i = 0; i < n_listed; ++i) some += sh.listed[i] != 0;
      }
      if (tid >= some) {
        ids[tid] = -1;
        lps[tid] = -INFINITY;
      }
    }
    place_alternatives(sh, n_listed, n, [&](int place, uint64_t key) {
      ids[place] = key_index(key);
      lps[place] = tally_logprob(a, key_score(key), scale);
    });
  }
}

template <typename T, bool TOP>
static int launch_token_logprobs(const ScoreParams& p, int rows, int split, cudaStream_t s) {
  auto kernel = token_logprobs_kernel<T, TOP>;
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

// Parts of a row.  A cluster's barriers and reads cost some 2 us, and larger clusters start later: a block for each of some 400 places, of
// 4096 scores at least (64 x 151936, 20 alternatives: 25.7 us whole, 13.6 in 4 parts, 17.4 in 8; 150 x 32768: 8.0 us whole, 10.1 in 4).
static int score_split(int rows, int V) {
  int split = 1;
  while (split < kScoreMaxSplit && (int64_t)rows * split * 2 <= 400 && V / (split * 2) >= 4096) split *= 2;
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
