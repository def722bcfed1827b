// Log-probabilities of given tokens with the entropy and the most likely alternatives of their rows (contract: ops/score.py).
#include "logprob_math.cuh"
#include "vec_io.cuh"

namespace xllm {

constexpr int kScoreThreads = 256;

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

template <typename T>
__global__ void __launch_bounds__(kScoreThreads) token_logprobs_kernel(ScoreParams p) {
  __shared__ float red[32];
  __shared__ float redv[32];
  __shared__ int redi[32];
  const int row = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  pdl_wait();
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;
  const float scale = row_scale(p.temperature, row), c = scale * kLog2e;
  Tally a = tally_empty();
  for (int i = threadIdx.x; i < p.V; i += kScoreThreads) a.m = fmaxf(a.m, to_f32(x[i]));
  a.m = block_max(a.m, red);
  for (int i = threadIdx.x; i < p.V; i += kScoreThreads) {
    const float t = bounded((to_f32(x[i]) - a.m) * c), e = exp2_fast(t);
    a.z += e;
    a.s += e * t;
  }
  a.z = block_sum(a.z, red);
  a.s = block_sum(a.s, red);
  if (threadIdx.x == 0) {
    const int64_t id = p.ids[row];
    p.out_lp[row] = id < 0 ? 0.f : id >= p.V ? -INFINITY : tally_logprob(a, to_f32(x[id]), scale);
    p.out_entropy[row] = tally_entropy(a);
  }
  // one pass a place: the largest of what comes behind the last one in the order (score, lowest index first)
  float pv = INFINITY;
  int pi = -1;
  for (int k = 0; k < p.n_top; ++k) {
    float v = -INFINITY;
    int idx = 0x7fffffff;
    for (int i = threadIdx.x; i < p.V; i += kScoreThreads) {
      const float u = to_f32(x[i]);
      if ((u < pv || (u == pv && i > pi)) && u > v) { v = u; idx = i; }
    }
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, v, o);
      const int oi = __shfl_xor_sync(0xffffffffu, idx, o);
      if (ov > v || (ov == v && oi < idx)) { v = ov; idx = oi; }
    }
    if (lane == 0) { redv[wid] = v; redi[wid] = idx; }
    __syncthreads();
    v = redv[0];
    idx = redi[0];
    for (int w = 1; w < kScoreThreads / 32; ++w)
      if (redv[w] > v || (redv[w] == v && redi[w] < idx)) { v = redv[w]; idx = redi[w]; }
    __syncthreads();
    const bool none = idx == 0x7fffffff;
    if (threadIdx.x == 0) {
      p.out_ids[(int64_t)row * p.n_top + k] = none ? -1 : idx;
      p.out_lps[(int64_t)row * p.n_top + k] = none ? -INFINITY : tally_logprob(a, v, scale);
    }
    pv = v;
    pi = idx;
  }
}

}  // namespace xllm

// dtype: 0 = bf16 logits, 1 = fp32 logits; ids int64 [rows], temperature fp32 [rows] or null; out_ids, out_lps [rows, n_top].
XLLM_API int xllm_token_logprobs(const void* logits, int64_t row_stride, int dtype, int rows, int vocab, const void* ids,
                                 const void* temperature, int n_top, void* out_lp, void* out_entropy, void* out_ids,
                                 void* out_lps, void* stream) {
  using namespace xllm;
  if (rows == 0) return 0;
  if (rows < 0 || vocab < 1 || n_top < 0 || n_top > vocab || (dtype != 0 && dtype != 1)) return (int)cudaErrorInvalidValue;
  const ScoreParams p{logits, row_stride, vocab, n_top, (const int64_t*)ids, (const float*)temperature, (float*)out_lp,
                      (float*)out_entropy, (int32_t*)out_ids, (float*)out_lps};
  if (dtype == 0) launch_pdl(token_logprobs_kernel<bf16>, dim3(rows), dim3(kScoreThreads), 0, (cudaStream_t)stream, p);
  else launch_pdl(token_logprobs_kernel<float>, dim3(rows), dim3(kScoreThreads), 0, (cudaStream_t)stream, p);
  return XLLM_LAUNCH_CHECK();
}
