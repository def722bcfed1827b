// Log-probabilities and entropies straight from hidden states and the output projection (contract: ops/score.py): the scores
// x = h W^T of a tile are tallied where they are computed and never stored.
//
//   head_tally_kernel  one tile of rows x vocabulary: the rows' tallies (logprob_math.cuh) of the tile's columns, and the
//                      given token's score from whichever tile holds it
//   head_join_kernel   a row's tallies over all tiles, joined in a fixed order
#include "logprob_math.cuh"
#include "vec_io.cuh"

namespace xllm {

constexpr int kHeadTile = 64, kHeadK = 32;

// workspace: tallies [column tiles][rows] and the given tokens' scores [rows]
struct HeadParams {
  const bf16* h;
  int64_t ldh;
  const bf16* w;
  int64_t ldw;
  int T, V, K, n_tiles;
  const int64_t* ids;
  const float* temperature;
  Tally* tallies;
  float* given;
};

__global__ void __launch_bounds__(256) head_tally_kernel(HeadParams p) {
  __shared__ float sa[kHeadK][kHeadTile + 1], sb[kHeadK][kHeadTile + 1];
  __shared__ float sx[kHeadTile][kHeadTile + 1];
  pdl_wait();
  const int m0 = blockIdx.y * kHeadTile, n0 = blockIdx.x * kHeadTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kHeadK) {
    for (int i = threadIdx.x; i < kHeadTile * kHeadK; i += 256) {
      const int r = i / kHeadK, k = i % kHeadK;
      sa[k][r] = m0 + r < p.T && k0 + k < p.K ? to_f32(p.h[(m0 + r) * p.ldh + k0 + k]) : 0.f;
      sb[k][r] = n0 + r < p.V && k0 + k < p.K ? to_f32(p.w[(n0 + r) * p.ldw + k0 + k]) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kHeadK; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) sx[ty * 4 + i][tx * 4 + j] = acc[i][j];
  __syncthreads();
  const int row = m0 + threadIdx.x;
  if (threadIdx.x >= kHeadTile || row >= p.T) return;
  const float c = row_scale(p.temperature, row) * kLog2e;
  const int n = min(kHeadTile, p.V - n0);
  Tally a = tally_empty();
  for (int j = 0; j < n; ++j) a.m = fmaxf(a.m, sx[threadIdx.x][j]);
  for (int j = 0; j < n; ++j) {
    const float t = bounded((sx[threadIdx.x][j] - a.m) * c), e = exp2_fast(t);
    a.z += e;
    a.s += e * t;
  }
  p.tallies[(int64_t)blockIdx.x * p.T + row] = a;
  const int64_t id = p.ids[row];
  if (id >= n0 && id < n0 + n) p.given[row] = sx[threadIdx.x][id - n0];
}

__global__ void __launch_bounds__(128) head_join_kernel(HeadParams p, float* out_lp, float* out_entropy) {
  pdl_wait();
  const int row = blockIdx.x * 128 + threadIdx.x;
  if (row >= p.T) return;
  const float scale = row_scale(p.temperature, row), c = scale * kLog2e;
  Tally a = tally_empty();
  for (int i = 0; i < p.n_tiles; ++i) a = tally_join(a, p.tallies[(int64_t)i * p.T + row], c);
  const int64_t id = p.ids[row];
  out_lp[row] = id < 0 ? 0.f : id >= p.V ? -INFINITY : tally_logprob(a, p.given[row], scale);
  out_entropy[row] = tally_entropy(a);
}

}  // namespace xllm

// Bytes of workspace of xllm_head_logprobs.
XLLM_API int64_t xllm_head_logprobs_workspace(int rows, int vocab) {
  using namespace xllm;
  const int64_t tiles = (vocab + kHeadTile - 1) / kHeadTile;
  return ((tiles * sizeof(Tally) + sizeof(float)) * rows + 15) / 16 * 16;
}

XLLM_API int xllm_head_logprobs_error_status() { return 0; }

XLLM_API int xllm_head_logprobs(const void* hidden, int64_t ldh, const void* weight, int64_t ldw, int rows, int vocab, int width,
                                const void* ids, const void* temperature, void* workspace, void* out_lp, void* out_entropy,
                                void* stream) {
  using namespace xllm;
  if (rows == 0) return 0;
  if (rows < 0 || vocab < 1 || width < 1) return (int)cudaErrorInvalidValue;
  const int n_tiles = (vocab + kHeadTile - 1) / kHeadTile;
  Tally* tallies = (Tally*)workspace;
  const HeadParams p{(const bf16*)hidden, ldh, (const bf16*)weight, ldw, rows, vocab, width, n_tiles, (const int64_t*)ids,
                     (const float*)temperature, tallies, (float*)(tallies + (int64_t)n_tiles * rows)};
  cudaStream_t s = (cudaStream_t)stream;
  launch_pdl(head_tally_kernel, dim3(n_tiles, (rows + kHeadTile - 1) / kHeadTile), dim3(256), 0, s, p);
  launch_pdl(head_join_kernel, dim3((rows + 127) / 128), dim3(128), 0, s, p, (float*)out_lp, (float*)out_entropy);
  return XLLM_LAUNCH_CHECK();
}
