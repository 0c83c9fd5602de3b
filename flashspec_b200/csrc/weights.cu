// Second half of the weighted decode: the attention weight of every cached token.
//
// The decode kernels leave the scores x = log2(e) * sm_scale * q.k and the rows' LSEs; here
//   weights[page, kv head, t] += sum_g 2^(x_g - LSE_g log2 e)   (g: the kv head's queries),
// the softmax weight each token received, summed over the queries that share the kv head.
// A weight needs the LSE of the whole row, known only when the decode has ended, so the
// scores make one round trip (4 bytes a query and token, against the 256 of a token's K
// and V) instead of K being read and multiplied again (128 bytes).
//
// Bound by memory: 4 G bytes of scores and 8 of weights a token (14 us for 64 ragged requests
// of 32 / 8 heads, 16 us for 2 x 131072 tokens of 64 / 8 heads, under a profiler with cold
// caches; the decodes before them take 141 and 121).  A lane takes four tokens
// of one request and walks the kv head's queries, so a warp reads 512 consecutive bytes a
// query.  Sums go out as reductions: pages shared by requests add up correctly (their order
// then varies), and a page of one request gets exactly one addition a call, so its sums are
// the same in every run.
#include <cuda_runtime.h>

#include <math.h>
#include <stdint.h>

#include "common.h"
#include "ptx.cuh"
#include "weights.h"

namespace fsb {

constexpr int kWThreads = 256;
constexpr int kWTokens = 4 * kWThreads;  // tokens of a CTA
constexpr int kWMaxG = 8;

struct AddWeightsParams {
  const float* scores;
  const float* lse;
  const int64_t* table;
  const int64_t* lengths;
  float* weights;
  int64_t stride, num_pages, max_seq_len;
  int64_t rows;  // B * Hq
  int Hq, Hkv, G, cols, page, parts;
};

// kVec: pages of a multiple of four tokens and a 16-byte aligned weights array, so four
// tokens are one vector reduction.
template <bool kVec>
__global__ void __launch_bounds__(kWThreads) add_weights_kernel(const AddWeightsParams p) {
  __shared__ float lse2[kWMaxG];
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const int64_t cap = (int64_t)p.cols * p.page;
  const int64_t len = min(min(p.lengths[b], p.max_seq_len), cap);
  const int64_t tok0 = (int64_t)blockIdx.y * kWTokens;
  if (tok0 >= len) return;
  const size_t row0 = (size_t)b * p.Hq + (size_t)h * p.G;
  if (threadIdx.x < p.G) {
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < p.parts; ++s) M = fmaxf(M, p.lse[(size_t)s * p.rows + row0 + threadIdx.x]);
    if (p.parts > 1 && M != -INFINITY) {
      for (int s = 0; s < p.parts; ++s) L += expf(p.lse[(size_t)s * p.rows + row0 + threadIdx.x] - M);
      M += logf(L);
    }
    lse2[threadIdx.x] = M * 1.4426950408889634f;
  }
  __syncthreads();
  const int64_t tok = tok0 + 4 * threadIdx.x;
  if (tok >= len) return;
  // rows are padded to whole 16-token groups, so the last load stays inside its row
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* sp = p.scores + row0 * p.stride + tok;
#pragma unroll 8
  for (int g = 0; g < p.G; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(sp + g * p.stride);
    const float l = lse2[g];
    w.x += ex2_approx(x.x - l);
    w.y += ex2_approx(x.y - l);
    w.z += ex2_approx(x.z - l);
    w.w += ex2_approx(x.w - l);
  }
  const int64_t lp = tok / p.page;
  if (kVec) {
    const int64_t phys = p.table[(size_t)b * p.cols + lp];
    if (phys < 0 || phys >= p.num_pages) return;
    // tokens behind the length add nothing (their scores may never have been written)
    if (tok + 1 >= len) w.y = 0.f;
    if (tok + 2 >= len) w.z = 0.f;
    if (tok + 3 >= len) w.w = 0.f;
    float* dst = p.weights + (phys * p.Hkv + h) * p.page + (tok - lp * p.page);
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "f"(w.x), "f"(w.y), "f"(w.z), "f"(w.w)
                 : "memory");
    return;
  }
  const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (tok + k >= len) break;
    const int64_t pg = (tok + k) / p.page;
    const int64_t phys = p.table[(size_t)b * p.cols + pg];
    if (phys < 0 || phys >= p.num_pages) continue;
    atomicAdd(p.weights + (phys * p.Hkv + h) * p.page + (tok + k - pg * p.page), v[k]);
  }
}

int launch_add_weights(const FsDecodeArgs* a, const ScoreTarget& t, const float* lse, int parts, float* weights,
                       void* stream) {
  AddWeightsParams p{};
  p.scores = t.scores;
  p.lse = lse;
  p.table = a->block_table;
  p.lengths = a->lengths;
  p.weights = weights;
  p.stride = t.stride;
  p.num_pages = a->num_blocks;
  p.max_seq_len = a->max_seq_len;
  p.rows = (int64_t)a->batch * a->q_heads;
  p.Hq = a->q_heads;
  p.Hkv = a->kv_heads;
  p.G = a->q_heads / a->kv_heads;
  p.cols = a->table_cols;
  p.page = a->page_size > 0 ? a->page_size : a->block_size;
  p.parts = parts;
  const int64_t chunks = (t.stride + kWTokens - 1) / kWTokens, pairs = (int64_t)a->batch * a->kv_heads;
  if (chunks == 0) return FS_OK;  // no token can be live
  if (chunks > 65535) return FS_ERR_UNSUPPORTED;  // 67M tokens; refused before the decode by its plan
  const dim3 grid((unsigned)pairs, (unsigned)chunks);
  const bool vec = p.page % 4 == 0 && (reinterpret_cast<uintptr_t>(weights) & 15) == 0;
  auto kernel = vec ? add_weights_kernel<true> : add_weights_kernel<false>;
  kernel<<<grid, kWThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("attention weights kernel launch");
}

}  // namespace fsb
