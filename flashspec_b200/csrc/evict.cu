// Eviction from the paged cache by accumulated attention weight: two kernels.
//
// select_tokens_kernel, per (request, kv head) with n > budget live tokens: the first
// `sinks` and the last `recent` tokens stay, and of the n - sinks - recent between them the
// K = budget - sinks - recent with the largest weights (ties: the lower position).  A
// cluster of CTAs takes one row.  It reads the row's weights once, as order-preserving
// 32-bit keys, into shared memory; three counting passes (11 + 11 + 10 bits) over those
// find the K-th largest key, the CTAs' histograms being summed over distributed shared
// memory; then an ordered pass numbers the kept tokens, writes their positions to `kept`
// and their weights to their new places (zeros behind them).
//
// move_tokens_kernel moves the kept tokens' K and V, in place, into the first pages of the
// request.  In place is what a cache under pressure needs, and the order makes it safe: a
// kept token never moves up (kept[i] >= i), so page j's sources lie in pages >= j.  A
// cluster takes one (request, kv head, K|V) and walks its pages in rounds: every warp loads
// its pages' source tokens into registers, the cluster synchronises, then the warps write.
// A round writes pages below all that later rounds read.  Affine pages are dequantized and
// requantized by the format's rule (quant_math.cuh, as fs_page_update does), symmetric ones
// keep their codes and scales.  A page whose kept tokens stand in it already is left as it
// is.
//
// Memory traffic is the floor: 4 bytes of weights for every live token, then 2 (D + a scale)
// bytes read and written for every kept one.  Measured: 64 requests of up to 8192 tokens and 8
// heads cut to 1000 (floor 38 us): selection 38 us, affine move 148 us, 83 M warp
// instructions; 2 x 131072 tokens cut to 16384 (floor 23 us): selection 51 us,
// symmetric move 54 us, in clusters of 8 CTAs for each of the 16 rows, one or two CTAs an SM.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <math.h>
#include <stdint.h>
#include <algorithm>

#include "../../include/flashspec_b200.h"
#include "common.h"
#include "quant_math.cuh"

namespace fsb {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 512;
constexpr int kBins = 2048;
constexpr int kSelMaxCluster = 8;
// keys of one CTA held in shared memory at most (192 KB); longer rows keep them in the workspace
constexpr int kSelSmemKeys = 48 * 1024;
constexpr int kEvictFill = 296;  // CTAs that keep the GPU busy: two on each of 148 SMs

// Division by a page's tokens or a head's dims: a shift where it is a power of two.
struct Divisor {
  int d, shift;  // shift < 0: not a power of two
  __device__ __forceinline__ int quot(int x) const { return shift >= 0 ? x >> shift : x / d; }
};

struct EvictParams {
  const int64_t* table;
  const int64_t* lengths;
  const float* weights;
  float* weights_out;
  int32_t* kept;
  int64_t* new_lengths;
  uint32_t* keys;  // workspace [rows, cluster * chunk_cap], or null
  uint32_t* status;
  int8_t* values[2];
  float* scale[2];
  int16_t* zero[2];
  int64_t num_pages, max_seq_len;
  Divisor by_page, by_dim;
  int Hkv, cols, page, D, budget, recent, sinks;
  int chunk_cap;  // keys of one CTA at most
  int vec;        // pages of whole groups of four tokens, weights 16-byte aligned
  int sym;
};

__device__ __forceinline__ int64_t live_tokens(const EvictParams& p, int b) {
  return max((int64_t)0, min(min(p.lengths[b], p.max_seq_len), (int64_t)p.cols * p.page));
}

// Page of the pool behind logical page lp of request b (fs_evict_tokens keeps pools below 2^31
// pages); -1 when unallocated (any negative entry) or outside the pool.
__device__ __forceinline__ int page_at(const EvictParams& p, int b, int lp) {
  const int64_t phys = p.table[(size_t)b * p.cols + lp];
  if (phys >= p.num_pages) {
    if (p.status != nullptr) atomicOr(p.status, FS_DEV_BAD_PAGE);
    return -1;
  }
  return phys < 0 ? -1 : (int)phys;
}

// Larger weight <-> larger key; -0 counts as +0, NaN (of either sign) is above all, and 0 is
// left for tokens without a page.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? max(~u, 1u) : (u | 0x80000000u);
}
__device__ __forceinline__ float weight_of(uint32_t key) {
  if (key == 0u) return 0.f;
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// Inclusive scan of v over the block; *total receives the block's sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // warp_sums is free
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const uint32_t x = warp_sums[w];
    if (w < warp) before += x;
    all += x;
  }
  *total = all;
  return v + before;
}

// kSmem: the keys live in shared memory, else in the workspace (each CTA in its own part).
template <bool kSmem>
__global__ void __launch_bounds__(kSelThreads) select_tokens_kernel(const EvictParams p) {
  extern __shared__ __align__(16) uint32_t sel_smem[];
  __shared__ __align__(16) uint32_t hist[kBins];
  __shared__ uint32_t warp_sums[kSelThreads / 32];
  __shared__ uint32_t found[2];   // bin of the K-th key, keys above that bin
  __shared__ uint32_t counts[2];  // this CTA's keys above and equal to the threshold
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / C, b = row / p.Hkv, h = row % p.Hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cap = p.cols * p.page;
  const int n = (int)live_tokens(p, b);
  const int count = min(n, p.budget);
  if (h == 0 && rank == 0 && tid == 0) p.new_lengths[b] = count;
  int32_t* kept = p.kept + (size_t)row * p.budget;
  const bool cut = n > p.budget;
  const int lo = p.sinks, hi = n - p.recent;  // the contested range of a row that is cut
  const int K = cut ? p.budget - p.sinks - p.recent : 0;

  // ---- the row's weights, as keys of positions [c0, c1); the chunk is padded to groups of four
  const int chunk = (n + 4 * C - 1) / (4 * C) * 4;  // <= chunk_cap
  const int c0 = min(rank * chunk, n), c1 = min(c0 + chunk, n);
  uint32_t* keys = kSmem ? sel_smem : p.keys + (size_t)blockIdx.x * p.chunk_cap;
  if (p.vec) {
    // four positions of one page a thread, four independent groups in flight
#pragma unroll 4
    for (int i = c0 + 4 * tid; i < c1; i += 4 * kSelThreads) {
      const int lp = p.by_page.quot(i);
      const int64_t phys = page_at(p, b, lp);
      uint4 k = make_uint4(0u, 0u, 0u, 0u);
      if (phys >= 0) {
        const float4 w = *reinterpret_cast<const float4*>(p.weights + (phys * p.Hkv + h) * p.page + (i - lp * p.page));
        k = make_uint4(key_of(w.x), key_of(w.y), key_of(w.z), key_of(w.w));
      }
      *reinterpret_cast<uint4*>(keys + (i - c0)) = k;
    }
  } else {
#pragma unroll 4
    for (int i = c0 + tid; i < c1; i += kSelThreads) {
      const int lp = p.by_page.quot(i);
      const int64_t phys = page_at(p, b, lp);
      keys[i - c0] = phys < 0 ? 0u : key_of(p.weights[(phys * p.Hkv + h) * p.page + (i - lp * p.page)]);
    }
  }

  if (cut && K > 0) {
    // ---- the K-th largest key T of the contested range, and how many equal to T stay
    uint32_t prefix = 0, need = (uint32_t)K;
    const int a0 = max(c0, lo), a1 = min(c1, hi);
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      *reinterpret_cast<uint4*>(hist + 4 * tid) = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
#pragma unroll 2
      for (int i = c0 + 4 * tid; i < c1; i += 4 * kSelThreads) {
        const uint4 k4 = *reinterpret_cast<const uint4*>(keys + (i - c0));
        const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j >= a0 && i + j < a1 && (pass == 0 || (k[j] >> (shift + bits)) == prefix))
            atomicAdd(hist + ((k[j] >> shift) & ((1u << bits) - 1)), 1u);
      }
      cluster.sync();  // every CTA's histogram is complete
      // thread t sums bins [top, top + 4) over the cluster, the highest bins first
      const int top = kBins - 4 * (tid + 1);
      uint32_t v[4] = {0, 0, 0, 0};
      for (int r = 0; r < C; ++r) {
        const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, r) + top);
        v[3] += x.x, v[2] += x.y, v[1] += x.z, v[0] += x.w;
      }
      const uint32_t mine = v[0] + v[1] + v[2] + v[3];
      uint32_t total;
      uint32_t before = block_scan(mine, warp_sums, &total) - mine;
      if (before < need && before + mine >= need) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (before < need && before + v[j] >= need) {
            found[0] = (uint32_t)(top + 3 - j);
            found[1] = before;
          }
          before += v[j];
        }
      }
      cluster.sync();  // found is written; no CTA reads a histogram that is cleared next
      prefix = (prefix << bits) | found[0];
      need -= found[1];
    }
    const uint32_t T = prefix, quota = need;  // kept: key > T, and the first `quota` keys == T

    // ---- each warp counts a contiguous part of the chunk, then numbers what it keeps
    const int part = (chunk + 128 * (kSelThreads / 32) - 1) / (128 * (kSelThreads / 32)) * 128;
    const int w0 = min(c0 + warp * part, c1), w1 = min(w0 + part, c1);
    uint32_t above = 0, equal = 0;
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
      const uint4 k4 = *reinterpret_cast<const uint4*>(keys + (i - c0));
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = i + j >= a0 && i + j < a1;
        above += in && k[j] > T;
        equal += in && k[j] == T;
      }
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    uint32_t n_above, n_equal;
    const uint32_t at_above = block_scan(lane == 31 ? above : 0u, warp_sums, &n_above);
    const uint32_t at_equal = block_scan(lane == 31 ? equal : 0u, warp_sums, &n_equal);
    // before this warp: the scan at the previous warp's last lane
    uint32_t base_above = __shfl_sync(0xffffffffu, at_above, 31) - above;
    uint32_t base_equal = __shfl_sync(0xffffffffu, at_equal, 31) - equal;
    if (tid == 0) counts[0] = n_above, counts[1] = n_equal;
    cluster.sync();  // counts are written
    for (int r = 0; r < rank; ++r) {
      const uint32_t* c = cluster.map_shared_rank(counts, r);
      base_above += c[0];
      base_equal += c[1];
    }
    for (int i0 = w0; i0 < w1; i0 += 128) {
      const int i = i0 + 4 * lane;
      uint32_t k[4] = {0u, 0u, 0u, 0u}, packed = 0;  // above in the low half, equal in the high half
      if (i < w1) {
        const uint4 k4 = *reinterpret_cast<const uint4*>(keys + (i - c0));
        k[0] = k4.x, k[1] = k4.y, k[2] = k4.z, k[3] = k4.w;
      }
      bool gt[4], eq[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = i + j >= a0 && i + j < a1;
        gt[j] = in && k[j] > T;
        eq[j] = in && k[j] == T;
        packed += (gt[j] ? 1u : 0u) + (eq[j] ? 0x10000u : 0u);
      }
      if (!__any_sync(0xffffffffu, packed != 0u)) continue;
      uint32_t incl = packed;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const uint32_t sum = __shfl_sync(0xffffffffu, incl, 31), at = incl - packed;
      uint32_t a = base_above + (at & 0xffffu), e = base_equal + (at >> 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (gt[j] || (eq[j] && e < quota)) kept[lo + (int)(a + min(e, quota))] = i + j;
        a += gt[j];
        e += eq[j];
      }
      base_above += sum & 0xffffu;
      base_equal += sum >> 16;
    }
  }
  // ---- the tokens that are kept anyway, and nothing behind them
  for (int i = rank * kSelThreads + tid; i < p.budget; i += C * kSelThreads) {
    if (!cut)
      kept[i] = i < n ? i : -1;
    else if (i < p.sinks)
      kept[i] = i;
    else if (i >= p.budget - p.recent)
      kept[i] = n - (p.budget - i);
  }
  cluster.sync();  // `kept` is complete; every weight of the row has been read

  // ---- the kept tokens' weights at their new places, zeros at the others
  auto weight_at = [&](int dst) -> float {
    if (dst >= count) return 0.f;
    const int src = kept[dst], r = src / chunk;
    const uint32_t* k = kSmem ? cluster.map_shared_rank(sel_smem, r) : p.keys + (size_t)(blockIdx.x - rank + r) * p.chunk_cap;
    return weight_of(k[src - r * chunk]);
  };
  if (p.vec) {
    for (int i = 4 * (rank * kSelThreads + tid); i < cap; i += 4 * C * kSelThreads) {
      const int lp = p.by_page.quot(i);
      const int64_t phys = page_at(p, b, lp);
      const float4 w = make_float4(weight_at(i), weight_at(i + 1), weight_at(i + 2), weight_at(i + 3));
      if (phys >= 0)
        *reinterpret_cast<float4*>(p.weights_out + (phys * p.Hkv + h) * p.page + (i - lp * p.page)) = w;
    }
  } else {
    for (int i = rank * kSelThreads + tid; i < cap; i += C * kSelThreads) {
      const int lp = p.by_page.quot(i);
      const int64_t phys = page_at(p, b, lp);
      const float w = weight_at(i);
      if (phys >= 0) p.weights_out[(phys * p.Hkv + h) * p.page + (i - lp * p.page)] = w;
    }
  }
  cluster.sync();  // no CTA leaves while its keys and counts may still be read
}


// Affine pages of up to four chunks a lane: registers for 28 resident warps an SM.
template <int kCh, int kWarps, bool kSym>
constexpr int move_min_blocks() {
  return kCh <= 4 && !kSym ? 28 / kWarps : 1;
}

// One page of K or V on its way through a warp: kCh 16-byte chunks a lane, chunk c of lane l
// being bytes [16 (32 c + l), ...) of the page's [page, D] block.  The sources (page of the
// pool and row in it, -1: zeros) are looked up a round ahead, behind the data loads of the
// round before.
template <int kCh, bool kSym>
struct PageMove {
  int sp[kCh], sr[kCh];              // source of each chunk
  int tp[kSym ? 2 : 1], tr[kSym ? 2 : 1];  // symmetric: source of tokens `lane` and `lane + 32`
  int dst;                           // page of the pool, -1: nothing to write

  __device__ __forceinline__ void plan(const EvictParams& p, int b, const int32_t* kept, int pg, int npg, int lane) {
    dst = -1;
    if (pg >= npg) return;
    const int rows = min(p.page, p.budget - pg * p.page);  // kept tokens of the page
    bool stays = true;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = lane + 32 * u;
      int src = -1;
      if (t < rows) {
        src = kept[pg * p.page + t];
        stays = stays && src == pg * p.page + t;
      }
      if (kSym) tp[u] = src;
    }
    if (__all_sync(0xffffffffu, stays)) return;
    dst = page_at(p, b, pg);
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int e = 16 * (32 * c + lane), t = p.by_dim.quot(e);
      sp[c] = -1;
      if (e < p.page * p.D && t < rows) {
        const int src = kept[pg * p.page + t], lp = p.by_page.quot(src);
        sp[c] = page_at(p, b, lp);
        sr[c] = src - lp * p.page;
      }
    }
    if (kSym) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (tp[u] < 0) continue;
        const int lp = p.by_page.quot(tp[u]);
        tr[u] = tp[u] - lp * p.page;
        tp[u] = page_at(p, b, lp);
      }
    }
  }
};

// Byte j of an XOR-ed word (a code u) as the float 2^23 + u.
__device__ __forceinline__ float code_float(uint32_t w, int j) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 | j));
}

// 16 codes through (u - zp) * scale and the destination's rounding, bit for bit as dequant16
// followed by quantize16_fast, with one multiplication for the two.  With d = u - zp exact the
// code is rint(clamp(t)), t = RN(RN(RN(d s) / S) + Z); here ta = RN(d RN(s RN(1/S)) + Z).
// Where ta lies in [0, 255], |d s / S| <= 255 (1 + 2^-15), each side is off from d s / S + Z by
// two roundings of it (255 * 2^-23) and half an ulp of 255 (2^-17): together less than 7.7e-5.
// So a ta farther than 2^-13 (1.2e-4) from a half-integer has the same rint, and one outside
// [0, 255] clamps the same way.  The others, 0.025% of them, take the exact path.
constexpr float kNearHalf = 0.5f - 1.220703125e-4f;

// Out of line: the codes of a chunk that has one near a half-integer, those by the format's
// own steps.
static __device__ __noinline__ uint4 requantize16_careful(uint4 raw, float scale, float base, float ratio, float to_scale,
                                                          float to_zero) {
  const QParams q{to_scale, to_zero};
  uint32_t w4[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t out = 0u;
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
      const float d = __fsub_rn(__uint_as_float(0x4B000000u | ((w4[k] >> (8 * j)) & 0xffu)), base);
      const float tc = fminf(fmaxf(__fmaf_rn(d, ratio, q.zp), 0.0f), 255.0f);
      uint32_t code = (uint32_t)rintf(tc);
      if (fabsf(__fsub_rn(tc, rintf(tc))) >= kNearHalf)
        code = (uint32_t)((int)quantize_one(__fmul_rn(d, scale), q) + 128);
      out |= code << (8 * j);
    }
    w4[k] = out ^ 0x80808080u;
  }
  return make_uint4(w4[0], w4[1], w4[2], w4[3]);
}

__device__ __forceinline__ uint4 requantize16(uint4 raw, float scale, int16_t zp, float ratio, QParams q) {
  const float base = __fadd_rn(8388608.0f, (float)zp);
  const uint32_t w4[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
  uint32_t w[4];
  float worst = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t bits[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float ta = __fmaf_rn(__fsub_rn(code_float(w4[k], j), base), ratio, q.zp);
      const float tc = fminf(fmaxf(ta, 0.0f), 255.0f);
      const float r = __fadd_rn(tc, kMagic);
      worst = fmaxf(worst, fabsf(__fsub_rn(tc, __fsub_rn(r, kMagic))));
      bits[j] = __float_as_uint(r);  // low byte = rint(tc)
    }
    const uint32_t lo = __byte_perm(bits[0], bits[1], 0x0040), hi = __byte_perm(bits[2], bits[3], 0x0040);
    w[k] = __byte_perm(lo, hi, 0x5410) ^ 0x80808080u;
  }
  if (worst >= kNearHalf) return requantize16_careful(raw, scale, base, ratio, q.scale, q.zp);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Smallest and largest of 16 codes u, as floats 2^23 + u.  (u - zp) times a positive scale is
// monotone, rounding included, so they give the chunk's extremes.
__device__ __forceinline__ void minmax16(uint4 raw, float& lo, float& hi) {
  const uint32_t w4[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
  lo = hi = code_float(w4[0], 0);
#pragma unroll
  for (int j = 1; j < 16; ++j) {
    const float f = code_float(w4[j >> 2], j & 3);
    lo = fminf(lo, f);
    hi = fmaxf(hi, f);
  }
}

template <int kCh, int kPages, int kWarps, bool kSym>
__global__ void __launch_bounds__(kWarps * 32, move_min_blocks<kCh, kWarps, kSym>()) move_tokens_kernel(const EvictParams p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int item = blockIdx.x / C, kv = item & 1, row = item >> 1, b = row / p.Hkv, h = row % p.Hkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n = live_tokens(p, b);
  if (n <= p.budget) return;  // the whole cluster: nothing moves
  const int page = p.page, D = p.D, E = page * D, npg = (p.budget + page - 1) / page;
  const int32_t* kept = p.kept + (size_t)row * p.budget;
  int8_t* values = p.values[kv];
  float* scale = p.scale[kv];
  int16_t* zero = p.zero[kv];
  const int per_round = C * kWarps * kPages;
  const int pg0 = (rank * kWarps + warp) * kPages;
  PageMove<kCh, kSym> mv[kPages];
#pragma unroll
  for (int q = 0; q < kPages; ++q) mv[q].plan(p, b, kept, pg0 + q, npg, lane);
  for (int r0 = 0; r0 < npg; r0 += per_round) {
    uint4 raw[kPages][kCh];
    float sc[kPages][kSym ? 2 : kCh];  // affine: of each chunk's source block; symmetric: of two tokens
    int16_t zp[kPages][kSym ? 1 : kCh];
    int64_t dst[kPages];
#pragma unroll
    for (int q = 0; q < kPages; ++q) {
      const PageMove<kCh, kSym>& m = mv[q];
      dst[q] = m.dst < 0 ? -1 : (int64_t)m.dst * p.Hkv + h;
      if (m.dst < 0) continue;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        const int e = 16 * (32 * c + lane);
        raw[q][c] = make_uint4(0u, 0u, 0u, 0u);
        if (!kSym) sc[q][c] = 0.f, zp[q][c] = 128;  // an absent token dequantizes to 0
        if (m.sp[c] >= 0) {
          const int64_t blk = (int64_t)m.sp[c] * p.Hkv + h;
          raw[q][c] = *reinterpret_cast<const uint4*>(values + blk * E + m.sr[c] * D + (e - p.by_dim.quot(e) * D));
          if (!kSym) sc[q][c] = scale[blk], zp[q][c] = zero[blk];
        }
      }
      if (kSym) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          sc[q][u] = m.tp[u] >= 0 ? scale[((int64_t)m.tp[u] * p.Hkv + h) * page + m.tr[u]] : 1.0e-8f;
      }
    }
    cluster.barrier_arrive();  // this warp's sources of the round are read
#pragma unroll
    for (int q = 0; q < kPages; ++q) mv[q].plan(p, b, kept, r0 + per_round + pg0 + q, npg, lane);
    QParams qp[kPages];
    if (!kSym) {  // the new codes, in place of the old ones, while the others arrive
#pragma unroll
      for (int q = 0; q < kPages; ++q) {
        if (dst[q] < 0) continue;
        float mn = INFINITY, mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          if (16 * (32 * c + lane) >= E) continue;
          float lo, hi;
          minmax16(raw[q][c], lo, hi);
          const float base = __fadd_rn(8388608.0f, (float)zp[q][c]);
          mn = fminf(mn, __fmul_rn(__fsub_rn(lo, base), sc[q][c]));
          mx = fmaxf(mx, __fmul_rn(__fsub_rn(hi, base), sc[q][c]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        qp[q] = qparams_from_range(mn, mx);
        const float rcp = __frcp_rn(qp[q].scale);
#pragma unroll
        for (int c = 0; c < kCh; ++c)
          raw[q][c] = requantize16(raw[q][c], sc[q][c], zp[q][c], __fmul_rn(sc[q][c], rcp), qp[q]);
      }
    }
    cluster.barrier_wait();  // all sources of the round are read
#pragma unroll
    for (int q = 0; q < kPages; ++q) {
      if (dst[q] < 0) continue;
      int8_t* out = values + dst[q] * E;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        const int e = 16 * (32 * c + lane);
        if (e < E) *reinterpret_cast<uint4*>(out + e) = raw[q][c];
      }
      if (kSym) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (lane + 32 * u < page) scale[dst[q] * page + lane + 32 * u] = sc[q][u];
      } else if (lane == 0) {
        scale[dst[q]] = qp[q].scale;
        zero[dst[q]] = (int16_t)qp[q].zp;
      }
    }
  }
}

// Cluster of a row of `tokens` positions, and the keys of one of its CTAs.  Rows that alone
// fill the GPU take one CTA each; few long rows are spread, down to 2048 keys a CTA.
static int select_cluster(int64_t tokens, int64_t rows, int* chunk_cap) {
  int C = 1;
  while (C < kSelMaxCluster && rows * C < kEvictFill && tokens > (int64_t)C * 2048) C *= 2;
  *chunk_cap = (int)((tokens + 4 * C - 1) / (4 * C) * 4);
  while (C < kSelMaxCluster && *chunk_cap > kSelSmemKeys) {  // keep the keys in shared memory
    C *= 2;
    *chunk_cap = (int)((tokens + 4 * C - 1) / (4 * C) * 4);
  }
  return C;
}

static Divisor divisor(int d) {
  Divisor x{d, -1};
  if ((d & (d - 1)) == 0)
    for (x.shift = 0; (1 << x.shift) < d;) ++x.shift;
  return x;
}

static int evict_check(const FsEvictArgs* a) {
  if (a == nullptr || a->block_table == nullptr || a->lengths == nullptr || a->weights == nullptr ||
      a->weights_out == nullptr || a->kept == nullptr || a->new_lengths == nullptr || a->k_values == nullptr ||
      a->v_values == nullptr || a->k_scale == nullptr || a->v_scale == nullptr)
    return FS_ERR_INVALID_ARGUMENT;
  if (a->kv_format != FS_KV_AFFINE_BLOCK && a->kv_format != FS_KV_SYMMETRIC) return FS_ERR_INVALID_ARGUMENT;
  if (a->kv_format == FS_KV_AFFINE_BLOCK && (a->k_zero == nullptr || a->v_zero == nullptr))
    return FS_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->kv_heads <= 0 || a->num_pages <= 0 || a->table_cols <= 0 || a->max_seq_len < 0 ||
      a->budget <= 0 || a->recent < 0 || a->sinks < 0 || (int64_t)a->recent + a->sinks > a->budget)
    return FS_ERR_INVALID_ARGUMENT;
  // the kernels read `lengths` while new_lengths is being written
  if (static_cast<const int64_t*>(a->new_lengths) == a->lengths) return FS_ERR_INVALID_ARGUMENT;
  // K and V move at the same time
  if (a->k_values == a->v_values || a->k_scale == a->v_scale) return FS_ERR_INVALID_ARGUMENT;
  if (a->page_size <= 0 || a->page_size > 64 || a->head_dim <= 0 || a->head_dim % 16 ||
      a->page_size * (a->head_dim + 16) > 12 * 1024)
    return FS_ERR_UNSUPPORTED;
  if (a->num_pages >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  if ((int64_t)a->batch * a->kv_heads * 2 * kSelMaxCluster >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  // positions are counted in 32 bits, strides of the loops over them included
  if ((int64_t)a->table_cols * a->page_size >= (1ll << 30) || a->budget >= (1 << 30)) return FS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->k_values) | reinterpret_cast<uintptr_t>(a->v_values)) & 15)
    return FS_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(a->weights) | reinterpret_cast<uintptr_t>(a->weights_out) |
       reinterpret_cast<uintptr_t>(a->k_scale) | reinterpret_cast<uintptr_t>(a->v_scale)) & 3)
    return FS_ERR_ALIGNMENT;
  return FS_OK;
}

static int64_t evict_tokens_at_most(const FsEvictArgs* a) {
  return std::min<int64_t>(a->max_seq_len, (int64_t)a->table_cols * a->page_size);
}

static size_t evict_workspace(const FsEvictArgs* a) {
  int chunk = 0;
  const int C = select_cluster(evict_tokens_at_most(a), (int64_t)a->batch * a->kv_heads, &chunk);
  return chunk <= kSelSmemKeys ? 0 : (size_t)a->batch * a->kv_heads * C * chunk * 4;
}

template <typename Kernel>
static int launch_cluster(Kernel kernel, const char* what, int64_t rows, int cluster, int threads, size_t smem,
                          const EvictParams& p, void* stream) {
  if (smem > 0) {
    // always the largest size: a call on another host thread may be between this and its launch
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmemKeys * 4);
        e != cudaSuccess)
      return fail_cuda(what, e);
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p); e != cudaSuccess) return fail_cuda(what, e);
  return FS_OK;
}

// Rows that fill the GPU by themselves take one CTA of four warps each (few warps wait for
// each other, no long tail); fewer rows are spread over clusters of CTAs of eight warps, up to
// one round of their pages.
template <int kCh, int kPages, bool kSym>
static int launch_move_chunks(const FsEvictArgs* a, const EvictParams& p, void* stream) {
  const int npg = (a->budget + a->page_size - 1) / a->page_size;
  const int64_t rows = (int64_t)a->batch * a->kv_heads * 2;
  const char* what = "token move kernel launch";
  if (rows >= 2 * kEvictFill) return launch_cluster(move_tokens_kernel<kCh, kPages, 4, kSym>, what, rows, 1, 128, 0, p, stream);
  int C = 1;
  while (C < 8 && rows * C < 2 * kEvictFill && npg > C * 8 * kPages) C *= 2;
  return launch_cluster(move_tokens_kernel<kCh, kPages, 8, kSym>, what, rows, C, 256, 0, p, stream);
}

template <bool kSym>
static int launch_move(const FsEvictArgs* a, const EvictParams& p, void* stream) {
  const int chunks = (a->page_size * a->head_dim + 511) / 512;
  if (chunks <= 1) return launch_move_chunks<1, 2, kSym>(a, p, stream);
  if (chunks <= 2) return launch_move_chunks<2, 2, kSym>(a, p, stream);
  if (chunks <= 4) return launch_move_chunks<4, kSym ? 2 : 1, kSym>(a, p, stream);
  if (chunks <= 8) return launch_move_chunks<8, 1, kSym>(a, p, stream);
  if (chunks <= 16) return launch_move_chunks<16, 1, kSym>(a, p, stream);
  return launch_move_chunks<24, 1, kSym>(a, p, stream);
}

}  // namespace fsb

extern "C" {

int fs_evict_workspace_size(const FsEvictArgs* a, size_t* bytes) {
  if (bytes == nullptr) return FS_ERR_INVALID_ARGUMENT;
  if (int st = fsb::evict_check(a); st != FS_OK) return st;
  *bytes = fsb::evict_workspace(a);
  return FS_OK;
}

int fs_evict_tokens(const FsEvictArgs* a, void* stream) {
  using namespace fsb;
  if (int st = evict_check(a); st != FS_OK) return st;
  const size_t need = evict_workspace(a);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return FS_ERR_WORKSPACE;
  if (need > 0 && (reinterpret_cast<uintptr_t>(a->workspace) & 255)) return FS_ERR_ALIGNMENT;  // keys go by 16 bytes
  EvictParams p{};
  p.table = a->block_table;
  p.lengths = a->lengths;
  p.weights = a->weights;
  p.weights_out = a->weights_out;
  p.kept = a->kept;
  p.new_lengths = a->new_lengths;
  p.status = a->device_status;
  p.values[0] = a->k_values;
  p.values[1] = a->v_values;
  p.scale[0] = a->k_scale;
  p.scale[1] = a->v_scale;
  p.zero[0] = a->k_zero;
  p.zero[1] = a->v_zero;
  p.num_pages = a->num_pages;
  p.max_seq_len = a->max_seq_len;
  p.Hkv = a->kv_heads;
  p.cols = a->table_cols;
  p.page = a->page_size;
  p.D = a->head_dim;
  p.budget = a->budget;
  p.recent = a->recent;
  p.sinks = a->sinks;
  p.by_page = divisor(a->page_size);
  p.by_dim = divisor(a->head_dim);
  p.sym = a->kv_format == FS_KV_SYMMETRIC;
  p.vec = a->page_size % 4 == 0 && ((reinterpret_cast<uintptr_t>(a->weights) | reinterpret_cast<uintptr_t>(a->weights_out)) & 15) == 0;
  const int C = select_cluster(evict_tokens_at_most(a), (int64_t)a->batch * a->kv_heads, &p.chunk_cap);
  const int64_t rows = (int64_t)a->batch * a->kv_heads;
  int st;
  if (need > 0) {
    p.keys = static_cast<uint32_t*>(a->workspace);
    st = launch_cluster(select_tokens_kernel<false>, "token selection kernel launch", rows, C, kSelThreads, 0, p, stream);
  } else {
    st = launch_cluster(select_tokens_kernel<true>, "token selection kernel launch", rows, C, kSelThreads,
                        (size_t)std::max(p.chunk_cap, 4) * 4, p, stream);
  }
  if (st != FS_OK) return st;
  // no request can be longer than the budget: nothing to move
  if (evict_tokens_at_most(a) <= a->budget) return FS_OK;
  return p.sym ? launch_move<true>(a, p, stream) : launch_move<false>(a, p, stream);
}

}  // extern "C"
