// The latent cache: keys and values of all heads from one shared vector a token.
//
// A token holds a latent vector c (dc values, INT8 with one fp32 scale, symmetric) and a
// rotary part r (dr values, 16 bit).  Absorbed attention works on the latents themselves:
//   score(t, h, j) = sm_scale * (scale_j * q_latent[t, h] . code_j + q_rope[t, h] . r_j)
//   out[t, h]      = sum_j softmax_j(score) * scale_j * code_j
// so every token is read once, dc + 4 + 2 dr bytes, for all heads: 16-row calls are bound by
// memory, calls of 64 and more rows by the tensor cores.
//
// latent_attention_kernel.  Rows (t, h) of a request are cut into blocks of up to 16, 32 or
// 64; the flattened list of (request, row block, tile of 64 tokens) is cut into equal
// contiguous shares, one per CTA (lengths are read on the device).  A CTA keeps three tiles
// in flight with cp.async.  Per tile:
//   1. S = Q C^T on the int8 tensor cores, straight from the stored bytes: q is held as
//      16-bit fixed point in two signed bytes (error max|q| 2^-16 of a row), two exact
//      MMAs; the rotary part on 16-bit MMAs.  The eight warps split rows, dims and tokens
//      (kMT x kKS x kTS), so q stays in registers; their partial sums meet in shared memory.
//   2. softmax: running maximum m of score + log2(scale) and sum of 2^(score - m) per row in
//      fp32; P = 2^(score - m) * scale in fp16, scaled by 2^14 to use its range whatever the
//      scale (the largest P is 2^14).
//   3. O += P C: each warp owns dc / 8 dims of all rows.  A byte becomes the exact fp16
//      integer (XOR and byte permute against 0x64 exponent bytes, minus 1152).
// A share that holds a whole (request, row block) writes the output; others leave normalised
// (O, LSE) partials that latent_merge_kernel joins.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <math.h>
#include <stdint.h>
#include <algorithm>
#include <mutex>

#include "../../include/flashspec_b200.h"
#include "common.h"
#include "ptx.cuh"

namespace fsb {

// ---------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------

struct LatentAppendParams {
  const void* latent;
  const void* rope;
  int64_t ls_b, ls_t, rs_b, rs_t;  // element strides of latent and rope [B, T, .]
  const int64_t* table;
  const int64_t* lengths;
  const int64_t* counts;
  int8_t* values;
  float* scale;
  void* ropes;
  void* held;
  int64_t* new_lengths;
  uint32_t* status;
  int64_t num_pages;
  int B, T, dc, dr, page, cols, bf16;
};

__device__ __forceinline__ float lat_f32(uint16_t x, int bf16) {
  return bf16 ? __bfloat162float(__ushort_as_bfloat16(x)) : __half2float(__ushort_as_half(x));
}
__device__ __forceinline__ uint16_t lat_b16(float x, int bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}

constexpr int kAppendWarps = 8;

// One warp per new token: lane l takes the elements l, l + 32, ... in groups of kVec.  The
// code and the scale are the symmetric format's (fs_quantize_symmetric): every operation is
// rounded once, as 32-bit arithmetic does.
__global__ void __launch_bounds__(kAppendWarps * 32) latent_append_kernel(const LatentAppendParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  if (item >= (int64_t)p.B * p.T) return;
  const int b = (int)(item / p.T), t = (int)(item % p.T);
  const int64_t count = p.counts != nullptr ? min(max(p.counts[b], (int64_t)0), (int64_t)p.T) : p.T;
  const int64_t len = max(p.lengths[b], (int64_t)0);
  if (t == 0 && lane == 0) p.new_lengths[b] = len + count;
  const uint16_t* src = static_cast<const uint16_t*>(p.latent) + b * p.ls_b + t * p.ls_t;
  uint16_t* held = p.held != nullptr ? static_cast<uint16_t*>(p.held) + item * p.dc : nullptr;
  if (t >= count) {
    if (held != nullptr)
      for (int e = lane; e < p.dc; e += 32) held[e] = 0;
    return;
  }
  const int64_t pos = len + t, lp = pos / p.page;
  int64_t phys = lp < p.cols ? p.table[(size_t)b * p.cols + lp] : -1;
  if (phys < 0 || phys >= p.num_pages) {  // no page to write to
    if (lane == 0 && p.status != nullptr) atomicOr(p.status, FS_DEV_BAD_PAGE);
    phys = -1;
  }
  float amax = 0.f;
  for (int e = lane; e < p.dc; e += 32) amax = fmaxf(amax, fabsf(lat_f32(src[e], p.bf16)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float scale = fmaxf(__fdiv_rn(amax, 127.0f), 1.0e-8f);
  const size_t row = phys < 0 ? 0 : (size_t)phys * p.page + (size_t)(pos - lp * p.page);
  for (int e = lane; e < p.dc; e += 32) {
    const float q = fminf(fmaxf(rintf(__fdiv_rn(lat_f32(src[e], p.bf16), scale)), -127.f), 127.f);
    if (phys >= 0) p.values[row * p.dc + e] = (int8_t)(int)q;
    if (held != nullptr) held[e] = lat_b16(__fmul_rn(q, scale), p.bf16);
  }
  if (phys < 0) return;
  if (lane == 0) p.scale[row] = scale;
  const uint16_t* rsrc = static_cast<const uint16_t*>(p.rope) + b * p.rs_b + t * p.rs_t;
  uint16_t* rdst = static_cast<uint16_t*>(p.ropes) + row * p.dr;
  for (int e = lane; e < p.dr; e += 32) rdst[e] = rsrc[e];
}

// ---------------------------------------------------------------------------------
// absorbed attention
// ---------------------------------------------------------------------------------

constexpr int kLatThreads = 256;
constexpr int kLatWarps = 8;
constexpr int kTile = 64;  // tokens
constexpr int kLatStages = 3;
constexpr int kSPad = 72;  // floats a row of partial scores
constexpr int kPPad = 72;  // halves a row of P
constexpr int kLatMaxBatch = 4096;
constexpr float kPTop = 16384.f;

struct LatentParams {
  const uint16_t* q;       // [B, T, H, dc]
  const uint16_t* q_rope;  // [B, T, H, dr]
  const int8_t* values;    // [P, page, dc]
  const float* scale;      // [P, page]
  const uint16_t* ropes;   // [P, page, dr]
  const int64_t* table;
  const int64_t* lengths;
  uint16_t* out;  // [B, T, H, dc]
  float* part_o;  // [ctas][2][rows of a block][dc]
  float* part_lse;  // [ctas][2][rows of a block], log2 domain
  int* prefix;  // [B + 1] tiles before each request (row blocks not counted)
  uint32_t* status;
  int64_t num_pages, max_seq_len;
  float scale_log2;  // sm_scale * log2(e)
  int B, T, H, R, row_blocks, page, cols, bf16;
};

__device__ __forceinline__ int latent_len(const LatentParams& p, int b) {
  return (int)max((int64_t)0, min(min(p.lengths[b], p.max_seq_len), (int64_t)p.cols * p.page));
}

// Bank swizzle of the 16-byte chunks of a row: rows r and r + 1 differ by 4 chunks (two rows
// of four chunks are read together), eight rows by eight different amounts.
__device__ __forceinline__ int lat_swz(int row) { return ((row & 1) << 2) | ((row >> 1) & 3); }

template <int kDC, int kDR, int kMT>
struct LatentShape {
  static constexpr int kRows = 16 * kMT;
  // warps = kMT row groups x kKS slices of the dims (64 at least) x kTS token groups
  static constexpr int kKS = (8 / kMT) < (kDC / 64) ? (8 / kMT) : (kDC / 64);
  static constexpr int kTS = 8 / (kMT * kKS);
  static constexpr int kSlice = kDC / kKS;        // dims of a warp's QK slice
  static constexpr int kQSteps = kSlice / 32;     // int8 MMA steps
  static constexpr int kNT = kTile / 8 / kTS;     // n-tiles of 8 tokens a warp
  static constexpr int kRSteps = kDR / 16;        // rotary MMA steps, dealt to the slices
  static constexpr int kRPer = (kRSteps + kKS - 1) / kKS;
  static constexpr int kDW = kDC / 8;             // dims of a warp's O
  static constexpr int kOT = kDW / 8;             // n-tiles of O
  static constexpr int kTPR = kLatThreads / kRows;  // softmax threads a row
  static constexpr int kSeg = kTile / 4 / kTPR;     // groups of four tokens a softmax thread
  static constexpr int kValBytes = kTile * kDC, kRopeBytes = kTile * kDR * 2;
  static constexpr int kStage = kValBytes + kRopeBytes + kTile * 4;
  static constexpr int kSBytes = kKS * kRows * kSPad * 4;
  static constexpr int kPBytes = kRows * kPPad * 2;
  static constexpr int kOffS = kLatStages * kStage;
  static constexpr int kOffP = kOffS + kSBytes;
  static constexpr int kOffMisc = kOffP + kPBytes;  // alpha [rows], qscale [rows], lam [tile], prefix
  static constexpr int kMiscFloats = 2 * kRows + kTile;
  static constexpr __host__ __device__ int smem(int batch) { return kOffMisc + kMiscFloats * 4 + (batch + 1) * 4; }
};

__device__ __forceinline__ void lat_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void mma_16816_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

// Tiles before each request, into pre[0 .. B] (shared memory); every thread calls it.
__device__ __forceinline__ void latent_prefix(const LatentParams& p, int* pre) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int r = tid; r < p.B; r += kLatThreads) pre[r + 1] = (latent_len(p, r) + kTile - 1) / kTile;
  __syncthreads();
  if (tid < 32) {
    int carry = 0;
    for (int base = 0; base < p.B; base += 32) {
      int x = base + lane < p.B ? pre[base + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (base + lane < p.B) pre[base + lane + 1] = carry + x;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  __syncthreads();
}

// Share k of C of n flat tiles starts here.
__device__ __forceinline__ int64_t latent_share(int64_t n, int k, int C) { return n * k / C; }

template <int kDC, int kDR, int kMT, bool kBf16>
__global__ void __launch_bounds__(kLatThreads, 1) latent_attention_kernel(const LatentParams p) {
  using L = LatentShape<kDC, kDR, kMT>;
  extern __shared__ __align__(1024) uint8_t lat_smem[];
  const uint32_t smem_s = smem_u32(lat_smem);
  float* s_part = reinterpret_cast<float*>(lat_smem + L::kOffS);  // [kKS][rows][kSPad]
  __half* s_p = reinterpret_cast<__half*>(lat_smem + L::kOffP);   // [rows][kPPad]
  float* s_alpha = reinterpret_cast<float*>(lat_smem + L::kOffMisc);
  float* s_qscale = s_alpha + L::kRows;
  float* s_lam = s_qscale + L::kRows;
  int* pre = reinterpret_cast<int*>(s_lam + kTile);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int mt = warp % kMT, ks = (warp / kMT) % L::kKS, ts = warp / (kMT * L::kKS);

  latent_prefix(p, pre);
  if (blockIdx.x == 0)
    for (int r = tid; r <= p.B; r += kLatThreads) p.prefix[r] = pre[r];
  const int64_t total = (int64_t)pre[p.B] * p.row_blocks;
  const int64_t f_begin = latent_share(total, blockIdx.x, gridDim.x);
  const int64_t f_end = latent_share(total, blockIdx.x + 1, gridDim.x);
  bool first = true;

  // softmax thread: row and its token groups
  const int srow = tid / L::kTPR, sj = tid % L::kTPR;

  for (int64_t f = f_begin; f < f_end;) {
    // ---- the piece: tiles [t0, t1) of row block rb of request b
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)pre[mid] * p.row_blocks <= f) lo = mid; else hi = mid;
    }
    const int b = lo, nt = pre[b + 1] - pre[b];
    const int64_t off = f - (int64_t)pre[b] * p.row_blocks;
    const int rb = (int)(off / nt), t0 = (int)(off % nt);
    const int t1 = (int)min((int64_t)nt, t0 + (f_end - f));
    f += t1 - t0;
    const int len = latent_len(p, b);
    const int row0 = rb * L::kRows, rows = min(L::kRows, p.R - row0);
    const uint16_t* qb = p.q + ((size_t)b * p.R + row0) * kDC;
    const uint16_t* qrb = p.q_rope + ((size_t)b * p.R + row0) * kDR;
    const int64_t* trow = p.table + (size_t)b * p.cols;

    // ---- tile loader: values, rotary parts and scales of tile t into stage t % kLatStages
    auto load_tile = [&](int t) {
      const int st = t % kLatStages;
      const uint32_t base = smem_s + st * L::kStage;
      const int tok0 = t * kTile;
      constexpr int kVC = kDC / 16, kRC = kDR / 8;  // 16-byte chunks of a row
#pragma unroll
      for (int i = tid; i < kTile * kVC; i += kLatThreads) {
        const int r = i / kVC, ch = i % kVC, tok = tok0 + r;
        if (tok < len) {
          const int lp = tok / p.page;
          const int64_t phys = trow[lp];
          if (phys >= 0 && phys < p.num_pages)
            lat_cp16(base + r * kDC + ((ch ^ lat_swz(r)) << 4),
                     p.values + ((size_t)phys * p.page + (tok - lp * p.page)) * kDC + 16 * ch);
        }
      }
#pragma unroll
      for (int i = tid; i < kTile * kRC; i += kLatThreads) {
        const int r = i / kRC, ch = i % kRC, tok = tok0 + r;
        if (tok < len) {
          const int lp = tok / p.page;
          const int64_t phys = trow[lp];
          if (phys >= 0 && phys < p.num_pages)
            lat_cp16(base + L::kValBytes + r * kDR * 2 + ((ch ^ (lat_swz(r) & (kRC - 1))) << 4),
                     p.ropes + ((size_t)phys * p.page + (tok - lp * p.page)) * kDR + 8 * ch);
        }
      }
      if (tid < kTile) {  // a token that is not there gets scale -1
        const int tok = tok0 + tid;
        const uint32_t dst = base + L::kValBytes + L::kRopeBytes + 4 * tid;
        int64_t phys = -1;
        int lp = 0;
        if (tok < len) {
          lp = tok / p.page;
          phys = trow[lp];
          if (phys >= p.num_pages) {
            if (p.status != nullptr) atomicOr(p.status, FS_DEV_BAD_PAGE);
            phys = -1;
          }
        }
        if (phys >= 0)
          cp_async_4(dst, p.scale + (size_t)phys * p.page + (tok - lp * p.page));
        else
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst), "f"(-1.f) : "memory");
      }
    };

    __syncthreads();  // the previous piece is done with the stages and the row state
    load_tile(t0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (t0 + 1 < t1) load_tile(t0 + 1);
    asm volatile("cp.async.commit_group;" ::: "memory");

    // ---- q as 16-bit fixed point: row scales, then this warp's fragments
    for (int r = warp; r < L::kRows; r += kLatWarps) {
      float amax = 0.f;
      bool bad = false;
      if (r < rows) {
        for (int e = 4 * lane; e < kDC; e += 128) {
          const uint2 w = *reinterpret_cast<const uint2*>(qb + (size_t)r * kDC + e);
          const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = fabsf(lat_f32((uint16_t)(ww[j >> 1] >> (16 * (j & 1))), kBf16));
            bad |= !(v < INFINITY);
            amax = fmaxf(amax, v);
          }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      bad = __any_sync(0xffffffffu, bad);
      // a row with infinities or NaN has no scale: its output is NaN
      if (lane == 0) s_qscale[r] = bad ? __int_as_float(0x7fc00000) : amax / 32639.0f;
    }
    __syncthreads();
    uint32_t qhi[L::kQSteps][4], qlo[L::kQSteps][4];  // a0..a3 of the m16n8k32 MMAs
    float fq[2];                                       // row scale * sm_scale * log2 e, rows g and g + 8
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      const int r = 16 * mt + g + 8 * r2;
      const float qs = s_qscale[r], inv = qs > 0.f ? 1.f / qs : 0.f;
      fq[r2] = qs * p.scale_log2;
#pragma unroll
      for (int j = 0; j < L::kQSteps; ++j) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {  // the words b0 / b1 of step j: dims 64 (j / 2) + 16 c + 8 (j & 1) + 4 w
          const int d = ks * L::kSlice + 64 * (j >> 1) + 16 * c + 8 * (j & 1) + 4 * w;
          uint2 raw = make_uint2(0u, 0u);
          if (r < rows) raw = *reinterpret_cast<const uint2*>(qb + (size_t)r * kDC + d);
          const uint32_t ww[2] = {raw.x, raw.y};
          uint32_t h = 0u, l = 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = lat_f32((uint16_t)(ww[e >> 1] >> (16 * (e & 1))), kBf16);
            const int q16 = max(-32639, min(32639, __float2int_rn(v * inv)));
            const int qh = (q16 + 128) >> 8;
            h |= (uint32_t)(qh & 0xff) << (8 * e);
            l |= (uint32_t)((q16 - (qh << 8)) & 0xff) << (8 * e);
          }
          qhi[j][2 * w + r2] = h;
          qlo[j][2 * w + r2] = l;
        }
      }
    }
    uint32_t qr[L::kRPer][4];  // rotary fragments of steps ks, ks + kKS, ...: dims 16 s + 4 c .. + 3
#pragma unroll
    for (int i = 0; i < L::kRPer; ++i) {
      const int s = ks + i * L::kKS;
#pragma unroll
      for (int r2 = 0; r2 < 2; ++r2) {
        const int r = 16 * mt + g + 8 * r2;
        uint2 raw = make_uint2(0u, 0u);
        if (r < rows && s < L::kRSteps) raw = *reinterpret_cast<const uint2*>(qrb + (size_t)r * kDR + 16 * s + 4 * c);
        qr[i][r2] = raw.x;
        qr[i][2 + r2] = raw.y;
      }
    }

    float acc[kMT][L::kOT][4];
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int j = 0; j < L::kOT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][j][k] = 0.f;
    float m_run = -1.0e30f, l_run = 0.f;
    // tokens that this softmax thread's row sees: query t sees the first len - T + t + 1
    const int limit = len - p.T + 1 + (row0 + srow) / p.H;

    for (int t = t0; t < t1; ++t) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();  // tile t is here; every warp is done with tile t - 1
      if (t + 2 < t1) load_tile(t + 2);
      asm volatile("cp.async.commit_group;" ::: "memory");
      const uint32_t base = smem_s + (t % kLatStages) * L::kStage;
      const float* tok_scale =
          reinterpret_cast<const float*>(lat_smem + (t % kLatStages) * L::kStage + L::kValBytes + L::kRopeBytes);
      if (tid < kTile) s_lam[tid] = fmaxf(lg2_approx(fmaxf(tok_scale[tid], 0.f)), -100.f);

      // ---- 1. partial scores of this warp's rows, dims and tokens
#pragma unroll
      for (int n = 0; n < L::kNT; ++n) {
        const int tok = (ts * L::kNT + n) * 8;
        int sh[4] = {0, 0, 0, 0}, sl[4] = {0, 0, 0, 0};
        const int brow = tok + g;
#pragma unroll
        for (int j2 = 0; j2 < L::kQSteps / 2; ++j2) {
          const int ch = (ks * L::kSlice + 64 * j2) / 16 + c;
          const uint4 kv = lds128(base + brow * kDC + ((ch ^ lat_swz(brow)) << 4));
          mma_16832_s8(sh, qhi[2 * j2][0], qhi[2 * j2][1], qhi[2 * j2][2], qhi[2 * j2][3], kv.x, kv.y);
          mma_16832_s8(sl, qlo[2 * j2][0], qlo[2 * j2][1], qlo[2 * j2][2], qlo[2 * j2][3], kv.x, kv.y);
          mma_16832_s8(sh, qhi[2 * j2 + 1][0], qhi[2 * j2 + 1][1], qhi[2 * j2 + 1][2], qhi[2 * j2 + 1][3], kv.z, kv.w);
          mma_16832_s8(sl, qlo[2 * j2 + 1][0], qlo[2 * j2 + 1][1], qlo[2 * j2 + 1][2], qlo[2 * j2 + 1][3], kv.z, kv.w);
        }
        float rp[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < L::kRPer; ++i) {
          const int s = ks + i * L::kKS;
          if (s < L::kRSteps) {
            constexpr int kRC = kDR / 8;
            const int ch = 2 * s + (c >> 1);
            const uint32_t at = base + L::kValBytes + brow * kDR * 2 + ((ch ^ (lat_swz(brow) & (kRC - 1))) << 4) + 8 * (c & 1);
            const float2 w = lds64f(at);
            const uint32_t b0 = __float_as_uint(w.x), b1 = __float_as_uint(w.y);
            if (kBf16)
              mma_16816_bf16(rp, qr[i][0], qr[i][1], qr[i][2], qr[i][3], b0, b1);
            else
              mma_16816(rp, qr[i][0], qr[i][1], qr[i][2], qr[i][3], b0, b1);
          }
        }
        const float2 sc = *reinterpret_cast<const float2*>(tok_scale + tok + 2 * c);
        float* dst = s_part + ((size_t)ks * L::kRows + 16 * mt + g) * kSPad + tok + 2 * c;
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          const float x0 = fmaf(256.f, (float)sh[2 * r2], (float)sl[2 * r2]) * (fq[r2] * sc.x);
          const float x1 = fmaf(256.f, (float)sh[2 * r2 + 1], (float)sl[2 * r2 + 1]) * (fq[r2] * sc.y);
          *reinterpret_cast<float2*>(dst + 8 * r2 * kSPad) =
              make_float2(fmaf(rp[2 * r2], p.scale_log2, x0), fmaf(rp[2 * r2 + 1], p.scale_log2, x1));
        }
      }
      __syncthreads();

      // ---- 2. softmax of row srow, four tokens at a time
      float z[L::kSeg][4];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < L::kSeg; ++i) {
        const int tk = 4 * (sj + L::kTPR * i);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k2 = 0; k2 < L::kKS; ++k2) {
          const float4 x = *reinterpret_cast<const float4*>(s_part + ((size_t)k2 * L::kRows + srow) * kSPad + tk);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        const float vv[4] = {v.x, v.y, v.z, v.w};
        const float4 sc = *reinterpret_cast<const float4*>(tok_scale + tk);
        const float scs[4] = {sc.x, sc.y, sc.z, sc.w};
        const float4 lm = *reinterpret_cast<const float4*>(s_lam + tk);
        const float lms[4] = {lm.x, lm.y, lm.z, lm.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool seen = t * kTile + tk + k < limit && !(scs[k] < 0.f);
          z[i][k] = seen ? vv[k] : -INFINITY;
          mx = fmaxf(mx, z[i][k] + lms[k]);
        }
      }
#pragma unroll
      for (int o = L::kTPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(m_run, mx);
      const float alpha = ex2_approx(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < L::kSeg; ++i) {
        const int tk = 4 * (sj + L::kTPR * i);
        const float4 sc = *reinterpret_cast<const float4*>(tok_scale + tk);
        const float scs[4] = {sc.x, sc.y, sc.z, sc.w};
        float pr[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = ex2_approx(z[i][k] - m_new);
          l_run += e;
          pr[k] = e * (scs[k] * kPTop);
        }
        uint2 w;
        w.x = pack_half2(pr[0], pr[1]);
        w.y = pack_half2(pr[2], pr[3]);
        *reinterpret_cast<uint2*>(s_p + srow * kPPad + tk) = w;
      }
      if (sj == 0) s_alpha[srow] = alpha;
      __syncthreads();

      // ---- 3. O += P C for this warp's dims
      float al[kMT][2];
      bool rescale = false;
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          al[i][r2] = s_alpha[16 * i + g + 8 * r2];
          rescale |= al[i][r2] != 1.f;
        }
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int j = 0; j < L::kOT; ++j) {
            acc[i][j][0] *= al[i][0];
            acc[i][j][1] *= al[i][0];
            acc[i][j][2] *= al[i][1];
            acc[i][j][3] *= al[i][1];
          }
      }
      const uint32_t p_s = smem_s + L::kOffP;
#pragma unroll
      for (int kk = 0; kk < kTile / 16; ++kk) {
        uint32_t pa[kMT][4];
#pragma unroll
        for (int i = 0; i < kMT; ++i)
          ldsm_x4(p_s + ((16 * i + (lane & 15)) * kPPad + 16 * kk + 8 * (lane >> 4)) * 2, pa[i][0], pa[i][1], pa[i][2],
                  pa[i][3]);
        // matrices of a transposed load: (tokens 0-7 | 8-15 of the step) x (chunk ch | ch + 1)
        constexpr int kChunks = L::kDW / 16;
        static_assert(kChunks >= 1, "a warp owns whole 16-dim chunks");
        const int r = 16 * kk + (lane & 7) + 8 * ((lane >> 3) & 1);
#pragma unroll
        for (int ch0 = 0; ch0 < kChunks; ch0 += 2) {
          uint32_t v[4];
          // with one chunk a warp (dc = 128) the second pair of matrices repeats the first
          const int ch = warp * kChunks + ch0 + (kChunks > 1 ? (lane >> 4) : 0);
          ldsm_x4_trans(base + r * kDC + ((ch ^ lat_swz(r)) << 4), v[0], v[1], v[2], v[3]);
#pragma unroll
          for (int u = 0; u < (kChunks > 1 ? 2 : 1); ++u) {
            // bytes [token 2c: dims 2g, 2g + 1][token 2c + 1: the same]; even dims form one
            // n-tile, odd dims the next
            const uint32_t x0 = v[2 * u] ^ 0x80808080u, x1 = v[2 * u + 1] ^ 0x80808080u;
            const __half2 base2 = __half2half2(__ushort_as_half((unsigned short)0x6480));  // 1152
            auto cvt = [&](uint32_t x, uint32_t sel) -> uint32_t {
              const uint32_t h = prmt(x, 0x64646464u, sel);
              const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), base2);
              return *reinterpret_cast<const uint32_t*>(&d);
            };
            const uint32_t e0 = cvt(x0, 0x4240u), e1 = cvt(x1, 0x4240u), o0 = cvt(x0, 0x4341u), o1 = cvt(x1, 0x4341u);
#pragma unroll
            for (int i = 0; i < kMT; ++i) {
              mma_16816(acc[i][2 * (ch0 + u)], pa[i][0], pa[i][1], pa[i][2], pa[i][3], e0, e1);
              mma_16816(acc[i][2 * (ch0 + u) + 1], pa[i][0], pa[i][1], pa[i][2], pa[i][3], o0, o1);
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- close the piece: normalise
    float l = l_run;
#pragma unroll
    for (int o = L::kTPR / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncthreads();  // every warp has read the last alphas
    if (sj == 0) {
      s_alpha[srow] = l > 0.f ? 1.f / (l * kPTop) : (l == 0.f ? 0.f : l);  // NaN stays
      s_qscale[srow] = l > 0.f ? m_run + log2f(l) : (l == 0.f ? -INFINITY : l);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    const size_t slot = ((size_t)blockIdx.x * 2 + (first ? 0 : 1)) * L::kRows;
    first = false;
    if (!whole && tid < rows) p.part_lse[slot + tid] = s_qscale[tid];
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int r2 = 0; r2 < 2; ++r2) {
        const int r = 16 * i + g + 8 * r2;
        if (r >= rows) continue;
        const float inv = s_alpha[r];
#pragma unroll
        for (int j = 0; j < L::kOT; j += 2) {  // dims 16 (j / 2) + 4c .. + 3: even tile, odd tile interleaved
          const int d = warp * L::kDW + 8 * j + 4 * c;
          const float o0 = acc[i][j][2 * r2] * inv, o1 = acc[i][j + 1][2 * r2] * inv;
          const float o2 = acc[i][j][2 * r2 + 1] * inv, o3 = acc[i][j + 1][2 * r2 + 1] * inv;
          if (whole) {
            uint2 w;
            w.x = (uint32_t)lat_b16(o0, kBf16) | ((uint32_t)lat_b16(o1, kBf16) << 16);
            w.y = (uint32_t)lat_b16(o2, kBf16) | ((uint32_t)lat_b16(o3, kBf16) << 16);
            *reinterpret_cast<uint2*>(p.out + ((size_t)b * p.R + row0 + r) * kDC + d) = w;
          } else {
            *reinterpret_cast<float4*>(p.part_o + (slot + r) * kDC + d) = make_float4(o0, o1, o2, o3);
          }
        }
      }
  }
}

// Joins the partials of each (request, row block) that several shares hold, and writes zeros
// for requests without tokens.  One CTA per (request, row block, 4 rows); a warp a row.
constexpr int kMergeWarps = 4;

__global__ void __launch_bounds__(kMergeWarps * 32) latent_merge_kernel(const LatentParams p, int block_rows, int dc,
                                                                       int ctas) {
  const int groups = (block_rows + kMergeWarps - 1) / kMergeWarps;
  const int grp = blockIdx.x % groups, item = blockIdx.x / groups, rb = item % p.row_blocks, b = item / p.row_blocks;
  const int lane = threadIdx.x & 31;
  const int r = grp * kMergeWarps + (threadIdx.x >> 5), row = rb * block_rows + r;
  if (r >= block_rows || row >= p.R) return;
  const int nt = p.prefix[b + 1] - p.prefix[b];
  uint16_t* out = p.out + ((size_t)b * p.R + row) * dc;
  if (nt == 0) {
    for (int d = 4 * lane; d < dc; d += 128) *reinterpret_cast<uint2*>(out + d) = make_uint2(0u, 0u);
    return;
  }
  const int64_t total = (int64_t)p.prefix[p.B] * p.row_blocks;
  const int64_t f0 = (int64_t)p.prefix[b] * p.row_blocks + (int64_t)rb * nt, f1 = f0 + nt;
  // the share that holds flat tile f: the last one that starts at or before it
  auto owner = [&](int64_t f) -> int {
    int k = (int)min((int64_t)ctas - 1, (f + 1) * ctas / total);
    while (k > 0 && latent_share(total, k, ctas) > f) --k;
    while (k + 1 < ctas && latent_share(total, k + 1, ctas) <= f) ++k;
    return k;
  };
  const int k0 = owner(f0), k1 = owner(f1 - 1);
  if (k0 == k1) return;  // one share wrote the output itself
  // the first share's piece is its first one only if the share starts in this row block
  auto slot = [&](int k) -> size_t {
    const bool is_first = k > k0 || latent_share(total, k, ctas) >= f0;
    return ((size_t)k * 2 + (is_first ? 0 : 1)) * block_rows + r;
  };
  float M = -INFINITY;
  bool nan = false;
  for (int k = k0 + lane; k <= k1; k += 32) {
    if (latent_share(total, k, ctas) == latent_share(total, k + 1, ctas)) continue;  // an empty share
    const float x = p.part_lse[slot(k)];
    nan |= isnan(x);
    M = fmaxf(M, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (__any_sync(0xffffffffu, nan)) M = __int_as_float(0x7fc00000);
  float W = 0.f;
  float4 acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (M != -INFINITY) {
    for (int k = k0; k <= k1; ++k) {
      if (latent_share(total, k, ctas) == latent_share(total, k + 1, ctas)) continue;
      const size_t s = slot(k);
      const float w = exp2f(p.part_lse[s] - M);
      W += w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 4 * lane + 128 * j;
        if (d >= dc) break;
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + s * dc + d);
        acc[j].x = fmaf(w, v.x, acc[j].x);
        acc[j].y = fmaf(w, v.y, acc[j].y);
        acc[j].z = fmaf(w, v.z, acc[j].z);
        acc[j].w = fmaf(w, v.w, acc[j].w);
      }
    }
  }
  const float inv = W > 0.f ? 1.f / W : (W == 0.f ? 0.f : W);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = 4 * lane + 128 * j;
    if (d >= dc) break;
    uint2 w;
    w.x = (uint32_t)lat_b16(acc[j].x * inv, p.bf16) | ((uint32_t)lat_b16(acc[j].y * inv, p.bf16) << 16);
    w.y = (uint32_t)lat_b16(acc[j].z * inv, p.bf16) | ((uint32_t)lat_b16(acc[j].w * inv, p.bf16) << 16);
    *reinterpret_cast<uint2*>(out + d) = w;
  }
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------

static bool latent_dims_ok(int dc, int dr, int page) {
  return (dc == 128 || dc == 256 || dc == 512) && (dr == 32 || dr == 64) &&
         (page == 16 || page == 32 || page == 64 || page == 128);
}

static int latent_check(const FsLatentArgs* a) {
  if (a == nullptr || a->q == nullptr || a->q_rope == nullptr || a->values == nullptr || a->scale == nullptr ||
      a->ropes == nullptr || a->block_table == nullptr || a->lengths == nullptr || a->out == nullptr)
    return FS_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->tokens <= 0 || a->heads <= 0 || a->table_cols <= 0 || a->num_pages <= 0 ||
      a->max_seq_len < 0)
    return FS_ERR_INVALID_ARGUMENT;
  if (a->dtype != FS_F16 && a->dtype != FS_BF16) return FS_ERR_UNSUPPORTED;
  if (!latent_dims_ok(a->latent_dim, a->rope_dim, a->page_size) || a->batch > kLatMaxBatch) return FS_ERR_UNSUPPORTED;
  if ((int64_t)a->tokens * a->heads > (1 << 20)) return FS_ERR_UNSUPPORTED;
  if ((int64_t)a->table_cols * a->page_size >= (1ll << 31) - kTile) return FS_ERR_UNSUPPORTED;
  // flat tiles are counted in 32 bits before the row blocks
  const int64_t longest = std::min<int64_t>(a->max_seq_len, (int64_t)a->table_cols * a->page_size);
  if ((longest / kTile + 1) * a->batch >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_rope) |
       reinterpret_cast<uintptr_t>(a->values) | reinterpret_cast<uintptr_t>(a->ropes) |
       reinterpret_cast<uintptr_t>(a->out)) & 15)
    return FS_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(a->scale) & 3) return FS_ERR_ALIGNMENT;
  return FS_OK;
}

struct LatentPlan {
  int mt, row_blocks, ctas;
  size_t o, lse, prefix;
};

static LatentPlan latent_plan(const FsLatentArgs* a, int device) {
  LatentPlan pl{};
  const int R = a->tokens * a->heads;
  pl.mt = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int rows = 16 * pl.mt;
  pl.row_blocks = (R + rows - 1) / rows;
  pl.ctas = device_sm_count(device);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  pl.o = up((size_t)pl.ctas * 2 * rows * a->latent_dim * 4);
  pl.lse = up((size_t)pl.ctas * 2 * rows * 4);
  pl.prefix = up((size_t)(a->batch + 1) * 4);
  return pl;
}

template <int kDC, int kDR, int kMT>
static int launch_latent(const LatentParams& p, const LatentPlan& pl, void* stream) {
  using L = LatentShape<kDC, kDR, kMT>;
  static_assert(L::smem(kLatMaxBatch) <= 227 * 1024, "shared memory of a CTA");
  const int smem = L::smem(p.B);
  auto kernel = p.bf16 ? latent_attention_kernel<kDC, kDR, kMT, true> : latent_attention_kernel<kDC, kDR, kMT, false>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(kLatMaxBatch));
      e != cudaSuccess)
    return fail_cuda("shared-memory limit of the latent attention kernel", e);
  kernel<<<pl.ctas, kLatThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  if (int st = launch_status("latent attention kernel launch"); st != FS_OK) return st;
  const int64_t blocks = (int64_t)p.B * p.row_blocks * ((L::kRows + kMergeWarps - 1) / kMergeWarps);
  latent_merge_kernel<<<(unsigned)blocks, kMergeWarps * 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      p, L::kRows, kDC, pl.ctas);
  return launch_status("latent merge kernel launch");
}

template <int kDC, int kDR>
static int launch_latent_rows(const LatentParams& p, const LatentPlan& pl, void* stream) {
  switch (pl.mt) {
    case 1: return launch_latent<kDC, kDR, 1>(p, pl, stream);
    case 2: return launch_latent<kDC, kDR, 2>(p, pl, stream);
    default: return launch_latent<kDC, kDR, 4>(p, pl, stream);
  }
}

template <int kDC>
static int launch_latent_rope(const LatentParams& p, const LatentPlan& pl, int dr, void* stream) {
  return dr == 64 ? launch_latent_rows<kDC, 64>(p, pl, stream) : launch_latent_rows<kDC, 32>(p, pl, stream);
}

}  // namespace fsb

extern "C" {

int fs_latent_append(const FsLatentAppendArgs* a, void* stream) {
  using namespace fsb;
  if (a == nullptr || a->latent == nullptr || a->rope == nullptr || a->values == nullptr || a->scale == nullptr ||
      a->ropes == nullptr || a->block_table == nullptr || a->lengths == nullptr || a->new_lengths == nullptr)
    return FS_ERR_INVALID_ARGUMENT;
  if (static_cast<const int64_t*>(a->new_lengths) == a->lengths) return FS_ERR_INVALID_ARGUMENT;
  if (a->batch <= 0 || a->tokens <= 0 || a->table_cols <= 0 || a->num_pages <= 0) return FS_ERR_INVALID_ARGUMENT;
  if (a->dtype != FS_F16 && a->dtype != FS_BF16) return FS_ERR_UNSUPPORTED;
  if (!latent_dims_ok(a->latent_dim, a->rope_dim, a->page_size)) return FS_ERR_UNSUPPORTED;
  const int64_t blocks = ((int64_t)a->batch * a->tokens + kAppendWarps - 1) / kAppendWarps;
  if (blocks >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->latent) | reinterpret_cast<uintptr_t>(a->rope) |
       reinterpret_cast<uintptr_t>(a->ropes) | reinterpret_cast<uintptr_t>(a->held)) & 1)
    return FS_ERR_ALIGNMENT;
  LatentAppendParams p{};
  p.latent = a->latent;
  p.rope = a->rope;
  p.ls_b = a->latent_stride_b;
  p.ls_t = a->latent_stride_t;
  p.rs_b = a->rope_stride_b;
  p.rs_t = a->rope_stride_t;
  p.table = a->block_table;
  p.lengths = a->lengths;
  p.counts = a->counts;
  p.values = a->values;
  p.scale = a->scale;
  p.ropes = a->ropes;
  p.held = a->held;
  p.new_lengths = a->new_lengths;
  p.status = a->device_status;
  p.num_pages = a->num_pages;
  p.B = a->batch;
  p.T = a->tokens;
  p.dc = a->latent_dim;
  p.dr = a->rope_dim;
  p.page = a->page_size;
  p.cols = a->table_cols;
  p.bf16 = a->dtype == FS_BF16;
  latent_append_kernel<<<(unsigned)blocks, kAppendWarps * 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("latent append kernel launch");
}

int fs_latent_workspace_size(const FsLatentArgs* a, size_t* bytes) {
  if (bytes == nullptr) return FS_ERR_INVALID_ARGUMENT;
  if (int st = fsb::latent_check(a); st != FS_OK) return st;
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return fsb::fail_cuda("cudaGetDevice", e);
  const fsb::LatentPlan pl = fsb::latent_plan(a, device);
  *bytes = pl.o + pl.lse + pl.prefix;
  return FS_OK;
}

int fs_latent_attention(const FsLatentArgs* a, void* stream) {
  using namespace fsb;
  if (int st = latent_check(a); st != FS_OK) return st;
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return fail_cuda("cudaGetDevice", e);
  const LatentPlan pl = latent_plan(a, device);
  if (a->workspace == nullptr || a->workspace_bytes < pl.o + pl.lse + pl.prefix) return FS_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return FS_ERR_ALIGNMENT;
  if ((int64_t)a->batch * pl.row_blocks * 16 >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  LatentParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_rope = static_cast<const uint16_t*>(a->q_rope);
  p.values = a->values;
  p.scale = a->scale;
  p.ropes = static_cast<const uint16_t*>(a->ropes);
  p.table = a->block_table;
  p.lengths = a->lengths;
  p.out = static_cast<uint16_t*>(a->out);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_lse = reinterpret_cast<float*>(ws + pl.o);
  p.prefix = reinterpret_cast<int*>(ws + pl.o + pl.lse);
  p.status = a->device_status;
  p.num_pages = a->num_pages;
  p.max_seq_len = a->max_seq_len;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.B = a->batch;
  p.T = a->tokens;
  p.H = a->heads;
  p.R = a->tokens * a->heads;
  p.row_blocks = pl.row_blocks;
  p.page = a->page_size;
  p.cols = a->table_cols;
  p.bf16 = a->dtype == FS_BF16;
  switch (a->latent_dim) {
    case 128: return launch_latent_rope<128>(p, pl, a->rope_dim, stream);
    case 256: return launch_latent_rope<256>(p, pl, a->rope_dim, stream);
    default: return launch_latent_rope<512>(p, pl, a->rope_dim, stream);
  }
}

}  // extern "C"
