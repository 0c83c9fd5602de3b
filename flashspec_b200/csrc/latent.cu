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
// contiguous shares, one per CTA (lengths are read on the device).  Warp 0 keeps two or three
// tiles in flight with TMA (128-byte swizzle; page lookups run a tile ahead).  Per tile:
//   1. S = Q C^T on the int8 tensor cores, straight from the stored bytes: q is held as
//      16-bit fixed point in two signed bytes (error max|q| 2^-16 of a row), two exact
//      MMAs; the rotary part on 16-bit MMAs.  The warps split rows, dims and tokens (kMT x
//      kKS x kTS), so q stays in registers; their partial sums meet in shared memory.
//   2. softmax: reference m, a running maximum of score + log2(scale) that moves only when the
//      true one is past it by more than 2^4, and the sum of 2^(score - m), per row in fp32; P =
//      2^(score - m) * scale * 2^11 in fp16, so that P uses fp16's range whatever the scale: at
//      most 2^15, in full precision down to 2^-25 of the reference (many far tokens make the
//      dims in which one near token is zero).
//   3. O += P C: each warp owns its part of the dims, of all rows.  A byte becomes the exact fp16
//      integer (XOR and byte permute against 0x64 exponent bytes, minus 1152).
// A share that holds a whole (request, row block) writes the output; others leave normalised
// (O, LSE) partials that latent_merge_kernel joins.
// Measured: 64 ragged requests (8192 -> 128 tokens) x 16 rows 61.5 us (2.8 TB/s; the memory
// floor is 26.6), 16 requests (8192 -> 4096) x 128 rows 131 us (209 TFLOP/s; warp-level MMAs
// end at a measured 557); both issue in under half of the cycles, at 16 and 8 warps an SM.
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
#include "tensor_map.h"

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

// N consecutive 16-bit elements, in vector words where kVec (16-byte aligned rows).
template <int N, bool kVec>
__device__ __forceinline__ void lat_load(const uint16_t* src, uint16_t (&x)[N]) {
  if (kVec && N >= 8) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) *reinterpret_cast<uint4*>(x + 8 * i) = reinterpret_cast<const uint4*>(src)[i];
  } else if (kVec) {
    *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(src);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = src[i];
  }
}

// Out of line: the code by the format's own steps.
static __device__ __noinline__ float latent_code_exact(float x, float scale) {
  return fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.f), 127.f);
}

// One warp per new token; lane l takes elements [N l, N l + N), N = dc / 32.  The code and the
// scale are the symmetric format's (fs_quantize_symmetric): scale = max(amax / 127, 1e-8), code
// = rint(RN(x / scale)) clamped.  Bound by memory (2 dc read, dc and, with `held`, 2 dc written
// a token), so the division is done once a token: RN(x RN(1 / scale)) is within 127 * 2^-23 +
// 2^-18 < 2.1e-5 of RN(x / scale), and one farther than 2^-15 (3.1e-5) from a half-integer has
// the same rint; the others (0.006%) divide.
template <int kDC, bool kVec>
__global__ void __launch_bounds__(kAppendWarps * 32) latent_append_kernel(const LatentAppendParams p) {
  constexpr int N = kDC / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
  if (item >= (int64_t)p.B * p.T) return;
  const int b = (int)(item / p.T), t = (int)(item - (int64_t)b * p.T);
  const int64_t count = p.counts != nullptr ? min(max(p.counts[b], (int64_t)0), (int64_t)p.T) : p.T;
  const int64_t len = max(p.lengths[b], (int64_t)0);
  if (t == 0 && lane == 0) p.new_lengths[b] = len + count;
  uint16_t* held = p.held != nullptr ? static_cast<uint16_t*>(p.held) + item * kDC + N * lane : nullptr;
  alignas(16) uint16_t x[N], hv[N];
  auto put_held = [&]() {
    if (held == nullptr) return;
    if (kVec && N >= 8) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) reinterpret_cast<uint4*>(held)[i] = *reinterpret_cast<const uint4*>(hv + 8 * i);
    } else if (kVec) {
      *reinterpret_cast<uint2*>(held) = *reinterpret_cast<const uint2*>(hv);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) held[i] = hv[i];
    }
  };
  if (t >= count) {
#pragma unroll
    for (int i = 0; i < N; ++i) hv[i] = 0;
    put_held();
    return;
  }
  lat_load<N, kVec>(static_cast<const uint16_t*>(p.latent) + b * p.ls_b + t * p.ls_t + N * lane, x);
  const uint16_t* rsrc = static_cast<const uint16_t*>(p.rope) + b * p.rs_b + t * p.rs_t;
  const uint16_t r0 = rsrc[lane], r1 = p.dr > 32 ? rsrc[lane + 32] : 0;  // dr is 32 or 64; read
  // beside the latent, not behind the codes' stores: kernel 21 -> 19 us for 8 ragged prompts of up to 4096 tokens
  // unsigned: a length near the type's largest value must not wrap to a column of the table
  const uint64_t pos = (uint64_t)len + t, lp = pos / (uint32_t)p.page;
  int64_t phys = lp < (uint64_t)p.cols ? p.table[(size_t)b * p.cols + lp] : -1;
  if (phys < 0 || phys >= p.num_pages) {  // no page to write to
    if (lane == 0 && p.status != nullptr) atomicOr(p.status, FS_DEV_BAD_PAGE);
    phys = -1;
  }
  float v[N], amax = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lat_f32(x[i], p.bf16);
    amax = fmaxf(amax, fabsf(v[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float scale = fmaxf(__fdiv_rn(amax, 127.0f), 1.0e-8f), rcp = __frcp_rn(scale);
  alignas(16) int8_t code[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float q = __fmul_rn(v[i], rcp);
    float r = rintf(q);
    // NaN and what infinities leave fail the comparison and take the exact steps too
    if (!(fabsf(__fsub_rn(q, r)) < 0.5f - 3.0517578125e-5f)) r = latent_code_exact(v[i], scale);
    r = fminf(fmaxf(r, -127.f), 127.f);
    code[i] = (int8_t)(int)r;
    hv[i] = lat_b16(__fmul_rn(r, scale), p.bf16);
  }
  put_held();
  if (phys < 0) return;
  const size_t row = (size_t)phys * p.page + (size_t)(pos - lp * p.page);
  int8_t* dst = p.values + row * kDC + N * lane;  // a row starts on a 128-byte boundary of the pool
  if (N == 16)
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(code);
  else if (N == 8)
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(code);
  else
    *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(code);
  if (lane == 0) p.scale[row] = scale;
  uint16_t* rdst = static_cast<uint16_t*>(p.ropes) + row * p.dr;
  rdst[lane] = r0;
  if (p.dr > 32) rdst[lane + 32] = r1;
}

// ---------------------------------------------------------------------------------
// absorbed attention
// ---------------------------------------------------------------------------------

constexpr int kTile = 64;  // tokens
constexpr int kSPad = 72;  // floats a row of partial scores
constexpr int kPPad = 72;  // halves a row of P
constexpr int kLatMaxBatch = 4096;
constexpr float kPTop = 2048.f;   // P of the reference maximum
constexpr float kLatSlack = 4.f;  // log2 of what the true maximum may be past the reference: P <= 2^15
constexpr uint64_t kLatTimeoutNs = 2000000000ull;

struct LatentParams {
  const uint16_t* q;       // [B, T, H, dc]
  const uint16_t* q_rope;  // [B, T, H, dr]
  const float* scale;      // [P, page]
  const int64_t* table;
  const int64_t* lengths;
  uint16_t* out;    // [B, T, H, dc]
  float* part_o;    // [ctas][2][rows of a block][dc]
  float* part_lse;  // [ctas][2][rows of a block], log2 domain
  int* prefix;      // [B + 1] units before each request (row blocks not counted)
  uint32_t* status;
  int64_t num_pages, max_seq_len;
  float scale_log2;  // sm_scale * log2(e)
  int B, T, H, R, row_blocks, page, cols, bf16;
};

__device__ __forceinline__ int latent_len(const LatentParams& p, int b) {
  return (int)max((int64_t)0, min(min(p.lengths[b], p.max_seq_len), (int64_t)p.cols * p.page));
}

// Column n of a tile's scores is token lat_token(n): inside each group of eight, even columns
// are tokens 0-3 and odd ones 4-7.  The two rows that a quarter warp reads together then
// differ in bit 2, so the 128-byte swizzle puts their four chunks on different banks.
__device__ __forceinline__ int lat_token(int n) { return (n & ~7) | ((n >> 1) & 3) | ((n & 1) << 2); }

template <int kDC, int kDR, int kMT>
struct LatentShape {
  // One 16-row block: two CTAs of 8 warps an SM, whose phases overlap; more rows: one CTA of
  // 16 warps (the scores' partial sums and O would not fit twice).
  static constexpr int kCtas = kMT == 1 ? 2 : 1;
  static constexpr int kStages = kMT == 1 ? 2 : 3;
  static constexpr int kWarps = kMT == 2 && kDC >= 256 ? 16 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRows = 16 * kMT;
  // warps = kMT row groups x kKS slices of the dims (64 at least) x kTS token groups
  static constexpr int kMaxKS = kWarps / kMT < 4 ? kWarps / kMT : 4;
  static constexpr int kKS = kMaxKS < kDC / 64 ? kMaxKS : kDC / 64;
  static constexpr int kTS = kWarps / (kMT * kKS);
  static constexpr int kSlice = kDC / kKS;     // dims of a warp's QK slice
  static constexpr int kQSteps = kSlice / 32;  // int8 MMA steps
  static constexpr int kNT = kTile / 8 / kTS;  // n-tiles of 8 tokens a warp
  static constexpr int kRSteps = kDR / 16;     // rotary MMA steps, dealt to the slices
  static constexpr int kRPer = (kRSteps + kKS - 1) / kKS;
  static constexpr int kDW = kDC / kWarps;     // dims of a warp's O
  static constexpr int kOT = kDW / 8;          // n-tiles of O
  static constexpr int kTPR = kThreads / kRows;  // softmax threads a row
  static constexpr int kGV = kTile / kTPR < 4 ? kTile / kTPR : 4;  // columns a softmax thread reads together
  static constexpr int kSeg = kTile / kTPR / kGV;
  static constexpr int kValBytes = kTile * kDC, kRopeBytes = kTile * kDR * 2;
  static constexpr int kStage = (kValBytes + kRopeBytes + kTile * 4 + 1023) / 1024 * 1024;
  static constexpr int kSBytes = kKS * kRows * kSPad * 4;
  static constexpr int kPBytes = kRows * kPPad * 2;
  static constexpr int kOffS = kStages * kStage;
  static constexpr int kOffP = kOffS + kSBytes;
  static constexpr int kOffMisc = kOffP + kPBytes;  // alpha, lse, amax [rows], scale and lam [tile], prefix
  static constexpr int kMiscFloats = 3 * kRows + 2 * kTile;
  static_assert(kTS >= 1 && kMT * kKS * kTS == kWarps, "every warp has a part of the scores");
  static constexpr __host__ __device__ int smem(int batch) {
    return 1024 /* alignment */ + kOffMisc + kMiscFloats * 4 + (batch + 1) * 4;
  }
};

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

// The work is divided in a cost space where every (request, row block) is charged kLatPiece
// virtual tiles ahead of its real ones, for what a piece costs whatever its length (reading the
// queries, closing it): without it the shares with many short requests ended last (64 ragged
// requests x 16 heads: 70 us with 0, 61.5 with 1 or 2, 62 with 3; 16 requests x 128 rows: 135,
// 131, 129.5, 129).  n units on C = min(CTAs, n) shares of n / C units, the first n % C of
// them one longer.
constexpr int kLatPiece = 2;

struct LatentShares {
  int per, rem;
  __device__ __forceinline__ LatentShares(int n, int ctas) {
    const int C = min(ctas, n);
    per = C > 0 ? n / C : 1;
    rem = n - per * C;
  }
  __device__ __forceinline__ int start(int k) const { return k * per + min(k, rem); }
  __device__ __forceinline__ int owner(int x) const {  // the share that holds unit x
    const int head = rem * (per + 1);
    return x < head ? x / (per + 1) : rem + (x - head) / per;
  }
};

// Units of a request, for each of its row blocks.
__device__ __forceinline__ int latent_units(int tiles) { return tiles > 0 ? tiles + kLatPiece : 0; }

// Units before each request (row blocks not counted), into pre[0 .. B] (shared memory); every
// thread calls it.
template <int kThreads>
__device__ __forceinline__ void latent_prefix(const LatentParams& p, int* pre) {
  const int tid = threadIdx.x, lane = tid & 31;
  for (int r = tid; r < p.B; r += kThreads) pre[r + 1] = latent_units((latent_len(p, r) + kTile - 1) / kTile);
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

template <int kDC, int kDR, int kMT, bool kBf16>
__global__ void __launch_bounds__(LatentShape<kDC, kDR, kMT>::kThreads, LatentShape<kDC, kDR, kMT>::kCtas)
    latent_attention_kernel(const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_r,
                            const LatentParams p) {
  using L = LatentShape<kDC, kDR, kMT>;
  extern __shared__ uint8_t lat_raw[];
  __shared__ alignas(8) uint64_t s_full[L::kStages];
  __shared__ uint32_t s_pages[L::kStages];  // which of a tile's pages are there, one bit each
  const uint32_t raw_s = smem_u32(lat_raw);
  const uint32_t smem_s = (raw_s + 1023u) & ~1023u;
  uint8_t* lat_smem = lat_raw + (smem_s - raw_s);
  float* s_part = reinterpret_cast<float*>(lat_smem + L::kOffS);  // [kKS][rows][kSPad]
  __half* s_p = reinterpret_cast<__half*>(lat_smem + L::kOffP);   // [rows][kPPad]
  float* s_alpha = reinterpret_cast<float*>(lat_smem + L::kOffMisc);
  float* s_lse = s_alpha + L::kRows;
  uint32_t* s_amax = reinterpret_cast<uint32_t*>(s_lse + L::kRows);
  float* s_scale = s_lse + 2 * L::kRows;  // by column, -1 where there is no token
  float* s_lam = s_scale + kTile;        // by column, log2 of it
  int* pre = reinterpret_cast<int*>(s_lam + kTile);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int mt = warp % kMT, ks = (warp / kMT) % L::kKS, ts = warp / (kMT * L::kKS);

  if (tid == 0) {
    for (int i = 0; i < L::kStages; ++i) mbar_init(smem_u32(&s_full[i]), 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  latent_prefix<L::kThreads>(p, pre);
  if (blockIdx.x == 0)
    for (int r = tid; r <= p.B; r += L::kThreads) p.prefix[r] = pre[r];
  const int total = pre[p.B] * p.row_blocks;
  if ((int)blockIdx.x >= min((int)gridDim.x, total)) return;
  const LatentShares shares(total, gridDim.x);
  const int f_begin = shares.start(blockIdx.x), f_end = shares.start(blockIdx.x + 1);
  bool first = true;
  uint32_t issued = 0, used = 0;  // tiles put into the ring and taken out of it, over all pieces

  const int srow = tid / L::kTPR, sj = tid % L::kTPR;  // softmax thread: row and its columns
  const int box_rows = min(p.page, kTile), per_tile = kTile / box_rows;  // pages (or halves of one) a tile

  for (int f = f_begin; f < f_end;) {
    // ---- the piece: tiles [t0, t1) of row block rb of request b
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] * p.row_blocks <= f) lo = mid; else hi = mid;
    }
    const int b = lo, units = pre[b + 1] - pre[b], nt = units - kLatPiece;
    const int off = f - pre[b] * p.row_blocks, rb = off / units, o0 = off - rb * units;
    const int o1 = min(units, o0 + (f_end - f));
    f += o1 - o0;
    const int t0 = max(0, o0 - kLatPiece), t1 = o1 - kLatPiece;
    if (t1 <= t0) continue;  // the share ends within the piece's charge
    const int len = latent_len(p, b);
    const int row0 = rb * L::kRows, rows = min(L::kRows, p.R - row0);
    const uint16_t* qb = p.q + ((size_t)b * p.R + row0) * kDC;
    const uint16_t* qrb = p.q_rope + ((size_t)b * p.R + row0) * kDR;
    const int64_t* trow = p.table + (size_t)b * p.cols;

    // ---- producer (warp 0): page lookups run a tile ahead of the copies
    auto lookup = [&](int t) -> int64_t {  // lane i: the pool page of part i of tile t, -1: none
      const int tok = t * kTile + lane * box_rows;
      if (t >= t1 || lane >= per_tile || tok >= len) return -1;
      const int64_t phys = trow[tok / p.page];
      if (phys >= p.num_pages) {
        if (p.status != nullptr) atomicOr(p.status, FS_DEV_BAD_PAGE);
        return -1;
      }
      return phys;
    };
    auto issue = [&](int t, int64_t phys) {  // tile t into the ring
      const int st = (int)(issued % L::kStages);
      const uint32_t base = smem_s + st * L::kStage, bar = smem_u32(&s_full[st]);
      const uint32_t there = __ballot_sync(0xffffffffu, phys >= 0);
      if (lane == 0) {
        s_pages[st] = there;
        mbar_arrive_expect_tx(bar, (uint32_t)__popc(there) * box_rows * (kDC + 2 * kDR + 4));
      }
      __syncwarp();
      if (phys >= 0) {
        const int r = lane * box_rows, in_page = (t * kTile + r) % p.page;
        const int64_t row = phys * p.page + in_page;
        const uint64_t policy = l2_policy_evict_first();
#pragma unroll
        for (int j = 0; j < kDC / 128; ++j)
          tma_load_2d(base + j * (kTile * 128) + r * 128, &map_v, 128 * j, (int32_t)row, bar, policy);
        tma_load_2d(base + L::kValBytes + r * 2 * kDR, &map_r, 0, (int32_t)row, bar, policy);
        bulk_load(base + L::kValBytes + L::kRopeBytes + 4 * r, p.scale + row, (uint32_t)(4 * box_rows), bar);
      }
      ++issued;
    };
    int64_t next_phys = -1;
    if (tid < L::kRows) s_amax[tid] = 0u;
    __syncthreads();  // the previous piece is done with the stages and the row state
    if (warp == 0) {
      int64_t phys[L::kStages];
#pragma unroll
      for (int i = 0; i < L::kStages; ++i) phys[i] = lookup(t0 + i);
#pragma unroll
      for (int i = 0; i < L::kStages - 1; ++i)
        if (t0 + i < t1) issue(t0 + i, phys[i]);
      next_phys = phys[L::kStages - 1];
    }

    // ---- q as 16-bit fixed point: this warp's words, the rows' largest magnitudes (16-bit
    // patterns, monotone, NaN above infinity above the rest) over all warps, then the bytes
    uint32_t qhi[L::kQSteps][4], qlo[L::kQSteps][4];  // a0..a3 of the m16n8k32 MMAs
    float fq[2];                                       // row scale * sm_scale * log2 e, rows g and g + 8
    {
      uint2 raw[2][L::kQSteps][2];
#pragma unroll
      for (int r2 = 0; r2 < 2; ++r2) {
        const int r = 16 * mt + g + 8 * r2;
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < L::kQSteps; ++j)
#pragma unroll
          for (int w = 0; w < 2; ++w) {  // the words b0 / b1 of step j: dims 64 (j / 2) + 16 c + 8 (j & 1) + 4 w
            const int d = ks * L::kSlice + 64 * (j >> 1) + 16 * c + 8 * (j & 1) + 4 * w;
            raw[r2][j][w] = make_uint2(0u, 0u);
            if (r < rows) raw[r2][j][w] = *reinterpret_cast<const uint2*>(qb + (size_t)r * kDC + d);
          }
#pragma unroll
        for (int j = 0; j < L::kQSteps; ++j)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t ww[2] = {raw[r2][j][w].x, raw[r2][j][w].y};
#pragma unroll
            for (int e = 0; e < 2; ++e) top = max(top, max(ww[e] & 0x7fffu, (ww[e] >> 16) & 0x7fffu));
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (c == 0) atomicMax(s_amax + r, top);
      }
      __syncthreads();
#pragma unroll
      for (int r2 = 0; r2 < 2; ++r2) {
        const uint32_t top = s_amax[16 * mt + g + 8 * r2];
        // a row with infinities or NaN has no scale: its output is NaN
        const float qs = top >= (kBf16 ? 0x7f80u : 0x7c00u) ? __int_as_float(0x7fc00000)
                                                            : lat_f32((uint16_t)top, kBf16) / 32639.0f;
        const float inv = qs > 0.f ? 1.f / qs : 0.f;
        fq[r2] = qs * p.scale_log2;
#pragma unroll
        for (int j = 0; j < L::kQSteps; ++j)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t ww[2] = {raw[r2][j][w].x, raw[r2][j][w].y};
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
    // tokens that this softmax thread's row sees: query t sees the first lengths - T + t + 1, as
    // far as they are in the table
    const int limit = (int)max((int64_t)0, min((int64_t)len, p.lengths[b] - p.T + 1 + (row0 + srow) / p.H));

    for (int t = t0; t < t1; ++t, ++used) {
      const int st = (int)(used % L::kStages);
      const uint32_t base = smem_s + st * L::kStage;
      const float* tok_scale =
          reinterpret_cast<const float*>(lat_smem + st * L::kStage + L::kValBytes + L::kRopeBytes);
      const bool here = mbar_wait_bounded(smem_u32(&s_full[st]), (used / L::kStages) & 1u, kLatTimeoutNs);

      // ---- 1. partial scores of this warp's rows, dims and tokens
      const int prow = lat_token(g);  // row of column g of a group
#pragma unroll 4
      for (int n = 0; n < L::kNT; ++n) {
        const int col = (ts * L::kNT + n) * 8, brow = col + prow;
        int sh[4] = {0, 0, 0, 0}, sl[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j2 = 0; j2 < L::kQSteps / 2; ++j2) {
          const int d16 = (ks * L::kSlice + 64 * j2) / 16 + c;  // 16-byte chunk of the row
          const uint4 kv = lds128(base + (d16 >> 3) * (kTile * 128) + brow * 128 + (((d16 & 7) ^ prow) << 4));
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
            const int ch = 2 * s + (c >> 1);
            const int swz = kDR == 64 ? prow : (prow >> 1) & 3;  // the 128- or 64-byte swizzle
            const float2 w = lds64f(base + L::kValBytes + brow * kDR * 2 + ((ch ^ swz) << 4) + 8 * (c & 1));
            const uint32_t b0 = __float_as_uint(w.x), b1 = __float_as_uint(w.y);
            if (kBf16)
              mma_16816_bf16(rp, qr[i][0], qr[i][1], qr[i][2], qr[i][3], b0, b1);
            else
              mma_16816(rp, qr[i][0], qr[i][1], qr[i][2], qr[i][3], b0, b1);
          }
        }
        const float sc0 = tok_scale[col + c], sc1 = tok_scale[col + c + 4];  // columns 2c and 2c + 1
        float* dst = s_part + ((size_t)ks * L::kRows + 16 * mt + g) * kSPad + col + 2 * c;
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {  // at most 256 dims: 256 hi + lo stays within 31 bits
          const float x0 = (float)((sh[2 * r2] << 8) + sl[2 * r2]) * (fq[r2] * sc0);
          const float x1 = (float)((sh[2 * r2 + 1] << 8) + sl[2 * r2 + 1]) * (fq[r2] * sc1);
          *reinterpret_cast<float2*>(dst + 8 * r2 * kSPad) =
              make_float2(fmaf(rp[2 * r2], p.scale_log2, x0), fmaf(rp[2 * r2 + 1], p.scale_log2, x1));
        }
      }
      if (tid < kTile) {
        const int tok = lat_token(tid);
        const bool there = t * kTile + tok < len && ((s_pages[st] >> (tok / box_rows)) & 1u);
        const float sc = there ? tok_scale[tok] : -1.f;
        s_scale[tid] = sc;
        s_lam[tid] = fmaxf(lg2_approx(fmaxf(sc, 0.f)), -100.f);
      }
      if (__syncthreads_or(here ? 0 : 1)) {  // a copy that never came: give up, outputs are invalid
        if (tid == 0) {
          if (p.status != nullptr) atomicOr(p.status, FS_DEV_TIMEOUT);
          // shared memory is given back only behind the copies still on their way to it
          for (uint32_t i = used; i != issued; ++i)
            mbar_wait_bounded(smem_u32(&s_full[i % L::kStages]), (i / L::kStages) & 1u, kLatTimeoutNs);
        }
        __syncthreads();
        return;
      }
      // every warp is done with tile t - 1: its stage takes tile t + L::kStages - 1
      if (warp == 0 && t + L::kStages - 1 < t1) {
        issue(t + L::kStages - 1, next_phys);
        next_phys = lookup(t + L::kStages);
      }

      // ---- 2. softmax of row srow
      float z[L::kSeg][L::kGV], sc[L::kSeg][L::kGV];
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < L::kSeg; ++i) {
        const int n0 = L::kGV * (sj + L::kTPR * i);
        float v[L::kGV], lm[L::kGV];
        auto load = [&](const float* src, float (&dst)[L::kGV]) {
          if (L::kGV == 4) {
            const float4 x = *reinterpret_cast<const float4*>(src);
            dst[0] = x.x, dst[1] = x.y, dst[L::kGV - 2] = x.z, dst[L::kGV - 1] = x.w;
          } else {
            const float2 x = *reinterpret_cast<const float2*>(src);
            dst[0] = x.x, dst[1] = x.y;
          }
        };
        load(s_part + (size_t)srow * kSPad + n0, v);
#pragma unroll
        for (int k2 = 1; k2 < L::kKS; ++k2) {
          float x[L::kGV];
          load(s_part + ((size_t)k2 * L::kRows + srow) * kSPad + n0, x);
#pragma unroll
          for (int k = 0; k < L::kGV; ++k) v[k] += x[k];
        }
        load(s_scale + n0, sc[i]);
        load(s_lam + n0, lm);
#pragma unroll
        for (int k = 0; k < L::kGV; ++k) {
          const bool seen = t * kTile + lat_token(n0 + k) < limit && !(sc[i][k] < 0.f);
          z[i][k] = seen ? v[k] : -INFINITY;
          sc[i][k] = seen ? sc[i][k] : 0.f;  // P of an unseen token is 0 whatever its scale
          mx = fmaxf(mx, z[i][k] + lm[k]);
        }
      }
#pragma unroll
      for (int o = L::kTPR / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // a row's first maximum is its reference; later ones only when far past it, so that O is
      // rescaled seldom
      const bool move = mx > m_run + (m_run == -1.0e30f ? 0.f : kLatSlack);
      const float m_new = move ? mx : m_run, alpha = ex2_approx(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < L::kSeg; ++i) {
        float pr[L::kGV];
#pragma unroll
        for (int k = 0; k < L::kGV; ++k) {
          const float e = ex2_approx(z[i][k] - m_new);
          l_run += e;
          pr[k] = e * (sc[i][k] * kPTop);
        }
        __half* dst = s_p + srow * kPPad + L::kGV * (sj + L::kTPR * i);
#pragma unroll
        for (int k = 0; k < L::kGV; k += 2) *reinterpret_cast<uint32_t*>(dst + k) = pack_half2(pr[k], pr[k + 1]);
      }
      if (sj == 0) s_alpha[srow] = alpha;
      const bool rescale = __syncthreads_or(move && t > t0 ? 1 : 0) != 0;

      // ---- 3. O += P C for this warp's dims
      if (rescale) {
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
          const float a0 = s_alpha[16 * i + g], a1 = s_alpha[16 * i + g + 8];
#pragma unroll
          for (int j = 0; j < L::kOT; ++j) {
            acc[i][j][0] *= a0;
            acc[i][j][1] *= a0;
            acc[i][j][2] *= a1;
            acc[i][j][3] *= a1;
          }
        }
      }
      const uint32_t p_s = smem_s + L::kOffP;
#pragma unroll
      for (int kk = 0; kk < kTile / 16; ++kk) {
        // matrices of a transposed load: (columns 0-7 | 8-15 of the step) x (chunk ch | ch + 1)
        constexpr int kChunks = L::kDW / 16;
        static_assert(kChunks == 1 || kChunks % 2 == 0, "a warp owns whole pairs of 16-dim chunks, or one chunk");
        constexpr int kPair = kChunks > 1 ? 2 : 1;
        const int in8 = lat_token(lane & 7), r = 16 * kk + 8 * ((lane >> 3) & 1) + in8;
#pragma unroll
        for (int ch0 = 0; ch0 < kChunks; ch0 += 2) {
          uint32_t v[4], bf[kPair][4];
          // with one chunk a warp the second pair of matrices repeats the first
          const int ch = warp * kChunks + ch0 + (kChunks > 1 ? (lane >> 4) : 0);
          ldsm_x4_trans(base + (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ in8) << 4), v[0], v[1], v[2], v[3]);
#pragma unroll
          for (int u = 0; u < kPair; ++u) {
            // bytes [column 2c: dims 2g, 2g + 1][column 2c + 1: the same]; even dims form one
            // n-tile, odd dims the next
            const uint32_t x0 = v[2 * u] ^ 0x80808080u, x1 = v[2 * u + 1] ^ 0x80808080u;
            const __half2 base2 = __half2half2(__ushort_as_half((unsigned short)0x6480));  // 1152
            auto cvt = [&](uint32_t x, uint32_t sel) -> uint32_t {
              const uint32_t h = prmt(x, 0x64646464u, sel);
              const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&h), base2);
              return *reinterpret_cast<const uint32_t*>(&d);
            };
            bf[u][0] = cvt(x0, 0x4240u), bf[u][1] = cvt(x1, 0x4240u);
            bf[u][2] = cvt(x0, 0x4341u), bf[u][3] = cvt(x1, 0x4341u);
          }
#pragma unroll
          for (int i = 0; i < kMT; ++i) {
            uint32_t pa[4];
            ldsm_x4(p_s + ((16 * i + (lane & 15)) * kPPad + 16 * kk + 8 * (lane >> 4)) * 2, pa[0], pa[1], pa[2], pa[3]);
#pragma unroll
            for (int u = 0; u < kPair; ++u) {
              mma_16816(acc[i][2 * (ch0 + u)], pa[0], pa[1], pa[2], pa[3], bf[u][0], bf[u][1]);
              mma_16816(acc[i][2 * (ch0 + u) + 1], pa[0], pa[1], pa[2], pa[3], bf[u][2], bf[u][3]);
            }
          }
        }
      }
    }

    // ---- close the piece: normalise
    float l = l_run;
#pragma unroll
    for (int o = L::kTPR / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncthreads();  // every warp has read the last alphas
    if (sj == 0) {
      s_alpha[srow] = l > 0.f ? 1.f / (l * kPTop) : (l == 0.f ? 0.f : l);  // NaN stays
      s_lse[srow] = l > 0.f ? m_run + log2f(l) : (l == 0.f ? -INFINITY : l);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    const size_t slot = ((size_t)blockIdx.x * 2 + (first ? 0 : 1)) * L::kRows;
    first = false;
    if (!whole && tid < rows) p.part_lse[slot + tid] = s_lse[tid];
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
// for requests without tokens.  One CTA a row, four dims a thread; the weights of up to
// kMergeChunk shares at a time are formed together, then their rows are added up.
constexpr int kMergeChunk = 128;

__global__ void __launch_bounds__(128) latent_merge_kernel(const LatentParams p, int block_rows, int dc, int ctas) {
  __shared__ float s_w[kMergeChunk];
  __shared__ float s_max[4];
  cudaGridDependencySynchronize();  // behind it the shares' results are there
  const int row = blockIdx.x % p.R, b = blockIdx.x / p.R, rb = row / block_rows, r = row - rb * block_rows;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int before = p.prefix[b], units = p.prefix[b + 1] - before, total = p.prefix[p.B] * p.row_blocks;
  uint16_t* out = p.out + ((size_t)b * p.R + row) * dc + 4 * tid;
  if (units == 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(0u, 0u);
    return;
  }
  const LatentShares shares(total, ctas);
  const int u0 = before * p.row_blocks + rb * units;  // the row block's first unit
  const int k0 = shares.owner(u0 + kLatPiece), k1 = shares.owner(u0 + units - 1);
  if (k0 == k1) return;  // one share wrote the output itself
  // a share's first piece is in slot 0; the first share's piece is a later one where the
  // share starts before this row block
  const size_t late = shares.start(k0) < u0 ? 1 : 0;
  auto slot = [&](int k) -> size_t { return ((size_t)k * 2 + (k == k0 ? late : 0)) * block_rows + r; };
  float M = -INFINITY;
  bool nan = false;
  for (int k = k0 + tid; k <= k1; k += threads) {
    const float x = p.part_lse[slot(k)];
    nan |= isnan(x);
    M = fmaxf(M, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) s_max[tid >> 5] = M;
  nan = __syncthreads_or(nan ? 1 : 0) != 0;
  for (int i = 0; i < threads / 32; ++i) M = fmaxf(M, s_max[i]);
  if (nan) M = __int_as_float(0x7fc00000);
  float W = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (M != -INFINITY) {
    for (int c0 = k0; c0 <= k1; c0 += kMergeChunk) {
      const int n = min(kMergeChunk, k1 + 1 - c0);
      __syncthreads();
      for (int i = tid; i < n; i += threads) s_w[i] = exp2f(p.part_lse[slot(c0 + i)] - M);
      __syncthreads();
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float w = s_w[i];
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot(c0 + i) * dc + 4 * tid);
        W += w;
        acc.x = fmaf(w, v.x, acc.x);
        acc.y = fmaf(w, v.y, acc.y);
        acc.z = fmaf(w, v.z, acc.z);
        acc.w = fmaf(w, v.w, acc.w);
      }
    }
  }
  const float inv = W > 0.f ? 1.f / W : (W == 0.f ? 0.f : W);
  uint2 w;
  w.x = (uint32_t)lat_b16(acc.x * inv, p.bf16) | ((uint32_t)lat_b16(acc.y * inv, p.bf16) << 16);
  w.y = (uint32_t)lat_b16(acc.z * inv, p.bf16) | ((uint32_t)lat_b16(acc.w * inv, p.bf16) << 16);
  *reinterpret_cast<uint2*>(out) = w;
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
  if ((int64_t)a->tokens * a->heads > (1 << 20) || (int64_t)a->tokens * a->heads * a->batch >= (1ll << 31))
    return FS_ERR_UNSUPPORTED;
  if (a->num_pages * a->page_size >= (1ll << 31) || a->num_pages >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  if ((int64_t)a->table_cols * a->page_size >= (1ll << 30)) return FS_ERR_UNSUPPORTED;  // positions in 32 bits
  // units of work (64 tokens of 16 to 64 rows) are counted in 32 bits
  const int64_t longest = std::min<int64_t>(a->max_seq_len, (int64_t)a->table_cols * a->page_size);
  const int64_t rows = (int64_t)a->tokens * a->heads;
  if ((longest / kTile + 1 + kLatPiece) * a->batch * ((rows + 15) / 16) >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_rope) |
       reinterpret_cast<uintptr_t>(a->values) | reinterpret_cast<uintptr_t>(a->ropes) |
       reinterpret_cast<uintptr_t>(a->scale) | reinterpret_cast<uintptr_t>(a->out)) & 15)
    return FS_ERR_ALIGNMENT;
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
  pl.ctas = device_sm_count(device) * (pl.mt == 1 ? 2 : 1);  // LatentShape::kCtas on every SM
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  pl.o = up((size_t)pl.ctas * 2 * rows * a->latent_dim * 4);
  pl.lse = up((size_t)pl.ctas * 2 * rows * 4);
  pl.prefix = up((size_t)(a->batch + 1) * 4);
  return pl;
}

template <int kDC, int kDR, int kMT>
static int launch_latent(const FsLatentArgs* a, const LatentParams& p, const LatentPlan& pl, void* stream) {
  using L = LatentShape<kDC, kDR, kMT>;
  static_assert(L::smem(kLatMaxBatch) <= 227 * 1024 && L::kCtas * (L::smem(1024) + 1024) <= 228 * 1024, "shared memory of a CTA");
  CUtensorMap map_v, map_r;
  const uint64_t rows = (uint64_t)a->num_pages * a->page_size;
  const uint32_t box_rows = (uint32_t)std::min(a->page_size, kTile);
  if (int st = make_byte_map(&map_v, a->values, rows, kDC, box_rows, 128); st != FS_OK) return st;
  if (int st = make_byte_map(&map_r, a->ropes, rows, 2 * kDR, box_rows, 2 * kDR); st != FS_OK) return st;
  auto kernel = p.bf16 ? latent_attention_kernel<kDC, kDR, kMT, true> : latent_attention_kernel<kDC, kDR, kMT, false>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(kLatMaxBatch));
      e != cudaSuccess)
    return fail_cuda("shared-memory limit of the latent attention kernel", e);
  kernel<<<pl.ctas, L::kThreads, L::smem(p.B), reinterpret_cast<cudaStream_t>(stream)>>>(map_v, map_r, p);
  if (int st = launch_status("latent attention kernel launch"); st != FS_OK) return st;
  // the merge may be set up before the shares have ended; nothing triggers it earlier, so this
  // hides its launch latency and no more
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.B * p.R));
  cfg.blockDim = dim3(kDC / 4);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, latent_merge_kernel, p, L::kRows, kDC, pl.ctas); e != cudaSuccess)
    return fail_cuda("latent merge kernel launch", e);
  return FS_OK;
}

template <int kDC, int kDR>
static int launch_latent_rows(const FsLatentArgs* a, const LatentParams& p, const LatentPlan& pl, void* stream) {
  switch (pl.mt) {
    case 1: return launch_latent<kDC, kDR, 1>(a, p, pl, stream);
    case 2: return launch_latent<kDC, kDR, 2>(a, p, pl, stream);
    default: return launch_latent<kDC, kDR, 4>(a, p, pl, stream);
  }
}

template <int kDC>
static int launch_latent_rope(const FsLatentArgs* a, const LatentParams& p, const LatentPlan& pl, void* stream) {
  return a->rope_dim == 64 ? launch_latent_rows<kDC, 64>(a, p, pl, stream)
                           : launch_latent_rows<kDC, 32>(a, p, pl, stream);
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
  if ((reinterpret_cast<uintptr_t>(a->values) & 15) || (reinterpret_cast<uintptr_t>(a->scale) & 3)) return FS_ERR_ALIGNMENT;
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
  // vector words need 16-byte aligned rows (a view of a packed projection may have none)
  const bool vec = a->latent_stride_b % 8 == 0 && a->latent_stride_t % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a->latent) | reinterpret_cast<uintptr_t>(a->held)) & 15) == 0;
  auto go = [&](auto kernel) {
    kernel<<<(unsigned)blocks, kAppendWarps * 32, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return launch_status("latent append kernel launch");
  };
  switch (a->latent_dim) {
    case 128: return vec ? go(latent_append_kernel<128, true>) : go(latent_append_kernel<128, false>);
    case 256: return vec ? go(latent_append_kernel<256, true>) : go(latent_append_kernel<256, false>);
    default: return vec ? go(latent_append_kernel<512, true>) : go(latent_append_kernel<512, false>);
  }
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
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  LatentParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_rope = static_cast<const uint16_t*>(a->q_rope);
  p.scale = a->scale;
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
    case 128: return launch_latent_rope<128>(a, p, pl, stream);
    case 256: return launch_latent_rope<256>(a, p, pl, stream);
    default: return launch_latent_rope<512>(a, p, pl, stream);
  }
}

}  // extern "C"
