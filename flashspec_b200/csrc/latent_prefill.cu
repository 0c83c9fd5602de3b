// Expanded latent attention for prompts: per-head keys and values that the caller expanded
// from the latents, one rotary key shared by all heads, ragged packed requests, causal and
// aligned at the end (the last query of a request sees its last key).
//
//   score(i, h, j) = sm_scale * (q[i, h, :dn] . kv[j, h, :dn] + q[i, h, dn:] . k_rope[j])
//   out[i, h]      = sum_j softmax_j(score) kv[j, h, dn:]
//
// A CTA takes 128 queries of one head, 16 a warp, and walks the keys in tiles of 64, two
// tiles in flight with cp.async.  The shared rotary key is read beside each head's own part,
// so it is never copied per head.  Running maximum and sum in fp32, P rounds to 16 bits
// before P V.  Bound by the tensor cores for long prompts.
//
// A value that is not finite must not reach queries that do not see its key (0 * inf is NaN).
// Only tiles on the causal edge are seen by some of a CTA's queries and not by others: there
// such values are set to zero and the first key that has one is noted per dim; the queries
// that see that key get NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "../../include/flashspec_b200.h"
#include "common.h"
#include "ptx.cuh"

namespace fsb {

constexpr int kPreThreads = 256;
constexpr int kPreQ = 128;  // queries of a CTA
constexpr int kPreK = 64;   // keys of a tile

struct PrefillParams {
  const uint16_t* q;       // [Nq, H, dn + dr]
  const uint16_t* kv;      // [Nk, H, dn + dv]
  const uint16_t* k_rope;  // [Nk, dr]
  const int64_t* q_off;    // [B + 1]
  const int64_t* k_off;
  uint16_t* out;  // [Nq, H, dv]
  int64_t nq, nk;
  float scale_log2;
  int B, H;
};

template <int kDN, int kDR, int kDV>
struct PrefillShape {
  static constexpr int kDQ = kDN + kDR;
  static constexpr int kQRow = kDQ * 2 + 16;  // padded rows: an odd number of 16-byte chunks
  static constexpr int kVRow = kDV * 2 + 16;
  static constexpr int kQBytes = kPreQ * kQRow, kKBytes = kPreK * kQRow, kVBytes = kPreK * kVRow;
  static constexpr int kStage = kKBytes + kVBytes;
  static constexpr int kSmem = kQBytes + 2 * kStage;
};

__device__ __forceinline__ void pre_cp16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // absent rows become zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void pre_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <bool kBf16>
__device__ __forceinline__ void pre_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pre_pack(float lo, float hi) {
  if (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}

// Offsets are the caller's device data: whatever they hold, a request's rows stay in [0, n].
__device__ __forceinline__ void pre_range(const int64_t* off, int b, int64_t n, int64_t& lo, int& count) {
  lo = min(max(off[b], (int64_t)0), n);
  count = (int)max((int64_t)0, min(off[b + 1], n) - lo);
}

template <int kDN, int kDR, int kDV, bool kBf16>
__global__ void __launch_bounds__(kPreThreads, 1) latent_prefill_kernel(const PrefillParams p) {
  using L = PrefillShape<kDN, kDR, kDV>;
  extern __shared__ __align__(128) uint8_t pre_smem[];
  __shared__ int s_find[2];
  __shared__ int s_bad[kDV];  // per dim: first key of an edge tile whose value is not finite
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.x % p.H;
  // the tile: counted from the last request's last one back, so that long tiles start first
  const int want = (int)(gridDim.x / p.H) - 1 - (int)(blockIdx.x / p.H);
  if (tid < 32) {
    int carry = 0, fb = -1, ft = 0;
    for (int base = 0; base < p.B && fb < 0; base += 32) {
      int64_t lo;
      int n = 0;
      if (base + lane < p.B) pre_range(p.q_off, base + lane, p.nq, lo, n);
      int x = (n + kPreQ - 1) / kPreQ;
      const int mine = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int before = carry + x - mine;
      const unsigned hit = __ballot_sync(0xffffffffu, want >= before && want < before + mine);
      if (hit) {
        const int l = __ffs(hit) - 1;
        fb = base + l;
        ft = want - __shfl_sync(0xffffffffu, before, l);
      }
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) s_find[0] = fb, s_find[1] = ft;
  }
  if (tid < kDV) s_bad[tid] = INT_MAX;
  __syncthreads();
  const int b = s_find[0];
  if (b < 0) return;  // more CTAs than tiles: the host knows only an upper bound
  int64_t q0, k0;
  int nq, nk;
  pre_range(p.q_off, b, p.nq, q0, nq);
  pre_range(p.k_off, b, p.nk, k0, nk);
  const int i0 = s_find[1] * kPreQ;           // first query of the tile, within the request
  const int rows = min(kPreQ, nq - i0);
  const int shift = nk - nq;                  // query i sees keys j <= i + shift
  const int last = min(nk, i0 + rows + shift);  // keys that any of the tile's queries sees
  const int tiles = last > 0 ? (last + kPreK - 1) / kPreK : 0;

  const uint32_t smem = smem_u32(pre_smem);
  constexpr int kQC = L::kDQ / 8, kNC = kDN / 8, kVC = kDV / 8, kRC = kDR / 8;
  for (int i = tid; i < kPreQ * kQC; i += kPreThreads) {
    const int r = i / kQC, ch = i % kQC;
    const int rr = min(r, rows - 1);
    pre_cp16(smem + r * L::kQRow + 16 * ch, p.q + ((size_t)(q0 + i0 + rr) * p.H + h) * L::kDQ + 8 * ch, r < rows);
  }
  auto load = [&](int t) {
    const uint32_t base = smem + L::kQBytes + (t & 1) * L::kStage;
    for (int i = tid; i < kPreK * (kNC + kVC); i += kPreThreads) {
      const int r = i / (kNC + kVC), ch = i % (kNC + kVC), j = t * kPreK + r;
      const uint16_t* src = p.kv + ((size_t)(k0 + min(j, nk - 1)) * p.H + h) * (kDN + kDV) + 8 * ch;
      pre_cp16(ch < kNC ? base + r * L::kQRow + 16 * ch : base + L::kKBytes + r * L::kVRow + 16 * (ch - kNC), src, j < nk);
    }
    for (int i = tid; i < kPreK * kRC; i += kPreThreads) {
      const int r = i / kRC, ch = i % kRC, j = t * kPreK + r;
      pre_cp16(base + r * L::kQRow + kDN * 2 + 16 * ch, p.k_rope + (size_t)(k0 + min(j, nk - 1)) * kDR + 8 * ch, j < nk);
    }
  };
  if (tiles > 0) load(0);
  asm volatile("cp.async.commit_group;" ::: "memory");

  float o[kDV / 8][4];
#pragma unroll
  for (int n = 0; n < kDV / 8; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) o[n][k] = 0.f;
  float m[2] = {-1.0e30f, -1.0e30f}, l[2] = {0.f, 0.f};
  const int row = 16 * warp + g;  // and row + 8
  bool any_bad = false;
  for (int t = 0; t < tiles; ++t) {
    if (t + 1 < tiles) load(t + 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const uint32_t kb = smem + L::kQBytes + (t & 1) * L::kStage, vb = kb + L::kKBytes;
    const int j0 = t * kPreK;
    float s[kPreK / 8][4];
#pragma unroll
    for (int n = 0; n < kPreK / 8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[n][k] = 0.f;
#pragma unroll
    for (int kk = 0; kk < L::kDQ / 16; ++kk) {
      uint32_t a[4];
      pre_ldsm(smem + (16 * warp + (lane & 15)) * L::kQRow + 32 * kk + 16 * (lane >> 4), a);
#pragma unroll
      for (int n = 0; n < kPreK / 16; ++n) {  // 16 keys: matrices (keys 0-7 | 8-15) x (dims 0-7 | 8-15)
        uint32_t kf[4];
        pre_ldsm(kb + (16 * n + (lane & 7) + 8 * (lane >> 4)) * L::kQRow + 32 * kk + 16 * ((lane >> 3) & 1), kf);
        pre_mma<kBf16>(s[2 * n], a, kf[0], kf[1]);
        pre_mma<kBf16>(s[2 * n + 1], a, kf[2], kf[3]);
      }
    }
    if (j0 + kPreK > i0 + shift + 1) {  // some of the CTA's queries do not see the whole tile
      constexpr uint16_t kExp = kBf16 ? 0x7f80 : 0x7c00;
      bool found = false;
      for (int i = tid; i < kPreK * kVC; i += kPreThreads) {
        const int r = i / kVC, ch = i % kVC;
        uint4* at = reinterpret_cast<uint4*>(pre_smem + (vb - smem) + r * L::kVRow + 16 * ch);
        uint4 v = *at;
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
        bool here = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint16_t x = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
          if ((x & kExp) == kExp) {
            atomicMin(s_bad + 8 * ch + k, j0 + r);
            w[k >> 1] &= (k & 1) ? 0x0000ffffu : 0xffff0000u;
            here = true;
          }
        }
        if (here) *at = make_uint4(w[0], w[1], w[2], w[3]);
        found |= here;
      }
      any_bad = __syncthreads_or(found ? 1 : 0) || any_bad;
    }
    // scores to the log2 domain; keys behind a row's last one, or behind the request, are masked
    const bool edge = j0 + kPreK > i0 + 16 * warp + shift + 1 || j0 + kPreK > nk;
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < kPreK / 8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x = s[n][k] * p.scale_log2;
        if (edge) {
          const int j = j0 + 8 * n + 2 * c + (k & 1);
          if (j > i0 + row + 8 * (k >> 1) + shift || j >= nk) x = -INFINITY;
        }
        s[n][k] = x;
        mx[k >> 1] = fmaxf(mx[k >> 1], x);
      }
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      mx[r2] = fmaxf(mx[r2], __shfl_xor_sync(0xffffffffu, mx[r2], 1));
      mx[r2] = fmaxf(mx[r2], __shfl_xor_sync(0xffffffffu, mx[r2], 2));
      const float alpha = ex2_approx(m[r2] - mx[r2]);
      m[r2] = mx[r2];
      l[r2] *= alpha;
#pragma unroll
      for (int n = 0; n < kDV / 8; ++n) {
        o[n][2 * r2] *= alpha;
        o[n][2 * r2 + 1] *= alpha;
      }
    }
#pragma unroll
    for (int n = 0; n < kPreK / 8; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[n][k] = ex2_approx(s[n][k] - m[k >> 1]);
        l[k >> 1] += s[n][k];
      }
#pragma unroll
    for (int kk = 0; kk < kPreK / 16; ++kk) {
      const uint32_t a[4] = {pre_pack<kBf16>(s[2 * kk][0], s[2 * kk][1]), pre_pack<kBf16>(s[2 * kk][2], s[2 * kk][3]),
                             pre_pack<kBf16>(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                             pre_pack<kBf16>(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int n = 0; n < kDV / 16; ++n) {  // matrices (keys 0-7 | 8-15) x (dims 0-7 | 8-15), transposed
        uint32_t v[4];
        ldsm_x4_trans(vb + (16 * kk + (lane & 15)) * L::kVRow + 32 * n + 16 * (lane >> 4), v[0], v[1], v[2], v[3]);
        pre_mma<kBf16>(o[2 * n], a, v[0], v[1]);
        pre_mma<kBf16>(o[2 * n + 1], a, v[2], v[3]);
      }
    }
    __syncthreads();  // the stage may be filled again
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int r2 = 0; r2 < 2; ++r2) {
    float x = l[r2];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    const float inv = x == 0.f ? 0.f : 1.f / x;
    const int r = row + 8 * r2;
    if (r >= rows) continue;
    uint16_t* dst = p.out + ((size_t)(q0 + i0 + r) * p.H + h) * kDV;
#pragma unroll
    for (int n = 0; n < kDV / 8; ++n) {
      if (any_bad) {
        if (s_bad[8 * n + 2 * c] <= i0 + r + shift) o[n][2 * r2] = __int_as_float(0x7fc00000);
        if (s_bad[8 * n + 2 * c + 1] <= i0 + r + shift) o[n][2 * r2 + 1] = __int_as_float(0x7fc00000);
      }
      *reinterpret_cast<uint32_t*>(dst + 8 * n + 2 * c) = pre_pack<kBf16>(o[n][2 * r2] * inv, o[n][2 * r2 + 1] * inv);
    }
  }
}

template <int kDN, int kDR, int kDV>
static int launch_prefill(const PrefillParams& p, int64_t tiles, bool bf16, void* stream) {
  using L = PrefillShape<kDN, kDR, kDV>;
  auto kernel = bf16 ? latent_prefill_kernel<kDN, kDR, kDV, true> : latent_prefill_kernel<kDN, kDR, kDV, false>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
      e != cudaSuccess)
    return fail_cuda("shared-memory limit of the latent prefill kernel", e);
  kernel<<<(unsigned)(tiles * p.H), kPreThreads, L::kSmem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return launch_status("latent prefill kernel launch");
}

template <int kDN, int kDR>
static int launch_prefill_v(const PrefillParams& p, int64_t tiles, int dv, bool bf16, void* stream) {
  return dv == 64 ? launch_prefill<kDN, kDR, 64>(p, tiles, bf16, stream)
                  : launch_prefill<kDN, kDR, 128>(p, tiles, bf16, stream);
}

}  // namespace fsb

extern "C" int fs_latent_prefill(const FsLatentPrefillArgs* a, void* stream) {
  using namespace fsb;
  if (a == nullptr || a->q_offsets == nullptr || a->k_offsets == nullptr || a->batch <= 0 || a->heads <= 0 ||
      a->q_rows < 0 || a->k_rows < 0)
    return FS_ERR_INVALID_ARGUMENT;
  if (a->dtype != FS_F16 && a->dtype != FS_BF16) return FS_ERR_UNSUPPORTED;
  if ((a->nope_dim != 64 && a->nope_dim != 128) || (a->rope_dim != 32 && a->rope_dim != 64) ||
      (a->value_dim != 64 && a->value_dim != 128))
    return FS_ERR_UNSUPPORTED;
  if (a->q_rows == 0) return FS_OK;  // no query, nothing to write
  if (a->q == nullptr || a->out == nullptr || (a->k_rows > 0 && (a->kv == nullptr || a->k_rope == nullptr)))
    return FS_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->kv) | reinterpret_cast<uintptr_t>(a->k_rope) |
       reinterpret_cast<uintptr_t>(a->out)) & 15)
    return FS_ERR_ALIGNMENT;
  if (a->q_rows >= (1ll << 30) || a->k_rows >= (1ll << 30)) return FS_ERR_UNSUPPORTED;
  const int64_t tiles = a->q_rows / kPreQ + a->batch;  // at least as many as the requests have
  if (tiles * a->heads >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  PrefillParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.kv = static_cast<const uint16_t*>(a->kv);
  p.k_rope = static_cast<const uint16_t*>(a->k_rope);
  p.q_off = a->q_offsets;
  p.k_off = a->k_offsets;
  p.out = static_cast<uint16_t*>(a->out);
  p.nq = a->q_rows;
  p.nk = a->k_rows;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.B = a->batch;
  p.H = a->heads;
  const bool bf16 = a->dtype == FS_BF16;
  if (a->nope_dim == 64)
    return a->rope_dim == 32 ? launch_prefill_v<64, 32>(p, tiles, a->value_dim, bf16, stream)
                             : launch_prefill_v<64, 64>(p, tiles, a->value_dim, bf16, stream);
  return a->rope_dim == 32 ? launch_prefill_v<128, 32>(p, tiles, a->value_dim, bf16, stream)
                           : launch_prefill_v<128, 64>(p, tiles, a->value_dim, bf16, stream);
}
