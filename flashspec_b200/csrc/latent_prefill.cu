// Expanded latent attention for prompts: per-head keys and values that the caller expanded
// from the latents, one rotary key shared by all heads, ragged packed requests, causal and
// aligned at the end (the last query of a request sees its last key).
//
//   score(i, h, j) = sm_scale * (q[i, h, :dn] . kv[j, h, :dn] + q[i, h, dn:] . k_rope[j])
//   out[i, h]      = sum_j softmax_j(score) kv[j, h, dn:]
//
// A CTA takes 128 queries of one head and walks the keys in tiles of 128.  Roles:
//   warp 0      TMA: Q once, then K (the head's own chunks and the shared rotary one, side by
//               side, so it is never copied per head) and V tiles, two of each in flight
//   warp 1      tcgen05.mma: S = Q K^T into one of two TMEM buffers, O += P V with P read
//               from TMEM; S of the next tile is issued before P V of this one, so the tensor
//               cores work while the softmax of a tile runs
//   warps 4-11  softmax: two threads a row, 64 keys each (they meet over the row's maximum).
//               P goes back to TMEM in 16 bits over the scores.  The reference maximum moves
//               only when the true one is past it by more than 2^8 (P then stays below 256,
//               sums are in fp32, and O is rescaled seldom instead of once a tile).
// Bound by the tensor cores for long prompts: a tile is 128 x 128 x (dn + dr + dv) MACs.
//
// A value that is not finite must not reach queries that do not see its key (0 * inf is NaN).
// Only tiles on the causal edge are seen by some of a CTA's queries and not by others (and
// only they may hold rows of the next request): there such values are set to zero and the
// first key that has one is noted per dim; the queries that see that key get NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "../../include/flashspec_b200.h"
#include "common.h"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace fsb {

constexpr int kPreThreads = 384;
constexpr int kPreSoft = 256;  // softmax threads (warps 4 .. 11)
constexpr int kPreQ = 128;     // queries of a CTA
constexpr int kPreK = 128;     // keys of a tile
constexpr int kChunk = kPreK * 128;  // bytes of a 64-element chunk of a tile: 128 rows of 128 bytes
constexpr float kPreSlack = 8.f;     // log2 of what the true maximum may be past the reference
constexpr uint64_t kPreTimeoutNs = 2000000000ull;

struct PrefillParams {
  const int64_t* q_off;  // [B + 1]
  const int64_t* k_off;
  uint16_t* out;  // [Nq, H, dv]
  uint32_t* status;
  int64_t nq, nk;
  float scale_log2;
  int B, H;
};

template <int kDN, int kDR, int kDV>
struct PrefillShape {
  static constexpr int kDQ = kDN + kDR;
  static constexpr int kQKChunks = kDN / 64 + 1;  // the last one is the rotary part, 32 or 64 wide
  static constexpr int kVChunks = kDV / 64;
  static constexpr int kQ = 0, kK = kQKChunks * kChunk, kV = kK + 2 * kQKChunks * kChunk;
  static constexpr int kSmem = kV + 2 * kVChunks * kChunk + 1024;  // 1024: alignment
  // TMEM columns: two score buffers (P over their first half) and O
  static constexpr uint32_t kTmemS = 0, kTmemO = 2 * kPreK, kTmemCols = 512;
};

struct PreBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], pv_done;
};

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

// Bounded wait that also ends when another role gave up.
__device__ __forceinline__ bool pre_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t a = smem_u32(bar);
  if (mbar_try_wait(a, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    for (int i = 0; i < 16; ++i)
      if (mbar_try_wait_sleep(a, parity, 1000u)) return true;
    if (*abort != 0) return false;
    if (globaltimer_ns() - t0 > kPreTimeoutNs) {
      *abort = 1;
      return false;
    }
  }
}

template <int kDN, int kDR, int kDV, bool kBf16>
__global__ void __launch_bounds__(kPreThreads, 1)
    latent_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                          const __grid_constant__ CUtensorMap map_r, const PrefillParams p) {
  using L = PrefillShape<kDN, kDR, kDV>;
  extern __shared__ uint8_t pre_raw[];
  __shared__ PreBars bars;
  __shared__ int s_find[2];
  __shared__ volatile int s_abort;
  __shared__ uint32_t s_tmem;
  __shared__ float s_half[2][2][kPreQ];  // [tile parity][half][row]: maxima, and sums at the end
  __shared__ int s_bad[kDV];             // per dim: first key of an edge tile whose value is not finite
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = blockIdx.x % p.H;
  // the tile: counted from the last request's last one back, so that long tiles start first
  const int want = (int)(gridDim.x / p.H) - 1 - (int)(blockIdx.x / p.H);
  if (warp == 0) {
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
  if (tid == 32) {
    mbar_init(smem_u32(&bars.q_full), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.k_full[i]), 1);
      mbar_init(smem_u32(&bars.k_empty[i]), 1);
      mbar_init(smem_u32(&bars.v_full[i]), 1);
      mbar_init(smem_u32(&bars.v_empty[i]), 1);
      mbar_init(smem_u32(&bars.s_full[i]), 1);
      mbar_init(smem_u32(&bars.p_ready[i]), kPreSoft);
    }
    mbar_init(smem_u32(&bars.pv_done), 1);
    s_abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (tid < kDV) s_bad[tid] = INT_MAX;
  __syncthreads();
  const int b = s_find[0];
  if (b < 0) return;  // more CTAs than tiles: the host knows only an upper bound
  if (warp == 2) tmem_alloc(smem_u32(&s_tmem), L::kTmemCols);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = s_tmem;
  const uint32_t smem = (smem_u32(pre_raw) + 1023u) & ~1023u;
  uint8_t* smem_p = pre_raw + (smem - smem_u32(pre_raw));

  int64_t q0, k0;
  int nq, nk;
  pre_range(p.q_off, b, p.nq, q0, nq);
  pre_range(p.k_off, b, p.nk, k0, nk);
  const int i0 = s_find[1] * kPreQ;             // first query of the tile, within the request
  const int rows = min(kPreQ, nq - i0);
  const int shift = nk - nq;                    // query i sees keys j <= i + shift
  const int last = min(nk, i0 + rows + shift);  // keys that any of the tile's queries sees
  const int tiles = last > 0 ? (last + kPreK - 1) / kPreK : 0;

  if (warp == 0) {
    // ================================ TMA ==================================
    if (lane == 0 && tiles > 0) {
      auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int64_t y, uint64_t* bar) {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"((int)y), "r"(smem_u32(bar))
            : "memory");
      };
      mbar_arrive_expect_tx(smem_u32(&bars.q_full), L::kQKChunks * kChunk);
      for (int c = 0; c < L::kQKChunks; ++c) load(smem + L::kQ + c * kChunk, &map_q, h * L::kDQ + 64 * c, q0 + i0, &bars.q_full);
      for (int j = 0; j < tiles; ++j) {
        const int st = j & 1;
        const uint32_t ph = ((j >> 1) & 1) ^ 1;  // the stage's previous use is over (none: passes)
        const int64_t y = k0 + (int64_t)j * kPreK;
        const int x = h * (kDN + kDV);
        if (j >= 2 && !pre_wait(&bars.k_empty[st], ph, &s_abort)) break;
        mbar_arrive_expect_tx(smem_u32(&bars.k_full[st]), L::kQKChunks * kChunk);
        const uint32_t kb = smem + L::kK + st * L::kQKChunks * kChunk;
        for (int c = 0; c < kDN / 64; ++c) load(kb + c * kChunk, &map_kv, x + 64 * c, y, &bars.k_full[st]);
        load(kb + (kDN / 64) * kChunk, &map_r, 0, y, &bars.k_full[st]);
        if (j >= 2 && !pre_wait(&bars.v_empty[st], ph, &s_abort)) break;
        mbar_arrive_expect_tx(smem_u32(&bars.v_full[st]), L::kVChunks * kChunk);
        const uint32_t vb = smem + L::kV + st * L::kVChunks * kChunk;
        for (int c = 0; c < L::kVChunks; ++c) load(vb + c * kChunk, &map_kv, x + kDN + 64 * c, y, &bars.v_full[st]);
      }
    }
  } else if (warp == 1) {
    // ================================ MMA ==================================
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t kIdS = mma_idesc(kPreQ, kPreK, kBf16, false);
      constexpr uint32_t kIdO = mma_idesc(kPreQ, kDV, kBf16, true);
      auto scores = [&](int j) {  // S of tile j
        const uint32_t kb = smem + L::kK + (j & 1) * L::kQKChunks * kChunk;
        const uint32_t d = tmem + L::kTmemS + (j & 1) * kPreK;
#pragma unroll
        for (int s = 0; s < L::kDQ / 16; ++s) {  // 16 dims a step: 32 bytes of a chunk's rows
          const uint32_t off = (s >> 2) * kChunk + (s & 3) * 32;
          mma_ss(d, mma_desc_sw128(smem + L::kQ + off, 0, 1024), mma_desc_sw128(kb + off, 0, 1024), kIdS, s > 0);
        }
        mma_commit(smem_u32(&bars.s_full[j & 1]));
        mma_commit(smem_u32(&bars.k_empty[j & 1]));
      };
      bool ok = pre_wait(&bars.q_full, 0, &s_abort) && pre_wait(&bars.k_full[0], 0, &s_abort);
      tcgen05_fence_after();
      if (ok) scores(0);
      for (int j = 0; j < tiles && ok; ++j) {
        const int st = j & 1;
        if (j + 1 < tiles) {
          ok = pre_wait(&bars.k_full[st ^ 1], ((j + 1) >> 1) & 1, &s_abort);
          tcgen05_fence_after();
          if (!ok) break;
          scores(j + 1);
        }
        ok = pre_wait(&bars.p_ready[st], (j >> 1) & 1, &s_abort) && pre_wait(&bars.v_full[st], (j >> 1) & 1, &s_abort);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t vb = smem + L::kV + st * L::kVChunks * kChunk, a = tmem + L::kTmemS + st * kPreK;
#pragma unroll
        for (int s = 0; s < kPreK / 16; ++s)  // 16 keys a step: 8 columns of P, 16 rows of V
          mma_ts(tmem + L::kTmemO, a + 8 * s, mma_desc_sw128(vb + s * 16 * 128, kChunk, 1024), kIdO, j > 0 || s > 0);
        mma_commit(smem_u32(&bars.v_empty[st]));
        mma_commit(smem_u32(&bars.pv_done));
      }
    }
  } else if (warp >= 4) {
    // ============================== softmax ================================
    const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane, st_tid = tid - 128;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int limit = i0 + row + shift;  // last key that this row sees
    float m_ref = -1.0e30f, l = 0.f;
    // a wait that gave up is shared at the next barrier, where all 256 threads leave together
    bool any_bad = false, ok = true;
    auto any_of = [](bool x) -> bool {  // OR over the softmax threads; also orders their shared memory
      uint32_t r;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, 1, 256, p;\n selp.b32 %0, 1, 0, q;\n}\n"
          : "=r"(r)
          : "r"((uint32_t)x)
          : "memory");
      return r != 0;
    };
    for (int j = 0; j < tiles; ++j) {
      const int st = j & 1, j0 = j * kPreK;
      ok = pre_wait(&bars.s_full[st], (j >> 1) & 1, &s_abort) && ok;
      __syncwarp();
      tcgen05_fence_after();
      const uint32_t sb = tmem + lanes + L::kTmemS + st * kPreK;
      const bool edge = j0 + kPreK > i0 + shift + 1;  // some of the CTA's queries do not see the whole tile
      uint32_t raw[2][32];
      tmem_ld32(sb + 64 * half, raw[0]);
      tmem_ld32(sb + 64 * half + 32, raw[1]);
      tmem_wait_ld();
      // tiles that every query sees whole keep the raw scores (the scale joins in the exponent's
      // FMA); edge tiles are scaled and masked here
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (edge) {
        const int seen = limit - j0 - 64 * half;  // this thread's keys 0 .. seen
#pragma unroll
        for (int k = 0; k < 64; ++k) {
          const float x = k > seen ? -INFINITY : __uint_as_float(raw[k >> 5][k & 31]) * p.scale_log2;
          raw[k >> 5][k & 31] = __float_as_uint(x);
          m4[k & 3] = fmaxf(m4[k & 3], x);
        }
      } else if (p.scale_log2 >= 0.f) {
#pragma unroll
        for (int k = 0; k < 64; ++k) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(raw[k >> 5][k & 31]));
      } else {
#pragma unroll
        for (int k = 0; k < 64; ++k) m4[k & 3] = fmaxf(m4[k & 3], -__uint_as_float(raw[k >> 5][k & 31]));
      }
      const float mul = edge ? 1.f : p.scale_log2;
      float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * fabsf(mul);
      s_half[st][half][row] = mx;
      if (any_of(!ok)) {  // after it, both halves have read their scores
        ok = false;
        break;
      }
      mx = fmaxf(mx, s_half[st][half ^ 1][row]);
      // a row's first maximum is its reference; later ones only when far past it
      const bool move = mx > m_ref + (m_ref == -1.0e30f ? 0.f : kPreSlack);
      if (__any_sync(0xffffffffu, move)) {
        const float m_new = move ? mx : m_ref;
        if (j > 0) {  // O is there: bring it to the new reference
          const float alpha = ex2_approx(m_ref - m_new);
          l *= alpha;
          ok = pre_wait(&bars.pv_done, (j - 1) & 1, &s_abort) && ok;
          __syncwarp();
          tcgen05_fence_after();
          const uint32_t ob = tmem + lanes + L::kTmemO + half * (kDV / 2);
#pragma unroll
          for (int c = 0; c < kDV / 64; ++c) {
            uint32_t o[32];
            tmem_ld32(ob + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st32(ob + 32 * c, o);
          }
        }
        m_ref = m_new;
      }
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t packed[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const float p0 = ex2_approx(fmaf(__uint_as_float(raw[k >> 4][(2 * k) & 31]), mul, -m_ref));
        const float p1 = ex2_approx(fmaf(__uint_as_float(raw[k >> 4][(2 * k + 1) & 31]), mul, -m_ref));
        l4[k & 3] += p0 + p1;
        packed[k] = pre_pack<kBf16>(p0, p1);
      }
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tmem_st32(sb + 32 * half, packed);
      if (edge) {
        constexpr uint16_t kExp = kBf16 ? 0x7f80 : 0x7c00;
        ok = pre_wait(&bars.v_full[st], (j >> 1) & 1, &s_abort) && ok;
        uint8_t* vb = smem_p + L::kV + st * L::kVChunks * kChunk;
        for (int i = st_tid; i < L::kVChunks * kPreK * 8; i += kPreSoft) {
          const int ch = i / (kPreK * 8), r = (i >> 3) & (kPreK - 1), u = i & 7;
          uint4* at = reinterpret_cast<uint4*>(vb + ch * kChunk + r * 128 + 16 * u);
          const uint4 v = *at;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool here = false;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint16_t e = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
            if ((e & kExp) == kExp) {
              atomicMin(s_bad + 64 * ch + 8 * (u ^ (r & 7)) + k, j0 + r);
              w[k >> 1] &= (k & 1) ? 0x0000ffffu : 0xffff0000u;
              here = true;
            }
          }
          if (here) *at = make_uint4(w[0], w[1], w[2], w[3]);
          any_bad |= here;
        }
        fence_proxy_async_smem();  // the MMA reads V through the async proxy
        __syncwarp();
      }
      tmem_wait_st();
      tcgen05_fence_before();
      mbar_arrive(smem_u32(&bars.p_ready[st]));
    }
    if (tiles > 0 && ok) ok = pre_wait(&bars.pv_done, (tiles - 1) & 1, &s_abort);
    __syncwarp();
    s_half[0][half][row] = l;
    const bool failed = any_of(!ok);
    any_bad = any_of(any_bad);
    if (failed) {
      if (st_tid == 0 && p.status != nullptr) atomicOr(p.status, FS_DEV_TIMEOUT);
    } else {
      tcgen05_fence_after();
      l += s_half[0][half ^ 1][row];
      const float inv = l == 0.f ? 0.f : 1.f / l;
      uint16_t* dst = p.out + ((size_t)(q0 + i0 + min(row, rows - 1)) * p.H + h) * kDV + half * (kDV / 2);
#pragma unroll
      for (int c = 0; c < kDV / 64; ++c) {
        uint32_t o[32];
        if (tiles > 0) {
          tmem_ld32(tmem + lanes + L::kTmemO + half * (kDV / 2) + 32 * c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (row < rows) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v0 = __uint_as_float(o[k + 2 * e]) * inv, v1 = __uint_as_float(o[k + 2 * e + 1]) * inv;
              if (any_bad) {
                const int d = half * (kDV / 2) + 32 * c + k + 2 * e;
                if (s_bad[d] <= limit) v0 = __int_as_float(0x7fc00000);
                if (s_bad[d + 1] <= limit) v1 = __int_as_float(0x7fc00000);
              }
              w[e] = pre_pack<kBf16>(v0, v1);
            }
            *reinterpret_cast<uint4*>(dst + 32 * c + k) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
      }
    }
    tcgen05_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Rows [n, heads * width] of 16-bit elements as boxes of 128 rows by 64 elements; what lies
// behind a row's end or behind the last row reads as zero.
static int pre_map(CUtensorMap* map, const void* base, int64_t n, int64_t row_elems) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail_cuda("cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)row_elems, (cuuint64_t)n};
  cuuint64_t strides[1] = {(cuuint64_t)row_elems * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)kPreK};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FS_OK : fail_cuda("cuTensorMapEncodeTiled", r);
}

template <int kDN, int kDR, int kDV>
static int launch_prefill(const FsLatentPrefillArgs* a, const PrefillParams& p, int64_t tiles, void* stream) {
  using L = PrefillShape<kDN, kDR, kDV>;
  CUtensorMap mq, mkv, mr;
  if (int st = pre_map(&mq, a->q, a->q_rows, (int64_t)a->heads * L::kDQ); st != FS_OK) return st;
  if (a->k_rows > 0) {
    if (int st = pre_map(&mkv, a->kv, a->k_rows, (int64_t)a->heads * (kDN + kDV)); st != FS_OK) return st;
    if (int st = pre_map(&mr, a->k_rope, a->k_rows, kDR); st != FS_OK) return st;
  } else {
    mkv = mr = mq;  // no key tile is ever loaded
  }
  auto kernel = a->dtype == FS_BF16 ? latent_prefill_kernel<kDN, kDR, kDV, true> : latent_prefill_kernel<kDN, kDR, kDV, false>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
      e != cudaSuccess)
    return fail_cuda("shared-memory limit of the latent prefill kernel", e);
  kernel<<<(unsigned)(tiles * p.H), kPreThreads, L::kSmem, reinterpret_cast<cudaStream_t>(stream)>>>(mq, mkv, mr, p);
  return launch_status("latent prefill kernel launch");
}

template <int kDN, int kDR>
static int launch_prefill_v(const FsLatentPrefillArgs* a, const PrefillParams& p, int64_t tiles, void* stream) {
  return a->value_dim == 64 ? launch_prefill<kDN, kDR, 64>(a, p, tiles, stream)
                            : launch_prefill<kDN, kDR, 128>(a, p, tiles, stream);
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
  if (a->q_rows >= (1ll << 30) || a->k_rows >= (1ll << 30) || a->heads > (1 << 20)) return FS_ERR_UNSUPPORTED;
  const int64_t tiles = a->q_rows / kPreQ + a->batch;  // at least as many as the requests have
  if (tiles * a->heads >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  PrefillParams p{};
  p.q_off = a->q_offsets;
  p.k_off = a->k_offsets;
  p.out = static_cast<uint16_t*>(a->out);
  p.status = a->device_status;
  p.nq = a->q_rows;
  p.nk = a->k_rows;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.B = a->batch;
  p.H = a->heads;
  if (a->nope_dim == 64)
    return a->rope_dim == 32 ? launch_prefill_v<64, 32>(a, p, tiles, stream) : launch_prefill_v<64, 64>(a, p, tiles, stream);
  return a->rope_dim == 32 ? launch_prefill_v<128, 32>(a, p, tiles, stream) : launch_prefill_v<128, 64>(a, p, tiles, stream);
}
