// Expanded latent attention for prompts: per-head keys and values that the caller expanded
// from the latents, one rotary key shared by all heads, ragged packed requests, causal and
// aligned at the end (the last query of a request sees its last key).
//
//   score(i, h, j) = sm_scale * (q[i, h, :dn] . kv[j, h, :dn] + q[i, h, dn:] . k_rope[j])
//   out[i, h]      = sum_j softmax_j(score) kv[j, h, dn:]
//
// A CTA takes 256 queries of one head, as two blocks of 128, and walks the keys in tiles of
// 96, so that two K and two V tiles fit beside the queries.  Four packed prompts (4096 -> 500
// tokens, 16 heads) take 198 us, 732 TFLOP/s of useful work.  Measured and dropped: 128 queries
// a CTA (220 us), an O each for even and odd tiles (230), 128 keys a tile with P over S (222),
// 80 keys with P beside S (244).  Spinning in place of sleeping waits cost 5% of the kernel.
// The MMA thread takes its descriptors from precomputed words: building them bound it.  Roles:
//   warp 0      TMA: the queries once, then K (the head's own chunks and the shared rotary
//               one, side by side, so it is never copied per head) and V tiles
//   warp 1      tcgen05.mma: S = Q K^T into TMEM, O += P V with P read from TMEM
//   warps 4-7   softmax of the first block, one thread a row; warps 8-11 of the second
// The blocks do not wait for each other: the tensor cores work on one's tile while the other
// forms exponentials.  P goes back to TMEM in 16 bits over the scores.  The reference maximum
// moves only when the true one is far past it (PreRange; sums are in fp32, and O is rescaled
// seldom instead of once a tile).
//
// A value that is not finite must not reach queries that do not see its key (0 * inf is NaN).
// Only tiles on the causal edge are seen by some of a block's queries and not by others (and
// only they may hold rows of the next request): there such values are set to zero.  Elsewhere
// they go through the MMA, where a probability that 16 bits round to zero makes NaN of an
// infinity.  A CTA that met one either way looks its values over once more (pre_mend) and gives
// each query what the definition gives: infinity where it sees infinities of one sign, else NaN.
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
constexpr int kPreSoft = 128;  // threads of a softmax group
constexpr int kPreQ = 128;     // queries of a block, two blocks a CTA
constexpr int kPreK = 96;      // keys of a tile
constexpr int kQChunk = kPreQ * 128;  // bytes of a 64-element chunk: rows of 128 bytes
constexpr int kChunk = kPreK * 128;
// P = 2^(score - reference + kLift).  The true maximum may be 2^kSlack past the reference.  fp16
// ends at 2^16 and loses bits below 2^-14: the lift keeps all of them down to 2^-25 of the
// maximum, where many far keys beside one near key of small value still make the output
// (without it 30000 keys at 2^-24.5 were rounded to nothing, and the output with them).  bf16 has
// the range of fp32 and needs no lift.
template <bool kBf16>
struct PreRange {
  static constexpr float kSlack = kBf16 ? 8.f : 4.f, kLift = kBf16 ? 0.f : 11.f;
};
constexpr uint64_t kPreTimeoutNs = 2000000000ull;

struct PrefillParams {
  const uint16_t* kv;    // [Nk, H, dn + dv]
  const int64_t* q_off;  // [B + 1]
  const int64_t* k_off;
  uint16_t* out;  // [Nq, H, dv]
  uint32_t* status;
  int64_t nq, nk;
  float scale_log2;
  int B, H;
  int tile_ctas;  // CTAs that may have queries; the ones behind them clear rows of no request
};

template <int kDN, int kDR, int kDV>
struct PrefillShape {
  static constexpr int kDQ = kDN + kDR;
  static constexpr int kQKChunks = kDN / 64 + 1;  // the last one is the rotary part, 32 or 64 wide
  static constexpr int kVChunks = kDV / 64;
  static constexpr int kQ = 0, kK = 2 * kQKChunks * kQChunk, kV = kK + 2 * kQKChunks * kChunk;
  static constexpr int kSmem = kV + 2 * kVChunks * kChunk + 1024;  // 1024: alignment
  // TMEM columns of a block: scores (P over their first half), and O
  static constexpr uint32_t kTmemS = 0, kTmemO = 256, kTmemStep = 128, kTmemCols = 512;
};

struct PreBars {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], pv_done[2], drained;
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

// The w-th piece of work, one warp: (request, its 256-query tile), the request -1 when there
// is none.
//
// Up to kPreDealt requests are dealt by descending tile index, so that tiles with many keys start
// first: f(t) = tiles with an index of at least t; the w-th one has the largest t with f(t) > w.
// (One prompt of 4096 tokens 104 us, 143 in ascending order; 32 ragged ones 1370, 1230.)
//
// More are found by a search of 32 probes a round: piece w belongs to the last request with
// base(b) = first row / 256 + b <= w.  base grows by at least the request's tiles, as n rows from
// row 256 a + r on pass (r + n) / 256 multiples of 256, and ends at the CTAs that the host
// launches.  (64 ragged prompts of up to 2048 tokens 438 us, 482 dealt; 4096 requests of one token
// 3.1 ms, 28 dealt: dealing looks at all requests in every CTA.)
//
// Offsets that fall at the end (a batch padded with zeros) would mislead the search; they are
// dealt as well, up to kPreFalling requests, where that takes tens of milliseconds; a larger batch
// of them is not computed.
constexpr int kPreDealt = 32, kPreFalling = 4096;

__device__ __forceinline__ int2 pre_find(const PrefillParams& p, int w, int lane) {
  auto tiles_of = [&](int b) -> int {
    int64_t lo;
    int n = 0;
    if (b < p.B) pre_range(p.q_off, b, p.nq, lo, n);
    return (n + 2 * kPreQ - 1) / (2 * kPreQ);
  };
  auto row_of = [&](int b) -> int64_t { return min(max(p.q_off[b], (int64_t)0), p.nq); };
  if (p.B > kPreDealt) {
    const int64_t last = row_of(p.B);
    bool falls = false;
    int lo = 0, hi = p.B;  // the request lies in [lo, hi), if there is one
    for (int step = hi; step > 1 && !falls;) {
      step = (int)(((int64_t)hi - lo + 31) / 32);
      const int64_t at = lo + (int64_t)lane * step;
      const int64_t row = at < hi ? row_of((int)at) : 0;
      falls = __any_sync(0xffffffffu, row > last);
      const int below = __popc(__ballot_sync(0xffffffffu, at < hi && row / (2 * kPreQ) + at <= w));
      if (below == 0) break;
      lo += (below - 1) * step;
      hi = min(hi, lo + step);
    }
    if (!falls) {
      const int64_t t = w - (row_of(lo) / (2 * kPreQ) + lo);  // negative: rows before the first request
      return t >= 0 && t < tiles_of(lo) ? make_int2(lo, (int)t) : make_int2(-1, 0);
    }
    if (p.B > kPreFalling) return make_int2(-1, 0);
  }
  const int mine = tiles_of(lane);  // up to 32 requests are one look
  auto count = [&](int t) -> int {  // f(t)
    int x = max(0, mine - t);
    for (int b = 32 + lane; b < p.B; b += 32) x += max(0, tiles_of(b) - t);
    return (int)__reduce_add_sync(0xffffffffu, (uint32_t)x);
  };
  if (count(0) <= w) return make_int2(-1, 0);
  int lo = 0, hi = (int)(p.nq / (2 * kPreQ)) + 1;  // f(lo) > w, f(hi) = 0
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) > w) lo = mid; else hi = mid;
  }
  int k = w - count(lo + 1);  // the k-th request that has a tile of this index
  for (int base = 0; base < p.B; base += 32) {
    const uint32_t has = __ballot_sync(0xffffffffu, (base == 0 ? mine : tiles_of(base + lane)) > lo);
    const int n = __popc(has);
    if (k < n) return make_int2(base + (int)__fns(has, 0, k + 1), lo);
    k -= n;
  }
  return make_int2(-1, 0);
}

// Zeros in the rows of out that no request covers, 1024 rows a CTA.  Ascending offsets leave
// only rows before the first and behind the last; others are looked up row by row.
constexpr int kClearRows = 1024;

template <int kDV>
__device__ __forceinline__ void pre_clear(const PrefillParams& p, int chunk) {
  const int64_t r0 = (int64_t)chunk * kClearRows, r1 = min(p.nq, r0 + kClearRows);
  const int64_t first = p.q_off[0], last = p.q_off[p.B];
  bool falls = false;
  for (int b = threadIdx.x; b < p.B; b += kPreThreads) falls |= p.q_off[b + 1] < p.q_off[b];
  falls = __syncthreads_or(falls ? 1 : 0) != 0;
  if (!falls && first <= r0 && last >= r1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = r0 + warp; r < r1; r += kPreThreads / 32) {
    bool covered = r >= first && r < last;
    if (falls) {
      covered = false;
      for (int b = lane; b < p.B; b += 32) covered |= r >= p.q_off[b] && r < p.q_off[b + 1];
      covered = __any_sync(0xffffffffu, covered);
    }
    if (covered) continue;
    uint4* row = reinterpret_cast<uint4*>(p.out + (size_t)r * p.H * kDV);
    for (int i = lane; i < p.H * kDV / 8; i += 32) row[i] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// OR of x over the two softmax groups; also orders their shared memory.
__device__ __forceinline__ bool pre_any(bool x) {
  __syncwarp();  // the barrier wants whole warps; loops before it may end lane by lane
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.or.pred q, 1, 256, p;\n selp.b32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// The softmax groups of a CTA that met values that are not finite: the first key of each dim
// whose value is NaN, +inf and -inf (first [3][kDV], shared), among the keys that any query of
// the CTA sees; then this thread's output row, whose last key is `limit` (-1: no row), gets its
// infinities and NaN.  Out of line: it costs the kernel no registers, and a V pass when it runs.
// v0: the first key's value of this head; stride: elements from key to key.
template <int kDV, bool kBf16>
static __device__ __noinline__ void pre_mend(const uint16_t* v0, int64_t stride, int keys, int* first, int limit,
                                             uint16_t* dst) {
  constexpr int kThreads = 2 * kPreSoft, kUnits = kDV / 8;
  constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
  const int t = threadIdx.x - (kPreThreads - kThreads);
  for (int i = t; i < 3 * kDV; i += kThreads) first[i] = INT_MAX;
  pre_any(false);
  for (int64_t i = t; i < (int64_t)keys * kUnits; i += kThreads) {
    const int key = (int)(i / kUnits), u = (int)(i % kUnits);
    const uint4 v = *reinterpret_cast<const uint4*>(v0 + key * stride + 8 * u);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = (w[k >> 1] >> (16 * (k & 1))) & 0xffffu;
      if ((e & 0x7fffu) < kInf) continue;
      int* at = first + ((e & 0x7fffu) > kInf ? 0 : (e >> 15) + 1) * kDV + 8 * u + k;
      if (key < *reinterpret_cast<volatile int*>(at)) atomicMin(at, key);
    }
  }
  pre_any(false);
  for (int d = 0; d < kDV; ++d) {
    const bool nan = first[d] <= limit, pos = first[kDV + d] <= limit, neg = first[2 * kDV + d] <= limit;
    if (nan || pos || neg) dst[d] = (uint16_t)(nan || (pos && neg) ? 0x7fffu : pos ? kInf : 0x8000u | kInf);
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
  __shared__ int s_first[3 * kDV];  // pre_mend's
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= p.tile_ctas) {
    pre_clear<kDV>(p, (int)blockIdx.x - p.tile_ctas);
    return;
  }
  const int h = blockIdx.x % p.H;
  if (warp == 0) {
    const int2 at = pre_find(p, (int)(blockIdx.x / p.H), lane);
    if (lane == 0) s_find[0] = at.x, s_find[1] = at.y;
  }
  if (tid == 32) {
    mbar_init(smem_u32(&bars.q_full), 1);
    mbar_init(smem_u32(&bars.drained), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.k_full[i]), 1);
      mbar_init(smem_u32(&bars.k_empty[i]), 1);
      mbar_init(smem_u32(&bars.v_full[i]), 1);
      mbar_init(smem_u32(&bars.v_empty[i]), 1);
      mbar_init(smem_u32(&bars.s_full[i]), 1);
      mbar_init(smem_u32(&bars.p_ready[i]), kPreSoft);
      mbar_init(smem_u32(&bars.pv_done[i]), 1);
    }
    s_abort = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
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
  const int i0 = s_find[1] * 2 * kPreQ;  // first query of the CTA, within the request
  const int shift = nk - nq;             // query i sees keys j <= i + shift
  // key tiles that any query of block g sees
  auto tiles_of = [&](int g) -> int {
    const int first = i0 + g * kPreQ, rows = min(kPreQ, nq - first), last = rows > 0 ? min(nk, first + rows + shift) : 0;
    return last > 0 ? (last + kPreK - 1) / kPreK : 0;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), tiles = max(n0, n1);
  int k_sent = 0, v_sent = 0;  // of the TMA thread: tiles whose copies were issued

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
      mbar_arrive_expect_tx(smem_u32(&bars.q_full), 2 * L::kQKChunks * kQChunk);
      for (int c = 0; c < 2 * L::kQKChunks; ++c)  // block 0's chunks, then block 1's (rows behind the last read as zero)
        load(smem + L::kQ + c * kQChunk, &map_q, h * L::kDQ + 64 * (c % L::kQKChunks),
             q0 + i0 + (c / L::kQKChunks) * kPreQ, &bars.q_full);
      for (int j = 0; j < tiles; ++j) {
        const int st = j & 1;
        const uint32_t ph = ((j >> 1) & 1) ^ 1;  // the stage's previous use is over (none: passes)
        const int64_t y = k0 + (int64_t)j * kPreK;
        const int x = h * (kDN + kDV);
        if (j >= 2 && !pre_wait(&bars.k_empty[st], ph, &s_abort)) break;
        mbar_arrive_expect_tx(smem_u32(&bars.k_full[st]), L::kQKChunks * kChunk);
        k_sent = j + 1;
        const uint32_t kb = smem + L::kK + st * L::kQKChunks * kChunk;
        for (int c = 0; c < kDN / 64; ++c) load(kb + c * kChunk, &map_kv, x + 64 * c, y, &bars.k_full[st]);
        load(kb + (kDN / 64) * kChunk, &map_r, 0, y, &bars.k_full[st]);
        if (j >= 2 && !pre_wait(&bars.v_empty[st], ph, &s_abort)) break;
        mbar_arrive_expect_tx(smem_u32(&bars.v_full[st]), L::kVChunks * kChunk);
        v_sent = j + 1;
        const uint32_t vb = smem + L::kV + st * L::kVChunks * kChunk;
        for (int c = 0; c < L::kVChunks; ++c) load(vb + c * kChunk, &map_kv, x + kDN + 64 * c, y, &bars.v_full[st]);
      }
    }
  } else if (warp == 1) {
    // ================================ MMA ==================================
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t kIdS = mma_idesc(kPreQ, kPreK, kBf16, false);
      constexpr uint32_t kIdO = mma_idesc(kPreQ, kDV, kBf16, true);
      constexpr uint32_t kHi = mma_desc_hi_sw128(1024);
      const uint32_t q_lo = mma_desc_lo(smem + L::kQ, 0), k_lo = mma_desc_lo(smem + L::kK, 0);
      const uint32_t v_lo = mma_desc_lo(smem + L::kV, kChunk);
      auto scores = [&](int g, int j) {  // S of block g and tile j
        const uint32_t q = q_lo + g * (L::kQKChunks * kQChunk / 16), k = k_lo + (j & 1) * (L::kQKChunks * kChunk / 16);
        const uint32_t d = tmem + L::kTmemS + g * L::kTmemStep;
#pragma unroll
        for (int s = 0; s < L::kDQ / 16; ++s)  // 16 dims a step: 32 bytes of a chunk's rows
          mma_ss(d, mma_desc(q + ((s >> 2) * kQChunk + (s & 3) * 32) / 16, kHi),
                 mma_desc(k + ((s >> 2) * kChunk + (s & 3) * 32) / 16, kHi), kIdS, s > 0);
        mma_commit(smem_u32(&bars.s_full[g]));
      };
      bool ok = pre_wait(&bars.q_full, 0, &s_abort) && pre_wait(&bars.k_full[0], 0, &s_abort);
      tcgen05_fence_after();
      if (ok) {
        if (n0 > 0) scores(0, 0);
        if (n1 > 0) scores(1, 0);
        // a stage is reported free only to a later tile: no arrival is under way when the CTA ends
        if (tiles > 2) mma_commit(smem_u32(&bars.k_empty[0]));
      }
      for (int j = 0; j < tiles && ok; ++j) {
        const int st = j & 1;
        const uint32_t v = v_lo + st * (L::kVChunks * kChunk / 16);
        ok = pre_wait(&bars.v_full[st], (j >> 1) & 1, &s_abort);
        if (ok && j + 1 < tiles) ok = pre_wait(&bars.k_full[st ^ 1], ((j + 1) >> 1) & 1, &s_abort);
        for (int g = 0; g < 2 && ok; ++g) {
          const int n = g == 0 ? n0 : n1;
          if (j >= n) continue;
          ok = pre_wait(&bars.p_ready[g], j & 1, &s_abort);
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t a = tmem + L::kTmemS + g * L::kTmemStep, d = tmem + L::kTmemO + g * L::kTmemStep;
#pragma unroll
          for (int s = 0; s < kPreK / 16; ++s)  // 16 keys a step: 8 columns of P, 16 rows of V
            mma_ts(d, a + 8 * s, mma_desc(v + s * (16 * 128 / 16), kHi), kIdO, j > 0 || s > 0);
          if (j + 1 == n) mma_commit(smem_u32(&bars.pv_done[g]));
          if (j + 1 < n) scores(g, j + 1);  // over the P that was just read
        }
        if (j + 2 < tiles) mma_commit(smem_u32(&bars.v_empty[st]));
        if (j + 3 < tiles) mma_commit(smem_u32(&bars.k_empty[st ^ 1]));  // of tile j + 1
      }
    }
  } else if (warp >= 4) {
    // ============================== softmax ================================
    const int grp = (warp - 4) >> 2, row = (warp & 3) * 32 + lane, grp_tid = tid & (kPreSoft - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int first = i0 + grp * kPreQ, rows = min(kPreQ, nq - first), n = grp == 0 ? n0 : n1;
    const int limit = first + row + shift;  // last key that this row sees
    const uint32_t sb = tmem + lanes + L::kTmemS + grp * L::kTmemStep;
    const uint32_t ob = tmem + lanes + L::kTmemO + grp * L::kTmemStep;
    float m_ref = -1.0e30f, l = 0.f;
    bool any_bad = false, ok = true;
    for (int j = 0; j < n; ++j) {
      const int j0 = j * kPreK;
      ok = pre_wait(&bars.s_full[grp], j & 1, &s_abort);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tcgen05_fence_after();
      const bool edge = j0 + kPreK > first + shift + 1;  // some of the block's queries do not see the whole tile
      uint32_t raw[kPreK / 32][32];
#pragma unroll
      for (int c = 0; c < kPreK / 32; ++c) tmem_ld32(sb + 32 * c, raw[c]);
      tmem_wait_ld();
      // tiles that every query sees whole keep the raw scores (the scale joins in the exponent's
      // FMA); edge tiles are scaled and masked here
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (edge) {
        const int seen = limit - j0;  // this row's keys 0 .. seen
#pragma unroll
        for (int k = 0; k < kPreK; ++k) {
          const float x = k > seen ? -INFINITY : __uint_as_float(raw[k >> 5][k & 31]) * p.scale_log2;
          raw[k >> 5][k & 31] = __float_as_uint(x);
          m4[k & 3] = fmaxf(m4[k & 3], x);
        }
      } else if (p.scale_log2 >= 0.f) {
#pragma unroll
        for (int k = 0; k < kPreK; ++k) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(raw[k >> 5][k & 31]));
      } else {
#pragma unroll
        for (int k = 0; k < kPreK; ++k) m4[k & 3] = fmaxf(m4[k & 3], -__uint_as_float(raw[k >> 5][k & 31]));
      }
      const float mul = edge ? 1.f : p.scale_log2;
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * fabsf(mul);
      // a row's first maximum is its reference; later ones only when far past it
      const bool move = mx > m_ref + (m_ref == -1.0e30f ? 0.f : PreRange<kBf16>::kSlack);
      if (__any_sync(0xffffffffu, move)) {
        const float m_new = move ? mx : m_ref;
        if (j > 0) {  // O is there (its MMAs were issued before this tile's): bring it to the new reference
          const float alpha = ex2_approx(m_ref - m_new);
          l *= alpha;
#pragma unroll
          for (int c = 0; c < kDV / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(ob + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st16(ob + 16 * c, o);
          }
        }
        m_ref = m_new;
      }
      const float up = PreRange<kBf16>::kLift - m_ref;
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kPreK / 32; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float p0 = ex2_approx(fmaf(__uint_as_float(raw[c][2 * k]), mul, up));
          const float p1 = ex2_approx(fmaf(__uint_as_float(raw[c][2 * k + 1]), mul, up));
          l4[k & 3] += p0 + p1;
          packed[k] = pre_pack<kBf16>(p0, p1);
        }
        tmem_st16(sb + 16 * c, packed);
      }
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      if (edge) {
        constexpr uint16_t kExp = kBf16 ? 0x7f80 : 0x7c00;
        ok = pre_wait(&bars.v_full[j & 1], (j >> 1) & 1, &s_abort);
        uint8_t* vb = smem_p + L::kV + (j & 1) * L::kVChunks * kChunk;
#pragma unroll 2
        for (int i = grp_tid; i < L::kVChunks * kPreK * 8; i += kPreSoft) {
          uint4* at = reinterpret_cast<uint4*>(vb + 16 * i);  // [chunk][key][16-byte unit]
          const uint4 v = *at;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool here = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // an exponent of all ones carries out of its field when its lowest bit is added
            constexpr uint32_t kLow = kBf16 ? 0x00800080u : 0x04000400u, kMask = kBf16 ? 0x7f807f80u : 0x7c007c00u;
            here |= (((w[k] & kMask) + kLow) & 0x80008000u) != 0u;
          }
          if (here) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint16_t e = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
              if ((e & kExp) == kExp) w[k >> 1] &= (k & 1) ? 0x0000ffffu : 0xffff0000u;
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
            any_bad = true;
          }
        }
        fence_proxy_async_smem();  // the MMA reads V through the async proxy
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
      }
      tmem_wait_st();
      tcgen05_fence_before();
      mbar_arrive(smem_u32(&bars.p_ready[grp]));
    }
    if (n > 0 && ok) ok = pre_wait(&bars.pv_done[grp], 0, &s_abort);
    __syncwarp();
    const bool failed = pre_any(!ok);
    uint16_t* dst = p.out + ((size_t)(q0 + first + row) * p.H + h) * kDV;
    if (failed) {
      if (grp == 0 && grp_tid == 0 && p.status != nullptr) atomicOr(p.status, FS_DEV_TIMEOUT);
    } else {
      tcgen05_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < kDV / 16; ++c) {
        uint32_t o[16];
        if (n > 0) {
          tmem_ld16(ob + 16 * c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = 0u;
        }
        if (row < rows) {
#pragma unroll
          for (int k = 0; k < 16; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float v[2];
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                v[u] = __uint_as_float(o[k + 2 * e + u]) * inv;
                bad |= !(fabsf(v[u]) < INFINITY);
              }
              w[e] = pre_pack<kBf16>(v[0], v[1]);
            }
            *reinterpret_cast<uint4*>(dst + 16 * c + k) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
      }
      any_bad |= bad && l == l;  // a row whose probabilities are undefined is NaN throughout already
    }
    if (pre_any(any_bad && !failed)) {
      const int keys = min(nk, i0 + min(2 * kPreQ, nq - i0) + shift);
      const int64_t stride = (int64_t)p.H * (kDN + kDV);
      pre_mend<kDV, kBf16>(p.kv + k0 * stride + (int64_t)h * (kDN + kDV) + kDN, stride, keys, s_first,
                           row < rows && l == l ? limit : -1, dst);
    }
    tcgen05_fence_before();
  }
  __syncthreads();
  if (s_abort != 0) {  // a wait gave up: memory is given back behind the copies and MMAs in flight
    if (warp == 0 && lane == 0 && tiles > 0) {
      mbar_wait_bounded(smem_u32(&bars.q_full), 0, kPreTimeoutNs);
      for (int j = max(0, k_sent - 2); j < k_sent; ++j)
        mbar_wait_bounded(smem_u32(&bars.k_full[j & 1]), (j >> 1) & 1, kPreTimeoutNs);
      for (int j = max(0, v_sent - 2); j < v_sent; ++j)
        mbar_wait_bounded(smem_u32(&bars.v_full[j & 1]), (j >> 1) & 1, kPreTimeoutNs);
    }
    if (warp == 1 && lane == 0) {  // the thread that issued the MMAs
      mma_commit(smem_u32(&bars.drained));
      mbar_wait_bounded(smem_u32(&bars.drained), 0, kPreTimeoutNs);
    }
    __syncthreads();
  }
  if (warp == 2) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// Rows [n, heads * width] of 16-bit elements as boxes of box_rows rows by 64 elements; what lies
// behind a row's end or behind the last row reads as zero.
static int pre_map(CUtensorMap* map, const void* base, int64_t n, int64_t row_elems, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return fail_cuda("cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)row_elems, (cuuint64_t)n};
  cuuint64_t strides[1] = {(cuuint64_t)row_elems * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FS_OK : fail_cuda("cuTensorMapEncodeTiled", r);
}

template <int kDN, int kDR, int kDV>
static int launch_prefill(const FsLatentPrefillArgs* a, const PrefillParams& p, void* stream) {
  using L = PrefillShape<kDN, kDR, kDV>;
  CUtensorMap mq, mkv, mr;
  if (int st = pre_map(&mq, a->q, a->q_rows, (int64_t)a->heads * L::kDQ, kPreQ); st != FS_OK) return st;
  if (a->k_rows > 0) {
    if (int st = pre_map(&mkv, a->kv, a->k_rows, (int64_t)a->heads * (kDN + kDV), kPreK); st != FS_OK) return st;
    if (int st = pre_map(&mr, a->k_rope, a->k_rows, kDR, kPreK); st != FS_OK) return st;
  } else {
    mkv = mr = mq;  // no key tile is ever loaded
  }
  auto kernel = a->dtype == FS_BF16 ? latent_prefill_kernel<kDN, kDR, kDV, true> : latent_prefill_kernel<kDN, kDR, kDV, false>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
      e != cudaSuccess)
    return fail_cuda("shared-memory limit of the latent prefill kernel", e);
  const int64_t ctas = p.tile_ctas + (a->clear_rest ? (a->q_rows + kClearRows - 1) / kClearRows : 0);
  kernel<<<(unsigned)ctas, kPreThreads, L::kSmem, reinterpret_cast<cudaStream_t>(stream)>>>(mq, mkv, mr, p);
  return launch_status("latent prefill kernel launch");
}

template <int kDN, int kDR>
static int launch_prefill_v(const FsLatentPrefillArgs* a, const PrefillParams& p, void* stream) {
  return a->value_dim == 64 ? launch_prefill<kDN, kDR, 64>(a, p, stream)
                            : launch_prefill<kDN, kDR, 128>(a, p, stream);
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
  const int64_t tiles = a->q_rows / (2 * kPreQ) + a->batch;  // at least as many as the requests have
  if (tiles * a->heads + a->q_rows / kClearRows + 1 >= (1ll << 31)) return FS_ERR_UNSUPPORTED;
  PrefillParams p{};
  p.kv = static_cast<const uint16_t*>(a->kv);
  p.q_off = a->q_offsets;
  p.k_off = a->k_offsets;
  p.out = static_cast<uint16_t*>(a->out);
  p.status = a->device_status;
  p.nq = a->q_rows;
  p.nk = a->k_rows;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.B = a->batch;
  p.H = a->heads;
  p.tile_ctas = (int)(tiles * a->heads);
  if (a->nope_dim == 64)
    return a->rope_dim == 32 ? launch_prefill_v<64, 32>(a, p, stream) : launch_prefill_v<64, 64>(a, p, stream);
  return a->rope_dim == 32 ? launch_prefill_v<128, 32>(a, p, stream) : launch_prefill_v<128, 64>(a, p, stream);
}
