// Tensor-core kernels of the int8 product (tcgen05.mma.kind::i8, int8 x int8
// into int32 accumulators in TMEM), operands brought in by tiled TMA copies with
// the 128-byte swizzle: one stage of the shared-memory ring is 128 bytes of K of
// an operand tile's rows, four MMAs of K = 32.
//
//   split_kernel  few tokens: weights are the M = 128 operand, tokens the N
//                 operand, and the CTAs of a cluster split K (their sums, whole
//                 numbers, meet over distributed shared memory).
//   pair_kernel   many tokens: persistent pairs of CTAs (cta_group::2), 256
//                 tokens x BN weight rows per tile, two accumulators so that one
//                 tile's epilogue runs under the next one's MMAs.
#pragma once

#include <cuda.h>

#include "qx_tc.cuh"

namespace qx {
namespace i8 {

constexpr uint32_t KST = 128;            // K bytes per stage (one swizzle span)

// ---- descriptors -----------------------------------------------------------------
// Shared-memory descriptor of a K-major tile with the 128-byte swizzle: rows 128
// bytes apart, 8-row groups 1024 bytes apart. A step of 32 K bytes advances the
// start address by 32 (the swizzle is a function of the address bits).
__device__ __forceinline__ uint64_t sdesc128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}

// Instruction descriptor of kind::i8: int32 accumulators, signed A and B, both
// K-major, dense, no saturation.
__host__ __device__ constexpr uint32_t idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// ---- TMA, clusters ----------------------------------------------------------------
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
// As tma_2d; the barrier may be the pair's other CTA's.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int4 ld_cluster_int4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrive on `bar` in both CTAs of the pair when the tcgen05 operations issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

// Bounded wait (cluster scope): false once the deadline has passed, with
// QX_DEV_TIMEOUT recorded; the caller then stops consuming.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, uint64_t deadline) {
  for (uint32_t it = 0;; ++it) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 15u) == 15u && globaltimer_ns() > deadline) {
      atomicOr(&g_status, (uint32_t)QX_DEV_TIMEOUT);
      return false;
    }
  }
}

// ---- accumulator loads ---------------------------------------------------------------
__device__ __forceinline__ void tm_ld16(uint32_t taddr, int32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Eight consecutive outputs of one row from column n (valid up to p.n): one
// 16-byte (two for FP32) store when the row allows it (vec), else element by element.
__device__ __forceinline__ void store8(const Args& p, int64_t row, int n, const float (&v)[8], bool vec) {
  const int64_t i = row * p.os + n;
  if (vec && n + 8 <= p.n) {
    if (p.type == QX_T_F32) {
      float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + i);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (p.type == QX_T_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (n + j < p.n) store_out(p.out, i + j, p.type, v[j]);
}

// ------------------------------------------------------------------ few tokens
// Grid: (row tile of 128 weight rows, token tile of BN tokens, K piece), the K
// pieces of one tile in one cluster. Warp 0 copies, warp 1 issues the MMAs, warps
// 2-5 bring the accumulator to shared memory; then every CTA of the cluster adds
// a share of the tile over the pieces and writes it. With SwiGLU the 128 rows are
// 64 gate rows and their 64 up rows. The ring is small enough for two CTAs per SM.
template <int BN>
struct Split {
  static constexpr uint32_t A_BYTES = 128 * KST, B_BYTES = BN * KST, STAGE = A_BYTES + B_BYTES;
  static constexpr int NS = BN <= 32 ? 5 : BN == 64 ? 4 : 3;
  static constexpr uint32_t COLS = BN < 32 ? 32 : BN;
  static constexpr size_t SMEM = NS * STAGE + 1024;      // 1024: alignment of the swizzled tiles
  static_assert(BN * 128 * 4 <= NS * STAGE, "the accumulator fits the drained ring");
};
constexpr int SPLIT_THR = 192;

template <int BN>
__global__ void __launch_bounds__(SPLIT_THR) split_kernel(const __grid_constant__ CUtensorMap tw,
                                                          const __grid_constant__ CUtensorMap ta, Args p, int pieces,
                                                          uint64_t timeout) {
  using L = Split<BN>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[L::NS], empty[L::NS], done;
  __shared__ uint32_t tmem;
  uint8_t* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = pieces > 1 ? (int)cluster_rank() : 0;
  const int half = p.swiglu ? 64 : 128;                  // output columns of a tile
  const int n0 = (int)(blockIdx.x / pieces) * half, m0 = blockIdx.y * BN;
  const int chunks = (p.k + (int)KST - 1) / (int)KST;
  const int c0 = (int)((int64_t)chunks * rank / pieces), c1 = (int)((int64_t)chunks * (rank + 1) / pieces);
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem, L::COLS);
    tc::tmem_relinquish();
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint64_t deadline = globaltimer_ns() + timeout;
  bool ok = true;
  if (warp == 0 && lane == 0) {
    int s = 0;
    uint32_t ph = 1;
    for (int c = c0; c < c1; ++c) {
      if (!(ok = wait_phase(&empty[s], ph, deadline))) break;
      const uint32_t dst = smem_u32(ring + (size_t)s * L::STAGE), bar = smem_u32(&full[s]);
      mbar_arrive_expect_tx(&full[s], L::STAGE);
      tma_2d(dst, &tw, c * (int)KST, n0, bar);
      tma_2d(dst + 64 * KST, &tw, c * (int)KST, p.swiglu ? p.n + n0 : n0 + 64, bar);
      tma_2d(dst + L::A_BYTES, &ta, c * (int)KST, m0, bar);
      if (++s == L::NS) s = 0, ph ^= 1;
    }
    if (!ok) {                                            // copies still in flight land before the CTA leaves
      const uint64_t grace = globaltimer_ns() + timeout;
      for (int i = 0; i < L::NS; ++i) wait_phase(&full[i], 0, grace);
    }
  } else if (warp == 1 && lane == 0) {
    int s = 0;
    uint32_t ph = 0;
    for (int c = c0; c < c1; ++c) {
      if (!(ok = wait_phase(&full[s], ph, deadline))) break;
      tc::fence_after_sync();
      const uint64_t da = sdesc128(smem_u32(ring + (size_t)s * L::STAGE)), db = da + (L::A_BYTES >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_i8<1>(tmem, da + 2 * j, db + 2 * j, idesc_i8(128, BN), c > c0 || j > 0);
      tc::commit(&empty[s]);
      if (++s == L::NS) s = 0, ph ^= 1;
    }
    tc::commit(&done);
  }
  __syncwarp();
  const int cols = min(BN, p.m - m0);                     // tokens of the tile
  int32_t* red = reinterpret_cast<int32_t*>(ring);        // [token][128 weight rows]
  if (warp >= 2) {
    ok = wait_phase(&done, 0, deadline + timeout);
    tc::fence_after_sync();
    if (__all_sync(0xffffffffu, ok)) {
      const int q = warp & 3;
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        int32_t v[16];
        tm_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < cols) red[(c + i) * 128 + q * 32 + lane] = v[i];
      }
    }
    tc::fence_before_sync();
  }
  if (pieces > 1) cluster_sync(); else __syncthreads();
  // items: (token, four weight rows), dealt to the cluster's CTAs in even runs
  const int per = half / 4, items = cols * per;
  const int i0 = items * rank / pieces, i1 = items * (rank + 1) / pieces;
  const uint32_t mine = smem_u32(red);
  for (int i = i0 + (int)threadIdx.x; i < i1; i += SPLIT_THR) {
    const int t = i / per, r = (i - t * per) * 4, n = n0 + r;
    int4 g = make_int4(0, 0, 0, 0), u = g;
    for (int s = 0; s < pieces; ++s) {
      const uint32_t at = (pieces > 1 ? mapa(mine, s) : mine) + (uint32_t)(t * 128 + r) * 4u;
      const int4 a = ld_cluster_int4(at);
      g.x += a.x; g.y += a.y; g.z += a.z; g.w += a.w;
      if (p.swiglu) {
        const int4 b = ld_cluster_int4(at + 64 * 4);
        u.x += b.x; u.y += b.y; u.z += b.z; u.w += b.w;
      }
    }
    const float sa = p.sa[m0 + t];
    const int gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (n + j >= p.n) break;
      float v = scaled(gv[j], sa, __ldg(&p.sw[n + j]));
      if (p.swiglu) v = swiglu(v, scaled(uv[j], sa, __ldg(&p.sw[p.n + n + j])), p.limit, p.has_limit);
      store_out(p.out, (int64_t)(m0 + t) * p.os + n + j, p.type, v);
    }
  }
  if (pieces > 1) cluster_sync(); else __syncthreads();   // the others have read this CTA's sums
  if (warp == 1) tc::tmem_dealloc(tmem, L::COLS);
}

// ------------------------------------------------------------------ many tokens
// Barrier of the 128 epilogue threads that also ANDs a predicate, so that all of
// them leave together after a wait that ran out for one.
__device__ __forceinline__ bool epilogue_and(bool pred) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.and.pred q, 1, 128, p; selp.u32 %0, 1, 0, q; }"
               : "=r"(r)
               : "r"((uint32_t)pred)
               : "memory");
  return r != 0u;
}

template <int BN>
struct Pair {
  static constexpr uint32_t A_BYTES = 128 * KST, B_BYTES = BN / 2 * KST, STAGE = A_BYTES + B_BYTES;
  static constexpr int NS = BN == 256 ? 6 : 8;
  static constexpr uint32_t COLS = 2 * BN;
  static constexpr size_t SMEM = NS * STAGE + 1024;
};
constexpr int PAIR_THR = 192;

// A pair of CTAs (the cluster) works on tiles of 256 tokens x BN weight rows:
// CTA r holds tokens [128 r, 128 r + 128) and weight rows [BN/2 r, BN/2 (r + 1))
// of the tile in its shared memory and its tokens' accumulators in its TMEM; CTA
// 0's warp 1 issues the MMAs of both. With SwiGLU the tile's weight rows are BN/2
// gate rows (CTA 0's copies) and their up rows (CTA 1's).
template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THR, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap ta, Args p, int tiles_m,
                int tiles, uint64_t timeout) {
  using L = Pair<BN>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[L::NS], empty[L::NS], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem;
  __shared__ __align__(16) float sws[2][BN];
  uint8_t* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int chunks = (p.k + (int)KST - 1) / (int)KST;
  const int cols = p.swiglu ? BN / 2 : BN;                // output columns of a tile
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);
    }
    mbar_init(&drained, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem)),
                 "r"(L::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  tc::fence_before_sync();
  cluster_sync();
  tc::fence_after_sync();
  const uint64_t deadline = globaltimer_ns() + timeout;
  bool ok = true;
  if (warp == 0 && lane == 0) {
    int s = 0;
    uint32_t ph = 1;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      const int m0 = tile % tiles_m * 256 + (int)rank * 128;
      const int nt = tile / tiles_m * cols;
      const int n0 = rank == 0 ? nt : p.swiglu ? p.n + nt : nt + BN / 2;
      for (int c = 0; c < chunks; ++c) {
        if (!(ok = wait_phase(&empty[s], ph, deadline))) break;
        const uint32_t dst = smem_u32(ring + (size_t)s * L::STAGE), bar = mapa(smem_u32(&full[s]), 0);
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE);
        tma_2d_pair(dst, &ta, c * (int)KST, m0, bar);
        tma_2d_pair(dst + L::A_BYTES, &tw, c * (int)KST, n0, bar);
        if (++s == L::NS) s = 0, ph ^= 1;
      }
    }
    // Copies still in flight after a wait that ran out count on CTA 0's barriers;
    // the cluster barrier below holds CTA 1 until CTA 0 has waited for them.
    if (!ok && rank == 0) {
      const uint64_t grace = globaltimer_ns() + timeout;
      for (int i = 0; i < L::NS; ++i) wait_phase(&full[i], 0, grace);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    int s = 0, it = 0;
    uint32_t ph = 0;
    for (int tile = pair; ok && tile < tiles; tile += pairs, ++it) {
      const int b = it & 1;
      if (!(ok = wait_phase(&acc_empty[b], ((it >> 1) & 1) ^ 1, deadline))) break;
      tc::fence_after_sync();
      for (int c = 0; c < chunks; ++c) {
        if (!(ok = wait_phase(&full[s], ph, deadline))) break;
        tc::fence_after_sync();
        const uint64_t da = sdesc128(smem_u32(ring + (size_t)s * L::STAGE)), db = da + (L::A_BYTES >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_i8<2>(tmem + (uint32_t)(b * BN), da + 2 * j, db + 2 * j, idesc_i8(256, BN), c > 0 || j > 0);
        commit_pair(&empty[s]);
        if (++s == L::NS) s = 0, ph ^= 1;
      }
      commit_pair(&acc_full[b]);
    }
    commit_pair(&drained);
    wait_phase(&drained, 0, deadline + timeout);          // no MMA is in flight when TMEM is released
  } else if (warp >= 2) {
    const int q = warp & 3, et = threadIdx.x - 64;
    const int osz = p.type == QX_T_F32 ? 4 : 2;
    const bool vec = (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0 && (p.os * osz) % 16 == 0;
    int it = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++it) {
      const int b = it & 1;
      const int n0 = tile / tiles_m * cols;
      const int64_t row = (int64_t)(tile % tiles_m) * 256 + rank * 128 + q * 32 + lane;
      for (int i = et; i < BN; i += 128) {
        const int n = n0 + (i < cols ? i : i - cols);
        sws[b][i] = n < p.n ? __ldg(&p.sw[i < cols ? n : p.n + n]) : 0.f;
      }
      const float sa = row < p.m ? __ldg(&p.sa[row]) : 0.f;
      ok = wait_phase(&acc_full[b], (it >> 1) & 1, deadline);
      if (!epilogue_and(ok)) break;                       // also: sws of this tile is written
      tc::fence_after_sync();
      const uint32_t t0 = tmem + (uint32_t)(b * BN) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        int32_t g[16], u[16];
        tm_ld16(t0 + c, g);
        if (p.swiglu) tm_ld16(t0 + BN / 2 + c, u);
        if (row < p.m) {
#pragma unroll
          for (int h = 0; h < 16; h += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] = scaled(g[h + j], sa, sws[b][c + h + j]);
              if (p.swiglu)
                v[j] = swiglu(v[j], scaled(u[h + j], sa, sws[b][BN / 2 + c + h + j]), p.limit, p.has_limit);
            }
            store8(p, row, n0 + c + h, v, vec);
          }
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_cluster(mapa(smem_u32(&acc_empty[b]), 0));
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  cluster_sync();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::COLS) : "memory");
}

}  // namespace i8
}  // namespace qx
