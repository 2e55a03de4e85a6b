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
__device__ __forceinline__ void tm_ld32(uint32_t taddr, int32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t taddr, int32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Two outputs of a 16-bit type in one word.
__device__ __forceinline__ uint32_t pack2(int type, float a, float b) {
  if (type == QX_T_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
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
                                                          int prefetch, uint64_t timeout) {
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
  pdl_launch_dependents();
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
    auto weights = [&](int c, int s) {
      const uint32_t dst = smem_u32(ring + (size_t)s * L::STAGE), bar = smem_u32(&full[s]);
      mbar_arrive_expect_tx(&full[s], L::STAGE);
      tma_2d(dst, &tw, c * (int)KST, n0, bar);
      tma_2d(dst + 64 * KST, &tw, c * (int)KST, p.swiglu ? p.n + n0 : n0 + 64, bar);
    };
    const int ahead = prefetch ? min(L::NS, c1 - c0) : 0;
    for (int s = 0; s < ahead; ++s) weights(c0 + s, s);
    pdl_wait();
    int s = 0;
    uint32_t ph = 1;
    for (int c = c0; c < c1; ++c) {
      if (!(ok = wait_phase(&empty[s], ph, deadline))) break;
      if (c - c0 >= ahead) weights(c, s);
      tma_2d(smem_u32(ring + (size_t)s * L::STAGE) + L::A_BYTES, &ta, c * (int)KST, m0, smem_u32(&full[s]));
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
  pdl_wait();                                             // the tokens' scales, and the output's place
  if (pieces > 1) cluster_sync(); else __syncthreads();
  // items: (token, four weight rows), dealt to the cluster's CTAs in even runs
  const int per = half / 4, items = cols * per;
  const int i0 = items * rank / pieces, i1 = items * (rank + 1) / pieces;
  const uint32_t mine = smem_u32(red);
  const int four = p.type == QX_T_F32 ? 16 : 8;           // bytes of four outputs
  const bool vec = reinterpret_cast<uintptr_t>(p.out) % four == 0 && p.os % 4 == 0;
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
    const float sa = __ldcg(&p.sa[m0 + t]);
    const int gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int nj = min(n + j, p.n - 1);
      v[j] = scaled(gv[j], sa, __ldcg(&p.sw[nj]));
      if (p.swiglu) v[j] = swiglu(v[j], scaled(uv[j], sa, __ldcg(&p.sw[p.n + nj])), p.limit, p.has_limit);
    }
    const int64_t at = (int64_t)(m0 + t) * p.os + n;
    if (vec && n + 4 <= p.n) {
      if (p.type == QX_T_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
      else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) =
               make_uint2(pack2(p.type, v[0], v[1]), pack2(p.type, v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < p.n) store_out(p.out, at + j, p.type, v[j]);
    }
  }
  if (pieces > 1) cluster_sync(); else __syncthreads();   // the others have read this CTA's sums
  if (warp == 1) tc::tmem_dealloc(tmem, L::COLS);
}

// ------------------------------------------------------------------ many tokens
// Barrier of the 256 epilogue threads that also ANDs a predicate, so that all of
// them leave together after a wait that ran out for one.
__device__ __forceinline__ bool epilogue_and(bool pred) {
  uint32_t r;
  asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.and.pred q, 1, 256, p; selp.u32 %0, 1, 0, q; }"
               : "=r"(r)
               : "r"((uint32_t)pred)
               : "memory");
  return r != 0u;
}

// Staging row of one token: 32 outputs, padded so that 16-byte accesses of
// consecutive rows fall into different banks (144 bytes for FP32, 80 for 16-bit types).
constexpr int PAIR_ROW = 32 * 4 + 16;

// 32 tokens x 32 output columns from column n on, each lane holding its token's
// values: through shared memory, so that a warp's stores cover whole row segments
// (16 bytes per lane where the rows are aligned, else one element per lane).
__device__ __forceinline__ void store_block(const Args& p, uint8_t* stage, int64_t row0, int n, const float (&v)[32],
                                            bool vec, int lane) {
  const bool wide = p.type == QX_T_F32;
  const int rowb = wide ? PAIR_ROW : 32 * 2 + 16;
  uint8_t* mine = stage + lane * rowb;
  if (wide) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      *reinterpret_cast<float4*>(mine + 4 * j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 8)
      *reinterpret_cast<uint4*>(mine + 2 * j) =
          make_uint4(pack2(p.type, v[j], v[j + 1]), pack2(p.type, v[j + 2], v[j + 3]), pack2(p.type, v[j + 4], v[j + 5]),
                     pack2(p.type, v[j + 6], v[j + 7]));
  }
  __syncwarp();
  const int rows = (int)min((int64_t)32, p.m - row0), cols = min(32, p.n - n);
  const int osz = wide ? 4 : 2;
  uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + (row0 * p.os + n) * osz;
  if (vec && cols == 32) {
    const int per = wide ? 8 : 4, part = lane % per;      // lanes per row segment
#pragma unroll 4
    for (int r = lane / per; r < rows; r += 32 / per)
      *reinterpret_cast<uint4*>(out + (int64_t)r * p.os * osz + part * 16) =
          *reinterpret_cast<const uint4*>(stage + r * rowb + part * 16);
  } else if (lane < cols) {
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      if (wide) *reinterpret_cast<float*>(out + ((int64_t)r * p.os + lane) * 4) =
                    *reinterpret_cast<const float*>(stage + r * rowb + lane * 4);
      else *reinterpret_cast<uint16_t*>(out + ((int64_t)r * p.os + lane) * 2) =
               *reinterpret_cast<const uint16_t*>(stage + r * rowb + lane * 2);
    }
  }
  __syncwarp();
}

// Epilogue warps: two per quarter of the accumulator's lanes, each half of the columns
// (one per quarter kept the tensor cores waiting: 87 us against 79 at 8192 x 5120 x 2304).
constexpr int PAIR_EPI = 8;

// The scaled values of two neighbouring columns (packed multiplications, each
// rounded as the scalar ones are).
__device__ __forceinline__ float2 scaled2(int32_t a, int32_t b, float sa, float2 sw) {
  uint64_t v, t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(__int2float_rn(a)), "f"(__int2float_rn(b)));
  asm("mov.b64 %0, {%1, %1};" : "=l"(t) : "f"(sa));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(t));
  asm("mov.b64 %0, {%1, %2};" : "=l"(t) : "f"(sw.x), "f"(sw.y));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(t));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

template <int BN>
struct Pair {
  static constexpr uint32_t A_BYTES = 128 * KST, B_BYTES = BN / 2 * KST, STAGE = A_BYTES + B_BYTES;
  static constexpr int NS = BN == 256 ? 5 : 7;
  static constexpr uint32_t COLS = 2 * BN;
  // ring, the epilogue warps' staging rows, alignment of the swizzled tiles
  static constexpr size_t SMEM = NS * STAGE + PAIR_EPI * 32 * PAIR_ROW + 1024;
};
constexpr int PAIR_THR = 64 + 32 * PAIR_EPI;

// A pair of CTAs (the cluster) works on tiles of 256 tokens x BN weight rows:
// CTA r holds tokens [128 r, 128 r + 128) and weight rows [BN/2 r, BN/2 (r + 1))
// of the tile in its shared memory and its tokens' accumulators in its TMEM; CTA
// 0's warp 1 issues the MMAs of both. With SwiGLU the tile's weight rows are BN/2
// gate rows (CTA 0's copies) and their up rows (CTA 1's).
template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THR, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap ta, Args p, int tiles_m,
                int tiles, int prefetch, uint64_t timeout) {
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
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * PAIR_EPI);
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
    auto weights = [&](int tile, int c, int s) {
      const int nt = tile / tiles_m * cols;
      const int n0 = rank == 0 ? nt : p.swiglu ? p.n + nt : nt + BN / 2;
      if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE);
      tma_2d_pair(smem_u32(ring + (size_t)s * L::STAGE) + L::A_BYTES, &tw, c * (int)KST, n0, mapa(smem_u32(&full[s]), 0));
    };
    int ahead = prefetch ? min(L::NS, chunks) : 0;        // stages whose weights are on their way
    for (int s = 0; s < ahead; ++s) weights(pair, s, s);
    pdl_wait();
    int s = 0;
    uint32_t ph = 1;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      const int m0 = tile % tiles_m * 256 + (int)rank * 128;
      for (int c = 0; c < chunks; ++c) {
        if (!(ok = wait_phase(&empty[s], ph, deadline))) break;
        if (ahead > 0) --ahead;
        else weights(tile, c, s);
        tma_2d_pair(smem_u32(ring + (size_t)s * L::STAGE), &ta, c * (int)KST, m0, mapa(smem_u32(&full[s]), 0));
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
    uint8_t* stage = ring + L::NS * L::STAGE + (warp - 2) * 32 * PAIR_ROW;
    const int c_lo = warp >= 6 ? cols / 2 : 0, c_hi = c_lo + cols / 2;
    pdl_wait();                                           // the tokens' scales, and the output's place
    auto row_of = [&](int tile) { return (int64_t)(tile % tiles_m) * 256 + rank * 128 + q * 32; };
    // one tile ahead: thread et's weight scale and the lane's token scale
    auto scale_w = [&](int tile) {
      const int n = tile / tiles_m * cols + (et < cols ? et : et - cols);
      return tile < tiles && et < BN && n < p.n ? __ldcg(&p.sw[et < cols ? n : p.n + n]) : 0.f;
    };
    auto scale_a = [&](int tile) {
      return tile < tiles && row_of(tile) + lane < p.m ? __ldcg(&p.sa[row_of(tile) + lane]) : 0.f;
    };
    float next_w = scale_w(pair), next_a = scale_a(pair);
    int it = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++it) {
      const int b = it & 1;
      const int n0 = tile / tiles_m * cols;
      const int64_t row0 = row_of(tile);
      const float sa = next_a;
      if (et < BN) sws[b][et] = next_w;
      next_w = scale_w(tile + pairs);
      next_a = scale_a(tile + pairs);
      ok = wait_phase(&acc_full[b], (it >> 1) & 1, deadline);
      if (!epilogue_and(ok)) break;                       // also: sws of this tile is written
      tc::fence_after_sync();
      const uint32_t t0 = tmem + (uint32_t)(b * BN) + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
      for (int c = c_lo; c < c_hi && n0 + c < p.n; c += 32) {
        int32_t g[32];
        float v[32];
        tm_ld32(t0 + c, g);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 r = scaled2(g[j], g[j + 1], sa, *reinterpret_cast<const float2*>(&sws[b][c + j]));
          v[j] = r.x;
          v[j + 1] = r.y;
        }
        if (p.swiglu) {
          tm_ld32(t0 + BN / 2 + c, g);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 r = scaled2(g[j], g[j + 1], sa, *reinterpret_cast<const float2*>(&sws[b][BN / 2 + c + j]));
            v[j] = swiglu(v[j], r.x, p.limit, p.has_limit);
            v[j + 1] = swiglu(v[j + 1], r.y, p.limit, p.has_limit);
          }
        }
        if (row0 < p.m) store_block(p, stage, row0, n0 + c, v, vec, lane);
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
