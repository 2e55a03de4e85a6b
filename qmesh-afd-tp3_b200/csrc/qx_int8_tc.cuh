// Tensor-core kernels of the int8 product (tcgen05.mma.kind::i8, int8 x int8
// into int32 accumulators in TMEM), operands brought in by tiled TMA copies with
// the 128-byte swizzle: a stage of the shared-memory ring is one or two spans of 128
// bytes of K of the operand tiles' rows, four MMAs of K = 32 each.
//
//   split_kernel  few tokens: weights are the M = 128 operand, tokens the N
//                 operand, and the CTAs of a cluster split K (their sums, whole
//                 numbers, meet over distributed shared memory).
//   pair_kernel   many tokens: persistent pairs of CTAs (cta_group::2), 256
//                 tokens x up to 256 weight rows per tile, two accumulators so that
//                 one tile's epilogue runs under the next one's MMAs.
#pragma once

#include <cuda.h>

#include "qx_tc.cuh"

namespace qx {
namespace i8 {

// K bytes of one tiled copy: a swizzle span. K past the end reads as 0.
constexpr uint32_t KST = 128;

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

// One lane of a converged warp, chosen so that the compiler knows it is one: the
// copies and MMAs of a lane picked by its number go through a loop over the
// active lanes (about 80 cycles each).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0u;
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
// The barrier in two halves and without memory order: nothing that was written before
// it is read after it, and the ordered form would wait for the global stores (2 us).
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int32_t v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// Arrive on another CTA's barrier. CTA scope: it says that accumulator reads are
// done and publishes no memory; at cluster scope it would first wait for this
// thread's global stores (1,400 cycles per tile).
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrive on `bar` in both CTAs of the pair when the tcgen05 operations issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ bool try_phase(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0u;
}

// Bounded wait: false once `limit` ns have passed, with QX_DEV_TIMEOUT recorded; the
// caller then stops consuming. The time runs from this wait's own start, and no thread
// waits here for what depends on the kernel in front before that one has ended
// (pdl_wait), so neither a long product nor a long kernel in front uses it up.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, uint64_t limit) {
  const uint64_t deadline = globaltimer_ns() + limit;
  for (uint32_t it = 0;; ++it) {
    if (try_phase(bar, parity)) return true;
    if ((it & 15u) == 15u && globaltimer_ns() > deadline) {
      atomicOr(&g_status, (uint32_t)QX_DEV_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, uint64_t limit) {
  return try_phase(bar, parity) || wait_long(bar, parity, limit);
}

// Bytes that stand for copies which were never issued.
__device__ __forceinline__ void complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// After the MMA thread has given up: waits (each bounded) until the copies in flight have
// landed, so that none writes into shared memory after the CTAs have left. A stage's fill
// is brought in by n copy threads, weights and tokens in turn, thread i having issued its
// `wb` or `tb` bytes of the first issued[i] fills; thread 0 also announces the bytes of all.
// No thread is more than one round of the ring ahead of the MMAs, so the last ns fills are
// in ns different stages. A fill that only some threads have issued is made to complete with
// those: the bytes of the others are counted as if they had come, or, where thread 0 is
// behind, the bytes that are under way are announced in its place.
__device__ __noinline__ void drain_copies(uint64_t* full, uint32_t ns, const uint32_t* issued, int n, uint32_t wb,
                                          uint32_t tb, uint64_t timeout) {
  uint32_t last = 0;
  for (int i = 0; i < n; ++i) last = max(last, issued[i]);
  for (uint32_t f = last > ns ? last - ns : 0u; f < last; ++f) {
    uint32_t in = 0, out = 0;
    for (int i = 0; i < n; ++i) (f < issued[i] ? in : out) += i & 1 ? tb : wb;
    uint64_t* bar = &full[f % ns];
    if (f >= issued[0]) mbar_arrive_expect_tx(bar, in);
    else if (out) complete_tx(bar, out);
    wait_phase(bar, (f / ns) & 1, timeout);
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
// Grid: (row tile of 128 weight rows) x (K piece), all tokens in one tile of BN, the K
// pieces of a row tile in one cluster. Warps 0 and 6 copy weights and tokens (one
// thread's copies for both took longer than their flight), warp 1 issues the MMAs.
// Token t's sums meet in CTA t mod pieces: warps 2-5 of every CTA store theirs into
// that CTA's shared memory, which adds them and writes the outputs. (Reading the
// others' sums instead needs a second cluster barrier before a CTA may leave, 1.5 us.)
// With SwiGLU the 128 rows are 64 gate rows and their 64 up rows. The weights' bytes
// bound it, and at a few us the launch: 4608 x 5120 for one token streams 23.6 MB in
// 3.8 of the kernel's 7.7 us. The ring takes half an SM, so that two CTAs run side by side.
template <int BN>
struct Split {
  static constexpr uint32_t A_BYTES = 128 * KST, STAGE = A_BYTES + BN * KST;
  static constexpr uint32_t COLS = BN < 32 ? 32 : BN;
  static constexpr uint32_t SUMS = (BN + 8) * 512;       // [piece][own token][128 rows], up to 8 pieces
  static constexpr int NS = (114688 - SUMS) / STAGE;     // two CTAs per SM
  static constexpr size_t SMEM = (size_t)NS * STAGE + SUMS + 1024;   // 1024: alignment of the swizzled tiles
};
constexpr int SPLIT_THR = 224;

template <int BN>
__global__ void __launch_bounds__(SPLIT_THR) split_kernel(const __grid_constant__ CUtensorMap tw,
                                                          const __grid_constant__ CUtensorMap ta, Args p, int pieces,
                                                          int prefetch, uint64_t timeout, int hold) {
  using L = Split<BN>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[L::NS], empty[L::NS], done;
  __shared__ uint32_t tmem, gave_up, issued[2];          // issued: fills whose weights, tokens were sent for
  uint8_t* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const uint32_t sums = smem_u32(ring) + L::NS * L::STAGE;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int half = p.swiglu ? 64 : 128;                  // output columns of a tile
  const int n0 = (int)(blockIdx.x / pieces) * half;
  const int chunks = (p.k + (int)KST - 1) / (int)KST;
  const int c0 = chunks * rank / pieces, c1 = chunks * (rank + 1) / pieces;
  const int own = (p.m + pieces - 1) / pieces;           // tokens per CTA at most
  pdl_launch_dependents();
  cluster_arrive_relaxed();                              // this CTA's shared memory may be written
  if (threadIdx.x == 0) {
    prefetch_map(&tw);
    prefetch_map(&ta);
    for (int s = 0; s < L::NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, hold == 1 ? 2 : 1);
    gave_up = issued[0] = issued[1] = 0;
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
  bool ok = true;
  uint32_t fills = 0;                                     // of a copy thread: stages it has sent for
  if (warp == 0 && elect_one()) {
    if (!prefetch) pdl_wait();
    const uint32_t base = smem_u32(ring), bars = smem_u32(full);
    int s = 0;
    uint32_t ph = 1;
    for (int c = c0; c < c1; ++c) {
      if (c == c0 + L::NS) pdl_wait();
      if (!(ok = wait_phase(&empty[s], ph, timeout))) break;
      mbar_arrive_expect_tx(&full[s], L::STAGE);
      tma_2d(base + s * L::STAGE, &tw, c * (int)KST, n0, bars + 8 * s);
      if (p.swiglu) tma_2d(base + s * L::STAGE + 64 * KST, &tw, c * (int)KST, p.n + n0, bars + 8 * s);
      ++fills;
      if (++s == L::NS) s = 0, ph ^= 1;
    }
  } else if (warp == 6 && elect_one()) {
    pdl_wait();
    const uint32_t base = smem_u32(ring) + L::A_BYTES, bars = smem_u32(full);
    int s = 0;
    uint32_t ph = 1;
    for (int c = c0; c < c1; ++c) {
      if (!(ok = wait_phase(&empty[s], ph, timeout))) break;
      tma_2d(base + s * L::STAGE, &ta, c * (int)KST, 0, bars + 8 * s);
      ++fills;
      if (++s == L::NS) s = 0, ph ^= 1;
    }
  } else if (warp == 1 && elect_one()) {
    pdl_wait();
    int s = 0;
    uint32_t ph = 0;
    if (hold == 2) ok = wait_phase(&done, 0, timeout);
    for (int c = c0; ok && c < c1; ++c) {
      if (!(ok = wait_phase(&full[s], ph, timeout))) break;
      tc::fence_after_sync();
      const uint64_t da = sdesc128(smem_u32(ring) + s * L::STAGE), db = da + (L::A_BYTES >> 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_i8<1>(tmem, da + 2 * j, db + 2 * j, idesc_i8(128, BN), c > c0 || j > 0);
      tc::commit(&empty[s]);
      if (++s == L::NS) s = 0, ph ^= 1;
    }
    if (!ok) gave_up = 1;
    tc::commit(&done);
  }
  __syncwarp();
  const bool epi = warp >= 2 && warp < 6;
  pdl_wait();                                             // also: the tokens' scales, and the output's place
  if (epi) ok = wait_phase(&done, 0, 2 * timeout);
  __syncwarp();                                           // a warp's lanes may have polled a different number of times
  cluster_wait();                                         // every CTA of the cluster has started
  if (epi && __all_sync(0xffffffffu, ok)) {
    tc::fence_after_sync();
    const int q = warp & 3;
    uint32_t to = sums + (uint32_t)(rank * own * 128 + q * 32 + lane) * 4u;   // token t's place in its CTA
    int dst = 0;                                          // t mod pieces
#pragma unroll 1
    for (int c = 0; c < p.m; c += 16) {
      int32_t v[16];
      tm_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (c + i < p.m) {
          st_cluster(mapa(to, dst), v[i]);
          if (++dst == pieces) dst = 0, to += 512;
        }
      }
    }
    tc::fence_before_sync();
  }
  cluster_sync();
  if (warp == 1) tc::tmem_dealloc(tmem, L::COLS);
  if (gave_up) {                                          // copies may still be in flight to this CTA
    if (fills) issued[warp == 0 ? 0 : 1] = fills;
    __syncthreads();
    if (threadIdx.x == 0) drain_copies(full, L::NS, issued, 2, L::A_BYTES, L::STAGE - L::A_BYTES, timeout);
  }
  // items of this CTA: (own token, four weight rows)
  const int per = half / 4, items = (p.m - rank + pieces - 1) / pieces * per;
  const int four = p.type == QX_T_F32 ? 16 : 8;           // bytes of four outputs
  const bool vec = reinterpret_cast<uintptr_t>(p.out) % four == 0 && p.os % 4 == 0;
  const int32_t* sum = reinterpret_cast<const int32_t*>(ring + L::NS * L::STAGE);
  for (int i = threadIdx.x; i < items; i += SPLIT_THR) {
    const int tl = i / per, r = (i - tl * per) * 4, n = n0 + r, t = tl * pieces + rank;
    int4 g = make_int4(0, 0, 0, 0), u = g;
    for (int s = 0; s < pieces; ++s) {
      const int32_t* from = sum + (s * own + tl) * 128 + r;
      const int4 a = *reinterpret_cast<const int4*>(from);
      g.x += a.x; g.y += a.y; g.z += a.z; g.w += a.w;
      if (p.swiglu) {
        const int4 b = *reinterpret_cast<const int4*>(from + 64);
        u.x += b.x; u.y += b.y; u.z += b.z; u.w += b.w;
      }
    }
    const float sa = __ldcg(&p.sa[t]);
    const int gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int nj = min(n + j, p.n - 1);
      v[j] = scaled(gv[j], sa, __ldcg(&p.sw[nj]));
      if (p.swiglu) v[j] = swiglu(v[j], scaled(uv[j], sa, __ldcg(&p.sw[p.n + nj])), p.limit, p.has_limit);
    }
    const int64_t at = (int64_t)t * p.os + n;
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

// Output staging of one epilogue warp: 32 tokens x 64 bytes (32 outputs of a 16-bit
// type, 16 FP32), 16-byte pieces permuted as the copy engine's 64-byte swizzle does
// (piece j of row r at j ^ (r / 2 mod 4)), which also keeps the lanes' accesses in
// different banks. Two buffers, so that a store drains while the next block is written.
constexpr int PAIR_BLOCK = 32 * 64;

// Up to 32 tokens (rows) x COLS output columns from column n on, each lane holding its
// token's values. Rows on 16-byte boundaries (tma): one tiled store, which leaves out rows
// past the tensor's end, but writes its last columns in whole pieces of 16 bytes: a block
// whose row ends inside such a piece, and rows on other boundaries, are stored element by
// element, 64 bytes of a row at a time.
template <int COLS>
__device__ __forceinline__ void store_block(const Args& p, const CUtensorMap* to, uint8_t* stage, int64_t row0, int rows,
                                            int n, const float* v, int tma, int lane) {
  constexpr int OSZ = 64 / COLS;
  uint8_t* mine = stage + lane * 64;
  const int sw = (lane >> 1) & 3;
  if (tma) {                                             // the store before last has left this buffer
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (OSZ == 4)
      *reinterpret_cast<float4*>(mine + 16 * (j ^ sw)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    else
      *reinterpret_cast<uint4*>(mine + 16 * (j ^ sw)) =
          make_uint4(pack2(p.type, v[8 * j], v[8 * j + 1]), pack2(p.type, v[8 * j + 2], v[8 * j + 3]),
                     pack2(p.type, v[8 * j + 4], v[8 * j + 5]), pack2(p.type, v[8 * j + 6], v[8 * j + 7]));
  }
  if (tma && (n + COLS <= p.n || p.n * OSZ % 16 == 0)) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(to), "r"(n),
                   "r"((int)row0), "r"(smem_u32(stage))
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return;
  }
  __syncwarp();
  const int c = lane % COLS;
  const int64_t step = p.os * OSZ;
  uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + row0 * step + (int64_t)(n + c) * OSZ;
  if (n + c < p.n) {
#pragma unroll 4
    for (int r = lane / COLS; r < rows; r += 32 / COLS) {
      const uint8_t* from = stage + r * 64 + 16 * ((c * OSZ / 16) ^ ((r >> 1) & 3)) + c * OSZ % 16;
      if constexpr (OSZ == 4) *reinterpret_cast<float*>(out + r * step) = *reinterpret_cast<const float*>(from);
      else *reinterpret_cast<uint16_t*>(out + r * step) = *reinterpret_cast<const uint16_t*>(from);
    }
  }
  __syncwarp();
  // An empty group stands for this block, so that the next wait still counts two buffers.
  if (tma && lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// Epilogue warps: two per quarter of the accumulator's lanes.
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

constexpr size_t PAIR_RING = 196608;
constexpr int MAX_NS = 12;               // stages of the pair kernel's ring at most
// ring, the epilogue warps' staging blocks, alignment of the swizzled tiles
constexpr size_t PAIR_SMEM = PAIR_RING + PAIR_EPI * 2 * PAIR_BLOCK + 1024;
constexpr int PAIR_THR = 96 + 32 * PAIR_EPI;         // weight copies, MMAs, epilogue, token copies
static_assert(PAIR_SMEM + 1536 <= 232448, "with the static part, one SM's memory");

// A pair of CTAs (the cluster) works on tiles of 2 tb tokens x bn weight rows (tb a
// multiple of 32, at most 128; bn a multiple of 32, of 64 with SwiGLU, at most 256):
// CTA r holds tokens [tb r, tb (r + 1)) and weight rows [bn/2 r, bn/2 (r + 1)) of the
// tile in its shared memory and its tokens' accumulators in its TMEM; CTA 0's warp 1
// issues the MMAs of both (always M = 256: the rows from tb on read whatever follows
// in shared memory and are not used). With SwiGLU the tile's weight rows are bn/2 gate
// rows (CTA 0's copies) and their up rows (CTA 1's). The ring holds as many stages as
// fit (6 of one span for tb = 128, bn = 256). Measured: 8192 x 5120 x 5120 160 us, the
// power cap's rate; 8192 x 5120 x 2304 68 us (2.8 POP/s); 2048 x 5120 x 2304 20.6. Tiles of 512 tokens (every weight copy used twice, one
// accumulator per block) were slower from 2048 tokens up: their epilogues run alone,
// and all at once.
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THR, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap ta,
                const __grid_constant__ CUtensorMap to, Args p, int tb, int bn, int spans, int tiles_m, int tiles,
                int prefetch, int tma, uint64_t timeout, int hold) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[MAX_NS], empty[MAX_NS], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem, gave_up, issued[4];          // issued: as in the other kernel, by CTA 0's copies, then CTA 1's
  __shared__ __align__(16) float sws[256];              // the tile's weight scales
  uint8_t* ring = raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int kst = spans * (int)KST, stages = (p.k + kst - 1) / kst;   // K of a stage, stages of a tile
  const int cols = p.swiglu ? bn / 2 : bn;                // output columns of a tile
  // a stage: its spans of the tokens, then of the weight rows
  const uint32_t a_span = (uint32_t)tb * KST, b_span = (uint32_t)bn / 2 * KST;
  const uint32_t stage_bytes = spans * (a_span + b_span);
  const int ns = min(MAX_NS, (int)(PAIR_RING / stage_bytes));
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_map(&tw);
    prefetch_map(&ta);
    if (tma) prefetch_map(&to);
    for (int s = 0; s < ns; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], hold == 1 ? 2 : 1);
      mbar_init(&acc_empty[b], 2 * PAIR_EPI);
    }
    mbar_init(&drained, 1);
    gave_up = issued[0] = issued[1] = issued[2] = issued[3] = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  tc::fence_before_sync();
  cluster_sync();
  tc::fence_after_sync();
  bool ok = true;
  uint32_t fills = 0;                                     // of a copy thread: stages it has sent for
  if (warp == 0 && elect_one()) {
    const uint32_t bytes = 2 * stage_bytes;               // both CTAs' copies
    // Weights (and CTA 0's count of both CTAs' bytes of a stage). Weights that are
    // complete already need not wait for the kernel in front.
    if (!prefetch) pdl_wait();
    const uint32_t base = smem_u32(ring) + spans * a_span, bars = mapa(smem_u32(full), 0);
    int s = 0;
    uint32_t ph = 1;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      const int nt = tile / tiles_m * cols;
      const int n0 = rank == 0 ? nt : p.swiglu ? p.n + nt : nt + bn / 2;
      for (int c = 0; c < stages; ++c) {
        if (tile > pair || c >= ns) pdl_wait();
        if (!(ok = wait_phase(&empty[s], ph, timeout))) break;
        if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
        for (int g = 0; g < spans; ++g)
          tma_2d_pair(base + s * stage_bytes + g * b_span, &tw, c * kst + g * (int)KST, n0, bars + 8 * s);
        ++fills;
        if (++s == ns) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 2 + PAIR_EPI && elect_one()) {
    pdl_wait();
    const uint32_t base = smem_u32(ring), bars = mapa(smem_u32(full), 0);
    int s = 0;
    uint32_t ph = 1;
    for (int tile = pair; ok && tile < tiles; tile += pairs) {
      const int m0 = (tile % tiles_m * 2 + (int)rank) * tb;
      for (int c = 0; c < stages; ++c) {
        if (!(ok = wait_phase(&empty[s], ph, timeout))) break;
        for (int g = 0; g < spans; ++g)
          tma_2d_pair(base + s * stage_bytes + g * a_span, &ta, c * kst + g * (int)KST, m0, bars + 8 * s);
        ++fills;
        if (++s == ns) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 1 && rank == 0 && elect_one()) {
    const uint32_t idesc = idesc_i8(256, (uint32_t)bn);
    pdl_wait();
    int s = 0, it = 0;
    uint32_t ph = 0;
    if (hold == 2) ok = wait_phase(&drained, 0, timeout);
    for (int tile = pair; ok && tile < tiles; tile += pairs, ++it) {
      const int b = it & 1;
      if (!(ok = wait_phase(&acc_empty[b], ((it >> 1) & 1) ^ 1, timeout))) break;
      tc::fence_after_sync();
      for (int c = 0; c < stages; ++c) {
        if (!(ok = wait_phase(&full[s], ph, timeout))) break;
        tc::fence_after_sync();
        const uint64_t da = sdesc128(smem_u32(ring) + s * stage_bytes), db = da + (spans * a_span >> 4);
        for (int g = 0; g < spans; ++g) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_i8<2>(tmem + (uint32_t)(b * 256), da + g * (a_span >> 4) + 2 * j, db + g * (b_span >> 4) + 2 * j, idesc,
                      c > 0 || g > 0 || j > 0);
        }
        commit_pair(&empty[s]);
        if (++s == ns) s = 0, ph ^= 1;
      }
      if (ok) commit_pair(&acc_full[b]);                  // else the tile's outputs are not written
    }
    if (!ok) {                                            // seen in both CTAs behind the cluster barrier below
      for (uint32_t r = 0; r < 2; ++r) st_cluster(mapa(smem_u32(&gave_up), r), 1);
      asm volatile("fence.acq_rel.cluster;" ::: "memory");
    }
    commit_pair(&drained);
    wait_phase(&drained, 0, 2 * timeout);          // no MMA is in flight when TMEM is released
  } else if (warp >= 2 && warp < 2 + PAIR_EPI) {
    const int q = warp & 3, et = threadIdx.x - 64, h = warp >= 6;   // lane quarter, thread, warp group
    uint8_t* stage = ring + PAIR_RING + (warp - 2) * 2 * PAIR_BLOCK;
    int buf = 0;
    pdl_wait();                                           // the tokens' scales, and the output's place
    // The scales one tile ahead: thread et's of a weight row, the lane's of a token.
    float next_w = 0.f, next_a = 0.f;
    int64_t next_row = 0;
    int next_n = 0;
    auto look_ahead = [&](int tile) {
      if (tile >= tiles) return;
      const int tn = tile / tiles_m, n = tn * cols + (et < cols ? et : et - cols);
      next_n = tn * cols;
      next_row = (int64_t)((tile - tn * tiles_m) * 2 + (int)rank) * tb + q * 32;
      next_w = et < bn && n < p.n ? __ldcg(&p.sw[et < cols ? n : p.n + n]) : 0.f;
      next_a = next_row + lane < p.m ? __ldcg(&p.sa[next_row + lane]) : 0.f;
    };
    look_ahead(pair);
    int it = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++it) {
      const int b = it & 1;                               // accumulator
      const int n0 = next_n;
      const int64_t row0 = next_row;
      const float sa = next_a;
      asm volatile("bar.sync 1, 256;" ::: "memory");      // the last tile's sws have been read
      sws[et] = next_w;
      look_ahead(tile + pairs);
      if (!epilogue_and(ok)) break;                       // this tile's sws are written; a wait that ran out ends all
      ok = __all_sync(0xffffffffu, wait_phase(&acc_full[b], (it >> 1) & 1, timeout));
      if (!ok) continue;
      tc::fence_after_sync();
      const uint32_t t0 = tmem + (uint32_t)(b * 256) + ((uint32_t)(q * 32) << 16);
      const int rows = q * 32 < tb ? (int)min((int64_t)32, p.m - row0) : 0;   // this warp's tokens
#pragma unroll 1
      for (int c = 32 * h; rows > 0 && c < cols && n0 + c < p.n; c += 64) {   // the groups' alternate pieces
        int32_t g[32];
        float v[32];
        tm_ld32(t0 + c, g);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 r = scaled2(g[j], g[j + 1], sa, *reinterpret_cast<const float2*>(sws + c + j));
          v[j] = r.x;
          v[j + 1] = r.y;
        }
        if (p.swiglu) {
          tm_ld32(t0 + cols + c, g);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 r = scaled2(g[j], g[j + 1], sa, *reinterpret_cast<const float2*>(sws + cols + c + j));
            v[j] = swiglu(v[j], r.x, p.limit, p.has_limit);
            v[j + 1] = swiglu(v[j + 1], r.y, p.limit, p.has_limit);
          }
        }
        if (p.type != QX_T_F32) {
          store_block<32>(p, &to, stage + buf * PAIR_BLOCK, row0, rows, n0 + c, v, tma, lane);
          buf ^= 1;
        } else {
          store_block<16>(p, &to, stage + buf * PAIR_BLOCK, row0, rows, n0 + c, v, tma, lane);
          if (n0 + c + 16 < p.n) store_block<16>(p, &to, stage + (buf ^ 1) * PAIR_BLOCK, row0, rows, n0 + c + 16, v + 16, tma, lane);
          else buf ^= 1;
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_cluster(mapa(smem_u32(&acc_empty[b]), 0));
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the stores are in memory
    // CTA 0's last arrival on this CTA's barriers has come before this CTA may leave.
    if (rank == 1 && warp == 2 && lane == 0) wait_phase(&drained, 0, 2 * timeout);
  }
  __syncwarp();
  tc::fence_before_sync();
  cluster_arrive_relaxed();
  cluster_wait();
  if (gave_up) {
    // Copies may still be in flight to either CTA; all of them count on CTA 0's barriers,
    // which waits for them, and neither CTA leaves before.
    if (fills) st_cluster(mapa(smem_u32(&issued[2 * rank + (warp == 0 ? 0 : 1)]), 0), (int32_t)fills);
    __syncwarp();
    cluster_sync();
    if (rank == 0 && threadIdx.x == 0) drain_copies(full, ns, issued, 4, spans * b_span, spans * a_span, timeout);
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace i8
}  // namespace qx
