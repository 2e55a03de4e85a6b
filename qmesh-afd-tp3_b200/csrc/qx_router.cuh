// The router of a whole MoE layer, part of qx_decode_tc.cu (included inside its
// namespace): the logits beside the x terms in moe_front_kernel, the selection of
// the experts in every CTA of the decode kernel.

// ------------------------------------------------------------------ logits
// One CTA: 16 rows x 8 experts over all of K, on warp-level BF16 tensor-core products
// (m16n8k16; the 16 x 8 tile is too small for a TMEM accumulator to pay). Warp w takes
// an eighth of K in 20 blocks of 32; a lane reads 8 consecutive elements of its row
// and of its expert, which are the operands of two products under one and the same
// permutation of K. Products of BF16 values are exact; FP32 router weights enter as
// three BF16 parts, w = hi + mid + lo to 2^-26. Each block's sum starts from zero and
// is added in FP32, so that a logit's error stays near 2^-24 of its partial sums.
// Bound by latency: the tile's weights and rows are asked into L2 at once, so that the
// blocks' loads wait for L2 only (13 -> 7 us with one row).
constexpr int RE = 8, RR = 16, RWARPS = PREP_THR / 32, RK = HID / RWARPS;
static_assert(RK % 32 == 0, "whole blocks of K per warp");

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Eight activations of row xr from k on, as the slice reads them, in BF16.
__device__ __forceinline__ uint4 load_x8(const Params& p, const uint8_t* xr, int k, float inv) {
  if (p.x_fmt == QX_X_BF16) return *reinterpret_cast<const uint4*>(xr + 2 * (size_t)k);
  const uint2 w = *reinterpret_cast<const uint2*>(xr + k);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t f2 = e4m3x2_to_f16x2((i & 2 ? w.y : w.x) >> (16 * (i & 1)));
    o[i] = bf16_pair(__fmul_rn(f16lo_to_f32(f2), inv), __fmul_rn(f16hi_to_f32(f2), inv));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A run of memory towards L2 (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void prefetch_l2(const uint8_t* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// c += a b over 16 elements of K (the k-th pairs of both operands belong together).
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int GT>
__device__ __forceinline__ void router_unit(const Params& p, int e0, int r0) {
  __shared__ __align__(8) float part[RWARPS][RR][RE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool two = r0 + 8 < p.rows;                      // the tile has rows 8..15
  const int ra = min(r0 + g, p.rows - 1), rb = min(r0 + g + 8, p.rows - 1);
  const uint8_t* x = reinterpret_cast<const uint8_t*>(p.x);
  const uint8_t *xa = x + (size_t)ra * p.x_stride, *xb = x + (size_t)rb * p.x_stride;
  float ia = 1.f, ib = 1.f;
  if (p.x_fmt == QX_X_E4M3) ia = p.x_scale[ra], ib = p.x_scale[rb];
  else if (p.x_fmt == QX_X_E4M3_POST) ia = ib = p.x_scale[0];
  const size_t at = (size_t)min(e0 + g, p.E - 1) * p.gate_stride;
  constexpr int GB = GT == QX_T_BF16 ? 2 : 4;
  if ((int)threadIdx.x < RE) {
    if (e0 + (int)threadIdx.x < p.E)
      prefetch_l2(reinterpret_cast<const uint8_t*>(p.gate) + (size_t)(e0 + threadIdx.x) * p.gate_stride * GB, HID * GB);
  } else if ((int)threadIdx.x < RE + RR && r0 + (int)threadIdx.x - RE < p.rows) {
    prefetch_l2(x + (size_t)(r0 + threadIdx.x - RE) * p.x_stride, p.x_fmt == QX_X_BF16 ? 2 * HID : HID);
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll (GT == QX_T_BF16 ? 10 : 5)
  for (int k = warp * RK + 8 * t; k < (warp + 1) * RK; k += 32) {
    const uint4 va = load_x8(p, xa, k, ia), vb = two ? load_x8(p, xb, k, ib) : make_uint4(0u, 0u, 0u, 0u);
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (GT == QX_T_BF16) {
      const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.gate) + at + k);
      mma16(c, va.x, vb.x, va.y, vb.y, w.x, w.y);
      mma16(c, va.z, vb.z, va.w, vb.w, w.z, w.w);
    } else {
      const float4* f = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.gate) + at + k);
      const float4 f0 = f[0], f1 = f[1];
      float v[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
      uint32_t w[3][4];
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[q][i] = bf16_pair(v[2 * i], v[2 * i + 1]);
          v[2 * i] -= bf16_lo(w[q][i]);
          v[2 * i + 1] -= bf16_hi(w[q][i]);
        }
#pragma unroll
      for (int q = 2; q >= 0; --q) {                      // the small parts first
        mma16(c, va.x, vb.x, va.y, vb.y, w[q][0], w[q][1]);
        mma16(c, va.z, vb.z, va.w, vb.w, w[q][2], w[q][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += c[i];
  }
  *reinterpret_cast<float2*>(&part[warp][g][2 * t]) = make_float2(acc[0], acc[1]);
  *reinterpret_cast<float2*>(&part[warp][g + 8][2 * t]) = make_float2(acc[2], acc[3]);
  __syncthreads();
  const int r = threadIdx.x / RE, e = threadIdx.x % RE;
  if (r < RR && r0 + r < p.rows && e0 + e < p.E) {
    float s = part[0][r][e];
#pragma unroll
    for (int w = 1; w < RWARPS; ++w) s += part[w][r][e];
    p.logits[(size_t)(r0 + r) * ((p.E + 3) & ~3) + e0 + e] = p.gate_bias ? s + __ldg(&p.gate_bias[e0 + e]) : s;
  }
}

// CTAs [0, rows * NXCH): the x terms; then one per (8 experts, 16 rows).
template <int GT>
__global__ void __launch_bounds__(PREP_THR) moe_front_kernel(Params p) {
  pdl_launch_dependents();
  const int prep = p.rows * NXCH;
  if ((int)blockIdx.x < prep) {
    prep_unit(p, prep, false);
    return;
  }
  const int u = blockIdx.x - prep, ne = (p.E + RE - 1) / RE;
  router_unit<GT>(p, u % ne * RE, u / ne * RR);
}

static void front_launch(const Params& p, int gate_type, cudaStream_t st) {
  const int grid = p.rows * NXCH + (p.E + RE - 1) / RE * ((p.rows + RR - 1) / RR);
  if (gate_type == QX_T_BF16) moe_front_kernel<QX_T_BF16><<<grid, PREP_THR, 0, st>>>(p);
  else moe_front_kernel<QX_T_F32><<<grid, PREP_THR, 0, st>>>(p);
}

// ------------------------------------------------------------------ selection
// A logit as an unsigned key in its order: NaN above everything, -0 equal to +0.
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;
__device__ __forceinline__ uint32_t logit_key(float l) {
  if (l != l) return 0xffffffffu;
  const uint32_t b = __float_as_uint(l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k == 0xffffffffu ? 0x7fc00000u : k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The topk experts of one row by one warp: the keys go to shared memory (`keys`, E4
// words) while each lane keeps the best of its own; a round takes the largest over
// the lanes (the lowest id of equals) and the lane it came from looks for its next.
// Short loops rather than unrolled ones: every SM fetches this code cold, once per
// call. Slot j's id and weight go to ids[j], tw[j].
__device__ void select_row(const float* l, int E, int topk, int lane, uint32_t* keys, int32_t* ids, float* tw) {
  uint32_t bk = 0u;                                       // 0: no key (every logit's is above it)
  int be = INT_MAX;
#pragma unroll 4
  for (int e = 4 * lane; e < E; e += 128) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(l + e));
    const uint4 k = make_uint4(logit_key(v.x), e + 1 < E ? logit_key(v.y) : 0u, e + 2 < E ? logit_key(v.z) : 0u,
                               e + 3 < E ? logit_key(v.w) : 0u);
    *reinterpret_cast<uint4*>(keys + e) = k;
    if (k.x > bk) bk = k.x, be = e;
    if (k.y > bk) bk = k.y, be = e + 1;
    if (k.z > bk) bk = k.z, be = e + 2;
    if (k.w > bk) bk = k.w, be = e + 3;
  }
  uint32_t my_key = 0u;
  int my_id = -1;
#pragma unroll 1
  for (int j = 0; j < topk; ++j) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
    const int id = __reduce_min_sync(0xffffffffu, bk == best ? be : INT_MAX);
    if (lane == j) my_key = best, my_id = best > KEY_NEG_INF ? id : -1;
    if (be == id) {                                       // this lane's: out, and its next best
      keys[id] = 0u;
      bk = 0u;
      be = INT_MAX;
#pragma unroll 1
      for (int e = 4 * lane; e < E; e += 128) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + e);
        if (k.x > bk) bk = k.x, be = e;
        if (k.y > bk) bk = k.y, be = e + 1;
        if (k.z > bk) bk = k.z, be = e + 2;
        if (k.w > bk) bk = k.w, be = e + 3;
      }
    }
    __syncwarp();
  }
  const float l0 = __shfl_sync(0xffffffffu, key_logit(my_key), 0);
  const float w = my_id >= 0 ? expf(key_logit(my_key) - l0) : 0.f;
  float sum = 0.f;
#pragma unroll 1
  for (int j = 0; j < topk; ++j) sum += __shfl_sync(0xffffffffu, w, j);
  if (lane < topk) {
    ids[lane] = my_id;
    tw[lane] = my_id >= 0 ? w / sum : 0.f;
  }
}

// Every row of the call into shared memory (ids[P], tw[P]), a warp per row; `keys`:
// E4 words per warp.
__device__ void select_rows(const Params& p, uint32_t* keys, int32_t* ids, float* tw, int warp, int warps) {
  const int lane = threadIdx.x & 31, E4 = (p.E + 3) & ~3;
  if (warp >= warps) return;
#pragma unroll 1
  for (int r = warp; r < p.rows; r += warps) {
    int32_t* ir = ids + r * p.topk;
    float* wr = tw + r * p.topk;
    select_row(p.logits + (size_t)r * E4, p.E, p.topk, lane, keys + warp * E4, ir, wr);
    if (blockIdx.x == 0 && lane < p.topk) {
      if (p.ids_out) p.ids_out[r * p.topk + lane] = ir[lane];
      if (p.tw_out) p.tw_out[r * p.topk + lane] = wr[lane];
    }
  }
}
