// The router of a whole MoE layer, part of qx_decode_tc.cu (included inside its
// namespace): the logits beside the x terms in moe_front_kernel, the selection of
// the experts in every CTA of the decode kernel.

// ------------------------------------------------------------------ logits
// One CTA: RE experts x up to RR rows over all of K. Warp w takes an eighth of K
// (640 elements, 80 pieces of 8), lane l its pieces l, l + 32, l + 64; products
// of BF16 values are exact in FP32, and a logit is 24 terms in a lane, then a
// tree over 32 lanes and 8 warps, so its rounding error stays near 2^-24 of the
// partial sums. The weights are read once per RR rows.
constexpr int RE = 3, RR = 8, RWARPS = PREP_THR / 32, RK = HID / RWARPS, RPIECES = RK / 8;
static_assert(RE * RR <= 32 && RK % 8 == 0, "one lane per sum");

__device__ __forceinline__ void bf16x8(const uint4& w, float (&v)[8]) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a[i] << 16);
    v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
  }
}

// Eight activations of row xr from k on, as the slice reads them.
__device__ __forceinline__ void load_x8(const Params& p, const uint8_t* xr, int k, float inv, float (&v)[8]) {
  if (p.x_fmt == QX_X_BF16) {
    bf16x8(*reinterpret_cast<const uint4*>(xr + 2 * (size_t)k), v);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(xr + k);
    const uint32_t a[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t f2 = e4m3x2_to_f16x2(a[i >> 1] >> (16 * (i & 1)));
      v[2 * i] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(f16lo_to_f32(f2), inv)));
      v[2 * i + 1] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(f16hi_to_f32(f2), inv)));
    }
  }
}

template <int GT>
__device__ __forceinline__ void router_unit(const Params& p, int e0, int r0) {
  __shared__ float part[RWARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nr = min(RR, p.rows - r0);
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
#pragma unroll
  for (int i = 0; i < (RPIECES + 31) / 32; ++i) {
    const int piece = lane + 32 * i;
    if (piece >= RPIECES) break;
    const int k = warp * RK + piece * 8;
    float w[RE][8];
#pragma unroll
    for (int e = 0; e < RE; ++e) {
      const size_t at = (size_t)min(e0 + e, p.E - 1) * p.gate_stride + k;
      if constexpr (GT == QX_T_BF16) {
        bf16x8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.gate) + at), w[e]);
      } else {
        const float4* g = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.gate) + at);
        const float4 a = g[0], b = g[1];
        w[e][0] = a.x; w[e][1] = a.y; w[e][2] = a.z; w[e][3] = a.w;
        w[e][4] = b.x; w[e][5] = b.y; w[e][6] = b.z; w[e][7] = b.w;
      }
    }
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      if (r < nr) {
        const float inv = p.x_fmt == QX_X_E4M3 ? p.x_scale[r0 + r] : p.x_fmt == QX_X_E4M3_POST ? p.x_scale[0] : 1.f;
        float x[8];
        load_x8(p, reinterpret_cast<const uint8_t*>(p.x) + (size_t)(r0 + r) * p.x_stride, k, inv, x);
#pragma unroll
        for (int e = 0; e < RE; ++e)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[e * RR + r] = fmaf(x[j], w[e][j], acc[e * RR + r]);
      }
    }
  }
  // Sums over the lanes, halving the values a lane carries at each step: lane i
  // ends with value i.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = up ? acc[i] : acc[i + o], keep = up ? acc[i + o] : acc[i];
      acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  part[warp][lane] = acc[0];
  __syncthreads();
  if (threadIdx.x < RE * RR) {
    const int e = e0 + threadIdx.x / RR, r = threadIdx.x % RR;
    if (e < p.E && r < nr) {
      float s = part[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < RWARPS; ++w) s += part[w][threadIdx.x];
      p.logits[(size_t)(r0 + r) * p.E + e] = p.gate_bias ? s + __ldg(&p.gate_bias[e]) : s;
    }
  }
}

// CTAs [0, rows * NXCH): the x terms; then one per (RE experts, RR rows).
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

// The topk experts of one row by one warp, each the largest (key, lowest id) after
// the one before; keys of up to 32 KEYS experts stay in registers, more are read
// again for every slot. Slot j's id and weight go to ids[j], tw[j].
template <int KEYS>
__device__ void select_row(const float* l, int E, int topk, int lane, int32_t* ids, float* tw) {
  uint32_t key[KEYS > 0 ? KEYS : 1];
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int e = lane + 32 * i;
      key[i] = e < E ? logit_key(__ldcg(l + e)) : 0u;
    }
  }
  uint32_t pk = 0xffffffffu, my_key = 0u;
  int pe = -1, my_id = -1;
  for (int j = 0; j < topk; ++j) {
    uint32_t bk = 0u;
    int be = INT_MAX;
    auto take = [&](uint32_t k, int e) {
      if ((k < pk || (k == pk && e > pe)) && k > bk) bk = k, be = e;   // ids ascend: the first of equals stays
    };
    if constexpr (KEYS > 0) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i) take(key[i], lane + 32 * i);
    } else {
#pragma unroll 4
      for (int e = lane; e < E; e += 32) take(logit_key(__ldcg(l + e)), e);
    }
    const uint32_t best = __reduce_max_sync(0xffffffffu, bk);
    const int e = __reduce_min_sync(0xffffffffu, bk == best ? be : INT_MAX);
    pk = best;
    pe = e;
    if (lane == j) my_key = best, my_id = best > KEY_NEG_INF ? e : -1;
  }
  const float l0 = __shfl_sync(0xffffffffu, key_logit(my_key), 0);
  const float w = my_id >= 0 ? expf(key_logit(my_key) - l0) : 0.f;
  float sum = 0.f;
  for (int j = 0; j < topk; ++j) sum += __shfl_sync(0xffffffffu, w, j);
  if (lane < topk) {
    ids[lane] = my_id;
    tw[lane] = my_id >= 0 ? w / sum : 0.f;
  }
}

// Every row of the call into shared memory (ids[P], tw[P]), a warp per row.
__device__ void select_rows(const Params& p, int32_t* ids, float* tw, int warp, int warps) {
  const int lane = threadIdx.x & 31;
  for (int r = warp; r < p.rows; r += warps) {
    const float* l = p.logits + (size_t)r * p.E;
    int32_t* ir = ids + r * p.topk;
    float* wr = tw + r * p.topk;
    if (p.E <= 128) select_row<4>(l, p.E, p.topk, lane, ir, wr);
    else if (p.E <= 512) select_row<16>(l, p.E, p.topk, lane, ir, wr);
    else select_row<0>(l, p.E, p.topk, lane, ir, wr);
    if (blockIdx.x == 0 && lane < p.topk) {
      if (p.ids_out) p.ids_out[r * p.topk + lane] = ir[lane];
      if (p.tw_out) p.tw_out[r * p.topk + lane] = wr[lane];
    }
  }
}
