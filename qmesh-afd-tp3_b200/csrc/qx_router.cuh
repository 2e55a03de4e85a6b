// The router of a whole MoE layer, part of qx_decode_tc.cu (included inside its
// namespace): the logits (moe_router_kernel), the selection beside the x terms
// (moe_prep_kernel) and the decode kernel's routing tables from it (route_pairs).

// ------------------------------------------------------------------ logits
// One CTA: 16 rows x 8 experts over a quarter of K, on warp-level BF16 tensor-core
// products (m16n8k16; the 16 x 8 tile is too small for a TMEM accumulator to pay).
// Each of its 8 warps takes 160 elements in 5 blocks of 32, every load of which is in
// flight at once: the weights' way from memory, paid once, is all that bounds it (one
// CTA over all of K, four rounds of loads, took 9 us with one row). A lane reads 8
// consecutive elements of its row and of its expert, which are the operands of two
// products under one and the same permutation of K. Products of BF16 values are exact;
// FP32 router weights enter as three BF16 parts, w = hi + mid + lo exactly (24 bits are
// three times 8). What PTX promises of the sums inside a product is single precision in
// an unspecified order and rounding, 2^-23 an addition: each block's 32 products start from
// zero, and the blocks, warps, quarters and the bias are added in FP32 (16 additions), so a
// logit is within (2 * 32 + 16) 2^-24 of its sum |x w| (a little over one more for FP32
// weights, whose smaller parts are added first). The quarters' sums are added where the logits
// are read.
constexpr int RE = 8, RR = 16, RWARPS = PREP_THR / 32, RSPLIT = 4, RK = HID / RSPLIT / RWARPS, RB = RK / 32;
static_assert(RK % 32 == 0, "whole blocks of K per warp");

// Floats between the quarters' logits, [rows][E rounded up to 4] each.
__host__ __device__ __forceinline__ int logit_row(const Params& p) { return (p.E + 3) & ~3; }

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

// c += a b over 16 elements of K (the k-th pairs of both operands belong together).
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int GT>
__device__ __forceinline__ void router_unit(const Params& p, int e0, int r0, int quarter) {
  __shared__ __align__(8) float part[RWARPS][RR][RE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool two = r0 + 8 < p.rows;                      // the tile has rows 8..15
  const int ra = min(r0 + g, p.rows - 1), rb = min(r0 + g + 8, p.rows - 1);
  const uint8_t* x = reinterpret_cast<const uint8_t*>(p.x);
  float ia = 1.f, ib = 1.f;
  if (p.x_fmt == QX_X_E4M3) ia = p.x_scale[ra], ib = p.x_scale[rb];
  else if (p.x_fmt == QX_X_E4M3_POST) ia = ib = p.x_scale[0];
  const int k0 = (quarter * RWARPS + warp) * RK + 8 * t;
  const size_t at = (size_t)min(e0 + g, p.E - 1) * p.gate_stride + k0;
  constexpr int GV = GT == QX_T_BF16 ? 1 : 2;            // 16-byte pieces of 8 weights
  uint4 va[RB], vb[RB], wv[RB][GV];
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const uint8_t* gp = reinterpret_cast<const uint8_t*>(p.gate) + (at + 32 * i) * (8 * GV / 4);
#pragma unroll
    for (int v = 0; v < GV; ++v) wv[i][v] = *reinterpret_cast<const uint4*>(gp + 16 * v);
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    va[i] = load_x8(p, x + (size_t)ra * p.x_stride, k0 + 32 * i, ia);
    vb[i] = make_uint4(0u, 0u, 0u, 0u);
    if (two) vb[i] = load_x8(p, x + (size_t)rb * p.x_stride, k0 + 32 * i, ib);
  }
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    const uint4 a = va[i], b = vb[i];
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    if constexpr (GT == QX_T_BF16) {
      const uint4 w = wv[i][0];
      mma16(c, a.x, b.x, a.y, b.y, w.x, w.y);
      mma16(c, a.z, b.z, a.w, b.w, w.z, w.w);
    } else {
      const uint32_t f[8] = {wv[i][0].x, wv[i][0].y, wv[i][0].z, wv[i][0].w,
                             wv[i][GV - 1].x, wv[i][GV - 1].y, wv[i][GV - 1].z, wv[i][GV - 1].w};
      uint32_t w[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo = __uint_as_float(f[2 * j]), hi = __uint_as_float(f[2 * j + 1]);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          w[q][j] = bf16_pair(lo, hi);
          lo -= bf16_lo(w[q][j]);
          hi -= bf16_hi(w[q][j]);
        }
      }
#pragma unroll
      for (int q = 2; q >= 0; --q) {                      // the small parts first
        mma16(c, a.x, b.x, a.y, b.y, w[q][0], w[q][1]);
        mma16(c, a.z, b.z, a.w, b.w, w[q][2], w[q][3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] += c[j];
  }
  *reinterpret_cast<float2*>(&part[warp][g][2 * t]) = make_float2(acc[0], acc[1]);
  *reinterpret_cast<float2*>(&part[warp][g + 8][2 * t]) = make_float2(acc[2], acc[3]);
  __syncthreads();
  const int r = threadIdx.x / RE, e = threadIdx.x % RE;
  if (r < RR && r0 + r < p.rows && e0 + e < p.E) {
    float s = part[0][r][e];
#pragma unroll
    for (int w = 1; w < RWARPS; ++w) s += part[w][r][e];
    if (quarter == 0 && p.gate_bias) s += __ldg(&p.gate_bias[e0 + e]);
    p.logits[((size_t)quarter * p.rows + r0 + r) * logit_row(p) + e0 + e] = s;
  }
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

// The two largest (key, lowest id of equals) that a lane has seen, ids ascending.
struct Top2 {
  uint32_t k0 = 0u, k1 = 0u;                              // 0: none (every logit's key is above it)
  int e0 = INT_MAX, e1 = INT_MAX;
  __device__ __forceinline__ void add(uint32_t k, int e) {
    if (k > k0) k1 = k0, e1 = e0, k0 = k, e0 = e;
    else if (k > k1) k1 = k, e1 = e;
  }
  __device__ __forceinline__ void add4(const uint4& k, int e) {
    add(k.x, e);
    add(k.y, e + 1);
    add(k.z, e + 2);
    add(k.w, e + 3);
  }
};

// The topk experts of one row by one warp: the keys go to shared memory (`keys`, one
// row of logits) while each lane keeps its two best; a round takes the largest over
// the lanes (the lowest id of equals), and a lane that has given both looks through
// its keys again. Short loops rather than unrolled ones: every SM fetches this code
// cold, once per call. `l`: the row's logits of the first quarter of K, the others'
// `step` floats apart. Lane j returns slot j's id and weight.
__device__ void select_row(const float* l, size_t step, int E, int topk, int lane, uint32_t* keys, int& id_out,
                           float& w_out) {
  Top2 best;
#pragma unroll 3
  for (int e = 4 * lane; e < E; e += 128) {
    float4 v = __ldcg(reinterpret_cast<const float4*>(l + e));
#pragma unroll
    for (int q = 1; q < RSPLIT; ++q) {
      const float4 w = __ldcg(reinterpret_cast<const float4*>(l + q * step + e));
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
    const uint4 k = make_uint4(logit_key(v.x), e + 1 < E ? logit_key(v.y) : 0u, e + 2 < E ? logit_key(v.z) : 0u,
                               e + 3 < E ? logit_key(v.w) : 0u);
    *reinterpret_cast<uint4*>(keys + e) = k;
    best.add4(k, e);
  }
  uint32_t my_key = 0u;
  int my_id = -1;
#pragma unroll 1
  for (int j = 0; j < topk; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best.k0);
    const int id = __reduce_min_sync(0xffffffffu, best.k0 == top ? best.e0 : INT_MAX);
    if (lane == j) my_key = top, my_id = top > KEY_NEG_INF ? id : -1;
    if (best.e0 == id) {
      keys[id] = 0u;
      best.k0 = best.k1, best.e0 = best.e1;
      best.k1 = 0u, best.e1 = INT_MAX;
      if (best.e0 == INT_MAX) {
#pragma unroll 1
        for (int e = 4 * lane; e < E; e += 128) best.add4(*reinterpret_cast<const uint4*>(keys + e), e);
      }
    }
    __syncwarp();
  }
  const float l0 = __shfl_sync(0xffffffffu, key_logit(my_key), 0);
  const float w = my_id >= 0 ? expf(key_logit(my_key) - l0) : 0.f;
  float sum = 0.f;
#pragma unroll 1
  for (int j = 0; j < topk; ++j) sum += __shfl_sync(0xffffffffu, w, j);
  id_out = my_id;
  w_out = my_id >= 0 ? w / sum : 0.f;
}

// Whether row r of the activations holds a NaN or an infinity (a whole warp asks). Only
// rows for which nothing was selected need it: an infinity times router weights of one
// sign makes every logit -infinity, as masks of all experts do.
__device__ __forceinline__ bool row_nonfinite(const Params& p, int r, int lane) {
  const float inv = p.x_fmt == QX_X_E4M3 ? p.x_scale[r] : p.x_fmt == QX_X_E4M3_POST ? p.x_scale[0] : 1.f;
  const uint8_t* xr = reinterpret_cast<const uint8_t*>(p.x) + (size_t)r * p.x_stride;
  bool bad = false;
#pragma unroll 1
  for (int k = 8 * lane; k < HID; k += 256) {
    const uint4 v = load_x8(p, xr, k, inv);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  }
  return __any_sync(0xffffffffu, bad);
}

// ------------------------------------------------------------------ kernels in front
// CTAs: one per (8 experts, 16 rows, quarter of K).
template <int GT>
__global__ void __launch_bounds__(PREP_THR) moe_router_kernel(Params p) {
  pdl_launch_dependents();
  const int ne = (p.E + RE - 1) / RE, u = blockIdx.x, tile = u / RSPLIT;
  router_unit<GT>(p, tile % ne * RE, tile / ne * RR, u % RSPLIT);
}

// Started with the router (everything the call reads is complete then): the first CTAs
// wait for its logits and select, a warp per row; the others compute the x terms
// meanwhile. (Selecting in every CTA of the decode kernel took 11 us with 48 rows;
// x terms in the router's kernel ran at its registers, 13 us against 7.)
// A CTA selects as many rows (8 at most) as their keys fit 24 KB of shared memory.
constexpr int SEL_BYTES = 24576;
__host__ __device__ __forceinline__ int select_per_cta(const Params& p) {
  const int fit = SEL_BYTES / (((p.E + 3) & ~3) * 4);
  return fit < RWARPS ? fit : RWARPS;
}
__global__ void __launch_bounds__(PREP_THR) moe_prep_kernel(Params p, int nsel) {
  pdl_launch_dependents();
  if ((int)blockIdx.x >= nsel) {
    prep_unit(p, blockIdx.x - nsel, gridDim.x - nsel, false);
    return;
  }
  __shared__ __align__(16) uint32_t keys[SEL_BYTES / 4];   // a row of logits per warp
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E4 = logit_row(p);
  const int per = select_per_cta(p), r = blockIdx.x * per + warp;
  if (warp >= per || r >= p.rows) return;
  int id;
  float w;
  select_row(p.logits + (size_t)r * E4, (size_t)p.rows * E4, p.E, p.topk, lane, keys + warp * E4, id, w);
  if (__shfl_sync(0xffffffffu, id, 0) < 0 && row_nonfinite(p, r, lane)) {   // a NaN row, as if its logits were NaN
    id = lane;
    w = __uint_as_float(0x7fc00000u);
  }
  if (lane < p.topk) {
    const int q = r * p.topk + lane;
    p.sel_ids[q] = id;
    p.sel_tw[q] = w;
    if (p.ids_out) p.ids_out[q] = id;
    if (p.tw_out) p.tw_out[q] = w;
  }
}

static cudaError_t front_launch(const Params& p, int gate_type, cudaStream_t st) {
  const int grid = (p.E + RE - 1) / RE * ((p.rows + RR - 1) / RR) * RSPLIT;
  if (gate_type == QX_T_BF16) moe_router_kernel<QX_T_BF16><<<grid, PREP_THR, 0, st>>>(p);
  else moe_router_kernel<QX_T_F32><<<grid, PREP_THR, 0, st>>>(p);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const int per = select_per_cta(p), nsel = (p.rows + per - 1) / per;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(nsel + p.rows * NXCH, 1, 1);
  cfg.blockDim = dim3(PREP_THR, 1, 1);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, moe_prep_kernel, p, nsel);
}

// ------------------------------------------------------------------ routing tables
// The routing tables of route_sort (unique experts ascending, an expert's pairs in
// order, split evenly into groups of at most gmax) from the ids in shared memory, by
// all threads of the CTA instead of one warp: a pair's place is the number of smaller
// keys (expert << 9 | pair), its run's ends are found by walking the sorted keys, a
// group's number is a sum over the places before its run. `scratch`: 3 MAXP words. (In
// one warp, sorting network and scans took 41 us for 288 pairs.)
__device__ void route_pairs(const Params& p, const int32_t* ids, uint32_t* scratch, GroupS* gs, PairS* ps,
                            RouteHdr* hdr) {
  constexpr uint32_t NONE = 0xffffffffu;                  // no expert: after every key
  constexpr int PT = (MAXP + NTHR - 1) / NTHR;            // pairs (then places) per thread
  const int P4 = (p.P + 3) & ~3, gmax = min(GMAX, p.rows), tid = threadIdx.x;
  uint32_t *keys = scratch, *sorted = scratch + MAXP, *runs = scratch + 2 * MAXP;   // runs: groups, at a run's start
  int mine = 0;                                           // this thread's pairs with an expert
  for (int i = tid; i < P4; i += NTHR) {
    const bool has = i < p.P && ids[i] >= 0;
    keys[i] = has ? (uint32_t)ids[i] << 9 | (uint32_t)i : NONE;
    sorted[i] = NONE;
    runs[i] = 0u;
    mine += has;
  }
  if (tid == 0) hdr->n_groups = hdr->n_pairs = hdr->b_max = 0;
  __syncthreads();
  if (mine) atomicAdd(&hdr->n_pairs, mine);
  for (int i = tid; i < p.P; i += NTHR) {
    const uint32_t k = keys[i];
    int place = 0;
#pragma unroll 4
    for (int j = 0; j < P4; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(keys + j);
      place += (int)(o.x < k) + (int)(o.y < k) + (int)(o.z < k) + (int)(o.w < k);
    }
    if (k != NONE) sorted[place] = k;
  }
  __syncthreads();
  const int valid = hdr->n_pairs;
  int start[PT], count[PT];
#pragma unroll
  for (int u = 0; u < PT; ++u) {
    const int i = tid + u * NTHR;
    start[u] = count[u] = 0;
    if (i >= valid) continue;
    const uint32_t k = sorted[i], e = k >> 9;
    int a = i, b = i + 1;
    while (a > 0 && sorted[a - 1] >> 9 == e) --a;
    while (b < valid && sorted[b] >> 9 == e) ++b;
    start[u] = a;
    count[u] = b - a;
    ps[i].pq = (int)(k & 511u);
    ps[i].row = div_small((int)(k & 511u), p.topk);
    if (a == i) runs[i] = (uint32_t)div_small(b - a + gmax - 1, gmax);
  }
  __syncthreads();
  const int abs = ((p.NT + SK - 1) / SK) * XT_STAGE;      // down-operand bytes per pair
#pragma unroll
  for (int u = 0; u < PT; ++u) {
    const int i = tid + u * NTHR, c = count[u];
    if (c == 0) continue;
    const int r = i - start[u], ng = div_small(c + gmax - 1, gmax);
    const int gk = div_small((r + 1) * ng - 1, c);        // the k with k c / ng <= r < (k + 1) c / ng
    const int lo = div_small(gk * c, ng);
    if (r != lo) continue;                                // the group's first pair writes its record
    int g = gk;
    for (int j = 0; j < start[u]; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(runs + j);
      g += (int)o.x + (j + 1 < start[u] ? (int)o.y : 0) + (j + 2 < start[u] ? (int)o.z : 0) +
           (j + 3 < start[u] ? (int)o.w : 0);
    }
    GroupS d;
    d.expert = (int)(sorted[i] >> 9);
    d.gsz = div_small((gk + 1) * c, ng) - lo;
    d.pair_off = i;
    d.n = XTERMS * d.gsz;
    d.sbs = d.gsz * XT_STAGE;
    d.ab_off = i * abs;
    d.shared = 0;
    d.pad = 0;
    gs[g] = d;
    atomicMax(&hdr->b_max, d.sbs);
    if (i + d.gsz == valid) hdr->n_groups = g + 1;        // the last group of the call
  }
}
