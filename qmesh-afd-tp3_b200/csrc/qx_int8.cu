// 8-bit integer products with one scale per token and one per channel, and the
// per-token quantiser that feeds them:
//   quantise   m = max |x[r, :]|, s[r] = max(m, 1e-30) / 127,
//              q[r, k] = round_half_even(127 x[r, k] / max(m, 1e-30))
//   product    y[m, n] = (sum_k a[m, k] w[n, k]) a_scale[m] w_scale[n]
//   SwiGLU     g, u = the product's columns n and n + N of w's gate rows, then up
//              rows; g = min(g, L), u = clamp(u, -L, L); y = g / (1 + exp(-g)) u
// The sums are whole numbers of at most 32 bits (k <= QX_INT8_MAX_K keeps
// 128 * 128 * k below 2^31), so their order does not matter and every variant
// below gives the same bytes. The scales are applied in FP32, ((float)sum *
// a_scale) * w_scale, and the result is rounded once to the output's type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdlib.h>

#include "qmesh_b200.h"
#include "qx_ptx.cuh"

namespace qx {
namespace i8 {

constexpr float QMAX = 127.f;
constexpr float AMAX_FLOOR = 1e-30f;   // rows below it quantise to whole multiples of 1e-30 / 127
constexpr uint32_t INF_BITS = 0x7f800000u;

// QX_DEV_* bits of this file's kernels since the last qx_int8_status.
__device__ uint32_t g_status;

// ------------------------------------------------------------------ outputs
__device__ __forceinline__ void store_out(void* out, int64_t i, int type, float v) {
  if (type == QX_T_BF16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else if (type == QX_T_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(out)[i] = v;
}

__device__ __forceinline__ float scaled(int32_t sum, float sa, float sw) {
  return __fmul_rn(__fmul_rn(__int2float_rn(sum), sa), sw);
}

// Comparisons, not fminf: a NaN (a row the quantiser refused) stays one.
__device__ __forceinline__ float swiglu(float g, float u, float limit, bool has_limit) {
  if (has_limit) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
  }
  return (g / (1.f + expf(-g))) * u;
}

// ------------------------------------------------------------------ quantiser
// Four elements of a row from k on (k % 4 == 0; those past the row's end read as 0),
// as FP32: BF16 / FP16 / FP32 values, or the slice's FP8 form bf16(float(e4m3) inv).
template <int T, bool VEC>
__device__ __forceinline__ void load4(const void* x, int64_t row_off, int k, int n, float inv, float (&v)[4]) {
  if constexpr (T == QX_T_F32) {
    const float* p = reinterpret_cast<const float*>(x) + row_off + k;
    if (VEC) {
      const float4 w = *reinterpret_cast<const float4*>(p);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = k + i < n ? p[i] : 0.f;
    }
  } else if constexpr (T == QX_T_E4M3) {
    const uint8_t* p = reinterpret_cast<const uint8_t*>(x) + row_off + k;
    uint32_t w = 0;
    if (VEC) w = *reinterpret_cast<const uint32_t*>(p);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (k + i < n ? (uint32_t)p[i] : 0u) << (8 * i);
    const uint32_t a = e4m3x2_to_f16x2(w & 0xffffu), b = e4m3x2_to_f16x2(w >> 16);
    const float f[4] = {f16lo_to_f32(a), f16hi_to_f32(a), f16lo_to_f32(b), f16hi_to_f32(b)};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(f[i], inv)));
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + row_off + k;
    uint16_t h[4];
    if (VEC) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      h[0] = w.x & 0xffffu; h[1] = w.x >> 16; h[2] = w.y & 0xffffu; h[3] = w.y >> 16;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = k + i < n ? p[i] : (uint16_t)0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = T == QX_T_BF16 ? __uint_as_float((uint32_t)h[i] << 16) : __half2float(__ushort_as_half(h[i]));
  }
}

// round_half_even(p / m) for p = 127 x, 0 < m: the rounded estimate p * (1 / m)
// is at most one off, and p - n m is exact for 8- and 11-bit x (p and n m both
// fit 24 bits), so one comparison with half of m settles it; BF16 values often
// sit on the half itself (x = m / 2 gives 63.5), where an inexact quotient would
// fall to either side.
__device__ __forceinline__ int quotient(float p, float m, float rm) {
  float n = rintf(p * rm);
  const float d = fmaf(-n, m, p), a2 = 2.f * fabsf(d);
  if (a2 > m || (a2 == m && ((int)n & 1))) n += d > 0.f ? 1.f : -1.f;
  return (int)fminf(fmaxf(n, -QMAX), QMAX);
}

constexpr int QTHR = 256;

template <int T, bool VEC>
__global__ void __launch_bounds__(QTHR) quant_kernel(const void* x, int64_t xs, const float* x_scale, int per_row,
                                                     int k, int8_t* q, int64_t qs, float* scale) {
  const int64_t r = blockIdx.x;
  const float inv = T == QX_T_E4M3 ? x_scale[per_row ? r : 0] : 1.f;
  float v[4];
  uint32_t m = 0;                                  // |x| as bits: a NaN or infinity is the largest
  for (int i = threadIdx.x * 4; i < k; i += QTHR * 4) {
    load4<T, VEC>(x, r * xs, i, k, inv, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t sm[QTHR / 32];
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QTHR / 32; ++i) m = max(m, sm[i]);
  const bool bad = m >= INF_BITS;
  const float mc = fmaxf(__uint_as_float(m), AMAX_FLOOR);
  const float f = mc > 1e30f ? 0x1p-20f : 1.f;     // 127 x must not overflow: a power of two changes no quotient
  const float qm = QMAX * f, mf = mc * f, rm = __frcp_rn(mf);
  if (threadIdx.x == 0) {
    scale[r] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(mc, QMAX);
    if (bad) atomicOr(&g_status, (uint32_t)QX_DEV_NONFINITE);
  }
  int8_t* qr = q + r * qs;
  for (int i = threadIdx.x * 4; i < k; i += QTHR * 4) {
    load4<T, VEC>(x, r * xs, i, k, inv, v);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w |= ((uint32_t)(bad ? 0 : quotient(__fmul_rn(v[j], qm), mf, rm)) & 0xffu) << (8 * j);
    if (VEC) *reinterpret_cast<uint32_t*>(qr + i) = w;
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < k) qr[i + j] = (int8_t)(w >> (8 * j));
  }
}

// ------------------------------------------------------------------ product
struct Args {
  const int8_t* a;
  const int8_t* w;
  const float* sa;
  const float* sw;
  void* out;
  int64_t as, ws, os;
  int m, n, k, type;
  int swiglu, has_limit;
  float limit;
};

// Any alignment: 64 x 64 sums per CTA by dp4a over 64-byte pieces of K staged in
// shared memory byte by byte. Serves rows whose address or stride the copy
// engine cannot take (not a multiple of 16 bytes).
constexpr int ST = 64, SKB = 64;
__global__ void __launch_bounds__(256) plain_kernel(Args p) {
  __shared__ __align__(16) int8_t sa[ST][SKB + 4], sw[ST][SKB + 4];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int half = p.swiglu ? ST / 2 : ST;               // output columns of the tile
  const int n0 = blockIdx.x * half, m0 = blockIdx.y * ST;
  int32_t acc[4][4] = {};                                // tokens ty + 16 i, weight rows tx + 16 j
  for (int k0 = 0; k0 < p.k; k0 += SKB) {
    for (int i = tid; i < ST * SKB; i += 256) {
      const int r = i / SKB, c = i % SKB;
      const int wr = r < half ? n0 + r : p.n + n0 + r - half;
      const bool w_ok = (r < half ? n0 + r : n0 + r - half) < p.n;
      sa[r][c] = (m0 + r < p.m && k0 + c < p.k) ? p.a[(int64_t)(m0 + r) * p.as + k0 + c] : (int8_t)0;
      sw[r][c] = (w_ok && k0 + c < p.k) ? p.w[(int64_t)wr * p.ws + k0 + c] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < SKB; c += 4) {
      int av[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        av[i] = *reinterpret_cast<const int*>(&sa[ty + 16 * i][c]);
        wv[i] = *reinterpret_cast<const int*>(&sw[tx + 16 * i][c]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], wv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 16 * i;
    if (m >= p.m) continue;
    const float s = p.sa[m];
    if (p.swiglu) {                                      // rows j < 2 are gates, j + 2 their ups
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n < p.n)
          store_out(p.out, (int64_t)m * p.os + n, p.type,
                    swiglu(scaled(acc[i][j], s, p.sw[n]), scaled(acc[i][j + 2], s, p.sw[p.n + n]), p.limit,
                           p.has_limit));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n < p.n) store_out(p.out, (int64_t)m * p.os + n, p.type, scaled(acc[i][j], s, p.sw[n]));
      }
    }
  }
}

}  // namespace i8
}  // namespace qx

#include "qx_int8_tc.cuh"

using namespace qx::i8;

namespace {
// SMs of the current device, with the kernels' shared memory set up; 0 if it is no sm_100.
int device_sms() {
  static int cached[64] = {0};
  int dev = 0, major = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev]) return cached[dev];
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10) return 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
  if (cudaFuncSetAttribute(split_kernel<16>, attr, (int)Split<16>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(split_kernel<32>, attr, (int)Split<32>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(split_kernel<64>, attr, (int)Split<64>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(split_kernel<128>, attr, (int)Split<128>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(pair_kernel<128>, attr, (int)Pair<128>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(pair_kernel<256>, attr, (int)Pair<256>::SMEM) != cudaSuccess)
    return 0;
  return cached[dev] = sms;
}

uint64_t wait_limit_ns() {
  const char* e = getenv("QX_TIMEOUT_MS");
  const long ms = e ? atol(e) : 1000;
  return (uint64_t)(ms < 10 ? 10 : ms) * 1000000ull;
}

// Tiled-copy descriptor of int8 rows [rows, k], boxes of 128 bytes x box_rows with
// the 128-byte swizzle; places outside the tensor read as 0.
bool row_map(CUtensorMap* map, const int8_t* base, int64_t rows, int k, int64_t stride, int box_rows) {
  static decltype(&cuTensorMapEncodeTiled) encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {KST, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
int split_launch(const Args& p, const CUtensorMap& tw, const CUtensorMap& ta, int pieces, cudaStream_t st) {
  const int half = p.swiglu ? 64 : 128;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pieces;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.n + half - 1) / half * pieces), (unsigned)((p.m + BN - 1) / BN), 1);
  cfg.blockDim = dim3(SPLIT_THR, 1, 1);
  cfg.dynamicSmemBytes = Split<BN>::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, split_kernel<BN>, tw, ta, p, pieces, wait_limit_ns()) == cudaSuccess
             ? QX_OK : QX_ERR_LAUNCH;
}

template <int BN>
int pair_launch(const Args& p, const CUtensorMap& tw, const CUtensorMap& ta, int sms, cudaStream_t st) {
  const int cols = p.swiglu ? BN / 2 : BN;
  const int tiles_m = (p.m + 255) / 256;
  const int64_t tiles = (int64_t)tiles_m * ((p.n + cols - 1) / cols);
  if (tiles > 0x7fffffff) return QX_ERR_SHAPE;
  const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2);
  pair_kernel<BN><<<2 * pairs, PAIR_THR, Pair<BN>::SMEM, st>>>(tw, ta, p, tiles_m, (int)tiles, wait_limit_ns());
  return cudaGetLastError() == cudaSuccess ? QX_OK : QX_ERR_LAUNCH;
}

// K pieces of the split kernel: the count (1..8) that leaves the busiest SM the
// fewest K chunks, the smallest of equals.
int pieces_of(int tiles, int chunks, int sms) {
  int best = 1;
  int64_t least = -1;
  for (int s = 1; s <= 8 && s <= chunks; ++s) {
    const int64_t c = (int64_t)((int64_t)tiles * s + sms - 1) / sms * ((chunks + s - 1) / s);
    if (least < 0 || c < least) best = s, least = c;
  }
  return best;
}

int tc_launch(const Args& p, int sms, cudaStream_t st) {
  CUtensorMap tw, ta;
  const int64_t w_rows = p.swiglu ? 2ll * p.n : p.n;
  if (p.m <= 128) {
    const int bn = p.m <= 16 ? 16 : p.m <= 32 ? 32 : p.m <= 64 ? 64 : 128;
    if (!row_map(&tw, p.w, w_rows, p.k, p.ws, 64) || !row_map(&ta, p.a, p.m, p.k, p.as, bn)) return QX_ERR_DEVICE;
    const int half = p.swiglu ? 64 : 128;
    const int s = pieces_of((p.n + half - 1) / half, (p.k + (int)KST - 1) / (int)KST, sms);
    return bn == 16 ? split_launch<16>(p, tw, ta, s, st) : bn == 32 ? split_launch<32>(p, tw, ta, s, st)
         : bn == 64 ? split_launch<64>(p, tw, ta, s, st) : split_launch<128>(p, tw, ta, s, st);
  }
  // 256 or 128 weight rows per tile: whichever leaves the busiest pair fewer of them
  const int tiles_m = (p.m + 255) / 256, pairs = sms / 2, h = p.swiglu ? 2 : 1;
  auto waves = [&](int bn) {
    const int64_t t = (int64_t)tiles_m * ((p.n * (int64_t)h + bn - 1) / bn);
    return (t + pairs - 1) / pairs * bn;
  };
  const int bn = waves(128) < waves(256) ? 128 : 256;
  if (!row_map(&tw, p.w, w_rows, p.k, p.ws, bn / 2) || !row_map(&ta, p.a, p.m, p.k, p.as, 128)) return QX_ERR_DEVICE;
  return bn == 128 ? pair_launch<128>(p, tw, ta, sms, st) : pair_launch<256>(p, tw, ta, sms, st);
}

template <int T>
void quant_launch(const void* x, int64_t xs, const float* x_scale, int per_row, int64_t rows, int k, int8_t* q,
                  int64_t qs, float* scale, bool vec, cudaStream_t st) {
  if (vec) quant_kernel<T, true><<<(unsigned)rows, QTHR, 0, st>>>(x, xs, x_scale, per_row, k, q, qs, scale);
  else quant_kernel<T, false><<<(unsigned)rows, QTHR, 0, st>>>(x, xs, x_scale, per_row, k, q, qs, scale);
}
}  // namespace

extern "C" {

int qx_quant_int8(const void* x, int64_t x_stride, int32_t x_type, const float* x_scale, int32_t n_scale,
                  int64_t rows, int32_t k, int8_t* q, int64_t q_stride, float* scale, void* stream) {
  if (rows < 0 || rows > 0x7fffffffll || k < 1 || k > QX_INT8_MAX_K) return QX_ERR_SHAPE;
  if (x_type < QX_T_BF16 || x_type > QX_T_E4M3) return QX_ERR_ARG;
  if (rows == 0) return QX_OK;
  if (!x || !q || !scale) return QX_ERR_ARG;
  if (x_type == QX_T_E4M3 && (!x_scale || (n_scale != 1 && n_scale != rows))) return QX_ERR_ARG;
  if (x_stride < k || q_stride < k) return QX_ERR_SHAPE;
  const int esz = x_type == QX_T_F32 ? 4 : x_type == QX_T_E4M3 ? 1 : 2;
  if (reinterpret_cast<uintptr_t>(x) % esz || reinterpret_cast<uintptr_t>(scale) % 4) return QX_ERR_ALIGN;
  if (device_sms() <= 0) return QX_ERR_DEVICE;
  // four elements per access where every row starts on that boundary and has a multiple of four
  const bool vec = k % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * esz) == 0 && x_stride % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_stride % 4 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int per_row = n_scale == rows && rows > 1;
  if (x_type == QX_T_BF16) quant_launch<QX_T_BF16>(x, x_stride, x_scale, per_row, rows, k, q, q_stride, scale, vec, st);
  else if (x_type == QX_T_F16) quant_launch<QX_T_F16>(x, x_stride, x_scale, per_row, rows, k, q, q_stride, scale, vec, st);
  else if (x_type == QX_T_F32) quant_launch<QX_T_F32>(x, x_stride, x_scale, per_row, rows, k, q, q_stride, scale, vec, st);
  else quant_launch<QX_T_E4M3>(x, x_stride, x_scale, per_row, rows, k, q, q_stride, scale, vec, st);
  return cudaGetLastError() == cudaSuccess ? QX_OK : QX_ERR_LAUNCH;
}

int qx_int8_matmul(const QxInt8Args* a, void* stream) {
  if (!a) return QX_ERR_ARG;
  if (a->m < 0 || a->n < 1 || a->n > (1 << 24) || a->m > (1 << 24) || a->k < 1 || a->k > QX_INT8_MAX_K)
    return QX_ERR_SHAPE;
  if (a->out_type < QX_T_BF16 || a->out_type > QX_T_F32) return QX_ERR_ARG;
  if (a->m == 0) return QX_OK;
  if (!a->a || !a->w || !a->a_scale || !a->w_scale || !a->out) return QX_ERR_ARG;
  if (a->a_stride < a->k || a->w_stride < a->k || a->out_stride < a->n) return QX_ERR_SHAPE;
  const int osz = a->out_type == QX_T_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->out) % osz || reinterpret_cast<uintptr_t>(a->a_scale) % 4 ||
      reinterpret_cast<uintptr_t>(a->w_scale) % 4)
    return QX_ERR_ALIGN;
  const int sms = device_sms();
  if (sms <= 0) return QX_ERR_DEVICE;
  Args p;
  p.a = a->a; p.w = a->w; p.sa = a->a_scale; p.sw = a->w_scale; p.out = a->out;
  p.as = a->a_stride; p.ws = a->w_stride; p.os = a->out_stride;
  p.m = a->m; p.n = a->n; p.k = a->k; p.type = a->out_type;
  p.swiglu = a->swiglu ? 1 : 0; p.has_limit = a->has_limit ? 1 : 0; p.limit = a->limit;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Tiled copies need rows that start on 16-byte boundaries (a single row: its address only).
  auto aligned = [](const int8_t* b, int64_t stride, int64_t rows) {
    return reinterpret_cast<uintptr_t>(b) % 16 == 0 && (stride % 16 == 0 || rows == 1);
  };
  if (aligned(p.a, p.as, p.m) && aligned(p.w, p.ws, p.swiglu ? 2 : p.n)) {
    if (p.m == 1) p.as = (p.as + 15) / 16 * 16;          // never stepped
    if (p.n == 1 && !p.swiglu) p.ws = (p.ws + 15) / 16 * 16;
    return tc_launch(p, sms, st);
  }
  const int half = p.swiglu ? ST / 2 : ST;
  const int64_t gy = (p.m + ST - 1) / ST;
  if (gy > 65535) return QX_ERR_SHAPE;
  plain_kernel<<<dim3((unsigned)((p.n + half - 1) / half), (unsigned)gy), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? QX_OK : QX_ERR_LAUNCH;
}

int qx_int8_status(uint32_t* status, void* stream) {
  if (!status) return QX_ERR_ARG;
  void* addr = nullptr;
  if (cudaGetSymbolAddress(&addr, g_status) != cudaSuccess) return QX_ERR_DEVICE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (cudaMemcpyAsync(status, addr, sizeof(uint32_t), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaMemsetAsync(addr, 0, sizeof(uint32_t), st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess)
    return QX_ERR_LAUNCH;
  return QX_OK;
}

}  // extern "C"
