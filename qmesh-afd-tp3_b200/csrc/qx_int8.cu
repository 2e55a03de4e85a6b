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

#include <atomic>
#include <thread>

#include "qmesh_b200.h"
#include "qx_ptx.cuh"

namespace qx {
namespace i8 {

constexpr float QMAX = 127.f;
constexpr float AMAX_FLOOR = 1e-30f;   // rows below it quantise to whole multiples of 1e-30 / 127
constexpr uint32_t INF_BITS = 0x7f800000u;

// QX_DEV_* bits of this file's kernels since the last qx_int8_status.
__device__ uint32_t g_status;

// Read and cleared in one step, so that no bit set beside a read is lost, into a word
// that belongs to the read until it returns.
constexpr int STATUS_READS = 64;
__device__ uint32_t g_taken[STATUS_READS];
__global__ void take_status_kernel(int slot) { g_taken[slot] = atomicExch(&g_status, 0u); }

// ------------------------------------------------------------------ outputs
__device__ __forceinline__ void store_out(void* out, int64_t i, int type, float v) {
  if (type == QX_T_BF16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else if (type == QX_T_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(out)[i] = v;
}

__device__ __forceinline__ float scaled(int32_t sum, float sa, float sw) {
  return __fmul_rn(__fmul_rn(__int2float_rn(sum), sa), sw);
}

// Comparisons, not fminf: a NaN (from a row that the quantiser refused) stays one. The
// quotient is the full-range approximation, within 2 units of its last place (2^-22) for
// every denominator that FP32 holds: 0 only for gates below -88.7, where exp(-g) is past
// FP32. An exactly rounded division, which branches per element, makes the pair kernel's
// epilogue 1.4 to 3 us longer (64 x 2304 x 5120: 13.0 us against 11.5; 333 x 1111 x 2000: 10.6
// against 9.2) for 3 of the 10 roundings of 2^-24 behind an output.
__device__ __forceinline__ float quotient_full(float a, float b) {
  float q;
  asm("div.full.f32 %0, %1, %2;" : "=f"(q) : "f"(a), "f"(b));
  return q;
}
__device__ __forceinline__ float swiglu(float g, float u, float limit, bool has_limit) {
  if (has_limit) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
  }
  return quotient_full(g, 1.f + expf(-g)) * u;
}

// ------------------------------------------------------------------ quantiser
// Elements of type T per 16-byte load.
template <int T>
__host__ __device__ constexpr int per16() { return T == QX_T_F32 ? 4 : T == QX_T_E4M3 ? 16 : 8; }

// The FP32 values of one 16-byte load: BF16 / FP16 / FP32 values, or the slice's
// FP8 form bf16(float(e4m3) inv).
template <int T>
__device__ __forceinline__ void unpack(const uint4& raw, float inv, float (&v)[per16<T>()]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == QX_T_F32) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (T == QX_T_BF16) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else if constexpr (T == QX_T_F16) {
      v[2 * i] = f16lo_to_f32(w[i]);
      v[2 * i + 1] = f16hi_to_f32(w[i]);
    } else {
      const uint32_t lo = e4m3x2_to_f16x2(w[i] & 0xffffu), hi = e4m3x2_to_f16x2(w[i] >> 16);
      const float f[4] = {f16lo_to_f32(lo), f16hi_to_f32(lo), f16lo_to_f32(hi), f16hi_to_f32(hi)};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(f[j], inv)));
    }
  }
}

// 16 bytes of a row's elements from index k on; one load where the row is aligned
// and the piece full, else element by element, those past n reading as 0.
template <int T, bool VEC>
__device__ __forceinline__ uint4 load16(const void* x, int64_t off, int k, int n) {
  constexpr int E = per16<T>(), B = 16 / E;
  const uint8_t* p = reinterpret_cast<const uint8_t*>(x) + (off + k) * B;
  if (VEC && k + E <= n) return __ldcg(reinterpret_cast<const uint4*>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < E; ++j) {
    uint32_t e = 0u;
    if (k + j < n) {
      if constexpr (B == 4) e = reinterpret_cast<const uint32_t*>(p)[j];
      else if constexpr (B == 2) e = reinterpret_cast<const uint16_t*>(p)[j];
      else e = p[j];
    }
    w[j * B / 4] |= e << (8 * (j * B % 4));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// round_half_even(127 x / m) as the low byte of the result, c = 127 / m rounded: the
// whole number comes from adding 1.5 * 2^23. BF16 and FP16 values often sit on a half
// (x = m / 2 gives 63.5), where an inexact quotient falls to either side: x c is within 2
// units of its last place of the true quotient, a half has at most 8 significant bits,
// and any other quotient of 8- or 11-bit numbers is at least 1 / (127 * 4094) of itself
// (16 units) away from one, so rounding x c to 21 bits first restores the halves and
// moves nothing over one (for m >= AMAX_FLOOR, below which c is not 127 over such a
// number). FP32 values are rounded as they come, at most 2^-24 off.
template <int T>
__device__ __forceinline__ uint32_t quotient(float x, float c) {
  constexpr float WHOLE = 12582912.f;
  if constexpr (T == QX_T_F32) return __float_as_uint(fmaf(x, c, WHOLE));
  const uint32_t t = (__float_as_uint(__fmul_rn(x, c)) + 4u) & ~7u;
  return __float_as_uint(__uint_as_float(t) + WHOLE);
}

// Largest |x| of one 16-byte piece, as the bits of its type (16-bit types: of one of
// two halves): a NaN or an infinity is above every number.
template <int T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m, const uint4& raw, float inv) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (T == QX_T_BF16 || T == QX_T_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  } else if constexpr (T == QX_T_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, w[i] & 0x7fffffffu);
  } else {
    float v[16];
    unpack<T>(raw, inv, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  return m;
}

// One CTA per row, about four 16-byte pieces per thread. The row is read once and
// kept in registers (raw) between the maximum and the quantisation; what is longer
// than NV pieces per thread is read again. Bound by the bytes (8192 x 5120 BF16: 24.3 us,
// 5.2 TB/s; 8192 x 2304 FP32: 17.8 us, 5.3 TB/s; a persistent form, the next row's loads
// ahead, took 48 us where this one then took 35). early: 1 lets the
// kernels behind this one start before it has waited for the ones in front (their
// weights are then known to be complete).
constexpr int QTHR = 512, NV = 4;

template <int T, bool VEC>
__global__ void __launch_bounds__(QTHR) quant_kernel(const void* x, int64_t xs, const float* x_scale, int per_row,
                                                     int k, int8_t* q, int64_t qs, float* scale, int q_vec,
                                                     int early) {
  constexpr int E = per16<T>();
  if (early) pdl_launch_dependents();
  pdl_wait();
  if (!early) pdl_launch_dependents();
  const int64_t r = blockIdx.x, off = r * xs;
  const float inv = T == QX_T_E4M3 ? __ldcg(&x_scale[per_row ? r : 0]) : 1.f;
  const int pieces = (k + E - 1) / E, thr = blockDim.x;
  uint4 raw[NV];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int g = threadIdx.x + i * thr;
    raw[i] = g < pieces ? load16<T, VEC>(x, off, g * E, k) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) m = top_bits<T>(m, raw[i], inv);
  for (int g = threadIdx.x + NV * thr; g < pieces; g += thr) m = top_bits<T>(m, load16<T, VEC>(x, off, g * E, k), inv);
  if constexpr (T == QX_T_BF16) m = max(m << 16, m & 0xffff0000u);
  if constexpr (T == QX_T_F16)                     // FP16's largest as FP32 bits (infinity and NaN stay so)
    m = __float_as_uint(__half2float(__ushort_as_half((uint16_t)max(m & 0xffffu, m >> 16))));
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t sm[QTHR / 32];
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < thr / 32; ++i) m = max(m, sm[i]);
  const bool bad = m >= INF_BITS;
  const float mc = fmaxf(__uint_as_float(m), AMAX_FLOOR);
  const float c = __fdiv_rn(QMAX, mc);
  const uint32_t keep = bad ? 0u : 0xffffffffu;
  if (threadIdx.x == 0) {
    scale[r] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(mc, QMAX);
    if (bad) atomicOr(&g_status, (uint32_t)QX_DEV_NONFINITE);
  }
  int8_t* qr = q + r * qs;
  auto put = [&](const uint4& w, int g) {
    float v[E];
    unpack<T>(w, inv, v);
    uint32_t o[E / 4];
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      uint32_t n[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = quotient<T>(v[j + i], c);
      o[j / 4] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410) & keep;
    }
    if (q_vec && (g + 1) * E <= k) {
      if constexpr (E == 16) *reinterpret_cast<uint4*>(qr + g * E) = make_uint4(o[0], o[1], o[2], o[3]);
      else if constexpr (E == 8) *reinterpret_cast<uint2*>(qr + g * E) = make_uint2(o[0], o[1]);
      else *reinterpret_cast<uint32_t*>(qr + g * E) = o[0];
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (g * E + j < k) qr[g * E + j] = (int8_t)(o[j / 4] >> (8 * (j % 4)));
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (threadIdx.x + i * thr < pieces) put(raw[i], threadIdx.x + i * thr);
  for (int g = threadIdx.x + NV * thr; g < pieces; g += thr) put(load16<T, VEC>(x, off, g * E, k), g);
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

// 16 bytes of a row from byte address p on, the first n >= 1 of them valid (the others 0):
// aligned words that overlap the valid bytes, shifted into place.
__device__ __forceinline__ uint4 load16_any(const int8_t* p, int n) {
  const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3u);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p - sh);
  uint32_t v[5], o[4];
#pragma unroll
  for (int j = 0; j < 5; ++j) v[j] = 4 * j < (int)sh + n ? __ldcg(w + j) : 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int left = n - 4 * j;                          // valid bytes of this word and those behind it
    o[j] = __funnelshift_r(v[j], v[j + 1], 8 * sh) & (left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << 8 * left) - 1u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Any alignment: 64 x 64 sums per CTA by dp4a over 64-byte pieces of K in shared
// memory, the next piece's loads under way meanwhile. Serves rows whose address or
// stride the copy engine cannot take (not a multiple of 16 bytes); bound by dp4a's
// rate (2048 x 5120 x 2303: 669 us against 20.6 for aligned rows) and with few tokens
// by the latency of its rounds over K (1 x 2222 x 1111: 25 us; byte loads took 76).
constexpr int ST = 64, SKB = 64;
__global__ void __launch_bounds__(256) plain_kernel(Args p) {
  __shared__ __align__(16) int8_t sa[ST][SKB + 4], sw[ST][SKB + 4];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int half = p.swiglu ? ST / 2 : ST;               // output columns of the tile
  const int n0 = blockIdx.x * half, m0 = blockIdx.y * ST;
  int32_t acc[4][4] = {};                                // tokens ty + 16 i, weight rows tx + 16 j
  const int r = tid >> 2, c = (tid & 3) * 16;            // this thread's row of both operands, its 16 bytes
  const int nr = n0 + (r < half ? r : r - half);         // output column of its weight row
  const int8_t* pa = m0 + r < p.m ? p.a + (int64_t)(m0 + r) * p.as + c : nullptr;
  const int8_t* pw = nr < p.n ? p.w + (int64_t)(r < half ? nr : p.n + nr) * p.ws + c : nullptr;
  uint4 va, vw;
  auto fetch = [&](int k0) {
    const int left = p.k - k0 - c, n = left < 16 ? left : 16;
    va = pa && n > 0 ? load16_any(pa + k0, n) : make_uint4(0u, 0u, 0u, 0u);
    vw = pw && n > 0 ? load16_any(pw + k0, n) : make_uint4(0u, 0u, 0u, 0u);
  };
  auto put = [&](int8_t* to, const uint4& v) {
    uint32_t* t = reinterpret_cast<uint32_t*>(to);
    t[0] = v.x; t[1] = v.y; t[2] = v.z; t[3] = v.w;
  };
  fetch(0);
  for (int k0 = 0; k0 < p.k; k0 += SKB) {
    put(&sa[r][c], va);
    put(&sw[r][c], vw);
    __syncthreads();
    if (k0 + SKB < p.k) fetch(k0 + SKB);
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
      cudaFuncSetAttribute(pair_kernel, attr, (int)PAIR_SMEM) != cudaSuccess)
    return 0;
  return cached[dev] = sms;
}

uint64_t wait_limit_ns() {
  const char* e = getenv("QX_TIMEOUT_MS");
  const long ms = e ? atol(e) : 1000;
  return (uint64_t)(ms < 10 ? 10 : ms) * 1000000ull;
}

// Test hook QX_TEST_INT8_HOLD: bounded waits that run out, with QX_DEV_TIMEOUT recorded. 1:
// the barriers behind which the epilogues read the sums expect one arrival too many; 2: the
// thread that issues the MMAs waits for something that does not come before it takes the
// first stage, and gives up with a ring full of copies in flight.
int test_hold() {
  const char* e = getenv("QX_TEST_INT8_HOLD");
  return e ? atoi(e) : 0;
}

int element_size(int type) { return type == QX_T_F32 ? 4 : type == QX_T_E4M3 ? 1 : 2; }

// Tiled-copy descriptor of rows x cols elements of 1, 2 or 4 bytes; places outside
// the tensor read as 0 and are not written.
bool tiled_map(CUtensorMap* map, const void* base, int esz, int64_t rows, int64_t cols, int64_t stride_bytes, int box_cols,
               int box_rows, CUtensorMapSwizzle swizzle) {
  static decltype(&cuTensorMapEncodeTiled) encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
  }();
  if (!encode) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUtensorMapDataType type = esz == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : esz == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                              : CU_TENSOR_MAP_DATA_TYPE_UINT32;
  return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Of int8 rows [rows, k]: boxes of one 128-byte swizzle span x box_rows.
bool row_map(CUtensorMap* map, const int8_t* base, int64_t rows, int k, int64_t stride, int box_rows) {
  return tiled_map(map, base, 1, rows, k, stride, KST, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Every kernel here is launched so that it may start while the one in front of it
// on the stream still runs (programmatic dependent launch): it sets itself up,
// then waits for that one before it touches global memory.
struct Launch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  Launch(dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster = 1) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
  }
  template <typename... P, typename... A>
  int operator()(void (*kernel)(P...), A... args) {
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) == cudaSuccess ? QX_OK : QX_ERR_LAUNCH;
  }
};

// Tile of the pair kernel: tokens per CTA (the tokens spread evenly over the fewest
// tiles of 256) and the weight rows with the smallest estimated time. A wave of tiles
// over the pairs takes, per 128-byte chunk of K, the longer of the MMAs (1.3 ns a weight
// row) and the copies into one SM (64 bytes a clock: 1.05 ns a row of its operands, 60 ns
// at least), or an epilogue (1.4 us for 256 rows) if that is longer; the last epilogue
// comes on top. Measured at 2048 x 5120 x 2304: 20.4 us with 224 rows, 20.6 with 192 (which the
// estimate takes), 21.1 with 256 (each 3 waves), 21.9 with 128 (5).
void pair_tile(const Args& p, int sms, int* tb, int* bn) {
  const int tiles_m = (p.m + 255) / 256, pairs = sms / 2, chunks = (p.k + (int)KST - 1) / (int)KST;
  const int h = p.swiglu ? 2 : 1, step = 32 * h;
  *tb = (p.m + 64 * tiles_m - 1) / (64 * tiles_m) * 32;
  double least = 0;
  for (int b = 256; b >= 64; b -= step) {
    const int64_t tiles = (int64_t)tiles_m * ((p.n + b / h - 1) / (b / h));
    const double mma = 1.3 * b, copy = 1.05 * (*tb + b / 2), epi = 1400.0 * b / 256;
    const double chunk = mma > copy ? (mma > 60 ? mma : 60) : (copy > 60 ? copy : 60), loop = chunks * chunk;
    const double ns = (double)((tiles + pairs - 1) / pairs) * (loop > epi ? loop : epi) + epi;
    if (least == 0 || ns < least) *bn = b, least = ns;
  }
}

int pair_launch(const Args& p, int prefetch, int sms, cudaStream_t st) {
  int tb = 0, bn = 0;
  pair_tile(p, sms, &tb, &bn);
  const int cols = p.swiglu ? bn / 2 : bn, tiles_m = (p.m + 2 * tb - 1) / (2 * tb);
  const int64_t tiles = (int64_t)tiles_m * ((p.n + cols - 1) / cols);
  if (tiles > 0x7fffffff) return QX_ERR_SHAPE;
  const int pairs = (int)(tiles < sms / 2 ? tiles : sms / 2), osz = element_size(p.type);
  CUtensorMap tw, ta, to = {};
  if (!row_map(&tw, p.w, p.swiglu ? 2ll * p.n : p.n, p.k, p.ws, bn / 2) || !row_map(&ta, p.a, p.m, p.k, p.as, tb))
    return QX_ERR_DEVICE;
  const int spans = bn >= 160 ? 1 : 2;   // from 160 rows on the MMAs of one span outlast the issuing threads' loop
  // Tiled stores where the output's rows start on 16-byte boundaries.
  const int tma = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.os * osz % 16 == 0 &&
                  tiled_map(&to, p.out, osz, p.m, p.n, p.os * osz, 64 / osz, 32, CU_TENSOR_MAP_SWIZZLE_64B);
  return Launch(dim3(2 * pairs, 1, 1), PAIR_THR, PAIR_SMEM, st, 2)(pair_kernel, tw, ta, to, p, tb, bn, spans, tiles_m,
                                                                  (int)tiles, prefetch, tma, wait_limit_ns(), test_hold());
}

// K pieces of the split kernel (1..8): the fewest that leave a CTA the least of K while
// all clusters fit on the GPU at once (two CTAs per SM, less what clusters leave unused of
// a group of SMs: 1.65 per SM; 5120 x 5120 with one token: 8.0 us in 5 pieces, 8.2 in 6, 11.4 in 7).
int pieces_of(int64_t tiles, int chunks, int sms) {
  int best = 1;
  for (int s = 2; s <= 8 && s <= chunks; ++s)
    if (tiles * s * 20 <= (int64_t)sms * 33 && (chunks + s - 1) / s < (chunks + best - 1) / best) best = s;
  return best;
}

template <int BN>
int split_launch(const Args& p, int prefetch, int sms, cudaStream_t st) {
  using L = Split<BN>;
  const int half = p.swiglu ? 64 : 128, tiles = (p.n + half - 1) / half;
  const int pieces = pieces_of(tiles, (p.k + (int)KST - 1) / (int)KST, sms);
  CUtensorMap tw, ta;
  if (!row_map(&tw, p.w, p.swiglu ? 2ll * p.n : p.n, p.k, p.ws, half) || !row_map(&ta, p.a, p.m, p.k, p.as, BN))
    return QX_ERR_DEVICE;
  return Launch(dim3((unsigned)(tiles * pieces), 1, 1), SPLIT_THR, L::SMEM, st, pieces)(
      split_kernel<BN>, tw, ta, p, pieces, prefetch, wait_limit_ns(), test_hold());
}

// A checked product. prefetch: the weights are complete when this kernel starts,
// so their copies may go out before it waits for the kernel in front.
int product(Args p, int prefetch, int sms, cudaStream_t st) {
  // Tiled copies need rows that start on 16-byte boundaries (a single row: its address only).
  auto aligned = [](const int8_t* b, int64_t stride, int64_t rows) {
    return reinterpret_cast<uintptr_t>(b) % 16 == 0 && (stride % 16 == 0 || rows == 1);
  };
  if (aligned(p.a, p.as, p.m) && aligned(p.w, p.ws, p.swiglu ? 2 : p.n)) {
    if (p.m == 1) p.as = (p.as + 15) / 16 * 16;          // never stepped
    if (p.n == 1 && !p.swiglu) p.ws = (p.ws + 15) / 16 * 16;
    // Up to 32 tokens by K pieces, more by pairs (4608 x 5120: 7.7 us against 10.5
    // with 1 token, 9.0 against 9.6 with 32; 5120 x 2304: 6.1 against 7.0, 7.1 against 6.6).
    if (p.m > 32) return pair_launch(p, prefetch, sms, st);
    return p.m <= 16 ? split_launch<16>(p, prefetch, sms, st) : split_launch<32>(p, prefetch, sms, st);
  }
  const int half = p.swiglu ? ST / 2 : ST;
  int rc = QX_OK;
  for (int64_t left = p.m; rc == QX_OK && left > 0; left -= p.m) {   // row blocks of what a grid's y counts
    p.m = (int)(left < 65535ll * ST ? left : 65535ll * ST);
    rc = Launch(dim3((unsigned)((p.n + half - 1) / half), (unsigned)((p.m + ST - 1) / ST), 1), 256, 0, st)(plain_kernel, p);
    p.a += p.m * p.as;
    p.sa += p.m;
    p.out = reinterpret_cast<uint8_t*>(p.out) + p.m * p.os * element_size(p.type);
  }
  return rc;
}

template <int T>
int quant_launch(const void* x, int64_t xs, const float* x_scale, int per_row, int64_t rows, int k, int8_t* q,
                 int64_t qs, float* scale, int early, cudaStream_t st) {
  constexpr int E = per16<T>(), B = 16 / E;
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && xs * B % 16 == 0;
  const int q_vec = reinterpret_cast<uintptr_t>(q) % E == 0 && qs % E == 0;
  const int pieces = (k + E - 1) / E, want = ((pieces + NV - 1) / NV + 31) / 32 * 32;
  Launch l(dim3((unsigned)rows, 1, 1), want < QTHR ? want : QTHR, 0, st);
  return vec ? l(quant_kernel<T, true>, x, xs, x_scale, per_row, k, q, qs, scale, q_vec, early)
             : l(quant_kernel<T, false>, x, xs, x_scale, per_row, k, q, qs, scale, q_vec, early);
}

int quantise(const void* x, int64_t xs, int type, const float* x_scale, int per_row, int64_t rows, int k, int8_t* q,
             int64_t qs, float* scale, int early, cudaStream_t st) {
  if (type == QX_T_BF16) return quant_launch<QX_T_BF16>(x, xs, x_scale, per_row, rows, k, q, qs, scale, early, st);
  if (type == QX_T_F16) return quant_launch<QX_T_F16>(x, xs, x_scale, per_row, rows, k, q, qs, scale, early, st);
  if (type == QX_T_F32) return quant_launch<QX_T_F32>(x, xs, x_scale, per_row, rows, k, q, qs, scale, early, st);
  return quant_launch<QX_T_E4M3>(x, xs, x_scale, per_row, rows, k, q, qs, scale, early, st);
}

int check_x(const void* x, int64_t x_stride, int type, const float* x_scale, int64_t n_scale, int64_t rows, int k) {
  if (!x) return QX_ERR_ARG;
  if (type == QX_T_E4M3 && (!x_scale || (n_scale != 1 && n_scale != rows))) return QX_ERR_ARG;
  if (x_stride < k) return QX_ERR_SHAPE;
  return reinterpret_cast<uintptr_t>(x) % element_size(type) ? QX_ERR_ALIGN : QX_OK;
}

constexpr int MAX_DIM = 1 << 24;

// Rows of q, its scales, h, q2 and its scales in an expert's workspace, each on a
// 16-byte boundary with rows a multiple of 16 bytes apart.
struct ExpertLayout {
  int64_t qs, hs, q2s;
  size_t q, s, h, q2, s2, total;
  ExpertLayout(int64_t rows, int k, int inter) {
    qs = (k + 15) / 16 * 16;
    hs = (inter + 3) / 4 * 4;
    q2s = (inter + 15) / 16 * 16;
    auto al = [](size_t v) { return (v + 255) & ~size_t(255); };
    q = 0;
    s = al(q + (size_t)rows * qs);
    h = al(s + (size_t)rows * 4);
    q2 = al(h + (size_t)rows * hs * 4);
    s2 = al(q2 + (size_t)rows * q2s);
    total = al(s2 + (size_t)rows * 4);
  }
};
}  // namespace

extern "C" {

int qx_quant_int8(const void* x, int64_t x_stride, int32_t x_type, const float* x_scale, int64_t n_scale,
                  int64_t rows, int32_t k, int8_t* q, int64_t q_stride, float* scale, void* stream) {
  if (rows < 0 || rows > 0x7fffffffll || k < 1 || k > QX_INT8_MAX_K) return QX_ERR_SHAPE;
  if (x_type < QX_T_BF16 || x_type > QX_T_E4M3) return QX_ERR_ARG;
  if (rows == 0) return QX_OK;
  if (!q || !scale) return QX_ERR_ARG;
  if (const int rc = check_x(x, x_stride, x_type, x_scale, n_scale, rows, k)) return rc;
  if (q_stride < k) return QX_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(scale) % 4) return QX_ERR_ALIGN;
  if (device_sms() <= 0) return QX_ERR_DEVICE;
  return quantise(x, x_stride, x_type, x_scale, n_scale == rows, rows, k, q, q_stride, scale, 0,
                  reinterpret_cast<cudaStream_t>(stream));
}

int qx_int8_matmul(const QxInt8Args* a, void* stream) {
  if (!a) return QX_ERR_ARG;
  if (a->m < 0 || a->n < 1 || a->n > MAX_DIM || a->m > MAX_DIM || a->k < 1 || a->k > QX_INT8_MAX_K)
    return QX_ERR_SHAPE;
  if (a->out_type < QX_T_BF16 || a->out_type > QX_T_F32) return QX_ERR_ARG;
  if (a->m == 0) return QX_OK;
  if (!a->a || !a->w || !a->a_scale || !a->w_scale || !a->out) return QX_ERR_ARG;
  if (a->a_stride < a->k || a->w_stride < a->k || a->out_stride < a->n) return QX_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(a->out) % element_size(a->out_type) ||
      reinterpret_cast<uintptr_t>(a->a_scale) % 4 || reinterpret_cast<uintptr_t>(a->w_scale) % 4)
    return QX_ERR_ALIGN;
  const int sms = device_sms();
  if (sms <= 0) return QX_ERR_DEVICE;
  Args p;
  p.a = a->a; p.w = a->w; p.sa = a->a_scale; p.sw = a->w_scale; p.out = a->out;
  p.as = a->a_stride; p.ws = a->w_stride; p.os = a->out_stride;
  p.m = a->m; p.n = a->n; p.k = a->k; p.type = a->out_type;
  p.swiglu = a->swiglu ? 1 : 0; p.has_limit = a->has_limit ? 1 : 0; p.limit = a->limit;
  return product(p, 0, sms, reinterpret_cast<cudaStream_t>(stream));
}

size_t qx_int8_expert_workspace_bytes(int32_t rows, int32_t k, int32_t inter) {
  if (rows < 0 || rows > MAX_DIM || k < 1 || k > QX_INT8_MAX_K || inter < 1 || inter > QX_INT8_MAX_K) return 0;
  return ExpertLayout(rows, k, inter).total;
}

int qx_int8_expert(const QxInt8ExpertArgs* a, void* stream) {
  if (!a) return QX_ERR_ARG;
  if (a->rows < 0 || a->rows > MAX_DIM || a->k < 1 || a->k > QX_INT8_MAX_K || a->inter < 1 ||
      a->inter > QX_INT8_MAX_K)
    return QX_ERR_SHAPE;
  if (a->x_type < QX_T_BF16 || a->x_type > QX_T_E4M3 || a->out_type < QX_T_BF16 || a->out_type > QX_T_F32)
    return QX_ERR_ARG;
  if (a->rows == 0) return QX_OK;
  if (!a->w13 || !a->w13_scale || !a->w2 || !a->w2_scale || !a->out || !a->workspace) return QX_ERR_ARG;
  if (const int rc = check_x(a->x, a->x_stride, a->x_type, a->x_scale, a->n_scale, a->rows, a->k)) return rc;
  if (a->w13_stride < a->k || a->w2_stride < a->inter || a->out_stride < a->k) return QX_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(a->out) % element_size(a->out_type) ||
      reinterpret_cast<uintptr_t>(a->w13_scale) % 4 || reinterpret_cast<uintptr_t>(a->w2_scale) % 4 ||
      reinterpret_cast<uintptr_t>(a->workspace) % 16)
    return QX_ERR_ALIGN;
  const ExpertLayout L(a->rows, a->k, a->inter);
  if (a->workspace_bytes < L.total) return QX_ERR_WORKSPACE;
  const int sms = device_sms();
  if (sms <= 0) return QX_ERR_DEVICE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* ws = reinterpret_cast<uint8_t*>(a->workspace);
  Args p;
  p.a = reinterpret_cast<int8_t*>(ws + L.q); p.as = L.qs; p.sa = reinterpret_cast<float*>(ws + L.s);
  p.w = a->w13; p.ws = a->w13_stride; p.sw = a->w13_scale;
  p.out = ws + L.h; p.os = L.hs; p.type = QX_T_F32;
  p.m = a->rows; p.n = a->inter; p.k = a->k;
  p.swiglu = 1; p.has_limit = a->has_limit ? 1 : 0; p.limit = a->limit;
  Args d = p;
  d.a = reinterpret_cast<int8_t*>(ws + L.q2); d.as = L.q2s; d.sa = reinterpret_cast<float*>(ws + L.s2);
  d.w = a->w2; d.ws = a->w2_stride; d.sw = a->w2_scale;
  d.out = a->out; d.os = a->out_stride; d.type = a->out_type;
  d.n = a->k; d.k = a->inter; d.swiglu = 0;
  int rc = quantise(a->x, a->x_stride, a->x_type, a->x_scale, a->n_scale == a->rows, a->rows, a->k,
                    reinterpret_cast<int8_t*>(ws + L.q), L.qs, reinterpret_cast<float*>(ws + L.s), 0, st);
  // The first quantiser lets the products start only after everything queued before
  // this call is complete, the weights included: their copies go out at once.
  if (rc == QX_OK) rc = product(p, 1, sms, st);
  if (rc == QX_OK)
    rc = quantise(ws + L.h, L.hs, QX_T_F32, nullptr, 0, a->rows, a->inter, reinterpret_cast<int8_t*>(ws + L.q2), L.q2s,
                  reinterpret_cast<float*>(ws + L.s2), 1, st);
  if (rc == QX_OK) rc = product(d, 1, sms, st);
  return rc;
}

int qx_int8_status(uint32_t* status, void* stream) {
  if (!status) return QX_ERR_ARG;
  if (device_sms() <= 0) return QX_ERR_DEVICE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> busy{0};                   // words of g_taken in use
  uint64_t b = busy.load();
  int slot = 0;
  do {
    while (b == ~0ull) std::this_thread::yield(), b = busy.load();
    slot = __builtin_ctzll(~b);
  } while (!busy.compare_exchange_weak(b, b | 1ull << slot));
  take_status_kernel<<<1, 1, 0, st>>>(slot);
  bool ok = cudaGetLastError() == cudaSuccess;
  ok = ok && cudaMemcpyFromSymbolAsync(status, g_taken, sizeof(uint32_t), slot * sizeof(uint32_t), cudaMemcpyDeviceToHost,
                                       st) == cudaSuccess;
  ok = cudaStreamSynchronize(st) == cudaSuccess && ok;
  busy.fetch_and(~(1ull << slot));
  return ok ? QX_OK : QX_ERR_LAUNCH;
}

}  // extern "C"
