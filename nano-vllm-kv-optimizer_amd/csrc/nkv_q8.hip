// 8-bit projections of the decoder (the Qwen3 modules that call the sparse
// layer-step): rows held as signed 8-bit codes with one fp32 scale a row, and
// products of such rows in integers.
//
//  * A row y[n] is held as q = rne(y * 127 / a), s = a / 127 with a = max |y|:
//    y ~ q s, off by at most s / 2.  Rows with a < 2^-119 (where 127 / a would
//    leave fp32's range) are zero: s = 0.  A row with a NaN or an infinity has
//    s = NaN and q = 0, so whatever is computed from it is NaN.
//  * A weight [n][k] is held the same way, one scale an output channel.
//  * Y[m][c] = (sum_k xq[m][k] wq[c][k]) sx[m] sw[c] (+ bias[c]): the sum is
//    exact in 32-bit integers (k <= 131056 codes of magnitude <= 128), so it
//    does not depend on how it is cut over lanes, wavefronts or tiles.
#include <algorithm>

#include "nkv_common.h"

namespace nkv {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr float kTiny = 0x1p-119f;       // rows whose largest magnitude is below are zero
constexpr int kMaxRow = 32768;           // longest row that is quantised
constexpr int kMaxDepth = 131056;        // longest product: 131056 * 128 * 128 < 2^31

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}

// The magnitude's bits, whose order as integers is the magnitudes' order with
// the infinities and NaN on top.
__device__ __forceinline__ uint32_t mag(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// 4 codes: rne(v * inv) for |v * inv| <= 127.5, in the low byte of the sum with
// 1.5 * 2^23 (one fma, its rounding to nearest even); NaN gives 0.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t x = __float_as_uint(__builtin_fmaf(a, inv, kMagic)), y = __float_as_uint(__builtin_fmaf(b, inv, kMagic));
  const uint32_t z = __float_as_uint(__builtin_fmaf(c, inv, kMagic)), w = __float_as_uint(__builtin_fmaf(d, inv, kMagic));
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400u), __builtin_amdgcn_perm(y, x, 0x0c0c0400u), 0x05040100u);
}

// scale and its inverse for a row whose largest magnitude is `top` (as bits)
struct RowScale {
  float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float a = __uint_as_float(top);
  if (top >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
  if (a < kTiny) return {0.0f, 0.0f};
  return {a / 127.0f, 127.0f / a};
}

// The same for a row t * r, r = rsqrt(mean(t^2) + eps), given the largest |t w|:
// the codes do not depend on r.  NaN also where the squares pass fp32's range.
__device__ __forceinline__ RowScale norm_row_scale(uint32_t top, float ss, int n, float eps) {
  RowScale rs = row_scale(top);
  const float r = rsqrtf(ss / static_cast<float>(n) + eps);
  const float a = __uint_as_float(top) * r;
  if (rs.scale == 0.0f || a < kTiny) rs = {0.0f, 0.0f};
  else rs.scale = a / 127.0f;
  if (mag(ss) >= 0x7f800000u || mag(a) >= 0x7f800000u) rs = {__uint_as_float(0x7fc00000u), 0.0f};
  return rs;
}

// One workgroup of THREADS a row; NCH 8-element chunks a thread.
constexpr int kRowChunks = 4;
template <int THREADS, bool NORM>
__global__ __launch_bounds__(THREADS) void rows_q8_kernel(const uint16_t* __restrict__ x, int64_t x_stride,
                                                          const uint16_t* __restrict__ res,
                                                          const uint16_t* __restrict__ w, float eps,
                                                          int8_t* __restrict__ q, float* __restrict__ scale,
                                                          uint16_t* __restrict__ res_out, int n) {
  __shared__ float s_sum[THREADS / kWave];
  __shared__ uint32_t s_top[THREADS / kWave];
  const int64_t row = blockIdx.x;
  const int nc = n >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * x_stride);
  const uint4* rr = NORM && res ? reinterpret_cast<const uint4*>(res + row * n) : nullptr;
  uint4* ro = NORM && res_out ? reinterpret_cast<uint4*>(res_out + row * n) : nullptr;
  float v[kRowChunks][8];
  float ss = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kRowChunks; ++j) {
    const int c = threadIdx.x + j * THREADS;
    if (c < nc) {
      unpack8(xr[c], v[j]);
      if constexpr (NORM) {
        float wf[8];
        unpack8(reinterpret_cast<const uint4*>(w)[c], wf);
        if (rr) {
          float r[8];
          unpack8(rr[c], r);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] += r[e];
        }
        if (ro) ro[c] = pack8(v[j]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss += v[j][e] * v[j][e];
          v[j][e] *= wf[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, mag(v[j][e]));
    }
  }
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    ss += __shfl_xor(ss, o);
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
  }
  if constexpr (THREADS > kWave) {
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) s_sum[wave] = ss, s_top[wave] = top;
    __syncthreads();
    ss = 0.0f;
    top = 0;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) ss += s_sum[i], top = max(top, s_top[i]);
  }
  const RowScale rs = NORM ? norm_row_scale(top, ss, n, eps) : row_scale(top);
  uint2* qr = reinterpret_cast<uint2*>(q + row * n);
#pragma unroll
  for (int j = 0; j < kRowChunks; ++j) {
    const int c = threadIdx.x + j * THREADS;
    if (c < nc)
      qr[c] = make_uint2(codes4(v[j][0], v[j][1], v[j][2], v[j][3], rs.inv), codes4(v[j][4], v[j][5], v[j][6], v[j][7], rs.inv));
  }
  if (threadIdx.x == 0) scale[row] = rs.scale;
}

// One thread per 16 codes.
__global__ __launch_bounds__(256) void dequantize_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                         uint16_t* __restrict__ out, int64_t chunks, int n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int64_t row = i / (n >> 4);
  const float s = scale[row];
  const i32x4 c = reinterpret_cast<const i32x4*>(q)[i];
  uint4* o = reinterpret_cast<uint4*>(out) + 2 * i;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = s * static_cast<float>(static_cast<int8_t>(c[2 * h + (e >> 2)] >> (8 * (e & 3))));
    o[h] = pack8(f);
  }
}

// SiLU(g) * u in fp32.
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// A product's sum in fp32, scaled by token and channel: every kernel rounds alike.
__device__ __forceinline__ float scaled(int acc, float sx, float sw, float bias) {
  return __builtin_fmaf(static_cast<float>(acc) * sx, sw, bias);
}

struct Product {
  const int8_t* w;        // [n][k], or with SILU gate|up [2 n][k]
  const float* sw;
  const int8_t* x;        // [m][k]
  const float* sx;
  const uint16_t* bias;   // [n] bf16, or null
  uint16_t* y;            // [m][n]
  int m, n, k;
};

// A wavefront owns 16 channels x 16 rows and reads its operands from memory.
template <bool SILU>
__global__ __launch_bounds__(256) void product_kernel(const Product p) {
  const int lane = threadIdx.x & (kWave - 1);
  const int c0 = blockIdx.x * 64 + static_cast<int>(threadIdx.x / kWave) * 16;
  const int m0 = blockIdx.y * 16;
  if (c0 >= p.n) return;
  const int r = lane & 15, g = lane >> 4;
  const int8_t* wr = p.w + static_cast<int64_t>(min(c0 + r, p.n - 1)) * p.k;
  const int8_t* ur = wr + static_cast<int64_t>(p.n) * p.k;   // SILU: the up row
  const int8_t* xr = p.x + static_cast<int64_t>(min(m0 + r, p.m - 1)) * p.k;
  i32x4 acc = {0, 0, 0, 0}, up = {0, 0, 0, 0};
  for (int k = 16 * g; k < p.k + 16 * g; k += 64) {
    i32x4 a = {0, 0, 0, 0}, b = a, u = a;
    if (k < p.k) {
      a = *reinterpret_cast<const i32x4*>(wr + k);
      b = *reinterpret_cast<const i32x4*>(xr + k);
      if constexpr (SILU) u = *reinterpret_cast<const i32x4*>(ur + k);
    }
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
    if constexpr (SILU) up = __builtin_amdgcn_mfma_i32_16x16x64_i8(u, b, up, 0, 0, 0);
  }
  const int m = m0 + r;
  if (m >= p.m) return;
  const float sx = p.sx[m];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = c0 + 4 * g + e;
    if (c >= p.n) break;
    float v = scaled(acc[e], sx, p.sw[c], p.bias ? bf16_to_f32(p.bias[c]) : 0.0f);
    if constexpr (SILU) v = silu_mul(v, scaled(up[e], sx, p.sw[p.n + c], 0.0f));
    p.y[static_cast<int64_t>(m) * p.n + c] = f32_to_bf16(v);
  }
}

__device__ __forceinline__ int dot16(const i32x4& a, const i32x4& b, int acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_sdot4(a[e], b[e], acc, false);
  return acc;
}

// The same product for 1-4 rows that are still bf16, with the rows' norm
// (NORM) and quantisation in the same launch: every workgroup quantises the rows
// into LDS, then each of its wavefronts takes channel pairs (SILU: a gate
// channel and its up channel), lanes along k.
struct Token {
  const int8_t* w;
  const float* sw;
  const uint16_t* x;      // [m][k] bf16
  const uint16_t* res;    // NORM: residual added first, or null
  const uint16_t* nw;     // NORM: norm weight
  const uint16_t* bias;
  uint16_t* y;
  uint16_t* res_out;      // NORM: bf16(x + res), or null
  float eps;
  int n, k;
};
constexpr int kTokenThreads = 256;
constexpr int kTokenWaves = kTokenThreads / kWave;

template <int MR, bool NORM, bool SILU>
__global__ __launch_bounds__(kTokenThreads) void token_kernel(const Token p) {
  extern __shared__ uint4 s_codes[];     // [MR][k / 16]
  __shared__ float s_sum[kTokenWaves][MR];
  __shared__ uint32_t s_top[kTokenWaves][MR];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1);
  const int nc = p.k >> 3;
  float ss[MR];
  uint32_t top[MR];
  auto load = [&](int m, int c, float (&v)[8], bool first) {
    const int64_t at = static_cast<int64_t>(m) * nc + c;
    unpack8(reinterpret_cast<const uint4*>(p.x)[at], v);
    if constexpr (NORM) {
      if (p.res) {
        float r[8];
        unpack8(reinterpret_cast<const uint4*>(p.res)[at], r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      }
      if (first && p.res_out && blockIdx.x == 0) reinterpret_cast<uint4*>(p.res_out)[at] = pack8(v);
      if (first)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[m] += v[e] * v[e];
      float wf[8];
      unpack8(reinterpret_cast<const uint4*>(p.nw)[c], wf);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= wf[e];
    }
  };
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    ss[m] = 0.0f;
    top[m] = 0;
    for (int c = threadIdx.x; c < nc; c += kTokenThreads) {
      float v[8];
      load(m, c, v, true);
#pragma unroll
      for (int e = 0; e < 8; ++e) top[m] = max(top[m], mag(v[e]));
    }
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) {
      ss[m] += __shfl_xor(ss[m], o);
      top[m] = max(top[m], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[m]), o)));
    }
    if (lane == 0) s_sum[wave][m] = ss[m], s_top[wave][m] = top[m];
  }
  __syncthreads();
  float sx[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    float sum = 0.0f;
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < kTokenWaves; ++i) sum += s_sum[i][m], all = max(all, s_top[i][m]);
    const RowScale rs = NORM ? norm_row_scale(all, sum, p.k, p.eps) : row_scale(all);
    sx[m] = rs.scale;
    for (int c = threadIdx.x; c < nc; c += kTokenThreads) {
      float v[8];
      load(m, c, v, false);
      reinterpret_cast<uint2*>(s_codes)[m * nc + c] =
          make_uint2(codes4(v[0], v[1], v[2], v[3], rs.inv), codes4(v[4], v[5], v[6], v[7], rs.inv));
    }
  }
  __syncthreads();

  const int nq = p.k >> 4;
  const i32x4* xv = reinterpret_cast<const i32x4*>(s_codes);
  const int units = SILU ? p.n : (p.n + 1) >> 1;
  for (int u = blockIdx.x * kTokenWaves + wave; u < units; u += gridDim.x * kTokenWaves) {
    const i32x4* w0 = reinterpret_cast<const i32x4*>(p.w + static_cast<int64_t>(SILU ? u : 2 * u) * p.k);
    const i32x4* w1 = reinterpret_cast<const i32x4*>(p.w + static_cast<int64_t>(SILU ? u + p.n : min(2 * u + 1, p.n - 1)) * p.k);
    int acc[MR][2] = {};
    for (int c = lane; c < nq; c += kWave) {
      const i32x4 a = w0[c], b = w1[c];
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const i32x4 xm = xv[m * nq + c];
        acc[m][0] = dot16(a, xm, acc[m][0]);
        acc[m][1] = dot16(b, xm, acc[m][1]);
      }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int o = kWave / 2; o > 0; o >>= 1) acc[m][j] += __shfl_xor(acc[m][j], o);
    if (lane != 0) continue;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      uint16_t* y = p.y + static_cast<int64_t>(m) * p.n;
      if constexpr (SILU) {
        y[u] = f32_to_bf16(silu_mul(scaled(acc[m][0], sx[m], p.sw[u], 0.0f), scaled(acc[m][1], sx[m], p.sw[p.n + u], 0.0f)));
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = 2 * u + j;
          if (c < p.n) y[c] = f32_to_bf16(scaled(acc[m][j], sx[m], p.sw[c], p.bias ? bf16_to_f32(p.bias[c]) : 0.0f));
        }
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether two ranges of bytes have none in common (NULL: no range).
bool apart(const void* a, int64_t na, const void* b, int64_t nb) {
  const char *pa = static_cast<const char*>(a), *pb = static_cast<const char*>(b);
  return !a || !b || pa + na <= pb || pb + nb <= pa;
}

template <bool NORM>
void launch_rows(const uint16_t* x, int64_t x_stride, const uint16_t* res, const uint16_t* w, float eps, int8_t* q,
                 float* scale, uint16_t* res_out, int rows, int n, hipStream_t s) {
  auto go = [&](auto kern, int threads) {
    hipLaunchKernelGGL(kern, dim3(rows), dim3(threads), 0, s, x, x_stride, res, w, eps, q, scale, res_out, n);
  };
  if (n <= 256 * kRowChunks * 8) go(rows_q8_kernel<256, NORM>, 256);
  else go(rows_q8_kernel<1024, NORM>, 1024);
}

template <bool SILU>
void launch_product(const Product& p, hipStream_t s) {
  hipLaunchKernelGGL(product_kernel<SILU>, dim3((p.n + 63) / 64, (p.m + 15) / 16), dim3(256), 0, s, p);
}

template <bool NORM, bool SILU>
void launch_token(const Token& p, int m, hipStream_t s) {
  const int cus = device_cus();
  const int units = SILU ? p.n : (p.n + 1) / 2;
  auto go = [&](auto kern) {
    const int grid = std::min(4 * (cus > 0 ? cus : 256), (units + kTokenWaves - 1) / kTokenWaves);
    hipLaunchKernelGGL(kern, dim3(grid), dim3(kTokenThreads), m * p.k, s, p);
  };
  switch (m) {
    case 1: go(token_kernel<1, NORM, SILU>); break;
    case 2: go(token_kernel<2, NORM, SILU>); break;
    case 3: go(token_kernel<3, NORM, SILU>); break;
    default: go(token_kernel<4, NORM, SILU>); break;
  }
}

constexpr int kTokenCodes = 49152;   // m * k of a token launch: its rows' codes lie in LDS

int check_rows(const char* who, const void* x, const int8_t* q, const float* scale, int rows, int n) {
  NKV_CHECK_ARG(x != nullptr && q != nullptr && scale != nullptr, "%s: every pointer must be non-NULL", who);
  NKV_CHECK_ARG(rows >= 1 && n >= 16 && n % 16 == 0 && n <= kMaxRow,
                "%s: rows >= 1 and n a multiple of 16 in [16, %d] (got %d, %d)", who, kMaxRow, rows, n);
  NKV_CHECK_ARG(aligned16(x) && aligned16(q), "%s: rows must be 16-byte aligned", who);
  return NKV_OK;
}

int check_product(const char* who, const Product& p, int outputs_per_channel) {
  NKV_CHECK_ARG(p.w != nullptr && p.sw != nullptr && p.x != nullptr && p.sx != nullptr && p.y != nullptr,
                "%s: weight, w_scale, x, x_scale and y must be non-NULL", who);
  NKV_CHECK_ARG(p.m >= 1 && p.n >= 1 && p.k >= 16 && p.k % 16 == 0 && p.k <= kMaxDepth,
                "%s: m and n >= 1 and k a multiple of 16 in [16, %d] (got %d, %d, %d)", who, kMaxDepth, p.m, p.n, p.k);
  NKV_CHECK_ARG(p.n <= INT32_MAX / 2 - 512 && p.m <= INT32_MAX - 512, "%s: m or n too large (got %d, %d)", who, p.m, p.n);
  NKV_CHECK_ARG(aligned16(p.w) && aligned16(p.x), "%s: weight and x must be 16-byte aligned", who);
  const int64_t out = 2 * static_cast<int64_t>(p.m) * p.n, channels = static_cast<int64_t>(p.n) * outputs_per_channel;
  NKV_CHECK_ARG(apart(p.y, out, p.w, channels * p.k) && apart(p.y, out, p.sw, 4 * channels) &&
                    apart(p.y, out, p.x, static_cast<int64_t>(p.m) * p.k) && apart(p.y, out, p.sx, 4 * static_cast<int64_t>(p.m)) &&
                    apart(p.y, out, p.bias, 2 * channels),
                "%s: y must not overlap an input", who);
  return NKV_OK;
}

template <bool NORM, bool SILU>
int token(const char* who, const Token& p, int m, void* stream) {
  NKV_CHECK_ARG(p.w != nullptr && p.sw != nullptr && p.x != nullptr && p.y != nullptr && (!NORM || p.nw != nullptr),
                "%s: weight, w_scale, x%s and y must be non-NULL", who, NORM ? ", norm_weight" : "");
  NKV_CHECK_ARG(m >= 1 && m <= 4, "%s: m must be in [1, 4] (got %d)", who, m);
  NKV_CHECK_ARG(p.n >= 1 && p.n <= INT32_MAX / 2 - 512 && p.k >= 16 && p.k % 16 == 0 && p.k <= kMaxRow,
                "%s: n >= 1 and k a multiple of 16 in [16, %d] (got %d, %d)", who, kMaxRow, p.n, p.k);
  NKV_CHECK_ARG(m * p.k <= kTokenCodes, "%s: m * k must be at most %d (got %d * %d)", who, kTokenCodes, m, p.k);
  NKV_CHECK_ARG(aligned16(p.w) && aligned16(p.x) && (!p.res || aligned16(p.res)) && (!p.nw || aligned16(p.nw)) &&
                    (!p.res_out || aligned16(p.res_out)),
                "%s: weight, the rows, norm_weight and residual_out must be 16-byte aligned", who);
  // every workgroup reads the rows, norm_weight and its scales while others write y and one writes residual_out
  const int64_t row = 2 * static_cast<int64_t>(p.k), rows = m * row, out = 2 * static_cast<int64_t>(m) * p.n;
  const int64_t channels = static_cast<int64_t>(p.n) * (SILU ? 2 : 1);
  struct Out {
    const char* name;
    const void* at;
    int64_t bytes;
  };
  for (const Out& o : {Out{"y", p.y, out}, Out{"residual_out", p.res_out, rows}})
    NKV_CHECK_ARG(apart(o.at, o.bytes, p.x, rows) && apart(o.at, o.bytes, p.res, rows) && apart(o.at, o.bytes, p.nw, row) &&
                      apart(o.at, o.bytes, p.w, channels * p.k) && apart(o.at, o.bytes, p.sw, 4 * channels) &&
                      apart(o.at, o.bytes, p.bias, 2 * channels),
                  "%s: %s must not overlap an input", who, o.name);
  NKV_CHECK_ARG(apart(p.y, out, p.res_out, rows), "%s: y must not overlap residual_out", who);
  launch_token<NORM, SILU>(p, m, reinterpret_cast<hipStream_t>(stream));
  return launch_status(who);
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int nkv_quantize_q8(const uint16_t* x, int64_t x_stride, int8_t* q, float* scale, int rows, int n,
                               void* stream) {
  const int rc = check_rows("nkv_quantize_q8", x, q, scale, rows, n);
  if (rc != NKV_OK) return rc;
  NKV_CHECK_ARG(x_stride % 8 == 0 && (rows == 1 || x_stride >= n),
                "nkv_quantize_q8: x_stride must be a multiple of 8, at least n (got %lld)", static_cast<long long>(x_stride));
  const int64_t in = 2 * ((rows - 1) * x_stride + n), codes = static_cast<int64_t>(rows) * n, sc = 4 * static_cast<int64_t>(rows);
  NKV_CHECK_ARG(apart(q, codes, x, in) && apart(scale, sc, x, in) && apart(q, codes, scale, sc),
                "nkv_quantize_q8: the outputs must overlap neither x nor each other");
  launch_rows<false>(x, x_stride, nullptr, nullptr, 0.0f, q, scale, nullptr, rows, n, reinterpret_cast<hipStream_t>(stream));
  return launch_status("nkv_quantize_q8");
}

extern "C" int nkv_dequantize_q8(const int8_t* q, const float* scale, uint16_t* out, int rows, int n, void* stream) {
  NKV_CHECK_ARG(q != nullptr && scale != nullptr && out != nullptr, "nkv_dequantize_q8: every pointer must be non-NULL");
  NKV_CHECK_ARG(rows >= 1 && n >= 16 && n % 16 == 0, "nkv_dequantize_q8: rows >= 1 and n a positive multiple of 16 (got %d, %d)",
                rows, n);
  NKV_CHECK_ARG(aligned16(q) && aligned16(out), "nkv_dequantize_q8: q and out must be 16-byte aligned");
  const int64_t codes = static_cast<int64_t>(rows) * n, chunks = codes / 16;
  NKV_CHECK_ARG(chunks <= INT64_C(256) * INT32_MAX, "nkv_dequantize_q8: too many elements");
  NKV_CHECK_ARG(apart(out, 2 * codes, q, codes) && apart(out, 2 * codes, scale, 4 * static_cast<int64_t>(rows)),
                "nkv_dequantize_q8: out must not overlap an input");
  hipLaunchKernelGGL(dequantize_kernel, dim3(static_cast<unsigned>((chunks + 255) / 256)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), q, scale, out, chunks, n);
  return launch_status("nkv_dequantize_q8");
}

extern "C" int nkv_rmsnorm_q8(const uint16_t* x, const uint16_t* residual, const uint16_t* weight, float eps, int8_t* q,
                              float* scale, uint16_t* residual_out, int rows, int n, void* stream) {
  const int rc = check_rows("nkv_rmsnorm_q8", x, q, scale, rows, n);
  if (rc != NKV_OK) return rc;
  NKV_CHECK_ARG(weight != nullptr && aligned16(weight) && (!residual || aligned16(residual)) && (!residual_out || aligned16(residual_out)),
                "nkv_rmsnorm_q8: weight must be non-NULL, and every buffer 16-byte aligned");
  const int64_t codes = static_cast<int64_t>(rows) * n, sc = 4 * static_cast<int64_t>(rows);
  // (a row's residual_out may replace its own inputs: every element is read by the thread that writes it, before)
  for (const uint16_t* in : {x, residual})
    NKV_CHECK_ARG(apart(q, codes, in, 2 * codes) && apart(scale, sc, in, 2 * codes) &&
                      (residual_out == in || apart(residual_out, 2 * codes, in, 2 * codes)),
                  "nkv_rmsnorm_q8: an output overlaps an input (residual_out may be x or residual itself)");
  NKV_CHECK_ARG(apart(q, codes, weight, 2 * n) && apart(scale, sc, weight, 2 * n) && apart(residual_out, 2 * codes, weight, 2 * n) &&
                    apart(q, codes, scale, sc) && apart(residual_out, 2 * codes, q, codes) && apart(residual_out, 2 * codes, scale, sc),
                "nkv_rmsnorm_q8: the outputs must overlap neither weight nor each other");
  launch_rows<true>(x, n, residual, weight, eps, q, scale, residual_out, rows, n, reinterpret_cast<hipStream_t>(stream));
  return launch_status("nkv_rmsnorm_q8");
}

extern "C" int nkv_linear_q8(const int8_t* weight, const float* w_scale, const int8_t* x, const float* x_scale,
                             const uint16_t* bias, uint16_t* y, int m, int n, int k, void* stream) {
  const Product p{weight, w_scale, x, x_scale, bias, y, m, n, k};
  const int rc = check_product("nkv_linear_q8", p, 1);
  if (rc != NKV_OK) return rc;
  launch_product<false>(p, reinterpret_cast<hipStream_t>(stream));
  return launch_status("nkv_linear_q8");
}

extern "C" int nkv_linear_silu_mul_q8(const int8_t* gate_up_weight, const float* w_scale, const int8_t* x,
                                      const float* x_scale, uint16_t* y, int m, int intermediate, int k, void* stream) {
  const Product p{gate_up_weight, w_scale, x, x_scale, nullptr, y, m, intermediate, k};
  const int rc = check_product("nkv_linear_silu_mul_q8", p, 2);
  if (rc != NKV_OK) return rc;
  launch_product<true>(p, reinterpret_cast<hipStream_t>(stream));
  return launch_status("nkv_linear_silu_mul_q8");
}

extern "C" int nkv_gemv_q8(const int8_t* weight, const float* w_scale, const uint16_t* x, const uint16_t* bias, uint16_t* y,
                           int m, int n, int k, void* stream) {
  return token<false, false>("nkv_gemv_q8", Token{weight, w_scale, x, nullptr, nullptr, bias, y, nullptr, 0.0f, n, k}, m, stream);
}

extern "C" int nkv_gemv_silu_mul_q8(const int8_t* gate_up_weight, const float* w_scale, const uint16_t* x, uint16_t* y, int m,
                                    int intermediate, int k, void* stream) {
  return token<false, true>("nkv_gemv_silu_mul_q8",
                            Token{gate_up_weight, w_scale, x, nullptr, nullptr, nullptr, y, nullptr, 0.0f, intermediate, k}, m,
                            stream);
}

extern "C" int nkv_norm_gemv_q8(const int8_t* weight, const float* w_scale, const uint16_t* x, const uint16_t* residual,
                                const uint16_t* norm_weight, float eps, const uint16_t* bias, uint16_t* y,
                                uint16_t* residual_out, int m, int n, int k, void* stream) {
  return token<true, false>("nkv_norm_gemv_q8",
                            Token{weight, w_scale, x, residual, norm_weight, bias, y, residual_out, eps, n, k}, m, stream);
}

extern "C" int nkv_norm_gemv_silu_mul_q8(const int8_t* gate_up_weight, const float* w_scale, const uint16_t* x,
                                         const uint16_t* residual, const uint16_t* norm_weight, float eps, uint16_t* y,
                                         uint16_t* residual_out, int m, int intermediate, int k, void* stream) {
  return token<true, true>("nkv_norm_gemv_silu_mul_q8",
                           Token{gate_up_weight, w_scale, x, residual, norm_weight, nullptr, y, residual_out, eps, intermediate, k},
                           m, stream);
}
