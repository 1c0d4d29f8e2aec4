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

// 4 codes: v * inv rounded to whole numbers, to nearest even, in the low byte of its sum with
// 1.5 * 2^23; NaN gives 0.  v * inv is off by less than 127 * 2^-23 < 2^-16 (inv and the product
// are rounded once each, no fma).  bf16 v and peak put v * 127 / peak half way between two codes or
// more than 2^-16 off (all pairs of mantissas were tried), so with EXACT (rows that are bf16) the
// product is rounded to 2^-15 first -- the sum with 1.5 * 2^8, whose last bit that is -- which
// makes a half way one exact again: the codes are rne(v * 127 / peak) itself.  (Rounded at once,
// 14 of the 254 half way pairs of mantissas went to the other code.)  Behind a norm v is fp32,
// half way means nothing, and the step would only move small values (4096 x 2560: 140 codes
// off the nearest against 10).
template <bool EXACT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
#pragma clang fp contract(off)
  constexpr float kSnap = EXACT ? 384.0f : 0.0f, kMagic = 12582912.0f - kSnap;
  float p[4] = {a * inv, b * inv, c * inv, d * inv};
  if constexpr (EXACT) p[0] += kSnap, p[1] += kSnap, p[2] += kSnap, p[3] += kSnap;
  const uint32_t x = __float_as_uint(p[0] + kMagic), y = __float_as_uint(p[1] + kMagic);
  const uint32_t z = __float_as_uint(p[2] + kMagic), w = __float_as_uint(p[3] + kMagic);
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
// the codes do not depend on r.  NaN also where the squares or |t w| pass fp32's range.
__device__ __forceinline__ RowScale norm_row_scale(uint32_t top, float ss, int n, float eps) {
  RowScale rs = row_scale(top);
  const float r = rsqrtf(ss / static_cast<float>(n) + eps);
  const float a = __uint_as_float(top) * r;
  if (rs.scale == 0.0f || a < kTiny) rs = {0.0f, 0.0f};
  else rs.scale = a / 127.0f;
  if (mag(ss) >= 0x7f800000u || mag(a) >= 0x7f800000u) rs = {__uint_as_float(0x7fc00000u), 0.0f};
  return rs;
}

// WPR wavefronts a row, NCH 8-element chunks a lane, held in registers between the
// pass that finds the row's peak (and sum of squares) and the one that writes its
// codes: every byte is moved once.  Bound by HBM for many rows (quantise 4096 x
// 9728 22.1 us, 5.4 TB/s; norm with residual 50.9-56.9 us, 4.9-5.5 TB/s; a large copy runs at
// 5.1), by the launch for few (1 x 2560 2.5 and 3.2 us in a captured chain).  Rows
// of up to 512 take a wavefront each, no barrier (4096 x 512 5.0 -> 3.9 us, 16384
// x 128 12 -> 5.8); longer ones more, in the steps of launch_rows (a fixed four: 1 x
// 2560 3.0 us, 4096 x 9728 26.5; just above a step up to half of the lanes have no
// chunk).  (x, res and res_out may be one buffer.)
constexpr int row_threads(int wpr) { return kWave * (wpr == 1 ? 4 : wpr); }
template <int WPR, int NCH, bool NORM>
__global__ __launch_bounds__(row_threads(WPR)) void rows_q8_kernel(const uint16_t* x, int64_t x_stride,
                                                                   const uint16_t* res, const uint16_t* __restrict__ w,
                                                                   float eps, int8_t* __restrict__ q,
                                                                   float* __restrict__ scale, uint16_t* res_out,
                                                                   int rows, int n) {
  constexpr int kRows = row_threads(WPR) / (WPR * kWave), kLanes = WPR * kWave;
  __shared__ float s_sum[WPR];
  __shared__ uint32_t s_top[WPR];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / kLanes : 0);
  if (kRows > 1 && row >= rows) return;                // (no barrier follows)
  const int t = kRows > 1 ? threadIdx.x % kLanes : threadIdx.x;
  const int nc = n >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * x_stride);
  const uint4* rr = NORM && res ? reinterpret_cast<const uint4*>(res + row * n) : nullptr;
  uint4* ro = NORM && res_out ? reinterpret_cast<uint4*>(res_out + row * n) : nullptr;
  float v[NCH][8];
  float ss = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int c = t + j * kLanes;
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
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) s_sum[wave] = ss, s_top[wave] = top;
    __syncthreads();
    ss = 0.0f;
    top = 0;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += s_sum[i], top = max(top, s_top[i]);
  }
  const RowScale rs = NORM ? norm_row_scale(top, ss, n, eps) : row_scale(top);
  uint2* qr = reinterpret_cast<uint2*>(q + row * n);
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int c = t + j * kLanes;
    if (c < nc)
      qr[c] = make_uint2(codes4<!NORM>(v[j][0], v[j][1], v[j][2], v[j][3], rs.inv), codes4<!NORM>(v[j][4], v[j][5], v[j][6], v[j][7], rs.inv));
  }
  if (t == 0) scale[row] = rs.scale;
}

// One thread per 16 codes (4096 x 9728: 23.6 us, 5.1 TB/s).
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

// SiLU(g) * u in fp32.  The hardware's exp2 and reciprocal (1 ulp each; the argument's
// rounding makes it |g| 2^-24 relative, far below the output's 2^-8): with
// expf and a division the epilogue of a 256 x 256 tile cost a tenth of the product
// (gate|up of 4096 rows 236 -> 207 us).
__device__ __forceinline__ float silu_mul(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.442695041f)) * u;
}

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

// Products stage rows in pieces of 128 codes, one 128-byte LDS row each.
constexpr int kTileK = 128;
constexpr int kRsrcWord3 = 0x00020000;   // raw buffer, 32-bit data format
// LDS row r's 16-byte piece c lies at piece c ^ swizzle(r): the 16 lanes that
// are served together (of 16 rows, at c or, for lanes 16 on, at c ^ 1) hit
// the 16 pieces of 256 bytes.
__device__ __forceinline__ int swizzle(int r) { return (r >> 1) & 7; }

// Workgroup barrier behind this wavefront's LDS operations; its loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);                  // lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

// Few rows (16 NB a workgroup): the product is bound by reading the weight once.
// A workgroup owns 16 channels (SILU: and their up channels); its wavefronts
// take 128-code pieces of k in turn, each on its own: whole 128-byte lines into
// registers, kDeep pieces in flight, turned through the wavefront's own LDS rows
// into the matrix instruction's operands (no barrier), and the partial sums are
// joined through LDS at the end: exact, being integers.  In a captured chain over
// 512 MB of weights and more (us): 6 x 2560 -> 6144 8.8, 6 x 9728 -> 2560 11.1 (2.2 TB/s), gate|up of
// 6 rows 15.9 (3.1 TB/s), 37 x 9728 -> 2560 16.7, where reading the rows, once a
// workgroup, counts as much as the weight.  Over 380 to 600 MB, in part from the 256 MB cache, 6.1, 8.4,
// 12.9 and 13.3, and what was compared there: operands read straight from memory as
// the matrix instruction wants them (64 bytes of 16 rows a load) took 11.5, 16.8 and 20.9
// for the last three; refills under a branch made the compiler wait for every
// load (8.4 -> 15.1); 8 wavefronts a workgroup: gate|up 15.8.
//
// NCH > 0: up to 8 rows that are still bf16 (p.x and p.sx are not read), of up to
// 512 NCH elements: every workgroup normalises (NORM) and quantises them itself, a
// wavefront one or two rows, while its first weights are in flight, and keeps their codes
// in LDS, in pieces like the weight's.  Over cold weights (us, with the rows' own launch
// before the product / in one): 4 x 2560 -> 6144 with a norm 9.0 / 7.9, 4 x 4096 -> 2560 8.2 / 6.5,
// 4 x 1024 -> 1024 5.7 / 3.7, gate|up of 9728 for 6 rows 16.0 / 15.5, with a norm 16.4 / 17.4 (what every
// workgroup does again).  All first weights fetched before a norm spilled registers
// (gate|up for 4 rows 18.0 against 15.2).
constexpr int kFewWaves = 4;
constexpr int kDraftRows = 2 * kFewWaves;
constexpr int kDraftMaxK = 4096;
constexpr int few_bytes(int tiles) { return tiles * kFewWaves * 16 * kTileK; }
struct Rows {
  const uint16_t* x;      // [m][k] bf16
  const uint16_t* res;    // NORM: residual added first, or null
  const uint16_t* nw;     // NORM: norm weight
  uint16_t* res_out;      // NORM: bf16(x + res), or null
  float eps;
};
template <int NB, bool SILU, int NCH = 0, bool NORM = false>
__global__ __launch_bounds__(64 * kFewWaves, NCH == 0 ? 1 : NCH <= 5 ? 3 : 2) void few_kernel(const Product p, const Rows in) {
  static_assert(NCH == 0 || NB == 1, "");
  constexpr int kHalves = SILU ? 2 : 1, kTiles = kHalves + (NCH ? 0 : NB);   // 16-row tiles of a piece: channels, then rows
  constexpr int kDeep = kTiles <= 3 ? 5 : kTiles <= 5 ? 4 : 3;
  extern __shared__ __align__(128) char s_few[];       // [wave][kTiles][16 rows][128]; then the partial sums
  constexpr int waves = kFewWaves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1);
  const int r = lane & 15, g = lane >> 4;
  const int c0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * NB;
  // lane u fetches 16 bytes, piece u & 7 of row u >> 3, of each 8-row half of a tile; past a
  // matrix's or a row's end the loads give zeros
  const int sub = lane >> 3, kc = 16 * (lane & 7);
  const int voff = sub * p.k + kc;
  __amdgpu_buffer_rsrc_t rs[kHalves + 1];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
    rs[h] = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.w + (static_cast<int64_t>(h) * p.n + c0) * p.k), 0,
                                              min(p.n - c0, 16) * p.k, kRsrcWord3);
  if constexpr (NCH == 0)
    rs[kHalves] = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.x + static_cast<int64_t>(m0) * p.k), 0,
                                                    min(p.m - m0, 16 * NB) * p.k, kRsrcWord3);
  char* mine_lds = s_few + wave * kTiles * 16 * kTileK;
  const int put_at = sub * kTileK + 16 * ((lane & 7) ^ swizzle(sub));       // (row 8 + sub: 8 rows on, its swizzle ^ 4)
  const int get_at = r * kTileK + 16 * (g ^ swizzle(r));
  i32x4 acc[kHalves][NB];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[h][j] = i32x4{0, 0, 0, 0};
  i32x4 st[kDeep][kTiles][2];
  auto fetch = [&](int d, int q) {
    const bool in_row = kTileK * q + kc < p.k;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int off = voff + ((t < kHalves ? 0 : 16 * (t - kHalves)) + 8 * e) * p.k + kTileK * q;
        st[d][t][e] = __builtin_bit_cast(
            i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs[min(t, kHalves)], in_row ? off : 0x7fffffff, 0, 0));
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  // NCH: the rows' codes, [piece][8 rows][128] (columns 8 on of a product repeat the first 8 and are not used)
  __shared__ __align__(128) char s_rows[NCH ? 512 * NCH * kDraftRows : 16];
  __shared__ float s_row_scale[kDraftRows];
  const int row_at = (r & 7) * kTileK + 16 * (g ^ swizzle(r & 7));
  auto products = [&](int d, int q) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<i32x4*>(mine_lds + (16 * t + 8 * e) * kTileK + (put_at ^ (64 * e))) = st[d][t][e];
    wave_lds_sync();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      i32x4 f[kHalves + NB];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) f[t] = *reinterpret_cast<const i32x4*>(mine_lds + 16 * t * kTileK + (get_at ^ (64 * e)));
      if constexpr (NCH > 0) f[kHalves] = *reinterpret_cast<const i32x4*>(s_rows + q * kDraftRows * kTileK + (row_at ^ (64 * e)));
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[h][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[h], f[kHalves + j], acc[h][j], 0, 0, 0);
    }
    wave_lds_sync();
  };
  const int pieces = (p.k + kTileK - 1) / kTileK;
  const int mine = (pieces - wave + waves - 1) / waves;   // pieces wave, wave + waves, ...
  // (fetches past the last piece read no row; made without a branch, so that the waits stay exact)
  if constexpr (NCH == 0) {
#pragma unroll
    for (int d = 0; d < kDeep; ++d) fetch(d, wave + d * waves);
  } else {
    constexpr int kNorm = NORM ? NCH : 1;
    const int nc = p.k >> 3;
    constexpr int kShare = NORM ? (NCH + waves - 1) / waves : 1;
    static_assert(kShare <= 2, "");
    uint4 xv[2][NCH], rv[2][kNorm], nv0, nv1;
    __shared__ uint4 s_nw[NORM ? kWave * waves * kShare : 1];
    if constexpr (NORM) {                              // (past the row: its last, not used)
      nv0 = reinterpret_cast<const uint4*>(in.nw)[min(static_cast<int>(threadIdx.x), nc - 1)];
      if constexpr (kShare > 1) nv1 = reinterpret_cast<const uint4*>(in.nw)[min(static_cast<int>(threadIdx.x) + kWave * waves, nc - 1)];
    }
    // past the row, past the last row, and without a residual: zeros, and nothing is read
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(in.x), 0, 2 * p.m * p.k, kRsrcWord3);
    const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(NORM ? in.res : in.x), 0,
                                                                        NORM && in.res ? 2 * p.m * p.k : 0, kRsrcWord3);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = lane + kWave * j;
        const int off = c < nc ? 2 * (wave + waves * h) * p.k + 16 * c : 0x7fffffff;
        xv[h][j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 0, 0));
        if constexpr (NORM) rv[h][j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rr, off, 0, 0));
      }
    __builtin_amdgcn_sched_barrier(0);
    // (the rest behind the first row, whose registers they take)
    constexpr int kFirst = NORM ? (SILU ? 1 : 2) : kDeep;
#pragma unroll
    for (int d = 0; d < kFirst; ++d) fetch(d, wave + d * waves);
    if constexpr (NORM) {
      s_nw[threadIdx.x] = nv0;
      if constexpr (kShare > 1) s_nw[threadIdx.x + kWave * waves] = nv1;
      lds_barrier();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = wave + waves * h;
      if (h == 1) {
#pragma unroll
        for (int d = kFirst; d < kDeep; ++d) fetch(d, wave + d * waves);
      }
      if (row >= p.m) continue;
      float v[NCH][8], ss = 0.0f;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = lane + kWave * j;
        unpack8(xv[h][j], v[j]);
        if constexpr (NORM) {
          if (in.res) {
            float t[8];
            unpack8(rv[h][j], t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] += t[e];
          }
          if (in.res_out && blockIdx.x == 0 && c < nc)
            reinterpret_cast<uint4*>(in.res_out)[static_cast<int64_t>(row) * nc + c] = pack8(v[j]);
          float wf[8];
          unpack8(s_nw[c], wf);                        // (past the row: its last)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (c < nc) ss += v[j][e] * v[j][e];
            v[j][e] *= wf[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, mag(v[j][e]));
      }
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) {
        if constexpr (NORM) ss += __shfl_xor(ss, o);
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
      }
      const RowScale sc = NORM ? norm_row_scale(top, ss, p.k, in.eps) : row_scale(top);
      if (lane == 0) s_row_scale[row] = sc.scale;
#pragma unroll
      for (int j = 0; j < NCH; ++j) {
        const int c = lane + kWave * j;                // 8 codes: half of 16-byte unit (c / 2) % 8 of piece c / 16
        if (c < nc)
          *reinterpret_cast<uint2*>(s_rows + (c >> 4) * kDraftRows * kTileK + row * kTileK + 16 * (((c >> 1) & 7) ^ swizzle(row)) + 8 * (c & 1)) =
              make_uint2(codes4<!NORM>(v[j][0], v[j][1], v[j][2], v[j][3], sc.inv), codes4<!NORM>(v[j][4], v[j][5], v[j][6], v[j][7], sc.inv));
      }
    }
    lds_barrier();
  }
  int i = 0;
  for (; i + kDeep < mine; i += kDeep)
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      products(d, wave + (i + d) * waves);
      fetch(d, wave + (i + d + kDeep) * waves);
    }
#pragma unroll
  for (int d = 0; d < kDeep; ++d)
    if (i + d < mine) products(d, wave + (i + d) * waves);
  // the joined sums: [wave][kHalves NB][lane]
  i32x4* s_part = reinterpret_cast<i32x4*>(s_few);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int j = 0; j < NB; ++j) s_part[((wave * kHalves + h) * NB + j) * kWave + lane] = acc[h][j];
  __syncthreads();
  for (int j = wave; j < NB; j += waves) {
    i32x4 sum[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      sum[h] = s_part[(h * NB + j) * kWave + lane];
      for (int v = 1; v < waves; ++v) sum[h] += s_part[((v * kHalves + h) * NB + j) * kWave + lane];
    }
    const int m = m0 + 16 * j + r;
    if (m >= p.m) continue;
    const float sx = NCH ? s_row_scale[m & (kDraftRows - 1)] : p.sx[m];
    uint16_t* y = p.y + static_cast<int64_t>(m) * p.n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = c0 + 4 * g + e;
      if (c >= p.n) break;
      float v = scaled(sum[0][e], sx, p.sw[c], p.bias ? bf16_to_f32(p.bias[c]) : 0.0f);
      if constexpr (SILU) v = silu_mul(v, scaled(sum[kHalves - 1][e], sx, p.sw[p.n + c], 0.0f));
      y[c] = f32_to_bf16(v);
    }
  }
}

// Tiles of 32 NA channels (SILU: 16 NA gate channels and their up channels) x
// 16 NB WM rows, one a workgroup of 2 x WM wavefronts (channels x rows); a
// wavefront owns NA x NB products of 16 x 16.
//
// 8192^3: 447 us, 2.46 PFLOP/s (a library's int8 product 2.09); a 4096-token chunk:
// 4096 -> 2560 46 us (1.87), 9728 -> 2560 96 (2.13), gate|up with SiLU 192 (2.12).
// The large ones are bound by the chip's power: the clock falls to 1.9-2.06 GHz, and
// matrix instructions on registers alone reach 3.2-3.5 PFLOP/s there.  8192^3 with
// parts taken out (us, timing copies): no loads 364, no LDS writes 396, no LDS reads 347,
// neither loads nor writes 337, against 420-447.  Measured on the way (8192^3): LDS
// rows that conflict two ways and direct copies into LDS 516; fragments read ahead
// 485; copies through registers 480; scales from LDS in the epilogue 447.  No gain:
// 128 x 128 a wavefront with one a SIMD (686), fragments read further ahead, two
// stages in registers, one workgroup a CU taking tile after tile with the next
// one's loads under the epilogue (480), wave priorities.
//
// LDS rows of a stage (weight rows, then x rows), rounded up to whole rounds of copies
constexpr int tile_rows(int na, int nb, int wm) { return (32 * na + 16 * nb * wm + 16 * wm - 1) / (16 * wm) * (16 * wm); }

// With PART, gridDim.y workgroups share a tile, each a run of its stages, and the
// sums go to part[blockIdx.y][m][n] for join_kernel.
// With KS = 2 a workgroup has two groups of wavefronts, which take the stages in turn,
// each in buffers of its own, and add their sums through LDS at the end: for the
// small tiles, whose one wavefront a SIMD waits for LDS between products (us, KS = 1 / 2:
// 200 x 2560 -> 6144 14.8 / 13.3, 200 x 4096 -> 2560 11.8 / 10.1, 65 x 4096 -> 2560 11.1 / 9.2;
// fragments read a whole stage ahead instead: no gain.  128 x 128 18.2 / 17.5).
template <int NA, int NB, int WM, int DEPTH, bool SILU, bool PART = false, int KS = 1>
__global__ __launch_bounds__(128 * WM * KS) void tile_kernel(const Product p, int mt, int nt, bool wide, int* part) {
  static_assert(!(SILU && PART) && (KS == 1 || (KS == 2 && NB % 2 == 0)), "");
  extern __shared__ __align__(128) char s_lds[];
  constexpr int kTileM = 16 * NB * WM, kWaves = 2 * WM;
  __shared__ __align__(16) float s_scale[32 * NA], s_bias[SILU ? 4 : 32 * NA], s_x[kTileM];
  constexpr int kStage = tile_rows(NA, NB, WM) * kTileK;
  constexpr int kCopies = tile_rows(NA, NB, WM) / (8 * kWaves);   // 8-row pieces a wavefront copies
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) % kWaves;
  const int group = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) / kWaves : 0;
  char* s_tile = s_lds + group * 2 * kStage;
  const int lane = threadIdx.x & (kWave - 1);
  // tiles: a run of them per XCD, 8 row tiles by all channel tiles at a time
  int t;
  {
    const int total = mt * nt, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    const int per = total >> 3, more = total & 7;
    t = xcd * per + min(xcd, more) + at;
  }
  const int band = t / (8 * nt), in = t - band * 8 * nt;
  const int rows_of_band = min(8, mt - band * 8);
  const int m0 = (band * 8 + in % rows_of_band) * kTileM;
  const int c0 = (in / rows_of_band) * (SILU ? 16 : 32) * NA;

  const int cn = min(p.n - c0, (SILU ? 16 : 32) * NA), mn = min(p.m - m0, kTileM);

  const int all = (p.k + kTileK - 1) / kTileK;
  const int first = PART ? static_cast<int>(static_cast<int64_t>(all) * blockIdx.y / gridDim.y) : 0;
  const int end = PART ? static_cast<int>(static_cast<int64_t>(all) * (blockIdx.y + 1) / gridDim.y) : all;
  const int stages = (end - first + KS - 1) / KS;      // of a group (KS = 2: the other's last one may be empty)

  // A wavefront's share of a stage: 8-row pieces wave, wave + kWaves, ..., lane u with
  // 16 bytes of row u >> 3.  They go through registers: loaded a stage ahead of
  // the step that puts them into LDS.  (Copies straight into LDS reach 61 B/ns
  // a CU, loads into registers 89: two 256-row tiles a stage want 64.)
  const int sub = lane >> 3;
  const int kc = 16 * (lane & 7);
  const int voff = sub * p.k + kc;
  const int lds_at = sub * kTileK + 16 * ((lane & 7) ^ swizzle(8 * wave + sub));   // (kWaves groups on: the same swizzle)
  i32x4 st[DEPTH][kCopies];
  auto fetch = [&](int set, int s, int i) {
    int row = 8 * (wave + kWaves * i);                 // of the stage (rows past its last: zeros)
    const int8_t* base = p.w + static_cast<int64_t>(c0) * p.k;
    int rows = cn;
    if (row >= 32 * NA) {
      row -= 32 * NA;
      base = p.x + static_cast<int64_t>(m0) * p.k;
      rows = mn;
    } else if constexpr (SILU) {                       // of a wavefront's 16 NA rows half are gate rows, half up rows
      constexpr int half = 8 * NA;
      if ((row / half) & 1) base += static_cast<int64_t>(p.n) * p.k;
      row = (row / (2 * half)) * half + row % half;
    }
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, rows * p.k, kRsrcWord3);
    const int kb = (first + s * KS + group) * kTileK;
    const int past = PART && KS > 1 ? min(p.k, end * kTileK) : p.k;       // past the row's (or run's) end: zeros
    const int off = kc < past - kb ? voff + row * p.k + kb : 0x7fffffff;
    st[set][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
  };
  auto put = [&](int set, int buf, int i) {
    const int row = 8 * (wave + kWaves * i);
    *reinterpret_cast<i32x4*>(s_tile + buf + row * kTileK + lds_at) = st[set][i];
  };

  // the scales of the tile's weight rows and x rows, and its bias
  for (int row = threadIdx.x; !PART && row < 32 * NA; row += 64 * kWaves * KS) {
    const int64_t up = SILU && (row / (8 * NA)) & 1 ? p.n : 0;
    const int c = c0 + min(SILU ? (row / (16 * NA)) * 8 * NA + row % (8 * NA) : row, cn - 1);
    s_scale[row] = p.sw[up + c];
    if constexpr (!SILU) s_bias[row] = p.bias ? bf16_to_f32(p.bias[c]) : 0.0f;
  }
  for (int row = threadIdx.x; !PART && row < kTileM; row += 64 * kWaves * KS) s_x[row] = p.sx[m0 + min(row, mn - 1)];

  const int wc = wave & 1, wm = wave >> 1;
  const int r = lane & 15, g = lane >> 4;
  const int at = r * kTileK + 16 * (g ^ swizzle(r));
  i32x4 acc[NA][NB];
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

  // A stage is 2 NA steps of NB products, step i with weight fragment i % NA of
  // the k half i / NA.  Fragments are read kAhead steps ahead (a ring of
  // registers).  Meanwhile the next stage goes into the other buffer, and the
  // one after it into the registers.  Before the last kAhead steps a wavefront has
  // read all of its stage and written its share of the next: behind the one
  // barrier there the next stage's first fragments are read under these steps.
  constexpr int kSteps = 2 * NA, kRing = NA % 2 == 0 ? 4 : 5, kAhead = NA > 2 ? kRing - 1 : 2;
  static_assert(kSteps % kRing == 0 && NB <= NA && NB + kAhead <= kSteps, "");
  i32x4 a[kRing], b[2][NB];
  const char* base_a = s_tile + wc * 16 * NA * kTileK;
  const char* base_b = s_tile + (32 * NA + wm * 16 * NB) * kTileK;
  auto read_a = [&](int buf, int i) {
    a[i % kRing] = *reinterpret_cast<const i32x4*>(base_a + buf + (i % NA) * 16 * kTileK + (at ^ (64 * (i / NA))));
  };
  auto read_b = [&](int buf, int ks, int j) {
    b[ks][j] = *reinterpret_cast<const i32x4*>(base_b + buf + j * 16 * kTileK + (at ^ (64 * ks)));
  };
  auto products = [&](int i) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
      acc[i % NA][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i % kRing], b[i / NA][j], acc[i % NA][j], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll
  for (int i = 0; i < kCopies; ++i) fetch(0, 0, i);
#pragma unroll
  for (int d = 1; d < DEPTH; ++d)
#pragma unroll
    for (int i = 0; i < kCopies; ++i) fetch(d, d, i);
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    put(0, 0, i);
    fetch(0, DEPTH, i);
  }
  lds_barrier();
#pragma unroll
  for (int j = 0; j < NB; ++j) read_b(0, 0, j);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) read_a(0, i);
  auto stage = [&](int s, int set) {                   // set: registers that hold stage s + 1
    const int buf = (s & 1) * kStage, next = kStage - buf;
#pragma unroll
    for (int i = 0; i < kSteps - kAhead; ++i) {
      read_a(buf, i + kAhead);
      if (i < NB) read_b(buf, 1, i);
#pragma unroll
      for (int c = 0; c < kCopies; ++c)
        if (c * (kSteps - kAhead) / kCopies == i) {
          put(set, next, c);
          fetch(set, s + 1 + DEPTH, c);
        }
      products(i);
    }
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // (past the last stage these read what lies in the other buffer, and nothing uses it)
#pragma unroll
    for (int j = 0; j < NB; ++j) read_b(next, 0, j);
#pragma unroll
    for (int i = kSteps - kAhead; i < kSteps; ++i) {
      read_a(next, i + kAhead - kSteps);
      products(i);
    }
  };
  for (int s = 0; s < stages; s += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (d > 0 && s + d >= stages) break;
      stage(s + d, (d + 1) % DEPTH);
    }
  }

  // the groups' sums: each finishes half of the row tiles
  auto mine = [&](int j) { return KS == 1 || j / (NB / KS) == group; };
  if constexpr (KS > 1) {
    static_assert(2 * kWaves * NA * NB * kWave * 16 / KS <= 2 * KS * kStage, "");
    i32x4* s_join = reinterpret_cast<i32x4*>(s_lds) + wave * NA * (NB / KS) * kWave + lane;
    constexpr int kGroup = kWaves * NA * (NB / KS) * kWave;
    lds_barrier();
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (!mine(j))
#pragma unroll
        for (int i = 0; i < NA; ++i) s_join[(1 - group) * kGroup + (i * (NB / KS) + j % (NB / KS)) * kWave] = acc[i][j];
    lds_barrier();
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (mine(j))
#pragma unroll
        for (int i = 0; i < NA; ++i) acc[i][j] += s_join[group * kGroup + (i * (NB / KS) + j % (NB / KS)) * kWave];
  }

  if constexpr (PART) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int mj = (wm * NB + j) * 16 + r;
      if (!mine(j) || mj >= mn) continue;
      int* o = part + (static_cast<int64_t>(blockIdx.y) * p.m + m0 + mj) * p.n;
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int c = c0 + (wc * NA + i) * 16 + 4 * g;
        if (wide) {
          if (c < p.n) *reinterpret_cast<i32x4*>(o + c) = acc[i][j];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < p.n) o[c + e] = acc[i][j][e];
        }
      }
    }
    return;
  }

  constexpr int kOut = SILU ? NA / 2 : NA;             // channel groups of 16 that are written
  const float4* my_scale = reinterpret_cast<const float4*>(s_scale + wc * 16 * NA + 4 * g);
  const float4* my_bias = reinterpret_cast<const float4*>(s_bias + wc * 16 * NA + 4 * g);
  float4 sw[NA], sb[SILU ? 1 : NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    sw[i] = my_scale[4 * i];
    if constexpr (!SILU) sb[i] = my_bias[4 * i];
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int mj = (wm * NB + j) * 16 + r;
    if (!mine(j) || mj >= mn) continue;
    const float sx = s_x[mj];
    uint16_t* y = p.y + static_cast<int64_t>(m0 + mj) * p.n;
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      const int c = c0 + (wc * kOut + i) * 16 + 4 * g;
      const float ws[4] = {sw[i].x, sw[i].y, sw[i].z, sw[i].w};
      float v[4];
      if constexpr (SILU) {
        const float4 u4 = sw[NA / 2 + i];
        const float us[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = silu_mul(scaled(acc[i][j][e], sx, ws[e], 0.0f), scaled(acc[NA / 2 + i][j][e], sx, us[e], 0.0f));
      } else {
        const float bs[4] = {sb[i].x, sb[i].y, sb[i].z, sb[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled(acc[i][j][e], sx, ws[e], bs[e]);
      }
      const uint2 o = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
      if (wide) {                                      // (rows of y are 8-byte aligned, and c + 4 <= n or c >= n)
        if (c < p.n) *reinterpret_cast<uint2*>(y + c) = o;
      } else {
        if (c < p.n) y[c] = static_cast<uint16_t>(o.x);
        if (c + 1 < p.n) y[c + 1] = static_cast<uint16_t>(o.x >> 16);
        if (c + 2 < p.n) y[c + 2] = static_cast<uint16_t>(o.y);
        if (c + 3 < p.n) y[c + 3] = static_cast<uint16_t>(o.y >> 16);
      }
    }
  }
}

// The sums of a product whose k was cut over `parts` workgroups, joined: y of
// channels c .. c + V - 1 of a row a thread.  part: [parts][m][n], with SILU [parts]
// [m][2 n] (gate, then up).
template <int V, bool SILU>
__global__ __launch_bounds__(256) void join_kernel(const Product p, const int* __restrict__ part, int parts) {
  const int width = SILU ? 2 * p.n : p.n;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int per = (p.n + V - 1) / V;
  const int64_t m = i / per;
  if (m >= p.m) return;
  const int c = static_cast<int>(i - m * per) * V;
  const int* at = part + m * width + c;
  const int64_t stride = static_cast<int64_t>(p.m) * width;
  int sum[SILU ? 2 : 1][V] = {};
  for (int s = 0; s < parts; ++s, at += stride)
#pragma unroll
    for (int h = 0; h < (SILU ? 2 : 1); ++h) {
      if constexpr (V == 4) {
        const i32x4 v = *reinterpret_cast<const i32x4*>(at + h * p.n);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[h][e] += v[e];
      } else {
        sum[h][0] += at[h * p.n];
      }
    }
  const float sx = p.sx[m];
  uint16_t* y = p.y + m * p.n + c;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float v = scaled(sum[0][e], sx, p.sw[c + e], p.bias ? bf16_to_f32(p.bias[c + e]) : 0.0f);
    if constexpr (SILU) v = silu_mul(v, scaled(sum[SILU ? 1 : 0][e], sx, p.sw[p.n + c + e], 0.0f));
    y[e] = f32_to_bf16(v);
  }
}

// Sum of the products of 16 codes, added to acc.
__device__ __forceinline__ int dot16(const i32x4& a, const i32x4& b, int acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_sdot4(a[e], b[e], acc, false);
  return acc;
}

// Sum of x over the wavefront, in every lane, without the LDS pipeline.
__device__ __forceinline__ int wave_sum(int x) {
#define NKV_ROR_ADD(n) x += __builtin_amdgcn_update_dpp(0, x, 0x120 + n, 0xf, 0xf, true)
  NKV_ROR_ADD(8);
  NKV_ROR_ADD(4);
  NKV_ROR_ADD(2);
  NKV_ROR_ADD(1);
#undef NKV_ROR_ADD
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = static_cast<int>(a[0]) + static_cast<int>(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return static_cast<int>(b[0]) + static_cast<int>(b[1]);
}

// The same product for one row that is still bf16 (a decode token), with its norm
// (NORM) and quantisation in the same launch.  Resident workgroups (one round)
// take two channels a wavefront at a time -- consecutive ones (long rows: one), or
// with SILU a gate channel and its up channel -- lanes along k, the weight rows'
// NCH = ceil(k / 1024) 16-byte chunks a lane in flight at once.  Each workgroup quantises the row
// for itself while its first weights are in flight.
struct Token {
  const int8_t* w;
  const float* sw;
  const uint16_t* x;      // [k] bf16
  const uint16_t* res;    // NORM: residual added first, or null
  const uint16_t* nw;     // NORM: norm weight
  const uint16_t* bias;
  uint16_t* y;
  uint16_t* res_out;      // NORM: bf16(x + res), or null
  float eps;
  int n, k;
};
constexpr int kTokenWaves = 4;
constexpr int kTokenThreads = kTokenWaves * kWave;
constexpr int kTokenMaxK = 12288;
constexpr int token_rows(int nch, bool silu) { return silu || nch <= 4 ? 2 : 1; }
// resident wavefronts per SIMD the kernel is built for and launched with
constexpr int token_waves(int nch, bool silu) { return nch <= 6 ? 4 : silu ? (nch <= 8 ? 3 : 2) : nch <= 8 ? 4 : 3; }

template <int NCH, bool NORM, bool SILU>
__global__ __launch_bounds__(kTokenThreads, token_waves(NCH, SILU)) void token_kernel(const Token p) {
  constexpr int R = token_rows(NCH, SILU);
  constexpr int XC = (NCH * 1024 + 8 * kTokenThreads - 1) / (8 * kTokenThreads);   // 8-element chunks of x a thread
  __shared__ i32x4 s_codes[NCH * kWave];
  __shared__ float s_sum[kTokenWaves];
  __shared__ uint32_t s_top[kTokenWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1);
  const int nc = p.k >> 3, nq = p.k >> 4;

  uint4 xv[XC], rv[XC], nv[XC];
#pragma unroll
  for (int j = 0; j < XC; ++j) {
    const int c = min(static_cast<int>(threadIdx.x) + j * kTokenThreads, nc - 1);   // past the row: its last, not used
    xv[j] = reinterpret_cast<const uint4*>(p.x)[c];
    if constexpr (NORM) {
      if (p.res) rv[j] = reinterpret_cast<const uint4*>(p.res)[c];
      nv[j] = reinterpret_cast<const uint4*>(p.nw)[c];
    }
  }
  const int units = SILU ? p.n : (p.n + R - 1) / R;
  const int stride = gridDim.x * kTokenWaves;
  int u = static_cast<int>(blockIdx.x) * kTokenWaves + wave;
  i32x4 b[R][NCH];
  auto load = [&](int unit) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int row = SILU ? unit + j * p.n : min(R * unit + j, p.n - 1);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<int8_t*>(p.w + static_cast<int64_t>(row) * p.k), 0, p.k, kRsrcWord3);
#pragma unroll
      for (int i = 0; i < NCH; ++i)                    // past the row: zeros
        b[j][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * lane + 1024 * i, 0, 0));
    }
  };
  load(min(u, units - 1));

  // the row: its scale, and its codes into LDS, with zeros behind them
  float v[XC][8];
  float ss = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < XC; ++j) {
    const int c = threadIdx.x + j * kTokenThreads;
    unpack8(xv[j], v[j]);
    if constexpr (NORM) {
      float wf[8];
      unpack8(nv[j], wf);
      if (p.res) {
        float t[8];
        unpack8(rv[j], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += t[e];
      }
      if (p.res_out && blockIdx.x == 0 && c < nc) reinterpret_cast<uint4*>(p.res_out)[c] = pack8(v[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (c < nc) ss += v[j][e] * v[j][e];
        v[j][e] *= wf[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, mag(v[j][e]));
  }
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    ss += __shfl_xor(ss, o);
    top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
  }
  if (lane == 0) s_sum[wave] = ss, s_top[wave] = top;
  lds_barrier();
  ss = 0.0f;
  top = 0;
#pragma unroll
  for (int i = 0; i < kTokenWaves; ++i) ss += s_sum[i], top = max(top, s_top[i]);
  const RowScale rs = NORM ? norm_row_scale(top, ss, p.k, p.eps) : row_scale(top);
#pragma unroll
  for (int j = 0; j < XC; ++j) {
    const int c = threadIdx.x + j * kTokenThreads;
    if (XC * kTokenThreads == NCH * kWave * 2 || c < NCH * kWave * 2)
      reinterpret_cast<uint2*>(s_codes)[c] =
          c < nc ? make_uint2(codes4<!NORM>(v[j][0], v[j][1], v[j][2], v[j][3], rs.inv), codes4<!NORM>(v[j][4], v[j][5], v[j][6], v[j][7], rs.inv))
                 : make_uint2(0u, 0u);
  }
  lds_barrier();
  while (u < units) {
    int acc[R] = {};
    if constexpr (NCH > 4) asm volatile("" ::: "memory");   // (a long row's codes are read again, not held in registers)
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const i32x4 x = s_codes[i * kWave + lane];
#pragma unroll
      for (int j = 0; j < R; ++j) acc[j] = dot16(b[j][i], x, acc[j]);
    }
    const int now = u;
    u += stride;
    if (u < units) load(u);
#pragma unroll
    for (int j = 0; j < R; ++j) acc[j] = wave_sum(acc[j]);
    if (lane != 0) continue;
    if constexpr (SILU) {
      p.y[now] = f32_to_bf16(silu_mul(scaled(acc[0], rs.scale, p.sw[now], 0.0f), scaled(acc[R - 1], rs.scale, p.sw[p.n + now], 0.0f)));
    } else {
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int c = R * now + j;
        if (c < p.n) p.y[c] = f32_to_bf16(scaled(acc[j], rs.scale, p.sw[c], p.bias ? bf16_to_f32(p.bias[c]) : 0.0f));
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
  // (a launch holds less than 2^32 threads: 2^21 rows of at most 1024)
  auto go = [&](auto kern, int wpr) {
    const int per = wpr == 1 ? 4 : 1;
    for (int64_t at = 0; at < rows; at += 1 << 21) {
      const int some = static_cast<int>(std::min<int64_t>(rows - at, 1 << 21));
      hipLaunchKernelGGL(kern, dim3((some + per - 1) / per), dim3(row_threads(wpr)), 0, s, x + at * x_stride, x_stride,
                         res ? res + at * n : nullptr, w, eps, q + at * n, scale + at, res_out ? res_out + at * n : nullptr, some, n);
    }
  };
  // many rows: half the wavefronts a row, two chunks in flight a lane (us, 4096 rows of 2560: 16.4
  // against 17.2 with a norm, 8.7 / 9.6 without; of 4096: 22.6 / 24.0, 11.6 / 12.6); few: one chunk
  // a lane (1 x 2560: 3.2 against 3.5 and 2.5 / 3.0).  The steps of n: powers of two, and the widths
  // that were measured (2560, 9728)
  const bool many = rows >= 1024;
  if (n <= 512) go(rows_q8_kernel<1, 1, NORM>, 1);
  else if (n <= 1024) many ? go(rows_q8_kernel<1, 2, NORM>, 1) : go(rows_q8_kernel<2, 1, NORM>, 2);
  else if (n <= 2048) many ? go(rows_q8_kernel<2, 2, NORM>, 2) : go(rows_q8_kernel<4, 1, NORM>, 4);
  else if (n <= 2560) many ? go(rows_q8_kernel<3, 2, NORM>, 3) : go(rows_q8_kernel<5, 1, NORM>, 5);
  else if (n <= 4096) many ? go(rows_q8_kernel<4, 2, NORM>, 4) : go(rows_q8_kernel<8, 1, NORM>, 8);
  else if (n <= 8192) go(rows_q8_kernel<8, 2, NORM>, 8);
  else if (n <= 12288) go(rows_q8_kernel<8, 3, NORM>, 8);
  else if (n <= 16384) go(rows_q8_kernel<8, 4, NORM>, 8);
  else go(rows_q8_kernel<16, 4, NORM>, 16);
}

template <int NB, bool SILU>
int launch_few(const Product& p, hipStream_t s) {
  const int mt = (p.m + 16 * NB - 1) / (16 * NB);
  hipLaunchKernelGGL((few_kernel<NB, SILU>), dim3((p.n + 15) / 16, mt), dim3(64 * kFewWaves), few_bytes(NB + (SILU ? 2 : 1)),
                     s, p, Rows{});
  return NKV_OK;
}

template <int NCH, bool NORM, bool SILU>
void launch_draft(const Product& p, const Rows& in, hipStream_t s) {
  hipLaunchKernelGGL((few_kernel<1, SILU, NCH, NORM>), dim3((p.n + 15) / 16), dim3(64 * kFewWaves), few_bytes(SILU ? 2 : 1), s, p, in);
}

template <int NA, int NB, int WM, int DEPTH, bool SILU, bool PART = false, int KS = 1>
int launch_tile(const Product& p, hipStream_t s, int parts = 1, int* part = nullptr) {
  constexpr int kLds = 2 * KS * tile_rows(NA, NB, WM) * kTileK;
  const auto kern = tile_kernel<NA, NB, WM, DEPTH, SILU, PART, KS>;
  if (kLds > 65536) {   // beyond the default limit of a launch (per device, so asked each time: it is a table lookup)
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      set_error("nkv_linear_q8: %d bytes of LDS refused: %s", kLds, hipGetErrorString(e));
      return NKV_ERR_HIP;
    }
  }
  constexpr int kM = 16 * NB * WM, kN = (SILU ? 16 : 32) * NA;
  const int mt = (p.m + kM - 1) / kM, nt = (p.n + kN - 1) / kN;
  const bool wide = p.n % 4 == 0 && (PART || reinterpret_cast<uintptr_t>(p.y) % 8 == 0);
  hipLaunchKernelGGL(kern, dim3(mt * nt, parts), dim3(128 * WM * KS), kLds, s, p, mt, nt, wide, part);
  return NKV_OK;
}

// How a product runs.  Few rows, few enough 16-channel groups for one round of
// workgroups and a k that is not too long for one, or at most 32 rows (us, few-row
// kernel / tiles: 48 x 4096 -> 4096 9.1 / 11.1, 33 x 2560 -> 6144 9.7 / 8.7, 37 x 9728 ->
// 2560 13.4 / 13.7, 64 16.8 / 14.8): the kernel that cuts k over wavefronts.  Otherwise the tile whose busiest CU is done first: ceil(tiles /
// CUs) tiles of the shape's time for a stage of 128 codes (us, plus what one
// tile alone waits), as measured at 20-76 stages and 65-4096 rows.  Larger
// tiles do more products a byte (2.5 PFLOP/s at 256 x 256, 1.9 at 128 x 128 on
// 8192^3), smaller ones leave fewer CUs idle.  A long k of few tiles is cut over
// workgroups where that gains more than joining the sums costs.
struct Shape {
  int channels, rows;   // (SILU: half as many channels of y)
  float us, wait_us;
  int threads;          // a workgroup
};
constexpr Shape kShapes[] = {{256, 256, 1.35f, 0.0f, 512}, {192, 256, 1.20f, 0.0f, 512}, {160, 256, 1.00f, 0.0f, 512},
                             {128, 256, 0.88f, 0.0f, 512}, {128, 128, 0.58f, 0.0f, 512}, {128, 64, 0.40f, 0.0f, 512},
                             {64, 64, 0.19f, 0.04f, 512},  {64, 32, 0.13f, 0.06f, 256}};
constexpr int kParted[] = {4, 6};     // the shapes of products whose k is cut
constexpr int kMaxParts = 8;
struct Plan {
  int few;      // 16-row tiles of the few-row kernel, or 0
  int shape;    // kShapes
  int parts;    // workgroups a tile
};
Plan plan_product(int m, int n, int k, bool silu) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int stages = (k + kTileK - 1) / kTileK;
  if (m <= 32 || (m <= 64 && (n + 15) / 16 <= cus && m * stages <= 4000)) return {std::min(4, (m + 15) / 16), 0, 1};
  auto tiles = [&](const Shape& sh, int channels) {
    return static_cast<int64_t>((channels + sh.channels - 1) / sh.channels) * ((m + sh.rows - 1) / sh.rows);
  };
  const int64_t channels = silu ? 2 * static_cast<int64_t>(n) : n;
  int best = 0;
  float least = 0.0f;
  for (int i = 0; i < static_cast<int>(sizeof(kShapes) / sizeof(kShapes[0])); ++i) {
    const Shape& sh = kShapes[i];
    if (silu && sh.channels == 160) continue;          // (an odd number of 16-channel groups a wavefront)
    const float us = static_cast<float>(stages) * (static_cast<float>((tiles(sh, channels) + cus - 1) / cus) * sh.us + sh.wait_us);
    if (i == 0 || us < least) best = i, least = us;
  }
  Plan plan{0, best, 1};
  for (const int i : kParted)
    for (int parts = 2; parts <= kMaxParts && stages >= 8 * parts; ++parts) {
      const Shape& sh = kShapes[i];
      // the join: a launch behind the tiles' last stores, and every sum written and read once at 6 TB/s
      // (us, cut / whole: 65 x 9728 -> 2560 14.9 / 19.4, 128 17.0 / 21.0, 512 28.8 / 35.2; 200 x 4096 -> 2560
      // 14.2 / 9.8.  128 x 128 tiles alone: 65 rows 17.1, 128 19.5)
      const float join = 3.0f + static_cast<float>(parts) * static_cast<float>(m) * static_cast<float>(channels) * 8.0f / 6.0e6f;
      const float us = static_cast<float>((stages + parts - 1) / parts) *
                           (static_cast<float>((tiles(sh, channels) * parts + cus - 1) / cus) * sh.us + sh.wait_us) + join;
      if (us < least) least = us, plan = {0, i, parts};
    }
  return plan;
}

// A launch holds less than 2^32 threads.
constexpr int64_t kMaxThreads = (INT64_C(1) << 32) - 1;
int64_t few_threads(int n) { return (static_cast<int64_t>(n) + 15) / 16 * (64 * kFewWaves); }
// Threads of a product's largest launch.
int64_t product_threads(int m, int n, int k, bool silu) {
  const Plan plan = plan_product(m, n, k, silu);
  if (plan.few) return few_threads(n);
  const Shape& sh = kShapes[plan.shape];
  const int64_t channels = silu ? 2 * static_cast<int64_t>(n) : n;
  const int64_t tiles = (channels + sh.channels - 1) / sh.channels * ((static_cast<int64_t>(m) + sh.rows - 1) / sh.rows);
  return std::max(tiles * sh.threads, plan.parts > 1 ? static_cast<int64_t>(m) * n + 255 : 0);   // (the join: at most an output each)
}

template <bool SILU>
int launch_product(const Product& p, int* workspace, hipStream_t s) {
  const Plan plan = plan_product(p.m, p.n, p.k, SILU);
  switch (plan.few) {
    case 0: break;
    case 1: return launch_few<1, SILU>(p, s);
    case 2: return launch_few<2, SILU>(p, s);
    case 3: return launch_few<3, SILU>(p, s);
    default: return launch_few<4, SILU>(p, s);
  }
  if (plan.parts > 1) {
    Product q = p;                                     // (gate and up rows are one matrix here)
    if (SILU) q.n = 2 * p.n;
    const int rc = plan.shape == kParted[0] ? launch_tile<4, 2, 4, 1, false, true>(q, s, plan.parts, workspace)
                                            : launch_tile<2, 2, 2, 4, false, true, 2>(q, s, plan.parts, workspace);
    if (rc != NKV_OK) return rc;
    const int v = p.n % 4 == 0 ? 4 : 1;
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>((p.n + v - 1) / v) * p.m + 255) / 256);
    if (v == 4) hipLaunchKernelGGL((join_kernel<4, SILU>), dim3(grid), dim3(256), 0, s, p, workspace, plan.parts);
    else hipLaunchKernelGGL((join_kernel<1, SILU>), dim3(grid), dim3(256), 0, s, p, workspace, plan.parts);
    return NKV_OK;
  }
  switch (plan.shape) {
    case 0: return launch_tile<8, 4, 4, 1, SILU>(p, s);
    case 1: return launch_tile<6, 4, 4, 1, SILU>(p, s);
    case 2:
      if constexpr (!SILU) return launch_tile<5, 4, 4, 1, SILU>(p, s);
      return NKV_ERR_UNSUPPORTED;                      // (never chosen)
    case 3: return launch_tile<4, 4, 4, 1, SILU>(p, s);
    case 4: return launch_tile<4, 2, 4, 1, SILU>(p, s);
    case 5: return launch_tile<4, 2, 2, 2, SILU, false, 2>(p, s);
    case 6: return launch_tile<2, 2, 2, 4, SILU, false, 2>(p, s);
    default: return launch_tile<2, 2, 1, 4, SILU, false, 2>(p, s);
  }
}

int64_t workspace_ints(int m, int n, int k, bool silu) {
  const Plan plan = plan_product(m, n, k, silu);
  return plan.parts > 1 ? static_cast<int64_t>(plan.parts) * m * n * (silu ? 2 : 1) : 0;
}

template <int NCH, bool NORM, bool SILU>
void launch_token(const Token& p, hipStream_t s) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  constexpr int R = token_rows(NCH, SILU);
  const int units = SILU ? p.n : (p.n + R - 1) / R;
  const int grid = std::min(token_waves(NCH, SILU) * cus, (units + kTokenWaves - 1) / kTokenWaves);   // waves per SIMD = workgroups per CU
  hipLaunchKernelGGL((token_kernel<NCH, NORM, SILU>), dim3(grid), dim3(kTokenThreads), 0, s, p);
}

template <bool NORM, bool SILU>
void launch_token(const Token& p, hipStream_t s) {
  const int nch = (p.k + 1023) / 1024;
  if (nch <= 1) launch_token<1, NORM, SILU>(p, s);
  else if (nch <= 2) launch_token<2, NORM, SILU>(p, s);
  else if (nch <= 3) launch_token<3, NORM, SILU>(p, s);
  else if (nch <= 4) launch_token<4, NORM, SILU>(p, s);
  else if (nch <= 6) launch_token<6, NORM, SILU>(p, s);
  else if (nch <= 8) launch_token<8, NORM, SILU>(p, s);
  else if (nch <= 10) launch_token<10, NORM, SILU>(p, s);
  else launch_token<12, NORM, SILU>(p, s);
}

int check_rows(const char* who, const void* x, const int8_t* q, const float* scale, int rows, int n) {
  NKV_CHECK_ARG(x != nullptr && q != nullptr && scale != nullptr, "%s: every pointer must be non-NULL", who);
  NKV_CHECK_ARG(rows >= 1 && n >= 16 && n % 16 == 0 && n <= kMaxRow,
                "%s: rows >= 1 and n a multiple of 16 in [16, %d] (got %d, %d)", who, kMaxRow, rows, n);
  NKV_CHECK_ARG(aligned16(x) && aligned16(q), "%s: rows must be 16-byte aligned", who);
  return NKV_OK;
}

int check_product(const char* who, const Product& p, int outputs_per_channel, const int* workspace) {
  NKV_CHECK_ARG(p.w != nullptr && p.sw != nullptr && p.x != nullptr && p.sx != nullptr && p.y != nullptr,
                "%s: weight, w_scale, x, x_scale and y must be non-NULL", who);
  NKV_CHECK_ARG(p.m >= 1 && p.n >= 1 && p.k >= 16 && p.k % 16 == 0 && p.k <= kMaxDepth,
                "%s: m and n >= 1 and k a multiple of 16 in [16, %d] (got %d, %d, %d)", who, kMaxDepth, p.m, p.n, p.k);
  NKV_CHECK_ARG(p.n <= INT32_MAX / 2 - 512 && p.m <= INT32_MAX - 512 &&
                    product_threads(p.m, p.n, p.k, outputs_per_channel == 2) <= kMaxThreads,
                "%s: m or n too large for a launch (got %d, %d)", who, p.m, p.n);
  NKV_CHECK_ARG(aligned16(p.w) && aligned16(p.x), "%s: weight and x must be 16-byte aligned", who);
  const int64_t out = 2 * static_cast<int64_t>(p.m) * p.n, channels = static_cast<int64_t>(p.n) * outputs_per_channel;
  NKV_CHECK_ARG(apart(p.y, out, p.w, channels * p.k) && apart(p.y, out, p.sw, 4 * channels) &&
                    apart(p.y, out, p.x, static_cast<int64_t>(p.m) * p.k) && apart(p.y, out, p.sx, 4 * static_cast<int64_t>(p.m)) &&
                    apart(p.y, out, p.bias, 2 * channels),
                "%s: y must not overlap an input", who);
  const int64_t ws = 4 * workspace_ints(p.m, p.n, p.k, outputs_per_channel == 2);
  NKV_CHECK_ARG(ws == 0 || (workspace != nullptr && aligned16(workspace)),
                "%s: this product needs a 16-byte aligned workspace of %lld bytes", who, static_cast<long long>(ws));
  NKV_CHECK_ARG(ws == 0 || (apart(workspace, ws, p.y, out) && apart(workspace, ws, p.w, channels * p.k) &&
                            apart(workspace, ws, p.sw, 4 * channels) && apart(workspace, ws, p.x, static_cast<int64_t>(p.m) * p.k) &&
                            apart(workspace, ws, p.sx, 4 * static_cast<int64_t>(p.m)) && apart(workspace, ws, p.bias, 2 * channels)),
                "%s: the workspace must not overlap an input or y", who);
  return NKV_OK;
}

template <bool NORM, bool SILU>
int token(const char* who, const Token& p, int m, void* stream) {
  NKV_CHECK_ARG(p.w != nullptr && p.sw != nullptr && p.x != nullptr && p.y != nullptr && (!NORM || p.nw != nullptr),
                "%s: weight, w_scale, x%s and y must be non-NULL", who, NORM ? ", norm_weight" : "");
  NKV_CHECK_ARG(m >= 1 && m <= kDraftRows && p.n >= 1 && p.n <= INT32_MAX / 2 - 512 && p.k >= 16 && p.k % 16 == 0 &&
                    p.k <= (m == 1 ? kTokenMaxK : kDraftMaxK),
                "%s: 1 <= m <= %d, n >= 1 and k a multiple of 16 in [16, %d], with one row [16, %d] (got %d, %d, %d)", who,
                kDraftRows, kDraftMaxK, kTokenMaxK, m, p.n, p.k);
  NKV_CHECK_ARG(m == 1 || few_threads(p.n) <= kMaxThreads, "%s: n too large for a launch (got %d)", who, p.n);
  NKV_CHECK_ARG(aligned16(p.w) && aligned16(p.x) && (!p.res || aligned16(p.res)) && (!p.nw || aligned16(p.nw)) &&
                    (!p.res_out || aligned16(p.res_out)),
                "%s: weight, x, residual, norm_weight and residual_out must be 16-byte aligned", who);
  // every workgroup reads the rows, norm_weight and its scales while others write y and one writes residual_out
  const int64_t rows = 2 * static_cast<int64_t>(m) * p.k, out = 2 * static_cast<int64_t>(m) * p.n, vec = 2 * static_cast<int64_t>(p.k);
  const int64_t channels = static_cast<int64_t>(p.n) * (SILU ? 2 : 1);
  struct Out {
    const char* name;
    const void* at;
    int64_t bytes;
  };
  for (const Out& o : {Out{"y", p.y, out}, Out{"residual_out", p.res_out, rows}})
    NKV_CHECK_ARG(apart(o.at, o.bytes, p.x, rows) && apart(o.at, o.bytes, p.res, rows) && apart(o.at, o.bytes, p.nw, vec) &&
                      apart(o.at, o.bytes, p.w, channels * p.k) && apart(o.at, o.bytes, p.sw, 4 * channels) &&
                      apart(o.at, o.bytes, p.bias, 2 * channels),
                  "%s: %s must not overlap an input", who, o.name);
  NKV_CHECK_ARG(apart(p.y, out, p.res_out, rows), "%s: y must not overlap residual_out", who);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (m == 1) {
    launch_token<NORM, SILU>(p, s);
  } else {
    const Product q{p.w, p.sw, nullptr, nullptr, p.bias, p.y, m, p.n, p.k};
    const Rows in{p.x, p.res, p.nw, p.res_out, p.eps};
    if (p.k <= 1024) launch_draft<2, NORM, SILU>(q, in, s);
    else if (p.k <= 2560) launch_draft<5, NORM, SILU>(q, in, s);
    else launch_draft<8, NORM, SILU>(q, in, s);
  }
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
  NKV_CHECK_ARG(chunks <= INT64_C(256) * ((1 << 24) - 1), "nkv_dequantize_q8: at most 2^36 - 2^12 elements (a launch's threads)");
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

extern "C" int64_t nkv_linear_q8_workspace(int m, int n, int k, int gated) {
  if (m < 1 || n < 1 || k < 16 || m > INT32_MAX - 512 || n > INT32_MAX / 2 - 512 || k > kMaxDepth) return 0;
  return workspace_ints(m, n, k, gated != 0);
}

extern "C" int nkv_linear_q8_tile(int m, int n, int k, int gated) {
  if (m < 1 || n < 1 || k < 16 || m > INT32_MAX - 512 || n > INT32_MAX / 2 - 512 || k > kMaxDepth) return 0;
  const Plan plan = plan_product(m, n, k, gated != 0);
  return plan.few ? 0 : kShapes[plan.shape].channels | kShapes[plan.shape].rows << 10 | plan.parts << 20;
}

extern "C" int nkv_linear_q8(const int8_t* weight, const float* w_scale, const int8_t* x, const float* x_scale,
                             const uint16_t* bias, uint16_t* y, int m, int n, int k, int32_t* workspace,
                             void* stream) {
  const Product p{weight, w_scale, x, x_scale, bias, y, m, n, k};
  const int rc = check_product("nkv_linear_q8", p, 1, workspace);
  if (rc != NKV_OK) return rc;
  const int launched = launch_product<false>(p, workspace, reinterpret_cast<hipStream_t>(stream));
  return launched != NKV_OK ? launched : launch_status("nkv_linear_q8");
}

extern "C" int nkv_linear_silu_mul_q8(const int8_t* gate_up_weight, const float* w_scale, const int8_t* x,
                                      const float* x_scale, uint16_t* y, int m, int intermediate, int k, int32_t* workspace,
                                      void* stream) {
  const Product p{gate_up_weight, w_scale, x, x_scale, nullptr, y, m, intermediate, k};
  const int rc = check_product("nkv_linear_silu_mul_q8", p, 2, workspace);
  if (rc != NKV_OK) return rc;
  const int launched = launch_product<true>(p, workspace, reinterpret_cast<hipStream_t>(stream));
  return launched != NKV_OK ? launched : launch_status("nkv_linear_silu_mul_q8");
}

extern "C" int nkv_gemv_q8(const int8_t* weight, const float* w_scale, const uint16_t* x, const uint16_t* bias, uint16_t* y,
                           int m, int n, int k, void* stream) {
  return token<false, false>("nkv_gemv_q8", Token{weight, w_scale, x, nullptr, nullptr, bias, y, nullptr, 0.0f, n, k}, m, stream);
}

extern "C" int nkv_gemv_silu_mul_q8(const int8_t* gate_up_weight, const float* w_scale, const uint16_t* x, uint16_t* y, int m,
                                    int intermediate, int k, void* stream) {
  return token<false, true>("nkv_gemv_silu_mul_q8",
                            Token{gate_up_weight, w_scale, x, nullptr, nullptr, nullptr, y, nullptr, 0.0f, intermediate, k}, m, stream);
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
                           Token{gate_up_weight, w_scale, x, residual, norm_weight, nullptr, y, residual_out, eps, intermediate, k}, m,
                           stream);
}
