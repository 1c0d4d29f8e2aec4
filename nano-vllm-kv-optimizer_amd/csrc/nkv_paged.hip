// Writing, reading and moving rows of the dense path's paged cache.
//
//  * append_kernel: the fused projection's rows q|k|v: per head of q and k an
//    RMSNorm over the head's dims (optional) and the rotation of the first R
//    dims by the row's position, then q goes out, and k and v go to the row's
//    slot of the cache, in one pass:
//      x' = x rsqrt(mean(x^2) + eps) w,
//      (a, b) -> (a cos - b sin, b cos + a sin) for the pairs (i, i + R/2), or
//      (2i, 2i + 1) when interleaved, all in fp32 and rounded once: to bf16, or
//      to the codes rne(y 127 / a) with the scale a / 127, a = max |y|.
//  * read_kernel: rows of the cache at given slots as bf16.
//  * move_kernel: rows from slots to slots, bit by bit, through a workspace
//    (the slots may overlap: a drafted tree's accepted path closes up in place).
// All are bound by their reads and writes of each row once (small calls: by the launch).  Measured, 8 KV heads
// of 128 dims: append with 32 query heads, norms and rotation, 4096 rows 20.2 us (102 MB: 5.0 TB/s), one
// row 2.9; read of 4096 scattered rows 8.7 us (7.2 in 8 bits), move of 4096 6.6 + 6.5, of 5 2.6 + 2.7.
#include <algorithm>

#include "nkv_paged.h"

namespace nkv {

int fill_paged(const char* who, void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
               int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size, int head_dim,
               PagedCache* c) {
  NKV_CHECK_SUPPORTED(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128 (got %d)", who, head_dim);
  NKV_CHECK_SUPPORTED(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                      "%s: page_size must be a power of two from 16 to 4096 (got %d)", who, page_size);
  NKV_CHECK_ARG(k && v, "%s: the cache is NULL", who);
  NKV_CHECK_ARG((k_scale != nullptr) == (v_scale != nullptr), "%s: keys and values have both scales or none", who);
  NKV_CHECK_ARG((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 16 == 0,
                "%s: scales must lie on a 16-byte boundary", who);
  NKV_CHECK_ARG(pages >= 1 && num_kv_heads >= 1, "%s: pages and num_kv_heads must be positive", who);
  NKV_CHECK_ARG(static_cast<int64_t>(pages) * page_size <= INT32_MAX, "%s: a cache holds fewer than 2^31 tokens", who);
  const int elem = k_scale ? 1 : 2;
  NKV_CHECK_ARG(page_stride >= 0 && head_stride >= 0 && token_stride >= head_dim,
                "%s: strides must not be negative, rows not overlap", who);
  NKV_CHECK_ARG((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                    (page_stride * elem | head_stride * elem | token_stride * elem) % 16 == 0,
                "%s: rows must lie on 16-byte boundaries", who);
  // (the attention's 32-bit offsets inside a page)
  NKV_CHECK_ARG(token_stride * elem <= (1 << 26), "%s: rows lie too far apart", who);
  c->k = static_cast<char*>(k);
  c->v = static_cast<char*>(v);
  c->ks = k_scale;
  c->vs = v_scale;
  c->sp = page_stride;
  c->sh = head_stride;
  c->st = token_stride;
  c->pages = pages;
  c->hkv = num_kv_heads;
  c->page = page_size;
  c->shift = 0;
  while ((1 << c->shift) < page_size) ++c->shift;
  return NKV_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxUnits = 1 << 27;   // (16 lanes each: a launch has fewer than 2^32 threads)

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}

struct AppendParams {
  const uint16_t* q_in;   // rows of heads: [q |] k | v, or k and v apart
  const uint16_t* k_in;
  const uint16_t* v_in;
  int64_t q_ls, k_ls, v_ls;   // elements from row to row
  const int32_t* slots;
  const int64_t* positions;
  const float* cos_t;     // [max_pos][R / 2]
  const float* sin_t;
  const uint16_t* q_w;
  const uint16_t* k_w;
  uint16_t* q_out;        // [rows][hq][D]
  uint32_t units;         // rows * (hq + 2 hkv)
  int hq, rot, max_pos, interleaved;
  float eps;
};

// The 8 values of y as int8 codes rne(y 127 / a), inv = 127 / a.  inv and y * inv
// are off by half a step of fp32 each, which a tie of bf16 values (rows as they came)
// does not bear: those are rounded to 2^-15 first, which makes their ties exact.
__device__ __forceinline__ uint2 codes8(const float (&y)[8], float inv, float top) {
  constexpr float kSnap = 0x1.8p8f, kMagic = 0x1.8p23f;   // sums with them are rounded to 2^-15, to whole numbers
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = y[e] * inv;
    const bool bf16s = ((__float_as_uint(y[e]) | __float_as_uint(top)) & 0xffffu) == 0;
    const float r = bf16s ? ((x + kSnap) + (kMagic - kSnap)) - kMagic : __builtin_rintf(x);
    w[e >> 2] |= (static_cast<uint32_t>(static_cast<int>(r)) & 0xffu) << (8 * (e & 3));
  }
  return make_uint2(w[0], w[1]);
}

// D / 16 lanes a (row, head): lane j holds two 8-dim chunks.  In the rotated
// part they are the two halves' chunks j and j + R/16 (the pairs i, i + R/2 meet in a
// lane), behind it, and when neighbouring dims are paired, two that follow one
// another; either way pairs 8 j .. 8 j + 7 are the lane's, so cos and sin come as 32 bytes each.
template <int D, bool INT8>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendParams p, const PagedCache c) {
  constexpr int L = D / 16;
  const uint32_t unit = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const int j = threadIdx.x % L;
  const int nh = p.hq + 2 * c.hkv;
  const uint32_t at = min(unit, p.units - 1);
  const int64_t t = at / static_cast<uint32_t>(nh);
  const int head = static_cast<int>(at % static_cast<uint32_t>(nh));
  const bool isq = head < p.hq, isv = head >= p.hq + c.hkv;
  const int hk = isv ? head - p.hq - c.hkv : head - p.hq;   // head of the cache
  const uint16_t* src = isq ? p.q_in + t * p.q_ls + head * D : (isv ? p.v_in + t * p.v_ls : p.k_in + t * p.k_ls) + hk * D;
  const int half = p.rot >> 4;   // lanes that rotate
  const bool turns = j < half && !isv;
  const int ca = p.interleaved ? 2 * j : (j < half ? j : 2 * j);
  const int cb = p.interleaved ? 2 * j + 1 : (j < half ? j + half : 2 * j + 1);
  const uint4 xa = reinterpret_cast<const uint4*>(src)[ca];
  const uint4 xb = reinterpret_cast<const uint4*>(src)[cb];
  const int slot = p.slots ? p.slots[t] : -1;
  float a[8], b[8];
  unpack8(xa, a);
  unpack8(xb, b);
  const uint16_t* w = isq ? p.q_w : p.k_w;
  if (!isv && w != nullptr) {
    float wa[8], wb[8];
    unpack8(reinterpret_cast<const uint4*>(w)[ca], wa);
    unpack8(reinterpret_cast<const uint4*>(w)[cb], wb);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    // (a root and a division: rsqrtf is off by up to 2 ulp)
    const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] *= r * wa[e];
      b[e] *= r * wb[e];
    }
  }
  if (turns) {
    int64_t pos = p.positions[t];
    pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
    const float4* ct = reinterpret_cast<const float4*>(p.cos_t + pos * (p.rot / 2) + 8 * j);
    const float4* st = reinterpret_cast<const float4*>(p.sin_t + pos * (p.rot / 2) + 8 * j);
    const float4 c0 = ct[0], c1 = ct[1], s0 = st[0], s1 = st[1];
    const float cc[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    float y[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // pair i: (a[i], b[i]), or when interleaved neighbours of a, then of b
      const float u = p.interleaved ? (i < 4 ? a[2 * (i & 3)] : b[2 * (i & 3)]) : a[i];
      const float v = p.interleaved ? (i < 4 ? a[2 * (i & 3) + 1] : b[2 * (i & 3) + 1]) : b[i];
      y[i] = u * cc[i] - v * sn[i];
      z[i] = v * cc[i] + u * sn[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = p.interleaved ? (i & 1 ? z[i >> 1] : y[i >> 1]) : y[i];
      b[i] = p.interleaved ? (i & 1 ? z[4 + (i >> 1)] : y[4 + (i >> 1)]) : z[i];
    }
  }
  float top = 0.0f;
  bool odd = false;
  if (INT8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, fmaxf(fabsf(a[e]), fabsf(b[e])));
      odd = odd || a[e] != a[e] || b[e] != b[e];
    }
    top = odd ? INFINITY : top;   // (a maximum passes a NaN over)
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  }
  if (unit >= p.units) return;   // (behind the shuffles)
  if (isq) {
    uint4* dst = reinterpret_cast<uint4*>(p.q_out + (t * p.hq + head) * D);
    dst[ca] = pack8(a);
    dst[cb] = pack8(b);
    return;
  }
  if (!paged_slot_ok(c, slot)) return;
  const int64_t row = paged_row(c, slot, hk);
  if (INT8) {
    const bool none = !(top >= kTinyRow) || top == INFINITY;
    const float inv = none ? 0.0f : 127.0f / top;
    if (top == INFINITY) {   // (an infinite value times 0 is no code)
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = b[e] = 0.0f;
    }
    uint2* dst = reinterpret_cast<uint2*>((isv ? c.v : c.k) + row);
    dst[ca] = codes8(a, inv, top);
    dst[cb] = codes8(b, inv, top);
    if (j == 0)
      (isv ? c.vs : c.ks)[paged_scale(c, slot, hk)] = top == INFINITY ? NAN : (none ? 0.0f : top / 127.0f);
  } else {
    uint4* dst = reinterpret_cast<uint4*>((isv ? c.v : c.k) + 2 * row);
    dst[ca] = pack8(a);
    dst[cb] = pack8(b);
  }
}

// 16-byte pieces of a row as they lie in the cache.
template <int D, bool INT8>
constexpr int kPieces = D * (INT8 ? 1 : 2) / 16;

// One lane a piece: unit (row, key or value, head) of the slots.
template <int D, bool INT8>
__global__ __launch_bounds__(kThreads) void read_kernel(const PagedCache c, const int32_t* slots, uint32_t units,
                                                        uint16_t* k_out, uint16_t* v_out) {
  constexpr int L = kPieces<D, INT8>;
  const uint32_t unit = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (unit >= units) return;
  const int j = threadIdx.x % L;
  const int h = static_cast<int>(unit % static_cast<uint32_t>(c.hkv));
  const uint32_t x = unit / static_cast<uint32_t>(c.hkv);
  const bool isv = x & 1;
  const int64_t t = x >> 1;
  const int slot = slots[t];
  uint16_t* out = (isv ? v_out : k_out) + (t * c.hkv + h) * D;
  const bool ok = paged_slot_ok(c, slot);
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  if (ok) w = reinterpret_cast<const uint4*>((isv ? c.v : c.k) + paged_row(c, slot, h) * (INT8 ? 1 : 2))[j];
  if (!INT8) {
    reinterpret_cast<uint4*>(out)[j] = w;
    return;
  }
  const float s = ok ? (isv ? c.vs : c.ks)[paged_scale(c, slot, h)] : 0.0f;
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
  float f[2][8];
#pragma unroll
  for (int e = 0; e < 16; ++e)
    f[e >> 3][e & 7] = static_cast<float>(static_cast<int8_t>((q[e >> 2] >> (8 * (e & 3))) & 0xffu)) * s;
  reinterpret_cast<uint4*>(out)[2 * j] = pack8(f[0]);
  reinterpret_cast<uint4*>(out)[2 * j + 1] = pack8(f[1]);
}

// Rows to the workspace (OUT false) or from it to their new slots: two
// launches, so that a slot that is read and written keeps neither half old.  A
// pair with a slot outside the cache moves nothing.  Workspace: the rows [n][2][hkv][D],
// then in 8 bits their scales.
template <int D, bool INT8, bool OUT>
__global__ __launch_bounds__(kThreads) void move_kernel(const PagedCache c, const int32_t* src, const int32_t* dst,
                                                        uint32_t units, char* ws) {
  constexpr int L = kPieces<D, INT8>;
  const uint32_t unit = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (unit >= units) return;
  const int j = threadIdx.x % L;
  const int h = static_cast<int>(unit % static_cast<uint32_t>(c.hkv));
  const uint32_t x = unit / static_cast<uint32_t>(c.hkv);
  const bool isv = x & 1;
  const int from = src[x >> 1], to = dst[x >> 1];
  if (!paged_slot_ok(c, from) || !paged_slot_ok(c, to)) return;
  const int slot = OUT ? to : from;
  uint4* row = reinterpret_cast<uint4*>((isv ? c.v : c.k) + paged_row(c, slot, h) * (INT8 ? 1 : 2)) + j;
  uint4* held = reinterpret_cast<uint4*>(ws) + static_cast<int64_t>(unit) * L + j;
  if (OUT) *row = *held; else *held = *row;
  if (INT8 && j == 0) {
    float* s = (isv ? c.vs : c.ks) + paged_scale(c, slot, h);
    float* hs = reinterpret_cast<float*>(ws + static_cast<int64_t>(units) * L * 16) + unit;
    if (OUT) *s = *hs; else *hs = *s;
  }
}

template <typename F>
void by_format(int head_dim, bool int8, F&& f) {
  using std::integral_constant;
  if (head_dim == 128)
    int8 ? f(integral_constant<int, 128>{}, integral_constant<bool, true>{})
         : f(integral_constant<int, 128>{}, integral_constant<bool, false>{});
  else
    int8 ? f(integral_constant<int, 64>{}, integral_constant<bool, true>{})
         : f(integral_constant<int, 64>{}, integral_constant<bool, false>{});
}

unsigned groups_of(int64_t units, int lanes) {
  const int64_t per = kThreads / lanes;
  return static_cast<unsigned>((units + per - 1) / per);
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int nkv_paged_append(void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
                                int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size,
                                int head_dim, const uint16_t* q_rows, int64_t q_stride, const uint16_t* k_rows,
                                int64_t k_stride, const uint16_t* v_rows, int64_t v_stride, int rows, int num_heads,
                                const int32_t* slots, const int64_t* positions, const float* cos_table,
                                const float* sin_table, int max_position, int rotary_dim, int interleaved,
                                const uint16_t* q_weight, const uint16_t* k_weight, float eps, uint16_t* q_out,
                                void* stream) {
  PagedCache c;
  if (int rc = fill_paged("nkv_paged_append", k, v, k_scale, v_scale, page_stride, head_stride, token_stride, pages,
                          num_kv_heads, page_size, head_dim, &c))
    return rc;
  NKV_CHECK_ARG(rows >= 0 && num_heads >= 0, "nkv_paged_append: rows and num_heads must not be negative");
  const int64_t units = static_cast<int64_t>(rows) * (num_heads + 2LL * num_kv_heads);
  NKV_CHECK_ARG(units <= kMaxUnits, "nkv_paged_append: at most 2^27 rows of heads");
  NKV_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 16 == 0,
                "nkv_paged_append: rotary_dim must be a multiple of 16 up to head_dim (got %d)", rotary_dim);
  if (rows == 0) return NKV_OK;
  NKV_CHECK_ARG(k_rows && v_rows && slots, "nkv_paged_append: k_rows, v_rows and slots must be non-NULL");
  NKV_CHECK_ARG(num_heads == 0 || (q_rows && q_out), "nkv_paged_append: q_rows and q_out must be non-NULL");
  NKV_CHECK_ARG(rotary_dim == 0 || (positions && cos_table && sin_table && max_position >= 1),
                "nkv_paged_append: a rotation needs positions and tables");
  NKV_CHECK_ARG((reinterpret_cast<uintptr_t>(q_rows) | reinterpret_cast<uintptr_t>(k_rows) |
                 reinterpret_cast<uintptr_t>(v_rows) | reinterpret_cast<uintptr_t>(q_out) |
                 reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table) |
                 reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight)) % 16 == 0 &&
                    (q_stride | k_stride | v_stride) % 8 == 0,
                "nkv_paged_append: rows, tables and weights must lie on 16-byte boundaries");
  const AppendParams p{q_rows,    k_rows,    v_rows,    q_stride, k_stride,
                       v_stride,  slots,     positions, cos_table, sin_table,
                       q_weight,  k_weight,  q_out,     static_cast<uint32_t>(units), num_heads,
                       rotary_dim, max_position, interleaved, eps};
  by_format(head_dim, k_scale != nullptr, [&](auto d, auto i8) {
    append_kernel<decltype(d)::value, decltype(i8)::value>
        <<<groups_of(units, decltype(d)::value / 16), kThreads, 0, static_cast<hipStream_t>(stream)>>>(p, c);
  });
  return launch_status("nkv_paged_append");
}

extern "C" int nkv_paged_read(void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
                              int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size,
                              int head_dim, const int32_t* slots, int rows, uint16_t* k_out, uint16_t* v_out,
                              void* stream) {
  PagedCache c;
  if (int rc = fill_paged("nkv_paged_read", k, v, k_scale, v_scale, page_stride, head_stride, token_stride, pages,
                          num_kv_heads, page_size, head_dim, &c))
    return rc;
  const int64_t units = static_cast<int64_t>(rows) * 2 * num_kv_heads;
  NKV_CHECK_ARG(rows >= 0 && units <= kMaxUnits, "nkv_paged_read: from 0 to 2^27 rows of heads");
  if (rows == 0) return NKV_OK;
  NKV_CHECK_ARG(slots && k_out && v_out, "nkv_paged_read: slots and outputs must be non-NULL");
  NKV_CHECK_ARG((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0,
                "nkv_paged_read: outputs must lie on 16-byte boundaries");
  by_format(head_dim, k_scale != nullptr, [&](auto d, auto i8) {
    constexpr int D = decltype(d)::value;
    constexpr bool I8 = decltype(i8)::value;
    read_kernel<D, I8><<<groups_of(units, kPieces<D, I8>), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
        c, slots, static_cast<uint32_t>(units), k_out, v_out);
  });
  return launch_status("nkv_paged_read");
}

extern "C" int64_t nkv_paged_move_workspace(int num_kv_heads, int head_dim, int int8, int rows) {
  return static_cast<int64_t>(rows) * 2 * num_kv_heads * (int8 ? head_dim + 4 : 2 * head_dim);
}

extern "C" int nkv_paged_move(void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
                              int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size,
                              int head_dim, const int32_t* src, const int32_t* dst, int rows, void* workspace,
                              void* stream) {
  PagedCache c;
  if (int rc = fill_paged("nkv_paged_move", k, v, k_scale, v_scale, page_stride, head_stride, token_stride, pages,
                          num_kv_heads, page_size, head_dim, &c))
    return rc;
  const int64_t units = static_cast<int64_t>(rows) * 2 * num_kv_heads;
  NKV_CHECK_ARG(rows >= 0 && units <= kMaxUnits, "nkv_paged_move: from 0 to 2^27 rows of heads");
  if (rows == 0) return NKV_OK;
  NKV_CHECK_ARG(src && dst && workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                "nkv_paged_move: src, dst and a workspace on a 16-byte boundary are needed");
  const auto s = static_cast<hipStream_t>(stream);
  by_format(head_dim, k_scale != nullptr, [&](auto d, auto i8) {
    constexpr int D = decltype(d)::value;
    constexpr bool I8 = decltype(i8)::value;
    const unsigned grid = groups_of(units, kPieces<D, I8>);
    char* ws = static_cast<char*>(workspace);
    move_kernel<D, I8, false><<<grid, kThreads, 0, s>>>(c, src, dst, static_cast<uint32_t>(units), ws);
    move_kernel<D, I8, true><<<grid, kThreads, 0, s>>>(c, src, dst, static_cast<uint32_t>(units), ws);
  });
  return launch_status("nkv_paged_move");
}
