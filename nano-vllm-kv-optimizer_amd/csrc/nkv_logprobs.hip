// Log probabilities of given tokens, the entropy of their distribution and its
// most likely alternatives, from rows of logits, in one pass over each row.
//
// With m the row's maximum, s the sum of e^(x - m) over all elements but the
// maximum, and w the sum of (m - x) e^(x - m):
//   log Z = m + log1p(s),  log p(t) = (x_t - m) - log1p(s),
//   H = log1p(s) + w / (1 + s).
// The maximum's own term, 1, stays out of s: the sum keeps the digits that a
// confident row's entropy and log probability are made of (1 + 1e-9 is 1).
// Pieces (m, s, w) join exactly: with d = m1 - m2 >= 0 and r = e^-d,
//   s = s1 + r (s2 + 1),  w = w1 + r (w2 + d (s2 + 1)).
//
// Work split: a wavefront takes a run of its row; its maximum is the same in
// all lanes and moves rarely, so an element costs a product, an exp2, two
// additions and the comparisons.  Alternatives: elements that reach the
// wavefront's bar go to its list of up to 256 in LDS; a list grown long is
// cut to its best.  The bar lies below the n-th largest of the lanes' maxima so
// far, so few elements ever reach it.  Order:
// value descending (NaN above all), index ascending.  Bound by reading the
// logits once, or by the launches (one row).  Measured, rows of 151936: 2048 in bf16 with 5
// alternatives 143 us (4.3 TB/s; 127 with none, 196 with 50: the vector instructions, 6 and an exp2 an
// element, run beside the loads and are not all hidden); one row of fp32 with 20: 9.3 and 7.1 us.
//
// Exponents are in log2 units: 2^-z with z = M - x log2 e in one fused operation, M = m
// log2 e rounded.  What M's rounding is off by, e, scales every term by 2^e alike, and adds
// to every z: both are mended in the sums (settle), not in the terms.  e is up to half an ulp of M: 2^-8
// for |m| < 2^16.  Larger maxima (runs that hold nothing but a mask's value) take m - x itself, since 2^e
// leaves the range from |m| = 2^32 on.
#include <algorithm>

#include "nkv_common.h"

namespace nkv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kList = 256;       // candidates a wavefront keeps at most
constexpr int kMaxTop = 64;      // alternatives: one a lane in the final order
constexpr int kEach = 16;        // elements a lane takes per iteration
constexpr int kMaxSplits = 128;  // pieces of a row
constexpr int kMaxRows = (1 << 24) - 1;   // (a launch has fewer than 2^32 threads)
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFar = 0x1p16f;  // maxima from here on are subtracted directly

enum Kind { kF32 = 0, kBf16 = 1, kF16 = 2 };

struct Params {
  const char* x;
  int64_t stride;          // elements from row to row
  int rows, vocab, top, splits;
  int per;                 // 16-byte pieces of a wavefront's run
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_lp;           // [rows][top]
  int64_t* top_ids;
  float* ws;               // [rows][splits][4 + 2 top]: m, s, w, entries, then their keys and ids
};

template <int K> constexpr int kBytes = K == kF32 ? 4 : 2;

template <int K>
__device__ __forceinline__ float element(const char* row, int64_t i) {
  if (K == kF32) return reinterpret_cast<const float*>(row)[i];
  const uint16_t b = reinterpret_cast<const uint16_t*>(row)[i];
  return K == kBf16 ? bf16_to_f32(b) : f16_bits_to_f32(b);
}

struct Stat { float m, s, w; };

__device__ __forceinline__ float exp_neg(float y) { return __builtin_amdgcn_exp2f(y * -kLog2e); }
// The maximum that keeps a NaN (v_maximum3_f32: two elements an instruction, none quieted first).
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ Stat join(Stat a, Stat b) {
  if (b.m > a.m) { const Stat t = a; a = b; b = t; }
  if (b.m == -INFINITY) return Stat{a.m, a.s + b.s, a.w + b.w};   // nothing, or a NaN that stays
  // (past 200 r is 0; d itself, 3e38 behind rows masked with the lowest value, times a sum would be infinite)
  const float d = fminf(a.m - b.m, 200.0f), r = exp_neg(d);
  return Stat{a.m, a.s + r * (b.s + 1.0f), a.w + r * (b.w + d * (b.s + 1.0f))};
}

__device__ __forceinline__ int count(uint64_t mask) { return __popcll(mask); }
__device__ __forceinline__ int below(uint64_t mask) {   // set bits under this lane's
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
}

// A reduction over the lanes of the wavefront (row shifts, then the rows' ends carried on), `none` its
// neutral element.
template <typename F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x, uint32_t none, F&& f) {
#define NKV_STEP(ctrl, rows) \
  x = f(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(x), ctrl, rows, 0xf, false)))
  NKV_STEP(0x111, 0xf);
  NKV_STEP(0x112, 0xf);
  NKV_STEP(0x114, 0xf);
  NKV_STEP(0x118, 0xf);
  NKV_STEP(0x142, 0xa);
  NKV_STEP(0x143, 0xc);
#undef NKV_STEP
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), kWave - 1));
}
__device__ __forceinline__ float lane_total(float x) {
  return __uint_as_float(over_lanes(__float_as_uint(x), 0u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ float lane_top(float x) {   // (a NaN gives way)
  return __uint_as_float(over_lanes(__float_as_uint(x), 0xff800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ uint32_t lane_max(uint32_t x) {
  return over_lanes(x, 0u, [](uint32_t a, uint32_t b) { return max(a, b); });
}
// What keys from lo to hi have in common, as the least number that has it; bit: the first in which they differ (-1: none).
__device__ __forceinline__ uint32_t prefix_of(uint32_t lo, uint32_t hi, int& bit) {
  bit = lo == hi ? -1 : 31 - __builtin_clz(lo ^ hi);
  return bit < 0 ? hi : hi & ~((2u << bit) - 1);
}

// A wavefront's candidates: (key, id) in LDS, and the bar that a new one has to
// beat: a larger key, or the same with a lower id.
struct List {
  uint32_t* keys;
  int* ids;
  int cnt, top;
  uint32_t bar;
  int bar_id;

  __device__ __forceinline__ bool beats(uint32_t key, int id) const { return key > bar || (key == bar && id < bar_id); }

  // Of up to four candidates a lane (an empty one has key 0, below every element's) the
  // best: at least `top` of them and at most `most` (top <= most <= 64).  They become the
  // list, and the bar keeps out what would not be among them.
  __device__ void keep_best(const uint32_t (&k)[4], const int (&id)[4], int have, int most) {
    auto above = [&](auto&& f) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) n += count(__ballot(f(k[i], id[i])));
      return n;
    };
    uint32_t t = 1;      // the smallest key kept (all candidates when there are few)
    int last = INT32_MAX;
    if (have > most) {
      // at least `top` keys are t or more, bit by bit, until they are few enough
      const uint32_t hi = lane_max(max(max(k[0], k[1]), max(k[2], k[3])));
      const uint32_t lo = ~lane_max(max(max(~(k[0] - 1), ~(k[1] - 1)), max(~(k[2] - 1), ~(k[3] - 1)))) + 1;   // (of those not 0)
      int kept = have, bit;
      for (t = prefix_of(lo, hi, bit); bit >= 0 && kept > most; --bit) {
        const uint32_t c = t | (1u << bit);
        const int n = above([&](uint32_t a, int) { return a >= c; });
        if (n >= top) {
          t = c;
          kept = n;
        }
      }
      if (kept > most) {   // too many are equal: of those the lowest ids
        const int more = above([&](uint32_t a, int) { return a > t; });
        last = 0;
        for (bit = 30; bit >= 0; --bit) {
          const int c = last | (1 << bit);
          // ids below c are too few: the (top - more)-th lowest is c or more
          if (above([&](uint32_t a, int i) { return a == t && i < c; }) < top - more) last = c;
        }
      }
      bar = t;
      bar_id = last;
    }
    wave_lds_sync();   // (the list has been read)
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool stays = k[i] > t || (k[i] == t && id[i] <= last);
      const uint64_t mask = __ballot(stays);
      if (stays) {
        keys[n + below(mask)] = k[i];
        ids[n + below(mask)] = id[i];
      }
      n += count(mask);
    }
    cnt = n;
    wave_lds_sync();
  }
  __device__ void cut(int lane, int most) {
    wave_lds_sync();
    uint32_t k[4];
    int id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = i * kWave + lane < cnt;
      k[i] = in ? keys[i * kWave + lane] : 0u;
      id[i] = in ? ids[i * kWave + lane] : INT32_MAX;
    }
    keep_best(k, id, cnt, most);
  }
  // Every lane's candidate (if it has one that beats the bar); the whole wavefront calls it.
  __device__ __forceinline__ void add(bool has, uint32_t key, int id, int lane) {
    has = has && beats(key, id);
    uint64_t mask = __ballot(has);
    if (mask == 0) return;
    if (cnt + count(mask) > kList) {
      cut(lane, kWave);
      has = has && beats(key, id);
      mask = __ballot(has);
    }
    if (has) {
      keys[cnt + below(mask)] = key;
      ids[cnt + below(mask)] = id;
    }
    cnt += count(mask);
  }
};

// The logit of the row's token (NaN: no such token).
template <int K>
__device__ __forceinline__ float token_logit(const Params& p, int row, const char* x) {
  const int64_t tok = p.tokens[row];
  return tok >= 0 && tok < p.vocab ? element<K>(x, tok) : NAN;
}
// The lanes' best `top` (key, id) in order and the row's numbers, by one wavefront; xt: the token's logit.
__device__ __forceinline__ void finish(const Params& p, int row, float xt, Stat t, const List& list, int lane) {
  const float z = t.m == INFINITY ? NAN : log1pf(t.s);   // (inf - inf: no probabilities)
  const bool none = t.m == -INFINITY;                    // every element is -inf: no distribution
  if (lane == 0) {
    p.logprob[row] = (xt - t.m) - z;
    p.entropy[row] = none ? NAN : z + t.w / (1.0f + t.s);
  }
  if (p.top == 0) return;
  wave_lds_sync();
  const uint32_t key = lane < p.top ? list.keys[lane] : 0u;
  const int id = lane < p.top ? list.ids[lane] : INT32_MAX;
  int rank = 0;
  for (int i = 0; i < p.top; ++i) {
    const uint32_t k = list.keys[i];
    rank += k > key || (k == key && list.ids[i] < id) ? 1 : 0;
  }
  if (lane < p.top) {
    const int64_t at = static_cast<int64_t>(row) * p.top + rank;
    p.top_lp[at] = (key_score(key) - t.m) - z;
    p.top_ids[at] = id;
  }
}

// The wavefronts' lists (up to 64 each) and numbers as one: in wavefront 0.
__device__ __forceinline__ void join_waves(uint32_t (&keys)[kWaves][kList], int (&ids)[kWaves][kList],
                                           Stat (&stats)[kWaves], int (&counts)[kWaves], int wave, int lane, Stat& t,
                                           List& list) {
  if (lane == 0) {
    stats[wave] = t;
    counts[wave] = list.cnt;
  }
  __syncthreads();
  if (wave != 0) return;
  t = stats[0];   // (in all lanes)
#pragma unroll
  for (int i = 1; i < kWaves; ++i) t = join(t, stats[i]);
  uint32_t k[4];
  int id[4], have = 0;
  static_assert(kWaves == 4, "one list a slot");
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const bool in = lane < counts[i];
    k[i] = in ? keys[i][lane] : 0u;
    id[i] = in ? ids[i][lane] : INT32_MAX;
    have += counts[i];
  }
  list.keep_best(k, id, have, list.top);
}

template <int K>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const Params p) {
  constexpr int E = 16 / kBytes<K>;    // elements a load
  constexpr int U = kEach / E;         // loads an iteration
  __shared__ uint32_t keys[kWaves][kList];
  __shared__ int ids[kWaves][kList];
  __shared__ Stat stats[kWaves];
  __shared__ int counts[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x / static_cast<unsigned>(p.splits);
  const int split = blockIdx.x % static_cast<unsigned>(p.splits);
  const char* x = p.x + static_cast<int64_t>(row) * p.stride * kBytes<K>;
  // 16-byte pieces from the boundary at or before the row: element i is in piece (i + head) / E
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / kBytes<K>);
  const int64_t pieces = (static_cast<int64_t>(p.vocab) + head + E - 1) / E;
  const int64_t lo = min(static_cast<int64_t>(p.per) * (split * kWaves + wave), pieces), hi = min(lo + p.per, pieces);

  // (early: two round trips that nothing waits for)
  const float xt = p.splits == 1 && wave == 0 ? token_logit<K>(p, row, x) : 0.0f;
  List list{keys[wave], ids[wave], 0, p.top, 0u, INT32_MAX};
  int until = 1, iterations = 1;                  // iterations until the bar is set anew
  float best = -INFINITY;                         // the lane's maximum so far
  float bar = p.top > 0 ? -INFINITY : INFINITY;   // the list's, as a value
  float m = -INFINITY, s = 0.0f, w = 0.0f;        // m is the wavefront's, s and w the lane's part
  // since m moved: the sums of 2^-z and z 2^-z, big_m = m log2 e rounded (0 of -inf), off what it lacks
  float sz = 0.0f, wz = 0.0f, big_m = 0.0f, off = 0.0f;
  auto settle = [&]() {
    const float f = __builtin_amdgcn_exp2f(-off);
    s += sz * f;
    w += (wz + off * sz) * f * (1.0f / kLog2e);
    sz = wz = 0.0f;
  };
  auto widen = [&](const uint4& raw, float (&f)[E]) {
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < E; ++e)
      f[e] = K == kF32 ? __uint_as_float(r[e & 3])
                       : K == kBf16 ? (e & 1 ? bf16_hi(r[(e >> 1) & 3]) : bf16_lo(r[(e >> 1) & 3]))
                                    : f16_bits_to_f32(static_cast<uint16_t>(r[(e >> 1) & 3] >> (16 * (e & 1))));
  };
  // a piece whose elements do not all exist (the row's ends, the run's end)
  auto load_some = [&](int64_t q, float (&f)[E]) {
    const int64_t first = q * E - head;
    if (q < hi && first >= 0 && first + E <= p.vocab) {
      widen(*reinterpret_cast<const uint4*>(x + first * kBytes<K>), f);
      return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t i = first + e;
      f[e] = q < hi && i >= 0 && i < p.vocab ? element<K>(x, i) : -INFINITY;
    }
  };
  for (int64_t q0 = lo; q0 < hi; q0 += U * kWave) {
    float v[U][E];
    const int64_t first = q0 * E - head;
    if (first >= 0 && q0 + U * kWave <= hi && first + U * kWave * E <= p.vocab) {
      const uint4* src = reinterpret_cast<const uint4*>(x + first * kBytes<K>) + lane;
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = src[u * kWave];
#pragma unroll
      for (int u = 0; u < U; ++u) widen(raw[u], v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) load_some(q0 + u * kWave + lane, v[u]);
    }
    float top = v[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) top = max_nan(top, v[u][e]);
    if (__any(top > m) || !(fabsf(m) < kFar)) {
      const float t = fmaxf(lane_top(top), m);
      settle();
      // the sums move to the new maximum; the old one becomes an element like others (lane 0 has it)
      const bool moves = t > m;
      if (m != -INFINITY && moves) {
        const float d = fminf(t - m, 200.0f), r = exp_neg(d);
        w = r * (w + d * s);
        s = r * s;
        if (lane == 0) {
          s += r;
          w += d * r;
        }
      }
      m = t;
      big_m = m * kLog2e;
      off = __builtin_fmaf(m, kLog2e, -big_m);
      if (!(fabsf(m) < kFar)) big_m = off = 0.0f;
      // one element that is the maximum stays out
      const uint64_t owners = moves ? __ballot(top == m) : 0;
      const float ref = m == -INFINITY ? 0.0f : m;
      bool skip = owners != 0 && lane == __ffsll(static_cast<long long>(owners)) - 1;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y = ref - v[u][e];
          float ex = exp_neg(y);
          if (skip && v[u][e] == m) {
            ex = 0.0f;
            skip = false;
          }
          s += ex;
          w += fminf(y, 200.0f) * ex;   // (e^-200 is 0: an infinite y adds nothing)
        }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float z = __builtin_fmaf(v[u][e], -kLog2e, big_m);
          const float ex = __builtin_amdgcn_exp2f(-z);
          sz += ex;
          wz += fminf(z, 300.0f) * ex;   // (likewise 2^-300)
        }
    }
    if (p.top == 0) continue;
    best = max_nan(best, top);
    if (--until == 0) {
      // the bar from the lanes' maxima so far: `top` lanes have one that reaches it, and not many
      // more; again after 1, 2, 4, ... iterations, so that an octave brings few candidates
      until = iterations += iterations;
      const uint32_t k = score_key(best);
      int n = kWave, bit;
      uint32_t t = prefix_of(~lane_max(~k), lane_max(k), bit);
      for (; bit >= 0 && n > p.top + 2; --bit) {
        const uint32_t c = t | (1u << bit);
        const int a = count(__ballot(k >= c));
        if (a >= p.top) {
          t = c;
          n = a;
        }
      }
      if (t > list.bar) {
        list.bar = t;
        list.bar_id = INT32_MAX;
      }
      bar = list.bar <= score_key(-INFINITY) ? -INFINITY : key_score(list.bar);
    }
    const uint64_t lanes = __ballot(top >= bar);
    if (lanes == 0) continue;
    int most = kEach * count(lanes);   // candidates at most, or where that is too many, as they are
    if (list.cnt + most > kList) {
      most = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) most += count(__ballot(v[u][e] >= bar));
    }
    if (first >= 0 && q0 + U * kWave <= hi && first + U * kWave * E <= p.vocab && list.cnt + most <= kList) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool has = v[u][e] >= bar;
          const uint64_t mask = __ballot(has);
          if (mask == 0) continue;
          if (has) {
            list.keys[list.cnt + below(mask)] = score_key(v[u][e]);
            list.ids[list.cnt + below(mask)] = static_cast<int>((q0 + u * kWave + lane) * E - head + e);
          }
          list.cnt += count(mask);
        }
      if (list.cnt > 2 * p.top + 32) {
        list.cut(lane, min(p.top + 8, kWave));
        bar = key_score(list.bar);
      }
    } else {
      // (all 64 lanes' element e at once; an element outside the row or run is none)
#pragma unroll 1
      for (int j = 0; j < U * E; ++j) {
        float f = v[0][0];
#pragma unroll
        for (int i = 1; i < U * E; ++i) f = i == j ? v[i / E][i % E] : f;
        if (!__any(f >= bar)) continue;
        const int64_t q = q0 + j / E * kWave + lane, i = q * E - head + j % E;
        list.add(f >= bar && q < hi && i >= 0 && i < p.vocab, score_key(f), static_cast<int>(i), lane);
        bar = list.bar <= score_key(-INFINITY) ? -INFINITY : key_score(list.bar);
      }
    }
  }
  settle();
  s = lane_total(s);
  w = lane_total(w);
  Stat t{m, s, w};
  if (p.top > 0 && s != s) {
    // a NaN or +inf: the row has no probabilities, but an order (NaN first): by keys
    list.cnt = 0;
    list.bar = 0;
    list.bar_id = INT32_MAX;
    for (int64_t q0 = lo; q0 < hi; q0 += kWave) {
      float v[E];
      load_some(q0 + lane, v);
      for (int e = 0; e < E; ++e) {
        float f = v[0];
#pragma unroll
        for (int j = 1; j < E; ++j) f = e == j ? v[j] : f;
        const int64_t i = (q0 + lane) * E - head + e;
        list.add(q0 + lane < hi && i >= 0 && i < p.vocab, score_key(f), static_cast<int>(i), lane);
      }
    }
  }
  if (list.cnt > kWave) list.cut(lane, kWave);
  join_waves(keys, ids, stats, counts, wave, lane, t, list);
  if (wave != 0) return;
  if (p.splits == 1) {
    finish(p, row, xt, t, list, lane);
    return;
  }
  float* rec = p.ws + static_cast<int64_t>(blockIdx.x) * (4 + 2 * p.top);
  wave_lds_sync();
  if (lane == 0) {
    rec[0] = t.m;
    rec[1] = t.s;
    rec[2] = t.w;
    rec[3] = __int_as_float(list.cnt);
  }
  if (lane < list.cnt) {
    rec[4 + lane] = __uint_as_float(list.keys[lane]);
    rec[4 + p.top + lane] = __int_as_float(list.ids[lane]);
  }
}

// The pieces of a row joined: wavefront i takes records i, i + 4, ...
template <int K>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(const Params p) {
  __shared__ uint32_t keys[kWaves][kList];
  __shared__ int ids[kWaves][kList];
  __shared__ Stat stats[kWaves];
  __shared__ int counts[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x;
  const float* recs = p.ws + static_cast<int64_t>(row) * p.splits * (4 + 2 * p.top);
  List list{keys[wave], ids[wave], 0, p.top, 0u, INT32_MAX};
  const float xt = wave == 0 ? token_logit<K>(p, row, p.x + static_cast<int64_t>(row) * p.stride * kBytes<K>) : 0.0f;
  Stat t{-INFINITY, 0.0f, 0.0f};   // a record a lane
  const int mine = wave + kWaves * lane;
  if (mine < p.splits) {
    const float* r = recs + static_cast<int64_t>(mine) * (4 + 2 * p.top);
    t = Stat{r[0], r[1], r[2]};
  }
  // the records' candidates as one run, three of each lane beside the best 64 so far
  const int size = 4 + 2 * p.top, all = p.splits * p.top;
  for (int e0 = 0; e0 < all; e0 += 3 * kThreads) {
    uint32_t key[4];
    int id[4], have = list.cnt;
    key[0] = lane < list.cnt ? keys[wave][lane] : 0u;
    id[0] = lane < list.cnt ? ids[wave][lane] : INT32_MAX;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const int x = e0 + (i - 1) * kThreads + static_cast<int>(threadIdx.x), e = min(x, all - 1);
      const int rec = static_cast<int>(static_cast<uint32_t>(e) / static_cast<uint32_t>(p.top)), at = e - rec * p.top;
      const float* r = recs + rec * size;
      const int entries = __float_as_int(r[3]);
      key[i] = __float_as_uint(r[4 + at]);   // (what lies behind the entries may be anything)
      id[i] = __float_as_int(r[4 + p.top + at]);
      const bool in = x < all && at < entries;
      key[i] = in ? key[i] : 0u;
      id[i] = in ? id[i] : INT32_MAX;
      have += count(__ballot(in));
    }
    list.keep_best(key, id, have, kWave);
  }
  // the lanes that have a record joined
  int lanes = 1;
  while (lanes * kWaves < p.splits) lanes <<= 1;
  for (int o = lanes >> 1; o > 0; o >>= 1)
    t = join(t, Stat{__shfl_xor(t.m, o), __shfl_xor(t.s, o), __shfl_xor(t.w, o)});
  join_waves(keys, ids, stats, counts, wave, lane, t, list);
  if (wave == 0) finish(p, row, xt, t, list, lane);
}

// Pieces of a row: rows alone fill the device from about 1024 workgroups on, and a
// piece is at least one iteration of its four wavefronts (us with 512 / 1024 / 2048 workgroups: 200 rows of
// 151936 50 / 42 / -, 400 69 / 60.5 / -, 64 33 / 32.7 / 36.2, 300 rows of 32000 29.1 / 31.7 / 32.5).
int splits_of(int rows, int vocab) {
  const int most = (vocab + 8 + kThreads * kEach - 1) / (kThreads * kEach);   // (8: up to the boundary before the row)
  return std::max(1, std::min({1024 / std::max(rows, 1), most, kMaxSplits}));
}

template <int K>
void launch(Params p, hipStream_t s) {
  // runs are whole iterations but for the row's end (which may lie a piece further than it need)
  constexpr int E = 16 / kBytes<K>, step = kEach / E * kWave;
  const int64_t pieces = (p.vocab + 2LL * (E - 1)) / E, runs = static_cast<int64_t>(p.splits) * kWaves * step;
  p.per = static_cast<int>((pieces + runs - 1) / runs * step);
  logprobs_kernel<K><<<static_cast<unsigned>(p.rows) * p.splits, kThreads, 0, s>>>(p);
  if (p.splits > 1) logprobs_join_kernel<K><<<p.rows, kThreads, 0, s>>>(p);
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int64_t nkv_token_logprobs_workspace(int rows, int vocab, int top) {
  const int s = splits_of(rows, vocab);
  return s > 1 ? static_cast<int64_t>(rows) * s * (4 + 2 * top) : 0;
}

extern "C" int nkv_token_logprobs(const void* logits, int kind, int64_t row_stride, int rows, int vocab,
                                  const int64_t* tokens, int top, float* logprob, float* entropy, float* top_logprobs,
                                  int64_t* top_ids, float* workspace, void* stream) {
  NKV_CHECK_ARG(kind >= kF32 && kind <= kF16, "nkv_token_logprobs: unknown type of logits %d", kind);
  NKV_CHECK_ARG(rows >= 0 && vocab >= 1 && vocab <= INT32_MAX - 65536,
                "nkv_token_logprobs: rows must not be negative, vocab from 1 to 2^31 - 65537");
  NKV_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= vocab,
                "nkv_token_logprobs: top must be from 0 to %d and at most vocab (got %d)", kMaxTop, top);
  if (rows == 0) return NKV_OK;
  NKV_CHECK_ARG(rows <= kMaxRows, "nkv_token_logprobs: at most 2^24 - 1 rows");
  NKV_CHECK_ARG(logits && tokens && logprob && entropy && (top == 0 || (top_logprobs && top_ids)),
                "nkv_token_logprobs: NULL input or output");
  NKV_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % (kind == kF32 ? 4 : 2) == 0 && row_stride >= 0,
                "nkv_token_logprobs: logits must be aligned to their elements");
  const int splits = splits_of(rows, vocab);
  NKV_CHECK_ARG(splits == 1 || workspace, "nkv_token_logprobs: these sizes need a workspace");
  const Params p{static_cast<const char*>(logits), row_stride, rows,    vocab,   top,          splits,  0,
                 tokens,                           logprob,    entropy, top_logprobs, top_ids, workspace};
  const auto s = static_cast<hipStream_t>(stream);
  if (kind == kF32) launch<kF32>(p, s);
  else if (kind == kBf16) launch<kBf16>(p, s);
  else launch<kF16>(p, s);
  return launch_status("nkv_token_logprobs");
}
