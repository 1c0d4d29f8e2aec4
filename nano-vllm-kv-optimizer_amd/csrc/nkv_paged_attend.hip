// Attention of every sequence's new tokens over its keys in a paged cache.
//
// Sequence b holds L keys (its page table's first L slots), the last n of them its new
// tokens'; query i of it sees the keys up to L - n + i, or with a tree the keys before
// L - n and those new ones whose bit its mask has.  o = softmax(scale q k^T) v with the
// softmax in fp32, one pass over the keys with a running maximum; a query that sees nothing gives 0.
//
// The G query heads of a KV head share its keys, so (query, head) pairs are the columns of
// one product S^T = K Q^T and O^T = V^T P^T on the matrix cores (16x16x32 bf16):
//   * few_kernel, up to 16 columns (a token, a short draft): bound by reading the keys once.
//     Every wavefront works on 32-key tiles by itself: K goes from HBM to the operand
//     registers, V through the wavefront's LDS (read back transposed), both a tile
//     ahead; P enters the second product as bf16 high and low parts, as good as fp32.
//     Measured, 32 query and 8 KV heads of 128 dims: 64 sequences of up to 8192 keys (1.2 GB)
//     195 us (6.1 TB/s); 3 of up to 131072 in 8 bits (575 MB) 100 us (5.7); one of 2048 6.5 + 4.
//   * many_kernel, tiles of 64 or 128 columns (trees, prompts): 64-key tiles staged in LDS
//     for all four wavefronts, the next one on its way; bound by the matrix cores for
//     long prompts, by the keys for trees.  P is rounded to bf16 for the second product (2^-8
//     of each weight, as the output's own rounding), in 16 bits numerator and denominator alike.
//     Measured: 4096 tokens behind 12288 791-845 us by box (1.14-1.22 PFLOP/s; of 64 dims 528 and 0.91), at
//     the chip's power limit; 7 prompts of up to 2000, 16 heads of 64 dims, 50 us (0.59: a CU may hold several of the longest tiles);
//     5 trees of 26 over up to 16384 keys (243 MB) 60 + 9 us.
// 8-bit caches: the codes are bf16 exactly; a key's scale multiplies its logits, a
// value's its weights, both in fp32.
//
// Work split, from the lengths, which are in device memory: the key tiles of all (sequence, KV
// head, query tile) units are one list, and every worker of one resident round (a wavefront of
// few_kernel, a workgroup of many_kernel) takes an equal run of it, whatever the sequences' lengths.
// A unit that several workers share is joined from their partial sums by a second
// kernel.  Query tiles that fill the device for several rounds are not cut: a workgroup each.
//
// Hidden keys get weight 0, which times an infinite or NaN value is NaN: such rows of V are zeros in LDS and
// are added to the columns that see them one by one from the cache, when a run is done a second time because it
// gave NaN (4096 tokens behind 12288, one of them NaN: 1040 us; 4 x 16384 keys 100, without 63).  In 8 bits the
// codes are finite, and the weight 0 of a scale stays 0.  Keys past the length are never read (rows are
// clamped or bounds-checked), page ids outside the cache hide their keys.
#include <algorithm>
#include <type_traits>

#include "nkv_paged.h"
#include "nkv_stage.h"

namespace nkv {
namespace {
using attend_detail::bf16x8;
using attend_detail::f32x4;
using attend_detail::i8x8_to_bf16x8;
using attend_detail::max_over_rows;
using attend_detail::sum_over_rows;
using namespace stage;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = 64;          // keys of a tile, the unit of runs
constexpr int kFewCols = 16;
constexpr int kMaxTree = 64;       // tokens of a tree: bits of a mask
constexpr float kHeadroom = 8.0f;  // a running maximum moves once a logit passes it by 2^8 (log2 units)

struct Plan {
  int few, nct, cols, tpw, qtiles;   // columns and tokens of a workgroup's tile, tiles of max_new tokens
  int workers;                       // wavefronts (few columns) or workgroups that share the list; 0: nothing is cut
};

struct Params {
  PagedCache c;
  const uint16_t* q;
  int64_t q_ls;
  uint16_t* out;
  const int32_t* tables;
  int64_t table_ls;
  int max_pages;
  const int32_t* lengths;
  const int32_t* starts;     // nullptr: n tokens each
  const uint64_t* tree;      // nullptr: in order
  int B, T, n, hq, G;
  float scale_log2;
  float* part;
  Plan plan;
};

// The arguments loaded again: what only a kernel's end or its rare paths use would
// otherwise be held in registers all along.
__device__ __forceinline__ const Params& again() {
  typedef __attribute__((address_space(4))) const Params kernarg;
  kernarg* k = (kernarg*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  return *(const Params*)k;
}

// Workspace: a note of each unit that has queries, then two records of each worker: a column's
// m, l, two floats of padding and its sums.  A unit that several workers share has
// record 2 w + 1 of the first one and 2 w of each that follows.
struct Note {
  int records, worker;   // records 1: the unit is whole
};
__host__ __device__ __forceinline__ int64_t note_floats(int64_t units) { return (2 * units + 3) & ~int64_t{3}; }
__device__ __forceinline__ Note* note_of(const Params& p, int unit) { return reinterpret_cast<Note*>(p.part) + unit; }
template <int D> constexpr int kPart = D + 4;
template <int D>
__device__ __forceinline__ float* record_of(const Params& p, int record, int c) {
  return p.part + note_floats(static_cast<int64_t>(p.B) * p.plan.qtiles * p.c.hkv) +
         (static_cast<int64_t>(record) * p.plan.cols + c) * kPart<D>;
}

typedef __attribute__((address_space(4))) const int32_t cint32;

struct Seq {
  int begin, count, len, older;   // first row of q, new tokens, keys, keys before the new tokens
};
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq s;
  int end;
  if (p.starts) {
    s.begin = min(max(((const cint32*)p.starts)[b], 0), p.T);
    end = min(max(((const cint32*)p.starts)[b + 1], s.begin), p.T);
  } else {
    s.begin = b * p.n;
    end = s.begin + p.n;
  }
  s.count = end - s.begin;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(((const cint32*)p.lengths)[b], 0)),
                               static_cast<int64_t>(p.max_pages) << p.c.shift));
  s.older = s.len - s.count;
  return s;
}

// The same for a sequence of the lane's own.
__device__ __forceinline__ Seq lane_seq(const Params& p, int b) {
  Seq s;
  int end;
  if (p.starts) {
    s.begin = min(max(p.starts[b], 0), p.T);
    end = min(max(p.starts[b + 1], s.begin), p.T);
  } else {
    s.begin = b * p.n;
    end = s.begin + p.n;
  }
  s.count = end - s.begin;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(p.lengths[b], 0)), static_cast<int64_t>(p.max_pages) << p.c.shift));
  s.older = s.len - s.count;
  return s;
}

// Keys that the queries [t0, t1] of a sequence may see: [0, this).
__device__ __forceinline__ int keys_of(const Params& p, const Seq& s, int t1) {
  return p.tree ? s.len : min(max(s.older + t1 + 1, 0), s.len);
}

// The page of the 16-key group that starts at key0 (-1: none); key0 is the same in all lanes.
__device__ __forceinline__ int page_of(const Params& p, const cint32* table, const Seq& s, int key0) {
  if (key0 >= s.len) return -1;
  const int id = table[key0 >> p.c.shift];
  return id >= 0 && id < p.c.pages ? id : -1;
}

// The keys of [key0, key0 + 64) that a query of sequence s sees, as bits: those up
// to `limit`, or with a tree the ones before its tokens and those that its mask names.
__device__ __forceinline__ uint64_t seen_bits(uint64_t mask, bool tree, int limit, const Seq& s, int key0) {
  if (tree) {
    const int at = key0 - s.older;   // the first key's place among the new tokens
    const uint64_t bits = at >= kMaxTree ? 0 : at >= 0 ? mask >> at : at <= -64 ? ~0ull : mask << -at | ((1ull << -at) - 1);
    const int rows = s.len - key0;
    return rows >= 64 ? bits : rows <= 0 ? 0 : bits & ((1ull << rows) - 1);
  }
  const int last = limit - key0;
  return last >= 63 ? ~0ull : last < 0 ? 0 : (2ull << last) - 1;
}
// x where the bit holds, else -inf.
__device__ __forceinline__ float where_bit(float x, uint32_t bits, int bit) {
  const uint32_t keep = static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - bit)) >> 31);
  return __uint_as_float((__float_as_uint(x) & keep) | (0xff800000u & ~keep));
}

// Whether one of 8 bf16 values is infinite or NaN.
__device__ __forceinline__ bool not_finite(u32x4 v) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd = odd || (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
  return odd;
}
// The bits of rows (L lanes each) that have a lane in `lanes`.
template <int L>
__device__ __forceinline__ uint32_t rows_of(uint64_t lanes) {
  uint32_t rows = 0;
#pragma unroll
  for (int r = 0; r < kWave / L; ++r) rows |= ((lanes >> (r * L)) & ((1ull << L) - 1)) != 0 ? 1u << r : 0u;
  return rows;
}
// 0, or NaN if one of the values is infinite or NaN, in four chains (comparisons would each pass a scalar register).
template <typename F>
__device__ __forceinline__ float zero_if_finite(int n, F&& at) {
  f32x4 z = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const f32x4 a = at(i);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = __builtin_fmaf(a[e], 0.0f, z[e]);
  }
  return (z[0] + z[1]) + (z[2] + z[3]);
}
// acc += w V for a row of V as it lies in the cache; acc[i][e] is dim 16 i + 4 lg + e.
template <int DT, typename F>
__device__ __forceinline__ void add_row(const char* row, int lg, float w, F&& acc) {
#pragma unroll
  for (int i = 0; i < DT; ++i) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(row + 32 * i + 8 * lg);
    f32x4& a = acc(i);
    a[0] += w * bf16_lo(v[0]);
    a[1] += w * bf16_hi(v[0]);
    a[2] += w * bf16_lo(v[1]);
    a[3] += w * bf16_hi(v[1]);
  }
}

__device__ __forceinline__ bf16x8 as_bf16(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// ---------------------------------------------------------------- few columns --
// A key or value is read by one workgroup: its line need not stay in the caches.
__device__ __forceinline__ u32x4 load_once(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// Operand layout of the 16x16x32 product: lane (ln, lg) holds A[ln][8 lg ..] and
// B[8 lg ..][ln], and of the result rows 4 lg .. + 3 of column ln.  The 32 keys of the
// second product are ordered as the first one's results lie: 4 lg + e of the
// first 16, then of the second, so P never leaves its lane.  In 8 bits a lane takes 16
// neighbouring codes of a row for two steps of the first product, and q is laid out alike.
constexpr int kFewKeys = 32;       // keys of a wavefront's tile

// Inclusive sum over the lanes of the wavefront (row shifts, then the rows' ends carried on).
__device__ __forceinline__ int lane_sums(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// Key tiles of query tile qt of a sequence: none without queries, at least one with.
__device__ __forceinline__ int key_tiles(const Params& p, const Seq& s, int qt, int keys) {
  const int count = min(s.count, p.n), t0 = qt * p.plan.tpw;
  return t0 >= count ? 0 : max(1, (keys_of(p, s, min(t0 + p.plan.tpw, count) - 1) + keys - 1) / keys);
}
// The list of all units' tiles (fewer than 2^31: the caller checked), of which the
// workers [0, active) take equal runs.
struct List {
  int total, active, share, more;   // the first `more` workers take share + 1
  __device__ __forceinline__ void split(int tiles, int workers) {
    total = tiles;
    active = min(total, workers);
    share = active == total ? 1 : static_cast<int>(static_cast<uint32_t>(total) / static_cast<uint32_t>(active));
    more = total - share * active;
  }
  __device__ __forceinline__ int lo(int w) const { return w * share + min(w, more); }
  __device__ __forceinline__ int worker_of(int x) const {
    if (share == 1 && more == 0) return x;
    const uint32_t edge = static_cast<uint32_t>(more) * (share + 1), at = x;
    return at < edge ? at / static_cast<uint32_t>(share + 1) : more + (at - edge) / static_cast<uint32_t>(share);
  }
};
// The tiles of all units of one KV head, `keys` keys each.  Unit u is query tile u % qtiles of
// sequence u / qtiles; a wavefront sums chunks of 64 units, a lane each, and goes over them once: lane
// i keeps the sum up to the end of block i (a 64th of the chunks, or one), which leaves few chunks to look
// through again for a tile's unit, however many sequences there are (a token each of 1024 / 4096 / 16384
// sequences of up to 300, 300 and 64 keys: 172 / 615 / 969 us; all chunks again for each chunk
// passed: 234 / 1629 / 18111).
struct Units {
  int chunks, per;      // chunks in all, of a block
  int ends;             // lane i: tiles up to the end of block i
  int before, inc;      // tiles before the chunk looked at, the inclusive sums of its units
  Seq mine;             // the lane's sequence there

  __device__ __forceinline__ void look(const Params& p, int keys, int lane, int c) {
    const int units = p.B * p.plan.qtiles, at = c * kWave + lane, u = min(at, units - 1);
    const int b = p.plan.qtiles == 1 ? u : static_cast<int>(static_cast<uint32_t>(u) / static_cast<uint32_t>(p.plan.qtiles));
    mine = lane_seq(p, b);
    inc = lane_sums(at < units ? key_tiles(p, mine, u - b * p.plan.qtiles, keys) : 0);
  }
  // All tiles.
  __device__ __forceinline__ int sum(const Params& p, int keys, int lane) {
    chunks = (p.B * p.plan.qtiles + kWave - 1) / kWave;
    per = (chunks + kWave - 1) / kWave;
    before = ends = 0;
    int all = 0;
    for (int c = 0, block = 0, left = per; c < chunks; ++c) {
      look(p, keys, lane, c);
      all += __builtin_amdgcn_readlane(inc, kWave - 1);
      ends = lane >= block ? all : ends;   // (those past the last block have all)
      if (--left == 0) {
        left = per;
        ++block;
      }
    }
    return all;
  }
  // The unit that holds tile x of the list in which every tile counts `each` times; -1: none (the lengths
  // have changed under the call).  `before` and `inc` are those of its chunk.
  __device__ __forceinline__ int find(const Params& p, int keys, int lane, int each, int x) {
    const uint64_t blocks = __ballot(ends * each > x);
    if (blocks == 0) return -1;
    const int block = __ffsll(static_cast<long long>(blocks)) - 1;
    before = block > 0 ? __builtin_amdgcn_readlane(ends, block - 1) : 0;
    for (int c = block * per; c < min((block + 1) * per, chunks); ++c) {
      if (chunks > 1) look(p, keys, lane, c);   // (one: as it was summed)
      const uint64_t past = __ballot((before + inc) * each > x);
      if (past != 0) return c * kWave + __ffsll(static_cast<long long>(past)) - 1;
      before += __builtin_amdgcn_readlane(inc, kWave - 1);
    }
    return -1;
  }
};

// Zeros for the rows of no sequence and those behind a sequence's max_new-th: by `waves` wavefronts,
// 16 rows at a time (4096 rows of 32 heads of 128 dims, all but one of padding, one over 2048 keys: 17 us; by
// one wavefront 830).
constexpr int kClearRows = 16;
__device__ __forceinline__ void clear_rest(const Params& p, int64_t wave, int64_t waves, int lane, int d) {
  const int64_t per = p.hq * d / 8;   // 16-byte pieces of a row
  for (int64_t r0 = wave * kClearRows; r0 < p.T; r0 += waves * kClearRows) {
    const int row = static_cast<int>(min(r0 + lane % kClearRows, static_cast<int64_t>(p.T) - 1));
    int b = -1, end = p.B + 1;        // the last sequence that starts at the row or before it (p.B: none)
    while (end - b > 1) {
      const int mid = (b + end) / 2;
      if (p.starts[mid] <= row) b = mid; else end = mid;
    }
    const bool none = b < 0 || b == p.B || row - max(p.starts[b], 0) >= p.n;
    uint32_t rows = static_cast<uint32_t>(__ballot(none && lane < kClearRows && r0 + lane < p.T));
    for (; rows != 0; rows &= rows - 1) {
      uint4* dst = reinterpret_cast<uint4*>(p.out) + (r0 + __builtin_ctz(rows)) * per;
      for (int64_t i = lane; i < per; i += kWave) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}
// Workgroups beside those that attend.
int clear_groups(const Params& p) {
  return p.starts ? std::min((p.T + kWaves * kClearRows - 1) / (kWaves * kClearRows), 256) : 0;
}

template <int D, bool INT8>
__global__ __launch_bounds__(kThreads, 2) void few_kernel(const Params args) {
  const Params& p = args;
  constexpr int KS = D / 32;                    // steps of the first product
  constexpr int DT = D / 16;                    // 16-dim tiles of the second
  constexpr int RB = 2 * D;                     // bytes of a V row in LDS
  constexpr int KL = INT8 ? D / 64 : D / 32;    // 16-byte loads of a K row's quarter
  constexpr int VR = INT8 ? 1024 / D : 512 / D; // V rows a load of the wavefront covers
  constexpr int VL = 16 / VR;                   // loads of a 16-key group
  constexpr int kBuf = kFewKeys * RB;
  constexpr int E = INT8 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kBuf];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int ln = lane & 15, lg = lane >> 4;
  const int groups = p.plan.workers / kWaves;
  if (static_cast<int>(blockIdx.x) >= groups) {   // (there are more with starts)
    clear_rest(p, (blockIdx.x - groups) * kWaves + wave, (gridDim.x - groups) * kWaves, lane, D);
    return;
  }
  const bool cut = p.part != nullptr;
  // wavefront w: the first ones of all workgroups, then the second ones (few tiles lie on all CUs)
  const int w = blockIdx.x + groups * wave;
  Units units;
  List list;
  list.split(units.sum(p, kFewKeys, lane) * p.c.hkv, p.plan.workers);
  if (w >= list.active) return;
  const int from = list.lo(w);
  // the sequence that holds the run's first tile
  int b = units.find(p, kFewKeys, lane, p.c.hkv, from);
  if (b < 0) return;
  const int at = b % kWave;
  const int before = units.before + (at > 0 ? __builtin_amdgcn_readlane(units.inc, at - 1) : 0);
  Seq s;
  s.begin = __builtin_amdgcn_readlane(units.mine.begin, at);
  s.count = __builtin_amdgcn_readlane(units.mine.count, at);
  s.len = __builtin_amdgcn_readlane(units.mine.len, at);
  s.older = s.len - s.count;
  char* buf = lds + wave * kBuf;
  // transposing read: keys 4 lg .. + 3 (+ 16 g) of dims 16 dt + ln
  int vtr[4];
#pragma unroll
  for (int x = 0; x < 4; ++x)
    vtr[x] = (4 * lg + (ln >> 2)) * RB + ((2 * (x ^ (ln >> 2)) + ((ln & 3) >> 1)) << 4) + 8 * (ln & 1);
  const int t = ln / p.G;   // column ln: query token, head of its group
  const int e0 = ln % p.G;

  int left = list.lo(w + 1) - from, done = 0;  // tiles to do, done
  int first = from - before * p.c.hkv;         // the first one's place in the sequence
  while (left > 0) {
    const Params& p = again();
    const int count = min(s.count, p.n);
    const int keys = keys_of(p, s, count - 1);
    const int per_head = max(1, (keys + kFewKeys - 1) / kFewKeys);
    const cint32* table = (const cint32*)(p.tables + b * p.table_ls);
    const bool mine = t < count;
    const int limit = mine ? s.older + t : -1;
    const bool tree = p.tree != nullptr;
    const uint64_t mask = tree && mine ? p.tree[s.begin + t] : 0;
    const int older = tree ? s.older - 1 : s.older;   // all columns see the keys up to here
    const float scale_log2 = p.scale_log2;
    for (int h = first / per_head; h < p.c.hkv && left > 0; ++h) {
      const int tile0 = first - h * per_head;       // (0 from the second pair on)
      const int ntile = min(per_head - tile0, left);
      first = (h + 1) * per_head;
      left -= ntile;
      const int lo = tile0 * kFewKeys, hi = min(lo + ntile * kFewKeys, keys);
      const int head = h * p.G + e0;
      bf16x8 bq[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 v = u32x4{0u, 0u, 0u, 0u};
        const int d0 = INT8 ? 64 * (ks >> 1) + 16 * lg + 8 * (ks & 1) : 32 * ks + 8 * lg;
        if (mine) v = *reinterpret_cast<const u32x4*>(p.q + static_cast<int64_t>(s.begin + t) * p.q_ls + head * D + d0);
        bq[ks] = __builtin_bit_cast(bf16x8, v);
      }
      u32x4 kr[2][KL], vr[2][VL];
      f32x4 ksc[2], vsc[2];
      // 16 keys of one page from key0; whether they have one (page 0 is read where not: loads
      // without branches leave the compiler nothing to merge behind them, 30 registers less)
      auto load_group = [&](int key0, u32x4 (&kd)[KL], u32x4 (&vd)[VL], f32x4& kss, f32x4& vss) {
        const int id = page_of(p, table, s, key0);
        const int page = max(id, 0);
        const int in = key0 & (p.c.page - 1);
        const int64_t base = (p.c.sp * page + p.c.sh * h + p.c.st * in) * E;
        const int last = max(s.len - 1 - key0, 0);     // rows behind it are read as it is
        const int row_bytes = static_cast<int>(p.c.st) * E;
        const char* kp = p.c.k + base + min(ln, last) * row_bytes + lg * 16;
#pragma unroll
        for (int i = 0; i < KL; ++i) kd[i] = load_once(kp + i * 64);
        constexpr int PC = 64 / VR;            // 16-byte pieces of a row
#pragma unroll
        for (int i = 0; i < VL; ++i)
          vd[i] = load_once(p.c.v + base + min(VR * i + lane / PC, last) * row_bytes + (lane % PC) * 16);
        if (INT8) {
          const int64_t at = ((static_cast<int64_t>(page) * p.c.hkv + h) << p.c.shift) + in + 4 * lg;
          kss = *reinterpret_cast<const f32x4*>(p.c.ks + at);
          vss = *reinterpret_cast<const f32x4*>(p.c.vs + at);
        }
        return id >= 0;
      };
      // a tile of 32: bit g of the result: its group g has a page
      auto load = [&](int key, u32x4 (&kd)[2][KL], u32x4 (&vd)[2][VL], f32x4 (&kss)[2], f32x4 (&vss)[2]) {
        const bool a = load_group(key, kd[0], vd[0], kss[0], vss[0]);
        const bool b = load_group(key + 16, kd[1], vd[1], kss[1], vss[1]);
        return (a ? 1 : 0) | (b ? 2 : 0);
      };
      // Zeros for the tile's rows of V that are not finite: their bits.
      auto clean = [&](u32x4 (&vd)[2][VL]) {
        constexpr int PC = 64 / VR;
        uint32_t rows = 0;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < VL; ++i) {
            const uint64_t lanes = __ballot(not_finite(vd[g][i]));
            if (lanes == 0) continue;
            const uint32_t odd = rows_of<PC>(lanes);
            if ((odd >> (lane / PC)) & 1) vd[g][i] = u32x4{0u, 0u, 0u, 0u};
            rows |= odd << (16 * g + VR * i);
          }
        return rows;
      };
      // V rows to LDS: row r at r RB, its 16-byte chunk c at position c ^ 2 (r & 3)
      auto put = [&](const u32x4 (&vd)[2][VL]) {
        constexpr int PC = 64 / VR;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < VL; ++i) {
            const int row = 16 * g + VR * i + lane / PC;
            const int c = lane % PC;
            if (INT8) {
              const u32x4 w = vd[g][i];
              *reinterpret_cast<uint4*>(buf + row * RB + (((2 * c) ^ (2 * (row & 3))) << 4)) = i8x8_to_bf16x8(w[0], w[1]);
              *reinterpret_cast<uint4*>(buf + row * RB + (((2 * c + 1) ^ (2 * (row & 3))) << 4)) = i8x8_to_bf16x8(w[2], w[3]);
            } else {
              *reinterpret_cast<u32x4*>(buf + row * RB + ((c ^ (2 * (row & 3))) << 4)) = vd[g][i];
            }
          }
      };
      f32x4 acc[DT];
      float m, l;   // the column's maximum (log2 units), the lane's part of its sum
      auto run = [&](auto care) {
        constexpr bool careful = decltype(care)::value;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = -INFINITY;
        l = 0.0f;
        int key = lo, have = 0;
        uint32_t apart = 0;             // rows of V that lie in LDS as zeros
        if (key < hi) {
          have = load(key, kr, vr, ksc, vsc);
          if (careful) apart = clean(vr);
          put(vr);
        }
        while (key < hi) {
          const int next = key + kFewKeys;
          u32x4 kn[2][KL], vn[2][VL];
          f32x4 ksn[2], vsn[2];
          int have_n = 0;
          if (next < hi) have_n = load(next, kn, vn, ksn, vsn);
          if (INT8) {
            // (an empty asm: the compiler would take the codes apart an iteration ahead, in 64 more
            // registers than there are)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int i = 0; i < KL; ++i) asm volatile("" : "+v"(kr[g][i]));
          }
          f32x4 S[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              bf16x8 a;
              if (INT8) {
                const u32x4 w = kr[g][ks >> 1];
                a = as_bf16(ks & 1 ? i8x8_to_bf16x8(w[2], w[3]) : i8x8_to_bf16x8(w[0], w[1]));
              } else {
                a = __builtin_bit_cast(bf16x8, kr[g][ks % KL]);
              }
              S[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, bq[ks], S[g], 0, 0, 0);
            }
          float y[2][4];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const f32x4 sc = ksc[g];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[g][e] = S[g][e] * (INT8 ? sc[e] * scale_log2 : scale_log2);
          }
          if (have != 3 || key + 31 > older) {
            uint64_t bits = mine ? seen_bits(mask, tree, limit, s, key) : 0;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (!((have >> g) & 1)) bits &= ~(0xffffull << (16 * g));
              const uint32_t own = static_cast<uint32_t>(bits >> (16 * g + 4 * lg));
#pragma unroll
              for (int e = 0; e < 4; ++e) y[g][e] = where_bit(y[g][e], own, e);
            }
          }
          float top = y[0][0];
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, y[g][e]);
          if (__any((top > m + kHeadroom) | ((m == -INFINITY) & (top > m)))) {
            const float mn = fmaxf(m, max_over_rows(top));
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= alpha;
          }
          const float base = m == -INFINITY ? 0.0f : m;
          bf16x8 hi8, lo8;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const f32x4 sc = vsc[g];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float w = __builtin_amdgcn_exp2f(y[g][e] - base);
              l += w;
              if (INT8) w = w == 0.0f ? 0.0f : w * sc[e];   // (the scale of a hidden key may be anything)
              const __bf16 a = static_cast<__bf16>(w);
              hi8[4 * g + e] = a;
              // (8 bits: behind a scale that is infinite the low part is finite, and so are its products with codes)
              const float rest = w - static_cast<float>(a);
              lo8[4 * g + e] = static_cast<__bf16>(INT8 ? fmaxf(rest, -1e34f) : rest);
            }
          }
          if (careful) {
            for (uint32_t todo = apart; todo != 0; todo &= todo - 1) {
              const int r = __builtin_ctz(todo);
              const int id = page_of(p, table, s, key + r);
              if (id < 0) continue;
              float w = 0.0f;   // the row's weight: in the lanes that hold keys 4 (r / 4) .. + 3 of its group
#pragma unroll
              for (int x = 0; x < 8; ++x)
                if (x == 4 * (r >> 4) + (r & 3)) w = static_cast<float>(hi8[x]) + static_cast<float>(lo8[x]);
              w = __shfl(w, 16 * ((r >> 2) & 3) + ln);
              const char* row = p.c.v + (p.c.sp * id + p.c.sh * h + p.c.st * ((key + r) & (p.c.page - 1))) * E;
              if (mine && (seen_bits(mask, tree, limit, s, key + r) & 1))
                add_row<DT>(row, lg, w, [&](int i) -> f32x4& { return acc[i]; });
            }
          }
          wave_lds_sync();
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            const char* vp = buf + vtr[i & 3] + (i >> 2) * 128;
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vp));
            const i16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vp + 16 * RB));
            const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7));
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, hi8, acc[i], 0, 0, 0);
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, lo8, acc[i], 0, 0, 0);
          }
          wave_lds_sync();
          if (next < hi) {
            if (careful) apart = clean(vn);
            if (INT8) {
              // (likewise the values' codes, right behind their loads)
#pragma unroll
              for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < VL; ++i) asm volatile("" : "+v"(vn[g][i]));
            }
            put(vn);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
#pragma unroll
              for (int i = 0; i < KL; ++i) kr[g][i] = kn[g][i];
              ksc[g] = ksn[g];
              vsc[g] = vsn[g];
            }
          }
          have = have_n;
          key = next;
        }
        l = sum_over_rows(l);
      };
      run(std::false_type{});
      if constexpr (!INT8) {
        // A sum that is not finite (l is NaN if a logit is) may be one of a value that its column does not see, or
        // of an infinite one, whose product with P's low part has any sign: again, such rows by themselves.
        const float z = zero_if_finite(DT, [&](int i) { return acc[i]; });
        if (__builtin_expect(__any((z != z) & mine & (l == l)), 0)) run(std::true_type{});
      }

      // ---- the pair's result, or this wavefront's part of it
      const Params& p = again();
      const bool whole = ntile == per_head;
      if (cut && tile0 == 0 && lane == 0)
        *note_of(p, b * p.c.hkv + h) = Note{whole ? 1 : list.worker_of(from + done + per_head - 1) - w + 1, w};
      done += ntile;
      if (ln < count * p.G) {
        if (whole) {
          uint16_t* dst = p.out + (static_cast<int64_t>(s.begin + t) * p.hq + head) * D + 4 * lg;
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int i = 0; i < DT; ++i)
            *reinterpret_cast<u32x2*>(dst + 16 * i) =
                u32x2{pack_bf16(acc[i][0] * inv, acc[i][1] * inv), pack_bf16(acc[i][2] * inv, acc[i][3] * inv)};
        } else {
          float* r = record_of<D>(p, 2 * w + (tile0 > 0 ? 0 : 1), ln);
          if (lg == 0) {
            r[0] = m;
            r[1] = l;
          }
#pragma unroll
          for (int i = 0; i < DT; ++i) *reinterpret_cast<f32x4*>(r + 4 + 16 * i + 4 * lg) = acc[i];
        }
      }
      wave_lds_sync();
    }
    first = 0;
    if (left <= 0 || b + 1 >= p.B) break;
    do s = seq_of(p, ++b); while (s.count == 0 && b + 1 < p.B);
  }
}

// --------------------------------------------------------------- many columns --
// LDS of a stage: K tile, V tile (64 rows of 2 D bytes each), in 8 bits the 64
// keys' and values' scales.  K row r's 16-byte chunk c lies at position c ^ (r mod chunks), V's
// at c ^ 2 (r & 3): the 16-byte reads of 8 keys and the transposing reads of
// 4 keys x 16 dims touch every bank once.
template <int D> constexpr int kTile = kKeys * 2 * D;
template <int D> constexpr int kStage = 2 * kTile<D> + 2 * kKeys * 4;

// The maximum that keeps a NaN (v_maximum3_f32 on pairs: no quieting of the operands first).
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Softmax state of a column: nm is minus the reference maximum (log2 units), a logit above
// thr moves it (both as before any key: 0 and -inf).
struct Col {
  float nm, thr;
};

// SHARED: the workgroups share the list; else one a unit: grid (KV head, query tile, sequence).
// (64 dims in bf16 fit three workgroups a CU, which plan_of counts on, with at most 168 registers.)
template <int D, bool INT8, int NCT, bool SHARED>
__global__ __launch_bounds__(kThreads, D == 64 && !INT8 ? 3 : 2) void many_kernel(const Params args) {
  const Params& p = args;
  constexpr int KS = D / 32, DT = D / 16, CH = D / 8, RB = 2 * D;
  constexpr int KT = INT8 && NCT > 1 ? 2 : 4;   // 16-key groups a pass: half the logits live
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage<D>];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int ln = lane & 15, lg = lane >> 4;
  const int tpw = p.plan.tpw, qtiles = p.plan.qtiles;

  // ---- the workgroup's first unit (KV head, sequence, query tile), its tile there, its run
  int h, b, qt, tile0 = 0, left = INT32_MAX, worker = 0;
  List list;
  if (!SHARED) {
    h = blockIdx.x;
    b = blockIdx.z;
    qt = qtiles - 1 - static_cast<int>(blockIdx.y);   // the longest first
    if (p.starts) {   // (the shortest units' workgroups come first here)
      const int64_t at = (static_cast<int64_t>(qt) * p.B + b) * p.c.hkv + h, all = static_cast<int64_t>(qtiles) * p.B * p.c.hkv;
      clear_rest(p, at * kWaves + wave, all * kWaves, lane, D);
    }
  } else {
    if (static_cast<int>(blockIdx.x) >= p.plan.workers) {   // (there are more with starts)
      clear_rest(p, (blockIdx.x - p.plan.workers) * kWaves + wave, (gridDim.x - p.plan.workers) * kWaves, lane, D);
      return;
    }
    // runs that follow one another on one XCD (workgroups go round them): units of a head share its keys in that L2
    const int per = p.plan.workers / 8;
    worker = p.plan.workers % 8 == 0 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
    Units units;
    const int sum = units.sum(p, kKeys, lane);
    list.split(sum * p.c.hkv, p.plan.workers);
    if (worker >= list.active) return;
    const int from = list.lo(worker);
    left = list.lo(worker + 1) - from;
    h = static_cast<int>(static_cast<uint32_t>(from) / static_cast<uint32_t>(sum));
    const int rest = from - h * sum;
    const int unit = units.find(p, kKeys, lane, 1, rest);
    if (unit < 0) return;
    const int at = unit % kWave;
    tile0 = rest - units.before - (at > 0 ? __builtin_amdgcn_readlane(units.inc, at - 1) : 0);
    b = unit / qtiles;
    qt = unit - b * qtiles;
  }

  const uint32_t lds_base = lds_address(lds);
  // operand addresses of the lane in a stage
  int koff[KS], vtr[4];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = ln * RB + (((4 * ks + lg) ^ (ln & (CH - 1))) << 4);
#pragma unroll
  for (int x = 0; x < 4; ++x)
    vtr[x] = kTile<D> + (4 * lg + (ln >> 2)) * RB + ((2 * (x ^ (ln >> 2)) + ((ln & 3) >> 1)) << 4) + 8 * (ln & 1);

  for (;;) {
    const Params& p = SHARED ? again() : args;
    const Seq s = seq_of(p, b);
    const int t0 = qt * tpw;
    const int tiles = key_tiles(p, s, qt, kKeys);
    if (!SHARED && tiles == 0) return;   // (the list has units with queries only)
    const int t_last = min(t0 + tpw, min(s.count, p.n)) - 1;
    const int lo = tile0, hi = min(tiles, left < tiles ? lo + left : tiles);
    const int32_t* table = p.tables + b * p.table_ls;
    const float sl = INT8 ? 1.0f : p.scale_log2;   // (8 bits: in the keys' scales)
    // the head's rows in a page
    constexpr int E = INT8 ? 1 : 2;
    const char* kbase = p.c.k + p.c.sh * h * E;
    const char* vbase = p.c.v + p.c.sh * h * E;
    const int row_bytes = static_cast<int>(p.c.st) * E;

    // column c = 16 NCT wave + 16 ct + ln: token t0 + c / G, head c % G
    int tcol[NCT];
    bf16x8 bq[NCT][KS];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      const int c = wave * 16 * NCT + ct * 16 + ln;
      const int t = t0 + static_cast<int>(static_cast<uint32_t>(c) / static_cast<uint32_t>(p.G));
      tcol[ct] = t;
      const uint16_t* qrow = p.q + static_cast<int64_t>(s.begin + t) * p.q_ls + (h * p.G + c - (t - t0) * p.G) * D;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 v = u32x4{0u, 0u, 0u, 0u};
        if (t <= t_last) v = *reinterpret_cast<const u32x4*>(qrow + 32 * ks + 8 * lg);
        bq[ct][ks] = __builtin_bit_cast(bf16x8, v);
      }
    }
    f32x4 acc[DT][NCT], lsum[NCT];
    Col col[NCT];

    // Staging of a tile: wavefront w brings its keys 16 w .. + 15, which lie in one page.
    // bf16 goes to LDS without registers, rows past the length (or of a page outside the
    // cache) as zeros; 8-bit codes through registers, widened on the way.
    constexpr int PC = INT8 ? D / 16 : D / 8;     // 16-byte pieces of a row in the cache
    constexpr int RL = kWave / PC;                // rows a load of the wavefront covers
    constexpr int NL = 16 / RL;                   // loads of its 16 rows
    u32x4 kreg[NL], vreg[NL];
    float sreg = 0.0f;
    // the pages of the 64 16-key groups from tile id0, one a lane (-1: none), and who has one
    int ids = -1, id0 = lo;
    uint64_t paged = 0;
    auto fetch_ids = [&](int tile) {
      const int key0 = tile * kKeys + 16 * lane;
      ids = key0 < s.len ? table[key0 >> p.c.shift] : -1;
      paged = __ballot(ids >= 0 && ids < p.c.pages);
      id0 = tile;
    };
    int have = 0;                                 // bit g: the tile's 16-key group g has a page
    auto begin_stage = [&](int tile, char* buf) {
      if (tile - id0 >= 16) fetch_ids(tile);
      const int at = (tile - id0) * 4;
      have = static_cast<int>(paged >> at) & 15;
      const int id = (have >> wave) & 1 ? __builtin_amdgcn_readlane(ids, at + wave) : 0;
      const int key0 = tile * kKeys + 16 * wave;
      const int rows = (have >> wave) & 1 ? min(16, s.len - key0) : 0;
      const int in = key0 & (p.c.page - 1);
      const int64_t row0 = p.c.sp * E * id + static_cast<int64_t>(in) * row_bytes;
      if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = RL * i + lane / PC;
          kreg[i] = vreg[i] = u32x4{0u, 0u, 0u, 0u};
          if (r < rows) {
            kreg[i] = *reinterpret_cast<const u32x4*>(kbase + row0 + static_cast<int64_t>(r) * row_bytes + (lane % PC) * 16);
            vreg[i] = *reinterpret_cast<const u32x4*>(vbase + row0 + static_cast<int64_t>(r) * row_bytes + (lane % PC) * 16);
          }
        }
        // lanes 0 .. 15 the keys' scales, 16 .. 31 the values'
        sreg = 0.0f;
        if (lane < 32 && ln < rows)
          sreg = (lane < 16 ? p.c.ks : p.c.vs)[((static_cast<int64_t>(id) * p.c.hkv + h) << p.c.shift) + in + ln];
      } else {
        const uint32_t bytes = static_cast<uint32_t>(rows) * row_bytes;
        const rsrc_words rk = rsrc_of(kbase + row0, bytes);
        const rsrc_words rv = rsrc_of(vbase + row0, bytes);
        // (made opaque: the offsets of all loads, kept from tile to tile, would not fit the registers)
        int row = lane / PC;
        asm volatile("" : "+v"(row));
        const int c = lane % PC, ko = (c ^ (row & (CH - 1))) << 4, vo = (c ^ (2 * (row & 3))) << 4;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(static_cast<int>(lds_base + (buf - lds) + 16 * wave * RB));
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int at_row = (row + RL * i) * row_bytes;
          lds_copy16(rk, dst + i * RL * RB, at_row + (ko ^ ((RL * i & (CH - 1)) << 4)));
          lds_copy16(rv, dst + i * RL * RB + kTile<D>, at_row + vo);
        }
      }
    };
    // From here on keys are hidden from some column (others that have no page are zeros).
    const int tail = max(p.tree ? s.older : s.older + t0 + 1, 0);
    auto finish_stage = [&](auto careful, int tile, char* buf) {
      if constexpr (INT8) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int r = 16 * wave + RL * i + lane / PC, c = 2 * (lane % PC);
          char* kd = buf + r * RB;
          char* vd = kd + kTile<D>;
          *reinterpret_cast<uint4*>(kd + ((c ^ (r & (CH - 1))) << 4)) = i8x8_to_bf16x8(kreg[i][0], kreg[i][1]);
          *reinterpret_cast<uint4*>(kd + (((c + 1) ^ (r & (CH - 1))) << 4)) = i8x8_to_bf16x8(kreg[i][2], kreg[i][3]);
          *reinterpret_cast<uint4*>(vd + ((c ^ (2 * (r & 3))) << 4)) = i8x8_to_bf16x8(vreg[i][0], vreg[i][1]);
          *reinterpret_cast<uint4*>(vd + (((c + 1) ^ (2 * (r & 3))) << 4)) = i8x8_to_bf16x8(vreg[i][2], vreg[i][3]);
        }
        if (lane < 32)
          reinterpret_cast<float*>(buf + 2 * kTile<D>)[(lane < 16 ? 0 : kKeys) + 16 * wave + ln] =
              lane < 16 ? sreg * p.scale_log2 : sreg;
      } else {
        __builtin_amdgcn_s_waitcnt(0);   // the copies have landed
        if (decltype(careful)::value && tile * kKeys + kKeys > tail) {
          // zeros for the wavefront's rows of V that are not finite; their bits lie behind the tiles
          asm volatile("" ::: "memory");   // (no read above the wait)
          char* vd = buf + kTile<D> + 16 * wave * RB + lane * 16;
          uint32_t rows = 0;
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            u32x4* piece = reinterpret_cast<u32x4*>(vd + i * RL * RB);
            const uint64_t lanes = __ballot(not_finite(*piece));
            if (lanes == 0) continue;
            const uint32_t odd = rows_of<PC>(lanes);
            if ((odd >> (lane / PC)) & 1) *piece = u32x4{0u, 0u, 0u, 0u};
            rows |= odd << (RL * i);
          }
          if (lane == 0) reinterpret_cast<uint32_t*>(buf + 2 * kTile<D>)[wave] = rows;
        }
      }
      __syncthreads();
    };

    // One tile in `buf`.  Operand reads run two products ahead through a ring of three
    // registers; the scheduling barriers keep that order.  The priority takes one of a SIMD's
    // wavefronts through its products, so that the others' softmax falls beside them (4096 tokens behind
    // 12288: 871 us without, 823 with it).
    auto attend = [&](auto careful, int tile, int got, const char* buf) {
      const float* scales = reinterpret_cast<const float*>(buf + 2 * kTile<D>);
      const bool hidden = tile * kKeys + kKeys > tail, mask = got != 15 || hidden;
#pragma unroll
      for (int pass = 0; pass < 4 / KT; ++pass) {
        constexpr int kQ = KS * KT;
        auto read_k = [&](int i) {   // ks outer, kt inner
          return *reinterpret_cast<const bf16x8*>(buf + (pass * KT + i % KT) * 16 * RB + koff[i / KT]);
        };
        auto read_v = [&](int i) {   // 32-key group outer, 16 dims inner
          const char* vp = buf + vtr[(i % DT) & 3] + ((i % DT) >> 2) * 128 + (pass * (KT / 2) + i / DT) * 32 * RB;
          const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vp));
          const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(vp + 16 * RB));
          return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // ---- S^T = K Q^T: S[kt][ct][e] is key 16 kt + 4 lg + e of the pass, column ct
        __builtin_amdgcn_s_setprio(1);
        f32x4 S[KT][NCT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) S[kt][ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        bf16x8 ka[3];
        ka[0] = read_k(0);
        ka[1] = read_k(1);
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
          if (i + 2 < kQ) ka[(i + 2) % 3] = read_k(i + 2);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
            S[i % KT][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[i % 3], bq[ct][i / KT], S[i % KT][ct], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        // the first values load while the softmax runs
        constexpr int kV = DT * (KT / 2);
        bf16x8 va[3];
        va[0] = read_v(0);
        va[1] = read_v(1);
        __builtin_amdgcn_sched_barrier(0);
        if (INT8) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const f32x4 sc = *reinterpret_cast<const f32x4*>(scales + 16 * (pass * KT + kt) + 4 * lg);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) S[kt][ct] *= sc;
          }
        }
        if (mask) {
          const Params& p = again();
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            const bool mine = tcol[ct] <= t_last;
            const uint64_t names = p.tree && mine ? p.tree[s.begin + tcol[ct]] : 0;
            uint64_t bits = seen_bits(names, p.tree != nullptr, mine ? s.older + tcol[ct] : -1, s, tile * kKeys);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
              const int g = pass * KT + kt;
              if (!((got >> g) & 1)) bits &= ~(0xffffull << (16 * g));
              const uint32_t own = static_cast<uint32_t>(bits >> (16 * g + 4 * lg));
#pragma unroll
              for (int e = 0; e < 4; ++e) S[kt][ct][e] = where_bit(S[kt][ct][e], own, e);
            }
          }
        }
        __builtin_amdgcn_s_setprio(0);
        // ---- softmax: a maximum moves only where a logit passes it by 2^8
        float top[NCT];
        bool move = false;
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          top[ct] = S[0][ct][0];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[ct] = max_nan(top[ct], S[kt][ct][e]);
          move = move || top[ct] > col[ct].thr;
        }
        if (__any(move)) {
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            const float old = col[ct].thr == -INFINITY ? -INFINITY : -col[ct].nm;
            const float cand = max_over_rows(top[ct]) * sl;
            const float m = cand > old + kHeadroom ? cand : old;
            const float ref = m == -INFINITY ? 0.0f : m;
            const float alpha = old == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(old - ref);
            col[ct].nm = -ref;
            col[ct].thr = m == -INFINITY ? -INFINITY : (m + kHeadroom) / sl;
            lsum[ct] *= alpha;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i][ct] *= alpha;
          }
        }
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              S[kt][ct][e] = __builtin_amdgcn_exp2f(INT8 ? S[kt][ct][e] + col[ct].nm : __builtin_fmaf(S[kt][ct][e], sl, col[ct].nm));
        if (INT8) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const f32x4 sc = *reinterpret_cast<const f32x4*>(scales + kKeys + 16 * (pass * KT + kt) + 4 * lg);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              lsum[ct] += S[kt][ct];
              // (the scale of a hidden key may be anything)
#pragma unroll
              for (int e = 0; e < 4; ++e) S[kt][ct][e] = S[kt][ct][e] == 0.0f ? 0.0f : S[kt][ct][e] * sc[e];
            }
          }
        }
        if (decltype(careful)::value && hidden) {
          const uint32_t* bits = reinterpret_cast<const uint32_t*>(buf + 2 * kTile<D>);
#pragma unroll 1
          for (int kt = 0; kt < 4; ++kt) {
            uint32_t todo = __builtin_amdgcn_readfirstlane(static_cast<int>(bits[kt]));
#pragma unroll 1
            for (; todo != 0; todo &= todo - 1) {
              const int r = __builtin_ctz(todo), key = tile * kKeys + 16 * kt + r;
              const Params& p = again();
              const int id = page_of(p, (const cint32*)(p.tables + b * p.table_ls), s, key);   // (it has one)
              const char* row = p.c.v + (p.c.sp * max(id, 0) + p.c.sh * h + p.c.st * (key & (p.c.page - 1))) * E;
#pragma unroll
              for (int ct = 0; ct < NCT; ++ct) {
                float w = 0.0f;   // the row's weight: in the lanes that hold keys 4 (r / 4) .. + 3 of the group
#pragma unroll
                for (int x = 0; x < 4 * KT; ++x)
                  if (x == 4 * kt + (r & 3)) w = S[x >> 2][ct][x & 3];
                w = __shfl(w, 16 * (r >> 2) + ln);
                const bool mine = tcol[ct] <= t_last;
                const uint64_t names = p.tree && mine ? p.tree[s.begin + tcol[ct]] : 0;
                if (mine && (seen_bits(names, p.tree != nullptr, s.older + tcol[ct], s, key) & 1))
                  add_row<DT>(row, lg, w, [&](int i) -> f32x4& { return acc[i][ct]; });
              }
            }
          }
        }
        // ---- O^T += V^T P^T, the row sums a product with ones
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const int j = i / DT, dt = i % DT;
          if (dt == 0) __builtin_amdgcn_sched_barrier(0);
          bf16x8 bp[NCT];
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            const f32x4 a0 = S[2 * j][ct], a1 = S[2 * j + 1][ct];
            const u32x4 w = u32x4{pack_bf16(a0[0], a0[1]), pack_bf16(a0[2], a0[3]), pack_bf16(a1[0], a1[1]), pack_bf16(a1[2], a1[3])};
            bp[ct] = __builtin_bit_cast(bf16x8, w);
            if (!INT8 && dt == 0) {
              const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
              lsum[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, bp[ct], lsum[ct], 0, 0, 0);
            }
          }
          if (i + 2 < kV) va[(i + 2) % 3] = read_v(i + 2);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
            acc[dt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[i % 3], bp[ct], acc[dt][ct], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    };

    auto run = [&](auto careful) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i][ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        lsum[ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        col[ct] = Col{0.0f, -INFINITY};
      }
      fetch_ids(lo);
      begin_stage(lo, lds);
      finish_stage(careful, lo, lds);
      for (int tile = lo; tile < hi; ++tile) {
        char* buf = lds + ((tile - lo) & 1) * kStage<D>;
        char* other = lds + ((tile - lo + 1) & 1) * kStage<D>;
        const int got = have;
        if (tile + 1 < hi) begin_stage(tile + 1, other);
        attend(careful, tile, got, buf);
        if (tile + 1 < hi) finish_stage(careful, tile + 1, other);
      }
    };
    run(std::false_type{});
    if (!INT8 && hi * kKeys > tail) {
      // A sum that is not finite may be one of a value that its column does not see.
      bool odd = false;
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        const float z = zero_if_finite(DT, [&](int i) { return acc[i][ct]; });
        odd |= (z != z) & (tcol[ct] <= t_last);
      }
      int* flags = reinterpret_cast<int*>(lds + 2 * kTile<D>) + kWaves;
      const bool any = __any(odd);
      if (lane == 0) flags[wave] = any;
      __syncthreads();
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]), 0)) {
        // the values in question (all wavefronts look through all of them)
        bool found = false;
        for (int key0 = max(tail, lo * kKeys) & -16; key0 < min(hi * kKeys, s.len) && !found; key0 += 16) {
          const int id = page_of(p, (const cint32*)table, s, key0);
          if (id < 0) continue;
          const int in = key0 & (p.c.page - 1);
#pragma unroll
          for (int i = 0; i < NL; ++i) {
            const int r = RL * i + lane / PC;
            if (key0 + r < s.len)
              found = found || not_finite(*reinterpret_cast<const u32x4*>(
                                   vbase + p.c.sp * E * id + static_cast<int64_t>(in + r) * row_bytes + (lane % PC) * 16));
          }
          found = __any(found);
        }
        __syncthreads();   // (the flags have been read)
        if (found) run(std::true_type{});
      }
    }

    // ---- store: acc[i][ct][e] is dim 16 i + 4 lg + e
    const bool whole = hi - lo == tiles;
    const Params& late = again();
    if (SHARED && lo == 0 && threadIdx.x == 0)   // (one that is cut is the run's last)
      *note_of(late, (h * late.B + b) * qtiles + qt) =
          Note{whole ? 1 : list.worker_of(list.lo(worker + 1) - hi + tiles - 1) - worker + 1, worker};
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      const int c0 = wave * 16 * NCT + ct * 16;
      const int c = c0 + ln;
      const bool mine = tcol[ct] <= t_last;
      const float l = INT8 ? sum_over_rows(lsum[ct][0] + lsum[ct][1] + lsum[ct][2] + lsum[ct][3]) : lsum[ct][0];
      if (!mine) continue;
      if (!SHARED || whole) {
        const int head = h * late.G + c - (tcol[ct] - t0) * late.G;
        uint16_t* dst = late.out + (static_cast<int64_t>(s.begin + tcol[ct]) * late.hq + head) * D + 4 * lg;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          const f32x4 o = acc[i][ct];
          *reinterpret_cast<u32x2*>(dst + 16 * i) = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
        }
      } else {
        float* r = record_of<D>(late, 2 * worker + (lo > 0 ? 0 : 1), c);
        if (lg == 0) {
          r[0] = col[ct].thr == -INFINITY ? -INFINITY : -col[ct].nm;
          r[1] = l;
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) *reinterpret_cast<f32x4*>(r + 4 + 16 * i + 4 * lg) = acc[i][ct];
      }
    }
    left -= hi - lo;
    if (!SHARED || left <= 0) return;
    // ---- the next unit of the list
    tile0 = 0;
    if (++qt * tpw >= min(s.count, late.n)) {
      qt = 0;
      do {
        if (++b == late.B) {
          b = 0;
          if (++h == late.c.hkv) return;   // (as in few_kernel)
        }
      } while (seq_of(late, b).count == 0);   // (there is a unit: the run goes on)
    }
    __syncthreads();   // (the stages have been read)
  }
}

// ----------------------------------------------------------------- the join --
// A wavefront a column of a unit that is cut, or with WIDE (few columns, which may be cut
// into many runs) a workgroup: D / 4 lanes a record, 8 records of each such group
// of lanes in flight.  Bound by the launch and three round trips, or by reading the records once
// (4 us behind one token over 2048 keys, 9 behind 5 trees: 28 MB of records).
template <int D, bool WIDE>
__global__ __launch_bounds__(kThreads) void merge_kernel(const Params p) {
  constexpr int L = D / 4, N = (WIDE ? kThreads : kWave) / L;
  const int lane = WIDE ? threadIdx.x : threadIdx.x & 63;
  const int unit = blockIdx.x, col = WIDE ? blockIdx.y : blockIdx.y * kWaves + static_cast<int>(threadIdx.x >> 6);
  int h, u;
  if (WIDE) {   // (the list of few columns goes sequence by sequence)
    u = unit / p.c.hkv;
    h = unit - u * p.c.hkv;
  } else {
    h = unit / (p.B * p.plan.qtiles);
    u = unit - h * p.B * p.plan.qtiles;
  }
  const Note note = *note_of(p, unit);
  const Seq s = seq_of(p, u / p.plan.qtiles);
  const int t0 = u % p.plan.qtiles * p.plan.tpw;
  // (a unit without queries has no note; one that points past the records was never written: the lengths
  // have changed under the call)
  if (col >= (min(s.count, min(t0 + p.plan.tpw, p.n)) - t0) * p.G || note.records <= 1 || note.worker < 0 ||
      note.records > p.plan.workers - note.worker)
    return;
  const int slot = lane / L, j = lane % L;
  float m = -INFINITY, l = 0.0f;
  f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 8;
  for (int i0 = slot; i0 - slot < note.records; i0 += U * N) {
    float mi[U], li[U];
    f32x4 a[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = min(i0 + k * N, note.records - 1);
      const float* r = record_of<D>(p, 2 * (note.worker + i) + (i == 0 ? 1 : 0), col);
      mi[k] = r[0];
      li[k] = r[1];
      a[k] = *reinterpret_cast<const f32x4*>(r + 4 + 4 * j);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < U; ++k) mn = fmaxf(mn, mi[k]);
    const float old = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= old;
    o *= old;
    m = mn;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      // (one that saw nothing, or one past the last, read again: nothing)
      const bool none = i0 + k * N >= note.records || (mi[k] == -INFINITY && li[k] == 0.0f);
      const float wt = __builtin_amdgcn_exp2f(mi[k] - mn);
      l += none ? 0.0f : li[k] * wt;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += none ? 0.0f : a[k][e] * wt;
    }
  }
  __shared__ float sm[kWaves], sl[kWaves];
  __shared__ f32x4 so[kWaves][L];
#pragma unroll
  for (int x = L; x < kWave; x <<= 1) {
    const float mo = __shfl_xor(m, x), lo = __shfl_xor(l, x);
    const float mn = fmaxf(m, mo);
    const float wa = m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float wb = mo == -INFINITY && lo == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mo - mn);
    l = l * wa + lo * wb;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * wa + __shfl_xor(o[e], x) * wb;
    m = mn;
  }
  if (WIDE) {
    if (lane % kWave < L) {
      sm[lane / kWave] = m;
      sl[lane / kWave] = l;
      so[lane / kWave][j] = o;
    }
    __syncthreads();
    if (slot != 0) return;
    m = -INFINITY;
    l = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = fmaxf(m, sm[i]);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float wt = sm[i] == -INFINITY && sl[i] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(sm[i] - m);
      l += sl[i] * wt;
      o += so[i][j] * wt;
    }
  }
  if (slot != 0) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const uint32_t t = static_cast<uint32_t>(col) / static_cast<uint32_t>(p.G);
  uint16_t* dst = p.out + (static_cast<int64_t>(s.begin + t0 + t) * p.hq + h * p.G + col - t * p.G) * D + 4 * j;
  *reinterpret_cast<u32x2*>(dst) = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
}

// ----------------------------------------------------------------- the plan --
Plan plan_of(int B, int T, int n, int hkv, int G, int head_dim, bool int8, int64_t cap_tokens, bool ragged) {
  Plan q{};
  const int64_t rows = static_cast<int64_t>(n) * G;
  const int cus = std::max(1, device_cus());
  q.few = rows <= kFewCols;
  if (q.few) {
    q.cols = static_cast<int>(rows);
    q.tpw = n;
    q.qtiles = 1;
    // Workgroups a CU by the bytes of a row, which a tile's loads in flight go by (us with 1 / 2 / 3: 256 bytes,
    // 64 x 8192 keys 195 / 201 / 208, 32768 38.7 / 40.8 / 47.5; 128 bytes, int8 3 x 131072 146 / 111 / 127,
    // bf16 64 x 8192 122 / 107 / 112; 64 bytes, 64 x 8192 131 / 87 / 79)
    const int row_bytes = int8 ? head_dim : 2 * head_dim;
    const int groups = row_bytes == 256 ? 1 : row_bytes == 128 ? 2 : 3;
    q.workers = cap_tokens > kFewKeys ? groups * kWaves * cus : 0;
    return q;
  }
  q.nct = rows <= 64 ? 1 : 2;
  q.cols = 64 * q.nct;
  q.tpw = q.cols / G;
  q.qtiles = (n + q.tpw - 1) / q.tpw;
  // A workgroup a unit takes as long as the longest unit; shared, the units take their mean
  // share of the slots, and about 32 tiles' time more for records of 64 KiB, written and
  // read (us, a workgroup a unit / shared: 500 tokens 21 / 37, 2000 56 / 97, 1000 behind 8192
  // 187 / 176, 2 x 947 behind 9882 217 / 137, 200 behind 32768 638 / 151)
  const int slots = (head_dim == 128 ? 2 : 3) * cus;   // workgroups that the CUs hold
  const int64_t cap = (cap_tokens + kKeys - 1) / kKeys;
  const int64_t units = std::max<int64_t>(ragged ? 1 : B, (static_cast<int64_t>(T) + q.tpw - 1) / q.tpw) * hkv;   // at least
  const bool fits = static_cast<int64_t>(B) * q.qtiles <= 1024 && hkv <= 1024 && cap * B * q.qtiles * hkv <= INT32_MAX;
  q.workers = fits && units < slots && cap * (slots - units) > 32 * static_cast<int64_t>(slots) ? slots : 0;
  return q;
}

template <int D, bool I8, int NCT>
void launch_many(const Params& p, hipStream_t s) {
  const Plan& q = p.plan;
  if (q.workers > 0)
    many_kernel<D, I8, NCT, true><<<q.workers + clear_groups(p), kThreads, 0, s>>>(p);
  else
    many_kernel<D, I8, NCT, false><<<dim3(p.c.hkv, q.qtiles, p.B), kThreads, 0, s>>>(p);
}

template <int D, bool I8>
void launch(const Params& p, hipStream_t s) {
  const Plan& q = p.plan;
  if (q.few) {
    // (where no pair has two tiles a wavefront takes some of them)
    Params f = p;
    if (q.workers == 0) f.part = nullptr;
    if (q.workers == 0)
      f.plan.workers = kWaves * static_cast<int>(std::min<int64_t>((static_cast<int64_t>(p.B) * p.c.hkv + kWaves - 1) / kWaves, 4096));
    few_kernel<D, I8><<<f.plan.workers / kWaves + clear_groups(p), kThreads, 0, s>>>(f);
  } else {
    q.nct == 1 ? launch_many<D, I8, 1>(p, s) : launch_many<D, I8, 2>(p, s);
  }
  if (q.workers == 0) return;
  const unsigned units = static_cast<unsigned>(p.B) * q.qtiles * p.c.hkv;
  if (q.few)
    merge_kernel<D, true><<<dim3(units, q.cols), kThreads, 0, s>>>(p);
  else
    merge_kernel<D, false><<<dim3(units, q.cols / kWaves), kThreads, 0, s>>>(p);
}

// Floats of the workspace: the notes and two records a worker.
int64_t part_floats(const Plan& q, int B, int hkv, int head_dim) {
  if (q.workers == 0) return 0;
  return note_floats(static_cast<int64_t>(B) * q.qtiles * hkv) + 2 * static_cast<int64_t>(q.workers) * q.cols * (head_dim + 4);
}

int check_sizes(const char* who, int batch, int rows, int max_new, int num_heads, int num_kv_heads, int max_pages,
                int page_size) {
  NKV_CHECK_ARG(batch >= 0 && batch <= 65535, "%s: from 0 to 65535 sequences (got %d)", who, batch);
  NKV_CHECK_ARG(rows >= 0 && max_new >= 1 && max_new <= (1 << 20), "%s: max_new must be from 1 to 2^20 (got %d)", who, max_new);
  NKV_CHECK_ARG(num_kv_heads >= 1 && num_heads >= num_kv_heads && num_heads % num_kv_heads == 0 && num_kv_heads <= 65535,
                "%s: num_heads (%d) must be a positive multiple of num_kv_heads (%d)", who, num_heads, num_kv_heads);
  NKV_CHECK_SUPPORTED(num_heads / num_kv_heads <= 64, "%s: at most 64 query heads a KV head", who);
  // (a launch has fewer than 2^32 threads)
  NKV_CHECK_ARG(static_cast<int64_t>(batch) * num_kv_heads < 1 << 24, "%s: fewer than 2^24 pairs of a sequence and a KV head", who);
  NKV_CHECK_ARG(max_pages >= 1 && static_cast<int64_t>(max_pages) * page_size <= INT32_MAX - 4096,
                "%s: a page table covers from 1 page to 2^31 - 4097 tokens", who);
  const int64_t tiles = (static_cast<int64_t>(max_pages) * page_size / kFewKeys + 1) * num_kv_heads;
  NKV_CHECK_ARG(tiles * std::max(batch, 1) <= INT32_MAX,
                "%s: the page tables cover 2^31 pieces of 32 keys of a KV head or more", who);
  return NKV_OK;
}

}  // namespace
}  // namespace nkv

using namespace nkv;

extern "C" int64_t nkv_paged_attend_workspace(int batch, int rows, int max_new, int num_heads, int num_kv_heads,
                                              int head_dim, int max_pages, int page_size, int ragged) {
  if (batch <= 0 || rows <= 0 || check_sizes("", batch, rows, max_new, num_heads, num_kv_heads, max_pages, page_size)) return 0;
  // (an 8-bit cache has as many workers as one of bf16, or more)
  const Plan q = plan_of(batch, rows, max_new, num_kv_heads, num_heads / num_kv_heads, head_dim, true,
                         static_cast<int64_t>(max_pages) * page_size, ragged != 0);
  return part_floats(q, batch, num_kv_heads, head_dim);
}

extern "C" int nkv_paged_attend(void* k, void* v, float* k_scale, float* v_scale, int64_t page_stride,
                                int64_t head_stride, int64_t token_stride, int pages, int num_kv_heads, int page_size,
                                int head_dim, const uint16_t* q, int64_t q_stride, int rows, int num_heads,
                                const int32_t* tables, int64_t table_stride, int max_pages, const int32_t* lengths,
                                int batch, const int32_t* starts, int max_new, const int64_t* tree, float scale,
                                uint16_t* out, float* workspace, void* stream) {
  const char* who = "nkv_paged_attend";
  Params p{};
  if (int rc = fill_paged(who, k, v, k_scale, v_scale, page_stride, head_stride, token_stride, pages, num_kv_heads,
                          page_size, head_dim, &p.c))
    return rc;
  if (int rc = check_sizes(who, batch, rows, max_new, num_heads, num_kv_heads, max_pages, page_size)) return rc;
  NKV_CHECK_ARG(starts != nullptr || static_cast<int64_t>(batch) * max_new == rows,
                "%s: without starts every sequence has max_new rows", who);
  NKV_CHECK_ARG(tree == nullptr || max_new <= kMaxTree, "%s: a tree has at most %d tokens (got %d)", who, kMaxTree, max_new);
  NKV_CHECK_ARG(scale > 0.0f && scale < INFINITY, "%s: scale must be positive and finite", who);
  if (rows == 0) return NKV_OK;
  NKV_CHECK_ARG(batch >= 1, "%s: rows need a sequence", who);
  NKV_CHECK_ARG(q && out && tables && lengths, "%s: q, out, tables and lengths must be non-NULL", who);
  NKV_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 && q_stride % 8 == 0,
                "%s: rows must lie on 16-byte boundaries", who);
  const int G = num_heads / num_kv_heads;
  p.plan = plan_of(batch, rows, max_new, num_kv_heads, G, head_dim, k_scale != nullptr,
                   static_cast<int64_t>(max_pages) * page_size, starts != nullptr);
  NKV_CHECK_ARG(p.plan.qtiles <= 65535, "%s: at most 65535 query tiles of a sequence (max_new is %d)", who, max_new);
  NKV_CHECK_ARG(part_floats(p.plan, batch, num_kv_heads, head_dim) == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "%s: these sizes need a workspace on a 16-byte boundary", who);
  p.q = q;
  p.q_ls = q_stride;
  p.out = out;
  p.tables = tables;
  p.table_ls = table_stride;
  p.max_pages = max_pages;
  p.lengths = lengths;
  p.starts = starts;
  p.tree = reinterpret_cast<const uint64_t*>(tree);
  p.B = batch;
  p.T = rows;
  p.n = max_new;
  p.hq = num_heads;
  p.G = G;
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.part = workspace;
  const auto s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    k_scale ? launch<128, true>(p, s) : launch<128, false>(p, s);
  else
    k_scale ? launch<64, true>(p, s) : launch<64, false>(p, s);
  return launch_status(who);
}
