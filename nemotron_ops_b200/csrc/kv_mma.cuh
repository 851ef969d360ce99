// What KvAttention and KvScore share: the division of the work over the blocks, and 16-token steps of
// codes as matrix-unit operands.
//
// Both read the cache in steps of 16 positions (16-position steps never straddle a page).  A step's
// codes go to the registers of one warp and become fp16 operands of mma.m16n8k16 there, with the
// positions (for logits) or the value axis (for outputs) as the 16 and the query rows as the 8: a
// sequence's rows that share a head are few, and tiles of 8 leave the least of the unit idle.  fp16
// holds every int8 and e4m3 value exactly, and a permutation of the contraction index, applied to both
// operands, lets every lane load 16 consecutive bytes.  Query rows are scaled by a power of two to the top of
// fp16's range and the power goes into the row's logit factor: a value's 8 significant bits fit down to 2^-31 of the
// row's largest, and smaller ones err by at most 2^-39 of it (of 2^-112, if that is more).
#pragma once

#include "kv.cuh"
#include "tensor_map.h"

namespace bolt {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The rows m0 .. m0 + rows - 1 of a sequence (row m = r * G + head of the group; R * G < 2^31) and the
// steps that they see: `sink` steps from position 0 on, then the steps lo ..; `n` in all.
struct KvSpan {
  int first, last;  // positions of the first and the last row that exist; last < first: none
  int sink, lo, n;
  __device__ __forceinline__ int base(int i) const { return (i < sink ? i : lo + i - sink) << 4; }
};

__device__ __forceinline__ KvSpan kv_span(const KvAttnParams& p, const KvSeq& q, unsigned m0, unsigned rows) {
  const unsigned G = p.G, most = static_cast<unsigned>(p.rows.R) - 1;
  const unsigned r0 = m0 / G, r1 = min((m0 + rows - 1) / G, most);
  KvSpan t;
  // start <= 2^30 and R <= 2^30
  t.first = min(q.start + static_cast<int>(min(r0, most + 1)), q.len);
  t.last = min(q.start + static_cast<int>(r1), q.len - 1);
  t.sink = t.lo = t.n = 0;
  if (t.last < t.first) return t;
  if (p.mask.window) {
    t.lo = max(0, t.first - p.mask.window + 1) >> 4;
    t.sink = min((min(p.mask.sinks, t.last + 1) + 15) >> 4, t.lo);
  }
  t.n = t.sink + (t.last >> 4) - t.lo + 1;
  return t;
}

// a / b of non-negative numbers; 64-bit division costs several times the 32-bit one's instructions
__device__ __forceinline__ int64_t kv_div(int64_t a, int b) {
  if (a <= 0xFFFFFFFFll) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The blocks share the steps of all (sequence, row block, head) items evenly.  The items lie one after
// another on one axis (head fastest within a (sequence, row block) pair), each behind `item_cost` units that
// stand for a block's set-up of an item, and each block takes a piece of `per` consecutive units of it.
// Where there are few items (at most a quarter of the blocks), pieces do not cross from one item to the
// next and there is nothing to level: a piece of two items costs its block a second set-up, which takes
// longer than the few steps that the last pieces of the items leave idle.  Lengths are only known on the
// device, so every block adds them up itself.
constexpr int kMostItemCost = 64;

struct KvShare {
  int64_t per;   // units of a piece
  int64_t left;  // units of this block's piece, from here on:
  int64_t off;   // of its first unit within its pair
  int64_t at;    // of its first unit on the axis (pieces that cross items)
  int pair;
  int cost;      // units in front of an item's steps: 0 where pieces do not cross items
  bool cross;
};

template <int THREADS>
__device__ __forceinline__ KvShare kv_share(const KvAttnParams& p, int row_blocks, unsigned block_rows, int round,
                                            int item_cost) {
  __shared__ int64_t s_sum[THREADS / 32], s_off;
  __shared__ int s_pair;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned pairs = static_cast<unsigned>(p.c.S) * row_blocks, q = (pairs + THREADS - 1) / THREADS;
  const auto steps = [&](unsigned i) -> int {
    const unsigned s = row_blocks == 1 ? i : i / row_blocks, m0 = (i - s * row_blocks) * block_rows;
    return kv_span(p, kv_seq(p.c, p.rows.start, p.rows.lens, s), m0, block_rows).n;
  };
  const int64_t items = static_cast<int64_t>(pairs) * p.c.heads;
  const int blocks = static_cast<int>(gridDim.x);
  KvShare w{0, 0, 0, 0, 0, 0, items * 4 > blocks};
  w.cost = w.cross ? item_cost : 0;
  const auto units = [&](unsigned i) {
    const int n = steps(i);
    return n > 0 ? n + w.cost : 0;
  };
  const unsigned i0 = min(tid * q, pairs), i1 = min(i0 + q, pairs);
  // the sum over this thread's pairs, the sum over those of the threads before it, and over all
  const auto scan = [&](auto&& of, int64_t& mine, int64_t& before, int64_t& all) {
    mine = 0;
    for (unsigned i = i0; i < i1; ++i) mine += of(i);
    int64_t pre = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += up;
    }
    __syncthreads();  // s_sum may hold another scan's
    if (lane == 31) s_sum[warp] = pre;
    __syncthreads();
    before = pre - mine;
    all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += s_sum[i];
      all += s_sum[i];
    }
  };
  if (p.few_steps && pairs <= 32) {
    // the same in each warp by itself: no barriers, 32-bit sums
    const int n = lane < static_cast<int>(pairs) ? units(lane) : 0, heads = p.c.heads;
    const int all = __reduce_add_sync(0xffffffffu, n * heads);
    if (all == 0) return w;
    const int pieces = w.cross ? blocks : blocks - static_cast<int>(items);
    const int per = ((all + pieces - 1) / pieces + round - 1) / round * round;
    const int parts = (n + per - 1) / per;  // of this lane's pair
    int pre = w.cross ? n * heads : parts * heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += up;
    }
    const int64_t at = w.cross ? static_cast<int64_t>(blockIdx.x) * per : blockIdx.x;
    const unsigned past = __ballot_sync(0xffffffffu, at < pre);
    w.per = per;
    w.at = at;
    if (past == 0) return w;
    w.pair = __ffs(past) - 1;
    const int size = __shfl_sync(0xffffffffu, n, w.pair), ps = __shfl_sync(0xffffffffu, parts, w.pair);
    const int off = static_cast<int>(at) - (__shfl_sync(0xffffffffu, pre, w.pair) - (w.cross ? size : ps) * heads);
    if (w.cross) {
      w.off = off;
      w.left = min(per, all - static_cast<int>(at));
    } else {
      const int h = off / ps, part = off - h * ps;
      w.off = static_cast<int64_t>(h) * size + part * per;
      w.left = min(per, size - part * per);
    }
    return w;
  }
  int64_t mine, before, total;
  scan([&](unsigned i) { return static_cast<int64_t>(units(i)) * p.c.heads; }, mine, before, total);
  if (total == 0) return w;
  const int pieces = w.cross ? blocks : blocks - static_cast<int>(items);  // each item may leave a piece unfilled
  w.per = kv_div(total + pieces - 1, pieces);
  w.per = kv_div(w.per + round - 1, round) * round;
  // this block's place: on the axis, or among the pieces
  w.at = w.cross ? blockIdx.x * w.per : blockIdx.x;
  const auto pieces_of = [&](unsigned i) { return kv_div(steps(i) + w.per - 1, static_cast<int>(w.per)) * p.c.heads; };
  if (!w.cross) scan([&](unsigned i) { return pieces_of(i); }, mine, before, total);
  if (w.at >= total) return w;
  if (w.at >= before && w.at < before + mine) {
    unsigned i = i0;
    int64_t n;
    while (w.at >= before + (n = w.cross ? static_cast<int64_t>(units(i)) * p.c.heads : pieces_of(i))) {
      before += n;
      ++i;
    }
    s_pair = static_cast<int>(i);
    s_off = w.at - before;
  }
  __syncthreads();
  w.pair = s_pair;
  w.off = s_off;
  if (w.cross) {
    w.left = min(w.per, total - w.at);
  } else {
    const int n = steps(w.pair), parts = static_cast<int>(kv_div(n + w.per - 1, static_cast<int>(w.per)));
    const int h = static_cast<int>(w.off) / parts, part = static_cast<int>(w.off) % parts;
    w.off = static_cast<int64_t>(h) * n + part * w.per;
    w.left = min(w.per, n - part * w.per);
  }
  return w;
}

// The segments of a block: one item's consecutive steps i0 .. i1 - 1 each.
struct KvSegment {
  int s, mb, h, pair, i0, i1;
  unsigned m0;   // the row block's first row
  int64_t end;   // on the axis, behind the item (pieces that cross items)
  KvSeq seq;
  KvSpan span;
  __device__ __forceinline__ bool whole_item() const { return i0 == 0 && i1 == span.n; }
};

struct KvWalk {
  KvShare share;
  int64_t left, off, at;
  int pair;
  __device__ __forceinline__ void start(const KvShare& w) {
    share = w;
    left = w.left;
    off = w.off;
    at = w.at;
    pair = w.pair;
  }
  __device__ __forceinline__ bool next(const KvAttnParams& p, int row_blocks, unsigned block_rows, KvSegment& t) {
    while (left > 0) {
      t.pair = pair;
      t.s = row_blocks == 1 ? pair : pair / row_blocks;
      t.mb = pair - t.s * row_blocks;
      t.m0 = static_cast<unsigned>(t.mb) * block_rows;
      t.seq = kv_seq(p.c, p.rows.start, p.rows.lens, t.s);
      t.span = kv_span(p, t.seq, t.m0, block_rows);
      if (t.span.n == 0) {
        ++pair;
        continue;
      }
      // units u0 .. u1 - 1 of the item, of which those from share.cost on are its steps
      const int size = t.span.n + share.cost;
      t.h = static_cast<int>(kv_div(off, size));
      const int u0 = static_cast<int>(off - static_cast<int64_t>(t.h) * size);
      const int u1 = static_cast<int>(min(static_cast<int64_t>(size), u0 + left));
      t.i0 = max(0, u0 - share.cost);
      t.i1 = max(0, u1 - share.cost);
      t.end = at - u0 + size;
      left -= u1 - u0;
      at += u1 - u0;
      off += u1 - u0;
      if (off == static_cast<int64_t>(size) * p.c.heads) {
        ++pair;
        off = 0;
      }
      if (t.i0 < t.i1) return true;
    }
    return false;
  }
};

// Page and scales of 32 of a warp's steps, one a lane.
struct KvPages {
  int page;
  float ks, vs;
  __device__ __forceinline__ void load_page(const KvCache& c, int s, bool live, int base) {
    // -1 stands for no page; an entry that is negative is one past every cache's last
    page = -1;
    if (live)
      page = static_cast<int>(
          min(static_cast<unsigned>(c.table[static_cast<int64_t>(s) * c.width + (base >> c.tshift)]), 0x7fffffffu));
  }
  __device__ __forceinline__ void check_page(const KvCache& c) {
    if (page >= c.pages) {
      set_status(kStatusKvPage);
      page = -1;
    }
  }
  template <bool V>
  __device__ __forceinline__ void load_scales(const KvCache& c, int h) {
    ks = vs = 0.f;
    if (page < 0) return;
    const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
    ks = c.ks[unit];
    if (V) vs = c.vs[unit];
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A step's codes lie in the ring as the tensor copy writes them: lines of 128 bytes (a position of 128
// values, or two of 64: a copy's rate goes by its lines), the 16-byte chunks of line i exchanged by XOR with
// i % 8.  Row index i of a tile of 8 positions stands for position place<D>(i): with this order the 8
// (16, for 8-byte loads) lanes of a shared-memory phase fall into different banks both when they read K
// (rows i = lane / 4) and V (rows i = 2 (lane % 4) and + 1).
template <int D>
__device__ __forceinline__ int place(int i) {
  return D == 128 ? i ^ ((i & 1) << 2) : (i & 4) | ((i & 1) << 1) | (((i >> 1) ^ i) & 1);
}

// Byte offset of byte `b` of position t < 8 of a step; position 8 + t is at kv_next_tile of it.
template <int D>
__device__ __forceinline__ int kv_at(int t, int b) {
  if (D == 128) return t * 128 + (((b >> 4) ^ t) << 4 | (b & 15));
  return (t >> 1) * 128 + ((((t & 1) * 4 + (b >> 4)) ^ (t >> 1)) << 4 | (b & 15));
}
template <int D>
__device__ __forceinline__ int kv_next_tile(int at) {
  return D == 128 ? at + 1024 : (at ^ 64) + 512;
}

// The map of a cache's codes by lines, with a box of one step; row r of the cache (of D bytes) is line r D / 128.
inline bool kv_code_map(CUtensorMap* out, const KvCache& c, const uint8_t* codes) {
  return encode_row_tile_map(out, codes, c.pages * c.heads * c.T * c.D / 128, 128, 1, 128, 16 * c.D / 128);
}

// Four codes (a word) as two fp16 pairs, exact.
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kKvInt8) {
    // a byte under the exponent of 1024 is 1024 + code
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152 = 1024 + 128
    uint32_t a = prmt(w, 0x64646464u, 0x4140u), b = prmt(w, 0x64646464u, 0x4342u);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), off), y = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// The bytes of a word of e4m3 codes that are NaN, all ones.
__device__ __forceinline__ uint32_t kv_nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// Four K codes as fp16 pairs: an int8 code's byte alone is the subnormal 2^-24 code, and its offset of 128 comes off the logit as 128 times the sum of the query row
// (kv_make_q), which costs one operation a row instead of one a pair.
template <int FMT>
__device__ __forceinline__ void k_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kKvInt8) {
    lo = prmt(w, 0, 0x4140u);
    hi = prmt(w, 0, 0x4342u);
  } else {
    codes_to_half<FMT>(w, lo, hi);
  }
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 8 query rows m0 .. of kv head h: lane (g, c) = (lane / 4, lane % 4) loads the values 64 i + 16 c ..
// + 15 of row g.  Rows that do not exist are 0.
template <int D>
__device__ __forceinline__ void kv_fetch_q(const KvAttnParams& p, const KvSeq& seq, int s, int h, unsigned m0,
                                           uint4 (&raw)[D / 64][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const unsigned m = m0 + g, r = m / static_cast<unsigned>(p.G);
  const bool live = r < static_cast<unsigned>(p.rows.R) && seq.start + static_cast<int>(r) < seq.len;
  const bf16* from = p.q + s * p.qs + r * p.qr + (h * static_cast<int64_t>(p.G) + (m - r * p.G)) * D + 16 * c;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      raw[i][k] = make_uint4(0, 0, 0, 0);
      if (live) raw[i][k] = *reinterpret_cast<const uint4*>(from + 64 * i + 8 * k);
    }
}

// ... and as B operands: for the contraction step 4 i + y the lane holds the values 64 i + 16 c + 4 y .. + 3
// of row g -- the order in which a lane's 16 loaded K codes lie.  logit / log 2 = (sum of products) * f - t,
// times the page's K scale; f and t are those of row g.  A row with a value that is not finite has a t of NaN,
// so that all its logits are.
template <int D, int FMT>
__device__ __forceinline__ void kv_make_q(const KvAttnParams& p, const uint4 (&raw)[D / 64][2], uint2 (&q)[D / 16],
                                          float& f, float& t) {
  uint32_t amax = 0;  // the largest magnitude's bits: those of infinities and NaN are the largest of all
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w[4] = {raw[i][k].x, raw[i][k].y, raw[i][k].z, raw[i][k].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) amax = max(amax, max((w[x] << 16) & 0x7FFF0000u, w[x] & 0x7FFF0000u));
    }
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  // 2^-x brings the largest value into [2^14, 2^15); the power is kept within fp32's normal range
  const int x = max(static_cast<int>(amax >> 23) - 127 - 14, -126);
  const float down = __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w[4] = {raw[i][k].x, raw[i][k].y, raw[i][k].z, raw[i][k].w};
      uint32_t u[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const __half2 v = __floats2half2_rn(__uint_as_float(w[y] << 16) * down, __uint_as_float(w[y] & 0xFFFF0000u) * down);
        sum += __low2float(v) + __high2float(v);
        u[y] = *reinterpret_cast<const uint32_t*>(&v);
      }
      q[4 * i + 2 * k] = make_uint2(u[0], u[1]);
      q[4 * i + 2 * k + 1] = make_uint2(u[2], u[3]);
    }
  f = __uint_as_float(static_cast<uint32_t>(127 + x) << 23) * (p.scale * kLog2e);
  t = 0.f;
  if constexpr (FMT == kKvInt8) {
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    t = 128.f * f * sum;
    f *= 0x1p24f;
  }
  if (amax >= 0x7F800000u) t = NAN;
}

// The same with sums that start at 0.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

}  // namespace bolt
