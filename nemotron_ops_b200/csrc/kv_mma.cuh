// What KvAttention and KvScore share: the division of the work over the blocks, and 16-token steps of
// codes as matrix-unit operands.
//
// Both read the cache in steps of 16 positions (16-position steps never straddle a page).  A step's
// codes go from global memory to the registers of one warp and become fp16 operands of
// mma.m16n8k16 there: fp16 holds every int8 and e4m3 value exactly, and a permutation of the
// contraction index, applied to both operands, lets every lane load 16 consecutive bytes.  Query rows
// are scaled by a power of two into fp16's range (their 8 significant bits fit) and the power goes
// into the row's logit factor.
#pragma once

#include "kv.cuh"

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
// another on one axis (head fastest within a (sequence, row block) pair), and each block takes a piece
// of `per` consecutive steps of it.  Where there are few items (at most a quarter of the blocks), pieces
// do not cross from one item to the next: a piece of two items costs its block a second set-up, which
// takes longer than the few steps that the last pieces of the items leave idle.  Lengths are only known
// on the device, so every block adds them up itself.
struct KvShare {
  int64_t per;   // steps of a piece
  int64_t left;  // steps of this block's piece, from here on:
  int64_t off;   // of its first step within its pair
  int64_t at;    // of its first step on the axis (pieces that cross items)
  int pair;
  bool cross;
};

template <int THREADS>
__device__ __forceinline__ KvShare kv_share(const KvAttnParams& p, int row_blocks, unsigned block_rows, int round) {
  __shared__ int64_t s_sum[THREADS / 32], s_off;
  __shared__ int s_pair;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned pairs = static_cast<unsigned>(p.c.S) * row_blocks, q = (pairs + THREADS - 1) / THREADS;
  const auto steps = [&](unsigned i) -> int {
    const unsigned s = row_blocks == 1 ? i : i / row_blocks, m0 = (i - s * row_blocks) * block_rows;
    return kv_span(p, kv_seq(p.c, p.rows.start, p.rows.lens, s), m0, block_rows).n;
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
  int64_t mine, before, total;
  scan([&](unsigned i) { return static_cast<int64_t>(steps(i)) * p.c.heads; }, mine, before, total);
  const int64_t items = static_cast<int64_t>(pairs) * p.c.heads;
  const int blocks = static_cast<int>(gridDim.x);
  KvShare w{0, 0, 0, 0, 0, items * 4 > blocks};
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
    while (w.at >= before + (n = w.cross ? static_cast<int64_t>(steps(i)) * p.c.heads : pieces_of(i))) {
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

// Page and scales of 32 of a warp's steps, one a lane.  The pages come first: the copies of the codes
// wait for them alone.
struct KvPages {
  int page;
  float ks, vlog, vinv;
};

__device__ __forceinline__ KvPages kv_pages(const KvCache& c, int s, bool live, int base) {
  return KvPages{live ? kv_page(c.table, c.width, c.pages, s, base >> c.tshift) : -1, 0.f, 0.f, 0.f};
}

// The value scale enters the logits as a power of two (vlog), so that the weights of every page share
// one reference whatever its scale; a scale of 0 (a page of zeros) is taken as 2^-96.
template <bool V>
__device__ __forceinline__ void kv_scales(const KvCache& c, int h, KvPages& m) {
  if (m.page < 0) return;
  const int64_t unit = static_cast<int64_t>(m.page) * c.heads + h;
  m.ks = c.ks[unit];
  if constexpr (V) {
    const float vs = fmaxf(c.vs[unit], 0x1p-96f);
    m.vlog = log2f(vs);
    m.vinv = 1.f / vs;
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous copies to shared memory, and plain loads: an earlier kernel of the stream may have written
// the codes while this one was starting.
__device__ __forceinline__ void cp_async16(void* dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(void* dst, const uint8_t* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 ld128(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
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

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The 16 query rows m0 .. of kv head h as A operands: lane (g, c) = (lane / 4, lane % 4) holds, for the
// contraction step 4 i + w, the values 64 i + 16 c + 4 w .. + 3 of the rows g and g + 8 -- the order
// in which a lane's 16 loaded K codes lie.  One warp writes D / 16 steps of 32 lanes to `sq` and the
// rows' logit factors (the power of two taken out, times scale * log2 e) to `sf`.  Rows that do not
// exist are 0.
template <int D>
__device__ __forceinline__ void kv_load_q(const KvAttnParams& p, const KvSeq& seq, int s, int h, unsigned m0, uint4* sq,
                                          float* sf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint32_t half[2][D / 64][8];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned m = m0 + g + 8 * e, r = m / static_cast<unsigned>(p.G);
    const bool live = r < static_cast<unsigned>(p.rows.R) && seq.start + static_cast<int>(r) < seq.len;
    const bf16* from = p.q + s * p.qs + r * p.qr + (h * static_cast<int64_t>(p.G) + (m - r * p.G)) * D + 16 * c;
    uint4 raw[D / 64][2];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        raw[i][k] = make_uint4(0, 0, 0, 0);
        if (live)
          raw[i][k] = *reinterpret_cast<const uint4*>(from + 64 * i + 8 * k);
        const uint32_t w[4] = {raw[i][k].x, raw[i][k].y, raw[i][k].z, raw[i][k].w};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xFFFF0000u))));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // 2^-x brings the largest value into [1, 2); the power is kept within fp32's normal range
    const int x = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 120);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t w[4] = {raw[i][k].x, raw[i][k].y, raw[i][k].z, raw[i][k].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const __half2 v = __floats2half2_rn(__uint_as_float(w[y] << 16) * down,
                                              __uint_as_float(w[y] & 0xFFFF0000u) * down);
          half[e][i][4 * k + y] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
    if (c == 0) sf[g + 8 * e] = __uint_as_float(static_cast<uint32_t>(127 + x) << 23) * (p.scale * kLog2e);
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      sq[(4 * i + w) * 32 + lane] =
          make_uint4(half[0][i][2 * w], half[1][i][2 * w], half[0][i][2 * w + 1], half[1][i][2 * w + 1]);
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

}  // namespace bolt
