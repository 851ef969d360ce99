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

// The rows m0 .. m0 + rows - 1 of a sequence (row m = r * G + head of the group) and the steps that
// they see: `sink` steps from position 0 on, then the steps lo ..; `n` in all.
struct KvSpan {
  int first, last;  // positions of the first and the last row that exist; last < first: none
  int sink, lo, n;
  __device__ __forceinline__ int base(int i) const { return (i < sink ? i : lo + i - sink) << 4; }
};

__device__ __forceinline__ KvSpan kv_span(const KvAttnParams& p, const KvSeq& q, int64_t m0, int rows) {
  const int r0 = static_cast<int>(m0 / p.G);
  const int64_t r1 = min((m0 + rows - 1) / p.G, static_cast<int64_t>(p.rows.R) - 1);
  KvSpan t;
  t.first = static_cast<int>(min(static_cast<int64_t>(q.start) + r0, static_cast<int64_t>(q.len)));
  t.last = static_cast<int>(min(q.start + r1, static_cast<int64_t>(q.len) - 1));
  t.sink = t.lo = t.n = 0;
  if (t.last < t.first) return t;
  if (p.mask.window) {
    t.lo = max(0, t.first - p.mask.window + 1) >> 4;
    t.sink = min((min(p.mask.sinks, t.last + 1) + 15) >> 4, t.lo);
  }
  t.n = t.sink + (t.last >> 4) - t.lo + 1;
  return t;
}

// The blocks share the steps of all (sequence, row block, head) items evenly: the items lie one after
// another on one axis (head fastest within a (sequence, row block) pair), and block i takes the i-th
// piece of `per` steps of it.  Lengths are only known on the device, so every block adds them up itself.
struct KvShare {
  int64_t total;  // steps on the axis
  int64_t per;    // steps of a block
  int64_t off;    // of this block's first step within its pair
  int pair;       // of this block's first step
};

template <int THREADS>
__device__ __forceinline__ KvShare kv_share(const KvAttnParams& p, int row_blocks, int block_rows, int round) {
  __shared__ int64_t s_sum[THREADS / 32];
  __shared__ int64_t s_off;
  __shared__ int s_pair;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t pairs = static_cast<int64_t>(p.c.S) * row_blocks, q = (pairs + THREADS - 1) / THREADS;
  const auto steps = [&](int64_t i) -> int64_t {
    const int s = static_cast<int>(i / row_blocks);
    const int64_t m0 = (i % row_blocks) * block_rows;
    return static_cast<int64_t>(kv_span(p, kv_seq(p.c, p.rows.start, p.rows.lens, s), m0, block_rows).n) * p.c.heads;
  };
  const int64_t i0 = min(tid * q, pairs), i1 = min(i0 + q, pairs);
  int64_t mine = 0;
  for (int64_t i = i0; i < i1; ++i) mine += steps(i);
  int64_t pre = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, pre, o);
    if (lane >= o) pre += up;
  }
  if (lane == 31) s_sum[warp] = pre;
  __syncthreads();
  KvShare w{0, 0, 0, 0};
  int64_t before = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) before += s_sum[i];
    w.total += s_sum[i];
  }
  pre += before - mine;
  w.per = (w.total + gridDim.x - 1) / gridDim.x;
  w.per = max((w.per + round - 1) / round, static_cast<int64_t>(1)) * round;
  const int64_t a = blockIdx.x * w.per;
  if (mine > 0 && a >= pre && a < pre + mine) {
    int64_t i = i0, n;
    while (a >= pre + (n = steps(i))) {
      pre += n;
      ++i;
    }
    s_pair = static_cast<int>(i);
    s_off = a - pre;
  }
  __syncthreads();
  w.pair = s_pair;
  w.off = s_off;
  return w;
}

// Page and scales of 32 of a warp's steps, one a lane.
struct KvMeta {
  int page;
  float ks, vlog, vinv;
};

// The value scale enters the logits as a power of two (vlog), so that the weights of every page share
// one reference whatever its scale; a scale of 0 (a page of zeros) is taken as 2^-96.
template <bool V>
__device__ __forceinline__ KvMeta kv_meta(const KvCache& c, int s, int h, bool live, int base) {
  KvMeta m{-1, 0.f, 0.f, 0.f};
  if (!live) return m;
  m.page = kv_page(c.table, c.width, c.pages, s, base >> c.tshift);
  if (m.page < 0) return m;
  const int64_t unit = static_cast<int64_t>(m.page) * c.heads + h;
  m.ks = c.ks[unit];
  if constexpr (V) {
    const float vs = fmaxf(c.vs[unit], 0x1p-96f);
    m.vlog = log2f(vs);
    m.vinv = 1.f / vs;
  }
  return m;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Plain loads: an earlier kernel of the stream may have written the codes while this one was starting.
template <bool KEEP>
__device__ __forceinline__ uint4 ld128(const uint8_t* p) {
  uint4 v;
  if constexpr (KEEP)
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}
template <bool KEEP>
__device__ __forceinline__ uint2 ld64(const uint8_t* p) {
  uint2 v;
  if constexpr (KEEP)
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
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
__device__ __forceinline__ void kv_load_q(const KvAttnParams& p, const KvSeq& seq, int s, int h, int64_t m0, uint4* sq,
                                          float* sf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint32_t half[2][D / 64][8];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int64_t m = m0 + g + 8 * e;
    const int64_t r = m / p.G;
    const bool live = r < p.rows.R && seq.start + r < seq.len;
    uint4 raw[D / 64][2];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        raw[i][k] = make_uint4(0, 0, 0, 0);
        if (live)
          raw[i][k] = *reinterpret_cast<const uint4*>(p.q + s * p.qs + r * p.qr + (h * p.G + m % p.G) * D + 64 * i +
                                                      16 * c + 8 * k);
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

// A step's K codes: lane (g, c) holds the codes 64 i + 16 c .. + 15 of the positions g and 8 + g.
template <int D, bool KEEP>
__device__ __forceinline__ void kv_load_k(const uint8_t* k, int64_t at, uint4 (&raw)[2][D / 64]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) raw[t][i] = ld128<KEEP>(k + (at + 8 * t + g) * D + 64 * i + 16 * c);
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

}  // namespace bolt
