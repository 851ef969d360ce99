// KvAttention over the paged 8-bit key/value cache (layout in kv.h).
//
//   l_j = scale * q . k_j over the positions j that the row sees;  lse = log sum_j exp(l_j)
//   o = sum_j exp(l_j - lse) v_j (bf16) and lse (f32); a row that sees nothing gives 0 and -inf
//
// One pass with the running maximum and sum of a softmax (kv_mma.cuh has the operands).  The rows of a
// sequence that read one kv head -- R rows times G query heads -- are the M axis of the products, so
// the codes are read once for all of them.  A block holds MW x MR tiles of 16 rows and splits their
// steps over TW warps; the blocks share all steps evenly (kv_share), a segment being one
// (sequence, row block, head)'s consecutive steps in one block.  At its end the TW partial results
// are joined through shared memory.  A segment that is a whole item writes the result; the others
// leave (max, sum, values) in the workspace for kv_combine_kernel, which joins them in block order, so
// results do not depend on scheduling.
//
// Rounding: logits, maxima, sums and values are fp32; a weight is rounded to fp16 (11 bits) once, as
// the second product's operand.  Weights are kept as 2^15 times their share of the row's largest, so
// that those down to 2^-29 of it have all 11 bits.
#include "kv_mma.cuh"

namespace bolt {

namespace {

constexpr float kWeightLog = 15.f;

struct Split {   // segments of one item: the first in block `block`'s slot 2 block + 1, the i-th in 2 (block + i)
  int s, mb, h, block, parts;
};

struct Work {
  float* part;    // [2 blocks][rows of a block][D]
  float2* ml;     // [2 blocks][rows of a block]: max and sum
  Split* split;   // [splits]
  int splits;     // min(items, blocks): an entry an item, or an entry a block
  int row_blocks;
};

template <int D, int MR, int MW, int TW, int STAGES>
struct Tile {
  static constexpr int kRows = MR * MW * 16, kThreads = MW * TW * 32;
  static constexpr int kQ = MR * MW * (D / 16) * 32;      // uint4 of query operands
  static constexpr int kStep = D * 2;                     // uint4 of a warp's step: 16 positions, K and V
  static constexpr int kRing = MW * TW * STAGES * kStep;  // uint4
  static constexpr int kJoin = TW * kRows * D / 4;        // uint4, in the ring's place
  static constexpr size_t kSmem = (kQ + (kRing > kJoin ? kRing : kJoin)) * 16 + kRows * 4 + TW * kRows * 8;
};

// float4 index f of a row's values in the joining buffer, spread over the banks
template <int D>
__device__ __forceinline__ int swizzle(int row, int f) {
  return f ^ ((f >> 3) | ((row & 1) << (D == 128 ? 2 : 1)));
}

// A warp's step in its ring: every lane copies the bytes that it will use itself, so that no other
// lane waits for them.  K: lane (g, c) takes the codes 64 i + 16 c .. + 15 of the positions g and 8 + g.
// V: the codes (D / 8) g .. of the positions 2 c, 2 c + 1, 8 + 2 c and 8 + 2 c + 1.
template <int D>
__device__ __forceinline__ void copy_step(uint4* to, const uint8_t* k, const uint8_t* v) {
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) cp_async16(to + (t * (D / 64) + i) * 32 + lane, k + (8 * t + g) * D + 64 * i + 16 * c);
  to += D / 32 * 32;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* from = v + ((i >> 1) * 8 + 2 * c + (i & 1)) * D + D / 8 * g;
    if constexpr (D == 128)
      cp_async16(to + i * 32 + lane, from);
    else
      cp_async8(reinterpret_cast<uint2*>(to) + i * 32 + lane, from);
  }
}

template <int D>
struct VCodes {
  uint32_t w[4][D / 32];  // position, word
  __device__ __forceinline__ void load(const uint4* from) {
    const int lane = threadIdx.x & 31;
    from += D / 32 * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (D == 128) {
        const uint4 x = from[i * 32 + lane];
        w[i][0] = x.x;
        w[i][1] = x.y;
        w[i][2] = x.z;
        w[i][3] = x.w;
      } else {
        const uint2 x = reinterpret_cast<const uint2*>(from)[i * 32 + lane];
        w[i][0] = x.x;
        w[i][1] = x.y;
      }
    }
  }
};

template <int D, int FMT, int MR, int MW, int TW, int STAGES, int CPS>
__global__ void __launch_bounds__(MW * TW * 32, CPS) kv_attention_kernel(const KvAttnParams p, const Work w) {
  using L = Tile<D, MR, MW, TW, STAGES>;
  extern __shared__ uint4 smem[];
  uint4* sq = smem;                                                                  // [MW * MR][D / 16][32]
  float4* so = reinterpret_cast<float4*>(smem + L::kQ);                              // [TW][rows][D / 4]
  float* sf = reinterpret_cast<float*>(smem + L::kSmem / 16) - L::kRows * (1 + 2 * TW);  // [rows]
  float* sm = sf + L::kRows;                                                         // [TW][rows]
  float* sl = sm + TW * L::kRows;                                                    // [TW][rows]
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int mw = warp % MW, tk = warp / MW;
  uint4* ring = smem + L::kQ + warp * STAGES * L::kStep;
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G, G = p.G;
  const int pairs = c.S * w.row_blocks;
  const bool by_item = static_cast<int64_t>(pairs) * c.heads == w.splits;
  const KvShare share = kv_share<L::kThreads>(p, w.row_blocks, L::kRows, TW);

  if (!by_item && tid == 0) w.split[blockIdx.x].parts = 0;
  // items without steps: their rows see nothing
  for (int i = blockIdx.x; i < pairs; i += gridDim.x) {
    const int s = i / w.row_blocks;
    const unsigned m0 = (i - s * w.row_blocks) * L::kRows;
    if (kv_span(p, kv_seq(c, p.rows.start, p.rows.lens, s), m0, L::kRows).n > 0) continue;
    const unsigned rows = min(M - m0, static_cast<unsigned>(L::kRows)) * c.heads;
    for (unsigned e = tid; e < rows * (D / 8); e += L::kThreads) {
      const unsigned row = e / (D / 8), h = row % c.heads, m = m0 + row / c.heads, r = m / G;
      const int64_t out = (static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * G + (m - r * G);
      reinterpret_cast<uint4*>(p.o + out * D)[e % (D / 8)] = make_uint4(0, 0, 0, 0);
      if (e % (D / 8) == 0) p.lse[out] = -INFINITY;
    }
    if (by_item)
      for (int h = tid; h < c.heads; h += L::kThreads) w.split[static_cast<int64_t>(i) * c.heads + h].parts = 0;
  }

  int64_t left = share.left, off = share.off, at = share.at;
  for (int pair = share.pair; left > 0;) {
    const int s = pair / w.row_blocks, mb = pair - s * w.row_blocks;
    const unsigned m0 = static_cast<unsigned>(mb) * L::kRows;
    const KvSeq seq = kv_seq(c, p.rows.start, p.rows.lens, s);
    const KvSpan span = kv_span(p, seq, m0, L::kRows);
    if (span.n == 0) {
      ++pair;
      continue;
    }
    const int h = static_cast<int>(kv_div(off, span.n)), i0 = static_cast<int>(off - static_cast<int64_t>(h) * span.n);
    const int i1 = static_cast<int>(min(static_cast<int64_t>(span.n), i0 + left));

    // ---- the segment: steps i0 .. i1 - 1, this warp's are i0 + tk, + TW, ...
    const KvSpan mine = kv_span(p, seq, min(m0 + mw * MR * 16, M), MR * 16);
    const int steps = mine.n > 0 ? max(0, (i1 - i0 - tk + TW - 1) / TW) : 0;
    const auto base_of = [&](int n) { return span.base(i0 + tk + n * TW); };
    const uint8_t* kc = c.k + static_cast<int64_t>(h) * c.T * D;
    const uint8_t* vc = c.v + static_cast<int64_t>(h) * c.T * D;
    const int64_t page_codes = static_cast<int64_t>(c.heads) * c.T * D;
    KvPages meta = kv_pages(c, s, lane < steps, base_of(lane)), next{-1};
    const auto fetch = [&](int n, int page) {  // step n into its slot of the ring; an empty group where there is none
      if (page >= 0) {
        const int64_t from = page * page_codes + (base_of(n) & (c.T - 1)) * D;
        copy_step<D>(ring + n % STAGES * L::kStep, kc + from, vc + from);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) {
      const int page = __shfl_sync(0xffffffffu, meta.page, n);
      fetch(n, n < steps ? page : -1);
    }
    kv_scales<true>(c, h, meta);
    if (tk == 0)
#pragma unroll
      for (int r = 0; r < MR; ++r)
        kv_load_q<D>(p, seq, s, h, m0 + (mw * MR + r) * 16, sq + (mw * MR + r) * (D / 16) * 32, sf + (mw * MR + r) * 16);
    int pos[MR][2];
    float o[MR][D / 8][4], m_run[MR][2], l_run[MR][2];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const unsigned m = m0 + (mw * MR + r) * 16 + 8 * e + g;
        const int row = seq.start + static_cast<int>(m / G);
        pos[r][e] = m < M && row < seq.len ? row : -1;
      }
#pragma unroll
      for (int t = 0; t < D / 8; ++t)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[r][t][x] = 0.f;
      m_run[r][0] = m_run[r][1] = -INFINITY;
      l_run[r][0] = l_run[r][1] = 0.f;
    }
    __syncthreads();  // the query operands
    float qf[MR][2];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      qf[r][0] = sf[(mw * MR + r) * 16 + g];
      qf[r][1] = sf[(mw * MR + r) * 16 + 8 + g];
    }
    const uint4* q = sq + mw * MR * (D / 16) * 32 + lane;

    const auto compute = [&](int n) {
      const uint4* b = ring + n % STAGES * L::kStep;
      const int page = __shfl_sync(0xffffffffu, meta.page, n & 31);
      const float ks = __shfl_sync(0xffffffffu, meta.ks, n & 31);
      const float vlog = __shfl_sync(0xffffffffu, meta.vlog, n & 31);
      const float vinv = __shfl_sync(0xffffffffu, meta.vinv, n & 31);
      const int j0 = base_of(n);
      if (page < 0 || j0 > mine.last) return;
      // logits of 16 positions, in units of log 2, with the value scale's logarithm added
      float x[MR][2][4];
      uint4 kw[2];
#pragma unroll
      for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][t][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        if ((kk & 3) == 0)
#pragma unroll
          for (int t = 0; t < 2; ++t) kw[t] = b[(t * (D / 64) + (kk >> 2)) * 32 + lane];
        uint32_t b0[2], b1[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) codes_to_half<FMT>(word_of(kw[t], kk & 3), b0[t], b1[t]);
#pragma unroll
        for (int r = 0; r < MR; ++r) {
          const uint4 a = q[(r * (D / 16) + kk) * 32];
          mma16816(x[r][0], a, b0[0], b1[0]);
          mma16816(x[r][1], a, b0[1], b1[1]);
        }
      }
      const bool whole = j0 + 15 <= mine.first && (p.mask.window == 0 || j0 > mine.last - p.mask.window ||
                                                   j0 + 15 < p.mask.sinks);
#pragma unroll
      for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][t][e] = x[r][t][e] * (qf[r][e >> 1] * ks) + vlog;
      if (!whole) {
#pragma unroll
        for (int r = 0; r < MR; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!kv_sees(p.mask, pos[r][e >> 1], j0 + 8 * t + 2 * q4 + (e & 1))) x[r][t][e] = -INFINITY;
      }
      uint4 a[MR];
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        float top[2], ref[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float y = fmaxf(fmaxf(x[r][0][2 * e], x[r][0][2 * e + 1]), fmaxf(x[r][1][2 * e], x[r][1][2 * e + 1]));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
          top[e] = fmaxf(m_run[r][e], y);
          ref[e] = top[e] == -INFINITY ? 0.f : top[e];
        }
        if (__any_sync(0xffffffffu, top[0] > m_run[r][0] || top[1] > m_run[r][1])) {
          const float f0 = ex2(m_run[r][0] - ref[0]), f1 = ex2(m_run[r][1] - ref[1]);
#pragma unroll
          for (int t = 0; t < D / 8; ++t) {
            o[r][t][0] *= f0;
            o[r][t][1] *= f0;
            o[r][t][2] *= f1;
            o[r][t][3] *= f1;
          }
          l_run[r][0] *= f0;
          l_run[r][1] *= f1;
          m_run[r][0] = top[0];
          m_run[r][1] = top[1];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][t][e] = ex2(x[r][t][e] - (ref[e >> 1] - kWeightLog));
#pragma unroll
        for (int e = 0; e < 2; ++e)
          l_run[r][e] += (x[r][0][2 * e] + x[r][0][2 * e + 1] + (x[r][1][2 * e] + x[r][1][2 * e + 1])) * vinv;
        const __half2 h0 = __floats2half2_rn(x[r][0][0], x[r][0][1]), h1 = __floats2half2_rn(x[r][0][2], x[r][0][3]);
        const __half2 h2 = __floats2half2_rn(x[r][1][0], x[r][1][1]), h3 = __floats2half2_rn(x[r][1][2], x[r][1][3]);
        a[r] = make_uint4(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1),
                          *reinterpret_cast<const uint32_t*>(&h2), *reinterpret_cast<const uint32_t*>(&h3));
      }
      VCodes<D> v;
      v.load(b);
      if (FMT == kKvE4m3 && !whole) {
        // what no row of the warp sees may be a NaN code
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = j0 + (i >> 1) * 8 + 2 * q4 + (i & 1);
          if (j > mine.last || (p.mask.window && j <= mine.first - p.mask.window && j >= p.mask.sinks))
#pragma unroll
            for (int wd = 0; wd < D / 32; ++wd) v.w[i][wd] = 0;
        }
      }
      // values: column g of tile t is value (D / 8) g + t; a word holds 4 tiles of one position
#pragma unroll
      for (int wd = 0; wd < D / 32; ++wd) {
        uint32_t b0[4], b1[4];
        {
          const uint32_t lo = prmt(v.w[0][wd], v.w[1][wd], 0x5140u);
          const uint32_t hi = prmt(v.w[0][wd], v.w[1][wd], 0x7362u);
          codes_to_half<FMT>(lo, b0[0], b0[1]);
          codes_to_half<FMT>(hi, b0[2], b0[3]);
        }
        {
          const uint32_t lo = prmt(v.w[2][wd], v.w[3][wd], 0x5140u);
          const uint32_t hi = prmt(v.w[2][wd], v.w[3][wd], 0x7362u);
          codes_to_half<FMT>(lo, b1[0], b1[1]);
          codes_to_half<FMT>(hi, b1[2], b1[3]);
        }
#pragma unroll
        for (int x4 = 0; x4 < 4; ++x4)
#pragma unroll
          for (int r = 0; r < MR; ++r) mma16816(o[r][4 * wd + x4], a[r], b0[x4], b1[x4]);
      }
    };
    for (int n = 0; n < steps; ++n) {
      if ((n & 31) == 0) {
        if (n > 0) meta = next;
        next = kv_pages(c, s, n + 32 + lane < steps, base_of(min(n + 32 + lane, steps)));
      }
      if ((n & 31) == 16) kv_scales<true>(c, h, next);
      const int ahead = n + STAGES - 1;
      const int page = __shfl_sync(0xffffffffu, (ahead ^ n) < 32 ? meta.page : next.page, ahead & 31);
      fetch(ahead, ahead < steps ? page : -1);
      cp_async_wait<STAGES - 1>();
      compute(n);
    }
    cp_async_wait<0>();

    // ---- join the TW warps of each row
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[r][e];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (pos[r][e] < 0) m_run[r][e] = -INFINITY;  // rows that do not exist
        if (q4 == 0) {
          const int row = (mw * MR + r) * 16 + 8 * e + g;
          sm[tk * L::kRows + row] = m_run[r][e];
          sl[tk * L::kRows + row] = l;
        }
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = (mw * MR + r) * 16 + 8 * e + g;
        float top = sm[row];
#pragma unroll
        for (int k = 1; k < TW; ++k) top = fmaxf(top, sm[k * L::kRows + row]);
        const float f = m_run[r][e] == -INFINITY ? 0.f : ex2(m_run[r][e] - top);
        float4* to = so + (tk * L::kRows + row) * (D / 4);
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int t = 0; t < D / 32; ++t) {
            float4 v;
            v.x = o[r][4 * t][2 * e + y] * f;
            v.y = o[r][4 * t + 1][2 * e + y] * f;
            v.z = o[r][4 * t + 2][2 * e + y] * f;
            v.w = o[r][4 * t + 3][2 * e + y] * f;
            if (f == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
            to[swizzle<D>(row, (D / 32) * (2 * q4 + y) + t)] = v;
          }
      }
    __syncthreads();
    const bool item = i0 == 0 && i1 == span.n;
    const int slot = 2 * blockIdx.x + (i0 == 0);
    if (!item && i0 == 0 && tid == 0) {
      const int parts = share.cross ? static_cast<int>((at + span.n - 1) / share.per) - static_cast<int>(blockIdx.x) + 1
                                    : static_cast<int>((span.n + share.per - 1) / share.per);
      w.split[by_item ? static_cast<int64_t>(pair) * c.heads + h : blockIdx.x] =
          Split{s, mb, h, static_cast<int>(blockIdx.x), parts};
    }
    if (item && by_item && tid == 0) w.split[static_cast<int64_t>(pair) * c.heads + h].parts = 0;
    for (int e = tid; e < L::kRows * (D / 8); e += L::kThreads) {
      const int row = e / (D / 8), f = 2 * (e % (D / 8));
      const unsigned m = m0 + row;
      if (m >= M) break;
      float top = sm[row];
#pragma unroll
      for (int k = 1; k < TW; ++k) top = fmaxf(top, sm[k * L::kRows + row]);
      float l = 0.f;
      float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
      for (int k = 0; k < TW; ++k) {
        const float mk = sm[k * L::kRows + row];
        if (mk != -INFINITY) l += sl[k * L::kRows + row] * ex2(mk - top);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float4 z = so[(k * L::kRows + row) * (D / 4) + swizzle<D>(row, f + y)];
          v[y].x += z.x;
          v[y].y += z.y;
          v[y].z += z.z;
          v[y].w += z.w;
        }
      }
      if (item) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const unsigned r = m / G;
        const int64_t out = (static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * G + (m - r * G);
        uint4 u;
        __nv_bfloat162 y0 = __floats2bfloat162_rn(v[0].x * inv, v[0].y * inv);
        __nv_bfloat162 y1 = __floats2bfloat162_rn(v[0].z * inv, v[0].w * inv);
        __nv_bfloat162 y2 = __floats2bfloat162_rn(v[1].x * inv, v[1].y * inv);
        __nv_bfloat162 y3 = __floats2bfloat162_rn(v[1].z * inv, v[1].w * inv);
        u.x = *reinterpret_cast<uint32_t*>(&y0);
        u.y = *reinterpret_cast<uint32_t*>(&y1);
        u.z = *reinterpret_cast<uint32_t*>(&y2);
        u.w = *reinterpret_cast<uint32_t*>(&y3);
        *reinterpret_cast<uint4*>(p.o + out * D + 4 * f) = u;
        if (f == 0) p.lse[out] = l > 0.f ? (top - kWeightLog + log2f(l)) * kLn2 : -INFINITY;
      } else {
        float4* to = reinterpret_cast<float4*>(w.part + (static_cast<int64_t>(slot) * L::kRows + row) * D) + f;
        to[0] = v[0];
        to[1] = v[1];
        if (f == 0) w.ml[static_cast<int64_t>(slot) * L::kRows + row] = make_float2(top, l);
      }
    }
    __syncthreads();  // the next segment writes the shared buffers
    left -= i1 - i0;
    at += i1 - i0;
    off += i1 - i0;
    if (off == static_cast<int64_t>(span.n) * c.heads) {
      ++pair;
      off = 0;
    }
  }
}

// Joins the parts of the items that lie in several blocks: WPR warps a row, a lane D / 32 values.
template <int D, int WPR>
__global__ void __launch_bounds__(256) kv_combine_kernel(const KvAttnParams p, const Work w, int rows) {
  constexpr int E = D / 32, RPB = 8 / WPR;
  __shared__ float s_l[8], s_o[8][D];
  pdl_wait();
  pdl_trigger();
  const Split t = w.split[blockIdx.x];
  if (t.parts == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y * RPB + warp / WPR;
  const int64_t m = static_cast<int64_t>(t.mb) * rows + row;
  const bool live = row < rows && m < static_cast<int64_t>(p.rows.R) * p.G;
  const auto slot = [&](int i) { return (2 * static_cast<int64_t>(t.block + i) + (i == 0)) * rows + row; };
  float top = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  if (live) {
    for (int i = lane; i < t.parts; i += 32) top = fmaxf(top, w.ml[slot(i)].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
#pragma unroll 8
    for (int i = warp % WPR; i < t.parts; i += WPR) {
      const float2 ml = w.ml[slot(i)];
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
      l += f * ml.y;
      const float* from = w.part + slot(i) * D + lane * E;
      if constexpr (E == 4) {
        const float4 v = *reinterpret_cast<const float4*>(from);
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(from);
        o[0] += f * v.x;
        o[1] += f * v.y;
      }
    }
  }
  if constexpr (WPR > 1) {
    if (lane == 0) s_l[warp] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    __syncthreads();
    if (warp % WPR != 0) return;
#pragma unroll
    for (int k = 1; k < WPR; ++k) {
      l += s_l[warp + k];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += s_o[warp + k][lane * E + e];
    }
  }
  if (!live) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t out = (static_cast<int64_t>(t.s) * p.rows.R + m / p.G) * p.Hq + t.h * p.G + m % p.G;
  uint32_t u[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
    u[e] = *reinterpret_cast<const uint32_t*>(&y);
  }
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(p.o + out * D + lane * E) = make_uint2(u[0], u[1]);
  else
    *reinterpret_cast<uint32_t*>(p.o + out * D + lane * E) = u[0];
  if (lane == 0) p.lse[out] = l > 0.f ? (top - kWeightLog + log2f(l)) * kLn2 : -INFINITY;
}

// The tiling for M = R * G rows a kv head: at most 16 rows: one tile whose steps four warps share, three
// blocks an SM; more: two tiles a warp, so that a converted operand serves both, one block an SM.
struct Plan {
  int rows, tw, per_sm;
};
Plan plan_of(int64_t M) {
  if (M <= 16) return Plan{16, 4, 3};
  if (M <= 32) return Plan{32, 8, 1};
  if (M <= 64) return Plan{64, 4, 1};
  return Plan{128, 2, 1};
}

template <int D, int FMT, int MR, int MW, int TW, int STAGES, int CPS>
cudaError_t launch(const KvAttnParams& p, const Work& w, unsigned blocks, const LaunchCfg& cfg) {
  using L = Tile<D, MR, MW, TW, STAGES>;
  static SmemOptIn opt;
  auto kern = kv_attention_kernel<D, FMT, MR, MW, TW, STAGES, CPS>;
  const cudaError_t e = allow_smem(kern, L::kSmem, opt);
  if (e != cudaSuccess) return e;
  return launch_kernel(kern, dim3(blocks), dim3(L::kThreads), L::kSmem, cfg, p, w);
}

template <int D, int FMT>
cudaError_t launch_rows(const KvAttnParams& p, const Work& w, int rows, unsigned blocks, const LaunchCfg& cfg) {
  switch (rows) {
    case 16: return launch<D, FMT, 1, 1, 4, 4, 3>(p, w, blocks, cfg);
    case 32: return launch<D, FMT, 2, 1, 8, 4, 1>(p, w, blocks, cfg);
    case 64: return launch<D, FMT, 2, 2, 4, 4, 1>(p, w, blocks, cfg);
    default: return launch<D, FMT, 2, 4, 2, 4, 1>(p, w, blocks, cfg);
  }
}

int64_t align16(int64_t n) { return (n + 15) & ~int64_t(15); }

}  // namespace

int64_t kv_attention_workspace(int64_t rows, int D, int sms) {
  const Plan t = plan_of(rows);
  const int64_t blocks = static_cast<int64_t>(sms) * t.per_sm;
  return align16(blocks * 2 * t.rows * D * 4) + align16(blocks * 2 * t.rows * 8) + blocks * static_cast<int64_t>(sizeof(Split));
}

cudaError_t launch_kv_attention(const KvAttnParams& p, void* workspace, const LaunchCfg& cfg) {
  const int64_t M = static_cast<int64_t>(p.rows.R) * p.G;
  const Plan t = plan_of(M);
  const int64_t row_blocks = (M + t.rows - 1) / t.rows, items = p.c.S * row_blocks * p.c.heads;
  if (M > 0x7fffffff || p.c.S * row_blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  // no more blocks than the longest sequences could fill
  const int64_t steps = std::max<int64_t>(items * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16), 1);
  const int64_t blocks = std::min<int64_t>(static_cast<int64_t>(cfg.sms) * t.per_sm, (steps + t.tw - 1) / t.tw);
  Work w{};
  w.row_blocks = static_cast<int>(row_blocks);
  w.splits = static_cast<int>(std::min(items, blocks));
  char* at = static_cast<char*>(workspace);
  w.part = reinterpret_cast<float*>(at);
  at += align16(blocks * 2 * t.rows * p.c.D * 4);
  w.ml = reinterpret_cast<float2*>(at);
  at += align16(blocks * 2 * t.rows * 8);
  w.split = reinterpret_cast<Split*>(at);
  const unsigned n = static_cast<unsigned>(blocks);
  const bool i8 = p.c.fmt == kKvInt8;
  cudaError_t e = p.c.D == 128 ? (i8 ? launch_rows<128, kKvInt8>(p, w, t.rows, n, cfg) : launch_rows<128, kKvE4m3>(p, w, t.rows, n, cfg))
                               : (i8 ? launch_rows<64, kKvInt8>(p, w, t.rows, n, cfg) : launch_rows<64, kKvE4m3>(p, w, t.rows, n, cfg));
  if (e != cudaSuccess) return e;
  LaunchCfg c2 = cfg;
  c2.pdl = true;  // same op: the kernel waits for its predecessor with griddepcontrol.wait
  const int64_t rows = std::min<int64_t>(M, t.rows);
  // few rows to join: eight warps a row, since each may have many parts
  const bool few = w.splits * rows <= 8 * cfg.sms;
  const dim3 grid(static_cast<unsigned>(w.splits), static_cast<unsigned>(few ? rows : (rows + 7) / 8));
  auto kern = p.c.D == 128 ? (few ? kv_combine_kernel<128, 8> : kv_combine_kernel<128, 1>)
                           : (few ? kv_combine_kernel<64, 8> : kv_combine_kernel<64, 1>);
  return launch_kernel(kern, grid, dim3(256), 0, c2, p, w, t.rows);
}

}  // namespace bolt
