// KvAttention over the paged 8-bit key/value cache (layout in kv.h).
//
//   l_j = scale * q . k_j over the positions j that the row sees;  lse = log sum_j exp(l_j)
//   o = sum_j exp(l_j - lse) v_j (bf16) and lse (f32); a row that sees nothing gives 0 and -inf,
//   one with a logit of NaN gives NaN
//
// One pass with the running maximum and sum of a softmax (kv_mma.cuh has the operands).  The rows of a
// sequence that read one kv head -- R rows times G query heads -- are the M axis of the products, so
// the codes are read once for all of them.  A block holds NT tiles of 8 rows and splits their steps over
// four warps; the blocks share all steps evenly (kv_share), a segment being one (sequence, row block,
// head)'s consecutive steps in one block.  At its end the four partial results are joined through shared
// memory.  A segment that is a whole item writes the result; the others leave (max, sum, values) in the
// workspace for kv_combine_kernel, which joins them in block order, so results do not depend on scheduling.
// More than 16 rows go to the tensor-memory kernel (kv_attention_umma.cu).
//
// Rounding: logits, maxima, sums and values are fp32; a weight is rounded to fp16 (11 bits) once, as
// the second product's operand.  A row's weights are 2^(x - m + 8) for its logits x (in units of log 2)
// and a reference m that is raised to the row's maximum only when some x passes m + 7: weights stay
// below 2^15, those down to 2^-22 of the largest keep all 11 bits and smaller ones err by at most 2^-33 of
// it, and most steps need neither the maximum over the row's lanes nor a rescaling.
//
// HBM bounds it where there is enough to read: 64 sequences of up to 8,192 positions, 8 heads, 4 rows a head
// take 95 us with the joining, 5.7 TB/s.  Tensor copies into a ring, because the codes must be on their way well
// ahead of their use and 16-byte copies by the lanes do not get there: with the arithmetic taken out they read
// 3.8 TB/s at any ring depth, tensor copies 5.9.  One sequence of 131,001 positions (16 rows a head, 2 heads)
// takes 30 us, 22 of them here: the way from the length to the first product, 37 steps a warp, and the parts'
// 2.4 MB.  Short items (48 sequences, 16 heads of 64 values, 68 steps an item: 37 us) are bound by their set-up.
#include "kv_split.cuh"

namespace bolt {

namespace {

// Of an item's set-up, in steps: about 6 us, measured in a batch of 64 sequences of up to 8,192 positions.
constexpr int kItemCost = 16;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kStages = 4;  // steps of a warp's ring

// NT tiles of 8 rows.
template <int D, int NT>
struct Tile {
  static constexpr int kRows = NT * 8;
  static constexpr int kStep = 32 * D;                       // bytes of a warp's step: 16 positions, K and V
  static constexpr int kRing = kWarps * kStages * kStep;
  static constexpr int kJoin = kWarps * kRows * D * 4;       // in the ring's place
  static_assert(kJoin <= kRing, "the joining buffer takes the ring's place");
  static constexpr size_t kSmem = kRing + kWarps * (64 * 20 + kStages * 8) + kWarps * kRows * 8 +
                                  1024;  // the ring starts on a 1,024-byte boundary
};

// float4 index f of a row's values in the joining buffer, spread over the banks
template <int D>
struct Swizzle {
  __device__ __forceinline__ int operator()(int row, int f) const {
    const int c = (row >> 1) & 3;
    return f ^ (D == 128 ? c : (c & 1) | (c >> 1) << 2);
  }
};

// An 8 x 8 matrix of halves, two neighbours of a row a lane, transposed.
__device__ __forceinline__ uint32_t transpose8(__half2 x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
  return y;
}

template <int D>
struct VCodes {
  uint32_t w[4][D / 32];  // position, word
  // `at`: this lane's places of the positions 2 c and 2 c + 1 in the step's V lines; the others are 8 positions on
  __device__ __forceinline__ void load(const uint8_t* v, const int (&at)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* from = v + (i < 2 ? at[i & 1] : kv_next_tile<D>(at[i & 1]));
      if constexpr (D == 128) {
        const uint4 x = lds128(from);
        w[i][0] = x.x;
        w[i][1] = x.y;
        w[i][2] = x.z;
        w[i][3] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(from);
        w[i][0] = x.x;
        w[i][1] = x.y;
      }
    }
  }
};

template <int D, int FMT, int NT, int CPS>
__global__ void __launch_bounds__(kThreads, CPS) kv_attention_kernel(
    const KvAttnParams p, const Work w, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using L = Tile<D, NT>;
  extern __shared__ uint4 smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float4* so = reinterpret_cast<float4*>(smem);                         // [warps][rows][D / 4]
  float4* s_scale = reinterpret_cast<float4*>(smem + L::kRing);         // [warps][64]: K scale, log2 and 1 / V scale, position and flags
  int* s_row = reinterpret_cast<int*>(s_scale + kWarps * 64);           // [warps][64]: first line of the codes, or -1
  uint64_t* s_full = reinterpret_cast<uint64_t*>(s_row + kWarps * 64);  // [warps][kStages]: barriers of the ring
  float* sm = reinterpret_cast<float*>(s_full + kWarps * kStages);      // [warps][rows]
  float* sl = sm + kWarps * L::kRows;                                   // [warps][rows]
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  uint8_t* ring = smem + warp * kStages * L::kStep;
  const uint32_t ring_at = smem_u32(ring);
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G, G = p.G;
  s_scale += warp * 64;
  s_row += warp * 64;
  s_full += warp * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(s_full + i), 1);
    fence_barrier_init();
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  __syncwarp();
  unsigned taken = 0;   // steps that this warp has put into its ring, of all segments
  bool stuck = false;   // a copy did not arrive in time: the rest of the work is left
  const int k_at = kv_at<D>(place<D>(g), 16 * q4);  // the codes 64 i + 16 q4 .. are at k_at ^ 64 i
  const int v_at[2] = {kv_at<D>(place<D>(2 * q4), D / 8 * g), kv_at<D>(place<D>(2 * q4 + 1), D / 8 * g)};
  const KvShare share = kv_share<kThreads>(p, w.row_blocks, L::kRows, kWarps, kItemCost);

  kv_empty_items<D, L::kRows, kThreads>(p, w);

  KvWalk walk;
  walk.start(share);
  for (KvSegment seg; walk.next(p, w.row_blocks, L::kRows, seg);) {
    const int s = seg.s, h = seg.h, i0 = seg.i0, i1 = seg.i1;
    const unsigned m0 = seg.m0;
    const KvSeq& seq = seg.seq;
    const KvSpan& span = seg.span;

    // ---- the segment: steps i0 .. i1 - 1; this warp's k-th is i0 + k kWarps + warp
    const int steps = max(0, (i1 - i0 - warp + kWarps - 1) / kWarps) * !stuck;
    const auto step_of = [&](int k) { return i0 + k * kWarps + warp; };
    uint4 raw_q[NT][D / 64][2];
#pragma unroll
    for (int r = 0; r < NT; ++r) kv_fetch_q<D>(p, seq, s, h, m0 + r * 8, raw_q[r]);
    // offsets and scales of 32 steps, one a lane, made in three stages so that the loads of one are under way
    // while steps are computed
    KvPages meta;
    const auto look_up_page = [&](int k) {
      meta.load_page(c, s, k < steps, span.base(min(step_of(k), i1 - 1)));
    };
    const auto look_up_scales = [&](int k) {
      meta.check_page(c);
      meta.load_scales<true>(c, h);
      s_row[k & 63] = meta.page < 0 ? -1 : ((meta.page * c.heads + h) * c.T + (span.base(step_of(k)) & (c.T - 1))) / (128 / D);
    };
    constexpr int kDead = 1, kWhole = 2;  // none of the rows sees the step, or all see all of it
    const auto keep = [&](int k) {
      const int j0 = span.base(min(step_of(k), i1 - 1));
      int flags = 0;
      if (meta.page < 0 || j0 > span.last)
        flags = kDead;
      else if (j0 + 15 <= span.first &&
               (p.mask.window == 0 || j0 > span.last - p.mask.window || j0 + 15 < p.mask.sinks))
        flags = kWhole;
      const float2 vs = kv_v_scale(meta.vs);
      s_scale[k & 63] = make_float4(meta.ks, vs.x, vs.y, __int_as_float(j0 | flags));
    };
    const auto fetch = [&](int k) {  // step k into its place in the ring
      __syncwarp();  // which no lane reads any more
      if (lane != 0 || k >= steps) return;
      const unsigned slot = (taken + k) % kStages;
      const int row = s_row[k & 63];
      const uint32_t bar = smem_u32(s_full + slot), to = ring_at + slot * L::kStep;
      if (row >= 0) {
        mbar_arrive_expect_tx(bar, 32 * D);
        tma_load_3d(to, &map_k, 0, row, 0, bar);
        tma_load_3d(to + 16 * D, &map_v, 0, row, 0, bar);
      } else {
        mbar_arrive(bar);
      }
    };
    constexpr int kAhead = kStages - 1;
    look_up_page(lane);
    look_up_scales(lane);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k);
    keep(lane);
    uint2 q[NT][D / 16];
    float qf[NT][2], qt[NT][2];  // of the rows 2 q4 and 2 q4 + 1 of each tile, as all that follow
    int pos[NT][2];
    float o[NT][D / 16][4], l_run[NT][2];
    float m_ref[NT][2], m_top[NT][2];  // the reference m - 8, and how far a logit may pass it: not at all until there is one
#pragma unroll
    for (int r = 0; r < NT; ++r) {
      float f, t;
      kv_make_q<D, FMT>(p, raw_q[r], q[r], f, t);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qf[r][e] = __shfl_sync(0xffffffffu, f, (2 * q4 + e) * 4);
        qt[r][e] = __shfl_sync(0xffffffffu, t, (2 * q4 + e) * 4);
        const unsigned m = m0 + r * 8 + 2 * q4 + e;
        const int row = seq.start + static_cast<int>(m / G);
        pos[r][e] = m < M && row < seq.len ? row : -1;
        m_ref[r][e] = 0.f;
        m_top[r][e] = -INFINITY;
        l_run[r][e] = 0.f;
      }
#pragma unroll
      for (int t2 = 0; t2 < D / 16; ++t2)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[r][t2][x] = 0.f;
    }
    __syncwarp();

    for (int k = 0; k < steps; ++k) {
      if ((k & 7) == 0) {
        const int later = (k & ~31) + 32 + lane;
        __syncwarp();  // no lane reads the entries of 32 steps ago any more
        if ((k & 31) == 0) look_up_page(later);
        if ((k & 31) == 8) look_up_scales(later);
        if ((k & 31) == 16) keep(later);
        __syncwarp();
      }
      fetch(k + kAhead);
      const unsigned at = taken + k;
      stuck |= !mbar_wait(smem_u32(s_full + at % kStages), (at / kStages) & 1, kStatusFullWait);
      if (__any_sync(0xffffffffu, stuck)) {
        // wait, within limits, for what else is on its way into the ring
        for (int i = k; i < min(k + kAhead + 1, steps); ++i)
          mbar_wait(smem_u32(s_full + (taken + i) % kStages), ((taken + i) / kStages) & 1, kStatusDrainWait);
        stuck = true;
        break;
      }

      const uint8_t* b = ring + at % kStages * L::kStep;
      const float4 sc = s_scale[k & 63];
      const int j0 = __float_as_int(sc.w) & ~15, flags = __float_as_int(sc.w);
      if (flags & kDead) continue;
      const bool whole = flags & kWhole;
      // logits in units of log 2, with the value scale's logarithm added, less the reference: lane (g, q4) has
      // the positions place(g) and 8 + place(g) (index 2 i) and the rows 2 q4 and 2 q4 + 1 (index e)
      float x[NT][4];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 lo = lds128(b + (k_at ^ (64 * i))), hi = lds128(b + (kv_next_tile<D>(k_at) ^ (64 * i)));
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t a0, a1, a2, a3;
          k_to_half<FMT>(word_of(lo, y), a0, a2);
          k_to_half<FMT>(word_of(hi, y), a1, a3);
#pragma unroll
          for (int r = 0; r < NT; ++r) {
            const uint2 qb = q[r][4 * i + y];
            if (i + y == 0)
              mma16816_first(x[r], a0, a1, a2, a3, qb.x, qb.y);
            else
              mma16816(x[r], a0, a1, a2, a3, qb.x, qb.y);
          }
        }
      }
      bool over = false;
#pragma unroll
      for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
          const float f = qf[r][e] * sc.x, d = sc.y - m_ref[r][e] - qt[r][e] * sc.x;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float& z = x[r][2 * i + e];
            z = z * f + d;
            if (!whole && !kv_sees(p.mask, pos[r][e], j0 + 8 * i + place<D>(g))) z = -INFINITY;
            top = fmaxf(top, z);
          }
          over |= top > m_top[r][e];
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int r = 0; r < NT; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(x[r][e], x[r][2 + e]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const bool fresh = m_top[r][e] == -INFINITY;
            // a row that sees nothing new keeps its reference
            if (top == -INFINITY) continue;
            const float up = fresh ? top - kWeightLog : fmaxf(0.f, top - kWeightLog), f = fresh ? 0.f : ex2(-up);
            x[r][e] -= up;
            x[r][2 + e] -= up;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
              o[r][t][e] *= f;
              o[r][t][2 + e] *= f;
            }
            l_run[r][e] *= f;
            m_ref[r][e] += up;
            m_top[r][e] = kWeightTop;
          }
      }
      // weights, as the second product's B operand: positions and rows change places
      uint32_t w0[NT], w1[NT];
#pragma unroll
      for (int r = 0; r < NT; ++r) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ex2(x[r][e]);
        l_run[r][0] += (y[0] + y[2]) * sc.z;
        l_run[r][1] += (y[1] + y[3]) * sc.z;
        w0[r] = transpose8(__floats2half2_rn(y[0], y[1]));
        w1[r] = transpose8(__floats2half2_rn(y[2], y[3]));
      }
      VCodes<D> v;
      v.load(b + 16 * D, v_at);
      if (FMT == kKvE4m3 && !whole) {
        // weights of 0 must not meet a NaN code (a stale one that no row sees, or one that some rows see): it becomes
        // 0, and the rows that see its position get a sum of NaN
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t any = 0;
#pragma unroll
          for (int wd = 0; wd < D / 32; ++wd) {
            const uint32_t bytes = kv_nan_bytes(v.w[i][wd]);
            any |= bytes;
            v.w[i][wd] &= ~bytes;
          }
          if (any) nan |= 1u << ((i >> 1) * 8 + place<D>(2 * q4 + (i & 1)));
        }
        nan = __reduce_or_sync(0xffffffffu, nan);
        if (nan) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = 8 * i + place<D>(g);
            if (nan >> at & 1)
#pragma unroll
              for (int r = 0; r < NT; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (kv_sees(p.mask, pos[r][e], j0 + at)) l_run[r][e] = NAN;
          }
        }
      }
      // the value axis: rows g and 8 + g of tile t are the values (D / 8) g + 2 t and + 1
#pragma unroll
      for (int wd = 0; wd < D / 32; ++wd)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t sel = i ? 0x7362u : 0x5140u;
          uint32_t a0, a1, a2, a3;
          codes_to_half<FMT>(prmt(v.w[0][wd], v.w[1][wd], sel), a0, a1);
          codes_to_half<FMT>(prmt(v.w[2][wd], v.w[3][wd], sel), a2, a3);
#pragma unroll
          for (int r = 0; r < NT; ++r) mma16816(o[r][2 * wd + i], a0, a1, a2, a3, w0[r], w1[r]);
        }
    }
    taken += steps;

    // ---- join the warps of each row
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[r][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        // the maximum's place takes the reference; none for rows that do not exist.  NaN among the logits passed
        // by the maximum and is in the sum, also of a row that has no reference.
        m_ref[r][e] = pos[r][e] < 0                  ? -INFINITY
                      : l != l                       ? NAN
                      : m_top[r][e] == -INFINITY     ? -INFINITY
                                                     : m_ref[r][e] + kWeightLog;
        if (g == 0) {
          const int row = r * 8 + 2 * q4 + e;
          sm[warp * L::kRows + row] = m_ref[r][e];
          sl[warp * L::kRows + row] = l;
        }
      }
    __syncthreads();  // and all rings are idle
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = r * 8 + 2 * q4 + e;
        float top = sm[row];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) top = fmaxf(top, sm[k * L::kRows + row]);
        const float f = m_ref[r][e] == -INFINITY ? 0.f : ex2(m_ref[r][e] - top);
        float4* to = so + (warp * L::kRows + row) * (D / 4);
#pragma unroll
        for (int t = 0; t < D / 16; t += 2) {
          float4 v = make_float4(o[r][t][e] * f, o[r][t][2 + e] * f, o[r][t + 1][e] * f, o[r][t + 1][2 + e] * f);
          if (f == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
          to[Swizzle<D>()(row, D / 32 * g + t / 2)] = v;
        }
      }
    __syncthreads();
    kv_finish<D, L::kRows, kWarps, kThreads>(p, w, share, seg, sm, sl, so, Swizzle<D>());
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next segment's copies come after these reads and writes
    __syncthreads();
  }
}

// Joins the parts of the items that lie in several blocks: WPR warps a row, a lane D / 32 values.  Latency bounds
// it (the item, the parts' maxima, the parts), so that a row of many parts has 32 warps: 6 us for 148 parts.
template <int D, int WPR>
__global__ void __launch_bounds__(WPR > 8 ? WPR * 32 : 256) kv_combine_kernel(const KvAttnParams p, const Work w, int rows) {
  constexpr int E = D / 32, W = WPR > 8 ? WPR : 8, RPB = W / WPR;
  __shared__ float s_l[W], s_o[W][D];
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
  const float inv = l == 0.f ? 0.f : 1.f / l;
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
  if (lane == 0) p.lse[out] = l == 0.f ? -INFINITY : (top - kWeightLog + log2f(l)) * kLn2;
}

// The tiling for M = R * G rows a kv head.  Up to 16 rows: tiles of 8 or 16 rows whose steps four warps share,
// several blocks an SM.  More: 128 rows, the tensor-memory kernel, one block an SM.  It costs much the same for 17
// rows as for 128, the other the more the more rows it has.  Both sides, in us, with tiles of 32 and 64 rows for the
// first, which it had before ("window": 1,024 positions and 4 sinks of 48 sequences of up to 20,000):
//   heads of 128 values           16 rows     24         32         48         64
//     32 x 8,192 positions, 8 heads  76   154 : 137  159 : 137  239 : 141  244 : 144
//     8 x 16,384, 2 heads            22              29 : 31    44 : 31    45 : 32
//     window, 16 heads               75   155 : 151  159 : 154  232 : 161  234 : 165
//     window, 4 heads                29    52 : 51    53 : 52    71 : 55    73 : 57
//   heads of 64 values
//     32 x 8,192 positions, 8 heads  61   111 : 121  114 : 123  171 : 124  173 : 126
//     8 x 16,384, 2 heads            19              24 : 27    34 : 28    34 : 28
//     window, 16 heads               61   113 : 134  115 : 135  173 : 139  172 : 141
//     window, 4 heads                23    38 : 44    39 : 44    53 : 46    54 : 47
// One rule for both head sizes: with 17 to 32 rows it costs heads of 64 values 7 to 19% (their weights' exponentials
// are as many as those of 128 values, over half the bytes), and a window of 256 positions in 4 sequences, where
// set-up is all, 10 to 20% for either; tiles of 32 rows for them alone would be a third form of this kernel.
// Registers set the blocks an SM.
struct Plan {
  int rows, round, per_sm;
};
Plan plan_of(int64_t M, int D) {
  if (M <= 8) return Plan{8, kWarps, D == 64 ? 4 : 3};
  if (M <= 16) return Plan{16, kWarps, 2};
  return Plan{128, 8, 1};
}

template <int D, int FMT, int NT, int CPS>
cudaError_t launch(const KvAttnParams& p, const Work& w, unsigned blocks, const LaunchCfg& cfg) {
  using L = Tile<D, NT>;
  static SmemOptIn opt;
  auto kern = kv_attention_kernel<D, FMT, NT, CPS>;
  const cudaError_t e = allow_smem(kern, L::kSmem, opt);
  if (e != cudaSuccess) return e;
  CUtensorMap map_k, map_v;
  if (!kv_code_map(&map_k, p.c, p.c.k) || !kv_code_map(&map_v, p.c, p.c.v)) return cudaErrorInvalidValue;
  return launch_kernel(kern, dim3(blocks), dim3(kThreads), L::kSmem, cfg, p, w, map_k, map_v);
}

template <int D, int FMT>
cudaError_t launch_rows(const KvAttnParams& p, const Work& w, int rows, unsigned blocks, const LaunchCfg& cfg) {
  switch (rows) {
    case 8: return launch<D, FMT, 1, D == 64 ? 4 : 3>(p, w, blocks, cfg);
    case 16: return launch<D, FMT, 2, 2>(p, w, blocks, cfg);
    default: return launch_kv_attention_umma(p, w, blocks, cfg);
  }
}

int64_t align16(int64_t n) { return (n + 15) & ~int64_t(15); }

}  // namespace

int64_t kv_attention_workspace(int64_t rows, int D, int sms) {
  const Plan t = plan_of(rows, D);
  const int64_t blocks = static_cast<int64_t>(sms) * t.per_sm;
  return align16(blocks * 2 * t.rows * D * 4) + align16(blocks * 2 * t.rows * 8) + blocks * static_cast<int64_t>(sizeof(Split));
}

cudaError_t launch_kv_attention(const KvAttnParams& params, void* workspace, const LaunchCfg& cfg) {
  KvAttnParams p = params;
  const int64_t M = static_cast<int64_t>(p.rows.R) * p.G;
  const Plan t = plan_of(M, p.c.D);
  const int64_t row_blocks = (M + t.rows - 1) / t.rows, items = p.c.S * row_blocks * p.c.heads;
  if (p.c.S * row_blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  p.few_steps = items * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16 + kMostItemCost) <= 0x7fffffff;
  // no more blocks than the longest sequences could fill
  const int64_t steps = std::max<int64_t>(items * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16), 1);
  const int64_t blocks = std::min<int64_t>(static_cast<int64_t>(cfg.sms) * t.per_sm, (steps + t.round - 1) / t.round);
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
  // few rows to join: 32 warps a row, since each may have many parts
  const bool few = w.splits * rows <= 2 * cfg.sms;
  const dim3 grid(static_cast<unsigned>(w.splits), static_cast<unsigned>(few ? rows : (rows + 7) / 8));
  auto kern = p.c.D == 128 ? (few ? kv_combine_kernel<128, 32> : kv_combine_kernel<128, 1>)
                           : (few ? kv_combine_kernel<64, 32> : kv_combine_kernel<64, 1>);
  return launch_kernel(kern, grid, dim3(few ? 1024 : 256), 0, c2, p, w, t.rows);
}

}  // namespace bolt
