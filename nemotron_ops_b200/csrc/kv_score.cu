// KvScore: score[s, h, j] += sum over the rows and the query heads of cache head h of
// exp(scale * q . k_j - lse), the attention weights that KvAttention gave position j.
//
// The steps of all (sequence, head) pairs are shared evenly over the blocks (kv_mma.cuh).  A step's
// 16 positions belong to one warp, which copies their K codes into a ring of its own ahead of time and
// keeps them as fp16 operands in registers while it goes through the row tiles: a sum is made by one warp
// in one order and added to the score once for each kRowTiles * 8 rows, by a reduction in memory that
// nothing waits for and no other warp makes for these positions.  Instruction issue bounds it where there is
// enough to do: 32 sequences of up to 8,192 positions, 8 heads of 64 values, 16 rows a head take 41 us, 290
// instructions a KB of codes.  One sequence of 65,536 positions, 2 heads of 128, 16 rows: 11 us, of which the
// bytes are 2.7 and the way from the length to the first codes most of the rest.
#include "kv_mma.cuh"

namespace bolt {

namespace {

constexpr int kWarps = 8;
constexpr int kItemCost = 16;  // of an item's set-up, in steps (kv_attention.cu has the measurement)
constexpr int kRowTiles = 16;  // tiles of 8 query rows in shared memory at a time
// Steps that a warp takes at a time and steps of its ring.  Steps of 64 values are too short for one alone
// (32 sequences of up to 8,192 positions, 8 heads, 16 rows a head: 47 us one at a time, with a ring of 3, 4 or 6, and
// 41 us two; 4 rows a head 41 and 36; one sequence of 65,536, 2 heads, 9.9 and 9.3).  Two of 128 values spill, and
// gain little (54 and 51 us for the batch, 28 and 28 for 8 sequences, 11.2 and 11.0 for one) with a ring of 4; one of
// 6 leaves one block an SM (83, 43 and 18 us).
template <int D>
constexpr int kTogether = D == 64 ? 2 : 1;
template <int D>
constexpr int kRing = D == 64 ? 6 : 4;
template <int D>
constexpr size_t kScoreSmem = kWarps * (kRing<D> * (16 * D + 8) + 64 * 12) + 1024;

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 2) kv_score_kernel(const KvAttnParams p, const __grid_constant__ CUtensorMap map_k) {
  constexpr int kPairs = kTogether<D>, kStages = kRing<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint2 sq[kRowTiles * (D / 16) * 32];
  __shared__ float4 srow[kRowTiles * 8];  // a row's logit factor and shift, lse / log 2 (of no row: infinite, so that its weights are 0), and position or -1
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + warp * kStages * 16 * D;
  uint64_t* s_full = reinterpret_cast<uint64_t*>(smem + kWarps * kStages * 16 * D) + warp * kStages;  // the ring's barriers
  // of 64 of the warp's steps: first line of the codes or -1, and the page's scale and the first position
  float2* s_scale = reinterpret_cast<float2*>(smem + kWarps * kStages * (16 * D + 8)) + warp * 64;
  int* s_row = reinterpret_cast<int*>(smem + kWarps * (kStages * (16 * D + 8) + 64 * 8)) + warp * 64;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(s_full + i), 1);
    fence_barrier_init();
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  __syncwarp();
  unsigned taken = 0;  // steps that this warp has put into its ring, of all segments
  bool stuck = false;  // a copy did not arrive in time: the rest of the work is left
  const int k_at = kv_at<D>(place<D>(g), 16 * q4);  // the codes 64 i + 16 q4 .. are at k_at ^ 64 i
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G;
  const KvShare share = kv_share<kWarps * 32>(p, 1, M, kWarps * kPairs, kItemCost);
  KvWalk walk;
  walk.start(share);
  for (KvSegment seg; walk.next(p, 1, M, seg);) {
    const int s = seg.s, h = seg.h, i0 = seg.i0, i1 = seg.i1;
    const KvSeq& seq = seg.seq;
    const KvSpan& span = seg.span;
    float* score = p.score + (static_cast<int64_t>(s) * c.heads + h) * p.score_width;
    // this warp's k-th step is the k % kPairs-th of the group k / kPairs * kWarps + warp
    const int most = max(0, (i1 - i0 - warp * kPairs + kWarps * kPairs - 1) / (kWarps * kPairs));
    const auto step_of = [&](int k) { return i0 + (k / kPairs * kWarps + warp) * kPairs + k % kPairs; };
    for (unsigned m0 = 0; m0 < M; m0 += kRowTiles * 8) {
      const int tiles = min((M - m0 + 7) / 8, static_cast<unsigned>(kRowTiles));
      const KvSpan chunk = kv_span(p, seq, m0, kRowTiles * 8);
      if (chunk.n == 0) break;  // rows past the sequence's end, here and in every later chunk
      const int rounds = stuck ? 0 : most;
      KvPages meta;
      const auto look_up = [&](int k) {
        const int i = step_of(k);
        meta.load_page(c, s, k < rounds * kPairs && i < i1, span.base(min(i, i1 - 1)));
      };
      const auto look_up_scales = [&](int k) {
        meta.check_page(c);
        meta.load_scales<false>(c, h);
        s_row[k & 63] = meta.page < 0 ? -1 : ((meta.page * c.heads + h) * c.T + (span.base(step_of(k)) & (c.T - 1))) / (128 / D);
      };
      constexpr int kDead = 1, kWhole = 2;  // no row of the chunk sees the step, or all see all of it
      const auto keep = [&](int k) {
        const int j0 = span.base(min(step_of(k), i1 - 1));
        int flags = 0;
        if (meta.page < 0 || j0 > chunk.last)
          flags = kDead;
        else if (j0 + 15 <= chunk.first &&
                 (p.mask.window == 0 || j0 > chunk.last - p.mask.window || j0 + 15 < p.mask.sinks))
          flags = kWhole;
        s_scale[k & 63] = make_float2(meta.ks, __int_as_float(j0 | flags));
      };
      const auto fetch = [&](int n) {
        __syncwarp();  // no lane reads its places in the ring any more
        if (lane != 0 || n >= rounds) return;
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          const unsigned slot = (taken + n * kPairs + u) % kStages;
          const int row = s_row[(n * kPairs + u) & 63];
          const uint32_t bar = smem_u32(s_full + slot);
          if (row >= 0) {
            mbar_arrive_expect_tx(bar, 16 * D);
            tma_load_3d(smem_u32(ring + slot * 16 * D), &map_k, 0, row, 0, bar);
          } else {
            mbar_arrive(bar);
          }
        }
      };
      constexpr int kAhead = kStages / kPairs - 1;
      look_up(lane);
      look_up_scales(lane);
      __syncwarp();
#pragma unroll
      for (int n = 0; n < kAhead; ++n) fetch(n);
      __syncthreads();  // the previous chunk's operands have been read
      for (int t = warp; t < tiles; t += kWarps) {
        uint2 x[D / 16];
        float f, sh;
        uint4 rq[D / 64][2];
        kv_fetch_q<D>(p, seq, s, h, m0 + t * 8, rq);
        const unsigned m = m0 + t * 8 + g, r = m / static_cast<unsigned>(p.G);
        const bool live = m < M && seq.start + static_cast<int>(r) < seq.len;
        const float z = live ? p.lse[(static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * p.G + (m - r * p.G)] * kLog2e : INFINITY;
        kv_make_q<D, FMT>(p, rq, x, f, sh);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) sq[(t * (D / 16) + kk) * 32 + lane] = x[kk];
        if (q4 == 0) srow[t * 8 + g] = make_float4(f, sh, z, __int_as_float(live ? seq.start + static_cast<int>(r) : -1));
      }
      keep(lane);
      __syncthreads();
      for (int n = 0; n < rounds; ++n) {
        const int k0 = n * kPairs;
        if ((k0 & 7) == 0) {
          const int later = (k0 & ~31) + 32 + lane;
          __syncwarp();  // no lane reads the entries of 32 steps ago any more
          if ((k0 & 31) == 0) look_up(later);
          if ((k0 & 31) == 8) look_up_scales(later);
          if ((k0 & 31) == 16) keep(later);
          __syncwarp();
        }
        fetch(n + kAhead);
        bool late = false;
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          const unsigned i = taken + k0 + u;
          late |= !mbar_wait(smem_u32(s_full + i % kStages), (i / kStages) & 1, kStatusFullWait);
        }
        if (__any_sync(0xffffffffu, late)) {
          // wait, within limits, for what else is on its way into the ring
          for (int k = k0; k < min(n + kAhead + 1, rounds) * kPairs; ++k)
            mbar_wait(smem_u32(s_full + (taken + k) % kStages), ((taken + k) / kStages) & 1, kStatusDrainWait);
          stuck = true;
          break;
        }
        float ks[kPairs];
        int j0[kPairs], all = kDead | kWhole;
        uint32_t a[kPairs][D / 16][4];
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
          const float2 sc = s_scale[(k0 + u) & 63];
          ks[u] = sc.x;
          j0[u] = __float_as_int(sc.y);
          all &= j0[u];
          // a step that was not copied holds anything; its weights are left out below
          const uint8_t* b = ring + (taken + k0 + u) % kStages * 16 * D;
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 lo = lds128(b + (k_at ^ (64 * i))), hi = lds128(b + (kv_next_tile<D>(k_at) ^ (64 * i)));
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              k_to_half<FMT>(word_of(lo, y), a[u][4 * i + y][0], a[u][4 * i + y][2]);
              k_to_half<FMT>(word_of(hi, y), a[u][4 * i + y][1], a[u][4 * i + y][3]);
            }
          }
        }
        if (all & kDead) continue;
        const bool whole = all & kWhole;
        float sum[kPairs][2] = {};  // positions place(g) and 8 + place(g)
        for (int t = 0; t < tiles; ++t) {
          float x[kPairs][4];
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint2 b = sq[(t * (D / 16) + kk) * 32 + lane];
#pragma unroll
            for (int u = 0; u < kPairs; ++u) {
              if (kk == 0)
                mma16816_first(x[u], a[u][kk][0], a[u][kk][1], a[u][kk][2], a[u][kk][3], b.x, b.y);
              else
                mma16816(x[u], a[u][kk][0], a[u][kk][1], a[u][kk][2], a[u][kk][3], b.x, b.y);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 row = srow[t * 8 + 2 * q4 + e];
#pragma unroll
            for (int u = 0; u < kPairs; ++u) {
              const float f = row.x * ks[u], d = -row.y * ks[u] - row.z;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float w = ex2(x[u][2 * i + e] * f + d);
                if (!whole && ((j0[u] & kDead) || !kv_sees(p.mask, __float_as_int(row.w), (j0[u] & ~15) + 8 * i + place<D>(g))))
                  w = 0.f;
                sum[u][i] += w;
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < kPairs; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v = sum[u][i];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            const int j = (j0[u] & ~15) + 8 * i + place<D>(g);
            if (q4 == 0 && !(j0[u] & kDead) && j <= chunk.last) atomicAdd(score + j, v);
          }
      }
      taken += rounds * kPairs;
    }
  }
}

template <int D, int FMT>
cudaError_t launch(const KvAttnParams& p, const CUtensorMap& map_k, unsigned blocks, const LaunchCfg& cfg) {
  static SmemOptIn opt;
  const cudaError_t e = allow_smem(kv_score_kernel<D, FMT>, kScoreSmem<D>, opt);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv_score_kernel<D, FMT>, dim3(blocks), dim3(kWarps * 32), kScoreSmem<D>, cfg, p, map_k);
}

}  // namespace

cudaError_t launch_kv_score(const KvAttnParams& params, const LaunchCfg& cfg) {
  KvAttnParams p = params;
  const int64_t steps = std::max<int64_t>(
      static_cast<int64_t>(p.c.S) * p.c.heads * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16), 1);
  p.few_steps = steps + static_cast<int64_t>(p.c.S) * p.c.heads * kMostItemCost <= 0x7fffffff;
  const int round = kWarps * (p.c.D == 64 ? kTogether<64> : kTogether<128>);
  const int64_t blocks = std::min<int64_t>(cfg.sms * 2, (steps + round - 1) / round);
  CUtensorMap map_k;
  if (!kv_code_map(&map_k, p.c, p.c.k)) return cudaErrorInvalidValue;
  const unsigned n = static_cast<unsigned>(blocks);
  const bool i8 = p.c.fmt == kKvInt8;
  if (p.c.D == 128) return i8 ? launch<128, kKvInt8>(p, map_k, n, cfg) : launch<128, kKvE4m3>(p, map_k, n, cfg);
  return i8 ? launch<64, kKvInt8>(p, map_k, n, cfg) : launch<64, kKvE4m3>(p, map_k, n, cfg);
}

}  // namespace bolt
