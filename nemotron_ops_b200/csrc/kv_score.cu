// KvScore: score[s, h, j] += sum over the rows and the query heads of cache head h of
// exp(scale * q . k_j - lse), the attention weights that KvAttention gave position j.
//
// The steps of all (sequence, head) pairs are shared evenly over the blocks (kv_mma.cuh); a step's
// 16 positions belong to one warp, which keeps their K codes as fp16 operands in registers while it
// goes through the row tiles, so a sum is made by one warp in one order and added to the score once
// for each kRowTiles * 8 rows.
#include "kv_mma.cuh"

namespace bolt {

namespace {

constexpr int kWarps = 8;
constexpr int kRowTiles = 16;  // tiles of 8 query rows in shared memory at a time

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 2) kv_score_kernel(const KvAttnParams p) {
  __shared__ uint2 sq[kRowTiles * (D / 16) * 32];
  __shared__ float4 srow[kRowTiles * 8];  // a row's logit factor and shift, lse / log 2, and position or -1
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G;
  const KvShare share = kv_share<kWarps * 32>(p, 1, M, kWarps);
  int64_t left = share.left, off = share.off;
  for (int next_s = share.pair; left > 0;) {
    const int s = next_s;
    const KvSeq seq = kv_seq(c, p.rows.start, p.rows.lens, s);
    const KvSpan span = kv_span(p, seq, 0, M);
    if (span.n == 0) {
      ++next_s;
      continue;
    }
    // units u0 .. u1 - 1 of the item, of which those from share.cost on are its steps
    const int size = span.n + share.cost;
    const int h = static_cast<int>(kv_div(off, size)), u0 = static_cast<int>(off - static_cast<int64_t>(h) * size);
    const int u1 = static_cast<int>(min(static_cast<int64_t>(size), u0 + left));
    const int i0 = max(0, u0 - share.cost), i1 = max(0, u1 - share.cost);
    left -= u1 - u0;
    off += u1 - u0;
    if (off == static_cast<int64_t>(size) * c.heads) {
      ++next_s;
      off = 0;
    }
    if (i0 == i1) continue;
    float* score = p.score + (static_cast<int64_t>(s) * c.heads + h) * p.score_width;
    const int steps = max(0, (i1 - i0 - warp + kWarps - 1) / kWarps);
    const auto base_of = [&](int n) { return span.base(i0 + warp + n * kWarps); };
    const uint8_t* kc = c.k + static_cast<int64_t>(h) * c.T * D;
    const int64_t page_codes = static_cast<int64_t>(c.heads) * c.T * D;
    for (unsigned m0 = 0; m0 < M; m0 += kRowTiles * 8) {
      const int tiles = min((M - m0 + 7) / 8, static_cast<unsigned>(kRowTiles));
      const KvSpan chunk = kv_span(p, seq, m0, kRowTiles * 8);
      if (chunk.n == 0) break;  // rows past the sequence's end, here and in every later chunk
      __syncthreads();          // the previous chunk's operands are still read
      for (int t = warp; t < tiles; t += kWarps) {
        uint2 x[D / 16];
        float f, sh;
        uint4 rq[D / 64][2];
        kv_fetch_q<D>(p, seq, s, h, m0 + t * 8, rq);
        kv_make_q<D, FMT>(p, rq, x, f, sh);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) sq[(t * (D / 16) + kk) * 32 + lane] = x[kk];
        if (q4 == 0) {
          const unsigned m = m0 + t * 8 + g, r = m / static_cast<unsigned>(p.G);
          const bool live = m < M && seq.start + static_cast<int>(r) < seq.len;
          const float z = live ? p.lse[(static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * p.G + (m - r * p.G)] * kLog2e : 0.f;
          srow[t * 8 + g] = make_float4(f, sh, z, __int_as_float(live ? seq.start + static_cast<int>(r) : -1));
        }
      }
      KvPages meta{-1, 0.f, 0.f}, next;
      next.load_page(c, s, lane < steps, base_of(lane));
      next.check_page(c);
      next.load_scales<false>(c, h);
      uint4 raw[2][D / 64], ahead[2][D / 64];
      const auto fetch = [&](int n, const KvPages& of) {
        const int page = __shfl_sync(0xffffffffu, of.page, n & 31);
        if (page < 0) return;
        // lane (g, q4) takes the codes 64 i + 16 q4 .. + 15 of the positions g and 8 + g
        const uint8_t* from = kc + page * page_codes + ((base_of(n) & (c.T - 1)) + g) * D + 16 * q4;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) ahead[t][i] = ld128(from + 8 * t * D + 64 * i);
      };
      if (steps > 0) fetch(0, next);
      __syncthreads();
      for (int n = 0; n < steps; ++n) {
        if ((n & 31) == 0) {
          meta = next;
          next.load_page(c, s, n + 32 + lane < steps, base_of(min(n + 32 + lane, steps)));
        }
        if ((n & 31) == 8) {
          next.check_page(c);
          next.load_scales<false>(c, h);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) raw[t][i] = ahead[t][i];
        if (n + 1 < steps) fetch(n + 1, ((n + 1) & 31) == 0 ? next : meta);
        const int page = __shfl_sync(0xffffffffu, meta.page, n & 31);
        const float ks = __shfl_sync(0xffffffffu, meta.ks, n & 31);
        const int j0 = base_of(n);
        if (page < 0 || j0 > chunk.last) continue;
        uint32_t a[D / 16][4];
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          k_to_half<FMT>(word_of(raw[0][kk >> 2], kk & 3), a[kk][0], a[kk][2]);
          k_to_half<FMT>(word_of(raw[1][kk >> 2], kk & 3), a[kk][1], a[kk][3]);
        }
        float sum[2] = {0.f, 0.f};  // positions g and 8 + g
        for (int t = 0; t < tiles; ++t) {
          float x[4];
          const uint2 b0 = sq[t * (D / 16) * 32 + lane];
          mma16816_first(x, a[0][0], a[0][1], a[0][2], a[0][3], b0.x, b0.y);
#pragma unroll
          for (int kk = 1; kk < D / 16; ++kk) {
            const uint2 b = sq[(t * (D / 16) + kk) * 32 + lane];
            mma16816(x, a[kk][0], a[kk][1], a[kk][2], a[kk][3], b.x, b.y);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 row = srow[t * 8 + 2 * q4 + e];
            const int pos = __float_as_int(row.w);
            const float f = row.x * ks, d = -row.y * ks - row.z;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float w = ex2(x[2 * i + e] * f + d);
              if (kv_sees(p.mask, pos, j0 + 8 * i + g)) sum[i] += w;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = sum[i];
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          const int j = j0 + 8 * i + g;
          if (q4 == 0 && j <= chunk.last) score[j] += v;
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_kv_score(const KvAttnParams& params, const LaunchCfg& cfg) {
  KvAttnParams p = params;
  const int64_t steps = std::max<int64_t>(
      static_cast<int64_t>(p.c.S) * p.c.heads * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16), 1);
  p.few_steps = steps + static_cast<int64_t>(p.c.S) * p.c.heads * kItemCost <= 0x7fffffff;
  const int64_t blocks = std::min<int64_t>(cfg.sms * 2, (steps + kWarps - 1) / kWarps);
  auto kern = p.c.D == 128 ? (p.c.fmt == kKvInt8 ? kv_score_kernel<128, kKvInt8> : kv_score_kernel<128, kKvE4m3>)
                           : (p.c.fmt == kKvInt8 ? kv_score_kernel<64, kKvInt8> : kv_score_kernel<64, kKvE4m3>);
  return launch_kernel(kern, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0, cfg, p);
}

}  // namespace bolt
