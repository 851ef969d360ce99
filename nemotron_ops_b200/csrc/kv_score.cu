// KvScore: score[s, h, j] += sum over the rows and the query heads of cache head h of
// exp(scale * q . k_j - lse), the attention weights that KvAttention gave position j.
//
// The steps of all (sequence, head) pairs are shared evenly over the blocks (kv_mma.cuh); a step's
// 16 positions belong to one warp, which keeps their K codes as fp16 operands in registers while it
// goes through the row tiles, so a sum is made by one warp in one order and added to the score once
// for each kRowTiles * 16 rows.
#include "kv_mma.cuh"

namespace bolt {

namespace {

constexpr int kWarps = 8;
constexpr int kRowTiles = 8;  // tiles of 16 query rows in shared memory at a time

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 2) kv_score_kernel(const KvAttnParams p) {
  __shared__ uint4 sq[kRowTiles * (D / 16) * 32];
  __shared__ float sf[kRowTiles * 16], sz[kRowTiles * 16];
  __shared__ int spos[kRowTiles * 16];
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G;
  const KvShare share = kv_share<kWarps * 32>(p, 1, M, kWarps);
  int64_t left = share.left, off = share.off;
  for (int s = share.pair; left > 0;) {
    const KvSeq seq = kv_seq(c, p.rows.start, p.rows.lens, s);
    const KvSpan span = kv_span(p, seq, 0, M);
    if (span.n == 0) {
      ++s;
      continue;
    }
    const int h = static_cast<int>(kv_div(off, span.n)), i0 = static_cast<int>(off - static_cast<int64_t>(h) * span.n);
    const int i1 = static_cast<int>(min(static_cast<int64_t>(span.n), i0 + left));
    float* score = p.score + (static_cast<int64_t>(s) * c.heads + h) * p.score_width;
    const int steps = max(0, (i1 - i0 - warp + kWarps - 1) / kWarps);
    const auto base_of = [&](int n) { return span.base(i0 + warp + n * kWarps); };
    const uint8_t* kc = c.k + static_cast<int64_t>(h) * c.T * D;
    const int64_t page_codes = static_cast<int64_t>(c.heads) * c.T * D;
    for (unsigned m0 = 0; m0 < M; m0 += kRowTiles * 16) {
      const int tiles = min((M - m0 + 15) / 16, static_cast<unsigned>(kRowTiles));
      const KvSpan chunk = kv_span(p, seq, m0, kRowTiles * 16);
      if (chunk.n == 0) break;  // rows past the sequence's end, here and in every later chunk
      __syncthreads();          // the previous chunk's operands are still read
      for (int t = warp; t < tiles; t += kWarps)
        kv_load_q<D>(p, seq, s, h, m0 + t * 16, sq + t * (D / 16) * 32, sf + t * 16);
      for (int i = tid; i < tiles * 16; i += kWarps * 32) {
        const unsigned m = m0 + i, r = m / static_cast<unsigned>(p.G);
        const bool live = m < M && seq.start + static_cast<int>(r) < seq.len;
        spos[i] = live ? seq.start + static_cast<int>(r) : -1;
        sz[i] = live ? p.lse[(static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * p.G + (m - r * p.G)] * kLog2e : 0.f;
      }
      KvPages meta{-1}, next = kv_pages(c, s, lane < steps, base_of(lane));
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
          if (n == 0) kv_scales<false>(c, h, meta);
          next = kv_pages(c, s, n + 32 + lane < steps, base_of(min(n + 32 + lane, steps)));
        }
        if ((n & 31) == 16) kv_scales<false>(c, h, next);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) raw[t][i] = ahead[t][i];
        if (n + 1 < steps) fetch(n + 1, ((n + 1) & 31) == 0 ? next : meta);
        const int page = __shfl_sync(0xffffffffu, meta.page, n & 31);
        const float ks = __shfl_sync(0xffffffffu, meta.ks, n & 31);
        const int j0 = base_of(n);
        if (page < 0 || j0 > chunk.last) continue;
        uint32_t b[2][D / 16][2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) codes_to_half<FMT>(word_of(raw[t][kk >> 2], kk & 3), b[t][kk][0], b[t][kk][1]);
        float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        for (int mt = 0; mt < tiles; ++mt) {
          float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint4 a = sq[(mt * (D / 16) + kk) * 32 + lane];
            mma16816(x[0], a, b[0][kk][0], b[0][kk][1]);
            mma16816(x[1], a, b[1][kk][0], b[1][kk][1]);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = mt * 16 + 8 * e + g, pos = spos[row];
            const float f = sf[row] * ks, z = sz[row];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const float w = ex2(x[t][2 * e + y] * f - z);
                if (kv_sees(p.mask, pos, j0 + 8 * t + 2 * q4 + y)) sum[t][y] += w;
              }
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float v = sum[t][y];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            const int j = j0 + 8 * t + 2 * q4 + y;
            if (g == 0 && j <= chunk.last) score[j] += v;
          }
      }
    }
    left -= i1 - i0;
    off += i1 - i0;
    if (off == static_cast<int64_t>(span.n) * c.heads) {
      ++s;
      off = 0;
    }
  }
}

}  // namespace

cudaError_t launch_kv_score(const KvAttnParams& p, const LaunchCfg& cfg) {
  const int64_t steps = std::max<int64_t>(
      static_cast<int64_t>(p.c.S) * p.c.heads * (((static_cast<int64_t>(p.c.width) << p.c.tshift) + 15) / 16), 1);
  const int64_t blocks = std::min<int64_t>(cfg.sms * 2, (steps + kWarps - 1) / kWarps);
  auto kern = p.c.D == 128 ? (p.c.fmt == kKvInt8 ? kv_score_kernel<128, kKvInt8> : kv_score_kernel<128, kKvE4m3>)
                           : (p.c.fmt == kKvInt8 ? kv_score_kernel<64, kKvInt8> : kv_score_kernel<64, kKvE4m3>);
  return launch_kernel(kern, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0, cfg, p);
}

}  // namespace bolt
