// KvAttention and KvScore over the paged 8-bit key/value cache (layout in kv.h).
//
//   l_j = scale * q . k_j over the positions j that the row sees;  lse = log sum_j exp(l_j)
//   KvAttention: o = sum_j exp(l_j - lse) v_j (bf16) and lse (f32); a row that sees nothing gives 0 and -inf
//   KvScore:     score[j] += sum over the rows and query heads of a kv head of exp(l_j - lse)
#include "kv.cuh"

namespace bolt {

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

// One block per (sequence, row, query head); a warp takes every fourth position, a lane D / 32 values.
template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) kv_attention_kernel(const KvAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float so[kWarps][D];
  __shared__ float sm[kWarps], sl[kWarps];
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  int64_t u = blockIdx.x;
  const int hq = static_cast<int>(u % p.Hq);
  u /= p.Hq;
  const int r = static_cast<int>(u % p.rows.R), s = static_cast<int>(u / p.rows.R), h = hq / p.G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const KvSeq seq = kv_seq(c, p.rows.start, p.rows.lens, s);
  const int64_t at = static_cast<int64_t>(seq.start) + r;
  const int pos = at < seq.len ? static_cast<int>(at) : -1;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[s * p.qs + r * p.qr + static_cast<int64_t>(hq) * D + lane * E + e]);
    acc[e] = 0.f;
  }
  for (int j = warp; j <= pos; j += kWarps) {
    if (!kv_sees(p.mask, pos, j)) continue;
    const int page = kv_page(c.table, c.width, c.pages, s, j >> c.tshift);
    if (page < 0) continue;
    const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
    const int64_t base = (unit * c.T + (j & (c.T - 1))) * D + lane * E;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dot += q[e] * kv_decode<FMT>(c.k[base + e]);
    const float t = warp_sum(dot) * (c.ks[unit] * p.scale * kLog2e);
    const float m2 = fmaxf(m, t), alpha = exp2f(m - m2), w = exp2f(t - m2);
    m = m2;
    l = l * alpha + w;
    const float wv = w * c.vs[unit];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * alpha + wv * kv_decode<FMT>(c.v[base + e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = acc[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  float top = sm[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += sl[w] * exp2f(sm[w] - ref);
  const int64_t row = (static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + hq;
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x += so[w][d] * exp2f(sm[w] - ref);
    p.o[row * D + d] = __float2bfloat16(total > 0.f ? x / total : 0.f);
  }
  if (threadIdx.x == 0) p.lse[row] = (top + log2f(total)) / kLog2e;
}

// One warp per (sequence, kv head, position).
template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32) kv_score_kernel(const KvAttnParams p) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * kWarps + warp, h = blockIdx.y;
  for (int s = blockIdx.z; s < c.S; s += gridDim.z) {
    const KvSeq seq = kv_seq(c, p.rows.start, p.rows.lens, s);
    if (j >= seq.len || j >= p.score_width) continue;
    const int page = kv_page(c.table, c.width, c.pages, s, j >> c.tshift);
    if (page < 0) continue;
    const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
    const int64_t base = (unit * c.T + (j & (c.T - 1))) * D + lane * E;
    float k[E], sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) k[e] = kv_decode<FMT>(c.k[base + e]);
    const float f = c.ks[unit] * p.scale * kLog2e;
    for (int r = 0; r < p.rows.R && seq.start + r < seq.len; ++r) {
      if (!kv_sees(p.mask, seq.start + r, j)) continue;
      for (int g = 0; g < p.G; ++g) {
        const int hq = h * p.G + g;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
          dot += k[e] * __bfloat162float(p.q[s * p.qs + r * p.qr + static_cast<int64_t>(hq) * D + lane * E + e]);
        const float z = p.lse[(static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + hq];
        sum += exp2f(warp_sum(dot) * f - z * kLog2e);
      }
    }
    if (lane == 0) p.score[(static_cast<int64_t>(s) * c.heads + h) * p.score_width + j] += sum;
  }
}

}  // namespace

cudaError_t launch_kv_attention(const KvAttnParams& p, const LaunchCfg& cfg) {
  const int64_t grid = static_cast<int64_t>(p.c.S) * p.rows.R * p.Hq;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  auto kern = p.c.D == 128 ? (p.c.fmt == kKvInt8 ? kv_attention_kernel<128, kKvInt8> : kv_attention_kernel<128, kKvE4m3>)
                           : (p.c.fmt == kKvInt8 ? kv_attention_kernel<64, kKvInt8> : kv_attention_kernel<64, kKvE4m3>);
  return launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(kWarps * 32), 0, cfg, p);
}

cudaError_t launch_kv_score(const KvAttnParams& p, const LaunchCfg& cfg) {
  const int64_t n = std::min<int64_t>(static_cast<int64_t>(p.c.width) << p.c.tshift, p.score_width);
  const dim3 grid(static_cast<unsigned>((n + kWarps - 1) / kWarps), static_cast<unsigned>(p.c.heads),
                  static_cast<unsigned>(std::min(p.c.S, 65535)));
  auto kern = p.c.D == 128 ? (p.c.fmt == kKvInt8 ? kv_score_kernel<128, kKvInt8> : kv_score_kernel<128, kKvE4m3>)
                           : (p.c.fmt == kKvInt8 ? kv_score_kernel<64, kKvInt8> : kv_score_kernel<64, kKvE4m3>);
  return launch_kernel(kern, grid, dim3(kWarps * 32), 0, cfg, p);
}

}  // namespace bolt
