// KvAppend and KvRead: writing and reading the paged 8-bit key/value cache (layout in kv.h).
//
// KvAppend quantises the rows of a call into their pages.  For each (page, head) that takes new rows:
//   s' = max(s, max|x| / Q)    over the new finite values x; s = the page's scale if it holds
//                              positions before the call's first, else 0; Q = 127 (int8), 448 (e4m3)
//   new codes = round(x / s'); the page's older codes become round(c * (s / s')) where s' > s
// A page's scale never shrinks, so its older codes are rewritten only when a new value is larger
// than all before it.  Infinities and NaN do not count towards the scale: they are stored as
// +-Q * s' and 0, and leave the rest of the page as it is.
#include "kv.cuh"

namespace bolt {

namespace {

constexpr int kThreads = 128;

// max over the block of a non-negative value, for every thread
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, red[w]);
  return v;
}

struct AppendParams {
  KvCache c;
  KvRows rows;
  const bf16 *k, *v;
  int64_t k_seq, k_row, v_seq, v_row;
  int blocks;  // most pages that a sequence's rows touch
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// one block per (sequence, touched page, head, K or V)
template <int FMT>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendParams p) {
  __shared__ float red[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  int64_t u = blockIdx.x;
  const bool is_v = u & 1;
  u >>= 1;
  const int h = static_cast<int>(u % c.heads);
  u /= c.heads;
  const int b = static_cast<int>(u % p.blocks), s = static_cast<int>(u / p.blocks);
  const KvSeq q = kv_seq(c, p.rows.start, p.rows.lens, s);
  const int end = min(static_cast<int64_t>(q.len), static_cast<int64_t>(q.start) + p.rows.R);
  const int blk = (q.start >> c.tshift) + b;
  const int lo = blk << c.tshift;
  if (q.start >= end || lo >= end) return;
  const int page = kv_page(c.table, c.width, c.pages, s, blk);
  if (page < 0) return;
  const int hi = min(lo + c.T, end), first = max(lo, q.start);
  const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
  uint8_t* codes = (is_v ? c.v : c.k) + unit * c.T * c.D;
  float* scale = (is_v ? c.vs : c.ks) + unit;
  const bf16* src = (is_v ? p.v : p.k) + s * (is_v ? p.v_seq : p.k_seq) + static_cast<int64_t>(h) * c.D;
  const int64_t row_stride = is_v ? p.v_row : p.k_row;
  const int vecs = c.D >> 3;  // vectors of 8 values a row
  float amax = 0.f;
  for (int i = threadIdx.x; i < (hi - first) * vecs; i += kThreads) {
    const int r = first - q.start + i / vecs, d = (i % vecs) * 8;
    float x[8];
    unpack8(*reinterpret_cast<const uint4*>(src + r * row_stride + d), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(x[e]);
      if (a < INFINITY) amax = fmaxf(amax, a);
    }
  }
  const float before = lo < q.start ? *scale : 0.f;
  amax = block_max(amax, red);
  const float after = fmaxf(before, amax / kv_qmax<FMT>());
  if (threadIdx.x == 0) *scale = after;
  if (first > lo && after > before) {
    const float ratio = before / after;
    uint32_t* w = reinterpret_cast<uint32_t*>(codes);
    for (int i = threadIdx.x; i < (first - lo) * c.D / 4; i += kThreads) {
      const uint32_t x = w[i];
      uint32_t y = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) y |= kv_encode<FMT>(kv_decode<FMT>((x >> (8 * e)) & 255) * ratio) << (8 * e);
      w[i] = y;
    }
  }
  for (int i = threadIdx.x; i < (hi - first) * vecs; i += kThreads) {
    const int t = first + i / vecs, d = (i % vecs) * 8;
    float x[8];
    unpack8(*reinterpret_cast<const uint4*>(src + (t - q.start) * row_stride + d), x);
    uint32_t y[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e >> 2] |= kv_encode<FMT>(after > 0.f ? x[e] / after : 0.f) << (8 * (e & 3));
    *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(t - lo) * c.D + d) = make_uint2(y[0], y[1]);
  }
}

// one thread per 8 values of a (sequence, row, head)
template <int FMT>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvCache c, const KvRows rows, bf16* k, bf16* v,
                                                           int64_t n) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const int vecs = c.D >> 3;
  int64_t u = i;
  const int d = static_cast<int>(u % vecs) * 8;
  u /= vecs;
  const int h = static_cast<int>(u % c.heads);
  u /= c.heads;
  const int r = static_cast<int>(u % rows.R), s = static_cast<int>(u / rows.R);
  const KvSeq q = kv_seq(c, rows.start, rows.lens, s);
  const int64_t pos = static_cast<int64_t>(q.start) + r;
  const int page = pos < q.len ? kv_page(c.table, c.width, c.pages, s, static_cast<int>(pos >> c.tshift)) : -1;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint4 out = make_uint4(0, 0, 0, 0);
    if (page >= 0) {
      const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
      const float sc = (kv ? c.vs : c.ks)[unit];
      const uint2 x = *reinterpret_cast<const uint2*>((kv ? c.v : c.k) + (unit * c.T + (pos & (c.T - 1))) * c.D + d);
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = (e < 2 ? x.x : x.y) >> (16 * (e & 1));
        const __nv_bfloat162 pair =
            __floats2bfloat162_rn(kv_decode<FMT>(w & 255) * sc, kv_decode<FMT>((w >> 8) & 255) * sc);
        y[e] = *reinterpret_cast<const uint32_t*>(&pair);
      }
      out = make_uint4(y[0], y[1], y[2], y[3]);
    }
    *reinterpret_cast<uint4*>((kv ? v : k) + i * 8) = out;
  }
}

}  // namespace

cudaError_t launch_kv_append(const KvCache& c, const KvRows& rows, const bf16* k, int64_t k_seq, int64_t k_row,
                             const bf16* v, int64_t v_seq, int64_t v_row, const LaunchCfg& cfg) {
  AppendParams p{c, rows, k, v, k_seq, k_row, v_seq, v_row, 0};
  // a first row in the last slot of its page touches the most
  p.blocks = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(rows.R) + c.T - 2) / c.T + 1, c.width));
  const int64_t grid = static_cast<int64_t>(c.S) * p.blocks * c.heads * 2;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_kernel(c.fmt == kKvInt8 ? kv_append_kernel<kKvInt8> : kv_append_kernel<kKvE4m3>,
                       dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, cfg, p);
}

cudaError_t launch_kv_read(const KvCache& c, const KvRows& rows, bf16* k, bf16* v, const LaunchCfg& cfg) {
  const int64_t n = static_cast<int64_t>(c.S) * rows.R * c.heads * (c.D >> 3);
  const int64_t grid = (n + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_kernel(c.fmt == kKvInt8 ? kv_read_kernel<kKvInt8> : kv_read_kernel<kKvE4m3>,
                       dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, cfg, c, rows, k, v, n);
}

}  // namespace bolt
