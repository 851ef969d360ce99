// KvAppend and KvRead: writing and reading the paged 8-bit key/value cache (layout in kv.h).
//
// KvAppend quantises the rows of a call into their pages.  For each (page, head) that takes new rows:
//   s' = max(s, max|x| / Q)    over the new finite values x; s = the page's scale if it holds
//                              positions before the call's first, else 0; Q = 127 (int8), 448 (e4m3)
//   new codes = round(x / s'); the page's older codes become round(c * (s / s')) where s' > s
// A page's scale never shrinks, so its older codes are rewritten only when a new value is larger
// than all before it.  Infinities and NaN do not count towards the scale: they are stored as
// +-Q * s' and 0, and leave the rest of the page as it is.
//
// Both are streams of HBM bytes (append 2 in, 1 out a value; read 1 in, 2 out).  KvAppend gives a block the
// new rows of one (page, head), which it holds in registers between the maximum and the rounding, so each
// value is read once.  2 sequences of 6,000 rows, 8 heads of 128 values, K and V: 38 us to write and read them
// back.  KvAppend by itself takes 24, bound by the instructions of the rounding (2.7 issued a cycle; 29 us with a
// division a value); KvRead goes at HBM's rate.  One row of each of 64 sequences: 10 us, latency.
#include "kv.cuh"

namespace bolt {

namespace {

constexpr int kThreads = 256;

// max over the block of a value that is not negative (NaN, if any is), for every thread
__device__ __forceinline__ float block_max(float v, float* red) {
  // of such values the bits are in their order, and NaN's the largest
  unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
  __syncthreads();  // red may hold an earlier maximum
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(m);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max(m, __float_as_uint(red[w]));
  return __uint_as_float(m);
}

__device__ __forceinline__ void unpack4(uint32_t a, uint32_t b, float (&x)[4]) {
  x[0] = __uint_as_float(a << 16);
  x[1] = __uint_as_float(a & 0xFFFF0000u);
  x[2] = __uint_as_float(b << 16);
  x[3] = __uint_as_float(b & 0xFFFF0000u);
}

// Codes of four finite bf16 values of at most Q * s, by the definition round(x / s), where they are the same at
// x * lo and x * hi, lo and hi being 1 / s less and more 2^-21 of it: x / s and its rounding to fp32 lie
// between.  Otherwise (a value that close to a tie; rare) sets bits of `near`.  A division for every value
// takes several times the operations, and these are what bounds the kernel.
template <int FMT>
__device__ __forceinline__ uint32_t quantise4(uint32_t a, uint32_t b, float lo, float hi, uint32_t& near) {
  float x[4];
  unpack4(a, b, x);
  if constexpr (FMT == kKvInt8) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // 1.5 * 2^23 more: the low byte is the rounded value
      c[e] = __float_as_uint(fmaf(x[e], lo, 12582912.f));
      near |= c[e] ^ __float_as_uint(fmaf(x[e], hi, 12582912.f));
    }
    return prmt(prmt(c[0], c[1], 0x0040u), prmt(c[2], c[3], 0x0040u), 0x5410u) ^ 0x80808080u;
  } else {
    float y[4], z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = x[e] * lo;
      z[e] = x[e] * hi;
    }
    const uint32_t c = kv_encode4_finite<FMT>(y);
    near |= c ^ kv_encode4_finite<FMT>(z);
    return c;
  }
}

// ... and by the division itself; any x.
template <int FMT>
__device__ __forceinline__ uint32_t divide4(uint32_t a, uint32_t b, float s) {
  float x[4];
  unpack4(a, b, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = s > 0.f ? x[e] / s : 0.f;
  return kv_encode4<FMT>(x);
}

struct AppendParams {
  KvCache c;
  KvRows rows;
  const bf16 *k, *v;
  int64_t k_seq, k_row, v_seq, v_row;
  int blocks;  // most pages that a sequence's rows touch
};

// one block per (sequence, touched page, head, K or V); a thread holds up to NV vectors of 8 values
template <int FMT, int NV>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendParams p) {
  __shared__ float red[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  unsigned u = blockIdx.x;
  const bool is_v = u & 1;
  u >>= 1;
  const int h = static_cast<int>(u % c.heads);
  u /= c.heads;
  const int s = static_cast<int>(u / p.blocks), b = static_cast<int>(u - s * p.blocks);
  const KvSeq q = kv_seq(c, p.rows.start, p.rows.lens, s);
  const int end = static_cast<int>(min(static_cast<int64_t>(q.len), static_cast<int64_t>(q.start) + p.rows.R));
  const int blk = (q.start >> c.tshift) + b;
  const int lo = blk << c.tshift;
  if (q.start >= end || lo >= end) return;
  const int hi = min(lo + c.T, end), first = max(lo, q.start);
  const int64_t row_stride = is_v ? p.v_row : p.k_row;
  const bf16* src = (is_v ? p.v : p.k) + s * (is_v ? p.v_seq : p.k_seq) + static_cast<int64_t>(h) * c.D +
                    (first - q.start) * row_stride;
  const int shift = c.D == 128 ? 4 : 3, n = (hi - first) << shift;  // vectors of 8 values
  uint4 x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * kThreads;
    x[i] = make_uint4(0, 0, 0, 0);
    if (at < n) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + (at >> shift) * row_stride) + (at & ((1 << shift) - 1)));
  }
  const int page = kv_page(c.table, c.width, c.pages, s, blk);
  if (page < 0) return;
  const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
  uint8_t* codes = (is_v ? c.v : c.k) + unit * c.T * c.D;
  float* scale = (is_v ? c.vs : c.ks) + unit;
  const float before = lo < q.start ? *scale : 0.f;
  __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t a = w[e] & 0x7FFF7FFFu;
      top = __hmax2_nan(top, *reinterpret_cast<const __nv_bfloat162*>(&a));
    }
  }
  float amax = block_max(__bfloat162float(__hmax_nan(top.x, top.y)), red);
  const bool odd = !(amax < INFINITY);  // an infinity or a NaN among the values: the largest of the others
  if (odd) {
    amax = 0.f;
#pragma unroll 1
    for (int i = threadIdx.x; i < n * 8; i += kThreads) {
      const float a = fabsf(__bfloat162float(src[(i >> (shift + 3)) * row_stride + (i & ((8 << shift) - 1))]));
      if (a < INFINITY) amax = fmaxf(amax, a);
    }
    amax = block_max(amax, red);
  }
  const float after = fmaxf(before, amax / kv_qmax<FMT>());
  if (threadIdx.x == 0) *scale = after;  // every thread has read it: block_max has a barrier
  if (first > lo && after > before) {
    const float ratio = before / after;
    uint4* w = reinterpret_cast<uint4*>(codes);
    for (int i = threadIdx.x; i < (first - lo) * c.D / 16; i += kThreads) {
      const uint4 y = w[i];
      w[i] = make_uint4(kv_rescale4<FMT>(y.x, ratio), kv_rescale4<FMT>(y.y, ratio), kv_rescale4<FMT>(y.z, ratio),
                        kv_rescale4<FMT>(y.w, ratio));
    }
  }
  uint2* out = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(first - lo) * c.D);
  const bool exact = odd || !(after >= 0x1p-100f);  // every value by division
  const float inv = 1.f / after, inv_lo = inv * (1.f - 0x1p-21f), inv_hi = inv * (1.f + 0x1p-21f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * kThreads;
    if (at >= n) break;
    uint32_t near = exact;
    uint2 y;
    y.x = quantise4<FMT>(x[i].x, x[i].y, inv_lo, inv_hi, near);
    y.y = quantise4<FMT>(x[i].z, x[i].w, inv_lo, inv_hi, near);
    if (near) {
      y.x = divide4<FMT>(x[i].x, x[i].y, after);
      y.y = divide4<FMT>(x[i].z, x[i].w, after);
    }
    out[at] = y;
  }
}

// Block y: a sequence.  A thread takes 16 values of a (row, head), of K and of V.
template <int FMT>
__global__ void __launch_bounds__(kThreads, 8) kv_read_kernel(const KvCache c, const KvRows rows, bf16* k, bf16* v) {
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, shift = c.D == 128 ? 3 : 2;
  const KvSeq q = kv_seq(c, rows.start, rows.lens, s);
  const int64_t n = static_cast<int64_t>(rows.R) * c.heads << shift;  // vectors of the sequence
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (at >= n) return;
  const int64_t rh = at >> shift;
  const int r = rh <= 0x7fffffff ? static_cast<int>(static_cast<unsigned>(rh) / static_cast<unsigned>(c.heads))
                                 : static_cast<int>(rh / c.heads);
  const int h = static_cast<int>(rh - static_cast<int64_t>(r) * c.heads);
  const int64_t pos = static_cast<int64_t>(q.start) + r;
  uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  float sc[2] = {0.f, 0.f};  // also where there is nothing to read
  const int page = pos < q.len ? kv_page(c.table, c.width, c.pages, s, static_cast<int>(pos >> c.tshift)) : -1;
  if (page >= 0) {
    const int64_t unit = static_cast<int64_t>(page) * c.heads + h;
    const int64_t from = ((unit << c.tshift) + (pos & (c.T - 1))) * c.D + (at & ((1 << shift) - 1)) * 16;
    x[0] = *reinterpret_cast<const uint4*>(c.k + from);
    x[1] = *reinterpret_cast<const uint4*>(c.v + from);
    sc[0] = c.ks[unit];
    sc[1] = c.vs[unit];
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const uint32_t w[4] = {x[kv].x, x[kv].y, x[kv].z, x[kv].w};
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float z[4];
      kv_decode4<FMT>(w[e], z);
      const __nv_bfloat162 a = __floats2bfloat162_rn(z[0] * sc[kv], z[1] * sc[kv]);
      const __nv_bfloat162 b = __floats2bfloat162_rn(z[2] * sc[kv], z[3] * sc[kv]);
      y[2 * e] = *reinterpret_cast<const uint32_t*>(&a);
      y[2 * e + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
    uint4* out = reinterpret_cast<uint4*>((kv ? v : k) + (static_cast<int64_t>(s) * n + at) * 16);
    __stcs(out, make_uint4(y[0], y[1], y[2], y[3]));
    __stcs(out + 1, make_uint4(y[4], y[5], y[6], y[7]));
  }
}

template <int FMT>
cudaError_t append(const AppendParams& p, unsigned grid, const LaunchCfg& cfg) {
  const int per_thread = (p.c.T * p.c.D / 8 + kThreads - 1) / kThreads;  // vectors of a page: 1 .. 16
  auto kern = per_thread <= 1   ? kv_append_kernel<FMT, 1>
              : per_thread <= 2 ? kv_append_kernel<FMT, 2>
              : per_thread <= 4 ? kv_append_kernel<FMT, 4>
              : per_thread <= 8 ? kv_append_kernel<FMT, 8>
                                : kv_append_kernel<FMT, 16>;
  return launch_kernel(kern, dim3(grid), dim3(kThreads), 0, cfg, p);
}

}  // namespace

cudaError_t launch_kv_append(const KvCache& c, const KvRows& rows, const bf16* k, int64_t k_seq, int64_t k_row,
                             const bf16* v, int64_t v_seq, int64_t v_row, const LaunchCfg& cfg) {
  AppendParams p{c, rows, k, v, k_seq, k_row, v_seq, v_row, 0};
  // a first row in the last slot of its page touches the most
  p.blocks = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(rows.R) + c.T - 2) / c.T + 1, c.width));
  const int64_t grid = static_cast<int64_t>(c.S) * p.blocks * c.heads * 2;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const unsigned n = static_cast<unsigned>(grid);
  return c.fmt == kKvInt8 ? append<kKvInt8>(p, n, cfg) : append<kKvE4m3>(p, n, cfg);
}

cudaError_t launch_kv_read(const KvCache& c, const KvRows& rows, bf16* k, bf16* v, const LaunchCfg& cfg) {
  const int64_t n = static_cast<int64_t>(rows.R) * c.heads * (c.D >> 4);
  const int64_t grid = (n + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_kernel(c.fmt == kKvInt8 ? kv_read_kernel<kKvInt8> : kv_read_kernel<kKvE4m3>,
                       dim3(static_cast<unsigned>(grid), static_cast<unsigned>(c.S)), dim3(kThreads), 0, cfg, c, rows, k, v);
}

}  // namespace bolt
