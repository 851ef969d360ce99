// Device helpers of the paged 8-bit key/value cache.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "kv.h"

namespace bolt {

template <int FMT>
__device__ __forceinline__ constexpr float kv_qmax() {
  return FMT == kKvInt8 ? 127.f : 448.f;
}

// The values (in units of the scale) of a word's four codes, exact.
template <int FMT>
__device__ __forceinline__ void kv_decode4(uint32_t w, float (&x)[4]) {
  if constexpr (FMT == kKvInt8) {
    // a byte under the exponent of 2^23 is 2^23 + code
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(prmt(w, 0x4B000000u, 0x7440u + e)) - 8388736.f;  // 2^23 + 128
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const __half2 h(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * e)), __NV_E4M3));
      x[2 * e] = __low2float(h);
      x[2 * e + 1] = __high2float(h);
    }
  }
}

// The codes nearest to x (in units of the scale; finite), ties to even.
template <int FMT>
__device__ __forceinline__ uint32_t kv_encode4_finite(const float (&x)[4]) {
  if constexpr (FMT == kKvInt8) {
    // adding 1.5 * 2^23 rounds to a whole number, which the low byte then holds; 128 more for the offset
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(fminf(fmaxf(x[e], -127.f), 127.f) + 12582912.f);
    return prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u) ^ 0x80808080u;
  } else {
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3)) << 16;
  }
}

// The same of any x: infinities give the largest codes, NaN the code of 0.
template <int FMT>
__device__ __forceinline__ uint32_t kv_encode4(const float (&x)[4]) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = x[e] != x[e] ? 0.f : x[e];
  return kv_encode4_finite<FMT>(y);
}

// A word's codes at ratio times their values.
template <int FMT>
__device__ __forceinline__ uint32_t kv_rescale4(uint32_t w, float ratio) {
  float x[4];
  kv_decode4<FMT>(w, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] *= ratio;
  return kv_encode4<FMT>(x);
}

// Length of sequence s, and the position of its first row (the length, where it would lie beyond).
// Values that the table cannot hold leave the sequence empty and set a status bit.
struct KvSeq {
  int start, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvCache& c, const int* start, const int* lens, int s) {
  KvSeq q{start ? start[s] : 0, lens[s]};
  if (q.len < 0 || q.len > (static_cast<int64_t>(c.width) << c.tshift) || q.start < 0) {
    set_status(kStatusKvRange);
    q = KvSeq{0, 0};
  }
  q.start = min(q.start, q.len);
  return q;
}

// Page of a sequence's block b, or -1 (and a status bit) where the table names none of the cache's.
__device__ __forceinline__ int kv_page(const int* table, int width, int64_t pages, int s, int b) {
  const int page = table[static_cast<int64_t>(s) * width + b];
  if (static_cast<unsigned>(page) < static_cast<uint64_t>(pages)) return page;
  set_status(kStatusKvPage);
  return -1;
}

__device__ __forceinline__ bool kv_sees(const KvMask& m, int pos, int j) {
  return j <= pos && (m.window == 0 || j > pos - m.window || j < m.sinks);
}

}  // namespace bolt
