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

// The value (in units of the scale) of a code.
template <int FMT>
__device__ __forceinline__ float kv_decode(uint32_t code) {
  if constexpr (FMT == kKvInt8) {
    return static_cast<float>(static_cast<int>(code) - 128);
  } else {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3)));
  }
}

// The code nearest to x (in units of the scale), ties to even; NaN gives the code of 0.
template <int FMT>
__device__ __forceinline__ uint32_t kv_encode(float x) {
  if constexpr (FMT == kKvInt8) {
    if (x != x) x = 0.f;
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f)) + 128);
  } else {
    if (x != x) x = 0.f;
    return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  }
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
