// What the attention kernels share: the parts of items that several blocks hold, and the writing of results.
#pragma once

#include "kv_mma.cuh"

namespace bolt {

// Weights are 2^(x - reference + kWeightLog) of their logits x, fp16 operands: at most 2^kWeightTop, and a row's
// largest at least 2^kWeightLog when its reference was last raised.
constexpr float kWeightLog = 8.f, kWeightTop = 15.f;

// A page's V scale is part of its positions' weights: its logarithm, to add to their logits, and the factor that
// takes it off again in the sums.  A scale of 0 counts as 2^-96 (its values are far below any others'); one that is
// not finite makes the logits NaN and leaves the factor finite, for the rows that do not see the page.
__device__ __forceinline__ float2 kv_v_scale(float scale) {
  const float s = fmaxf(scale, 0x1p-96f);
  return make_float2(scale < INFINITY ? log2f(s) : NAN, 1.f / s);
}

struct Split {  // segments of one item: the first in block `block`'s slot 2 block + 1, the i-th in 2 (block + i)
  int s, mb, h, block, parts;
};

struct Work {
  float* part;    // [2 blocks][rows of a block][D]
  float2* ml;     // [2 blocks][rows of a block]: max and sum
  Split* split;   // [splits]
  int splits;     // min(items, blocks): an entry an item, or an entry a block
  int row_blocks;
};

// Joins, for each of a segment's ROWS rows, the TW partial results in shared memory: sm the references, sl the
// sums, so [TW][ROWS][D / 4] the values, already on the scale of the row's largest reference, float4 f of row r
// at swizzle(r, f).  A segment that is a whole item writes the result; others leave their part in the workspace.
// All threads of the block, between barriers.
template <int D, int ROWS, int TW, int THREADS, typename Swz>
__device__ __forceinline__ void kv_finish(const KvAttnParams& p, const Work& w, const KvShare& share,
                                          const KvSegment& seg, const float* sm, const float* sl, const float4* so,
                                          Swz&& swizzle) {
  const int tid = threadIdx.x;
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G, G = p.G;
  const bool by_item = static_cast<int64_t>(p.c.S) * w.row_blocks * p.c.heads == w.splits, item = seg.whole_item();
  const int slot = 2 * blockIdx.x + (seg.i0 == 0);
  if (tid == 0 && seg.i0 == 0) {
    const int64_t at = by_item ? static_cast<int64_t>(seg.pair) * p.c.heads + seg.h : blockIdx.x;
    if (!item) {
      const int parts = share.cross ? static_cast<int>((seg.end - 1) / share.per) - static_cast<int>(blockIdx.x) + 1
                                    : static_cast<int>((seg.span.n + share.per - 1) / share.per);
      w.split[at] = Split{seg.s, seg.mb, seg.h, static_cast<int>(blockIdx.x), parts};
    } else if (by_item) {
      w.split[at].parts = 0;
    }
  }
  for (int e = tid; e < ROWS * (D / 8); e += THREADS) {
    const int row = e / (D / 8), f = 2 * (e % (D / 8));
    const unsigned m = seg.m0 + row;
    if (m >= M) break;
    float top = sm[row];
#pragma unroll
    for (int k = 1; k < TW; ++k) top = fmaxf(top, sm[k * ROWS + row]);
    float l = 0.f;
    float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < TW; ++k) {
      const float mk = sm[k * ROWS + row];
      if (mk != -INFINITY) l += sl[k * ROWS + row] * ex2(mk - top);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float4 z = so[(k * ROWS + row) * (D / 4) + swizzle(row, f + y)];
        v[y].x += z.x;
        v[y].y += z.y;
        v[y].z += z.z;
        v[y].w += z.w;
      }
    }
    if (item) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const unsigned r = m / G;
      const int64_t out = (static_cast<int64_t>(seg.s) * p.rows.R + r) * p.Hq + seg.h * G + (m - r * G);
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
      if (f == 0) p.lse[out] = l == 0.f ? -INFINITY : (top - kWeightLog + log2f(l)) * kLn2;
    } else {
      float4* to = reinterpret_cast<float4*>(w.part + (static_cast<int64_t>(slot) * ROWS + row) * D) + f;
      to[0] = v[0];
      to[1] = v[1];
      if (f == 0) w.ml[static_cast<int64_t>(slot) * ROWS + row] = make_float2(top, l);
    }
  }
}

// Before a block's segments: no item is split yet, and the rows of items without steps see nothing.
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ void kv_empty_items(const KvAttnParams& p, const Work& w) {
  const int tid = threadIdx.x, pairs = p.c.S * w.row_blocks;
  const unsigned M = static_cast<unsigned>(p.rows.R) * p.G, G = p.G;
  const bool by_item = static_cast<int64_t>(pairs) * p.c.heads == w.splits;
  if (!by_item && tid == 0) w.split[blockIdx.x].parts = 0;
  for (int i = blockIdx.x; i < pairs; i += gridDim.x) {
    const int s = i / w.row_blocks;
    const unsigned m0 = (i - s * w.row_blocks) * ROWS;
    if (kv_span(p, kv_seq(p.c, p.rows.start, p.rows.lens, s), m0, ROWS).n > 0) continue;
    const unsigned rows = min(M - m0, static_cast<unsigned>(ROWS)) * p.c.heads;
    for (unsigned e = tid; e < rows * (D / 8); e += THREADS) {
      const unsigned row = e / (D / 8), h = row % p.c.heads, m = m0 + row / p.c.heads, r = m / G;
      const int64_t out = (static_cast<int64_t>(s) * p.rows.R + r) * p.Hq + h * G + (m - r * G);
      reinterpret_cast<uint4*>(p.o + out * D)[e % (D / 8)] = make_uint4(0, 0, 0, 0);
      if (e % (D / 8) == 0) p.lse[out] = -INFINITY;
    }
    if (by_item)
      for (int h = tid; h < p.c.heads; h += THREADS) w.split[static_cast<int64_t>(i) * p.c.heads + h].parts = 0;
  }
}

// The kernel for more than 16 rows a kv head (kv_attention_umma.cu): 128 rows a block, one block an SM.
cudaError_t launch_kv_attention_umma(const KvAttnParams& p, const Work& w, unsigned blocks, const LaunchCfg& cfg);

}  // namespace bolt
