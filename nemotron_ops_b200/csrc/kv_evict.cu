// KvEvict: keep the `keep` most attended positions of every (sequence, kv head) and lay their codes
// out in pages of their own (cache layout in kv.h).
//
// A sequence of n <= keep positions keeps all of them.  Otherwise each of its heads keeps the first
// `sinks` positions, the last `recent`, and of the rest those with the largest accumulated weights
// (KvScore), the lower position first where two are equal; a NaN ranks above every number.  Kept
// positions stay in order.  A new page's scale is the largest of its positions' old scales s', and a
// code c of a position with scale s becomes round(c * (s / s')), so codes whose scale is the page's
// largest stay as they are.
//
// Two kernels: one block per (sequence, head) selects and compacts, then one block per (sequence,
// new page, head, K or V) moves the codes.
#include "kv.cuh"

namespace bolt {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 128;

// A weight's rank as an unsigned number: larger weights larger, NaN the largest, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// exclusive prefix of (a, b) over the block, and their totals; every thread calls it
__device__ __forceinline__ int2 block_prefix(int a, int b, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int px = __shfl_up_sync(0xffffffffu, x, o), py = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += px;
      y += py;
    }
  }
  __syncthreads();  // warp_sums may hold an earlier call's values
  if (lane == 31) warp_sums[warp] = make_int2(x, y);
  __syncthreads();
  int2 before = make_int2(0, 0);
  total = make_int2(0, 0);
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const int2 t = warp_sums[w];
    if (w < warp) {
      before.x += t.x;
      before.y += t.y;
    }
    total.x += t.x;
    total.y += t.y;
  }
  return make_int2(before.x + x - a, before.y + y - b);
}

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const KvEvictParams p) {
  __shared__ int hist[256];
  __shared__ int2 sums[kSelThreads / 32];
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const KvSeq seq = kv_seq(p.c, nullptr, p.lens, s);
  const int n = min(static_cast<int64_t>(seq.len), p.score_width);
  const int64_t unit = static_cast<int64_t>(s) * p.c.heads + h;
  const float* score = p.score + unit * p.score_width;
  int* kept = p.kept + unit * p.keep;
  float* out = p.new_score + unit * p.keep;
  if (h == 0 && tid == 0) p.new_lens[s] = min(n, p.keep);
  if (n <= p.keep) {
    for (int i = tid; i < p.keep; i += kSelThreads) {
      kept[i] = i < n ? i : -1;
      out[i] = i < n ? score[i] : 0.f;
    }
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;
  int left = p.keep - p.sinks - p.recent;  // positions to take of [lo, hi)
  // the left-th largest rank, eight bits at a time: `cut` holds the bits found so far
  uint32_t cut = 0;
  for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const uint32_t r = rank_of(score[i]);
      if (shift == 24 || (r >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&hist[(r >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, need = left;
      while (d > 0 && need > hist[d]) need -= hist[d--];
      s_digit = d;
      s_left = need;
    }
    __syncthreads();
    cut |= s_digit << shift;
    left = s_left;
  }
  // all ranks above `cut` are kept, and the first `left` that equal it
  const bool some = p.keep > p.sinks + p.recent;
  const int per = (n + kSelThreads - 1) / kSelThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
  int above = 0, equal = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t r = rank_of(score[i]);
    const bool forced = i < lo || i >= hi;
    above += forced || (some && r > cut);
    equal += !forced && some && r == cut;
  }
  int2 total;
  const int2 before = block_prefix(above, equal, sums, total);
  int a = before.x, e = before.y;
  for (int i = i0; i < i1; ++i) {
    const float x = score[i];
    const uint32_t r = rank_of(x);
    const bool forced = i < lo || i >= hi;
    const bool up = forced || (some && r > cut), eq = !forced && some && r == cut;
    if (up || (eq && e < left)) {
      const int at = a + min(e, left);
      kept[at] = i;
      out[at] = x;
    }
    a += up;
    e += eq;
  }
}

template <int FMT>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const KvEvictParams p) {
  __shared__ int64_t src[256];  // byte offset of each slot's codes, -1 for none
  __shared__ float unit_of[256];
  __shared__ float red[kMoveThreads / 32];
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x;
  int64_t u = blockIdx.x;
  const bool is_v = u & 1;
  u >>= 1;
  const int h = static_cast<int>(u % c.heads);
  u /= c.heads;
  const int blocks = (p.keep + c.T - 1) >> c.tshift;
  const int b = static_cast<int>(u % blocks), s = static_cast<int>(u / blocks);
  const int n = min(p.new_lens[s] - (b << c.tshift), c.T);
  if (n <= 0) return;
  const int to = kv_page(p.new_table, p.new_width, c.pages, s, b);
  if (to < 0) return;
  const float* scale = is_v ? c.vs : c.ks;
  const uint8_t* codes = is_v ? c.v : c.k;
  const int* kept = p.kept + (static_cast<int64_t>(s) * c.heads + h) * p.keep + (static_cast<int64_t>(b) << c.tshift);
  float top = 0.f;
  for (int i = tid; i < n; i += kMoveThreads) {
    const int j = kept[i];
    const int page = kv_page(c.table, c.width, c.pages, s, j >> c.tshift);
    const int64_t from = static_cast<int64_t>(page) * c.heads + h;
    src[i] = page < 0 ? -1 : (from * c.T + (j & (c.T - 1))) * c.D;
    unit_of[i] = page < 0 ? 0.f : scale[from];
    top = fmaxf(top, unit_of[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMoveThreads / 32; ++w) top = fmaxf(top, red[w]);
  const int64_t dst = static_cast<int64_t>(to) * c.heads + h;
  if (tid == 0) (is_v ? c.vs : c.ks)[dst] = top;
  uint8_t* out = (is_v ? c.v : c.k) + dst * c.T * c.D;
  const int vecs = c.D >> 4;  // 16 codes a vector
  for (int i = tid; i < n * vecs; i += kMoveThreads) {
    const int t = i / vecs, d = (i % vecs) * 16;
    const float unit = unit_of[t];
    uint4 x = src[t] < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(codes + src[t] + d);
    if (unit != top || src[t] < 0) {
      const float ratio = top > 0.f ? unit / top : 0.f;
      uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t y = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) y |= kv_encode<FMT>(kv_decode<FMT>((w[k] >> (8 * e)) & 255) * ratio) << (8 * e);
        w[k] = y;
      }
      x = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(out + static_cast<int64_t>(t) * c.D + d) = x;
  }
}

}  // namespace

cudaError_t launch_kv_evict(const KvEvictParams& p, const LaunchCfg& cfg) {
  const KvCache& c = p.c;
  cudaError_t e = launch_kernel(kv_select_kernel, dim3(static_cast<unsigned>(c.heads), static_cast<unsigned>(c.S)),
                                dim3(kSelThreads), 0, cfg, p);
  if (e != cudaSuccess) return e;
  LaunchCfg c2 = cfg;
  c2.pdl = true;  // same op: the kernel waits for its predecessor with griddepcontrol.wait
  const int64_t grid = static_cast<int64_t>(c.S) * ((p.keep + c.T - 1) / c.T) * c.heads * 2;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return launch_kernel(c.fmt == kKvInt8 ? kv_move_kernel<kKvInt8> : kv_move_kernel<kKvE4m3>,
                       dim3(static_cast<unsigned>(grid)), dim3(kMoveThreads), 0, c2, p);
}

}  // namespace bolt
