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
// Two kernels.  Selection, one block per (sequence, head): the weights go to shared memory once (up to
// kSelKeys positions), the cut is found eleven bits at a time by histograms, and the kept positions are
// written in order.  Then the codes move, one block per (sequence, head, 128 positions or one page of 256):
// look-ups of positions, pages and scales serve K and V, and the copies are 16 bytes a thread.  32 sequences of
// 4,096 positions cut to 1,000, 8 heads of 128 values: 22 us for the selection (passes over shared memory) and 31
// for the moves, 116 MB at 3.7 TB/s, which the instructions of the requantising bound (2.3 issued a cycle, the ALU
// busy half the time).  One of 20,000, cut to 8,192, 2 heads: the selection takes 29 us, on two SMs, and the moves
// 13, latency; a split of the selection over more SMs would need an exchange of histograms in each pass.
#include "kv.cuh"

namespace bolt {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 48 * 1024;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

// A weight's rank as an unsigned number: larger weights larger, NaN the largest, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum of the first `warp` of 32 sums, one a warp of the block.
__device__ __forceinline__ unsigned sum_before(const unsigned* sums, int warp) {
  const int lane = threadIdx.x & 31;
  return __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0u);
}

// Of the 32-bit ranks get(i), lo <= i < hi: the left-th largest; `left` becomes the number of those equal
// to it that belong to the largest.  1 <= left <= hi - lo.
template <typename Get>
__device__ __forceinline__ uint32_t find_cut(Get&& get, int lo, int hi, int& left, unsigned* hist, unsigned* warp_sums,
                                             uint2* found) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t cut = 0, known = 0;  // the bits found so far, and which they are
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const uint32_t r = get(i);
      if ((r & known) == cut) atomicAdd(&hist[(r >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // thread t has the bins from the top: bins - 1 - 2 t and the one below
    const int top = bins - 1 - 2 * tid;
    const unsigned a = top >= 0 ? hist[top] : 0, b = top >= 1 ? hist[top - 1] : 0;
    unsigned sum = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    const unsigned before = sum - a - b + sum_before(warp_sums, warp);
    const unsigned need = static_cast<unsigned>(left);
    if (before < need && need <= before + a)
      *found = make_uint2(top, need - before);
    else if (before + a < need && need <= before + a + b)
      *found = make_uint2(top - 1, need - before - a);
    __syncthreads();
    cut |= found->x << shift;
    left = static_cast<int>(found->y);
    known |= static_cast<uint32_t>(bins - 1) << shift;
    __syncthreads();  // hist, warp_sums and found are written again
  }
  return cut;
}

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const KvEvictParams p, int key_room) {
  extern __shared__ float keys[];  // [key_room]
  __shared__ unsigned hist[kBins], warp_sums[kSelThreads / 32], above_sums[kSelThreads / 32], equal_sums[kSelThreads / 32];
  __shared__ uint2 found;
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const KvSeq seq = kv_seq(p.c, nullptr, p.lens, s);
  const int n = seq.len;  // at most width * T, which score_width covers
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
  const bool some = left > 0, in_smem = n <= key_room;
  if (in_smem) {
#pragma unroll 8
    for (int i = tid; i < n; i += kSelThreads) keys[i] = score[i];
    __syncthreads();
  }
  const auto weight = [&](int i) { return in_smem ? keys[i] : score[i]; };
  const auto get = [&](int i) { return rank_of(weight(i)); };
  const uint32_t cut = some ? find_cut(get, lo, hi, left, hist, warp_sums, &found) : 0;
  // every rank above `cut` is kept, and the first `left` equal to it; a warp takes consecutive positions
  const int per = ((n + kSelThreads - 1) / kSelThreads) * 32, i0 = min(warp * per, n), i1 = min(i0 + per, n);
  const auto class_of = [&](int i) {  // 2: kept, 1: equal to the cut
    if (i < lo || i >= hi) return 2;
    const uint32_t r = get(i);
    return some ? (r > cut ? 2 : r == cut ? 1 : 0) : 0;
  };
  int above = 0, equal = 0;
  for (int i = i0; i < i1; i += 32) {
    const int k = i + lane < i1 ? class_of(i + lane) : 0;
    above += __popc(__ballot_sync(0xffffffffu, k == 2));
    equal += __popc(__ballot_sync(0xffffffffu, k == 1));
  }
  if (lane == 0) {
    above_sums[warp] = above;
    equal_sums[warp] = equal;
  }
  __syncthreads();
  int a = sum_before(above_sums, warp), e = sum_before(equal_sums, warp);
  const unsigned lower = (1u << lane) - 1;
  for (int i = i0; i < i1; i += 32) {
    const int k = i + lane < i1 ? class_of(i + lane) : 0;
    const unsigned ma = __ballot_sync(0xffffffffu, k == 2), me = __ballot_sync(0xffffffffu, k == 1);
    const int my_e = e + __popc(me & lower);
    if (k == 2 || (k == 1 && my_e < left)) {
      const int at = a + __popc(ma & lower) + min(my_e, left);
      kept[at] = i + lane;
      out[at] = weight(i + lane);
    }
    a += __popc(ma);
    e += __popc(me);
  }
}

// Block: (sequence, head, group of `group` kept positions); group = max(T, 128) <= 256.
template <int FMT>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const KvEvictParams p, int groups) {
  __shared__ int64_t src[256];   // a slot's first code, -1: none
  __shared__ float ratio[2][256];
  __shared__ int top[2][8];      // the new pages' scales: the largest of their positions', as their bits
  __shared__ int to[8];          // the new pages
  pdl_wait();
  pdl_trigger();
  const KvCache& c = p.c;
  const int tid = threadIdx.x, group = max(c.T, 128);
  unsigned u = blockIdx.x;
  const int h = static_cast<int>(u % c.heads);
  u /= c.heads;
  const int s = static_cast<int>(u / groups), i0 = static_cast<int>(u - s * groups) * group;
  const int n = min(p.new_lens[s] - i0, group);
  if (n <= 0) return;
  const int pages = (n + c.T - 1) >> c.tshift;
  if (tid < 16) top[tid >> 3][tid & 7] = 0;
  if (tid < pages) to[tid] = kv_page(p.new_table, p.new_width, c.pages, s, (i0 >> c.tshift) + tid);
  float ks = 0.f, vs = 0.f;
  if (tid < n) {
    const int j = p.kept[(static_cast<int64_t>(s) * c.heads + h) * p.keep + i0 + tid];
    const int page = kv_page(c.table, c.width, c.pages, s, j >> c.tshift);
    const int64_t from = static_cast<int64_t>(page) * c.heads + h;
    src[tid] = page < 0 ? -1 : ((from << c.tshift) + (j & (c.T - 1))) * c.D;
    if (page >= 0) {
      ks = c.ks[from];
      vs = c.vs[from];
    }
  }
  __syncthreads();
  if (tid < n) {
    // scales are not negative, so their bits are in their order
    atomicMax(&top[0][tid >> c.tshift], ks > 0.f ? __float_as_int(ks) : 0);
    atomicMax(&top[1][tid >> c.tshift], vs > 0.f ? __float_as_int(vs) : 0);
  }
  __syncthreads();
  if (tid < n) {
    const float kt = __int_as_float(top[0][tid >> c.tshift]), vt = __int_as_float(top[1][tid >> c.tshift]);
    ratio[0][tid] = kt > 0.f ? ks / kt : 0.f;
    ratio[1][tid] = vt > 0.f ? vs / vt : 0.f;
  }
  if (tid < 2 * pages) {
    const int i = tid >> 1, kv = tid & 1;
    if (to[i] >= 0) (kv ? c.vs : c.ks)[static_cast<int64_t>(to[i]) * c.heads + h] = __int_as_float(top[kv][i]);
  }
  __syncthreads();
  const int shift = c.D == 128 ? 3 : 2, vecs = n << shift;  // 16 codes a vector
#pragma unroll 4
  for (int i = tid; i < 2 * vecs; i += kMoveThreads) {
    const bool is_v = i >= vecs;
    const int at = is_v ? i - vecs : i, t = at >> shift, d = (at & ((1 << shift) - 1)) * 16;
    const int page = to[t >> c.tshift];
    if (page < 0) continue;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (src[t] >= 0) x = *reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + src[t] + d);
    const float r = ratio[is_v][t];
    if (r != 1.f)
      x = make_uint4(kv_rescale4<FMT>(x.x, r), kv_rescale4<FMT>(x.y, r), kv_rescale4<FMT>(x.z, r),
                     kv_rescale4<FMT>(x.w, r));
    uint8_t* out = (is_v ? c.v : c.k) + (((static_cast<int64_t>(page) * c.heads + h) << c.tshift) + (t & (c.T - 1))) * c.D;
    *reinterpret_cast<uint4*>(out + d) = x;
  }
}

}  // namespace

cudaError_t launch_kv_evict(const KvEvictParams& p, const LaunchCfg& cfg) {
  const KvCache& c = p.c;
  const int group = std::max(c.T, 128), groups = (p.keep + group - 1) / group;
  const int64_t grid = static_cast<int64_t>(c.S) * groups * c.heads;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  // shared memory for the longest sequence of the table, as far as it goes
  const int room = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(c.width) << c.tshift, kSelKeys));
  static SmemOptIn opt;
  cudaError_t e = allow_smem(kv_select_kernel, room * sizeof(uint32_t), opt);
  if (e != cudaSuccess) return e;
  e = launch_kernel(kv_select_kernel, dim3(static_cast<unsigned>(c.heads), static_cast<unsigned>(c.S)),
                    dim3(kSelThreads), room * sizeof(uint32_t), cfg, p, room);
  if (e != cudaSuccess) return e;
  LaunchCfg c2 = cfg;
  c2.pdl = true;  // same op: the kernel waits for its predecessor with griddepcontrol.wait
  return launch_kernel(c.fmt == kKvInt8 ? kv_move_kernel<kKvInt8> : kv_move_kernel<kKvE4m3>,
                       dim3(static_cast<unsigned>(grid)), dim3(kMoveThreads), 0, c2, p, groups);
}

}  // namespace bolt
