// KvAttention for more than 16 rows a kv head (drafted rows of large groups, chunks of prompts) on the
// 5th-generation tensor cores: 128 rows a block, tiles of 128 positions (8 steps of 16).
//
//   S = Q K^T      tcgen05.mma, 128 x 128, both operands fp16 in shared memory, S fp32 in tensor memory
//   P = exp2(...)  a thread a row: no exchange between threads for the maxima and the sums
//   O += P V       tcgen05.mma, P fp16 in tensor memory (in S's place), V fp16 in shared memory, O in tensor memory
//
// One block an SM, 18 warps:
//   * two groups of 4 softmax warps.  Group i takes the segment's tiles i, i + 2, ... as a stream of its own
//     with its own S / P, O, references and sums (2 x 256 of the 512 tensor-memory columns), so that one
//     stream's products run while the other's weights are made; the streams are joined at the segment's end.
//   * 8 conversion warps, one step of each tile each: codes from a ring of tensor copies, a tile ahead, to
//     exact fp16 in shared memory (K's int8 codes as subnormals, their offset taken off the logits), and one
//     warp that issues the copies, a lane a ring.
//   * one warp that issues the products.
// Both operands have one shared-memory image, 8 positions x 8 values a core matrix: it is K-major for S and
// MN-major (transposed in the instruction) for O.  The weights' exponentials are its
// floor (128 x 128 a tile at 16 a cycle and SM are 1,024 cycles, the tile's two products 512), but the latency of
// a stream's chain S -> weights -> O bounds it: about 4,000 cycles a tile with two streams, products and
// exponentials a quarter of the time each.  Two sequences of 4,000 positions, 1,500 rows, 16 query heads on 4:
// 184 us with the joining, 440 TFLOP/s; 8 sequences of up to 16,384, 128 rows a head, 2 heads: 34 us.
#include <type_traits>

#include "kv_split.cuh"

namespace bolt {

namespace {

constexpr int kRows = 128, kSteps = 8, kTileTokens = kSteps * 16;
constexpr int kSoftWarps = 8, kConvWarps = kSteps;
constexpr int kSlots = 3;  // of a conversion warp's ring: the next tile's K and V are under way
constexpr int kMmaWarp = kSoftWarps + kConvWarps, kCopyWarp = kMmaWarp + 1;
constexpr int kThreads = (kCopyWarp + 1) * 32;
constexpr int kMetaTiles = 64;
constexpr int kItemCost = 48;  // of an item's set-up, in steps

constexpr int kDead = 1, kWhole = 2;  // of a step: no row of the block sees it; all see all of it

template <int D>
struct Smem {
  static constexpr int kTile = 128 * D * 2;  // bytes of 128 rows of fp16
  static constexpr int kGroup = D * 16;      // bytes of 8 rows: D / 8 core matrices of 128 bytes
  static constexpr int kQ = 0, kK = kTile, kV = 3 * kTile, kMeta = 5 * kTile;  // K and V: one tile a stream
  static constexpr int kFactor = kMeta + kMetaTiles * kSteps * 16, kRef = kFactor + kRows * 8, kSum = kRef + 2 * kRows * 4;
  static constexpr int kBars = kSum + 2 * kRows * 4, kLine = kBars + (11 + 2 * kConvWarps * kSlots) * 8;
  // per conversion warp a ring of kSlots copies of a step's K or V codes, on 1,024-byte boundaries
  static constexpr int kRing = (kLine + kConvWarps * kMetaTiles * 4 + 1023) / 1024 * 1024, kSlot = 16 * D;
  static constexpr int kBytes = kRing + kConvWarps * kSlots * kSlot + 1024;
  static_assert(2 * kRows * D * 4 == 4 * kTile, "the joining buffer takes the place of K and V");
};

// fp32 D, fp16 A and B; 128 rows, N columns; B K-major (S) or MN-major (O)
__device__ constexpr uint32_t idesc(int n, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
// shared-memory descriptor without swizzle: byte strides along the descriptor's leading and other axis
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// products and commits: the whole warp, warp-uniform operands, one elected lane
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
      : "memory");
}
// 16 columns of this thread's row: begun, and arrived (the values pass through the wait, so that no use of
// them comes before it)
__device__ __forceinline__ void tm_begin16(uint32_t at, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tm_arrived16(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t at, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(at),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The positions of a step (16 from j0 on) that a row at `pos` sees, as bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1; }
__device__ __forceinline__ uint32_t seen_bits(const KvMask& m, int pos, int j0) {
  uint32_t seen = low_bits(pos - j0 + 1);
  if (m.window) seen &= ~low_bits(pos - m.window + 1 - j0) | low_bits(m.sinks - j0);
  return seen;
}

// Every row of the span sees all of the step from j0 on.
__device__ __forceinline__ bool sees_whole(const KvMask& m, const KvSpan& span, int j0) {
  return j0 + 15 <= span.first && (m.window == 0 || j0 > span.last - m.window || j0 + 15 < m.sinks);
}

// 16 codes as 16 halves in order: exact V codes, or K's (k_to_half).
template <int FMT, bool V>
__device__ __forceinline__ void convert16(const uint4& x, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (V)
      codes_to_half<FMT>(w[e], y[2 * e], y[2 * e + 1]);
    else
      k_to_half<FMT>(w[e], y[2 * e], y[2 * e + 1]);
  }
  lo = make_uint4(y[0], y[1], y[2], y[3]);
  hi = make_uint4(y[4], y[5], y[6], y[7]);
}

struct SwizzleRow {
  __device__ __forceinline__ int operator()(int row, int f) const { return f ^ (row & 7); }
};

template <int D, int FMT>
__global__ void __launch_bounds__(kThreads, 1) kv_attention_umma_kernel(
    const KvAttnParams p, const Work w, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using L = Smem<D>;
  extern __shared__ uint4 smem_raw[];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_lost;
  // the block's place in its work is kept here: the roles need the registers
  __shared__ KvWalk s_walk;
  __shared__ KvSegment s_seg;
  __shared__ int s_more;
  __shared__ unsigned s_nan[kRows / 32];  // the rows that see a NaN among V's codes of a step that not all rows see
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float4* s_meta = reinterpret_cast<float4*>(smem + L::kMeta);  // [tile % 64][step]: K scale, log2 and 1 / V scale, position and flags
  float2* sf = reinterpret_cast<float2*>(smem + L::kFactor);    // [row]: logit factor and shift (kv_make_q)
  float* sm = reinterpret_cast<float*>(smem + L::kRef);         // [stream][row]
  float* sl = reinterpret_cast<float*>(smem + L::kSum);         // [stream][row]
  float4* so = reinterpret_cast<float4*>(smem + L::kK);         // [stream][row][D / 4], when the products are done
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  const auto k_full = [&](int i) { return smem_u32(bars + i); };      // 8: K of the stream's next tile is in place
  const auto v_full = [&](int i) { return smem_u32(bars + 2 + i); };  // 8: its V
  const auto s_full = [&](int i) { return smem_u32(bars + 4 + i); };  // 2: its S is complete (and K free)
  const auto p_full = [&](int i) { return smem_u32(bars + 6 + i); };  // 4: its P is in place
  const auto o_full = [&](int i) { return smem_u32(bars + 8 + i); };  // its part of O is added (V, S and P free)
  const uint32_t drained = smem_u32(bars + 10);  // after a lost wait: the products are complete
  constexpr uint32_t kZero = FMT == kKvInt8 ? 0x80808080u : 0u;  // four codes of 0
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full(i), kConvWarps);
      mbar_init(v_full(i), kConvWarps);
      mbar_init(s_full(i), 2);
      mbar_init(p_full(i), 4);
      mbar_init(o_full(i), 1);
    }
    mbar_init(drained, 1);
    for (int i = 0; i < 2 * kConvWarps * kSlots; ++i) mbar_init(smem_u32(bars + 11 + i), 1);
    fence_barrier_init();
    s_lost = 0;
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s_tmem;
  const auto s_col = [&](int i) { return tmem + 128u * i; };
  const auto o_col = [&](int i) { return tmem + 256u + 128u * i; };
  pdl_wait();
  pdl_trigger();
  {
    const KvShare share = kv_share<kThreads>(p, w.row_blocks, kRows, kSteps, kItemCost);
    if (tid == 0) s_walk.start(share);
  }
  kv_empty_items<D, kRows, kThreads>(p, w);
  unsigned done0 = 0, done1 = 0;  // tiles of each stream, of all segments so far
  unsigned taken = 0;             // copies into each conversion warp's ring, of all segments
  bool lost = false;          // a wait ran out: the remaining segments are written as if their rows saw nothing
  const auto wait = [&](uint32_t bar, unsigned n) {  // for the completion of phase n
    const bool ok = mbar_wait(bar, n & 1, kStatusFullWait);
    if (!ok) s_lost = 1;
    return __all_sync(0xffffffffu, ok);
  };

  while (true) {
    if (tid == 0) s_more = s_walk.next(p, w.row_blocks, kRows, s_seg);
    if (FMT == kKvE4m3 && tid < kRows / 32) s_nan[tid] = 0;
    __syncthreads();
    if (!s_more) break;
    const int i0 = s_seg.i0, i1 = s_seg.i1, tiles = (i1 - i0 + kSteps - 1) / kSteps;
    // conversion warp cw, lane l: the entries of step cw of tile t0 + l
    const auto meta_table = [&](int t0) {
      const KvSpan span = s_seg.span;
      const int cw = warp - kSoftWarps, t = t0 + lane, step = i0 + t * kSteps + cw;
      const int j0 = span.base(min(step, i1 - 1));
      KvPages meta;
      meta.load_page(c, s_seg.s, step < i1 && j0 <= span.last, j0);
      meta.check_page(c);
      meta.load_scales<true>(c, s_seg.h);
      int flags = 0;
      if (meta.page < 0)
        flags = kDead;
      else if (sees_whole(p.mask, span, j0))
        flags = kWhole;
      const float2 vs = kv_v_scale(meta.vs);
      s_meta[t % kMetaTiles * kSteps + cw] = make_float4(meta.ks, vs.x, vs.y, __int_as_float(j0 | flags));
      reinterpret_cast<int*>(smem + L::kLine)[cw * kMetaTiles + t % kMetaTiles] =
          meta.page < 0 ? -1 : ((meta.page * c.heads + s_seg.h) * c.T + (j0 & (c.T - 1))) / (128 / D);
    };
    if (warp >= kSoftWarps && warp < kMmaWarp) meta_table(0);
    // the query rows: a warp takes tiles of 8 rows
    for (int tile = warp; tile < kRows / 8; tile += kCopyWarp + 1) {
      uint4 raw[D / 64][2];
      uint2 q[D / 16];
      float f, t;
      kv_fetch_q<D>(p, s_seg.seq, s_seg.s, s_seg.h, s_seg.m0 + tile * 8, raw);
      kv_make_q<D, FMT>(p, raw, q, f, t);
      const uint32_t flip = f < 0.f ? 0x80008000u : 0u;  // a negative scale goes into the rows: factors are not negative
      const int g = lane >> 2, q4 = lane & 3;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint2 a = q[4 * i + 2 * y], b = q[4 * i + 2 * y + 1];
          *reinterpret_cast<uint4*>(smem + L::kQ + tile * L::kGroup + (8 * i + 2 * q4 + y) * 128 + g * 16) =
              make_uint4(a.x ^ flip, a.y ^ flip, b.x ^ flip, b.y ^ flip);
        }
      if (q4 == 0) sf[tile * 8 + g] = make_float2(fabsf(f), t);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();

    if (lost) {
      if (warp < kSoftWarps) sm[tid] = -INFINITY;
    } else if (warp == kMmaWarp) {
      // ---- the products
      const auto scores = [&](int t) {  // S of tile t
        const int i = t & 1;
        const unsigned n = (i ? done1 : done0) + (t >> 1);
        if (!wait(k_full(i), n)) return false;
        if (n > 0 && !wait(o_full(i), n - 1)) return false;
        tc_after();
        const uint32_t kt = smem_u32(smem + L::kK + i * L::kTile), qt = smem_u32(smem + L::kQ);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(s_col(i), sdesc(qt + kk * 256, 128, L::kGroup), sdesc(kt + kk * 256, 128, L::kGroup),
                 idesc(kTileTokens, false), kk > 0);
        tc_commit(s_full(i));
        if (lane == 0) mbar_arrive(s_full(i));  // hands on what the conversion warps wrote for the softmax warps
        return true;
      };
      bool ok = scores(0) && (tiles < 2 || scores(1));
      for (int t = 0; ok && t < tiles; ++t) {
        const int i = t & 1;
        const unsigned n = (i ? done1 : done0) + (t >> 1);
        ok = wait(p_full(i), n) && wait(v_full(i), n);
        if (!ok) break;
        tc_after();
        const uint32_t vt = smem_u32(smem + L::kV + i * L::kTile);
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk)
          mma_ts(o_col(i), s_col(i) + 8 * kk, sdesc(vt + kk * 2 * L::kGroup, L::kGroup, 128), idesc(D, true),
                 t >= 2 || kk > 0);
        tc_commit(o_full(i));
        ok = t + 2 >= tiles || scores(t + 2);
      }
    } else if (warp == kCopyWarp) {
      // ---- copies into the rings, lane i for conversion warp i: unit 2 t is its step of tile t's K, 2 t + 1 of V
      const int* lines = reinterpret_cast<const int*>(smem + L::kLine) + (lane & 7) * kMetaTiles;
      uint64_t* full = bars + 11 + (lane & 7) * kSlots;
      uint64_t* empty = full + kConvWarps * kSlots;
      for (int u = 0; u < 2 * tiles; ++u) {
        const unsigned n = taken + u, slot = n % kSlots, round = n / kSlots;
        // the first kSlots units find their places free; the wait also orders the reading of `lines` behind
        // its writing: unit u's line was written before unit u - kSlots was handed back
        if (round > 0 && !wait(smem_u32(empty + slot), round - 1)) break;
        if (lane < kConvWarps) {
          const int line = lines[(u >> 1) % kMetaTiles];
          const uint32_t bar = smem_u32(full + slot);
          if (line >= 0) {
            mbar_arrive_expect_tx(bar, L::kSlot);
            tma_load_3d(smem_u32(smem + L::kRing + (lane * kSlots + slot) * L::kSlot), u & 1 ? &map_v : &map_k, 0, line, 0,
                        bar);
          } else {
            mbar_arrive(bar);
          }
        }
        __syncwarp();
      }
    } else if (warp >= kSoftWarps) {
      // ---- codes to fp16: this warp's step of each tile
      const int cw = warp - kSoftWarps, r = lane & 7, chunk = lane >> 3;
      const KvSpan span = s_seg.span;
      const uint8_t* ring = smem + L::kRing + cw * kSlots * L::kSlot;
      uint64_t* full = bars + 11 + cw * kSlots;
      uint64_t* empty = full + kConvWarps * kSlots;
      const int* lines = reinterpret_cast<const int*>(smem + L::kLine) + cw * kMetaTiles;
      const int from_at = kv_at<D>(r, chunk * 16), to_at = 2 * cw * L::kGroup + 2 * chunk * 128 + r * 16;
      const auto convert = [&](int u, auto is_v, bool dead, bool whole, int j0, uint8_t* tile) {
        constexpr bool V = decltype(is_v)::value;
        const unsigned n = taken + u, slot = n % kSlots;
        if (!wait(smem_u32(full + slot), n / kSlots)) return false;
        const uint8_t* from = ring + slot * L::kSlot;
        uint4 x[D / 32];
#pragma unroll
        for (int v = 0; v < D / 32; ++v) x[v] = lds128(from + ((v & 1 ? kv_next_tile<D>(from_at) : from_at) ^ (v >> 1) * 64));
        if (dead) {  // no codes
#pragma unroll
          for (int v = 0; v < D / 32; ++v) x[v] = make_uint4(kZero, kZero, kZero, kZero);
        } else if (FMT == kKvE4m3 && V && !whole) {
          // weights of 0 must not meet a NaN code (a stale one that no row sees, or one that some rows see): it
          // becomes 0, and the rows that see its position are marked
          uint32_t nan = 0;
#pragma unroll
          for (int v = 0; v < D / 32; ++v) {
            const uint4 b = make_uint4(kv_nan_bytes(x[v].x), kv_nan_bytes(x[v].y), kv_nan_bytes(x[v].z), kv_nan_bytes(x[v].w));
            if (b.x | b.y | b.z | b.w) nan |= 1u << ((v & 1) * 8 + r);
            x[v] = make_uint4(x[v].x & ~b.x, x[v].y & ~b.y, x[v].z & ~b.z, x[v].w & ~b.w);
          }
          nan = __reduce_or_sync(0xffffffffu, nan);
          if (nan) {
#pragma unroll 1
            for (int k = 0; k < kRows / 32; ++k) {
              const int at_row = s_seg.seq.start + static_cast<int>((s_seg.m0 + 32 * k + lane) / static_cast<unsigned>(p.G));
              const unsigned rows = __ballot_sync(0xffffffffu, seen_bits(p.mask, at_row, j0) & nan);
              if (lane == 0) atomicOr(&s_nan[k], rows);
            }
          }
        }
#pragma unroll
        for (int v = 0; v < D / 32; ++v) {
          uint4 lo, hi;
          convert16<FMT, V>(x[v], lo, hi);
          uint8_t* to = tile + to_at + (v & 1) * L::kGroup + (v >> 1) * 8 * 128;
          *reinterpret_cast<uint4*>(to) = lo;
          *reinterpret_cast<uint4*>(to + 128) = hi;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(empty + slot));
        return true;
      };
      for (int t = 0; t < tiles; ++t) {
        const int i = t & 1;
        const unsigned n = (i ? done1 : done0) + (t >> 1);
        // the entries of the next 32 tiles, when no role reads those of 32 tiles ago any more: K of this tile
        // can be replaced only when S of the last but one, and so the weights before it, are made
        if ((t & 31) == 8) meta_table(t + 24);
        if (n > 0 && !wait(s_full(i), n - 1)) break;
        const bool dead = lines[t % kMetaTiles] < 0;
        const int j0 = span.base(min(i0 + t * kSteps + cw, i1 - 1));
        const bool whole = sees_whole(p.mask, span, j0);
        if (!convert(2 * t, std::false_type(), dead, whole, j0, smem + L::kK + i * L::kTile)) break;
        if (lane == 0) mbar_arrive(k_full(i));
        if (n > 0 && !wait(o_full(i), n - 1)) break;
        if (!convert(2 * t + 1, std::true_type(), dead, whole, j0, smem + L::kV + i * L::kTile)) break;
        if (lane == 0) mbar_arrive(v_full(i));
      }
    } else {
      // ---- weights: stream i, this thread's row
      const int i = warp >> 2, row = tid & 127;
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 rows a warp, in the address's upper half
      const unsigned m = s_seg.m0 + row, G = p.G;
      const int at_row = s_seg.seq.start + static_cast<int>(m / G);
      const int pos = m < static_cast<unsigned>(p.rows.R) * G && at_row < s_seg.seq.len ? at_row : -1;
      const float qf = sf[row].x, qt = sf[row].y;
      float ref = 0.f, top_off = -INFINITY, l = 0.f;  // the reference m - 8; how far a logit may pass it: not at all until there is one
      bool ok = true;
      int n_tiles = 0;
      for (int t = i; t < tiles; t += 2, ++n_tiles) {
        const unsigned n = (i ? done1 : done0) + (t >> 1);
        ok = wait(s_full(i), n);
        if (!ok) break;
        tc_after();
        const float4* meta = s_meta + t % kMetaTiles * kSteps;
        float xa[16], xb[16];
        // the row's largest logit: of a step's sums before their factor, which is not negative
        float most = -INFINITY;
        int whole = kWhole;
        const auto largest = [&](int k, const float (&x)[16]) {
          const float4 sc = meta[k];
          const int j0 = __float_as_int(sc.w);
          whole &= j0;
          float top;
          if (j0 & kWhole) {
            top = max3(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[8])),
                       max3(x[9], x[10], x[11]), max3(max3(x[12], x[13], x[14]), x[15], x[15]));
          } else {
            const uint32_t seen = j0 & kDead ? 0u : seen_bits(p.mask, pos, j0 & ~15);
            top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, seen >> e & 1 ? x[e] : -INFINITY);
          }
          const float z = top * (qf * sc.x) + (sc.y - ref - qt * sc.x);
          most = fmaxf(most, top > -INFINITY ? z : -INFINITY);
        };
        tm_begin16(s_col(i) + lanes, xa);
#pragma unroll 1
        for (int k = 0; k < kSteps; k += 2) {
          tm_arrived16(xa);
          tm_begin16(s_col(i) + 16 * (k + 1) + lanes, xb);
          largest(k, xa);
          tm_arrived16(xb);
          tm_begin16(s_col(i) + (k + 2 < kSteps ? 16 * (k + 2) : 0) + lanes, xa);  // at the end: the first again
          largest(k + 1, xb);
        }
        if (__any_sync(0xffffffffu, most > top_off)) {
          const bool fresh = top_off == -INFINITY, move = most > -INFINITY;
          const float up = !move ? 0.f : fresh ? most - kWeightLog : fmaxf(0.f, most - kWeightLog);
          const float g = fresh ? 0.f : ex2(-up);
          l *= g;
          ref += up;
          if (move) top_off = kWeightTop;
          if (t != i) {  // the stream's O: all its products so far are complete, this S came after them
            float y[16];
#pragma unroll 1
            for (int z = 0; z < D / 16; ++z) {
              tm_begin16(o_col(i) + 16 * z + lanes, y);
              tm_arrived16(y);
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] *= g;
              tm_st16(o_col(i) + 16 * z + lanes, y);
            }
          }
        }
        const auto weigh = [&](int k, auto all, float (&x)[16]) {  // step k of the tile: 16 logits to 16 weights
          const float4 sc = meta[k];
          const float f = qf * sc.x, d = sc.y - ref - qt * sc.x;
          const float2 f2 = make_float2(f, f), d2 = make_float2(d, d);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float2 y = ffma2(make_float2(x[e], x[e + 1]), f2, d2);
            x[e] = ex2(y.x);
            x[e + 1] = ex2(y.y);
          }
          if constexpr (!decltype(all)::value) {
            const int j0 = __float_as_int(sc.w);
            const uint32_t seen = j0 & kWhole ? 0xFFFFu : j0 & kDead ? 0u : seen_bits(p.mask, pos, j0 & ~15);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = seen >> e & 1 ? x[e] : 0.f;
          }
          uint32_t h[8];
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            sum[(e >> 1) & 1] = fadd2(sum[(e >> 1) & 1], make_float2(x[e], x[e + 1]));
            const __half2 z = __floats2half2_rn(x[e], x[e + 1]);
            h[e / 2] = *reinterpret_cast<const uint32_t*>(&z);
          }
          const float2 both = fadd2(sum[0], sum[1]);
          l += (both.x + both.y) * sc.z;
          tm_st8(s_col(i) + 8 * k + lanes, h);  // columns that have been read
        };
        const auto weigh_all = [&](auto all) {
#pragma unroll 1
          for (int k = 0; k < kSteps; k += 2) {
            tm_arrived16(xa);
            tm_begin16(s_col(i) + 16 * (k + 1) + lanes, xb);
            weigh(k, all, xa);
            tm_arrived16(xb);
            if (k + 2 < kSteps) tm_begin16(s_col(i) + 16 * (k + 2) + lanes, xa);
            weigh(k + 1, all, xb);
          }
        };
        if (whole)
          weigh_all(std::true_type());
        else
          weigh_all(std::false_type());
        tm_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(i));
      }
      if (ok && n_tiles > 0) ok = wait(o_full(i), (i ? done1 : done0) + n_tiles - 1);
      tc_after();
      // NaN among the logits passed by the maximum and is in the sum, also of a row that has no reference
      ref = pos < 0 || !ok ? -INFINITY : l != l ? NAN : top_off == -INFINITY ? -INFINITY : ref + kWeightLog;
      sm[i * kRows + row] = ref;
      sl[i * kRows + row] = l;
    }
    done0 += (tiles + 1) / 2;
    done1 += tiles / 2;
    taken += 2 * tiles;
    __syncthreads();  // all products are complete: K and V make room for the values
    if (!lost && s_lost && warp == kCopyWarp && lane < kConvWarps)
      // wait, within limits, for what is on its way into the rings
      for (unsigned i = 0; i < kSlots; ++i) mbar_wait(smem_u32(bars + 11 + lane * kSlots + i), ((taken + i) / kSlots) & 1, kStatusDrainWait);
    lost |= s_lost != 0;
    if (warp < kSoftWarps) {
      const int i = warp >> 2, row = tid & 127;
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
      const float ref = sm[i * kRows + row], top = fmaxf(sm[row], sm[kRows + row]);
      const float f = ref == -INFINITY ? 0.f : ex2(ref - top);
      if (FMT == kKvE4m3 && (s_nan[row >> 5] >> (row & 31) & 1)) sl[i * kRows + row] = NAN;
#pragma unroll 1
      for (int q = 0; q < D / 16; ++q) {
        float x[16];
        if (i < tiles) {
          tm_begin16(o_col(i) + 16 * q + lanes, x);
          tm_arrived16(x);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (f != 0.f) v = make_float4(x[e] * f, x[e + 1] * f, x[e + 2] * f, x[e + 3] * f);
          so[(i * kRows + row) * (D / 4) + SwizzleRow()(row, 4 * q + e / 4)] = v;
        }
      }
      tc_before();
    }
    __syncthreads();
    kv_finish<D, kRows, 2, kThreads>(p, w, s_walk.share, s_seg, sm, sl, so, SwizzleRow());
    __syncthreads();  // the next segment writes the shared buffers
    tc_after();
  }
  if (lost && warp == kMmaWarp) {
    // products may be under way: wait for them, within the limit, before the tensor memory is released
    tc_commit(drained);
    mbar_wait(drained, 0, kStatusDrainWait);
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == kMmaWarp) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int D, int FMT>
cudaError_t launch(const KvAttnParams& p, const Work& w, unsigned blocks, const LaunchCfg& cfg) {
  static SmemOptIn opt;
  auto kern = kv_attention_umma_kernel<D, FMT>;
  const cudaError_t e = allow_smem(kern, Smem<D>::kBytes, opt);
  if (e != cudaSuccess) return e;
  CUtensorMap map_k, map_v;
  if (!kv_code_map(&map_k, p.c, p.c.k) || !kv_code_map(&map_v, p.c, p.c.v)) return cudaErrorInvalidValue;
  return launch_kernel(kern, dim3(blocks), dim3(kThreads), Smem<D>::kBytes, cfg, p, w, map_k, map_v);
}

}  // namespace

cudaError_t launch_kv_attention_umma(const KvAttnParams& p, const Work& w, unsigned blocks, const LaunchCfg& cfg) {
  const bool i8 = p.c.fmt == kKvInt8;
  if (p.c.D == 128) return i8 ? launch<128, kKvInt8>(p, w, blocks, cfg) : launch<128, kKvE4m3>(p, w, blocks, cfg);
  return i8 ? launch<64, kKvInt8>(p, w, blocks, cfg) : launch<64, kKvE4m3>(p, w, blocks, cfg);
}

}  // namespace bolt
