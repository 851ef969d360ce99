// The paged 8-bit key/value cache: host-side parameters and launchers (kv_cache.cu, kv_attention.cu,
// kv_evict.cu).
//
// K and V are u8 [pages, heads, T, D] each, with an f32 scale per (page, head) beside them:
//   value = scale * (code - 128)   (kKvInt8; a byte is q + 128, as in Q8Gemv's weights)
//   value = scale * e4m3(code)     (kKvE4m3)
// Position j of sequence s is slot j % T of page table[s][j / T].
#pragma once

#include "kernels.h"

namespace bolt {

enum KvFmt : int { kKvInt8 = 0, kKvE4m3 = 1 };

struct KvCache {
  uint8_t *k, *v;        // [pages, heads, T, D]
  float *ks, *vs;        // [pages, heads]
  const int* table;      // [S, width]
  int64_t pages;
  int heads, T, tshift, D, fmt;
  int S, width;
};

// The rows of a call: row r of sequence s is position start[s] + r and exists while that is below lens[s].
struct KvRows {
  const int *start, *lens;  // [S]
  int R;
};

// What a row at position p sees of its sequence: j <= p and, under a window, j > p - window or j < sinks.
struct KvMask {
  int window, sinks;  // window 0: none
};

struct KvAttnParams {
  KvCache c;
  KvRows rows;
  KvMask mask;
  const bf16* q;            // [S, R, Hq, D], strides qs (sequence) and qr (row)
  int64_t qs, qr;
  int Hq, G;                // G = Hq / heads
  float scale;
  bf16* o;                  // [S, R, Hq, D]
  float* lse;               // [S, R, Hq]; KvScore reads it
  float* score;             // [S, heads, score_width] (KvScore)
  int64_t score_width;
  bool few_steps;           // the 16-position steps of all items are fewer than 2^31 whatever the lengths
};

cudaError_t launch_kv_append(const KvCache& c, const KvRows& rows, const bf16* k, int64_t k_seq, int64_t k_row,
                             const bf16* v, int64_t v_seq, int64_t v_row, const LaunchCfg& cfg);
cudaError_t launch_kv_read(const KvCache& c, const KvRows& rows, bf16* k, bf16* v, const LaunchCfg& cfg);
// Bytes of the scratch memory that launch_kv_attention takes (16-byte aligned).
// `rows`: R * G, the rows that read one head of the cache.
int64_t kv_attention_workspace(int64_t rows, int D, int sms);
cudaError_t launch_kv_attention(const KvAttnParams& p, void* workspace, const LaunchCfg& cfg);
cudaError_t launch_kv_score(const KvAttnParams& p, const LaunchCfg& cfg);

struct KvEvictParams {
  KvCache c;
  const int* lens;        // [S]
  const float* score;     // [S, heads, score_width]
  int64_t score_width;
  const int* new_table;   // [S, new_width]
  int new_width;
  int keep, sinks, recent;
  int* kept;              // [S, heads, keep]
  int* new_lens;          // [S]
  float* new_score;       // [S, heads, keep]
};
cudaError_t launch_kv_evict(const KvEvictParams& p, const LaunchCfg& cfg);

}  // namespace bolt
