#pragma once

// Arguments of the 8-bit KV cache kernels (kv_fp8.hip, kv_fp8_attention.hip), shared with the host
// code that launches them (csrc/hip/kv_fp8_ops.cc).
#include <stdint.h>

// The pages of a cache and the sequences in them (layout in include/dli_hip.h).
struct Kv8Pages {
  uint8_t* key;     // [num_blocks, heads, block_size, head_dim]
  uint8_t* value;   // [num_blocks, heads, head_dim, block_size]
  uint8_t* scales;  // [num_blocks, heads, 2, block_size]: the keys', then the values'
  const int32_t* table;  // [batch, max_blocks]; an id outside [0, num_blocks): a page that holds nothing
  int64_t num_blocks;
  int64_t max_blocks;
  const void* positions;  // [batch] int32 or int64, or NULL: every sequence at `start`
  int64_t start;
  int pos64;
  int block_size;
  int heads;
  int head_dim;
};

// kv_append: k, v [batch, heads, seq, head_dim]. rope_append: qkv [batch, seq, (q_heads + 2 heads)
// * head_dim], q and k rotated by cos/sin [max_pos, pairs]; q goes to q_out [batch, q_heads, seq,
// head_dim].
struct Kv8WriteArgs {
  Kv8Pages pages;
  const void* k;
  const void* v;
  const void* qkv;
  const float* cos;
  const float* sin;
  void* q_out;
  int64_t max_pos;
  int64_t batch;
  int64_t seq;
  int pairs;
  int q_heads;
};

// kv_read: key, value [batch, heads, seq, head_dim] of the tokens from start (or positions[b]) on.
struct Kv8ReadArgs {
  Kv8Pages pages;
  void* k;
  void* v;
  int64_t batch;
  int64_t seq;
};

// Attention of q [batch, q_heads, seq_q, head_dim]; pages.start / positions: the tokens that a
// sequence holds before the first query. splits workgroups share the keys of one row tile; with
// splits > 1 each leaves, per row, (maximum, sum) and the normalised output of its keys.
struct Kv8AttentionArgs {
  Kv8Pages pages;
  const void* q;
  void* out;
  float* part_ml;  // [rows of the call][splits][2]
  float* part_o;   // [rows of the call][splits][head_dim]
  int64_t capacity;  // tokens a sequence's pages hold
  int batch;
  int q_heads;
  int seq_q;
  int causal;
  int out_bshd;  // out is [batch, seq_q, q_heads, head_dim]
  int splits;
  float scale_log2;  // scale * log2(e)
};
