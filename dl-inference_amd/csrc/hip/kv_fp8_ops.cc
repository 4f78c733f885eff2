// Entry points of the 8-bit paged KV cache (declared in include/dli_hip.h): argument checks, the
// choice of kernel and launch geometry.
#include <cmath>
#include <string>

#include "../kernels/kv_fp8_args.h"
#include "runtime.h"

namespace dli::hip {
namespace {

int badArg(const char* op, const std::string& what) {
  return fail(DLI_HIP_EINVAL, std::string(op) + ": " + what);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int dtypeIndex(int dtype) {
  return dtype == DLI_F32 ? 0 : dtype == DLI_BF16 ? 1 : dtype == DLI_F16 ? 2 : -1;
}

#define KV8_DTYPES(module, base) \
  { {module, base "_f32"}, {module, base "_bf16"}, {module, base "_f16"} }

// [head_dim 64, 128][dtype]
#define KV8_DIMS(module, base, tail) \
  { KV8_DTYPES(module, base "d64" tail), KV8_DTYPES(module, base "d128" tail) }

DeviceKernel k_append[2][3] = KV8_DIMS("kv_fp8", "kv8_append_", "");
DeviceKernel k_append_few[2][3] = KV8_DIMS("kv_fp8", "kv8_append_few_", "");
DeviceKernel k_append_any[3] = KV8_DTYPES("kv_fp8", "kv8_append_any");
DeviceKernel k_rope[2][3] = KV8_DIMS("kv_fp8", "kv8_rope_", "");
DeviceKernel k_rope_few[2][3] = KV8_DIMS("kv_fp8", "kv8_rope_few_", "");
DeviceKernel k_rope_any[3] = KV8_DTYPES("kv_fp8", "kv8_rope_any");
DeviceKernel k_read[2][3] = KV8_DIMS("kv_fp8", "kv8_read_", "");
DeviceKernel k_read_any[3] = KV8_DTYPES("kv_fp8", "kv8_read_any");
// [small pages][head_dim][dtype]
DeviceKernel k_decode[2][2][3] = {KV8_DIMS("kv_fp8_attention", "kv8_decode_", ""),
                                  KV8_DIMS("kv_fp8_attention", "kv8_decode_small_", "")};
// [small pages][head_dim][dtype], 64 rows a workgroup
DeviceKernel k_chunk[2][2][3] = {KV8_DIMS("kv_fp8_attention", "kv8_chunk_", "_r64"),
                                 KV8_DIMS("kv_fp8_attention", "kv8_chunk_small_", "_r64")};
// [small pages]: 128 rows, bf16 of head_dim 64 and 128, f16 of 128
#define KV8_LARGE(base)                                                                          \
  { {"kv_fp8_attention", base "d64_r128_bf16"}, {"kv_fp8_attention", base "d128_r128_bf16"},      \
    {"kv_fp8_attention", base "d128_r128_f16"} }
DeviceKernel k_chunk_large[2][3] = {KV8_LARGE("kv8_chunk_"), KV8_LARGE("kv8_chunk_small_")};
DeviceKernel k_phased = {"kv_fp8_attention", "kv8_phased_d128_bf16"};  // 256 rows
DeviceKernel k_merge[2][3] = KV8_DIMS("kv_fp8_attention", "kv8_merge_", "");
DeviceKernel k_rows[3] = KV8_DTYPES("kv_fp8_attention", "kv8_rows");

constexpr int64_t kMostTokens = int64_t{1} << 30;  // of a sequence, and rows of a pair: 32-bit indexes
constexpr int64_t kMostPairs = int64_t{1} << 40;   // of a call's tokens: products with heads stay in range
constexpr int64_t kMostGrid = 65535;               // of a grid's y and z

// What every call has in common; fills `pages`. 0, or the recorded error.
int pagesOf(const char* op, int dtype, const void* key_codes, const void* value_codes,
            const void* scales, const int32_t* block_table, int64_t num_blocks, int64_t batch,
            int64_t heads, int64_t seq, int64_t head_dim, int64_t block_size, int64_t max_blocks,
            int64_t start, const void* positions, int positions_dtype, Kv8Pages* pages) {
  if (dtypeIndex(dtype) < 0)
    return badArg(op, "unsupported dtype code " + std::to_string(dtype));
  if (batch < 0 || seq < 0 || heads <= 0) return badArg(op, "batch and seq must be >= 0, heads > 0");
  if (head_dim <= 0 || head_dim > 256) return badArg(op, "head_dim must be in [1, 256]");
  if (block_size <= 0 || max_blocks <= 0 || num_blocks <= 0)
    return badArg(op, "block_size, max_blocks and num_blocks must be positive");
  if (block_size >= kMostTokens || max_blocks >= kMostTokens || block_size * max_blocks >= kMostTokens)
    return badArg(op, "a sequence's pages must hold fewer than 2^30 tokens");
  if (heads > kMostGrid / 2 || batch >= kMostTokens || seq >= kMostTokens || batch * seq >= kMostPairs)
    return badArg(op, "batch, seq or heads too large");
  if (positions != nullptr && positions_dtype != DLI_I64 && positions_dtype != DLI_I32)
    return badArg(op, "positions must be int64 or int32");
  if (batch > 0 && seq > 0 &&
      (key_codes == nullptr || value_codes == nullptr || scales == nullptr || block_table == nullptr))
    return badArg(op, "null cache pointer");
  pages->key = static_cast<uint8_t*>(const_cast<void*>(key_codes));
  pages->value = static_cast<uint8_t*>(const_cast<void*>(value_codes));
  pages->scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  pages->table = block_table;
  pages->num_blocks = num_blocks;
  pages->max_blocks = max_blocks;
  pages->positions = positions;
  pages->start = start;
  pages->pos64 = positions_dtype == DLI_I64;
  pages->block_size = static_cast<int>(block_size);
  pages->heads = static_cast<int>(heads);
  pages->head_dim = static_cast<int>(head_dim);
  return 0;
}

int dimIndex(int64_t head_dim) { return head_dim == 64 ? 0 : head_dim == 128 ? 1 : -1; }

// The tile kernels of append, rope and read: head_dim 64 or 128, runs of 16 tokens in one page,
// 16-byte loads and stores.
bool tileForm(const Kv8Pages& p, int64_t batch, int64_t grid_rows) {
  return dimIndex(p.head_dim) >= 0 && p.block_size % 16 == 0 && batch <= kMostGrid &&
         grid_rows <= kMostGrid && aligned16(p.key) && aligned16(p.value);
}

unsigned rowBlocks(int64_t rows) {  // of 4 waves, a row each; the kernels go on from row to row
  const int64_t blocks = (rows + 3) / 4;
  return static_cast<unsigned>(blocks < 65536 ? blocks : 65536);
}

// Tiles of `tokens` that a sequence's new tokens touch, wherever it starts in one.
unsigned tilesOf(int64_t seq, int64_t tokens) {
  return static_cast<unsigned>((seq + 2 * tokens - 2) / tokens);
}

// 64 tokens to a workgroup, 16 for up to 16 of them (more workgroups, none waiting for empty waves).
int launchWrite(const Kv8WriteArgs& a, bool tiles, int rows, int di, DeviceKernel (&many)[2][3],
                DeviceKernel (&few)[2][3], DeviceKernel (&any)[3], void* stream) {
  if (!tiles)
    return launch(any[di], {rowBlocks(a.batch * a.seq * rows)}, {256}, 0, stream, a);
  const int dim = dimIndex(a.pages.head_dim);
  const unsigned y = static_cast<unsigned>(rows), z = static_cast<unsigned>(a.batch);
  if (a.seq <= 16) return launch(few[dim][di], {tilesOf(a.seq, 16), y, z}, {64}, 0, stream, a);
  return launch(many[dim][di], {tilesOf(a.seq, 64), y, z}, {256}, 0, stream, a);
}

// How attention runs: 0 one wave per row, 1 decode (at most 16 rows of a pair), 2 chunk.
struct AttentionPlan {
  int form;
  int size;  // chunk: 64 << size rows a workgroup; 2 is the phased kernel
  int64_t splits;
};

// reach: tokens that a sequence holds at most, queries included, as far as the host knows: all that its pages
// take where the positions are on the device. phased: whether that kernel may be chosen.
AttentionPlan attentionPlan(int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t seq_q,
                            int64_t head_dim, int64_t block_size, int64_t reach, bool phased = true) {
  const int64_t units = batch * kv_heads, rows = q_heads / kv_heads * seq_q;
  const bool paged = block_size % 64 == 0 || block_size == 16 || block_size == 32;
  // offsets within a page's head are 32 bits
  const bool near = block_size * head_dim < int64_t{1} << 31;
  if (dimIndex(head_dim) < 0 || !paged || !near || units > kMostGrid || units == 0 || rows >= kMostTokens)
    return {0, 0, 1};
  const int64_t tiles = (reach + 63) / 64;
  if (rows <= 16) {
    // About one workgroup of 8 waves per CU, each wave with a tile at least if the sequences are that
    // long. Joining the splits is a launch of its own, which costs more than two tiles to a wave: 1000
    // tokens of one sequence (14 / 2 heads x 64) 7.6 us undivided and 8.9 in 2 splits; 8 x 2000 (28 / 4 x
    // 128) 18.6, 15.5 and, in 4, 12.2. (Joined by the split that arrives last, in the same launch: 13.1 us
    // for 32 x 4096 where two launches take 12.6, and 20.6 for 16 splits where they take 11.5.)
    if (tiles <= 16) return {1, 0, 1};
    int64_t splits = (256 + units - 1) / units;
    const int64_t most = (tiles + 7) / 8;
    splits = splits < most ? splits : most;
    return {1, 0, splits < 32 ? splits : 32};
  }
  // 128 rows share a staged tile where they still fill half the card. 64 and 128 rows, us: bf16, 2 x
  // 300 tokens over 3000 (28 / 4 heads x 128, 136 workgroups of 128) 87 and 64; 1 x 2048 over 8192 465 and
  // 339; 4 x 2048 tokens (14 / 2 x 64) 60 and 51. f16 holds its weights in two terms and pays from more
  // workgroups on, with head_dim 128 only: 2 x 500 over 2000 77 and 84, 1 x 2000 over 3000 235 and 209,
  // 4 x 1000 over 500 (x 64) 45 and 47. fp32 (three terms of q) never: 92 and 113, 36 and 40.
  const int64_t large = units * ((rows + 127) / 128);
  const int size = dtype == DLI_BF16  ? large >= 128
                   : dtype == DLI_F16 ? large >= 384 && head_dim == 128
                                      : 0;
  const auto blocksOf = [&](int s) { return units * ((rows + (int64_t{64} << s) - 1) / (int64_t{64} << s)); };
  // keys split until two workgroups stand on every CU, each with 4 tiles at least (as above); a split's
  // results are written and read again, so none where the rows fill the card (2 x 1000 prompt tokens, 28 / 4
  // heads x 128: 37 us, 61 in two splits)
  const auto splitsOf = [&](int64_t blocks, int64_t places) {
    int64_t splits = places / blocks;
    const int64_t most = tiles / 4;
    splits = splits < most ? splits : most;
    splits = splits < 32 ? splits : 32;
    return splits > 1 ? splits : 1;
  };
  if (phased && dtype == DLI_BF16 && head_dim == 128 && size == 1 && block_size % 64 == 0 &&
      reach > 2500) {
    // A phased workgroup has a CU to itself, so it pays over long contexts, where its first and last
    // steps count little, and where its rounds fill the card by two thirds. 128 rows and phased, us (28 / 4
    // heads): 2 x 1000 tokens over nothing 37 and 42, over 1000 67 and 72, 2000 101 and 96, 4000 170 and
    // 149; 1 x 4096 155 and 130; 2 x 300 over 3000 63 and 60; 8 x 300 over 3000, 288 workgroups, 185 and 191.
    const int64_t blocks = blocksOf(2), splits = splitsOf(blocks, 256), all = blocks * splits;
    if ((all + 255) / 256 * 256 * 2 <= all * 3) return {2, 2, splits};
  }
  return {2, size, splitsOf(blocksOf(size), 512)};
}

size_t partBytes(int64_t rows, int64_t head_dim, int64_t splits) {
  return splits > 1 ? static_cast<size_t>(rows * splits * (head_dim + 2)) * sizeof(float) : 0;
}

}  // namespace
}  // namespace dli::hip

using namespace dli::hip;

extern "C" {

int dli_hip_kv_append_fp8(int dtype, const void* key, const void* value, void* key_codes,
                          void* value_codes, void* scales, const int32_t* block_table,
                          int64_t num_blocks, int64_t batch, int64_t heads, int64_t seq,
                          int64_t head_dim, int64_t block_size, int64_t max_blocks, int64_t start,
                          const void* positions, int positions_dtype, void* stream) {
  const char* op = "kv_append_fp8";
  Kv8WriteArgs a{};
  if (int rc = pagesOf(op, dtype, key_codes, value_codes, scales, block_table, num_blocks, batch, heads,
                       seq, head_dim, block_size, max_blocks, start, positions, positions_dtype, &a.pages))
    return rc;
  if (batch == 0 || seq == 0) return 0;
  if (key == nullptr || value == nullptr) return badArg(op, "null input");
  a.k = key;
  a.v = value;
  a.batch = batch;
  a.seq = seq;
  const bool tiles = tileForm(a.pages, batch, 2 * heads) && aligned16(key) && aligned16(value);
  return launchWrite(a, tiles, static_cast<int>(2 * heads), dtypeIndex(dtype), k_append, k_append_few,
                     k_append_any, stream);
}

int dli_hip_rope_append_fp8(int dtype, const void* qkv, const float* cos_table, const float* sin_table,
                            int64_t max_pos, int64_t pairs, void* q_out, void* key_codes,
                            void* value_codes, void* scales, const int32_t* block_table,
                            int64_t num_blocks, int64_t batch, int64_t seq, int64_t q_heads,
                            int64_t kv_heads, int64_t head_dim, int64_t block_size,
                            int64_t max_blocks, int64_t start, const void* positions,
                            int positions_dtype, void* stream) {
  const char* op = "rope_append_fp8";
  Kv8WriteArgs a{};
  if (int rc = pagesOf(op, dtype, key_codes, value_codes, scales, block_table, num_blocks, batch, kv_heads,
                       seq, head_dim, block_size, max_blocks, start, positions, positions_dtype, &a.pages))
    return rc;
  if (q_heads <= 0 || q_heads > kMostGrid) return badArg(op, "q_heads must be in [1, 65535]");
  if (pairs <= 0 || 2 * pairs > head_dim || max_pos < 0)
    return badArg(op, "cos/sin must have at most head_dim / 2 pairs");
  if (batch == 0 || seq == 0) return 0;
  if (qkv == nullptr || q_out == nullptr || (max_pos > 0 && (cos_table == nullptr || sin_table == nullptr)))
    return badArg(op, "null input or output");
  a.qkv = qkv;
  a.cos = cos_table;
  a.sin = sin_table;
  a.q_out = q_out;
  a.max_pos = max_pos;
  a.batch = batch;
  a.seq = seq;
  a.pairs = static_cast<int>(pairs);
  a.q_heads = static_cast<int>(q_heads);
  const int64_t rows = q_heads + 2 * kv_heads;
  const bool tiles = tileForm(a.pages, batch, rows) && 2 * pairs == head_dim && aligned16(qkv) &&
                     aligned16(q_out) && aligned16(cos_table) && aligned16(sin_table);
  return launchWrite(a, tiles, static_cast<int>(rows), dtypeIndex(dtype), k_rope, k_rope_few, k_rope_any,
                     stream);
}

int dli_hip_kv_read_fp8(int dtype, const void* key_codes, const void* value_codes, const void* scales,
                        const int32_t* block_table, int64_t num_blocks, void* key, void* value,
                        int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                        int64_t block_size, int64_t max_blocks, int64_t start, const void* positions,
                        int positions_dtype, void* stream) {
  const char* op = "kv_read_fp8";
  Kv8ReadArgs a{};
  if (int rc = pagesOf(op, dtype, key_codes, value_codes, scales, block_table, num_blocks, batch, heads,
                       seq, head_dim, block_size, max_blocks, start, positions, positions_dtype, &a.pages))
    return rc;
  if (batch == 0 || seq == 0) return 0;
  if (key == nullptr || value == nullptr) return badArg(op, "null output");
  a.k = key;
  a.v = value;
  a.batch = batch;
  a.seq = seq;
  const int di = dtypeIndex(dtype);
  if (!tileForm(a.pages, batch, 2 * heads) || !aligned16(key) || !aligned16(value))
    return launch(k_read_any[di], {rowBlocks(batch * heads * seq)}, {256}, 0, stream, a);
  return launch(k_read[dimIndex(head_dim)][di],
                {tilesOf(seq, 64), static_cast<unsigned>(2 * heads), static_cast<unsigned>(batch)}, {256},
                0, stream, a);
}

size_t dli_hip_paged_attention_fp8_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                             int64_t seq_q, int64_t head_dim, int64_t block_size,
                                             int64_t max_blocks) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || seq_q <= 0 ||
      block_size <= 0 || max_blocks <= 0 || batch >= kMostTokens || q_heads > kMostGrid ||
      seq_q >= kMostTokens || block_size >= kMostTokens || max_blocks >= kMostTokens ||
      block_size * max_blocks >= kMostTokens)
    return 0;
  int64_t splits = 1;  // the most of any data type and number of tokens held
  for (int dtype : {DLI_F32, DLI_BF16, DLI_F16}) {
    for (bool phased : {false, true}) {
      const AttentionPlan plan = attentionPlan(dtype, batch, q_heads, kv_heads, seq_q, head_dim, block_size,
                                               block_size * max_blocks, phased);
      splits = splits > plan.splits ? splits : plan.splits;
    }
  }
  return partBytes(batch * q_heads * seq_q, head_dim, splits);
}

int dli_hip_paged_attention_fp8(int dtype, const void* q, const void* key_codes,
                                const void* value_codes, const void* scales,
                                const int32_t* block_table, int64_t num_blocks, void* out,
                                int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t seq_q,
                                int64_t head_dim, int64_t block_size, int64_t max_blocks,
                                int64_t past, const void* positions, int positions_dtype, int causal,
                                float scale, int out_bshd, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* op = "paged_attention_fp8";
  Kv8AttentionArgs a{};
  if (int rc = pagesOf(op, dtype, key_codes, value_codes, scales, block_table, num_blocks, batch, kv_heads,
                       seq_q, head_dim, block_size, max_blocks, past, positions, positions_dtype,
                       &a.pages))
    return rc;
  if (q_heads <= 0 || q_heads > kMostGrid || q_heads % kv_heads != 0)
    return badArg(op, "q_heads must be a multiple of kv_heads, at most 65535");
  if (batch == 0 || seq_q == 0) return 0;
  if (q == nullptr || out == nullptr) return badArg(op, "null input or output");
  const int64_t rows = batch * q_heads * seq_q;
  if (rows >= (int64_t{1} << 31)) return badArg(op, "too many query rows");
  const int64_t capacity = block_size * max_blocks, before = past < 0 ? 0 : past;
  const int64_t reach =
      positions != nullptr || before >= capacity || before + seq_q > capacity ? capacity : before + seq_q;
  AttentionPlan plan =
      attentionPlan(dtype, batch, q_heads, kv_heads, seq_q, head_dim, block_size, reach);
  // the MFMA forms take 16-byte loads and put masked scores to -inf before the scale's sign could
  // matter, as the other attention kernels do
  if (!(scale > 0.f) || !std::isfinite(scale) || !aligned16(q) || !aligned16(out) ||
      !aligned16(key_codes) || !aligned16(value_codes))
    plan = {0, 0, 1};
  while (plan.splits > 1 &&
         (workspace == nullptr || !aligned16(workspace) ||
          workspace_bytes < partBytes(rows, head_dim, plan.splits)))
    --plan.splits;
  a.q = q;
  a.out = out;
  a.splits = static_cast<int>(plan.splits);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = plan.splits > 1 ? a.part_o + rows * plan.splits * head_dim : nullptr;
  a.capacity = capacity;
  a.batch = static_cast<int>(batch);
  a.q_heads = static_cast<int>(q_heads);
  a.seq_q = static_cast<int>(seq_q);
  a.causal = causal != 0;
  a.out_bshd = out_bshd != 0;
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  const int di = dtypeIndex(dtype);
  if (plan.form == 0)
    return launch(k_rows[di], {static_cast<unsigned>(rows < 65536 ? rows : 65536)}, {64}, 0, stream, a);
  const int small = block_size % 64 == 0 ? 0 : 1, dim = dimIndex(head_dim);
  const unsigned units = static_cast<unsigned>(batch * kv_heads);
  int rc;
  if (plan.form == 1) {
    rc = launch(k_decode[small][dim][di], {static_cast<unsigned>(plan.splits), units}, {512}, 0, stream,
                a);
  } else {
    const int64_t tile = int64_t{64} << plan.size, pair_rows = q_heads / kv_heads * seq_q;
    DeviceKernel& chunk = plan.size == 0   ? k_chunk[small][dim][di]
                          : plan.size == 1 ? k_chunk_large[small][dtype == DLI_F16 ? 2 : dim]
                                           : k_phased;
    rc = launch(chunk,
                {static_cast<unsigned>((pair_rows + tile - 1) / tile), units,
                 static_cast<unsigned>(plan.splits)},
                {plan.size == 2 ? 512u : 256u}, 0, stream, a);
  }
  if (rc != 0 || plan.splits == 1) return rc;
  return launch(k_merge[dim][di], {blocksFor(rows, 4)}, {256}, 0, stream, a);
}

}  // extern "C"
