// Entry points of the microscaled operators (declared in include/dli_hip.h): argument checks,
// launch geometry and the launch of the matching gfx950 kernel.
#include <string>

#include "runtime.h"

namespace dli::hip {
namespace {

int badArg(const char* op, const std::string& what) {
  return fail(DLI_HIP_EINVAL, std::string(op) + ": " + what);
}

bool aligned(const void* p, uintptr_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

int dtypeIndex(int dtype) {
  return dtype == DLI_F32 ? 0 : dtype == DLI_BF16 ? 1 : dtype == DLI_F16 ? 2 : -1;
}

// The kernels <base>_<fp8|fp4>_<f32|bf16|f16> and, for data of any alignment, <...>_any.
struct MxKernels {
  DeviceKernel k[2][2][3];  // [any][format][dtype]
#define DLI_MX_NAMES(base, any)                                                          \
  {                                                                                      \
    {{"mx_quantize", base "_fp8_f32" any}, {"mx_quantize", base "_fp8_bf16" any},        \
     {"mx_quantize", base "_fp8_f16" any}},                                              \
        {{"mx_quantize", base "_fp4_f32" any}, {"mx_quantize", base "_fp4_bf16" any},    \
         {"mx_quantize", base "_fp4_f16" any}}                                           \
  }
};

MxKernels k_quantize{{DLI_MX_NAMES("mx_quantize", ""), DLI_MX_NAMES("mx_quantize", "_any")}};
MxKernels k_dequantize{{DLI_MX_NAMES("mx_dequantize", ""), DLI_MX_NAMES("mx_dequantize", "_any")}};
MxKernels k_rms_norm{{DLI_MX_NAMES("rms_norm_mx", ""), DLI_MX_NAMES("rms_norm_mx", "_any")}};
MxKernels k_silu_mul{{DLI_MX_NAMES("silu_mul_mx", ""), DLI_MX_NAMES("silu_mul_mx", "_any")}};
#define DLI_MX_LINEAR(form, odd)                                                                 \
  {                                                                                              \
    {{"mx_linear", form "_fp8_f32" odd}, {"mx_linear", form "_fp8_bf16" odd},                    \
     {"mx_linear", form "_fp8_f16" odd}},                                                        \
        {{"mx_linear", form "_fp4_f32" odd}, {"mx_linear", form "_fp4_bf16" odd},                \
         {"mx_linear", form "_fp4_f16" odd}}                                                     \
  }
#define DLI_MX_STREAM(rows, odd)                                                            \
  {                                                                                         \
    DLI_MX_LINEAR("mx_stream_r" rows "_k1", odd), DLI_MX_LINEAR("mx_stream_r" rows "_k2", odd), \
        DLI_MX_LINEAR("mx_stream_r" rows "_k4", odd),                                       \
        DLI_MX_LINEAR("mx_stream_r" rows "_k8", odd)                                        \
  }
// [rows of scales that are not whole words][activation rows: 1, 4, 16][log2 of the waves that
// split K][format][dtype]
DeviceKernel k_stream[2][3][4][2][3] = {
    {DLI_MX_STREAM("1", ""), DLI_MX_STREAM("4", ""), DLI_MX_STREAM("16", "")},
    {DLI_MX_STREAM("1", "_odd"), DLI_MX_STREAM("4", "_odd"), DLI_MX_STREAM("16", "_odd")}};

// [tile: 256 x 256, 128 x 128, 64 x 128, then the last two and 64 x up to 256 on scales as they are]
// [format][dtype]
DeviceKernel k_tile[6][2][3] = {DLI_MX_LINEAR("mx_tile_256", ""), DLI_MX_LINEAR("mx_tile_128", ""),
                                DLI_MX_LINEAR("mx_tile_64", ""), DLI_MX_LINEAR("mx_tile_128r", ""),
                                DLI_MX_LINEAR("mx_tile_64r", ""), DLI_MX_LINEAR("mx_tile_64w", "")};
DeviceKernel k_sum_parts[3] = {{"mx_linear", "mx_sum_parts_f32"},
                               {"mx_linear", "mx_sum_parts_bf16"},
                               {"mx_linear", "mx_sum_parts_f16"}};
DeviceKernel k_scale_words("mx_linear", "mx_scale_words");

// Words of 4 scales per row as the tiles read them: whole stages of 256 columns.
int64_t scaleWords(int64_t k) { return (k + 255) / 256 * 2; }

int64_t padded256(int64_t rows) { return (rows + 255) / 256 * 256; }

// Scales laid out for the tiles (mx_scale_words).
int64_t scaleWordBytes(int64_t m, int64_t n, int64_t k) {
  return scaleWords(k) * 4 * (padded256(m) + padded256(n));
}

// How a product runs: the tile (-1: the weight stream), the parts of K, and whether the tile kernel
// reads the scales as they are.
struct Plan {
  int tile, parts;
  bool rows;
  int64_t width;  // columns of a tile
};
constexpr int kTileRows[4] = {256, 128, 64, 64}, kTileColumns[3] = {256, 128, 128};

int64_t tilesOf(int tile, int64_t m, int64_t n) {
  return (m + kTileRows[tile] - 1) / kTileRows[tile] *
         ((n + kTileColumns[tile] - 1) / kTileColumns[tile]);
}

// words: the scales are rows of aligned words (K % 128 == 0).
Plan planFor(int64_t m, int64_t n, int64_t k, bool words) {
  // Row offsets within a tile are 32-bit.
  if (m <= 16 || k > (int64_t{1} << 23)) return {-1, 1, false, 0};
  // Small products stay on the stream, which takes about 3 us and one for 1000 of its units (16 x 16
  // outputs, 256 columns): 64 x 512 x 3584 5.3 us, 9.0 in tiles and their parts; 32 x 3584 x 3584 7.1
  // and 9.9 (64 rows 11.7 and 10.8); 64 x 896 x 4864 5.9 and 10.5; 200 x 896 x 896 5.7 and 6.8; 20 x 9728
  // x 896 8.7 and 6.2. The tiles' time grows with the columns that one walks, and by a launch where
  // their scales have to be laid out (333 x 1003 x 928 in fp4, a call: 8.0 and 21.6).
  const int64_t units = (m + 15) / 16 * ((n + 15) / 16) * ((k + 255) / 256);
  if (units < (words ? 3000 + (k < 5000 ? k : 5000) : 10000)) return {-1, 1, false, 0};
  // Large tiles run one to a CU, so their time goes by whole rounds of 256, whatever part of a tile's
  // rows is there; tiles of 128 run two to a CU and even out. Large ones pay where tiles of 128 would
  // take at least 1.2 + 500 / k rounds to one of theirs (their scales are laid out by a launch, and first
  // loads and the epilogue weigh more over a short K; from 1.9 rounds on they pay over any). Large tiles
  // and tiles of 128, us, fp8: 257 x 24576 x 896 22.9 and 16.9; 2048 x 9728 x 896 37.0 and 27.0, over K =
  // 8192 199 and 165; 512 x 37888 x 3584 97 and 90; 1025 x 9856 x 3584 50.9 and 55.5; 768 x 18944 x 3584 57
  // and 73, x 896 22.9 and 22.6; 8192 x 37888 x 288 238 and 263. Fewer than 192 leave too many CUs empty
  // (2000 x 3584 x 18944, 112 tiles: 205 and 138).
  const int64_t large = tilesOf(0, m, n), rounds = (large + 255) / 256, deep_k = k < 720 ? 720 : k;
  if (m > 128 && large >= 192 &&
      tilesOf(1, m, n) * deep_k * 10 >= rounds * 512 * (12 * deep_k + 5000))
    return {0, 1, false, 256};
  // Up to 64 rows are bound by what one CU can load. Where tiles of 128 columns would fall on some CUs
  // twice and on others once, every CU takes an equal run of columns instead. In tiles and in runs, us:
  // 64 x 37888 x 3584 31.1 and 24.0; over K = 8192, 33000 columns 59.7 and 49.7, 65536 89.6 and 79.8;
  // K = 18944, 33000 columns 116.7 and 98.7, 65536 166.2 and 149.3. Past two tiles to a CU both take as
  // long (70000 x 3584: 46.4 and 45.8), and over a short K the tiles' smaller stages start as soon or
  // sooner (K = 1024: 33000 columns 11.2 and 10.4, 65536 13.2 and 13.6).
  const int64_t tiles64 = tilesOf(2, m, n);
  if (m <= 64 && words && tiles64 > 256 && tiles64 <= 512 && k >= 2048)
    return {3, 1, true, ((n + 255) / 256 + 7) / 8 * 8};
  // Parts of K until the small tiles are about two to a CU (one of 64 rows), each part at least 2048
  // columns (1024): 484 x 3584 x 18944 in 1, 2, 4 and 8 parts 85.6, 58.2, 53.6 and 62.4 us; 64 rows
  // 60.0, 37.4, 26.1, 22.7 and, in 16, 26.6; 700 x 4608 x 3584 24.3 whole and 30.1 in 2.
  const int tile = m > 64 ? 1 : 2;
  const int64_t most = (tile == 1 ? 512 : 256) / tilesOf(tile, m, n);
  const int64_t deep = k / (tile == 1 ? 2048 : 1024), fit = most < deep ? most : deep;
  const int64_t parts = fit < 1 ? 1 : fit;
  // Reading scales as they are takes a cache line for every 8 bytes, over a long K more than the launch
  // that lays them out (64 x 9728 x 896: 6.5 us as they are, 9.7 laid out; 700 x 4608 x 3584: 21.1 and
  // 24.7; 484 x 3584 x 18944 in 4 parts 60.2 and 52.8; 2000 x 3584 x 18944 180 and 139).
  return {tile, static_cast<int>(parts), words && k / parts <= 4096, 128};
}

// The form of a product that has no workspace for `plan`. Tiles that read the scales as they are and
// walk all of K take about 4.5 us for 1000 of its columns and round of workgroups, the stream 0.65 us for
// 1000 of its units: 484 x 3584 x 18944 84.7 and 323 us (54.8 with the workspace), 2000 x 3584 x 18944 168
// and 1287 (140), 70 x 9728 x 8192 38.9 and 54.9, 64 x 20000 x 8192 41.4 and 82; 100 x 3584 x 18944 88 and 79,
// 64 x 3584 x 18944 77 and 47, 100 x 896 x 8192 28.6 and 11.7. Other scales than rows of words go to the
// stream, whatever it takes.
Plan planWithout(const Plan& plan, int64_t m, int64_t n, int64_t k, bool words) {
  if (plan.tile < 0 || (plan.rows && plan.parts == 1)) return plan;
  const int tile = m > 64 ? 1 : 2;
  const int64_t at_once = tile == 1 ? 512 : 256;
  const int64_t rounds = (tilesOf(tile, m, n) + at_once - 1) / at_once;
  const int64_t units = (m + 15) / 16 * ((n + 15) / 16) * ((k + 255) / 256);
  if (words && units > 7 * k * rounds) return {tile, 1, true, 128};
  return {-1, 1, false, 0};
}

size_t workspaceOf(const Plan& plan, int64_t m, int64_t n, int64_t k) {
  if (plan.tile < 0) return 0;
  return static_cast<size_t>((plan.rows ? 0 : scaleWordBytes(m, n, k)) +
                             (plan.parts > 1 ? plan.parts * m * n * 4 : 0));
}

// 0 when dtype and format are valid and [rows, k] is a shape of whole blocks.
int checkTensor(const char* op, int dtype, int format, int64_t rows, int64_t k, const char* name) {
  if (dtypeIndex(dtype) < 0)
    return badArg(op, "unsupported dtype code " + std::to_string(dtype));
  if (format != DLI_MX_FP8 && format != DLI_MX_FP4)
    return badArg(op, "unsupported format " + std::to_string(format));
  if (rows < 0 || k < 0) return badArg(op, "negative size");
  if (k % 32 != 0) return badArg(op, std::string(name) + " must be a multiple of 32");
  // element counts, offsets in bytes and chunk counts stay far inside 63 bits
  if (k > 0 && rows > (int64_t{1} << 56) / k) return badArg(op, "tensor is too large");
  return 0;
}

// 0 when mx_linear takes a product of these sizes (planFor's arithmetic stays inside 63 bits then).
int checkProduct(const char* op, int out_dtype, int x_format, int64_t m, int64_t n, int64_t k) {
  if (int rc = checkTensor(op, out_dtype, x_format, m, k, "k")) return rc;
  if (int rc = checkTensor(op, out_dtype, x_format, n, k, "k")) return rc;
  if (k == 0) return badArg(op, "k must be positive");
  if (m == 0 || n == 0) return 0;
  if (m > (int64_t{1} << 56) / n) return badArg(op, "output is too large");
  // (a launch has fewer than 2^32 threads along x: 4 per output column at most)
  if (m > 65535 * int64_t{16} || n > int64_t{1} << 29)
    return badArg(op, "m must be at most 1048560, n at most 2^29");
  if (k > int64_t{1} << 28) return badArg(op, "k must be at most 2^28");
  return 0;
}

// Grid-stride launches of one chunk (8 values) per thread: enough blocks to fill 256 CUs.
unsigned chunkBlocks(int64_t chunks) {
  const int64_t blocks = (chunks + 255) / 256;
  return static_cast<unsigned>(blocks < 8192 ? blocks : 8192);
}

}  // namespace
}  // namespace dli::hip

using namespace dli::hip;

extern "C" {

int dli_hip_mx_quantize(int dtype, int format, const void* x, void* codes, void* scales,
                        int64_t rows, int64_t k, void* stream) {
  const char* op = "mx_quantize";
  if (int rc = checkTensor(op, dtype, format, rows, k, "k")) return rc;
  if (rows == 0 || k == 0) return 0;
  if (x == nullptr || codes == nullptr || scales == nullptr) return badArg(op, "NULL pointer");
  const int any = aligned(x, 16) && aligned(codes, 8) ? 0 : 1;
  const int64_t chunks = rows * (k / 8);
  return launch(k_quantize.k[any][format][dtypeIndex(dtype)], {chunkBlocks(chunks)}, {256}, 0,
                stream, x, codes, scales, chunks);
}

int dli_hip_mx_dequantize(int dtype, int format, const void* codes, const void* scales, void* out,
                          int64_t rows, int64_t k, void* stream) {
  const char* op = "mx_dequantize";
  if (int rc = checkTensor(op, dtype, format, rows, k, "k")) return rc;
  if (rows == 0 || k == 0) return 0;
  if (out == nullptr || codes == nullptr || scales == nullptr) return badArg(op, "NULL pointer");
  const int any = aligned(out, 16) && aligned(codes, 8) ? 0 : 1;
  const int64_t chunks = rows * (k / 8);
  return launch(k_dequantize.k[any][format][dtypeIndex(dtype)], {chunkBlocks(chunks)}, {256}, 0,
                stream, codes, scales, out, chunks);
}

int dli_hip_rms_norm_mx(int dtype, int format, const void* x, const void* residual,
                        const void* weight, void* hidden_out, void* codes, void* scales,
                        int64_t rows, int64_t hidden, float eps, void* stream) {
  const char* op = "rms_norm_mx";
  if (int rc = checkTensor(op, dtype, format, rows, hidden, "hidden")) return rc;
  if (hidden == 0) return badArg(op, "hidden must be positive");
  if (rows == 0) return 0;
  if (x == nullptr || weight == nullptr || codes == nullptr || scales == nullptr)
    return badArg(op, "NULL pointer");
  const int any = aligned(x, 16) && aligned(residual, 16) && aligned(weight, 16) &&
                          aligned(hidden_out, 16) && aligned(codes, 8)
                      ? 0
                      : 1;
  const unsigned blocks = static_cast<unsigned>(rows < 65535 ? rows : 65535);
  // A chunk of 8 values per thread, up to 4 waves. 8192 rows of 896: 21.6 us with 4 waves, 17.1 with
  // 2 or 1; 333 of 4864: 16.8 with 1, 10.7 with 2, 7.2 with 4.
  const unsigned threads = hidden <= 512 ? 64 : hidden <= 1024 ? 128 : 256;
  return launch(k_rms_norm.k[any][format][dtypeIndex(dtype)], {blocks}, {threads}, 0, stream, x,
                residual, weight, hidden_out, codes, scales, rows, hidden,
                1.0 / static_cast<double>(hidden), eps);
}

int dli_hip_silu_mul_mx(int dtype, int format, const void* gate, const void* up, int64_t stride,
                        void* codes, void* scales, int64_t rows, int64_t ffn, void* stream) {
  const char* op = "silu_mul_mx";
  if (int rc = checkTensor(op, dtype, format, rows, ffn, "ffn")) return rc;
  if (stride < ffn) return badArg(op, "stride must be at least ffn");
  if (stride > 0 && rows > (int64_t{1} << 56) / stride) return badArg(op, "tensor is too large");
  if (rows == 0 || ffn == 0) return 0;
  if (gate == nullptr || up == nullptr || codes == nullptr || scales == nullptr)
    return badArg(op, "NULL pointer");
  const int any = aligned(gate, 16) && aligned(up, 16) && aligned(codes, 8) &&
                          (dtype == DLI_F32 ? stride % 4 : stride % 8) == 0
                      ? 0
                      : 1;
  const int64_t row_chunks = ffn / 8;
  return launch(k_silu_mul.k[any][format][dtypeIndex(dtype)], {chunkBlocks(rows * row_chunks)},
                {256}, 0, stream, gate, up, stride, codes, scales, rows, row_chunks);
}

size_t dli_hip_mx_linear_workspace(int x_format, int64_t m, int64_t n, int64_t k) {
  if (checkProduct("mx_linear", DLI_F32, x_format, m, n, k) != 0 || m == 0 || n == 0) return 0;
  return workspaceOf(planFor(m, n, k, k % 128 == 0), m, n, k);
}

int dli_hip_mx_linear(int x_format, int out_dtype, const void* x_codes, const void* x_scales,
                      const void* w_codes, const void* w_scales, const void* bias,
                      const void* residual, void* out, int64_t m, int64_t n, int64_t k,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "mx_linear";
  if (int rc = checkProduct(op, out_dtype, x_format, m, n, k)) return rc;
  if (m == 0 || n == 0) return 0;
  if (x_codes == nullptr || x_scales == nullptr || w_codes == nullptr || w_scales == nullptr ||
      out == nullptr)
    return badArg(op, "NULL pointer");
  if (!aligned(x_codes, 16) || !aligned(w_codes, 16))
    return badArg(op, "codes must be 16-byte aligned");
  const bool words = k % 128 == 0 && aligned(x_scales, 4) && aligned(w_scales, 4);
  Plan plan = planFor(m, n, k, words);
  if (workspace == nullptr || workspace_bytes < workspaceOf(plan, m, n, k) || !aligned(workspace, 16))
    plan = planWithout(plan, m, n, k, words);
  if (plan.tile >= 0) {
    const int64_t scale_bytes = plan.rows ? 0 : scaleWordBytes(m, n, k);
    const int64_t m_pad = padded256(m), n_pad = padded256(n), row_words = scaleWords(k);
    auto* const parts = plan.parts > 1 ? static_cast<char*>(workspace) + scale_bytes : nullptr;
    const void *xw = x_scales, *ww = w_scales;
    if (!plan.rows) {
      auto* const to = static_cast<uint32_t*>(workspace);
      xw = to;
      ww = to + row_words * m_pad;
      if (int rc = launch(k_scale_words,
                          {static_cast<unsigned>((m_pad + n_pad) / 64), blocksFor(row_words, 16)},
                          {256}, 0, stream, x_scales, w_scales, xw, ww, m, n,
                          static_cast<int>(k / 32), m_pad, n_pad))
        return rc;
    }
    const unsigned threads = plan.tile == 3 || (plan.tile == 0 && x_format == DLI_MX_FP8) ? 512 : 256;
    if (int rc = launch(k_tile[plan.tile + (plan.rows ? 2 : 0)][x_format][dtypeIndex(out_dtype)],
                        {blocksFor(n, plan.width), blocksFor(m, kTileRows[plan.tile]),
                         static_cast<unsigned>(plan.parts)},
                        {threads}, 0, stream, x_codes, xw, w_codes, ww, bias, residual, out, parts,
                        m, n, k, m_pad, n_pad, static_cast<int>(plan.width)))
      return rc;
    if (parts == nullptr) return 0;
    return launch(k_sum_parts[dtypeIndex(out_dtype)], {chunkBlocks((m * n + 7) / 8)}, {256}, 0,
                  stream, parts, plan.parts, bias, residual, out, m, n);
  }
  const int odd = words ? 0 : 1;
  const int form = m == 1 ? 0 : m <= 4 ? 1 : 2, rows = form == 0 ? 1 : form == 1 ? 4 : 16;
  // The waves that share K: about 2048 in all, up to two for a unit of 256 columns and four for 512 (half
  // of them without a unit then: their places hold fewer tiles to a workgroup, which is no slower for few
  // outputs). us: 1152 outputs, 16 rows, K = 256 on one wave and two 3.63 and 3.42, K = 512 on two and four
  // 3.85 and 3.61; 9728, one row, 3.60 and 3.46, 3.86 and 3.87; but 9728, 16 rows in fp8, K = 512 on two and
  // four 4.24 and 5.73, as the workgroups of four no longer fit on the card at once. Eight share from 4096
  // on (4608 x 3584, one row: 7.8 us on 8, 5.4 on 4; 3584 x 18944: 9.9 and 10.6).
  const int64_t tiles = (n + 15) / 16;
  int split = 0;
  while (split < 3 && (tiles << split) < 2048 && k >= (split < 2 ? 256 << split : 4096)) ++split;
  const int waves = split < 3 ? 4 : 8;
  return launch(k_stream[odd][form][split][x_format][dtypeIndex(out_dtype)],
                {blocksFor(n, 16 * (waves >> split)), blocksFor(m, rows)},
                {static_cast<unsigned>(64 * waves)}, 0, stream, x_codes, x_scales, w_codes,
                w_scales, bias, residual, out, m, n, k);
}

}  // extern "C"
