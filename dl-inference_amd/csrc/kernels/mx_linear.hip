// Linears on microscaled 4-bit weights on gfx950:
//   out[m, n] = sum_k x[m, k] * w[n, k] (+ bias[n]) (+ residual[m, n])
// on v_mfma_scale_f32_16x16x128_f8f6f4, which takes e4m3 or e2m1 elements with their blocks' scale
// codes and multiplies and scales in one instruction.
//
// Operand layout (lane l, g = l / 16): e2m1, 16 bytes: row l % 16, k = 32 g .. 32 g + 31; e4m3,
// 2 x 16 bytes: k = 16 g .. 16 g + 15, then the same + 64. The scale byte of lane l is that of row
// l % 16, block g of the 128 columns, for either element type. D[(l / 16) * 4 + i][l % 16].
#include "gemm_tiles.h"
#include "mx.h"

using namespace dk;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The 16 or 32 bytes of one operand row that a lane feeds to one instruction (128 columns).
template <class F>
struct Frag {
  U32x4 q[F::kWords];
};

template <class F>
__device__ __forceinline__ i32x8 operand(const Frag<F>& f) {
  i32x8 v;
  const U32x4 lo = f.q[0], hi = f.q[F::kWords - 1];  // e2m1: the upper four registers are not read
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = static_cast<int>(lo[i]);
    v[4 + i] = static_cast<int>(hi[i]);
  }
  return v;
}

// x = lo + hi, the elements of exponent fields 0..8 and 9..15 (see mma)
template <class F>
__device__ __forceinline__ void splitFp8(const Frag<F>& x, Frag<F>& lo, Frag<F>& hi) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // per byte: bit 7 of field + 0x38 is set from exponent field 9 (0x48) on
      const uint32_t top = ((x.q[j][i] & 0x78787878u) + 0x38383838u) & 0x80808080u;
      const uint32_t mask = (top - (top >> 7)) | top;
      hi.q[j][i] = x.q[j][i] & mask;
      lo.q[j][i] = x.q[j][i] & ~mask;
    }
}

// c + w x, w a fragment of 16 weight rows (e2m1), x one of 16 activation rows.
//
// Precision: the unit adds the products of 8 neighbouring columns after aligning them to the largest
// of the 8 and drops what lies below 2^-13 of it, at most 7 x 2^-13 of the largest; further sums are
// fp32. Products of two e2m1 values span less than that and are exact. With e4m3 rows the relative
// 2-norm error is 4e-6, a fiftieth of what rounding a result to f16 adds and less of bf16's. One group
// can lose more: less than half a step of bf16 (2^-8), up to 1.75 halves of f16's (2^-11), of its largest
// product, and beside large products that cancel the small ones go. kSplit loses nothing: the e4m3
// values of exponent fields 0..8 and 9..15 are multiplied by themselves; within each group the products
// of 8 columns span at most 13 bits. It takes the matrix unit twice, so only fp32 results have it (bf16
// results without and with, us: 1 x 37888 x 3584 14.9 and 18.6, 64 rows 26.1 and 33.6, 2000 x 3584 x 18944
// 131 and 250, 8192 x 37888 x 3584 932 and 2310): a caller that needs it takes fp32.
template <class F, bool kSplit>
__device__ __forceinline__ f32x4 mma(const Frag<MxFp4>& w, uint32_t sw, const Frag<F>& x,
                                     uint32_t sx, f32x4 c) {
  constexpr int kFp8 = 0, kFp4 = 4;
  constexpr int kX = F::kWords == 2 ? kFp8 : kFp4;
  if constexpr (kSplit && F::kWords == 2) {
    Frag<F> lo, hi;
    splitFp8(x, lo, hi);
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(lo), c, kFp4, kX, 0,
                                                         sw, 0, sx);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(hi), c, kFp4, kX,
                                                            0, sw, 0, sx);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w), operand(x), c, kFp4, kX, 0,
                                                            sw, 0, sx);
  }
}

template <int V>
struct Int {
  static constexpr int value = V;
};

// ---- loads straight into LDS ---------------------------------------------------------------------
// global_load_lds writes the wave's 64 x 16 (or 4) bytes to consecutive LDS addresses from m0 on and
// holds no registers while in flight. As inline assembly with explicit waits: for the builtin the
// compiler waits for every load in flight before any LDS read, which would empty the pipeline. The
// statements have no outputs; "memory" keeps LDS reads on their side of a wait or a load.
template <int kBytes, bool kStream>
__device__ __forceinline__ void loadLds(const uint8_t* base, uint32_t offset, uint32_t lds) {
  if constexpr (kBytes == 16 && kStream)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
  else if constexpr (kBytes == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :: "s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}

// All but the last n of the wave's vector memory operations are done.
template <int n>
__device__ __forceinline__ void waitLoads() {
  static_assert(n < 64, "vmcnt has 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(n) : "memory");
}

__device__ __forceinline__ void waitLdsReads() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

__device__ __forceinline__ uint32_t ldsAddress(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) void*)p));
}

__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// ---- few rows: a weight stream ---------------------------------------------------------------
// A wave owns 16 weight rows, up to kRows activation rows and a run of K in units of 256 columns (a
// 128-byte line of every weight row). KW waves share the rows and split K; their tiles are summed
// through LDS in order. Each wave streams its units through a ring of its own in LDS: no barrier, and
// kDepth units in flight.
//
// Why through LDS: an instruction that loads a fragment directly touches 16 rows x 64 bytes, and the
// cache handles a line per 4 cycles, so 8 units of 256 columns took a CU 2400 cycles (16 activation
// rows: 4600) however many were in flight. Staged, an instruction covers 8 whole lines.
//
// One row of 37888 x 3584 from memory: 16 us, 4.5 TB/s of weights; of 1152 x 896 3.0 us, where the chain
// of a load, the MFMAs, the join of the waves and a store is all there is. 16 rows of 37888 x 3584: 23
// us; every wave reads all activation rows, twice the bytes of its weights.
constexpr int kMaxRun = 16;  // units whose scales a wave holds at once (128 bytes per row)

template <class F, int kRows>
struct Stream {
  static constexpr int kXRow = 128 * F::kWords;                 // bytes of a row's unit
  static constexpr int kXBytes = kRows * kXRow < 256 ? 256 : kRows * kXRow;
  static constexpr int kXLoads = kRows == 1 ? 1 : (kXBytes + 1023) / 1024;
  static constexpr int kXSlot = kRows == 1 ? 256 : kXLoads * 1024;
  static constexpr int kSlot = 2048 + kXSlot, kLoads = 2 + kXLoads;
  static constexpr int kScales = (16 + kRows) * kMaxRun * 8;
};

template <class F, class T, int kRows, int KW, int kDepth, bool kScales4>
__device__ __forceinline__ void mx_linear_stream(const uint8_t* x, const uint8_t* xs,
                                                 const uint8_t* w, const uint8_t* ws,
                                                 const void* bias, const void* residual, void* out,
                                                 int64_t M, int64_t N, int64_t K) {
  using S = Stream<F, kRows>;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int kWaves = KW > 4 ? KW : 4, kTiles = kWaves / KW;
  constexpr int kWaveBytes = kDepth * S::kSlot + S::kScales;
  static_assert(kWaveBytes >= 1024, "room for the wave's sums");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kWaves * kWaveBytes];
  const int lane = threadIdx.x % kWave, g = lane / 16, r = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int kw = wave % KW;
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) * kTiles + wave / KW) * 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kRows;
  const int64_t blocks = K / kMxBlock;
  const int units = static_cast<int>((K + 255) / 256);
  const int last = static_cast<int>(blocks) - (units - 1) * 8;  // blocks of the last unit, 1 to 8
  // the wave's units: a run of units / KW, one more for the last waves
  const int more = KW - units % KW;
  const int mine = units / KW + (kw >= more ? 1 : 0);
  const int first = units / KW * kw + (kw >= more ? kw - more : 0);
  const int partial = last < 8 && first + mine == units ? mine - 1 : -1;  // of the wave's units
  uint8_t* const ring = smem + wave * kWaveBytes;
  uint32_t* const sw = reinterpret_cast<uint32_t*>(ring + kDepth * S::kSlot);
  uint32_t* const sx = sw + 16 * kMaxRun * 2;
  const uint32_t ringAt = __builtin_amdgcn_readfirstlane(ldsAddress(ring));
  // rows past the last one stand for it: their results are dropped
  const int64_t wBase = n0 < N ? n0 : N - 1;
  const int64_t wLast = N - 1 - wBase, xLast = M - 1 - m0;
  auto wRow = [&](int row) { return static_cast<uint32_t>(row < wLast ? row : wLast); };
  auto xRow = [&](int row) { return static_cast<uint32_t>(row < xLast ? row : xLast); };
  const uint32_t wStride = static_cast<uint32_t>(K / 2);
  const uint32_t xStride = static_cast<uint32_t>(K * F::kWords / 2);
  const uint8_t* const wTile = uniform(w + wBase * (K / 2) + static_cast<int64_t>(first) * 128);
  const uint8_t* const xTile = uniform(x + m0 * (K * F::kWords / 2) +
                                      static_cast<int64_t>(first) * S::kXRow);
  // chunk (16 bytes) p of a row of 128 bytes sits at p ^ ((row / 2) % 8), of 256 bytes at
  // p ^ (row % 16): the 16 rows of a fragment read then fall on different banks
  uint32_t wOff[2], xOff[S::kXLoads];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = i * 8 + lane / 8;
    wOff[i] = wRow(row) * wStride + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
  }
#pragma unroll
  for (int i = 0; i < S::kXLoads; ++i) {
    if constexpr (kRows == 1) {
      xOff[i] = (lane * 4) % S::kXRow;
    } else {
      constexpr int kPer = S::kXRow / 16;  // chunks per row
      const int row = (i * 64 + lane) / kPer % kRows, c = lane % kPer;
      xOff[i] = xRow(row) * xStride + (c ^ (kPer == 8 ? (row >> 1) & 7 : row)) * 16;
    }
  }
  auto issue = [&](int u, int slot) {  // unit u of the wave's
    const uint32_t at = ringAt + slot * S::kSlot;
    const uint8_t* const pw = wTile + static_cast<int64_t>(u) * 128;
    const uint8_t* const px = xTile + static_cast<int64_t>(u) * S::kXRow;
    if (u != partial) {
#pragma unroll
      for (int i = 0; i < 2; ++i) loadLds<16, true>(pw, wOff[i], at + i * 1024);
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i)
        loadLds<kRows == 1 ? 4 : 16, false>(px, xOff[i], at + 2048 + i * 1024);
    } else {  // columns past the last one stand for it: their weights are multiplied as zeros
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = i * 8 + lane / 8, c = (lane % 8) ^ ((row >> 1) & 7);
        loadLds<16, true>(pw, wRow(row) * wStride + (c < last ? c : last - 1) * 16, at + i * 1024);
      }
      const int xBytes = last * 16 * F::kWords;
#pragma unroll
      for (int i = 0; i < S::kXLoads; ++i) {
        uint32_t off = xOff[i];
        if constexpr (kRows == 1) {
          off = off < xBytes - 4u ? off : xBytes - 4u;
        } else {
          constexpr int kPer = S::kXRow / 16;
          const int row = (i * 64 + lane) / kPer % kRows;
          const uint32_t in = off - xRow(row) * xStride;
          off = off - in + (in < xBytes - 16u ? in : xBytes - 16u);
        }
        loadLds<kRows == 1 ? 4 : 16, false>(px, off, at + 2048 + i * 1024);
      }
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  int pad = 2;  // words of scales per row of the run, a power of two
  auto multiply = [&](int u, int slot, int live = 8) {  // unit u of the run, `live` blocks of 8
    const uint8_t* const at = ring + slot * S::kSlot;
    const int xr = r % kRows;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Frag<MxFp4> fw;
      Frag<F> fx;
      fw.q[0] = *reinterpret_cast<const U32x4*>(at + r * 128 + ((h * 4 + g) ^ ((r >> 1) & 7)) * 16);
#pragma unroll
      for (int j = 0; j < F::kWords; ++j) {
        const int c = F::kWords == 2 ? h * 8 + j * 4 + g : h * 4 + g;
        fx.q[j] = *reinterpret_cast<const U32x4*>(
            at + 2048 + xr * S::kXRow + (c ^ (F::kWords == 2 ? xr : (xr >> 1) & 7)) * 16);
      }
      if (h * 4 + g >= live) fw.q[0] = U32x4{0u, 0u, 0u, 0u};
      const int d = u * 2 + h;
      const uint32_t a = sw[r * pad + ((d + 2 * r) & (pad - 1))];
      const uint32_t b = sx[xr * pad + ((d + 2 * xr) & (pad - 1))];
      acc = mma<F, kSplit>(fw, a >> (8 * g), fx, b >> (8 * g), acc);
    }
  };
  for (int done = 0; done < mine; done += kMaxRun) {
    const int n = mine - done < kMaxRun ? mine - done : kMaxRun;
    pad = 2;
    while (pad < 2 * n) pad *= 2;
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (d < n) issue(done + d, d);
    // The run's scales. Word d of row `row` sits at (d + 2 row) % pad, so that a word of all rows
    // is read from different banks; blocks past the run repeat its last one.
    const int b0 = (first + done) * 8, left = static_cast<int>(blocks) - b0;
    const int there = left < n * 8 ? left : n * 8;
    auto stage = [&](const uint8_t* base, int64_t row0, auto rows, uint32_t* to, auto rowOf) {
      constexpr int kRuns = (decltype(rows)::value * kMaxRun * 2 + kWave - 1) / kWave;
      const int words = decltype(rows)::value * pad;
      uint32_t v[kRuns];
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
        const int i = j * kWave + lane;
        if (j * kWave >= words) break;
        const int at = i < words ? i : words - 1, row = at / pad;
        const int b = (((at % pad) - 2 * row) & (pad - 1)) * 4;  // the word's first block
        const uint8_t* p = base + (row0 + rowOf(row)) * blocks + b0;
        if constexpr (kScales4) {
          v[j] = *gp(reinterpret_cast<const uint32_t*>(p + (b < there ? b : there - 4)));
        } else {
          v[j] = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            v[j] |= static_cast<uint32_t>(gp(p)[b + q < there ? b + q : there - 1]) << (8 * q);
        }
      }
#pragma unroll
      for (int j = 0; j < kRuns; ++j)
        if (j * kWave + lane < words) to[j * kWave + lane] = v[j];
    };
    stage(ws, wBase, Int<16>{}, sw, wRow);
    stage(xs, m0, Int<kRows>{}, sx, xRow);
    int slot = 0, u = 0;
    for (; u + kDepth <= n; ++u) {  // kDepth - 1 units in flight behind this one
      waitLoads<(kDepth - 1) * S::kLoads>();
      multiply(u, slot);
      waitLdsReads();
      if (u + kDepth < n) issue(done + u + kDepth, slot);
      slot = slot + 1 == kDepth ? 0 : slot + 1;
    }
    auto drain = [&](auto behind) {
      constexpr int kBehind = decltype(behind)::value;
      if (kBehind < kDepth - 1 && kBehind < n) {
        waitLoads<kBehind * S::kLoads>();
        if (kBehind == 0 && done + u == partial) multiply(u, slot, last);
        else multiply(u, slot);
        ++u;
        slot = slot + 1 == kDepth ? 0 : slot + 1;
      }
    };
    static_assert(kDepth >= 2 && kDepth <= 4, "units in flight (the partial one is drained)");
    drain(Int<2>{});
    drain(Int<1>{});
    drain(Int<0>{});
    waitLdsReads();
  }
  auto finish = [&](int64_t m, int64_t n, float v) {
    if (m >= M || n >= N) return;
    if (bias != nullptr) v += ld(static_cast<const T*>(bias) + n);
    if (residual != nullptr) v += ld(static_cast<const T*>(residual) + m * N + n);
    st(static_cast<T*>(out) + m * N + n, v);
  };
  if constexpr (KW == 1) {
    if (r < kRows)
#pragma unroll
      for (int i = 0; i < 4; ++i) finish(m0 + r, n0 + g * 4 + i, acc[i]);
  } else {
    // [m][n] over the wave's ring: 4 consecutive n of one m per lane
    *reinterpret_cast<f32x4*>(ring + (r * 16 + g * 4) * 4) = acc;
    __syncthreads();
    for (int e = threadIdx.x; e < kTiles * kRows * 16; e += kWaves * kWave) {
      const int tile = e / (kRows * 16), at = e % (kRows * 16);
      const uint8_t* const p = smem + tile * KW * kWaveBytes + at * 4;
      float v = *reinterpret_cast<const float*>(p);
#pragma unroll
      for (int q = 1; q < KW; ++q) v += *reinterpret_cast<const float*>(p + q * kWaveBytes);
      finish(m0 + at / 16, (static_cast<int64_t>(blockIdx.x) * kTiles + tile) * 16 + at % 16, v);
    }
  }
}

// ---- many rows: tiles on the matrix units ------------------------------------------------------
// A workgroup of WM x WN waves owns a BM x BN tile of out, each wave BM / WM x BN / WN of it as 32 x 32
// MFMA tiles (v_mfma_scale_f32_32x32x64_f8f6f4; lane l, g = l / 32: e2m1 k = 32 g .. 32 g + 31,
// e4m3 16 bytes from k = 16 g and 16 from 32 + 16 g, scale byte of row l % 32 and block g).
// K goes by in stages of KS columns through ST buffers in LDS, loaded straight into them; fragments
// are read from LDS one step of 64 columns ahead of the MFMAs that use them.
//
// A 256 x 256 tile takes 64 KB from L2 per 256 columns and 2048 cycles of e2m1 MFMAs, 32 bytes a
// cycle, and 64 of the 128 bytes a cycle that LDS can read. The sums fill 256 registers of a wave,
// so one wave runs per SIMD.
//
// 8192 x 37888 x 3584 on e2m1 rows: 640 us, 3.5 PFLOP/s, MFMA busy 43% at 1.96 GHz, no LDS conflicts. A
// stage of 256 columns takes 1.9 us (MFMAs alone, limited by power, about 1.3; with every load hitting
// one line the whole product takes 540 us), and a round of tiles about 9 us for its first loads and its
// epilogue (one workgroup per CU that loads the next tile's first stage during the epilogue: 2% less).
// 2000 x 3584 x 18944 on e4m3 rows in 128 x 128 tiles: 133 us and 5 for the scales, MFMA busy 49%; the
// 448 tiles leave an eighth of the places empty, and LDS serves 141 bytes a cycle at full rate, more
// than it has (128 x 256 tiles: 5% less here, 15% more at 4096 x 3584 x 3584).
//
// Scales: one word (4 blocks, 128 columns) per row and step pair, read as xw / ww[word][row] (rows of
// mPad / nPad words, mx_scale_words below), so that a load of them is contiguous.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class F, bool kSplit, int kHalf>
__device__ __forceinline__ f32x16 mma32(const Frag<MxFp4>& w, uint32_t sw, const Frag<F>& x,
                                        uint32_t sx, f32x16 c) {
  constexpr int kX = F::kWords == 2 ? 0 : 4;
  if constexpr (kSplit && F::kWords == 2) {
    Frag<F> lo, hi;
    splitFp8(x, lo, hi);
    c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(lo), c, 4, kX,
                                                        2 * kHalf, sw, 2 * kHalf, sx);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(hi), c, 4, kX,
                                                           2 * kHalf, sw, 2 * kHalf, sx);
  } else {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w), operand(x), c, 4, kX,
                                                           2 * kHalf, sw, 2 * kHalf, sx);
  }
}

template <class F, int BM, int BN, int KS, int kWaves, bool kRowScales>
struct Big {
  static constexpr int kXRow = KS * F::kWords / 2, kWRow = KS / 2;  // bytes of a row's stage
  static constexpr int kX = BM * kXRow, kW = BN * kWRow, kWordsK = KS / 128;
  static constexpr int kScales = kWordsK * (BM + BN) * 4;
  static constexpr int kStage = kX + kW + kScales;
  static constexpr int kSBytes = !kRowScales && kScales % (1024 * kWaves) == 0 ? 16 : 4;  // of a lane
  static constexpr int kSRows = kRowScales ? 64 / kWordsK : 16 * kSBytes;  // rows of a load of scales
  static constexpr int kXLoads = kX / (1024 * kWaves), kWLoads = kW / (1024 * kWaves);
  static constexpr int kSAll = kScales / (64 * kSBytes);  // loads of scales
  static constexpr int kSLoads = (kSAll + kWaves - 1) / kWaves;
  static constexpr int kLoads = kXLoads + kWLoads + kSLoads;  // of a wave, per stage
  static_assert(kX % (1024 * kWaves) == 0 && kW % (1024 * kWaves) == 0 &&
                    kScales % (64 * kSBytes) == 0 && BM % kSRows == 0 && BN % kSRows == 0,
                "whole loads");
};

__device__ __forceinline__ U32x4 ldsRead16(uint32_t at) {
  return *(const __attribute__((address_space(3))) U32x4*)at;
}
__device__ __forceinline__ uint32_t ldsRead4(uint32_t at) {
  return *(const __attribute__((address_space(3))) uint32_t*)at;
}

// Chunk (16 bytes) c of row `row` of a stage sits at c ^ chunkSwizzle: the 16 rows that LDS serves at
// once then fall on different banks.
template <int kRow>
__device__ __forceinline__ int chunkSwizzle(int row) {
  return kRow == 256 ? row & 15 : kRow == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
}

template <class F, class T, int BM, int BN, int WM, int WN, int KS, int ST, bool kRowScales>
__device__ __forceinline__ void mx_linear_big(const uint8_t* x, const uint32_t* xw,
                                              const uint8_t* w, const uint32_t* ww,
                                              const void* bias, const void* residual, void* out,
                                              float* parts, int64_t M, int64_t N, int64_t K,
                                              int64_t mPad, int64_t nPad, int width) {
  constexpr int kWaves = WM * WN, kM = BM / WM, kN = BN / WN;  // a wave's part of the tile
  using B = Big<F, BM, BN, KS, kWaves, kRowScales>;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int TM = kM / 32, TN = kN / 32, NK = KS / 64;
  static_assert(NK % 2 == 0 && ST >= 2 && ST <= 3 && kN % 64 == 0, "stages, and the epilogue's runs");
  constexpr int kPitch = kN + 4;  // floats of a row of the epilogue's slab (32 rows per wave)
  constexpr int kEpilogue = kWaves * 32 * kPitch * 4;
  constexpr int kBytes = ST * B::kStage > kEpilogue ? ST * B::kStage : kEpilogue;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kBytes];
  const int lane = threadIdx.x % kWave, r = lane % 32, g = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  int64_t m0, n0;
  const int bn = kRowScales && BM == 64 ? width : BN;  // the tile's columns, a multiple of 8
  groupedTile(BM, bn, m0, n0);
  const int blocks = static_cast<int>(K / kMxBlock);
  // the stages of this part of K (blockIdx.z of gridDim.z), and the blocks of its last one
  const int all = static_cast<int>((K + KS - 1) / KS);
  const int from = static_cast<int>(static_cast<int64_t>(all) * blockIdx.z / gridDim.z);
  const int stages = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.z + 1) / gridDim.z) - from;
  const int live = from + stages == all ? blocks - (all - 1) * (KS / kMxBlock) : KS / kMxBlock;
  const uint32_t ldsAt = __builtin_amdgcn_readfirstlane(ldsAddress(smem));
  const uint32_t xStride = static_cast<uint32_t>(K * F::kWords / 2);
  const uint32_t wStride = static_cast<uint32_t>(K / 2);
  const uint8_t* const xTile = uniform(x + m0 * (K * F::kWords / 2) + static_cast<int64_t>(from) * B::kXRow);
  const uint8_t* const wTile = uniform(w + n0 * (K / 2) + static_cast<int64_t>(from) * B::kWRow);
  // the rows' scales as they are, of x and w (kRowScales)
  const uint8_t* const xsTile = uniform(reinterpret_cast<const uint8_t*>(xw) + (kRowScales ? m0 * blocks : 0));
  const uint8_t* const wsTile = uniform(reinterpret_cast<const uint8_t*>(ww) + (kRowScales ? n0 * blocks : 0));
  const int mLast = static_cast<int>(M - 1 - m0 < BM ? M - 1 - m0 : BM - 1);
  const int nLast = static_cast<int>(N - 1 - n0 < bn ? N - 1 - n0 : bn - 1);
  const int64_t nEnd = n0 + nLast + 1;

  // ---- loads ----
  constexpr int kXPer = B::kXRow / 16, kWPer = B::kWRow / 16;  // chunks per row
  uint32_t xOff[B::kXLoads], wOff[B::kWLoads];
  // the lane's rows lie whole multiples of 16 rows apart, so its chunk is the same in each
  const int xRow0 = wave * (64 / kXPer) + lane / kXPer, wRow0 = wave * (64 / kWPer) + lane / kWPer;
  const int xChunk = (lane % kXPer) ^ chunkSwizzle<B::kXRow>(xRow0);
  const int wChunk = (lane % kWPer) ^ chunkSwizzle<B::kWRow>(wRow0);
  static_assert(kWaves * 64 / kXPer % 16 == 0 && kWaves * 64 / kWPer % 16 == 0, "rows of a load");
#pragma unroll
  for (int i = 0; i < B::kXLoads; ++i) {
    const int row = xRow0 + i * (kWaves * 64 / kXPer);
    xOff[i] = static_cast<uint32_t>(row < mLast ? row : mLast) * xStride + xChunk * 16;
  }
#pragma unroll
  for (int i = 0; i < B::kWLoads; ++i) {
    const int row = wRow0 + i * (kWaves * 64 / kWPer);
    wOff[i] = static_cast<uint32_t>(row < nLast ? row : nLast) * wStride + wChunk * 16;
  }
  // before stage s is loaded: the last stage's columns past K stand for its last block
  auto prepare = [&](int s) {
    if (s + 1 == stages && live < KS / kMxBlock) {
      const int xMost = live * F::kWords - 1, wMost = live - 1;
      const uint32_t xBack = xChunk > xMost ? (xChunk - xMost) * 16 : 0;
      const uint32_t wBack = wChunk > wMost ? (wChunk - wMost) * 16 : 0;
#pragma unroll
      for (int i = 0; i < B::kXLoads; ++i) xOff[i] -= xBack;
#pragma unroll
      for (int i = 0; i < B::kWLoads; ++i) wOff[i] -= wBack;
    }
  };
  // load i of stage s into its buffer
  auto issue = [&](int s, int buffer, int i) {
    const uint32_t at = ldsAt + buffer * B::kStage;
    if (i < B::kXLoads) {
      loadLds<16, false>(xTile + static_cast<int64_t>(s) * B::kXRow, xOff[i],
                         at + (i * kWaves + wave) * 1024);
    } else if (i < B::kXLoads + B::kWLoads) {
      const int j = i - B::kXLoads;
      loadLds<16, false>(wTile + static_cast<int64_t>(s) * B::kWRow, wOff[j],
                         at + B::kX + (j * kWaves + wave) * 1024);
    } else {
      // (with fewer loads than waves to make them, some are made twice)
      int q = (i - B::kXLoads - B::kWLoads) * kWaves + wave;
      if constexpr (B::kSAll % kWaves != 0) q = q < B::kSAll ? q : B::kSAll - 1;
      const uint32_t to = at + B::kX + B::kW + q * 256 * (B::kSBytes / 4);
      if constexpr (kRowScales) {
        // [x rows | w rows][word] from the scales as they are: rows of whole words (K % 128 == 0),
        // words past the last one stand for it
        const int row = q * B::kSRows + lane / B::kWordsK, here = row < BM ? row : row - BM;
        const int most = row < BM ? mLast : nLast;
        int word = (from + s) * B::kWordsK + lane % B::kWordsK;
        word = word < blocks / 4 ? word : blocks / 4 - 1;
        const bool isX = q * B::kSRows < BM;
        loadLds<4, false>(isX ? xsTile : wsTile,
                          static_cast<uint32_t>(here < most ? here : most) * blocks + word * 4, to);
      } else {
        // [word][x rows | w rows]
        constexpr int kPerWord = (BM + BN) / B::kSRows;
        const int64_t word = static_cast<int64_t>(from + s) * B::kWordsK + q / kPerWord;
        const int row = q % kPerWord * B::kSRows;
        const uint32_t* p = row < BM ? xw + word * mPad + m0 + row : ww + word * nPad + n0 + row - BM;
        loadLds<B::kSBytes, false>(uniform(reinterpret_cast<const uint8_t*>(p)), lane * B::kSBytes, to);
      }
    }
  };

  // ---- fragments ----
  struct Frags {
    Frag<MxFp4> w[TN];
    Frag<F> x[TM];
  };
  struct Scales {
    uint32_t w[TN], x[TM];
  };
  // LDS addresses of the lane's row in a buffer, and its chunk of step 0; another chunk of the row is
  // an exclusive or away, since rows are whole multiples of 64 bytes. Passed through an empty asm
  // once per stage, so that the compiler does not hold one address per step and buffer.
  const int xr = wm * kM + r, wr = wn * kN + r;
  const uint32_t xBase = ldsAt + xr * B::kXRow + ((g ^ chunkSwizzle<B::kXRow>(xr)) * 16);
  const uint32_t wBase = ldsAt + B::kX + wr * B::kWRow + ((g ^ chunkSwizzle<B::kWRow>(wr)) * 16);
  constexpr int kSRow = kRowScales ? 4 * B::kWordsK : 4;         // bytes from row to row
  constexpr int kSWord = kRowScales ? 4 : (BM + BN) * 4;  // and from word to word
  const uint32_t sBase = ldsAt + B::kX + B::kW + xr * kSRow;
  struct At {
    uint32_t x, w, s;
  };
  auto atBuffer = [&](int buffer) {
    const uint32_t off = buffer * B::kStage;
    At at = {xBase + off, wBase + off, sBase + off};
    asm volatile("" : "+v"(at.x), "+v"(at.w), "+v"(at.s));
    return at;
  };
  // read i of the fragments of a step (kReads of them), then of the scale words of a step pair
  constexpr int kReads = TN + TM * F::kWords;
  auto read = [&](const At& at, auto step, int i, Frags& f) {
    constexpr int kStep = decltype(step)::value;
    if (i < TN) {
      f.w[i].q[0] = ldsRead16((at.w ^ (kStep * 32)) + i * 32 * B::kWRow);
    } else {
      const int q = (i - TN) / F::kWords, h = (i - TN) % F::kWords;
      f.x[q].q[h] = ldsRead16((at.x ^ (kStep * 32 * F::kWords + h * 32)) + q * 32 * B::kXRow);
    }
  };
  const int wFromX = (BM + wr - xr) * kSRow;
  auto readScale = [&](const At& at, int word, int i, Scales& s) {
    const uint32_t p = at.s + word * kSWord;
    if (i < TN) s.w[i] = ldsRead4(p + wFromX + i * 32 * kSRow);
    else s.x[i - TN] = ldsRead4(p + (i - TN) * 32 * kSRow);
  };
  auto shiftScales = [&](Scales& s) {  // the lane's blocks to bytes 0 and 2
#pragma unroll
    for (int i = 0; i < TN; ++i) s.w[i] >>= 8 * g;
#pragma unroll
    for (int i = 0; i < TM; ++i) s.x[i] >>= 8 * g;
  };
  f32x16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;

  // ---- the pipeline ----
  auto issueAll = [&](int s, int buffer) {
    prepare(s);
#pragma unroll
    for (int i = 0; i < B::kLoads; ++i) issue(s, buffer, i);
  };
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < stages) issueAll(s, s);
  auto waitStage = [&](int after) {  // `after`: stages issued behind the awaited one
    if (ST > 2 && after >= 2) waitLoads<ST < 3 ? 0 : 2 * B::kLoads>();
    else if (after >= 1) waitLoads<B::kLoads>();
    else waitLoads<0>();
  };
  waitStage(stages - 1 < ST - 1 ? stages - 1 : ST - 1);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  Frags f[2];
  Scales sc[2];
  At here = atBuffer(0);
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(here, Int<0>{}, i, f[0]);
#pragma unroll
  for (int i = 0; i < TN + TM; ++i) readScale(here, 0, i, sc[0]);
  int buffer = 0;
  // Stage s from its buffer; f[0] and sc[0] hold its first step. mode 0: stage s + ST is loaded; 1:
  // another stage follows; 2: the last one. The order of MFMAs, LDS reads and loads is the one
  // written (sched_barrier, and no branch in a stage): left to itself the compiler reads a whole
  // stage, waits, and then multiplies.
  auto stage = [&](int s, auto mode) {
    constexpr bool kLast = decltype(mode)::value == 2, kMore = decltype(mode)::value == 0;
    const int next = buffer + 1 == ST ? 0 : buffer + 1;
    const At there = atBuffer(next);
    auto step = [&](auto j) {
      constexpr int kJ = decltype(j)::value, kWord = kJ / 2;
      constexpr bool kTurn = kJ + 1 == NK;  // the next step is the next stage's first
      Frags& now = f[kJ % 2];
      Frags& then = f[1 - kJ % 2];
      Scales& k = sc[kWord % 2];
      Scales& kThen = sc[1 - kWord % 2];
      if constexpr (kTurn && !kLast) {
        // every wave has read this stage: its buffer takes stage s + ST
        waitLdsReads();
        waitLoads<kMore ? (ST - 2) * B::kLoads : 0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if constexpr (kLast) {
        // blocks past K: their weights are zeros
        if (kJ * 2 + g >= live)
#pragma unroll
          for (int i = 0; i < TN; ++i) now.w[i].q[0] = U32x4{0u, 0u, 0u, 0u};
      }
      if constexpr (kJ % 2 == 0) shiftScales(k);
      constexpr int kMm = TM * TN;
#pragma unroll
      for (int i = 0; i < kMm; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!kTurn || !kLast) {
#pragma unroll
          for (int q = i * kReads / kMm; q < (i + 1) * kReads / kMm; ++q) {
            if constexpr (kTurn) read(there, Int<0>{}, q, then);
            else read(here, Int<(kTurn ? 0 : kJ + 1)>{}, q, then);
          }
          if constexpr (kJ % 2 == 1)
#pragma unroll
            for (int q = i * (TN + TM) / kMm; q < (i + 1) * (TN + TM) / kMm; ++q)
              readScale(kTurn ? there : here, kTurn ? 0 : kWord + 1, q, kThen);
        }
        if constexpr (kTurn && kMore)
#pragma unroll
          for (int q = i * B::kLoads / kMm; q < (i + 1) * B::kLoads / kMm; ++q)
            issue(s + ST, buffer, q);
        __builtin_amdgcn_sched_barrier(0);
        acc[i / TM][i % TM] = mma32<F, kSplit, kJ % 2>(now.w[i / TM], k.w[i / TM], now.x[i % TM],
                                                       k.x[i % TM], acc[i / TM][i % TM]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kTurn && kWord % 2 == 0 && !kLast) sc[0] = sc[1];
    };
    step(Int<0>{});
    step(Int<1>{});
    if constexpr (NK == 4) {
      step(Int<2>{});
      step(Int<3>{});
    }
    buffer = next;
    here = there;
  };
  int s = 0;
  for (; s + ST < stages; ++s) {
    prepare(s + ST);
    stage(s, Int<0>{});
  }
  for (; s + 1 < stages; ++s) stage(s, Int<1>{});
  stage(s, Int<2>{});

  // ---- epilogue: through LDS, so that rows of out are written whole ----
  // Every wave has read the last stage. The wait is written out: the compiler moves MFMAs of the last
  // step behind the barrier and, with them, its own wait for the fragments that they use.
  waitLdsReads();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  float* const slab = reinterpret_cast<float*>(smem) + wave * 32 * kPitch;
  float* const part = parts == nullptr ? nullptr : parts + blockIdx.z * M * N;
  const bool vec = N % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(bias) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(residual) & 15) == 0;
#pragma unroll
  for (int q = 0; q < TM; ++q) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<f32x4*>(&slab[r * kPitch + i * 32 + v * 8 + g * 4]) =
            f32x4{acc[i][q][4 * v], acc[i][q][4 * v + 1], acc[i][q][4 * v + 2],
                  acc[i][q][4 * v + 3]};
    const int64_t mq = m0 + wm * kM + q * 32;
    if (vec) {
      constexpr int kRuns = kN / 8, kRows = kWave / kRuns;  // 8 columns per lane
      const int c = (lane % kRuns) * 8;
      const int64_t n = n0 + wn * kN + c;
      float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (bias != nullptr && part == nullptr && n < nEnd)
        mxLoad8<T, true>(static_cast<const T*>(bias) + n, b);
#pragma unroll 4
      for (int p = 0; p < 32; p += kRows) {
        const int row = p + lane / kRuns;
        const f32x4 lo = *reinterpret_cast<const f32x4*>(&slab[row * kPitch + c]);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(&slab[row * kPitch + c + 4]);
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = lo[e] + b[e];
          v[4 + e] = hi[e] + b[4 + e];
        }
        if (mq + row >= M || n >= nEnd) continue;
        const int64_t at = (mq + row) * N + n;
        if (part != nullptr) {
          mxStore8<float, true>(part + at, v);
          continue;
        }
        if (residual != nullptr) {
          float s[8];
          mxLoad8<T, true>(static_cast<const T*>(residual) + at, s);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += s[e];
        }
        mxStore8<T, true>(static_cast<T*>(out) + at, v);
      }
    } else {
      // a lane takes one column of a run of 64, 8 rows at a time: their loads are in flight together
#pragma unroll
      for (int run = 0; run < kN / 64; ++run) {
        const int c = run * 64 + lane;
        const int64_t n = n0 + wn * kN + c;
        if (n >= nEnd) continue;
        const float b = bias != nullptr && part == nullptr ? ld(static_cast<const T*>(bias) + n) : 0.f;
        const T* const pr = part == nullptr ? static_cast<const T*>(residual) : nullptr;
        for (int p = 0; p < 32; p += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t m = mq + p + e < M ? mq + p + e : M - 1;
            v[e] = pr != nullptr ? ld(pr + m * N + n) : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int64_t m = mq + p + e;
            if (m >= M) break;
            const float sum = slab[(p + e) * kPitch + c] + b + v[e];
            if (part != nullptr) part[m * N + n] = sum;
            else st(static_cast<T*>(out) + m * N + n, sum);
          }
        }
      }
    }
  }
}

// out = the sum of `count` parts [M, N] (+ bias) (+ residual), in order.
template <class T>
__device__ __forceinline__ void mx_sum_parts(const float* parts, int count, const void* bias,
                                             const void* residual, void* out, int64_t M, int64_t N) {
  const int64_t total = M * N, step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const bool vec = N % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(bias) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(residual) & 15) == 0;
  T* const po = static_cast<T*>(out);
  const T *const pb = static_cast<const T*>(bias), *const pr = static_cast<const T*>(residual);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (vec) {
    for (int64_t i = first; i < total / 8; i += step) {
      float v[8], a[8];
      mxLoad8<float, true>(parts + i * 8, v);
      for (int q = 1; q < count; ++q) {
        mxLoad8<float, true>(parts + q * total + i * 8, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += a[e];
      }
      if (bias != nullptr) {
        mxLoad8<T, true>(pb + i * 8 % N, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += a[e];
      }
      if (residual != nullptr) {
        mxLoad8<T, true>(pr + i * 8, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += a[e];
      }
      mxStore8<T, true>(po + i * 8, v);
    }
  } else {
    for (int64_t i = first; i < total; i += step) {
      float v = parts[i];
      for (int q = 1; q < count; ++q) v += parts[q * total + i];
      if (bias != nullptr) v += ld(pb + i % N);
      if (residual != nullptr) v += ld(pr + i);
      st(po + i, v);
    }
  }
}

// The scales of x [M, blocks] and w [N, blocks] as words of 4 blocks, [word][row] with rows padded to
// mPad and nPad (multiples of 256), columns to whole stages of 256: what the tiles read. Blocks and
// rows past the end are 1. A workgroup turns 64 rows x 16 words through LDS; blockIdx.x counts row
// groups, x's first. Bound by a launch's latency: 5 us for 37888 + 8192 rows of 3584 columns.
__device__ __forceinline__ void scaleWords(const uint8_t* xs, const uint8_t* ws, uint32_t* xw,
                                           uint32_t* ww, int64_t M, int64_t N, int blocks,
                                           int64_t mPad, int64_t nPad) {
  __shared__ uint32_t tile[16][65];
  const bool isX = blockIdx.x < mPad / 64;
  const uint8_t* const from = isX ? xs : ws;
  uint32_t* const to = isX ? xw : ww;
  const int64_t rows = isX ? M : N, pad = isX ? mPad : nPad;
  const int64_t row0 = (isX ? blockIdx.x : blockIdx.x - mPad / 64) * 64;
  const int there = (blocks + 3) / 4, word0 = blockIdx.y * 16;
  const int words = (blocks + 7) / 8 * 2;  // whole stages of 256 columns
  const bool whole = blocks % 4 == 0 && (reinterpret_cast<uintptr_t>(from) & 3) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 16 + threadIdx.x / 16, word = threadIdx.x % 16;
    uint32_t v = 0x7F7F7F7Fu;
    if (row0 + row < rows && word0 + word < there) {
      const uint8_t* p = from + (row0 + row) * blocks + (word0 + word) * 4;
      if (whole) {
        v = *gp(reinterpret_cast<const uint32_t*>(p));
      } else {
        const int n = blocks - (word0 + word) * 4;
        v = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          v |= (b < n ? static_cast<uint32_t>(gp(p)[b]) : 0x7Fu) << (8 * b);
      }
    }
    tile[word][row] = v;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int word = i * 4 + threadIdx.x / 64, row = threadIdx.x % 64;
    if (word0 + word < words) to[(word0 + word) * pad + row0 + row] = tile[word][row];
  }
}

}  // namespace

#define MX_LINEAR_ARGS                                                                           \
  (const uint8_t* x, const uint8_t* xs, const uint8_t* w, const uint8_t* ws, const void* bias,   \
   const void* residual, void* out, int64_t M, int64_t N, int64_t K)
#define MX_STREAM(name, F, T, ROWS, KW, DEPTH)                                                   \
  extern "C" __global__ void __launch_bounds__(64 * (KW > 4 ? KW : 4)) name MX_LINEAR_ARGS {    \
    mx_linear_stream<F, T, ROWS, KW, DEPTH, true>(x, xs, w, ws, bias, residual, out, M, N, K);  \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(64 * (KW > 4 ? KW : 4))                          \
      name##_odd MX_LINEAR_ARGS {                                                               \
    mx_linear_stream<F, T, ROWS, KW, DEPTH, false>(x, xs, w, ws, bias, residual, out, M, N, K); \
  }
#define MX_STREAM_FORMS(ROWS, KW, DEPTH)                                            \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp8_f32, MxFp8, float, ROWS, KW, DEPTH)     \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp8_bf16, MxFp8, bf16, ROWS, KW, DEPTH)     \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp8_f16, MxFp8, f16, ROWS, KW, DEPTH)       \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp4_f32, MxFp4, float, ROWS, KW, DEPTH)     \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp4_bf16, MxFp4, bf16, ROWS, KW, DEPTH)     \
  MX_STREAM(mx_stream_r##ROWS##_k##KW##_fp4_f16, MxFp4, f16, ROWS, KW, DEPTH)
#define MX_STREAM_ROWS(ROWS, DEPTH) \
  MX_STREAM_FORMS(ROWS, 1, DEPTH)   \
  MX_STREAM_FORMS(ROWS, 2, DEPTH)   \
  MX_STREAM_FORMS(ROWS, 4, DEPTH)   \
  MX_STREAM_FORMS(ROWS, 8, DEPTH)
MX_STREAM_ROWS(1, 4)
MX_STREAM_ROWS(4, 4)
MX_STREAM_ROWS(16, 2)

#define MX_BIG(name, F, T, BM, BN, WM, WN, KS, ST, PER, RS)                                          \
  extern "C" __global__ void __launch_bounds__(64 * WM * WN)                                     \
      __attribute__((amdgpu_waves_per_eu(PER, PER)))                                             \
      name(const uint8_t* x, const uint32_t* xw, const uint8_t* w, const uint32_t* ww,           \
           const void* bias, const void* residual, void* out, float* parts, int64_t M,           \
           int64_t N, int64_t K, int64_t mPad, int64_t nPad, int width) {                        \
    mx_linear_big<F, T, BM, BN, WM, WN, KS, ST, RS>(x, xw, w, ww, bias, residual, out, parts, M, \
                                                    N, K, mPad, nPad, width);                    \
  }
#define MX_BIG_FORMS(name, F, BM, BN, WM, WN, KS, ST, PER, RS)         \
  MX_BIG(name##_f32, F, float, BM, BN, WM, WN, KS, ST, PER, RS)        \
  MX_BIG(name##_bf16, F, bf16, BM, BN, WM, WN, KS, ST, PER, RS)        \
  MX_BIG(name##_f16, F, f16, BM, BN, WM, WN, KS, ST, PER, RS)
// 256 x 256. e2m1 rows: 4 waves, stages of 256 columns (two fill LDS). e4m3 rows: 8 waves of 64 x 128,
// whose MFMAs leave time for their fragments twice over, stages of 128 columns (8192 rows x 8192 x
// 8192: 441 us, 488 with 4 waves; e2m1 on 8 waves ran out of registers).
MX_BIG_FORMS(mx_tile_256_fp8, MxFp8, 256, 256, 4, 2, 128, 3, 2, false)
MX_BIG_FORMS(mx_tile_256_fp4, MxFp4, 256, 256, 2, 2, 256, 2, 1, false)
// smaller tiles, two workgroups to a CU
MX_BIG_FORMS(mx_tile_128_fp8, MxFp8, 128, 128, 2, 2, 128, 3, 2, false)
MX_BIG_FORMS(mx_tile_128_fp4, MxFp4, 128, 128, 2, 2, 256, 2, 2, false)
MX_BIG_FORMS(mx_tile_64_fp8, MxFp8, 64, 128, 2, 2, 256, 2, 2, false)
MX_BIG_FORMS(mx_tile_64_fp4, MxFp4, 64, 128, 2, 2, 256, 3, 2, false)
MX_BIG_FORMS(mx_tile_128r_fp8, MxFp8, 128, 128, 2, 2, 128, 3, 2, true)
MX_BIG_FORMS(mx_tile_128r_fp4, MxFp4, 128, 128, 2, 2, 256, 2, 2, true)
MX_BIG_FORMS(mx_tile_64r_fp8, MxFp8, 64, 128, 2, 2, 256, 2, 2, true)
MX_BIG_FORMS(mx_tile_64r_fp4, MxFp4, 64, 128, 2, 2, 256, 3, 2, true)
// One workgroup to a CU, of as many columns as the launch says: three stages of 48 KB. 64 x 37888 x 3584
// from memory: 24.0 us, 3.2 TB/s (e2m1 rows 23.4). The cache hands a CU about a line per 2 cycles, and
// of the 704 of a stage 320 are for 8 bytes of scales each (3 us in all).
MX_BIG_FORMS(mx_tile_64w_fp8, MxFp8, 64, 256, 2, 4, 256, 3, 2, true)
MX_BIG_FORMS(mx_tile_64w_fp4, MxFp4, 64, 256, 2, 4, 256, 3, 2, true)

#define MX_SUM_PARTS(name, T)                                                                 \
  extern "C" __global__ void __launch_bounds__(256)                                           \
      name(const float* parts, int count, const void* bias, const void* residual, void* out,  \
           int64_t M, int64_t N) {                                                            \
    mx_sum_parts<T>(parts, count, bias, residual, out, M, N);                                 \
  }
MX_SUM_PARTS(mx_sum_parts_f32, float)
MX_SUM_PARTS(mx_sum_parts_bf16, bf16)
MX_SUM_PARTS(mx_sum_parts_f16, f16)

extern "C" __global__ void __launch_bounds__(256)
    mx_scale_words(const uint8_t* xs, const uint8_t* ws, uint32_t* xw, uint32_t* ww, int64_t M,
                   int64_t N, int blocks, int64_t mPad, int64_t nPad) {
  scaleWords(xs, ws, xw, ww, M, N, blocks, mPad, nPad);
}
