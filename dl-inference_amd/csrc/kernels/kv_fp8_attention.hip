// Attention over the 8-bit paged KV cache on gfx950 (formats in kv_fp8.h): softmax(q k^T * scale
// [+ causal mask]) v with k and v = element * scale of the token, in T = bf16, f16 or fp32.
//
// The elements (4 bits of significand) are exact in bf16 and f16, so both products run on the 16-bit
// MFMA with fp32 sums and lose nothing to the cache's format:
//   S^T = K Q^T    elements as bf16 (T bf16 and fp32, whose q is the exact sum of three bf16 terms)
//                  or f16 (T f16); the token's key scale multiplies the score in fp32.
//   O^T += V^T P^T elements as f16, P as f16: one term (11 bits) where the output is bf16 (8 bits),
//                  two terms (22 bits) else. The largest is 2^11 to 2^15.5, so that f16's normal range reaches
//                  down to 2^-25 of it. The token's value scale goes into P (few rows, RowSum), or into V
//                  relative to the largest seen (many, if their values are not too far apart: kNear).
// A token whose row was not finite (scale 255) makes the score NaN, so rows that
// see it are NaN and rows that do not see it are untouched.
#include "kv_fp8.h"
#include "skinny.h"

using namespace dk;

namespace {

constexpr int kTileK = 64;
// log2 of a probability at the running reference, and what the reference lags behind at most: a lag of
// 2 (and 2^13 at the reference) moves it more often, 53.8 us for 4 x 2048 prompt tokens (52.2)
constexpr float kLift = 11.f, kSlack = 4.5f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// T's part in the products: the type that K's elements and q's terms take, q's and P's terms
template <class T>
struct Kv8Type;
template <>
struct Kv8Type<bf16> {
  static constexpr int kQ = 1, kP = 1;
};
template <>
struct Kv8Type<f16> {
  static constexpr int kQ = 1, kP = 2;
};
template <>
struct Kv8Type<float> {
  static constexpr int kQ = 3, kP = 2;
};

// 8 codes -> the 16-bit values that they stand for, exactly
__device__ __forceinline__ U128 codesToF16(uint32_t w0, uint32_t w1) {
  return U128{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, true))};
}
__device__ __forceinline__ U128 codesToBf16(uint32_t w0, uint32_t w1) {
  return U128{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, true))};
}

template <class T>
__device__ __forceinline__ U128 keyFragment(uint32_t w0, uint32_t w1) {
  if constexpr (__is_same(T, f16))
    return codesToF16(w0, w1);
  else
    return codesToBf16(w0, w1);
}

template <class T>
__device__ __forceinline__ f32x4 keyMma(const U128& a, const U128& b, const f32x4& c) {
  if constexpr (__is_same(T, f16))
    return F16::mma(a, b, c);
  else
    return Bf16::mma(a, b, c);
}

// 8 elements of q as terms: q itself, or three bf16 numbers (8 bits each, cut off) that add up to it;
// an infinity and two zeros, NaN and two zeros
template <class T>
__device__ __forceinline__ void queryFragment(const T* q, U128 (&f)[Kv8Type<T>::kQ]) {
  if constexpr (sizeof(T) == 2) {
    f[0] = gload16(q);
  } else {
    const U128 lo = gload16(q), hi = gload16(q + 4);
    uint32_t x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
    for (int i = 0; i < 8; ++i)  // a NaN stays one without its low bits
      if (__builtin_isnan(__uint_as_float(x[i]))) x[i] = 0x7FC00000u;
#pragma unroll
    for (int u = 0; u < 3; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[u][j] = (x[2 * j] >> 16) | (x[2 * j + 1] & 0xFFFF0000u);
#pragma unroll
        for (int i = 2 * j; i < 2 * j + 2; ++i)
          x[i] = u == 0 && !__builtin_isfinite(__uint_as_float(x[i]))
                     ? 0u
                     : __float_as_uint(__uint_as_float(x[i]) - __uint_as_float(x[i] & 0xFFFF0000u));
      }
  }
}

// Queries of 2^100 and more are taken 2^-32 times as large where scores are summed before the key's scale is
// applied: a sum of 256 products with elements of up to 448 stays finite. Elements that this loses are below
// 2^-194 of their row's largest.
constexpr float kLargeQuery = 0x1p100f, kQueryDown = 0x1p-32f, kQueryUp = 0x1p32f;

// Bits 0..14 of the largest magnitude among the halves of w, which are 16-bit floats, or of `most`.
typedef uint16_t U16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ U16x2 largestHalf(U16x2 most, uint32_t w) {
  return __builtin_elementwise_max(most, __builtin_bit_cast(U16x2, w & 0x7FFF7FFFu));
}

// Two bf16 times a power of two, cut to bf16 again.
__device__ __forceinline__ uint32_t timesBf16(uint32_t w, float f) {
  return (__float_as_uint(__uint_as_float(w << 16) * f) >> 16) |
         (__float_as_uint(__uint_as_float(w & 0xFFFF0000u) * f) & 0xFFFF0000u);
}

// The value of lane 16 g + n in the lanes 16 g .. 16 g + 15; n is a constant once loops are unrolled,
// and the move becomes an operand of the multiplication it feeds.
template <int n>
__device__ __forceinline__ float rowLane(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x150 + n, 0xF, 0xF, true));
}

// s[kk][i] *= the factor of key 16 g + 4 kk + i of the lane's row of lanes
template <int n = 0>
__device__ __forceinline__ void timesKeys(f32x4 (&s)[4], float factor) {
  if constexpr (n < 16) {
    s[n / 4][n % 4] *= rowLane<n>(factor);
    timesKeys<n + 1>(s, factor);
  }
}

// The score factor and value scale of the lane's key. nan: neither finite
struct KeyScales {
  float k;      // 2^(key scale) * the given scale; NaN where a scale is 255
  uint32_t v;   // value scale code, 0 where a scale is 255 or the key is not live
};
__device__ __forceinline__ KeyScales keyScales(uint32_t kc, uint32_t vc, bool live,
                                               float scale) {
  const bool bad = kc == 255u || vc == 255u;
  return {mxScaleValue(bad ? 255u : kc) * scale, bad || !live ? 0u : vc};
}

// 2^(code - top) for code <= top
__device__ __forceinline__ float valueFactor(uint32_t code, uint32_t top) {
  const int e = 127 + static_cast<int>(code) - static_cast<int>(top);
  return e > 0 ? __uint_as_float(static_cast<uint32_t>(e) << 23) : 0.f;
}

// The largest of the wave's values in each half of a word: over 16 lanes by rotation, then over their rows.
typedef uint16_t U16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t waveMaxHalves(uint32_t v) {
  auto larger = [](uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(U16x2, x),
                                                                  __builtin_bit_cast(U16x2, y)));
  };
  v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, true));
  v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, true));
  v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, true));
  v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, true));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = larger(a[0], a[1]);
  const auto c = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(larger(c[0], c[1]));
}

// t for a second run over the same work: what the first computed from it is not kept in registers.
__device__ __forceinline__ int againOf(int t) {
  asm volatile("" : "+v"(t));
  return t;
}

// In a branch that is seldom taken: keeps the compiler from computing both sides and selecting.
__device__ __forceinline__ void rarely() { asm volatile(""); }

// Bytes i < 16 of w whose bit i is clear become 0.
__device__ __forceinline__ void keepBytes(U128& w, uint32_t bits) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = bits >> (4 * j);
    w[j] &= ((b & 1u) ? 0xFFu : 0u) | ((b & 2u) ? 0xFF00u : 0u) | ((b & 4u) ? 0xFF0000u : 0u) |
            ((b & 8u) ? 0xFF000000u : 0u);
  }
}

// Probabilities of 16 keys -> two B fragments of f16 (keys 0..7 and 8..15), kP terms
template <int kP>
__device__ __forceinline__ void packWeights(const f32x4 (&w)[4], U128 (&f)[kP][2]) {
#pragma unroll
  for (int st = 0; st < 2; ++st)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = w[2 * st + j / 2][2 * (j % 2)], b = w[2 * st + j / 2][2 * (j % 2) + 1];
      const f16x2 hi = {static_cast<f16>(a), static_cast<f16>(b)};
      f[0][st][j] = __builtin_bit_cast(uint32_t, hi);
      if constexpr (kP == 2) {
        const f16x2 lo = {static_cast<f16>(a - static_cast<float>(hi[0])),
                          static_cast<f16>(b - static_cast<float>(hi[1]))};
        f[1][st][j] = __builtin_bit_cast(uint32_t, lo);
      }
    }
}

// A row's softmax and the unit that its output is summed in, as powers of two. Value scales may lie 2^247
// apart, f16 holds 2^40: weights for the products are taken relative to the largest weight times value scale
// that the row has seen, so neither a token that it does not see nor one that weighs nothing costs the others
// a bit.
struct RowSum {
  float m = -INFINITY;     // reference of the scores
  float l = 0.f;           // this lane's part of the sum of 2^(score - m)
  float unit = 0.f;        // a whole number: the output is sum * 2^(unit - 127)
  float peak = -INFINITY;  // the largest log2 of a weight in o, at m and unit
};

// u[n] = s[n] + the scale code of key n - unit
template <int n = 0>
__device__ __forceinline__ void inUnit(const f32x4 (&s)[4], float code, float unit, f32x4 (&u)[4]) {
  if constexpr (n < 16) {
    u[n / 4][n % 4] = s[n / 4][n % 4] + (rowLane<n>(code) - unit);
    inUnit<n + 1>(s, code, unit, u);
  }
}

__device__ __forceinline__ float largestOf(const f32x4 (&s)[4]) {
  float most = -INFINITY;
#pragma unroll
  for (int n = 0; n < 16; ++n) most = fmaxf(most, s[n / 4][n % 4]);
  return most;
}

// Scores of 16 keys (-infinity where masked) -> their weights 2^(score - m + code - unit), between 2^kLift and
// 2^(kLift + kSlack) at the peak; code: the value scale code of this lane's key. o follows m and unit.
template <int DT>
__device__ __forceinline__ void weigh(f32x4 (&s)[4], float code, RowSum& row, f32x4 (&o)[DT]) {
  FP_EXACT;  // a large score less its reference, in one step with the score's own product, would not be 0
  const float top = rowsMax(largestOf(s));
  const bool grow = top > row.m + kSlack;  // false while top is -inf
  bool changed = __builtin_amdgcn_ballot_w64(grow) != 0;
  float shift = 0.f;
  if (changed) {
    shift = grow ? row.m - top : 0.f;
    row.m = grow ? top : row.m;
    row.l *= __builtin_amdgcn_exp2f(shift);  // 0 from -inf
    row.peak += shift;
  }
  // the reference alone first: from 2^24 on its sum with anything is rounded
  const float base = row.m == -INFINITY ? 0.f : row.m;
#pragma unroll
  for (int n = 0; n < 16; ++n) s[n / 4][n % 4] -= base;
  f32x4 u[4];
  inUnit(s, code, row.unit, u);
  row.peak = fmaxf(row.peak, rowsMax(largestOf(u)));
  // it falls only where the reference moves
  const bool low = grow && row.peak < kLift && row.peak != -INFINITY;
  const bool move = row.peak > kLift + kSlack || low;
  if (__builtin_amdgcn_ballot_w64(move)) {
    const float by = move ? floorf(row.peak - kLift) : 0.f;
    row.unit += by;
    row.peak -= by;
    shift -= by;
    changed = true;
    inUnit(s, code, row.unit, u);
  }
  if (changed) {
    const float alpha = __builtin_amdgcn_exp2f(shift);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
  }
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    sum += __builtin_amdgcn_exp2f(s[n / 4][n % 4]);
    s[n / 4][n % 4] = __builtin_amdgcn_exp2f(u[n / 4][n % 4]);
  }
  row.l += sum;
}

// keys that row i of the queries sees, in [0, capacity]
__device__ __forceinline__ int visibleKeys(const Kv8AttentionArgs& a, int64_t past, int i) {
  const int64_t n = past + (a.causal ? i + 1 : a.seq_q);
  return static_cast<int>(n < 0 ? 0 : (n > a.capacity ? a.capacity : n));
}

// Row p of a (sequence, KV head) pair: query p / group of head p % group.
struct RowAt {
  int i, h;
};
__device__ __forceinline__ RowAt rowAt(int p, int group, int kvh) {
  const int i = p / group;
  return {i, kvh * group + p - i * group};
}

// element 0 of a row in q, [batch, q_heads, seq_q, D], and in out
__device__ __forceinline__ int64_t queryAt(const Kv8AttentionArgs& a, int64_t b, RowAt r, int D) {
  return ((b * a.q_heads + r.h) * a.seq_q + r.i) * D;
}
__device__ __forceinline__ int64_t outAt(const Kv8AttentionArgs& a, int64_t b, RowAt r, int D) {
  return a.out_bshd ? ((b * a.seq_q + r.i) * a.q_heads + r.h) * D : queryAt(a, b, r, D);
}

// ---------------------------------------------------------------------------------------------
// Few rows (at most 16 of a (sequence, KV head) pair: the group's heads of one new token, or of a
// few): each key is used once, so the keys stream from memory into registers. A workgroup of
// kDecWaves waves takes split blockIdx.x of pair blockIdx.y; its waves take 64-key tiles in turn, the
// next one's loads in flight while one is computed, and join their results in LDS. A lane (r, g) of a
// wave loads 16-byte runs: of K the row of key 16 (r / 4) + 4 kk + r % 4 at the dims 16 g + 64 j, of
// V the dims 16 dt + r at the keys 16 g. The order in which the MFMA takes dims and keys is free as
// long as both operands share it, so those runs are its fragments as they come, and the scores come
// out as 16 consecutive keys a lane: V's order.
//
// Long calls are bound by the stream of the cache: 64 sequences of 8192 tokens (28 / 4 heads x 128) 83 us,
// 511 MB at 6.2 TB/s (part of it from the 256 MB cache). Short ones by latency: 32 of 4096 (14 / 2 x 64)
// 13.0 us, 32 MB, of which two launches take 7.4; one of 1000 tokens 7.6, three trips to memory (table and
// position, the tile, the store) and a join of 8 waves.
// ---------------------------------------------------------------------------------------------
constexpr int kDecWaves = 8;

// Loads of lines that are read once. They pay where an instruction covers whole 128-byte lines: V's
// rows of 64 keys stand one behind the other, and so do 4 rows of K with head_dim 64; with 128 an
// instruction takes half of each line of K. 64 sequences of 8192 tokens (28 / 4 heads x 128): 91.6 us with
// cached loads, 83.4 with V streamed, 84.2 with K too; 32 of 4096 (14 / 2 x 64) 14.0, 14.0 and 13.1.
__device__ __forceinline__ U128 streamed16(const uint8_t* p) {
  return __builtin_nontemporal_load(gp(reinterpret_cast<const U128*>(p)));
}
template <int D>
__device__ __forceinline__ U128 keyLoad(const uint8_t* p) {
  return D == 64 ? streamed16(p) : gload16(p);
}

// A tile's codes and this lane's key's scales; ids of its pages, -1 where a page holds nothing
template <int D>
struct KeyTile {
  U128 k[4][D / 64];
  U128 v[D / 16];
  uint32_t kc, vc;
  bool live;  // the lane's key is in a page
};

template <class T, int D>
struct DecodeLds {
  // q's terms where there are several: in registers they would push the tiles out (fp32, head_dim 128,
  // 64 sequences of 4096 tokens: 80.7 us with 43 registers spilled, 50 so). The same of what a row has
  // beside them: the wait for a register that comes back from memory is one for the tile on its way (10 of
  // them: 57).
  U128 q[Kv8Type<T>::kQ > 1 ? D / 64 * 2 * Kv8Type<T>::kQ : 1][kWave];
  float row_scale[kWave];
  int lim[kWave];
  float m[kDecWaves][16];
  float l[kDecWaves][16];
  float unit[kDecWaves][16];
  float o[kDecWaves][D][17];
};

// kSmall: pages of 16 or 32 tokens (else a multiple of 64)
template <class T, int D, bool kSmall>
__device__ __forceinline__ void kv8_decode(const Kv8AttentionArgs& a) {
  using Ty = Kv8Type<T>;
  constexpr int J = D / 64, DT = D / 16;
  __shared__ DecodeLds<T, D> lds;
  const Kv8Pages& pg = a.pages;
  const int t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int r = lane % 16, g = lane / 16;
  const int pair = blockIdx.y, b = pair / pg.heads, kvh = pair - b * pg.heads;
  const int group = a.q_heads / pg.heads, rows = group * a.seq_q;
  const int bs = pg.block_size;
  const int stride = a.splits * kDecWaves, first = blockIdx.x * kDecWaves + wave;
  const int32_t* table = pg.table + static_cast<int64_t>(b) * pg.max_blocks;
  // Page ids, a lane each: of kIds tiles of this wave (kSmall: 4 runs of 16 keys a tile).
  constexpr int kIds = kSmall ? 16 : 64;
  int ids = -1;
  auto loadIds = [&](int ordinal) {  // of the tiles ordinal .. ordinal + kIds - 1
    const int64_t tile = first + static_cast<int64_t>(ordinal + (kSmall ? lane / 4 : lane)) * stride;
    const int64_t key = tile * kTileK + (kSmall ? 16 * (lane % 4) : 0);
    ids = -1;
    // whatever the sequence holds: the ids are on their way while its position is
    if (key < a.capacity) ids = gp(table)[static_cast<uint32_t>(key) / static_cast<uint32_t>(bs)];
    if (ids >= pg.num_blocks) ids = -1;
  };
  loadIds(0);
  const int64_t past = kv8First(pg, b);
  const int most = visibleKeys(a, past, a.seq_q - 1);
  const int tiles = (most + kTileK - 1) / kTileK;
  KeyTile<D> buf[2];
  auto fetch = [&](KeyTile<D>& x, int tile, int ordinal) {
    const int64_t head = static_cast<int64_t>(bs) * D;
    int id_k, id_v, slot_k, slot_v;
    if constexpr (kSmall) {
      const int at = (ordinal % kIds) * 4;
      id_k = __shfl(ids, at + r / 4, kWave);
      id_v = __shfl(ids, at + g, kWave);
      slot_k = 16 * (r / 4) % bs;
      slot_v = 16 * g % bs;
    } else {
      id_k = id_v = __builtin_amdgcn_readlane(ids, ordinal % kIds);
      const int in_page = static_cast<int>(static_cast<uint32_t>(tile) * kTileK % static_cast<uint32_t>(bs));
      slot_k = in_page + 16 * (r / 4);
      slot_v = in_page + 16 * g;
    }
    x.live = id_v >= 0;
    // a page that holds nothing: page 0 is read in its place and masked
    const int64_t hk = static_cast<int64_t>(id_k < 0 ? 0 : id_k) * pg.heads + kvh;
    const int64_t hv = static_cast<int64_t>(id_v < 0 ? 0 : id_v) * pg.heads + kvh;
    const uint8_t* kb = pg.key + hk * head + static_cast<int64_t>(slot_k + r % 4) * D + 16 * g;
    const uint8_t* vb = pg.value + hv * head + static_cast<int64_t>(r) * bs + slot_v;
    const uint8_t* sb = pg.scales + hv * 2 * bs + slot_v + r;
    x.kc = gp(sb)[0];
    x.vc = gp(sb)[bs];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int j = 0; j < J; ++j) x.k[kk][j] = keyLoad<D>(kb + 4 * kk * D + 64 * j);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) x.v[dt] = streamed16(vb + static_cast<int64_t>(16 * dt) * bs);
  };

  // q: rows past the last are zero and not stored
  constexpr bool kSharedQ = Ty::kQ > 1;
  U128 qf[J][2][Ty::kQ];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int u = 0; u < Ty::kQ; ++u) qf[j][half][u] = zero16();
  int lim = most;  // keys of this lane's row
  if (r < rows) {
    const RowAt at = rowAt(r, group, kvh);
    lim = visibleKeys(a, past, at.i);
    const T* q = static_cast<const T*>(a.q) + queryAt(a, b, at, D) + 16 * g;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) queryFragment<T>(q + 64 * j + 8 * half, qf[j][half]);
  }
  // What brings the row's sums back to their size, times the softmax scale: a key's scale alone may then be as
  // small as it gets. f16 has no queries that large.
  float row_scale = a.scale_log2;
  if constexpr (!__is_same(T, f16)) {
    U16x2 largest = {0, 0};
#pragma unroll
    for (int x = 0; x < J * 8; ++x) largest = largestHalf(largest, qf[x / 8][x / 4 % 2][0][x % 4]);
    const float of_lane = __uint_as_float(
        static_cast<uint32_t>(largest[0] > largest[1] ? largest[0] : largest[1]) << 16);
    // one lane of the row is enough; a NaN counts for nothing, its row is NaN in any case
    const bool up = rowsMax(of_lane) >= kLargeQuery;
    if (__builtin_amdgcn_ballot_w64(up)) {
      rarely();
      row_scale *= up ? kQueryUp : 1.f;
      const float down = up ? kQueryDown : 1.f;
#pragma unroll
      for (int x = 0; x < J * 8; ++x)
#pragma unroll
        for (int u = 0; u < Ty::kQ; ++u)
          qf[x / 8][x / 4 % 2][u][x % 4] = timesBf16(qf[x / 8][x / 4 % 2][u][x % 4], down);
    }
  }
  if constexpr (kSharedQ) {
    if (wave == 0) {
      lds.row_scale[lane] = row_scale;
      lds.lim[lane] = lim;
#pragma unroll
      for (int x = 0; x < J * 2 * Ty::kQ; ++x)
        lds.q[x][lane] = qf[x / (2 * Ty::kQ)][x / Ty::kQ % 2][x % Ty::kQ];
    }
    __syncthreads();
  }
  auto query = [&](int at, int j, int half, int u) {
    return kSharedQ ? lds.q[(j * 2 + half) * Ty::kQ + u][at] : qf[j][half][u];
  };
  const int all_see = visibleKeys(a, past, 0);  // keys that every row sees

  RowSum row;
  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto attend = [&](KeyTile<D>& x, int tile) {
    const int k0 = tile * kTileK;
    int q_lane = lane;
    if constexpr (kSharedQ) asm volatile("" : "+v"(q_lane));  // read per tile, not held in registers
    f32x4 s[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      s[kk] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const U128 ka = keyFragment<T>(x.k[kk][j][2 * half], x.k[kk][j][2 * half + 1]);
#pragma unroll
          for (int u = Ty::kQ - 1; u >= 0; --u) s[kk] = keyMma<T>(ka, query(q_lane, j, half, u), s[kk]);
        }
    }
    const bool live = x.live && k0 + lane < most;
    const uint64_t lives = __builtin_amdgcn_ballot_w64(live);
    constexpr bool kRowScale = !__is_same(T, f16);
    const KeyScales sc = keyScales(x.kc, x.vc, live, kRowScale ? 1.f : a.scale_log2);
    timesKeys(s, sc.k);
    if constexpr (kRowScale) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) s[kk] *= kSharedQ ? lds.row_scale[q_lane] : row_scale;
    }
    if (lives != ~uint64_t{0} || k0 + kTileK > all_see) {  // uniform
      const uint32_t mine = static_cast<uint32_t>(lives >> (16 * g)) & 0xFFFFu;
      const int key0 = k0 + 16 * g, end = kSharedQ ? lds.lim[q_lane] : lim;
#pragma unroll
      for (int n = 0; n < 16; ++n)
        if (!(mine >> n & 1u) || key0 + n >= end) s[n / 4][n % 4] = -INFINITY;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) keepBytes(x.v[dt], mine);
    }
    weigh(s, static_cast<float>(sc.v), row, o);
    U128 pf[Ty::kP][2];
    packWeights<Ty::kP>(s, pf);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const U128 va = codesToF16(x.v[dt][2 * st], x.v[dt][2 * st + 1]);
#pragma unroll
        for (int u = Ty::kP - 1; u >= 0; --u) o[dt] = F16::mma(va, pf[u][st], o[dt]);
      }
  };

  if (first < tiles) fetch(buf[0], first, 0);
  for (int tile = first, n = 0; tile < tiles; tile += 2 * stride, n += 2) {
    const int second = tile + stride, third = second + stride;
    if (second < tiles) fetch(buf[1], second, n + 1);
    attend(buf[0], tile);
    if (second >= tiles) break;
    if (third < tiles) {
      if ((n + 2) % kIds == 0) loadIds(n + 2);
      fetch(buf[0], third, n + 2);
    }
    attend(buf[1], second);
  }

  // join the waves at the row's largest reference, and the largest unit at it
  const float l_row = rowsSum(row.l);
  if (g == 0) {
    lds.m[wave][r] = row.m;
    lds.l[wave][r] = l_row;
    lds.unit[wave][r] = row.unit;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) lds.o[wave][16 * dt + 4 * g + i][r] = o[dt][i];
  __syncthreads();
  for (int e = t; e < rows * D; e += kDecWaves * kWave) {
    const int p = e / D, d = e % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) M = fmaxf(M, lds.m[w][p]);
    float L = 0.f, unit = -INFINITY, past_m[kDecWaves];
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
      const float m = lds.m[w][p], l = lds.l[w][p];
      // a wave that saw no key has no part; a NaN sum stays one whatever its reference
      past_m[w] = m == -INFINITY ? (l == 0.f ? -INFINITY : 0.f) : m - M;
      L += __builtin_amdgcn_exp2f(past_m[w]) * l;
      unit = fmaxf(unit, lds.unit[w][p] + rintf(past_m[w]));
    }
    float acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w)
      acc += __builtin_amdgcn_exp2f(past_m[w] + (lds.unit[w][p] - unit)) * lds.o[w][d][p];
    const RowAt at = rowAt(p, group, kvh);
    // the quotient first, so that neither overflows
    const float result = L == 0.f ? 0.f : __builtin_ldexpf(acc / L, static_cast<int>(unit) - 127);
    if (a.splits == 1) {
      st(static_cast<T*>(a.out) + outAt(a, b, at, D) + d, result);
    } else {
      const int64_t part = (queryAt(a, b, at, 1) * a.splits + blockIdx.x);
      if (d == 0) {
        a.part_ml[part * 2] = M;
        a.part_ml[part * 2 + 1] = L;
      }
      a.part_o[part * D + d] = result;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Many rows (a chunk of new tokens, a prompt): the group's heads and the queries are one row index,
// so a staged tile serves every head of the group. A workgroup of 4 waves owns 64 QB rows of a pair
// (16 QB a wave) and a range of 64-key tiles; grid.z splits the keys where rows alone leave CUs idle.
// A tile's codes are converted once, on their way into LDS: K [key][dim], keys in the order in which
// the scores come out as 16 consecutive keys a lane, and V^T [dim][key] as it lies in the page, its 16-byte
// chunks permuted by dim so that the 16 rows of a fragment read fall on distinct banks. One barrier a
// tile: two buffers, and two workgroups on a CU that need not keep step.
//
// 2048 tokens over 8192 (28 / 4 heads x 128, bf16) take 339 us, 270 GFLOP at 798 TFLOP/s (291 phased, below).
// No unit is full: MFMA 33% busy, vector instructions 43%, LDS 33% (a quarter of it conflicts); a wave waits
// for its own chain (scores, weights, products) and for the tile, and two waves a SIMD hide half of
// that. Left out one at a time, staging saves 100 us, the softmax 60, the loads 42. Tried, in us: 64 rows a
// wave at one wave a SIMD 635; 256 rows and 8 waves a workgroup in step 354; the next tile's scores between
// this one's softmax 331 to 350, and slower with head_dim 64; wave priorities 342 to 361; scales read by
// their users, without LDS, 343.
// ---------------------------------------------------------------------------------------------
constexpr int kChunkWaves = 4;
constexpr int kAhead = 3;  // LDS fragments read before they are needed
// exponent of a staged value's factor at the largest value scale: elements reach 448 * 2^7 there, and a
// token's elements stay exact in f16 down to 2^-22 of that scale
constexpr int kValueLift = 7;
// a row's shift before its first key: any finite score added to it passes the slack, and -infinity
// stays what it is
constexpr float kNoReference = 0x1.fffffep127f;

// A weight's exponent is score * scale + shift in one fma. From 2^23 on the shift's own rounding would show
// in it (and past 2^27 pass what f16 holds): rows whose reference lies there subtract the score at the
// reference first. Their scores are rounded to whole units and more, so only the largest matters.
constexpr float kFarShift = 8388608.f;
__device__ __forceinline__ bool farRow(float shift) {
  return fabsf(shift) >= kFarShift && shift != kNoReference;
}
__device__ __forceinline__ float farExponent(float score, float ref, float shift, float scale) {
  return farRow(shift) ? fmaf(score - ref, scale, kLift) : fmaf(score, scale, shift);
}
// Scores of a far row become those past its reference; what brings score * scale to its exponent.
__device__ __forceinline__ float fromReference(f32x4 (&s)[4], float ref, float shift) {
  const bool away = farRow(shift);
#pragma unroll
  for (int n = 0; n < 16; ++n) s[n / 4][n % 4] -= away ? ref : 0.f;
  return away ? kLift : shift;
}
// Moves a row's reference to its largest score `most` if its weight would pass 2^(kLift + kSlack); the factor
// of what was summed so far.
__device__ __forceinline__ float moveReference(float most, float scale, float& ref, float& shift) {
  const float top = rowsMax(most);  // the same in a row's four lanes
  if (!(farExponent(top, ref, shift, scale) > kLift + kSlack)) return 1.f;
  const float next = kLift - top * scale;
  const float alpha =
      __builtin_amdgcn_exp2f(farRow(shift) ? (ref - top) * scale : next - shift);  // 0 at first
  ref = top;
  shift = next;
  return alpha;
}

// Places of 16-byte chunks (8 elements) in LDS. A ds_read_b128 serves 16 lanes a cycle: lanes 0-3,
// 12-15 and 20-27 together, then 4-11, 16-19 and 28-31, and the upper half alike (found by timing pairs
// of lanes on one bank). With r the row of a fragment read and g or g + 4 st the chunk, chunk ^ r over rows
// of 16 chunks and chunk ^ r / 2 over rows of 8 put those lanes on distinct banks.
template <int D>
__device__ __forceinline__ int keyChunk(int row, int chunk) {
  return row * D + (chunk ^ (D == 128 ? row & 15 : (row >> 1) & 7)) * 8;
}
// keys 8 half .. 8 half + 7 of the run of 16
__device__ __forceinline__ int valueChunk(int d, int run, int half) {
  return d * kTileK + ((run + 4 * half) ^ ((d >> 1) & 7)) * 8;
}

// 2^(code - top + kValueLift) as f16, 0 below its least subnormal
__device__ __forceinline__ uint16_t valueFactorF16(uint32_t code, uint32_t top) {
  int e = 127 + kValueLift + static_cast<int>(code) - static_cast<int>(top);
  e = e > 0 ? e : 0;
  return __builtin_bit_cast(uint16_t,
                            static_cast<f16>(__uint_as_float(static_cast<uint32_t>(e) << 23)));
}

// 8 value codes times their tokens' factors
__device__ __forceinline__ U128 valueFragment(uint32_t w0, uint32_t w1, const U128& factors) {
  return __builtin_bit_cast(U128, __builtin_bit_cast(f16x8, codesToF16(w0, w1)) *
                                      __builtin_bit_cast(f16x8, factors));
}

// 8 key codes times 2^e as bf16 (exact: a bf16 has fp32's exponents)
__device__ __forceinline__ U128 scaledKey(uint32_t w0, uint32_t w1, float scale) {
  return U128{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true))};
}

// A row's sum of weights 2^(score - m) and its reference m; its output is o / l * 2^e.
struct RowEnd {
  float l, m;
  int e;
};

// Of rows weighed by their reference and shift, o in units of the value scale top; sum: their lifted sum.
__device__ __forceinline__ RowEnd endOf(float sum, float ref, float shift, float scale, uint32_t top) {
  // the shift is what the weights have in them, but for far rows
  return {__builtin_ldexpf(sum, -static_cast<int>(kLift)), farRow(shift) ? ref * scale : kLift - shift,
          static_cast<int>(top) - 127 - kValueLift - static_cast<int>(kLift)};
}
__device__ __forceinline__ RowEnd endOf(const RowSum& row) {
  return {rowsSum(row.l), row.m, static_cast<int>(row.unit) - 127};
}

// Rows first .. first + 16 QB - 1 of a wave: stored, or left with their maximum and sum for the join.
template <class T, int D, int QB>
__device__ __forceinline__ void storeRows(const Kv8AttentionArgs& a, int b, int kvh, int group, int rows,
                                          int first, const f32x4 (&o)[QB][D / 16],
                                          const RowEnd (&end)[QB]) {
  constexpr int DT = D / 16;
  const int lane = threadIdx.x % kWave, r = lane % 16, g = lane / 16;
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float L = end[qb].l;
    const int p = first + qb * 16 + r, e = end[qb].e;
    if (p >= rows) continue;
    const RowAt at = rowAt(p, group, kvh);
    const float inv = L == 0.f ? 0.f : 1.f / L;  // no key, or none of any weight: zeros
    if (a.splits == 1) {
      T* out = static_cast<T*>(a.out) + outAt(a, b, at, D) + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st(out + 16 * dt + i, __builtin_ldexpf(o[qb][dt][i] * inv, e));
    } else {
      const int64_t part = queryAt(a, b, at, 1) * a.splits + blockIdx.z;
      if (g == 0) {
        a.part_ml[part * 2] = L == 0.f ? -INFINITY : fminf(end[qb].m, kNoReference);
        a.part_ml[part * 2 + 1] = L;
      }
      float* out = a.part_o + part * D + 4 * g;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          out[16 * dt + i] = __builtin_ldexpf(o[qb][dt][i] * inv, e);
    }
  }
}

// How far apart the value scales of a workgroup's keys may lie (powers of two) for V to be staged relative to
// the largest: its elements are exact in f16 down to 2^-22, and a weight is one down to 2^-36 of its row's
// largest, so what is lost is below 2^-22 of the smallest scale an element. Past that the workgroup starts again
// with weights in units of their rows (RowSum): 2048 tokens over 8192 take 712 us in place of 294, 4 x 2048
// prompt tokens (14 / 2 x 64) 107 in place of 53. Scale code 0 is left out, since rows of zeros have it: next
// to a value scale above 2^-113 such rows, which are below 2^-118, may count for zeros.
constexpr uint32_t kNear = 14;
struct ValueScales {  // uniform
  uint32_t top = 0, bottom = 255;  // of the codes seen so far
  // Whether the lanes' codes (0 for keys that are not there) lie outside what was seen.
  __device__ __forceinline__ bool news(uint32_t code) const {
    return __builtin_amdgcn_ballot_w64(code > top || (code != 0 && code < bottom)) != 0;
  }
  // Takes them in; 2^(top before - top).
  __device__ __forceinline__ float add(uint32_t code) {
    const uint32_t before = top;
    const uint32_t most = waveMaxHalves(code | (code != 0 ? 255u - code : 0u) << 16);
    const uint32_t high = most & 0xFFFFu, low = 255u - (most >> 16);
    top = high > top ? high : top;
    bottom = low < bottom ? low : bottom;
    return valueFactor(before, top);
  }
  __device__ __forceinline__ bool apart() const { return top > bottom + kNear; }
};

template <int D>
struct ChunkLds {
  uint16_t k[2][kTileK * D];
  uint16_t v[2][D * kTileK];
  float kf[kChunkWaves][kTileK];     // each wave's own copy of the tile's key scales
  uint16_t vf[kChunkWaves][kTileK];  // and of the value factors
};

// kInRows: weights in units of their rows. Returns false, the same in every wave and with nothing stored, where
// the other form finds value scales too far apart. t: the thread.
template <class T, int D, int QB, bool kSmall, bool kInRows>
__device__ __forceinline__ bool kv8_chunk_rows(const Kv8AttentionArgs& a, ChunkLds<D>& lds, const int t) {
  using Ty = Kv8Type<T>;
  // f16 keys stay unscaled (their range would not hold a scaled one), the score takes the scale
  constexpr bool kScaleKeys = !__is_same(T, f16);
  constexpr int DT = D / 16, DK = D / 32, kThreads = kChunkWaves * kWave, kRows = 16 * QB * kChunkWaves;
  constexpr int kParts = D / 16;         // 16-code chunks of a key
  constexpr int kPer = 4 * D / kThreads;  // chunks of K, and of V^T, a thread
  const Kv8Pages& pg = a.pages;
  const int lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int r = lane % 16, g = lane / 16;
  const int group = a.q_heads / pg.heads, rows = a.seq_q * group, bs = pg.block_size;
  // the pair is the fast index (consecutive workgroups go to different XCDs), the row tile the slow
  // one, last tile first: under a causal mask the longest workgroups start first
  const uint32_t lin = blockIdx.x + gridDim.x * blockIdx.y;
  const int pair = static_cast<int>(lin % gridDim.y), b = pair / pg.heads, kvh = pair - b * pg.heads;
  const int p0 = static_cast<int>(gridDim.x - 1 - lin / gridDim.y) * kRows;
  const int pw = p0 + wave * 16 * QB;  // the wave's first row
  const bool active = pw < rows;       // uniform over the wave
  const int64_t past = kv8First(pg, b);
  auto clamped = [&](int p) { return p < rows ? p : rows - 1; };

  U128 qf[QB][DK][Ty::kQ];
  int lim[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const RowAt at = rowAt(clamped(pw + qb * 16 + r), group, kvh);  // clamped: not stored
    const T* q = static_cast<const T*>(a.q) + queryAt(a, b, at, D) + g * 8;
#pragma unroll
    for (int c = 0; c < DK; ++c) queryFragment<T>(q + c * 32, qf[qb][c]);
    lim[qb] = visibleKeys(a, past, at.i);
  }
  const int wg_keys = visibleKeys(a, past, clamped(p0 + kRows - 1) / group);
  const int wave_full = visibleKeys(a, past, clamped(pw) / group);  // keys every row of the wave sees

  const int all_tiles = (wg_keys + kTileK - 1) / kTileK;
  const int per = (all_tiles + a.splits - 1) / a.splits;
  const int kt0 = static_cast<int>(blockIdx.z) * per;
  const int kt1 = kt0 + per < all_tiles ? kt0 + per : all_tiles;

  // Where a tile lies: the page ids of its four runs of 16 keys (one page where pages are not small),
  // -1 for a page that holds nothing, and its first slot. Tiles past the last one repeat it; runs past
  // the pages repeat the last one and are masked.
  struct Where {
    int id[4];
    int slot;
  };
  const int32_t* table = pg.table + static_cast<int64_t>(b) * pg.max_blocks;
  const int kt_last = kt1 - 1;
  const int tiles_per_page = kSmall ? 1 : bs / kTileK;
  const int last_run = static_cast<int>((a.capacity - 1) / 16), run_shift = bs == 32 ? 1 : 0;
  int next_kt = kt0, next_page = kSmall ? 0 : kt0 / tiles_per_page;
  int next_slot = kSmall ? 0 : (kt0 - next_page * tiles_per_page) * kTileK;
  Where coming;  // as loaded
  auto loadIds = [&] {  // of tile next_kt, which then moves on
#pragma unroll
    for (int u = 0; u < (kSmall ? 4 : 1); ++u) {
      int page = next_page;
      if constexpr (kSmall) {
        const int run = next_kt * 4 + u;
        page = (run < last_run ? run : last_run) >> run_shift;
      }
      coming.id[u] = gp(table)[page];
    }
    coming.slot = next_slot;
    if (next_kt < kt_last) {
      ++next_kt;
      next_slot += kTileK;
      if (next_slot >= bs) {
        next_slot = 0;
        ++next_page;
      }
    }
  };
  auto takeIds = [&] {  // once they are there; the same in every lane
    Where w = coming;
#pragma unroll
    for (int u = 0; u < (kSmall ? 4 : 1); ++u) {
      const int x = __builtin_amdgcn_readfirstlane(coming.id[u]);
      w.id[u] = x < pg.num_blocks ? x : -1;
    }
    return w;
  };
  auto pick = [&](const Where& w, int u) {
    return !kSmall || u == 0 ? w.id[0] : u == 1 ? w.id[1] : u == 2 ? w.id[2] : w.id[3];
  };
  auto headOf = [&](int page) {  // a page that holds nothing: page 0 is read in its place and masked
    return static_cast<int64_t>(page < 0 ? 0 : page) * pg.heads + kvh;
  };
  // offsets of this thread's chunks within a page's head
  const int64_t head = static_cast<int64_t>(bs) * D;
  uint32_t ko[kPer], vo[kPer];
  auto chunkOf = [&](int i) { return t + i * kThreads; };
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = chunkOf(i);
    ko[i] = kSmall ? static_cast<uint32_t>(c / kParts % bs * D + c % kParts * 16)
                   : static_cast<uint32_t>(c * 16);
    vo[i] = static_cast<uint32_t>(c / 4) * static_cast<uint32_t>(bs) +
            static_cast<uint32_t>(kSmall ? 16 * (c % 4) % bs : 16 * (c % 4));
  }
  // A tile's codes on their way to LDS, and the scales of this lane's key.
  U128 kr[kPer], vr[kPer];
  uint32_t kc = 0, vc = 0;
  bool in_page = false;
  auto fetchScales = [&](const Where& w) {
    const int page = pick(w, g);
    in_page = page >= 0;
    const uint8_t* sb = pg.scales + headOf(page) * 2 * bs + (kSmall ? 0 : w.slot);
    const uint32_t at = static_cast<uint32_t>(kSmall ? lane % bs : lane);
    kc = gp(sb)[at];
    vc = gp(sb + bs)[at];
  };
  auto fetchKeys = [&](const Where& w) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint8_t* kb = pg.key + headOf(pick(w, (chunkOf(i)) / kParts / 16)) * head +
                          (kSmall ? 0 : static_cast<int64_t>(w.slot) * D);
      kr[i] = gload16(kb + ko[i]);
    }
  };
  auto fetchValues = [&](const Where& w) {
    const uint8_t* vb = pg.value + headOf(pick(w, t % 4)) * head + (kSmall ? 0 : w.slot);
#pragma unroll
    for (int i = 0; i < kPer; ++i) vr[i] = gload16(vb + vo[i]);
  };

  const float score_scale = kScaleKeys ? a.scale_log2 : 1.f;
  const uint32_t one = r == 0 ? 0x3C003C00u : 0u;
  const U128 ones = U128{one, one, one, one};  // A fragment of one row of ones

  f32x4 o[QB][DT];
  f32x4 ls[QB];      // element 0 of the lanes g = 0: the sum of row r's weights
  float shift[QB];   // kLift less the row's reference, times the scale
  float ref[QB];     // the reference, a score
  bool far = false;  // a row of the wave has been farRow
  ValueScales scales;  // o is kept in units of the largest
  RowSum row[QB];    // in place of these where kInRows
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    shift[qb] = kNoReference;
    ref[qb] = 0.f;
    ls[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[qb][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  Where at{};
  auto fetch = [&] {
    at = takeIds();
    loadIds();
    fetchScales(at);
    fetchKeys(at);
    fetchValues(at);
  };
  if (kt0 < kt1) {
    loadIds();
    fetch();
  }
  int end = kt1;
  for (int kt = kt0; kt < end; ++kt) {
    const int k0 = kt * kTileK, buf = kt & 1;
    const bool live = in_page && k0 + lane < wg_keys;
    const bool bad = kc == 255u || vc == 255u;
    const uint64_t lives = __builtin_amdgcn_ballot_w64(live);
    const uint64_t bads = __builtin_amdgcn_ballot_w64(live && bad);
    const uint32_t vcode = bad || !live ? 0u : vc;
    if constexpr (!kInRows) {
      if (scales.news(vcode)) {  // every wave comes to the same
        const float down = scales.add(vcode);
        if (scales.apart()) end = kt;  // the last tile
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= down;
      }
      lds.vf[wave][lane] = valueFactorF16(vcode, scales.top);
    }
    const float kf = mxScaleValue(bad ? 255u : kc) * (kScaleKeys ? 1.f : a.scale_log2);
    if constexpr (kScaleKeys) lds.kf[wave][lane] = kf;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes' factors are read below
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = chunkOf(i);
      const int key = c / kParts, part = c % kParts;
      // the score of row 4 g + i of the 16-key group kk is that of key 16 g + 4 kk + i
      const int row = 16 * (key % 16 / 4) + 4 * (key / 16) + key % 4;
      U128 k0v, k1v;
      if constexpr (kScaleKeys) {
        const float f = lds.kf[wave][key];
        k0v = scaledKey(kr[i][0], kr[i][1], f);
        k1v = scaledKey(kr[i][2], kr[i][3], f);
        if (bads != 0) {
          rarely();
          if (bads >> key & 1) k0v = k1v = U128{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
        }
      } else {
        k0v = keyFragment<T>(kr[i][0], kr[i][1]);
        k1v = keyFragment<T>(kr[i][2], kr[i][3]);
      }
      *reinterpret_cast<U128*>(&lds.k[buf][keyChunk<D>(row, 2 * part)]) = k0v;
      *reinterpret_cast<U128*>(&lds.k[buf][keyChunk<D>(row, 2 * part + 1)]) = k1v;
    }
    U128 vf[2];
    if constexpr (!kInRows) {
      vf[0] = load16(&lds.vf[wave][16 * (t % 4)]);
      vf[1] = load16(&lds.vf[wave][16 * (t % 4) + 8]);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = chunkOf(i) / 4, run = t % 4;
      if (lives != ~uint64_t{0}) {
        rarely();
        keepBytes(vr[i], static_cast<uint32_t>(lives >> (16 * run)) & 0xFFFFu);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w0 = vr[i][2 * half], w1 = vr[i][2 * half + 1];
        *reinterpret_cast<U128*>(&lds.v[buf][valueChunk(d, run, half)]) =
            kInRows ? codesToF16(w0, w1) : valueFragment(w0, w1, vf[half]);
      }
    }
    fetch();
    // one barrier a tile: the other buffer was last read before the previous one
    __syncthreads();
    if (!active) continue;

    f32x4 s[QB][4];
    U128 frag[kAhead + 1];
    constexpr int kSteps = 4 * DK;
    auto keyRead = [&](int i) {
      return load16(&lds.k[buf][keyChunk<D>(i / DK * 16 + r, 4 * (i % DK) + g)]);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag[i] = keyRead(i);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < kSteps) frag[(i + kAhead) % (kAhead + 1)] = keyRead(i + kAhead);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
        if (i % DK == 0) s[qb][i / DK] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = Ty::kQ - 1; u >= 0; --u)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
          s[qb][i / DK] = keyMma<T>(frag[i % (kAhead + 1)], qf[qb][i % DK][u], s[qb][i / DK]);
    }
    __builtin_amdgcn_sched_barrier(0);
    auto valueRead = [&](int i) {
      return load16(&lds.v[buf][valueChunk(16 * (i % DT) + r, g, i / DT)]);
    };
    const bool full = lives == ~uint64_t{0} && k0 + kTileK <= wave_full;
    U128 pf[QB][Ty::kP][2];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      if constexpr (!kScaleKeys) timesKeys(s[qb], kf);
      if constexpr (kInRows && kScaleKeys) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) s[qb][kk] *= score_scale;
      }
      if (!full) {
        const int seen = lim[qb] - k0 - 16 * g;
        const uint32_t mine = static_cast<uint32_t>(lives >> (16 * g)) & 0xFFFFu &
                              (seen >= 16 ? 0xFFFFu : seen > 0 ? (1u << seen) - 1u : 0u);
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (!(mine >> n & 1u)) s[qb][n / 4][n % 4] = -INFINITY;
      }
      if constexpr (kInRows) {
        weigh(s[qb], static_cast<float>(vcode), row[qb], o[qb]);
      } else {
        const float smax = largestOf(s[qb]);
        // the reference moves only when a weight would pass 2^(kLift + kSlack)
        bool over = fmaf(smax, score_scale, shift[qb]) > kLift + kSlack;
        if (far) {
          rarely();
          over = farExponent(smax, ref[qb], shift[qb], score_scale) > kLift + kSlack;
        }
        if (__builtin_amdgcn_ballot_w64(over)) {
          rarely();
          const float alpha = moveReference(smax, score_scale, ref[qb], shift[qb]);
          far = far || __builtin_amdgcn_ballot_w64(farRow(shift[qb])) != 0;
          ls[qb] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= alpha;
        }
        float to_lift = shift[qb];
        if (far) {
          rarely();
          to_lift = fromReference(s[qb], ref[qb], shift[qb]);
        }
#pragma unroll
        for (int n = 0; n < 16; ++n)
          s[qb][n / 4][n % 4] =
              __builtin_amdgcn_exp2f(fmaf(s[qb][n / 4][n % 4], score_scale, to_lift));
      }
      packWeights<Ty::kP>(s[qb], pf[qb]);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag[i] = valueRead(i);
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < 2 * DT) frag[(i + kAhead) % (kAhead + 1)] = valueRead(i + kAhead);
#pragma unroll
      for (int u = Ty::kP - 1; u >= 0; --u)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          if (!kInRows && i % DT == 0) ls[qb] = F16::mma(ones, pf[qb][u][i / DT], ls[qb]);
          o[qb][i % DT] = F16::mma(frag[i % (kAhead + 1)], pf[qb][u][i / DT], o[qb][i % DT]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (scales.apart()) return false;
  RowEnd ends[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    ends[qb] = kInRows ? endOf(row[qb])
                       : endOf(__shfl(ls[qb][0], r, kWave), ref[qb], shift[qb], score_scale, scales.top);
  storeRows<T, D, QB>(a, b, kvh, group, rows, pw, o, ends);
  return true;
}

template <class T, int D, int QB, bool kSmall>
__device__ __forceinline__ void kv8_chunk(const Kv8AttentionArgs& a) {
  __shared__ __attribute__((aligned(16))) ChunkLds<D> lds;
  if (kv8_chunk_rows<T, D, QB, kSmall, false>(a, lds, threadIdx.x)) return;
  __syncthreads();  // waves still read the last tile
  kv8_chunk_rows<T, D, QB, kSmall, true>(a, lds, againOf(threadIdx.x));
}

// ---------------------------------------------------------------------------------------------
// Many rows over long contexts (bf16, head_dim 128, pages of a multiple of 64): 8 waves and 256 rows a
// workgroup, in two halves that run a phase apart, a barrier between phases. In its matrix phase a
// half adds the values of tile kt - 1 and takes the scores of tile kt, and between those products it
// stages its part of the keys of kt + 1 and the values of kt; in the other phase it asks for the codes of the
// tile after and turns the scores into weights. So one wave of a SIMD feeds the matrix unit while the other
// has its softmax, where the kernel above leaves it to chance:
//   phase     0     1     2     3     4
//   half 0   M(0)  S(0)  M(1)  S(1)  M(2)
//   half 1         M(0)  S(0)  M(1)  S(1)
// A tile's buffers are written by both halves in their M(kt - 1), two phases in a row, and read in their M of
// the keys' tile, or the one after for values: each has two. Wave priority goes with the matrix phase.
//
// 2048 tokens over 8192 (28 / 4 heads x 128) 291 us, 930 TFLOP/s; above 339. A phase takes 1800 cycles
// either way (products alone: 1455, of which the unit needs 1088). Steps, in us: everything staged in the
// softmax phase 357, between the products 416, the scales read by their users and page offsets in 32 bits
// 335, priority 309, loads issued in the softmax phase 295.
// ---------------------------------------------------------------------------------------------
constexpr int kPhasedWaves = 8;

template <int D>
struct PhasedLds {
  uint16_t k[2][kTileK * D];
  uint16_t v[2][D * kTileK];
  uint16_t vf[kPhasedWaves][kTileK];  // each wave's own copy of a tile's value factors
};

template <bool kBoth>
struct Products {
  static constexpr bool kKeys = kBoth;
};

// As kv8_chunk_rows.
template <bool kInRows>
__device__ __forceinline__ bool kv8_phased_rows(const Kv8AttentionArgs& a, PhasedLds<128>& lds, const int t) {
  using T = bf16;
  constexpr int D = 128, QB = 2, DT = D / 16, DK = D / 32, kRows = 16 * QB * kPhasedWaves;
  constexpr int kParts = D / 16;  // 16-code chunks of a key; a thread stages one of K and one of V^T
  static_assert(kTileK * kParts == kPhasedWaves * kWave);
  const Kv8Pages& pg = a.pages;
  const int lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int r = lane % 16, g = lane / 16;
  const int group = a.q_heads / pg.heads, rows = a.seq_q * group, bs = pg.block_size;
  // pairs, row tiles and clamped rows as in kv8_chunk
  const uint32_t lin = blockIdx.x + gridDim.x * blockIdx.y;
  const int pair = static_cast<int>(lin % gridDim.y), b = pair / pg.heads, kvh = pair - b * pg.heads;
  const int p0 = static_cast<int>(gridDim.x - 1 - lin / gridDim.y) * kRows;
  const int pw = p0 + wave * 16 * QB;  // the wave's first row
  const bool late = wave >= kPhasedWaves / 2;
  const int64_t past = kv8First(pg, b);
  auto clamped = [&](int p) { return p < rows ? p : rows - 1; };

  U128 qf[QB][DK][1];
  int lim[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const RowAt at = rowAt(clamped(pw + qb * 16 + r), group, kvh);  // clamped: not stored
    const T* q = static_cast<const T*>(a.q) + queryAt(a, b, at, D) + g * 8;
#pragma unroll
    for (int c = 0; c < DK; ++c) queryFragment<T>(q + c * 32, qf[qb][c]);
    lim[qb] = visibleKeys(a, past, at.i);
  }
  const int wg_keys = visibleKeys(a, past, clamped(p0 + kRows - 1) / group);
  const int wave_full = visibleKeys(a, past, clamped(pw) / group);  // keys every row of the wave sees
  const int all_tiles = (wg_keys + kTileK - 1) / kTileK;
  const int per = (all_tiles + a.splits - 1) / a.splits;
  const int kt0 = static_cast<int>(blockIdx.z) * per;
  const int kt1 = kt0 + per < all_tiles ? kt0 + per : all_tiles;

  // The page id of tile next_kt is read a tile ahead of the loads that use it. Tiles past the last one
  // repeat it.
  const int32_t* table = pg.table + static_cast<int64_t>(b) * pg.max_blocks;
  const int tiles_per_page = bs / kTileK;
  int next_kt = kt0, next_page = kt0 / tiles_per_page;
  int next_slot = (kt0 - next_page * tiles_per_page) * kTileK;
  int coming_id = 0, coming_slot = 0;
  auto loadId = [&] {
    coming_id = gp(table)[next_page];
    coming_slot = next_slot;
    if (next_kt < kt1 - 1) {
      ++next_kt;
      next_slot += kTileK;
      if (next_slot >= bs) {
        next_slot = 0;
        ++next_page;
      }
    }
  };
  const uint32_t held = static_cast<uint32_t>(pg.num_blocks < INT32_MAX ? pg.num_blocks : INT32_MAX);
  const uint32_t head = static_cast<uint32_t>(bs) * D;  // attentionPlan: below 2^31
  const uint64_t page_codes = static_cast<uint64_t>(pg.heads) * head;
  const uint64_t page_scales = static_cast<uint64_t>(pg.heads) * 2u * static_cast<uint32_t>(bs);
  const uint8_t* const keys = pg.key + static_cast<uint64_t>(kvh) * head;
  const uint8_t* const values = pg.value + static_cast<uint64_t>(kvh) * head;
  const uint8_t* const scales = pg.scales + static_cast<uint64_t>(kvh) * 2u * static_cast<uint32_t>(bs);
  // This thread's chunks: part of key t / kParts, and the run of 16 keys t % 4 of dim t / 4.
  const int key = t / kParts, part = t % kParts, dim = t / 4, run = t % 4;
  const uint32_t vo = static_cast<uint32_t>(dim) * static_cast<uint32_t>(bs) + 16u * run;
  const int key_row = 16 * (key % 16 / 4) + 4 * (key / 16) + key % 4;  // as in kv8_chunk
  // On their way: the keys of a tile and the scales of this thread's key, the value scale of this lane's
  // key, and the values and value scales of the tile before.
  U128 kr, vr;
  uint32_t own_k = 0, own_v = 0, vc = 0, vc_before = 0;
  bool in = false, in_before = false;  // those tiles' pages hold something
  uint64_t value_page = 0;
  auto fetch = [&] {
    const uint32_t id = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(coming_id));
    const uint32_t slot = static_cast<uint32_t>(coming_slot);
    in_before = in;
    in = id < held;  // else page 0 is read in its place and masked
    const uint64_t page = in ? id : 0u;
    loadId();
    const uint8_t* sb = scales + page * page_scales + slot;
    own_k = gp(sb)[static_cast<uint32_t>(key)];
    own_v = gp(sb + bs)[static_cast<uint32_t>(key)];
    vc_before = vc;
    vc = gp(sb + bs)[static_cast<uint32_t>(lane)];
    kr = gload16(keys + page * page_codes + static_cast<uint64_t>(slot) * D + static_cast<uint32_t>(t) * 16);
    vr = gload16(values + value_page + vo);
    value_page = page * page_codes + slot;
  };

  f32x4 o[QB][DT];
  RowSum row[QB];   // in place of the next four where kInRows
  f32x4 ls[QB];     // element 0 of the lanes g = 0: the sum of row r's weights
  float shift[QB];  // kLift less the row's reference, times the scale
  float ref[QB];    // the reference, a score
  bool far = false;  // a row of the wave has been farRow
  f32x4 s[QB][4];
  U128 pf[QB][1][2];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    shift[qb] = kNoReference;
    ref[qb] = 0.f;
    ls[qb] = f32x4{0.f, 0.f, 0.f, 0.f};
    pf[qb][0][0] = pf[qb][0][1] = zero16();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[qb][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one = r == 0 ? 0x3C003C00u : 0u;
  const U128 ones = U128{one, one, one, one};  // A fragment of one row of ones

  // The value scales up to the tile whose factors were written last, the largest up to the one before, and
  // the one that o is kept in.
  ValueScales seen_scales;
  uint32_t top_before = 0, top_o = 0;
  auto codeIn = [&](int kt, bool there, uint32_t code) {  // this lane's of tile kt, 0 where nothing is
    return code == 255u || !there || kt * kTileK + lane >= wg_keys ? 0u : code;
  };
  auto factors = [&](int kt, bool there, uint32_t raw) {  // of tile kt
    if constexpr (kInRows) return;
    const uint32_t code = codeIn(kt, there, raw);
    top_before = seen_scales.top;
    if (seen_scales.news(code)) {  // every wave comes to the same
      rarely();
      seen_scales.add(code);
    }
    lds.vf[wave][lane] = valueFactorF16(code, seen_scales.top);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes' factors are read
  };
  uint64_t lives = 0;  // the keys of the tile staged last that are there
  U128 vf[2] = {zero16(), zero16()};
  uint32_t nan = 0;
  float key_scale = 1.f;
  auto keyScale = [&] {
    const bool bad = own_k == 255u || own_v == 255u;
    nan = bad ? 0x7FC07FC0u : 0u;  // the codes of such a row are 0
    key_scale = mxScaleValue(bad ? 127u : own_k);
  };
  auto stageKeys = [&](int buf, int half) {
    U128 w = scaledKey(kr[2 * half], kr[2 * half + 1], key_scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] |= nan;
    *reinterpret_cast<U128*>(&lds.k[buf][keyChunk<D>(key_row, 2 * part + half)]) = w;
  };
  auto stageValues = [&](int buf, int half) {
    const uint32_t w0 = vr[2 * half], w1 = vr[2 * half + 1];
    *reinterpret_cast<U128*>(&lds.v[buf][valueChunk(dim, run, half)]) =
        kInRows ? codesToF16(w0, w1) : valueFragment(w0, w1, vf[half]);
  };
  // The keys of kt + 1 and the values of kt, in pieces that fit between products.
  constexpr int kPieces = 5, kPieceSteps = 3;
  auto stage = [&](int kt, int piece) {
    const int vbuf = kt & 1, kbuf = vbuf ^ 1;
    if (piece == 0) {
      if constexpr (!kInRows) {
        vf[0] = load16(&lds.vf[wave][16 * run]);
        vf[1] = load16(&lds.vf[wave][16 * run + 8]);
      }
      const int n = wg_keys - kt * kTileK;
      lives = !in_before || n <= 0 ? uint64_t{0} : n >= kTileK ? ~uint64_t{0} : (uint64_t{1} << n) - 1;
    } else if (piece == 1) {
      keyScale();
      stageKeys(kbuf, 0);
    } else if (piece == 2) {
      stageKeys(kbuf, 1);
    } else if (piece == 3) {
      if (lives != ~uint64_t{0}) {
        rarely();
        keepBytes(vr, static_cast<uint32_t>(lives >> (16 * run)) & 0xFFFFu);
      }
      stageValues(vbuf, 0);
    } else {
      stageValues(vbuf, 1);
    }
  };
  auto products = [&](int kt, auto which) {  // the values of kt - 1, and the scores of kt
    constexpr bool kKeys = decltype(which)::kKeys;
    constexpr int kValueSteps = 2 * DT, kSteps = kValueSteps + (kKeys ? 4 * DK : 0);
    const int kbuf = kt & 1, vbuf = kbuf ^ 1;
    auto read = [&](int i) {
      if (i < kValueSteps) return load16(&lds.v[vbuf][valueChunk(16 * (i % DT) + r, g, i / DT)]);
      const int n = i - kValueSteps;
      return load16(&lds.k[kbuf][keyChunk<D>(n / DK * 16 + r, 4 * (n % DK) + g)]);
    };
    if (top_before != top_o) {
      rarely();
      const float down = valueFactor(top_o, top_before);
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= down;
      top_o = top_before;
    }
    U128 frag[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) frag[i] = read(i);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < kSteps) frag[(i + kAhead) % (kAhead + 1)] = read(i + kAhead);
      if (kKeys && i % kPieceSteps == 0 && i / kPieceSteps < kPieces) stage(kt, i / kPieceSteps);
      const U128& f = frag[i % (kAhead + 1)];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        if (i < kValueSteps) {
          if (!kInRows && i % DT == 0) ls[qb] = F16::mma(ones, pf[qb][0][i / DT], ls[qb]);
          o[qb][i % DT] = F16::mma(f, pf[qb][0][i / DT], o[qb][i % DT]);
        } else {
          const int n = i - kValueSteps;
          if (n % DK == 0) s[qb][n / DK] = f32x4{0.f, 0.f, 0.f, 0.f};
          s[qb][n / DK] = keyMma<T>(f, qf[qb][n % DK][0], s[qb][n / DK]);
        }
      }
    }
  };

  if (kt0 < kt1) {
    // the first tile's keys; zeros in place of the values before it, whose weights are 0
    loadId();
    fetch();
    keyScale();
    stageKeys(kt0 & 1, 0);
    stageKeys(kt0 & 1, 1);
    factors(kt0, in, vc);
    vr = zero16();
    stageValues((kt0 & 1) ^ 1, 0);
    stageValues((kt0 & 1) ^ 1, 1);
    fetch();
    __syncthreads();
    if (late) __syncthreads();
    for (int kt = kt0; kt < kt1; ++kt) {
      const int k0 = kt * kTileK;
      __builtin_amdgcn_s_setprio(1);
      products(kt, Products<true>{});
      __builtin_amdgcn_s_setprio(0);
      __syncthreads();
      const float code = static_cast<float>(codeIn(kt, in_before, vc_before));
      fetch();
      if constexpr (kInRows) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) s[qb][kk] *= a.scale_log2;
      }
      if (lives != ~uint64_t{0} || k0 + kTileK > wave_full) {
        rarely();
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const int seen = lim[qb] - k0 - 16 * g;
          const uint32_t mine = static_cast<uint32_t>(lives >> (16 * g)) & 0xFFFFu &
                                (seen >= 16 ? 0xFFFFu : seen > 0 ? (1u << seen) - 1u : 0u);
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (!(mine >> n & 1u)) s[qb][n / 4][n % 4] = -INFINITY;
        }
      }
      if constexpr (kInRows) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          weigh(s[qb], code, row[qb], o[qb]);
          packWeights<1>(s[qb], pf[qb]);
        }
      } else {
        float most[QB];
        bool over = false;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          most[qb] = -INFINITY;
#pragma unroll
          for (int n = 0; n < 16; ++n) most[qb] = fmaxf(most[qb], s[qb][n / 4][n % 4]);
          over |= fmaf(most[qb], a.scale_log2, shift[qb]) > kLift + kSlack;
        }
        if (far) {
          rarely();
          over = false;
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
            over |= farExponent(most[qb], ref[qb], shift[qb], a.scale_log2) > kLift + kSlack;
        }
        // the references move only when a weight would pass 2^(kLift + kSlack)
        if (__builtin_amdgcn_ballot_w64(over)) {
          rarely();
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) {
            const float alpha = moveReference(most[qb], a.scale_log2, ref[qb], shift[qb]);
            far = far || __builtin_amdgcn_ballot_w64(farRow(shift[qb])) != 0;
            ls[qb] *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[qb][dt] *= alpha;
          }
        }
        float to_lift[QB];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) to_lift[qb] = shift[qb];
        if (far) {
          rarely();
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) to_lift[qb] = fromReference(s[qb], ref[qb], shift[qb]);
        }
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
          for (int n = 0; n < 16; ++n)
            s[qb][n / 4][n % 4] =
                __builtin_amdgcn_exp2f(fmaf(s[qb][n / 4][n % 4], a.scale_log2, to_lift[qb]));
          packWeights<1>(s[qb], pf[qb]);
        }
      }
      factors(kt + 1, in_before, vc_before);
      __syncthreads();
    }
    products(kt1, Products<false>{});
    if (!late) __syncthreads();
  }
  if (seen_scales.apart()) return false;
  RowEnd ends[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
    ends[qb] = kInRows ? endOf(row[qb])
                       : endOf(__shfl(ls[qb][0], r, kWave), ref[qb], shift[qb], a.scale_log2, top_o);
  storeRows<T, D, QB>(a, b, kvh, group, rows, pw, o, ends);
  return true;
}

__device__ __forceinline__ void kv8_phased(const Kv8AttentionArgs& a) {
  __shared__ __attribute__((aligned(16))) PhasedLds<128> lds;
  if (kv8_phased_rows<false>(a, lds, threadIdx.x)) return;
  __syncthreads();  // waves still read the last tile
  kv8_phased_rows<true>(a, lds, againOf(threadIdx.x));
}

// ---------------------------------------------------------------------------------------------
// The splits' results of a row joined, one wave a row: every lane's loads go out before the first is
// used (a merge is a launch and one trip to memory). D / 4 lanes hold a split's row, 256 / D splits are
// read at a time, their sums joined at the end in a fixed order.
// ---------------------------------------------------------------------------------------------
template <class T, int D>
__device__ __forceinline__ void kv8_merge(const Kv8AttentionArgs& a) {
  constexpr int kLanes = D / 4, kAtOnce = kWave / kLanes, kDepth = 8;
  const int lane = threadIdx.x % kWave, mine = lane / kLanes, d = 4 * (lane % kLanes);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (row >= static_cast<int64_t>(a.batch) * a.q_heads * a.seq_q) return;
  const float* ml = a.part_ml + row * a.splits * 2;
  const float* o = a.part_o + row * a.splits * D + d;
  const bool have = lane < a.splits;
  const float m = have ? gp(ml)[2 * lane] : -INFINITY, l = have ? gp(ml)[2 * lane + 1] : 0.f;
  f32x4 x[kDepth];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int s = s0 + u * kAtOnce + mine;
      x[u] = s < a.splits ? *gp(reinterpret_cast<const f32x4*>(o + static_cast<int64_t>(s) * D))
                          : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  load(0);
  const float M = waveMax(m);
  // no key, or none of any weight: 0; a NaN sum stays one whatever its maximum
  const float f = (m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - M)) * l;
  const float L = waveSum(f);
  // divided before they meet the values: a sum of L times a value may pass the largest number
  float share = L == 0.f ? 0.f : f / L;
  // a share below what fp32 holds may meet values that make up for it: half of its exponent first
  const bool small = m - M < -100.f && m != -INFINITY;
  float half = 1.f;
  const bool any_small = __builtin_amdgcn_ballot_w64(small) != 0;
  if (any_small) {
    rarely();
    const float h = __builtin_amdgcn_exp2f(0.5f * (m - M));
    half = small ? h : 1.f;
    share = small ? h * (l / L) : share;
  }
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += kDepth * kAtOnce) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int s = s0 + u * kAtOnce + mine;
      const float w = __shfl(share, s % kWave, kWave);
      if (any_small) {
        rarely();
        x[u] *= __shfl(half, s % kWave, kWave);
      }
      if (s < a.splits) acc += x[u] * w;
    }
  }
#pragma unroll
  for (int off = kLanes; off < kWave; off *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], off, kWave);
  if (mine != 0) return;
  const int i = static_cast<int>(row % a.seq_q);
  const int64_t bh = row / a.seq_q, b = bh / a.q_heads;
  const RowAt at = {i, static_cast<int>(bh % a.q_heads)};
  T* out = static_cast<T*>(a.out) + outAt(a, b, at, D) + d;
#pragma unroll
  for (int u = 0; u < 4; ++u) st(out + u, acc[u]);
}

// ---------------------------------------------------------------------------------------------
// Any head_dim up to 256, page size, scale and alignment: one wave per row, 64 keys a round.
// ---------------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ void kv8_rows(const Kv8AttentionArgs& a) {
  FP_EXACT;  // as in weigh
  __shared__ float q_lds[256];
  __shared__ float p_lds[kWave];
  __shared__ int64_t at_lds[kWave];
  const Kv8Pages& pg = a.pages;
  const int lane = threadIdx.x, D = pg.head_dim;
  const int64_t total = static_cast<int64_t>(a.batch) * a.q_heads * a.seq_q;
  for (int64_t row = blockIdx.x; row < total; row += gridDim.x) {
    const int i = static_cast<int>(row % a.seq_q);
    const int64_t bh = row / a.seq_q, b = bh / a.q_heads;
    const int h = static_cast<int>(bh % a.q_heads), kvh = h / (a.q_heads / pg.heads);
    const int lim = visibleKeys(a, kv8First(pg, b), i);
    const T* q = static_cast<const T*>(a.q) + row * D;
    float largest = 0.f;
    for (int d = lane; d < D; d += kWave) largest = fmaxf(largest, fabsf(ld(q + d)));
    const bool up = waveMax(largest) >= kLargeQuery;
    for (int d = lane; d < D; d += kWave) q_lds[d] = ld(q + d) * (up ? kQueryDown : 1.f);
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    float unit = 0.f, peak = -INFINITY;  // as in RowSum
    for (int j0 = 0; j0 < lim; j0 += kWave) {
      const int j = j0 + lane;
      float s = -INFINITY;
      uint32_t code = 0;
      int64_t at = -1;
      if (j < lim) {
        const int64_t page = kv8Page(pg, b, j);
        if (page >= 0) {
          const int slot = j % pg.block_size;
          const int64_t head = page * pg.heads + kvh;
          const uint32_t kc = pg.scales[head * 2 * pg.block_size + slot];
          const uint32_t vc = pg.scales[(head * 2 + 1) * pg.block_size + slot];
          const uint8_t* k = pg.key + (head * pg.block_size + slot) * D;
          float dot = 0.f;
          for (int d = 0; d < D; ++d)
            dot = fmaf(q_lds[d], __builtin_amdgcn_cvt_f32_fp8(k[d], 0), dot);
          s = dot * mxScaleValue(kc == 255u || vc == 255u ? 255u : kc) *
              (up ? kQueryUp * a.scale_log2 : a.scale_log2);
          code = vc == 255u ? 0u : vc;
          at = head * D * pg.block_size + slot;
        }
      }
      const float next = fmaxf(m, waveMax(s));
      const float base = next == -INFINITY ? 0.f : next;
      const float past = s - base, fall = m - base;  // fall: -infinity on the first round
      l = l * __builtin_amdgcn_exp2f(fall) + waveSum(at >= 0 ? __builtin_amdgcn_exp2f(past) : 0.f);
      m = next;
      const float key_unit = static_cast<float>(code) - unit;
      peak = fmaxf(peak + fall, waveMax(past + key_unit));  // -infinity where s is
      const float by = peak == -INFINITY ? 0.f : rintf(peak);
      unit += by;
      peak -= by;
      const float down = __builtin_amdgcn_exp2f(fall - by);
      p_lds[lane] = at >= 0 ? __builtin_amdgcn_exp2f(past + (key_unit - by)) : 0.f;
      at_lds[lane] = at;
      __syncthreads();
      const int n = lim - j0 < kWave ? lim - j0 : kWave;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + u * kWave;
        if (d >= D) break;
        float x = acc[u] * down;
        for (int jj = 0; jj < n; ++jj)
          if (at_lds[jj] >= 0)
            x = fmaf(p_lds[jj], __builtin_amdgcn_cvt_f32_fp8(
                                    pg.value[at_lds[jj] + static_cast<int64_t>(d) * pg.block_size], 0), x);
        acc[u] = x;
      }
      __syncthreads();
    }
    T* out = static_cast<T*>(a.out) + outAt(a, b, {i, h}, D);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (lane + u * kWave < D)
        st(out + lane + u * kWave,
           l == 0.f ? 0.f : __builtin_ldexpf(acc[u] / l, static_cast<int>(unit) - 127));
  }
}

}  // namespace

// 64 or 128 rows a workgroup. WAVES of a SIMD at least: what LDS allows with head_dim 128, and with 64 what
// the registers that the loop needs do.
#define KV8_CHUNK(suffix, T, D, ROWS, WAVES)                                                     \
  extern "C" __global__ void __launch_bounds__(kChunkWaves* kWave, WAVES)                       \
      kv8_chunk_d##D##_r##ROWS##_##suffix(Kv8AttentionArgs a) {                                 \
    kv8_chunk<T, D, ROWS / 64, false>(a);                                                       \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(kChunkWaves* kWave, WAVES)                       \
      kv8_chunk_small_d##D##_r##ROWS##_##suffix(Kv8AttentionArgs a) {                           \
    kv8_chunk<T, D, ROWS / 64, true>(a);                                                        \
  }

#define KV8_ATTENTION(suffix, T)                                                                \
  extern "C" __global__ void __launch_bounds__(kDecWaves * kWave)                               \
      kv8_decode_d64_##suffix(Kv8AttentionArgs a) {                                             \
    kv8_decode<T, 64, false>(a);                                                                \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(kDecWaves * kWave)                               \
      kv8_decode_d128_##suffix(Kv8AttentionArgs a) {                                            \
    kv8_decode<T, 128, false>(a);                                                               \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(kDecWaves * kWave)                               \
      kv8_decode_small_d64_##suffix(Kv8AttentionArgs a) {                                       \
    kv8_decode<T, 64, true>(a);                                                                 \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(kDecWaves * kWave)                               \
      kv8_decode_small_d128_##suffix(Kv8AttentionArgs a) {                                      \
    kv8_decode<T, 128, true>(a);                                                                \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(256) kv8_merge_d64_##suffix(Kv8AttentionArgs a) { \
    kv8_merge<T, 64>(a);                                                                        \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(256)                                             \
      kv8_merge_d128_##suffix(Kv8AttentionArgs a) {                                             \
    kv8_merge<T, 128>(a);                                                                       \
  }                                                                                             \
  extern "C" __global__ void __launch_bounds__(64) kv8_rows_##suffix(Kv8AttentionArgs a) {      \
    kv8_rows<T>(a);                                                                             \
  }

KV8_ATTENTION(f32, float)
KV8_ATTENTION(bf16, bf16)
KV8_ATTENTION(f16, f16)

// attentionPlan (csrc/hip/kv_fp8_ops.cc) chooses the rows
KV8_CHUNK(f32, float, 64, 64, 3)
KV8_CHUNK(f32, float, 128, 64, 2)
KV8_CHUNK(bf16, bf16, 64, 64, 4)
KV8_CHUNK(bf16, bf16, 64, 128, 3)
KV8_CHUNK(bf16, bf16, 128, 64, 2)
KV8_CHUNK(bf16, bf16, 128, 128, 2)
KV8_CHUNK(f16, f16, 64, 64, 4)
KV8_CHUNK(f16, f16, 128, 64, 2)
KV8_CHUNK(f16, f16, 128, 128, 2)
extern "C" __global__ void __launch_bounds__(kPhasedWaves* kWave, 1)
    kv8_phased_d128_bf16(Kv8AttentionArgs a) {
  kv8_phased(a);
}
