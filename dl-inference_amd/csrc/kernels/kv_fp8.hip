// Writing and reading the 8-bit paged KV cache on gfx950 (formats in kv_fp8.h).
//
//  kv8_append   rows k, v [B, H, S, D] -> e4m3 elements and a scale per row, in the pages
//  kv8_rope     the same from the joined q|k|v projection: RoPE on q and k, q to its own tensor
//  kv8_read     the pages' rows back as T
//
// A row's scale needs its largest magnitude, so a row stays with the four lanes of a quad: 16
// elements each per 64 of head_dim, two DPP steps to the maximum. Keys go out as they lie, 16 bytes
// a lane; the value pool is dim-major, so a tile's value codes are turned in LDS and leave as runs
// of 16 tokens. Tiles start at multiples of their size in the cache, so a run never crosses a page.
//
// Bound by the bytes they move: 3.7 us for a launch in a graph taken off, 4 x 2048 tokens (4 heads x 128,
// bf16) are written in 5.0 us (25 MB, as fast as a large copy), 2 x 1000 tokens of q|k|v (28 / 4 heads x
// 128, f16) in 7.8 (36 MB, 4.6 TB/s), 8 x 8192 tokens (4 heads x 128) read back in 41.6 (202 MB, 4.9 TB/s).
// Short calls are bound by the chain of position, block table and store: 64 x 1 token 4.7 us with the
// launch, 32 x 1 of q|k|v 4.0, 300 tokens read 3.3.
#include "kv_fp8.h"

using namespace dk;

namespace {

template <class T>
__device__ __forceinline__ void load16Values(const T* p, float (&v)[16]) {
  mxLoad8<T, true>(p, *reinterpret_cast<float(*)[8]>(&v[0]));
  mxLoad8<T, true>(p + 8, *reinterpret_cast<float(*)[8]>(&v[8]));
}

template <class T>
__device__ __forceinline__ void store16Values(T* p, const float (&v)[16]) {
  mxStore8<T, true>(p, *reinterpret_cast<const float(*)[8]>(&v[0]));
  mxStore8<T, true>(p + 8, *reinterpret_cast<const float(*)[8]>(&v[8]));
}

// The pair (a, b) turned by the angle of (c, s): each product rounded by itself, as the plain
// arithmetic has it (a contraction would make codes depend on the kernel that computes them).
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  FP_EXACT;
  const float x = a * c - b * s, y = a * s + b * c;
  a = x;
  b = y;
}

// One workgroup: kTokens tokens of one row kind (grid.y: a head of k or v; with kRope a head of q, k
// or v) of sequence blockIdx.z, four threads per token.
template <class T, int D, int kTokens, bool kRope>
__device__ __forceinline__ void kv8_write(const Kv8WriteArgs& a) {
  constexpr int kGroups = D / 64;       // 16-element groups of a thread
  constexpr int kRuns = kTokens / 16;   // runs of 16 tokens in a tile
  constexpr int kPitch = kTokens + 8;  // bytes between dims in LDS: a quad's rows start on other banks
  __shared__ __attribute__((aligned(16))) uint8_t vs[D * kPitch];
  const Kv8Pages& p = a.pages;
  const int t = threadIdx.x, tok = t / 4, part = t % 4;
  const int row = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int64_t first = kv8First(p, b);
  const int64_t tile = (first & ~static_cast<int64_t>(kTokens - 1)) +
                       static_cast<int64_t>(blockIdx.x) * kTokens;
  const int64_t capacity = p.max_blocks * p.block_size;
  const int64_t pos = tile + tok, s = pos - first;
  const bool given = s >= 0 && s < a.seq;
  const int q_rows = kRope ? a.q_heads : 0;
  const bool is_q = kRope && row < q_rows;
  const bool is_v = row >= q_rows + p.heads;
  const int h = row - q_rows - (is_v ? p.heads : 0);
  int64_t page = -1;
  if (!is_q && given && pos >= 0 && pos < capacity) page = kv8Page(p, b, pos);
  // the run of 16 tokens that this thread writes of the values
  const int64_t run = tile + 16 * (t % kRuns);
  const int64_t low = first > 0 ? first : 0;
  const int64_t high = first + a.seq < capacity ? first + a.seq : capacity;
  int64_t run_page = -1;
  if (is_v && run + 16 > low && run < high) run_page = kv8Page(p, b, run > low ? run : low);

  float x[kGroups][16];
  if (given) {
    const T* src;
    if constexpr (kRope)
      src = static_cast<const T*>(a.qkv) +
            ((b * a.seq + s) * (q_rows + 2 * p.heads) + row) * static_cast<int64_t>(D);
    else
      src = static_cast<const T*>(is_v ? a.v : a.k) +
            ((b * p.heads + h) * a.seq + s) * static_cast<int64_t>(D);
#pragma unroll
    for (int j = 0; j < kGroups; ++j) load16Values(src + 16 * (part + 4 * j), x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[j][i] = 0.f;
  }
  if constexpr (kRope) {
    if (!is_v && given && pos >= 0 && pos < a.max_pos) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const int64_t at = pos * (D / 2) + 8 * (part + 4 * j);
        float c[8], sn[8];
        mxLoad8<float, true>(a.cos + at, c);
        mxLoad8<float, true>(a.sin + at, sn);
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(x[j][2 * i], x[j][2 * i + 1], c[i], sn[i]);
      }
    }
    if (is_q) {
      if (!given) return;
      T* out = static_cast<T*>(a.q_out) + ((b * a.q_heads + row) * a.seq + s) * D;
#pragma unroll
      for (int j = 0; j < kGroups; ++j) store16Values(out + 16 * (part + 4 * j), x[j]);
      return;
    }
    // a rotated key is rounded to T before it is quantised, as where the rotation is a node
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[j][i] = Num<T>::round(x[j][i]);
  }

  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) most = mxMax(most, x[j][i]);
  const uint32_t code = kv8Scale(mxQuadMax(most));
  const float inverse = mxInverse(code);
  uint32_t w[kGroups][4];
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[j][8 * half + i] * inverse;
      uint32_t word[2];
      MxFp8::pack(y, word);
      w[j][2 * half] = code == 255u ? 0u : word[0];
      w[j][2 * half + 1] = code == 255u ? 0u : word[1];
    }
  if (page >= 0) {
    const int64_t slot = pos % p.block_size;
    const int64_t at = page * p.heads + h;
    if (part == 0)
      gp(p.scales)[(at * 2 + (is_v ? 1 : 0)) * p.block_size + slot] = static_cast<uint8_t>(code);
    if (!is_v) {
      uint8_t* out = p.key + (at * p.block_size + slot) * D;
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
        *gp(reinterpret_cast<U32x4*>(out + 16 * (part + 4 * j))) =
            U32x4{w[j][0], w[j][1], w[j][2], w[j][3]};
    }
  }
  if (!is_v) return;  // the same for the whole workgroup
#pragma unroll
  for (int j = 0; j < kGroups; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      vs[(16 * (part + 4 * j) + i) * kPitch + tok] = static_cast<uint8_t>(w[j][i / 4] >> (8 * (i % 4)));
  __syncthreads();
  if (run_page < 0) return;
  const int slot = static_cast<int>(run > 0 ? run % p.block_size : 0);
  const bool whole = run >= low && run + 16 <= high;
  for (int e = t / kRuns; e < D; e += kTokens * 4 / kRuns) {
    const uint8_t* from = &vs[e * kPitch + 16 * (t % kRuns)];
    uint8_t* to = p.value + ((run_page * p.heads + h) * D + e) * p.block_size + slot;
    if (whole) {
      const U32x2 a0 = *reinterpret_cast<const U32x2*>(from);
      const U32x2 a1 = *reinterpret_cast<const U32x2*>(from + 8);
      *gp(reinterpret_cast<U32x4*>(to)) = U32x4{a0[0], a0[1], a1[0], a1[1]};
    } else {
      for (int i = 0; i < 16; ++i)
        if (run + i >= low && run + i < high) gp(to)[i] = from[i];
    }
  }
}

// Any head_dim up to 256, page size, number of rotated pairs and alignment: one wave per row, two
// elements a lane and 128 of head_dim.
template <class T, bool kRope>
__device__ __forceinline__ void kv8_write_any(const Kv8WriteArgs& a) {
  const Kv8Pages& p = a.pages;
  const int lane = threadIdx.x % kWave, D = p.head_dim;
  const int q_rows = kRope ? a.q_heads : 0, rows = q_rows + 2 * p.heads;
  const int64_t total = a.batch * rows * a.seq, capacity = p.max_blocks * p.block_size;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / kWave);
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWave) + threadIdx.x / kWave;
       at < total; at += step) {
    const int64_t s = at % a.seq, b = at / a.seq / rows;
    const int row = static_cast<int>(at / a.seq % rows);
    const bool is_q = row < q_rows, is_v = row >= q_rows + p.heads;
    const int h = row - q_rows - (is_v ? p.heads : 0);
    const int64_t pos = kv8First(p, b) + s;
    const T* src = kRope ? static_cast<const T*>(a.qkv) + ((b * a.seq + s) * rows + row) * D
                         : static_cast<const T*>(is_v ? a.v : a.k) + ((b * p.heads + h) * a.seq + s) * D;
    float x[2][2];
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int pair = lane + u * kWave, d = 2 * pair;
#pragma unroll
      for (int i = 0; i < 2; ++i) x[u][i] = d + i < D ? ld(src + d + i) : 0.f;
      if (kRope && !is_v && pair < a.pairs && pos >= 0 && pos < a.max_pos)
        turn(x[u][0], x[u][1], a.cos[pos * a.pairs + pair], a.sin[pos * a.pairs + pair]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kRope) x[u][i] = Num<T>::round(x[u][i]);
        if (is_q && d + i < D)
          st(static_cast<T*>(a.q_out) + ((b * a.q_heads + row) * a.seq + s) * D + d + i, x[u][i]);
        most = mxMax(most, x[u][i]);
      }
    }
    if (is_q) continue;
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
      const uint32_t other = __shfl_xor(most, off, kWave);
      most = other > most ? other : most;
    }
    if (pos < 0 || pos >= capacity) continue;
    const int64_t page = kv8Page(p, b, pos);
    if (page < 0) continue;
    const uint32_t code = kv8Scale(most);
    const float inverse = mxInverse(code);
    const int64_t slot = pos % p.block_size, head = page * p.heads + h;
    if (lane == 0)
      p.scales[(head * 2 + (is_v ? 1 : 0)) * p.block_size + slot] = static_cast<uint8_t>(code);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float y[8] = {x[u][0] * inverse, x[u][1] * inverse, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      uint32_t w[2];
      MxFp8::pack(y, w);
      if (code == 255u) w[0] = 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = 2 * (lane + u * kWave) + i;
        const uint8_t c = static_cast<uint8_t>(w[0] >> (8 * i));
        if (d < D) {
          if (is_v)
            p.value[(head * D + d) * p.block_size + slot] = c;
          else
            p.key[(head * p.block_size + slot) * D + d] = c;
        }
      }
    }
  }
}

// One workgroup: kTokens tokens of one head's keys or values (grid.y) of sequence blockIdx.z.
template <class T, int D, int kTokens>
__device__ __forceinline__ void kv8_read_tile(const Kv8ReadArgs& a) {
  constexpr int kGroups = D / 64, kRuns = kTokens / 16, kPitch = kTokens + 8;
  __shared__ __attribute__((aligned(16))) uint8_t vs[D * kPitch];
  const Kv8Pages& p = a.pages;
  const int t = threadIdx.x, tok = t / 4, part = t % 4;
  const bool is_v = static_cast<int>(blockIdx.y) >= p.heads;
  const int h = blockIdx.y - (is_v ? p.heads : 0);
  const int64_t b = blockIdx.z, first = kv8First(p, b);
  const int64_t tile = (first & ~static_cast<int64_t>(kTokens - 1)) +
                       static_cast<int64_t>(blockIdx.x) * kTokens;
  const int64_t capacity = p.max_blocks * p.block_size;
  const int64_t pos = tile + tok, s = pos - first;
  const bool wanted = s >= 0 && s < a.seq;
  int64_t page = -1;
  if (wanted && pos >= 0 && pos < capacity) page = kv8Page(p, b, pos);
  uint32_t code = 0;
  uint32_t w[kGroups][4] = {};
  if (page >= 0) {
    const int64_t slot = pos % p.block_size, at = page * p.heads + h;
    code = gp(p.scales)[(at * 2 + (is_v ? 1 : 0)) * p.block_size + slot];
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const U32x4 v = *gp(reinterpret_cast<const U32x4*>(
            p.key + (at * p.block_size + slot) * D + 16 * (part + 4 * j)));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = v[i];
      }
    }
  }
  if (is_v) {
    // runs of 16 tokens of one dim; what lies outside the pages is not read
    const int64_t run = tile + 16 * (t % kRuns);
    const int64_t run_page = run >= 0 && run < capacity ? kv8Page(p, b, run) : -1;
    if (run_page >= 0) {
      const int64_t slot = run % p.block_size;
      for (int e = t / kRuns; e < D; e += kTokens * 4 / kRuns) {
        const U32x4 v = *gp(reinterpret_cast<const U32x4*>(
            p.value + ((run_page * p.heads + h) * D + e) * p.block_size + slot));
        U32x2* to = reinterpret_cast<U32x2*>(&vs[e * kPitch + 16 * (t % kRuns)]);
        to[0] = U32x2{v[0], v[1]};
        to[1] = U32x2{v[2], v[3]};
      }
    }
    __syncthreads();
    if (page >= 0) {
#pragma unroll
      for (int j = 0; j < kGroups; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          w[j][i / 4] |= static_cast<uint32_t>(vs[(16 * (part + 4 * j) + i) * kPitch + tok]) << (8 * (i % 4));
    }
  }
  if (!wanted) return;
  const float scale = mxScaleValue(code);
  T* out = static_cast<T*>(is_v ? a.v : a.k) + ((b * p.heads + h) * a.seq + s) * D;
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    float v[16];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t pair[2] = {w[j][2 * half], w[j][2 * half + 1]};
      MxFp8::unpack(pair, *reinterpret_cast<float(*)[8]>(&v[8 * half]));
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = page >= 0 ? v[i] * scale : 0.f;
    store16Values(out + 16 * (part + 4 * j), v);
  }
}

template <class T>
__device__ __forceinline__ void kv8_read_any(const Kv8ReadArgs& a) {
  const Kv8Pages& p = a.pages;
  const int lane = threadIdx.x % kWave, D = p.head_dim;
  const int64_t total = a.batch * p.heads * a.seq, capacity = p.max_blocks * p.block_size;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x / kWave);
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWave) + threadIdx.x / kWave;
       at < total; at += step) {
    const int64_t s = at % a.seq, bh = at / a.seq, b = bh / p.heads, h = bh % p.heads;
    const int64_t pos = kv8First(p, b) + s;
    const int64_t page = pos >= 0 && pos < capacity ? kv8Page(p, b, pos) : -1;
    const int64_t slot = page >= 0 ? pos % p.block_size : 0, head = page * p.heads + h;
    float ks = 0.f, vs = 0.f;
    if (page >= 0) {
      ks = mxScaleValue(p.scales[head * 2 * p.block_size + slot]);
      vs = mxScaleValue(p.scales[(head * 2 + 1) * p.block_size + slot]);
    }
    for (int d = lane; d < D; d += kWave) {
      float k = 0.f, v = 0.f;
      if (page >= 0) {
        k = __builtin_amdgcn_cvt_f32_fp8(p.key[(head * p.block_size + slot) * D + d], 0) * ks;
        v = __builtin_amdgcn_cvt_f32_fp8(p.value[(head * D + d) * p.block_size + slot], 0) * vs;
      }
      st(static_cast<T*>(a.k) + at * D + d, k);
      st(static_cast<T*>(a.v) + at * D + d, v);
    }
  }
}

}  // namespace

#define KV8_KERNELS(suffix, T)                                                                    \
  extern "C" __global__ void __launch_bounds__(256) kv8_append_d64_##suffix(Kv8WriteArgs a) {     \
    kv8_write<T, 64, 64, false>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_append_d128_##suffix(Kv8WriteArgs a) {    \
    kv8_write<T, 128, 64, false>(a);                                                              \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64) kv8_append_few_d64_##suffix(Kv8WriteArgs a) {  \
    kv8_write<T, 64, 16, false>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64) kv8_append_few_d128_##suffix(Kv8WriteArgs a) { \
    kv8_write<T, 128, 16, false>(a);                                                              \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_append_any_##suffix(Kv8WriteArgs a) {     \
    kv8_write_any<T, false>(a);                                                                   \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_rope_d64_##suffix(Kv8WriteArgs a) {       \
    kv8_write<T, 64, 64, true>(a);                                                                \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_rope_d128_##suffix(Kv8WriteArgs a) {      \
    kv8_write<T, 128, 64, true>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64) kv8_rope_few_d64_##suffix(Kv8WriteArgs a) {    \
    kv8_write<T, 64, 16, true>(a);                                                                \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(64) kv8_rope_few_d128_##suffix(Kv8WriteArgs a) {   \
    kv8_write<T, 128, 16, true>(a);                                                               \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_rope_any_##suffix(Kv8WriteArgs a) {       \
    kv8_write_any<T, true>(a);                                                                    \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_read_d64_##suffix(Kv8ReadArgs a) {        \
    kv8_read_tile<T, 64, 64>(a);                                                                  \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_read_d128_##suffix(Kv8ReadArgs a) {       \
    kv8_read_tile<T, 128, 64>(a);                                                                 \
  }                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kv8_read_any_##suffix(Kv8ReadArgs a) {        \
    kv8_read_any<T>(a);                                                                           \
  }

KV8_KERNELS(f32, float)
KV8_KERNELS(bf16, bf16)
KV8_KERNELS(f16, f16)
