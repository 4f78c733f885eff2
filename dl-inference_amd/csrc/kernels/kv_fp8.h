#pragma once

// The 8-bit paged KV cache on gfx950: e4m3 elements, and per token and KV head one power-of-two
// scale for the key and one for the value.
#include "kv_fp8_args.h"
#include "mx.h"

namespace dk {

// Scale code of a row: the least c with largest / 2^(c - 127) <= 448, at least 0; 255 where the
// row holds an infinity or a NaN. `most`: bits of the largest magnitude (mxMax). Unlike the
// microscaled blocks' rule nothing saturates: a cached row is read by every later token, and an
// element's error stays within the half step of its format, 2^-4 of its value.
__device__ __forceinline__ uint32_t kv8Scale(uint32_t most) {
  const int e = static_cast<int>(most >> 23);
  const int c = e - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e == 255 ? 255u : static_cast<uint32_t>(c > 0 ? c : 0);
}

// Position of sequence b's first token. Cut to +-2^40, past any page and any number of tokens, so that
// sums with it stay in range.
__device__ __forceinline__ int64_t kv8First(const Kv8Pages& p, int64_t b) {
  constexpr int64_t kFar = int64_t{1} << 40;
  const int64_t at = p.positions != nullptr ? loadIndex(p.positions, p.pos64, b) : p.start;
  return at < -kFar ? -kFar : (at > kFar ? kFar : at);
}

// Page of position pos (0 <= pos < capacity) of sequence b, or -1: it holds nothing.
__device__ __forceinline__ int64_t kv8Page(const Kv8Pages& p, int64_t b, int64_t pos) {
  const int64_t id = gp(p.table)[b * p.max_blocks + pos / p.block_size];
  return id >= 0 && id < p.num_blocks ? id : -1;
}

}  // namespace dk
