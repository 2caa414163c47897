// The 4-bit paged KV cache (gfx950): its layout, and the conversions its kernels share.
//
// A row x[D] of one (token, kv head), K and V alike, is held as codes c[D] in 0..15 and a
// pair of fp16 numbers, its scale s and minimum m, that stand for the values s * c + m:
//   m   = fp16(min x)                   (saturated at +-65504)
//   s   = fp16((max x - min x) / 15)    (saturated at 65504)
//   c_d = clamp(rne((x_d - m) / s), 0, 15), 0 where s = 0.
// A row that holds an infinity or a NaN gets s = m = NaN and codes 0: it reads back as NaN.
//
// Layout, K and V alike:
//   codes   uint8 [num_blocks, num_kv_heads, block_size / 4, head_dim / 8, 4, 4]
//   scales  fp16  [num_blocks, num_kv_heads, block_size, 2]   (scale, minimum)
// The innermost 4 bytes are 8 consecutive dims of one token, dim e in bits 4e..4e+3; 4
// consecutive tokens (a quad) of the same 8 dims are 16 consecutive bytes.  A lane of the
// decode kernel takes one such 16-byte cell by one load: 4 tokens of a K row group (4
// matrix instructions' rows), or 4 tokens of the 8 dims of V that the lane's output rows
// are, so neither product needs a transpose across lanes, and a new token is written
// without reading what its neighbours hold.
#pragma once

#include "pa_device.hpp"
#include "pa_internal.hpp"

namespace pa {

// Byte offset of the quad that holds token `off` of a block, from the (block, head)'s first byte.
__device__ __forceinline__ int quad_offset(int off, int chunks) { return (off >> 2) * chunks * 16; }

// The two 16-bit elements of a word, widened to fp32 (exactly).
template <bool BF>
__device__ __forceinline__ float widen_lo(uint32_t w) {
  if constexpr (BF) return bitsf(w << 16);
  else return (float)__builtin_bit_cast(half2_t, w).x;
}
template <bool BF>
__device__ __forceinline__ float widen_hi(uint32_t w) {
  if constexpr (BF) return bitsf(w & 0xFFFF0000u);
  else return (float)__builtin_bit_cast(half2_t, w).y;
}

// Two fp32 values rounded (to nearest even) to a packed pair.
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (BF) {
    const bf2_t v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return pack_h2(a, b);
  }
}

}  // namespace pa
