// Rows into the 4-bit paged cache (quantizing write) and back out of it (gfx950).
// Layout and quantizer: pa_int4.hpp.
//
// Work.  A row (token, kv head) is GL lanes of 8 dims; a wave holds 64 / GL rows and
// walks ITERS groups of consecutive tokens of one head, K and V.  All loads of a wave go
// out before the first is used.  Neighbouring waves take the heads of the same tokens,
// whose rows are neighbours in the input.  A code store puts the 4 bytes of 8 dims into
// their token's place of a quad: 4 consecutive tokens at head_dim 128 fill 256
// consecutive bytes with one instruction.
#include "pa_int4.hpp"

namespace pa {

constexpr int kRowsThreads = 256;

template <class Op, int GL>
__device__ __forceinline__ float row_reduce(float v, Op op) {
  if constexpr (GL >= 2) v = op(v, dpp_mov<kQuadXor1>(v));
  if constexpr (GL >= 4) v = op(v, dpp_mov<kQuadXor2>(v));
  if constexpr (GL >= 8) v = op(v, dpp_mov<kRowHalfMirror>(v));
  if constexpr (GL >= 16) v = op(v, dpp_mov<kRowMirror>(v));
  if constexpr (GL >= 32) v = cross_row16(v, op);
  return v;
}
struct OpMin {
  __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); }
};

struct RowsArgs {
  const int64_t* slots;
  int num_tokens, num_kv_heads, chunks, num_blocks, bs_log2, groups;  // groups: of tokens
  int64_t kts, khs, vts, vhs;   // row strides in elements
};

// One row's 8 dims per lane, quantized: the word of codes; (s, m) packed in `sm`, the same
// in all lanes of the row.  `live`: the lane holds dims of the row.
template <bool BF, int GL>
__device__ __forceinline__ uint32_t quantize_row(uint4 w, bool live, uint32_t& sm) {
  const uint32_t wv[4] = {w.x, w.y, w.z, w.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = widen_lo<BF>(wv[i]);
    x[2 * i + 1] = widen_hi<BF>(wv[i]);
  }
  float lo = INFINITY, hi = -INFINITY, bad = 0.f;
  if (live) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
      bad = __builtin_fmaf(x[i], 0.f, bad);   // NaN from an infinity or a NaN
    }
  }
  bad = bad != bad ? 1.f : 0.f;
  lo = row_reduce<OpMin, GL>(lo, OpMin());
  hi = row_reduce<OpMax, GL>(hi, OpMax());
  bad = row_reduce<OpMax, GL>(bad, OpMax());
  const half_t mh = (half_t)fminf(fmaxf(lo, -65504.f), 65504.f);
  const half_t sh = (half_t)fminf((hi - lo) / 15.f, 65504.f);
  const float m = (float)mh, s = (float)sh;
  const half2_t pair = {sh, mh};
  sm = bad != 0.f ? 0x7E007E00u : __builtin_bit_cast(uint32_t, pair);
  // The quotient's two nearest codes k, k + 1 come from a reciprocal; which of them is
  // nearer is decided on x - m against (k + 1/2) s, whose product is exact (15 bits), so a
  // value on the border of two codes goes to the even one as by an exact division.
  const float r = 1.f / s;
  uint32_t c8 = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - m;
    const float k = fminf(fmaxf(floorf(d * r), 0.f), 15.f);
    const float t = (k + 0.5f) * s;
    const uint32_t kc = (uint32_t)k;
    uint32_t c = kc + ((d > t || (d == t && (kc & 1u))) ? 1u : 0u);
    c = c > 15u ? 15u : c;
    c8 |= c << (4 * i);
  }
  return (s > 0.f && bad == 0.f) ? c8 : 0u;
}

template <bool BF, int GL, int ITERS>
__global__ void __launch_bounds__(kRowsThreads)
int4_write_kernel(const uint16_t* __restrict__ key, const uint16_t* __restrict__ value,
                  uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, uint32_t* __restrict__ ks,
                  uint32_t* __restrict__ vs, RowsArgs a) {
  constexpr int RW = kWave / GL;           // rows of one step
  const int wave = blockIdx.x * (kRowsThreads / kWave) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & (kWave - 1);
  const int g = wave / a.num_kv_heads, h = wave - g * a.num_kv_heads;
  if (g >= a.groups) return;
  const int chunk = lane % GL, row = lane / GL;
  const bool live = chunk < a.chunks;
  const int ch = live ? chunk : 0;
  const int t0 = g * (RW * ITERS);
  uint4 kx[ITERS], vx[ITERS];
  int64_t slot[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    int t = t0 + i * RW + row;
    const bool in = t < a.num_tokens;
    t = in ? t : a.num_tokens - 1;
    slot[i] = a.slots[t];
    if (!in) slot[i] = -1;
    kx[i] = *reinterpret_cast<const uint4*>(key + t * a.kts + h * a.khs + ch * 8);
    vx[i] = *reinterpret_cast<const uint4*>(value + t * a.vts + h * a.vhs + ch * 8);
  }
  const int64_t pool = (int64_t)a.num_blocks << a.bs_log2;
  const size_t tile = (size_t)a.chunks * 4 << a.bs_log2;   // bytes of a (block, head)
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    uint32_t ksm, vsm;
    const uint32_t kcode = quantize_row<BF, GL>(kx[i], live, ksm);
    const uint32_t vcode = quantize_row<BF, GL>(vx[i], live, vsm);
    if (slot[i] < 0 || slot[i] >= pool) continue;
    const int64_t blk = slot[i] >> a.bs_log2;
    const int off = (int)(slot[i] & ((1 << a.bs_log2) - 1));
    const size_t bh = (size_t)blk * a.num_kv_heads + h;
    const size_t at = bh * tile + quad_offset(off, a.chunks) + chunk * 16 + (off & 3) * 4;
    if (live) {
      *reinterpret_cast<uint32_t*>(kc + at) = kcode;
      *reinterpret_cast<uint32_t*>(vc + at) = vcode;
    }
    if (chunk == 0) {
      ks[(bh << a.bs_log2) + off] = ksm;
      vs[(bh << a.bs_log2) + off] = vsm;
    }
  }
}

template <bool BF>
__device__ __forceinline__ uint4 dequantize8(uint32_t c, float s, float m) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (s * c is exact in fp32: one rounding to fp32 in the sum, one to the output type)
    const float a = __builtin_fmaf((float)((c >> (8 * i)) & 15u), s, m);
    const float b = __builtin_fmaf((float)((c >> (8 * i + 4)) & 15u), s, m);
    w[i] = pack2<BF>(a, b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool BF, int GL, int ITERS>
__global__ void __launch_bounds__(kRowsThreads)
int4_gather_kernel(uint16_t* __restrict__ key, uint16_t* __restrict__ value,
                   const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                   const uint32_t* __restrict__ ks, const uint32_t* __restrict__ vs, RowsArgs a) {
  constexpr int RW = kWave / GL;
  const int wave = blockIdx.x * (kRowsThreads / kWave) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & (kWave - 1);
  const int g = wave / a.num_kv_heads, h = wave - g * a.num_kv_heads;
  if (g >= a.groups) return;
  const int chunk = lane % GL, row = lane / GL;
  const bool live = chunk < a.chunks;
  const int ch = live ? chunk : 0;
  const int t0 = g * (RW * ITERS);
  const int64_t pool = (int64_t)a.num_blocks << a.bs_log2;
  const size_t tile = (size_t)a.chunks * 4 << a.bs_log2;
  int64_t slot[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) slot[i] = a.slots[min(t0 + i * RW + row, a.num_tokens - 1)];
  uint32_t kw[ITERS], vw[ITERS], ksm[ITERS], vsm[ITERS];
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    kw[i] = vw[i] = ksm[i] = vsm[i] = 0;      // a slot outside the pool: zeros
    if (slot[i] >= 0 && slot[i] < pool) {
      const int off = (int)(slot[i] & ((1 << a.bs_log2) - 1));
      const size_t bh = (size_t)(slot[i] >> a.bs_log2) * a.num_kv_heads + h;
      const size_t at = bh * tile + quad_offset(off, a.chunks) + ch * 16 + (off & 3) * 4;
      kw[i] = *reinterpret_cast<const uint32_t*>(kc + at);
      vw[i] = *reinterpret_cast<const uint32_t*>(vc + at);
      ksm[i] = ks[(bh << a.bs_log2) + off];
      vsm[i] = vs[(bh << a.bs_log2) + off];
    }
  }
#pragma unroll
  for (int i = 0; i < ITERS; ++i) {
    const int t = t0 + i * RW + row;
    if (t >= a.num_tokens || !live) continue;
    *reinterpret_cast<uint4*>(key + t * a.kts + h * a.khs + chunk * 8) =
        dequantize8<BF>(kw[i], widen_lo<false>(ksm[i]), widen_hi<false>(ksm[i]));
    *reinterpret_cast<uint4*>(value + t * a.vts + h * a.vhs + chunk * 8) =
        dequantize8<BF>(vw[i], widen_lo<false>(vsm[i]), widen_hi<false>(vsm[i]));
  }
}

namespace {

template <bool WRITE, bool BF, int GL, int ITERS>
hipError_t launch_rows_iters(const Int4Rows& l) {
  constexpr int per_wave = kWave / GL * ITERS;
  RowsArgs a;
  a.slots = l.slot_mapping;
  a.num_tokens = l.num_tokens;
  a.num_kv_heads = l.num_kv_heads;
  a.chunks = l.head_dim / 8;
  a.num_blocks = l.num_blocks;
  a.bs_log2 = __builtin_ctz((unsigned)l.block_size);
  a.groups = (l.num_tokens + per_wave - 1) / per_wave;
  a.kts = l.key_token_stride;
  a.khs = l.key_head_stride;
  a.vts = l.value_token_stride;
  a.vhs = l.value_head_stride;
  const int64_t waves = (int64_t)a.groups * l.num_kv_heads;
  const int64_t grid = (waves + kRowsThreads / kWave - 1) / (kRowsThreads / kWave);
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  if constexpr (WRITE)
    int4_write_kernel<BF, GL, ITERS><<<(unsigned)grid, kRowsThreads, 0, l.stream>>>(
        static_cast<const uint16_t*>(l.key), static_cast<const uint16_t*>(l.value),
        static_cast<uint8_t*>(l.k_cache), static_cast<uint8_t*>(l.v_cache),
        static_cast<uint32_t*>(l.k_scales), static_cast<uint32_t*>(l.v_scales), a);
  else
    int4_gather_kernel<BF, GL, ITERS><<<(unsigned)grid, kRowsThreads, 0, l.stream>>>(
        static_cast<uint16_t*>(l.key), static_cast<uint16_t*>(l.value),
        static_cast<const uint8_t*>(l.k_cache), static_cast<const uint8_t*>(l.v_cache),
        static_cast<const uint32_t*>(l.k_scales), static_cast<const uint32_t*>(l.v_scales), a);
  return hipGetLastError();
}

template <bool WRITE, bool BF>
hipError_t launch_rows(const Int4Rows& l) {
  const int chunks = l.head_dim / 8;
  if (chunks <= 4) return launch_rows_iters<WRITE, BF, 4, 1>(l);
  if (chunks <= 8) return launch_rows_iters<WRITE, BF, 8, 2>(l);
  if (chunks <= 16) return launch_rows_iters<WRITE, BF, 16, 4>(l);
  return launch_rows_iters<WRITE, BF, 32, 4>(l);
}

}  // namespace

hipError_t launch_int4_write(const Int4Rows& l) {
  return l.bf16 ? launch_rows<true, true>(l) : launch_rows<true, false>(l);
}
hipError_t launch_int4_gather(const Int4Rows& l) {
  return l.bf16 ? launch_rows<false, true>(l) : launch_rows<false, false>(l);
}

}  // namespace pa
