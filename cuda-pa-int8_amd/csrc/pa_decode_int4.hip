// Decode attention over the 4-bit paged cache (gfx950).  Layout: pa_int4.hpp.
//
//   out[h] = sum_t p_t (s_t c_t + m_t) / sum_t p_t,
//   p_t = exp(scale * (s'_t (q . c'_t) + m'_t sum(q)))     (primed: K's codes, scale and minimum)
//
// One wave per (sequence, query head): 64 tokens at a time, a lane to a token for the
// scores, a lane to dims for the weighted sum, the running maximum and sum in fp32.
#include "pa_int4.hpp"

namespace pa {

template <bool BF>
__global__ void __launch_bounds__(kWave)
decode_int4_kernel(uint16_t* __restrict__ out, const uint16_t* __restrict__ q,
                   const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                   const half2_t* __restrict__ ks, const half2_t* __restrict__ vs,
                   const int32_t* __restrict__ bt, const int32_t* __restrict__ ctxl,
                   Int4DecodeShape sh) {
  __shared__ float qs[256];
  __shared__ float ps[kWave], pm[kWave];
  __shared__ int blk_of[kWave];
  const int lane = threadIdx.x;
  const int seq = blockIdx.x / sh.num_heads, head = blockIdx.x - seq * sh.num_heads;
  const int kvh = head / sh.group, D = sh.head_dim, chunks = D / 8, bs = 1 << sh.bs_log2;
  const uint16_t* qr = q + ((size_t)seq * sh.num_heads + head) * D;
  float qsum = 0.f;
  for (int d = lane; d < D; d += kWave) {
    const float v = widen_lo<BF>((uint32_t)qr[d]);
    qs[d] = v;
    qsum += v;
  }
  qsum = wave_sum(qsum);
  __syncthreads();
  const int cap = sh.max_blocks * bs;
  int ctx = ctxl[seq];
  ctx = ctx < 0 ? 0 : (ctx > cap ? cap : ctx);
  const size_t tile = (size_t)chunks * 4 * bs;
  float M = -INFINITY, L = 0.f, bias = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < ctx; t0 += kWave) {
    const int t = t0 + lane;
    int blk = t < ctx ? bt[(size_t)seq * sh.max_blocks + (t >> sh.bs_log2)] : -1;
    if (blk >= sh.num_blocks) blk = -1;
    const int off = t & (bs - 1);
    float score = -INFINITY, s = 0.f, m = 0.f;
    if (blk >= 0) {
      const size_t bh = (size_t)blk * sh.num_kv_heads + kvh;
      const uint8_t* row = kc + bh * tile + quad_offset(off, chunks) + (off & 3) * 4;
      float dot = 0.f;
      for (int c = 0; c < chunks; ++c) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(row + c * 16);
        for (int e = 0; e < 8; ++e) dot += qs[8 * c + e] * (float)((w >> (4 * e)) & 15u);
      }
      const half2_t ksm = ks[(bh << sh.bs_log2) + off], vsm = vs[(bh << sh.bs_log2) + off];
      score = ((float)ksm.x * dot + (float)ksm.y * qsum) * sh.scale_log2;
      s = (float)vsm.x;
      m = (float)vsm.y;
    }
    const float mx = fmaxf(M, wave_max(score));
    const float f = M == -INFINITY ? 0.f : exp2f(M - mx);
    const float p = blk >= 0 ? exp2f(score - mx) : 0.f;
    L = L * f + wave_sum(p);
    bias = bias * f + wave_sum(p * m);
    M = mx == -INFINITY ? M : mx;
    __syncthreads();
    ps[lane] = p * s;
    blk_of[lane] = blk;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + i * kWave;
      acc[i] *= f;
      if (d < D)
        for (int j = 0; j < kWave; ++j) {
          if (blk_of[j] < 0) continue;
          const int o = (t0 + j) & (bs - 1);
          const size_t bh = (size_t)blk_of[j] * sh.num_kv_heads + kvh;
          const uint8_t byte = vc[bh * tile + quad_offset(o, chunks) + (d >> 3) * 16 + (o & 3) * 4 +
                                  ((d & 7) >> 1)];
          acc[i] += ps[j] * (float)((byte >> (4 * (d & 1))) & 15u);
        }
    }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  for (int i = 0; i < 4; ++i) {
    const int d = lane + i * kWave;
    if (d < D)
      out[((size_t)seq * sh.num_heads + head) * D + d] =
          (uint16_t)pack2<BF>((acc[i] + bias) * inv, 0.f);
  }
}

hipError_t launch_int4_decode(const Int4Decode& l) {
  const unsigned grid = (unsigned)(l.shape.num_seqs * l.shape.num_heads);
  auto* k = l.bf16 ? decode_int4_kernel<true> : decode_int4_kernel<false>;
  k<<<grid, kWave, 0, l.stream>>>(
      static_cast<uint16_t*>(l.out), static_cast<const uint16_t*>(l.q),
      static_cast<const uint8_t*>(l.k_cache), static_cast<const uint8_t*>(l.v_cache),
      static_cast<const half2_t*>(l.k_scales), static_cast<const half2_t*>(l.v_scales),
      l.block_table, l.context_lens, l.shape);
  return hipGetLastError();
}

size_t int4_decode_workspace_bytes(const Int4DecodeShape&) { return 0; }
size_t int4_decode_counter_bytes() { return 256; }

}  // namespace pa
