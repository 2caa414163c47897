// Rows into the 4-bit paged cache (quantizing write) and back out of it (gfx950).
// Layout and quantizer: pa_int4.hpp.
//
// Work.  A row (token, kv head) is GL lanes of 8 or 16 dims, a wave 64 / GL consecutive
// tokens of one head, K and V; neighbouring waves take the heads of the same tokens,
// whose rows are neighbours in the input.  A code store puts the 4 bytes of 8 dims into
// their token's place of a quad: 4 consecutive tokens of 16-lane rows fill 256 consecutive
// bytes by one instruction.  The work-groups are dealt so that each XCD has
// consecutive ones, whose parts of a line of codes or scales then meet in one L2 (read-back of
// 16 prefixes, 60 k rows of 8 heads: 51 -> 46 us).
//
// What bounds it: HBM, and for the write the vector ALU beside it.  MI355X, head_dim 128, 8
// heads: read-back of 16 ragged prefixes (312 MB) 44 us, 7.1 TB/s, with non-temporal
// stores (73 us without); write of 48 ragged bf16 prompts (247 MB) 48 us, 5.1 TB/s.  The
// write began at 70 us: exact codes for every element, minimum and maximum in fp32, a
// scan for infinities.  Fast codes with a check (below) took it to 53, the ordered-integer
// reduction and 16 dims a lane, which halve the row's work on scale and minimum, to 48.  Two
// steps of rows a wave were 2-4% slower than one.
#include "pa_int4.hpp"

namespace pa {

constexpr int kRowsThreads = 256;
constexpr int64_t kManyRows = 16384;   // 2 to 4 waves a SIMD

// fp16 and bf16 bit patterns as 16-bit integers in the numbers' order, two at a time (and
// back: the map is its own inverse): the bits below a set sign are turned over.
typedef short s2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ s2_t ordered(s2_t v) { return v ^ ((v >> 15) & (short)0x7FFF); }

// Min over the GL lanes of a row, of both halves.
template <int GL>
__device__ __forceinline__ s2_t row_min(s2_t v) {
  auto step = [&](uint32_t w) { v = __builtin_elementwise_min(v, __builtin_bit_cast(s2_t, w)); };
  auto bits = [&] { return __builtin_bit_cast(uint32_t, v); };
  if constexpr (GL >= 2) step(dpp_mov_u<kQuadXor1>(bits()));
  if constexpr (GL >= 4) step(dpp_mov_u<kQuadXor2>(bits()));
  if constexpr (GL >= 8) step(dpp_mov_u<kRowHalfMirror>(bits()));
  if constexpr (GL >= 16) step(dpp_mov_u<kRowMirror>(bits()));
  if constexpr (GL >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(bits(), bits(), false, false);
    v = __builtin_elementwise_min(__builtin_bit_cast(s2_t, (uint32_t)r[0]),
                                  __builtin_bit_cast(s2_t, (uint32_t)r[1]));
  }
  return v;
}

// A store of rows that this kernel does not read again.
__device__ __forceinline__ void store_stream(void* p, uint4 v) {
  typedef uint32_t v4_t __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(__builtin_bit_cast(v4_t, v), reinterpret_cast<v4_t*>(p));
}
// Work-groups go round the 8 XCDs in turn: consecutive items for each XCD, so that the parts of
// a cache line that different waves write meet in one L2.
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int q = n >> 3, r = n & 7, x = b & 7;
  return x * q + min(x, r) + (b >> 3);
}
struct RowsArgs {
  const int64_t* slots;
  int num_tokens, num_kv_heads, chunks, num_blocks, bs_log2, grid, groups;  // groups: of tokens
  int64_t kts, khs, vts, vhs;   // row strides in elements
};

// Where a slot's row of head h lies: bytes from the codes' base to its first word, words from
// the scales'.  (Blocks times heads fit 32 bits: the host has checked.)
struct Cell {
  uint64_t codes, scales;
  bool ok;
};
__device__ __forceinline__ Cell locate(const RowsArgs& a, int64_t slot, int h) {
  Cell c;
  const uint64_t blk = (uint64_t)slot >> a.bs_log2;
  c.ok = blk < (uint64_t)a.num_blocks;             // (also no for a negative slot)
  const int off = (int)slot & ((1 << a.bs_log2) - 1);
  const uint32_t bh = (uint32_t)blk * (uint32_t)a.num_kv_heads + (uint32_t)h;
  const uint32_t tile = (uint32_t)(a.chunks * 4) << a.bs_log2;   // bytes of a (block, head)
  c.codes = (uint64_t)bh * tile + (uint32_t)(quad_offset(off, a.chunks) + (off & 3) * 4);
  c.scales = ((uint64_t)bh << a.bs_log2) + (uint32_t)off;
  return c;
}

// Exact codes of d = x - m against s > 0: of the two nearest codes k, k + 1 that an
// approximate quotient gives, the nearer, decided on d against (k + 1/2) s, whose product is
// exact (15 bits); a value on the border goes to the even one, as by an exact division.
__device__ __forceinline__ uint32_t exact_code(float d, float r, float s) {
  const float k = fminf(fmaxf(floorf(d * r), 0.f), 15.f);
  const float t = (k + 0.5f) * s;
  const uint32_t kc = (uint32_t)k;
  const uint32_t c = kc + ((d > t || (d == t && (kc & 1u))) ? 1u : 0u);
  return c > 15u ? 15u : c;
}

constexpr float kRoundMagic = 12582912.f;   // 1.5 * 2^23: y + magic holds rne(y) in its low bits
// The fast codes are rne(d r), r the hardware reciprocal of s (within 1 ulp): off the exact
// quotient, at most 15.01, by less than 15.01 * 2^-22.9 < 2e-6.  A product farther than that
// from every border of two codes rounds as the exact quotient does.
constexpr float kBorder = 0.5f - 4e-6f;

// A row's 8 EL dims per lane, quantized: a word of codes for each 8; (s, m) packed in `sm`,
// the same in all lanes of the row.  (Lanes past the row's end repeat its last 8.)
template <bool BF, int GL, int EL>
__device__ __forceinline__ void quantize_row(const uint4 (&w)[EL], uint32_t (&code)[EL],
                                             uint32_t& sm) {
  // (minimum, complement of the maximum) as ordered integers: one reduction for both
  s2_t mn, mx;
#pragma unroll
  for (int j = 0; j < EL; ++j) {
    const uint32_t wv[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const s2_t k = ordered(__builtin_bit_cast(s2_t, wv[i]));
      mn = i + j == 0 ? k : __builtin_elementwise_min(mn, k);
      mx = i + j == 0 ? k : __builtin_elementwise_max(mx, k);
    }
  }
  const uint32_t a = __builtin_bit_cast(uint32_t, mn), b = ~__builtin_bit_cast(uint32_t, mx);
  const s2_t both = row_min<GL>(__builtin_elementwise_min(
      __builtin_bit_cast(s2_t, __builtin_amdgcn_perm(b, a, 0x05040100u)),
      __builtin_bit_cast(s2_t, __builtin_amdgcn_perm(b, a, 0x07060302u))));
  const uint32_t key = __builtin_bit_cast(uint32_t, both) ^ 0xFFFF0000u;
  const s2_t kk = __builtin_bit_cast(s2_t, key);
  constexpr short kInf = BF ? 0x7F80 : 0x7C00;      // infinities and NaN lie outside these
  const bool bad = kk.y >= kInf || kk.x <= (short)~kInf;
  const uint32_t ext = __builtin_bit_cast(uint32_t, ordered(kk));
  const float lo = widen_lo<BF>(ext), hi = widen_hi<BF>(ext);
  const half_t mh = (half_t)__builtin_amdgcn_fmed3f(lo, -65504.f, 65504.f);
  // fl((hi - lo) / 15): a product, then one step on its exact remainder.  (Where that is
  // subnormal, s is 0 all the same; an infinite range gives a NaN here and 65504 by the min.)
  const float range = hi - lo, q0 = range * (1.f / 15.f);
  const float q1 = __builtin_fmaf(__builtin_fmaf(-15.f, q0, range), 1.f / 15.f, q0);
  const half_t sh = (half_t)fminf(q1, 65504.f);
  const float m = (float)mh, s = (float)sh;
  const half2_t pair = {sh, mh};
  sm = bad ? 0x7E007E00u : __builtin_bit_cast(uint32_t, pair);
  const float r = __builtin_amdgcn_rcpf(s);
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < EL; ++j) {
    const uint32_t wv[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float d0 = widen_lo<BF>(wv[i]) - m, d1 = widen_hi<BF>(wv[i]) - m;
      const float y0 = __builtin_fmaf(d0, r, kRoundMagic), y1 = __builtin_fmaf(d1, r, kRoundMagic);
      off = __builtin_fmaxf(off, __builtin_fmaxf(fabsf(__builtin_fmaf(d0, r, -(y0 - kRoundMagic))),
                                                 fabsf(__builtin_fmaf(d1, r, -(y1 - kRoundMagic)))));
      p[i] = (fbits(y1) << 4) | fbits(y0);            // (the low byte counts)
    }
    code[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(p[3], p[2], 0x0c0c0400u),
                                    __builtin_amdgcn_perm(p[1], p[0], 0x0c0c0400u), 0x05040100u);
  }
  // Subnormal and saturated numbers, whose quotients may leave 0..15, take the exact codes too.
  const bool fast = off < kBorder && s >= 0x1p-14f && s < 65504.f && fabsf(m) < 65504.f;
  if (__any(!fast)) {
#pragma unroll
    for (int j = 0; j < EL; ++j) {
      const uint32_t wv[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
      code[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float d = ((i & 1) ? widen_hi<BF>(wv[i >> 1]) : widen_lo<BF>(wv[i >> 1])) - m;
        asm volatile("" : "+v"(d));   // (a branch to skip, not work to do beforehand)
        code[j] |= exact_code(d, r, s) << (4 * i);
      }
    }
  }
  const bool some = s > 0.f && !bad;
#pragma unroll
  for (int j = 0; j < EL; ++j) code[j] = some ? code[j] : 0u;
}

template <bool BF, int GL, int EL>
__global__ void __launch_bounds__(kRowsThreads)
int4_write_kernel(const uint16_t* __restrict__ key, const uint16_t* __restrict__ value,
                  uint8_t* __restrict__ kc, uint8_t* __restrict__ vc, uint32_t* __restrict__ ks,
                  uint32_t* __restrict__ vs, RowsArgs a) {
  constexpr int RW = kWave / GL;           // rows of a wave
  const int wave = xcd_order(blockIdx.x, a.grid) * (kRowsThreads / kWave) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & (kWave - 1);
  const int g = wave / a.num_kv_heads, h = wave - g * a.num_kv_heads;
  if (g >= a.groups) return;
  const int first = lane % GL, t = g * RW + lane / GL;
  const int t_in = min(t, a.num_tokens - 1);
  const uint16_t* kp = key + t_in * a.kts + h * a.khs;
  const uint16_t* vp = value + t_in * a.vts + h * a.vhs;
  const int64_t slot = t < a.num_tokens ? a.slots[t] : -1;
  uint4 kx[EL], vx[EL];
#pragma unroll
  for (int j = 0; j < EL; ++j) {
    const int c = min(first + j * GL, a.chunks - 1) * 8;
    kx[j] = load_stream<uint4>(kp + c);
    vx[j] = load_stream<uint4>(vp + c);
  }
  uint32_t ksm, vsm, kcode[EL], vcode[EL];
  quantize_row<BF, GL, EL>(kx, kcode, ksm);
  quantize_row<BF, GL, EL>(vx, vcode, vsm);
  const Cell c = locate(a, slot, h);
  if (!c.ok) return;
#pragma unroll
  for (int j = 0; j < EL; ++j) {
    const int chunk = first + j * GL;
    if (chunk < a.chunks) {
      *reinterpret_cast<uint32_t*>(kc + c.codes + chunk * 16) = kcode[j];
      *reinterpret_cast<uint32_t*>(vc + c.codes + chunk * 16) = vcode[j];
    }
  }
  if (first == 0) {
    ks[c.scales] = ksm;
    vs[c.scales] = vsm;
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

template <bool BF, int GL>
__global__ void __launch_bounds__(kRowsThreads)
int4_gather_kernel(uint16_t* __restrict__ key, uint16_t* __restrict__ value,
                   const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                   const uint32_t* __restrict__ ks, const uint32_t* __restrict__ vs, RowsArgs a) {
  constexpr int RW = kWave / GL;
  const int wave = xcd_order(blockIdx.x, a.grid) * (kRowsThreads / kWave) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & (kWave - 1);
  const int g = wave / a.num_kv_heads, h = wave - g * a.num_kv_heads;
  const int chunk = lane % GL, t = g * RW + lane / GL;
  if (g >= a.groups || chunk >= a.chunks || t >= a.num_tokens) return;
  const Cell c = locate(a, a.slots[t], h);
  uint32_t kw = 0, vw = 0, ksm = 0, vsm = 0;      // a slot outside the pool: zeros
  if (c.ok) {
    kw = *reinterpret_cast<const uint32_t*>(kc + c.codes + chunk * 16);
    vw = *reinterpret_cast<const uint32_t*>(vc + c.codes + chunk * 16);
    ksm = ks[c.scales];
    vsm = vs[c.scales];
  }
  store_stream(key + t * a.kts + h * a.khs + chunk * 8,
               dequantize8<BF>(kw, widen_lo<false>(ksm), widen_hi<false>(ksm)));
  store_stream(value + t * a.vts + h * a.vhs + chunk * 8,
               dequantize8<BF>(vw, widen_lo<false>(vsm), widen_hi<false>(vsm)));
}

namespace {

template <bool WRITE, bool BF, int GL, int EL>
hipError_t launch_rows(const Int4Rows& l) {
  constexpr int per_wave = kWave / GL;
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
  if (waves > INT32_MAX - kRowsThreads) return hipErrorInvalidValue;
  a.grid = (int)grid;
  if constexpr (WRITE)
    int4_write_kernel<BF, GL, EL><<<(unsigned)grid, kRowsThreads, 0, l.stream>>>(
        static_cast<const uint16_t*>(l.key), static_cast<const uint16_t*>(l.value),
        static_cast<uint8_t*>(l.k_cache), static_cast<uint8_t*>(l.v_cache),
        static_cast<uint32_t*>(l.k_scales), static_cast<uint32_t*>(l.v_scales), a);
  else
    int4_gather_kernel<BF, GL><<<(unsigned)grid, kRowsThreads, 0, l.stream>>>(
        static_cast<uint16_t*>(l.key), static_cast<uint16_t*>(l.value),
        static_cast<const uint8_t*>(l.k_cache), static_cast<const uint8_t*>(l.v_cache),
        static_cast<const uint32_t*>(l.k_scales), static_cast<const uint32_t*>(l.v_scales), a);
  return hipGetLastError();
}

// Lanes of a row: the next power of two of its 8-dim groups.  The write of many rows gives a
// lane two of the groups of heads wider than 64; few rows, where latency is all, keep
// one (256 appended tokens of 8 heads 3.8 us against 4.6; 48 prompts 49.7 against 48.2).
template <bool WRITE, bool BF>
hipError_t launch_rows_of(const Int4Rows& l) {
  const int chunks = l.head_dim / 8;
  const bool many = WRITE && (int64_t)l.num_tokens * l.num_kv_heads >= kManyRows;
  if (chunks <= 4) return launch_rows<WRITE, BF, 4, 1>(l);
  if (chunks <= 8) return launch_rows<WRITE, BF, 8, 1>(l);
  if (chunks <= 16)
    return many ? launch_rows<WRITE, BF, 8, 2>(l) : launch_rows<WRITE, BF, 16, 1>(l);
  return many ? launch_rows<WRITE, BF, 16, 2>(l) : launch_rows<WRITE, BF, 32, 1>(l);
}

}  // namespace

hipError_t launch_int4_write(const Int4Rows& l) {
  return l.bf16 ? launch_rows_of<true, true>(l) : launch_rows_of<true, false>(l);
}
hipError_t launch_int4_gather(const Int4Rows& l) {
  return l.bf16 ? launch_rows_of<false, true>(l) : launch_rows_of<false, false>(l);
}

}  // namespace pa
