// Decode attention over the 4-bit paged cache (gfx950).  Layout: pa_int4.hpp.
//
//   out[h] = sum_t p_t (s_t c_t + m_t) / sum_t p_t,
//   p_t = exp(scale (s'_t (q . c'_t) + m'_t sum(q)))      (primed: K's codes, scale and minimum)
//
// Both products are matrix instructions on the codes themselves (v_mfma_f32_16x16x32_f16); the
// scales and minima enter in fp32, at the scores and at the weights:
//   scores   S[token][head]  = C'[tokens][32 dims] x Q^T[dims][16 heads]
//   output   O^T[dim][head] += C^T[dims][32 tokens] x P^T[tokens][heads],  P = p s
// A code c sits in the low bits of an fp16 element, where it is the subnormal number
// c 2^-24, or 16 c 2^-24 from the upper half byte: masking is all the unpacking there is (5
// instructions for 8 codes of K, 6 of V), and the matrix core takes subnormal
// elements exactly.  The powers of two are put right in fp32, those of K in q (normalised
// per head to at most 2^15 so that none of its bits are lost).
//
// Lanes.  Lane l = (i = l & 15, g = l >> 4).  A tile is 64 tokens.  For K, lane (i, g) loads
// quad i (tokens 4i .. 4i+3) of 8 dims 8 (4 step + g) ..: matrix row i of instruction n is token
// 4i + n, and the scores of head h = i and tokens 16g + 4r + n come out in lane (h, g),
// register r.  For V, lane (i, g) loads tokens 16g .. 16g + 15 of the dims 8i .. 8i + 7:
// the weights that lane (h, g) holds are the operand as they are, no lane exchanges anything
// but the running maximum, and output row i of instruction n is dim 8i + n.
//
// Weights.  The reference point of the exponentials is the running maximum of score +
// log2(s), less kShift: the P = p s stay at or below 2^kShift whatever the rows' scales.  P
// enters as two fp16 numbers (its rounding and what that left), 22 bits together: with one
// the outputs' error would grow threefold, as the codes are not centred.  sum p and sum p m are
// fp32 sums of the unrounded weights.
//
// Work.  The tiles of all units (sequence, kv head, chunk of 16 HT query heads) form one list,
// in that order, and the N waves of the launch take the ranges [i W / N, (i + 1) W / N) of its W
// tiles: as even as tiles are, whatever the lengths, and found by every wave from
// context_lens alone.  A unit inside one wave's range needs no merge at all; the pieces of a
// unit that several waves share are merged through LDS, and those of a unit that several
// work-groups share through memory, by the last of them to arrive (in two levels above
// kMergeMax pieces).  All orders are fixed: the same bits every time.
#include <math.h>

#include "pa_decode_kernels.hpp"
#include "pa_int4.hpp"

namespace pa {

constexpr int kI4Waves = 8;          // waves of a work-group
constexpr int kI4Groups = kInt4Groups;   // work-groups of a launch, at most: one a CU
constexpr int kI4Tile = 64;          // tokens
constexpr int kI4MinTiles = 2;       // tiles of a wave before another work-group is used
constexpr int kMergeMax = 16;        // pieces merged at once
constexpr float kShift = 14.f;
constexpr float kCode24 = 16777216.f;   // 2^24: a code's element times this is the code

struct I4Args {
  const uint16_t* q;
  uint16_t* out;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint32_t* ks;
  const uint32_t* vs;
  const int32_t* bt;
  const int32_t* ctxl;
  float* ws;
  uint32_t* cnt;
  int nchunk;
  Int4DecodeShape sh;
};

// A tile of the list: unit `u` (kv head * chunks + chunk) of sequence `seq`, tile t of n.
struct I4Tile {
  int seq, u, t, n, ctx, ctx_next;
};

// float4s a lane keeps of a piece: [head tile][16-chunk tile][row r][half].
template <int STEPS, int HT>
struct I4Geo {
  static constexpr int T = (STEPS + 3) / 4;
  static constexpr int NF = 8 * T * HT;
  static constexpr int kPieceFloats = NF * kWave * 4;
  static constexpr int kMlFloats = 2 * 16 * HT;
  static constexpr size_t kSlotFloats = kPieceFloats + kMlFloats;
};

// The unit that a wave's first tile belongs to, where it was begun before the wave.
struct I4Unit {
  long long begin;   // its first tile in the list
  int n, seq, u;
};

template <int STEPS, int HT>
struct alignas(16) I4Smem {
  using G = I4Geo<STEPS, HT>;
  f4_t acc[kI4Waves][G::NF][kWave];
  f2_t ml[kI4Waves][16 * HT];
  I4Unit head[kI4Waves];
  int state[kI4Waves];
  // the pieces of units that other work-groups share: [0] begun earlier, [1] continued later
  struct {
    int active, first, count, seq, u, last;
  } piece[2];
  int last2;
};
constexpr int kHasTiles = 1, kHead = 2, kHeadEnds = 4, kTail = 8;

__device__ __forceinline__ int i4_clamp_ctx(int c, int cap) { return c < 0 ? 0 : (c > cap ? cap : c); }
__device__ __forceinline__ int i4_tiles(int ctx) { return ctx > 0 ? (ctx + kI4Tile - 1) / kI4Tile : 1; }

// 8 codes (a token's word) -> 8 fp16 elements in the order of dims 0 4 1 5 2 6 3 7; those of
// dims 1, 3, 5 and 7 are 16 times too large.
__device__ __forceinline__ h8_t codes_k(uint32_t w) {
  const uint32_t v = w >> 8;
  const u4_t d = {w & 0x000F000Fu, w & 0x00F000F0u, v & 0x000F000Fu, v & 0x00F000F0u};
  return __builtin_bit_cast(h8_t, d);
}

__device__ __forceinline__ f4_t dev_load4(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, kPolicyDevice));
}
__device__ __forceinline__ void dev_store4(__amdgpu_buffer_rsrc_t r, int off, f4_t v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v), r, off, 0, kPolicyDevice);
}

template <int STEPS, int HT, bool BF>
__global__ void __launch_bounds__(kI4Waves* kWave) __attribute__((amdgpu_waves_per_eu(2)))
decode_int4_kernel(I4Args a) {
  using G = I4Geo<STEPS, HT>;
  constexpr int T = G::T, NF = G::NF;
  __shared__ I4Smem<STEPS, HT> sm;
  const Int4DecodeShape& sh = a.sh;
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int S = sh.num_seqs, U = sh.num_kv_heads * a.nchunk, C = sh.head_dim / 8, D = sh.head_dim;
  const int bs = 1 << sh.bs_log2;
  const int cap = sh.max_blocks << sh.bs_log2;
  const size_t cell_bytes = (size_t)C * 4 << sh.bs_log2;   // bytes of a (block, head)

  // ---- the wave's range.  Lane l sums the tiles of sequences l per .. l per + per - 1.
  const int per = (S + kWave - 1) / kWave;
  long long mine = 0;
  for (int j = 0; j < per; ++j) {
    const int s = lane * per + j;
    if (s < S) mine += i4_tiles(i4_clamp_ctx(a.ctxl[s], cap));
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const long long y = __shfl_up(incl, o, kWave);
    if (lane >= o) incl += y;
  }
  const long long W = __shfl(incl, kWave - 1, kWave) * U;
  const long long want = (W + kI4Waves * kI4MinTiles - 1) / (kI4Waves * kI4MinTiles);
  const int groups = want < kI4Groups ? (int)want : kI4Groups;
  if ((int)blockIdx.x >= groups) return;
  const long long N = (long long)groups * kI4Waves;
  const long long widx = (long long)blockIdx.x * kI4Waves + wv;
  const long long x0 = widx * W / N, x1 = (widx + 1) * W / N;
  const int count = (int)(x1 - x0);

  I4Tile cur;
  {
    // The sequence that holds x0: its lane by a ballot, then a walk over that lane's.
    const unsigned long long before = __ballot(incl * U <= x0);
    const int l = __builtin_popcountll(before);
    long long base = l > 0 ? __shfl(incl, l - 1, kWave) : 0;
    int s = l * per;
    int ctx = 0, n = 1;
    for (int j = 0; j < per; ++j) {
      ctx = i4_clamp_ctx(a.ctxl[s < S ? s : S - 1], cap);
      n = i4_tiles(ctx);
      if (s >= S - 1 || (base + n) * U > x0) break;
      base += n;
      ++s;
    }
    const long long in = x0 - base * U;
    cur.seq = __builtin_amdgcn_readfirstlane(s < S ? s : S - 1);
    cur.ctx = __builtin_amdgcn_readfirstlane(ctx);
    cur.n = __builtin_amdgcn_readfirstlane(n);
    cur.u = __builtin_amdgcn_readfirstlane((int)(in / n));
    cur.t = __builtin_amdgcn_readfirstlane((int)(in % n));
    cur.ctx_next = i4_clamp_ctx(a.ctxl[min(cur.seq + 1, S - 1)], cap);
  }

  auto advance = [&](I4Tile& t) {
    if (++t.t < t.n) return;
    t.t = 0;
    if (++t.u < U) return;
    t.u = 0;
    t.seq = min(t.seq + 1, S - 1);
    t.ctx = t.ctx_next;
    t.n = i4_tiles(t.ctx);
    t.ctx_next = i4_clamp_ctx(a.ctxl[min(t.seq + 1, S - 1)], cap);
  };

  // ---- per-tile loads
  struct Ids {
    int k, v;
  };
  auto load_ids = [&](const I4Tile& t) -> Ids {
    Ids r{-1, -1};
    if (t.ctx > 0) {
      const int lastb = (t.ctx - 1) >> sh.bs_log2;
      const int32_t* row = a.bt + (size_t)t.seq * sh.max_blocks;
      r.k = row[min((t.t * kI4Tile + 4 * i16) >> sh.bs_log2, lastb)];
      r.v = row[min((t.t * kI4Tile + 16 * g) >> sh.bs_log2, lastb)];
    }
    return r;
  };
  auto safe = [&](int id) { return (uint32_t)id < (uint32_t)sh.num_blocks ? id : 0; };
  uint4 kr[STEPS], vr[T][4], ksr[4], vsr[4];
  const int k_last = min(4 * (STEPS - 1) + g, C - 1) * 16;
  int v_chunk[T];
#pragma unroll
  for (int tt = 0; tt < T; ++tt) v_chunk[tt] = min(16 * tt + i16, C - 1) * 16;
  auto load_k = [&](const I4Tile& t, int id) {
    const int off = (t.t * kI4Tile + 4 * i16) & (bs - 1);
    const uint8_t* p = a.kc + ((size_t)safe(id) * sh.num_kv_heads + t.u / a.nchunk) * cell_bytes +
                       quad_offset(off, C);
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      kr[j] = *reinterpret_cast<const uint4*>(p + (j < STEPS - 1 ? 64 * j + 16 * g : k_last));
  };
  auto load_scales = [&](const I4Tile& t, int id) {
    const size_t bh = (size_t)safe(id) * sh.num_kv_heads + t.u / a.nchunk;
    const size_t at = (bh << sh.bs_log2) + ((t.t * kI4Tile + 16 * g) & (bs - 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) ksr[j] = *reinterpret_cast<const uint4*>(a.ks + at + 4 * j);
#pragma unroll
    for (int j = 0; j < 4; ++j) vsr[j] = *reinterpret_cast<const uint4*>(a.vs + at + 4 * j);
  };
  auto load_v = [&](const I4Tile& t, int id) {
    const int off = (t.t * kI4Tile + 16 * g) & (bs - 1);
    const uint8_t* p = a.vc + ((size_t)safe(id) * sh.num_kv_heads + t.u / a.nchunk) * cell_bytes +
                       quad_offset(off, C);
#pragma unroll
    for (int tt = 0; tt < T; ++tt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        vr[tt][k] = *reinterpret_cast<const uint4*>(p + k * C * 16 + v_chunk[tt]);
  };

  // ---- the query of a unit: raw rows, then the matrix operand and its two factors
  uint4 qr[HT][STEPS];
  float cs[HT], qs[HT];
  auto load_q = [&](const I4Tile& t) {
    const int kvh = t.u / a.nchunk, ch = t.u - kvh * a.nchunk;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int hh = min(ch * 16 * HT + ht * 16 + i16, sh.group - 1);
      const uint16_t* row = a.q + ((size_t)t.seq * sh.num_heads + kvh * sh.group + hh) * D;
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
        qr[ht][j] = *reinterpret_cast<const uint4*>(row + min(4 * j + g, C - 1) * 8);
    }
  };
  auto convert_q = [&]() {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      float mx = 0.f, sum = 0.f;
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        if (4 * j + g >= C) qr[ht][j] = make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {qr[ht][j].x, qr[ht][j].y, qr[ht][j].z, qr[ht][j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float lo = widen_lo<BF>(w[k]), hi = widen_hi<BF>(w[k]);
          mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
          sum += lo + hi;
        }
      }
      mx = head_max(mx);
      sum = head_sum(sum);
      const int e = 15 - __builtin_amdgcn_frexp_expf(mx);   // |q| 2^e < 2^15
      cs[ht] = __builtin_amdgcn_ldexpf(sh.scale_log2 * kCode24, -e);
      qs[ht] = sh.scale_log2 * sum;
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const uint32_t w[4] = {qr[ht][j].x, qr[ht][j].y, qr[ht][j].z, qr[ht][j].w};
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = __builtin_amdgcn_ldexpf(widen_lo<BF>(w[k]), e);
          x[2 * k + 1] = __builtin_amdgcn_ldexpf(widen_hi<BF>(w[k]), e - 4);
        }
        qr[ht][j] = make_uint4(pack_h2(x[0], x[4]), pack_h2(x[1], x[5]), pack_h2(x[2], x[6]),
                               pack_h2(x[3], x[7]));
      }
    }
  };

  // ---- running state of the unit: reference point, sums over the lane's own tokens, output
  float M[HT], L[HT], B[HT];
  f4_t acc[HT][T][8];
  auto reset = [&]() {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      M[ht] = kNegInf;
      L[ht] = B[ht] = 0.f;
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[ht][tt][n] = (f4_t){0.f, 0.f, 0.f, 0.f};
    }
  };

  auto process = [&](const I4Tile& t, int idv, bool more, const I4Tile& nx, Ids idn) {
    // scores of the codes
    f4_t sc[HT][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) sc[ht][n] = (f4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const uint32_t w[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
        const h8_t ka = codes_k(w[n]);
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
          sc[ht][n] = mfma16(ka, __builtin_bit_cast(h8_t, qr[ht][j]), sc[ht][n]);
      }
    }
    if (more) {
      if (nx.t == 0) load_q(nx);
      load_k(nx, idn.k);
    }
    // tokens of the lane's 16 that exist
    int live = t.ctx - (t.t * kI4Tile + 16 * g);
    if ((uint32_t)idv >= (uint32_t)sh.num_blocks) live = 0;
    uint32_t kw[16], vw[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      kw[4 * k] = ksr[k].x, kw[4 * k + 1] = ksr[k].y, kw[4 * k + 2] = ksr[k].z, kw[4 * k + 3] = ksr[k].w;
      vw[4 * k] = vsr[k].x, vw[4 * k + 1] = vsr[k].y, vw[4 * k + 2] = vsr[k].z, vw[4 * k + 3] = vsr[k].w;
    }
    const bool full = __all(live >= 16);
    if (!full) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e >= live) kw[e] = vw[e] = 0;
    }
    h8_t phi[HT][2], plo[HT][2];
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      float z[16], mx = M[ht];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const half2_t k2 = __builtin_bit_cast(half2_t, kw[e]), v2 = __builtin_bit_cast(half2_t, vw[e]);
        z[e] = __builtin_fmaf((float)k2.x, sc[ht][e & 3][e >> 2] * cs[ht], (float)k2.y * qs[ht]);
        if (!full && e >= live) z[e] = kNegInf;
        // (2^-24: fp16's smallest step, for rows of one value, whose scale is 0)
        mx = fmaxf(mx, z[e] + __builtin_amdgcn_logf(fmaxf((float)v2.x, 0x1p-24f)));
      }
      mx = head_max(mx);
      const float f = M[ht] == kNegInf ? 0.f : exp2f_fast(M[ht] - mx);
      const float ref = mx == kNegInf ? 0.f : mx - kShift;
      if (__any(mx != M[ht])) {
#pragma unroll
        for (int tt = 0; tt < T; ++tt)
#pragma unroll
          for (int n = 0; n < 8; ++n) acc[ht][tt][n] *= f;
        L[ht] *= f;
        B[ht] *= f;
      }
      M[ht] = mx;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const half2_t v2 = __builtin_bit_cast(half2_t, vw[e]);
        const float p = exp2f_fast(z[e] - ref);
        L[ht] += p;
        B[ht] = __builtin_fmaf(p, (float)v2.y, B[ht]);
        const float ps = p * (float)v2.x;
        const half_t hi = (half_t)ps;
        phi[ht][e >> 3][e & 7] = hi;
        plo[ht][e >> 3][e & 7] = (half_t)(ps - (float)hi);
      }
    }
    if (more) load_scales(nx, idn.v);
    // weighted codes
#pragma unroll
    for (int tt = 0; tt < T; ++tt) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint4 a0 = vr[tt][2 * hf], a1 = vr[tt][2 * hf + 1];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x07060302u : 0x05040100u;
          u4_t w = {__builtin_amdgcn_perm(a0.y, a0.x, sel), __builtin_amdgcn_perm(a0.w, a0.z, sel),
                    __builtin_amdgcn_perm(a1.y, a1.x, sel), __builtin_amdgcn_perm(a1.w, a1.z, sel)};
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if (b == 2) w = w >> 8;
            const h8_t va = __builtin_bit_cast(h8_t, w & ((b & 1) ? 0x00F000F0u : 0x000F000Fu));
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
              f4_t& o = acc[ht][tt][4 * half + b];
              o = mfma16(va, phi[ht][hf], o);
              o = mfma16(va, plo[ht][hf], o);
            }
          }
        }
      }
    }
    if (more) load_v(nx, idn.v);
  };

  // The state as a piece: sums over the head's lanes, outputs in their own units.
  auto to_piece = [&]() {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      L[ht] = head_sum(L[ht]);
      B[ht] = head_sum(B[ht]);
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[ht][tt][n][r] =
                __builtin_fmaf(acc[ht][tt][n][r], (n & 1) ? kCode24 / 16.f : kCode24, B[ht]);
    }
  };
  auto piece4 = [&](int ht, int tt, int r, int half) {
    return (f4_t){acc[ht][tt][4 * half][r], acc[ht][tt][4 * half + 1][r],
                  acc[ht][tt][4 * half + 2][r], acc[ht][tt][4 * half + 3][r]};
  };
  auto write_out = [&](int seq, int u) {
    const int kvh = u / a.nchunk, ch = u - kvh * a.nchunk;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int hh = ch * 16 * HT + ht * 16 + i16;
      const float inv = L[ht] != 0.f ? 1.f / L[ht] : 0.f;
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int chunk = 16 * tt + 4 * g + r;
          if (hh >= sh.group || chunk >= C) continue;
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = pack2<BF>(acc[ht][tt][2 * k][r] * inv, acc[ht][tt][2 * k + 1][r] * inv);
          *reinterpret_cast<uint4*>(
              a.out + ((size_t)seq * sh.num_heads + kvh * sh.group + hh) * D + chunk * 8) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
  };

  // ---- the wave's tiles
  int state = count > 0 ? kHasTiles : 0;
  const int t0 = cur.t;
  if (count > 0) {
    if (t0 != 0) {
      state |= kHead;
      if (lane == 0) sm.head[wv] = I4Unit{x0 - t0, cur.n, cur.seq, cur.u};
    }
    reset();
    Ids id = load_ids(cur);
    load_q(cur);
    load_k(cur, id.k);
    load_scales(cur, id.v);
    load_v(cur, id.v);
    I4Tile nx = cur;
    Ids idn{-1, -1};
    if (count > 1) {
      advance(nx);
      idn = load_ids(nx);
    }
    bool fresh = true;
    for (int k = 0; k < count; ++k) {
      const bool more = k + 1 < count;
      if (fresh) convert_q();
      I4Tile nn = nx;
      Ids id2{-1, -1};
      if (k + 2 < count) {
        advance(nn);
        id2 = load_ids(nn);
      }
      process(cur, id.v, more, nx, idn);
      fresh = cur.t == cur.n - 1;                       // the unit ends here
      const bool head = (state & kHead) && cur.t == t0 + k;   // ... and was begun before the wave
      if (fresh || !more) {
        to_piece();
        if (head) {
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
            for (int tt = 0; tt < T; ++tt)
#pragma unroll
              for (int f = 0; f < 8; ++f)
                sm.acc[wv][(ht * T + tt) * 8 + f][lane] = piece4(ht, tt, f >> 1, f & 1);
            if (g == 0) sm.ml[wv][ht * 16 + i16] = (f2_t){M[ht], L[ht]};
          }
          if (fresh) state |= kHeadEnds;
        } else if (fresh) {
          write_out(cur.seq, cur.u);
        } else {
          state |= kTail;
        }
        if (more) reset();
      }
      if (more) {
        cur = nx;
        id = idn;
        nx = nn;
        idn = id2;
      }
    }
  }
  if (lane == 0) sm.state[wv] = state;
  if (threadIdx.x < 2) sm.piece[threadIdx.x].active = 0;
  __syncthreads();

  // ---- units that several waves share.  The wave that began one folds the waves' behind it.
  auto fold_slot = [&](int w) {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const f2_t ml = sm.ml[w][ht * 16 + i16];
      const float mx = fmaxf(M[ht], ml.x);
      const float f1 = M[ht] == kNegInf ? 0.f : exp2f_fast(M[ht] - mx);
      const float f2 = ml.x == kNegInf ? 0.f : exp2f_fast(ml.x - mx);
      M[ht] = mx;
      L[ht] = L[ht] * f1 + ml.y * f2;
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int f = 0; f < 8; ++f) {
          const f4_t v = sm.acc[w][(ht * T + tt) * 8 + f][lane];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f4_t& o = acc[ht][tt][4 * (f & 1) + k];
            o[f >> 1] = o[f >> 1] * f1 + v[k] * f2;
          }
        }
    }
  };
  // Folds the slots of waves w, w + 1, ..; whether the unit ends among them.
  auto fold_from = [&](int w) {
    for (; w < kI4Waves; ++w) {
      const int st = __builtin_amdgcn_readfirstlane(sm.state[w]);
      if (!(st & kHasTiles)) continue;
      fold_slot(w);
      if (st & kHeadEnds) return true;
    }
    return false;
  };
  auto worker_group = [&](long long x) {          // the work-group whose range holds tile x
    return (int)((((x + 1) * N - 1) / W) / kI4Waves);
  };
  // The piece of a unit that other work-groups share: into memory, to be counted below.
  auto share = [&](int which, long long begin, int n, int seq, int u) {
    float* slot = a.ws + (size_t)(2 * blockIdx.x + which) * G::kSlotFloats;
    const auto rs = buf_rsrc(slot, (uint32_t)(G::kSlotFloats * 4));
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int f = 0; f < 8; ++f)
          dev_store4(rs, (((ht * T + tt) * 8 + f) * kWave + lane) * 16, piece4(ht, tt, f >> 1, f & 1));
      if (g == 0) {
        const f2_t ml = {M[ht], L[ht]};
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2_t, ml), rs,
                                              G::kPieceFloats * 4 + (ht * 16 + i16) * 8, 0,
                                              kPolicyDevice);
      }
    }
    if (lane == 0) {
      auto& p = sm.piece[which];
      p.active = 1;
      p.first = worker_group(begin);
      p.count = worker_group(begin + n - 1) - p.first + 1;
      p.seq = seq;
      p.u = u;
    }
  };
  if (state & kTail) {
    if (fold_from(wv + 1)) write_out(cur.seq, cur.u);
    else share(1, x1 - 1 - cur.t, cur.n, cur.seq, cur.u);
  }
  if (wv == 0) {
    int w = 0;
    while (w < kI4Waves && !(sm.state[w] & kHasTiles)) ++w;
    w = __builtin_amdgcn_readfirstlane(w);
    if (w < kI4Waves && (sm.state[w] & kHead)) {
      reset();
      fold_from(w);
      share(0, sm.head[w].begin, sm.head[w].n, sm.head[w].seq, sm.head[w].u);
    }
  }
  // ---- units that several work-groups share: the last to arrive merges the pieces.
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  const int b = blockIdx.x;
  auto arrive = [&](uint32_t* c, int n) {
    const bool last = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                      (uint32_t)(n - 1);
    if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
  };
  if (threadIdx.x < 2) {
    auto& p = sm.piece[threadIdx.x];
    p.last = 0;
    if (p.active) {
      // groups of kMergeMax consecutive pieces; the first group's counter is the first
      // work-group's own, which no other unit has, a later group's its first member's
      const int gi = (b - p.first) / kMergeMax, m0 = p.first + gi * kMergeMax;
      p.last = arrive(a.cnt + (gi == 0 ? 0 : kI4Groups) + m0, min(kMergeMax, p.first + p.count - m0));
    }
  }
  __syncthreads();
  // Merges n pieces, those of work-groups m0, m0 + step, ..: the output, or one piece in
  // place of the first.
  auto merge = [&](int first, int m0, int step, int n, bool final_out, int seq, int u) {
    const int kvh = u / a.nchunk, ch = u - kvh * a.nchunk;
    auto slot_of = [&](int j) {
      const int m = m0 + j * step;
      return a.ws + (size_t)(2 * m + (m == first ? 1 : 0)) * G::kSlotFloats;
    };
    f4_t A[T * HT];
    float Mi[T * HT], Li[T * HT];
#pragma unroll
    for (int q = 0; q < T * HT; ++q) {
      const int f = wv + q * kI4Waves;                  // (ht * T + tt) * 8 + 2 r + half
      const int h = (f / (8 * T)) * 16 + i16;
      f4_t v[kMergeMax];
      f2_t ml[kMergeMax];
#pragma unroll
      for (int j = 0; j < kMergeMax; ++j) {
        // (past the last piece it is read again and weighted 0: every load is unconditional)
        const auto rs = buf_rsrc(slot_of(min(j, n - 1)), (uint32_t)(G::kSlotFloats * 4));
        v[j] = dev_load4(rs, (f * kWave + lane) * 16);
        ml[j] = __builtin_bit_cast(f2_t, __builtin_amdgcn_raw_buffer_load_b64(
                                             rs, G::kPieceFloats * 4 + h * 8, 0, kPolicyDevice));
      }
      float mx = kNegInf;
#pragma unroll
      for (int j = 0; j < kMergeMax; ++j)
        if (j < n) mx = fmaxf(mx, ml[j].x);
      f4_t s = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int j = 0; j < kMergeMax; ++j) {
        const float w = j >= n || ml[j].x == kNegInf ? 0.f : exp2f_fast(ml[j].x - mx);
        if (j < n) {
          s += v[j] * w;
          l += ml[j].y * w;
        }
      }
      A[q] = s;
      Mi[q] = mx;
      Li[q] = l;
    }
    if (final_out) {
#pragma unroll
      for (int q = 0; q < T * HT; ++q) {
        const int f = wv + q * kI4Waves;
        const int hh = ch * 16 * HT + (f / (8 * T)) * 16 + i16;
        const int chunk = ((f / 8) % T) * 16 + 4 * g + ((f & 7) >> 1);
        if (hh >= sh.group || chunk >= C) continue;
        const float inv = Li[q] != 0.f ? 1.f / Li[q] : 0.f;
        const uint2 w = make_uint2(pack2<BF>(A[q][0] * inv, A[q][1] * inv),
                                   pack2<BF>(A[q][2] * inv, A[q][3] * inv));
        *reinterpret_cast<uint2*>(a.out +
                                  ((size_t)seq * sh.num_heads + kvh * sh.group + hh) * D +
                                  chunk * 8 + 4 * (f & 1)) = w;
      }
    } else {
      // (each thread rewrites the items that it alone read; the pairs, which all read, after
      // a barrier)
      __syncthreads();
      const auto rs = buf_rsrc(slot_of(0), (uint32_t)(G::kSlotFloats * 4));
#pragma unroll
      for (int q = 0; q < T * HT; ++q) {
        const int f = wv + q * kI4Waves;
        dev_store4(rs, (f * kWave + lane) * 16, A[q]);
        if (f % (8 * T) == 0 && g == 0) {
          const f2_t ml = {Mi[q], Li[q]};
          __builtin_amdgcn_raw_buffer_store_b64(
              __builtin_bit_cast(u2_t, ml), rs,
              G::kPieceFloats * 4 + ((f / (8 * T)) * 16 + i16) * 8, 0, kPolicyDevice);
        }
      }
    }
  };
  for (int which = 0; which < 2; ++which) {
    const auto p = sm.piece[which];
    if (!__builtin_amdgcn_readfirstlane(p.last)) continue;
    const int first = __builtin_amdgcn_readfirstlane(p.first);
    const int np = __builtin_amdgcn_readfirstlane(p.count);
    const int seq = __builtin_amdgcn_readfirstlane(p.seq), u = __builtin_amdgcn_readfirstlane(p.u);
    const int gi = (b - first) / kMergeMax, m0 = first + gi * kMergeMax;
    const int n = min(kMergeMax, first + np - m0);
    if (np <= kMergeMax) {
      merge(first, m0, 1, n, true, seq, u);
      continue;
    }
    merge(first, m0, 1, n, false, seq, u);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    const int ng = (np + kMergeMax - 1) / kMergeMax;
    if (threadIdx.x == 0) sm.last2 = arrive(a.cnt + 2 * kI4Groups + first, ng);
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(sm.last2)) merge(first, first, kMergeMax, ng, true, seq, u);
    __syncthreads();   // (last2 is written again by the other piece)
  }
}

namespace {

template <int HT, bool BF>
hipError_t launch_tiles(const Int4Decode& l) {
  I4Args a{static_cast<const uint16_t*>(l.q), static_cast<uint16_t*>(l.out),
           static_cast<const uint8_t*>(l.k_cache), static_cast<const uint8_t*>(l.v_cache),
           static_cast<const uint32_t*>(l.k_scales), static_cast<const uint32_t*>(l.v_scales),
           l.block_table, l.context_lens, l.workspace, l.counters,
           (l.shape.group + 16 * HT - 1) / (16 * HT), l.shape};
  decode_int4_kernel<PA_INT4_STEPS, HT, BF><<<kI4Groups, kI4Waves * kWave, 0, l.stream>>>(a);
  return hipGetLastError();
}

}  // namespace

// Two head tiles where one unit then holds heads that would read its rows twice (their
// second set of outputs needs the registers that wider heads use).
template <>
hipError_t launch_int4_decode_steps<PA_INT4_STEPS>(const Int4Decode& l) {
#if PA_INT4_STEPS <= 4
  if (l.shape.group > 16) return l.bf16 ? launch_tiles<2, true>(l) : launch_tiles<2, false>(l);
#endif
  return l.bf16 ? launch_tiles<1, true>(l) : launch_tiles<1, false>(l);
}

template <>
size_t int4_decode_slot_bytes<PA_INT4_STEPS>(int group) {
  return sizeof(float) * (PA_INT4_STEPS <= 4 && group > 16 ? I4Geo<PA_INT4_STEPS, 2>::kSlotFloats
                                                           : I4Geo<PA_INT4_STEPS, 1>::kSlotFloats);
}

}  // namespace pa
