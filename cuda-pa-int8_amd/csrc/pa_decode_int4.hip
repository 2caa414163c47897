// Decode attention over the 4-bit paged cache (gfx950).  Layout: pa_int4.hpp.
//
//   out[h] = sum_t p_t (s_t c_t + m_t) / sum_t p_t,
//   p_t = exp(scale (s'_t (q . c'_t) + m'_t sum(q)))      (primed: K's codes, scale and minimum)
//
// Both products are matrix instructions on the codes themselves (v_mfma_f32_16x16x32_f16); the
// scales and minima enter in fp32, at the scores and at the weights:
//   scores   S[token][head]  = C'[tokens][32 dims] x Q^T[dims][16 heads]
//   output   O^T[dim][head] += C^T[dims][32 tokens] x P^T[tokens][heads],  P = p s
// A code c sits in the low bits of an fp16 element, where it is a subnormal number: for K
// c 2^-24, or 16 c 2^-24 from the upper half byte, and masks are all the unpacking there is (5
// instructions for 8 codes); for V, whose bytes are put in token order first, 4 c 2^-24 or
// 64 c 2^-24 (a shift and a mask each for the even and the odd dims).  The matrix core takes
// subnormal elements exactly.  The powers of two are put right in fp32: those of K in q
// (normalised per head to at most 2^15 so that none of its bits are lost), those of V when a
// piece is finished.
//
// Lanes.  Lane l = (i = l & 15, g = l >> 4).  A tile is 64 tokens.  For K, lane (i, g) loads
// quad i (tokens 4i .. 4i+3) of 8 dims 8 (4 step + g) ..: matrix row i of instruction n is token
// 4i + n, and the scores of head h = i and tokens 16g + 4r + n come out in lane (h, g),
// register r.  For V, lane (i, g) loads tokens 16g .. 16g + 15 of the dims 8i .. 8i + 7:
// the weights that lane (h, g) holds are the operand as they are, no lane exchanges anything
// but the running maximum, and output row i of instruction n is dim 8i + n.  A token's scale and
// minimum are in one lane of its row, from where the score and weight instructions read them.
//
// Weights.  The reference point of the exponentials is the running maximum of score +
// log2(s), less kShift: the P = p s stay at or below 2^(kShift + kSlack) whatever the rows'
// scales.  P enters as two fp16 numbers (its rounding and what that left), 22 bits together: with
// one the outputs' error would grow threefold, as the codes are not centred.  sum p and sum p m
// are fp32 sums of the unrounded weights.
//
// Work.  The tiles of all units (sequence, kv head, chunk of 16 HT query heads) form one list,
// in that order.  It is divided evenly among the work-groups, one a CU, and a work-group's part
// among its waves: as even as tiles are, whatever the lengths, and found by every wave from
// context_lens alone.  (Where units are few and short, a work-group takes one unit.)  A unit
// inside one wave's range needs no merge at all; the pieces of a unit that several waves share are merged
// through LDS, and those of a unit that several work-groups share through memory, by the last of
// them to arrive (in two levels above kMergeMax pieces).  All orders are fixed: the same bits
// every time.
//
// What bounds it.  Long lists, the reads: the next tile's rows are loaded as this one's
// registers fall free, eight waves a CU keep 64 to 128 KB under way, and the loop reads 6.3 to
// 6.7 TB/s (large reads reach 7.0); V is read without being kept in the caches, and the wave that
// is behind goes first on its SIMD.  A launch has about 2.5 us before its first rows arrive
// (lengths, block ids, rows: three loads that wait for each other) and 5 to 9 us from the last
// rows to the end where units are shared between work-groups, which is what bounds short ones.
// Measured, in us: 4 x 100-512 tokens, 8/8 heads of 64: 6.6; 32 x 4096, 12/2 of 128: 13.6 (36 MB);
// 8 x 32768, 32/8 of 128: 54 (5.3 TB/s); 192 ragged sequences (median 1024 tokens, at most 8192),
// 32/8 of 128: 65 (5.1 TB/s); 24 x 900-9000, 8/4 of 256: 32.8 (4.7 TB/s).
#include <math.h>

#include "pa_decode_kernels.hpp"
#include "pa_int4.hpp"

namespace pa {

constexpr int kI4Waves = 8;          // waves of a work-group
constexpr int kI4Groups = kInt4Groups;   // work-groups of a launch, at most: one a CU
constexpr int kI4Tile = 64;          // tokens
constexpr int kMergeMax = 16;        // pieces merged at once
// Tiles from which units of more than 16 heads take two head tiles (decode_int4_kernel).
constexpr uint32_t kI4TwoTiles = 6u * kI4Groups * kI4Waves;
constexpr float kShift = 14.f;       // the weights' upper end: 2^14 of fp16's 2^16, and
constexpr float kSlack = 1.5f;       // how far a score may pass the reference before that moves
constexpr float kCode24 = 16777216.f;   // 2^24: a code's element times this is the code

// A tile of the list: tile t of the n of a unit (sequence, kv head, chunk of query heads).
struct I4Tile {
  int seq, kvh, ch, t, n, ctx, ctx_next;
};

// Groups of at most 8 heads leave columns of the products free.
// kPack, heads wider than 64: a finished piece holds the second half of each 8 dims in columns
// 8 .. 15, so that pieces are half as large in LDS and memory.  kPack4, at most 4 such heads: the
// four quads of columns hold a quarter each.
// kPair, heads of at most 64 dims, which leave half of the rows of the output product free too:
// matrix rows i and i + 8 are chunk i of a lane row's tokens 16g .. 16g + 7 and 16g + 8 .., columns
// c and c + 8 head c's weights of the same, and the blocks where they meet count.  Half the
// softmax, the conversions of V and the products of a tile; a finished piece holds the second half
// of each 8 dims in lanes 32 ...
// (kPair: 64 x 2000-16000 tokens at 32/8 heads of 64 86 -> 73 us, 16 x 500-8000 at 14/2 14.2 -> 12.6.
// kPack and kPack4: 24 x 900-9000 at 8/4 heads of 256 37.1 -> 33.2, one of 131072 at 8/1 of 128
// 16.6 -> 14.4, 32 x 4096 at 12/2 14.4 -> 14.0.)
constexpr int kWhole = 0, kPack = 1, kPair = 2, kPack4 = 3;
// Items of a head tile and 16 chunks.
constexpr int mode_items(int mode) { return mode == kWhole ? 8 : (mode == kPack4 ? 2 : 4); }

// A piece: items of 64 lanes x 4 dims, [head tile][16-chunk tile][item], kWhole's [row r][half].
template <int STEPS, int HT, int MODE>
struct I4Geo {
  static constexpr int T = (STEPS + 3) / 4;
  static constexpr int NF = mode_items(MODE) * T * HT;
  static constexpr int kPieceFloats = NF * kWave * 4;
  static constexpr int kMlFloats = 2 * 16 * HT;
  static constexpr size_t kSlotFloats = kPieceFloats + kMlFloats;
};

// The unit that a wave's first tile belongs to, where it was begun before the wave.
struct I4Unit {
  uint32_t begin;   // its start in the list
  int n, seq, kvh, ch;
};

template <int STEPS, int HT, int MODE>
struct alignas(16) I4Smem {
  using G = I4Geo<STEPS, HT, MODE>;
  f4_t acc[kI4Waves][G::NF][kWave];
  f2_t ml[kI4Waves][16 * HT];
  I4Unit head[kI4Waves], tail[kI4Waves];
  int state[kI4Waves], progress[kI4Waves];
  // the pieces of units that other work-groups share: [0] begun earlier, [1] continued later
  struct {
    int active, first, count, seq, kvh, ch, last;
  } piece[2];
  int last2;
};
constexpr int kI4Check = 256;        // beside the block size's log2: a checked call
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

// Eight tokens' scores: lanes E0 .. E0 + 7 of a row hold their scale and minimum, which the
// instructions read from there (a row broadcast each).  z = m qn + s c.  The compiler does not
// see what is inside: both halves wait the two states that a broadcast of values just written
// needs, and the first (E0 = 0) waits out the matrix instructions behind c; the second comes
// after it.
template <int E0>
__device__ __forceinline__ void score8(float (&z)[16], float m, float s, float qn, const f4_t* c) {
#define PA_MUL(K, E) "v_mul_f32_dpp %" #K ", %8, %10 row_newbcast:" #E " row_mask:0xf bank_mask:0xf\n\t"
#define PA_FMAC(K, C, E) "v_fmac_f32_dpp %" #K ", %9, %" #C " row_newbcast:" #E " row_mask:0xf bank_mask:0xf\n\t"
#define PA_OUT(E) "=&v"(z[E]), "=&v"(z[E + 1]), "=&v"(z[E + 2]), "=&v"(z[E + 3]), "=&v"(z[E + 4]), \
                  "=&v"(z[E + 5]), "=&v"(z[E + 6]), "=&v"(z[E + 7])
#define PA_IN(R) "v"(m), "v"(s), "v"(qn), "v"(c[0][R]), "v"(c[1][R]), "v"(c[2][R]), "v"(c[3][R]), \
                 "v"(c[0][R + 1]), "v"(c[1][R + 1]), "v"(c[2][R + 1]), "v"(c[3][R + 1])
  if constexpr (E0 == 0)
    asm("s_nop 7\n\ts_nop 7\n\t" PA_MUL(0, 0) PA_MUL(1, 1) PA_MUL(2, 2) PA_MUL(3, 3) PA_MUL(4, 4) PA_MUL(5, 5)
        PA_MUL(6, 6) PA_MUL(7, 7) PA_FMAC(0, 11, 0) PA_FMAC(1, 12, 1) PA_FMAC(2, 13, 2)
        PA_FMAC(3, 14, 3) PA_FMAC(4, 15, 4) PA_FMAC(5, 16, 5) PA_FMAC(6, 17, 6) PA_FMAC(7, 18, 7)
        : PA_OUT(0) : PA_IN(0));
  else
    asm("s_nop 1\n\t" PA_MUL(0, 8) PA_MUL(1, 9) PA_MUL(2, 10) PA_MUL(3, 11) PA_MUL(4, 12)
        PA_MUL(5, 13) PA_MUL(6, 14) PA_MUL(7, 15) PA_FMAC(0, 11, 8) PA_FMAC(1, 12, 9)
        PA_FMAC(2, 13, 10) PA_FMAC(3, 14, 11) PA_FMAC(4, 15, 12) PA_FMAC(5, 16, 13)
        PA_FMAC(6, 17, 14) PA_FMAC(7, 18, 15)
        : PA_OUT(8) : PA_IN(2), "v"(z[0]));
#undef PA_IN
#undef PA_OUT
#undef PA_FMAC
#undef PA_MUL
}
// ... and their weights p: w = s p, B += m p.
template <int E0>
__device__ __forceinline__ void weight8(float (&w)[8], float& B, float m, float s,
                                        const float (&p)[8]) {
#define PA_MUL(K, P, E) "v_mul_f32_dpp %" #K ", %10, %" #P " row_newbcast:" #E " row_mask:0xf bank_mask:0xf\n\t"
#define PA_FMAC(P, E) "v_fmac_f32_dpp %8, %9, %" #P " row_newbcast:" #E " row_mask:0xf bank_mask:0xf\n\t"
#define PA_ARGS                                                                                 \
  : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), \
    "=&v"(w[7]), "+&v"(B) : "v"(m), "v"(s), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]),        \
    "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7])
  if constexpr (E0 == 0)
    asm("s_nop 1\n\t" PA_MUL(0, 11, 0) PA_FMAC(11, 0) PA_MUL(1, 12, 1) PA_FMAC(12, 1)
        PA_MUL(2, 13, 2) PA_FMAC(13, 2) PA_MUL(3, 14, 3) PA_FMAC(14, 3) PA_MUL(4, 15, 4)
        PA_FMAC(15, 4) PA_MUL(5, 16, 5) PA_FMAC(16, 5) PA_MUL(6, 17, 6) PA_FMAC(17, 6)
        PA_MUL(7, 18, 7) PA_FMAC(18, 7) PA_ARGS);
  else
    asm("s_nop 1\n\t" PA_MUL(0, 11, 8) PA_FMAC(11, 8) PA_MUL(1, 12, 9) PA_FMAC(12, 9)
        PA_MUL(2, 13, 10) PA_FMAC(13, 10) PA_MUL(3, 14, 11) PA_FMAC(14, 11) PA_MUL(4, 15, 12)
        PA_FMAC(15, 12) PA_MUL(5, 16, 13) PA_FMAC(16, 13) PA_MUL(6, 17, 14) PA_FMAC(17, 14)
        PA_MUL(7, 18, 15) PA_FMAC(18, 15) PA_ARGS);
#undef PA_ARGS
#undef PA_FMAC
#undef PA_MUL
}
// Max over the 16 lanes of a row.
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_mov<kQuadXor1>(v));
  v = fmaxf(v, dpp_mov<kQuadXor2>(v));
  v = fmaxf(v, dpp_mov<kRowHalfMirror>(v));
  return fmaxf(v, dpp_mov<kRowMirror>(v));
}
constexpr int kRowRor4 = 0x124, kRowRor8 = 0x128, kRowRor12 = 0x12C, kQuadReverse = 0x1B;
// Of a head's two columns.
__device__ __forceinline__ float pair_max8(float v) { return fmaxf(v, dpp_mov<kRowRor8>(v)); }
__device__ __forceinline__ float pair_sum8(float v) { return v + dpp_mov<kRowRor8>(v); }
// v, in columns 8 .. 15 u's of columns 0 .. 7.
template <int CTRL = kRowRor8, int BANKS = 0xC>
__device__ __forceinline__ float upper_from(float v, float u) {
  return bitsf((uint32_t)__builtin_amdgcn_update_dpp((int)fbits(v), (int)fbits(u), CTRL, 0xF, BANKS,
                                                     false));
}
// a, b, c and d of columns 0 .. 3 in the four quads of columns.
__device__ __forceinline__ float quads_from(float a, float b, float c, float d) {
  return upper_from<kRowRor12, 0x8>(
      upper_from<kRowRor8, 0x4>(upper_from<kRowRor4, 0x2>(a, b), c), d);
}
// v, in the quads of BANKS that of the lane 4 further or back in its 8.
template <int BANKS>
__device__ __forceinline__ uint32_t other_quad(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)dpp_mov_u<kRowHalfMirror>(v),
                                               kQuadReverse, 0xF, BANKS, false);
}
// The value that lane N of the quad holds.
template <int N>
__device__ __forceinline__ float quad_bcast(float v) {
  return dpp_mov<N * 0x55>(v);
}
__device__ __forceinline__ int select4(int a0, int a1, int a2, int a3, int k) {
  const int lo = (k & 1) ? a1 : a0, hi = (k & 1) ? a3 : a2;
  return (k & 2) ? hi : lo;
}

// Lengths and block table, which nothing in the launch writes: uniform reads stay scalar loads,
// whatever stores come before them.
typedef const __attribute__((address_space(4))) int32_t* const_i32;
__device__ __forceinline__ const_i32 as_const(const int32_t* p) {
  return (const_i32)reinterpret_cast<uintptr_t>(p);
}

// What a wave knows of the lengths.  Lane l has the tiles of sequences l per .. l per + per - 1.
struct I4Lens {
  int per, lane_ctx;        // sequences a lane; the context of the lane's last
  uint32_t incl, total;     // tiles of one (kv head, chunk): the lanes' running sum, and all
  uint32_t longest;         // tiles of a sequence: the longest of this lane's
  bool empty;               // whether one holds no token
};
__device__ __forceinline__ I4Lens i4_lens(const_i32 ctxl, int S, int cap) {
  I4Lens r;
  r.per = (S + kWave - 1) / kWave;
  uint32_t mine = 0;
  r.longest = 0;
  r.lane_ctx = 0;
  int least = 1;
  for (int j = 0; j < r.per; ++j) {
    const int s = (threadIdx.x & (kWave - 1)) * r.per + j;
    const int ctx = ctxl[min(s, S - 1)];
    least = min(least, ctx);
    r.lane_ctx = i4_clamp_ctx(ctx, cap);
    const uint32_t n = i4_tiles(r.lane_ctx);
    mine += s < S ? n : 0u;
    r.longest = max(r.longest, n);
  }
  r.incl = wave_scan_dpp(mine);
  r.total = (uint32_t)__builtin_amdgcn_readlane((int)r.incl, kWave - 1);
  r.empty = __any(least < 1);
  return r;
}

template <int STEPS, int HT, int MODE, bool BF>
__device__ __forceinline__ void decode_int4_body(
    I4Smem<STEPS, HT, MODE>& sm, const I4Lens& lens, const_i32 bt, const_i32 ctxl,
    const Int4DecodeShape& sh, const uint16_t* __restrict__ q,
    const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const uint32_t* __restrict__ ks, const uint32_t* __restrict__ vs, uint16_t* __restrict__ out,
    float* __restrict__ ws, uint32_t* __restrict__ cnt) {
  using G = I4Geo<STEPS, HT, MODE>;
  constexpr bool PAIR = MODE == kPair, PACK = MODE == kPack, PACK4 = MODE == kPack4;
  constexpr int T = G::T, I = mode_items(MODE);
  // The waves' pieces of one unit are folded by all of them where a piece is at most one float4 a
  // thread (32 x 4096 at 12/2 heads 15.7 -> 14.9 us; with two, slower than by their first wave: 64
  // sequences of median 2048 at 32/1 26.4 against 24.6).
  constexpr bool kTogether = G::NF <= kI4Waves;
  // the next unit's query is loaded a tile ahead where there are registers for it (with more, the
  // loop spills)
  constexpr bool kQueryAhead = STEPS * HT <= 4;
  const int nchunk = (sh.group + 16 * HT - 1) / (16 * HT);
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int S = sh.num_seqs, U = sh.num_kv_heads * nchunk, C = sh.head_dim / 8, D = sh.head_dim;
  const int bs = 1 << sh.bs_log2;
  const int cap = sh.max_blocks << sh.bs_log2;
  const uint32_t cell_bytes = (uint32_t)(C * 4) << sh.bs_log2;   // bytes of a (block, head)

  const int per = lens.per, lane_ctx = lens.lane_ctx;
  const uint32_t incl = lens.incl;
  const uint32_t tiles = lens.total * (uint32_t)U;
  // (another work-group as soon as every wave has a tile: with two each, 2000 tokens at 28/4 heads
  // 10.7 -> 13.0 us)
  const uint32_t want = (tiles + kI4Waves - 1) / kI4Waves;
  // Few short units get a work-group each: nothing then is merged through memory, which costs
  // about two tiles' time (4 x 100-512 tokens at 8/8 heads 10.4 -> 7.4 us).
  const uint32_t units = (uint32_t)(S * U);
  const uint32_t most = (tiles / (kI4Groups * kI4Waves) + 2) * kI4Waves;
  const bool whole = units <= (uint32_t)kI4Groups && !__any(lens.longest > most);
  const uint32_t groups = whole ? units : (want < kI4Groups ? want : kI4Groups);
  const uint32_t b = blockIdx.x;
  if (b >= groups) return;
  // Work-group b takes tiles / groups tiles of the list, the first tiles % groups one more; its
  // waves likewise.  (Divided by cost, half a tile for a unit's start and end, 192 ragged sequences
  // ran 66.1 -> 65.0 us and the other calls 0.2 us longer.)
  const uint32_t Q = tiles / groups, R = tiles - Q * groups;
  const uint32_t gn = Q + (b < R ? 1u : 0u);
  const uint32_t x0 = b * Q + min(b, R) + wv * (gn / kI4Waves) + min((uint32_t)wv, gn % kI4Waves);
  const uint32_t x1 = x0 + gn / kI4Waves + ((uint32_t)wv < gn % kI4Waves ? 1u : 0u);

  // Tile x of the list, and where its unit starts.
  const uint32_t lane_end = incl * (uint32_t)U;
  auto tile_at = [&](uint32_t x, I4Tile& t) {
    // The sequence: its lane by a ballot, then, where a lane has several, a walk over that
    // lane's.
    const unsigned long long before = __ballot(lane_end <= x);
    const int l = min((int)__builtin_popcountll(before), kWave - 1);
    uint32_t base = l > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)incl, l - 1) : 0u;
    int s = min(l * per, S - 1), n, ctx;
    if (per == 1) {
      ctx = __builtin_amdgcn_readlane(lane_ctx, s);
      n = i4_tiles(ctx);
      t.ctx_next = __builtin_amdgcn_readlane(lane_ctx, min(s + 1, S - 1));
    } else {
      for (int j = 0;; ++j) {
        ctx = i4_clamp_ctx(ctxl[s], cap);
        n = i4_tiles(ctx);
        if (j >= per - 1 || s >= S - 1 || (base + n) * U > x) break;
        base += n;
        ++s;
      }
      t.ctx_next = ctxl[min(s + 1, S - 1)];
    }
    const uint32_t in = x - base * U, u = in / (uint32_t)n;
    t.seq = s;
    t.ctx = ctx;
    t.n = n;
    t.t = (int)(in - u * n);
    t.kvh = (int)(u / (uint32_t)nchunk);
    t.ch = (int)u - t.kvh * nchunk;
    return x - (uint32_t)t.t;
  };
  I4Tile cur;
  uint32_t unit0 = 0;                // where the first tile's unit starts
  int count = (int)(x1 - x0);
  if (whole) {
    const int seq = (int)(b / (uint32_t)U), u = (int)b - seq * U;
    cur.seq = seq;
    cur.kvh = u / nchunk;
    cur.ch = u - cur.kvh * nchunk;
    cur.ctx = i4_clamp_ctx(ctxl[seq], cap);
    cur.n = i4_tiles(cur.ctx);
    cur.ctx_next = 0;
    cur.t = wv * (cur.n / kI4Waves) + min(wv, cur.n % kI4Waves);
    count = cur.n / kI4Waves + (wv < cur.n % kI4Waves ? 1 : 0);
  } else {
    unit0 = tile_at(x0, cur);
  }

  auto advance = [&](I4Tile& t) {
    if (++t.t < t.n) return;
    t.t = 0;
    if (++t.ch < nchunk) return;
    t.ch = 0;
    if (++t.kvh < sh.num_kv_heads) return;
    t.kvh = 0;
    t.seq = min(t.seq + 1, S - 1);
    t.ctx = i4_clamp_ctx(t.ctx_next, cap);
    t.n = i4_tiles(t.ctx);
    t.ctx_next = ctxl[min(t.seq + 1, S - 1)];
  };

  // ---- per-tile loads.  The block ids of a tile's four 16-token groups, in scalar registers.
  struct Ids {
    int b[4];
  };
  auto load_ids = [&](const I4Tile& t) {
    Ids r{{-1, -1, -1, -1}};
    if (t.ctx > 0) {
      const int lastb = (t.ctx - 1) >> sh.bs_log2;
      const const_i32 row = bt + (size_t)t.seq * sh.max_blocks;
#pragma unroll
      for (int j = 0; j < 4; ++j) r.b[j] = row[min((t.t * kI4Tile + 16 * j) >> sh.bs_log2, lastb)];
    }
    return r;
  };
  // The lane's block for K (tokens 4 i16 ..) and for V and the scales (16 g ..), 0 where the id
  // is outside the pool, and how many of its 16 tokens exist (none then).
  struct Where {
    int k, v, live;
  };
  auto locate = [&](const I4Tile& t, const Ids& id) {
    int sb[4], lv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = (uint32_t)id.b[j] < (uint32_t)sh.num_blocks;
      sb[j] = ok ? id.b[j] : 0;
      lv[j] = ok ? t.ctx - (t.t * kI4Tile + 16 * j) : 0;
    }
    return Where{select4(sb[0], sb[1], sb[2], sb[3], i16 >> 2),
                 select4(sb[0], sb[1], sb[2], sb[3], g), select4(lv[0], lv[1], lv[2], lv[3], g)};
  };
  constexpr int VQ = PAIR ? 2 : 4;         // quads of V's tokens a lane loads
  uint4 kr[STEPS], vr[T][VQ];
  uint32_t ksr, vsr;
  // Byte offset of step j's 8 dims of K (of a query) for this lane.  Opaque to the compiler,
  // which would otherwise keep each sum of such offsets in registers through the loop.
  const uint32_t k_first = 16 * g, k_last = min(4 * (STEPS - 1) + g, C - 1) * 16;
  auto k_chunk = [&](int j) {
    uint32_t c = j < STEPS - 1 ? k_first : k_last;
    asm volatile("" : "+v"(c));
    return j < STEPS - 1 ? c + 64 * j : c;
  };
  const int v_step = C * 16;
  auto load_k = [&](const I4Tile& t, const Where& w) {
    const int off = (t.t * kI4Tile + 4 * i16) & (bs - 1);
    const uint8_t* p = kc + (uint64_t)(uint32_t)(w.k * sh.num_kv_heads + t.kvh) * cell_bytes +
                       (uint32_t)quad_offset(off, C);
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      kr[j] = *reinterpret_cast<const uint4*>(p + k_chunk(j));
  };
  // (lane (i, g) holds token 16 g + i's pairs; the rows broadcast them)
  auto load_scales = [&](const I4Tile& t, const Where& w) {
    const uint32_t bh = (uint32_t)(w.v * sh.num_kv_heads + t.kvh);
    const uint64_t at = ((uint64_t)bh << sh.bs_log2) + ((t.t * kI4Tile + 16 * g) & (bs - 1)) + i16;
    ksr = ks[at];
    vsr = vs[at];
  };
  auto load_v = [&](const I4Tile& t, const Where& w) {
    const int off = (t.t * kI4Tile + 16 * g + (PAIR ? i16 & 8 : 0)) & (bs - 1);
    const uint8_t* p = vc + (uint64_t)(uint32_t)(w.v * sh.num_kv_heads + t.kvh) * cell_bytes +
                       (uint32_t)quad_offset(off, C);
#pragma unroll
    for (int tt = 0; tt < T; ++tt) {
      uint32_t c = min(16 * tt + (PAIR ? i16 & 7 : i16), C - 1) * 16;
      asm volatile("" : "+v"(c));
      const uint8_t* row = p + c;
#pragma unroll
      for (int k = 0; k < VQ; ++k) {
        vr[tt][k] = load_stream<uint4>(row);
        row += v_step;
      }
    }
  };

  // ---- the query of a unit: raw rows, then the matrix operand.  Scores in its units: those
  // of base 2 are cs z, cs >= 0 (a negative scale turns the query round).
  uint4 qr[HT][STEPS];
  u4_t qa[HT][STEPS];
  float cs[HT], qn[HT];
  auto load_q = [&](const I4Tile& t) {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int hh = min(t.ch * 16 * HT + ht * 16 + (PAIR ? i16 & 7 : i16), sh.group - 1);
      const uint8_t* row = reinterpret_cast<const uint8_t*>(
          q + ((size_t)t.seq * sh.num_heads + t.kvh * sh.group + hh) * D);
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
        qa[ht][j] = *reinterpret_cast<const u4_t*>(row + k_chunk(j));
    }
  };
  auto convert_q = [&]() {
    const float sgn = sh.scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      float mx = 0.f, sum = 0.f;
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        if (4 * j + g >= C) qa[ht][j] = (u4_t){0, 0, 0, 0};
        const uint32_t w[4] = {qa[ht][j].x, qa[ht][j].y, qa[ht][j].z, qa[ht][j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float lo = widen_lo<BF>(w[k]), hi = widen_hi<BF>(w[k]);
          mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
          sum += lo + hi;
        }
        // (the second pass widens the rows again, as there are no registers to keep them wide)
        asm volatile("" : "+v"(qa[ht][j]));
      }
      mx = head_max(mx);
      sum = head_sum(sum);
      const int e = 15 - __builtin_amdgcn_frexp_expf(mx);   // |q| 2^e < 2^15
      cs[ht] = __builtin_amdgcn_ldexpf(fabsf(sh.scale_log2), 24 - e);
      qn[ht] = __builtin_amdgcn_ldexpf(sgn * sum, e - 24);
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const uint32_t w[4] = {qa[ht][j].x, qa[ht][j].y, qa[ht][j].z, qa[ht][j].w};
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = __builtin_amdgcn_ldexpf(sgn * widen_lo<BF>(w[k]), e);
          x[2 * k + 1] = __builtin_amdgcn_ldexpf(sgn * widen_hi<BF>(w[k]), e - 4);
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

  // One tile, its rows in registers; MORE: the next one's loads go out as registers fall free.
  auto process = [&](auto MORE, int live, const I4Tile& nx, const Where& wn) {
    constexpr bool kMore = decltype(MORE)::value;
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
    if constexpr (kMore) {
      if (!kQueryAhead && nx.t == 0) load_q(nx);
      load_k(nx, wn);
    }
    // the lane's own token's scales; nothing of a token that does not exist
    const bool mine_live = i16 < live;
    const uint32_t kp = mine_live ? ksr : 0u, vp = mine_live ? vsr : 0u;
    const float s_k = widen_lo<false>(kp), m_k = widen_hi<false>(kp);
    const float s_v = widen_lo<false>(vp), m_v = widen_hi<false>(vp);
    // (PAIR: the pairs of the lane's 8 tokens, four in each quad of its 8 lanes)
    const uint32_t kpj[2] = {other_quad<0xA>(kp), other_quad<0x5>(kp)};
    const uint32_t vpj[2] = {other_quad<0xA>(vp), other_quad<0x5>(vp)};
    if constexpr (kMore) load_scales(nx, wn);
    // (2^-24: fp16's smallest step, for rows of one value, whose scale is 0)
    const float log_s = __builtin_amdgcn_logf(fmaxf(row_max(s_v), 0x1p-24f));
    const bool full = __all(live >= 16);
    h8_t phi[HT][VQ / 2], plo[HT][VQ / 2];
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      constexpr int E = PAIR ? 8 : 16;       // the lane's tokens
      float z[E];
      if constexpr (PAIR) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = (i16 & 8) ? sc[ht][n][2 + j] : sc[ht][n][j];
          const float mj = widen_hi<false>(kpj[j]), sj = widen_lo<false>(kpj[j]);
          z[4 * j + 0] = __builtin_fmaf(quad_bcast<0>(sj), x[0], quad_bcast<0>(mj) * qn[ht]);
          z[4 * j + 1] = __builtin_fmaf(quad_bcast<1>(sj), x[1], quad_bcast<1>(mj) * qn[ht]);
          z[4 * j + 2] = __builtin_fmaf(quad_bcast<2>(sj), x[2], quad_bcast<2>(mj) * qn[ht]);
          z[4 * j + 3] = __builtin_fmaf(quad_bcast<3>(sj), x[3], quad_bcast<3>(mj) * qn[ht]);
        }
      } else {
        score8<0>(z, m_k, s_k, qn[ht], sc[ht]);
        score8<8>(z, m_k, s_k, qn[ht], sc[ht]);
      }
      if (!full) {
        asm volatile("");   // (a branch: most tiles are full)
        const int mine = PAIR ? live - (i16 & 8) : live;
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = e < mine ? z[e] : kNegInf;
      }
      float mx = fmaxf(z[0], z[1]);
#pragma unroll
      for (int e = 2; e < E; e += 2) mx = fmaxf(fmaxf(mx, z[e]), z[e + 1]);
      // (a tile without tokens: -inf, also where cs is 0)
      mx = mx == kNegInf ? kNegInf : __builtin_fmaf(mx, cs[ht], log_s);
      mx = head_max(PAIR ? pair_max8(mx) : mx);
      // The reference moves when it is passed by kSlack: the weights then stay below 2^16.
      const bool move = mx > M[ht] + kSlack;
      if (__any(move)) {
        const float f = !move ? 1.f : (M[ht] == kNegInf ? 0.f : exp2f_fast(M[ht] - mx));
        M[ht] = move ? mx : M[ht];
#pragma unroll
        for (int tt = 0; tt < T; ++tt)
#pragma unroll
          for (int n = 0; n < 8; ++n) acc[ht][tt][n] *= f;
        L[ht] *= f;
        B[ht] *= f;
      }
      const float ref = M[ht] == kNegInf ? 0.f : M[ht] - kShift;
#pragma unroll
      for (int hf = 0; hf < E / 8; ++hf) {
        float p[8], w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = exp2f_fast(__builtin_fmaf(z[8 * hf + e], cs[ht], -ref));
          L[ht] += p[e];
        }
        if constexpr (PAIR) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float mj = widen_hi<false>(vpj[j]), sj = widen_lo<false>(vpj[j]);
            w[4 * j + 0] = quad_bcast<0>(sj) * p[4 * j + 0];
            w[4 * j + 1] = quad_bcast<1>(sj) * p[4 * j + 1];
            w[4 * j + 2] = quad_bcast<2>(sj) * p[4 * j + 2];
            w[4 * j + 3] = quad_bcast<3>(sj) * p[4 * j + 3];
            B[ht] = __builtin_fmaf(quad_bcast<0>(mj), p[4 * j + 0], B[ht]);
            B[ht] = __builtin_fmaf(quad_bcast<1>(mj), p[4 * j + 1], B[ht]);
            B[ht] = __builtin_fmaf(quad_bcast<2>(mj), p[4 * j + 2], B[ht]);
            B[ht] = __builtin_fmaf(quad_bcast<3>(mj), p[4 * j + 3], B[ht]);
          }
        } else if (hf == 0) {
          weight8<0>(w, B[ht], m_v, s_v, p);
        } else {
          weight8<8>(w, B[ht], m_v, s_v, p);
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          // (towards zero: the second number holds what that leaves)
          const auto hi = __builtin_amdgcn_cvt_pkrtz(w[e], w[e + 1]);
          const auto lo = __builtin_amdgcn_cvt_pkrtz(w[e] - (float)hi[0], w[e + 1] - (float)hi[1]);
          phi[ht][hf][e] = hi[0];
          phi[ht][hf][e + 1] = hi[1];
          plo[ht][hf][e] = lo[0];
          plo[ht][hf][e + 1] = lo[1];
        }
      }
    }
    // weighted codes
#pragma unroll
    for (int tt = 0; tt < T; ++tt) {
#pragma unroll
      for (int hf = 0; hf < VQ / 2; ++hf) {
        const uint4 a0 = vr[tt][2 * hf], a1 = vr[tt][2 * hf + 1];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x07060302u : 0x05040100u;
          const u4_t w = {
              __builtin_amdgcn_perm(a0.y, a0.x, sel), __builtin_amdgcn_perm(a0.w, a0.z, sel),
              __builtin_amdgcn_perm(a1.y, a1.x, sel), __builtin_amdgcn_perm(a1.w, a1.z, sel)};
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const u4_t x = d < 2 ? w << 2 : w >> 6;
            const h8_t va = __builtin_bit_cast(h8_t, x & ((d & 1) ? 0x03C003C0u : 0x003C003Cu));
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
              f4_t& o = acc[ht][tt][4 * half + d];
              o = mfma16(va, phi[ht][hf], o);
              o = mfma16(va, plo[ht][hf], o);
            }
          }
        }
      }
    }
    if constexpr (kMore) load_v(nx, wn);
  };

  // The state as a piece: sums over the head's lanes, outputs in their own units.
  auto to_piece = [&]() {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      L[ht] = head_sum(PAIR ? pair_sum8(L[ht]) : L[ht]);
      B[ht] = head_sum(PAIR ? pair_sum8(B[ht]) : B[ht]);
      if constexpr (PACK) {
        M[ht] = upper_from(M[ht], M[ht]);
        L[ht] = upper_from(L[ht], L[ht]);
        B[ht] = upper_from(B[ht], B[ht]);
      }
      if constexpr (PACK4) {
        M[ht] = quads_from(M[ht], M[ht], M[ht], M[ht]);
        L[ht] = quads_from(L[ht], L[ht], L[ht], L[ht]);
        B[ht] = quads_from(B[ht], B[ht], B[ht], B[ht]);
      }
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int n = 0; n < (MODE == kWhole ? 8 : 4); ++n)
#pragma unroll
          for (int r = 0; r < (PACK4 ? 2 : 4); ++r) {
            float v = acc[ht][tt][n][r];
            if constexpr (PAIR) {
              // both token halves' sums, dim n in lanes 0 - 31 and dim n + 4 in the others
              const auto w = __builtin_amdgcn_permlane32_swap(fbits(v), fbits(acc[ht][tt][n + 4][r]),
                                                              false, false);
              v = bitsf((uint32_t)w[0]) + dpp_mov<kRowRor8>(bitsf((uint32_t)w[1]));
            }
            if constexpr (PACK) v = upper_from(v, acc[ht][tt][n + 4][r]);
            if constexpr (PACK4)
              v = quads_from(v, acc[ht][tt][n + 4][r], acc[ht][tt][n][r + 2], acc[ht][tt][n + 4][r + 2]);
            acc[ht][tt][n][r] =
                __builtin_fmaf(v, (n & 1) ? kCode24 / 64.f : kCode24 / 4.f, B[ht]);
          }
    }
  };
  auto piece4 = [&](int ht, int tt, int r, int half) {
    return (f4_t){acc[ht][tt][4 * half][r], acc[ht][tt][4 * half + 1][r],
                  acc[ht][tt][4 * half + 2][r], acc[ht][tt][4 * half + 3][r]};
  };
  // Item f of a piece: four dims of the column's head.
  auto item4 = [&](int ht, int tt, int f) {
    return MODE != kWhole ? piece4(ht, tt, f, 0) : piece4(ht, tt, f >> 1, f & 1);
  };
  // Its head tile, and which 8 dims and which half of them it is.
  auto item_head = [&](int f) { return f / (I * T); };
  auto item_chunk = [&](int f) {
    if constexpr (PAIR) return 4 * (g & 1) + f;
    const int row = PACK4 ? (f & 1) + 2 * (i16 >> 3) : (PACK ? f & 3 : (f & 7) >> 1);
    return ((f / I) % T) * 16 + 4 * g + row;
  };
  auto item_half = [&](int f) {
    return PAIR ? g >> 1 : (PACK ? i16 >> 3 : (PACK4 ? (i16 >> 2) & 1 : f & 1));
  };
  const int column = PACK ? i16 & 7 : (PACK4 ? i16 & 3 : i16);   // the column's head
  auto write_out = [&](int seq, int kvh, int ch) {
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int hh = ch * 16 * HT + ht * 16 + column;
      const float inv = L[ht] != 0.f ? 1.f / L[ht] : 0.f;
      if constexpr (MODE != kWhole) {
#pragma unroll
        for (int f = 0; f < G::NF; ++f) {
          const int chunk = item_chunk(f);
          if (hh >= sh.group || chunk >= C) continue;
          const f4_t v = item4(ht, f / I, f % I);
          *reinterpret_cast<uint2*>(out + ((size_t)seq * sh.num_heads + kvh * sh.group + hh) * D +
                                    chunk * 8 + 4 * item_half(f)) =
              make_uint2(pack2<BF>(v[0] * inv, v[1] * inv), pack2<BF>(v[2] * inv, v[3] * inv));
        }
        continue;
      }
      int gq = g;
      asm volatile("" : "+v"(gq));   // (as k_chunk)
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int chunk = 16 * tt + 4 * gq + r;
          if (hh >= sh.group || chunk >= C) continue;
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = pack2<BF>(acc[ht][tt][2 * k][r] * inv, acc[ht][tt][2 * k + 1][r] * inv);
          *reinterpret_cast<uint4*>(
              out + ((size_t)seq * sh.num_heads + kvh * sh.group + hh) * D + chunk * 8) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
  };

  // ---- the wave's tiles
  // (relaxed atomics of the work-group: a volatile's system scope waits for every load under way,
  // the next tile's rows too; 8 x 1000 tokens at 32/8 heads 11.0 -> 10.4 us without that wait)
  auto set_progress = [&](int k) {
    __hip_atomic_store(&sm.progress[wv], k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  auto progress_of = [&](int w) {
    return __hip_atomic_load(&sm.progress[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  int state = count > 0 ? kHasTiles : 0;
  const int t0 = cur.t;
  if (count > 0) {
    if (t0 != 0) {
      state |= kHead;
      if (lane == 0) sm.head[wv] = I4Unit{unit0, cur.n, cur.seq, cur.kvh, cur.ch};
    }
    I4Tile nx = cur;
    Where w = locate(cur, load_ids(cur));
    load_q(cur);
    load_k(cur, w);
    load_scales(cur, w);
    load_v(cur, w);
    int live = w.live;
    Ids idn{{-1, -1, -1, -1}};
    if (count > 1) {
      advance(nx);
      idn = load_ids(nx);
    }
    set_progress(0);
    reset();
    convert_q();
    if (kQueryAhead && count > 1 && nx.t == 0) load_q(nx);
    auto to_slot = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int tt = 0; tt < T; ++tt)
#pragma unroll
          for (int f = 0; f < I; ++f)
            sm.acc[wv][(ht * T + tt) * I + f][lane] = item4(ht, tt, f);
        if (g == 0) sm.ml[wv][ht * 16 + i16] = (f2_t){M[ht], L[ht]};
      }
    };
    // What a unit's last tile, or the wave's, leaves to be done.
    auto finish = [&](bool ends, bool head) {
      to_piece();
      if (head) {
        to_slot();
        if (ends) state |= kHeadEnds;
      } else if (ends) {
        write_out(cur.seq, cur.kvh, cur.ch);
      } else {
        state |= kTail;
      }
    };
    // (head: the unit was begun before the wave, whose tiles it still holds without a break)
    for (int k = 0; k < count - 1; ++k) {
      // Of the SIMD's two waves the one behind goes first (left alone, the older does).
      const int other = __builtin_amdgcn_readfirstlane(progress_of(wv ^ 4));
      if (k <= other) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      set_progress(k + 1);
      w = locate(nx, idn);
      I4Tile nn = nx;
      if (k + 2 < count) {
        advance(nn);
        idn = load_ids(nn);
      }
      process(std::true_type(), live, nx, w);
      if (nx.t == 0) {
        finish(true, (state & kHead) && cur.t == t0 + k);
        reset();
        convert_q();
      }
      live = w.live;
      cur = nx;
      nx = nn;
      if (kQueryAhead && k + 2 < count && nx.t == 0) load_q(nx);
    }
    process(std::false_type(), live, nx, w);
    // (a query asked for may still be on its way as far as the compiler knows: were its registers
    // used for this tile, the tile would wait for it)
    if constexpr (kQueryAhead)
#pragma unroll
      for (int j = 0; j < STEPS; ++j) asm volatile("" : : "v"(qa[0][j]));
    finish(cur.t == cur.n - 1, (state & kHead) && cur.t == t0 + count - 1);
    if (kTogether && (state & (kHead | kTail)) == kTail) {
      to_slot();
      if (lane == 0) sm.tail[wv] = I4Unit{x1 - 1 - cur.t, cur.n, cur.seq, cur.kvh, cur.ch};
    }
  }
  if (lane == 0) sm.state[wv] = state;
  if (threadIdx.x < 2) sm.piece[threadIdx.x].active = 0;
  __syncthreads();

  // What the waves have, a bit each.
  const int st_lane = sm.state[lane & (kI4Waves - 1)];
  auto waves_with = [&](int bit) {
    return (uint32_t)__ballot(lane < kI4Waves && (st_lane & bit) != 0);
  };
  const uint32_t w_tiles = waves_with(kHasTiles), w_head = waves_with(kHead);
  const uint32_t w_ends = waves_with(kHeadEnds), w_tail = waves_with(kTail);
  // The waves with pieces of the unit that wave w has the first of, up to its end; and whether
  // it ends among them.
  auto behind_of = [&](int w, bool from_head, bool& ended) {
    const uint32_t later = from_head ? ~0u << w : ~0u << (w + 1);
    const uint32_t end = w_ends & later;
    ended = end != 0;
    return w_tiles & later & (ended ? (end ^ (end - 1)) : ~0u);   // up to the lowest end
  };

  // ---- units that several waves share.  The wave that began one folds the waves' behind it.
  // Folds the slots of n waves, K at most, into the wave's own state; the reads of all are
  // under way together (unused ones read the first again, weighted 0).
  auto fold_slots = [&](auto KC, const int (&slot)[4], int n) __attribute__((always_inline)) {
    constexpr int K = decltype(KC)::value;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      f2_t ml[K];
      float mx = M[ht], f[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        ml[k] = sm.ml[slot[k]][ht * 16 + i16];
        mx = fmaxf(mx, ml[k].x);
      }
      const float own = M[ht] == kNegInf ? 0.f : exp2f_fast(M[ht] - mx);
      M[ht] = mx;
      L[ht] *= own;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        f[k] = k >= n || ml[k].x == kNegInf ? 0.f : exp2f_fast(ml[k].x - mx);
        L[ht] = __builtin_fmaf(ml[k].y, f[k], L[ht]);
      }
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int i = 0; i < I; ++i) {
          const int n0 = MODE != kWhole ? 0 : 4 * (i & 1), r = MODE != kWhole ? i : i >> 1;
          f4_t s;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] = acc[ht][tt][n0 + e][r] * own;
#pragma unroll
          for (int k = 0; k < K; ++k) s += sm.acc[slot[k]][(ht * T + tt) * I + i][lane] * f[k];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[ht][tt][n0 + e][r] = s[e];
        }
    }
  };
  auto fold_waves = [&](uint32_t members) __attribute__((always_inline)) {
    while (members != 0) {
      int slot[4], n = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (members != 0) {
          slot[k] = __builtin_ctz(members);
          members &= members - 1;
          n = k + 1;
        } else {
          slot[k] = slot[0];
        }
      }
      if (n == 1) fold_slots(std::integral_constant<int, 1>(), slot, n);
      else fold_slots(std::integral_constant<int, 4>(), slot, n);
    }
  };
  auto worker_group = [&](uint32_t x) {          // the last work-group that starts at x or before
    const uint32_t big = R * (Q + 1);
    return (int)(x < big ? x / (Q + 1) : R + (x - big) / Q);
  };
  // The piece of a unit that other work-groups share: into memory, to be counted below.
  auto share = [&](int which) {
    float* slot = ws + (size_t)(2 * b + which) * G::kSlotFloats;
    const auto rs = buf_rsrc(slot, (uint32_t)(G::kSlotFloats * 4));
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
      for (int tt = 0; tt < T; ++tt)
#pragma unroll
        for (int f = 0; f < I; ++f)
          dev_store4(rs, (((ht * T + tt) * I + f) * kWave + lane) * 16, item4(ht, tt, f));
      if (g == 0) {
        const f2_t ml = {M[ht], L[ht]};
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2_t, ml), rs,
                                              G::kPieceFloats * 4 + (ht * 16 + i16) * 8, 0,
                                              kPolicyDevice);
      }
    }
  };
  // Four dims of a head (item f of a piece) as outputs.
  auto store_item = [&](int seq, int kvh, int ch, int f, f4_t s, float l) {
    const int hh = ch * 16 * HT + item_head(f) * 16 + column;
    const int chunk = item_chunk(f);
    if (hh >= sh.group || chunk >= C) return;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    *reinterpret_cast<uint2*>(out + ((size_t)seq * sh.num_heads + kvh * sh.group + hh) * D +
                              chunk * 8 + 4 * item_half(f)) =
        make_uint2(pack2<BF>(s[0] * inv, s[1] * inv), pack2<BF>(s[2] * inv, s[3] * inv));
  };
  auto note_shared = [&](int which, const I4Unit& u) {
    auto& p = sm.piece[which];
    p.active = 1;
    p.first = worker_group(u.begin);
    p.count = worker_group(u.begin + u.n - 1) - p.first + 1;
    p.seq = u.seq;
    p.kvh = u.kvh;
    p.ch = u.ch;
  };
  // A unit's first piece here: one begun, or the first wave's, of a unit begun before.
  const uint32_t lead = w_head & (w_tiles & (0u - w_tiles)), starts = w_tail | lead;
  if (kTogether && (w_head & w_tail) == 0 && (starts & (starts - 1)) == 0) {
    // One unit at most, and every wave's piece of it in its slot: all waves fold them
    // together, four dims of a head per lane.
    if (starts != 0) {
      const int w0 = __builtin_ctz(starts);
      const bool begun = w_tail != 0;
      bool ended;
      const uint32_t members = behind_of(w0, !begun, ended) | starts;
      const I4Unit unit = begun ? sm.tail[w0] : sm.head[w0];
      const int which = begun ? 1 : 0;
#pragma unroll
      for (int q2 = 0; q2 < T * HT; ++q2) {
        const int f = wv + q2 * kI4Waves, h = item_head(f) * 16 + i16;
        if (f >= G::NF) break;
        f2_t ml[kI4Waves];
        f4_t v[kI4Waves];
        float mx = kNegInf, l = 0.f;
#pragma unroll
        for (int k = 0; k < kI4Waves; ++k) {
          const int src = ((members >> k) & 1) ? k : w0;
          ml[k] = sm.ml[src][h];
          v[k] = sm.acc[src][f][lane];
          mx = fmaxf(mx, ml[k].x);
        }
        f4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kI4Waves; ++k) {
          const float e = !((members >> k) & 1) || ml[k].x == kNegInf ? 0.f : exp2f_fast(ml[k].x - mx);
          s += v[k] * e;
          l += ml[k].y * e;
        }
        if (begun && ended) {
          store_item(unit.seq, unit.kvh, unit.ch, f, s, l);
        } else {
          const auto rs = buf_rsrc(ws + (size_t)(2 * b + which) * G::kSlotFloats,
                                   (uint32_t)(G::kSlotFloats * 4));
          dev_store4(rs, (f * kWave + lane) * 16, s);
          if (f % (I * T) == 0 && g == 0) {
            const f2_t p = {mx, l};
            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2_t, p), rs,
                                                  G::kPieceFloats * 4 + h * 8, 0, kPolicyDevice);
          }
        }
      }
      if (!(begun && ended) && threadIdx.x == 0) note_shared(which, unit);
    }
  } else {
    bool ended;
    if (state & kTail) {
      const uint32_t behind = behind_of(wv, false, ended);
      fold_waves(behind);
      if (ended) {
        write_out(cur.seq, cur.kvh, cur.ch);
      } else {
        share(1);
        if (lane == 0) note_shared(1, I4Unit{x1 - 1 - cur.t, cur.n, cur.seq, cur.kvh, cur.ch});
      }
    }
    if (wv == 0 && lead != 0) {
      const int w = __builtin_ctz(lead);
      reset();
      fold_waves(behind_of(w, true, ended));
      share(0);
      if (lane == 0) note_shared(0, sm.head[w]);
    }
  }
  // ---- units that several work-groups share: the last to arrive merges the pieces.
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
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
      const int gi = ((int)b - p.first) / kMergeMax, m0 = p.first + gi * kMergeMax;
      p.last = arrive(cnt + (gi == 0 ? 0 : kI4Groups) + m0, min(kMergeMax, p.first + p.count - m0));
    }
  }
  __syncthreads();
  // Merges n pieces, those of work-groups m0, m0 + step, ..: the output, or one piece in
  // place of the first.
  auto merge_of = [&](auto KC, int first, int m0, int step, int n, bool final_out, int seq, int kvh,
                      int ch) __attribute__((always_inline)) {
    constexpr int K = decltype(KC)::value;
    auto slot_of = [&](int j) {
      const int m = m0 + j * step;
      return ws + (size_t)(2 * m + (m == first ? 1 : 0)) * G::kSlotFloats;
    };
    f4_t A[T * HT];
    float Mi[T * HT], Li[T * HT];
#pragma unroll
    for (int q = 0; q < T * HT; ++q) {
      const int f = wv + q * kI4Waves;
      const int h = item_head(f) * 16 + i16;
      if (f >= G::NF) break;
      float mx = kNegInf, l = 0.f;
      f4_t s = {0.f, 0.f, 0.f, 0.f};
      for (int j0 = 0; j0 < n; j0 += K) {
        f4_t v[K];
        f2_t ml[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
          // (past the last piece it is read again and weighted 0: every load is unconditional)
          const auto rs = buf_rsrc(slot_of(min(j0 + j, n - 1)), (uint32_t)(G::kSlotFloats * 4));
          v[j] = dev_load4(rs, (f * kWave + lane) * 16);
          ml[j] = __builtin_bit_cast(f2_t, __builtin_amdgcn_raw_buffer_load_b64(
                                               rs, G::kPieceFloats * 4 + h * 8, 0, kPolicyDevice));
        }
        const float old = mx;
#pragma unroll
        for (int j = 0; j < K; ++j) mx = fmaxf(mx, ml[j].x);
        const float keep = old == kNegInf ? 0.f : exp2f_fast(old - mx);
        s *= keep;
        l *= keep;
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const float w = j0 + j >= n || ml[j].x == kNegInf ? 0.f : exp2f_fast(ml[j].x - mx);
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
      for (int q = 0; q < T * HT; ++q)
        if (wv + q * kI4Waves < G::NF) store_item(seq, kvh, ch, wv + q * kI4Waves, A[q], Li[q]);
    } else {
      // (each thread rewrites the items that it alone read; the pairs, which all read, after
      // a barrier)
      __syncthreads();
      const auto rs = buf_rsrc(slot_of(0), (uint32_t)(G::kSlotFloats * 4));
#pragma unroll
      for (int q = 0; q < T * HT; ++q) {
        const int f = wv + q * kI4Waves;
        if (f >= G::NF) break;
        dev_store4(rs, (f * kWave + lane) * 16, A[q]);
        if (f % (I * T) == 0 && g == 0) {
          const f2_t ml = {Mi[q], Li[q]};
          __builtin_amdgcn_raw_buffer_store_b64(
              __builtin_bit_cast(u2_t, ml), rs,
              G::kPieceFloats * 4 + (item_head(f) * 16 + i16) * 8, 0, kPolicyDevice);
        }
      }
    }
  };
  auto merge = [&](int first, int m0, int step, int n, bool final_out, int seq, int kvh,
                   int ch) __attribute__((always_inline)) {
    if (n <= 4)
      merge_of(std::integral_constant<int, 4>(), first, m0, step, n, final_out, seq, kvh, ch);
    else
      merge_of(std::integral_constant<int, 8>(), first, m0, step, n, final_out, seq, kvh, ch);
  };
  for (int which = 0; which < 2; ++which) {
    const auto p = sm.piece[which];
    if (!__builtin_amdgcn_readfirstlane(p.last)) continue;
    const int first = __builtin_amdgcn_readfirstlane(p.first);
    const int np = __builtin_amdgcn_readfirstlane(p.count);
    const int seq = __builtin_amdgcn_readfirstlane(p.seq);
    const int kvh = __builtin_amdgcn_readfirstlane(p.kvh), ch = __builtin_amdgcn_readfirstlane(p.ch);
    const int gi = ((int)b - first) / kMergeMax, m0 = first + gi * kMergeMax;
    const int n = min(kMergeMax, first + np - m0);
    if (np <= kMergeMax) {
      merge(first, m0, 1, n, true, seq, kvh, ch);
      continue;
    }
    merge(first, m0, 1, n, false, seq, kvh, ch);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    const int ng = (np + kMergeMax - 1) / kMergeMax;
    if (threadIdx.x == 0) sm.last2 = arrive(cnt + 2 * kI4Groups + first, ng);
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(sm.last2)) merge(first, first, kMergeMax, ng, true, seq, kvh, ch);
    __syncthreads();   // (last2 is written again by the other piece)
  }
}

// MAX_HT = 2 is for groups of more than 16 heads.  Two head tiles read and unpack such a unit's
// rows once for both, but start, fold and merge twice the state, and one wave works where two
// would.  Long lists take them (64 x 16384 tokens at 128/4 heads 145 us against 181, 64 x 8192
// at 64/2 46.4 against 49.3), short ones do not (64 sequences of median 2048 at 32/1 21.8
// against 24.8, 16 of 100-700 10.1 against 16.2); they meet near four to eight tiles a wave.  Wider rows
// have no registers for a second set of outputs.
//
// The first arguments reach the waves in registers; the lengths are loaded while the rest come, whether
// the call is checked among the first.
template <int STEPS, int MAX_HT, int MODE, bool BF>
__global__ void __launch_bounds__(kI4Waves* kWave) __attribute__((amdgpu_waves_per_eu(2)))
decode_int4_kernel(const int32_t* __restrict__ lengths, int num_seqs, int max_blocks, int bs_check,
                   int num_kv_heads, int group, int head_dim, int num_blocks, float scale_log2,
                   const int32_t* __restrict__ table, const uint16_t* __restrict__ q,
                   const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                   const uint32_t* __restrict__ ks, const uint32_t* __restrict__ vs,
                   uint16_t* __restrict__ out, float* __restrict__ ws, uint32_t* __restrict__ cnt,
                   uint64_t* __restrict__ report, uint32_t tag) {
  const int bs_log2 = bs_check & 255;
  const Int4DecodeShape sh{num_seqs, num_kv_heads * group, num_kv_heads, group, head_dim, num_blocks,
                           max_blocks, bs_log2, scale_log2};
  __shared__ I4Smem<STEPS, MAX_HT, MODE> sm;
  const const_i32 ctxl = as_const(lengths), bt = as_const(table);
  const I4Lens lens = i4_lens(ctxl, sh.num_seqs, sh.max_blocks << sh.bs_log2);
  // A checked call's answer goes out at once, while the launch goes on; all leave where it is no.
  if (bs_check & kI4Check) {
    if (blockIdx.x == 0 && threadIdx.x == 0)
      __hip_atomic_store(report, ((uint64_t)tag << 32) | (lens.empty ? 0u : 1u), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_SYSTEM);
    if (lens.empty) return;
  }
  if constexpr (MAX_HT > 1) {
    if (lens.total * (uint32_t)sh.num_kv_heads >= kI4TwoTiles) {
      decode_int4_body<STEPS, 2, kWhole, BF>(sm, lens, bt, ctxl, sh, q, kc, vc, ks, vs, out, ws, cnt);
      return;
    }
  }
  decode_int4_body<STEPS, 1, MODE, BF>(reinterpret_cast<I4Smem<STEPS, 1, MODE>&>(sm), lens, bt, ctxl, sh, q, kc,
                                 vc, ks, vs, out, ws, cnt);
}

namespace {

template <int MAX_HT, int MODE, bool BF>
hipError_t launch_tiles(const Int4Decode& l) {
  decode_int4_kernel<PA_INT4_STEPS, MAX_HT, MODE, BF><<<kI4Groups, kI4Waves * kWave, 0, l.stream>>>(
      l.context_lens, l.shape.num_seqs, l.shape.max_blocks,
      l.shape.bs_log2 | (l.report != nullptr ? kI4Check : 0), l.shape.num_kv_heads, l.shape.group,
      l.shape.head_dim, l.shape.num_blocks, l.shape.scale_log2, l.block_table,
      static_cast<const uint16_t*>(l.q),
      static_cast<const uint8_t*>(l.k_cache), static_cast<const uint8_t*>(l.v_cache),
      static_cast<const uint32_t*>(l.k_scales), static_cast<const uint32_t*>(l.v_scales),
      static_cast<uint16_t*>(l.out), l.workspace, l.counters, l.report, l.tag);
  return hipGetLastError();
}

}  // namespace

template <>
hipError_t launch_int4_decode_steps<PA_INT4_STEPS>(const Int4Decode& l) {
#if PA_INT4_STEPS <= 4
  if (l.shape.group > 16)
    return l.bf16 ? launch_tiles<2, kWhole, true>(l) : launch_tiles<2, kWhole, false>(l);
#endif
#if PA_INT4_STEPS > 2
  if (l.shape.group <= 4)
    return l.bf16 ? launch_tiles<1, kPack4, true>(l) : launch_tiles<1, kPack4, false>(l);
#endif
  constexpr int kFewHeads = PA_INT4_STEPS <= 2 ? kPair : kPack;
  if (l.shape.group <= 8)
    return l.bf16 ? launch_tiles<1, kFewHeads, true>(l) : launch_tiles<1, kFewHeads, false>(l);
  return l.bf16 ? launch_tiles<1, kWhole, true>(l) : launch_tiles<1, kWhole, false>(l);
}

template <>
size_t int4_decode_slot_bytes<PA_INT4_STEPS>(int group) {
  return sizeof(float) * (PA_INT4_STEPS <= 4 && group > 16 ? I4Geo<PA_INT4_STEPS, 2, kWhole>::kSlotFloats
                                                           : I4Geo<PA_INT4_STEPS, 1, kWhole>::kSlotFloats);
}

}  // namespace pa
