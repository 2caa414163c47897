// Block tables, slots and positions of a batch's new tokens, on the device (gfx950).
//
//   have_s = ceil(ctx_s / bs),  need_s = ceil((ctx_s + new_s) / bs) - have_s
//   first_s = need_0 + .. + need_{s-1},  cu_s = new_0 + .. + new_{s-1}
//   table[s][have_s + j] = free[num_free - 1 - (first_s + j)],  j < need_s
//   row cu_s + i: position ctx_s + i, slot table[s][position / bs] * bs + position % bs
//
// One launch.  Every work-group scans the batch's lengths itself (a few KB from the
// caches).  Where no sequence gets more than kFew tokens (decode steps) the first one's
// threads place their own sequences' rows; else the prefix sums are kept in LDS and the token
// rows are dealt to all work-groups, each thread finding its sequence by a search there; a
// new block's first row enters it in the table.  A new block's id comes straight from the free
// list, so no work-group reads what another writes.  The lengths and the free count may be updated in place:
// the work-group that arrives last, when all others have read them, writes both.
//
// What bounds it is latency: the launch, two dependent loads, the scan and the stores.
// MI355X, replayed from a graph: one token for each of 256 sequences 3.3 us (6.1 with 1024
// threads, the searches and 64-bit shuffles of a first version), 64 prompts of 98,575 tokens 3.8
// (7.3), in place 6.8.
#include "pa_decode_kernels.hpp"

namespace pa {

constexpr int kExtThreads = 256;
constexpr int kExtPer = kExtendMaxSeqs / kExtThreads;   // sequences of one thread, at most
constexpr int kFew = 4;

struct ExtendArgs {
  int32_t* bt;
  const int32_t* free;
  int32_t *ctx_out, *num_free_out;
  int64_t *slots, *pos;
  int32_t *cu, *status;
  uint32_t* counter;
  int rows;
  bool in_place;
};

// The largest index i < n with pre[i] <= x (pre ascending, pre[0] = 0 <= x); of equal
// entries the last, so a sequence without new rows (blocks) is never found for one.
__device__ __forceinline__ int last_at_most(const int* pre, int n, int x) {
  int lo = 0, hi = n;           // pre[lo] <= x < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Inclusive prefix sum over the wave of counts below 2^31, in 64 bits.
__device__ __forceinline__ long long wave_scan64(uint32_t v) {
  return ((long long)wave_scan_dpp(v >> 16) << 16) + wave_scan_dpp(v & 0xFFFFu);
}

// (The first arguments reach the waves in registers; the lengths are loaded while the rest come.)
template <int PER>
__global__ void __launch_bounds__(kExtThreads)
extend_kernel(const int32_t* ctx_in, const int32_t* new_in, const int32_t* num_free, int seqs,
              int max_blocks, int bs_log2, int free_cap, ExtendArgs a) {
  constexpr int NW = kExtThreads / kWave;
  extern __shared__ int lds[];               // cu, first, ctx of each sequence
  __shared__ long long wsum[2][NW];
  __shared__ int wflag[NW];
  __shared__ bool last;
  const int S = seqs, tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid >> 6;
  const int s0 = tid * PER, bs = 1 << bs_log2;
  int z = 0;
  asm volatile("" : "+v"(z));      // (loaded as the lengths are, with them)
  const int nfree_lane = num_free[z];
  int c[PER], n[PER], need[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = min(s0 + i, S - 1);
    c[i] = ctx_in[s];
    n[i] = new_in[s];
  }
  const int nfree = __builtin_amdgcn_readfirstlane(nfree_lane);
  // (here by now; left alone, the compiler asks for them behind the barrier)
  asm volatile("" : : "s"(a.bt), "s"(a.free), "s"(a.slots), "s"(a.pos), "s"(a.cu), "s"(a.status),
               "s"(a.ctx_out), "s"(a.num_free_out), "s"(a.rows), "s"((int)a.in_place));
  int bad = nfree < 0 || nfree > free_cap ? kExtendBadLength : 0;
  bool many = false;
  long long xn = 0, xb = 0;   // inclusive sums up to this thread, within the wave
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    need[i] = 0;
    if (s0 + i >= S || c[i] < 0 || n[i] < 0) {
      if (s0 + i < S) bad |= kExtendBadLength;
      n[i] = 0;
    } else {
      const long long have = ((long long)c[i] + bs - 1) >> bs_log2;
      const long long want = ((long long)c[i] + n[i] + bs - 1) >> bs_log2;
      if (want > max_blocks || (long long)c[i] + n[i] > INT32_MAX) bad |= kExtendRowFull;
      need[i] = (int)(want - have);
      many |= n[i] > kFew;
    }
    xn += wave_scan64((uint32_t)n[i]);      // (a sum over i of scans is the scan of the sums)
    xb += wave_scan64((uint32_t)need[i]);
  }
  if (lane == kWave - 1) {
    wsum[0][wv] = xn;
    wsum[1][wv] = xb;
  }
  // (all reads of what may be updated in place are over at the barrier)
  // one bit for each reason, and one for a long row of new tokens
  const int f1 = __any(bad & kExtendBadLength) ? kExtendBadLength : 0;
  const int f2 = __any(bad & kExtendRowFull) ? kExtendRowFull : 0;
  const int f3 = __any(many) ? 16 : 0;
  if (lane == 0) wflag[wv] = f1 | f2 | f3;
  __syncthreads();
  long long alln = 0, allb = 0;
  int st = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wv) {
      xn += wsum[0][w];
      xb += wsum[1][w];
    }
    alln += wsum[0][w];
    allb += wsum[1][w];
    st |= wflag[w];
  }
  // (counted now, looked at in the end)
  uint32_t arrived = 0;
  if (tid == 0 && gridDim.x > 1 && a.in_place)
    arrived = __hip_atomic_fetch_add(a.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const bool search = (st & 16) != 0;
  st &= 15;
  if (nfree >= 0 && nfree <= free_cap && allb > nfree) st |= kExtendNoBlocks;
  if (alln > a.rows) st |= kExtendNoRows;
  const int live = st ? 0 : (int)alln, blocks = st ? 0 : (int)allb;
#pragma unroll
  for (int i = PER - 1; i >= 0; --i) {       // exclusive, from the thread's last sequence down
    xn -= n[i];
    xb -= need[i];
    if (search && s0 + i < S) {
      lds[s0 + i] = (int)xn;
      lds[S + s0 + i] = (int)xb;
      lds[2 * S + s0 + i] = c[i];
    }
    if (blockIdx.x == 0 && s0 + i < S) {
      if (a.cu) a.cu[s0 + i] = st ? 0 : (int)xn;
      if (!search && !st) {
        const int have = (c[i] + bs - 1) >> bs_log2;
        int32_t* row = a.bt + (size_t)(s0 + i) * max_blocks;
        for (int k = 0; k < n[i]; ++k) {
          const int p = c[i] + k, b = (p >> bs_log2) - have;
          const int blk = b < 0 ? row[p >> bs_log2] : a.free[nfree - 1 - ((int)xb + b)];
          if (b >= 0 && (p & (bs - 1)) == 0) row[p >> bs_log2] = blk;
          a.slots[(int)xn + k] = (int64_t)blk * bs + (p & (bs - 1));
          if (a.pos) a.pos[(int)xn + k] = p;
        }
      }
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    if (a.cu) a.cu[S] = live;
    *a.status = st;
  }
  const int stride = gridDim.x * kExtThreads;
  int r = blockIdx.x * kExtThreads + tid;
  if (search) {
    __syncthreads();
    const int *cu = lds, *first = lds + S, *ctx = lds + 2 * S;
    for (; r < live; r += stride) {
      const int s = last_at_most(cu, S, r);
      const int c0 = ctx[s], p = c0 + (r - cu[s]);
      const int b = (p >> bs_log2) - ((c0 + bs - 1) >> bs_log2);
      int32_t* entry = a.bt + (size_t)s * max_blocks + (p >> bs_log2);
      const int blk = b < 0 ? *entry : a.free[nfree - 1 - (first[s] + b)];
      if (b >= 0 && (p & (bs - 1)) == 0) *entry = blk;    // (a new block's first token)
      a.slots[r] = (int64_t)blk * bs + (p & (bs - 1));
      if (a.pos) a.pos[r] = p;
    }
  }
  // Rows behind the last token.
  for (; r < a.rows; r += stride)
    if (r >= live) {
      a.slots[r] = -1;
      if (a.pos) a.pos[r] = 0;
    }
  // The new lengths: by the first work-group; in place, when every one has read the old ones
  // (its waves before the barrier above), by the last to arrive.
  if (!a.in_place) {
    if (blockIdx.x != 0) return;
  } else if (gridDim.x > 1) {
    if (tid == 0) last = arrived == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) *a.counter = 0;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (s0 + i < S) a.ctx_out[s0 + i] = c[i] + (st ? 0 : n[i]);
  if (tid == 0) *a.num_free_out = nfree - blocks;
}

hipError_t launch_extend(const ExtendLaunch& l) {
  const bool in_place = l.context_lens_out == l.context_lens || l.num_free_out == l.num_free;
  ExtendArgs a{l.block_table, l.free_blocks, l.context_lens_out, l.num_free_out, l.slot_mapping,
               l.positions, l.cu_seqlens, l.status, l.counter, l.num_rows, in_place};
  // One row a thread; in place fewer work-groups, as their arrivals are counted in one word,
  // one after another (98,575 rows: 64 work-groups 8.3 us, 256 6.8).
  const int most = in_place ? 256 : 512;
  int grid = (l.num_rows + kExtThreads - 1) / kExtThreads;
  grid = grid < 1 ? 1 : (grid > most ? most : grid);
  const size_t lds = 3 * sizeof(int) * l.num_seqs;
  const int per = (l.num_seqs + kExtThreads - 1) / kExtThreads;
  auto* k = per <= 1 ? extend_kernel<1> : (per <= 4 ? extend_kernel<4> : extend_kernel<kExtPer>);
  k<<<grid, kExtThreads, lds, l.stream>>>(l.context_lens, l.new_lens, l.num_free, l.num_seqs,
                                         l.max_blocks, __builtin_ctz((unsigned)l.block_size),
                                         l.free_capacity, a);
  return hipGetLastError();
}

}  // namespace pa
