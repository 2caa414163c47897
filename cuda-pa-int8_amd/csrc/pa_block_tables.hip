// Block tables, slots and positions of a batch's new tokens, on the device (gfx950).
//
//   have_s = ceil(ctx_s / bs),  need_s = ceil((ctx_s + new_s) / bs) - have_s
//   first_s = need_0 + .. + need_{s-1},  cu_s = new_0 + .. + new_{s-1}
//   table[s][have_s + j] = free[num_free - 1 - (first_s + j)],  j < need_s
//   row cu_s + i: position ctx_s + i, slot table[s][position / bs] * bs + position % bs
//
// One launch.  Every work-group scans the batch's lengths itself (a few KB from the
// caches) and keeps the prefix sums in LDS; the token rows and the new table entries are then
// dealt to all of them, each finding its sequence by a search in LDS.  A new block's id
// comes straight from the free list, so no work-group reads what another writes.  The
// lengths and the free count may be updated in place: the work-group that arrives
// last, when all others have read them, writes both.  What bounds it is latency: the launch,
// two dependent loads, the scan and the stores.
#include "pa_int4.hpp"

namespace pa {

constexpr int kExtThreads = 1024;
constexpr int kExtPer = kExtendMaxSeqs / kExtThreads;   // sequences of one thread, at most

struct ExtendArgs {
  int32_t* bt;
  const int32_t *ctx, *nw, *free, *num_free;
  int32_t *ctx_out, *num_free_out;
  int64_t *slots, *pos;
  int32_t *cu, *status;
  uint32_t* counter;
  int seqs, max_blocks, bs_log2, rows, free_cap;
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

__global__ void __launch_bounds__(kExtThreads) extend_kernel(ExtendArgs a) {
  extern __shared__ int lds[];               // cu, first, ctx of each sequence
  __shared__ long long wsum[2][kExtThreads / kWave];
  __shared__ int flags;
  __shared__ bool last;
  const int S = a.seqs, tid = threadIdx.x, lane = tid & (kWave - 1), wv = tid >> 6;
  int *cu = lds, *first = lds + S, *ctx = lds + 2 * S;
  const int per = (S + kExtThreads - 1) / kExtThreads, s0 = tid * per;
  const int bs = 1 << a.bs_log2;
  if (tid == 0) flags = 0;
  const int nfree = *a.num_free;
  int n[kExtPer], need[kExtPer];
  long long tn = 0, tb = 0;
  int bad = 0;
#pragma unroll
  for (int i = 0; i < kExtPer; ++i) {
    n[i] = need[i] = 0;
    const int s = s0 + i;
    if (i < per && s < S) {
      const int c = a.ctx[s], w = a.nw[s];
      ctx[s] = c;
      if (c < 0 || w < 0) {
        bad |= kExtendBadLength;
      } else {
        const long long have = ((long long)c + bs - 1) >> a.bs_log2;
        const long long want = ((long long)c + w + bs - 1) >> a.bs_log2;
        if (want > a.max_blocks || (long long)c + w > INT32_MAX) bad |= kExtendRowFull;
        n[i] = w;
        need[i] = (int)(want - have);
        tn += w;
        tb += want - have;
      }
    }
  }
  // Exclusive scan over the threads: a wave's lanes by shuffles, the waves through LDS.
  long long xn = tn, xb = tb;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const long long yn = __shfl_up(xn, o, kWave), yb = __shfl_up(xb, o, kWave);
    if (lane >= o) {
      xn += yn;
      xb += yb;
    }
  }
  if (lane == kWave - 1) {
    wsum[0][wv] = xn;
    wsum[1][wv] = xb;
  }
  __syncthreads();
  long long alln = 0, allb = 0;
  for (int w = 0; w < kExtThreads / kWave; ++w) {
    if (w == wv) {
      xn += alln;
      xb += allb;
    }
    alln += wsum[0][w];
    allb += wsum[1][w];
  }
  if (nfree < 0 || nfree > a.free_cap) bad |= kExtendBadLength;
  else if (allb > nfree) bad |= kExtendNoBlocks;
  if (alln > a.rows) bad |= kExtendNoRows;
  if (bad) atomicOr(&flags, bad);
  long long en = xn - tn, eb = xb - tb;
#pragma unroll
  for (int i = 0; i < kExtPer; ++i) {
    const int s = s0 + i;
    if (i < per && s < S) {
      cu[s] = (int)en;
      first[s] = (int)eb;
      en += n[i];
      eb += need[i];
    }
  }
  __syncthreads();
  const int st = flags;
  const int live = st ? 0 : (int)alln, blocks = st ? 0 : (int)allb;
  const int stride = gridDim.x * kExtThreads;
  // New table entries, then the rows.
  for (int e = blockIdx.x * kExtThreads + tid; e < blocks; e += stride) {
    const int s = last_at_most(first, S, e);
    const int have = (ctx[s] + bs - 1) >> a.bs_log2;
    a.bt[(size_t)s * a.max_blocks + have + (e - first[s])] = a.free[nfree - 1 - e];
  }
  for (int r = blockIdx.x * kExtThreads + tid; r < a.rows; r += stride) {
    int64_t slot = -1, p = 0;
    if (r < live) {
      const int s = last_at_most(cu, S, r);
      const int c = ctx[s], pos = c + (r - cu[s]);
      const int j = (pos >> a.bs_log2) - ((c + bs - 1) >> a.bs_log2);
      const int blk = j < 0 ? a.bt[(size_t)s * a.max_blocks + (pos >> a.bs_log2)]
                            : a.free[nfree - 1 - (first[s] + j)];
      slot = (int64_t)blk * bs + (pos & (bs - 1));
      p = pos;
    }
    a.slots[r] = slot;
    if (a.pos) a.pos[r] = p;
  }
  if (blockIdx.x == 0) {
    if (a.cu) {
      for (int s = tid; s < S; s += kExtThreads) a.cu[s] = st ? 0 : cu[s];
      if (tid == 0) a.cu[S] = live;
    }
    if (tid == 0) *a.status = st;
  }
  // In-place outputs: by the last arrival, with every work-group's reads behind it (their
  // values have been used, in the scan above).
  if (gridDim.x > 1) {
    if (tid == 0)
      last = __hip_atomic_fetch_add(a.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) *a.counter = 0;
  }
#pragma unroll
  for (int i = 0; i < kExtPer; ++i) {
    const int s = s0 + i;
    if (i < per && s < S) a.ctx_out[s] = ctx[s] + (st ? 0 : n[i]);
  }
  if (tid == 0) *a.num_free_out = nfree - blocks;
}

hipError_t launch_extend(const ExtendLaunch& l) {
  ExtendArgs a{l.block_table, l.context_lens, l.new_lens, l.free_blocks, l.num_free,
               l.context_lens_out, l.num_free_out, l.slot_mapping, l.positions, l.cu_seqlens,
               l.status, l.counter, l.num_seqs, l.max_blocks,
               __builtin_ctz((unsigned)l.block_size), l.num_rows, l.free_capacity};
  // (two rows a thread; the scan, repeated by each work-group, is what more of them cost)
  int grid = (l.num_rows + 2 * kExtThreads - 1) / (2 * kExtThreads);
  grid = grid < 1 ? 1 : (grid > 256 ? 256 : grid);
  extend_kernel<<<grid, kExtThreads, 3 * sizeof(int) * (l.num_seqs > 0 ? l.num_seqs : 1),
                  l.stream>>>(a);
  return hipGetLastError();
}

}  // namespace pa
