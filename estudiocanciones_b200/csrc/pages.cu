// Pages of a KV cache: growing, forking, freeing, copying and compacting them, and the
// RoPE / KV write into them (sm_100a).
//
// The static cache of the reference (app/engine.py:119-121) gives every row its own copy of
// the prompt.  Here K and V lie in a pool [layers, n_pages, Hk, page, hd]; row s of `table`
// lists the pages of sequence s in order (-1 = none), lens[s] is the number of positions it
// holds, refs[p] the number of sequences that hold page p (0 = free).
//
// Bookkeeping (one CTA of 1024 threads): every call first checks its whole list, then either
// applies all of it or sets a bit in `err` and changes nothing.  Free pages are handed out
// lowest number first, in the order of the list, so the result does not depend on scheduling.
// The r-th free page is found by ballots: 16 coalesced loads per thread, 16 x 32 warp counts
// scanned by one warp; a pool of 16384 pages is one round.  Bound by its chain of memory latencies and
// barriers: grow and free take 2.5 to 2.8 us in a graph, the list of a fork 5 to 8, that of a compaction 8 to 10 (it looks
// at the whole table too: 64 sequences of 512 pages cost it 6 more).
// Data (copy kernel, every SM): pure HBM traffic, 2 bytes moved per byte kept.  A warp takes a
// piece of 4 KB (8 x 16 bytes per lane in flight) of one (page, layer, K or V, head).  Only the
// rows that hold positions are copied.  Compacting 128 pages of 4 MB, half of them free (32 pages move, 268 MB
// read and written), takes 58 us with its list and two small copies that restore the table and the counts
// for the next pass (4.9 TB/s); eight forks of 600 positions in 28 layers 17 us.
// The copy kernel reads the list that the bookkeeping kernel wrote, so nothing returns to the
// host and both can be captured.
#include <cuda_bf16.h>

#include "hm_common.cuh"

namespace {

constexpr int kMeta = 1024;      // threads of the bookkeeping CTA, and the longest list
constexpr int kPer = 16;         // reference counts per thread and round
constexpr int kRound = kMeta * kPer;
constexpr int kPiece = 4096;     // bytes a warp copies at a time
constexpr int kCopyThreads = 256;
constexpr int kMaxPages = 1 << 30;  // rounds over the counts stay inside 32 bits

struct PageState {
  int* table;
  int64_t table_ld;
  int n_seqs, max_pages;
  int64_t* lens;
  int* refs;
  int n_pages, page;
  int* err;
};

struct Move {
  int src, dst, rows, pad;
};

// Workspace of the calls that move data: the count, then the list, then (compact) the new
// page numbers.
struct MoveList {
  int* count;
  Move* moves;
  int* map;
};

struct MetaSmem {
  int cnt[kPer][kMeta / 32];   // zero counts per load and warp, then their exclusive prefix
  int warp[kMeta / 32];
  int64_t len[kMeta];
  int a[kMeta], b[kMeta], off[kMeta + 1];
  int bad, total;
};

// Exclusive prefix sum of one value per thread over the CTA; the total goes to *total.
__device__ int block_scan(int v, int* warp_s, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_s and total may still be read from an earlier call
  if (lane == 31) warp_s[w] = x;
  __syncthreads();
  if (w == 0) {
    int s = warp_s[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_s[lane] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) *total = warp_s[31];
  const int before = w ? warp_s[w - 1] : 0;
  __syncthreads();
  return before + x - v;
}

// One round over the counts of pages base .. base + kRound - 1: pred(p) for each, their ranks
// in ascending page order given to use(p, rank) where pred held.  Returns how many held;
// use is called for none of them when they are fewer than `least`.  words (shared memory, if given): a bit
// for each page of the round, whether it held.
template <typename Pred, typename Use>
__device__ int ranked_round(MetaSmem& sm, const int* refs, int n_pages, int base, Pred pred, Use use, int least = 0,
                            uint32_t* words = nullptr) {
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  uint32_t mine[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int p = base + j * kMeta + tid;
    const bool in = p < n_pages;
    const int r = in ? refs[p] : 0;
    mine[j] = __ballot_sync(0xffffffffu, in && pred(p, r));
  }
  __syncthreads();  // sm.cnt and sm.total are free
  if (lane == 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      sm.cnt[j][w] = __popc(mine[j]);
      if (words) words[j * (kMeta / 32) + w] = mine[j];
    }
  }
  __syncthreads();
  if (w == 0) {  // exclusive prefix over the (load, warp) order: lane takes 16 consecutive counts
    int* c = &sm.cnt[0][0] + lane * kPer;
    int s = 0, v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      v[j] = s;
      s += c[j];
    }
    int x = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) c[j] = v[j] + x - s;
    if (lane == 31) sm.total = x;
  }
  __syncthreads();
  const int total = sm.total;
  if (total < least) return total;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if ((mine[j] >> lane) & 1u) use(base + j * kMeta + tid, sm.cnt[j][w] + __popc(mine[j] & ((1u << lane) - 1u)));
  return total;
}
static_assert(kMeta == 1024, "32 warps: one warp scans kPer counts per lane, and the warps' sums");

// give(rank, page) for the `need` lowest free pages, or false (and nothing given) when fewer are free.
// A pool of one round is read once; a larger one is counted first.
template <typename Give>
__device__ bool take_free(MetaSmem& sm, const PageState& P, int need, Give give) {
  auto is_free = [](int, int r) { return r == 0; };
  const bool once = P.n_pages <= kRound;
  int have = once ? need : 0;
  for (int base = 0; base < P.n_pages && have < need; base += kRound)
    have += ranked_round(sm, P.refs, P.n_pages, base, is_free, [](int, int) {});
  if (have < need) return false;
  have = 0;
  for (int base = 0; base < P.n_pages && have < need; base += kRound) {
    const int h = have;
    have += ranked_round(sm, P.refs, P.n_pages, base, is_free,
                         [&](int p, int rank) {
                           if (h + rank < need) give(h + rank, p);
                         },
                         once ? need : 0);
  }
  return have >= need;
}

// The list entry that owns rank r: the last i with off[i] <= r (off ascending, off[n] = total).
__device__ int owner_of(const int* off, int n, int r) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// All of a call or nothing: true when some thread found its part wrong.
__device__ bool any_bad(bool bad, int code, int* err) {
  const bool b = __syncthreads_or(bad);
  if (b && threadIdx.x == 0) report_error(err, code);
  return b;
}

// ------------------------------------------------------------------ grow
__global__ void __launch_bounds__(kMeta) pages_grow_kernel(PageState P, const int* __restrict__ seqs, int n, int add) {
  __shared__ MetaSmem sm;
  const int tid = threadIdx.x;
  int s = -1, need = 0;
  int64_t len = 0;
  bool bad = false;
  if (tid < n) s = seqs[tid];
  sm.a[tid] = s;
  __syncthreads();
  if (s >= 0) {
    bad = s >= P.n_seqs;
    for (int j = 0; j < tid && !bad; ++j) bad = sm.a[j] == s;
    if (!bad) {
      len = P.lens[s];
      bad = len < 0 || len + add > (int64_t)P.max_pages * P.page;
    }
    if (!bad) {
      const int have = static_cast<int>((len + P.page - 1) / P.page);
      need = static_cast<int>((len + add + P.page - 1) / P.page) - have;
      if (len % P.page && add > 0) {  // positions are added to this page: no other sequence may hold it
        const int last = P.table[s * P.table_ld + have - 1];
        bad = last < 0 || last >= P.n_pages || P.refs[last] != 1;
      }
    }
  }
  if (any_bad(bad, HM_ERR_BADINDEX, P.err)) return;
  __shared__ unsigned long long sum;  // 64 bits: the list may ask for more pages than there are
  if (tid == 0) sum = 0;
  __syncthreads();
  if (need) atomicAdd(&sum, static_cast<unsigned long long>(need));
  __syncthreads();
  bool enough = sum <= static_cast<unsigned long long>(P.n_pages);
  if (enough) {
    sm.off[tid] = block_scan(need, sm.warp, &sm.off[kMeta]);
    sm.len[tid] = len;
    __syncthreads();
    enough = take_free(sm, P, static_cast<int>(sum), [&](int rank, int p) {
      const int i = owner_of(sm.off, kMeta, rank);
      const int col = static_cast<int>((sm.len[i] + P.page - 1) / P.page) + rank - sm.off[i];
      P.table[sm.a[i] * P.table_ld + col] = p;
      P.refs[p] = 1;
    });
  }
  if (!enough) {
    if (tid == 0) report_error(P.err, HM_ERR_NOPAGES);
    return;
  }
  if (s >= 0) P.lens[s] = len + add;
}

// ------------------------------------------------------------------ free
__global__ void __launch_bounds__(kMeta) pages_free_kernel(PageState P, const int* __restrict__ seqs, int n) {
  __shared__ MetaSmem sm;
  const int tid = threadIdx.x;
  const int s = tid < n ? seqs[tid] : -1;
  sm.a[tid] = s;
  __syncthreads();
  bool bad = s >= P.n_seqs;
  if (s >= 0)
    for (int j = 0; j < tid && !bad; ++j) bad = sm.a[j] == s;
  if (any_bad(bad, HM_ERR_BADINDEX, P.err)) return;
  // The counts go down first: whether the listed rows hold a page more often than it is counted shows only then.
  // If they do (or name a page that is none), every count goes up again and no row has changed.
  const int64_t cells = (int64_t)n * P.max_pages;
  bad = false;
  for (int64_t c = tid; c < cells; c += kMeta) {
    const int q = sm.a[c / P.max_pages];
    if (q < 0) continue;
    const int p = P.table[q * P.table_ld + c % P.max_pages];
    if (p >= 0) bad |= p >= P.n_pages || atomicSub(&P.refs[p], 1) <= 0;
  }
  const bool undo = any_bad(bad, HM_ERR_BADINDEX, P.err);
  for (int64_t c = tid; c < cells; c += kMeta) {
    const int q = sm.a[c / P.max_pages];
    if (q < 0) continue;
    int* cell = &P.table[q * P.table_ld + c % P.max_pages];
    const int p = *cell;
    if (p < 0) continue;
    if (!undo)
      *cell = -1;
    else if (p < P.n_pages)
      atomicAdd(&P.refs[p], 1);
  }
  if (undo) return;
  if (s >= 0) P.lens[s] = 0;
}

// ------------------------------------------------------------------ fork
__global__ void __launch_bounds__(kMeta) pages_fork_kernel(PageState P, const int* __restrict__ src,
                                                           const int* __restrict__ dst, int n, MoveList W) {
  __shared__ MetaSmem sm;
  const int tid = threadIdx.x;
  pdl_trigger();
  if (tid == 0) *W.count = 0;
  int from = -1, to = -1, part = 0;
  int64_t len = 0;
  if (tid < n) {
    to = dst[tid];
    from = to >= 0 ? src[tid] : -1;
  }
  sm.a[tid] = from;
  sm.b[tid] = to;
  __syncthreads();
  bool bad = false;
  if (to >= 0) {
    bad = to >= P.n_seqs || from < 0 || from >= P.n_seqs;
    for (int j = 0; j < n && !bad; ++j) bad = (j < tid && sm.b[j] == to) || sm.a[j] == to;
    if (!bad) {
      len = P.lens[from];
      bad = P.lens[to] != 0 || len < 0 || len > (int64_t)P.max_pages * P.page;
      part = static_cast<int>(len % P.page);
    }
  }
  if (any_bad(bad, HM_ERR_BADINDEX, P.err)) return;
  sm.len[tid] = len;
  __syncthreads();
  const int64_t cells = (int64_t)n * P.max_pages;
  bad = false;
  for (int64_t c = tid; c < cells; c += kMeta) {
    const int i = static_cast<int>(c / P.max_pages), j = static_cast<int>(c % P.max_pages);
    if (sm.b[i] < 0) continue;
    if ((int64_t)j * P.page < sm.len[i]) {
      const int p = P.table[sm.a[i] * P.table_ld + j];
      bad |= p < 0 || p >= P.n_pages || P.refs[p] <= 0;
    }
  }
  if (any_bad(bad, HM_ERR_BADINDEX, P.err)) return;
  sm.off[tid] = block_scan(part > 0, sm.warp, &sm.off[kMeta]);
  __syncthreads();
  const int total = sm.off[kMeta];
  const bool enough = take_free(sm, P, total, [&](int rank, int p) {
    const int i = owner_of(sm.off, kMeta, rank);
    const int j = static_cast<int>(sm.len[i] / P.page);
    P.table[sm.b[i] * P.table_ld + j] = p;
    P.refs[p] = 1;
    W.moves[rank] = Move{P.table[sm.a[i] * P.table_ld + j], p, static_cast<int>(sm.len[i] % P.page), 0};
  });
  if (!enough) {
    if (tid == 0) report_error(P.err, HM_ERR_NOPAGES);
    return;
  }
  for (int64_t c = tid; c < cells; c += kMeta) {
    const int i = static_cast<int>(c / P.max_pages), j = static_cast<int>(c % P.max_pages);
    if (sm.b[i] < 0) continue;
    int* cell = &P.table[sm.b[i] * P.table_ld + j];
    if ((int64_t)(j + 1) * P.page <= sm.len[i]) {
      const int p = P.table[sm.a[i] * P.table_ld + j];
      atomicAdd(&P.refs[p], 1);
      *cell = p;
    } else if ((int64_t)j * P.page >= sm.len[i]) {
      *cell = -1;
    }
  }
  if (to >= 0) P.lens[to] = len;
  if (tid == 0) *W.count = total;
}

// ------------------------------------------------------------------ copy list
__global__ void __launch_bounds__(kMeta) pages_copy_list_kernel(const int* __restrict__ src, const int* __restrict__ dst,
                                                                int n, int n_pages, int page, MoveList W, int* err) {
  __shared__ MetaSmem sm;
  const int tid = threadIdx.x;
  pdl_trigger();
  if (tid == 0) *W.count = 0;
  const int to = tid < n ? dst[tid] : -1, from = to >= 0 ? src[tid] : -1;
  sm.a[tid] = from;
  sm.b[tid] = to;
  __syncthreads();
  bool bad = false;
  if (to >= 0) {
    bad = to >= n_pages || from < 0 || from >= n_pages;
    for (int j = 0; j < n && !bad; ++j) bad = (j < tid && sm.b[j] == to) || sm.a[j] == to;
  }
  if (any_bad(bad, HM_ERR_BADINDEX, err)) return;
  const int rank = block_scan(to >= 0, sm.warp, &sm.total);
  if (to >= 0) W.moves[rank] = Move{from, to, page, 0};
  __syncthreads();
  if (tid == 0) *W.count = sm.total;
}

// ------------------------------------------------------------------ compact
// Live pages at or above n_live move into the holes below it, i-th to i-th: the fewest moves,
// and sources and targets never overlap.  The table is looked over first: an entry that names a dead page would
// end up naming another sequence's.  Then nothing moves, and n_live is the size of the pool, so that the copy kernel
// renumbers nothing either.
__global__ void __launch_bounds__(kMeta) pages_compact_kernel(PageState P, MoveList W, int* n_live_out) {
  __shared__ MetaSmem sm;
  __shared__ uint32_t live_s[kRound / 32];
  const int tid = threadIdx.x;
  pdl_trigger();
  // The table's cells, kCells of a thread's requested at once, the first ones with the counts: a power of two of
  // threads to a row (no divisions), row by row.
  constexpr int kCells = 4;
  const int lg = P.max_pages <= 32 ? 5 : min(10, 32 - __clz(P.max_pages - 1));
  int col = tid & ((1 << lg) - 1), row = tid >> lg, cell[kCells];
  auto fetch = [&] {
#pragma unroll
    for (int i = 0; i < kCells; ++i) {
      cell[i] = col < P.max_pages && row < P.n_seqs ? P.table[row * P.table_ld + col] : -1;
      row += kMeta >> lg;
      if (row >= P.n_seqs) {
        row = tid >> lg;
        col += 1 << lg;
      }
    }
  };
  fetch();
  int n_live = 0;
  const bool once = P.n_pages <= kRound;  // live_s holds the whole pool
  for (int base = 0; base < P.n_pages; base += kRound)
    n_live += ranked_round(sm, P.refs, P.n_pages, base, [](int, int r) { return r > 0; }, [](int, int) {}, 0, live_s);
  bool bad = false;
  for (;;) {
#pragma unroll
    for (int i = 0; i < kCells; ++i) {
      const int p = cell[i];
      if (p >= 0) bad |= p >= P.n_pages || (once ? !((live_s[p >> 5] >> (p & 31)) & 1u) : P.refs[p] <= 0);
    }
    if (col >= P.max_pages) break;
    fetch();
  }
  if (any_bad(bad, HM_ERR_BADINDEX, P.err)) {
    if (tid == 0) {
      *W.count = 0;
      *n_live_out = P.n_pages;
    }
    return;
  }
  int holes = 0;
  for (int base = 0; base < n_live; base += kRound) {
    const int h = holes;
    holes += ranked_round(sm, P.refs, n_live, base, [](int, int r) { return r <= 0; },
                          [&](int p, int rank) { W.moves[h + rank].dst = p; });
  }
  int movers = 0;
  for (int base = n_live / kRound * kRound; base < P.n_pages; base += kRound) {
    const int h = movers;
    movers += ranked_round(sm, P.refs, P.n_pages, base,
                           [&](int p, int r) {
                             return p >= n_live && r > 0;
                           },
                           [&](int p, int rank) {
                             W.moves[h + rank].src = p;
                             W.moves[h + rank].rows = P.page;
                           });
  }
  __syncthreads();  // the list is complete (holes == movers)
  for (int i = tid; i < movers; i += kMeta) {
    const Move m = W.moves[i];
    W.map[m.src] = m.dst;
    P.refs[m.dst] = P.refs[m.src];
    P.refs[m.src] = 0;
  }
  if (tid == 0) {
    *W.count = movers;
    *n_live_out = n_live;
  }
}

// ------------------------------------------------------------------ data
struct CopyParams {
  uint8_t* k;
  uint8_t* v;
  int64_t layer_bytes, page_bytes;  // strides of the pool
  int layers, Hk, page, row_bytes;
  MoveList W;
  PageState P;   // compact: the table's new numbers (table NULL otherwise)
  const int* n_live;
};

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ CopyParams C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5);
  const int64_t warps = (int64_t)gridDim.x * (kCopyThreads / 32);
  const int count = *C.W.count;
  const int head_bytes = C.page * C.row_bytes;
  const int pieces = (head_bytes + kPiece - 1) / kPiece;
  const int64_t per_move = (int64_t)C.layers * 2 * C.Hk * pieces;
  for (int64_t u = warp; u < per_move * count; u += warps) {
    const Move m = C.W.moves[u / per_move];
    int64_t r = u % per_move;
    const int piece = static_cast<int>(r % pieces);
    r /= pieces;
    const int h = static_cast<int>(r % C.Hk);
    r /= C.Hk;
    uint8_t* const pool = (r & 1) ? C.v : C.k;
    const int64_t at = (r >> 1) * C.layer_bytes + (int64_t)h * head_bytes + (int64_t)piece * kPiece;
    const int left = min(kPiece, m.rows * C.row_bytes - piece * kPiece);  // row_bytes % 16 == 0
    const uint4* s = reinterpret_cast<const uint4*>(pool + m.src * C.page_bytes + at);
    uint4* d = reinterpret_cast<uint4*>(pool + m.dst * C.page_bytes + at);
    uint4 x[kPiece / 512];
#pragma unroll
    for (int i = 0; i < kPiece / 512; ++i)
      if (16 * (i * 32 + lane) < left) x[i] = __ldcs(s + i * 32 + lane);
#pragma unroll
    for (int i = 0; i < kPiece / 512; ++i)
      if (16 * (i * 32 + lane) < left) __stcs(d + i * 32 + lane, x[i]);
  }
  if (C.P.table) {
    const int n_live = *C.n_live;
    const int64_t cells = (int64_t)C.P.n_seqs * C.P.max_pages;
    for (int64_t c = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; c < cells; c += (int64_t)gridDim.x * kCopyThreads) {
      int* cell = &C.P.table[c / C.P.max_pages * C.P.table_ld + c % C.P.max_pages];
      const int p = *cell;
      if (p < n_live) continue;
      if (p < C.P.n_pages) *cell = C.W.map[p];  // (not so only in a table that was refused)
    }
  }
}

// ------------------------------------------------------------------ RoPE and write
template <typename T>
HM_DEV float2 to_f2(uint32_t v);
template <>
HM_DEV float2 to_f2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <>
HM_DEV float2 to_f2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
template <typename T>
HM_DEV uint32_t from_f2(float a, float b);
template <>
HM_DEV uint32_t from_f2<__half>(float a, float b) { return pack_h2(a, b); }
template <>
HM_DEV uint32_t from_f2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// (x0, x1) -> (x0 c - x1 s, x1 c + x0 s): 32 bits, products and sum rounded separately like the
// flat cache's write, then once to the cache's type
template <typename T>
HM_DEV uint32_t rotate2(uint32_t xv, float c, float sn) {
  const float2 x = to_f2<T>(xv);
  return from_f2<T>(__fsub_rn(__fmul_rn(x.x, c), __fmul_rn(x.y, sn)), __fadd_rn(__fmul_rn(x.y, c), __fmul_rn(x.x, sn)));
}

struct RopeParams {
  const void* qkv;
  int64_t ld_qkv;
  const float* rope;
  int rope_rows;
  const int64_t* pos;
  void* q_out;
  int64_t ld_q;
  void* k;
  void* v;
  const int* table;
  int64_t table_ld;
  const int* seqs;
  int n_table, max_pages, n_pages, page;
  int R, S, Hq, Hk, hd;
  int* err;
};

// 8 head dims per thread: a 16-byte load, two 16-byte table loads, a 16-byte store (and the
// V copy beside a K head), coalesced along the row.
template <typename T>
__global__ void __launch_bounds__(256) rope_pages_kernel(const __grid_constant__ RopeParams P) {
  const int cph = P.hd / 8, cpr = (P.Hq + P.Hk) * cph;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= (int64_t)P.R * cpr) return;
  const int r = static_cast<int>(idx / cpr), c = static_cast<int>(idx % cpr);
  const int h = c / cph, j = c % cph;
  const int64_t p = P.pos[r];
  const T* qkv = reinterpret_cast<const T*>(P.qkv) + r * P.ld_qkv + 8 * j;
  T* q_out = reinterpret_cast<T*>(P.q_out) + r * P.ld_q + (int64_t)h * P.hd + 8 * j;
  int page = -1;
  if (p >= 0 && p < (int64_t)P.max_pages * P.page && p < P.rope_rows) {
    const int b = r / P.S, s = P.seqs ? P.seqs[b] : b;
    if (s >= 0 && s < P.n_table) page = P.table[s * P.table_ld + p / P.page];
    if (page >= P.n_pages) page = -1;
  }
  if (page < 0) {  // a padding row (pos < 0), or a position without a page
    if (p >= 0 && c == 0) report_error(P.err, HM_ERR_BADINDEX);
    if (h < P.Hq) *reinterpret_cast<uint4*>(q_out) = make_uint4(0, 0, 0, 0);
    return;
  }
  const float4* t4 = reinterpret_cast<const float4*>(P.rope + (p * (P.hd / 2) + 4 * j) * 2);
  const float4 t0 = t4[0], t1 = t4[1];
  const uint4 xv = *reinterpret_cast<const uint4*>(qkv + (int64_t)h * P.hd);
  uint4 o;
  o.x = rotate2<T>(xv.x, t0.x, t0.y);
  o.y = rotate2<T>(xv.y, t0.z, t0.w);
  o.z = rotate2<T>(xv.z, t1.x, t1.y);
  o.w = rotate2<T>(xv.w, t1.z, t1.w);
  if (h < P.Hq) {
    *reinterpret_cast<uint4*>(q_out) = o;
  } else {
    const int64_t at = (((int64_t)page * P.Hk + (h - P.Hq)) * P.page + p % P.page) * P.hd + 8 * j;
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(P.k) + at) = o;
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(P.v) + at) =
        *reinterpret_cast<const uint4*>(qkv + (int64_t)(h + P.Hk) * P.hd);
  }
}

// ------------------------------------------------------------------ host side
bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }

bool state_ok(const hm_page_state* s) {
  return s && s->table && s->refs && s->n_seqs >= 1 && s->max_pages >= 1 && s->table_ld >= s->max_pages &&
         s->n_pages >= 1 && s->n_pages <= kMaxPages && s->page >= 1 && s->page <= 1024;
}

PageState state_of(const hm_page_state* s) {
  return PageState{s->table, s->table_ld, s->n_seqs, s->max_pages, s->lens, s->refs, s->n_pages, s->page, s->err};
}

bool pool_ok(const hm_page_pool* p) {
  return p && !bad16(p->k) && !bad16(p->v) && p->layers >= 1 && p->n_pages >= 1 && p->n_pages <= kMaxPages &&
         p->Hk >= 1 && p->page >= 1 && p->page <= 1024 && p->row_bytes >= 16 && p->row_bytes % 16 == 0 &&
         (int64_t)p->page * p->row_bytes <= (1 << 24);
}

MoveList list_of(void* ws, int64_t moves) {
  MoveList w;
  w.count = reinterpret_cast<int*>(ws);
  w.moves = reinterpret_cast<Move*>(reinterpret_cast<uint8_t*>(ws) + 16);
  w.map = reinterpret_cast<int*>(w.moves + moves);
  return w;
}

cudaError_t launch_copy(const hm_page_pool* p, MoveList w, int64_t max_moves, const PageState* st, const int* n_live,
                        cudaStream_t stream) {
  CopyParams c = {};
  c.k = reinterpret_cast<uint8_t*>(p->k);
  c.v = reinterpret_cast<uint8_t*>(p->v);
  const int64_t head = (int64_t)p->page * p->row_bytes;
  c.page_bytes = head * p->Hk;
  c.layer_bytes = c.page_bytes * p->n_pages;
  c.layers = p->layers;
  c.Hk = p->Hk;
  c.page = p->page;
  c.row_bytes = p->row_bytes;
  c.W = w;
  if (st) c.P = *st;
  c.n_live = n_live;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  // every warp one piece, at most 8 CTAs (64 warps) per SM
  const int64_t units = max_moves * p->layers * 2 * p->Hk * ((head + kPiece - 1) / kPiece);
  const int64_t want = (units + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  const int grid = static_cast<int>(want < 1 ? 1 : (want < 8 * sms ? want : 8 * sms));
  return hm_launch(pages_copy_kernel, dim3(grid), dim3(kCopyThreads), 0, stream, 1, c);
}

int rc_of(cudaError_t e) { return e == cudaSuccess ? HM_OK : static_cast<int>(e); }

}  // namespace

extern "C" size_t hm_pages_workspace_bytes(int n_moves, int n_pages) {
  if (n_moves < 0 || n_pages < 0) return 0;
  return 16 + (size_t)n_moves * sizeof(Move) + (size_t)n_pages * sizeof(int);
}

extern "C" int hm_pages_grow(const hm_page_state* s, const int* seqs, int n, int add, hm_stream_t stream) {
  if (!state_ok(s) || !s->lens || !seqs || n < 1 || n > kMeta || add < 0) return HM_EARG;
  return rc_of(hm_launch(pages_grow_kernel, dim3(1), dim3(kMeta), 0, stream, 0, state_of(s), seqs, n, add));
}

extern "C" int hm_pages_free(const hm_page_state* s, const int* seqs, int n, hm_stream_t stream) {
  if (!state_ok(s) || !s->lens || !seqs || n < 1 || n > kMeta) return HM_EARG;
  return rc_of(hm_launch(pages_free_kernel, dim3(1), dim3(kMeta), 0, stream, 0, state_of(s), seqs, n));
}

extern "C" int hm_pages_fork(const hm_page_state* s, const hm_page_pool* pool, const int* src, const int* dst, int n,
                             void* ws, size_t ws_bytes, hm_stream_t stream) {
  if (!state_ok(s) || !s->lens || !pool_ok(pool) || pool->n_pages != s->n_pages || pool->page != s->page || !src || !dst || n < 1 ||
      n > kMeta || bad16(ws) || ws_bytes < hm_pages_workspace_bytes(n, 0))
    return HM_EARG;
  const MoveList w = list_of(ws, n);
  cudaError_t e = hm_launch(pages_fork_kernel, dim3(1), dim3(kMeta), 0, stream, 0, state_of(s), src, dst, n, w);
  if (e == cudaSuccess) e = launch_copy(pool, w, n, nullptr, nullptr, stream);
  return rc_of(e);
}

extern "C" int hm_pages_copy(const hm_page_pool* pool, const int* src, const int* dst, int n, void* ws, size_t ws_bytes,
                             int* err, hm_stream_t stream) {
  if (!pool_ok(pool) || !src || !dst || n < 1 || n > kMeta || bad16(ws) || ws_bytes < hm_pages_workspace_bytes(n, 0))
    return HM_EARG;
  const MoveList w = list_of(ws, n);
  cudaError_t e =
      hm_launch(pages_copy_list_kernel, dim3(1), dim3(kMeta), 0, stream, 0, src, dst, n, pool->n_pages, pool->page, w, err);
  if (e == cudaSuccess) e = launch_copy(pool, w, n, nullptr, nullptr, stream);
  return rc_of(e);
}

extern "C" int hm_pages_compact(const hm_page_state* s, const hm_page_pool* pool, int* n_live, void* ws, size_t ws_bytes,
                                hm_stream_t stream) {
  if (!state_ok(s) || !pool_ok(pool) || pool->n_pages != s->n_pages || pool->page != s->page || !n_live || bad16(ws))
    return HM_EARG;
  const int moves = s->n_pages / 2;  // a hole below n_live for every page above it
  if (ws_bytes < hm_pages_workspace_bytes(moves, s->n_pages)) return HM_EARG;
  const MoveList w = list_of(ws, moves);
  const PageState st = state_of(s);
  cudaError_t e = hm_launch(pages_compact_kernel, dim3(1), dim3(kMeta), 0, stream, 0, st, w, n_live);
  if (e == cudaSuccess) e = launch_copy(pool, w, moves, &st, n_live, stream);
  return rc_of(e);
}

extern "C" int hm_rope_pages(const void* qkv, int64_t ld_qkv, const float* rope, int rope_rows, const int64_t* pos,
                             void* q_out, int64_t ld_q, void* k, void* v, int dtype, const int* table, int64_t table_ld,
                             const int* seqs, int n_table, int max_pages, int n_pages, int page, int R, int S, int Hq,
                             int Hk, int hd, int* err, hm_stream_t stream) {
  if (bad16(qkv) || bad16(rope) || bad16(q_out) || bad16(k) || bad16(v) || !pos || !table) return HM_EARG;
  if (R < 1 || S < 1 || Hq < 1 || Hk < 1 || hd < 8 || hd % 8 || rope_rows < 1 || page < 1 || n_pages < 1 ||
      max_pages < 1 || n_table < 1 || table_ld < max_pages)
    return HM_EARG;
  if ((!seqs && (R + S - 1) / S > n_table) || ld_qkv < (int64_t)(Hq + 2 * Hk) * hd || ld_qkv % 8 ||
      ld_q < (int64_t)Hq * hd || ld_q % 8 || (dtype != HM_DT_F16 && dtype != HM_DT_BF16))
    return HM_EARG;
  const RopeParams p{qkv,  ld_qkv, rope,    rope_rows, pos,     q_out, ld_q, k, v,  table, table_ld,
                     seqs, n_table, max_pages, n_pages, page, R,    S,    Hq, Hk, hd,    err};
  const int64_t threads = (int64_t)R * (Hq + Hk) * (hd / 8);
  if ((threads + 255) / 256 > 0x7fffffff) return HM_EARG;
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  return rc_of(dtype == HM_DT_F16 ? hm_launch(rope_pages_kernel<__half>, grid, dim3(256), 0, stream, 0, p)
                                  : hm_launch(rope_pages_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, 0, p));
}
