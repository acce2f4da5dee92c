// Decode attention of a batch whose sequences share a long prefix, over a paged KV cache (sm_100a).
//
//   o[r, h] = sum_{p <= pos[r]} softmax_p(q[r, h] . k[p] * scale) v[p],  k, v of KV head h / G
//
// Positions [0, plen[g]) of group g are the same pages for every sequence of the group, so they
// are read once and multiplied with the queries of all its rows; positions [plen[g], pos[r]] are
// the sequence's own.  The two ranges, and every split of them, leave partial results
//   m = max_p s_p,  l = sum_p 2^(s_p - m),  a = sum_p 2^(s_p - m) v[p]     (s in units of log 2)
// which join exactly: with M = max m_i,  o = sum_i a_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
//
// What bounds it: K and V are read once per group and once per sequence, 4 * Hk * hd bytes a
// position, against 4 * Hq * hd operations a (row, position).  The kernel is built to keep the
// memory busy and the tensor cores off the critical path:
//  * The work is a list of jobs (one sequence's own positions or a group's prefix, cut into blocks
//    of query rows) x KV heads x tiles of 64 positions.  Lengths live on the device, so every CTA
//    builds the list itself (one pass over pos, a scan in shared memory) and takes an equal share
//    of the tiles: a long prefix next to short sequences leaves no SM idle, whatever the lengths.
//  * One producer warp fetches page numbers 32 at a time and issues one TMA box per page and
//    operand (128-byte swizzle) into a ring of 96 KB per CTA, two CTAs per SM, across job
//    boundaries, so the ring never drains.  It also works out what each run of tiles belongs to
//    and hands that over before the tiles arrive.
//  * Blocks of up to 16 query rows (the G heads of a KV head x rows; every sequence's own positions
//    in a decode step): mma.sync, each of the four consumer warps takes 16 of the tile's
//    positions, so K and V leave shared memory once; the four partial results meet there.
//  * Blocks of up to 128 rows (a prefix and the rows that share it): tcgen05.  Q and the
//    probabilities are the TMEM operands A of S = Q K^T and O += P V, K and V are read where TMA put
//    them; one thread per row does the softmax.  P replaces S in TMEM, so S, Q and O of a CTA take
//    256 columns (hd 128) and two CTAs share an SM: one's softmax runs beside the other's products.
//    O is rescaled only when a row's maximum has grown by more than 2^8 (its reference stays a
//    little behind: P <= 256, the result does not depend on it), which is rare after a few tiles.
//    Calls in a graph, us (1 row on 512 positions / 8 rows, two prefixes of 600 / 64 rows on 4096 / 16 rows, two
//    prefixes of 30001): 10.0 / 14.5 / 42.6 / 68.9; with every block on mma.sync, 16 rows each, 10.0 / 19.6 /
//    91.5 / 108; with every block on tcgen05 12.4 / 18.6 / 58.1 / 78.8.  Several rows a sequence: 8 x 8 rows behind a prefix of
//    600 26.9, two prompts of 512 65, one of 1024 84.
//  * A second small kernel joins the partial results of a row in a fixed order (results do not
//    depend on scheduling) and writes o; its launch overlaps the first kernel's tail.
//  * A row that ends inside its group's prefix takes no part in it and reads all its pages itself, so
//    every row of a prefix job sees all of it. Where the rows of one sequence (S > 1) end at different
//    positions, a V that is not finite must not reach the rows that do not see it (0 * inf): tiles
//    that some row sees only in part are looked over, and the products of such a V are added row by
//    row. Calls with one row per sequence run a variant without that code (kSpread): its registers
//    and instructions cost a call of 16 sequences on long prefixes 11 % although it never ran.
//  * What it spends now: the ring alone (no products) takes 22.3 of the 42.6 us and 53.8 of the 68.7 (312 MB: 5.8
//    TB/s; 4.5 TB/s with the products); a tile of 16 rows costs a CTA ~1500 cycles, one of 24 rows ~2600, one of 128
//    ~3800, a run of a large block ~9000 more (Q waits behind the ring's loads, the result is 64 KB). Shares
//    weighted by these costs were slower (49.6 and 77.4 us): they make more such runs.
// Scores, m, l and a are fp32; the probabilities are rounded to the cache's type for the product
// with V, as the flat decode attention does (l keeps the unrounded sum).  V rows outside a job's
// range are zeroed (in registers, in shared memory for tcgen05), so whatever stands there (NaN
// included) has no effect.
#include <cuda_bf16.h>

#include <atomic>

#include "hm_common.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int kTile = 64;       // positions per tile
constexpr int kMaxJobs = 1024;  // jobs of a call (the list lives in shared memory)
constexpr int kMaxPre = 640;    // prefix jobs, and groups, of a call
constexpr int kMaxRows = 16384; // query rows of a call
constexpr int kThreads = 192;   // 4 consumer warps, the producer, the tcgen05 issuer
constexpr int kCons = 128;
constexpr int kBig = 128;       // rows of a tcgen05 block

struct Params {
  const void* q;
  int64_t ld_q;
  void* o;
  int64_t ld_o;
  const int64_t* pos;
  const int* table;
  int64_t table_ld;
  const int* seqs;
  const int* gstart;
  const int* owner;
  const int* plen;
  int R, S, B, Hq, Hk, G, n_table, max_pages, n_pages, page, n_groups;
  int sub_shift;      // log2 of the positions per TMA box (at most a page, at most a tile)
  float scale;        // scale * log2(e)
  int n_jobs;         // own jobs, then room for the prefix jobs
  int own_blocks;     // row blocks of one sequence's own job
  int own_rows;       // row capacity of an own partial
  int pre_rows;       // row capacity of a prefix partial
  int big;            // some block may have more than 16 rows
  int64_t pre_slots;  // prefix partials come first
  int* plan;          // what the join needs of the job list
  float* pm;          // [rows] maxima, [rows] sums, [rows][hd] accumulators
  float* pl;
  float* pa;
  int* err;
};

// plan: 0 a CTA's share of the tiles, 1 groups unusable; then the tiles before every job (per KV head)
constexpr int kPlanScan = 2, kPlanInts = 2 + kMaxJobs + 1;
#define HM_HD __host__ __device__ __forceinline__

// ---------------------------------------------------------------- types
template <typename T>
struct Ty;
template <>
struct Ty<__half> {
  static constexpr uint32_t kFormat = 0;  // of tcgen05 operands A and B
  static constexpr uint32_t kExp = 0x7c00u;
  static HM_DEV float2 f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static HM_DEV uint32_t pack(float a, float b) { return pack_h2(a, b); }
  static HM_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <>
struct Ty<__nv_bfloat16> {
  static constexpr uint32_t kFormat = (1u << 7) | (1u << 10);
  static constexpr uint32_t kExp = 0x7f80u;
  static HM_DEV float2 f2(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
  static HM_DEV uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static HM_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Whether one of 8 values is an infinity or NaN.
template <typename T>
HM_DEV bool odd16(uint4 v) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    odd |= (u[i] & Ty<T>::kExp) == Ty<T>::kExp || ((u[i] >> 16) & Ty<T>::kExp) == Ty<T>::kExp;
  return odd;
}

// Whether 64 bytes of each 64-dim part of a V row (from `row`, parts `half` bytes apart) hold an infinity
// or NaN.  Out of line, like the products of such values below: their registers and instructions stay
// out of the loops that hardly ever need them.
template <typename T, int PARTS>
__device__ __noinline__ bool odd_row(const uint8_t* row, uint32_t half) {
  bool odd = false;
  for (int h = 0; h < PARTS; ++h)
    for (int k = 0; k < 4; ++k) odd |= odd16<T>(*reinterpret_cast<const uint4*>(row + h * half + 16 * k));
  return odd;
}

// Barrier over the first `n` threads of the CTA that returns whether any of them passed true.
HM_DEV bool named_bar_or(int id, int n, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(static_cast<uint32_t>(p))
      : "memory");
  return r != 0;
}

HM_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- lengths and groups
// Block size of a job with `rows` query rows per KV head.
HM_HD int block_rows(int rows) { return rows <= 16 ? 16 : kBig; }
// Positions that row r attends to: 0 for a padding row and for one whose position or table row
// is out of range (reported).
HM_DEV int row_len(const Params& P, int r) {
  const int64_t p = P.pos[r];
  const int b = r / P.S, s = P.seqs ? P.seqs[b] : b;
  if (p < 0) return 0;
  if (p >= (int64_t)P.max_pages * P.page || s < 0 || s >= P.n_table) {
    report_error(P.err, HM_ERR_BADINDEX);
    return 0;
  }
  return static_cast<int>(p) + 1;
}

// Prefix length of a group: 0 when its entry is out of range (reported).
HM_DEV int group_plen(const Params& P, int g) {
  const int n = P.plen[g], own = P.owner[g];
  if (n == 0) return 0;
  if (n < 0 || n > (int64_t)P.max_pages * P.page || own < 0 || own >= P.n_table) {
    report_error(P.err, HM_ERR_BADINDEX);
    return 0;
  }
  return n;
}

// The group of sequence b (gs: ascending boundaries), -1 for none.
HM_DEV int group_of(const int* gs, int n_groups, int b) {
  int lo = 0, hi = n_groups;  // the first boundary above b
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (gs[mid + 1] <= b)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < n_groups && gs[lo] <= b ? lo : -1;
}

// One job: query rows i0 .. i0 + M - 1 of `row0` (i -> row row0 + i / G, head kh * G + i % G) over
// the positions [lo, hi) of table row `trow`.  mt: rows of the block; plen: the group's prefix.
struct Job {
  int row0, i0, M, lo, hi, trow, mt, plen;
};

// The first prefix job of a group whose sequences start at a: a group of n rows has at most
// n / 128 + 1 jobs, so these numbers leave room for all of them without a scan.
HM_DEV int group_job(const Params& P, int n_own, int g, int a) { return n_own + a * P.S * P.G / kBig + g; }

// Block blk of a group's prefix (sequences a .. b - 1), and of sequence b's own positions behind it.
// Their ranges follow from the rows' lengths, see own_range and prefix_range.
HM_DEV Job prefix_job(const Params& P, int blk, int a, int b, int plen) {
  Job J;
  const int rows = (b - a) * P.S * P.G;
  J.row0 = a * P.S;
  J.lo = J.hi = 0;
  J.plen = plen;
  J.mt = block_rows(rows);
  J.i0 = blk * J.mt;
  J.M = min(J.mt, rows - J.i0);
  return J;
}
HM_DEV Job own_job(const Params& P, int blk, int b, int plen) {
  Job J;
  const int rows = P.S * P.G;
  J.row0 = b * P.S;
  J.lo = J.hi = 0;
  J.plen = plen;
  J.mt = block_rows(rows);
  J.i0 = blk * J.mt;
  J.M = min(J.mt, rows - J.i0);
  return J;
}
// top: the largest length of the job's rows, low: the smallest of those above 0 (else INT_MAX).
HM_DEV void own_range(Job& J, int top, int low) {
  J.lo = low < J.plen ? 0 : J.plen;  // a row that ends inside the prefix reads its own pages from the start
  J.hi = top;
}
HM_DEV void prefix_range(Job& J, int top) { J.hi = top >= J.plen ? J.plen : 0; }
HM_DEV int low_of(int len) { return len > 0 ? len : 0x7fffffff; }
// First and last query row of a job.
HM_DEV int row_first(const Params& P, const Job& J) { return J.row0 + J.i0 / P.G; }
HM_DEV int row_last(const Params& P, const Job& J) { return J.row0 + (J.i0 + J.M - 1) / P.G; }
HM_DEV int tiles_of(const Job& J) { return J.hi > J.lo ? (J.hi - 1) / kTile - J.lo / kTile + 1 : 0; }

// ---------------------------------------------------------------- shared memory
template <int HD>
struct Cfg {
  static constexpr int kOperand = kTile * HD * 2;  // bytes of a K (or V) tile
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kCtas = HD <= 128 ? 2 : 1;  // per SM
  static constexpr bool kQSmem = HD > 128;         // query fragments: registers, or shared memory
  static constexpr int kQPitch = HD * 2 + 16;
  // TMEM columns of a tcgen05 block: S (then P) 64, Q hd / 2, O hd
  static constexpr uint32_t kTmem = HD <= 128 ? 256 : 512, kTmemQ = 64, kTmemO = 64 + HD / 2;
  static_assert(kTmemO + HD <= kTmem, "TMEM");
};

// A run of tiles of one (job, KV head), as the producer hands it to the consumers.
struct Run {
  Job J;
  int kh, tile, tiles;  // first tile (of the cache), their number
  int slot, prefix;     // number of the partial result among those of its kind
};
// Entries of the hand-over.  Entry n + 8 is written after the first tile of run n + 7 was issued, that
// is, after the tile kStages (<= 6) before it was consumed by all warps: run n is over by then.
constexpr int kRuns = 8;

template <int HD>
struct Smem {
  uint8_t kv[Cfg<HD>::kStages][2][Cfg<HD>::kOperand];
  // four rows of each warp's partial result; for blocks of up to 128 rows 16 columns (64 bytes) of each
  float red[4][4][HD < 128 ? 128 : HD];
  uint8_t q[Cfg<HD>::kQSmem ? 16 * Cfg<HD>::kQPitch : 16];
  int scan[kMaxJobs + 1];
  int ids[kMaxPre];     // prefix jobs: group and block
  Run run[kRuns];
  float mw[4][16], lw[4][16];
  uint64_t full[Cfg<HD>::kStages], empty[Cfg<HD>::kStages], run_full[kRuns];
  uint64_t s_full[2], o_full[2];  // tcgen05, a half tile: S = Q K^T, O += P V done
  uint64_t q_full, p_full[2];     // Q, P in TMEM (each consumer warp)
  uint32_t tmem;
  int bad[Cfg<HD>::kStages];  // 16-position blocks of the stage without a page
  int abort_flag;
};
static_assert(sizeof(Smem<64>::red) >= kBig * 64, "64 bytes of every row of a block");
static_assert(sizeof(Smem<128>) + 1024 <= 233472 / 2, "two CTAs per SM at hd 128");
static_assert(sizeof(Smem<64>) + 1024 <= 233472 / 2, "two CTAs per SM at hd 64");
static_assert(sizeof(Smem<256>) <= 227 * 1024, "shared memory at hd 256");
// the ring doubles as scratch while the job list is built: row lengths, group boundaries, prefixes
static_assert((kMaxRows + 2 * kMaxPre + 1) * sizeof(int) <= 6 * 2 * kTile * 64 * 2, "scratch");

// The job list: scan[j] = tiles of the jobs before j (per KV head), own jobs first.  All threads of the
// CTA; everything it needs from memory is requested first, in one go.  Returns whether the groups
// are unusable (their boundaries do not ascend inside the batch: reported, nobody shares anything).
template <int HD>
HM_DEV bool build_jobs(const Params& P, Smem<HD>& sm) {
  const int tid = threadIdx.x, lane = tid & 31;
  int* const len = reinterpret_cast<int*>(&sm.kv[0][0][0]);
  int* const gs = len + kMaxRows;
  int* const gp = gs + kMaxPre + 1;
  const int n_own = P.B * P.own_blocks, n_jobs = P.n_jobs;
  bool bad = false;
  // (rows from the first thread on, groups from the last: on small calls no thread waits twice)
  for (int g = kThreads - 1 - tid; g < P.n_groups; g += kThreads) {
    const int a = P.gstart[g], b = P.gstart[g + 1];
    gp[g] = group_plen(P, g);
    gs[g] = a;
    if (g == P.n_groups - 1) gs[g + 1] = b;
    bad |= a < 0 || a > b || b > P.B;
  }
  for (int r = tid; r < P.R; r += kThreads) len[r] = row_len(P, r);
  for (int j = n_own + tid; j < n_jobs; j += kThreads) sm.scan[j] = 0;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) report_error(P.err, HM_ERR_BADINDEX);
  // eight lanes share a job's rows (one where a block is one row)
  const bool single = P.S == 1 && P.own_blocks == 1;
  const int step = single ? 1 : 8, mine = tid & (step - 1);
  for (int j0 = 0; j0 < n_own; j0 += kThreads / step) {
    const int j = j0 + tid / step;
    Job J = {};
    int top = 0, low = 0x7fffffff;
    if (j < n_own) {
      const int b = P.own_blocks == 1 ? j : j / P.own_blocks;
      const int g = bad ? -1 : group_of(gs, P.n_groups, b);
      J = own_job(P, j - b * P.own_blocks, b, g < 0 ? 0 : gp[g]);
      for (int r = single ? b : row_first(P, J) + mine, e = single ? b : row_last(P, J); r <= e; r += 8) {
        top = max(top, len[r]);
        low = min(low, low_of(len[r]));
      }
    }
    if (!single) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      }
    }
    own_range(J, top, low);
    if (j < n_own && mine == 0) sm.scan[j] = tiles_of(J);
  }
  // a warp per group (the last warp first, see above), eight lanes per block of its rows
  for (int g = (kThreads - 1 - tid) >> 5; g < P.n_groups && !bad; g += kThreads / 32) {
    const int plen = gp[g], a = gs[g], b = gs[g + 1];
    if (plen == 0) continue;
    const int rows = (b - a) * P.S * P.G, mt = block_rows(rows), first = group_job(P, n_own, g, a);
    for (int m0 = 0; m0 * mt < rows; m0 += 4) {
      const int blk = m0 + (lane >> 3);
      Job J = prefix_job(P, blk, a, b, plen);
      int top = 0;
      if (J.M > 0)
        for (int r = row_first(P, J) + (lane & 7); r <= row_last(P, J); r += 8) top = max(top, len[r]);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      prefix_range(J, top);
      if (J.M > 0 && (lane & 7) == 0) {
        sm.scan[first + blk] = tiles_of(J);
        sm.ids[first + blk - n_own] = g | (blk << 16);
      }
    }
  }
  __syncthreads();
  if (tid < 32) {
    const int per = (n_jobs + 31) / 32, j0 = min(lane * per, n_jobs), j1 = min(j0 + per, n_jobs);
    int s = 0;
    for (int j = j0; j < j1; ++j) s += sm.scan[j];
    int x = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    int at = x - s;
    for (int j = j0; j < j1; ++j) {
      const int t = sm.scan[j];
      sm.scan[j] = at;
      at += t;
    }
    if (lane == 31) sm.scan[n_jobs] = x;
  }
  // the scratch was written by threads; TMA writes it next
  fence_proxy_async_smem();
  __syncthreads();
  return bad;
}

// The job that holds tile x of the flat order (scan * Hk + kh * tiles + t): the last that starts at or
// before it (jobs without tiles in front of it share its start).
HM_DEV int job_at(const int* scan, int n_jobs, int64_t x, int Hk) {
  int lo = 0, hi = n_jobs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)scan[mid] * Hk <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Byte offset of positions 16 * b .. of a tile in its boxes of 2^shift positions, each
// [64-dim part][position][128 bytes].
template <int HD>
HM_DEV uint32_t block_at(int shift, int b) {
  const int p = 16 * b;
  return (static_cast<uint32_t>(p >> shift) << shift) * 128u * (HD / 64) + static_cast<uint32_t>(p & ((1 << shift) - 1)) * 128u;
}

// A lane's share of acc += P V in the MMA's layout (rows g and g + 8 of w, columns 8 n + 2 t, + 1 of V),
// over the positions in see0 / see1 only.
template <int HD, typename T>
__device__ __noinline__ void rows_product(float* acc, const float* w, const uint8_t* v, uint32_t half, uint32_t see0,
                                          uint32_t see1) {
  for (int p = 0; p < 16; ++p) {
    for (int n = 0; n < HD / 8; ++n) {
      const float2 x =
          Ty<T>::f2(*reinterpret_cast<const uint32_t*>(v + (n / 8) * half + p * 128 + (((n % 8) ^ (p & 7)) << 4)));
      if ((see0 >> p) & 1) {
        acc[4 * n] += w[p] * x.x;
        acc[4 * n + 1] += w[p] * x.y;
      }
      if ((see1 >> p) & 1) {
        acc[4 * n + 2] += w[128 + p] * x.x;
        acc[4 * n + 3] += w[128 + p] * x.y;
      }
    }
  }
}

// ---------------------------------------------------------------- blocks of up to 16 rows
// kSpread: the rows of a sequence (S > 1) may end at different positions.
template <int HD, typename T, bool kSpread>
struct Consumer {
  const Params& P;
  Smem<HD>& sm;
  int warp, lane, g, t, mi, ri;
  float acc[HD / 8][4];
  float m[2], l[2];
  int low[2], lim[2];  // positions [low, lim) that this lane's two rows see
  bool mixed;          // not the same for all rows of the job
  uint32_t qf[Cfg<HD>::kQSmem ? 1 : HD / 16][4];

  HM_DEV Consumer(const Params& p, Smem<HD>& s) : P(p), sm(s) {
    warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    g = lane >> 2;
    t = lane & 3;
    mi = lane >> 3;
    ri = lane & 7;
  }

  HM_DEV const T* q_ptr(const Job& J, int kh, int i) const {
    const int v = J.i0 + i;
    return reinterpret_cast<const T*>(P.q) + (int64_t)(J.row0 + v / P.G) * P.ld_q + (int64_t)(kh * P.G + v % P.G) * HD;
  }

  // Query fragments, limits and cleared statistics of a run.
  HM_DEV void begin(const Job& J, int kh, bool prefix) {
    int len[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = g + 8 * e;
      len[e] = kSpread && i < J.M && !prefix ? row_len(P, J.row0 + (J.i0 + i) / P.G) : J.hi;
      m[e] = -INFINITY;
      l[e] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    if constexpr (Cfg<HD>::kQSmem) {
      named_bar(1, kCons);  // the last run's fragments are no longer read
      for (int c = threadIdx.x; c < 16 * (HD / 8); c += kCons) {
        const int i = c / (HD / 8), d = c % (HD / 8);
        const uint4 v = i < J.M ? *reinterpret_cast<const uint4*>(q_ptr(J, kh, i) + 8 * d) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(sm.q + i * Cfg<HD>::kQPitch + 16 * d) = v;
      }
      named_bar(1, kCons);
    } else {
      const int i = g;
      const T* a = q_ptr(J, kh, i < J.M ? i : 0) + 2 * t;
      const T* b = q_ptr(J, kh, i + 8 < J.M ? i + 8 : 0) + 2 * t;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        qf[ks][0] = i < J.M ? *reinterpret_cast<const uint32_t*>(a + 16 * ks) : 0u;
        qf[ks][1] = i + 8 < J.M ? *reinterpret_cast<const uint32_t*>(b + 16 * ks) : 0u;
        qf[ks][2] = i < J.M ? *reinterpret_cast<const uint32_t*>(a + 16 * ks + 8) : 0u;
        qf[ks][3] = i + 8 < J.M ? *reinterpret_cast<const uint32_t*>(b + 16 * ks + 8) : 0u;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      low[e] = kSpread && g + 8 * e < J.M && len[e] >= J.plen && !prefix ? max(J.lo, J.plen) : J.lo;
      lim[e] = min(len[e], J.hi);
    }
    mixed = kSpread && __any_sync(0xffffffffu, low[0] != J.lo || low[1] != J.lo || lim[0] != J.hi || lim[1] != J.hi);
  }

  HM_DEV void q_frag(int ks, uint32_t (&a)[4]) const {
    if constexpr (Cfg<HD>::kQSmem) {
      ldsm_x4(a[0], a[1], a[2], a[3],
              smem_u32(sm.q + ((mi & 1) * 8 + ri) * Cfg<HD>::kQPitch + ks * 32 + (mi >> 1) * 16));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = qf[ks][e];
    }
  }

  // This warp's 16 positions of a tile from p0.
  HM_DEV void tile(int st, int p0, int lo, int hi, int bad) {
    const int b0 = p0 + 16 * warp;
    if (b0 >= hi || b0 + 16 <= lo) return;
    const uint32_t half = 128u << P.sub_shift;
    const uint32_t at = block_at<HD>(P.sub_shift, warp), kb = smem_u32(sm.kv[st][0]) + at, vb = smem_u32(sm.kv[st][1]) + at;
    // two sums a score: half the chain of dependent products
    float s[2][4] = {}, s2[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      uint32_t a[4], x0, x1, x2, x3;
      q_frag(ks, a);
      const int c = 2 * ks + (mi & 1);
      ldsm_x4(x0, x1, x2, x3, kb + (c >> 3) * half + ((mi >= 2 ? 8 : 0) + ri) * 128 + (((c & 7) ^ ri) << 4));
      Ty<T>::mma(ks & 1 ? s2[0] : s[0], a, x0, x1);
      Ty<T>::mma(ks & 1 ? s2[1] : s[1], a, x2, x3);
    }
    const bool no = (bad >> warp) & 1;
    const bool edge = b0 < lo || b0 + 16 > hi || no;  // V rows that are not the job's
    const bool mask = edge || (kSpread && mixed);
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p = b0 + 8 * n + 2 * t + (e & 1);
        const float x = (s[n][e] + s2[n][e]) * P.scale;
        s[n][e] = mask && (no || p < low[e >> 1] || p >= lim[e >> 1]) ? -INFINITY : x;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    float alpha[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
      const float mn = fmaxf(m[e], top[e]);
      // nothing seen yet: keep every weight at 0 (2^(-inf - 0)) instead of 2^(-inf + inf)
      alpha[e] = ex2(m[e] - (mn == -INFINITY ? 0.f : mn));
      m[e] = mn;
      top[e] = mn == -INFINITY ? 0.f : mn;
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2(s[n][e] - top[e >> 1]);
        sum[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) l[e] = l[e] * alpha[e] + sum[e];  // this lane's share; joined at the end of the run
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        acc[n][0] *= alpha[0];
        acc[n][1] *= alpha[0];
        acc[n][2] *= alpha[1];
        acc[n][3] *= alpha[1];
      }
    }
    const uint32_t a[4] = {Ty<T>::pack(s[0][0], s[0][1]), Ty<T>::pack(s[0][2], s[0][3]), Ty<T>::pack(s[1][0], s[1][1]),
                           Ty<T>::pack(s[1][2], s[1][3])};
    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // V rows of this lane that belong to the job
    if (edge) {
      const int p = b0 + 2 * t;
      auto in = [&](int x) { return !no && x >= lo && x < hi; };
      keep0 = (in(p) ? 0xffffu : 0u) | (in(p + 1) ? 0xffff0000u : 0u);
      keep1 = (in(p + 8) ? 0xffffu : 0u) | (in(p + 9) ? 0xffff0000u : 0u);
    }
    if constexpr (kSpread) {
      if (mixed && !no && partly_unseen(b0, lo, hi) && not_finite(sm.kv[st][1] + at, b0, lo, hi)) {
        add_rows(sm.kv[st][1] + at, b0, s);
        return;
      }
    }
#pragma unroll
    for (int nd = 0; nd < HD / 16; ++nd) {
      const int c = 2 * nd + (mi >> 1);
      uint32_t v0, v1, v2, v3;
      ldsm_x4_t(v0, v1, v2, v3, vb + (c >> 3) * half + ((mi & 1) * 8 + ri) * 128 + (((c & 7) ^ ri) << 4));
      if (edge) {
        v0 &= keep0;
        v1 &= keep1;
        v2 &= keep0;
        v3 &= keep1;
      }
      Ty<T>::mma(acc[2 * nd], a, v0, v1);
      Ty<T>::mma(acc[2 * nd + 1], a, v2, v3);
    }
  }

  // Whether some row of the block sees only a part of this warp's positions.
  HM_DEV bool partly_unseen(int b0, int lo, int hi) const {
    const int a = max(b0, lo), b = min(b0 + 16, hi);
    return __any_sync(0xffffffffu, low[0] > a || low[1] > a || lim[0] < b || lim[1] < b);
  }
  // Whether V of this warp's positions inside [lo, hi) holds an infinity or NaN.
  HM_DEV bool not_finite(const uint8_t* v, int b0, int lo, int hi) const {
    const int p = lane >> 1;
    const bool in = b0 + p >= lo && b0 + p < hi;
    return __any_sync(0xffffffffu, in && odd_row<T, HD / 64>(v + p * 128 + (lane & 1) * 64, 128u << P.sub_shift));
  }
  // acc += P V with every row's own positions only (weights in s).
  HM_DEV void add_rows(const uint8_t* v, int b0, const float (&s)[2][4]) {
    float* const w = &sm.red[warp][0][0];  // 16 rows x 16 positions, 0 where the row does not see
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[(g + 8 * (e >> 1)) * 16 + 8 * n + 2 * t + (e & 1)] = s[n][e];
    __syncwarp();
    uint32_t sees[2] = {0u, 0u};
    for (int p = 0; p < 16; ++p)
      for (int e = 0; e < 2; ++e) sees[e] |= (b0 + p >= low[e] && b0 + p < lim[e] ? 1u : 0u) << p;
    float a[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) a[n][e] = acc[n][e];
    rows_product<HD, T>(&a[0][0], w + g * 16, v + 4 * t, 128u << P.sub_shift, sees[0], sees[1]);
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = a[n][e];
    __syncwarp();
  }

  // The run's partial result goes to rows row_at .. row_at + M - 1 of the workspace: the four warps'
  // join with their common maximum, four rows at a time.
  HM_DEV void finish(int M, int64_t row_at) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (t == 0) {
        sm.mw[warp][g + 8 * e] = m[e];
        sm.lw[warp][g + 8 * e] = l[e];
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (4 * c >= M) break;
      if (c) named_bar(1, kCons);  // the last four rows have been read
      if ((g >> 2) == (c & 1)) {
        const int e = c >> 1;
        float* a = &sm.red[warp][g & 3][2 * t];
        if (g + 8 * e < M) {
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(a + 8 * n) = make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
        }
      }
      named_bar(1, kCons);
      // 4 rows x HD / 4 columns of 16 bytes
      for (int x = threadIdx.x; x < HD; x += kCons) {
        const int k = x / (HD / 4), i = 4 * c + k, d = 4 * (x % (HD / 4));
        if (i >= M) continue;
        const float top = fmaxf(fmaxf(sm.mw[0][i], sm.mw[1][i]), fmaxf(sm.mw[2][i], sm.mw[3][i]));
        const float top0 = top == -INFINITY ? 0.f : top;
        float den = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = ex2(sm.mw[w][i] - top0);
          const float4 v = *reinterpret_cast<const float4*>(&sm.red[w][k][d]);
          y.x += f * v.x;
          y.y += f * v.y;
          y.z += f * v.z;
          y.w += f * v.w;
          den += f * sm.lw[w][i];
        }
        *reinterpret_cast<float4*>(P.pa + (row_at + i) * HD + d) = y;
        if (d == 0) {
          P.pm[row_at + i] = top;
          P.pl[row_at + i] = den;
        }
      }
    }
  }
};

template <int HD>
HM_DEV void advance(int& st, int& ph) {
  if (++st == Cfg<HD>::kStages) {
    st = 0;
    ph ^= 1;
  }
}

// First workspace row of a run's partial result.
HM_DEV int64_t run_row(const Params& P, const Run& run) {
  return run.prefix ? (int64_t)run.slot * P.pre_rows : P.pre_slots * P.pre_rows + (int64_t)run.slot * P.own_rows;
}

// A run: its query rows first (the tiles are on their way), then all of its tiles.
template <int HD, typename T, bool kSpread>
HM_DEV void consume(const Params& P, Smem<HD>& sm, const Run& run, int& st, int& ph) {
  Consumer<HD, T, kSpread> C(P, sm);
  const Job J = run.J;
  const int64_t row_at = run_row(P, run);
  int left = run.tiles, p0 = run.tile * kTile;
  C.begin(J, run.kh, run.prefix);
  for (; left > 0; --left, p0 += kTile) {
    // on a timeout: carry on, the error is flagged (every warp has to reach finish's barriers)
    mbar_wait_short(&sm.full[st], ph, P.err, &sm.abort_flag);
    C.tile(st, p0, J.lo, J.hi, sm.bad[st]);
    __syncwarp();
    if (C.lane == 0) mbar_arrive(&sm.empty[st]);
    advance<HD>(st, ph);
  }
  C.finish(J.M, row_at);
}

// ---------------------------------------------------------------- blocks of up to 128 rows
// A tile is two halves of 32 positions whose S (and P over it) have 32 TMEM columns each: while the
// consumers work on one half, the issuer has the other half's products done.
//   issuer, half h of tile t: wait for P -> O += P V -> wait for it -> S of half h of tile t + 1.
constexpr int kHalf = 32;

// S of half h of the tile in stage st.
template <int HD, typename T>
HM_DEV void issue_s(const Params& P, Smem<HD>& sm, int st, int h) {
  const uint32_t half = 128u << P.sub_shift, kb = smem_u32(sm.kv[st][0]);
  const int sub = min(1 << P.sub_shift, kHalf);  // positions of a box inside this half
  const uint32_t id = idesc_f16(kBig, 8) - (1u << 17) + (static_cast<uint32_t>(sub >> 3) << 17) + Ty<T>::kFormat;
  if (elect_one()) {
    for (int p = 0; p < kHalf; p += sub) {
      const uint64_t b = sw128_desc(kb + block_at<HD>(P.sub_shift, (kHalf * h + p) / 16));
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        umma_f16_ts(sm.tmem + kHalf * h + p, sm.tmem + Cfg<HD>::kTmemQ + 8 * ks, b + (ks / 4) * (half >> 4) + 2 * (ks % 4), id,
                    ks != 0);
    }
    umma_commit(&sm.s_full[h]);
  }
  __syncwarp();
}

// hph: parity of the halves' barriers (each takes one phase per tile).
template <int HD, typename T, bool kSpread>
HM_DEV void issue_big(const Params& P, Smem<HD>& sm, const Run& run, int& st, int& ph, int& qph, int& hph) {
  const uint32_t half = 128u << P.sub_shift;
  constexpr uint32_t id_o = idesc_f16(kBig, HD, false, true) | Ty<T>::kFormat;
  mbar_wait_short(&sm.q_full, qph, P.err, &sm.abort_flag);
  qph ^= 1;
  mbar_wait_short(&sm.full[st], ph, P.err, &sm.abort_flag);
  tc_fence_after();
  issue_s<HD, T>(P, sm, st, 0);
  issue_s<HD, T>(P, sm, st, 1);
  for (int t = 0, n = run.tiles; t < n; ++t) {
    int st2 = st, ph2 = ph;
    advance<HD>(st2, ph2);
    const uint32_t vb = smem_u32(sm.kv[st][1]);
    bool ahead = false;  // the next tile's first S is issued between the halves when its K is there
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mbar_wait_short(&sm.p_full[h], hph, P.err, &sm.abort_flag);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int b = 0; b < kHalf / 16; ++b)
          umma_f16_ts(sm.tmem + Cfg<HD>::kTmemO, sm.tmem + kHalf * h + 8 * b,
                      sw128_mn_desc(vb + block_at<HD>(P.sub_shift, 2 * h + b), half), id_o,
                      kSpread || (t | h | b) != 0);  // (kSpread: the consumers cleared O)
        umma_commit(&sm.o_full[h]);
      }
      __syncwarp();
      mbar_wait_short(&sm.o_full[h], hph, P.err, &sm.abort_flag);
      tc_fence_after();
      if (h == 0) {
        ahead = t + 1 < n && __all_sync(0xffffffffu, mbar_try_wait(&sm.full[st2], ph2));
        if (ahead) issue_s<HD, T>(P, sm, st2, 0);
      } else {  // both halves are done with the stage
        if (elect_one()) mbar_arrive_n(&sm.empty[st], 5);
        __syncwarp();
        if (t + 1 < n) {
          if (!ahead) {
            mbar_wait_short(&sm.full[st2], ph2, P.err, &sm.abort_flag);
            issue_s<HD, T>(P, sm, st2, 0);
          }
          issue_s<HD, T>(P, sm, st2, 1);
        }
      }
    }
    hph ^= 1;
    st = st2;
    ph = ph2;
  }
}

// A column of this thread's TMEM lane (no wait).
HM_DEV void tmem_ld1_nowait(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
}

// O += P V of this thread's row for positions q0 .. q0 + 31 of the tile, those in `sees` only.
// Scores are read back from S.
template <int HD, typename T>
__device__ __noinline__ void add_row(const uint8_t* v, int sub_shift, uint32_t tmem, int q0, uint32_t sees, float m,
                                     float scale) {
#pragma unroll 1
  for (int c = 0; c < HD / 32; ++c) {
    uint32_t o[32];
    tmem_ld32_nowait(tmem + Cfg<HD>::kTmemO + 32 * c, o);
#pragma unroll 1
    for (int p = 0; p < kHalf; ++p) {
      uint32_t x;
      __syncwarp();
      tmem_ld1_nowait(tmem + q0 + p, x);
      tmem_wait_ld();
      if (!((sees >> p) & 1)) continue;
      const float w = ex2(fmaf(__uint_as_float(x), scale, -m));
      const int q = q0 + p;
      const uint8_t* row = v + block_at<HD>(sub_shift, q >> 4) + (c / 2) * (128u << sub_shift) + (q & 15) * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 y = *reinterpret_cast<const uint4*>(row + (((4 * (c & 1) + k) ^ (q & 7)) << 4));
        const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Ty<T>::f2(u[e]);
          o[8 * k + 2 * e] = __float_as_uint(__uint_as_float(o[8 * k + 2 * e]) + w * f.x);
          o[8 * k + 2 * e + 1] = __float_as_uint(__uint_as_float(o[8 * k + 2 * e + 1]) + w * f.y);
        }
      }
    }
    __syncwarp();
    tmem_st32(tmem + Cfg<HD>::kTmemO + 32 * c, o);
  }
}

// Consumers: thread = TMEM lane = row of the block.
template <int HD, typename T, bool kSpread>
HM_DEV void consume_big(const Params& P, Smem<HD>& sm, const Run& run, int& st, int& ph, int& hph) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = threadIdx.x;  // i: row of the block
  const Job J = run.J;
  const int64_t row_at = run_row(P, run);
  const uint32_t tmem = sm.tmem + (static_cast<uint32_t>(32 * warp) << 16);
  const bool mine = 32 * warp < J.M;  // whole warps: some rows of this one exist
  auto q_row = [&](int k) {         // of row k of this warp's 32 (clamped)
    const int v = J.i0 + min(32 * warp + k, J.M - 1);
    return reinterpret_cast<const T*>(P.q) + (int64_t)(J.row0 + v / P.G) * P.ld_q + (int64_t)(run.kh * P.G + v % P.G) * HD;
  };
  if (mine) {
    // Q: 32 rows x 64 bytes at a time through shared memory (four lanes a row, whole sectors), then
    // a row per lane into TMEM
    uint4 y[HD / 32][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4* q = reinterpret_cast<const uint4*>(q_row(8 * j + (lane >> 2))) + (lane & 3);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) y[c][j] = q[4 * c];
    }
    uint4* const buf = reinterpret_cast<uint4*>(&sm.red[0][0][0]) + 128 * warp;  // 2 KB of the 8
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) buf[(8 * j + (lane >> 2)) * 4 + ((lane & 3) ^ (lane >> 3))] = y[c][j];
      __syncwarp();
      uint32_t x[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 z = buf[lane * 4 + (k ^ ((lane >> 1) & 3))];
        x[4 * k] = z.x;
        x[4 * k + 1] = z.y;
        x[4 * k + 2] = z.z;
        x[4 * k + 3] = z.w;
      }
      tmem_st16(tmem + Cfg<HD>::kTmemQ + 16 * c, x);
    }
    if constexpr (kSpread) {  // O = 0: rows may be added to it before the first product
      uint32_t z[16] = {};
      for (int c = 0; c < HD / 16; ++c) tmem_st16(tmem + Cfg<HD>::kTmemO + 16 * c, z);
    }
    tmem_wait_st();
  }
  auto publish = [&](uint64_t* bar) {  // Q or P of this warp's rows
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  publish(&sm.q_full);
  // positions [low, lim) that this row sees
  int low = J.lo, lim = i < J.M ? J.hi : 0;
  bool mixed = false;  // not the same for all rows of the job
  if (kSpread && !run.prefix) {
    if (i < J.M) {
      const int len = row_len(P, J.row0 + (J.i0 + i) / P.G);
      if (len >= J.plen) low = max(J.lo, J.plen);
      lim = min(len, J.hi);
    }
    mixed = named_bar_or(1, kCons, i < J.M && (low != J.lo || lim != J.hi));
  }
  float m = 0.f, l = 0.f;  // m: the row's reference, at most 2^8 behind its maximum
  bool seen = false;
  for (int t = 0, n = run.tiles, p0 = run.tile * kTile; t < n; ++t, p0 += kTile) {
    mbar_wait_short(&sm.full[st], ph, P.err, &sm.abort_flag);
    const int bad = sm.bad[st];
    if (p0 < J.lo || p0 + kTile > J.hi) {
      // V rows that are not the job's: zero times whatever stands there must be zero
      const int p = threadIdx.x >> 1;
      if (p0 + p < J.lo || p0 + p >= J.hi) {
        uint8_t* row = sm.kv[st][1] + block_at<HD>(P.sub_shift, p >> 4) + (p & 15) * 128 + (threadIdx.x & 1) * 64;
        const uint32_t half = 128u << P.sub_shift;
#pragma unroll
        for (int h = 0; h < HD / 64; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(row + h * half + 16 * k) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
    }
    bool slow = false;  // a V that is not finite, and a row that must not see it
    if (kSpread && mixed && named_bar_or(1, kCons, i < J.M && (low > max(p0, J.lo) || lim < min(p0 + kTile, J.hi)))) {
      const int p = threadIdx.x >> 1;
      const uint8_t* row = sm.kv[st][1] + block_at<HD>(P.sub_shift, p >> 4) + (p & 15) * 128 + (threadIdx.x & 1) * 64;
      const bool in = p0 + p >= J.lo && p0 + p < J.hi;
      slow = named_bar_or(1, kCons, in && odd_row<T, HD / 64>(row, 128u << P.sub_shift));
    }
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      const int a0 = p0 + kHalf * h;
      mbar_wait_short(&sm.s_full[h], hph, P.err, &sm.abort_flag);
      tc_fence_after();
      __syncwarp();
      if (mine) {
        uint32_t x[kHalf];
        tmem_ld32_nowait(tmem + kHalf * h, x);
        // the columns that this row sees, a bit each
        const int from = max(low - a0, 0), to = min(lim - a0, kHalf);
        uint32_t sees = to > from ? (0xffffffffu >> (kHalf - (to - from))) << from : 0u;
        if (bad) sees &= ((bad >> (2 * h)) & 1 ? 0xffff0000u : 0xffffffffu) & ((bad >> (2 * h)) & 2 ? 0xffffu : 0xffffffffu);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, sees != 0xffffffffu && sees != 0u)) {
#pragma unroll
          for (int c = 0; c < kHalf; ++c)
            if (!((sees >> c) & 1)) x[c] = 0xff800000u;  // -infinity
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kHalf; ++c) tops[c & 3] = fmaxf(tops[c & 3], __uint_as_float(x[c]));
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * P.scale;
        if (sees == 0u) top = -INFINITY;
        bool grow = false;
        if (!seen) {  // the first positions that this row sees: nothing in O or l but zeros
          if (top > -INFINITY) {
            m = top;
            seen = true;
          }
        } else {
          grow = top > m + 8.f;
        }
        if (__any_sync(0xffffffffu, grow)) {
          // O at rest: the product before this half's (of the other half) has to be over
          mbar_wait_short(&sm.o_full[h ^ 1], h ? hph : hph ^ 1, P.err, &sm.abort_flag);
          tc_fence_after();
          const float f = grow ? ex2(m - top) : 1.f;
          if (grow) m = top;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld32_nowait(tmem + Cfg<HD>::kTmemO + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st32(tmem + Cfg<HD>::kTmemO + 32 * c, o);
          }
        }
        float sum[2] = {0.f, 0.f};
        uint32_t y[kHalf / 2];
#pragma unroll
        for (int c = 0; c < kHalf / 2; ++c) {
          const float y0 = ex2(fmaf(__uint_as_float(x[2 * c]), P.scale, -m));
          const float y1 = ex2(fmaf(__uint_as_float(x[2 * c + 1]), P.scale, -m));
          sum[0] += y0;
          sum[1] += y1;
          y[c] = sees ? Ty<T>::pack(y0, y1) : 0u;
        }
        if (sees) l += sum[0] + sum[1];
        __syncwarp();
        if (kSpread && slow) {
          mbar_wait_short(&sm.o_full[h ^ 1], h ? hph : hph ^ 1, P.err, &sm.abort_flag);  // O at rest, see above
          tc_fence_after();
          add_row<HD, T>(sm.kv[st][1], P.sub_shift, tmem, kHalf * h, sees, m, P.scale);
#pragma unroll
          for (int c = 0; c < kHalf / 2; ++c) y[c] = 0u;
        }
        tmem_st16(tmem + kHalf * h, y);
        tmem_wait_st();
      }
      if (kSpread && slow) {  // this half's products are in O: zero times zero for the tensor cores
        named_bar(1, kCons);
        const int p = kHalf * h + (threadIdx.x >> 2);
        uint8_t* row = sm.kv[st][1] + block_at<HD>(P.sub_shift, p >> 4) + (p & 15) * 128 + (threadIdx.x & 3) * 32;
        for (int k = 0; k < HD / 64; ++k) {
          *reinterpret_cast<uint4*>(row + k * (128u << P.sub_shift)) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(row + k * (128u << P.sub_shift) + 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      publish(&sm.p_full[h]);
    }
    hph ^= 1;
    advance<HD>(st, ph);
  }
  // both halves' last products
  mbar_wait_short(&sm.o_full[0], hph ^ 1, P.err, &sm.abort_flag);
  mbar_wait_short(&sm.o_full[1], hph ^ 1, P.err, &sm.abort_flag);
  tc_fence_after();
  if (!seen) m = -INFINITY;
  if (i < J.M) {
    P.pm[row_at + i] = m;
    P.pl[row_at + i] = l;
  }
  // 16 columns at a time through shared memory, where a lane's row becomes four lanes' (whole sectors)
  if (mine) {
    float4* const buf = reinterpret_cast<float4*>(&sm.red[0][0][0]) + 128 * warp;
    float* const out = P.pa + (row_at + 32 * warp + (lane >> 2)) * HD + 4 * (lane & 3);
#pragma unroll 1
    for (int c = 0; c < HD / 16; ++c) {
      float o[16];
      __syncwarp();  // the last columns have been read
      tmem_ld16(tmem + Cfg<HD>::kTmemO + 16 * c, o);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        buf[lane * 4 + (k ^ ((lane >> 1) & 3))] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      __syncwarp();
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int row = 8 * g + (lane >> 2);
        if (32 * warp + row < J.M)
          *reinterpret_cast<float4*>(out + 8 * g * HD + 16 * c) = buf[row * 4 + ((lane & 3) ^ ((row >> 1) & 3))];
      }
    }
  }
  tc_fence_before();
}

// ---------------------------------------------------------------- kernel
template <int HD, typename T, bool kSpread>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kCtas)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ Params P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {  // (the same for every CTA: all return, and the join finds jobs without tiles)
    if (threadIdx.x == 0) report_error(P.err, HM_ERR_TIMEOUT);
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < kPlanInts; i += kThreads) P.plan[i] = i == 0;
    return;
  }
  constexpr int NST = Cfg<HD>::kStages;
  static_assert(NST < kRuns, "run entries");
  const int tid = threadIdx.x, lane = tid & 31;
  pdl_trigger();  // the join may be launched; it waits for this grid's end
  if (tid == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < NST; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 5);  // the consumer warps and the issuer
    }
    for (int i = 0; i < kRuns; ++i) mbar_init(&sm.run_full[i], 1);
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sm.s_full[h], 1);
      mbar_init(&sm.o_full[h], 1);
      mbar_init(&sm.p_full[h], 4);
    }
    mbar_init(&sm.q_full, 4);
    fence_barrier_init();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (P.big && tid >= kThreads - 32) tmem_alloc(&sm.tmem, Cfg<HD>::kTmem);
  tc_fence_before();
  const bool no_groups = build_jobs(P, sm);  // (synchronises the CTA)
  tc_fence_after();
  const int n_jobs = P.n_jobs, n_own = P.B * P.own_blocks, Hk = P.Hk;
  const int64_t total = (int64_t)sm.scan[n_jobs] * Hk;
  const int64_t share = total > 0 ? (total + gridDim.x - 1) / gridDim.x : 1;
  if (blockIdx.x == 0) {  // for the join
    if (tid == 0) {
      P.plan[0] = static_cast<int>(share);
      P.plan[1] = no_groups;
    }
    for (int j = tid; j <= n_jobs; j += kThreads) P.plan[kPlanScan + j] = sm.scan[j];
  }

  if (tid >= kThreads - 32) {
    // ------------------------------------------------------------ tcgen05 issuer
    int st = 0, ph = 0, qph = 0, hph = 0;
    for (int n = 0;; ++n) {
      if (!mbar_wait_short(&sm.run_full[n % kRuns], (n / kRuns) & 1, P.err, &sm.abort_flag)) break;
      const Run& run = sm.run[n % kRuns];
      if (run.tiles == 0) break;
      if (run.J.mt > 16) {
        issue_big<HD, T, kSpread>(P, sm, run, st, ph, qph, hph);
      } else {  // follow the ring, so that an entry is not overwritten before this warp has read it
        for (int t = 0, k = run.tiles; t < k; ++t) {
          mbar_wait_short(&sm.full[st], ph, P.err, &sm.abort_flag);
          if (lane == 0) mbar_arrive(&sm.empty[st]);
          __syncwarp();
          advance<HD>(st, ph);
        }
      }
    }
  } else if (tid >= kCons) {
    // ------------------------------------------------------------ producer warp
    const int64_t x0 = share * blockIdx.x, x1 = min(total, x0 + share);
    const int sub = 1 << P.sub_shift, nsub = kTile >> P.sub_shift;
    const int batch = 32 / nsub;  // tiles whose page numbers the lanes fetch at once
    const int none = P.n_pages * Hk * P.page;  // a row behind the pool: TMA fills with zeros
    constexpr uint32_t bytes = 2 * Cfg<HD>::kOperand;
    int it = 0, runs = 0, st = 0, ph = 1;
    bool go = true;
    auto hand_over = [&](const Run& r) {  // the entry is free: see kRuns
      if (lane == 0) {
        sm.run[runs % kRuns] = r;
        mbar_arrive(&sm.run_full[runs % kRuns]);
      }
      ++runs;
    };
    int j = x0 < x1 ? job_at(sm.scan, n_jobs, x0, Hk) : n_jobs;
    int64_t base = x0 < x1 ? (int64_t)sm.scan[j] * Hk : x1;  // where the unit (j, kh) starts
    for (; base < x1 && go; ++j) {
      const int tiles = sm.scan[j + 1] - sm.scan[j];
      if (tiles == 0) continue;
      int kh = 0;
      if (base < x0) {  // the first job: the unit that holds x0
        kh = static_cast<int>((x0 - base) / tiles);
        base += (int64_t)kh * tiles;
      }
      Job J;
      if (j < n_own) {
        const int b = P.own_blocks == 1 ? j : j / P.own_blocks, g = no_groups ? -1 : group_of(P.gstart, P.n_groups, b);
        J = own_job(P, j - b * P.own_blocks, b, g < 0 ? 0 : group_plen(P, g));
        J.trow = P.seqs ? P.seqs[b] : b;
      } else {
        const int id = sm.ids[j - n_own], g = id & 0xffff;
        J = prefix_job(P, id >> 16, P.gstart[g], P.gstart[g + 1], P.plen[g]);
        J.trow = P.owner[g];
      }
      int top = 0, low = 0x7fffffff;
      for (int r = row_first(P, J) + lane; r <= row_last(P, J); r += 32) {
        const int len = row_len(P, r);
        top = max(top, len);
        low = min(low, low_of(len));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (j < n_own)
        own_range(J, top, __reduce_min_sync(0xffffffffu, low));
      else
        prefix_range(J, top);
      const int first = J.lo / kTile;
      const int* const trow = P.table + J.trow * P.table_ld;
      int have = -1, pg = 0, at = 0, bad = 0;  // the batch whose pages the lanes hold
      for (; kh < Hk && base < x1 && go; ++kh, base += tiles) {
        const int t0 = base < x0 ? static_cast<int>(x0 - base) : 0;
        const int t1 = x1 - base >= tiles ? tiles : static_cast<int>(x1 - base);
        // a run is one (job, KV head) of one CTA: along the flat order either grows, so their
        // sum numbers the runs of a kind without collisions
        hand_over(Run{J, kh, first + t0, t1 - t0, (j < n_own ? j : j - n_own) * Hk + kh + static_cast<int>(blockIdx.x),
                      j >= n_own});
        for (int tb = t0; tb < t1 && go;) {
          if (have < 0 || tb < have || tb >= have + batch) {
            have = tb;
            const int p = (first + tb + lane / nsub) * kTile + (lane % nsub) * sub;
            pg = -1;
            bad = 0;
            at = p % P.page;
            if (p + sub > J.lo && p < J.hi) {
              pg = trow[p / P.page];
              if (pg < 0 || pg >= P.n_pages) {
                pg = -1;
                bad = 1;
                report_error(P.err, HM_ERR_BADINDEX);
              }
            }
          }
          const uint32_t bads = __ballot_sync(0xffffffffu, bad);
          const int y = pg < 0 ? none : (pg * Hk + kh) * P.page + at;
          const int n = min(have + batch, t1) - tb;
          for (int i = tb - have, e = i + n; i < e; ++i, ++it, ++tb) {
            if (it >= NST) go = mbar_wait_short(&sm.empty[st], ph, P.err, &sm.abort_flag);
            if (!__all_sync(0xffffffffu, go)) {
              go = false;
              break;
            }
            if (lane == 0) {
              int mask = 0;  // a bit per 16 positions
              if (bads)
                for (int b = 0; b < kTile / 16; ++b) mask |= ((bads >> (i * nsub + ((16 * b) >> P.sub_shift))) & 1) << b;
              sm.bad[st] = mask;
              mbar_arrive_expect_tx(&sm.full[st], bytes);
            }
            __syncwarp();
            // lane i * nsub + s holds the row of sub-box s: it issues that box of K and of V
            if (lane / nsub == i) {
              const int off = (lane % nsub) * sub * HD * 2;
              tma_load_3d_plain(sm.kv[st][0] + off, &kmap, 0, y, 0, &sm.full[st]);
              tma_load_3d_plain(sm.kv[st][1] + off, &vmap, 0, y, 0, &sm.full[st]);
            }
            __syncwarp();
            if (++st == NST) {
              st = 0;
              ph ^= 1;
            }
          }
        }
      }
    }
    hand_over(Run{});  // no tiles: the end
  } else {
    // ------------------------------------------------------------ consumers
    int st = 0, ph = 0, hph = 0;
    for (int n = 0;; ++n) {
      const bool ok = mbar_wait_short(&sm.run_full[n % kRuns], (n / kRuns) & 1, P.err, &sm.abort_flag);
      // after a timeout (flagged) all four warps stop together: none waits for another at a barrier
      if (named_bar_or(1, kCons, !ok)) break;
      const Run& run = sm.run[n % kRuns];
      if (run.tiles == 0) break;
      if (run.J.mt == 16)
        consume<HD, T, kSpread>(P, sm, run, st, ph);
      else
        consume_big<HD, T, kSpread>(P, sm, run, st, ph, hph);
    }
  }
  settle(&sm.abort_flag);
  __syncthreads();
  if (P.big && tid >= kThreads - 32) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, Cfg<HD>::kTmem);
  }
}

// x / d for x >= 0: the 64-bit quotient only where it is needed (it takes a few hundred cycles).
HM_DEV int quotient(int64_t x, int d) {
  return (x >> 32) == 0 ? static_cast<int>(static_cast<uint32_t>(x) / static_cast<uint32_t>(d)) : static_cast<int>(x / d);
}

// Joins the partial results of a (row, head), WPR warps each: the sequence's own in order, then the
// prefix's, every WPR-th by one warp.  Nothing to join (a padding row): zeros.  The kernel is a chain
// of memory latencies, so everything that can be is requested at once: the job list's entries, then
// the maxima, sums and first columns together.  Four warps a pair while all pairs fit the SMs at once
// (16 x 24 pairs of ~17 splits: 69.1 us a call, 72.9 with one warp each), one where there are more
// (64 x 32 pairs of ~8 splits: 42.4 us, 45.5 with four).
template <int HD, typename T, int WPR>
__global__ void __launch_bounds__(128) prefix_join_kernel(const __grid_constant__ Params P) {
  __shared__ float part_s[WPR == 1 ? 1 : 4][HD];
  const int warp = (threadIdx.x >> 5) % WPR, lane = threadIdx.x & 31;
  const unsigned pair = blockIdx.x * (4 / WPR) + (threadIdx.x >> 5) / WPR;
  const bool live = pair < static_cast<unsigned>(P.R) * P.Hq;
  const int r = live ? pair / P.Hq : 0, h = pair % P.Hq, kh = h / P.G, b = r / P.S;
  // the call's inputs do not change while it runs: read them while the first kernel still works
  const int n_own = P.B * P.own_blocks;
  int g = group_of(P.gstart, P.n_groups, b), i = 0, mt = 16, j = 0;
  const int plen = g >= 0 ? group_plen(P, g) : 0;
  // (a bad boundary may be anything)
  if (plen > 0 && P.gstart[g] >= 0 && P.gstart[g + 1] <= P.B && row_len(P, r) >= plen) {
    const int a = P.gstart[g];
    mt = block_rows((P.gstart[g + 1] - a) * P.S * P.G);
    i = (r - a * P.S) * P.G + h % P.G;
    j = group_job(P, n_own, g, a) + i / mt;
  } else {
    g = -1;
  }
  const int omt = block_rows(P.S * P.G), oi = (r % P.S) * P.G + h % P.G, u = b * P.own_blocks + oi / omt;
  pdl_wait();
  if (WPR == 1 && !live) return;
  const int* scan = P.plan + kPlanScan;
  const int share = P.plan[0], bad = P.plan[1], o0 = scan[u], o1 = scan[u + 1];
  const int p0 = g >= 0 ? scan[j] : 0, p1 = g >= 0 ? scan[j + 1] : 0;
  // splits of the two jobs, and the workspace row of the first (the next one is a slot further)
  int cnt0 = 0, cnt1 = 0;
  int64_t at0 = 0, at1 = 0;
  if (o1 > o0) {
    const int64_t x = (int64_t)o0 * P.Hk + (int64_t)kh * (o1 - o0);
    const int c0 = quotient(x, share);
    cnt0 = quotient(x + (o1 - o0) - 1, share) - c0 + 1;
    at0 = P.pre_slots * P.pre_rows + ((int64_t)u * P.Hk + kh + c0) * P.own_rows + oi % omt;
  }
  if (p1 > p0 && !bad) {
    const int64_t x = (int64_t)p0 * P.Hk + (int64_t)kh * (p1 - p0);
    const int c0 = quotient(x, share);
    cnt1 = quotient(x + (p1 - p0) - 1, share) - c0 + 1;
    at1 = ((int64_t)(j - n_own) * P.Hk + kh + c0) * P.pre_rows + i % mt;
  }
  const int n = cnt0 + cnt1;
  auto row_of = [&](int s) { return s < cnt0 ? at0 + (int64_t)s * P.own_rows : at1 + (int64_t)(s - cnt0) * P.pre_rows; };
  constexpr int V = HD / 32, E = 6;  // columns of a lane; splits of a warp whose columns are requested early
  auto cols = [&](int s, float (&a)[V]) {
    const float* p = P.pa + row_of(s) * HD + V * lane;
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 f = *reinterpret_cast<const float2*>(p + e);
      a[e] = f.x;
      a[e + 1] = f.y;
    }
  };
  float m = -INFINITY, l = 0.f;  // of split `lane`
  if (lane < n) {
    const int64_t rw = row_of(lane);
    m = P.pm[rw];
    l = P.pl[rw];
  }
  float early[E][V];
#pragma unroll
  for (int k = 0; k < E; ++k)
    if (warp + WPR * k < n) cols(warp + WPR * k, early[k]);
  float M = m;
  for (int s = 32 + lane; s < n; s += 32) M = fmaxf(M, P.pm[row_of(s)]);
  M = warp_max(M);
  const float M0 = M == -INFINITY ? 0.f : M;
  float num[V] = {};
  float den = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    if (s0) {
      m = -INFINITY;
      l = 0.f;
      if (s0 + lane < n) {
        const int64_t rw = row_of(s0 + lane);
        m = P.pm[rw];
        l = P.pl[rw];
      }
    }
    const float w = ex2(m - M0);  // 0 for lanes without a split
    den += warp_sum(s0 + lane < n ? l * w : 0.f);
    int s = s0 + warp;
    if (s0 == 0) {
#pragma unroll
      for (int k = 0; k < E; ++k, s += WPR) {
        const float ws = __shfl_sync(0xffffffffu, w, warp + WPR * k);
        if (s < n) {
#pragma unroll
          for (int v = 0; v < V; ++v) num[v] += ws * early[k][v];
        }
      }
    }
    const int e = min(s0 + 32, n);
#pragma unroll 4
    for (; s < e; s += WPR) {
      const float ws = __shfl_sync(0xffffffffu, w, s - s0);
      float a[V];
      cols(s, a);
#pragma unroll
      for (int v = 0; v < V; ++v) num[v] += ws * a[v];
    }
  }
  const float inv = 1.f / den;  // NaN stays NaN
  T* o = reinterpret_cast<T*>(P.o) + r * P.ld_o + (int64_t)h * HD;
  if constexpr (WPR == 1) {
#pragma unroll
    for (int v = 0; v < V; v += 2)
      *reinterpret_cast<uint32_t*>(o + V * lane + v) = den == 0.f ? 0u : Ty<T>::pack(num[v] * inv, num[v + 1] * inv);
  } else {
    static_assert(WPR == 1 || WPR == 4, "the CTA's four warps");
#pragma unroll
    for (int v = 0; v < V; ++v) part_s[warp][V * lane + v] = num[v];
    __syncthreads();
    for (int d = 2 * threadIdx.x; d < HD; d += 256) {
      const float y0 = ((part_s[0][d] + part_s[1][d]) + part_s[2][d]) + part_s[3][d];
      const float y1 = ((part_s[0][d + 1] + part_s[1][d + 1]) + part_s[2][d + 1]) + part_s[3][d + 1];
      *reinterpret_cast<uint32_t*>(o + d) = den == 0.f ? 0u : Ty<T>::pack(y0 * inv, y1 * inv);
    }
  }
}

// ---------------------------------------------------------------- host side
struct Shape {
  int B, G, own_blocks, own_rows, pre_rows, big;
  int64_t pre_jobs, pre_slots, rows;
};

// Sizes that follow from the arguments alone (the lengths are on the device).
bool shape_of(int R, int S, int Hq, int Hk, int n_groups, int ctas, Shape* s) {
  if (R < 1 || S < 1 || R % S || Hk < 1 || Hq < Hk || Hq % Hk || n_groups < 0) return false;
  s->B = R / S;
  s->G = Hq / Hk;
  if (s->G > 64 || R > kMaxRows) return false;
  const int64_t own = (int64_t)S * s->G, all = (int64_t)R * s->G;
  const int own_mt = own <= 16 ? 16 : kBig;
  s->own_blocks = static_cast<int>((own + own_mt - 1) / own_mt);
  s->own_rows = static_cast<int>(own < own_mt ? own : own_mt);
  s->pre_rows = static_cast<int>(all < kBig ? all : kBig);
  // groups of up to 128 rows are one job, larger ones one per started 128 rows
  s->pre_jobs = n_groups == 0 ? 0 : all / kBig + n_groups;
  s->big = own > 16 || (n_groups > 0 && all > 16);
  if (s->pre_jobs + (int64_t)s->B * s->own_blocks > kMaxJobs || s->pre_jobs > kMaxPre) return false;
  s->pre_slots = s->pre_jobs ? s->pre_jobs * Hk + ctas : 0;
  s->rows = s->pre_slots * s->pre_rows + ((int64_t)s->B * s->own_blocks * Hk + ctas) * s->own_rows;
  return true;
}

constexpr int kMaxDevices = 64;

// SMs of the current device and its index.
cudaError_t device_sms(int* dev, int* sms) {
  static std::atomic<int> known[kMaxDevices];
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return e;
  if (*dev < kMaxDevices && (*sms = known[*dev].load()) > 0) return cudaSuccess;
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev);
  if (e == cudaSuccess && *dev < kMaxDevices) known[*dev].store(*sms);
  return e;
}

int ctas_per_sm(int hd) { return hd <= 128 ? 2 : 1; }

constexpr size_t kPlanBytes = (kPlanInts * sizeof(int) + 255) / 256 * 256;

// [rows of the pool, hd] as {64 dims, rows, hd / 64}, a box of `sub` rows and all dims
bool pool_map(const void* p, int64_t rows, int hd, int sub, bool bf16, CUtensorMap* out) {
  auto enc = hm_encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {64, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(hd / 64)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(hd) * 2, 128};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(sub), static_cast<cuuint32_t>(hd / 64)};
  cuuint32_t es[3] = {1, 1, 1};
  return enc(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p),
             dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, typename T, bool kSpread>
cudaError_t launch_main(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int grid, int dev, cudaStream_t st) {
  constexpr size_t smem = sizeof(Smem<HD>);
  static std::atomic<bool> configured[kMaxDevices];
  if (dev >= kMaxDevices || !configured[dev].load()) {
    const cudaError_t e = cudaFuncSetAttribute(prefix_attn_kernel<HD, T, kSpread>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) configured[dev].store(true);
  }
  return hm_launch(prefix_attn_kernel<HD, T, kSpread>, dim3(grid), dim3(kThreads), smem, st, 0, km, vm, p);
}

template <int HD, typename T>
cudaError_t launch(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int grid, int sms, int dev,
                   cudaStream_t st) {
  const cudaError_t e = p.S == 1 ? launch_main<HD, T, false>(km, vm, p, grid, dev, st)
                                 : launch_main<HD, T, true>(km, vm, p, grid, dev, st);
  if (e != cudaSuccess) return e;
  const unsigned pairs = static_cast<unsigned>(p.R) * p.Hq;
  if (pairs <= 4u * sms) return hm_launch(prefix_join_kernel<HD, T, 4>, dim3(pairs), dim3(128), 0, st, 1, p);
  return hm_launch(prefix_join_kernel<HD, T, 1>, dim3((pairs + 3) / 4), dim3(128), 0, st, 1, p);
}

template <int HD>
cudaError_t launch_t(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int grid, int sms, int dev,
                     cudaStream_t st, bool bf16) {
  return bf16 ? launch<HD, __nv_bfloat16>(km, vm, p, grid, sms, dev, st)
              : launch<HD, __half>(km, vm, p, grid, sms, dev, st);
}

bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }

}  // namespace

extern "C" size_t hm_prefix_attn_workspace_bytes(int R, int S, int Hq, int Hk, int hd, int n_groups, int sms) {
  Shape s;
  if ((hd != 64 && hd != 128 && hd != 256) || sms < 1 || !shape_of(R, S, Hq, Hk, n_groups, sms * ctas_per_sm(hd), &s))
    return 0;
  return kPlanBytes + (size_t)s.rows * (hd + 2) * sizeof(float);
}

extern "C" int hm_prefix_attn(const hm_prefix_attn_desc* d, hm_stream_t stream) {
  if (!d || bad16(d->q) || bad16(d->o) || bad16(d->k) || bad16(d->v) || bad16(d->ws) || !d->pos || !d->table)
    return HM_EARG;
  if ((d->dtype != HM_DT_F16 && d->dtype != HM_DT_BF16) || (d->hd != 64 && d->hd != 128 && d->hd != 256)) return HM_EARG;
  if (d->n_groups > 0 && (!d->gstart || !d->owner || !d->plen)) return HM_EARG;
  if (!(d->scale > 0.f) || !(d->scale < INFINITY)) return HM_EARG;
  const int pg = d->page;
  if (!(pg == 16 || pg == 32 || (pg >= 64 && pg % 64 == 0))) return HM_EARG;
  if (d->n_pages < 1 || d->max_pages < 1 || d->n_table < 1 || d->table_ld < d->max_pages || d->Hk < 1) return HM_EARG;
  // pool rows and positions are 32-bit TMA coordinates / lengths
  if ((int64_t)d->n_pages * d->Hk * pg > 0x7fffff00 || (int64_t)d->max_pages * pg > 0x7fffff00) return HM_EARG;
  if (d->ld_q % 8 || d->ld_o % 8 || d->ld_q < (int64_t)d->Hq * d->hd || d->ld_o < (int64_t)d->Hq * d->hd) return HM_EARG;
  // tile offsets are 32-bit
  if (((int64_t)d->max_pages * pg / kTile + 1) * kMaxJobs > 0x7fffffff) return HM_EARG;
  // before anything asks for the device: the sizes do not depend on the number of SMs
  Shape s;
  if (!shape_of(d->R, d->S, d->Hq, d->Hk, d->n_groups, 1, &s)) return HM_EARG;
  if (!d->seqs && s.B > d->n_table) return HM_EARG;
  int dev = 0, sms = 0;
  cudaError_t e = device_sms(&dev, &sms);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int ctas = sms * ctas_per_sm(d->hd);
  shape_of(d->R, d->S, d->Hq, d->Hk, d->n_groups, ctas, &s);
  if (d->ws_bytes < hm_prefix_attn_workspace_bytes(d->R, d->S, d->Hq, d->Hk, d->hd, d->n_groups, sms)) return HM_EARG;
  const bool bf16 = d->dtype == HM_DT_BF16;
  const int sub = pg < kTile ? pg : kTile;
  const int64_t rows = (int64_t)d->n_pages * d->Hk * pg;
  CUtensorMap km, vm;
  if (!pool_map(d->k, rows, d->hd, sub, bf16, &km) || !pool_map(d->v, rows, d->hd, sub, bf16, &vm)) return HM_EARG;
  Params p = {};
  p.q = d->q;
  p.ld_q = d->ld_q;
  p.o = d->o;
  p.ld_o = d->ld_o;
  p.pos = d->pos;
  p.table = d->table;
  p.table_ld = d->table_ld;
  p.seqs = d->seqs;
  p.gstart = d->gstart;
  p.owner = d->owner;
  p.plen = d->plen;
  p.R = d->R;
  p.S = d->S;
  p.B = s.B;
  p.Hq = d->Hq;
  p.Hk = d->Hk;
  p.G = s.G;
  p.n_table = d->n_table;
  p.max_pages = d->max_pages;
  p.n_pages = d->n_pages;
  p.page = pg;
  p.n_groups = d->n_groups;
  p.sub_shift = sub == 16 ? 4 : (sub == 32 ? 5 : 6);
  p.scale = d->scale * 1.4426950408889634f;
  p.n_jobs = static_cast<int>(s.B * (int64_t)s.own_blocks + s.pre_jobs);
  p.own_blocks = s.own_blocks;
  p.own_rows = s.own_rows;
  p.pre_rows = s.pre_rows;
  p.big = s.big;
  p.pre_slots = s.pre_slots;
  p.plan = reinterpret_cast<int*>(d->ws);
  p.pa = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(d->ws) + kPlanBytes);
  p.pm = p.pa + s.rows * d->hd;
  p.pl = p.pm + s.rows;
  p.err = d->err;
  // no more CTAs than there can be tiles
  const int64_t most = (s.pre_jobs + (int64_t)s.B * s.own_blocks) * d->Hk * (((int64_t)d->max_pages * pg) / kTile + 1);
  if (most / ctas > 0x7ffffffe) return HM_EARG;  // a CTA's share is a 32-bit number
  const int grid = static_cast<int>(most < ctas ? most : ctas);
  e = d->hd == 64    ? launch_t<64>(km, vm, p, grid, sms, dev, stream, bf16)
      : d->hd == 128 ? launch_t<128>(km, vm, p, grid, sms, dev, stream, bf16)
                     : launch_t<256>(km, vm, p, grid, sms, dev, stream, bf16);
  return e == cudaSuccess ? HM_OK : static_cast<int>(e);
}
