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
// position, against 4 * Hq * hd operations a (row, position).  Up to ~100 query rows per KV head
// that is less than the tensor cores do while the bytes arrive, so the kernel is built to keep
// the memory busy:
//  * The work is a list of jobs (group prefix or one sequence's own positions, cut into blocks
//    of query rows) x KV heads x tiles of 64 positions.  Lengths live on the device, so every CTA
//    builds the list itself (one pass over pos, a scan in shared memory) and takes an equal share
//    of the tiles: a long prefix next to short sequences leaves no SM idle, whatever the lengths.
//  * One producer warp fetches page numbers 32 at a time and issues one TMA box per page and
//    operand (128-byte swizzle) into a ring of 96 KB per CTA, two CTAs per SM, across job
//    boundaries, so the ring never drains.
//  * Four consumer warps.  Blocks of up to 16 query rows (the G heads of a KV head x rows): each
//    warp takes 16 of the tile's positions, so K and V leave shared memory once; the four
//    partial results meet in shared memory.  Blocks of up to 64 rows: each warp takes 16 rows and
//    all positions, K and V leave shared memory four times but HBM / L2 only once per 64 rows.
//  * A second small kernel joins the partial results of a row in a fixed order (results do not
//    depend on scheduling) and writes o; its launch overlaps the first kernel's tail.
// Scores, m, l and a are fp32; the probabilities are rounded to the cache's type for the product
// with V, as the flat decode attention does (they are at most 1; l keeps the unrounded sum).
// V rows outside a job's range are zeroed in registers, so whatever stands there (NaN included)
// has no effect.
#include <cuda_bf16.h>

#include <atomic>

#include "hm_common.cuh"

namespace {

constexpr int kTile = 64;       // positions per tile
constexpr int kMaxJobs = 1024;  // jobs of a call (the list lives in shared memory)
constexpr int kThreads = 160;   // 4 consumer warps + the producer
constexpr int kCons = 128;

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
  int own_blocks;     // row blocks of one sequence's own job
  int own_rows;       // row capacity of an own partial
  int pre_rows;       // row capacity of a prefix partial
  int64_t pre_slots;  // prefix partials come first
  int* plan;          // header, tile scan, first prefix job of every group (for the join)
  float* pm;          // [rows] maxima, [rows] sums, [rows][hd] accumulators
  float* pl;
  float* pa;
  int* err;
};

// plan: 0 prefix jobs, 1 jobs, 2 tiles per CTA, 3 groups unusable; then kMaxJobs + 1 tile offsets;
// then n_groups first jobs
constexpr int kPlanScan = 4, kPlanGroup = 4 + kMaxJobs + 1;

// ---------------------------------------------------------------- types
template <typename T>
struct Ty;
template <>
struct Ty<__half> {
  static HM_DEV uint32_t pack(float a, float b) { return pack_h2(a, b); }
  static HM_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <>
struct Ty<__nv_bfloat16> {
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

HM_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- lengths and groups
// Block size of a job with `rows` query rows per KV head: 16 rows while they fit one block.
HM_DEV int block_rows(int rows) { return rows <= 16 ? 16 : 64; }

// Positions that row r attends to: 0 for a padding row and for one whose position or table row
// is out of range (reported).
HM_DEV int row_len(const Params& P, int r) {
  const int64_t p = P.pos[r];
  if (p < 0) return 0;
  const int b = r / P.S, s = P.seqs ? P.seqs[b] : b;
  if (p >= (int64_t)P.max_pages * P.page || s < 0 || s >= P.n_table) {
    report_error(P.err, HM_ERR_BADINDEX);
    return 0;
  }
  return static_cast<int>(p) + 1;
}

// Prefix length of a group: 0 when its entry is out of range (reported).
HM_DEV int group_plen(const Params& P, int g) {
  const int n = P.plen[g];
  if (n == 0) return 0;
  const int own = P.owner[g];
  if (n < 0 || n > (int64_t)P.max_pages * P.page || own < 0 || own >= P.n_table) {
    report_error(P.err, HM_ERR_BADINDEX);
    return 0;
  }
  return n;
}

// The group of sequence b (gstart ascending, checked), -1 for none.
HM_DEV int group_of(const Params& P, int b) {
  int lo = 0, hi = P.n_groups;  // the first boundary above b
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (P.gstart[mid + 1] <= b)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < P.n_groups && P.gstart[lo] <= b ? lo : -1;
}

HM_DEV bool bad_boundary(const Params& P, int g) {
  const int a = P.gstart[g], b = P.gstart[g + 1];
  return a < 0 || a > b || b > P.B;
}

// One job: query rows i0 .. i0 + M - 1 of `row0` (i -> row row0 + i / G, head kh * G + i % G) over
// the positions [lo, hi) of table row `trow`.
struct Job {
  int row0, i0, M, lo, hi, trow, big;
};

HM_DEV Job job_of(const Params& P, int n_pre, const int* ids, int j, bool no_groups) {
  Job J;
  if (j < n_pre) {
    const int g = ids[j] & 0xffff, blk = ids[j] >> 16;
    const int a = P.gstart[g];
    const int rows = (P.gstart[g + 1] - a) * P.S * P.G, mt = block_rows(rows);
    J.row0 = a * P.S;
    J.i0 = blk * mt;
    J.M = min(mt, rows - J.i0);
    J.big = mt > 16;
    J.lo = 0;
    J.hi = P.plen[g];  // in range: groups with a bad entry have no job
    J.trow = P.owner[g];
  } else {
    const int u = j - n_pre, b = u / P.own_blocks, blk = u % P.own_blocks;
    const int rows = P.S * P.G, mt = block_rows(rows);
    J.row0 = b * P.S;
    J.i0 = blk * mt;
    J.M = min(mt, rows - J.i0);
    J.big = mt > 16;
    const int g = no_groups ? -1 : group_of(P, b);
    J.lo = g < 0 ? 0 : group_plen(P, g);
    J.hi = (int64_t)P.max_pages * P.page;
    J.trow = P.seqs ? P.seqs[b] : b;
  }
  return J;
}
// First and last query row of a job.
HM_DEV int row_first(const Params& P, const Job& J) { return J.row0 + J.i0 / P.G; }
HM_DEV int row_last(const Params& P, const Job& J) { return J.row0 + (J.i0 + J.M - 1) / P.G; }

// The job with hi cut to what its rows see.  Whole warps.
HM_DEV Job warp_job(const Params& P, int n_pre, const int* ids, int j, bool no_groups) {
  Job J = job_of(P, n_pre, ids, j, no_groups);
  int top = 0;
  for (int r = row_first(P, J) + (threadIdx.x & 31); r <= row_last(P, J); r += 32) top = max(top, row_len(P, r));
  J.hi = min(J.hi, __reduce_max_sync(0xffffffffu, top));
  return J;
}

HM_DEV int tiles_of(const Job& J) { return J.hi > J.lo ? (J.hi - 1) / kTile - J.lo / kTile + 1 : 0; }

// ---------------------------------------------------------------- shared memory
template <int HD>
struct Cfg {
  static constexpr int kOperand = kTile * HD * 2;  // bytes of a K (or V) tile
  static constexpr int kStages = HD == 64 ? 6 : (HD == 128 ? 3 : 2);
  static constexpr int kCtas = HD <= 128 ? 2 : 1;  // per SM
  static constexpr bool kQSmem = HD > 128;         // query fragments: registers, or shared memory
  static constexpr int kQPitch = HD * 2 + 16;
};

template <int HD>
struct Smem {
  uint8_t kv[Cfg<HD>::kStages][2][Cfg<HD>::kOperand];
  float red[16][HD];
  uint8_t q[Cfg<HD>::kQSmem ? 64 * Cfg<HD>::kQPitch : 16];
  int scan[kMaxJobs + 1];
  int ids[kMaxJobs];
  float mw[4][16], lw[4][16];
  uint64_t full[Cfg<HD>::kStages], empty[Cfg<HD>::kStages];
  int bad[Cfg<HD>::kStages];  // 16-position blocks of the stage without a page
  int n_pre, no_groups, abort_flag;
};
static_assert(sizeof(Smem<128>) + 1024 <= 233472 / 2, "two CTAs per SM at hd 128");
static_assert(sizeof(Smem<64>) + 1024 <= 233472 / 2, "two CTAs per SM at hd 64");
static_assert(sizeof(Smem<256>) <= 227 * 1024, "shared memory at hd 256");

// The job list: prefix jobs in group order, then own_blocks jobs per sequence; scan[j] = tiles
// of the jobs before j (per KV head).  All threads of the CTA.
template <int HD>
HM_DEV int build_jobs(const Params& P, Smem<HD>& sm) {
  const int tid = threadIdx.x, lane = tid & 31;
  bool bad = false;
  for (int g = tid; g < P.n_groups; g += kThreads) bad |= bad_boundary(P, g);
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) report_error(P.err, HM_ERR_BADINDEX);
  if (tid < 32) {
    int n = 0;
    for (int g0 = 0; g0 < P.n_groups && !bad; g0 += 32) {
      const int g = g0 + lane;
      int jobs = 0;
      if (g < P.n_groups && group_plen(P, g) > 0) {
        const int rows = (P.gstart[g + 1] - P.gstart[g]) * P.S * P.G, mt = block_rows(rows);
        jobs = (rows + mt - 1) / mt;
      }
      int x = jobs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int first = n + x - jobs;
      for (int m = 0; m < jobs; ++m) sm.ids[first + m] = g | (m << 16);
      if (blockIdx.x == 0 && g < P.n_groups) P.plan[kPlanGroup + g] = first;
      n += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      sm.n_pre = n;
      sm.no_groups = bad;
    }
  }
  __syncthreads();
  const int n_pre = sm.n_pre, n_jobs = n_pre + P.B * P.own_blocks;
  // a block of one row: a thread per job; else eight lanes share the job's rows
  const bool single = P.S == 1 && P.own_blocks == 1;
  for (int j0 = 0; j0 < (single ? n_pre : n_jobs); j0 += kThreads / 8) {
    const int j = j0 + tid / 8;
    Job J = {};
    int top = 0;
    if (j < n_jobs) {
      J = job_of(P, n_pre, sm.ids, j, bad);
      for (int r = row_first(P, J) + (tid & 7); r <= row_last(P, J); r += 8) top = max(top, row_len(P, r));
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    J.hi = min(J.hi, top);
    if (j < n_jobs && (tid & 7) == 0) sm.scan[j] = tiles_of(J);
  }
  __syncthreads();  // the last step above may have passed n_pre: the loop below writes the same values there
  if (single) {
    for (int j = n_pre + tid; j < n_jobs; j += kThreads) {
      Job J = job_of(P, n_pre, sm.ids, j, bad);
      J.hi = min(J.hi, row_len(P, J.row0));
      sm.scan[j] = tiles_of(J);
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
  __syncthreads();
  return n_jobs;
}

// The job that holds flat tile x (flat tile = scan * Hk + kh * tiles + t).
HM_DEV int job_at(const int* scan, int n_jobs, int64_t x, int Hk) {
  int lo = 0, hi = n_jobs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)scan[mid] * Hk <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;  // the last with scan <= x: jobs without tiles in front of it share its offset
}

// A run of tiles [t0, t1) of one (job, KV head), part of a CTA's share.
struct Run {
  int j, kh, t0, t1;
};
HM_DEV Run run_at(const int* scan, int n_jobs, int64_t x, int64_t end, int Hk) {
  Run r;
  r.j = job_at(scan, n_jobs, x, Hk);
  const int tiles = scan[r.j + 1] - scan[r.j];
  const int64_t in = x - (int64_t)scan[r.j] * Hk;
  r.kh = static_cast<int>(in / tiles);
  r.t0 = static_cast<int>(in % tiles);
  const int64_t left = end - x;
  r.t1 = left < tiles - r.t0 ? r.t0 + static_cast<int>(left) : tiles;
  return r;
}

// ---------------------------------------------------------------- consumer
template <int HD, typename T>
struct Consumer {
  const Params& P;
  Smem<HD>& sm;
  int warp, lane, g, t, mi, ri;
  float acc[HD / 8][4];
  float m[2], l[2];
  int lim[2];  // positions that this lane's two rows see
  uint32_t qf[Cfg<HD>::kQSmem ? 1 : HD / 16][4];
  int qrow;    // first query row of this warp in shared memory

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
  HM_DEV void begin(const Job& J, int kh) {
    qrow = J.big ? warp * 16 : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = qrow + g + 8 * e;
      lim[e] = i < J.M ? min(row_len(P, J.row0 + (J.i0 + i) / P.G), J.hi) : J.hi;
      m[e] = -INFINITY;
      l[e] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    if constexpr (Cfg<HD>::kQSmem) {
      named_bar(1, kCons);  // the last run's fragments are no longer read
      const int rows = J.big ? 64 : 16;
      for (int c = threadIdx.x; c < rows * (HD / 8); c += kCons) {
        const int i = c / (HD / 8), d = c % (HD / 8);
        const uint4 v = i < J.M ? *reinterpret_cast<const uint4*>(q_ptr(J, kh, i) + 8 * d) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(sm.q + i * Cfg<HD>::kQPitch + 16 * d) = v;
      }
      named_bar(1, kCons);
    } else {
      const int i = qrow + g;
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
  }

  HM_DEV void q_frag(int ks, uint32_t (&a)[4]) const {
    if constexpr (Cfg<HD>::kQSmem) {
      ldsm_x4(a[0], a[1], a[2], a[3],
              smem_u32(sm.q + (qrow + (mi & 1) * 8 + ri) * Cfg<HD>::kQPitch + ks * 32 + (mi >> 1) * 16));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = qf[ks][e];
    }
  }

  // One tile of 64 positions from p0; NB = 1: this warp's 16 positions, NB = 4: all of them.
  template <int NB>
  HM_DEV void tile(int st, int p0, const Job& J, int bad) {
    const int b0 = NB == 1 ? warp : 0;
    if (NB == 1 && (p0 + 16 * b0 >= J.hi || p0 + 16 * b0 + 16 <= J.lo)) return;
    const uint32_t kb = smem_u32(sm.kv[st][0]), vb = smem_u32(sm.kv[st][1]);
    const int sub = 1 << P.sub_shift;                         // positions of a box: [64-dim part][position][128 bytes]
    const uint32_t part = static_cast<uint32_t>(sub) * 128u;
    // byte offset of position 16 * b of the tile in its box
    auto block_at = [&](int b) {
      const int p = 16 * b;
      return static_cast<uint32_t>(p >> P.sub_shift) * part * (HD / 64) + static_cast<uint32_t>(p & (sub - 1)) * 128u;
    };
    float s[2 * NB][4];
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    {
      const int row = (mi >= 2 ? 8 : 0) + ri;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t a[4];
        q_frag(ks, a);
        const int c = 2 * ks + (mi & 1);
        const uint32_t off = (c >> 3) * part + row * 128 + (((c & 7) ^ ri) << 4);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t x0, x1, x2, x3;
          ldsm_x4(x0, x1, x2, x3, kb + block_at(b0 + b) + off);
          Ty<T>::mma(s[2 * b], a, x0, x1);
          Ty<T>::mma(s[2 * b + 1], a, x2, x3);
        }
      }
    }
    const bool edge = p0 < J.lo || p0 + kTile > J.hi || bad;  // the same for the whole CTA
    float top[2] = {-INFINITY, -INFINITY};
    if (edge || p0 + kTile > min(lim[0], lim[1])) {
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int b = b0 + n / 2, p = p0 + 16 * b + 8 * (n & 1) + 2 * t + (e & 1);
          const bool ok = p >= J.lo && p < lim[e >> 1] && !((bad >> b) & 1);
          s[n][e] = ok ? s[n][e] * P.scale : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
    } else {
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][e] *= P.scale;
          top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
        }
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
    for (int n = 0; n < 2 * NB; ++n)
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
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t a[4] = {Ty<T>::pack(s[2 * b][0], s[2 * b][1]), Ty<T>::pack(s[2 * b][2], s[2 * b][3]),
                             Ty<T>::pack(s[2 * b + 1][0], s[2 * b + 1][1]), Ty<T>::pack(s[2 * b + 1][2], s[2 * b + 1][3])};
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // V rows of this lane that belong to the job
      if (edge) {
        const int p = p0 + 16 * (b0 + b) + 2 * t;
        const bool no = (bad >> (b0 + b)) & 1;
        auto in = [&](int x) { return !no && x >= J.lo && x < J.hi; };
        keep0 = (in(p) ? 0xffffu : 0u) | (in(p + 1) ? 0xffff0000u : 0u);
        keep1 = (in(p + 8) ? 0xffffu : 0u) | (in(p + 9) ? 0xffff0000u : 0u);
      }
      const uint32_t base = vb + block_at(b0 + b);
      const int row = (mi & 1) * 8 + ri;
#pragma unroll
      for (int nd = 0; nd < HD / 16; ++nd) {
        const int c = 2 * nd + (mi >> 1);
        uint32_t v0, v1, v2, v3;
        ldsm_x4_t(v0, v1, v2, v3, base + (c >> 3) * part + row * 128 + (((c & 7) ^ ri) << 4));
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
  }

  // The run's partial result goes to rows row_at .. row_at + M - 1 of the workspace.
  HM_DEV void finish(const Job& J, int64_t row_at) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if (J.big) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = qrow + g + 8 * e;
        if (i >= J.M) continue;
        float* a = P.pa + (row_at + i) * HD + 2 * t;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(a + 8 * n) = make_float2(acc[n][2 * e], acc[n][2 * e + 1]);
        if (t == 0) {
          P.pm[row_at + i] = m[e];
          P.pl[row_at + i] = l[e];
        }
      }
      return;
    }
    // the four warps' partial results, added in warp order
    if (t == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sm.mw[warp][g + 8 * e] = m[e];
        sm.lw[warp][g + 8 * e] = l[e];
      }
    }
    named_bar(1, kCons);
    float f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = g + 8 * e;
      float M = fmaxf(fmaxf(sm.mw[0][i], sm.mw[1][i]), fmaxf(sm.mw[2][i], sm.mw[3][i]));
      const float M0 = M == -INFINITY ? 0.f : M;
      f[e] = ex2(m[e] - M0);
      if (warp == 0 && t == 0 && i < J.M) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += sm.lw[w][i] * ex2(sm.mw[w][i] - M0);
        P.pm[row_at + i] = M;
        P.pl[row_at + i] = s;
      }
    }
    for (int w = 0; w < 4; ++w) {
      if (warp == w) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (g + 8 * e >= J.M) continue;
          float* a = &sm.red[g + 8 * e][2 * t];
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            float2 x = make_float2(acc[n][2 * e] * f[e], acc[n][2 * e + 1] * f[e]);
            float2* d = reinterpret_cast<float2*>(a + 8 * n);
            if (w) {
              x.x += d->x;
              x.y += d->y;
            }
            *d = x;
          }
        }
      }
      named_bar(1, kCons);
    }
    for (int c = threadIdx.x; c < J.M * (HD / 4); c += kCons)
      *reinterpret_cast<float4*>(P.pa + row_at * HD + 4 * c) = *reinterpret_cast<const float4*>(&sm.red[0][0] + 4 * c);
  }
};

// ---------------------------------------------------------------- kernel
template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, Cfg<HD>::kCtas)
    prefix_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ Params P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<HD>& sm = *reinterpret_cast<Smem<HD>*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {  // (the same for every CTA: all return)
    if (threadIdx.x == 0) report_error(P.err, HM_ERR_TIMEOUT);
    return;
  }
  constexpr int NST = Cfg<HD>::kStages;
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < NST; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 4);
    }
    fence_barrier_init();
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  const int n_jobs = build_jobs(P, sm);
  const int n_pre = sm.n_pre;
  const bool no_groups = sm.no_groups;
  const int64_t total = (int64_t)sm.scan[n_jobs] * P.Hk;
  const int64_t share = (total + gridDim.x - 1) / gridDim.x;
  const int64_t x0 = share * blockIdx.x, x1 = min(total, x0 + share);
  if (blockIdx.x == 0) {  // for the join
    if (tid == 0) {
      P.plan[0] = n_pre;
      P.plan[1] = n_jobs;
      P.plan[2] = static_cast<int>(share);
      P.plan[3] = no_groups;
    }
    for (int j = tid; j <= n_jobs; j += kThreads) P.plan[kPlanScan + j] = sm.scan[j];
  }

  if (tid >= kCons) {
    // ------------------------------------------------------------ producer warp
    const int sub = 1 << P.sub_shift, nsub = kTile >> P.sub_shift;
    const int batch = 32 / nsub;  // tiles whose page numbers the lanes fetch at once
    const int none = P.n_pages * P.Hk * P.page;  // a row behind the pool: TMA fills with zeros
    constexpr uint32_t bytes = 2 * Cfg<HD>::kOperand;
    int it = 0;
    bool go = true;
    for (int64_t x = x0; x < x1 && go;) {
      const Run r = run_at(sm.scan, n_jobs, x, x1, P.Hk);
      const Job J = warp_job(P, n_pre, sm.ids, r.j, no_groups);
      const int first = J.lo / kTile;
      for (int tb = r.t0; tb < r.t1 && go; tb += batch) {
        const int my = tb + lane / nsub;
        int y = none, bad = 0;
        if (my < r.t1) {
          const int p = (first + my) * kTile + (lane % nsub) * sub;
          if (p + sub > J.lo && p < J.hi) {
            const int pg = P.table[J.trow * P.table_ld + p / P.page];
            if (pg >= 0 && pg < P.n_pages) {
              y = (pg * P.Hk + r.kh) * P.page + p % P.page;
            } else {
              bad = 1;
              report_error(P.err, HM_ERR_BADINDEX);
            }
          }
        }
        const int n = min(batch, r.t1 - tb);
        for (int i = 0; i < n; ++i, ++it) {
          const int st = it % NST;
          const uint32_t no = __ballot_sync(0xffffffffu, bad) >> (i * nsub);
          int ok = 1;
          if (lane == 0 && it >= NST) ok = mbar_wait_short(&sm.empty[st], ((it / NST) - 1) & 1, P.err, &sm.abort_flag);
          go = __shfl_sync(0xffffffffu, ok, 0);
          if (!go) break;
          if (lane == 0) {
            int mask = 0;  // a bit per 16 positions
            for (int b = 0; b < kTile / 16; ++b) mask |= ((no >> ((16 * b) >> P.sub_shift)) & 1) << b;
            sm.bad[st] = mask;
            mbar_arrive_expect_tx(&sm.full[st], bytes);
          }
          __syncwarp();
          // lane i * nsub + s holds the row of sub-box s: it issues that box of K and of V
          if (lane / nsub == i) {
            const int s = lane % nsub, off = s * sub * HD * 2;
            tma_load_3d_plain(sm.kv[st][0] + off, &kmap, 0, y, 0, &sm.full[st]);
            tma_load_3d_plain(sm.kv[st][1] + off, &vmap, 0, y, 0, &sm.full[st]);
          }
          __syncwarp();
        }
      }
      x += r.t1 - r.t0;
    }
  } else {
    // ------------------------------------------------------------ consumers
    Consumer<HD, T> C(P, sm);
    int it = 0;
    for (int64_t x = x0; x < x1;) {
      const Run r = run_at(sm.scan, n_jobs, x, x1, P.Hk);
      const Job J = warp_job(P, n_pre, sm.ids, r.j, no_groups);
      C.begin(J, r.kh);
      const int first = J.lo / kTile;
      for (int tt = r.t0; tt < r.t1; ++tt, ++it) {
        const int st = it % NST;
        mbar_wait_short(&sm.full[st], (it / NST) & 1, P.err, &sm.abort_flag);  // on timeout: carry on, error flagged
        const int bad = sm.bad[st], p0 = (first + tt) * kTile;
        if (J.big)
          C.template tile<4>(st, p0, J, bad);
        else
          C.template tile<1>(st, p0, J, bad);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[st]);
      }
      // a run is one (job, KV head) of one CTA: along the flat order either grows, so their sum
      // numbers the runs of a kind without collisions
      const int64_t slot = (int64_t)(r.j < n_pre ? r.j : r.j - n_pre) * P.Hk + r.kh + blockIdx.x;
      C.finish(J, r.j < n_pre ? slot * P.pre_rows : P.pre_slots * P.pre_rows + slot * P.own_rows);
      x += r.t1 - r.t0;
    }
  }
  pdl_trigger();
}

// Joins the partial results of a (row, head), one warp each: the prefix's in order, then the
// sequence's own.  Nothing to join (a padding row): zeros.
template <int HD, typename T>
__global__ void __launch_bounds__(128) prefix_join_kernel(const __grid_constant__ Params P) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (int64_t)P.R * P.Hq) return;
  const int r = static_cast<int>(id / P.Hq), h = static_cast<int>(id % P.Hq), kh = h / P.G;
  const int n_pre = P.plan[0], b = r / P.S;
  const int64_t share = P.plan[2];
  const int* scan = P.plan + kPlanScan;
  int64_t at[2] = {0, 0}, step[2] = {P.pre_rows, P.own_rows};  // workspace row of the first split, distance of the next
  int cnt[2] = {0, 0};
  auto splits = [&](int j, int unit, int row, int kind) {
    const int tiles = scan[j + 1] - scan[j];
    if (tiles == 0) return;
    const int64_t x = (int64_t)scan[j] * P.Hk + (int64_t)kh * tiles;
    const int64_t c0 = x / share, c1 = (x + tiles - 1) / share;
    cnt[kind] = static_cast<int>(c1 - c0) + 1;
    at[kind] = (kind ? P.pre_slots * P.pre_rows : 0) + ((int64_t)unit * P.Hk + kh + c0) * step[kind] + row;
  };
  const int g = P.plan[3] ? -1 : group_of(P, b);
  if (g >= 0 && group_plen(P, g) > 0) {
    const int a = P.gstart[g], mt = block_rows((P.gstart[g + 1] - a) * P.S * P.G);
    const int i = (r - a * P.S) * P.G + h % P.G, j = P.plan[kPlanGroup + g] + i / mt;
    splits(j, j, i % mt, 0);
  }
  {
    const int mt = block_rows(P.S * P.G), i = (r % P.S) * P.G + h % P.G;
    const int u = b * P.own_blocks + i / mt;
    splits(n_pre + u, u, i % mt, 1);
  }
  const int n = cnt[0] + cnt[1];
  auto row_of = [&](int s) { return s < cnt[0] ? at[0] + s * step[0] : at[1] + (s - cnt[0]) * step[1]; };
  float M = -INFINITY;
  for (int s = lane; s < n; s += 32) M = fmaxf(M, P.pm[row_of(s)]);
  M = warp_max(M);
  const float M0 = M == -INFINITY ? 0.f : M;
  constexpr int V = HD / 32;  // columns of a lane
  float num[V] = {};
  float den = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float w = 0.f, ls = 0.f;
    if (s0 + lane < n) {
      const int64_t rw = row_of(s0 + lane);
      w = ex2(P.pm[rw] - M0);
      ls = P.pl[rw] * w;
    }
    den += warp_sum(ls);
    const int e = min(32, n - s0);
#pragma unroll 4
    for (int s = 0; s < e; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const float* a = P.pa + row_of(s0 + s) * HD + V * lane;
#pragma unroll
      for (int i = 0; i < V; ++i) num[i] += ws * a[i];
    }
  }
  const float inv = den > 0.f ? 1.f / den : (den == 0.f ? 0.f : den);  // NaN stays NaN
  uint32_t out[V / 2];
#pragma unroll
  for (int i = 0; i < V; i += 2) out[i / 2] = Ty<T>::pack(den == 0.f ? 0.f : num[i] * inv, den == 0.f ? 0.f : num[i + 1] * inv);
  uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(P.o) + r * P.ld_o + (int64_t)h * HD + V * lane);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) o[i] = out[i];
}

// ---------------------------------------------------------------- host side
struct Shape {
  int B, G, own_blocks, own_rows, pre_rows;
  int64_t pre_jobs, pre_slots, rows;
};

// Sizes that follow from the arguments alone (the lengths are on the device).
bool shape_of(int R, int S, int Hq, int Hk, int n_groups, int ctas, Shape* s) {
  if (R < 1 || S < 1 || R % S || Hk < 1 || Hq < Hk || Hq % Hk || n_groups < 0) return false;
  s->B = R / S;
  s->G = Hq / Hk;
  if (s->G > 64 || R > (1 << 20)) return false;
  const int64_t own = (int64_t)S * s->G, all = (int64_t)R * s->G;
  const int own_mt = own <= 16 ? 16 : 64;
  s->own_blocks = static_cast<int>((own + own_mt - 1) / own_mt);
  s->own_rows = static_cast<int>(own < own_mt ? own : own_mt);
  s->pre_rows = all <= 16 ? static_cast<int>(all) : 64;
  // groups of up to 16 rows are one job, larger ones one per started 64 rows
  s->pre_jobs = n_groups == 0 ? 0 : (all + 63) / 64 + n_groups;
  if (s->pre_jobs + (int64_t)s->B * s->own_blocks > kMaxJobs || n_groups > kMaxJobs) return false;
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

size_t plan_bytes(int n_groups) { return ((kPlanGroup + n_groups) * sizeof(int) + 255) / 256 * 256; }

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

template <int HD, typename T>
cudaError_t launch(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int grid, int dev, cudaStream_t st) {
  constexpr size_t smem = sizeof(Smem<HD>);
  static std::atomic<bool> configured[kMaxDevices];
  if (dev >= kMaxDevices || !configured[dev].load()) {
    const cudaError_t e = cudaFuncSetAttribute(prefix_attn_kernel<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) configured[dev].store(true);
  }
  cudaError_t e = hm_launch(prefix_attn_kernel<HD, T>, dim3(grid), dim3(kThreads), smem, st, 0, km, vm, p);
  if (e != cudaSuccess) return e;
  const int64_t warps = (int64_t)p.R * p.Hq;
  return hm_launch(prefix_join_kernel<HD, T>, dim3(static_cast<unsigned>((warps + 3) / 4)), dim3(128), 0, st, 1, p);
}

template <int HD>
cudaError_t launch_t(const CUtensorMap& km, const CUtensorMap& vm, const Params& p, int grid, int dev, cudaStream_t st,
                     bool bf16) {
  return bf16 ? launch<HD, __nv_bfloat16>(km, vm, p, grid, dev, st) : launch<HD, __half>(km, vm, p, grid, dev, st);
}

bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }

}  // namespace

extern "C" size_t hm_prefix_attn_workspace_bytes(int R, int S, int Hq, int Hk, int hd, int n_groups, int sms) {
  Shape s;
  if ((hd != 64 && hd != 128 && hd != 256) || sms < 1 || !shape_of(R, S, Hq, Hk, n_groups, sms * ctas_per_sm(hd), &s))
    return 0;
  return plan_bytes(n_groups) + (size_t)s.rows * (hd + 2) * sizeof(float) + 16;
}

extern "C" int hm_prefix_attn(const hm_prefix_attn_desc* d, hm_stream_t stream) {
  if (!d || bad16(d->q) || bad16(d->o) || bad16(d->k) || bad16(d->v) || bad16(d->ws) || !d->pos || !d->table)
    return HM_EARG;
  if ((d->dtype != HM_DT_F16 && d->dtype != HM_DT_BF16) || (d->hd != 64 && d->hd != 128 && d->hd != 256)) return HM_EARG;
  if (d->n_groups > 0 && (!d->gstart || !d->owner || !d->plen)) return HM_EARG;
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
  p.own_blocks = s.own_blocks;
  p.own_rows = s.own_rows;
  p.pre_rows = s.pre_rows;
  p.pre_slots = s.pre_slots;
  p.plan = reinterpret_cast<int*>(d->ws);
  p.pa = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(d->ws) + plan_bytes(d->n_groups));
  p.pm = p.pa + s.rows * d->hd;
  p.pl = p.pm + s.rows;
  p.err = d->err;
  // no more CTAs than there can be tiles
  const int64_t most = (s.pre_jobs + (int64_t)s.B * s.own_blocks) * d->Hk * (((int64_t)d->max_pages * pg) / kTile + 1);
  const int grid = static_cast<int>(most < ctas ? most : ctas);
  e = d->hd == 64    ? launch_t<64>(km, vm, p, grid, dev, stream, bf16)
      : d->hd == 128 ? launch_t<128>(km, vm, p, grid, dev, stream, bf16)
                     : launch_t<256>(km, vm, p, grid, dev, stream, bf16);
  return e == cudaSuccess ? HM_OK : static_cast<int>(e);
}
