// Matrix product in 8-bit integers with a scale for each token and each output channel (sm_100a).
//
//   q[m, k] = round(127 x[m, k] / amax[m]),  sx[m] = amax[m] / 127,  amax[m] = max_k |x[m, k]|
//   acc[m, n] = sum_k q[m, k] * w[n, k]                              (int32, exact: K <= 131072)
//   STORE: c[m, n] = acc * s[n] * sx[m]  (+ res[m, n])
//   SILU : w = [w1; w3], c[m, f] = silu(a) * b,  a, b = the two halves' scaled sums
// Everything after the integers is fp32 and rounded once to the activations' type (fp16, bf16).
// The reference multiplies int8 weights with fp16 activations (app/kernels.py:20-54); with both
// operands in 8 bits the tensor cores run twice as fast and the activations take half the bytes.
//
// quant_kernel: one CTA per token; the row stays in registers between the maximum and the
// rounding, so x is read once (HBM: 3 bytes an element).  127 x is exact in fp32 (at most 18
// bits; bf16 rows above 2^120, where it would overflow, are divided with both sides times 2^-8), so
// one IEEE division decides the rounding; it is only taken where the product with the
// reciprocal lies within 2^-15 of a half (its error is below 127 * 2^-23), else the cheap product
// gives the same integer.  HBM-bound for many tokens: 4096 x 4096 in 11.2 us (4.5 TB/s), one token 2.4 us.
//
// Two products, both tcgen05.mma kind::i8 (K = 32 a step) fed by TMA (128-byte swizzle, K blocks of
// 128 bytes) with the int32 sums in TMEM:
//  * gemm_small: one MT x BN tile per CTA, MT = 64 or 128, BN = 32 .. 128.  For few tokens the weights are all the
//    traffic, so BN is chosen to put the weight stream on as many SMs as there are, and a CTA
//    keeps a ring of up to 200 KB in flight (106 KB where two CTAs share an SM).  Only the rows that exist are loaded: the MMA's
//    other rows read whatever lies behind them in shared memory, and nobody reads their sums.
//    In hm_int8_mm_a8 the weight stream starts before the quantisation has finished
//    (programmatic dependent launch; the weights do not depend on it).
//  * gemm_pair: persistent 256 x 256 tiles on SM pairs (cta_group::2), two accumulators per CTA so
//    that a tile's epilogue overlaps the next tile's products (the layout of gemm_f16w with twice
//    the depth per byte).
// Measured: 8 x 16384 x 4096 in 11.6 us (5.8 TB/s of weights), 1 x 5120 x 4096 in 7.3 (2.9 TB/s: 4.5 us are launch,
// first bytes and epilogue), 4096 x 16384 x 4096 in 164 us (3.36 POP/s, the tensor pipe 92 % busy).
// The integer sums do not depend on the order, so both give the same result bit for bit.
#include <cuda_bf16.h>

#include <atomic>

#include "hm_common.cuh"
#include "tcgen05.cuh"

namespace {

// ---------------------------------------------------------------- types
template <typename T>
struct Ty;
template <>
struct Ty<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  static HM_DEV float2 f2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static HM_DEV uint32_t pack(float a, float b) { return pack_h2(a, b); }
  static HM_DEV float f(__half v) { return __half2float(v); }
  static HM_DEV __half one(float v) { return __float2half_rn(v); }
};
template <>
struct Ty<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u;
  static HM_DEV float2 f2(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
  static HM_DEV uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static HM_DEV float f(__nv_bfloat16 v) { return __bfloat162float(v); }
  static HM_DEV __nv_bfloat16 one(float v) { return __float2bfloat16_rn(v); }
};

// ---------------------------------------------------------------- quantisation of the tokens
constexpr int kQChunks = 4;  // 8-element chunks a thread keeps in registers (K <= 32 * threads)

// Adding 1.5 * 2^23 rounds a small value half to even into the low mantissa bits, whose last byte is
// the integer's: no conversion instructions (they run at an eighth of the adds' rate).
constexpr float kRound = 12582912.f;

HM_DEV uint32_t quant1(float x, float inv, float amax) {
  const float t = __fmul_rn(x, inv), r = __fadd_rn(t, kRound);
  // near a half (or an overflowing reciprocal): the exact quotient decides
  if (!(fabsf(__fsub_rn(t, __fsub_rn(r, kRound))) < 0.5f - 3.0517578125e-5f)) {
    // 127 x has to stay finite: x is at least amax / 256 here, so the power of two costs no bits
    const float f = amax > 0x1p120f ? 0x1p-8f : 1.f;
    return __float_as_uint(__fadd_rn(__fdiv_rn(__fmul_rn(x * f, 127.f), amax * f), kRound));
  }
  return __float_as_uint(r);
}

template <typename T>
HM_DEV uint2 quant8(uint4 v, float inv, float amax) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 a = Ty<T>::f2(u[2 * h]), b = Ty<T>::f2(u[2 * h + 1]);
    out[h] = __byte_perm(__byte_perm(quant1(a.x, inv, amax), quant1(a.y, inv, amax), 0x0040),
                         __byte_perm(quant1(b.x, inv, amax), quant1(b.y, inv, amax), 0x0040), 0x5410);
  }
  return make_uint2(out[0], out[1]);
}

// The largest |x| of 8 elements as 16-bit patterns (ordered like the values; inf and NaN on top).
HM_DEV uint32_t top_bits(uint4 v, uint32_t top) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, u[i] & 0x7fff7fffu);
  return top;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) quant_kernel(const T* __restrict__ x, int64_t ldx, int K, int8_t* __restrict__ q,
                                                   int64_t ldq, float* __restrict__ sx) {
  __shared__ uint32_t red[NT / 32];
  pdl_trigger();
  const int tid = threadIdx.x, nc = K / 8;
  const uint4* row = reinterpret_cast<const uint4*>(x + blockIdx.x * ldx);
  uint2* out = reinterpret_cast<uint2*>(q + blockIdx.x * ldq);
  uint4 v[kQChunks];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) {
    const int c = tid + i * NT;
    v[i] = c < nc ? row[c] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) top = top_bits(v[i], top);
  for (int c = tid + kQChunks * NT; c < nc; c += NT) top = top_bits(row[c], top);  // K > 32 * NT: read twice
  top = max(top & 0xffffu, top >> 16);
  top = __reduce_max_sync(0xffffffffu, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) top = max(top, red[w]);
  const float amax = Ty<T>::f2(top).x;
  const bool zero = top == 0, bad = top >= Ty<T>::kInf;
  const float inv = __fdiv_rn(127.f, amax);
  // a row with an infinity or NaN has the scale NaN: its outputs are NaN, the other rows' are not
  if (tid == 0) sx[blockIdx.x] = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(amax, 127.f);
  const bool none = zero || bad;
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) {
    const int c = tid + i * NT;
    if (c < nc) out[c] = none ? make_uint2(0, 0) : quant8<T>(v[i], inv, amax);
  }
  for (int c = tid + kQChunks * NT; c < nc; c += NT) out[c] = none ? make_uint2(0, 0) : quant8<T>(row[c], inv, amax);
}

// ---------------------------------------------------------------- products
struct GemmParams {
  const __half* s;
  const float* sx;
  const void* res;
  int64_t ldr;
  void* c;
  int64_t ldc;
  int M, N, K;   // N: output columns (features for SILU)
  int w3;        // SILU: row of w3 inside W
  int ntiles;    // pair: tiles along N
  int n_fast;    // pair: consecutive tiles walk N
  int vec;       // rows of c and res start on 16 bytes and hold a multiple of 8 columns
  int m_box;     // small: rows of A that a CTA loads (a multiple of 8)
  int nst;       // small: ring stages
  int deep;      // small: K blocks per stage (one wait and one commit for 4 * deep MMAs)
  int* err;
};

constexpr int BK = 128;  // bytes (= int8 elements) of K per stage: one swizzle row
constexpr int BM = 128;

// kind::i8: D s32, A and B signed 8 bit, K-major
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
HM_DEV void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
HM_DEV void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// silu(a) = a c / (c + c e^-a) with the fast exponential and quotient.  c = 2^-8 keeps the divisor below 2^126, above
// which the fast quotient gives 0, down to a = -92.8; silu(a) leaves the normal numbers (bf16 has the same) at -91.9.  The
// exponent takes its -8 in the product with log2 e.  The exponential is off by about (2 + |a|) 2^-23, the result is rounded
// to 16 bits next.
HM_DEV float silu_f(float a) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(a, -1.4426950408889634f, -8.f)));
  return __fdividef(a * 0x1p-8f, 0x1p-8f + e);
}

// A TMEM integer, scaled.  The channel's scale comes first: an integer times an fp16 value is zero or a normal
// number, while the token's scale of a bf16 row may be anything that fits 32 bits (times the integer alone it can overflow
// where the result does not).
HM_DEV float scaled(float bits, float sx, float scl) { return static_cast<float>(__float_as_int(bits)) * scl * sx; }

// 16 residual values of one row from column `col` on (zero outside)
template <typename T>
HM_DEV void res16(const GemmParams& P, int m, int col, float (&r)[16]) {
  const T* p = reinterpret_cast<const T*>(P.res) + (int64_t)m * P.ldr + col;
  if (P.vec && col + 16 <= P.N) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = Ty<T>::f2(u[i]);
      r[2 * i] = f.x;
      r[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = col + i < P.N ? Ty<T>::f(p[i]) : 0.f;
  }
}

// ---------------------------------------------------------------- few tokens: one tile per CTA
// Warps: 0 streams W, 1 issues the MMAs, 2 streams A, 3-6 the epilogue.  MT = 64 or 128 rows per MMA
// (an MMA with 64 rows takes two thirds of the time of one with 128 at BN = 64).
constexpr int kSmallThreads = 224;
constexpr int kMaxStages = 16;

struct SmallBars {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

template <int BN, int EPI, int MT, typename T>
__global__ void __launch_bounds__(kSmallThreads) gemm_small_kernel(const __grid_constant__ CUtensorMap amap,
                                                                   const __grid_constant__ CUtensorMap wmap,
                                                                   const __grid_constant__ GemmParams P) {
  extern __shared__ uint8_t smem_raw[];  // A stages (deep blocks of m_box rows), then W stages (deep x BN rows)
  uint8_t* const ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ SmallBars sm;
  __shared__ float scl[BN];
  constexpr int W = EPI == HM_EPI_SILU ? BN / 2 : BN;  // output columns of the tile
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nt = blockIdx.x, m0 = blockIdx.y * BM;
  const int nst = P.nst, deep = P.deep;
  const int nb = (P.K + BK - 1) / BK, nk = (nb + deep - 1) / deep;  // K blocks, stages to fill
  constexpr uint32_t w_block = BN * BK;
  const uint32_t a_block = static_cast<uint32_t>(P.m_box) * BK, a_bytes = deep * a_block, w_bytes = deep * w_block;
  uint8_t* const wring = ring + nst * a_bytes;
  int* const err = P.err;
  volatile int* abort_s = &sm.abort_flag;
  if (tid == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < nst; ++i) {
      mbar_init(&sm.full[i], 2);  // both producers' expect_tx
      mbar_init(&sm.empty[i], 1);
    }
    mbar_init(&sm.acc_full, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&sm.tmem_base, BN);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------ TMA producers
    // the weights do not depend on the launch before, so only the tokens wait for it
    if (warp == 2) {
      pdl_wait();
      fence_proxy_async_global();  // the launch before wrote the tokens; TMA reads them
    }
    for (int kb = 0, s = 0, ph = 1; kb < nk; ++kb) {
      if (kb >= nst && !mbar_wait_short(&sm.empty[s], ph, err, abort_s)) break;
      if (elect_one()) {
        const int n = min(deep, nb - kb * deep);  // the last stage may hold fewer blocks
        if (warp == 0) {
          mbar_arrive_expect_tx(&sm.full[s], n * w_block);
          uint8_t* dst = wring + s * w_bytes;
          for (int d = 0; d < n; ++d, dst += w_block) {
            tma_load_2d_plain(dst, &wmap, (kb * deep + d) * BK, nt * W, &sm.full[s]);
            if (EPI == HM_EPI_SILU) tma_load_2d_plain(dst + W * BK, &wmap, (kb * deep + d) * BK, P.w3 + nt * W, &sm.full[s]);
          }
        } else {
          mbar_arrive_expect_tx(&sm.full[s], n * a_block);
          uint8_t* dst = ring + s * a_bytes;
          for (int d = 0; d < n; ++d, dst += a_block) tma_load_2d_plain(dst, &amap, (kb * deep + d) * BK, m0, &sm.full[s]);
        }
      }
      __syncwarp();
      if (++s == nst) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = idesc_i8(MT, BN);
    const uint64_t a0 = sw128_desc(smem_u32(ring)), b0 = sw128_desc(smem_u32(wring));
    for (int kb = 0, s = 0, ph = 0; kb < nk; ++kb) {
      mbar_wait_short(&sm.full[s], ph, err, abort_s);
      tc_fence_after();
      if (elect_one()) {
        const int n = min(deep, nb - kb * deep);
        uint64_t ad = a0 + s * (a_bytes >> 4), bd = b0 + s * (w_bytes >> 4);
        for (int d = 0; d < n; ++d, ad += a_block >> 4, bd += w_block >> 4) {
#pragma unroll
          for (int k = 0; k < BK / 32; ++k) umma_i8(tmem, ad + 2 * k, bd + 2 * k, idesc, (kb | d | k) != 0);
        }
        umma_commit(&sm.empty[s]);
        if (kb == nk - 1) umma_commit(&sm.acc_full);
      }
      __syncwarp();
      if (++s == nst) {
        s = 0;
        ph ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue: a row per thread
    const int et = tid - 96, quad = warp & 3;  // TMEM lanes 32 * (warp % 4) ..
    for (int i = et; i < BN; i += 128) {
      const int col = EPI == HM_EPI_SILU ? nt * W + i % W : nt * W + i;
      scl[i] = col < P.N ? __half2float(P.s[col + (EPI == HM_EPI_SILU && i >= W ? P.w3 : 0)]) : 0.f;
    }
    named_bar(1, 128);
    // rows of the accumulator: 32 per warp, or (64-row MMA) 16 in the lower lanes of each
    const int r0 = MT == 64 ? 16 * quad : 32 * quad;
    const int m = MT == 64 && lane >= 16 ? P.M : m0 + r0 + lane;
    pdl_wait();
    const float sx = m < P.M ? P.sx[m] : 0.f;
    mbar_wait_short(&sm.acc_full, 0, err, abort_s);
    tc_fence_after();
    if (m0 + r0 < P.M) {  // whole warps (tcgen05.ld is warp-wide)
      const uint32_t trow = tmem + (static_cast<uint32_t>(32 * quad) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < W; c0 += 16) {
        __syncwarp();  // rows behind the last one skipped the stores
        float y[16];
        if (EPI == HM_EPI_SILU) {
          float a[16], b[16];
          tmem_ld16(trow + c0, a);
          tmem_ld16(trow + W + c0, b);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            y[i] = silu_f(scaled(a[i], sx, scl[c0 + i])) * scaled(b[i], sx, scl[W + c0 + i]);
        } else {
          tmem_ld16(trow + c0, y);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = scaled(y[i], sx, scl[c0 + i]);
        }
        const int col = nt * W + c0;
        if (m >= P.M || col >= P.N) continue;
        if (EPI != HM_EPI_SILU && P.res) {
          float r[16];
          res16<T>(P, m, col, r);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] += r[i];
        }
        T* c = reinterpret_cast<T*>(P.c) + (int64_t)m * P.ldc + col;
        if (P.vec && col + 16 <= P.N) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            reinterpret_cast<uint4*>(c)[h] =
                make_uint4(Ty<T>::pack(y[8 * h], y[8 * h + 1]), Ty<T>::pack(y[8 * h + 2], y[8 * h + 3]),
                           Ty<T>::pack(y[8 * h + 4], y[8 * h + 5]), Ty<T>::pack(y[8 * h + 6], y[8 * h + 7]));
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (col + i < P.N) c[i] = Ty<T>::one(y[i]);
        }
      }
    }
  }
  settle(abort_s);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

// ---------------------------------------------------------------- many tokens: SM pairs
constexpr int BN2 = 256;
constexpr int kEpiW = 8;
constexpr int kPairThreads = 64 + 32 * kEpiW;
constexpr int NS2 = 5;
constexpr int kTileBytes = BM * BK;  // 16 KB: 128 rows of A, or a CTA's half of the weight tile

struct PairSmem {
  uint8_t a[NS2][kTileBytes];
  uint8_t b[NS2][kTileBytes];
  uint8_t stage[BM * 512];  // 128 rows x 256 results
  __half scl[2][BN2];
  uint64_t full[NS2], empty[NS2];      // full: used in the leader CTA only
  uint64_t acc_full[2], acc_empty[2];  // acc_empty: the leader's, the epilogue warps of both CTAs arrive
  uint32_t tmem_base;
  int abort_flag;
};

// The tile's results: warp w reads TMEM lanes 32 * (w % 4) .. +31 over half of the columns, scales
// (SiLU, residual), rounds and stages them (16-byte chunk c of row r at slot c ^ (r & 7)); then it
// copies its 32 rows out as whole row segments.  `release` hands the accumulator back.
template <int EPI, typename T, typename Release>
HM_DEV void pair_epilogue(const GemmParams& P, uint32_t tmem, int warp, int lane, int m_row0, int nt, uint8_t* stage,
                          __half* scl, Release release) {
  const int et = (warp - 2) * 32 + lane, quad = warp & 3, part = (warp - 2) / 4;
  constexpr int WT = EPI == HM_EPI_SILU ? BN2 / 2 : BN2;  // output columns of the tile
  constexpr int W = WT / 2;                               // of this warp
  constexpr int cpr = W / 8, rpi = 32 / cpr;              // 16-byte chunks per row, rows per copy step
  const int col0 = nt * WT;
  {
    const int col = EPI == HM_EPI_SILU ? col0 + (et & (WT - 1)) : col0 + et;
    scl[et] = col < P.N ? P.s[col + (EPI == HM_EPI_SILU && et >= WT ? P.w3 : 0)] : __float2half_rn(0.f);
  }
  named_bar(1, 32 * kEpiW);
  const int r = 32 * quad + lane, m = m_row0 + r;
  const float sx = m < P.M ? P.sx[m] : 0.f;
  const uint32_t trow = tmem + (static_cast<uint32_t>(32 * quad) << 16);
  uint8_t* const srow = stage + r * 512;
#pragma unroll 1
  for (int c0 = part * W; c0 < (part + 1) * W; c0 += 16) {
    float y[16];
    if (EPI == HM_EPI_SILU) {
      float a[16], b[16];
      tmem_ld16(trow + c0, a);
      tmem_ld16(trow + BN2 / 2 + c0, b);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        y[i] = silu_f(scaled(a[i], sx, __half2float(scl[c0 + i]))) *
               scaled(b[i], sx, __half2float(scl[BN2 / 2 + c0 + i]));
    } else {
      float rr[16];
      const bool add = P.res && m < P.M && col0 + c0 < P.N;
      if (add) res16<T>(P, m, col0 + c0, rr);
      __syncwarp();
      tmem_ld16(trow + c0, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = scaled(y[i], sx, __half2float(scl[c0 + i])) + (add ? rr[i] : 0.f);
    }
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = Ty<T>::pack(y[2 * i], y[2 * i + 1]);
    const int ch = c0 / 8;
    *reinterpret_cast<uint4*>(srow + ((ch ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(srow + (((ch + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
  }
  release();
  __syncwarp();
  T* const C = reinterpret_cast<T*>(P.c);
#pragma unroll 4
  for (int it = 0; it < 32 / rpi; ++it) {
    const int rr = 32 * quad + it * rpi + lane / cpr, ch = part * cpr + lane % cpr;
    const int mm = m_row0 + rr, col = col0 + 8 * ch;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 512 + ((ch ^ (rr & 7)) << 4));
    if (mm >= P.M || col >= P.N) continue;
    T* c = C + (int64_t)mm * P.ldc + col;
    if (P.vec) {
      *reinterpret_cast<uint4*>(c) = v;
    } else {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < P.N) c[i] = e[i];
    }
  }
}

static_assert(sizeof(PairSmem) + 1024 <= 227 * 1024, "one CTA per SM");

template <int EPI, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ GemmParams P) {
  extern __shared__ uint8_t smem_raw[];
  PairSmem& sm = *reinterpret_cast<PairSmem*>(smem_raw + ((1024 - (smem_u32(smem_raw) & 1023u)) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
  const int mpairs = (P.M + 2 * BM - 1) / (2 * BM), tiles = mpairs * P.ntiles;
  const int nk = (P.K + BK - 1) / BK;
  int* const err = P.err;
  constexpr int WT = EPI == HM_EPI_SILU ? BN2 / 2 : BN2;
  if (tid == 0) {
    sm.abort_flag = 0;
    for (int i = 0; i < NS2; ++i) {
      mbar_init(&sm.full[i], 1);   // the leader's producer (expect_tx) + both CTAs' copies (bytes)
      mbar_init(&sm.empty[i], 1);  // the leader's MMA commit
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.acc_full[i], 1);
      mbar_init(&sm.acc_empty[i], 2 * kEpiW);
    }
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_pair(&sm.tmem_base, 2 * BN2);
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_s = &sm.abort_flag;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      prefetch_tensormap(&amap);
      prefetch_tensormap(&wmap);
    }
    fence_proxy_async_global();  // the launch before wrote the tokens; TMA reads them
    __syncwarp();
    const uint32_t full0 = dsmem_addr(&sm.full[0], 0);
    int g = 0;
    for (int t = pair; t < tiles; t += npairs) {
      const int mp = P.n_fast ? t / P.ntiles : t % mpairs, nt = P.n_fast ? t % P.ntiles : t / mpairs;
      const int m_row0 = mp * 2 * BM + static_cast<int>(rank) * BM;
      const int brow = EPI == HM_EPI_SILU ? (rank == 0 ? 0 : P.w3) + nt * WT : nt * WT + static_cast<int>(rank) * BM;
      for (int kb = 0; kb < nk; ++kb, ++g) {
        const int s = g % NS2;
        if (g >= NS2) mbar_wait_short(&sm.empty[s], ((g / NS2) - 1) & 1, err, abort_s);
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], 4 * kTileBytes);
          tma_load_2d_pair(sm.a[s], &amap, kb * BK, m_row0, full0 + 8 * s);
          tma_load_2d_pair(sm.b[s], &wmap, kb * BK, brow, full0 + 8 * s);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA)
    if (rank == 0) {
      constexpr uint32_t idesc = idesc_i8(2 * BM, BN2);
      const uint64_t a0 = sw128_desc(smem_u32(sm.a[0])), b0 = sw128_desc(smem_u32(sm.b[0]));
      int g = 0, i = 0;
      for (int t = pair; t < tiles; t += npairs, ++i) {
        const int ab = i & 1;
        if (i >= 2 && !*abort_s && !mbar_wait_cluster(&sm.acc_empty[ab], ((i >> 1) - 1) & 1, err)) *abort_s = 1;
        tc_fence_after();
        const uint32_t acc = tmem + ab * BN2;
        for (int kb = 0; kb < nk; ++kb, ++g) {
          const int s = g % NS2;
          mbar_wait_short(&sm.full[s], (g / NS2) & 1, err, abort_s);
          tc_fence_after();
          if (elect_one()) {
            const uint64_t ad = a0 + s * (kTileBytes >> 4), bd = b0 + s * (kTileBytes >> 4);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k) umma_i8_pair(acc, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0);
            umma_commit_pair(&sm.empty[s]);
            if (kb == nk - 1) umma_commit_pair(&sm.acc_full[ab]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs: their 128 rows)
    const uint32_t acc_empty0 = dsmem_addr(&sm.acc_empty[0], 0);
    int i = 0;
    for (int t = pair; t < tiles; t += npairs, ++i) {
      const int ab = i & 1;
      const int mp = P.n_fast ? t / P.ntiles : t % mpairs, nt = P.n_fast ? t % P.ntiles : t / mpairs;
      const int m_row0 = mp * 2 * BM + static_cast<int>(rank) * BM;
      mbar_wait_short(&sm.acc_full[ab], (i >> 1) & 1, err, abort_s);
      tc_fence_after();
      pair_epilogue<EPI, T>(P, tmem + ab * BN2, warp, lane, m_row0, nt, sm.stage, sm.scl[ab], [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (rank == 0)
            mbar_arrive(&sm.acc_empty[ab]);
          else
            mbar_arrive_dsmem(acc_empty0 + 8 * ab);
        }
      });
    }
  }
  settle(abort_s);
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves while the pair's copies, MMAs or commits may touch its memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN2);
  }
}

// ---------------------------------------------------------------- host side
constexpr int kMaxDevices = 64;

cudaError_t device_sms(int* dev, int* sms) {
  static std::atomic<int> known[kMaxDevices];
  cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return e;
  if (*dev < kMaxDevices && (*sms = known[*dev].load()) > 0) return cudaSuccess;
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev);
  if (e == cudaSuccess && *dev < kMaxDevices) known[*dev].store(*sms);
  return e;
}

// int8 [rows, cols] with a row pitch of ld bytes: boxes of 128 bytes x box_rows, 128-byte swizzle
bool tile_map(const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows, CUtensorMap* out) {
  auto enc = hm_encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {BK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t es[2] = {1, 1};
  return enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
cudaError_t max_smem(K kernel, std::atomic<bool>* configured, int dev, size_t bytes) {
  if (dev < kMaxDevices && configured[dev].load()) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < kMaxDevices) configured[dev].store(true);
  return e;
}

// A small CTA's ring: two CTAs per SM, or one when the grid has no more CTAs than SMs (8 x 5120 x 4096:
// 7.2 us with 200 KB, 9.2 with 106; 64 x 16384 x 4096: 11.4, 13.9).
constexpr int kRingTwo = 106 * 1024, kRingOne = 200 * 1024;

template <int BN, int EPI, int MT, typename T>
cudaError_t launch_small(const CUtensorMap& am, const CUtensorMap& wm, GemmParams p, int sms, int dev, int pdl,
                         cudaStream_t st) {
  static std::atomic<bool> configured[kMaxDevices];
  const cudaError_t e = max_smem(gemm_small_kernel<BN, EPI, MT, T>, configured, dev, kRingOne + 1024);
  if (e != cudaSuccess) return e;
  constexpr int W = EPI == HM_EPI_SILU ? BN / 2 : BN;
  const dim3 grid((p.N + W - 1) / W, (p.M + BM - 1) / BM);
  const int room = (int64_t)grid.x * grid.y <= sms ? kRingOne : kRingTwo;
  const int block = (p.m_box + BN) * BK, nb = (p.K + BK - 1) / BK;
  p.deep = 4;
  while (p.deep > 1 && room / (p.deep * block) < 3) p.deep /= 2;
  const int nk = (nb + p.deep - 1) / p.deep;
  p.nst = room / (p.deep * block) < kMaxStages ? room / (p.deep * block) : kMaxStages;
  if (p.nst > nk) p.nst = nk;
  static_assert(kRingTwo / ((MT + BN) * BK) >= 3 && 2 * kRingTwo + 6 * 1024 <= 228 * 1024 && kRingOne + 3 * 1024 <= 227 * 1024,
                "ring");
  // from the last A block the MMA reads MT rows: they have to lie inside the allocation
  const int used = p.nst * p.deep * block, reach = (p.deep * p.nst - 1) * p.m_box * BK + MT * BK;
  return hm_launch(gemm_small_kernel<BN, EPI, MT, T>, grid, dim3(kSmallThreads),
                   static_cast<size_t>(used > reach ? used : reach) + 1024, st, pdl, am, wm, p);
}

template <int EPI, int MT, typename T>
cudaError_t launch_bn(const CUtensorMap& am, const CUtensorMap& wm, const GemmParams& p, int bn, int sms, int dev,
                      int pdl, cudaStream_t st) {
  switch (bn) {
    case 128: return launch_small<128, EPI, MT, T>(am, wm, p, sms, dev, pdl, st);
    case 64: return launch_small<64, EPI, MT, T>(am, wm, p, sms, dev, pdl, st);
    default: return launch_small<32, EPI, MT, T>(am, wm, p, sms, dev, pdl, st);
  }
}

template <int EPI, typename T>
cudaError_t launch_pair(const CUtensorMap& am, const CUtensorMap& wm, GemmParams p, int sms, int dev, int pdl,
                        cudaStream_t st) {
  static std::atomic<bool> configured[kMaxDevices];
  constexpr size_t smem = sizeof(PairSmem) + 1024;
  const cudaError_t e = max_smem(gemm_pair_kernel<EPI, T>, configured, dev, smem);
  if (e != cudaSuccess) return e;
  constexpr int WT = EPI == HM_EPI_SILU ? BN2 / 2 : BN2;
  p.ntiles = (p.N + WT - 1) / WT;
  // the tiles in flight share the larger operand's rows: 16384 x 4096 x 4096 in 170 us with N fast, 187 with M fast;
  // 4096 x 16384 x 4096 191 and 185; 8192 x 2048 x 4096 48.2 and 47.1 (both fit the L2)
  p.n_fast = p.M > (EPI == HM_EPI_SILU ? 2 * p.N : p.N);
  const int64_t tiles = (int64_t)((p.M + 2 * BM - 1) / (2 * BM)) * p.ntiles;
  const int pairs = static_cast<int>(tiles < sms / 2 ? tiles : sms / 2);
  return hm_launch(gemm_pair_kernel<EPI, T>, dim3(2 * pairs), dim3(kPairThreads), smem, st, pdl, am, wm, p);
}

template <int EPI, typename T>
cudaError_t launch_gemm(const int8_t* q, int64_t ldq, const int8_t* w, GemmParams p, int wrows, int pdl, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = device_sms(&dev, &sms);
  if (e != cudaSuccess) return e;
  CUtensorMap am, wm;
  const int64_t pair_tiles = (int64_t)((p.M + 255) / 256) * ((wrows + 255) / 256);
  // pairs once half of them have a tile; at K = N = 4096, us small / pairs: M 256 10.6 / 15.4, 512 12.6 / 15.8,
  // 640 17.8 / 16.1, 1024 18.3 / 16.5, 2048 34.0 / 25.9
  if (p.M > BM && pair_tiles >= sms / 4) {
    if (!tile_map(q, p.M, p.K, ldq, BM, &am) || !tile_map(w, wrows, p.K, p.K, BM, &wm)) return cudaErrorInvalidValue;
    return launch_pair<EPI, T>(am, wm, p, sms, dev, pdl, st);
  }
  const int mt = (p.M + BM - 1) / BM;
  p.m_box = p.M < BM ? (p.M + 7) / 8 * 8 : BM;
  // the tile width whose CTAs cost an SM the least: cycles per MMA (measured, with a share of the
  // waits) times the CTAs that an SM gets.  us at 32 / 64 / 128, K 4096, the rule's in brackets: 1 x 1024 [6.1] / 6.9 / 10.6,
  // 1 x 5120 8.1 / [7.2] / 10.7, 8 x 16384 14.2 / 11.1 / [11.4], 64 x 5120 9.3 / [7.6] / 11.1, 64 x 16384 17.8 / 11.0 / [11.8],
  // 128 x 5120 14.5 / [11.0] / 12.7, 128 x 16384 26.6 / 16.9 / [12.7], 333 x 4096 (K 2048) 15.2 / 10.5 / [8.3].
  const int64_t cycles[2][3] = {{37, 45, 77}, {53, 61, 77}};
  int bn = 0;
  int64_t best = INT64_MAX;
  for (int i = 2; i >= 0; --i) {
    const int64_t tiles = (int64_t)mt * ((wrows + (32 << i) - 1) / (32 << i));
    const int64_t cost = (tiles + sms - 1) / sms * cycles[p.M > 64][i];
    if (cost < best) {
      best = cost;
      bn = 32 << i;
    }
  }
  if (!tile_map(q, p.M, p.K, ldq, p.m_box, &am) ||
      !tile_map(w, wrows, p.K, p.K, EPI == HM_EPI_SILU ? bn / 2 : bn, &wm))
    return cudaErrorInvalidValue;
  return p.M <= 64 ? launch_bn<EPI, 64, T>(am, wm, p, bn, sms, dev, pdl, st)
                   : launch_bn<EPI, 128, T>(am, wm, p, bn, sms, dev, pdl, st);
}

bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15u); }
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

bool x_ok(const void* x, int64_t ldx, int dtype, int M, int K) {
  return !bad16(x) && (dtype == HM_DT_F16 || dtype == HM_DT_BF16) && M >= 1 && K >= 16 && K % 16 == 0 && K <= 131072 &&
         ldx >= K && ldx % 8 == 0;
}

bool out_ok(const int8_t* w, const void* s, const void* res, int64_t ldr, const void* c, int64_t ldc, int N, int epi) {
  if (bad16(w) || !s || !c || N < 1 || (epi != HM_EPI_STORE && epi != HM_EPI_SILU)) return false;
  if (epi == HM_EPI_SILU && (res || N % 2)) return false;
  const int nout = epi == HM_EPI_SILU ? N / 2 : N;
  return ldc >= nout && (!res || ldr >= nout) && !(reinterpret_cast<uintptr_t>(s) & 1u) &&
         !(reinterpret_cast<uintptr_t>(c) & 1u) && !(reinterpret_cast<uintptr_t>(res) & 1u);
}

template <typename T>
cudaError_t quantise(const void* x, int64_t ldx, int M, int K, int8_t* q, int64_t ldq, float* sx, cudaStream_t st) {
  const T* p = reinterpret_cast<const T*>(x);
  // as few threads as keep a row in registers: more rows in flight per SM (4096 rows, us with 128 / 256 / 512
  // threads: K 4096 11.2 / - / 17.2, K 8192 23.4 / 20.7 / 26.0, K 14336 47.8 / - / 36.2)
  if (K <= 128 * 8 * kQChunks) return hm_launch(quant_kernel<T, 128>, dim3(M), dim3(128), 0, st, 0, p, ldx, K, q, ldq, sx);
  if (K <= 256 * 8 * kQChunks) return hm_launch(quant_kernel<T, 256>, dim3(M), dim3(256), 0, st, 0, p, ldx, K, q, ldq, sx);
  return hm_launch(quant_kernel<T, 512>, dim3(M), dim3(512), 0, st, 0, p, ldx, K, q, ldq, sx);
}

cudaError_t multiply(const int8_t* q, int64_t ldq, const float* sx, int dtype, const int8_t* w, const void* s,
                     const void* res, int64_t ldr, void* c, int64_t ldc, int M, int N, int K, int epi, int* err, int pdl,
                     cudaStream_t st) {
  GemmParams p = {};
  p.s = reinterpret_cast<const __half*>(s);
  p.sx = sx;
  p.res = res;
  p.ldr = ldr;
  p.c = c;
  p.ldc = ldc;
  p.M = M;
  p.N = epi == HM_EPI_SILU ? N / 2 : N;
  p.K = K;
  p.w3 = epi == HM_EPI_SILU ? N / 2 : 0;
  p.vec = p.N % 8 == 0 && ldc % 8 == 0 && !off16(c) && (!res || (ldr % 8 == 0 && !off16(res)));
  p.err = err;
  if (epi == HM_EPI_SILU)
    return dtype == HM_DT_F16 ? launch_gemm<HM_EPI_SILU, __half>(q, ldq, w, p, N, pdl, st)
                              : launch_gemm<HM_EPI_SILU, __nv_bfloat16>(q, ldq, w, p, N, pdl, st);
  return dtype == HM_DT_F16 ? launch_gemm<HM_EPI_STORE, __half>(q, ldq, w, p, N, pdl, st)
                            : launch_gemm<HM_EPI_STORE, __nv_bfloat16>(q, ldq, w, p, N, pdl, st);
}

int rc_of(cudaError_t e) { return e == cudaSuccess ? HM_OK : static_cast<int>(e); }

size_t scale_bytes(int M) { return ((size_t)M * sizeof(float) + 255) / 256 * 256; }

}  // namespace

extern "C" int hm_quant_tokens(const void* x, int64_t ldx, int dtype, int M, int K, int8_t* q, int64_t ldq, float* sx,
                               hm_stream_t stream) {
  if (!x_ok(x, ldx, dtype, M, K) || bad16(q) || !sx || (reinterpret_cast<uintptr_t>(sx) & 3u) || ldq < K || ldq % 8)
    return HM_EARG;
  return rc_of(dtype == HM_DT_F16 ? quantise<__half>(x, ldx, M, K, q, ldq, sx, stream)
                                  : quantise<__nv_bfloat16>(x, ldx, M, K, q, ldq, sx, stream));
}

extern "C" int hm_gemm_i8a8(const int8_t* q, int64_t ldq, const float* sx, int dtype, const int8_t* w, const void* s,
                            const void* res, int64_t ldr, void* c, int64_t ldc, int M, int N, int K, int epi, int* err,
                            hm_stream_t stream) {
  if (bad16(q) || ldq < K || ldq % 16 || !sx || (reinterpret_cast<uintptr_t>(sx) & 3u) || M < 1 || K < 16 || K % 16 ||
      K > 131072 || (dtype != HM_DT_F16 && dtype != HM_DT_BF16) || !out_ok(w, s, res, ldr, c, ldc, N, epi))
    return HM_EARG;
  return rc_of(multiply(q, ldq, sx, dtype, w, s, res, ldr, c, ldc, M, N, K, epi, err, 0, stream));
}

extern "C" size_t hm_int8_mm_a8_workspace_bytes(int M, int K) {
  return M < 1 || K < 1 ? 0 : scale_bytes(M) + (size_t)M * K;
}

extern "C" int hm_int8_mm_a8(const void* x, int64_t ldx, int dtype, const int8_t* w, const void* s, const void* res,
                             int64_t ldr, void* c, int64_t ldc, int M, int N, int K, int epi, void* ws, size_t ws_bytes,
                             int* err, hm_stream_t stream) {
  if (!x_ok(x, ldx, dtype, M, K) || !out_ok(w, s, res, ldr, c, ldc, N, epi) || bad16(ws) ||
      ws_bytes < hm_int8_mm_a8_workspace_bytes(M, K))
    return HM_EARG;
  float* sx = reinterpret_cast<float*>(ws);
  int8_t* q = reinterpret_cast<int8_t*>(ws) + scale_bytes(M);
  cudaError_t e = dtype == HM_DT_F16 ? quantise<__half>(x, ldx, M, K, q, K, sx, stream)
                                     : quantise<__nv_bfloat16>(x, ldx, M, K, q, K, sx, stream);
  // the product may start beside the quantisation: that launch waits for everything before it, and
  // the product reads only the weights and their scales before it waits in turn
  if (e == cudaSuccess) e = multiply(q, K, sx, dtype, w, s, res, ldr, c, ldc, M, N, K, epi, err, 1, stream);
  return rc_of(e);
}
