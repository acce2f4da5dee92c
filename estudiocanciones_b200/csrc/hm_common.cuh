// Shared device helpers for the HeartMuLa sm_100a decode kernels.
//
// Everything here is plain inline PTX for features the kernels rely on:
// programmatic dependent launch (griddepcontrol), mbarriers with bounded waits,
// TMA tile loads (cp.async.bulk.tensor) and 1-D bulk copies (cp.async.bulk),
// the fp16 tensor-core MMA, and an exact int8 -> fp16 conversion.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdlib>
#include <mutex>
#include <utility>

#include "heartmula_b200.h"

// Upper bound for any wait inside a kernel (mbarrier, split-K fixup). A healthy
// wait ends in microseconds; after this the kernel records HM_ERR_TIMEOUT in the
// caller's error word and returns instead of spinning on.
#ifndef HM_WAIT_NS
#define HM_WAIT_NS 2000000000ull
#endif

#define HM_DEV __device__ __forceinline__

HM_DEV uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---------------------------------------------------------------- programmatic dependent launch
// wait: block until every grid this launch depends on has completed and its
// memory is visible.  Code before it may only read data no earlier kernel writes.
HM_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// trigger: let the next launch in the stream start its prologue early.
HM_DEV void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

HM_DEV uint64_t globaltimer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

HM_DEV void report_error(int* err, int code) {
  if (err) atomicOr(err, code);
}

// ---------------------------------------------------------------- mbarrier
HM_DEV void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
// make barrier initialisation visible to the async (TMA) proxy
HM_DEV void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
HM_DEV void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// order this thread's view of global memory (generic proxy) before its later async-proxy reads
HM_DEV void fence_proxy_async_global() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

HM_DEV void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

HM_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

HM_DEV void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}

HM_DEV bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded wait on phase `parity`.  Returns false (and records HM_ERR_TIMEOUT)
// when the phase does not complete within HM_WAIT_NS or 2^28 polls.
HM_DEV bool mbar_wait(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 28); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0 && globaltimer_ns() - t0 > HM_WAIT_NS) break;
  }
  report_error(err, HM_ERR_TIMEOUT);
  return false;
}

// Bounded wait that never strands a CTA: the first wait to time out sets a
// CTA-wide abort flag in shared memory and every later wait returns at once.
// Callers carry on (computing garbage that the error word flags) instead of
// returning early, so every thread still reaches every barrier and the kernel
// ends in bounded time.
HM_DEV bool mbar_wait_ab(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  if (*abort_flag) return false;
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 28); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > HM_WAIT_NS) break;
    }
  }
  *abort_flag = 1;
  report_error(err, HM_ERR_TIMEOUT);
  return false;
}

// mbar_wait_ab for waits that are mostly short: up to 64 polls before the timer is read.
HM_DEV bool mbar_wait_short(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait_ab(bar, parity, err, abort_flag);
}

// After a wait gave up, copies and matrix products that were issued may still be on their way, and a CTA must
// not hand its memory back before they land.  They take microseconds: each thread that sees the flag stays a millisecond
// (at most 2^20 looks at the clock) before the CTA's last barrier.
HM_DEV void settle(const volatile int* abort_flag) {
  if (!*abort_flag) return;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 20) && globaltimer_ns() - t0 < 1000000ull; ++i) {
  }
}

// ---------------------------------------------------------------- thread-block clusters
HM_DEV uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Every thread of every CTA of the cluster: arrive (release) and wait (acquire).
HM_DEV void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of the same shared-memory location in CTA `rank` of the cluster.
HM_DEV uint32_t dsmem_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
HM_DEV float ld_dsmem_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
HM_DEV void st_dsmem_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
// The 32-bit word at local shared address `p` in CTAs 0..7 of the cluster, the eight
// remote loads issued together (their latencies overlap).
HM_DEV void ld_dsmem_u32_x8(const void* p, uint32_t (&v)[8]) {
  asm volatile(
      "{\n\t.reg .u32 a<8>;\n\t"
      "mapa.shared::cluster.u32 a0, %8, 0;\n\tmapa.shared::cluster.u32 a1, %8, 1;\n\t"
      "mapa.shared::cluster.u32 a2, %8, 2;\n\tmapa.shared::cluster.u32 a3, %8, 3;\n\t"
      "mapa.shared::cluster.u32 a4, %8, 4;\n\tmapa.shared::cluster.u32 a5, %8, 5;\n\t"
      "mapa.shared::cluster.u32 a6, %8, 6;\n\tmapa.shared::cluster.u32 a7, %8, 7;\n\t"
      "ld.shared::cluster.u32 %0, [a0];\n\tld.shared::cluster.u32 %1, [a1];\n\t"
      "ld.shared::cluster.u32 %2, [a2];\n\tld.shared::cluster.u32 %3, [a3];\n\t"
      "ld.shared::cluster.u32 %4, [a4];\n\tld.shared::cluster.u32 %5, [a5];\n\t"
      "ld.shared::cluster.u32 %6, [a6];\n\tld.shared::cluster.u32 %7, [a7];\n\t}\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
      : "r"(smem_u32(p))
      : "memory");
}
HM_DEV void fence_acq_rel_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
// Arrive (release at cluster scope) on an mbarrier of another CTA of the cluster.
HM_DEV void mbar_arrive_dsmem(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}
HM_DEV bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait (acquire at cluster scope) for arrivals from other CTAs of the cluster;
// records HM_ERR_TIMEOUT and returns false after HM_WAIT_NS.
HM_DEV bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 28); ++i) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if ((i & 255u) == 0 && globaltimer_ns() - t0 > HM_WAIT_NS) break;
  }
  report_error(err, HM_ERR_TIMEOUT);
  return false;
}

// ---------------------------------------------------------------- TMA
// 2-D tiled load global -> shared, completion counted on `bar` (bytes).
// x is the innermost coordinate (elements); callers keep x*elem_size % 16 == 0.
HM_DEV void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// 3-D / 4-D tiled loads with an L2 cache hint (x innermost, same alignment rule).
HM_DEV void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}
HM_DEV void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar,
                        uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// Same without an L2 cache hint.
HM_DEV void tma_load_2d_plain(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

HM_DEV void tma_load_3d_plain(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// 1-D bulk copy global -> shared (16-byte aligned addresses, size % 16 == 0).
HM_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Ampere-style asynchronous copies (global -> shared), completed with wait_all.
HM_DEV void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
HM_DEV void cp_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
HM_DEV void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrive on `bar` once every cp.async this thread issued so far has landed
// (the barrier's expected count includes this arrival).
HM_DEV void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Barrier over the first `n` threads of the CTA (id 0 is __syncthreads').
HM_DEV void named_bar(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }

HM_DEV uint64_t policy_evict_first() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
HM_DEV uint64_t policy_evict_last() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}

HM_DEV void prefetch_tensormap(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ---------------------------------------------------------------- math helpers
// Exact int8 -> fp16 for four packed bytes: (b0,b1) -> lo, (b2,b3) -> hi.
// Each byte is biased to 0..255, placed in the mantissa of 1024.0 and the
// bias 1024+128 is subtracted; every int8 value is exactly representable.
HM_DEV void i8x4_to_h2x2(uint32_t v, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = v ^ 0x80808080u;
  lo = __byte_perm(u, 0x64646464u, 0x5140);
  hi = __byte_perm(u, 0x64646464u, 0x5342);
  const uint32_t bias = 0x64806480u;  // 1152.0 in both halves
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(bias));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(bias));
}

// D(16x8,f32) += A(16x16,f16,row) * B(16x8,f16,col)
HM_DEV void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ldmatrix: four 8x8 b16 matrices; lanes 8i..8i+7 give the row addresses of matrix i
HM_DEV void ldsm_x4(uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
HM_DEV void ldsm_x4_t(uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
// two floats -> fp16x2 (first in the low half), round to nearest even
HM_DEV uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

HM_DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
HM_DEV float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// fp16(a) * fp16(b) rounded once to fp16 (the product of two fp16 values is
// exact in fp32, so this equals an IEEE fp16 multiply).
// Sum over t < tiles of ss[t*ld + row] by one warp, lane-strided in increasing t
// (the same order as a plain strided loop), with 16 loads per lane in flight at
// once instead of one memory latency per 32 partials.
HM_DEV float warp_sum_partials(const float* ss, int tiles, int64_t ld, int row, int lane) {
  float a = 0.f;
  for (int base = 0; base < tiles; base += 512) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = base + lane + 32 * i;
      v[i] = t < tiles ? ss[(int64_t)t * ld + row] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) a += v[i];
  }
  return warp_sum(a);
}

// RMSNorm of two packed fp16 values: fp16(fp16(x * inv) * g), each product rounded once
// (register-only: no address-taken temporaries).
HM_DEV uint32_t rms_h2(uint32_t xv, uint32_t gv, float inv) {
  const float x0 = __half2float(__ushort_as_half(static_cast<unsigned short>(xv & 0xffffu)));
  const float x1 = __half2float(__ushort_as_half(static_cast<unsigned short>(xv >> 16)));
  const __half2 n = __floats2half2_rn(x0 * inv, x1 * inv);
  const __half2 g = __halves2half2(__ushort_as_half(static_cast<unsigned short>(gv & 0xffffu)),
                                   __ushort_as_half(static_cast<unsigned short>(gv >> 16)));
  const __half2 r = __hmul2(n, g);
  return static_cast<uint32_t>(__half_as_ushort(__low2half(r))) |
         (static_cast<uint32_t>(__half_as_ushort(__high2half(r))) << 16);
}

HM_DEV __half hmul_rn(__half a, __half b) { return __float2half_rn(__half2float(a) * __half2float(b)); }
HM_DEV __half hadd_rn(__half a, __half b) { return __hadd(a, b); }

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link).
static inline PFN_cuTensorMapEncodeTiled_v12000 hm_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// Every kernel asks for the maximum shared-memory carveout, so consecutive
// kernels never need a different L1/shared split on an SM (a change of split
// drains the SM and defeats overlapping launches).  HM_CARVEOUT=0 turns it off.
template <typename K>
static inline void hm_carveout(K kernel) {
  static const int on = [] {
    const char* e = getenv("HM_CARVEOUT");
    return e ? atoi(e) : 1;
  }();
  if (on) cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
}

// Launch helper: every kernel is launched with the programmatic-stream-
// serialisation attribute when `pdl` is set, so it may overlap the previous
// kernel's tail (its own griddepcontrol.wait keeps the data dependency).
template <typename... KArgs, typename... Args>
static inline cudaError_t hm_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                    cudaStream_t stream, int pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  static bool carved = false;  // once per kernel instantiation
  if (!carved) {
    hm_carveout(kernel);
    carved = true;
  }
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
