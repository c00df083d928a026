// qrb200 -- matrix product with bias, activation and residual in its epilogue, on tcgen05.
//
//   D_ij = act( p_i q_j sum_k P_ik Q_jk + b_j ) + R_ij
// P (i: tokens) and Q (j: features) are bf16, f16 or e4m3; the sum is float32 in tensor memory,
// the epilogue is float32 and D is rounded once.  For a layer's forward pass P = x, Q = W; its
// backward products are the same kernel on other views: dx = dz W is P = dz, Q = W^T and
// dW = dz^T x is P = dz^T, Q = x^T.  A transposed view is not copied: an operand is either
// contiguous along k ("k-major") or along its rows ("row-major"), and both have a tensor map and a
// tcgen05 descriptor form.
//
// Shared-memory operand tiles (128-byte swizzle, rows of 128 bytes, 1024-byte atoms):
//   k-major    [rows][128 B of k]: descriptor stride 1024 between 8-row groups; the next 32 bytes
//              of k start 32 bytes on.
//   row-major  chunks of 64 rows, each [64 k][64 rows = 128 B] = 8192 bytes: descriptor stride
//              1024 between groups of 8 k, 8192 between chunks; the next 16 k start 2048 bytes on.
// Boxes that reach past an edge are filled with zeros, which add nothing.
#pragma once
#include <cuda_fp8.h>

#include "qrb_f2.cuh"
#include "qrb_pdl.cuh"
#include "qrb_tc.cuh"
#include "qrb_tmap.cuh"

namespace qrb {
namespace lin {

enum Activation : int { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_COUNT };

// Bounded wait; false when it ran out.  The limit is that of the factorization's tiles; a library of its own,
// for a test, is built with waits that run out at once.
#ifndef QRB_LAYER_WAIT_LIMIT
#define QRB_LAYER_WAIT_LIMIT tc::kSpinLimit
#endif
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t phase) { return tc::mbar_wait_n(bar, phase, QRB_LAYER_WAIT_LIMIT); }

// Raised by a kernel whose bounded wait ran out; its tile is then filled with NaN.
__device__ int g_timeout;
// Takes it for the host in one step: what another stream raises meanwhile stays for the next time.
__device__ int g_taken;
__global__ void take_timeout() { g_taken = atomicExch(&g_timeout, 0); }

struct Epilogue {
  const float* row_scale;  // p (null: 1); 8-bit operands only
  const float* col_scale;  // q (null: 1); likewise
  const void* bias;        // b, in the output's type, or null
  const void* res;         // R, in the output's type, or null
  int64_t ldr;
  void* out;
  int64_t ldo;
  uint16_t* slope;         // act'(z), m x n contiguous, or null (see pack_slopes)
  int act;
};

struct Args {
  int m, n, k;             // D is m x n
  int splits;              // CTAs of a cluster that share a tile's sum
  int part;                // 128-byte blocks of k of each of them (the last may have fewer)
  uint32_t idesc;          // element types and operand majors
  int es;                  // bytes of an operand element
  int p_row, q_row;        // operand is row-major (contiguous along its rows)
  int vec;                 // out / res / bias / slope rows allow 4-element accesses
  Epilogue e;
};

struct Maps {
  CUtensorMap p, q;
};

// act' is kept for the backward pass in 16 bits: its root, with its sign, in fixed point, 2^15 (t + 3/8)
// with act' = t |t|.  act' lies in (-0.13, 1.13) for every activation here, t in (-0.37, 1.07); steps of
// 2^-15 hold 0 and 1 exactly and the rest to 2 |t| 2^-16, so to 3.3e-5 at most and to 2^-8 of its value, a
// bf16 dz's own rounding, down to 6e-5.  (act' itself in such steps is off by 1.6e-5 everywhere: a feature
// whose z all lie in a tail lost 3 % of its gradient at z = -4 of gelu and all of it at -5.  A bf16 act' or z
// would be off by up to 2e-3 of its value.)  65535 stands for NaN.
// Adding 2^23 rounds to an integer and leaves it in the low bits; those of a NaN are all ones.
__device__ __forceinline__ float signed_root(float s) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fabsf(s)));
  return copysignf(r, s);
}
__device__ __forceinline__ uint32_t pack_slopes(F2 s) {  // two of them
  float a, b;
  split(s, a, b);
  split(fma(f2(signed_root(a), signed_root(b)), f2(32768.f), f2(8388608.f + 12288.f)), a, b);
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
}
__device__ __forceinline__ float slope_value(uint32_t bits) {
  const float t = fmaf(__uint_as_float(0x4B000000u | bits), 1.f / 32768.f, -256.375f);
  return bits == 0xFFFFu ? __int_as_float(0x7FFFFFFF) : t * fabsf(t);
}

// 1 / x and 2^x of the special-function unit, good to about 2^-22 of the result.
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ F2 rcp(F2 x) {
  float a, b;
  split(x, a, b);
  return f2(rcp_fast(a), rcp_fast(b));
}
__device__ __forceinline__ F2 exp2_(F2 x) {
  float a, b;
  split(x, a, b);
  return f2(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// act(z) of two values; with SLOPE also act'(z).  The epilogue runs beside the MMAs and shares their
// power, so every instruction shows: two special functions and about seven others a value.  gelu
// takes the normal integral from Abramowitz and Stegun's approximation 7.1.26 of the error function
// (off by 1.5e-7 at most),
//   Phi(-|z|) = exp(-z^2 / 2) (a1 t + ... + a5 t^5) / 2,  t = 1 / (1 + p |z| / sqrt 2),
// as z Phi(z) = max(z, 0) - |z| Phi(-|z|); its slope needs the same exponential.
template <int ACT, bool SLOPE>
__device__ __forceinline__ F2 activate(F2 z, F2& slope) {
  constexpr float kLog2e = 1.4426950408889634f;
  float a, b;
  split(z, a, b);
  if constexpr (ACT == ACT_RELU) {
    if (SLOPE) slope = f2(a > 0.f ? 1.f : (a != a ? a : 0.f), b > 0.f ? 1.f : (b != b ? b : 0.f));
    return f2(max_nan(a, 0.f), max_nan(b, 0.f));
  } else if constexpr (ACT == ACT_GELU) {
    const float ma = fminf(fabsf(a), 1e18f), mb = fminf(fabsf(b), 1e18f);  // finite: times a tail of 0
    const F2 m = f2(ma, mb);
    const F2 t = rcp(fma(m, f2(0.3275911f * 0.70710678118654752f), f2(1.f)));
    const F2 ex = exp2_(mul(mul(z, z), f2(-0.5f * kLog2e)));
    F2 s = fma(t, f2(0.5f * 1.061405429f), f2(0.5f * -1.453152027f));
    s = fma(s, t, f2(0.5f * 1.421413741f));
    s = fma(s, t, f2(0.5f * -0.284496736f));
    s = fma(s, t, f2(0.5f * 0.254829592f));
    const F2 tail = mul(mul(s, t), ex);  // Phi(-|z|)
    if (SLOPE) {
      float ta, tb;
      split(tail, ta, tb);
      slope = fma(mul(z, ex), f2(0.3989422804014327f), f2(a > 0.f ? 1.f - ta : ta, b > 0.f ? 1.f - tb : tb));
    }
    return fma(f2(-ma, -mb), tail, f2(max_nan(a, 0.f), max_nan(b, 0.f)));
  } else if constexpr (ACT == ACT_GELU_TANH) {  // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    const F2 z2 = f2(fminf(a * a, 1e30f), fminf(b * b, 1e30f));  // its product with a vanished 1 - p stays 0
    const F2 p = rcp(add(exp2_(mul(mul(z, f2(-1.5957691216057308f * kLog2e)), fma(z2, f2(0.044715f), f2(1.f)))), f2(1.f)));
    const F2 y = mul(z, p);
    if (SLOPE) slope = fma(mul(mul(y, fma(p, f2(-1.f), f2(1.f))), f2(1.5957691216057308f)), fma(z2, f2(0.134145f), f2(1.f)), p);
    return y;
  } else if constexpr (ACT == ACT_SILU) {
    const F2 p = rcp(add(exp2_(mul(z, f2(-kLog2e))), f2(1.f)));
    if (SLOPE) slope = mul(p, fma(z, fma(p, f2(-1.f), f2(1.f)), f2(1.f)));
    return mul(z, p);
  } else {
    if (SLOPE) slope = f2(1.f);
    return z;
  }
}
template <int ACT, bool SLOPE, int N>
__device__ __forceinline__ void activate_as(F2 (&v)[N], F2 (&sl)[N]) {
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] = activate<ACT, SLOPE>(v[c], sl[c]);
}
// act() of 2N values, with the choice made once.
template <bool SLOPE, int N>
__device__ __forceinline__ void activate_all(int act, F2 (&v)[N], F2 (&sl)[N]) {
  switch (act) {
    case ACT_RELU: activate_as<ACT_RELU, SLOPE>(v, sl); break;
    case ACT_GELU: activate_as<ACT_GELU, SLOPE>(v, sl); break;
    case ACT_GELU_TANH: activate_as<ACT_GELU_TANH, SLOPE>(v, sl); break;
    case ACT_SILU: activate_as<ACT_SILU, SLOPE>(v, sl); break;
    default: activate_as<ACT_NONE, SLOPE>(v, sl);
  }
}

// Two 16-bit values <-> float32 pair.
__device__ __forceinline__ F2 widen2(uint32_t w, __nv_bfloat16) { return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ F2 widen2(uint32_t w, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2(f.x, f.y);
}
__device__ __forceinline__ uint32_t narrow2(F2 x, __nv_bfloat16) {
  float a, b;
  split(x, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(F2 x, __half) {
  float a, b;
  split(x, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- small PTX helpers on top of qrb_tc.cuh ----
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(tc::smem_u32(bar))
      : "memory");
}
// Instruction descriptor: D float32, both operands of one type (code: f16 0, bf16 1; e4m3 0).
__host__ __device__ constexpr uint32_t idesc(int type, int a_row, int b_row, int m, int n) {
  return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)a_row << 15) |
         ((uint32_t)b_row << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Shared-memory descriptor of an operand tile (see the layouts above).
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int row_major) {
  const uint64_t lead = row_major ? (8192u >> 4) : 1u;
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <int ES>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    uint32_t accumulate) {
  if (ES == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// 16 consecutive float32 columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(r[x]);
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(r)
               : "memory");
  return v;
}

// A role whose wait ran out: raises the flag and gives the loads and MMAs in flight, whose
// barriers may be another thread's or another CTA's to poll, about 10 ms to end.
__device__ __forceinline__ void give_up() {
  atomicExch(&g_timeout, 1);
  for (int i = 0; i < 1000; ++i) __nanosleep(10000);
}

// 4 adjacent elements of row i from column j, zero past the edge, as they are stored.
template <typename T>
__device__ __forceinline__ uint2 fetch4(const T* p, bool vec, int left) {
  if (vec && left >= 4) return *reinterpret_cast<const uint2*>(p);
  uint2 a = make_uint2(0, 0);
  T* e = reinterpret_cast<T*>(&a);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (c < left) e[c] = p[c];
  return a;
}
template <typename T>
__device__ __forceinline__ void widen4(uint2 a, float (&v)[4]) {
  const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = to_f32(e[c]);
}
// 4 adjacent elements of a row from column j, what lies past the edge left out.
__device__ __forceinline__ void put4(void* p, uint2 packed, bool vec, int left) {
  if (vec && left >= 4) {
    *reinterpret_cast<uint2*>(p) = packed;
  } else {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(&packed);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < left) static_cast<uint16_t*>(p)[c] = e[c];
  }
}

// ---- one 128 (j) x T (i) tile per cluster of `splits` CTAs ----
// Q's rows are the MMA's 128 rows, P's the T columns, so few tokens cost a narrow MMA and not a
// padded one; the CTAs of a cluster take equal parts of k, leave their float32 sums in shared
// memory, and each finishes T / splits of the tile's rows with its peers' sums read over the
// cluster, added in rank order.  Roles: warps 0-7 epilogue, warps 8 and 10 loads, warp 9 MMAs.  The loads
// start before anything else is set up, and the epilogue warps fetch bias and scales (and the
// residual, as far as the L2 cache) while the sums are made: these calls are short, and each wait
// for memory would show.  So would the time to fetch instructions that run once (with 16 rows
// unrolled, finishing a tile took 16 us): loops stay loops, and there are no divisions.  Bound by the
// rate at which an SM fetches its operands, and when short by set-up, exchange and epilogue, about
// 4 us: 16 x 8192 x 8192 in 8 bits 14.5 us (4.6 TB/s), 128 x 4096 x 4096 bf16 12.9 us.
constexpr int kTileThreads = 352;
constexpr int kTileQ = 128;

// RINGS = 2: half an SM's shared memory, two CTAs an SM; 1: all of it, for grids of one CTA an SM.
template <int T, int RINGS>
struct TileCfg {
  static constexpr int P_BYTES = T * 128, Q_BYTES = kTileQ * 128, STAGE = P_BYTES + Q_BYTES;
  static constexpr int STAGES = (T >= 128 ? 192 : 180) * 1024 / RINGS / STAGE;
  static constexpr int ACC_BYTES = T * kTileQ * 4;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int DATA = RING > ACC_BYTES ? RING : ACC_BYTES;
  static constexpr int SMEM = DATA + 1024;
  static constexpr int TMEM = T < 32 ? 32 : T;
};

template <typename Out, int ES, int T, bool SLOPE, int RINGS>
__global__ void __launch_bounds__(kTileThreads, RINGS)
    tile_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a) {
  using C = TileCfg<T, RINGS>;
  extern __shared__ char smraw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], done;
  __shared__ uint32_t tslot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = a.splits, rank = blockIdx.x;  // the cluster is the grid's x
  const int j0 = blockIdx.y * kTileQ, i0 = blockIdx.z * T;
  constexpr int BKE = 128 / ES;
  const int kb = rank * a.part, nk = max(0, min(a.part, (a.k + BKE - 1) / BKE - kb));
  const Epilogue& e = a.e;

  // block t of this CTA's k into ring slot s: Q's rows (which also announces the bytes of both), P's
  auto load_q = [&](int t, int s) {
    const uint32_t to = tc::smem_u32(sm + s * C::STAGE);
    const int k0 = (kb + t) * BKE;
    mbar_expect_tx(&full[s], C::STAGE);
    if (ES == 2 && a.q_row) {
#pragma unroll
      for (int c = 0; c < kTileQ / 64; ++c) tma_load_2d(to + 8192 * c, &maps.q, j0 + 64 * c, k0, &full[s]);
    } else {
      tma_load_2d(to, &maps.q, k0, j0, &full[s]);
    }
  };
  auto load_p = [&](int t, int s) {
    const uint32_t to = tc::smem_u32(sm + s * C::STAGE) + C::Q_BYTES;
    const int k0 = (kb + t) * BKE;
    if (ES == 2 && T >= 64 && a.p_row) {
#pragma unroll
      for (int c = 0; c < T / 64; ++c) tma_load_2d(to + 8192 * c, &maps.p, i0 + 64 * c, k0, &full[s]);
    } else {
      tma_load_2d(to, &maps.p, k0, i0, &full[s]);
    }
  };
  if (warp == 8 && lane == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    tc::mbar_init(&done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_async_smem();
    after_previous();
    for (int t = 0; t < nk && t < C::STAGES; ++t) {
      load_q(t, t);
      load_p(t, t);
    }
  } else if (warp == 9) {
    tc::tmem_alloc(&tslot, C::TMEM);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tslot;
  after_previous();

  // the tile's rows that this CTA finishes, two per warp at a time
  const int per = T / S, j = j0 + 4 * lane, left = a.n - j;
  float* acc = reinterpret_cast<float*>(sm);  // [T][128]; the ring is free when the sums are there
  float bias[4] = {}, cscale[4] = {1.f, 1.f, 1.f, 1.f};
  if (warp == 8 || warp == 10) {
    if (lane == 0) {
      bool ok = true;
      int s = 0;
      uint32_t phase = 0;  // of the wait for the slot's last use
      for (int t = C::STAGES; t < nk && ok; ++t) {
        ok = wait(&empty[s], phase);
        if (ok) {
          if (warp == 8) load_q(t, s);
          else load_p(t, s);
        }
        if (++s == C::STAGES) {
          s = 0;
          phase ^= 1;
        }
      }
      if (!ok) give_up();
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const uint32_t qstep = (a.q_row ? 2048 : 32) >> 4, pstep = (a.p_row ? 2048 : 32) >> 4;
      const uint64_t q0 = operand_desc(tc::smem_u32(sm), a.q_row), p0 = operand_desc(tc::smem_u32(sm) + C::Q_BYTES, a.p_row);
      bool ok = true;
      int s = 0;
      uint32_t phase = 0;
      for (int t = 0; t < nk; ++t) {
        ok = wait(&full[s], phase);
        if (!ok) break;
        tc::tc_fence_after();
        uint64_t dq = q0 + (uint64_t)(s * (C::STAGE >> 4)), dp = p0 + (uint64_t)(s * (C::STAGE >> 4));
#pragma unroll
        for (int c = 0; c < 4; ++c, dq += qstep, dp += pstep)
          mma<ES>(tmem, dq, dp, a.idesc, (t | c) ? 1u : 0u);
        tc::mma_commit(&empty[s]);
        if (++s == C::STAGES) {
          s = 0;
          phase ^= 1;
        }
      }
      if (ok && nk > 0) tc::mma_commit(&done);
      if (!ok) give_up();
    }
  } else {
    if (left > 0) {
      if (e.bias) widen4<Out>(fetch4(static_cast<const Out*>(e.bias) + j, a.vec, left), bias);
      if (ES == 1 && e.col_scale) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c < left) cscale[c] = e.col_scale[j + c];
      }
    }
    if (e.res) {  // 256 bytes a row: a lane for each half of the CTA's rows
      for (int x = 32 * warp + lane; x < 2 * per; x += 256) {
        const int i = i0 + rank * per + (x >> 1), c = j0 + 64 * (x & 1);
        if (i < a.m && c < a.n)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const Out*>(e.res) + (int64_t)i * e.ldr + c));
      }
    }
    bool ok = nk == 0 || wait(&done, 0);
    allow_next();
    if (!ok) give_up();  // loads in flight land where the sums' places are
    ok = __all_sync(0xffffffffu, ok);
    tc::tc_fence_after();
    // float32 sums to shared memory as acc[i][j]: a warp's 32 lanes are 32 adjacent j
    const int lq = warp & 3;
    constexpr int HALF = T < 32 ? T : T / 2;  // columns of a warp: its half, or all 16 of them
    if (T >= 32 || warp < 4) {
#pragma unroll
      for (int c = 0; c < HALF; c += 16) {
        const int col = (T >= 32 ? (warp >> 2) * HALF : 0) + c;
        float r[16];
        if (nk > 0 && ok) {
          tmem_ld16(tmem + ((uint32_t)(32 * lq) << 16) + col, r);
        } else {
#pragma unroll
          for (int x = 0; x < 16; ++x) r[x] = ok ? 0.f : __int_as_float(0x7FFFFFFF);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (i0 + col + x < a.m) acc[(col + x) * kTileQ + 32 * lq + lane] = r[x];
      }
    }
  }
  tc::tc_fence_before();
  __syncwarp();
  if (S > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 9) tc::tmem_dealloc(tmem, C::TMEM);
  if (warp < 8 && left > 0) {
#pragma unroll 1
    for (int x0 = warp; x0 < per; x0 += 16) {  // rows x0 and x0 + 8 of this CTA's
      uint2 res[2];
      F2 v[4], sl[4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int x = x0 + 8 * y, il = rank * per + x, i = i0 + il;
        const bool mine = x < per && i < a.m;
        res[y] = make_uint2(0, 0);
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
        float rs = 1.f;
        if (mine) {
          if (e.res) res[y] = fetch4(static_cast<const Out*>(e.res) + (int64_t)i * e.ldr + j, a.vec, left);
          if (ES == 1 && e.row_scale) rs = e.row_scale[i];
          const float* at = acc + il * kTileQ + 4 * lane;
          if (S > 1) {
#pragma unroll 1
            for (int s = 0; s < S; s += 2) {  // 2, 4 or 8 parts; two reads in flight, added in rank order
              const float4 p = ld_cluster(tc::smem_u32(at), s), q = ld_cluster(tc::smem_u32(at), s + 1);
              u.x = u.x + p.x + q.x; u.y = u.y + p.y + q.y; u.z = u.z + p.z + q.z; u.w = u.w + p.w + q.w;
            }
          } else {
            u = *reinterpret_cast<const float4*>(at);
          }
        }
        F2 lo = f2(u.x, u.y), hi = f2(u.z, u.w);
        if (ES == 1) {
          lo = mul(lo, mul(f2(rs), f2(cscale[0], cscale[1])));
          hi = mul(hi, mul(f2(rs), f2(cscale[2], cscale[3])));
        }
        v[2 * y] = add(lo, f2(bias[0], bias[1]));
        v[2 * y + 1] = add(hi, f2(bias[2], bias[3]));
      }
      activate_all<SLOPE>(e.act, v, sl);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int x = x0 + 8 * y, i = i0 + rank * per + x;
        if (x >= per || i >= a.m) continue;
        const uint2 packed = make_uint2(narrow2(add(v[2 * y], widen2(res[y].x, Out())), Out()),
                                        narrow2(add(v[2 * y + 1], widen2(res[y].y, Out())), Out()));
        put4(static_cast<Out*>(e.out) + (int64_t)i * e.ldo + j, packed, a.vec, left);
        if (SLOPE)
          put4(e.slope + (int64_t)i * a.n + j, make_uint2(pack_slopes(sl[2 * y]), pack_slopes(sl[2 * y + 1])), a.vec, left);
      }
    }
  }
  __syncwarp();
  if (S > 1) {  // the peers read this CTA's sums until here
    cluster_arrive();
    cluster_wait();
  }
}

// ---- a few tokens: a warp per R features, W read once, straight into registers ----
// Bound by W's bytes, and for small W by what a call costs at all: no tensor maps, no shared
// memory, no set-up.  A warp reads 512 bytes of each of its R rows of W at a time (32 lanes x 16
// bytes; single elements where rows start off 16 bytes), the same part of the M tokens from the L1
// cache, and adds the products in float32; SPLIT warps share a feature's k where there are too few
// features to fill the GPU.  One lane per (token, feature) finishes it.  Measured, bf16: 1 x 8192 x 8192
// 23.7 us (5.7 TB/s), 1 x 4096 x 4096 8.1 us, 1 x 512 x 512 2.0 us (tiles: 10.5, 4.4 for the last two).
template <typename T> struct Chunk;  // 16 bytes of an operand as float
template <> struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void widen(const uint4& a, float (&v)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <> struct Chunk<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void widen(const uint4& a, float (&v)[8]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <> struct Chunk<__nv_fp8_e4m3> {
  static constexpr int N = 16;
  static __device__ __forceinline__ void widen(const uint4& a, float (&v)[16]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> (16 * h)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        v[4 * i + 2 * h] = f.x;
        v[4 * i + 2 * h + 1] = f.y;
      }
  }
};
__device__ __forceinline__ float widen1(__nv_bfloat16 x) { return to_f32(x); }
__device__ __forceinline__ float widen1(__half x) { return to_f32(x); }
__device__ __forceinline__ float widen1(__nv_fp8_e4m3 x) { return float(x); }

struct TokenArgs {
  const void* x; int64_t ldx;
  const void* w; int64_t ldw;
  int m, n, k;
  Epilogue e;
};

template <typename Out, typename In, int M, int R, int SPLIT, bool VEC>
__global__ void __launch_bounds__(256) token_kernel(TokenArgs a) {
  after_previous();
  __shared__ float s_part[SPLIT == 1 ? 1 : 8][M * R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = SPLIT == 1 ? 0 : warp;
  const int j0 = (SPLIT == 1 ? blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x) * R;
  if (j0 >= a.n) return;  // SPLIT == 1 only: no barrier follows there
  const Epilogue& e = a.e;
  // this lane's output, if it has one: token i, feature j
  const int i = lane / R, j = j0 + lane % R;
  const bool mine = lane < M * R && i < a.m && j < a.n && part == 0;
  float bias = 0.f, res = 0.f, scale = 1.f;
  if (mine) {
    if (e.bias) bias = to_f32(static_cast<const Out*>(e.bias)[j]);
    if (e.res) res = to_f32(static_cast<const Out*>(e.res)[(int64_t)i * e.ldr + j]);
    if (e.row_scale) scale = e.row_scale[i];
    if (e.col_scale) scale *= e.col_scale[j];
  }
  const In* w[R];
  const In* x[M];
#pragma unroll
  for (int r = 0; r < R; ++r) w[r] = static_cast<const In*>(a.w) + (int64_t)min(j0 + r, a.n - 1) * a.ldw;
#pragma unroll
  for (int t = 0; t < M; ++t) x[t] = static_cast<const In*>(a.x) + (int64_t)min(t, a.m - 1) * a.ldx;
  float acc[M][R] = {};
  constexpr int N = VEC ? Chunk<In>::N : 1;
  constexpr int STEP = 32 * N * SPLIT;
  constexpr int U = VEC ? (R * M == 1 ? 8 : R * M >= 8 ? 2 : 4) : 8;  // steps in flight
  static_assert(STEP * U <= 32768, "k0 passes k by less than the margin below 2^31 that callers keep");
  for (int k0 = 32 * N * part + N * lane; k0 < a.k; k0 += STEP * U) {
    if constexpr (VEC) {
      uint4 wv[U][R];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int k = k0 + u * STEP;
          wv[u][r] = k < a.k ? __ldcs(reinterpret_cast<const uint4*>(w[r] + k)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * STEP;
        if (k >= a.k) break;
        float wf[R][N];
#pragma unroll
        for (int r = 0; r < R; ++r) Chunk<In>::widen(wv[u][r], wf[r]);
#pragma unroll
        for (int t = 0; t < M; ++t) {
          float xf[N];
          Chunk<In>::widen(*reinterpret_cast<const uint4*>(x[t] + k), xf);
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < N; ++c) acc[t][r] = fmaf(xf[c], wf[r][c], acc[t][r]);
        }
      }
    } else {
      float wf[U][R];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int k = k0 + u * STEP;
          wf[u][r] = k < a.k ? widen1(w[r][k]) : 0.f;
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * STEP;
        if (k >= a.k) break;
#pragma unroll
        for (int t = 0; t < M; ++t) {
          const float xf = widen1(x[t][k]);
#pragma unroll
          for (int r = 0; r < R; ++r) acc[t][r] = fmaf(xf, wf[u][r], acc[t][r]);
        }
      }
    }
  }
  allow_next();
  float sum = 0.f;  // of this lane's output
#pragma unroll
  for (int t = 0; t < M; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float v = acc[t][r];
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == t * R + r) sum = v;
    }
  if (SPLIT > 1) {
    if (lane < M * R) s_part[warp][lane] = sum;
    __syncthreads();
    if (!mine) return;
    sum = 0.f;
#pragma unroll
    for (int p = 0; p < SPLIT; ++p) sum += s_part[p][lane];
  }
  if (!mine) return;
  F2 v[1] = {f2(sum * scale + bias)}, slope[1];
  activate_all<false>(e.act, v, slope);
  float y, same;
  split(v[0], y, same);
  static_cast<Out*>(e.out)[(int64_t)i * e.ldo + j] = from_f32<Out>(y + res);
}

// ---- dz = dy act'(z), and the column sums of dz (the bias' gradient) ----
// Bound by memory: dy and the slope are read once, dz is written once; 8 columns a thread, 256 a
// block, a block takes every gridDim.y-th group of 8 rows.  The sums are of the float32 values,
// before dz is rounded to the operands' type for the two products.  8192 x 8192 bf16: 57 us for 402 MB.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    dz_kernel(const T* dy, int64_t lddy, const uint16_t* slope, T* dz, int64_t lddz, float* part,
              int64_t m, int64_t n) {
  after_previous();
  __shared__ float s[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j0 = (int64_t)blockIdx.x * 256;
  float sum[8] = {};
  for (int64_t i = (int64_t)blockIdx.y * 8 + warp; i < m; i += (int64_t)gridDim.y * 8) {
    const T* src = dy + i * lddy;
    const uint16_t* sl = slope ? slope + i * n : nullptr;
    T* dst = dz ? dz + i * lddz : nullptr;
    if (VEC) {
      const int64_t j = j0 + 8 * lane;
      if (j >= n) continue;
      const uint4 raw = *reinterpret_cast<const uint4*>(src + j);
      const T* e = reinterpret_cast<const T*>(&raw);
      float v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = to_f32(e[c]);
      if (sl) {
        const uint4 f = *reinterpret_cast<const uint4*>(sl + j);
        const uint16_t* g = reinterpret_cast<const uint16_t*>(&f);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] *= slope_value(g[c]);
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) sum[c] += v[c];
      if (dst) {
        uint4 o;
        T* w = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int c = 0; c < 8; ++c) w[c] = from_f32<T>(v[c]);
        *reinterpret_cast<uint4*>(dst + j) = o;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int64_t j = j0 + 32 * c + lane;
        if (j >= n) continue;
        float v = to_f32(src[j]);
        if (sl) v *= slope_value(sl[j]);
        sum[c] += v;
        if (dst) dst[j] = from_f32<T>(v);
      }
    }
  }
  allow_next();
  if (!part) return;
#pragma unroll
  for (int c = 0; c < 8; ++c) s[warp][VEC ? 8 * lane + c : 32 * c + lane] = sum[c];
  __syncthreads();
  const int64_t j = j0 + threadIdx.x;
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += s[w][threadIdx.x];
  if (j < n) part[blockIdx.y * n + j] = t;
}

// ---- rows of operands that TMA cannot address (a base or a stride off 16 bytes), copied into rows
// 16 bytes apart; bound by memory, 16 bytes written a thread; blockIdx.y is the operand ----
struct AlignJobs {
  struct { const void* src; int64_t ld, cols, rows; void* dst; int64_t ldd; } job[3];
};
template <typename T>
__global__ void __launch_bounds__(256) align_rows_kernel(AlignJobs jobs) {
  allow_next();
  after_previous();
  constexpr int V = 16 / sizeof(T);
  const auto& o = jobs.job[blockIdx.y];
  const T* src = static_cast<const T*>(o.src);
  const int64_t per = o.ldd / V, total = o.rows * per;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 256) {
    const int64_t r = x / per, c = x % per * V;
    T v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < o.cols ? src[r * o.ld + c + e] : T(0);
    *reinterpret_cast<uint4*>(static_cast<T*>(o.dst) + r * o.ldd + c) = *reinterpret_cast<const uint4*>(v);
  }
}

}  // namespace lin
}  // namespace qrb
