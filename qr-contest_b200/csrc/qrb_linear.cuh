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
#include "qrb_tc.cuh"
#include "qrb_tmap.cuh"

namespace qrb {
namespace lin {

enum Activation : int { ACT_NONE = 0, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU, ACT_COUNT };

// Raised by a kernel whose bounded wait ran out; its tile is then filled with NaN.
__device__ int g_timeout;

struct Epilogue {
  const float* row_scale;  // p (null: 1)
  const float* col_scale;  // q (null: 1)
  const void* bias;        // b, in the output's type, or null
  const void* res;         // R, in the output's type, or null
  int64_t ldr;
  void* out;
  int64_t ldo;
  int16_t* slope;          // act'(z), m x n contiguous, or null (see kSlopeOne)
  int act;
};

struct Args {
  int m, n, k;             // D is m x n
  int splits;              // CTAs of a cluster that share a tile's sum
  uint32_t idesc;          // element types and operand majors
  int es;                  // bytes of an operand element
  int p_row, q_row;        // operand is row-major (contiguous along its rows)
  int vec;                 // out / res / bias / slope rows allow 4-element accesses
  Epilogue e;
};

struct Maps {
  CUtensorMap p, q;
};

// act' is kept for the backward pass in 16 bits of fixed point: it lies in (-0.13, 1.13) for every
// activation here, so steps of 2^-14 hold 0 and 1 exactly and the rest to 3e-5, where a bf16 act'
// or z would be off by up to 2e-3 of its value.  -32768 stands for NaN.
constexpr float kSlopeOne = 16384.f;
__device__ __forceinline__ int16_t slope_to_fixed(float s) {
  return s != s ? (int16_t)-32768 : (int16_t)__float2int_rn(s * kSlopeOne);
}
__device__ __forceinline__ float slope_from_fixed(int16_t f) {
  return f == -32768 ? __int_as_float(0x7FFFFFFF) : (float)f * (1.f / kSlopeOne);
}

// act(z); with SLOPE also act'(z).
template <bool SLOPE>
__device__ __forceinline__ float activate(int act, float z, float& slope) {
  switch (act) {
    case ACT_RELU:
      if (SLOPE) slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
      return z < 0.f ? 0.f : z;  // NaN stays
    case ACT_GELU: {
      const float phi = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      if (SLOPE) slope = phi + z * 0.3989422804014327f * __expf(-0.5f * z * z);
      return z * phi;
    }
    case ACT_GELU_TANH: {  // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
      const float z2 = z * z;
      const float p = 1.f / (1.f + __expf(-1.5957691216057308f * z * (1.f + 0.044715f * z2)));
      if (SLOPE) slope = p + z * p * (1.f - p) * 1.5957691216057308f * (1.f + 0.134145f * z2);
      return z * p;
    }
    case ACT_SILU: {
      const float p = 1.f / (1.f + __expf(-z));
      if (SLOPE) slope = p * (1.f + z * (1.f - p));
      return z * p;
    }
    default:
      if (SLOPE) slope = 1.f;
      return z;
  }
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

// ---- epilogue of 4 adjacent outputs (i, j .. j+3) ----
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {  // 16-bit types, 8 bytes
  uint2 a = *reinterpret_cast<const uint2*>(p);
  const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  uint2 a;
  T* e = reinterpret_cast<T*>(&a);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<uint2*>(p) = a;
}

template <typename Out, bool SLOPE>
__device__ __forceinline__ void finish4(const Args& a, int i, int j, const float (&acc)[4]) {
  const Epilogue& e = a.e;
  const int left = a.n - j;
  const bool vec = a.vec && left >= 4;
  const float rs = e.row_scale ? e.row_scale[i] : 1.f;
  float b[4] = {}, r[4] = {}, v[4];
  int16_t sl[4];
  const Out* bias = static_cast<const Out*>(e.bias);
  const Out* res = static_cast<const Out*>(e.res) + (e.res ? (int64_t)i * e.ldr : 0);
  if (vec) {
    if (bias) load4(bias + j, b);
    if (e.res) load4(res + j, r);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < left) {
        if (bias) b[c] = to_f32(bias[j + c]);
        if (e.res) r[c] = to_f32(res[j + c]);
      }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float z = acc[c];
    if (e.col_scale) z *= rs * (c < left ? e.col_scale[j + c] : 0.f);
    else if (e.row_scale) z *= rs;
    z += b[c];
    float slope;
    v[c] = activate<SLOPE>(e.act, z, slope) + r[c];
    if (SLOPE) sl[c] = slope_to_fixed(slope);
  }
  Out* out = static_cast<Out*>(e.out) + (int64_t)i * e.ldo + j;
  int16_t* so = SLOPE ? e.slope + (int64_t)i * a.n + j : nullptr;
  if (vec) {
    store4(out, v);
    if (SLOPE) *reinterpret_cast<short4*>(so) = make_short4(sl[0], sl[1], sl[2], sl[3]);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < left) {
        out[c] = from_f32<Out>(v[c]);
        if (SLOPE) so[c] = sl[c];
      }
  }
}

// ---- one 128 (j) x T (i) tile per cluster of `splits` CTAs ----
// Q's rows are the MMA's 128 rows, P's the T columns, so few tokens cost a narrow MMA and not a
// padded one; the CTAs of a cluster take equal parts of k, leave their float32 sums in shared
// memory, and each finishes T / splits of the tile's rows with its peers' sums read over the
// cluster, added in rank order.
constexpr int kTileThreads = 256;
constexpr int kTileQ = 128;

template <int T>
struct TileCfg {
  static constexpr int P_BYTES = T * 128, Q_BYTES = kTileQ * 128, STAGE = P_BYTES + Q_BYTES;
  // 2 CTAs per SM up to T = 128; one with four 48 KB stages for T = 256
  static constexpr int STAGES = T == 256 ? 4 : (T == 128 ? 3 : (T == 64 ? 4 : 5));
  static constexpr int ACC_BYTES = T * kTileQ * 4;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int DATA = RING > ACC_BYTES ? RING : ACC_BYTES;
  static constexpr int SMEM = DATA + 1024;
  static constexpr int TMEM = T < 32 ? 32 : T;
};

template <typename Out, int ES, int T, bool SLOPE>
__global__ void __launch_bounds__(kTileThreads)
    tile_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a) {
  using C = TileCfg<T>;
  extern __shared__ char smraw[];
  char* sm = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smraw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::STAGES], empty[C::STAGES], done;
  __shared__ uint32_t tslot;
  __shared__ int s_issued, s_committed, s_drained;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = a.splits, rank = blockIdx.x % S;
  const int tile = blockIdx.x / S, tiles_j = (a.n + kTileQ - 1) / kTileQ;
  const int j0 = tile % tiles_j * kTileQ, i0 = tile / tiles_j * T;
  constexpr int BKE = 128 / ES;
  const int nkb = (a.k + BKE - 1) / BKE;
  const int kb = (int)((int64_t)nkb * rank / S), nk = (int)((int64_t)nkb * (rank + 1) / S) - kb;

  if (warp == 0) {
    tc::tmem_alloc(&tslot, C::TMEM);
    tc::tmem_relinquish();
  }
  if (tid == 0) {
    s_issued = s_committed = 0;
    s_drained = 1;
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    tc::mbar_init(&done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tslot;
  bool ok = true;

  if (warp == 0 && lane == 0) {
    for (int t = 0; t < nk; ++t) {
      const int s = t % C::STAGES, k0 = (kb + t) * BKE;
      if (t >= C::STAGES && !tc::mbar_wait(&empty[s], ((t / C::STAGES) - 1) & 1)) { ok = false; break; }
      const uint32_t pq = tc::smem_u32(sm + s * C::STAGE), pp = pq + C::Q_BYTES;
      mbar_expect_tx(&full[s], C::STAGE);
      if (ES == 2 && a.q_row) {
#pragma unroll
        for (int c = 0; c < kTileQ / 64; ++c) tma_load_2d(pq + 8192 * c, &maps.q, j0 + 64 * c, k0, &full[s]);
      } else {
        tma_load_2d(pq, &maps.q, k0, j0, &full[s]);
      }
      if (ES == 2 && T >= 64 && a.p_row) {
#pragma unroll
        for (int c = 0; c < T / 64; ++c) tma_load_2d(pp + 8192 * c, &maps.p, i0 + 64 * c, k0, &full[s]);
      } else {
        tma_load_2d(pp, &maps.p, k0, i0, &full[s]);
      }
      s_issued = t + 1;
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t qstep = (a.q_row ? 2048 : 32) >> 4, pstep = (a.p_row ? 2048 : 32) >> 4;
    for (int t = 0; t < nk; ++t) {
      const int s = t % C::STAGES;
      if (!tc::mbar_wait(&full[s], (t / C::STAGES) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      const uint32_t pq = tc::smem_u32(sm + s * C::STAGE), pp = pq + C::Q_BYTES;
      uint64_t dq = operand_desc(pq, a.q_row), dp = operand_desc(pp, a.p_row);
#pragma unroll
      for (int c = 0; c < 4; ++c, dq += qstep, dp += pstep)
        mma<ES>(tmem, dq, dp, a.idesc, (t | c) ? 1u : 0u);
      tc::mma_commit(&empty[s]);
      s_committed = t + 1;
    }
    if (nk > 0 && ok) {
      tc::mma_commit(&done);
      if (!tc::mbar_wait(&done, 0)) ok = false;
    }
  }
  const bool failed = __syncthreads_or(!ok);
  if (failed && tid == 0) {
    // what is in flight ends (each wait again bounded) before the buffers and the TMEM are reused:
    // commit t completes phase t / STAGES of empty[t % STAGES], load t that of full[t % STAGES]
    const int nc = s_committed, ni = s_issued;
    if (nc > 0 && !tc::mbar_wait(&empty[(nc - 1) % C::STAGES], ((nc - 1) / C::STAGES) & 1)) s_drained = 0;
    for (int u = ni > C::STAGES ? ni - C::STAGES : 0; u < ni; ++u)
      if (!tc::mbar_wait(&full[u % C::STAGES], (u / C::STAGES) & 1)) s_drained = 0;
    atomicExch(&g_timeout, 1);
  }
  if (failed) __syncthreads();
  tc::tc_fence_after();

  // float32 sums to shared memory as acc[i][j]: a warp's 32 lanes are 32 adjacent j
  float* acc = reinterpret_cast<float*>(sm);
  {
    const int lq = warp & 3;
    constexpr int HALF = T < 64 ? T : T / 2;  // columns of a warp: all of them, or its half
    if (T >= 64 || warp < 4) {
#pragma unroll
      for (int c = 0; c < HALF; c += 16) {
        const int col = (T >= 64 ? (warp >> 2) * HALF : 0) + c;
        uint32_t r[16];
        if (nk > 0 && !failed) {
          asm volatile(
              "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
              "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
              : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
              : "r"(tmem + ((uint32_t)(32 * lq) << 16) + col));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        } else {
#pragma unroll
          for (int x = 0; x < 16; ++x) r[x] = 0;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
          acc[(col + x) * kTileQ + 32 * lq + lane] =
              failed ? __int_as_float(0x7FFFFFFF) : __uint_as_float(r[x]);
      }
    }
  }
  tc::tc_fence_before();
  if (S > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 0 && s_drained) tc::tmem_dealloc(tmem, C::TMEM);
  const int per = T / S;
  for (int x = warp; x < per; x += kTileThreads / 32) {
    const int il = rank * per + x, i = i0 + il, j = j0 + 4 * lane;
    if (i >= a.m) break;
    const uint32_t at = tc::smem_u32(acc + il * kTileQ + 4 * lane);
    float v[4] = {};
    for (int s = 0; s < S; ++s) {
      const float4 u = S > 1 ? ld_cluster(at, s) : *reinterpret_cast<const float4*>(acc + il * kTileQ + 4 * lane);
      v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
    }
    if (j < a.n) finish4<Out, SLOPE>(a, i, j, v);
  }
  __syncwarp();
  if (S > 1) {  // the peers read this CTA's sums until here
    cluster_arrive();
    cluster_wait();
  }
}

// ---- dz = dy act'(z), and the column sums of dz (the bias' gradient) ----
// Bound by memory: dy and the slope are read once, dz is written once; 8 columns a thread, 256 a
// block, a block takes every gridDim.y-th group of 8 rows.  The sums are of the float32 values,
// before dz is rounded to the operands' type for the two products.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    dz_kernel(const T* dy, int64_t lddy, const int16_t* slope, T* dz, int64_t lddz, float* part,
              int64_t m, int64_t n) {
  __shared__ float s[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j0 = (int64_t)blockIdx.x * 256;
  float sum[8] = {};
  for (int64_t i = (int64_t)blockIdx.y * 8 + warp; i < m; i += (int64_t)gridDim.y * 8) {
    const T* src = dy + i * lddy;
    const int16_t* sl = slope ? slope + i * n : nullptr;
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
        const int16_t* g = reinterpret_cast<const int16_t*>(&f);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] *= slope_from_fixed(g[c]);
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
        if (sl) v *= slope_from_fixed(sl[j]);
        sum[c] += v;
        if (dst) dst[j] = from_f32<T>(v);
      }
    }
  }
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

// ---- rows of an operand that TMA cannot address (a base or a stride off 16 bytes), copied into
// rows 16 bytes apart; bound by memory, 16 bytes written a thread ----
template <typename T>
__global__ void __launch_bounds__(256) align_rows_kernel(const T* src, int64_t ld, int64_t cols, T* dst, int64_t ldd, int64_t rows) {
  constexpr int V = 16 / sizeof(T);
  const int64_t per = ldd / V, total = rows * per;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < total; x += (int64_t)gridDim.x * 256) {
    const int64_t r = x / per, c = x % per * V;
    T v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < cols ? src[r * ld + c + e] : T(0);
    *reinterpret_cast<uint4*>(dst + r * ldd + c) = *reinterpret_cast<const uint4*>(v);
  }
}

}  // namespace lin
}  // namespace qrb
