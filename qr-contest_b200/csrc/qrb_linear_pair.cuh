// qrb200 -- the matrix product of qrb_linear.cuh for many tokens: a persistent kernel whose CTA pairs
// share 256 x TN output tiles (tcgen05 cta_group::2).
//
// Each CTA of a pair (a cluster of 2 on neighbouring SMs) loads 128 of the tile's 256 rows of P and
// TN / 2 of its TN rows of Q; one thread of the first CTA issues the MMAs for both, which read both
// CTAs' shared memory, so a byte of Q is fetched once per 256 rows instead of once per 128 and shared
// memory holds twice the k.  Each CTA's tensor memory holds its 128 rows x TN float32 sums twice:
// while 8 warps finish one tile (bias, activation, residual, rounding), the MMAs of the next run.
// Roles: warps 0-7 epilogue, warp 8 loads P, warp 10 loads Q, warp 9 (first CTA) MMAs.  Hand-offs are mbarriers:
//   full[s]       loads of both CTAs -> MMA        (in the first CTA; bytes of both)
//   empty[s]      MMA -> loads of both CTAs        (commit to both)
//   acc_full[a]   MMA -> epilogues of both CTAs    (commit to both)
//   acc_empty[a]  epilogues of both CTAs -> MMA    (in the first CTA; 16 warps)
// Results leave through shared memory: a warp writes 32 rows x 64 columns in the 128-byte swizzle
// and one TMA store puts them out (rows that TMA cannot address are copied from there by the warp,
// a row at a time); a residual comes in the same way before the sums are needed.  No multicast loads.
// Bound by power in long runs (4096 x 16384 x 4096 bf16: 356 us in short runs, 400 to 413 sustained, 1.3 to
// 1.4 PFLOP/s; with bias and gelu 430) and by the operands' way into shared memory in 8 bits
// (8192 x 8192 x 4096: 196 us, 2.8 PFLOP/s).  The tensor pipe is 80 % active.
//
// Every wait is bounded.  A role whose wait runs out raises g_timeout and stops; the epilogue then
// writes NaN for the tiles it still owes, and the loads in flight get time to land before the exit.
#pragma once
#include "qrb_linear.cuh"

namespace qrb {
namespace lin {

constexpr int kPairThreads = 352;
constexpr int kPairM = 256;  // tile rows of a pair

struct PairMaps {
  CUtensorMap p, q, out, res, slope;
};
struct PairArgs {
  int m, n, k;
  uint32_t idesc;
  int p_row, q_row;
  int tiles_i, tiles_j, group;  // tile order: `group` tiles along i, then along j
  int tma_out, tma_res, tma_slope;
  Epilogue e;
};

template <int TN>
struct PairCfg {
  static constexpr int P_BYTES = 128 * 128, Q_BYTES = TN / 2 * 128, STAGE = P_BYTES + Q_BYTES;
  static constexpr int STAGES = TN == 256 ? 5 : 6;
  static constexpr int STAGING = 8 * 2 * 4096;
  static constexpr int COLS = 8 * 2 * 32 * 4;  // a warp's bias and column scales, 32 columns at a time
  // All shared memory is dynamic, so its base is 1024-byte aligned.
  static constexpr int SMEM = STAGES * STAGE + STAGING + COLS + 256;
  static constexpr int TMEM = 2 * TN;
  static_assert(SMEM <= 227 * 1024, "pair kernel shared memory");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
// A load into this CTA's shared memory that reports to a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
template <int ES>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (ES == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Completion of the MMAs so far, reported to this barrier in both CTAs.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          tc::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Address of 16-byte chunk q of row r in a staged block of 32 rows x 128 bytes.
__device__ __forceinline__ char* staged(char* buf, int r, int q) { return buf + 128 * r + 16 * (q ^ (r & 7)); }

// Element-wise copies between a staged block and rows that TMA cannot address; T is 2 bytes wide.
template <typename T>
__device__ __forceinline__ void copy_out(char* buf, T* dst, int64_t ld, int i0, int j0, int m, int n, int lane) {
  for (int r = 0; r < 32 && i0 + r < m; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 32 * h + lane;
      if (j0 + c < n)
        dst[(int64_t)(i0 + r) * ld + j0 + c] = *reinterpret_cast<const T*>(staged(buf, r, c >> 3) + 2 * (c & 7));
    }
}
template <typename T>
__device__ __forceinline__ void copy_in(char* buf, const T* src, int64_t ld, int i0, int j0, int m, int n, int lane) {
#pragma unroll 4
  for (int r = 0; r < 32; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 32 * h + lane;
      T v = from_f32<T>(0.f);
      if (i0 + r < m && j0 + c < n) v = src[(int64_t)(i0 + r) * ld + j0 + c];
      *reinterpret_cast<T*>(staged(buf, r, c >> 3) + 2 * (c & 7)) = v;
    }
}

template <typename Out, int ES, int TN, bool SLOPE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairArgs a) {
  using C = PairCfg<TN>;
  extern __shared__ __align__(1024) char sm[];
  char* staging = sm + C::STAGES * C::STAGE;
  float(*s_col)[2][32] = reinterpret_cast<float(*)[2][32]>(staging + C::STAGING);
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING + C::COLS);
  uint64_t *empty = full + C::STAGES, *acc_full = empty + C::STAGES, *acc_empty = acc_full + 2, *res_bar = acc_empty + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(res_bar + 8);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  constexpr int BKE = 128 / ES;
  const int nk = (a.k + BKE - 1) / BKE;
  const int tiles = a.tiles_i * a.tiles_j;

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tslot)), "r"(C::TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      tc::mbar_init(&full[s], 1);
      tc::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&acc_full[b], 1);
      tc::mbar_init(&acc_empty[b], 16);
    }
    for (int w = 0; w < 8; ++w) tc::mbar_init(&res_bar[w], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  tc::tc_fence_after();
  const uint32_t tmem = *tslot;
  after_previous();

  // tile t of the order: groups of `group` tiles along i, all j of a group before the next one, so
  // that the pairs at work at one time share their rows of P and of Q in the L2 cache
  auto place = [&](int t, int& ti, int& tj) {
    const int per = a.group * a.tiles_j, g = t / per, first = g * a.group;
    const int height = min(a.group, a.tiles_i - first), in = t - g * per;
    ti = first + in % height;
    tj = in / height;
  };

  bool ok = true;
  if (warp == 8 || warp == 10) {  // P's rows, Q's rows: a thread each, which has little time a block
    if (lane == 0) {
      const bool is_p = warp == 8, by_rows = ES == 2 && (is_p ? a.p_row : a.q_row);
      const CUtensorMap* map = is_p ? &maps.p : &maps.q;
      const uint32_t base = tc::smem_u32(sm) + (is_p ? 0 : C::P_BYTES), full0 = in_rank(tc::smem_u32(full), 0);
      const int chunks = is_p ? 2 : TN / 128;
      int s = 0, first = 1;
      uint32_t phase = 0;  // of the wait for a slot's last use
      for (int t = pair; t < tiles && ok; t += pairs) {
        int ti, tj;
        place(t, ti, tj);
        const int r0 = is_p ? ti * kPairM + 128 * (int)rank : tj * TN + TN / 2 * (int)rank;
        for (int kb = 0, k0 = 0; kb < nk; ++kb, k0 += BKE) {
          if (!first && !lin::wait(&empty[s], phase)) { ok = false; break; }
          if (is_p && rank == 0) mbar_expect_tx(&full[s], 2 * C::STAGE);
          const uint32_t to = base + s * C::STAGE, bar = full0 + 8 * s;
          if (by_rows) {
            for (int c = 0; c < chunks; ++c) tma_load_2d_pair(to + 8192 * c, map, r0 + 64 * c, k0, bar);
          } else {
            tma_load_2d_pair(to, map, k0, r0, bar);
          }
          if (++s == C::STAGES) {
            s = 0;
            if (first) first = 0;
            else phase ^= 1;
          }
        }
      }
      if (!ok) give_up();
    }
    __syncwarp();
  } else if (warp == 9) {
    if (lane == 0 && rank == 0) {
      const uint32_t pstep = (a.p_row ? 2048 : 32) >> 4, qstep = (a.q_row ? 2048 : 32) >> 4;
      const uint64_t p0 = operand_desc(tc::smem_u32(sm), a.p_row), q0 = operand_desc(tc::smem_u32(sm) + C::P_BYTES, a.q_row);
      int s = 0, turn = 0;
      uint32_t phase = 0;
      for (int t = pair; t < tiles && ok; t += pairs, ++turn) {
        const int b = turn & 1;
        if (turn >= 2 && !lin::wait(&acc_empty[b], ((turn >> 1) - 1) & 1)) { ok = false; break; }
        tc::tc_fence_after();
        for (int kb = 0; kb < nk; ++kb) {
          if (!lin::wait(&full[s], phase)) { ok = false; break; }
          tc::tc_fence_after();
          uint64_t dp = p0 + (uint64_t)(s * (C::STAGE >> 4)), dq = q0 + (uint64_t)(s * (C::STAGE >> 4));
#pragma unroll
          for (int c = 0; c < 4; ++c, dp += pstep, dq += qstep)
            mma_pair<ES>(tmem + b * TN, dp, dq, a.idesc, (kb | c) ? 1u : 0u);
          commit_pair(&empty[s]);
          if (++s == C::STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) commit_pair(&acc_full[b]);
      }
      if (!ok) give_up();
    }
    __syncwarp();
  } else {
    const int lq = warp & 3, half = warp >> 2;
    const uint32_t lane_base = (uint32_t)(32 * lq) << 16;
    char* const bufs = staging + warp * 8192;
    const Epilogue& e = a.e;
    const uint32_t done_bar0 = in_rank(tc::smem_u32(&acc_empty[0]), 0), done_bar1 = in_rank(tc::smem_u32(&acc_empty[1]), 0);
    int turn = 0, chunk = 0, res_phase = 0;
    for (int t = pair; t < tiles; t += pairs, ++turn) {
      int ti, tj;
      place(t, ti, tj);
      const int b = turn & 1;
      const int i0 = ti * kPairM + 128 * rank + 32 * lq, i = i0 + lane;
      const float rs = e.row_scale && i < a.m ? e.row_scale[i] : 1.f;
      bool waited = false;
#pragma unroll 1
      for (int c0 = half * (TN / 2); c0 < (half + 1) * (TN / 2); c0 += 64, ++chunk) {
        const int j0 = tj * TN + c0;
        const bool live = i0 < a.m && j0 < a.n;
        // with a slope: block 0 holds the results, block 1 the slopes; otherwise in turn
        char* const buf = bufs + (SLOPE ? 0 : 4096 * (chunk & 1));
        if (lane == 0) {
          if (SLOPE) store_wait_read<0>();
          else store_wait_read<1>();
        }
        tc::fence_async_smem();  // this warp's own accesses to the block, before a load overwrites it
        __syncwarp();
        const bool fetch = e.res && live && ok;
        if (fetch) {
          if (a.tma_res) {
            if (lane == 0) {
              mbar_expect_tx(&res_bar[warp], 4096);
              tma_load_2d(tc::smem_u32(buf), &maps.res, j0, i0, &res_bar[warp]);
            }
          } else {
            copy_in(buf, static_cast<const Out*>(e.res), e.ldr, i0, j0, a.m, a.n, lane);
          }
        }
        float bias[2], cscale[2];  // of columns lane and 32 + lane
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = j0 + 32 * h + lane;
          bias[h] = e.bias && j < a.n ? to_f32(static_cast<const Out*>(e.bias)[j]) : 0.f;
          cscale[h] = ES == 1 && e.col_scale && j < a.n ? e.col_scale[j] : 1.f;
        }
        if (!waited) {
          if (ok && !lin::wait(&acc_full[b], (turn >> 1) & 1)) ok = false;
          tc::tc_fence_after();
          waited = true;
          if (t + pairs >= tiles) allow_next();  // this CTA's last sums
        }
        if (fetch && a.tma_res) {  // also where the sums have not come: it lands in the block
          if (!lin::wait(&res_bar[warp], res_phase)) {
            ok = false;
            give_up();
          }
          res_phase ^= 1;
        }
        ok = __all_sync(0xffffffffu, ok);
        // 16 columns at a time, in a loop: instructions that are fetched to run once cost more than
        // the loop does
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          float raw[16];
          if (ok) {
            tmem_ld16(tmem + b * TN + lane_base + c0 + 16 * h, raw);
          } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) raw[x] = __int_as_float(0x7FFFFFFF);
          }
          if (h == 3 && c0 + 64 == (half + 1) * (TN / 2)) {  // the sums are in registers
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(b ? done_bar1 : done_bar0);
          }
          if (!live) continue;
          if (!(h & 1)) {
            __syncwarp();
            s_col[warp][0][lane] = h ? bias[1] : bias[0];
            if (ES == 1) s_col[warp][1][lane] = h ? cscale[1] : cscale[0];
            __syncwarp();
          }
          const int hc = 16 * (h & 1);
          F2 v[8], sl[8];
#pragma unroll
          for (int x = 0; x < 8; x += 2) {
            const float4 bb = *reinterpret_cast<const float4*>(&s_col[warp][0][hc + 2 * x]);
            F2 lo = f2(raw[2 * x], raw[2 * x + 1]), hi = f2(raw[2 * x + 2], raw[2 * x + 3]);
            if (ES == 1) {
              const float4 cs = *reinterpret_cast<const float4*>(&s_col[warp][1][hc + 2 * x]);
              lo = mul(lo, mul(f2(rs), f2(cs.x, cs.y)));
              hi = mul(hi, mul(f2(rs), f2(cs.z, cs.w)));
            }
            v[x] = add(lo, f2(bb.x, bb.y));
            v[x + 1] = add(hi, f2(bb.z, bb.w));
          }
          activate_all<SLOPE>(e.act, v, sl);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint4* at = reinterpret_cast<uint4*>(staged(buf, lane, 2 * h + q));
            F2* w = v + 4 * q;
            if (e.res) {
              const uint4 r = *at;
              w[0] = add(w[0], widen2(r.x, Out())); w[1] = add(w[1], widen2(r.y, Out()));
              w[2] = add(w[2], widen2(r.z, Out())); w[3] = add(w[3], widen2(r.w, Out()));
            }
            *at = make_uint4(narrow2(w[0], Out()), narrow2(w[1], Out()), narrow2(w[2], Out()), narrow2(w[3], Out()));
            if (SLOPE)
              *reinterpret_cast<uint4*>(staged(bufs + 4096, lane, 2 * h + q)) =
                  make_uint4(pack_slopes(sl[4 * q]), pack_slopes(sl[4 * q + 1]), pack_slopes(sl[4 * q + 2]), pack_slopes(sl[4 * q + 3]));
          }
        }
        if (live) {
          tc::fence_async_smem();
          __syncwarp();
          if (!a.tma_out) copy_out(buf, static_cast<Out*>(e.out), e.ldo, i0, j0, a.m, a.n, lane);
          if (SLOPE && !a.tma_slope) copy_out(bufs + 4096, e.slope, a.n, i0, j0, a.m, a.n, lane);
          if (lane == 0) {
            if (a.tma_out) tma_store_2d(&maps.out, tc::smem_u32(buf), j0, i0);
            if (SLOPE && a.tma_slope) tma_store_2d(&maps.slope, tc::smem_u32(bufs + 4096), j0, i0);
          }
        }
        if (lane == 0) store_commit();
      }
    }
    if (lane == 0) store_wait_read<0>();
    if (!ok && lane == 0) atomicExch(&g_timeout, 1);
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  cluster_arrive();  // the pair's MMAs and signals have ended
  cluster_wait();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM));
}

}  // namespace lin
}  // namespace qrb
