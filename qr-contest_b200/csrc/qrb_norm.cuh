// qrb200 -- root-mean-square norm of rows, with the residual's addition and an 8-bit output.
//
//   h = x + residual        rounded to the stream's type, because it is kept; y is the norm of
//                           what is kept, so a backward pass or a later layer that reads h sees
//                           the numbers y was made from
//   r = (mean_j h_j^2 + eps)^-1/2,   y_j = h_j r w_j
//   8 bits: s = max(max_j |y_j| / 448, 2^-126),  q_j = e4m3(y_j / s), computed as r max |h w| / 448 and
//           y_j (1 / s): one reduction less and no division an element, for a rounding of float32 that
//           an e4m3 code shows only beside the middle between two of them
// and, with g = dy w and c = r^3 / D sum_j g_j h_j,
//   dx = dresidual = dh + r g - c h,      dw_j = sum_rows dy_j h_j r.
// All sums, r, s and c are float32; every output is rounded once, when it is stored.
//
// All of it is bound by memory: about 10 operations an element against 3 to 8 bytes.  So a row is
// read once and stays in registers, as it is stored, between its reductions: VPT 8-element vectors a
// thread (16 bytes of a 16-bit type each), blockDim.x threads a row.  Rows of up to 1024 elements take
// a warp or a part of one (blockDim.y rows a block, shuffles only); longer ones a block each, up to
// 16384 elements; longer rows still are read again for each pass.  Rows that start off a 16-byte
// boundary (odd widths, odd strides) use the same kernels with single-element accesses, thread t
// taking elements t, t + blockDim.x, ... so that a warp's accesses stay adjacent.
// Measured on one B200 (copy 6.46 TB/s), 8192 x 8192 bf16 with residual: 84 us to bf16 (6.4 TB/s), 78 us
// to 8 bits (6.0 TB/s); 8191 x 8191 to 8 bits 125 us; backward of 16384 x 4096 bf16 93 us (5.8 TB/s).
#pragma once
#include <cuda_fp8.h>

#include "qrb_common.cuh"
#include "qrb_f2.cuh"
#include "qrb_pdl.cuh"

namespace qrb {
namespace norm {

constexpr int kMaxThreads = 1024;
// Threads a row: 64 registers each, so 1024 of them fill an SM's register file whatever the shape.
constexpr int max_threads(int vpt) { return vpt == 4 ? 512 : kMaxThreads; }
constexpr int kRegDim = 16384;                      // longest row that stays in registers
constexpr float kFp8Max = 448.f;                    // largest e4m3 value
constexpr float kTiny = 1.17549435e-38f;            // 2^-126

// ---- 8 elements of a row, as they are stored: 4 registers for 16-bit types ----
template <typename T>
struct Vec8 {
  static constexpr int Q = sizeof(T) / 2;  // 16-byte parts
  uint4 q[Q];
};
__device__ __forceinline__ void unpack(const Vec8<float>& a, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(a.q[i].x); v[4 * i + 1] = __uint_as_float(a.q[i].y);
    v[4 * i + 2] = __uint_as_float(a.q[i].z); v[4 * i + 3] = __uint_as_float(a.q[i].w);
  }
}
__device__ __forceinline__ void unpack(const Vec8<__nv_bfloat16>& a, float (&v)[8]) {
  const uint32_t w[4] = {a.q[0].x, a.q[0].y, a.q[0].z, a.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack(const Vec8<__half>& a, float (&v)[8]) {
  const uint32_t w[4] = {a.q[0].x, a.q[0].y, a.q[0].z, a.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void pack(Vec8<float>& a, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    a.q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                        __float_as_uint(v[4 * i + 3]));
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void pack(Vec8<T>& a, const float (&v)[8]) {
  a.q[0] = make_uint4(pack2(T(), v[0], v[1]), pack2(T(), v[2], v[3]), pack2(T(), v[4], v[5]), pack2(T(), v[6], v[7]));
}
// Rows are read once: they need not stay in the caches (STREAM); a weight is read for every row.
template <bool STREAM, typename T>
__device__ __forceinline__ void load8(const T* p, Vec8<T>& a) {
#pragma unroll
  for (int i = 0; i < Vec8<T>::Q; ++i) {
    const uint4* at = reinterpret_cast<const uint4*>(p) + i;
    a.q[i] = STREAM ? __ldcs(at) : *at;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  Vec8<T> a;
  pack(a, v);
#pragma unroll
  for (int i = 0; i < Vec8<T>::Q; ++i) reinterpret_cast<uint4*>(p)[i] = a.q[i];
}
__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ void store8(uint8_t* p, const float (&v)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
template <typename T> __device__ __forceinline__ void store1(T* p, float v) { *p = from_f32<T>(v); }
__device__ __forceinline__ void store1(uint8_t* p, float v) { *p = to_e4m3(v); }

// ---- a thread's share of a row: VPT groups of 8 elements ----
// NT == 0: rows of 16-byte vectors; group i is the 8 adjacent elements from 8 (i nt + t), nt =
// blockDim.x.  Otherwise single elements, blockDim.x == NT: element (8 i + j) NT + t (a constant
// distance, so that the accesses of a group need one address).
template <int VPT, int NT>
struct Share {
  static constexpr bool VEC = NT == 0;
  int dim, nt, t;
  __device__ Share(int dim_) : dim(dim_), nt(VEC ? blockDim.x : NT), t(threadIdx.x) {}
  __device__ __forceinline__ int column(int i, int j) const { return VEC ? 8 * (i * nt + t) + j : (8 * i + j) * NT + t; }
  // group i of a row, zero beyond its end
  template <bool STREAM, typename T>
  __device__ __forceinline__ void load(const T* row, int i, Vec8<T>& a) const {
    if (VEC) {
      const int c = 8 * (i * nt + t);
      if (c < dim) load8<STREAM>(row + c, a);
      else {
#pragma unroll
        for (int x = 0; x < Vec8<T>::Q; ++x) a.q[x] = make_uint4(0, 0, 0, 0);
      }
    } else {
      T e[8];
      const T* p = row + 8 * i * NT + t;
      if (8 * (i + 1) * NT <= dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = p[j * NT];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = column(i, j) < dim ? p[j * NT] : from_f32<T>(0.f);
      }
      memcpy(&a, e, sizeof(a));
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, int i, const float (&v)[8]) const {
    if (VEC) {
      const int c = 8 * (i * nt + t);
      if (c < dim) store8(row + c, v);
    } else {
      T* p = row + 8 * i * NT + t;
      if (8 * (i + 1) * NT <= dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) store1(p + j * NT, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (column(i, j) < dim) store1(p + j * NT, v[j]);
      }
    }
  }
};

// ---- reductions over the blockDim.x threads of a row ----
// Shuffles among the threads of a warp that share the row (a power of two up to 32); with more than
// one warp a row (blockDim.y == 1 then) one exchange through `slots` and one barrier.  Every thread
// gets the result; the order of the additions is fixed.
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* slots) {
  for (int o = min(blockDim.x, 32u) >> 1; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (blockDim.x <= 32) return make_float2(a, b);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slots[warp] = make_float2(a, b);
  __syncthreads();
  const float2 s = lane < (int)(blockDim.x >> 5) ? slots[lane] : make_float2(0.f, 0.f);
  a = s.x;
  b = s.y;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
}
__device__ __forceinline__ float row_sum(float v, float* slots) {
  for (int o = min(blockDim.x, 32u) >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x <= 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  v = lane < (int)(blockDim.x >> 5) ? slots[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Largest |v| as bit patterns: without the sign they order like the numbers, with NaN above
// infinity, so a NaN in the row is the result.
__device__ __forceinline__ float row_absmax(uint32_t bits, uint32_t* slots) {
  if (blockDim.x < 32) {
    for (int o = blockDim.x >> 1; o; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    return __uint_as_float(bits);
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (blockDim.x > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slots[warp] = bits;
    __syncthreads();
    bits = __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? slots[lane] : 0u);
  }
  return __uint_as_float(bits);
}
// Sum and largest |v| of a row with one exchange.
struct SumMax { float sum, absmax; };
__device__ __forceinline__ SumMax row_sum_max(float v, uint32_t bits, uint2* slots) {
  for (int o = min(blockDim.x, 32u) >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x < 32) {
    for (int o = blockDim.x >> 1; o; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  } else {
    bits = __reduce_max_sync(0xffffffffu, bits);
  }
  if (blockDim.x > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slots[warp] = make_uint2(__float_as_uint(v), bits);
    __syncthreads();
    const uint2 s = lane < (int)(blockDim.x >> 5) ? slots[lane] : make_uint2(0, 0);
    v = __uint_as_float(s.x);
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    bits = __reduce_max_sync(0xffffffffu, s.y);
  }
  return {v, __uint_as_float(bits)};
}
// The row's scale; a NaN stays (fmaxf would drop it).
__device__ __forceinline__ float scale_of(float absmax) {
  const float s = absmax / kFp8Max;
  return s < kTiny ? kTiny : s;
}

struct FwdArgs {
  const void* x; int64_t ldx;
  const void* res; int64_t ldr;  // residual, or null
  const void* w; int w_f32;      // weight (null: ones), in float32 or in x's type
  void* y; float* scale;         // y in x's type, or e4m3 with a scale a row
  void* h;                       // x + residual (null without a residual)
  int64_t rows;
  int dim;
  float eps;
};

// Group i of the weight as float32.  One in x's type waits in registers; a float32 one is read
// from the cache where it is used.
template <typename TX, int VPT, int NT>
struct Weight {
  Vec8<TX> kept[VPT];
  __device__ __forceinline__ void load(const Share<VPT, NT>& mine, const void* w, bool f32) {
    if (w && !f32) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) mine.template load<false>(static_cast<const TX*>(w), i, kept[i]);
    }
  }
  __device__ __forceinline__ void get(const Share<VPT, NT>& mine, const void* w, bool f32, int i, float (&v)[8]) const {
    if (!w) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 1.f;
    } else if (f32) {
      Vec8<float> a;
      mine.template load<false>(static_cast<const float*>(w), i, a);
      unpack(a, v);
    } else {
      unpack(kept[i], v);
    }
  }
};

// TH is the type that the norm reads: the stream's with a residual, else x's.
template <typename TX, typename TH, bool RES, bool Q8, bool NORM, int VPT, int NT>
__global__ void __launch_bounds__(max_threads(VPT), kMaxThreads / max_threads(VPT)) fwd_kernel(FwdArgs a) {
  after_previous();
  __shared__ float s_sum[32];
  __shared__ uint2 s_both[32];
  __shared__ uint32_t s_max[32];
  // rows past the end are computed again from the last row and not stored: no thread leaves early
  const int64_t at = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = at < a.rows;
  const int64_t row = live ? at : a.rows - 1;
  const Share<VPT, NT> mine(a.dim);
  Vec8<TH> h[VPT];
  Weight<TX, VPT, NT> w;
  if constexpr (RES) {
    Vec8<TX> x[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      mine.template load<true>(static_cast<const TX*>(a.x) + row * a.ldx, i, x[i]);
      mine.template load<true>(static_cast<const TH*>(a.res) + row * a.ldr, i, h[i]);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float u[8], v[8];
      unpack(x[i], u);
      unpack(h[i], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += u[j];
      pack(h[i], v);  // rounded as it is kept
      if (live) mine.store(static_cast<TH*>(a.h) + row * a.dim, i, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) mine.template load<true>(static_cast<const TH*>(a.x) + row * a.ldx, i, h[i]);
  }
  float r = 1.f;
  if (NORM) w.load(mine, a.w, a.w_f32);
  allow_next();
  float absmax = 0.f;
  if (NORM || Q8) {
    // max |y| = r max |h w|, so the scale takes no reduction of its own after r is known
    float ss = 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float v[8], u[8];
      unpack(h[i], v);
      if (Q8 && NORM) w.get(mine, a.w, a.w_f32, i, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (NORM) ss = fmaf(v[j], v[j], ss);
        if (Q8) top = max(top, __float_as_uint(NORM ? v[j] * u[j] : v[j]) & 0x7FFFFFFFu);
      }
    }
    if (Q8) {
      const SumMax s = row_sum_max(ss, top, s_both);
      ss = s.sum;
      absmax = s.absmax;
    } else {
      ss = row_sum(ss, s_sum);
    }
    if (NORM) {
      r = rsqrtf(ss / a.dim + a.eps);
      absmax *= r;
    }
  }
  auto value = [&](int i, float (&v)[8]) {
    unpack(h[i], v);
    if (NORM) {
      float u[8];
      w.get(mine, a.w, a.w_f32, i, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * r * u[j];
    }
  };
  if (Q8) {
    if (NORM && __any_sync(0xffffffffu, !(absmax <= 3.402823466e38f))) {
      // h w may have left float32's range where y does not: the same question of y itself (the whole
      // row agrees on it)
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float v[8];
        value(i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
      absmax = row_absmax(top, s_max);
    }
    const float s = scale_of(absmax);
    const float inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float v[8];
      value(i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv;
      if (live) mine.store(static_cast<uint8_t*>(a.y) + row * a.dim, i, v);
    }
    if (live && threadIdx.x == 0) a.scale[row] = s;
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float v[8];
      value(i, v);
      if (live) mine.store(static_cast<TX*>(a.y) + row * a.dim, i, v);
    }
  }
}

// Rows too long for registers: one 1024-thread block a row, each pass reads the row again (h from
// where this thread has just written it).
template <typename TX, typename TR, bool Q8, bool NORM>
__global__ void __launch_bounds__(kMaxThreads) fwd_long_kernel(FwdArgs a) {
  allow_next();
  after_previous();
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TR* res = a.res ? static_cast<const TR*>(a.res) + row * a.ldr : nullptr;
  TR* h = a.res ? static_cast<TR*>(a.h) + row * a.dim : nullptr;
  const float* wf = a.w && a.w_f32 ? static_cast<const float*>(a.w) : nullptr;
  const TX* wx = a.w && !a.w_f32 ? static_cast<const TX*>(a.w) : nullptr;
  float ss = 0.f;
  if (NORM) {
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      float v = to_f32(x[c]);
      if (res) {
        const TR kept = from_f32<TR>(v + to_f32(res[c]));
        h[c] = kept;
        v = to_f32(kept);
      }
      ss = fmaf(v, v, ss);
    }
    ss = row_sum(ss, s_sum);
  }
  const float r = NORM ? rsqrtf(ss / a.dim + a.eps) : 1.f;
  auto value = [&](int c) {
    float v = (NORM && res) ? to_f32(h[c]) : to_f32(x[c]);
    if (NORM) v = v * r * (wf ? wf[c] : wx ? to_f32(wx[c]) : 1.f);
    return v;
  };
  if (Q8) {
    uint32_t top = 0;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x)
      top = max(top, __float_as_uint(value(c)) & 0x7FFFFFFFu);
    const float s = scale_of(row_absmax(top, s_max));
    const float inv = 1.f / s;
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.dim;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) q[c] = to_e4m3(value(c) * inv);
    if (threadIdx.x == 0) a.scale[row] = s;
  } else {
    TX* y = static_cast<TX*>(a.y) + row * a.dim;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) y[c] = from_f32<TX>(value(c));
  }
}

struct BwdArgs {
  const void* dy; int64_t lddy;
  const void* h; int64_t ldh;
  const void* dh; int64_t lddh;  // gradient of the stream, or null
  const void* w; int w_f32;
  void* dx;                      // in x's type
  void* dres;                    // in the stream's type where that is another one, else null
  float* part;                   // [gridDim.x][dim] partial weight gradients, or null
  int64_t rows;
  int dim;
  float eps;
};

__device__ __forceinline__ void pairs(const float (&v)[8], F2 (&p)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = f2(v[2 * j], v[2 * j + 1]);
}

// 16 bytes from global to shared memory, past the registers.
__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A block (or, for short rows, part of a warp) walks over rows a grid apart and keeps its part of the
// weight's gradient in registers; the parts are added in a fixed order by colsum_kernel, so the result
// does not depend on timing.  Rows of vectors (NT == 0): a thread copies its share of the next row to
// shared memory while it works on this one (`depth` rows in turn; only the thread itself reads it, so
// that takes no barrier), and reads it there before and after the reduction instead of holding 24
// floats a group.  What lies past a row's end, past the last row, or in an absent dh is zero there, so
// the arithmetic asks nothing: with questions in it the kernel was bound by its instructions (39 an
// element; 16384 x 4096: 110 us, now 93 with the column sums' 7).  With 2 groups a thread instead of 4 the
// reductions weigh more: 155 us.
template <typename TX, typename TH, typename TW, int VPT, int NT>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT == 256 ? 256 : 512, NT == 32 ? 8 : NT == 256 ? 4 : 1)
    bwd_kernel(BwdArgs a, int depth) {
  after_previous();
  constexpr bool VEC = NT == 0;
  extern __shared__ __align__(16) char ring[];
  __shared__ float2 s_sum[2][32];
  const Share<VPT, NT> mine(a.dim);
  const int threads = blockDim.x * blockDim.y, flat = threadIdx.y * blockDim.x + threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  // 16-byte part x of this thread's slot of a row (h, dh, dy in this order); the parts of one x are
  // adjacent over the threads
  constexpr int QH = Vec8<TH>::Q, QX = Vec8<TX>::Q, PARTS = VPT * (2 * QH + QX);
  const int pitch = 16 * threads;
  char* const slots = ring + 16 * flat;
  auto zero_slot = [&](int stage) {
    for (int x = 0; x < PARTS; ++x) *reinterpret_cast<uint4*>(slots + (stage * PARTS + x) * pitch) = make_uint4(0, 0, 0, 0);
  };
  auto fetch = [&](int64_t row, int stage) {
    const TH* h = static_cast<const TH*>(a.h) + row * a.ldh + 8 * mine.t;
    const TX* dy = static_cast<const TX*>(a.dy) + row * a.lddy + 8 * mine.t;
    const TH* dh = static_cast<const TH*>(a.dh) + row * a.lddh + 8 * mine.t;
    const uint32_t to = smem_at(slots + stage * PARTS * pitch);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = 8 * i * mine.nt;
      if (c + 8 * mine.t >= a.dim) continue;
#pragma unroll
      for (int x = 0; x < QH; ++x) {
        copy16(to + (i * QH + x) * pitch, h + c + 16 / sizeof(TH) * x);
        if (a.dh) copy16(to + (VPT * QH + i * QH + x) * pitch, dh + c + 16 / sizeof(TH) * x);
      }
#pragma unroll
      for (int x = 0; x < QX; ++x) copy16(to + (2 * VPT * QH + i * QX + x) * pitch, dy + c + 16 / sizeof(TX) * x);
    }
  };
  Vec8<TW> w[VPT];
  F2 dw[VPT][4];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (a.w) mine.template load<false>(static_cast<const TW*>(a.w), i, w[i]);
    else pack(w[i], {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f});
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[i][j] = f2(0.f, 0.f);
  }
  // every thread of a warp takes the same number of turns (the shuffles need them all)
  const int64_t turns = (a.rows + step - 1) / step;
  if (VEC) {
    for (int p = 0; p < depth; ++p) zero_slot(p);
    if (depth == 2) {
      if (first < a.rows) fetch(first, 0);
      copy_commit();
    }
  }
  int stage = 0;
  for (int64_t turn = 0; turn < turns; ++turn) {
    const int64_t row = first + turn * step;
    const bool live = row < a.rows;
    Vec8<TH> hr[VEC ? 1 : VPT], dr[VEC ? 1 : VPT];
    Vec8<TX> gr[VEC ? 1 : VPT];
    const char* from = slots + stage * PARTS * pitch;
    if (VEC) {
      const int64_t next = row + (depth - 1) * step;
      const int to = depth == 2 ? stage ^ 1 : 0;
      if (next < a.rows) fetch(next, to);
      else zero_slot(to);
      copy_commit();
      if (depth == 2) copy_wait<1>();
      else copy_wait<0>();
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int x = VEC ? 0 : i;
        hr[x] = dr[x] = Vec8<TH>{};
        gr[x] = Vec8<TX>{};
        if (live) {
          mine.template load<true>(static_cast<const TH*>(a.h) + row * a.ldh, i, hr[x]);
          mine.template load<true>(static_cast<const TX*>(a.dy) + row * a.lddy, i, gr[x]);
          if (a.dh) mine.template load<true>(static_cast<const TH*>(a.dh) + row * a.lddh, i, dr[x]);
        }
      }
    }
    // group i of the row: h (0) or dh (1), and dy
    auto stream = [&](int i, int which, F2 (&p)[4]) {
      Vec8<TH> h;
      if (VEC) {
#pragma unroll
        for (int x = 0; x < QH; ++x) h.q[x] = *reinterpret_cast<const uint4*>(from + (which * VPT * QH + i * QH + x) * pitch);
      } else h = which ? dr[VEC ? 0 : i] : hr[VEC ? 0 : i];
      float v[8];
      unpack(h, v);
      pairs(v, p);
    };
    auto grad = [&](int i, F2 (&p)[4]) {
      Vec8<TX> g;
      if (VEC) {
#pragma unroll
        for (int x = 0; x < QX; ++x) g.q[x] = *reinterpret_cast<const uint4*>(from + (2 * VPT * QH + i * QX + x) * pitch);
      } else g = gr[VEC ? 0 : i];
      float v[8];
      unpack(g, v);
      pairs(v, p);
    };
    auto weight = [&](int i, F2 (&p)[4]) {
      float v[8];
      unpack(w[i], v);
      pairs(v, p);
    };
    F2 hh2 = f2(0.f, 0.f), gh2 = hh2;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      F2 h[4], g[4], u[4];
      stream(i, 0, h);
      grad(i, g);
      weight(i, u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hh2 = fma(h[j], h[j], hh2);
        gh2 = fma(mul(g[j], u[j]), h[j], gh2);
      }
    }
    float hh, gh, hh1, gh1;
    split(hh2, hh, hh1);
    split(gh2, gh, gh1);
    // two sets of slots in turn: a slow warp may still read the last row's
    const float2 s = row_sum2(hh + hh1, gh + gh1, s_sum[turn & 1]);
    const float r = rsqrtf(s.x / a.dim + a.eps);
    const float c = r * (r * (r * (s.y / a.dim)));  // r^3 alone leaves float32 from |h| = 1e13 on, and below 1e-12 with eps 0
    const F2 r2 = f2(r, r), c2 = f2(-c, -c);
    TX* const dx = live ? static_cast<TX*>(a.dx) + row * a.dim : nullptr;
    TH* const dres = live ? static_cast<TH*>(a.dres) + row * a.dim : nullptr;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      F2 h[4], g[4], u[4], e[4];
      float d[8];
      stream(i, 0, h);
      grad(i, g);
      stream(i, 1, e);
      weight(i, u);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const F2 gr2 = mul(g[j], r2);
        if (live) dw[i][j] = fma(gr2, h[j], dw[i][j]);
        split(fma(gr2, u[j], fma(c2, h[j], e[j])), d[2 * j], d[2 * j + 1]);
      }
      if (live && a.dx) mine.store(dx, i, d);
      if (live && a.dres) mine.store(dres, i, d);
    }
    if (VEC && depth == 2) stage ^= 1;
  }
  allow_next();
  if (!a.part) return;
  float sum[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) split(dw[i][j], sum[i][2 * j], sum[i][2 * j + 1]);
  if (blockDim.y == 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) mine.store(a.part + (int64_t)blockIdx.x * a.dim, i, sum[i]);
    return;
  }
  // several rows a block: their parts are added through shared memory (the ring, or its size)
  copy_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(ring);  // [blockDim.y][dim]
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = mine.column(i, j);
      if (c < a.dim) sums[threadIdx.y * a.dim + c] = sum[i][j];
    }
  __syncthreads();
  for (int c = flat; c < a.dim; c += threads) {
    float v = 0.f;
    for (int y = 0; y < (int)blockDim.y; ++y) v += sums[y * a.dim + c];
    a.part[(int64_t)blockIdx.x * a.dim + c] = v;
  }
}

// Rows too long for registers; the partial weight gradients are added up in memory.
template <typename TX, typename TR>
__global__ void __launch_bounds__(kMaxThreads) bwd_long_kernel(BwdArgs a) {
  allow_next();
  after_previous();
  __shared__ float2 s_sum[2][32];
  const float* wf = a.w && a.w_f32 ? static_cast<const float*>(a.w) : nullptr;
  const TX* wx = a.w && !a.w_f32 ? static_cast<const TX*>(a.w) : nullptr;
  auto weight = [&](int c) { return wf ? wf[c] : wx ? to_f32(wx[c]) : 1.f; };
  float* part = a.part ? a.part + (int64_t)blockIdx.x * a.dim : nullptr;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const TR* h = static_cast<const TR*>(a.h) + row * a.ldh;
    const TX* dy = static_cast<const TX*>(a.dy) + row * a.lddy;
    const TR* dh = a.dh ? static_cast<const TR*>(a.dh) + row * a.lddh : nullptr;
    float hh = 0.f, gh = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const float v = to_f32(h[c]);
      hh = fmaf(v, v, hh);
      gh = fmaf(to_f32(dy[c]) * weight(c), v, gh);
    }
    const float2 s = row_sum2(hh, gh, s_sum[turn]);
    const float r = rsqrtf(s.x / a.dim + a.eps);
    const float k = r * (r * (r * (s.y / a.dim)));
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const float v = to_f32(h[c]), g = to_f32(dy[c]);
      const float d = (dh ? to_f32(dh[c]) : 0.f) + fmaf(r, g * weight(c), -k * v);
      if (a.dx) static_cast<TX*>(a.dx)[row * a.dim + c] = from_f32<TX>(d);
      if (a.dres) static_cast<TR*>(a.dres)[row * a.dim + c] = from_f32<TR>(d);
      if (part) part[c] = row == blockIdx.x ? g * (v * r) : fmaf(g, v * r, part[c]);
    }
  }
}

// out[c] = sum over p < parts of part[p][c], in a fixed order: 32 columns a block, 32 rows of
// threads that each add every 32nd part, then a tree.
template <typename T>
__global__ void __launch_bounds__(1024) colsum_kernel(const float* part, int64_t parts, int64_t cols, T* out) {
  allow_next();
  after_previous();
  __shared__ float s[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t p = threadIdx.y; p < parts; p += 32) v += part[p * cols + c];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  float t = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int64_t oc = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && oc < cols) out[oc] = from_f32<T>(t);
}

}  // namespace norm
}  // namespace qrb
