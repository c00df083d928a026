// qrb200 -- root-mean-square norm of rows, with the residual's addition and an 8-bit output.
//
//   h = x + residual        rounded to the stream's type, because it is kept; y is the norm of
//                           what is kept, so a backward pass or a later layer that reads h sees
//                           the numbers y was made from
//   r = (mean_j h_j^2 + eps)^-1/2,   y_j = h_j r w_j
//   8 bits: s = max(max_j |y_j| / 448, 2^-126),  q_j = e4m3(y_j / s)
// and, with g = dy w and c = r^3 / D sum_j g_j h_j,
//   dx = dresidual = dh + r g - c h,      dw_j = sum_rows dy_j h_j r.
// All sums, r, s and c are float32; every output is rounded once, when it is stored.
//
// All of it is bound by memory: about 10 operations an element against 3 to 8 bytes.  So a row is
// read once and stays in registers between its reductions: VPT 8-element vectors a thread
// (16 bytes of a 16-bit type each), blockDim.x threads a row.  Rows of up to 1024 elements take a
// warp each (blockDim.y rows a block, shuffles only); longer ones a block each, up to 16384
// elements; longer rows still are read again for each pass.  Rows that start off a 16-byte
// boundary (odd widths, odd strides) use the same kernels with single-element accesses, thread t
// taking elements t, t + blockDim.x, ... so that a warp's accesses stay adjacent.
#pragma once
#include <cuda_fp8.h>

#include "qrb_common.cuh"

namespace qrb {
namespace norm {

constexpr int kMaxThreads = 1024;
// threads a row: one vector each leaves room for 1024 of them, more vectors for 512
constexpr int max_threads(int vpt) { return vpt == 1 ? kMaxThreads : 512; }
constexpr int kRegDim = 512 * 4 * 8;                // longest row that stays in registers
constexpr float kFp8Max = 448.f;                    // largest e4m3 value
constexpr float kTiny = 1.17549435e-38f;            // 2^-126

// ---- 8 elements of a row <-> float ----
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T2, typename T>
__device__ __forceinline__ void store8_16(T* p, const float (&v)[8], T2 (*pack)(float, float)) {
  T2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  store8_16<__nv_bfloat162>(p, v, [](float a, float b) { return __floats2bfloat162_rn(a, b); });
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  store8_16<__half2>(p, v, [](float a, float b) { return __floats2half2_rn(a, b); });
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
// VEC: group i is the 8 adjacent elements from 8 (i NT + t); otherwise element (8 i + j) NT + t.
template <int VPT, bool VEC>
struct Share {
  int dim, nt, t;
  __device__ Share(int dim_) : dim(dim_), nt(blockDim.x), t(threadIdx.x) {}
  template <typename T> __device__ __forceinline__ void load(const T* row, float (&v)[VPT][8]) const {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (VEC) {
        const int c = 8 * (i * nt + t);
        if (c < dim) load8(row + c, v[i]);
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (8 * i + j) * nt + t;
          v[i][j] = c < dim ? to_f32(row[c]) : 0.f;
        }
      }
    }
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[VPT][8]) const {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (VEC) {
        const int c = 8 * (i * nt + t);
        if (c < dim) store8(row + c, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (8 * i + j) * nt + t;
          if (c < dim) store1(row + c, v[i][j]);
        }
      }
    }
  }
};

// ---- reductions over the blockDim.x threads of a row ----
// Warp shuffles; with more than one warp a row (blockDim.y == 1 then) one exchange through
// `slots` and one barrier.  Every thread gets the result; the order of the additions is fixed.
__device__ __forceinline__ float row_sum(float v, float* slots) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (blockDim.x == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  v = lane < (int)(blockDim.x >> 5) ? slots[lane] : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* slots) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (blockDim.x == 32) return make_float2(a, b);
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
// Largest |v| as bit patterns: without the sign they order like the numbers, with NaN above
// infinity, so a NaN in the row is the result.
__device__ __forceinline__ float row_absmax(uint32_t bits, uint32_t* slots) {
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (blockDim.x > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slots[warp] = bits;
    __syncthreads();
    bits = __reduce_max_sync(0xffffffffu, lane < (int)(blockDim.x >> 5) ? slots[lane] : 0u);
  }
  return __uint_as_float(bits);
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

// v as it is kept in the stream's type.
template <typename TR> __device__ __forceinline__ float as_kept(float v) { return to_f32(from_f32<TR>(v)); }

template <typename TX, typename TR, bool Q8, bool NORM, int VPT, bool VEC>
__global__ void __launch_bounds__(max_threads(VPT)) fwd_kernel(FwdArgs a) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;  // with several rows a block no barrier follows
  const Share<VPT, VEC> mine(a.dim);
  float v[VPT][8];
  mine.load(static_cast<const TX*>(a.x) + row * a.ldx, v);
  if (NORM) {
    if (a.res) {
      float u[VPT][8];
      mine.load(static_cast<const TR*>(a.res) + row * a.ldr, u);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = as_kept<TR>(v[i][j] + u[i][j]);
      mine.store(static_cast<TR*>(a.h) + row * a.dim, v);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    float w[VPT][8];
    if (!a.w) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = 1.f;
    } else if (a.w_f32) mine.load(static_cast<const float*>(a.w), w);
    else mine.load(static_cast<const TX*>(a.w), w);
    const float r = rsqrtf(row_sum(ss, s_sum) / a.dim + a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * w[i][j];
  }
  if (Q8) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
    const float s = scale_of(row_absmax(top, s_max));
    const float inv = 1.f / s;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= inv;
    mine.store(static_cast<uint8_t*>(a.y) + row * a.dim, v);
    if (threadIdx.x == 0) a.scale[row] = s;
  } else {
    mine.store(static_cast<TX*>(a.y) + row * a.dim, v);
  }
}

// Rows too long for registers: one 1024-thread block a row, each pass reads the row again (h from
// where this thread has just written it).
template <typename TX, typename TR, bool Q8, bool NORM>
__global__ void __launch_bounds__(kMaxThreads) fwd_long_kernel(FwdArgs a) {
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
  float* part;                   // [gridDim.x * blockDim.y][dim] partial weight gradients, or null
  int64_t rows;
  int dim;
  float eps;
};

// One row at a time as in the forward kernel; a block (or, for short rows, a warp) walks over
// rows a grid apart and keeps its part of the weight's gradient in registers.  The parts are added
// in a fixed order by colsum_kernel, so the result does not depend on timing.
template <typename TX, typename TR, int VPT, bool VEC>
__global__ void __launch_bounds__(max_threads(VPT)) bwd_kernel(BwdArgs a) {
  __shared__ float2 s_sum[2][32];
  const Share<VPT, VEC> mine(a.dim);
  const int64_t first = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  float dw[VPT][8] = {};
  int turn = 0;
  for (int64_t row = first; row < a.rows; row += step, turn ^= 1) {
    float h[VPT][8], g[VPT][8], w[VPT][8];
    mine.load(static_cast<const TR*>(a.h) + row * a.ldh, h);
    mine.load(static_cast<const TX*>(a.dy) + row * a.lddy, g);
    if (!a.w) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) w[i][j] = 1.f;
    } else if (a.w_f32) mine.load(static_cast<const float*>(a.w), w);
    else mine.load(static_cast<const TX*>(a.w), w);
    float hh = 0.f, gh = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hh = fmaf(h[i][j], h[i][j], hh);
        gh = fmaf(g[i][j] * w[i][j], h[i][j], gh);
      }
    // two slot sets in turn: a slow warp may still read the last row's
    const float2 s = row_sum2(hh, gh, s_sum[turn]);
    const float r = rsqrtf(s.x / a.dim + a.eps);
    const float c = r * r * r * (s.y / a.dim);
    float d[VPT][8];
    if (a.dh) mine.load(static_cast<const TR*>(a.dh) + row * a.lddh, d);
    else {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) d[i][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] = fmaf(g[i][j], h[i][j] * r, dw[i][j]);
        d[i][j] += fmaf(r, g[i][j] * w[i][j], -c * h[i][j]);
      }
    if (a.dx) mine.store(static_cast<TX*>(a.dx) + row * a.dim, d);
    if (a.dres) mine.store(static_cast<TR*>(a.dres) + row * a.dim, d);
  }
  if (a.part) mine.store(a.part + first * a.dim, dw);
}

// Rows too long for registers; the partial weight gradients are added up in memory.
template <typename TX, typename TR>
__global__ void __launch_bounds__(kMaxThreads) bwd_long_kernel(BwdArgs a) {
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
    const float k = r * r * r * (s.y / a.dim);
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
  __shared__ float s[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < cols)
    for (int64_t p = threadIdx.y; p < parts; p += 32) v += part[p * cols + c];
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
