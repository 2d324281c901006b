// bf16 rows to rows in 8 bits (hs_fp8_rows.h): hs_quantize_rows_fp8, and hs_rmsnorm_fp8 with
// the RMSNorm, and the residual's addition, before it. Both read each value once and are
// bound by memory; a group of 128 values is 16 lanes of 8.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_fp8_rows.h"

namespace hs {
namespace {

__device__ __forceinline__ void floats8(uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

constexpr int kQuantThreads = 256;

// 8 values a thread: 4096 rows of 4096 11.0 us (4.6 TB/s)
__global__ __launch_bounds__(kQuantThreads) void k_quantize_rows(
    const uint16_t* __restrict__ x, int64_t xs, int rows, int width, int groups,
    uint8_t* __restrict__ codes, int64_t cs, uint8_t* __restrict__ scales, int64_t ss) {
  const int64_t e = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  const int64_t at = e >> 4;  // the group
  if (at >= (int64_t)rows * groups) return;  // whole groups of lanes
  const int64_t row = at / groups;
  const int group = (int)(at % groups), k = group * kFp8Group + 8 * (int)(e & 15);
  uint4 u = make_uint4(0, 0, 0, 0);
  if (k < width) u = *reinterpret_cast<const uint4*>(x + row * xs + k);
  float v[8];
  floats8(u, v);
  uint2 c;
  const uint32_t byte = group_codes8(v, c);
  if (k < width) *reinterpret_cast<uint2*>(codes + row * cs + k) = c;
  if ((e & 15) == 0) scales[row * ss + group] = (uint8_t)byte;
}

struct NormArgs {
  const uint16_t* x;
  int64_t xs;
  uint16_t* res;
  int64_t rs;
  const uint16_t* w;
  float eps;
  int rows, hidden;
  uint8_t* codes;
  int64_t cs;
  uint8_t* scales;
  int64_t ss;
};

// rows of a workgroup of T-thread rows
constexpr int norm_rows(int T) { return T < 256 ? 256 / T : 1; }

// The sum over a row's T threads, in every one of them.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* s_sum) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += s_sum[i];
  }
  return v;
}

// A row whose sum of squares passes f32's range (4096 values of 2.9e17) is summed once more in
// these units: 2^24 values of up to 2^128 stay within it then, and what they lose are values far
// below the row's root mean square.
constexpr float kFar = 0x1p-80f;

// 1 / the row's root mean square, given its sum of squares; where that is an infinity, `squares`
// gives a thread's share in units of kFar. (The least such quotient, 2^-128, has 22 bits.)
template <int T, class F>
__device__ __forceinline__ float row_inverse(float sum, const NormArgs& a, float* s_sum,
                                             F squares) {
  if (sum != __builtin_inff()) return rsqrtf(sum / (float)a.hidden + a.eps);
  if constexpr (T > 64) __syncthreads();  // all threads of a row are here; s_sum has been read
  return rsqrtf(row_sum<T>(squares(), s_sum) / (float)a.hidden) * kFar;
}

__device__ __forceinline__ uint4 load8(const uint16_t* p, int k, bool live) {
  return live ? *reinterpret_cast<const uint4*>(p + k) : make_uint4(0, 0, 0, 0);
}

// the residual's row, and the codes of 8 normalised values a lane, at k of a row
__device__ __forceinline__ void norm_out(const NormArgs& a, int64_t row, int k, bool live,
                                         const float (&h)[8], uint4 weight, float inv) {
  float w[8], y[8];
  floats8(weight, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = live ? h[i] * inv * w[i] : 0.0f;
  if (a.res && live) {
    uint16_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = to_bf(h[i]);
    *reinterpret_cast<uint4*>(a.res + row * a.rs + k) = pack8(r);
  }
  uint2 c;
  const uint32_t byte = group_codes8(y, c);
  if (live) *reinterpret_cast<uint2*>(a.codes + row * a.cs + k) = c;
  if (live && (threadIdx.x & 15) == 0) a.scales[row * a.ss + k / kFp8Group] = (uint8_t)byte;
}

// T threads a row, each with C times 8 values that stay in registers from the one read to the
// writes: 4096 rows of 4096 with a residual 24.2 us (4.9 TB/s) over six sets of rows in turn, 20.3
// us over three, of which the cache keeps a part; 4 rows 2.9 us. (Read twice it took 28.5 us where
// this took 22.5.) T: a row in one piece or two a thread, in one wave where it fits.
template <int T, int C>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rmsnorm_fp8(NormArgs a) {
  __shared__ float s_sum[T / 64];
  const int64_t row = (int64_t)blockIdx.x * norm_rows(T) + threadIdx.x / T;
  if (row >= a.rows) return;  // whole waves, and T > 64 has one row a workgroup
  const int tid = threadIdx.x % T;
  const uint16_t* x = a.x + row * a.xs;
  const uint16_t* res = a.res + row * a.rs;
  uint4 xv[C], rv[C], wv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int k = 8 * (c * T + tid);
    const bool live = k < a.hidden;
    xv[c] = load8(x, k, live);
    if (a.res) rv[c] = load8(res, k, live);
    wv[c] = load8(a.w, k, live);
  }
  float h[C][8], ss = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    floats8(xv[c], h[c]);
    if (a.res) {
      float r[8];
      floats8(rv[c], r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[c][i] += r[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += h[c][i] * h[c][i];
  }
  const float inv = row_inverse<T>(row_sum<T>(ss, s_sum), a, s_sum, [&] {
    float far = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) far += h[c][i] * kFar * (h[c][i] * kFar);
    return far;
  });
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int k = 8 * (c * T + tid);
    norm_out(a, row, k, k < a.hidden, h[c], wv[c], inv);
  }
}

constexpr int kLongThreads = 1024, kLongRow = 16384;

// Rows that do not fit the registers are read twice, the second time from the cache.
__global__ __launch_bounds__(kLongThreads) void k_rmsnorm_fp8_long(NormArgs a) {
  __shared__ float s_sum[kLongThreads / 64];
  const int64_t row = blockIdx.x;
  const uint16_t* x = a.x + row * a.xs;
  const uint16_t* res = a.res + row * a.rs;
  auto load = [&](int k, float (&h)[8]) {
    floats8(load8(x, k, k < a.hidden), h);
    if (a.res) {
      float r[8];
      floats8(load8(res, k, k < a.hidden), r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
  };
  auto squares = [&](float unit) {
    float ss = 0.0f;
    for (int k = 8 * threadIdx.x; k < a.hidden; k += 8 * kLongThreads) {
      float h[8];
      load(k, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += h[i] * unit * (h[i] * unit);
    }
    return ss;
  };
  const float inv = row_inverse<kLongThreads>(row_sum<kLongThreads>(squares(1.0f), s_sum), a,
                                              s_sum, [&] { return squares(kFar); });
  const int padded = (a.hidden + kFp8Group - 1) / kFp8Group * kFp8Group;
  for (int k = 8 * threadIdx.x; k < padded; k += 8 * kLongThreads) {  // whole groups of lanes
    float h[8];
    load(k, h);
    norm_out(a, row, k, k < a.hidden, h, load8(a.w, k, k < a.hidden), inv);
  }
}

template <int T, int C>
void launch_norm(const NormArgs& a, hipStream_t s) {
  const int per = norm_rows(T);
  hipLaunchKernelGGL((k_rmsnorm_fp8<T, C>), dim3((unsigned)((a.rows + per - 1) / per)),
                     dim3(T < 256 ? 256 : T), 0, s, a);
}

constexpr int kMaxRows = (1 << 22) - 1;  // 1024 threads each in a grid of less than 2^32

// the limits that both entry points share: whole 16-byte pieces of bf16, 8-byte pieces of codes
int rows_status(const void* x, int64_t xs, int rows, int width, const void* codes, int64_t cs,
                int64_t ss) {
  if (width % 16 || width > (1 << 24) || rows > kMaxRows) return HS_ERR_UNSUPPORTED;
  if ((xs % 8) || (cs % 8) || xs < width || cs < width || ss < (width + kFp8Group - 1) / kFp8Group)
    return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)x & 15) || ((uintptr_t)codes & 7)) return HS_ERR_UNSUPPORTED;
  return HS_OK;
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

int hs_quantize_rows_fp8(const void* x, int64_t x_stride, int rows, int width, void* codes,
                         int64_t codes_stride, void* scales, int64_t scales_stride, void* stream) {
  if (rows == 0) return HS_OK;
  if (!x || !codes || !scales || rows < 0 || width < 1) return HS_ERR_INVALID;
  const int status = rows_status(x, x_stride, rows, width, codes, codes_stride, scales_stride);
  if (status != HS_OK) return status;
  const int groups = (width + kFp8Group - 1) / kFp8Group;
  const int64_t blocks = ((int64_t)rows * groups * 16 + kQuantThreads - 1) / kQuantThreads;
  if (blocks * kQuantThreads > UINT32_MAX) return HS_ERR_UNSUPPORTED;  // a grid's threads
  hipLaunchKernelGGL(k_quantize_rows, dim3((unsigned)blocks), dim3(kQuantThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), static_cast<const uint16_t*>(x),
                     x_stride, rows, width, groups, static_cast<uint8_t*>(codes), codes_stride,
                     static_cast<uint8_t*>(scales), scales_stride);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

int hs_rmsnorm_fp8(const void* x, int64_t x_stride, void* residual, int64_t residual_stride,
                   const void* weight, float eps, int rows, int hidden, void* codes,
                   int64_t codes_stride, void* scales, int64_t scales_stride, void* stream) {
  if (rows == 0) return HS_OK;
  if (!x || !weight || !codes || !scales || rows < 0 || hidden < 1) return HS_ERR_INVALID;
  const int status = rows_status(x, x_stride, rows, hidden, codes, codes_stride, scales_stride);
  if (status != HS_OK) return status;
  if (((uintptr_t)weight | (uintptr_t)residual) & 15) return HS_ERR_UNSUPPORTED;
  if (residual && ((residual_stride % 8) || residual_stride < hidden)) return HS_ERR_UNSUPPORTED;
  NormArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.xs = x_stride;
  a.res = static_cast<uint16_t*>(residual);
  a.rs = residual ? residual_stride : 0;
  a.w = static_cast<const uint16_t*>(weight);
  a.eps = eps;
  a.hidden = hidden;
  a.codes = static_cast<uint8_t*>(codes);
  a.cs = codes_stride;
  a.scales = static_cast<uint8_t*>(scales);
  a.ss = scales_stride;
  a.rows = rows;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (hidden <= 512) launch_norm<64, 1>(a, s);
  else if (hidden <= 1024) launch_norm<64, 2>(a, s);
  else if (hidden <= 2048) launch_norm<256, 1>(a, s);
  else if (hidden <= 4096) launch_norm<512, 1>(a, s);
  else if (hidden <= 8192) launch_norm<512, 2>(a, s);
  else if (hidden <= kLongRow) launch_norm<1024, 2>(a, s);
  else
    hipLaunchKernelGGL(k_rmsnorm_fp8_long, dim3((unsigned)rows), dim3(kLongThreads), 0, s, a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // extern "C"
