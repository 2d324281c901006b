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

// 8 values a thread
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
  int hidden;
  uint8_t* codes;
  int64_t cs;
  uint8_t* scales;
  int64_t ss;
};

constexpr int kNormThreads = 256;

// A workgroup a row.
__global__ __launch_bounds__(kNormThreads) void k_rmsnorm_fp8(NormArgs a) {
  __shared__ float s_sum[kNormThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const uint16_t* x = a.x + row * a.xs;
  uint16_t* res = a.res ? a.res + row * a.rs : nullptr;
  auto load = [&](int k, float (&h)[8]) {
    floats8(*reinterpret_cast<const uint4*>(x + k), h);
    if (res) {
      float r[8];
      floats8(*reinterpret_cast<const uint4*>(res + k), r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
  };
  float ss = 0.0f;
  for (int k = 8 * tid; k < a.hidden; k += 8 * kNormThreads) {
    float h[8];
    load(k, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += h[i] * h[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
  if ((tid & 63) == 0) s_sum[tid >> 6] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < kNormThreads / 64; ++i) ss += s_sum[i];
  const float inv = rsqrtf(ss / (float)a.hidden + a.eps);
  const int padded = (a.hidden + kFp8Group - 1) / kFp8Group * kFp8Group;
  for (int k = 8 * tid; k < padded; k += 8 * kNormThreads) {  // whole groups of lanes
    float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (k < a.hidden) {
      load(k, y);
      if (res) {
        uint16_t r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = to_bf(y[i]);
        *reinterpret_cast<uint4*>(res + k) = pack8(r);
      }
      float w[8];
      floats8(*reinterpret_cast<const uint4*>(a.w + k), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * w[i];
    }
    uint2 c;
    const uint32_t byte = group_codes8(y, c);
    if (k < a.hidden) *reinterpret_cast<uint2*>(a.codes + row * a.cs + k) = c;
    if ((tid & 15) == 0) a.scales[row * a.ss + k / kFp8Group] = (uint8_t)byte;
  }
}

// the limits that both entry points share: whole 16-byte pieces of bf16, 8-byte pieces of codes
int rows_status(const void* x, int64_t xs, int rows, int width, const void* codes, int64_t cs,
                int64_t ss) {
  if (width % 16 || width > (1 << 24) || rows > (1 << 24)) return HS_ERR_UNSUPPORTED;
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
  if (blocks > INT32_MAX) return HS_ERR_UNSUPPORTED;
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
  hipLaunchKernelGGL(k_rmsnorm_fp8, dim3((unsigned)rows), dim3(kNormThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // extern "C"
