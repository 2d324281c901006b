// Log-probabilities of given tokens with the rows' entropy and most likely tokens.
// Of a row y = logits / T with maximum m, S = sum exp(y - m), U = sum (y - m) exp(y - m):
//   log p(t) = (y_t - m) - ln S        entropy = ln S - U / S
// and the `top` largest logits in order, the lower index first among equal ones.
// One pass over the logits, which bound it: a workgroup takes a chunk of a row into
// registers, so its maximum, its two sums and its candidates come from one read.
//
// Candidates: a wave's n-th largest lane maximum is at most its n-th largest value, so
// only values from there on can be among the row's n largest; the lane maxima's n-th
// largest is found bit by bit with ballots. What passes is ranked by counting and the
// chunk's n best are written in order (one at a time where more pass than the list
// holds: many equal values). k_logprobs_join adds up a row's chunks (sums rescaled to
// the row's maximum, f32) and ranks their lists' values the same way.
//
// Order: values as the row holds them (a temperature does not change it), -0 as 0,
// and NaN above everything. A row with a NaN, with +inf, or with nothing but -inf gets
// NaN log-probabilities and entropy, as the formulas give.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_device.h"

namespace hs {
namespace {

constexpr int kLpT = 256;      // threads of a workgroup
constexpr int kMaxTop = 32;
constexpr int kListed = 512;   // candidates of a chunk that are ranked by counting
constexpr int kPerLane = 4;    // chunks of a row over the lanes of a wave: at most 256
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobArgs {
  const void* logits;
  int64_t stride;
  const int64_t* tokens;
  const float* temps;  // or null
  int rows, vocab, top, chunks;
  float* logprobs;
  float* entropy;
  int64_t* top_ids;
  float* top_logprobs;
  // per (row, chunk): m, S, U, unused; then top keys and ids
  float4* sums;
  uint32_t* keys;
  int32_t* ids;
};

// order of a value: larger is larger, -0 as 0, NaN the largest
__device__ __forceinline__ uint32_t order_key(float x) {
  return x != x ? 0xffffffffu : hs_key(x);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// maximum that keeps a NaN
__device__ __forceinline__ float nan_max(float a, float b) { return (a > b || a != a) ? a : b; }
__device__ __forceinline__ float wave_nan_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = nan_max(v, __shfl_xor(v, o, 64));
  return v;
}

template <typename T>
__device__ __forceinline__ float logit(const T* x, int64_t i) {
  if constexpr (sizeof(T) == 2) return bf16_to_f32(x[i]);
  else return x[i];
}

// value e of a thread's chunk share: element 8 * (i * kLpT + tid) + j, e = 8 i + j
__device__ __forceinline__ int elem_of(int e) {
  return 8 * ((e >> 3) * kLpT + (int)threadIdx.x) + (e & 7);
}

// E values a thread: a chunk is E * kLpT elements.
template <typename T, int E, bool kAligned>
__global__ __launch_bounds__(kLpT) void k_logprobs_chunk(LogprobArgs a) {
  constexpr int kChunkLen = E * kLpT;
  __shared__ float s_f[3][4];
  __shared__ uint32_t s_key[kListed];
  __shared__ int s_id[kListed];
  __shared__ int s_n;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.y, chunk = blockIdx.x;
  const int base = chunk * kChunkLen, len = min(kChunkLen, a.vocab - base);
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride + base;
  float v[E];
#pragma unroll
  for (int i = 0; i < E / 8; ++i) {
    const int at = elem_of(8 * i);
    if (kAligned && at + 8 <= len) {
      if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(x + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] = u2f(w[j] << 16);
          v[8 * i + 2 * j + 1] = u2f(w[j] & 0xffff0000u);
        }
      } else {
        const float4 f = *reinterpret_cast<const float4*>(x + at);
        const float4 h = *reinterpret_cast<const float4*>(x + at + 4);
        v[8 * i] = f.x, v[8 * i + 1] = f.y, v[8 * i + 2] = f.z, v[8 * i + 3] = f.w;
        v[8 * i + 4] = h.x, v[8 * i + 5] = h.y, v[8 * i + 6] = h.z, v[8 * i + 7] = h.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[8 * i + j] = at + j < len ? logit<T>(x, at + j) : -INFINITY;
      }
    }
  }
  if (threadIdx.x == 0) s_n = 0;

  // the largest value, the sums
  float most = v[0];
#pragma unroll
  for (int e = 1; e < E; ++e) most = nan_max(most, v[e]);
  const float lane_most = most;
  most = wave_nan_max(most);
  if (lane == 0) s_f[0][wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) most = nan_max(most, s_f[0][w]);
  const float inv_t = a.temps ? 1.0f / a.temps[row] : 1.0f;
  const float m = most * inv_t;
  float S = 0.0f, U = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = v[e] * inv_t - m;
    const float p = __builtin_amdgcn_exp2f(d * kLog2e);
    S += p;
    U += p == 0.0f ? 0.0f : p * d;  // an excluded token's -inf takes no part
  }
  S = wave_sum(S);
  U = wave_sum(U);
  if (lane == 0) s_f[1][wave] = S, s_f[2][wave] = U;

  if (a.top > 0) {
    // the top-th largest lane maximum of the wave, by its bits from the highest
    const uint32_t mine = order_key(lane_most);
    uint32_t bar = 0;
#pragma unroll
    for (int b = 31; b >= 0; --b) {
      const uint32_t trial = bar | (1u << b);
      if (__popcll(__ballot(mine >= trial)) >= a.top) bar = trial;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t key = order_key(v[e]);
      const int id = elem_of(e);
      if (key >= bar && id < len) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kListed) {
          s_key[at] = key;
          s_id[at] = id;
        }
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t o = (int64_t)row * a.chunks + chunk;
    a.sums[o] = make_float4(m, (s_f[1][0] + s_f[1][1]) + (s_f[1][2] + s_f[1][3]),
                            (s_f[2][0] + s_f[2][1]) + (s_f[2][2] + s_f[2][3]), 0.0f);
  }
  if (a.top > 0) {
    const int n = s_n;
    const int64_t o = ((int64_t)row * a.chunks + chunk) * a.top;
    if (n <= kListed) {
      for (int c = threadIdx.x; c < n; c += kLpT) {
        const uint32_t key = s_key[c];
        const int id = s_id[c];
        int rank = 0;
        for (int i = 0; i < n && rank < a.top; ++i)
          rank += s_key[i] > key || (s_key[i] == key && s_id[i] < id);
        if (rank < a.top) {
          a.keys[o + rank] = key;
          a.ids[o + rank] = base + id;
        }
      }
      // a short last chunk has fewer: key 0 stands for none (no value has it)
      for (int r = n + threadIdx.x; r < a.top; r += kLpT) {
        a.keys[o + r] = 0;
        a.ids[o + r] = 0x7fffffff;
      }
    } else {
      uint32_t last_key = 0xffffffffu;
      int last_id = -1;
      for (int r = 0; r < a.top; ++r) {
        uint32_t key = 0;
        int id = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t k = order_key(v[e]);
          const int i = elem_of(e);
          const bool behind = k < last_key || (k == last_key && i > last_id);
          if (behind && i < len && (k > key || (k == key && i < id))) key = k, id = i;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
          const uint32_t k = (uint32_t)__shfl_xor((int)key, d, 64);
          const int i = __shfl_xor(id, d, 64);
          if (k > key || (k == key && i < id)) key = k, id = i;
        }
        __syncthreads();  // the last round's reads
        if (lane == 0) s_key[wave] = key, s_id[wave] = id;
        __syncthreads();
        for (int w = 0; w < 4; ++w) {
          const uint32_t k = s_key[w];
          const int i = s_id[w];
          if (k > key || (k == key && i < id)) key = k, id = i;
        }
        if (threadIdx.x == 0) a.keys[o + r] = key, a.ids[o + r] = base + id;
        last_key = key;
        last_id = id;
      }
    }
  }
}

// One wave a row.
template <typename T>
__global__ __launch_bounds__(64) void k_logprobs_join(LogprobArgs a) {
  const int lane = threadIdx.x, row = blockIdx.x;
  const float4* sums = a.sums + (int64_t)row * a.chunks;
  float m = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) m = nan_max(m, sums[c].x);
  m = wave_nan_max(m);
  float S = 0.0f, U = 0.0f;
  for (int c = lane; c < a.chunks; c += 64) {
    const float4 s = sums[c];
    // sums under the chunk's maximum, moved to the row's
    const float d = s.x - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
    S += f == 0.0f ? 0.0f : f * s.y;
    U += f == 0.0f ? 0.0f : f * (s.z + d * s.y);
  }
  S = wave_sum(S);
  U = wave_sum(U);
  const float log_s = logf(S);
  const float inv_t = a.temps ? 1.0f / a.temps[row] : 1.0f;
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
  if (lane == 0) {
    if (a.entropy) a.entropy[row] = log_s - U / S;
    if (a.logprobs) {
      const int64_t tok = a.tokens[row];
      float lp = -INFINITY;  // a token that the vocabulary does not have
      if (tok >= 0 && tok < a.vocab) lp = (logit<T>(x, tok) * inv_t - m) - log_s;
      a.logprobs[row] = lp;
    }
  }
  if (a.top == 0) return;
  // The chunks' lists are in order and a lane's best is the first of one of its lists.
  // Only lanes whose best is among the `top` best ones can hold one of the row's.
  __shared__ uint32_t s_key[kMaxTop * kPerLane * kMaxTop];
  __shared__ int s_id[kMaxTop * kPerLane * kMaxTop];
  __shared__ int s_n;
  const uint32_t* keys = a.keys + (int64_t)row * a.chunks * a.top;
  const int32_t* ids = a.ids + (int64_t)row * a.chunks * a.top;
  if (lane == 0) s_n = 0;
  uint32_t key = 0;
  int id = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int c = lane + 64 * i;
    if (c < a.chunks) {
      const uint32_t k = keys[c * a.top];
      const int d = ids[c * a.top];
      if (k > key || (k == key && d < id)) key = k, id = d;
    }
  }
  uint32_t bar = 0;
#pragma unroll
  for (int b = 31; b >= 0; --b) {
    const uint32_t trial = bar | (1u << b);
    if (__popcll(__ballot(key >= trial)) >= a.top) bar = trial;
  }
  // of the lanes at the bar, as many as are left, those of the lowest ids
  const int left = a.top - __popcll(__ballot(key > bar));
  uint32_t first = 0;  // the ids below it are those of fewer than `left` lanes
#pragma unroll
  for (int b = 30; b >= 0; --b) {
    const uint32_t trial = first | (1u << b);
    if (__popcll(__ballot(key == bar && (uint32_t)id < trial)) < left) first = trial;
  }
  __syncthreads();
  if (key > bar || (key == bar && key != 0 && (uint32_t)id <= first)) {
    for (int i = 0; i < kPerLane; ++i) {
      const int c = lane + 64 * i;
      if (c >= a.chunks) break;
      for (int r = 0; r < a.top; ++r) {
        const uint32_t k = keys[c * a.top + r];
        if (k == 0 || k < bar) break;
        const int at = atomicAdd(&s_n, 1);
        s_key[at] = k;
        s_id[at] = ids[c * a.top + r];
      }
    }
  }
  __syncthreads();
  const int n = s_n;
  for (int c = lane; c < n; c += 64) {
    const uint32_t k = s_key[c];
    const int d = s_id[c];
    int rank = 0;
    for (int i = 0; i < n && rank < a.top; ++i)
      rank += s_key[i] > k || (s_key[i] == k && s_id[i] < d);
    if (rank < a.top) {
      a.top_ids[(int64_t)row * a.top + rank] = d;
      a.top_logprobs[(int64_t)row * a.top + rank] = (logit<T>(x, d) * inv_t - m) - log_s;
    }
  }
}

// values a thread: short chunks while there are few rows to fill the chip with, but
// at most 256 chunks a row
int elems_of(int rows, int vocab) {
  const int64_t small = (int64_t)rows * ((vocab + 8 * kLpT - 1) / (8 * kLpT));
  if (small <= 2048 && vocab <= 256 * 8 * kLpT) return 8;
  return 32;
}
int chunks_of(int rows, int vocab) {
  const int len = elems_of(rows, vocab) * kLpT;
  return (vocab + len - 1) / len;
}
bool sizes_ok(int rows, int vocab, int top) {
  return rows >= 1 && vocab >= 1 && top >= 0 && top <= kMaxTop && top <= vocab;
}

template <typename T, int E>
void launch(const LogprobArgs& a, bool aligned, hipStream_t s) {
  const dim3 grid((unsigned)a.chunks, (unsigned)a.rows);
  if (aligned) hipLaunchKernelGGL((k_logprobs_chunk<T, E, true>), grid, dim3(kLpT), 0, s, a);
  else hipLaunchKernelGGL((k_logprobs_chunk<T, E, false>), grid, dim3(kLpT), 0, s, a);
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

size_t hs_token_logprobs_workspace_size(int rows, int vocab, int top) {
  if (!sizes_ok(rows, vocab, top)) return 0;
  return (size_t)rows * chunks_of(rows, vocab) * (sizeof(float4) + (size_t)top * 8);
}

int hs_token_logprobs(const void* logits, int logits_dtype, int64_t logits_row_stride, int rows,
                      int vocab, const int64_t* tokens, const float* temperatures, int top,
                      float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs,
                      void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return HS_OK;
  if (!logits || !sizes_ok(rows, vocab, top)) return HS_ERR_INVALID;
  if (logits_dtype != HS_F32 && logits_dtype != HS_BF16) return HS_ERR_INVALID;
  if ((tokens == nullptr) != (logprobs == nullptr)) return HS_ERR_INVALID;
  if (top > 0 && (!top_ids || !top_logprobs)) return HS_ERR_INVALID;
  if (logits_row_stride < vocab) return HS_ERR_INVALID;
  const int esz = logits_dtype == HS_BF16 ? 2 : 4;
  if ((uintptr_t)logits & (esz - 1)) return HS_ERR_UNSUPPORTED;
  // 256 chunks of 8192 values a row, a grid's second dimension of rows
  if (rows > 65535 || vocab > 256 * 32 * kLpT) return HS_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < hs_token_logprobs_workspace_size(rows, vocab, top))
    return HS_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HS_ERR_UNSUPPORTED;
  LogprobArgs a;
  a.logits = logits;
  a.stride = logits_row_stride;
  a.tokens = tokens;
  a.temps = temperatures;
  a.rows = rows;
  a.vocab = vocab;
  a.top = top;
  a.chunks = chunks_of(rows, vocab);
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  const size_t n = (size_t)rows * a.chunks;
  a.sums = static_cast<float4*>(workspace);
  a.keys = reinterpret_cast<uint32_t*>(a.sums + n);
  a.ids = reinterpret_cast<int32_t*>(a.keys + n * top);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // 16-byte loads of every row
  const bool aligned = !(((uintptr_t)logits | (uint64_t)(logits_row_stride * esz)) & 15);
  const bool wide = elems_of(rows, vocab) == 32;
  if (esz == 2) {
    if (wide) launch<uint16_t, 32>(a, aligned, s);
    else launch<uint16_t, 8>(a, aligned, s);
  } else {
    if (wide) launch<float, 32>(a, aligned, s);
    else launch<float, 8>(a, aligned, s);
  }
  if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  if (esz == 2) hipLaunchKernelGGL(k_logprobs_join<uint16_t>, dim3((unsigned)rows), dim3(64), 0, s, a);
  else hipLaunchKernelGGL(k_logprobs_join<float>, dim3((unsigned)rows), dim3(64), 0, s, a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // extern "C"
