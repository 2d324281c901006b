// Log-probabilities of given tokens with the rows' entropy and most likely tokens.
// Of a row y = logits / T with maximum m, S = sum exp(y - m), U = sum (y - m) exp(y - m):
//   log p(t) = (y_t - m) - ln S        entropy = ln S - U / S
// and the `top` largest logits in order, the lower index first among equal ones.
// Exponents are powers of two: (x - max x) log2(e) / T.
// k_logprobs_chunk reads the logits, which bound it, once: a workgroup takes a chunk of
// a row into registers and leaves its maximum, its two sums and the maximum of every 32
// neighbouring logits. k_logprobs_join, a workgroup a row, adds up the chunks (sums
// rescaled to the row's maximum, f32) and finds the alternatives: the n-th largest of
// its 256 threads' shares of those maxima is at most the row's n-th largest value, so
// only values from there on can be among the n largest, and they lie in the groups of 32
// whose maxima reach it. It finds that bar bit by bit with ballots, reads those groups
// again (about n of them), and ranks what passes by counting. (256 rows of 151936 bf16
// logits, top 20: 39 us with the n largest of every chunk picked in the chunk's
// workgroup and merged, 30 us so, of which the join is about 9; 512 rows of f32
// logits, top 5: 67 us, 4.7 TB/s.) Where more passes than its
// list holds - many equal values - the row's values are taken one by one, and -inf, what
// a mask leaves of excluded tokens, only fills up.
//
// Order: values as the row holds them (a temperature does not change it), -0 as 0,
// and NaN above everything. A row with a NaN, with +inf, or with nothing but -inf gets
// NaN log-probabilities and entropy, as the formulas give.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_device.h"
#include "hs_model_dev.h"

namespace hs {
namespace {

constexpr int kLpT = 256;      // threads of a workgroup
constexpr int kMaxTop = 32;
constexpr int kListed = 1024;  // groups and values that are ranked by counting
constexpr int kKept = 20;      // group maxima of a row that a thread of the join keeps
constexpr int kGroup = 32;     // neighbouring logits with a maximum kept
constexpr float kLn2 = 0.6931471805599453f;
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
  float4* sums;    // [row][chunk]: largest logit, S, U (in powers of two), unused
  uint32_t* most;  // [row][groups]: order of the groups' maxima
  int groups;      // of a row: its chunks' logits over kGroup
};

// order of a value: larger is larger, -0 as 0, NaN the largest
__device__ __forceinline__ uint32_t order_key(float x) {
  return x != x ? 0xffffffffu : hs_key(x);
}

// a value and its place as one number: larger comes first
__device__ __forceinline__ uint64_t listing(uint32_t key, int id) {
  return ((uint64_t)key << 32) | (uint32_t)~(uint32_t)id;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}
// Over a wave, by lane swaps in the vector pipe (through LDS the three of a chunk took
// 1.2 us of the 256-row call): with f commutative and associative but for rounding, every
// lane gets the same result.
template <typename F>
__device__ __forceinline__ float over_wave(float v, F f) {
  v = f(v, row_xor1(v));
  v = f(v, row_xor2(v));
  v = f(v, row_mirror8(v));
  v = f(v, row_xor8(v));
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_max(float v) {
  return over_wave(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return over_wave(v, [](float a, float b) { return a + b; });
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

// The largest of three, in one instruction: fmaxf would quiet every operand before it.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// E values a thread: a chunk is E * kLpT elements.
template <typename T, int E, bool kAligned>
__global__ __launch_bounds__(kLpT) void k_logprobs_chunk(LogprobArgs a) {
  constexpr int kChunkLen = E * kLpT;
  __shared__ float s_f[3][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.y, chunk = blockIdx.x;
  const int base = chunk * kChunkLen, len = min(kChunkLen, a.vocab - base);
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride + base;
  float v[E];
  if (kAligned && len == kChunkLen) {  // every load of the chunk before the first wait
    constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
    uint32_t w[E / 8][kWords];
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
#pragma unroll
      for (int h = 0; h < kWords / 4; ++h) {
        const uint4 u = reinterpret_cast<const uint4*>(x + elem_of(8 * i))[h];
        w[i][4 * h] = u.x, w[i][4 * h + 1] = u.y, w[i][4 * h + 2] = u.z, w[i][4 * h + 3] = u.w;
      }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (sizeof(T) == 2)
        v[e] = u2f((e & 1) ? w[e >> 3][(e & 7) >> 1] & 0xffff0000u : w[e >> 3][(e & 7) >> 1] << 16);
      else
        v[e] = u2f(w[e >> 3][e & 7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = logit<T>(x, min(elem_of(e), len - 1));
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = elem_of(e) < len ? v[e] : -INFINITY;
  }
  // the largest values of the thread's groups of 8 (of a NaN, a number or NaN: the sums
  // are NaN then, and the group is marked below)
  float group[E / 8], most = -INFINITY;
#pragma unroll
  for (int i = 0; i < E / 8; ++i) {
    const float* e = v + 8 * i;
    group[i] = max3(max3(e[0], e[1], e[2]), max3(e[3], e[4], e[5]), max3(e[6], e[6], e[7]));
    most = fmaxf(most, group[i]);
  }
  most = wave_max(most);
  if (lane == 0) s_f[0][wave] = most;
  __syncthreads();
  most = fmaxf(fmaxf(s_f[0][0], s_f[0][1]), fmaxf(s_f[0][2], s_f[0][3]));
  const float c = a.temps ? kLog2e / a.temps[row] : kLog2e;
  const float ref = most == -INFINITY ? 0.0f : most;
  float S = 0.0f, U = 0.0f;
  auto add = [&](float d) {
    const float p = __builtin_amdgcn_exp2f(d);
    S += p;
    // far below, where p is 0, d may be -inf: it takes no part
    U = fmaf(p, fmaxf(d, -512.0f), U);
  };
  // The difference first: it is exact where it counts and cannot overflow, and the largest
  // logit's exponent is 0, so that S is 1 or more and no log-probability above 0. (v c - ref c
  // in one step is an instruction less, 28.3 us for 30.0 at 256 rows of 151936 bf16 logits, but
  // rounds ref c: a certain token came out at up to 2.6e-6.)
#pragma unroll
  for (int e = 0; e < E; ++e) add((v[e] - ref) * c);
  if (!(S < INFINITY)) {
    // a NaN among the thread's values, perhaps: its groups, and no others, count as
    // +inf, for they do hold a value that no other is above
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (v[e] != v[e]) group[e >> 3] = INFINITY;
  }
  S = wave_sum(S);
  U = wave_sum(U);
  if (lane == 0) s_f[1][wave] = S, s_f[2][wave] = U;
  if (a.top > 0) {
    // four neighbouring lanes hold a group, and lane i of them writes the i-th
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      float g = group[i];
      g = fmaxf(g, row_xor1(g));
      g = fmaxf(g, row_xor2(g));
      if ((lane & 3) == i) mine = g;
    }
    if ((lane & 3) < E / 8)
      a.most[(int64_t)row * a.groups + (base + 8 * ((lane & 3) * kLpT + ((int)threadIdx.x & ~3))) / kGroup] =
          order_key(mine);
  }
  __syncthreads();
  if (threadIdx.x == 0)
    a.sums[(int64_t)row * a.chunks + chunk] =
        make_float4(most, (s_f[1][0] + s_f[1][1]) + (s_f[1][2] + s_f[1][3]),
                    (s_f[2][0] + s_f[2][1]) + (s_f[2][2] + s_f[2][3]), 0.0f);
}

// The `top` largest of a row with many equal ones: value by value, the ids of one in
// order. s_n: a shared counter of four.
template <typename T>
__device__ void top_by_value(const LogprobArgs& a, const T* x, int64_t* ids, int* s_n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t last = 1ull << 32;  // orders from here on are done
  int filled = 0;
  while (filled < a.top) {
    uint32_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kLpT) {
      const uint32_t k = order_key(logit<T>(x, i));
      if (k < last && k > best) best = k;
    }
    best = wave_max_u32(best);
    __syncthreads();
    if (lane == 0) s_n[wave] = (int)best;
    __syncthreads();
    for (int w = 0; w < 4; ++w) best = max(best, (uint32_t)s_n[w]);
    for (int i = 0; i < a.vocab && filled < a.top; i += kLpT) {
      const int id = i + (int)threadIdx.x;
      const bool take = id < a.vocab && order_key(logit<T>(x, id)) == best;
      const uint64_t all = __ballot(take);
      __syncthreads();
      if (lane == 0) s_n[wave] = __popcll(all);
      __syncthreads();
      int to = filled + __popcll(all & ((1ull << lane) - 1));
      for (int w = 0; w < 4; ++w) {
        if (w < wave) to += s_n[w];
        filled += s_n[w];
      }
      if (take && to < a.top) ids[to] = id;
    }
    last = best;
  }
}

template <typename T>
__global__ __launch_bounds__(kLpT) void k_logprobs_join(LogprobArgs a) {
  __shared__ uint4 s_most[kLpT / 4];
  __shared__ int s_group[kListed];
  __shared__ uint64_t s_list[kListed];
  __shared__ int s_n[4];
  __shared__ float s_f[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.stride;
  const float c = a.temps ? kLog2e / a.temps[row] : kLog2e;
  const uint32_t* most = a.most + (int64_t)row * a.groups;
  // the thread's share, kept for the second look at it
  uint32_t share[kKept];
  if (a.top > 0) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int i = j * kLpT + (int)threadIdx.x;
      share[j] = most[min(i, a.groups - 1)];
    }
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      if (j * kLpT + (int)threadIdx.x >= a.groups) share[j] = 0;
      mine = max(mine, share[j]);
    }
#pragma unroll 8
    for (int i = kKept * kLpT + (int)threadIdx.x; i < a.groups; i += kLpT) mine = max(mine, most[i]);
    reinterpret_cast<uint32_t*>(s_most)[threadIdx.x] = mine;
    if (threadIdx.x < 4) s_n[threadIdx.x] = 0;
  }
  if (wave == 3) {
    const float4* sums = a.sums + (int64_t)row * a.chunks;
    float m = -INFINITY;
    for (int i = lane; i < a.chunks; i += 64) m = fmaxf(m, sums[i].x);
    m = wave_max(m);
    float S = 0.0f, U = 0.0f;
    for (int i = lane; i < a.chunks; i += 64) {
      const float4 s = sums[i];
      // sums under the chunk's maximum, moved to the row's
      const float d = (s.x - m) * c, f = __builtin_amdgcn_exp2f(d);
      // far below, where f is 0 and d may be -inf, a chunk's numbers take no part; a NaN,
      // which the chunk's maximum does not show, always does
      const bool none = f == 0.0f && s.y == s.y;
      S += none ? 0.0f : f * s.y;
      U += none ? 0.0f : f * (s.z + d * s.y);
    }
    S = wave_sum(S);
    U = wave_sum(U);
    if (lane == 0) {
      const float log_s = log2f(S);
      if (a.entropy) a.entropy[row] = (log_s - U / S) * kLn2;
      if (a.logprobs) {
        const int64_t tok = a.tokens[row];
        float lp = -INFINITY;  // a token that the vocabulary does not have
        if (tok >= 0 && tok < a.vocab) lp = ((logit<T>(x, tok) - m) * c - log_s) * kLn2;
        a.logprobs[row] = lp;
      }
      s_f[0] = m;
      s_f[1] = log_s;
    }
  }
  if (a.top == 0) return;
  __syncthreads();

  // the bar, by the upper half of the order's bits (a bf16's all; the lower bound that
  // is left of an f32's serves as well)
  const uint4 k = s_most[lane];
  uint32_t bits = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t trial = bits | (1u << b);
    if (__popcll(__ballot(k.x >= trial)) + __popcll(__ballot(k.y >= trial)) +
            __popcll(__ballot(k.z >= trial)) + __popcll(__ballot(k.w >= trial)) >= a.top)
      bits = trial;
  }
  float bar = hs_unkey(bits);
  // fewer than `top` threads' shares hold anything above -inf: all such values
  if (bar != bar || bar == -INFINITY) bar = -3.402823466e38f;
  const uint32_t reach = max(bits, order_key(-3.402823466e38f));
  auto reached = [&](uint32_t key, int i) {
    if (key >= reach) {
      const int at = atomicAdd(&s_n[0], 1);
      if (at < kListed) s_group[at] = i;
    }
  };
#pragma unroll
  for (int j = 0; j < kKept; ++j) reached(share[j], j * kLpT + (int)threadIdx.x);
  for (int i = kKept * kLpT + (int)threadIdx.x; i < a.groups; i += kLpT) reached(most[i], i);
  __syncthreads();
  const int groups = s_n[0];
  for (int i = threadIdx.x / kGroup; i < min(groups, kListed); i += kLpT / kGroup) {
    const int id = s_group[i] * kGroup + (threadIdx.x & (kGroup - 1));
    if (id < a.vocab) {
      const float f = logit<T>(x, id);
      if (!(f < bar)) {
        const int at = atomicAdd(&s_n[1], 1);
        if (at < kListed) s_list[at] = listing(order_key(f), id);
      }
    }
  }
  __syncthreads();
  const int n = s_n[1];
  int64_t* ids = a.top_ids + (int64_t)row * a.top;
  if (groups > kListed || n > kListed) {
    top_by_value<T>(a, x, ids, s_n);
  } else {
    for (int i = threadIdx.x; i < n; i += kLpT) {
      const uint64_t own = s_list[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += s_list[j] > own;
      if (rank < a.top) ids[rank] = (int)~(uint32_t)own;
    }
    if (n < a.top && wave == 0) {  // then the first of the -inf ones
      int filled = n;
      for (int i = 0; i < a.vocab && filled < a.top; i += 64) {
        const bool out = i + lane < a.vocab && logit<T>(x, min(i + lane, a.vocab - 1)) == -INFINITY;
        const uint64_t all = __ballot(out);
        const int to = filled + __popcll(all & ((1ull << lane) - 1));
        if (out && to < a.top) ids[to] = i + lane;
        filled += __popcll(all);
      }
    }
  }
  __syncthreads();  // the ids, written by this workgroup
  if (threadIdx.x < a.top) {
    // every place was written above; an index that comes from memory is bounded all the same
    const int64_t id = min(max(ids[threadIdx.x], (int64_t)0), (int64_t)a.vocab - 1);
    a.top_logprobs[(int64_t)row * a.top + threadIdx.x] =
        ((logit<T>(x, id) - s_f[0]) * c - s_f[1]) * kLn2;
  }
}

// values a thread: short chunks while there are few rows to fill the chip with (16 rows of
// 151936: 11.8 us either way; 64: 12.0 us, 13.0 us with 8; 32 values took as long as 16)
int elems_of(int rows, int vocab) {
  const int64_t chunks = ((int64_t)vocab + 8 * kLpT - 1) / (8 * kLpT);
  return rows * chunks <= 512 ? 8 : 16;
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
  const size_t chunks = chunks_of(rows, vocab);
  const size_t groups = top ? chunks * elems_of(rows, vocab) * kLpT / kGroup : 0;
  return rows * (chunks * sizeof(float4) + groups * 4);
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
  // a grid's second dimension of rows
  if (rows > 65535 || vocab > (1 << 21)) return HS_ERR_UNSUPPORTED;
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
  a.groups = a.chunks * elems_of(rows, vocab) * kLpT / kGroup;
  a.sums = static_cast<float4*>(workspace);
  a.most = reinterpret_cast<uint32_t*>(a.sums + (size_t)rows * a.chunks);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // 16-byte loads of every row
  const bool aligned = !(((uintptr_t)logits | (uint64_t)(logits_row_stride * esz)) & 15);
  const int e = elems_of(rows, vocab);
  if (esz == 2) {
    if (e == 16) launch<uint16_t, 16>(a, aligned, s);
    else launch<uint16_t, 8>(a, aligned, s);
  } else {
    if (e == 16) launch<float, 16>(a, aligned, s);
    else launch<float, 8>(a, aligned, s);
  }
  if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  if (esz == 2) hipLaunchKernelGGL(k_logprobs_join<uint16_t>, dim3((unsigned)rows), dim3(kLpT), 0, s, a);
  else hipLaunchKernelGGL(k_logprobs_join<float>, dim3((unsigned)rows), dim3(kLpT), 0, s, a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

}  // extern "C"
