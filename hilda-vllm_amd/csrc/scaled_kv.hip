// Store into an 8-bit (e4m3fn) paged KV cache that holds one f32 scale for every
// group of `group` consecutive slots of a block and kv head: the K/V rows of
// store_kvcache (mini_vllm/layers/attention.py:59-90) quantised against the
// values they stand with, instead of against one scale for the whole tensor.
//
// Of every (group, head) that the call writes to, over the call's rows in it:
//   a    = max |x| of the finite values
//   need = the smallest power of two >= a / 448, not below 2^-96
//   s    = need                where the call writes the group's first slot (a
//                              sequence fills its blocks in order, so what lies
//                              behind that slot is from an earlier owner) or no
//                              valid scale (finite and positive) is stored
//        = max(old, need)      otherwise; if that is above the old scale, the
//                              group's other codes c become e4m3(c * old / s)
//   code = e4m3(x / s), saturating at +-448; NaN stays NaN.
// Powers of two because a code's relative precision is the same at every scale
// (e4m3 is itself a floating type): a tighter scale would win nothing but range
// at the low end, and raising one by a power of two moves every other code of
// the group without rounding it, down to e4m3's subnormals.
//
// Launch: one workgroup per (chunk of tokens, kv head, K or V). A workgroup
// takes the tokens of its chunk whose predecessor in the call lies in another
// group, looks through the call's whole slot list for the group's other tokens
// (so the tokens of a group may stand anywhere in the call; the list is a few KB
// and read from L2), leaves the group to the workgroup of its first token, and
// otherwise does all of the group's work. No two workgroups write one group, and
// a slot that occurs twice takes the row of the higher token index, so the
// result does not depend on any order of execution.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_fp8.h"
#include "hs_model_dev.h"

namespace hs {
namespace {

constexpr int kSkT = 256;       // threads of a workgroup
constexpr int kSkMinExp = -96;  // smallest exponent of a computed scale

struct ScaledStoreArgs {
  const uint16_t* x[2];  // key, value rows
  int64_t x_st[2], x_sh[2];
  uint8_t* c[2];  // K, V cache
  float* s[2];    // their scales
  int64_t c_sb, c_st, c_sh;
  int64_t s_sb, s_sg, s_sh;
  const int32_t* slots;
  int N, chunk, block_size, num_blocks;
};

// e4m3 codes of 8 values times `inv`, or over `s` where inv is 0
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float s, float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float y = inv != 0.0f ? f[k] * inv : f[k] / s;
    w[k >> 2] |= (uint32_t)f32_to_e4m3fn_sat(y) << (8 * (k & 3));
  }
  return make_uint2(w[0], w[1]);
}

// 1 / s where that is exact (s a power of two with a normal inverse), else 0
__device__ __forceinline__ float exact_inverse(float s) {
  const uint32_t b = __float_as_uint(s), e = b >> 23;
  return ((b & 0x7fffffu) == 0 && e >= 1 && e <= 253) ? __uint_as_float((254u - e) << 23) : 0.0f;
}

template <int G>
__global__ __launch_bounds__(kSkT) void k_store_scaled(ScaledStoreArgs a) {
  constexpr int kPasses = G / 16;  // 16 rows of 16 lanes x 8 elements a pass
  __shared__ int s_owner[G];
  __shared__ int s_earlier;
  __shared__ uint32_t s_max[kSkT / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int head = blockIdx.y, kv = blockIdx.z;
  const int t0 = blockIdx.x * a.chunk;
  const uint16_t* x = a.x[kv] + head * a.x_sh[kv];
  uint8_t* cache = a.c[kv] + head * a.c_sh;

  // every wave finds the chunk's run starts for itself
  bool start = false;
  if (lane < a.chunk && t0 + lane < a.N) {
    const int slot = a.slots[t0 + lane];
    if (slot >= 0 && slot / a.block_size < a.num_blocks) {
      // groups do not cross blocks, and G divides the block size: a group is G
      // consecutive slots from a multiple of G
      start = t0 + lane == 0 || a.slots[t0 + lane - 1] < 0 ||
              a.slots[t0 + lane - 1] / G != slot / G;
    }
  }
  for (uint64_t runs = __ballot(start); runs; runs &= runs - 1) {
    const int first = t0 + __builtin_ctzll(runs);
    const int slot0 = a.slots[first] / G * G;
    __syncthreads();  // the last group's reads of the shared arrays
    for (int o = tid; o < G; o += kSkT) s_owner[o] = -1;
    if (tid == 0) s_earlier = 0;
    __syncthreads();
    bool earlier = false;
#pragma unroll 4
    for (int j = tid; j < a.N; j += kSkT) {
      const int slot = a.slots[j];
      const uint32_t o = (uint32_t)slot - (uint32_t)slot0;
      if (slot >= 0 && o < (uint32_t)G) {
        earlier |= j < first;
        atomicMax(&s_owner[o], j);
      }
    }
    if (earlier) s_earlier = 1;
    __syncthreads();
    if (s_earlier) continue;  // the workgroup of an earlier token has the group

    const int blk = slot0 / a.block_size, off0 = slot0 % a.block_size;
    uint8_t* rows = cache + (int64_t)blk * a.c_sb + (int64_t)off0 * a.c_st + 8 * (tid & 15);
    float* scale = a.s[kv] + (int64_t)blk * a.s_sb + (int64_t)(off0 / G) * a.s_sg + head * a.s_sh;
    const float old = *scale;
    uint4 raw[kPasses];
    int own[kPasses];
    uint32_t most = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      own[p] = s_owner[p * 16 + (tid >> 4)];
      raw[p] = make_uint4(0, 0, 0, 0);
      if (own[p] >= 0)
        raw[p] = *reinterpret_cast<const uint4*>(x + (int64_t)own[p] * a.x_st[kv] + 8 * (tid & 15));
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      uint16_t h[8];
      unpack8(raw[p], h);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = h[k] & 0x7fffu;  // finite bf16 values order as their bits
        if (m < 0x7f80u && m > most) most = m;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    if (lane == 0) s_max[tid >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSkT / 64; ++w) most = max(most, s_max[w]);
    // a = 1.f 2^(E - 127), 448 = 1.75 * 2^8: the exponent of the power of two
    const int E = (int)(most >> 7);
    int e = E - 135 + ((most & 0x7fu) > 0x60u ? 1 : 0);
    if (e < kSkMinExp) e = kSkMinExp;
    const float need = __uint_as_float((uint32_t)(e + 127) << 23);
    const bool fresh = s_owner[0] >= 0 || !(old > 0.0f && old < INFINITY);
    const float now = fresh ? need : fmaxf(old, need);
    const bool raise = !fresh && now > old;
    const float inv = exact_inverse(now);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      uint8_t* row = rows + (int64_t)(p * 16 + (tid >> 4)) * a.c_st;
      if (own[p] >= 0) {
        uint16_t h[8];
        float f[8];
        unpack8(raw[p], h);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = bf(h[k]);
        *reinterpret_cast<uint2*>(row) = encode8(f, now, inv);
      } else if (raise) {
        const uint2 c = *reinterpret_cast<const uint2*>(row);
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t b = (k < 4 ? c.x : c.y) >> (8 * (k & 3));
          f[k] = __builtin_amdgcn_cvt_f32_fp8((int)b, 0) * old;
        }
        *reinterpret_cast<uint2*>(row) = encode8(f, now, inv);
      }
    }
    if (tid == 0) *scale = now;  // every thread read the old one before the last barrier
  }
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" int hs_store_kvcache_scaled(
    const void* key, int64_t key_stride_tok, int64_t key_stride_head, const void* value,
    int64_t value_stride_tok, int64_t value_stride_head, void* k_cache, void* v_cache,
    int64_t cache_stride_block, int64_t cache_stride_tok, int64_t cache_stride_head,
    float* k_scales, float* v_scales, int64_t scale_stride_block, int64_t scale_stride_group,
    int64_t scale_stride_head, int group, const int32_t* slot_mapping, int num_tokens,
    int num_kv_heads, int head_dim, int block_size, int num_blocks, void* stream) {
  if (num_tokens == 0) return HS_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scales || !v_scales || !slot_mapping)
    return HS_ERR_INVALID;
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks <= 0 || group <= 0 ||
      block_size % group)
    return HS_ERR_INVALID;
  if (head_dim != 128) return HS_ERR_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128 && group != 256) return HS_ERR_UNSUPPORTED;
  if (num_kv_heads > 65535) return HS_ERR_UNSUPPORTED;
  // rows are read 16 bytes and written 8 bytes a lane
  if ((key_stride_tok | key_stride_head | value_stride_tok | value_stride_head) & 7)
    return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)key | (uintptr_t)value) & 15) return HS_ERR_UNSUPPORTED;
  if ((cache_stride_block | cache_stride_tok | cache_stride_head) & 7) return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 7) return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3) return HS_ERR_UNSUPPORTED;
  ScaledStoreArgs a;
  a.x[0] = static_cast<const uint16_t*>(key);
  a.x[1] = static_cast<const uint16_t*>(value);
  a.x_st[0] = key_stride_tok;
  a.x_st[1] = value_stride_tok;
  a.x_sh[0] = key_stride_head;
  a.x_sh[1] = value_stride_head;
  a.c[0] = static_cast<uint8_t*>(k_cache);
  a.c[1] = static_cast<uint8_t*>(v_cache);
  a.s[0] = k_scales;
  a.s[1] = v_scales;
  a.c_sb = cache_stride_block;
  a.c_st = cache_stride_tok;
  a.c_sh = cache_stride_head;
  a.s_sb = scale_stride_block;
  a.s_sg = scale_stride_group;
  a.s_sh = scale_stride_head;
  a.slots = slot_mapping;
  a.N = num_tokens;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  // Decode rows start a group each, so a workgroup takes one token of a small call
  // (64 tokens one by one: 16 workgroups each, all at once); prompts fill groups,
  // so a chunk of their tokens holds a start or two
  a.chunk = 1;
  while (a.chunk < 32 && num_tokens > 64 * a.chunk) a.chunk *= 2;
  const dim3 grid((unsigned)((num_tokens + a.chunk - 1) / a.chunk), (unsigned)num_kv_heads, 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (group) {
    case 32: hipLaunchKernelGGL(k_store_scaled<32>, grid, dim3(kSkT), 0, st, a); break;
    case 64: hipLaunchKernelGGL(k_store_scaled<64>, grid, dim3(kSkT), 0, st, a); break;
    case 128: hipLaunchKernelGGL(k_store_scaled<128>, grid, dim3(kSkT), 0, st, a); break;
    default: hipLaunchKernelGGL(k_store_scaled<256>, grid, dim3(kSkT), 0, st, a); break;
  }
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}
