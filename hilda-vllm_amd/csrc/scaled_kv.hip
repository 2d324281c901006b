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
// Launch: a workgroup per (chunk of tokens, kv head, K or V). It takes the tokens of its
// chunk whose predecessor in the call lies in another group, looks through the
// call's whole slot list for the group's other tokens (so the tokens of a group may
// stand anywhere in the call; read from L2, so that the reads grow with the square of the
// call's tokens: 4000 tokens of 8 heads 13.6 us, 8000 25.8 us, 24000 121 us, five times
// their bytes' time), leaves the group to
// the workgroup of its first token, and otherwise does all of the group's work, the rows
// held in registers from their maximum to their codes. No two workgroups write one group
// and head, and a slot that occurs twice takes the row of the higher token index, so the
// result does not depend on any order of execution. The call is bound by latency - the
// list, the rows, the codes, one after the other - and the rows that follow the first
// token in the call, which are nearly always the group's, are loaded during the search.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_fp8.h"
#include "hs_model_dev.h"

namespace hs {
namespace {

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

// e4m3 codes of 8 values times `inv`, or over `s` where inv is 0, that are at most 448, or
// infinities, which saturate (before the conversion: 448 s may be past f32's largest), or
// NaN (v_cvt_pk_fp8_f32: round to nearest even, the same codes as f32_to_e4m3fn_sat's for
// all of these; 2 instructions a value against about 25)
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float s, float inv) {
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    y[k] = inv != 0.0f ? f[k] * inv : f[k] / s;
    if (fabsf(f[k]) == INFINITY) y[k] = copysignf(448.0f, f[k]);
  }
  int w[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], w[h], false);
    w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w[h], true);
  }
  return make_uint2((uint32_t)w[0], (uint32_t)w[1]);
}

// 1 / s where that is exact (s a power of two with a normal inverse), else 0
__device__ __forceinline__ float exact_inverse(float s) {
  const uint32_t b = __float_as_uint(s), e = b >> 23;
  return ((b & 0x7fffffu) == 0 && e >= 1 && e <= 253) ? __uint_as_float((254u - e) << 23) : 0.0f;
}

// threads of a group's workgroup: 16 lanes x 8 elements to a row, 2 or 4 rows each
constexpr int threads_of(int G) { return G <= 64 ? 256 : 4 * G; }

template <int G>
__global__ __launch_bounds__(threads_of(G)) void k_store_scaled(ScaledStoreArgs a) {
  constexpr int kT = threads_of(G), kWaves = kT / 64;
  constexpr int kRowsAPass = kT / 16, kPasses = G / kRowsAPass;
  __shared__ int s_owner[G];
  __shared__ int s_earlier;
  __shared__ uint32_t s_max[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, col = 8 * (tid & 15);
  const int head = blockIdx.y, t0 = blockIdx.x * a.chunk;
  const int v = blockIdx.z & 1, odd = blockIdx.z >> 1;  // K or V; which of the chunk's starts
  const uint16_t* x = a.x[v] + head * a.x_sh[v] + col;

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
  // the chunk's starts in turn, or (two workgroups to a chunk) every other one
  uint64_t runs = __ballot(start);
  if (odd) runs &= runs - 1;
  for (; runs; runs &= runs - 1, runs = gridDim.z == 4 ? runs & (runs - 1) : runs) {
    const int first = t0 + __builtin_ctzll(runs);
    const int slot1 = a.slots[first], slot0 = slot1 / G * G;
    const int blk = slot0 / a.block_size, off0 = slot0 % a.block_size;
    const int64_t at = (int64_t)blk * a.c_sb + (int64_t)off0 * a.c_st + (int64_t)head * a.c_sh + col;
    const int64_t sat = (int64_t)blk * a.s_sb + (int64_t)(off0 / G) * a.s_sg + (int64_t)head * a.s_sh;
    float* scale = a.s[v] + sat;
    const float old = *scale;
    uint4 raw[kPasses];
    int own[kPasses];
    auto load = [&](int p) {
      raw[p] = make_uint4(0, 0, 0, 0);
      if (own[p] >= 0)
        raw[p] = *reinterpret_cast<const uint4*>(x + (int64_t)own[p] * a.x_st[v]);
    };
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int slot = slot0 + p * kRowsAPass + (tid >> 4), t = first + slot - slot1;
      own[p] = slot >= slot1 && t < a.N && a.slots[t] == slot ? t : -1;
      load(p);
    }
    __syncthreads();  // the last group's reads of the shared arrays
    for (int o = tid; o < G; o += kT) s_owner[o] = -1;
    if (tid == 0) s_earlier = 0;
    __syncthreads();
    bool earlier = false;
    auto look = [&](int j, int slot) {
      const uint32_t o = (uint32_t)slot - (uint32_t)slot0;
      if (j < a.N && slot >= 0 && o < (uint32_t)G) {
        earlier |= j < first;
        atomicMax(&s_owner[o], j);
      }
    };
    if (a.N <= kT) {
      look(tid, a.slots[min(tid, a.N - 1)]);
    } else {
      for (int j = tid; j < a.N; j += 8 * kT) {
        int slot[8];  // every load of the round before the first wait
#pragma unroll
        for (int i = 0; i < 8; ++i) slot[i] = a.slots[min(j + i * kT, a.N - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) look(j + i * kT, slot[i]);
      }
    }
    if (earlier) s_earlier = 1;
    __syncthreads();
    if (s_earlier) continue;  // the workgroup of an earlier token has the group

    uint32_t most = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int owner = s_owner[p * kRowsAPass + (tid >> 4)];
      if (owner != own[p]) {
        own[p] = owner;
        load(p);
      }
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
    for (int w = 0; w < kWaves; ++w) most = max(most, s_max[w]);
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
      uint8_t* row = a.c[v] + at + (int64_t)(p * kRowsAPass + (tid >> 4)) * a.c_st;
      if (own[p] >= 0) {
        uint16_t h[8];
        float f[8];
        unpack8(raw[p], h);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = bf(h[k]);  // |x| <= 448 s by the choice of s
        *reinterpret_cast<uint2*>(row) = encode8(f, now, inv);
      } else if (raise) {
        const uint2 c = *reinterpret_cast<const uint2*>(row);
        // the new scale is a power of two from 2^-96 to 2^120, so the quotient of the
        // scales rounds only where no code survives it; 448 old may overflow
        const float shrink = old * inv;
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t b = (k < 4 ? c.x : c.y) >> (8 * (k & 3));
          f[k] = __builtin_amdgcn_cvt_f32_fp8((int)b, 0) * shrink;
        }
        *reinterpret_cast<uint2*>(row) = encode8(f, 1.0f, 1.0f);
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
  // Decode rows start a group each, so a workgroup takes one token of a small call;
  // prompts fill groups, and a chunk of 32 of their tokens holds a start or, with groups
  // of 32, two for a workgroup each (2003 tokens: 15 us, 17.5 us with one workgroup;
  // chunks of 16 start twice as many workgroups, half of them for nothing: 4000 tokens
  // 20.5 us against 13.7 us)
  a.chunk = 1;
  while (a.chunk < 32 && num_tokens > 64 * a.chunk) a.chunk *= 2;
  const dim3 grid((unsigned)((num_tokens + a.chunk - 1) / a.chunk), (unsigned)num_kv_heads,
                  a.chunk > 1 && group == 32 ? 4 : 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (group) {
    case 32: hipLaunchKernelGGL(k_store_scaled<32>, grid, dim3(threads_of(32)), 0, st, a); break;
    case 64: hipLaunchKernelGGL(k_store_scaled<64>, grid, dim3(threads_of(64)), 0, st, a); break;
    case 128: hipLaunchKernelGGL(k_store_scaled<128>, grid, dim3(threads_of(128)), 0, st, a); break;
    default: hipLaunchKernelGGL(k_store_scaled<256>, grid, dim3(threads_of(256)), 0, st, a); break;
  }
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}
