// Projections of rows in 8 bits (hs_fp8_rows.h) by e4m3 weights with an f32 scale for every
// block of 128 x 128 on gfx950:
//   y[r, n] = sum_b sx[r, b] sw[n / 128, b] sum_{k in block b} cx[r, k] cw[n, k]
// with f32 accumulation, y in bf16; SwiGLU: silu(gate) * up of a [2F, K] weight, rounded
// once to bf16 or, with scales, to 8 bits.
//
// One 16x16x128 MFMA is one block of 128 inputs: its products leave in an accumulator of
// their own, with sx applied by the instruction as the operand's block exponent, and sw, the
// same for 128 features, multiplies them as they are added (one fused multiply-add an
// element, which the matrix unit's time covers). All sums are kept in units of 2^17, the
// weight operand's block exponent: 128 products of values up to 448 * 2^120, past bf16's
// largest, by codes up to 448 stay below 2^128 then, so that what sw brings back into range
// has not become an infinity before. The other end has room for it: sums before sw are multiples
// of 2^-132 instead of 2^-149.
//
// What the matrix unit adds is not quite f32: the products of 8 neighbouring inputs (the bytes
// of two registers) are added as multiples of 2^(e - 13), e the largest sum of two of their
// exponents, and what lies below is dropped; the 16 such sums of a block and the blocks' sums
// are added in f32. A block's relative error from it is 1.4e-5 by norm where the channels are
// alike and 7.3e-5 where they spread by e^1.5, at most a tenth of bf16's rounding. (The older
// 16x16x32 form adds alike, with the same two errors, at half the rate.)
//
// Times at the kernels are a trace's averages, over three inputs in turn; where variants are
// compared, each is one call among others of a replayed graph, the launch's gap included.
//
// A weight is kept as 16-feature tiles by 128-input steps, 2 KB each: lane l holds inputs
// 64 h + 16 (l / 16) .. + 15 of feature l % 16 as the 16 bytes at (h, l), h = 0 and 1. The
// order of the inputs within a step is free as long as the rows are read in the same one.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/hilda_spec.h"
#include "hs_fp8_rows.h"

namespace hs {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kStep = kFp8Group;  // inputs of a step

struct Fp8Args {
  const uint8_t* x;   // codes, or bf16 (k_fp8_rows)
  int64_t xs;
  const uint8_t* xe;  // exponent bytes [rows][xes]
  int64_t xes;
  const uint4* w;     // [tiles][steps][2][64]
  const float* sc;    // [tiles][steps]
  int rows, K, N;     // N: output features
  int steps;
  int units;          // 16-feature tiles of the output
  int up;             // first tile of the up rows (SwiGLU)
  uint16_t* y;        // bf16, or codes
  int64_t ys;
  int wide;           // y and ys in 16-byte pieces
  uint8_t* ye;        // exponent bytes of the codes
  int64_t yes;
  float* part;        // [split][rows][tiles * 16]
  int split_steps, nsplit;
  int cols, rowtiles;  // workgroups of the large tiles
};

__device__ __forceinline__ i32x8_t operand(uint4 a, uint4 b) {
  return i32x8_t{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

constexpr float kUnit = 1 << 17;  // of the sums
constexpr int kPerUnit = 127 - 17;  // the weights' block exponent

// 16 features by 16 rows, one step; the lane's row's exponent is byte B of xe
template <int B>
__device__ __forceinline__ f32x4_t mfma(i32x8_t w, i32x8_t x, uint32_t xe) {
  const f32x4_t zero = {0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, kPerUnit, B, (int)xe);
}

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}

// (the reciprocal instruction is good to one unit in f32's last place, but flushes what is below
// f32's normal numbers: of (1 + e) / 16 it stays above them up to f32's largest e)
__device__ __forceinline__ float silu(float g) {
  return g * 0.0625f * __builtin_amdgcn_rcpf(fmaf(__expf(-g), 0.0625f, 0.0625f));
}

// of sums
__device__ __forceinline__ float swiglu(float gate, float up) {
  return silu(gate * kUnit) * (up * kUnit);
}
template <bool kGate>
__device__ __forceinline__ uint16_t result(float v, float up) {
  return to_bf(kGate ? swiglu(v, up) : v * kUnit);
}

// 8 features of a row, n a multiple of 8; wide: outputs in 16-byte pieces
__device__ __forceinline__ void store8(const Fp8Args& a, int64_t row, int n, uint4 v) {
  uint16_t* y = a.y + row * a.ys + n;
  if (a.wide && n + 8 <= a.N) {
    *reinterpret_cast<uint4*>(y) = v;
    return;
  }
  uint16_t h[8];
  unpack8(v, h);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (n + j < a.N) y[j] = h[j];
  }
}

// The lane's 32 values of a bf16 row's step (inputs 64 h + 16 g .. + 15, h = 0 and 1) as codes
// under the scale of the step's 128, which the four lanes of a row share; its exponent's byte.
__device__ __forceinline__ i32x8_t row_codes(const uint4 (&raw)[4], uint32_t& byte) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  uint32_t v[16] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w,
                    raw[2].x, raw[2].y, raw[2].z, raw[2].w, raw[3].x, raw[3].y, raw[3].z, raw[3].w};
  // the bits of |v| order bf16 numbers
  auto most_of = [&] {
    u16x2_t most = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, v[i] & 0x7fff7fffu));
    uint32_t m = max((uint32_t)most[0], (uint32_t)most[1]);
    const auto p = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max(p[0], p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return max(q[0], q[1]);
  };
  uint32_t most = most_of();
  if (__any(most >= 0x7f80u)) {  // NaN and infinities take no part in the scale, and are NaN
    uint32_t nan[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      nan[i] = ((v[i] & 0x7f80u) == 0x7f80u ? 0x7fc0u : 0) |
               ((v[i] & 0x7f800000u) == 0x7f800000u ? 0x7fc00000u : 0);
      if (nan[i] & 0xffffu) v[i] &= 0xffff0000u;
      if (nan[i] >> 16) v[i] &= 0xffffu;
    }
    most = most_of();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] |= nan[i];
  }
  byte = scale_byte(most << 16);
  return scaled_codes32(v, byte);
}

// RT * 16 rows a workgroup. W: its waves, which share out the steps of its TN weight tiles
// (with SwiGLU half of them gate and half up tiles) and join their sums in LDS. kBf16: the
// rows are bf16 and go to 8 bits here, in every workgroup. Bound by the weights' stream: 16
// rows of 4096 by 151936 features 105 us (5.9 TB/s), by 2 x 12288 features 18.8 us (5.4 TB/s),
// one row by 4096 features 5.7 us, of which the launch's start and end are 2.
template <int W, int TN, int RT, bool kGate, bool kBf16>
__global__ __launch_bounds__(64 * W) void k_fp8_rows(Fp8Args a) {
  constexpr int kOut = kGate ? TN / 2 : TN;
  __shared__ float s_part[W][TN][16 * RT][16];  // [wave][tile][row][feature]
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u0 = blockIdx.x * kOut, r0 = blockIdx.y * 16 * RT;
  int tile[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) tile[t] = min(u0 + t % kOut, a.units - 1) + t / kOut * a.up;
  f32x4_t y[TN][RT];
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int r = 0; r < RT; ++r) y[t][r] = f32x4_t{0, 0, 0, 0};
  constexpr int kRaw = kBf16 ? 4 : 2;  // 16-byte pieces of a row's step in a lane
  struct Step {
    uint4 w[TN][2], x[RT][kRaw];
    uint32_t e[RT];
    float sc[TN];
  };
  auto load = [&](int step, Step& s) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int64_t at = (int64_t)tile[t] * a.steps + step;
      s.w[t][0] = load_once(a.w + at * 128 + lane);
      s.w[t][1] = load_once(a.w + at * 128 + 64 + lane);
      s.sc[t] = a.sc[at];
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = r0 + 16 * r + m;
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        const int k = kStep * step + 64 * (2 * i / kRaw) + 16 * g + (kBf16 ? 8 * (i & 1) : 0);
        s.x[r][i] = make_uint4(0, 0, 0, 0);
        if (row < a.rows && k < a.K)
          s.x[r][i] = *reinterpret_cast<const uint4*>(a.x + ((int64_t)row * a.xs + k) *
                                                                (kBf16 ? 2 : 1));
      }
      if (!kBf16) s.e[r] = a.xe[(int64_t)min(row, a.rows - 1) * a.xes + step];
    }
  };
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      uint32_t e = s.e[r];
      i32x8_t x;
      if constexpr (kBf16) x = row_codes(s.x[r], e);
      else x = operand(s.x[r][0], s.x[r][1]);
#pragma unroll
      for (int t = 0; t < TN; ++t)
        y[t][r] += s.sc[t] * mfma<0>(operand(s.w[t][0], s.w[t][1]), x, e);
    }
  };
  // one step's loads at a time: many waves hide them as well as many loads (16 waves 5.0 us, 8
  // waves with four steps' loads 5.1 us for a row of 4096, 4096 features)
  for (int step = wave; step < a.steps; step += W) {
    Step s;
    load(step, s);
    multiply(s);
  }
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int r = 0; r < RT; ++r)
      *reinterpret_cast<f32x4_t*>(&s_part[wave][t][16 * r + m][4 * g]) = y[t][r];
  __syncthreads();
  const int rows = min(16 * RT, a.rows - r0);
  for (int e = threadIdx.x; e < 16 * rows * kOut; e += 64 * W) {
    const int n = e & 15, t = (e >> 4) % kOut, r = (e >> 4) / kOut;
    float v = 0.0f, up = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      v += s_part[w][t][r][n];
      if (kGate) up += s_part[w][kOut + t][r][n];
    }
    const int col = (u0 + t) * 16 + n;
    if (a.part) {
      if (u0 + t >= a.units) continue;
      const int64_t width = (int64_t)a.units * (kGate ? 32 : 16);
      a.part[(r0 + r) * width + col] = v;
      if (kGate) a.part[(r0 + r) * width + (int64_t)a.units * 16 + col] = up;
    } else if (col < a.N) {
      a.y[(int64_t)(r0 + r) * a.ys + col] = result<kGate>(v, up);
    }
  }
}

// ---- many rows: 256 features by 256 rows a workgroup -----------------------------------

constexpr int kBig = 256;                   // features and rows of a workgroup
constexpr int kBigThreads = 512;            // 4 waves over the features, 2 over the rows
constexpr int kPast = INT32_MAX;            // a byte offset past any buffer: reads zeros
constexpr int kRange = INT32_MAX - 255;
constexpr int kStage = kBig * kStep;        // bytes of a step's rows, and of its weights
constexpr int kChunk = 64;                  // steps whose exponents and scales are held
// shared memory: two stages of rows, two of weights, the chunk's exponents and scales
constexpr int kAtW = 2 * kStage, kAtE = 4 * kStage, kAtS = kAtE + kChunk * kBig;
constexpr int kBigBytes = kAtS + kChunk * 4 * 16;

// 16 bytes a lane from a buffer straight to LDS, at lds + 16 lane. The compiler does not see
// the write: the wait before the barrier behind a step covers it. (Through the builtin it
// would wait for the load before the next read of any shared memory.) kOffset is added to
// both sides.
template <int kOffset = 0>
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t from, int offset, int at,
                                         uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\t"
               "buffer_load_dwordx4 %1, %2, %3 offen offset:%4 lds"
               :: "s"(lds), "v"(offset), "s"(from), "s"(at), "n"(kOffset)
               : "memory");
}
// 4 bytes a lane, at lds + 4 lane
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t from, int offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(lds), "v"(offset), "s"(from)
               : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
// waits for the wave's LDS traffic and all but its last kLoads loads, then for the other waves
template <int kLoads>
__device__ __forceinline__ void step_barrier() {
  static_assert(kLoads < 16, "the count's low four bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | kLoads);  // vmcnt(kLoads) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int I>
using Index = std::integral_constant<int, I>;

// the 16-byte piece of a row's step that lies at piece p of the row in LDS, and back
__device__ __forceinline__ int swizzle(int row, int p) { return p ^ (row & 7); }

// The end of a workgroup of WF x WR waves, each with 16 FT features (with SwiGLU half gate and
// half up) by 16 RT rows, from its first output tile u0 and row r0, `high` of its rows in the
// matrix: outputs through shared memory, so that whole lines go out.
template <int kEpilogue, int FT, int RT, int WF, int WR>
__device__ __forceinline__ void finish(const Fp8Args& a, f32x4_t (&acc)[FT][RT], uint8_t* s_bytes,
                                       int u0, int r0, int high) {
  constexpr bool kGate = kEpilogue != HS_LINEAR_PLAIN, kEight = kEpilogue == HS_LINEAR_SWIGLU_FP8;
  constexpr int OT = kGate ? FT / 2 : FT;  // output tiles of a wave
  constexpr int kRows = 16 * RT * WR, kTileRows = 16 * RT;
  constexpr int kRow = 16 * OT * WF * (kEight ? 1 : 2), kPitch = kRow + 16;  // bytes of a row
  static_assert(!kEight || kRow == kFp8Group, "a row's outputs are one group");
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wf = wave % WF, first = kTileRows * (wave / WF) + m;
  uint32_t bytes[RT];  // exponents of the rows' codes
  if constexpr (kEight) {
    uint32_t* s_max = reinterpret_cast<uint32_t*>(s_bytes + kRows * kPitch);  // [wf][row]
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float most = 0;
#pragma unroll
      for (int f = 0; f < OT; ++f) {
        float here = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[f][t][j] = swiglu(acc[f][t][j], acc[f + OT][t][j]);
          here = fmaxf(here, fabsf(acc[f][t][j]));  // (passes over NaN)
        }
        most = fmaxf(most, u0 + OT * wf + f < a.units ? here : 0.0f);
      }
      if (__any(most == __builtin_inff())) {  // the scale is that of the finite values
        uint32_t bits = 0;
#pragma unroll
        for (int f = 0; f < OT; ++f)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (u0 + OT * wf + f < a.units) bits = max(bits, finite_bits(acc[f][t][j]));
            acc[f][t][j] = nan_unless_finite(acc[f][t][j]);
          }
        most = __uint_as_float(bits);
      }
      most = quad_max(most);
      if (g == 0) s_max[wf * kRows + first + 16 * t] = __float_as_uint(most);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      uint32_t most = 0;
#pragma unroll
      for (int w = 0; w < WF; ++w) most = max(most, s_max[w * kRows + first + 16 * t]);
      bytes[t] = scale_byte(most);
      const float inv = scale_inverse(bytes[t]);
#pragma unroll
      for (int f = 0; f < OT; ++f) {
        const float v[4] = {acc[f][t][0], acc[f][t][1], acc[f][t][2], acc[f][t][3]};
        *reinterpret_cast<uint32_t*>(s_bytes + (first + 16 * t) * kPitch + 16 * (OT * wf + f) +
                                     4 * g) = finite_codes4(v, inv);
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int f = 0; f < OT; ++f) {
        uint16_t v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = result<kGate>(acc[f][t][j], kGate ? acc[f + FT - OT][t][j] : 0.0f);
        *reinterpret_cast<uint2*>(s_bytes + (first + 16 * t) * kPitch + 32 * (OT * wf + f) +
                                  8 * g) =
            make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
      }
    }
  }
  __syncthreads();
  constexpr int kLanes = kRow / 16;  // of a row
#pragma unroll
  for (int i = 0; i < kRows * kLanes / (64 * WF * WR); ++i) {
    const int e = (i * WF * WR + wave) * 64 + lane, in = e / kLanes, at = e % kLanes;
    const int64_t row = r0 + in;
    if (in >= high) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(s_bytes + in * kPitch + 16 * at);
    if constexpr (kEight) {
      const int n = 16 * (u0 + at);
      if (n < a.N)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.y) + row * a.ys + n) = v;
    } else {
      store8(a, row, 16 * u0 + 8 * at, v);
    }
  }
  if constexpr (kEight) {
    if (wf == 0 && g == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if (first + 16 * t < high)
          a.ye[(int64_t)(r0 + first + 16 * t) * a.yes + u0 / 8] = (uint8_t)bytes[t];
      }
    }
  }
}

// The workgroup's place in the order of the tiles: each XCD (workgroups go to them in turn)
// has a stretch of it, so that what its L2 holds is shared: 8 row tiles to a column.
__device__ __forceinline__ int order_of(int total) {
  const int id = blockIdx.x, x = id & 7, q = total >> 3, r = total & 7;
  return x * q + min(x, r) + (id >> 3);
}
__device__ __forceinline__ void place_of(const Fp8Args& a, int o, int& col, int& row) {
  const int group = o / (8 * a.cols), in = o % (8 * a.cols);
  const int tall = min(8, a.rowtiles - 8 * group);
  row = 8 * group + in % tall;
  col = in / tall;
}

// A chunk's exponents to shared memory at `e`, a word of four steps a row, [four steps][row], and
// its weights' scales at `s`, [gate, up][step][output tile]: SLOTS weight tiles from output tile
// u0, ROWS rows from r0 (the last ones are `high`), of WAVES waves. Past the last step both are
// zeros, but for bytes of a word that it ends in (trim).
template <bool kGate, int ROWS, int SLOTS, int WAVES>
__device__ __forceinline__ void load_chunk(const Fp8Args& a, int first, int u0, int r0, int high,
                                           uint32_t e, uint32_t s) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto eb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.xe + r0 * a.xes), 0, (high - 1) * (int)a.xes + (a.steps + 3) / 4 * 4,
      0x00027000);
  static_assert(ROWS / 4 % WAVES == 0, "");
#pragma unroll
  for (int i = 0; i < ROWS / 4 / WAVES; ++i) {
    const int j = i * WAVES + wave, d = 64 * j + lane, step = first + d / ROWS * 4;
    load_lds4(eb, step < a.steps ? d % ROWS * (int)a.xes + step : kPast, e + 256 * j);
  }
  constexpr int OUT = kGate ? SLOTS / 2 : SLOTS;
#pragma unroll
  for (int i = 0; i < (SLOTS + WAVES - 1) / WAVES; ++i) {
    const int j = i * WAVES + wave;
    if (SLOTS % WAVES && j >= SLOTS) break;
    const int half = kGate ? j / OUT : 0, d = 64 * (j - half * OUT) + lane;
    const int step = first + d / OUT;
    const auto sb = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(a.sc + (u0 + half * (int64_t)a.up) * a.steps), 0, kRange, 0x00027000);
    const int tile = min(d % OUT, a.units - 1 - u0);
    load_lds4(sb, step < a.steps ? 4 * (tile * a.steps + step) : kPast, s + 256 * j);
  }
}
// after the chunk has landed and all waves know: zeros for what follows the last step in its word
template <int ROWS>
__device__ __forceinline__ void trim_chunk(const Fp8Args& a, int first, uint8_t* e) {
  const int left = a.steps - first;
  if (left >= kChunk || left % 4 == 0) return;
  if (threadIdx.x < ROWS)
    reinterpret_cast<uint32_t*>(e)[left / 4 * ROWS + threadIdx.x] &= (1u << 8 * (left % 4)) - 1;
  __syncthreads();
}
// N consecutive scales of a wave's tiles at p
template <int N>
__device__ __forceinline__ void read_scales(const uint8_t* p, float* out) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  if constexpr (N == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    out[0] = v.x; out[1] = v.y; out[2] = v.z; out[3] = v.w;
  } else if constexpr (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    out[0] = v.x; out[1] = v.y;
  } else {
    out[0] = *reinterpret_cast<const float*>(p);
  }
}
__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// A wave has 64 features by 128 rows. Its step is 32 products of 32 cycles, two waves to a SIMD:
// 2048 cycles of the matrix unit, beside 256 KB to and from LDS (half of its 256 bytes a cycle)
// and 64 KB from L2 (half of a CU's 64 bytes a cycle). Measured are 2300 to 2500. 4096 rows of
// 4096 by 2 x 12288 features with 8-bit SwiGLU take 342 to 359 us among others (2300 to 2410
// TFLOP/s; in two traces 384 and 407), of which the first loads are 26 and the ends 28 (the
// exponential and the quotient); 325 us if all operands are zeros, for the card's power sets the
// clock.
template <int kEpilogue>
__global__ __launch_bounds__(kBigThreads, 2) void k_fp8_big(Fp8Args a) {
  constexpr bool kGate = kEpilogue != HS_LINEAR_PLAIN;
  extern __shared__ uint4 s_all[];  // [stage][x: row, piece | w: tile, half, lane]
  uint8_t* s_bytes = reinterpret_cast<uint8_t*>(s_all);
  const uint32_t lds = lds_address(s_all);
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wf = wave & 3, wr = wave >> 2;
  int u0, r0;
  place_of(a, order_of(a.cols * a.rowtiles), u0, r0);
  r0 *= kBig;
  u0 *= kGate ? 8 : 16;
  auto tile_of = [&](int slot) {  // weight tile of one of the workgroup's 16 slots
    const int f = slot & 3;
    const int u = kGate ? u0 + (slot >> 2) * 2 + (f & 1) : u0 + slot;
    return min(u, a.units - 1) + (kGate && f >= 2 ? a.up : 0);
  };
  // this wave's loads: 32 rows and two weight tiles
  const int piece = swizzle(lane >> 3, lane & 7);
  const int64_t tile_bytes = (int64_t)a.steps * (16 * kStep);
  uint8_t* wp = reinterpret_cast<uint8_t*>(const_cast<uint4*>(a.w));
  uint8_t* xp = const_cast<uint8_t*>(a.x + (int64_t)r0 * a.xs);
  uint8_t* wp0 = wp + tile_of(2 * wave) * tile_bytes;
  uint8_t* wp1 = wp + tile_of(2 * wave + 1) * tile_bytes;
  const int high = min(a.rows - r0, kBig);  // rows of the tile
  const int x_range = (high - 1) * (int)a.xs + a.K;  // rows behind the last one read zeros
  // A wave's eight loads of a step: i 0 and 1 the lower 64 rows of each half, 2 to 5 weights
  // (group A), 6 and 7 the upper rows (group B). Past the last step none reads memory.
  const int row0 = (wave >> 2) * 128 + (wave & 3) * 16 + (lane >> 3);
  auto load = [&](int step, auto index) {
    constexpr int i = decltype(index)::value;
    const uint32_t to = lds + (step & 1) * kStage;
    if constexpr (i < 2 || i >= 6) {
      constexpr int kRow = i < 2 ? 8 * i : 64 + 8 * (i - 6);
      const auto b = __builtin_amdgcn_make_buffer_rsrc(xp, 0, x_range, 0x00027000);
      const int k = kStep * step + 16 * piece;
      const int at = (row0 + kRow) * (int)a.xs + k;
      load_lds(b, k < a.K ? at : kPast, 0,
               to + ((wave >> 2) * 128 + (wave & 3) * 16 + kRow) * kStep);
    } else {
      const auto b = __builtin_amdgcn_make_buffer_rsrc(i < 4 ? wp0 : wp1, 0,
                                                       step < a.steps ? kRange : 0, 0x00027000);
      load_lds<1024 * (i & 1)>(b, 16 * lane, 16 * kStep * step,
                               to + kAtW + (wave * 4 + (i & 2 ? 0 : 2)) * 1024);
    }
  };
  auto load_a = [&](int step) {
    load(step, Index<0>()); load(step, Index<1>()); load(step, Index<2>()); load(step, Index<3>());
    load(step, Index<4>()); load(step, Index<5>());
  };
  auto load_b = [&](int step) { load(step, Index<6>()); load(step, Index<7>()); };

  // operands from LDS
  const uint8_t* sx0 = s_bytes + (128 * wr + m) * kStep + 16 * swizzle(m, g);
  const uint8_t* sx1 = s_bytes + (128 * wr + m) * kStep + 16 * swizzle(m, 4 + g);
  const uint8_t* sw0 = s_bytes + kAtW + wf * 4 * 2048 + 16 * lane;
  const uint8_t* se0 = s_bytes + kAtE + 4 * (128 * wr + m);
  auto read_x = [&](int step, int t) {
    const int at = (step & 1) * kStage + 16 * t * kStep;
    return operand(*reinterpret_cast<const uint4*>(sx0 + at),
                   *reinterpret_cast<const uint4*>(sx1 + at));
  };
  auto read_w = [&](int step, int f) {
    const uint8_t* p = sw0 + (step & 1) * kStage + 2048 * f;
    return operand(*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + 1024));
  };
  auto read_e = [&](int quad, int t) {
    return *reinterpret_cast<const uint32_t*>(se0 + quad * 4 * kBig + 64 * t);
  };

  f32x4_t acc[4][8], part[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    part[f] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[f][t] = f32x4_t{0, 0, 0, 0};
  }
  // the scales of the wave's tiles
  const uint8_t* ss = s_bytes + kAtS + 4 * (kGate ? 2 : 4) * wf;
  auto read_scale = [&](int in_chunk, float (&v)[4]) {
    if constexpr (kGate) {
      read_scales<2>(ss + 32 * in_chunk, v);
      read_scales<2>(ss + 32 * kChunk + 32 * in_chunk, v + 2);
    } else {
      read_scales<4>(ss + 64 * in_chunk, v);
    }
  };
  auto chunk = [&](int first) {
    load_chunk<kGate, kBig, 16, 8>(a, first, u0, r0, high, lds + kAtE, lds + kAtS);
  };
  chunk(0);
  load_a(0);
  load_b(0);
  load_a(1);
  load_b(1);
  step_barrier<8>();
  trim_chunk<kBig>(a, 0, s_bytes + kAtE);
  i32x8_t x[3], w[4];
  uint32_t e[3];
  x[2] = read_x(0, 0);
#pragma unroll
  for (int f = 0; f < 4; ++f) w[f] = read_w(0, f);
  float scale[4] = {0, 0, 0, 0};
  // One step, in an order that the compiler keeps: 32 products, each added three products
  // later; a row tile's operand is read one tile ahead. At the first barrier the lower rows
  // and the weights of the step have been read (by all waves): the step after the next loads
  // into their place (group A). At the second the upper rows have been, too (group B): the
  // next step's first operands are read in place of those used up. What a barrier waits for
  // was loaded one and a half steps before.
  auto one = [&](int step, int quad, auto quarter) {
    constexpr int kQ = decltype(quarter)::value;
    constexpr int kReg[8] = {2, 0, 1, 0, 1, 2, 0, 1};  // of the row tiles
    float before[4], next[4];
    read_scale(step & (kChunk - 1), next);
#pragma unroll
    for (int f = 0; f < 4; ++f) before[f] = scale[f];
    // tile and weight of product i: the last two row tiles by weights
    auto tile = [](int i) { return i < 24 ? i >> 2 : 6 + (i & 1); };
    auto weight = [](int i) { return i < 24 ? i & 3 : (i - 24) >> 1; };
    auto read = [&](int t) {
      x[kReg[t]] = read_x(kQ, t);
      e[kReg[t]] = read_e(quad, t);
    };
    auto product = [&](int i) {
      const int t = tile(i), f = weight(i), r = kReg[t];
      part[i & 3] = mfma<kQ>(w[f], x[r], e[r]);
      if (i == 2) {
#pragma unroll
        for (int q = 0; q < 4; ++q) scale[q] = uniform(next[q]);
      }
      const int j = (i + 29) & 31;
      acc[weight(j)][tile(j)] += (i < 3 ? before : scale)[weight(j)] * part[j & 3];
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      if ((i & 3) == 0) read((i >> 2) + 1);
      product(i);
    }
    step_barrier<8>();
    auto middle = [&](auto index) {
      constexpr int i = decltype(index)::value;
      if (i == 12) read(4);
      if (i == 16) read(5);
      if (i == 20) {
        read(6);
        read(7);
      }
      product(i);
      if constexpr (i < 18) {
        load(step + 2, Index<i - 12>());
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    middle(Index<12>()); middle(Index<13>()); middle(Index<14>()); middle(Index<15>());
    middle(Index<16>()); middle(Index<17>()); middle(Index<18>()); middle(Index<19>());
    middle(Index<20>()); middle(Index<21>()); middle(Index<22>()); middle(Index<23>());
    step_barrier<8>();
    x[2] = read_x(kQ + 1, 0);
    e[2] = read_e((quad + (kQ == 3)) & (kChunk / 4 - 1), 0);
#pragma unroll
    for (int i = 24; i < 32; ++i) {
      product(i);
      if (i & 1) w[weight(i)] = read_w(kQ + 1, weight(i));
      if (i == 25) load(step + 2, Index<6>());
      if (i == 27) load(step + 2, Index<7>());
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (int first = 0; first < a.steps; first += kChunk) {
    if (first) {
      step_barrier<0>();  // the last chunk's exponents have been read
      chunk(first);
      step_barrier<0>();
      trim_chunk<kBig>(a, first, s_bytes + kAtE);
    }
    e[2] = read_e(0, 0);
    // four steps at a time; past the last one the rows are zeros, and so is their scale
    const int until = min(first + kChunk, a.steps);
    for (int step = first; step < until; step += 4) {
      const int quad = (step & (kChunk - 1)) >> 2;
      one(step, quad, Index<0>());
      one(step + 1, quad, Index<1>());
      one(step + 2, quad, Index<2>());
      one(step + 3, quad, Index<3>());
    }
  }
#pragma unroll
  for (int j = 29; j < 32; ++j)
    acc[(j - 24) >> 1][6 + (j & 1)] += scale[(j - 24) >> 1] * part[j & 3];
  step_barrier<0>();  // the last loads, which bring zeros, have landed
  finish<kEpilogue, 4, 8, 4, 2>(a, acc, s_bytes, u0, r0, high);
}

// ---- fewer rows: smaller tiles, more stages, the steps split where there are few tiles ----

// The sizes of a workgroup: WF x WR waves, each with 16 FT features by 16 RT rows; S stages.
template <int kFT, int kRT, int kWF, int kWR, int kS>
struct Tile {
  static constexpr int FT = kFT, RT = kRT, WF = kWF, WR = kWR, S = kS;
  static constexpr int kWaves = WF * WR, kThreads = 64 * kWaves;
  static constexpr int kRows = 16 * RT * WR, kSlots = FT * WF;  // rows, 16-feature tiles
  static constexpr int kXLoads = kRows / 8 / kWaves, kWLoads = 2 * kSlots / kWaves;  // a wave's
  static constexpr int kXBytes = kRows * kStep, kStageBytes = kXBytes + kSlots * 16 * kStep;
  static constexpr int kAtE = S * kStageBytes, kAtS = kAtE + kChunk * kRows;
  static constexpr int kBytes = kAtS + kChunk * 4 * kSlots;
  static_assert(kXLoads * 8 * kWaves == kRows && (kWLoads == 2 || kWLoads == 4) &&
                kWLoads * kWaves == 2 * kSlots, "");
  static_assert(kRows * (32 * kSlots + 16) <= kBytes && kBytes <= 160 * 1024, "");
};

// Bound by what waves issue around the products (a step of 128 x 128 is 512 cycles of the matrix
// unit and 1000 in all, with some 107 instructions a wave), and by the card's power: with all CUs
// at work the clock falls from 2.4 to 1.9 GHz, zeros instead of data take a fifth less time, and
// 89 instructions a step make a lone workgroup 9% faster, all of them 2% at best. 531 rows of
// 4096 by 6144 features 23.9 us (240 workgroups), 64 rows of 12288 by 4096 features 12.9 us and
// 3.7 for the join.
template <int kEpilogue, class T>
__global__ __launch_bounds__(T::kThreads, 2) void k_fp8_tile(Fp8Args a) {
  constexpr bool kGate = kEpilogue != HS_LINEAR_PLAIN;
  constexpr int FT = T::FT, RT = T::RT, OT = kGate ? FT / 2 : FT;
  extern __shared__ uint4 s_all[];  // [stage][x: row, piece | w: tile, half, lane], exponents, scales
  uint8_t* s_bytes = reinterpret_cast<uint8_t*>(s_all);
  const uint32_t lds = lds_address(s_all);
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wf = wave % T::WF, wr = wave / T::WF;
  const int tiles = a.cols * a.rowtiles, order = order_of(tiles * a.nsplit);
  const int split = order / tiles;
  int u0, r0;
  place_of(a, order % tiles, u0, r0);
  r0 *= T::kRows;
  u0 *= OT * T::WF;
  const int begin = split * a.split_steps, end = min(a.steps, begin + a.split_steps);
  auto tile_of = [&](int slot) {  // weight tile of one of the workgroup's slots
    const int f = slot % FT, u = u0 + slot / FT * OT + f % OT;
    return min(u, a.units - 1) + f / OT * a.up;
  };
  const int64_t tile_bytes = (int64_t)a.steps * (16 * kStep);
  uint8_t* wp = reinterpret_cast<uint8_t*>(const_cast<uint4*>(a.w));
  uint8_t* xp = const_cast<uint8_t*>(a.x + (int64_t)r0 * a.xs);
  constexpr int kWLoads = T::kWLoads;
  uint8_t* wp0 = wp + tile_of(kWLoads / 2 * wave) * tile_bytes;
  uint8_t* wp1 = wp + tile_of(kWLoads / 2 * (wave + 1) - 1) * tile_bytes;
  const int high = min(a.rows - r0, T::kRows), k_end = min(a.K, kStep * end);
  const int x_range = (high - 1) * (int)a.xs + a.K;  // rows behind the last one read zeros
  const int piece = swizzle(lane >> 3, lane & 7);
  // load i of a step's into stage `to`; past the last step none reads memory
  constexpr int kLoads = T::kXLoads + kWLoads;
  auto load = [&](int step, uint32_t to, int i) {
    if (i < T::kXLoads) {
      const auto b = __builtin_amdgcn_make_buffer_rsrc(xp, 0, x_range, 0x00027000);
      const int k = kStep * step + 16 * piece, row = 8 * (T::kXLoads * wave + i);
      load_lds(b, k < k_end ? (row + (lane >> 3)) * (int)a.xs + k : kPast, 0,
               to + row * kStep);
      return;
    }
    i -= T::kXLoads;
    const auto b = __builtin_amdgcn_make_buffer_rsrc(i < 2 ? wp0 : wp1, 0, step < end ? kRange : 0,
                                                     0x00027000);
    const uint32_t tw = to + T::kXBytes + 1024 * (kWLoads * wave + (i & 2));
    if (i & 1) load_lds<1024>(b, 16 * lane, 16 * kStep * step, tw);
    else load_lds<0>(b, 16 * lane, 16 * kStep * step, tw);
  };
  auto stage = [&](int i) { return lds + i * T::kStageBytes; };
  const uint8_t* ss = s_bytes + T::kAtS + 4 * OT * wf;  // the scales of the wave's tiles
  constexpr int kOutTiles = OT * T::WF;
  auto chunk = [&](int first) {
    load_chunk<kGate, T::kRows, T::kSlots, T::kWaves>(a, first, u0, r0, high, lds + T::kAtE,
                                                      lds + T::kAtS);
  };

  f32x4_t acc[FT][RT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[f][t] = f32x4_t{0, 0, 0, 0};
  chunk(begin);
#pragma unroll
  for (int i = 0; i < T::S * kLoads; ++i) load(begin + i / kLoads, stage(i / kLoads), i % kLoads);
  const int in_rows = 16 * RT * wr + m;
  const uint8_t* sx0 = s_bytes + in_rows * kStep + 16 * swizzle(m, g);
  const uint8_t* sx1 = s_bytes + in_rows * kStep + 16 * swizzle(m, 4 + g);
  const uint8_t* sw = s_bytes + T::kXBytes + wf * FT * 2048 + 16 * lane;
  const uint8_t* se = s_bytes + T::kAtE + 4 * in_rows;
  struct Operands {
    i32x8_t x[RT], w[FT];
  };
  constexpr int kReads = FT + RT;
  auto read = [&](int at, Operands& o, int i) {  // operand i: the weights', then the rows'
    if (i < FT) {
      o.w[i] = operand(*reinterpret_cast<const uint4*>(sw + at + 2048 * i),
                       *reinterpret_cast<const uint4*>(sw + at + 2048 * i + 1024));
    } else {
      o.x[i - FT] = operand(*reinterpret_cast<const uint4*>(sx0 + at + 16 * (i - FT) * kStep),
                            *reinterpret_cast<const uint4*>(sx1 + at + 16 * (i - FT) * kStep));
    }
  };
  step_barrier<(T::S - 1) * kLoads>();
  trim_chunk<T::kRows>(a, begin, s_bytes + T::kAtE);
  Operands even, odd;
#pragma unroll
  for (int i = 0; i < kReads; ++i) read(0, even, i);
  int now = 0;  // the step's stage
  // A step, whose operands are in registers. Between its products the next one's are read
  // and the loads of the step that takes its stage go out: a wave issues in order. The barrier
  // sees that the next step has landed and that all waves have read this one. (With all CUs at
  // work a step of 128 x 128 takes 0.54 us with eight waves, 0.70 us with four of twice the
  // size, one to a SIMD.)
  auto one = [&](int step, int in_chunk, const Operands& o, Operands& next) {
    step_barrier<(T::S - 2) * kLoads>();
    uint32_t e[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
      e[t] = *reinterpret_cast<const uint32_t*>(se + (in_chunk >> 2) * 4 * T::kRows + 64 * t);
    const uint32_t to = stage(now);
    now = now == T::S - 1 ? 0 : now + 1;
    const int shift = 8 * (in_chunk & 3);
    float scale[FT];
    read_scales<OT>(ss + 4 * kOutTiles * in_chunk, scale);
    if constexpr (kGate)
      read_scales<OT>(ss + 4 * kOutTiles * (kChunk + in_chunk), scale + OT);
    // products, each added three products later
    f32x4_t part[4];
    auto add = [&](int j) { acc[j % FT][j / FT] += scale[j % FT] * part[j & 3]; };
#pragma unroll
    for (int i = 0; i < FT * RT; ++i) {
      const int t = i / FT, f = i % FT;
      if (f == 0) e[t] >>= shift;
      if (i >= 3) add(i - 3);
      part[i & 3] = mfma<0>(o.w[f], o.x[t], e[t]);
      constexpr int P = FT * RT;
#pragma unroll
      for (int j = i * kReads / P; j < (i + 1) * kReads / P; ++j)
        read(now * T::kStageBytes, next, j);
#pragma unroll
      for (int j = i * kLoads / P; j < (i + 1) * kLoads / P; ++j) load(step + T::S, to, j);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = FT * RT - 3; j < FT * RT; ++j) add(j);
  };
  for (int first = begin; first < end; first += kChunk) {
    if (first != begin) {
      step_barrier<0>();  // the last chunk's exponents have been read
      chunk(first);
      step_barrier<0>();
      trim_chunk<T::kRows>(a, first, s_bytes + T::kAtE);
    }
    // two steps at a time: past the last one the rows are zeros, and so is their scale
    const int count = min(kChunk, end - first);
    for (int i = 0; i < count; i += 2) {
      one(first + i, i, even, odd);
      one(first + i + 1, i + 1, odd, even);
    }
  }
  step_barrier<0>();  // the last loads, which bring zeros, have landed
  if (a.part) {
    const int64_t width = (int64_t)a.units * (kGate ? 32 : 16);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (in_rows + 16 * t >= high) continue;
      float* to = a.part + ((int64_t)split * a.rows + r0 + in_rows + 16 * t) * width;
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        const int u = u0 + wf * OT + f % OT;
        if (u < a.units)
          *reinterpret_cast<f32x4_t*>(to + (int64_t)(u + f / OT * a.units) * 16 + 4 * g) = acc[f][t];
      }
    }
    return;
  }
  if constexpr (kEpilogue != HS_LINEAR_SWIGLU_FP8)
    finish<kEpilogue, FT, RT, T::WF, T::WR>(a, acc, s_bytes, u0, r0, high);
  else if constexpr (OT * T::WF == 8)
    finish<kEpilogue, FT, RT, T::WF, T::WR>(a, acc, s_bytes, u0, r0, high);
}

constexpr int kJoinThreads = 256;

// Adds the parts of split steps and finishes them, 8 features a thread: bf16 or (kEight)
// codes, 16 lanes a group.
template <bool kGate, bool kEight>
__global__ __launch_bounds__(kJoinThreads) void k_fp8_join(Fp8Args a) {
  const int groups = (a.N + kFp8Group - 1) / kFp8Group;
  const int64_t e = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
  const int64_t at = e >> 4;
  if (at >= (int64_t)groups * a.rows) return;  // whole groups of lanes
  const int64_t row = at / groups;
  const int group = (int)(at % groups), n = group * kFp8Group + 8 * (int)(e & 15);
  const int64_t width = (int64_t)a.units * (kGate ? 32 : 16);
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (n < a.N) {
    for (int s = 0; s < a.nsplit; ++s) {
      const float* p = a.part + ((int64_t)s * a.rows + row) * width + n;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const f32x4_t q = *reinterpret_cast<const f32x4_t*>(p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i + j] += q[j];
        if (kGate) {
          const f32x4_t r = *reinterpret_cast<const f32x4_t*>(p + (int64_t)a.units * 16 + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) u[i + j] += r[j];
        }
      }
    }
  }
  if constexpr (kEight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = swiglu(v[i], u[i]);
    uint2 c;
    const uint32_t byte = group_codes8(v, c);
    if (n < a.N) *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.y) + row * a.ys + n) = c;
    if ((e & 15) == 0) a.ye[row * a.yes + group] = (uint8_t)byte;
  } else {
    uint16_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = result<kGate>(v[i], u[i]);
    store8(a, row, n, pack8(h));
  }
}

constexpr int kCus = 256;

using Tile256x128 = Tile<4, 4, 4, 2, 3>;  // features by rows
using Tile128x128 = Tile<2, 4, 4, 2, 4>;
using Tile128x64 = Tile<2, 2, 4, 2, 3>;
using Tile128x32 = Tile<2, 2, 4, 1, 3>;

enum Kernel { kRows, k128x32, k128x64, k128x128, k256x128, k256x256 };

// What a workgroup of a tile kernel takes, in us: a step, alone and with all CUs at work, and
// everything beside the steps. Fitted to 135 shapes (17 to 3000 rows, 1024 to 12288 inputs, 1024
// to 24576 features) with every kernel and up to 16 splits: the choices by these figures take
// 0.6% longer than the best ones on average, 7% at most.
struct TileTime {
  int features, rows;
  float step, full_step, rest;
};
constexpr TileTime kTileTimes[] = {{0, 0, 0, 0, 0},
                                   {128, 32, 0.23f, 0.28f, 3.4f},
                                   {128, 64, 0.30f, 0.38f, 3.5f},
                                   {128, 128, 0.37f, 0.54f, 4.1f},
                                   {256, 128, 0.66f, 0.78f, 6.7f},
                                   {256, 256, 1.12f, 1.35f, 6.7f}};

struct Fp8Plan {
  Kernel kernel;
  bool fused;          // bf16 rows go to 8 bits in the projection's kernel
  int split_steps, nsplit;
  size_t part_bytes;   // sums of split steps
  size_t codes_bytes;  // codes of bf16 rows
  size_t bytes;
};

size_t padded(size_t n) { return (n + 255) / 256 * 256; }
int64_t scales_row(int K) { return ((K + kStep - 1) / kStep + 3) / 4 * 4; }

// The few-row kernel's sizes for a call, none (0 waves) where the tiles serve it. Up to 16 rows
// take it always:
// - 16 waves for a tile of a weight of up to 256 (4 rows of 4096, 4096 features: 5.3 us, 5.9 with
//   8), 8 for more than 8 rows, whose operands weigh more (16 rows of 4096: 6.1 us, 6.4 with 16; of
//   12288: 12.9 and 14.5; 9 rows of 4096 would gain, 5.8 and 5.2);
// - two tiles to a workgroup that shares their rows for wider ones (4 rows of 4096, 6144 features:
//   7.0 us, 7.4 with one);
// - four of very wide ones with many rows, for the bf16 rows that each workgroup takes to 8 bits
//   (16 of 4096, with four and with two tiles: 40960 features 34.0 and 33.4 us, 49152 36.5 and
//   38.9, 65536 46.1 and 50.9, 151936 105 and 116). Rows in 8 bits take the same though two tiles
//   would be as fast or faster (16 rows, 151936 features 103 and 104; 9 rows 101 and 94): rows give
//   the same bits in either form.
// More rows take it
// - where the workgroups still fit the CUs: then each weight is read once or twice and nothing has
//   to be joined (4096 inputs, 4096 features: 64 rows 9.6 us, 10.5 in tiles; 32 rows 6.8 and 9.6);
//   with 32 rows a workgroup only up to 56 steps, past which the rows' reads cost more (64 rows by
//   4096 features: 7168 inputs 13.5 us, 13.8 in tiles, 8192 16.0 and 15.0, 12288 23.8 and 19.3; 128
//   rows by 2048: 7168 13.1 and 14.0, 8192 15.8 and 12.9);
// - up to 32 by very wide weights (24 rows of 4096: 49152 features 38.1 us, 40.8 in tiles, 151936
//   109 and 112; 32 rows 39.4 and 41.7, 116 and 113).
struct RowsKernel {
  int waves, tiles, row_tiles;
};
RowsKernel rows_of(int rows, int steps, int units, bool gate) {
  const int r16 = (rows + 15) / 16, r32 = (rows + 31) / 32;
  const int pairs = gate ? units : (units + 1) / 2;
  if (!gate && (int64_t)units * r16 <= kCus) return {rows <= 8 ? 16 : 8, 1, 1};
  if (rows <= 16 && !gate && units >= 12 * kCus && rows > 8) return {4, 4, 1};
  if (rows <= 16 || (int64_t)pairs * r16 <= kCus) return {8, 2, 1};
  if ((int64_t)pairs * r32 <= kCus && steps <= 56) return {8, 2, 2};
  if (rows <= 32 && !gate && units >= 12 * kCus) return {4, 4, 2};
  return {0, 0, 0};
}

Fp8Plan plan_of(int rows, int K, int N, int epilogue, bool bf16_rows) {
  Fp8Plan p = {};
  const bool gate = epilogue != HS_LINEAR_PLAIN, eight = epilogue == HS_LINEAR_SWIGLU_FP8;
  const int steps = (K + kStep - 1) / kStep, units = (N + 15) / 16;
  p.nsplit = 1;
  p.split_steps = steps;
  p.kernel = rows_of(rows, steps, units, gate).waves ? kRows : k128x32;
  if (p.kernel != kRows) {
    float best = 0;
    for (int k = k128x32; k <= k256x256; ++k) {
      const TileTime& t = kTileTimes[k];
      const int64_t tiles = (int64_t)((units * (gate ? 2 : 1) * 16 + t.features - 1) / t.features) *
                            ((rows + t.rows - 1) / t.rows);
      for (int want : {1, 2, 3, 4, 6, 8, 12, 16}) {
        // (exponents are read four steps at a time)
        const int split_steps = ((steps + want - 1) / want + 3) / 4 * 4;
        const int n = (steps + split_steps - 1) / split_steps;
        if (want > 1 && (k == k256x256 || tiles * n > 2 * kCus || split_steps >= steps)) break;
        const int64_t groups = tiles * n, rounds = (groups + kCus - 1) / kCus;
        const float fill = groups < kCus ? (float)groups / kCus : 1.0f;
        const float step = t.step + (t.full_step - t.step) * fill;
        float time = rounds * ((want > 1 ? split_steps : steps) * step + t.rest);
        // the weights' stream, from memory or the cache before it
        time = fmaxf(time, (float)units * (gate ? 2 : 1) * 16 * K / 8e6f + 2.0f);
        // sums that go through memory, and the launch that joins them
        if (n > 1 || (eight && k < k256x128))
          time += 3.6f + (float)n * rows * units * (gate ? 2 : 1) * 64 / 2.25e6f;
        if (best != 0 && time >= best) continue;
        best = time;
        p.kernel = (Kernel)k;
        p.nsplit = n;
        p.split_steps = n > 1 ? split_steps : steps;
      }
    }
  }
  const bool whole = p.kernel == k256x256 || p.kernel == k256x128;  // of a group of outputs
  if (p.nsplit > 1 || (eight && !whole))
    p.part_bytes = padded((size_t)p.nsplit * rows * units * (gate ? 32 : 16) * sizeof(float));
  p.fused = bf16_rows && p.kernel == kRows && rows_of(rows, steps, units, gate).row_tiles == 1;
  if (bf16_rows && !p.fused)
    p.codes_bytes = padded((size_t)rows * K) + padded((size_t)rows * scales_row(K));
  p.bytes = p.part_bytes + p.codes_bytes;
  return p;
}

template <int W, int TN, int RT, bool kGate>
void launch_rows(const Fp8Args& a, bool bf16_rows, hipStream_t s) {
  constexpr int kOut = kGate ? TN / 2 : TN;
  const dim3 grid((unsigned)((a.units + kOut - 1) / kOut), (unsigned)((a.rows + 16 * RT - 1) / (16 * RT)));
  if (bf16_rows) {
    if constexpr (RT == 1)
      hipLaunchKernelGGL((k_fp8_rows<W, TN, RT, kGate, true>), grid, dim3(64 * W), 0, s, a);
  } else {
    hipLaunchKernelGGL((k_fp8_rows<W, TN, RT, kGate, false>), grid, dim3(64 * W), 0, s, a);
  }
}

void dispatch_rows(const Fp8Args& a, bool gate, bool bf16_rows, hipStream_t s) {
  const RowsKernel k = rows_of(a.rows, a.steps, a.units, gate);
  if (gate && k.row_tiles == 1) launch_rows<8, 2, 1, true>(a, bf16_rows, s);
  else if (gate) launch_rows<8, 2, 2, true>(a, bf16_rows, s);
  else if (k.waves == 16) launch_rows<16, 1, 1, false>(a, bf16_rows, s);
  else if (k.tiles == 1) launch_rows<8, 1, 1, false>(a, bf16_rows, s);
  else if (k.tiles == 2 && k.row_tiles == 1) launch_rows<8, 2, 1, false>(a, bf16_rows, s);
  else if (k.tiles == 2) launch_rows<8, 2, 2, false>(a, bf16_rows, s);
  else if (k.row_tiles == 1) launch_rows<4, 4, 1, false>(a, bf16_rows, s);
  else launch_rows<4, 4, 2, false>(a, bf16_rows, s);
}

// a kernel of more than 64 KB of shared memory
template <class F>
int launch(F kernel, int64_t blocks, int threads, int bytes, const Fp8Args& a, hipStream_t s) {
  if (blocks * threads > UINT32_MAX) return HS_ERR_UNSUPPORTED;  // a grid's threads
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return HS_ERR_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), bytes, s, a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

template <int kEpilogue>
int launch_tiles(Fp8Args& a, Kernel kernel, hipStream_t s) {
  constexpr int kHalf = kEpilogue == HS_LINEAR_PLAIN ? 1 : 2;
  auto tiles = [&](int slots, int rows) {
    a.cols = (a.units + slots / kHalf - 1) / (slots / kHalf);
    a.rowtiles = (a.rows + rows - 1) / rows;
    return (int64_t)a.cols * a.rowtiles * a.nsplit;
  };
  auto go = [&](auto tile) {
    using T = decltype(tile);
    return launch(k_fp8_tile<kEpilogue, T>, tiles(T::kSlots, T::kRows), T::kThreads, T::kBytes, a, s);
  };
  if (kernel == k256x256)
    return launch(k_fp8_big<kEpilogue>, tiles(16, kBig), kBigThreads, kBigBytes, a, s);
  if (kernel == k256x128) return go(Tile256x128());
  if (kernel == k128x128) return go(Tile128x128());
  if (kernel == k128x64) return go(Tile128x64());
  return go(Tile128x32());
}

int join(const Fp8Args& a, int epilogue, hipStream_t s) {
  const int64_t groups = (a.N + kFp8Group - 1) / kFp8Group * (int64_t)a.rows;
  if (groups * 16 + kJoinThreads > UINT32_MAX) return HS_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((groups * 16 + kJoinThreads - 1) / kJoinThreads)), block(kJoinThreads);
  if (epilogue == HS_LINEAR_PLAIN)
    hipLaunchKernelGGL((k_fp8_join<false, false>), grid, block, 0, s, a);
  else if (epilogue == HS_LINEAR_SWIGLU)
    hipLaunchKernelGGL((k_fp8_join<true, false>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((k_fp8_join<true, true>), grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
}

constexpr int kMaxRows = 1 << 20;

bool sizes_ok(int rows, int K, int N, int epilogue) {
  return rows >= 1 && K >= 1 && N >= 1 && epilogue >= HS_LINEAR_PLAIN &&
         epilogue <= HS_LINEAR_SWIGLU_FP8;
}
// grids and 32-bit offsets of the kernels
bool sizes_fit(int rows, int K, int N) {
  return rows <= kMaxRows && K <= 1 << 22 && N <= 1 << 24;
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

size_t hs_linear_fp8_workspace_size(int rows, int in_features, int out_features, int epilogue,
                                    int bf16_rows) {
  if (!sizes_ok(rows, in_features, out_features, epilogue) ||
      !sizes_fit(rows, in_features, out_features))
    return 0;
  return plan_of(rows, in_features, out_features, epilogue, bf16_rows != 0).bytes;
}

int hs_linear_fp8_plan(int rows, int in_features, int out_features, int epilogue, int bf16_rows,
                       int* plan) {
  if (!plan || !sizes_ok(rows, in_features, out_features, epilogue)) return HS_ERR_INVALID;
  if (!sizes_fit(rows, in_features, out_features)) return HS_ERR_UNSUPPORTED;
  const Fp8Plan p = plan_of(rows, in_features, out_features, epilogue, bf16_rows != 0);
  if (p.kernel == kRows) {
    const RowsKernel k = rows_of(rows, (in_features + kStep - 1) / kStep, (out_features + 15) / 16,
                                 epilogue != HS_LINEAR_PLAIN);
    plan[0] = 16 * k.tiles;
    plan[1] = 16 * k.row_tiles;
    plan[2] = k.waves;
  } else {
    plan[0] = kTileTimes[p.kernel].features;
    plan[1] = kTileTimes[p.kernel].rows;
    plan[2] = p.kernel == k128x32 ? Tile128x32::kWaves : kBigThreads / 64;
  }
  plan[3] = p.split_steps;
  return HS_OK;
}

int hs_linear_fp8(const void* x, int64_t x_stride, const void* x_scales, int64_t x_scales_stride,
                  const void* packed, const float* scales, int rows, int in_features,
                  int out_features, int epilogue, void* out, int64_t out_stride, void* out_scales,
                  int64_t out_scales_stride, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (rows == 0) return HS_OK;
  const bool gate = epilogue != HS_LINEAR_PLAIN, eight = epilogue == HS_LINEAR_SWIGLU_FP8;
  if (!x || !packed || !scales || !out || (eight && !out_scales)) return HS_ERR_INVALID;
  if (!sizes_ok(rows, in_features, out_features, epilogue)) return HS_ERR_INVALID;
  if (in_features % 16) return HS_ERR_UNSUPPORTED;
  // gate and up halves start at a tile each
  if (gate && out_features % 16) return HS_ERR_UNSUPPORTED;
  if (!sizes_fit(rows, in_features, out_features)) return HS_ERR_UNSUPPORTED;
  const bool bf16_rows = !x_scales;
  if ((x_stride % (bf16_rows ? 8 : 16)) || x_stride < in_features || x_stride > (1 << 22))
    return HS_ERR_UNSUPPORTED;
  if (!bf16_rows && ((x_scales_stride % 4) || ((uintptr_t)x_scales & 3) ||
                     x_scales_stride < scales_row(in_features) || x_scales_stride > (1 << 22)))
    return HS_ERR_UNSUPPORTED;
  if (out_stride < out_features) return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)x | (uintptr_t)packed) & 15) return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)scales & 3) || ((uintptr_t)out & (eight ? 15 : 1))) return HS_ERR_UNSUPPORTED;
  if (eight && (out_stride % 16 || out_scales_stride < (out_features + kStep - 1) / kStep))
    return HS_ERR_UNSUPPORTED;
  const Fp8Plan p = plan_of(rows, in_features, out_features, epilogue, bf16_rows);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return HS_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HS_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Fp8Args a;
  a.x = static_cast<const uint8_t*>(x);
  a.xs = x_stride;
  a.xe = static_cast<const uint8_t*>(x_scales);
  a.xes = x_scales_stride;
  if (bf16_rows && !p.fused) {
    uint8_t* codes = ws + p.part_bytes;
    uint8_t* exps = codes + padded((size_t)rows * in_features);
    const int status = hs_quantize_rows_fp8(x, x_stride, rows, in_features, codes, in_features,
                                            exps, scales_row(in_features), stream);
    if (status != HS_OK) return status;
    a.x = codes;
    a.xs = in_features;
    a.xe = exps;
    a.xes = scales_row(in_features);
  }
  a.w = static_cast<const uint4*>(packed);
  a.sc = scales;
  a.rows = rows;
  a.K = in_features;
  a.N = out_features;
  a.steps = (in_features + kStep - 1) / kStep;
  a.units = (out_features + 15) / 16;
  a.up = a.units;
  a.y = static_cast<uint16_t*>(out);
  a.ys = out_stride;
  a.wide = !((uintptr_t)out & 15) && out_stride % 8 == 0;
  a.ye = static_cast<uint8_t*>(out_scales);
  a.yes = out_scales_stride;
  a.part = p.part_bytes ? reinterpret_cast<float*>(ws) : nullptr;
  a.split_steps = p.split_steps;
  a.nsplit = p.nsplit;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int status = HS_OK;
  if (p.kernel == kRows) {
    dispatch_rows(a, gate, p.fused, s);
    if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  } else if (epilogue == HS_LINEAR_PLAIN) {
    status = launch_tiles<HS_LINEAR_PLAIN>(a, p.kernel, s);
  } else if (epilogue == HS_LINEAR_SWIGLU) {
    status = launch_tiles<HS_LINEAR_SWIGLU>(a, p.kernel, s);
  } else {
    status = launch_tiles<HS_LINEAR_SWIGLU_FP8>(a, p.kernel, s);
  }
  if (status != HS_OK) return status;
  return a.part ? join(a, epilogue, s) : HS_OK;
}

}  // extern "C"
