// Projections with 4-bit weights and group scales on gfx950:
//   y[r, n] = sum_k x[r, k] (c[n, k] - 8) s[n, k / group]     (x, y bf16, s bf16)
// with f32 accumulation; SwiGLU: y = silu(gate) * up of a [2F, K] weight, rounded once.
//
// A weight is kept as 16-feature tiles by 128-input steps, 1 KB each: dword i of
// lane l holds the codes of feature l % 16, inputs 32 i + 8 (l / 16) .. + 7, so a
// wave loads a step with one 16-byte load a lane, contiguous over the tile, and
// each dword is one lane's share of a 16x16x32 MFMA A operand. The codes are not
// converted: shifted into the top four mantissa bits of a bf16 2^-8 they read
// (16 + c) 2^-12 (one shift and one and-or for two of them), and
//   sum x (c - 8) = 2^12 (sum x (16 + c) 2^-12 - sum x 24 2^-12),
// whose last sum is the same for every feature and enters as the accumulator's
// start. A group's products end in an accumulator of their own that its scales
// then multiply; 2^12 multiplies the output's sum: nothing is rounded below f32 before
// the output. (The offset costs the sums a factor of about 24 / 4.6, the size of 16 + c
// over that of c - 8, in f32's last bits. 2^-12, because the partial sums of a group then
// stay finite whatever finite x are: 128 products of at most 31 2^-12 |x|. An infinity in
// x gives NaN.)
//
// k_int4_rows (up to 16 rows): bound by the weights' stream. A workgroup's waves share
// out the steps of its one to four tiles and join their sums in LDS. The rows come from
// L2 in every workgroup, as B operands straight into registers.
// k_int4_tile (more rows): 128 features by 64 rows a workgroup, the rows' step in
// LDS as B operands shared by its four waves, each with 32 features of its own; where
// there are few workgroups the steps are split over two sets of waves and over
// workgroups, whose parts k_int4_join adds.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_model_dev.h"

namespace hs {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;  // inputs of a step

struct Int4Args {
  const uint16_t* x;
  int64_t xs;
  const uint4* w;       // [tiles][steps][64]
  const uint16_t* sc;   // [tiles][steps * groups][16]
  int rows, K, N;       // N: output features
  int steps;
  int units;            // 16-feature tiles of the output
  int up;               // first tile of the up rows (SwiGLU)
  uint16_t* y;
  int64_t ys;
  float* part;          // [split][rows][tiles * 16] (k_int4_tile with split steps)
  int split_steps, nsplit;
};

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

constexpr float kUnit = 4096.0f;  // the sums are kept in units of 2^12

// 8 codes -> bf16 (16 + c) 2^-12: a shift and an and-or for two, with the mask in a vector and the
// base in a scalar register (as two literals they would take an instruction more)
struct CodeMask {
  uint32_t mask, base;
  __device__ __forceinline__ CodeMask() : mask(0x00780078u), base(0x3b803b80u) {
    asm("" : "+v"(mask));
    asm("" : "+s"(base));
  }
};
__device__ __forceinline__ bf16x8_t codes8(uint32_t w, const CodeMask& m) {
  u32x4_t u;
  u.x = ((w << 3) & m.mask) | m.base;
  u.y = ((w >> 1) & m.mask) | m.base;
  u.z = ((w >> 5) & m.mask) | m.base;
  u.w = ((w >> 9) & m.mask) | m.base;
  return __builtin_bit_cast(bf16x8_t, u);
}
// -24 2^-12 in every element: the operand whose product with x is the accumulator's start
__device__ __forceinline__ bf16x8_t minus24() {
  const u32x4_t u = {0xbbc0bbc0u, 0xbbc0bbc0u, 0xbbc0bbc0u, 0xbbc0bbc0u};
  return __builtin_bit_cast(bf16x8_t, u);
}

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}

// inputs 128 step + 32 i + 8 g .. + 7 of a row as a B operand; zeros past the row or K
__device__ __forceinline__ bf16x8_t load_x(const Int4Args& a, int row, int step, int i, int g) {
  const int k = kStep * step + 32 * i + 8 * g;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (row < a.rows && k < a.K)
    v = *reinterpret_cast<const uint4*>(a.x + (int64_t)row * a.xs + k);
  return __builtin_bit_cast(bf16x8_t, v);
}

__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

// the output of sums in units of 2^12
template <bool kGate>
__device__ __forceinline__ uint16_t result(float v, float up) {
  return to_bf(kGate ? silu(v * kUnit) * (up * kUnit) : v * kUnit);
}

// a lane's share of one step of one tile: its codes, and the scales of features
// 4 g .. 4 g + 3 in the step's GP groups
template <int GP>
struct Step {
  uint4 w;
  uint2 s[GP];
};
template <int GP>
__device__ __forceinline__ void load_step(const Int4Args& a, int tile, int step, int lane,
                                          Step<GP>& st) {
  const int64_t at = (int64_t)tile * a.steps + step;
  st.w = load_once(a.w + at * 64 + lane);
#pragma unroll
  for (int p = 0; p < GP; ++p)
    st.s[p] = *reinterpret_cast<const uint2*>(a.sc + (at * GP + p) * 16 + 4 * (lane >> 4));
}

__device__ __forceinline__ void add_scaled(f32x4_t& y, const f32x4_t& acc, uint2 s) {
  y[0] += acc[0] * __uint_as_float(s.x << 16);
  y[1] += acc[1] * __uint_as_float(s.x & 0xffff0000u);
  y[2] += acc[2] * __uint_as_float(s.y << 16);
  y[3] += acc[3] * __uint_as_float(s.y & 0xffff0000u);
}

// y += the step's products. c0[p]: -24 2^-12 sum x of group p (the lane's column).
template <int GP>
__device__ __forceinline__ void multiply(const Step<GP>& st, const bf16x8_t (&x)[4],
                                         const float (&c0)[GP], const CodeMask& mask, f32x4_t& y) {
  const uint32_t w[4] = {st.w.x, st.w.y, st.w.z, st.w.w};
#pragma unroll
  for (int p = 0; p < GP; ++p) {
    f32x4_t acc = {c0[p], c0[p], c0[p], c0[p]};
#pragma unroll
    for (int i = p * 4 / GP; i < (p + 1) * 4 / GP; ++i) acc = mfma(codes8(w[i], mask), x[i], acc);
    add_scaled(y, acc, st.s[p]);
  }
}

// Up to 16 rows. W: waves of a workgroup; TN: its weight tiles (with SwiGLU half of them
// gate and half up tiles).
template <int GP, int W, int TN, bool kGate>
__global__ __launch_bounds__(64 * W) void k_int4_rows(Int4Args a) {
  constexpr int kOut = kGate ? TN / 2 : TN;
  __shared__ float s_part[W][TN][16][16];  // [wave][tile][row][feature]
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int u0 = blockIdx.x * kOut;
  const CodeMask mask;
  int tile[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) tile[t] = min(u0 + t % kOut, a.units - 1) + t / kOut * a.up;
  f32x4_t y[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) y[t] = f32x4_t{0, 0, 0, 0};
  // One step's loads at a time: many waves hide them better than many loads of few waves
  // (12288 features, SwiGLU, 4 rows: 20.8 us with 8 waves and two steps ahead, 17.3 us so
  // when that was measured; 16.0 us as the codes are decoded now)
  for (int step = wave; step < a.steps; step += W) {
    bf16x8_t x[4];
    Step<GP> w[TN];
#pragma unroll
    for (int t = 0; t < TN; ++t) load_step<GP>(a, tile[t], step, lane, w[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = load_x(a, m, step, i, g);
    float c0[GP];
#pragma unroll
    for (int p = 0; p < GP; ++p) {
      f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int i = p * 4 / GP; i < (p + 1) * 4 / GP; ++i) acc = mfma(minus24(), x[i], acc);
      c0[p] = acc[0];
    }
#pragma unroll
    for (int t = 0; t < TN; ++t) multiply<GP>(w[t], x, c0, mask, y[t]);
  }
  if (m < a.rows) {
#pragma unroll
    for (int t = 0; t < TN; ++t) *reinterpret_cast<f32x4_t*>(&s_part[wave][t][m][4 * g]) = y[t];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * a.rows * kOut; e += 64 * W) {
    const int n = e & 15, t = (e >> 4) % kOut, row = (e >> 4) / kOut;
    float v = 0.0f, up = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      v += s_part[w][t][row][n];
      if (kGate) up += s_part[w][kOut + t][row][n];
    }
    const int col = (u0 + t) * 16 + n;
    if (col < a.N) a.y[(int64_t)row * a.ys + col] = result<kGate>(v, up);
  }
}

constexpr int kTileRows = 64, kTileWaves = 4;
constexpr int kPast = INT32_MAX - 511;  // a byte offset past any row: reads zeros

// waits for the wave's LDS traffic only: the next step's loads stay in flight
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ uint4 as_uint4(u32x4_t v) { return make_uint4(v.x, v.y, v.z, v.w); }

// 32 output features a wave (with SwiGLU 16, gate and up) by 64 rows. The next step's loads
// are in flight during a step, issued alike whatever is left: past the end their buffers
// are empty and they touch no memory. Two and three steps ahead took the same time or
// longer; what bounds it is a wave's own chain of operand reads, code shifts and products.
// H = 2: two sets of waves, each with rows of its own in LDS, take the steps in turn and
// join their sums in LDS. 64 rows of 12288 inputs, 4096 features: 22.1 us (291 TFLOP/s), 4
// of them the join's launch; 600 rows of 4096 inputs, 2 x 12288 features: 167 us (723 TFLOP/s),
// 4096 rows 1021 us (808): every 64 rows decode the weights again.
template <int GP, bool kGate, int H>
__global__ __launch_bounds__(64 * kTileWaves * H, H == 1 && GP < 4 ? 3 : 2)
void k_int4_tile(Int4Args a) {
  constexpr int RT = kTileRows / 16;
  __shared__ uint4 s_xs[H][2][4][RT][64];      // [half][step parity][i][row tile][lane]
  __shared__ float s_cs[H][2][GP][kTileRows];  // -24 2^-12 sum x
  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kTileWaves;
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kTileWaves;
  auto& s_x = s_xs[half];
  auto& s_c = s_cs[half];
  const int r0 = blockIdx.y * kTileRows;
  const int first = blockIdx.z * a.split_steps;
  const int last = min(a.steps, first + a.split_steps);
  // the wave's two weight tiles; tiles past the end repeat the last one
  const int u0 = blockIdx.x * (kGate ? 1 : 2) * kTileWaves + wave * (kGate ? 1 : 2);
  const int ua = min(u0, a.units - 1);
  const int ub = kGate ? ua + a.up : min(u0 + 1, a.units - 1);

  const CodeMask mask;
  static_assert(RT == kTileWaves, "a wave stages one row tile");
  u32x4_t x[4];
  Step<GP> w[2];
  const int row_at = r0 + 16 * wave + m < a.rows ? (16 * wave + m) * (int)a.xs * 2 + 16 * g
                                                 : kPast;
  const int64_t wa0 = (int64_t)ua * a.steps, wb0 = (int64_t)ub * a.steps;
  auto load = [&](int step) {
    const bool live = step < last;
    const int k = kStep * min(step, a.steps - 1);
    const int64_t at = live ? step : 0;
    const auto xb = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.x + (int64_t)r0 * a.xs + k), 0, live ? kPast : 0, 0x00027000);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __builtin_amdgcn_raw_buffer_load_b128(
          xb, k + 32 * i + 8 * g < a.K && row_at != kPast ? row_at + 64 * i : kPast, 0, 0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t tile = (t ? wb0 : wa0) + at;
      const auto wb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint4*>(a.w + tile * 64), 0,
                                                        live ? 1024 : 0, 0x00027000);
      const auto sb = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(a.sc + tile * GP * 16), 0, live ? 32 * GP : 0, 0x00027000);
      w[t].w = as_uint4(__builtin_amdgcn_raw_buffer_load_b128(wb, 16 * lane, 0, 0));
#pragma unroll
      for (int p = 0; p < GP; ++p) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(sb, 32 * p + 8 * g, 0, 0);
        w[t].s[p] = make_uint2(v[0], v[1]);
      }
    }
  };
  f32x4_t y[2][RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) y[0][t] = y[1][t] = f32x4_t{0, 0, 0, 0};
  load(first + half);
  // the halves take turns, and as many steps (the last one may be empty)
  for (int step = first, par = 0; step < last; step += H, par ^= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s_x[par][i][wave][lane] = as_uint4(x[i]);
#pragma unroll
    for (int p = 0; p < GP; ++p) {
      f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int i = p * 4 / GP; i < (p + 1) * 4 / GP; ++i)
        acc = mfma(minus24(), __builtin_bit_cast(bf16x8_t, x[i]), acc);
      if (g == 0) s_c[par][p][16 * wave + m] = acc[0];
    }
    const Step<GP> ca = w[0], cb = w[1];
    load(step + H + half);
    lds_barrier();
    const uint32_t qa[4] = {ca.w.x, ca.w.y, ca.w.z, ca.w.w};
    const uint32_t qb[4] = {cb.w.x, cb.w.y, cb.w.z, cb.w.w};
#pragma unroll
    for (int p = 0; p < GP; ++p) {
      f32x4_t acc[2][RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float c = s_c[par][p][16 * t + m];
        acc[0][t] = acc[1][t] = f32x4_t{c, c, c, c};
      }
#pragma unroll
      for (int i = p * 4 / GP; i < (p + 1) * 4 / GP; ++i) {
        const bf16x8_t fa = codes8(qa[i], mask), fb = codes8(qb[i], mask);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const bf16x8_t b = __builtin_bit_cast(bf16x8_t, s_x[par][i][t][lane]);
          acc[0][t] = mfma(fa, b, acc[0][t]);
          acc[1][t] = mfma(fb, b, acc[1][t]);
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        add_scaled(y[0][t], acc[0][t], ca.s[p]);
        add_scaled(y[1][t], acc[1][t], cb.s[p]);
      }
    }
    // one barrier a step: the buffer written next was read before this step's barrier
  }
  if constexpr (H == 2) {
    // the second half's sums, through its own buffers of x
    static_assert(sizeof(s_xs[0]) == sizeof(y) * 64 * kTileWaves, "");
    f32x4_t* part = reinterpret_cast<f32x4_t*>(&s_xs[1]) + wave * 2 * RT * 64 + lane;
    __syncthreads();
    if (half) {
#pragma unroll
      for (int t = 0; t < 2 * RT; ++t) part[64 * t] = y[t / RT][t % RT];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int t = 0; t < 2 * RT; ++t) y[t / RT][t % RT] += part[64 * t];
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = r0 + 16 * t + m;
    if (row >= a.rows) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tile = u0 + (kGate ? 0 : h);
      if (tile >= a.units) continue;
      if (a.nsplit > 1) {
        const int64_t width = (int64_t)a.units * 16 * (kGate ? 2 : 1);
        const int64_t col = (int64_t)(kGate && h ? a.units + tile : tile) * 16 + 4 * g;
        *reinterpret_cast<f32x4_t*>(a.part + ((int64_t)blockIdx.z * a.rows + row) * width + col) =
            y[h][t];
        continue;
      }
      if (kGate && h) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = tile * 16 + 4 * g + j;
        if (n < a.N) a.y[(int64_t)row * a.ys + n] = result<kGate>(y[h][t][j], y[1][t][j]);
      }
    }
  }
}

// Adds the parts of split steps: 4 features a thread.
template <bool kGate>
__global__ __launch_bounds__(256) void k_int4_join(Int4Args a) {
  const int64_t quads = (int64_t)a.units * 4;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= quads * a.rows) return;
  const int64_t row = e / quads, n = 4 * (e % quads);
  const int64_t width = (int64_t)a.units * 16 * (kGate ? 2 : 1);
  f32x4_t v = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) {
    const float* p = a.part + ((int64_t)s * a.rows + row) * width + n;
    v += *reinterpret_cast<const f32x4_t*>(p);
    if (kGate) u += *reinterpret_cast<const f32x4_t*>(p + (int64_t)a.units * 16);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j < a.N) a.y[row * a.ys + n + j] = result<kGate>(v[j], u[j]);
  }
}

constexpr int kCus = 256;

struct Int4Plan {
  bool rows;  // k_int4_rows
  int halves;
  int split_steps, nsplit;
  size_t bytes;
};

Int4Plan plan_of(int rows, int K, int N, bool gate) {
  Int4Plan p = {};
  const int steps = (K + kStep - 1) / kStep, units = (N + 15) / 16;
  p.nsplit = 1;
  p.split_steps = steps;
  p.rows = rows <= 16;
  if (p.rows) return p;
  // split the steps until there are about two workgroups a CU, at least 4 steps a wave
  const int64_t groups = (int64_t)((units + (gate ? 4 : 8) - 1) / (gate ? 4 : 8)) *
                         ((rows + kTileRows - 1) / kTileRows);
  // With 8 steps for every CU, one workgroup a CU whose halves share its steps: half the
  // parts (64 rows of 12288 inputs, 4096 features: 21.0 us, 23.0 us with two workgroups),
  // or none (64 rows of 4096, 2 x 12288: 30.5 us, 33.9 us). Fewer steps go to more
  // workgroups (17 rows of 4096, 4096 features: 11.1 us, 12.9 us in halves).
  p.halves = groups < kCus && groups * steps >= 8 * kCus ? 2 : 1;
  int want = (int)(p.halves == 2 ? kCus / groups : (2 * kCus + groups - 1) / groups);
  const int least = 4 * p.halves;
  if (want > (steps + least - 1) / least) want = (steps + least - 1) / least;
  if (want > 1) {
    p.split_steps = (steps + want - 1) / want;
    p.nsplit = (steps + p.split_steps - 1) / p.split_steps;
  }
  if (p.nsplit > 1)
    p.bytes = (size_t)p.nsplit * rows * units * 16 * (gate ? 2 : 1) * sizeof(float);
  return p;
}

template <int GP, int W, int TN, bool kGate>
void launch_rows(const Int4Args& a, hipStream_t s) {
  constexpr int kOut = kGate ? TN / 2 : TN;
  hipLaunchKernelGGL((k_int4_rows<GP, W, TN, kGate>),
                     dim3((unsigned)((a.units + kOut - 1) / kOut)), dim3(64 * W), 0, s, a);
}

// Many tiles: workgroups of 4 waves, several of which fit a CU and hide each other's
// beginning and end, and of several tiles, which share the rows' loads (151936 features, 4
// rows: 67 us with 8 waves and 2 tiles, 71 us with 4 and 2, 60 us with 4 and 4: 5.4 TB/s).
// Few: 8 waves to one tile, so that each CU has its tile's steps in flight at once (4096 by
// 4096, 4 rows: 7.4 us, 9.8 us with 4), more where there are many steps (12288 inputs, 8
// rows: 12.4 us with 12, 14.3 us with 8).
template <int GP>
void dispatch_rows(const Int4Args& a, bool gate, hipStream_t s) {
  if (gate) launch_rows<GP, 4, 2, true>(a, s);
  else if (a.units >= 12 * kCus) launch_rows<GP, 4, 4, false>(a, s);
  else if (a.units >= 4 * kCus) launch_rows<GP, 4, 2, false>(a, s);
  else if (a.steps < 64) launch_rows<GP, 8, 1, false>(a, s);
  else launch_rows<GP, 12, 1, false>(a, s);
}

template <int GP>
int launch(const Int4Args& a, const Int4Plan& p, bool gate, hipStream_t s) {
  if (p.rows) {
    dispatch_rows<GP>(a, gate, s);
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
  }
  const int per = gate ? kTileWaves : 2 * kTileWaves;
  const dim3 grid((unsigned)((a.units + per - 1) / per),
                  (unsigned)((a.rows + kTileRows - 1) / kTileRows), (unsigned)p.nsplit);
  const dim3 block(64 * kTileWaves * p.halves);
  if (p.halves == 2) {
    if (gate) hipLaunchKernelGGL((k_int4_tile<GP, true, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_int4_tile<GP, false, 2>), grid, block, 0, s, a);
  } else {
    if (gate) hipLaunchKernelGGL((k_int4_tile<GP, true, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_int4_tile<GP, false, 1>), grid, block, 0, s, a);
  }
  if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  if (p.nsplit > 1) {
    const int64_t quads = (int64_t)a.units * 4 * a.rows;
    const dim3 jg((unsigned)((quads + 255) / 256));
    if (gate) hipLaunchKernelGGL(k_int4_join<true>, jg, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_int4_join<false>, jg, dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  }
  return HS_OK;
}

bool sizes_ok(int rows, int K, int N, int group, int epilogue) {
  return rows >= 1 && K >= 1 && N >= 1 && (group == 32 || group == 64 || group == 128) &&
         K % group == 0 && (epilogue == HS_LINEAR_PLAIN || epilogue == HS_LINEAR_SWIGLU);
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

size_t hs_linear_int4_workspace_size(int rows, int in_features, int out_features, int epilogue) {
  if (!sizes_ok(rows, in_features, out_features, 32, epilogue) || rows > (1 << 20)) return 0;
  return plan_of(rows, in_features, out_features, epilogue == HS_LINEAR_SWIGLU).bytes;
}

int hs_linear_int4(const void* x, int64_t x_stride, const void* packed, const void* scales,
                   int rows, int in_features, int out_features, int group, int epilogue, void* out,
                   int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows == 0) return HS_OK;
  if (!x || !packed || !scales || !out) return HS_ERR_INVALID;
  if (!sizes_ok(rows, in_features, out_features, group, epilogue)) return HS_ERR_INVALID;
  const bool gate = epilogue == HS_LINEAR_SWIGLU;
  // gate and up halves start at a tile each
  if (gate && out_features % 16) return HS_ERR_UNSUPPORTED;
  // grids and 32-bit element counts of the kernels
  if (rows > (1 << 20) || in_features > (1 << 23) || out_features > (1 << 24))
    return HS_ERR_UNSUPPORTED;
  if ((x_stride % 8) || x_stride < in_features || out_stride < out_features)
    return HS_ERR_UNSUPPORTED;
  if (x_stride > (1 << 23)) return HS_ERR_UNSUPPORTED;  // 64 rows within 1 GiB
  if (((uintptr_t)x | (uintptr_t)packed) & 15) return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)scales & 7) || ((uintptr_t)out & 1)) return HS_ERR_UNSUPPORTED;
  const Int4Plan p = plan_of(rows, in_features, out_features, gate);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return HS_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HS_ERR_UNSUPPORTED;
  Int4Args a;
  a.x = static_cast<const uint16_t*>(x);
  a.xs = x_stride;
  a.w = static_cast<const uint4*>(packed);
  a.sc = static_cast<const uint16_t*>(scales);
  a.rows = rows;
  a.K = in_features;
  a.N = out_features;
  a.steps = (in_features + kStep - 1) / kStep;
  a.units = (out_features + 15) / 16;
  a.up = a.units;
  a.y = static_cast<uint16_t*>(out);
  a.ys = out_stride;
  a.part = static_cast<float*>(workspace);
  a.split_steps = p.split_steps;
  a.nsplit = p.nsplit;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (group == 128) return launch<1>(a, p, gate, s);
  if (group == 64) return launch<2>(a, p, gate, s);
  return launch<4>(a, p, gate, s);
}

}  // extern "C"
