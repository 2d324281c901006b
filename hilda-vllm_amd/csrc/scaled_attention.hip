// Attention over an 8-bit (e4m3fn) paged KV cache with one f32 scale per group of
// tokens and kv head (written by scaled_kv.hip): decode, verify and prompt rows,
// causal with bottom-right alignment (query token i of a sequence with Lq queries
// and Lk keys sees keys 0 .. Lk - Lq + i), grouped heads, head size 128:
//   s_ij = softmax_scale * ks[g(j)] * <q_i, kc_j>
//   o_i  = sum_j p_ij vs[g(j)] vc_j / sum_j p_ij,  p_ij = exp(s_ij - max_j s_ij)
// Codes are decoded exactly to bf16 (every e4m3 value is one) and multiplied on
// the matrix cores with f32 accumulation; a window of 32 keys lies in one group,
// so its scales are two scalars: ks joins the softmax scale, and the power of two in vs
// the decoding of V (what a scale of another producer has besides is the unit that the
// outputs are kept in). Statistics, sums and partial results are f32. The probabilities are
// the product's second operand: in two bf16 parts (16 bits and more) for decode and verify
// rows and prompts of one tile a wave, where the second product is hidden by the loads (64
// verify steps 41.9 us, 41.6 us in one part; 32 decodes 85.7 and 85.4; one prompt of 509
// tokens 18.1 and 17.5). Longer prompts are bound by the vector and matrix pipes and round
// them to bf16 once (the listed prompts 175 us, 225 us in two parts): their error against
// 64-bit sums is 1.85e-3 of the outputs' size, root mean square, where the output's own
// rounding is 1.66e-3. The sum below takes the same rounded ones. (Scales that differ by more
// than powers of two from group to group cost long prompts the change of unit in every
// group: the listed prompts 209 us, 185 us with a second rounding of the weights instead.)
//
// A wave works on its own, without LDS in its loop. It takes a window's K rows as
// the A operand of S^T = K Q^T (lane l: key l % 16, dims 32 (l / 16) .. + 31, two
// 16-byte loads) and its V rows as 8 keys x 8 dims a lane (8 loads of 8 bytes, 16
// lanes to a cache line); byte permutes transpose those 8 x 8 codes in registers
// into the A operand of O^T = V^T P^T, whose key order is chosen so that the lane's
// own probabilities are its B operand. A window's K registers take the next window's K
// as soon as its scores are there, its V registers the next V after its product, so a
// window costs 32 registers and enough waves fit to hide the loads.
//
//  * k_scaled_split: decode and verify rows, 16 query rows (head of the kv head's
//    group, token) to a tile. A workgroup of 4 waves takes `split_len` keys of a
//    (sequence, kv head, tile), its waves interleaved over the windows, and joins
//    their results in LDS; k_scaled_combine joins the splits' partials. The partials
//    are written before they are read and nothing is counted between the launches,
//    so the workspace needs no preparation.
//    It is bound by the cache's stream, which it reads once: 256 decodes of 64 to 2048
//    keys of 8 heads 124 us (4.5 TB/s), 32 of 2048 to 8192 86 us (4.0), 64 verify steps of
//    64 to 2048 keys 41.9 us (3.4, of which the join's launch is about 5).
//  * k_scaled_rows: prompts. A wave takes 16 QT query rows and all of their keys; bound by
//    decoding and the softmax beside the products (prompts of up to 2043 tokens behind up
//    to 1000 keys: 176 us, 633 TFLOP/s). A call's longest prompt chooses the kernel for all of its
//    sequences: decodes beside a prompt are not split (31 of 8192 keys with one prompt of 130
//    tokens: 288 us, 115 us the decodes alone).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/hilda_spec.h"
#include "hs_model_dev.h"

namespace hs {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kD = 128;    // head size
constexpr int kWin = 32;   // keys of a window
constexpr int kRows = 16;  // query rows of a tile
constexpr int kSplitWaves = 4;
constexpr int kRowWaves = 4;

struct ScaledAttnArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  int64_t c_sb, c_st, c_sh;
  const float* ks;
  const float* vs;
  int64_t s_sb, s_sg, s_sh;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_width, num_blocks;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int num_seqs, Hkv, G, block_size;
  int bs_shift;  // log2(block_size) for powers of two, else -1
  int g_shift;   // log2(group)
  float scale_log2;  // softmax_scale * log2(e)
  uint16_t* out;
  int64_t o_st, o_sh;
  int qtiles, nsplit, split_len;
  float* part_o;   // [sequence, kv head, tile, split][16][128]
  float* part_ml;  // [sequence, kv head, tile, split][16][2]
};

// Sequence b's first query row and lengths, as the caller gives them: its query rows lie
// within q and out. Its keys go through the block table, which is checked entry by entry.
struct Seq {
  int qs, Lq, Lk;
};
__device__ __forceinline__ Seq seq_of(const ScaledAttnArgs& a, int b) {
  Seq s;
  s.qs = a.cu_q[b];
  s.Lq = a.cu_q[b + 1] - s.qs;
  s.Lk = a.cu_k[b + 1] - a.cu_k[b];
  return s;
}

// keys that row r (of the sequence's Lq * G) sees
__device__ __forceinline__ int row_keys(const Seq& s, int G, int r) {
  const int n = s.Lk - s.Lq + r / G + 1;
  return n < 0 ? 0 : (n > s.Lk ? s.Lk : n);
}

__device__ __forceinline__ float quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// two codes (of the lower or upper half) times the power of two in `scale`
__device__ __forceinline__ uint32_t bf16_pair(uint32_t codes, bool high, float scale) {
  const bf16x2_t p = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false);
  return __builtin_bit_cast(uint32_t, p);
}
typedef float f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t));
}
union Frag {
  uint32_t u[4];
  bf16x8_t v;
};
__device__ __forceinline__ bf16x8_t decode8(uint32_t lo, uint32_t hi) {
  Frag f;
  f.u[0] = bf16_pair(lo, false, 1.0f);
  f.u[1] = bf16_pair(lo, true, 1.0f);
  f.u[2] = bf16_pair(hi, false, 1.0f);
  f.u[3] = bf16_pair(hi, true, 1.0f);
  return f.v;
}

// A window as a lane holds it. K: rows l % 16 and 16 + l % 16, 32 bytes each. V: 8
// bytes (dims 8 (l % 16) ..) of keys 4g + e and 16 + 4g + e, g = l / 16, e < 4.
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
struct Win {
  u32x4_t k[4];
  u32x2_t v[8];
};

__device__ __forceinline__ int block_of(const ScaledAttnArgs& a, int key) {
  return a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
}

// The K or V rows of a window: `rows` rows from row `off` of block `blk`. The buffer ends
// behind its last row, so further ones read as zeros and, with none, the loads touch no
// memory: every window's loads are issued alike, whatever is left.
struct Source {
  int64_t base;
  int bytes;
};
__device__ __forceinline__ Source source_of(const ScaledAttnArgs& a, int head, int blk, int off,
                                            int rows) {
  Source s;
  s.base = (int64_t)blk * a.c_sb + (int64_t)off * a.c_st + (int64_t)head * a.c_sh;
  s.bytes = rows > 0 ? (min(rows, kWin) - 1) * (int)a.c_st + kD : 0;
  return s;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* cache, const Source& s) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(cache + s.base), 0, s.bytes,
                                           0x00027000);
}
// `at`: the lane's first offset, c * stride + 32 g for K and 4 g * stride + 8 c for V
// (c = l % 16). The others are sums that are cheaper than the registers to keep them in,
// so the compiler may not take them out of the loop.
__device__ __forceinline__ void load_k(const ScaledAttnArgs& a, const Source& s, int at, Win& w) {
  const auto r = buffer_of(a.kc, s);
  const int st = (int)a.c_st;
  asm volatile("" : "+v"(at));
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w.k[2 * t] = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * t * st, 0, 0);
    w.k[2 * t + 1] = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * t * st + 16, 0, 0);
  }
}
__device__ __forceinline__ void load_v(const ScaledAttnArgs& a, const Source& s, int at, Win& w) {
  const auto r = buffer_of(a.vc, s);
  const int st = (int)a.c_st;
  asm volatile("" : "+v"(at));
#pragma unroll
  for (int e = 0; e < 8; ++e)
    w.v[e] = __builtin_amdgcn_raw_buffer_load_b64(r, at + ((e & 4) * 4 + (e & 3)) * st, 0, 0);
}

// The V^T operand of dims 8 i + db (i = l % 16), db = 0 .. 7, from the lane's 8 x 8
// codes times the power of two in `scale`; emit(db, operand).
template <typename F>
__device__ __forceinline__ void transposed(const u32x2_t (&v)[8], float scale, F emit) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // keys (2 p, 2 p + 1) of dims 4 w + 2 h and the next
      const uint32_t sel = h ? 0x03070206u : 0x01050004u;
      uint32_t m[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t x = w ? v[2 * p].y : v[2 * p].x, y = w ? v[2 * p + 1].y : v[2 * p + 1].x;
        m[p] = __builtin_amdgcn_perm(x, y, sel);
      }
      Frag f;
#pragma unroll
      for (int p = 0; p < 4; ++p) f.u[p] = bf16_pair(m[p], false, scale);
      emit(4 * w + 2 * h, f.v);
#pragma unroll
      for (int p = 0; p < 4; ++p) f.u[p] = bf16_pair(m[p], true, scale);
      emit(4 * w + 2 * h + 1, f.v);
    }
  }
}

// 0xff in every byte of x that is a NaN code
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) {
  const uint32_t t = (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return t * 255u;
}

// The state of 16 QT query rows: per tile the lane's row (l % 16) has its maximum
// (log2 domain), its sum (in every element of l) and O[d = 32 (l / 16) + 8 j + db] in
// o[db][j], in units of `unit`.
template <int QT>
struct Rows {
  bf16x8_t q[QT][4];
  int lim[QT];  // keys that the row sees
  float m[QT], unit;
  f32x4_t l[QT], o[QT][8];
};

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// A window's v scale: the power of two in |vs|, which V's decoding takes for nothing, times
// the outputs' unit, 1 or what else a scale of another producer has (so that no probability
// is rounded again), times `rest`, which multiplies the probabilities. That is 1 but for
// scales that are zero, subnormal or not finite.
struct Split {
  float scale, unit, rest;
};
__device__ __forceinline__ Split split_of(float vs, float unit) {
  const uint32_t bits = __float_as_uint(vs), size = bits & 0x7fffffffu;
  if (size >= 0x00800000u && size < 0x7f800000u)
    return {__uint_as_float(size), __uint_as_float((bits & 0x807fffffu) | 0x3f800000u), 1.0f};
  if (size && size < 0x00800000u) return {0x1p-100f, unit, uniform(vs * 0x1p100f / unit)};
  return {1.0f, unit, uniform(vs / unit)};
}

template <int QT>
__device__ __forceinline__ void to_unit(float unit, Rows<QT>& R) {
  const float ratio = uniform(R.unit / unit);
#pragma unroll
  for (int u = 0; u < QT; ++u)
#pragma unroll
    for (int db = 0; db < 8; ++db) R.o[u][db] *= ratio;
  R.unit = unit;
}

template <int QT>
__device__ __forceinline__ void load_rows(const ScaledAttnArgs& a, const Seq& s, int head, int r0,
                                          int lane, Rows<QT>& R) {
  const int n = lane & 15, g = lane >> 4;
  R.unit = 1.0f;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = r0 + 16 * t + n;
    const bool live = r < s.Lq * a.G;
    R.lim[t] = live ? row_keys(s, a.G, r) : 0;
    R.m[t] = -INFINITY;
    R.l[t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int db = 0; db < 8; ++db) R.o[t][db] = f32x4_t{0, 0, 0, 0};
    const uint16_t* p = a.q;
    if (live)
      p += (int64_t)(s.qs + r / a.G) * a.q_st + (int64_t)(head * a.G + r % a.G) * a.q_sh + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (live) x = *reinterpret_cast<const uint4*>(p + 8 * i);
      R.q[t][i] = __builtin_bit_cast(bf16x8_t, x);
    }
  }
}

// S^T of a window: scores of keys 16 t + 4 g + j in s[u][t][j].
template <int QT>
__device__ __forceinline__ void scores(const Win& w, const Rows<QT>& R, f32x4_t (&s)[QT][2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4_t k = w.k[2 * t + (i >> 1)];
      const bf16x8_t ka = (i & 1) ? decode8(k.z, k.w) : decode8(k.x, k.y);
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const f32x4_t z = i ? s[u][t] : f32x4_t{0, 0, 0, 0};
        s[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, R.q[u][i], z, 0, 0, 0);
      }
    }
  }
}

// P^T as the product's operand: one bf16 part, or two whose sum is the probability
template <bool kTwo>
struct Probs {
  bf16x8_t part[kTwo ? 2 : 1];
};
template <bool kTwo>
__device__ __forceinline__ Probs<kTwo> probs_of(const float (&y)[8]) {
  Probs<kTwo> p;
  Frag f, rest;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f.u[e >> 1] = pk_bf16(y[e], y[e + 1]);
    if constexpr (kTwo)
      rest.u[e >> 1] = pk_bf16(y[e] - __uint_as_float(f.u[e >> 1] << 16),
                               y[e + 1] - __uint_as_float(f.u[e >> 1] & 0xffff0000u));
  }
  p.part[0] = f.v;
  if constexpr (kTwo) p.part[1] = rest.v;
  return p;
}
// c += a P^T
template <bool kTwo>
__device__ __forceinline__ f32x4_t times(bf16x8_t a, const Probs<kTwo>& p, f32x4_t c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p.part[0], c, 0, 0, 0);
  if constexpr (kTwo) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p.part[1], c, 0, 0, 0);
  return c;
}
template <int QT>
using WindowProbs = Probs<QT == 1>;

// The softmax step of the scores (times c), and the probabilities as P^T. kMask: some row may
// not see some key. A key that a row does not see takes no part in that row, whatever its
// codes and scales are: its probability is 0. Bit e of seen[u]: the row sees the lane's e-th
// key. The sum adds the probabilities as they are multiplied, in their bf16 parts, on the
// matrix cores (a row of ones), so that the weights of an output add up to one.
template <int QT, bool kMask>
__device__ __forceinline__ void weigh(const f32x4_t (&s)[QT][2], float c, int ws,
                                      int rows, int g, Rows<QT>& R, WindowProbs<QT> (&p)[QT],
                                      uint32_t (&seen)[QT]) {
  Frag one;
  one.u[0] = one.u[1] = one.u[2] = one.u[3] = 0x3f803f80u;
  const bf16x8_t ones = one.v;
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    seen[u] = 0xff;
    if constexpr (kMask) {
      // keys 4 g + j and 16 + 4 g + j of the window's first `rows`, below the row's limit
      const int left = min(R.lim[u] - ws, rows) - 4 * g;
      const uint32_t lo = left >= 4 ? 15u : (left <= 0 ? 0u : (1u << left) - 1);
      const uint32_t hi = left >= 20 ? 15u : (left <= 16 ? 0u : (1u << (left - 16)) - 1);
      seen[u] = lo | (hi << 4);
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = s[u][e >> 2][e & 3] * c;
      if constexpr (kMask) y[e] = (seen[u] >> e) & 1u ? y[e] : -INFINITY;
    }
    const float most = quad_max(fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])),
                                      fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7]))));
    const float m = fmaxf(R.m[u], most);
    const float ref = m == -INFINITY ? 0.0f : m;
    if (__any(m > R.m[u])) {
      const float f = __builtin_amdgcn_exp2f(R.m[u] - ref);
      R.l[u] *= f;
#pragma unroll
      for (int db = 0; db < 8; ++db) R.o[u][db] *= f;
      R.m[u] = m;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(y[e] - ref);
    p[u] = probs_of<QT == 1>(y);
    R.l[u] = times(ones, p[u], R.l[u]);
  }
}

// the probabilities times `rest`, where the rows see the keys
template <int QT>
__device__ __forceinline__ void multiply(float rest, const uint32_t (&seen)[QT],
                                         WindowProbs<QT> (&p)[QT]) {
#pragma unroll
  for (int u = 0; u < QT; ++u) {
#pragma unroll
    for (int h = 0; h < (int)(sizeof(p[u].part) / sizeof(bf16x8_t)); ++h) {
      // a second part is all of nothing where the product is not finite
      const bool none = h && !(fabsf(rest) < INFINITY);
      Frag f;
      f.v = p[u].part[h];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = __uint_as_float(f.u[e >> 1] << 16) * rest;
        const float b = __uint_as_float(f.u[e >> 1] & 0xffff0000u) * rest;
        f.u[e >> 1] = pk_bf16((seen[u] >> e) & 1u && !none ? a : 0.0f,
                              (seen[u] >> (e + 1)) & 1u && !none ? b : 0.0f);
      }
      p[u].part[h] = f.v;
    }
  }
}

// O^T += V^T P^T
template <int QT>
__device__ __forceinline__ void gather(const Win& w, float scale, const WindowProbs<QT> (&p)[QT],
                                       Rows<QT>& R) {
  transposed(w.v, scale, [&](int db, bf16x8_t va) {
#pragma unroll
    for (int u = 0; u < QT; ++u) R.o[u][db] = times(va, p[u], R.o[u][db]);
  });
}

// Takes the NaN codes, which a probability of zero does not cancel, out of V; true where
// there is one.
__device__ __forceinline__ bool drop_nan(Win& w) {
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const u32x2_t bad = {nan_bytes(w.v[e].x), nan_bytes(w.v[e].y)};
    w.v[e] &= ~bad;
    any |= bad.x | bad.y;
  }
  return __any(any != 0);
}

// Gives the NaN codes of V (as loaded) to the rows that see them, by a product of their
// own: 1 for a NaN code by 1 for a key that is seen.
template <int QT>
__device__ __forceinline__ void spread_nan(Win& w, const uint32_t (&seen)[QT], Rows<QT>& R) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    w.v[e] = u32x2_t{nan_bytes(w.v[e].x) & 0x38383838u, nan_bytes(w.v[e].y) & 0x38383838u};
#pragma unroll
  for (int u = 0; u < QT; ++u) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      f.u[e >> 1] = ((seen[u] >> e) & 1u ? 0x3f80u : 0u) |
                    ((seen[u] >> (e + 1)) & 1u ? 0x3f800000u : 0u);
    transposed(w.v, 1.0f, [&](int db, bf16x8_t va) {
      const f32x4_t n =
          __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, f.v, f32x4_t{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n[j] > 0.0f) R.o[u][db][j] = NAN;
    });
  }
}

// The windows of a walk, 64 at a time: lane i has looked up the i-th one's block (-1: the
// table has none there) and scales, so that no window waits for its own.
struct Batch {
  int n, ws0, stride, hi;
  int blk, off;
  float ks, vs;
};
__device__ __forceinline__ Batch look_up(const ScaledAttnArgs& a, const int32_t* bt, int head,
                                         int lane, int ws0, int stride, int hi) {
  Batch t;
  t.n = min(64, (hi - ws0 + stride - 1) / stride);
  t.ws0 = ws0;
  t.stride = stride;
  t.hi = hi;
  const int ws = ws0 + min(lane, t.n - 1) * stride, col = block_of(a, ws);
  t.off = ws - col * a.block_size;
  t.blk = col < a.bt_width ? bt[col] : -1;
  if (t.blk >= a.num_blocks || t.blk < 0) t.blk = -1;
  const int64_t at = (int64_t)max(t.blk, 0) * a.s_sb + (int64_t)(t.off >> a.g_shift) * a.s_sg +
                     (int64_t)head * a.s_sh;
  t.ks = a.ks[at];
  t.vs = a.vs[at];
  return t;
}
// rows of window i: none past the last window, and of a window without a block
__device__ __forceinline__ Source source(const ScaledAttnArgs& a, const Batch& t, int head, int i) {
  const int j = min(i, 63), blk = __builtin_amdgcn_readlane(t.blk, j);
  return source_of(a, head, max(blk, 0), __builtin_amdgcn_readlane(t.off, j),
                   i < t.n && blk >= 0 ? t.hi - (t.ws0 + i * t.stride) : 0);
}

// Window i, in registers, and the loads of the next one.
template <int QT, bool kMask>
__device__ __forceinline__ void window(const ScaledAttnArgs& a, const Batch& t, int head, int i,
                                       int at_k, int at_v, int lane, Win& w, Rows<QT>& R) {
  const int ws = t.ws0 + i * t.stride;
  const Source next = source(a, t, head, i + 1);
  const float ks = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t.ks), i));
  const float vs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t.vs), i));
  // The two steps for scales of another producer stand outside the tiles' loop, where a branch
  // would keep the tiles' steps from overlapping (the listed prompts: 201 us so).
  const Split v = split_of(vs, R.unit);
  if (__float_as_uint(v.unit) != __float_as_uint(R.unit)) to_unit<QT>(v.unit, R);
  f32x4_t s[QT][2];
  scores<QT>(w, R, s);
  load_k(a, next, at_k, w);  // in flight during the rest of this window
  WindowProbs<QT> p[QT];
  uint32_t seen[QT];
  const int rows = __builtin_amdgcn_readlane(t.blk, i) < 0 ? 0 : kWin;
  weigh<QT, kMask>(s, a.scale_log2 * ks, ws, rows, lane >> 4, R, p, seen);
  if (__float_as_uint(v.rest) != __float_as_uint(1.0f)) multiply<QT>(v.rest, seen, p);
  if constexpr (!kMask) {
    gather<QT>(w, v.scale, p, R);
  } else {
    const bool bad = drop_nan(w);
    gather<QT>(w, v.scale, p, R);
    if (bad) {
      load_v(a, source(a, t, head, i), at_v, w);
      spread_nan<QT>(w, seen, R);
    }
  }
  load_v(a, next, at_v, w);  // in flight during the next window's scores
}

// windows of a batch before the first one that some row does not see all of
__device__ __forceinline__ int free_windows(const Batch& t, int full) {
  if (full - t.ws0 < kWin || __any(t.blk < 0)) return 0;
  return min(t.n, (full - t.ws0 - kWin) / t.stride + 1);
}

// Windows at keys ws0, ws0 + stride, ... below hi; `full` is the number of keys that
// every row sees. Windows whose table entry is no block of the cache, or lies past the
// table, are left out.
template <int QT>
__device__ __forceinline__ void walk(const ScaledAttnArgs& a, const int32_t* bt, int head, int lane,
                                     int ws0, int stride, int hi, int full, Rows<QT>& R) {
  const int c = lane & 15, g = lane >> 4, st = (int)a.c_st;
  const int at_k = c * st + 32 * g, at_v = 4 * g * st + 8 * c;
  for (; ws0 < hi; ws0 += 64 * stride) {
    const Batch t = look_up(a, bt, head, lane, ws0, stride, hi);
    const int free = free_windows(t, full);
    Win w;
    const Source first = source(a, t, head, 0);
    load_k(a, first, at_k, w);
    load_v(a, first, at_v, w);
    int i = 0;
    for (; i < free; ++i) window<QT, false>(a, t, head, i, at_k, at_v, lane, w, R);
    for (; i < t.n; ++i) window<QT, true>(a, t, head, i, at_k, at_v, lane, w, R);
  }
  if (__float_as_uint(R.unit) != __float_as_uint(1.0f)) to_unit<QT>(1.0f, R);
}

// row r's 8 outputs of dims d .. d + 7
__device__ __forceinline__ uint16_t* out_row(const ScaledAttnArgs& a, const Seq& s, int head, int r) {
  return a.out + (int64_t)(s.qs + r / a.G) * a.o_st + (int64_t)(head * a.G + r % a.G) * a.o_sh;
}

__global__ __launch_bounds__(64 * kSplitWaves, 3) void k_scaled_split(ScaledAttnArgs a) {
  __shared__ float s_o[kSplitWaves][kRows][kD];
  __shared__ float s_ml[kSplitWaves][kRows][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go round the 8 XCDs in order. The heads of a (sequence, split) go to one of
  // them: side by side in memory, they take all of its L2 channels together. The splits
  // that every sequence has come first, in turn over the XCDs.
  const int tiles = a.Hkv * a.qtiles;
  const int pair = (int)(blockIdx.x >> 3) / tiles * 8 + (blockIdx.x & 7);
  const int at = (int)(blockIdx.x >> 3) % tiles;
  const int head = at % a.Hkv, tile = at / a.Hkv;
  const int split = pair / a.num_seqs, b = pair % a.num_seqs;
  if (split >= a.nsplit) return;
  const Seq s = seq_of(a, b);
  const int r0 = tile * kRows, rows = s.Lq * a.G - r0;  // rows of this tile, and behind it
  if (rows <= 0) return;
  const int live = min(rows, kRows);
  const int keys = row_keys(s, a.G, r0 + live - 1), full = row_keys(s, a.G, r0);
  const int lo = split * a.split_len;
  // the last split also takes the keys past the declared longest sequence
  const int hi = split == a.nsplit - 1 ? keys : min(keys, lo + a.split_len);
  if (lo >= hi && split) return;
  Rows<1> R;
  load_rows<1>(a, s, head, r0, lane, R);
  walk<1>(a, a.bt + (int64_t)b * a.bt_stride, head, lane, lo + wave * kWin, kSplitWaves * kWin, hi,
          full, R);
  const int n = lane & 15, g = lane >> 4;
  if (g == 0) {
    s_ml[wave][n][0] = R.m[0];
    s_ml[wave][n][1] = R.l[0][0];
  }
  if (n < live) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(&s_o[wave][n][32 * g + 8 * j + 4 * h]) =
            make_float4(R.o[0][4 * h][j], R.o[0][4 * h + 1][j], R.o[0][4 * h + 2][j],
                        R.o[0][4 * h + 3][j]);
    }
  }
  __syncthreads();
  // 32 threads a row, 4 dims each
  const int d = 4 * (threadIdx.x & 31);
  for (int row = threadIdx.x >> 5; row < live; row += 2 * kSplitWaves) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSplitWaves; ++w) m = fmaxf(m, s_ml[w][row][0]);
    const float ref = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kSplitWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_ml[w][row][0] - ref);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][row][d]);
      sum += f * s_ml[w][row][1];
      o[0] += f * x.x;
      o[1] += f * x.y;
      o[2] += f * x.z;
      o[3] += f * x.w;
    }
    if (a.nsplit == 1 || keys <= a.split_len) {  // the tile's only split
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint2 y;
      y.x = (uint32_t)to_bf(o[0] * inv) | ((uint32_t)to_bf(o[1] * inv) << 16);
      y.y = (uint32_t)to_bf(o[2] * inv) | ((uint32_t)to_bf(o[3] * inv) << 16);
      *reinterpret_cast<uint2*>(out_row(a, s, head, r0 + row) + d) = y;
    } else {
      const int64_t slot = (((int64_t)b * a.Hkv + head) * a.qtiles + tile) * a.nsplit + split;
      *reinterpret_cast<float4*>(a.part_o + (slot * kRows + row) * kD + d) =
          make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) {
        a.part_ml[(slot * kRows + row) * 2] = m;
        a.part_ml[(slot * kRows + row) * 2 + 1] = sum;
      }
    }
  }
}

// Joins the splits of 8 / P query rows: 32 threads a row and part of the splits (P: parts).
template <int P>
__global__ __launch_bounds__(256) void k_scaled_combine(ScaledAttnArgs a) {
  __shared__ float s_o[8][kD];
  __shared__ float s_ml[8][2];
  const int head = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv, b = blockIdx.y;
  const int part = (threadIdx.x >> 5) % P, d = 4 * (threadIdx.x & 31);
  const int row = blockIdx.z * (8 / P) + (threadIdx.x >> 5) / P;
  const Seq s = seq_of(a, b);
  const int r0 = tile * kRows, rows = s.Lq * a.G - r0;
  if (row >= rows) return;
  const int keys = row_keys(s, a.G, r0 + min(rows, kRows) - 1);
  if (keys <= a.split_len) return;  // written by its only split
  const int n = min(a.nsplit, (keys + a.split_len - 1) / a.split_len);
  const int64_t slot0 = (((int64_t)b * a.Hkv + head) * a.qtiles + tile) * a.nsplit;
  float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = part; i < n; i += P) {
    const int64_t at = (slot0 + i) * kRows + row;
    const float mi = a.part_ml[2 * at], li = a.part_ml[2 * at + 1];
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * kD + d);
    const float mn = fmaxf(m, mi), ref = mn == -INFINITY ? 0.0f : mn;
    const float f = __builtin_amdgcn_exp2f(m - ref), fi = __builtin_amdgcn_exp2f(mi - ref);
    m = mn;
    l = l * f + li * fi;
    o[0] = o[0] * f + x.x * fi;
    o[1] = o[1] * f + x.y * fi;
    o[2] = o[2] * f + x.z * fi;
    o[3] = o[3] * f + x.w * fi;
  }
  if constexpr (P > 1) {
    *reinterpret_cast<float4*>(&s_o[part][d]) = make_float4(o[0], o[1], o[2], o[3]);
    if (d == 0) s_ml[part][0] = m, s_ml[part][1] = l;
    __syncthreads();
    if (part) return;
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < P; ++i) m = fmaxf(m, s_ml[i][0]);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f;
    o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float f = __builtin_amdgcn_exp2f(s_ml[i][0] - ref);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[i][d]);
      l += f * s_ml[i][1];
      o[0] += f * x.x;
      o[1] += f * x.y;
      o[2] += f * x.z;
      o[3] += f * x.w;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 y;
  y.x = (uint32_t)to_bf(o[0] * inv) | ((uint32_t)to_bf(o[1] * inv) << 16);
  y.y = (uint32_t)to_bf(o[2] * inv) | ((uint32_t)to_bf(o[3] * inv) << 16);
  *reinterpret_cast<uint2*>(out_row(a, s, head, r0 + row) + d) = y;
}

template <int QT>
__global__ __launch_bounds__(64 * kRowWaves, QT == 1 ? 3 : 2) void k_scaled_rows(ScaledAttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // as k_scaled_split's workgroups, with the rows that see most keys first
  const int pair = (int)(blockIdx.x >> 3) / a.Hkv * 8 + (blockIdx.x & 7);
  const int head = (int)(blockIdx.x >> 3) % a.Hkv;
  const int tile = a.qtiles - 1 - pair / a.num_seqs, b = pair % a.num_seqs;
  if (tile < 0) return;
  const Seq s = seq_of(a, b);
  const int total = s.Lq * a.G;
  const int r0 = (tile * kRowWaves + wave) * kRows * QT;
  if (r0 >= total) return;
  Rows<QT> R;
  load_rows<QT>(a, s, head, r0, lane, R);
  walk<QT>(a, a.bt + (int64_t)b * a.bt_stride, head, lane, 0, kWin,
           row_keys(s, a.G, min(total, r0 + kRows * QT) - 1), row_keys(s, a.G, r0), R);
  const int n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float l = R.l[t][0];
    const int r = r0 + 16 * t + n;
    if (r >= total) continue;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* y = out_row(a, s, head, r) + 32 * g;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint16_t h[8];
#pragma unroll
      for (int db = 0; db < 8; ++db) h[db] = to_bf(R.o[t][db][j] * inv);
      *reinterpret_cast<uint4*>(y + 8 * j) = pack8(h);
    }
  }
}

struct ScaledPlan {
  int qt;  // tiles of a wave of k_scaled_rows, 0: k_scaled_split
  int qtiles, nsplit, split_len;
  size_t bytes;
};

ScaledPlan plan_of(int num_seqs, int Hkv, int G, int max_q, int max_k) {
  ScaledPlan p;
  const int64_t rows = (int64_t)max_q * G;
  const int64_t q = (rows + kRows - 1) / kRows;
  p.qtiles = (int)q;
  p.nsplit = 1;
  p.split_len = INT32_MAX;
  p.bytes = 0;
  const int64_t tiles = (int64_t)num_seqs * Hkv * q;
  // Prompts take k_scaled_rows once their tiles fill half the chip's SIMDs without
  // splitting keys (one prompt of 33 tokens, 72 tiles, behind 967 keys: 18.9 us split,
  // 26.7 us not). More tiles to a wave share a window's loads and decoding as long as the
  // waves still fill the chip: 509 tokens, 1024 tiles, take 17.4 / 20.9 / 25.4 us with 1 /
  // 2 / 3, 2000 tokens of 16 heads, 2000 tiles, 124 / 82 / 103 us, and 3500 of 32 heads,
  // 7100 tiles, 353 / 198 / 173 us.
  p.qt = tiles < 512 || rows <= 64 ? 0 : (tiles >= 6144 ? 3 : (tiles >= 1536 ? 2 : 1));
  if (p.qt) return p;
  // about 512 workgroups if every sequence is as long as declared, of at least one window
  // a wave and at most 512 keys (an eighth of the longest sequence up to 1024, so that long
  // ones leave few parts) unless that makes more than 4096 of them. 64 verify steps of 64
  // to 2048 keys: 41.4 us, 44.2 us with 1024 keys; 32 decodes of 2048 to 8192: 84.2 us,
  // 86.4 us with 512; one verify step of 40001 keys: 26.9 us, 28.3 us with 1024 workgroups.
  int64_t len = (max_k * tiles + 511) / 512;
  const int cap = max_k / 8 < 512 ? 512 : (max_k / 8 > 1024 ? 1024 : max_k / 8);
  if (len > cap) len = cap;
  const int64_t floor_len = (max_k * tiles + 4095) / 4096;
  if (len < floor_len) len = floor_len;
  // short sequences in one launch (16 verify steps of 500 keys: 10.2 us, 15.1 us split; one:
  // 8.9 us, 9.6 us), also up to 1024 keys where there are tiles enough (16 of up to 1000:
  // 12.7 us, 16.6 us split; with 4: 12.2 us, 11.5 us split)
  if (max_k <= 512 || (max_k <= 1024 && tiles >= 128)) len = max_k;
  const int64_t unit = kSplitWaves * kWin;
  len = (len + unit - 1) / unit * unit;
  p.split_len = (int)(len > INT32_MAX / 2 ? INT32_MAX / 2 : len);
  p.nsplit = (int)((max_k + (int64_t)p.split_len - 1) / p.split_len);
  if (p.nsplit > 1) p.bytes = (size_t)tiles * p.nsplit * kRows * (kD + 2) * sizeof(float);
  return p;
}

}  // namespace
}  // namespace hs

using namespace hs;

extern "C" {

size_t hs_verify_attention_scaled_workspace_size(int num_seqs, int num_q_heads, int num_kv_heads,
                                                 int max_seqlen_q, int max_seqlen_k) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || max_seqlen_q <= 0 ||
      max_seqlen_k <= 0)
    return 0;
  return plan_of(num_seqs, num_kv_heads, num_q_heads / num_kv_heads, max_seqlen_q, max_seqlen_k)
      .bytes;
}

int hs_verify_attention_scaled(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
    const void* v_cache, int64_t cache_stride_block, int64_t cache_stride_tok,
    int64_t cache_stride_head, const float* k_scales, const float* v_scales,
    int64_t scale_stride_block, int64_t scale_stride_group, int64_t scale_stride_head, int group,
    const int32_t* block_tables, int64_t block_table_stride, int block_table_width, int num_blocks,
    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int num_seqs, int max_seqlen_q,
    int max_seqlen_k, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
    float softmax_scale, void* out, int64_t out_stride_tok, int64_t out_stride_head,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !k_scales || !v_scales || !block_tables || !cu_seqlens_q ||
      !cu_seqlens_k || !out)
    return HS_ERR_INVALID;
  if (num_seqs <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_seqlen_q <= 0 ||
      max_seqlen_k <= 0 || num_blocks <= 0 || block_size <= 0 || group <= 0 ||
      block_table_width <= 0 || block_table_stride < block_table_width)
    return HS_ERR_INVALID;
  if (num_q_heads % num_kv_heads || block_size % group) return HS_ERR_INVALID;
  if (head_dim != kD) return HS_ERR_UNSUPPORTED;
  if (group != 32 && group != 64 && group != 128 && group != 256) return HS_ERR_UNSUPPORTED;
  const int G = num_q_heads / num_kv_heads;
  if (G > kRows) return HS_ERR_UNSUPPORTED;
  if ((q_stride_tok % 8) || (q_stride_head % 8) || (out_stride_tok % 8) || (out_stride_head % 8))
    return HS_ERR_UNSUPPORTED;
  if ((cache_stride_block % 16) || (cache_stride_tok % 16) || (cache_stride_head % 16))
    return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15)
    return HS_ERR_UNSUPPORTED;
  if (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3) return HS_ERR_UNSUPPORTED;
  // a window's rows lie within 2 GiB of its first (32-bit offsets of the lanes)
  if (cache_stride_tok < kD || cache_stride_tok > INT32_MAX / (2 * kWin)) return HS_ERR_UNSUPPORTED;
  const ScaledPlan p = plan_of(num_seqs, num_kv_heads, G, max_seqlen_q, max_seqlen_k);
  const int64_t tiles = (int64_t)num_kv_heads * p.qtiles;
  if (num_seqs > 65535 || (int64_t)max_seqlen_q * G > INT32_MAX / 2 || num_kv_heads > 65535)
    return HS_ERR_UNSUPPORTED;
  if (p.bytes && (!workspace || workspace_bytes < p.bytes)) return HS_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return HS_ERR_UNSUPPORTED;
  ScaledAttnArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.kc = static_cast<const uint8_t*>(k_cache);
  a.vc = static_cast<const uint8_t*>(v_cache);
  a.c_sb = cache_stride_block;
  a.c_st = cache_stride_tok;
  a.c_sh = cache_stride_head;
  a.ks = k_scales;
  a.vs = v_scales;
  a.s_sb = scale_stride_block;
  a.s_sg = scale_stride_group;
  a.s_sh = scale_stride_head;
  a.bt = block_tables;
  a.bt_stride = block_table_stride;
  a.bt_width = block_table_width;
  a.num_blocks = num_blocks;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs;
  a.Hkv = num_kv_heads;
  a.G = G;
  a.block_size = block_size;
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz((unsigned)block_size) : -1;
  a.g_shift = __builtin_ctz((unsigned)group);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_stride_tok;
  a.o_sh = out_stride_head;
  a.qtiles = p.qtiles;
  a.nsplit = p.nsplit;
  a.split_len = p.split_len;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o + (size_t)num_seqs * tiles * p.nsplit * kRows * kD;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p.qt) {
    const int64_t per = (int64_t)kRows * p.qt * kRowWaves;
    a.qtiles = (int)(((int64_t)max_seqlen_q * G + per - 1) / per);
    const int64_t groups = ((int64_t)num_seqs * a.qtiles + 7) / 8 * 8 * num_kv_heads;
    if (groups > INT32_MAX) return HS_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)groups), block(64 * kRowWaves);
    if (p.qt == 3) hipLaunchKernelGGL(k_scaled_rows<3>, grid, block, 0, st, a);
    else if (p.qt == 2) hipLaunchKernelGGL(k_scaled_rows<2>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(k_scaled_rows<1>, grid, block, 0, st, a);
    return hipGetLastError() == hipSuccess ? HS_OK : HS_ERR_LAUNCH;
  }
  const int64_t groups = ((int64_t)num_seqs * p.nsplit + 7) / 8 * 8 * tiles;
  if (groups > INT32_MAX) return HS_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(k_scaled_split, dim3((unsigned)groups), dim3(64 * kSplitWaves), 0, st, a);
  if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  if (p.nsplit > 1) {
    // a workgroup for 8 rows, or for each where there are many splits to share out
    if (p.nsplit <= 8)
      hipLaunchKernelGGL(k_scaled_combine<1>, dim3((unsigned)tiles, (unsigned)num_seqs, kRows / 8),
                         dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL(k_scaled_combine<8>, dim3((unsigned)tiles, (unsigned)num_seqs, kRows),
                         dim3(256), 0, st, a);
    if (hipGetLastError() != hipSuccess) return HS_ERR_LAUNCH;
  }
  return HS_OK;
}

}  // extern "C"
