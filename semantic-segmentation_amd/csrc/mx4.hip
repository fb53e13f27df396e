// 4-bit microscaled products (OCP MXFP4): e2m1 values with one power of two per 32 reduction elements on both sides,
//   y[m][n] = sum_b 2^(ex[m][b] - 127) 2^(ew[n][b] - 127) sum_(k in block b) qx[m][k] qw[n][k]
// v_mfma_scale_f32_32x32x64_f8f6f4 takes the codes and the two exponents as they are and sums in float32, so the product needs no
// arithmetic of its own: it is bound by the matrix unit for many rows (four times the bfloat16 rate), by the weights' bytes (half a
// byte each, a quarter of bfloat16's) for few.
// Quantisation: s = the smallest power of two >= 2^-111 with max |x| < 7 s, values rounded to nearest even (v_cvt_scalef32_pk_fp4).
#include "gemm_tile.h"
#include <algorithm>

#include "gate_act.h"

namespace ssmi {

typedef int i32x8 __attribute__((ext_vector_type(8)));
static constexpr int kBlock = 32;

// the block's biased exponent from the largest |x| pattern: 7 / 4 = 1.75, mantissas from there carry into the exponent; 255: not finite
__device__ __forceinline__ unsigned block_exponent(unsigned top) {
  const int e = max((int)((top + 0x200000u) >> 23) - 2, 16);
  return top < 0x7F800000u ? (unsigned)e : 255u;
}
// eight values -> eight codes, element 0 in the lowest half byte
__device__ __forceinline__ unsigned codes_of(const float (&v)[8], unsigned e) {
  if (e == 255u) return 0u;
  const float s = __builtin_bit_cast(float, e << 23);
  unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
}
__device__ __forceinline__ unsigned top_of(const float (&v)[8]) {
  unsigned t = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = max(t, __builtin_bit_cast(unsigned, v[i]) & 0x7FFFFFFFu);
  return t;
}
template <typename T, bool VEC>
__device__ __forceinline__ void take8(const T* p, int n, float (&v)[8]) {
  if constexpr (VEC) {
    const f32x4 a = Act<T>::gld4(p), b = Act<T>::gld4(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Act<T>::gld(p + i) : 0.f;
  }
}

// x [rows][ld] -> codes [rows][16 nb], scales [rows][nb]: four lanes a block, eight values a lane
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx4_quantize_kernel_rows(const T* __restrict__ x, int64_t ld, int64_t rows, int k, int nb, uint8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales) {
  const int64_t all = rows * nb;
  for (int64_t base = (int64_t)blockIdx.x * 64; base < all; base += (int64_t)gridDim.x * 64) {      // lanes of a block stay together
    const int64_t i = base + (threadIdx.x >> 2);
    const int part = threadIdx.x & 3;
    const bool here = i < all;
    const int64_t m = here ? i / nb : 0;
    const int b = here ? (int)(i - m * nb) : 0, at = b * kBlock + part * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (here && at < k) take8<T, VEC>(x + m * ld + at, k - at, v);
    unsigned top = top_of(v);
    top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
    const unsigned e = block_exponent(top);
    if (here) {
      *reinterpret_cast<unsigned*>(codes + (m * nb + b) * 16 + part * 4) = codes_of(v, e);
      if (part == 0) scales[m * nb + b] = (uint8_t)e;
    }
  }
}

// a Keras kernel w [k][n] -> codes and scales of its columns: a lane owns 32 k of one column (neighbouring lanes neighbouring columns)
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel_cols(const T* __restrict__ w, int k, int n, int nb, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), b = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (col >= n || b >= nb) return;
  float v[4][8];
  unsigned top = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int kk = b * kBlock + q * 8 + i;
      v[q][i] = kk < k ? Act<T>::gld(w + (int64_t)kk * n + col) : 0.f;
    }
    top = max(top, top_of(v[q]));
  }
  const unsigned e = block_exponent(top);
  u32x4 o;
#pragma unroll
  for (int q = 0; q < 4; ++q) o[q] = codes_of(v[q], e);
  *reinterpret_cast<u32x4*>(codes + ((int64_t)col * nb + b) * 16) = o;
  scales[(int64_t)col * nb + b] = (uint8_t)e;
}

__global__ __launch_bounds__(256) void mx4_dequantize_kernel_cols(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int k, int n, int nb,
                                                                  float* __restrict__ w) {
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), b = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (col >= n || b >= nb) return;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const unsigned e = scales[(int64_t)col * nb + b];
  const float s = __builtin_bit_cast(float, e == 255u ? 0x7FC00000u : e == 0u ? 0x00400000u : e << 23);      // 0: 2^-127
  for (int q = 0; q < 4; ++q) {
    unsigned c = *reinterpret_cast<const unsigned*>(codes + ((int64_t)col * nb + b) * 16 + q * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c >> (8 * i), 1.0f, 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int kk = b * kBlock + q * 8 + 2 * i + j;
        if (kk < k) w[(int64_t)kk * n + col] = v[j] * s;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------- many rows: tiles of the matrix unit

struct Mx4Args {
  const uint8_t *xc, *xs;                     // quantised x
  const uint8_t *wc[2], *ws[2];               // one weight, or gate and up
  const float* bias[2];
  void* y;
  int64_t rows, y_ld;
  int n, nb, act, vec_out, past;
  unsigned np, nq;
};

// Operand rows of 16 nb bytes of codes, eight blocks (128 bytes) of a row a step, swizzled like the tile engine's rows.  (Four blocks a
// step and twice the workgroups to a CU measured 4 % faster at a reduction of 512, 30 % slower at 4096.)
static constexpr int kBlocks = 8;
template <int N>
struct Mx4Operand {
  static constexpr int kBytes = N * kBlocks * 16, kLoads = kBytes / 4096, kRowsPerLoad = 256 / kBlocks;
  unsigned voff[kLoads];
  int piece;
  __amdgpu_buffer_rsrc_t rsrc;
  static __device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }
  __device__ __forceinline__ void init(const uint8_t* base, int64_t ld, int count) {
    rsrc = make_rsrc(base, 0x7FFFFFFFu);
    const int row = (int)threadIdx.x / kBlocks;
    piece = (int)(threadIdx.x % kBlocks) ^ swizzle(row);      // rows of the other loads lie multiples of sixteen on
#pragma unroll
    for (int j = 0; j < kLoads; ++j) voff[j] = row + kRowsPerLoad * j < count ? (unsigned)((row + kRowsPerLoad * j) * ld) + piece * 16u : kOOB;
  }
  __device__ __forceinline__ void request(lds_bytes lds, int t, int left) const {      // left: blocks from this step on
    const unsigned dst = (unsigned)(uintptr_t)lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) stage16(rsrc, piece < left ? voff[j] : kOOB, (unsigned)t * (kBlocks * 16u), dst + j * 4096);
  }
};

template <int SP, int SQ, bool GATE>
struct Mx4Shape {
  static constexpr int kP = SP * 64, kQ = SQ * 64, kHalf = GATE ? kP / 2 : kP, kRow = kBlocks * 16, kSub = 32 * kRow;
  static constexpr int kStage = (kP + kQ) * kRow, kRows = TileRows<SP, SQ, 64>::kBytes, kLds = 2 * kStage > kRows ? 2 * kStage : kRows;
};

// waves 2 x 2 as in the tile engine; exponents of a step are read from memory straight into registers, one step ahead
template <typename T, int SP, int SQ, bool GATE>
__global__ __launch_bounds__(256, 2) void mx4_kernel(Mx4Args a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  typedef Mx4Shape<SP, SQ, GATE> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, hh = lane >> 5;
  const int wp = wave >> 1, wq = wave & 1;
  const TileAt at = tile_at(spread_blocks(blockIdx.x, gridDim.x), a.np, a.nq);
  const int64_t m0 = (int64_t)at.q * S::kQ;
  const int n0 = at.p * S::kHalf;
  const int64_t ld = 16 * (int64_t)a.nb;
  lds_bytes lds = (lds_bytes)smem;

  Mx4Operand<S::kHalf> w0, w1;
  Mx4Operand<S::kQ> x;
  w0.init(a.wc[0] + n0 * ld, ld, a.n - n0);
  if constexpr (GATE) w1.init(a.wc[1] + n0 * ld, ld, a.n - n0);
  x.init(a.xc + m0 * ld, ld, (int)min((int64_t)S::kQ, a.rows - m0));
  auto request = [&](int t) __attribute__((always_inline)) {
    lds_bytes s = lds + (t & 1) * S::kStage;
    const int left = a.nb - t * kBlocks;
    w0.request(s, t, left);
    if constexpr (GATE) w1.request(s + S::kHalf * S::kRow, t, left);
    x.request(s + S::kP * S::kRow, t, left);
  };
  // rows of this lane's exponents; a row past the end reads the last one (its codes are zeros)
  const uint8_t *sp[SP], *sq[SQ];
#pragma unroll
  for (int i = 0; i < SP; ++i) {
    const int part = GATE ? i / (SP / 2) : 0, sub = GATE ? wp * (SP / 2) + i % (SP / 2) : wp * SP + i;
    sp[i] = a.ws[part] + (int64_t)min(n0 + sub * 32 + r, a.n - 1) * a.nb;
  }
#pragma unroll
  for (int j = 0; j < SQ; ++j) sq[j] = a.xs + min(m0 + (wq * SQ + j) * 32 + r, a.rows - 1) * a.nb;
  // a lane's half of the wave takes the first or the second half of a step's blocks, so its exponents are one (half) word of any alignment
  auto exponents = [&](const uint8_t* p, int t) __attribute__((always_inline)) {
    unsigned v = 0;
    const int at = t * kBlocks + kBlocks / 2 * hh;
    if (t * kBlocks + kBlocks <= a.nb) {
      __builtin_memcpy(&v, p + at, kBlocks / 2);
    } else {      // blocks past the last have zero codes: any of the row's exponents will do
#pragma unroll
      for (int k = 0; k < kBlocks / 2; ++k) v |= (unsigned)p[min(at + k, a.nb - 1)] << (8 * k);
    }
    return (int)v;
  };

  f32x16 acc[SP][SQ];
#pragma unroll
  for (int i = 0; i < SP; ++i)
#pragma unroll
    for (int j = 0; j < SQ; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;

  // The tile engine's loop: fragments one piece ahead of their arithmetic, a step's barrier in front of its last piece, two stages.  The
  // exponents of step t + 2 are asked for in front of its codes, so that waiting for the codes covers them.
  constexpr int kLoads = (S::kP + S::kQ) * S::kRow / 4096;
  const unsigned fr = (unsigned)(r * S::kRow + (((kBlocks / 2 * hh) ^ Mx4Operand<S::kQ>::swizzle(r)) << 4));
  const int steps = (a.nb + kBlocks - 1) / kBlocks;
  struct Exponents { int p[SP], q[SQ]; } e0, e1, e2;
  auto take = [&](Exponents& e, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < SP; ++i) e.p[i] = exponents(sp[i], t);
#pragma unroll
    for (int j = 0; j < SQ; ++j) e.q[j] = exponents(sq[j], t);
  };
  u32x4 p[2][SP], q[2][SQ];
  auto read = [&](int buf, lds_bytes stage, int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const int sub = GATE ? (i / (SP / 2)) * (S::kHalf / 32) + wp * (SP / 2) + i % (SP / 2) : wp * SP + i;
      p[buf][i] = *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(stage + sub * S::kSub + (fr ^ (unsigned)(ks << 4)));
    }
#pragma unroll
    for (int j = 0; j < SQ; ++j)
      q[buf][j] = *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(stage + S::kP * S::kRow + (wq * SQ + j) * S::kSub + (fr ^ (unsigned)(ks << 4)));
  };
  auto multiply = [&](auto which) __attribute__((always_inline)) {
    constexpr int ks = decltype(which)::value, buf = ks & 1;
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
      for (int j = 0; j < SQ; ++j) {
        const i32x8 pa = {(int)p[buf][i][0], (int)p[buf][i][1], (int)p[buf][i][2], (int)p[buf][i][3], 0, 0, 0, 0};
        const i32x8 qa = {(int)q[buf][j][0], (int)q[buf][j][1], (int)q[buf][j][2], (int)q[buf][j][3], 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(pa, qa, acc[i][j], 4, 4, ks, e0.p[i], ks, e0.q[j]);
      }
  };
  take(e0, 0);
  take(e1, min(1, steps - 1));
  e2 = e1;
  request(0);
  if (steps > 1) {
    request(1);
    stage_wait<kLoads>();
  } else {
    stage_wait<0>();
  }
  __syncthreads();
  read(0, lds, 0);
  for (int t = 0; t < steps; ++t) {
    lds_bytes cur = lds + (t & 1) * S::kStage, nxt = lds + ((t + 1) & 1) * S::kStage;
    read(1, cur, 1);
    multiply(ActIs<0>{});
    read(0, cur, 2);
    multiply(ActIs<1>{});
    read(1, cur, 3);
    multiply(ActIs<2>{});
    stage_wait<0>();
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    if (t + 2 < steps) {
      take(e2, t + 2);
      request(t + 2);
    }
    if (t + 1 < steps) read(0, nxt, 0);
    multiply(ActIs<3>{});
    e0 = e1;
    e1 = e2;
  }

  typedef TileRows<SP, SQ, S::kHalf> R;
  const int col = R::col(), f = n0 + col, n = a.n - f;
  float b0[4] = {0.f, 0.f, 0.f, 0.f}, b1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (a.bias[0] && e < n) b0[e] = a.bias[0][f + e];
    if (GATE && a.bias[1] && e < n) b1[e] = a.bias[1][f + e];
  }
  auto pos = [&](int i) __attribute__((always_inline)) { return GATE ? (i / (SP / 2)) * S::kHalf + (wp * (SP / 2) + i % (SP / 2)) * 32 : (wp * SP + i) * 32; };
  const bool whole = m0 + S::kQ <= a.rows && n0 + S::kHalf <= a.n && a.vec_out;
  T* const y = static_cast<T*>(a.y) + m0 * a.y_ld + n0;
  const unsigned lane_at = (unsigned)R::first() * (unsigned)a.y_ld + (unsigned)col;
  with_act(GATE ? a.act : kRelu, [&](auto which) __attribute__((always_inline)) {
    constexpr int kAct = decltype(which)::value;
    auto value = [&](const float* row) __attribute__((always_inline)) {
      f32x4 o = *reinterpret_cast<const f32x4*>(row);
      if constexpr (GATE) {
        const f32x4 u = *reinterpret_cast<const f32x4*>(row + S::kHalf);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = gate_act<T, kAct>(o[e] + b0[e]) * (u[e] + b1[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += b0[e];
      }
      return o;
    };
    if (whole && a.past) {
      R::template run<R::kRounds>(acc, reinterpret_cast<float*>(smem), wq, pos, [](int) {},
                                  [&](const float* row, int qc, int) __attribute__((always_inline)) { put4<T, true>(y + qc * a.y_ld + lane_at, value(row)); });
    } else if (whole) {
      R::template run<R::kRounds>(acc, reinterpret_cast<float*>(smem), wq, pos, [](int) {},
                                  [&](const float* row, int qc, int) __attribute__((always_inline)) { put4<T>(y + qc * a.y_ld + lane_at, value(row)); });
    } else {
      R::template run<1>(acc, reinterpret_cast<float*>(smem), wq, pos, [](int) {}, [&](const float* row, int qc, int) __attribute__((always_inline)) {
        const int64_t m = m0 + R::first() + qc;
        if (m >= a.rows || n <= 0) return;
        const f32x4 v = value(row);
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store4<T>(static_cast<T*>(a.y) + m * a.y_ld + f, o, n, a.vec_out);
      });
    }
  });
}

// ---------------------------------------------------------------------------------------------------------------------- a few rows
// Bound by reading the weights, or by latency: no staging, and x is quantised on the way in (each workgroup does it again, k values
// a row).  The matrix unit multiplies 32 columns by up to 32 rows; a workgroup's four waves share its 32 columns (of both weights when
// gated) and split the reduction, a step of 64 each in turn.
template <typename T, bool GATE, bool VEC>
__global__ __launch_bounds__(256) void mx4_rows_kernel(const T* __restrict__ x, int64_t x_ld, Mx4Args a, int k) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // codes [rows][16 nb + 16], then exponents [rows][nb]
  __shared__ float red[3][GATE ? 2 : 1][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, hh = lane >> 5;
  const int rows = (int)a.rows, ldc = 16 * a.nb + 16;
  uint8_t* const sc = smem + rows * ldc;
  for (int base = 0; base < rows * a.nb; base += 64) {
    const int i = base + ((int)threadIdx.x >> 2), part = threadIdx.x & 3;
    const bool here = i < rows * a.nb;
    const int m = here ? i / a.nb : 0, b = here ? i - m * a.nb : 0, pos = b * kBlock + part * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (here && pos < k) take8<T, VEC>(x + m * x_ld + pos, k - pos, v);
    unsigned top = top_of(v);
    top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
    const unsigned e = block_exponent(top);
    if (here) {
      *reinterpret_cast<unsigned*>(smem + m * ldc + b * 16 + part * 4) = codes_of(v, e);
      if (part == 0) sc[m * a.nb + b] = (uint8_t)e;
    }
  }
  __syncthreads();
  constexpr int kW = GATE ? 2 : 1;
  const int n0 = blockIdx.x * 32, col = min(n0 + r, a.n - 1);
  f32x16 acc[kW];
#pragma unroll
  for (int w = 0; w < kW; ++w)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[w][i] = 0.f;
  const int steps = (a.nb + 1) / 2;
  for (int t = wave; t < steps; t += 4) {
    const int b = 2 * t + hh;
    const bool in = b < a.nb;
    u32x4 q = {0u, 0u, 0u, 0u};
    int eq = 127;
    if (in && r < rows) {
      q = *reinterpret_cast<const u32x4*>(smem + r * ldc + b * 16);
      eq = sc[r * a.nb + b];
    }
    const i32x8 qa = {(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      u32x4 p = {0u, 0u, 0u, 0u};
      int ep = 127;
      if (in) {
        p = *reinterpret_cast<const u32x4*>(a.wc[w] + ((int64_t)col * a.nb + b) * 16);
        ep = a.ws[w][(int64_t)col * a.nb + b];
      }
      const i32x8 pa = {(int)p[0], (int)p[1], (int)p[2], (int)p[3], 0, 0, 0, 0};
      acc[w] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(pa, qa, acc[w], 4, 4, 0, ep, 0, eq);
    }
  }
  if (wave) {
#pragma unroll
    for (int w = 0; w < kW; ++w)
#pragma unroll
      for (int i = 0; i < 16; ++i) red[wave - 1][w][i][lane] = acc[w][i];
  }
  __syncthreads();
  if (wave || r >= rows) return;
#pragma unroll
  for (int w = 0; w < kW; ++w)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[w][i] += red[0][w][i][lane] + red[1][w][i][lane] + red[2][w][i][lane];
  with_act(GATE ? a.act : kRelu, [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int n = n0 + 8 * (i >> 2) + 4 * hh + (i & 3);
      if (n >= a.n) continue;
      float v = acc[0][i] + (a.bias[0] ? a.bias[0][n] : 0.f);
      if constexpr (GATE) v = gate_act<T, decltype(which)::value>(v) * (acc[kW - 1][i] + (a.bias[1] ? a.bias[1][n] : 0.f));
      Act<T>::gst(static_cast<T*>(a.y) + r * a.y_ld + n, v);
    }
  });
}

// --------------------------------------------------------------------------------------------------------------------- host side

static inline bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static inline int blocks_of(int k) { return (k + kBlock - 1) / kBlock; }
static constexpr size_t kFewBytes = 48 * 1024;             // of quantised x in LDS
static inline size_t few_bytes(int64_t rows, int nb) { return (size_t)rows * (17 * (size_t)nb + 16); }
// mx4_rows_kernel saves the launch that quantises x, but each of its workgroups quantises all of it: it pays up to 8 rows, and 6144 values more,
// of at most the 32 that a matrix instruction takes.  Its and the tiles' times in us, quantisation included: 1 x 512 -> 512 5.2 and 7.2,
// 16 x 512 7.1 and 7.6, 32 x 512 9.1 and 7.8; 8 x 2048 -> 2048 10.2 and 11.9, 16 x 2048 13.8 and 12.1; 32 x 96 -> 301 6.1 and 8.4.
static inline bool takes_few(int64_t rows, int k) { return rows <= std::min(32, 8 + 6144 / k) && few_bytes(rows, blocks_of(k)) <= kFewBytes; }
static inline size_t round256(size_t v) { return (v + 255) & ~(size_t)255; }

static ssmi_status check_mx4(const char* who, int64_t rows, int32_t k, int32_t n, int64_t ld, int32_t dtype) {
  SSMI_REQUIRE(rows > 0 && k > 0 && n > 0, SSMI_E_SHAPE, "%s: %lld rows, reduction %d, %d columns", who, (long long)rows, k, n);
  SSMI_REQUIRE(k <= 65536 && n <= 65536 && rows < (1ll << 31), SSMI_E_UNSUPPORTED, "%s: at most 65536 reduction elements and columns and 2^31 - 1 rows", who);
  SSMI_REQUIRE(ld >= k && ld <= (1 << 20), SSMI_E_SHAPE, "%s: row stride %lld under %d (or over 2^20)", who, (long long)ld, k);
  SSMI_REQUIRE(dtype == SSMI_F32 || dtype == SSMI_BF16, SSMI_E_UNSUPPORTED, "%s: unknown activation dtype %d", who, dtype);
  return SSMI_OK;
}

template <typename T>
static void quantize_rows(const T* x, int64_t ld, int64_t rows, int k, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  const int nb = blocks_of(k);
  const int64_t want = ceil_div64(rows * nb, 64);
  const dim3 grid((unsigned)(want < 16384 ? want : 16384));
  if (k % 8 == 0 && ld % 8 == 0 && at16(x)) hipLaunchKernelGGL((mx4_quantize_kernel_rows<T, true>), grid, dim3(256), 0, st, x, ld, rows, k, nb, codes, scales);
  else hipLaunchKernelGGL((mx4_quantize_kernel_rows<T, false>), grid, dim3(256), 0, st, x, ld, rows, k, nb, codes, scales);
}

template <typename T, bool GATE>
static ssmi_status launch_few(const T* x, int64_t x_ld, const Mx4Args& a, int k, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div64(a.n, 32));
  const size_t lds = few_bytes(a.rows, a.nb);
  if (k % 8 == 0 && x_ld % 8 == 0 && at16(x)) hipLaunchKernelGGL((mx4_rows_kernel<T, GATE, true>), grid, dim3(256), lds, st, x, x_ld, a, k);
  else hipLaunchKernelGGL((mx4_rows_kernel<T, GATE, false>), grid, dim3(256), lds, st, x, x_ld, a, k);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}
template <typename T, int SP, int SQ, bool GATE>
static ssmi_status launch_tiles(Mx4Args a, hipStream_t st) {
  typedef Mx4Shape<SP, SQ, GATE> S;
  a.np = (unsigned)ceil_div64(a.n, S::kHalf);
  a.nq = (unsigned)ceil_div64(a.rows, S::kQ);
  hipLaunchKernelGGL((mx4_kernel<T, SP, SQ, GATE>), dim3(a.np * a.nq), dim3(256), S::kLds, st, a);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}

template <bool GATE>
static ssmi_status mx4_product(const char* who, const void* x, int64_t x_ld, int64_t rows, int32_t k, int32_t n, int32_t dtype, Mx4Args a, void* ws, size_t ws_bytes,
                               void* stream) {
  const ssmi_status c = check_mx4(who, rows, k, n, x_ld, dtype);
  if (c != SSMI_OK) return c;
  SSMI_REQUIRE(x && a.y && a.wc[0] && a.ws[0] && (!GATE || (a.wc[1] && a.ws[1])), SSMI_E_INVALID_ARG, "%s: null pointer", who);
  SSMI_REQUIRE(a.y_ld >= n && a.y_ld <= (1 << 20), SSMI_E_SHAPE, "%s: row stride %lld under %d columns (or over 2^20)", who, (long long)a.y_ld, n);
  SSMI_REQUIRE(at16(a.wc[0]) && at16(a.wc[1]), SSMI_E_INVALID_ARG, "%s: codes must be 16-byte aligned", who);
  const size_t need = ssmi_mx4_workspace_bytes(rows, k);
  SSMI_REQUIRE(need == 0 || (ws && ws_bytes >= need), SSMI_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
  SSMI_REQUIRE(at16(ws), SSMI_E_INVALID_ARG, "%s: the workspace must be 16-byte aligned", who);
  SSMI_REQUIRE(ceil_div64(rows, Mx4Shape<2, 2, GATE>::kQ) * ceil_div64(n, Mx4Shape<2, 2, GATE>::kHalf) < kMostBlocks, SSMI_E_UNSUPPORTED,
               "%s: %lld rows of %d columns are too many for one launch", who, (long long)rows, n);
  a.rows = rows;
  a.n = n;
  a.nb = blocks_of(k);
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const T* xt = static_cast<const T*>(x);
    if (takes_few(rows, k)) return launch_few<T, GATE>(xt, x_ld, a, k, as_stream(stream));
    uint8_t* const codes = static_cast<uint8_t*>(ws);
    uint8_t* const scales = codes + round256((size_t)rows * 16 * a.nb);
    quantize_rows<T>(xt, x_ld, rows, k, codes, scales, as_stream(stream));
    SSMI_LAUNCH_CHECK();
    a.xc = codes;
    a.xs = scales;
    a.vec_out = a.y_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & (4 * sizeof(T) - 1)) == 0;
    // Results of 128 MB and more go past the caches: 64k x 512 -> 1024 float32 78 us, through them 97, with a reader behind it 173 and 193;
    // 32k rows 42 and 42, 85 and 90.  Under that the reader finds them there: 16k rows 24 and 25, 45.6 and 43.7.
    a.past = rows * n * (int64_t)sizeof(T) >= (128ll << 20);
    return launch_tiles<T, 2, 2, GATE>(a, as_stream(stream));
  });
}

}  // namespace ssmi

using namespace ssmi;

extern "C" {

ssmi_status ssmi_mx4_quantize(const void* x, int64_t ld, int64_t rows, int32_t k, int32_t dtype, uint8_t* codes, uint8_t* scales, void* stream) {
  const ssmi_status c = check_mx4("mx4_quantize", rows, k, 1, ld, dtype);
  if (c != SSMI_OK) return c;
  SSMI_REQUIRE(x && codes && scales, SSMI_E_INVALID_ARG, "mx4_quantize: null pointer");
  SSMI_REQUIRE(at16(codes), SSMI_E_INVALID_ARG, "mx4_quantize: codes must be 16-byte aligned");
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    quantize_rows<decltype(tag)>(static_cast<const decltype(tag)*>(x), ld, rows, k, codes, scales, as_stream(stream));
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

ssmi_status ssmi_mx4_quantize_kernel(const void* w, int32_t k, int32_t n, int32_t dtype, uint8_t* codes, uint8_t* scales, void* stream) {
  const ssmi_status c = check_mx4("mx4_quantize_kernel", 1, k, n, k, dtype);
  if (c != SSMI_OK) return c;
  SSMI_REQUIRE(w && codes && scales, SSMI_E_INVALID_ARG, "mx4_quantize_kernel: null pointer");
  SSMI_REQUIRE(at16(codes), SSMI_E_INVALID_ARG, "mx4_quantize_kernel: codes must be 16-byte aligned");
  const int nb = blocks_of(k);
  const dim3 grid((unsigned)ceil_div64(n, 64), (unsigned)ceil_div64(nb, 4));
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    hipLaunchKernelGGL((mx4_quantize_kernel_cols<T>), grid, dim3(256), 0, as_stream(stream), static_cast<const T*>(w), k, n, nb, codes, scales);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

ssmi_status ssmi_mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, int32_t k, int32_t n, float* w, void* stream) {
  const ssmi_status c = check_mx4("mx4_dequantize_kernel", 1, k, n, k, SSMI_F32);
  if (c != SSMI_OK) return c;
  SSMI_REQUIRE(w && codes && scales, SSMI_E_INVALID_ARG, "mx4_dequantize_kernel: null pointer");
  SSMI_REQUIRE(at16(codes), SSMI_E_INVALID_ARG, "mx4_dequantize_kernel: codes must be 16-byte aligned");
  const int nb = blocks_of(k);
  hipLaunchKernelGGL(mx4_dequantize_kernel_cols, dim3((unsigned)ceil_div64(n, 64), (unsigned)ceil_div64(nb, 4)), dim3(256), 0, as_stream(stream), codes, scales, k, n, nb, w);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}

size_t ssmi_mx4_workspace_bytes(int64_t rows, int32_t k) {
  if (rows <= 0 || k <= 0 || takes_few(rows, k)) return 0;
  const size_t nb = (size_t)blocks_of(k);
  return round256((size_t)rows * 16 * nb) + round256((size_t)rows * nb);
}

ssmi_status ssmi_mx4_dense(const void* x, int64_t x_ld, int64_t rows, int32_t k, int32_t n, int32_t dtype, const uint8_t* codes, const uint8_t* scales,
                           const float* bias, void* y, int64_t y_ld, void* ws, size_t ws_bytes, void* stream) {
  Mx4Args a = {};
  a.wc[0] = codes;
  a.ws[0] = scales;
  a.bias[0] = bias;
  a.y = y;
  a.y_ld = y_ld;
  return mx4_product<false>("mx4_dense", x, x_ld, rows, k, n, dtype, a, ws, ws_bytes, stream);
}

ssmi_status ssmi_mx4_gated(const void* x, int64_t x_ld, int64_t rows, int32_t k, int32_t n, int32_t dtype, int32_t act, const uint8_t* codes_gate,
                           const uint8_t* scales_gate, const uint8_t* codes_up, const uint8_t* scales_up, const float* b_gate, const float* b_up, void* y, int64_t y_ld,
                           void* ws, size_t ws_bytes, void* stream) {
  SSMI_REQUIRE(act >= SSMI_GATE_SWISH && act <= SSMI_GATE_SIGMOID, SSMI_E_INVALID_ARG, "mx4_gated: unknown activation %d", act);
  SSMI_REQUIRE(!b_gate == !b_up, SSMI_E_INVALID_ARG, "mx4_gated: both biases or none");
  Mx4Args a = {};
  a.wc[0] = codes_gate;
  a.ws[0] = scales_gate;
  a.wc[1] = codes_up;
  a.ws[1] = scales_up;
  a.bias[0] = b_gate;
  a.bias[1] = b_up;
  a.act = act;
  a.y = y;
  a.y_ld = y_ld;
  return mx4_product<true>("mx4_gated", x, x_ld, rows, k, n, dtype, a, ws, ws_bytes, stream);
}

}  // extern "C"
