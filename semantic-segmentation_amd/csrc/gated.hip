// Gated feed-forward unit on rows of channels (pixels):
//   g = x Wg + bg,  u = x Wu + bu,  y = act(g) * u                         x [rows, c], W [c, f] (Keras kernels), y [rows, f]
// Forward: both projections in one kernel; a wave holds the accumulators of the same 32 units of both, so activation and product
// happen in registers and g, u never reach memory.
// Backward: nothing but x is kept.  One kernel recomputes g and u (exact float32 in registers, where storing them would round them to
// the activation type or double the traffic) and forms in its epilogue, from dy,
//   dg = dy * u * act'(g),   du = dy * act(g)                              one row [dg | du] per pixel, float32 or two bfloat16 terms
// then  dx = dg Wg^T + du Wu^T  (one product over 2 f) and  dW = x^T dg, x^T du  (one product over the rows, split into strips whose
// float32 partial sums are added in a fixed order: results do not depend on the launch).
// All products run on gemm_tile.h: bfloat16 32x32x16 or float32 32x32x2 matrix instructions, float32 sums throughout.
#include <algorithm>

#include "gate_act.h"
#include "gemm_tile.h"

namespace ssmi {

__device__ __forceinline__ float param_at(const void* p, int bf, int64_t i) {
  return bf ? (float)static_cast<const bf16*>(p)[i] : static_cast<const float*>(p)[i];
}

// Stages, K step, q rows that the epilogue takes at once and workgroups to a CU (registers and LDS) of a tile shape.  The products of dx
// and dW run long K loops: 128-byte steps, fewer barriers (16k x 512 -> 2048 bfloat16: dx 147 us, with 64-byte steps 182).  The gate kernels run
// short ones with an epilogue as long: the 128 x 128 tile takes 64-byte steps and a quarter of the tile through LDS at a time, so three
// workgroups share a CU and one's epilogue runs under the others' products.
template <int SP, int SQ>
struct ProductShape {
  static constexpr int kStep = SP * SQ == 8 ? 64 : 128, kStages = SP * SQ == 8 ? 3 : 2, kAtOnce = SQ > 2 ? 2 : SQ;
  static constexpr int kPerCu = SP * SQ == 16 ? 1 : SQ == 1 ? 3 : 2;
  static constexpr bool kChunks = true;
};
template <int SP, int SQ>
struct GateShape {
  static constexpr int kStep = SQ == 1 ? 128 : 64, kStages = SQ == 4 ? 3 : 2, kAtOnce = SQ == 4 ? 2 : 1, kPerCu = SQ == 4 ? 2 : 3;
};
// float32 sums over more than kChunk channels go in chunks, whose registers leave two of the larger tiles to a CU (16k x 512 -> 1024 forward
// 259 -> 267 us, 8k x 1024 -> 1024 247 -> 258); shorter ones have one chunk and stay with three
template <typename T, int SP, int SQ, bool LONG> constexpr int gate_per_cu() { return LONG && sizeof(T) == 4 && SQ == 2 ? 2 : GateShape<SP, SQ>::kPerCu; }

struct GateArgs {
  const void *x, *wg, *wu;      // x [rows][x_ld], W [c][w_ld], activation type
  const void *bg, *bu;          // parameter type or nullptr
  const void* dy;               // backward
  void* out;                    // y, or [dg | du]
  int64_t rows, x_ld, w_ld, out_ld, dy_ld;
  int c, f, fp;                 // fp: units with the padding that [dg | du] rows have
  int act, bf_params, vec_out, vec_dy;      // see vec_of
  float* db;                    // backward: column sums of [dg | du] per row tile, or nullptr
  unsigned np, nq;
};

// Columns of the projections' gradients, in units of fp: float32 [dg | du], bfloat16 [dg | du | rest of dg | rest of du].  One bfloat16 of
// dg is off by up to 2^-8 of it and shows beside the results' own rounding (bfloat16 results of 9999 x 256 -> 682 off by 2.3e-3 of their norm
// instead of the 1.7e-3 of that rounding, float32 ones by 1.7e-3); the second term brings it to 2^-16 (1.7e-3 and 2.5e-6) for twice the
// arithmetic of dx and dW (64k x 512 -> 2048: with dg and du 420 -> 490 us, dx 233 -> 469, dW 253 -> 514).
template <typename T> constexpr int kGradSides = sizeof(T) == 2 ? 4 : 2;

// what the first bfloat16 term leaves; an infinity leaves nothing (inf - inf would turn it into a NaN), a NaN is one in the first term already
__device__ __forceinline__ float rest_of(float v) {
  const float first = (float)(bf16)v;
  return __builtin_fabsf(first) < INFINITY ? v - first : 0.f;
}

template <typename T, int SP, int SQ, bool LONG>
struct GateSides : GateShape<SP, SQ> {
  using GateShape<SP, SQ>::kStep;
  static constexpr bool kChunks = LONG;
  static constexpr int kHalf = SP * 32;      // units of a tile
  typedef Operand<T, kHalf, true, kStep> W;
  typedef Operand<T, SQ * 64, false, kStep> X;
  static constexpr int kStage = 2 * W::kBytes + X::kBytes, kLoads = 2 * W::kLoads + X::kLoads;
  W wg, wu;
  X x;
  typename W::Reader rw;
  typename X::Reader rx;
  int c, wp, wq;
  __device__ __forceinline__ void one(lds_bytes s, int t, int j) const {
    const int left = c - t * W::kStepK;
    if (j < W::kLoads) wg.one(s, t, j, left);
    else if (j < 2 * W::kLoads) wu.one(s + W::kBytes, t, j - W::kLoads, left);
    else x.one(s + 2 * W::kBytes, t, j - 2 * W::kLoads, left);
  }
  __device__ __forceinline__ u32x4 p(lds_bytes s, int i, int ks) const {
    return rw.get(s + (i / (SP / 2)) * W::kBytes, wp * (SP / 2) + i % (SP / 2), ks);
  }
  __device__ __forceinline__ u32x4 q(lds_bytes s, int j, int ks) const { return rx.get(s + 2 * W::kBytes, wq * SQ + j, ks); }
};

template <typename T, int SP, int SQ, bool BWD, bool LONG>
__global__ __launch_bounds__(256, (gate_per_cu<T, SP, SQ, LONG>())) void gate_kernel(GateArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  typedef GateSides<T, SP, SQ, LONG> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const TileAt at = tile_at(spread_blocks(blockIdx.x, gridDim.x), a.np, a.nq);
  const int64_t m0 = (int64_t)at.q * (SQ * 64);
  const int f0 = at.p * S::kHalf;
  S s;
  s.c = a.c;
  s.wp = wave >> 1;
  s.wq = wave & 1;
  s.wg.init(static_cast<const T*>(a.wg) + f0, a.w_ld, a.fp - f0);
  s.wu.init(static_cast<const T*>(a.wu) + f0, a.w_ld, a.fp - f0);
  s.x.init(static_cast<const T*>(a.x) + m0 * a.x_ld, a.x_ld, (int)min((int64_t)(SQ * 64), a.rows - m0));
  s.rw.init(lane);
  s.rx.init(lane);
  f32x16 acc[SP][SQ];
  tile_product<T, SP, SQ>(s, (lds_bytes)smem, (a.c + S::W::kStepK - 1) / S::W::kStepK, acc);

  // a thread keeps four units for the whole epilogue
  typedef TileRows<SP, SQ, S::kHalf, S::kAtOnce> R;
  const int col = R::col(), f = f0 + col, n = a.f - f;
  float bg[4] = {0.f, 0.f, 0.f, 0.f}, bu[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.bg) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bg[e] = e < n ? param_at(a.bg, a.bf_params, f + e) : 0.f;
      bu[e] = e < n ? param_at(a.bu, a.bf_params, f + e) : 0.f;
    }
  }
  const int wp = s.wp;
  auto pos = [&](int i) __attribute__((always_inline)) { return (i / (SP / 2)) * S::kHalf + (wp * (SP / 2) + i % (SP / 2)) * 32; };
  const bool whole = m0 + SQ * 64 <= a.rows && f0 + S::kHalf <= a.f && a.vec_out && (!BWD || a.vec_dy);      // uniform
  // the lane's place in a tile of `out` / dy; rounds add whole rows
  T* const out = static_cast<T*>(a.out) + m0 * a.out_ld + f0;
  const T* const dyt = static_cast<const T*>(a.dy) + (BWD ? m0 * a.dy_ld + f0 : 0);
  const unsigned o_lane = (unsigned)R::first() * (unsigned)a.out_ld + (unsigned)col, d_lane = (unsigned)R::first() * (unsigned)a.dy_ld + (unsigned)col;
  float sum[BWD ? 8 : 1] = {};
  // [dg | du] of four units of a pixel; behind them the parts that bfloat16 leaves
  auto put_gradients = [&](T* d, const float (&o)[4], const float (&v)[4]) __attribute__((always_inline)) {
    if constexpr (BWD) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { sum[e] += o[e]; sum[4 + e] += v[e]; }
      put4<T>(d, f32x4{o[0], o[1], o[2], o[3]});
      put4<T>(d + a.fp, f32x4{v[0], v[1], v[2], v[3]});
      if constexpr (sizeof(T) == 2) {
        f32x4 ro, rv;
#pragma unroll
        for (int e = 0; e < 4; ++e) { ro[e] = rest_of(o[e]); rv[e] = rest_of(v[e]); }
        put4<T>(d + 2 * a.fp, ro);
        put4<T>(d + 3 * a.fp, rv);
      }
    }
  };
  with_act(a.act, [&](auto which) __attribute__((always_inline)) {
    constexpr int kAct = decltype(which)::value;
    auto forward = [&](const float* row, float (&o)[4]) __attribute__((always_inline)) {
      const f32x4 g = *reinterpret_cast<const f32x4*>(row), u = *reinterpret_cast<const f32x4*>(row + S::kHalf);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = gate_act<T, kAct>(g[e] + bg[e]) * (u[e] + bu[e]);
    };
    auto backward = [&](const float* row, const float (&dy)[4], float (&o)[4], float (&v)[4]) __attribute__((always_inline)) {
      const f32x4 g = *reinterpret_cast<const f32x4*>(row), u = *reinterpret_cast<const f32x4*>(row + S::kHalf);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float h, d;
        gate_act_both<T, kAct>(g[e] + bg[e], h, d);
        o[e] = dy[e] * (u[e] + bu[e]) * d;
        v[e] = dy[e] * h;
      }
    };
    if constexpr (sizeof(T) == 2 && !BWD) {
      // The forward pass stores straight from the accumulators: no LDS, no barrier, 32 bytes of a row at a time (64k x 512 -> 2048: 306 us,
      // through LDS 317, 16k rows 74 and 78).  Where dy has to come the same way, or nothing but the store is to do (dx), whole rows through
      // LDS are faster (both measured with one bfloat16 term of dg and du: 64k x 512 -> 2048 with dg, du 421 against 476 us; 16k rows, dx 66
      // against 72).
      if (whole && a.vec_out == 2) {
        const int hh = lane >> 5, u0 = wp * (SP / 2) * 32;
        T* const y = out + (int64_t)(s.wq * SQ * 32) * a.out_ld + u0;
        const unsigned y_lane = (unsigned)(lane & 31) * (unsigned)a.out_ld;
#pragma unroll
        for (int i = 0; i < SP / 2; ++i)
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            float bg8[8] = {}, bu8[8] = {};
            if (a.bg) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int unit = f0 + u0 + i * 32 + 8 * (k + e / 4) + 4 * hh + e % 4;
                bg8[e] = param_at(a.bg, a.bf_params, unit);
                bu8[e] = param_at(a.bu, a.bf_params, unit);
              }
            }
#pragma unroll
            for (int j = 0; j < SQ; ++j) {
              f32x4 o[2];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e / 4][e % 4] = gate_act<T, kAct>(acc[i][j][4 * k + e] + bg8[e]) * (acc[i + SP / 2][j][4 * k + e] + bu8[e]);
              put8(y + j * 32 * a.out_ld + i * 32 + 8 * k + y_lane, hh, o[0], o[1]);
            }
          }
        return;
      }
    }
    if (whole) {
      typename Act<T>::raw4 dy[BWD ? R::kRounds : 1];
      R::template run<R::kRounds>(
          acc, reinterpret_cast<float*>(smem), s.wq, pos,
          [&](int pass) __attribute__((always_inline)) {
            if constexpr (BWD) {      // dy is on its way while the accumulators move
#pragma unroll
              for (int i = 0; i < R::kRounds; ++i) dy[i] = *reinterpret_cast<const typename Act<T>::raw4*>(dyt + R::q_of(pass, i) * a.dy_ld + d_lane);
            }
          },
          [&](const float* row, int qc, int i) __attribute__((always_inline)) {
            float o[4], v[4];
            T* const d = out + qc * a.out_ld + o_lane;
            if constexpr (!BWD) {
              forward(row, o);
              put4<T>(d, f32x4{o[0], o[1], o[2], o[3]});
            } else {
              const f32x4 y = Act<T>::up4(dy[i]);
              const float y4[4] = {y[0], y[1], y[2], y[3]};
              backward(row, y4, o, v);
              put_gradients(d, o, v);
            }
          });
    } else {
      R::template run<1>(
          acc, reinterpret_cast<float*>(smem), s.wq, pos, [](int) {},
          [&](const float* row, int qc, int) __attribute__((always_inline)) {
            const int64_t m = m0 + R::first() + qc;
            if (m >= a.rows || f >= (BWD ? a.fp : a.f)) return;
            float o[4], v[4];
            T* const d = static_cast<T*>(a.out) + m * a.out_ld + f;
            if constexpr (!BWD) {
              forward(row, o);
              store4<T>(d, o, n, a.vec_out);
            } else {
              float dy[4];
              fetch4<T>(static_cast<const T*>(a.dy) + m * a.dy_ld + f, dy, n, a.vec_dy);
              backward(row, dy, o, v);
#pragma unroll
              for (int e = 0; e < 4; ++e) {      // padded units are set, not multiplied: zero weights times an infinite x are no number
                o[e] = e < n ? o[e] : 0.f;
                v[e] = e < n ? v[e] : 0.f;
              }
              put_gradients(d, o, v);
            }
          });
    }
  });
  if constexpr (BWD) {
    if (a.db) {      // the tile's column sums, of the unrounded values: over the threads that share the units, then a row per tile
      float* const sh = reinterpret_cast<float*>(smem);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) sh[((e >> 2) * R::kPerRound + R::first()) * S::kHalf + col + (e & 3)] = sum[e];
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * S::kHalf; i += 256) {
        const int side = i / S::kHalf, unit = i - side * S::kHalf;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < R::kPerRound; ++k) t += sh[(side * R::kPerRound + k) * S::kHalf + unit];
        if (f0 + unit < a.fp) a.db[(int64_t)at.q * (2 * (int64_t)a.fp) + side * a.fp + f0 + unit] = t;
      }
    }
  }
}

// dx[m][c] = sum_f dg[m][f] Wg[c][f] + du[m][f] Wu[c][f]: K runs over the units of the first, then of the second projection (and again
// over the second terms of bfloat16).  Few tiles under a long K share it in strips, whose float32 sums [strip][rows][c4] are added
// in their order by the reduction behind dW.
struct GateDxArgs {
  const void *dgu, *wg, *wu;
  void* dx;
  float* part;      // more than one strip: instead of dx
  int64_t rows, w_ld, dx_ld;
  int c, fp, vec_out;
  int each, strips, c4;           // K steps of a strip
  unsigned np, nq;
};
template <typename T, int SP, int SQ>
struct DxSides : ProductShape<SP, SQ> {
  using ProductShape<SP, SQ>::kStep;
  typedef Operand<T, SP * 64, false, kStep> W;
  typedef Operand<T, SQ * 64, false, kStep> D;
  static constexpr int kStage = W::kBytes + D::kBytes, kLoads = W::kLoads + D::kLoads;
  W wg;
  D d;
  __amdgpu_buffer_rsrc_t wu;
  typename W::Reader rw;
  typename D::Reader rd;
  int fp, half, first, end, wp, wq;      // the strip's steps
  __device__ __forceinline__ void one(lds_bytes s, int step, int j) const {
    const int t = first + step, side = t >= 2 * half ? (t >= 3 * half ? 3 : 2) : t >= half ? 1 : 0;
    const int ts = t - side * half, left = t < end ? fp - ts * W::kStepK : 0;
    if (j < W::kLoads) {
      W w = wg;
      if (side & 1) w.rsrc = wu;
      w.one(s, ts, j, left);
    } else {
      d.one(s + W::kBytes, ts, j - W::kLoads, left, (unsigned)(side * fp * (int)sizeof(T)));
    }
  }
  __device__ __forceinline__ u32x4 p(lds_bytes s, int i, int ks) const { return rw.get(s, wp * SP + i, ks); }
  __device__ __forceinline__ u32x4 q(lds_bytes s, int j, int ks) const { return rd.get(s + W::kBytes, wq * SQ + j, ks); }
};
template <typename T, int SP, int SQ>
__global__ __launch_bounds__(256, (ProductShape<SP, SQ>::kPerCu)) void gate_dx_kernel(GateDxArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  typedef DxSides<T, SP, SQ> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned v = spread_blocks(blockIdx.x, gridDim.x), tiles = a.np * a.nq, strip = __builtin_amdgcn_readfirstlane(v / tiles);
  const TileAt at = tile_at(v - strip * tiles, a.np, a.nq);
  const int64_t m0 = (int64_t)at.q * (SQ * 64);
  const int c0 = at.p * (SP * 64);
  S s;
  s.fp = a.fp;
  s.half = (a.fp + S::W::kStepK - 1) / S::W::kStepK;
  s.first = (int)strip * a.each;
  s.end = min(s.first + a.each, kGradSides<T> * s.half);
  s.wp = wave >> 1;
  s.wq = wave & 1;
  s.wg.init(static_cast<const T*>(a.wg) + c0 * a.w_ld, a.w_ld, a.c - c0);
  s.wu = make_rsrc(static_cast<const T*>(a.wu) + c0 * a.w_ld, 0x7FFFFFFFu);
  s.d.init(static_cast<const T*>(a.dgu) + m0 * (kGradSides<T> * (int64_t)a.fp), kGradSides<T> * (int64_t)a.fp, (int)min((int64_t)(SQ * 64), a.rows - m0));
  s.rw.init(lane);
  s.rd.init(lane);
  f32x16 acc[SP][SQ];
  tile_product<T, SP, SQ>(s, (lds_bytes)smem, s.end - s.first, acc);
  typedef TileRows<SP, SQ, SP * 64, S::kAtOnce> R;
  const int wp = s.wp, c = c0 + R::col();
  auto pos = [&](int i) __attribute__((always_inline)) { return (wp * SP + i) * 32; };
  if (a.part) {
    float* const part = a.part + (strip * a.rows + m0 + R::first()) * a.c4 + c;
    R::template run<1>(acc, reinterpret_cast<float*>(smem), s.wq, pos, [](int) {}, [&](const float* row, int qc, int) __attribute__((always_inline)) {
      if (m0 + R::first() + qc < a.rows && c < a.c) *reinterpret_cast<f32x4*>(part + (int64_t)qc * a.c4) = *reinterpret_cast<const f32x4*>(row);
    });
  } else if (m0 + SQ * 64 <= a.rows && c0 + SP * 64 <= a.c && a.vec_out) {
    T* const dx = static_cast<T*>(a.dx) + m0 * a.dx_ld + c0;
    const unsigned lane_at = (unsigned)R::first() * (unsigned)a.dx_ld + (unsigned)R::col();
    R::template run<R::kRounds>(acc, reinterpret_cast<float*>(smem), s.wq, pos, [](int) {}, [&](const float* row, int qc, int) __attribute__((always_inline)) {
      put4<T>(dx + qc * a.dx_ld + lane_at, *reinterpret_cast<const f32x4*>(row));
    });
  } else {
    R::template run<1>(acc, reinterpret_cast<float*>(smem), s.wq, pos, [](int) {}, [&](const float* row, int qc, int) __attribute__((always_inline)) {
      const int64_t m = m0 + R::first() + qc;
      if (m >= a.rows || c >= a.c) return;
      const f32x4 v = *reinterpret_cast<const f32x4*>(row);
      const float o[4] = {v[0], v[1], v[2], v[3]};
      store4<T>(static_cast<T*>(a.dx) + m * a.dx_ld + c, o, a.c - c, a.vec_out);
    });
  }
}

// part[strip][c][2 fp] = sum over the strip's rows of x[m][c] [dg | du][m][p]; bfloat16 goes through the rows twice, the second time with the second terms
struct GateDwArgs {
  const void *x, *dgu;
  float* part;
  int64_t rows, x_ld, strip_rows;
  int c, cp, fp;                // cp: channels with the padding of x rows
  unsigned np, nq;
};
template <typename T, int SP, int SQ>
struct DwSides : ProductShape<SP, SQ> {
  using ProductShape<SP, SQ>::kStep;
  typedef Operand<T, SP * 64, true, kStep> D;
  typedef Operand<T, SQ * 64, true, kStep> X;
  static constexpr int kStage = D::kBytes + X::kBytes, kLoads = D::kLoads + X::kLoads;
  D d;
  X x;
  typename D::Reader rd;
  typename X::Reader rx;
  int rows, once, times, wp, wq;
  unsigned second;      // bytes from the first terms of a row to the second ones
  __device__ __forceinline__ void one(lds_bytes s, int t, int j) const {
    const bool again = t >= once;
    const int ts = again ? t - once : t, left = t < times * once ? rows - ts * D::kStepK : 0;
    if (j < D::kLoads) d.one(s, ts, j, left, again ? second : 0u);
    else x.one(s + D::kBytes, ts, j - D::kLoads, left);
  }
  __device__ __forceinline__ u32x4 p(lds_bytes s, int i, int ks) const { return rd.get(s, wp * SP + i, ks); }
  __device__ __forceinline__ u32x4 q(lds_bytes s, int j, int ks) const { return rx.get(s + D::kBytes, wq * SQ + j, ks); }
};
template <typename T, int SP, int SQ>
__global__ __launch_bounds__(256, (ProductShape<SP, SQ>::kPerCu)) void gate_dw_kernel(GateDwArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  typedef DwSides<T, SP, SQ> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned v = spread_blocks(blockIdx.x, gridDim.x), tiles = a.np * a.nq, strip = __builtin_amdgcn_readfirstlane(v / tiles);
  const TileAt at = tile_at(v - strip * tiles, a.np, a.nq);
  const int64_t m0 = (int64_t)strip * a.strip_rows;
  const int c0 = at.q * (SQ * 64), p0 = at.p * (SP * 64);
  S s;
  s.rows = (int)min(a.strip_rows, a.rows - m0);
  s.wp = wave >> 1;
  s.wq = wave & 1;
  s.d.init(static_cast<const T*>(a.dgu) + m0 * (kGradSides<T> * (int64_t)a.fp) + p0, kGradSides<T> * (int64_t)a.fp, 2 * a.fp - p0);
  s.once = (s.rows + S::D::kStepK - 1) / S::D::kStepK;
  s.times = kGradSides<T> / 2;
  s.second = 2u * (unsigned)a.fp * (unsigned)sizeof(T);
  s.x.init(static_cast<const T*>(a.x) + m0 * a.x_ld + c0, a.x_ld, a.cp - c0);
  s.rd.init(lane);
  s.rx.init(lane);
  f32x16 acc[SP][SQ];
  tile_product<T, SP, SQ>(s, (lds_bytes)smem, s.times * s.once, acc);
  typedef TileRows<SP, SQ, SP * 64, S::kAtOnce> R;
  const int wp = s.wp, p = p0 + R::col();
  float* const part = a.part + ((int64_t)strip * a.c + c0 + R::first()) * (2 * (int64_t)a.fp) + p;
  R::template run<R::kRounds>(acc, reinterpret_cast<float*>(smem), s.wq, [&](int i) __attribute__((always_inline)) { return (wp * SP + i) * 32; }, [](int) {},
                              [&](const float* row, int qc, int) __attribute__((always_inline)) {
                                if (c0 + R::first() + qc < a.c && p < 2 * a.fp) *reinterpret_cast<f32x4*>(part + qc * (2 * (int64_t)a.fp)) = *reinterpret_cast<const f32x4*>(row);
                              });
}

// sum of n partial sums of four values in their order, sixteen on their way at a time
__device__ __forceinline__ f32x4 ordered_sum(const float* s, int n, int64_t step) {
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  int k = 0;
  for (; k + 16 <= n; k += 16) {
    f32x4 v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = *reinterpret_cast<const f32x4*>(s + (k + e) * step);
#pragma unroll
    for (int e = 0; e < 16; ++e) sum += v[e];
  }
  for (; k + 4 <= n; k += 4) {
    f32x4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const f32x4*>(s + (k + e) * step);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += v[e];
  }
  for (; k < n; ++k) sum += *reinterpret_cast<const f32x4*>(s + k * step);
  return sum;
}
// dW = sum of the strips' partial sums in their order, db = that of the row tiles' column sums; four units a thread, the bias row last;
// behind them dx, where its sums lie in strips
struct ReduceArgs {
  const float *part, *db, *dx_part;
  void *dwg, *dwu, *dbg, *dbu, *dx;
  int64_t c, rows, dx_ld;
  int strips, db_tiles, f, fp, bf;
  int dx_strips, dx_c, c4, dx_vec;
  unsigned dw_blocks;
};
static constexpr int kReduce = 64;      // threads: a small dW still spreads over the card
template <typename T>
__global__ __launch_bounds__(kReduce) void gate_reduce_kernel(ReduceArgs a) {
  if (blockIdx.x >= a.dw_blocks) {
    const int64_t i = (int64_t)(blockIdx.x - a.dw_blocks) * kReduce + threadIdx.x, m = i / (a.c4 / 4);
    const int c = (int)(i - m * (a.c4 / 4)) * 4;
    if (m >= a.rows) return;
    const f32x4 v = ordered_sum(a.dx_part + m * a.c4 + c, a.dx_strips, a.rows * a.c4);
    const float o[4] = {v[0], v[1], v[2], v[3]};
    store4<T>(static_cast<T*>(a.dx) + m * a.dx_ld + c, o, a.dx_c - c, a.dx_vec);
    return;
  }
  const int64_t i = (int64_t)blockIdx.x * kReduce + threadIdx.x;
  const int quads = a.fp / 2;
  const int64_t ci = i / quads;
  const int p = (int)(i - ci * quads) * 4;
  const bool bias = ci == a.c;
  if (ci > a.c || (bias && !a.db)) return;
  const int fu = p < a.fp ? p : p - a.fp;
  char* const dst = static_cast<char*>(bias ? (p < a.fp ? a.dbg : a.dbu) : (p < a.fp ? a.dwg : a.dwu));
  if (!dst) return;
  const int n = bias ? a.db_tiles : a.strips;
  const int64_t step = (bias ? 1 : a.c) * 2 * a.fp;
  const float* s = bias ? a.db + p : a.part + ci * (2 * (int64_t)a.fp) + p;
  const f32x4 sum = ordered_sum(s, n, step);
  const int64_t at = (bias ? 0 : ci * a.f) + fu;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (fu + e < a.f) {
      if (a.bf) reinterpret_cast<bf16*>(dst)[at + e] = (bf16)sum[e];
      else reinterpret_cast<float*>(dst)[at + e] = sum[e];
    }
}

// memory rows brought to the tile engine's form: activation type, rows of cols_p >= cols values (16-byte multiples), zeros behind.
// Up to three matrices a launch (x, both kernels), one per blockIdx.y.  float32 kernels under bfloat16 rows become bfloat16 here, as the
// convolutions' bfloat16 packs do: the matrix instructions take one type, and a second term would double the products of the forward pass.
struct PadJob {
  const void* src;
  void* dst;
  int64_t ld, rows;
  int cols, cols_p, bf;      // bf: the source is bfloat16
};
struct PadJobs { PadJob job[3]; };
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadJobs jobs) {
  const PadJob j = jobs.job[blockIdx.y];
  const int quads = j.cols_p / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < j.rows * quads; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / quads;
    const int k = (int)(i - r * quads) * 4;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + e < j.cols ? param_at(j.src, j.bf, r * j.ld + k + e) : 0.f;
    Act<T>::gst4(static_cast<T*>(j.dst) + r * j.cols_p + k, v);
  }
}

// A few rows: bound by reading the weights (or by latency), so no tiles and no staging of W.  A workgroup owns 32 units of both
// projections.  Four lanes side by side hold eight units each, 16 bytes of bfloat16 or twice 16 of float32; the other 16 WAVES of them share
// the channels, so that all loads of a short reduction are on their way at once.
template <typename P, bool VEC>
__device__ __forceinline__ void fetch8(const P* p, int n, float (&v)[8]) {
  if constexpr (VEC) {
    if constexpr (sizeof(P) == 2) {
      const u32x4 r = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(r[e] << 16);
        v[2 * e + 1] = __uint_as_float(r[e] & 0xFFFF0000u);
      }
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : 0.f;
  }
}
// sums over the lanes that differ in bit 5, then 4, 3 and 2; each step sends half of the values and keeps the other, so lane 4 s + oct ends
// with the N / 16 values from s N / 16 on
template <int N, int BIT>
__device__ __forceinline__ void fold(float* v, int lane) {
  const bool up = lane & BIT;
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float keep = up ? v[N / 2 + i] : v[i], send = up ? v[i] : v[N / 2 + i];
    v[i] = keep + __shfl_xor(send, BIT, 64);
  }
  if constexpr (BIT > 4) fold<N / 2, BIT / 2>(v, lane);
}
template <typename T, typename P, int MB, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void gate_rows_kernel(GateArgs a) {
  extern __shared__ float xs[];                     // [c][MB]
  __shared__ float red[WAVES][MB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * MB;
  const int nm = (int)min((int64_t)MB, a.rows - m0);
  for (int k = threadIdx.x; k < a.c; k += 64 * WAVES) {
    float x[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) x[m] = Act<T>::gld(static_cast<const T*>(a.x) + (m0 + min(m, nm - 1)) * a.x_ld + k);      // all on their way at once
#pragma unroll
    for (int m = 0; m < MB; ++m) xs[k * MB + m] = x[m];      // rows behind the last repeat it and are not written
  }
  __syncthreads();
  const int oct = lane & 3, f = blockIdx.x * 32 + oct * 8, n = a.f - f;
  const P *wg = static_cast<const P*>(a.wg) + f, *wu = static_cast<const P*>(a.wu) + f;
  float sum[16 * MB];      // [side][unit][row]
#pragma unroll
  for (int i = 0; i < 16 * MB; ++i) sum[i] = 0.f;
  if (n > 0) {
    constexpr int kAhead = sizeof(P) == 2 ? 4 : 2;      // 32 registers of loads
#pragma unroll kAhead
    for (int k = wave * 16 + (lane >> 2); k < a.c; k += 16 * WAVES) {
      float w[2][8];
      fetch8<P, VEC>(wg + (int64_t)k * a.f, n, w[0]);
      fetch8<P, VEC>(wu + (int64_t)k * a.f, n, w[1]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // float32 parameters under bfloat16 activations are multiplied as bfloat16
        const float wv = sizeof(P) != sizeof(T) ? (float)(T)w[i / 8][i % 8] : w[i / 8][i % 8];
#pragma unroll
        for (int m = 0; m < MB; ++m) sum[i * MB + m] = fmaf(xs[k * MB + m], wv, sum[i * MB + m]);
      }
    }
  }
  fold<16 * MB, 32>(sum, lane);
#pragma unroll
  for (int m = 0; m < MB; ++m) red[wave][m][(lane >> 5) * 32 + oct * 8 + ((lane >> 2) & 7)] = sum[m];
  __syncthreads();
  for (int i = threadIdx.x; i < nm * 32; i += 64 * WAVES) {
    const int m = i >> 5, col = i & 31, ff = blockIdx.x * 32 + col;
    if (ff >= a.f) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      g += red[w][m][col];
      u += red[w][m][32 + col];
    }
    if (a.bg) {
      g += param_at(a.bg, a.bf_params, ff);
      u += param_at(a.bu, a.bf_params, ff);
    }
    with_act(a.act, [&](auto which) { g = gate_act<T, decltype(which)::value>(g); });
    Act<T>::gst(static_cast<T*>(a.out) + (m0 + m) * a.out_ld + ff, g * u);
  }
}

// --------------------------------------------------------------------------------------------------------------- host side

static inline int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
static inline size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// The tile loop asks for kStages K steps past the last one, at most 128 memory rows of an operand whose K runs over rows.  Their lanes are
// switched off by an offset past the descriptor's end, which holds as long as the step's own offset does not pass that end.
static constexpr int64_t kPastRows = 128, kReach = 0x7FFFFFFF;
template <typename S> constexpr int64_t past_rows(int es) { return (int64_t)S::kStages * S::kStep / es; }
static_assert(past_rows<GateShape<2, 1>>(2) <= kPastRows && past_rows<GateShape<2, 2>>(2) <= kPastRows && past_rows<GateShape<2, 4>>(2) <= kPastRows &&
              past_rows<ProductShape<2, 1>>(2) <= kPastRows && past_rows<ProductShape<2, 2>>(2) <= kPastRows && past_rows<ProductShape<2, 4>>(2) <= kPastRows, "");

// Tile shapes (columns p x rows q), chosen by how many workgroups they make: a card of 256 CUs wants 512 of those that go two to a CU.
//   gate: 128 x 256 where that makes 384 tiles (64k x 512 -> 2048 bfloat16: forward 301 us, with dg and du 464; 128 x 128 330 and 510), 128 x 128
//         where that makes 256, else 128 x 64
//   no tile of 128 rows or channels where there are 64 (131k x 64 -> 256 float32, dx 142 -> 103 us, dW 127 -> 90)
//   dx:   256 x 256 (one to a CU: no epilogue to hide; 64k x 512 -> 2048 bfloat16 477 us, 128 x 128 594) where that makes 192; 64 x 64 under 64
//         channels or where 128 x 64 makes under 384 (4096 x 512 -> 2048 bfloat16 76 -> 69 us, 16k x 128 -> 512 float32 46 -> 44); else as above
//   dW:   128 x 256 under strips of 4096 rows (64k x 512 -> 2048 bfloat16 538 us, 128 x 128 611); else as above, counting the strips
// float32 takes no wide tiles: its 64-cycle matrix instructions leave LDS time to spare, and its sums take twice the registers.
enum Tile { kTile64x64, kTile128x64, kTile128x128, kTile128x256, kTile256x256 };
static Tile tile_for(int64_t q, int64_t p, bool wide, int64_t times = 1) {
  if (wide && ceil_div64(q, 256) * ceil_div64(p, 128) * times >= 384 && q > 128) return kTile128x256;
  return q > 64 && ceil_div64(q, 128) * ceil_div64(p, 128) * times >= 256 ? kTile128x128 : kTile128x64;
}
static Tile tile_for_dx(int64_t rows, int64_t c, bool wide) {
  if (wide && c > 128 && ceil_div64(rows, 256) * ceil_div64(c, 256) >= 192) return kTile256x256;
  const Tile t = tile_for(rows, c, false);
  if (c <= 64) return kTile64x64;
  return t == kTile128x64 && ceil_div64(rows, 64) * ceil_div64(c, 128) < 384 ? kTile64x64 : t;
}
static Tile tile_for_dw(int64_t rows, int64_t c, int64_t p, bool wide, int64_t most_strips) {
  // the larger tile only under strips of 4096 rows, where its own speed outweighs the partial sums of twice the strips
  if (wide && c > 128 && rows / ceil_div64(512, ceil_div64(p, 128) * ceil_div64(c, 256)) >= 4096) return kTile128x256;
  return tile_for(c, p, false, most_strips);
}
// K steps that a strip of dx takes.  Its smallest tiles may leave the card idle under a long K; strips bring one or two workgroups to a CU, of
// four steps (256 bfloat16, 128 float32 values) at least.  By measurement a step takes a workgroup 0.4 us in bfloat16, two workgroups of a CU
// side by side, and 0.85 in float32, where the matrix unit is full with one of them; the strips' sums and their reduction take 6.
// Whole backward pass, one strip and so: 64 x 64 -> 4096 bfloat16 126 and 21 us, float32 205 and 26; 31 x 80 -> 944 43 and 18, 61 and 23;
// 2048 x 512 -> 512 bfloat16 43.5 and 42.1.  dx alone, one strip and two, where they do not pay: 16k x 64 -> 256 bfloat16 11.5 and 14, float32
// 16 and 19, 2048 x 512 -> 512 float32 27 and 28.
static int dx_each(Tile t, int64_t rows, int64_t c, int steps, bool bf) {
  const int64_t tiles = ceil_div64(rows, 64) * ceil_div64(c, 64);
  int best = steps;
  if (t != kTile64x64 || tiles > 256) return best;
  const int64_t step_ns = bf ? 400 : 850, strips_ns = 6000;
  int64_t least = steps * step_ns;
  for (int per_cu = 1; per_cu <= 2; ++per_cu) {
    const int64_t strips = 256 * per_cu / tiles;
    if (strips < 2) continue;
    const int64_t each = std::max<int64_t>(ceil_div64(steps, strips), 4), ns = each * step_ns * (bf ? 1 : per_cu) + strips_ns;
    if (ns < least) { least = ns; best = (int)each; }
  }
  return best;
}
static inline int64_t q_side(Tile t) { return t <= kTile128x64 ? 64 : t == kTile128x128 ? 128 : 256; }

struct GatePlan {
  int es, ce;                       // bytes of an activation, activations in 16 bytes
  int fp, cp;
  bool pad_w, pad_x;
  Tile gate_tile, dx_tile, dw_tile;
  int strips;
  int64_t strip_rows;
  int db_tiles;
  int dx_each, dx_strips, c4;
  size_t w_bytes, x_bytes, dgu_bytes, part_bytes, db_bytes, dx_bytes;
};

static GatePlan gate_plan(const ssmi_gated_desc* d) {
  GatePlan p = {};
  p.es = d->dtype == SSMI_BF16 ? 2 : 4;
  p.ce = 16 / p.es;
  p.fp = (int)up_to(d->f, p.ce);
  p.cp = (int)up_to(d->c, p.ce);

  const bool bf = d->dtype == SSMI_BF16;
  p.dx_tile = tile_for_dx(d->rows, d->c, bf);
  p.pad_w = p.fp != d->f || d->param_dtype != d->dtype;
  p.pad_x = p.cp != d->c || d->x_ld % p.ce != 0;
  p.w_bytes = p.pad_w ? 2 * up256((size_t)d->c * p.fp * p.es) : 0;
  p.x_bytes = p.pad_x ? up256((size_t)d->rows * p.cp * p.es) : 0;
  const int sides = bf ? kGradSides<bf16> : kGradSides<float>;
  p.gate_tile = tile_for(d->rows, 2 * (int64_t)d->f, bf);
  p.dgu_bytes = up256((size_t)d->rows * sides * p.fp * p.es);
  // strips of the weight gradient: one round of workgroups (two to a CU), each strip long enough to be worth its partial sums (512 rows)
  // and, in float32, short enough for the running sums (4096 rows: 2^-24 sqrt(4096) of a term)
  const int64_t most = ceil_div64(d->rows, 512), least = bf ? 1 : ceil_div64(d->rows, 4096);
  p.dw_tile = tile_for_dw(d->rows, d->c, 2 * p.fp, bf, most);
  int64_t strips = ceil_div64(512, ceil_div64(2 * p.fp, 128) * ceil_div64(d->c, q_side(p.dw_tile)));
  strips = strips < most ? strips : most;
  strips = strips > least ? strips : least;
  // a strip is addressed with 32-bit offsets from its first row, and the loop asks for kPastRows more of [dg | du] and of x
  const int64_t row_bytes = p.es * std::max<int64_t>(sides * (int64_t)p.fp, p.pad_x ? p.cp : d->x_ld);
  const int64_t reach = std::max<int64_t>((kReach / row_bytes - kPastRows) / 64 * 64, 64);
  p.strip_rows = std::min(up_to(ceil_div64(d->rows, strips), 64), reach);
  p.strips = (int)ceil_div64(d->rows, p.strip_rows);
  p.part_bytes = up256((size_t)p.strips * d->c * 2 * p.fp * 4);
  p.c4 = (int)up_to(d->c, 4);
  const int steps = sides * (int)ceil_div64(p.fp * p.es, ProductShape<1, 1>::kStep);
  p.dx_each = dx_each(p.dx_tile, d->rows, d->c, steps, bf);
  p.dx_strips = (int)ceil_div64(steps, p.dx_each);
  p.dx_bytes = p.dx_strips > 1 ? up256((size_t)p.dx_strips * d->rows * p.c4 * 4) : 0;
  p.db_tiles = (int)ceil_div64(d->rows, q_side(p.gate_tile));
  p.db_bytes = up256((size_t)p.db_tiles * 2 * p.fp * 4);
  return p;
}

static ssmi_status check_desc(const char* who, const ssmi_gated_desc* d) {
  SSMI_REQUIRE(d, SSMI_E_INVALID_ARG, "%s: null descriptor", who);
  SSMI_REQUIRE(d->rows > 0 && d->c > 0 && d->f > 0, SSMI_E_SHAPE, "%s: %lld rows, %d channels, %d units", who, (long long)d->rows, d->c, d->f);
  SSMI_REQUIRE(d->c <= 65536 && d->f <= 65536 && d->rows < (1ll << 31), SSMI_E_UNSUPPORTED, "%s: at most 65536 channels and units and 2^31 - 1 rows", who);
  SSMI_REQUIRE(d->x_ld >= d->c && d->y_ld >= d->f && d->x_ld <= (1 << 20) && d->y_ld <= (1 << 20), SSMI_E_SHAPE,
               "%s: row strides %lld, %lld under %d channels, %d units (or over 2^20)", who, (long long)d->x_ld, (long long)d->y_ld, d->c, d->f);
  SSMI_REQUIRE(d->act >= SSMI_GATE_SWISH && d->act <= SSMI_GATE_SIGMOID, SSMI_E_INVALID_ARG, "%s: unknown activation %d", who, d->act);
  SSMI_REQUIRE(d->dtype == SSMI_F32 || d->dtype == SSMI_BF16, SSMI_E_UNSUPPORTED, "%s: unknown activation dtype %d", who, d->dtype);
  SSMI_REQUIRE(d->param_dtype == SSMI_F32 || (d->param_dtype == SSMI_BF16 && d->dtype == SSMI_BF16), SSMI_E_UNSUPPORTED,
               "%s: parameters are float32, or bfloat16 under bfloat16 activations", who);
  SSMI_REQUIRE((d->c + kPastRows) * up_to(d->f, 8) * 4 <= kReach, SSMI_E_UNSUPPORTED, "%s: a kernel that comes within %lld rows of 2 GiB", who, (long long)kPastRows);
  return SSMI_OK;
}

// every launch of a call inside kMostBlocks, checked in front of the first
static ssmi_status check_launches(const char* who, const ssmi_gated_desc* d, const GatePlan& p, bool dx, bool dw) {
  int64_t most = ceil_div64(d->rows, q_side(p.gate_tile)) * ceil_div64(d->f, 64);
  const int64_t dx_side = p.dx_tile == kTile64x64 ? 64 : p.dx_tile == kTile256x256 ? 256 : 128;
  if (dx) most = std::max(most, ceil_div64(d->rows, q_side(p.dx_tile)) * ceil_div64(d->c, dx_side) * p.dx_strips);
  if (dw) most = std::max(most, ceil_div64(d->c, q_side(p.dw_tile)) * ceil_div64(2 * p.fp, 128) * p.strips);
  SSMI_REQUIRE(most < kMostBlocks, SSMI_E_UNSUPPORTED, "%s: %lld rows of %d channels and %d units are too many for one launch", who, (long long)d->rows, d->c, d->f);
  return SSMI_OK;
}

static inline bool aligned(const void* p, int b) { return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0; }

// how rows may be stored: 0 value by value, 1 four values at a time, 2 eight
static inline int vec_of(int64_t ld, const void* p, int es) { return ld % 4 || !aligned(p, 4 * es) ? 0 : ld % 8 || !aligned(p, 16) ? 1 : 2; }

// operands in the tile engine's form, padded copies in ws where they are not in it already
struct Staged {
  const void *x, *wg, *wu;
  int64_t x_ld, w_ld;
  char* ws;      // what is left of the workspace
};
template <typename T>
static Staged stage_operands(const ssmi_gated_desc* d, const GatePlan& p, const void* x, const void* wg, const void* wu, void* ws, hipStream_t st) {
  Staged s = {x, wg, wu, d->x_ld, d->f, static_cast<char*>(ws)};
  PadJobs jobs = {};
  int n = 0;
  int64_t most = 0;
  auto add = [&](const void* src, int64_t ld, int64_t rows, int cols, int cols_p, bool bf) {
    jobs.job[n++] = {src, s.ws, ld, rows, cols, cols_p, bf};
    most = most > rows * (cols_p / 4) ? most : rows * (cols_p / 4);
    const void* at = s.ws;
    s.ws += up256((size_t)rows * cols_p * sizeof(T));
    return at;
  };
  if (p.pad_w) {
    s.wg = add(wg, d->f, d->c, d->f, p.fp, d->param_dtype == SSMI_BF16);
    s.wu = add(wu, d->f, d->c, d->f, p.fp, d->param_dtype == SSMI_BF16);
    s.w_ld = p.fp;
  }
  if (p.pad_x) {
    s.x = add(x, d->x_ld, d->rows, d->c, p.cp, d->dtype == SSMI_BF16);
    s.x_ld = p.cp;
  }
  if (n) {
    const int64_t blocks = ceil_div64(most, 256);
    hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)n), dim3(256), 0, st, jobs);
  }
  return s;
}

template <typename S, int SP, int SQ>
static constexpr int tile_lds() {
  constexpr int stages = S::kStages * S::kStage, rows = TileRows<SP, SQ, 64, S::kAtOnce>::kBytes;
  return stages > rows ? stages : rows;
}

template <typename T, int SP, int SQ, bool BWD, bool LONG>
static ssmi_status launch_gate_long(GateArgs a, hipStream_t st) {
  typedef GateSides<T, SP, SQ, LONG> S;
  a.np = (unsigned)ceil_div64(a.f, S::kHalf);
  a.nq = (unsigned)ceil_div64(a.rows, SQ * 64);
  set_last_kernel("gate_kernel<%s, %d, %d, %s>", sizeof(T) == 2 ? "bf16" : "float", SP, SQ, BWD ? "backward" : "forward");
  hipLaunchKernelGGL((gate_kernel<T, SP, SQ, BWD, LONG>), dim3(a.np * a.nq), dim3(256), (tile_lds<S, SP, SQ>()), st, a);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}
template <typename T, int SP, int SQ, bool BWD>
static ssmi_status launch_gate_as(const GateArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 4) {
    if (a.c > kChunk) return launch_gate_long<T, SP, SQ, BWD, true>(a, st);
  }
  return launch_gate_long<T, SP, SQ, BWD, false>(a, st);
}
template <typename T, bool BWD>
static ssmi_status launch_gate(Tile t, const GateArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (t == kTile128x256) return launch_gate_as<T, 2, 4, BWD>(a, st);
  }
  return t == kTile128x128 ? launch_gate_as<T, 2, 2, BWD>(a, st) : launch_gate_as<T, 2, 1, BWD>(a, st);
}
template <typename T, int SP, int SQ>
static ssmi_status launch_dx_as(GateDxArgs a, hipStream_t st) {
  typedef DxSides<T, SP, SQ> S;
  a.np = (unsigned)ceil_div64(a.c, SP * 64);
  a.nq = (unsigned)ceil_div64(a.rows, SQ * 64);
  set_last_kernel("gate_dx_kernel<%s, %d, %d>", sizeof(T) == 2 ? "bf16" : "float", SP, SQ);
  hipLaunchKernelGGL((gate_dx_kernel<T, SP, SQ>), dim3(a.np * a.nq * (unsigned)a.strips), dim3(256), (tile_lds<S, SP, SQ>()), st, a);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}
template <typename T, int SP, int SQ>
static ssmi_status launch_dw_as(GateDwArgs a, int strips, hipStream_t st) {
  typedef DwSides<T, SP, SQ> S;
  a.np = (unsigned)ceil_div64(2 * a.fp, SP * 64);
  a.nq = (unsigned)ceil_div64(a.c, SQ * 64);
  set_last_kernel("gate_dw_kernel<%s, %d, %d>", sizeof(T) == 2 ? "bf16" : "float", SP, SQ);
  hipLaunchKernelGGL((gate_dw_kernel<T, SP, SQ>), dim3(a.np * a.nq * (unsigned)strips), dim3(256), (tile_lds<S, SP, SQ>()), st, a);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}

template <typename T>
static ssmi_status launch_dx(Tile t, const GateDxArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (t == kTile256x256) return launch_dx_as<T, 4, 4>(a, st);
  }
  if (t == kTile128x128) return launch_dx_as<T, 2, 2>(a, st);
  return t == kTile128x64 ? launch_dx_as<T, 2, 1>(a, st) : launch_dx_as<T, 1, 1>(a, st);
}
template <typename T>
static ssmi_status launch_dw(Tile t, const GateDwArgs& a, int strips, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (t == kTile128x256) return launch_dw_as<T, 2, 4>(a, strips, st);
  }
  return t == kTile128x128 ? launch_dw_as<T, 2, 2>(a, strips, st) : launch_dw_as<T, 2, 1>(a, strips, st);
}

template <typename T, typename P, int MB>
static void launch_rows_mb(const GateArgs& a, bool vec, hipStream_t st) {
  constexpr int kWaves = MB <= 2 ? 16 : 8;
  const dim3 grid((unsigned)ceil_div64(a.f, 32), (unsigned)ceil_div64(a.rows, MB)), block(64 * kWaves);
  const size_t lds = (size_t)MB * a.c * 4;
  if (vec) hipLaunchKernelGGL((gate_rows_kernel<T, P, MB, kWaves, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((gate_rows_kernel<T, P, MB, kWaves, false>), grid, block, lds, st, a);
}
template <typename T, typename P>
static ssmi_status launch_rows(const GateArgs& a, hipStream_t st) {
  const bool vec = a.f % 8 == 0 && aligned(a.wg, 16) && aligned(a.wu, 16);
  if (a.rows == 1) launch_rows_mb<T, P, 1>(a, vec, st);
  else if (a.rows == 2 || sizeof(P) == 2) launch_rows_mb<T, P, 2>(a, vec, st);      // bfloat16 parameters: see takes_rows_kernel
  else if (a.rows <= 4) launch_rows_mb<T, P, 4>(a, vec, st);
  else launch_rows_mb<T, P, 8>(a, vec, st);
  SSMI_LAUNCH_CHECK();
  return SSMI_OK;
}

// Rows that gate_rows_kernel takes: as many as it beats the tiles at.  Its and their times in us:
//   bfloat16                        1 x 512 -> 2048 3.9 and 5.9, 2 rows 4.7 and 5.9, 4 rows 6.1 and 5.9, 1 x 2048 -> 4096 14 and 19
//   bfloat16, float32 parameters    1 x 512 -> 2048 4.2 and 12.5, 16 rows 8.7 and 12.5: the tiles need a bfloat16 copy of the parameters;
//                                   4 x 96 -> 301 5.9 and 6.3, 8 rows 8.0 and 6.5
//   float32                         1 x 512 -> 2048 4.0 and 20, 24 rows 9.8 and 20.6, 48 rows 17 and 21: few tiles cannot hide a long reduction;
//                                   16 x 96 -> 301 7.6 and 8.7
// Its rows of x have to fit LDS: eight of 2048 float32.
static bool takes_rows_kernel(const ssmi_gated_desc* d) {
  const bool long_c = d->c >= 256;
  const int most = d->param_dtype == SSMI_BF16 ? 2 : d->dtype == SSMI_BF16 ? (long_c ? 16 : 4) : (long_c ? 32 : 16);
  return d->rows <= most && d->c <= 2048;
}

template <typename T>
static ssmi_status gated_fwd(const ssmi_gated_desc* d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* y, void* ws,
                             hipStream_t st) {
  GateArgs a = {};
  a.bg = bg; a.bu = bu; a.out = y; a.out_ld = d->y_ld; a.rows = d->rows; a.c = d->c; a.f = d->f; a.act = d->act;
  a.bf_params = d->param_dtype == SSMI_BF16;
  if (takes_rows_kernel(d)) {
    a.x = x; a.wg = wg; a.wu = wu; a.x_ld = d->x_ld;
    if constexpr (sizeof(T) == 2) {
      if (a.bf_params) return launch_rows<T, bf16>(a, st);
    }
    return launch_rows<T, float>(a, st);
  }
  const GatePlan p = gate_plan(d);
  const Staged s = stage_operands<T>(d, p, x, wg, wu, ws, st);
  SSMI_LAUNCH_CHECK();
  a.x = s.x; a.wg = s.wg; a.wu = s.wu; a.x_ld = s.x_ld; a.w_ld = s.w_ld; a.fp = p.fp;
  a.vec_out = vec_of(d->y_ld, y, p.es);
  return launch_gate<T, false>(p.gate_tile, a, st);
}

template <typename T>
static ssmi_status gated_bwd(const ssmi_gated_desc* d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, const void* dy, void* dx,
                             void* dwg, void* dwu, void* dbg, void* dbu, void* ws, hipStream_t st) {
  const GatePlan p = gate_plan(d);
  Staged s = stage_operands<T>(d, p, x, wg, wu, ws, st);
  void* const dgu = s.ws;
  float* const part = reinterpret_cast<float*>(s.ws + p.dgu_bytes);
  float* const dbp = reinterpret_cast<float*>(s.ws + p.dgu_bytes + p.part_bytes);
  float* const dxp = dx && p.dx_strips > 1 ? reinterpret_cast<float*>(s.ws + p.dgu_bytes + p.part_bytes + p.db_bytes) : nullptr;
  const int bf = d->param_dtype == SSMI_BF16;
  GateArgs a = {};
  a.x = s.x; a.wg = s.wg; a.wu = s.wu; a.bg = bg; a.bu = bu; a.dy = dy; a.out = dgu;
  SSMI_LAUNCH_CHECK();
  a.rows = d->rows; a.x_ld = s.x_ld; a.w_ld = s.w_ld; a.out_ld = kGradSides<T> * (int64_t)p.fp; a.dy_ld = d->y_ld;
  a.c = d->c; a.f = d->f; a.fp = p.fp; a.act = d->act; a.bf_params = bf;
  a.db = dbg || dbu ? dbp : nullptr;
  a.vec_out = 2;      // rows of whole 16 bytes
  a.vec_dy = vec_of(d->y_ld, dy, p.es);
  ssmi_status r = launch_gate<T, true>(p.gate_tile, a, st);
  if (r != SSMI_OK) return r;
  const int dx_vec = vec_of(d->x_ld, dx, p.es);
  if (dx) {
    GateDxArgs b = {};
    b.part = dxp; b.each = p.dx_each; b.strips = p.dx_strips; b.c4 = p.c4;
    b.dgu = dgu; b.wg = s.wg; b.wu = s.wu; b.dx = dx; b.rows = d->rows; b.w_ld = s.w_ld; b.dx_ld = d->x_ld; b.c = d->c; b.fp = p.fp;
    b.vec_out = dx_vec;
    r = launch_dx<T>(p.dx_tile, b, st);
    if (r != SSMI_OK) return r;
  }
  const bool dw = dwg || dwu;
  if (dw) {
    GateDwArgs b = {};
    b.x = s.x; b.dgu = dgu; b.part = part; b.rows = d->rows; b.x_ld = s.x_ld; b.strip_rows = p.strip_rows; b.c = d->c; b.cp = p.cp; b.fp = p.fp;
    r = launch_dw<T>(p.dw_tile, b, p.strips, st);
    if (r != SSMI_OK) return r;
  }
  if (dw || a.db || dxp) {
    ReduceArgs b = {};
    b.part = part; b.db = a.db; b.dwg = dwg; b.dwu = dwu; b.dbg = dbg; b.dbu = dbu; b.c = dw ? d->c : 0;
    b.strips = p.strips; b.db_tiles = p.db_tiles; b.f = d->f; b.fp = p.fp; b.bf = bf;
    b.dx_part = dxp; b.dx = dx; b.rows = d->rows; b.dx_ld = d->x_ld; b.dx_strips = p.dx_strips; b.dx_c = d->c; b.c4 = p.c4; b.dx_vec = dx_vec;
    b.dw_blocks = (unsigned)ceil_div64((b.c + (a.db ? 1 : 0)) * (p.fp / 2), kReduce);
    const unsigned dx_blocks = dxp ? (unsigned)ceil_div64(d->rows * (p.c4 / 4), kReduce) : 0;
    hipLaunchKernelGGL((gate_reduce_kernel<T>), dim3(b.dw_blocks + dx_blocks), dim3(kReduce), 0, st, b);
    SSMI_LAUNCH_CHECK();
  }
  return SSMI_OK;
}

}  // namespace ssmi

using namespace ssmi;

extern "C" {

size_t ssmi_gated_ff_workspace_bytes(const ssmi_gated_desc* d, int32_t backward) {
  if (check_desc("gated_ff_workspace_bytes", d) != SSMI_OK) return 0;
  const GatePlan p = gate_plan(d);
  if (!backward) return takes_rows_kernel(d) ? 0 : p.w_bytes + p.x_bytes;
  return p.w_bytes + p.x_bytes + p.dgu_bytes + p.part_bytes + p.db_bytes + p.dx_bytes;
}

ssmi_status ssmi_gated_ff_fwd(const ssmi_gated_desc* d, const void* x, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, void* y,
                              void* ws, size_t ws_bytes, void* stream) {
  const ssmi_status st = check_desc("gated_ff_fwd", d);
  if (st != SSMI_OK) return st;
  SSMI_REQUIRE(x && w_gate && w_up && y, SSMI_E_INVALID_ARG, "gated_ff_fwd: null pointer");
  SSMI_REQUIRE(!b_gate == !b_up, SSMI_E_INVALID_ARG, "gated_ff_fwd: both biases or none");
  const size_t need = ssmi_gated_ff_workspace_bytes(d, 0);
  SSMI_REQUIRE(need == 0 || (ws && ws_bytes >= need), SSMI_E_WORKSPACE, "gated_ff_fwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  SSMI_REQUIRE(aligned(ws, 16), SSMI_E_INVALID_ARG, "gated_ff_fwd: the workspace must be 16-byte aligned");
  SSMI_REQUIRE(takes_rows_kernel(d) || ((aligned(x, 16) || gate_plan(d).pad_x) && ((aligned(w_gate, 16) && aligned(w_up, 16)) || gate_plan(d).pad_w)), SSMI_E_INVALID_ARG,
               "gated_ff_fwd: x and the kernels must be 16-byte aligned");
  const ssmi_status fits = takes_rows_kernel(d) ? SSMI_OK : check_launches("gated_ff_fwd", d, gate_plan(d), false, false);
  if (fits != SSMI_OK) return fits;
  return dispatch_dtype(d->dtype, [&](auto tag) -> ssmi_status { return gated_fwd<decltype(tag)>(d, x, w_gate, w_up, b_gate, b_up, y, ws, as_stream(stream)); });
}

ssmi_status ssmi_gated_ff_bwd(const ssmi_gated_desc* d, const void* x, const void* w_gate, const void* w_up, const void* b_gate, const void* b_up, const void* dy,
                              void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, void* ws, size_t ws_bytes, void* stream) {
  const ssmi_status st = check_desc("gated_ff_bwd", d);
  if (st != SSMI_OK) return st;
  SSMI_REQUIRE(x && w_gate && w_up && dy, SSMI_E_INVALID_ARG, "gated_ff_bwd: null pointer");
  SSMI_REQUIRE(!b_gate == !b_up, SSMI_E_INVALID_ARG, "gated_ff_bwd: both biases or none");
  const size_t need = ssmi_gated_ff_workspace_bytes(d, 1);
  SSMI_REQUIRE(ws && ws_bytes >= need, SSMI_E_WORKSPACE, "gated_ff_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
  SSMI_REQUIRE(aligned(ws, 16), SSMI_E_INVALID_ARG, "gated_ff_bwd: the workspace must be 16-byte aligned");
  const GatePlan p = gate_plan(d);
  SSMI_REQUIRE((aligned(x, 16) || p.pad_x) && ((aligned(w_gate, 16) && aligned(w_up, 16)) || p.pad_w), SSMI_E_INVALID_ARG,
               "gated_ff_bwd: x and the kernels must be 16-byte aligned");
  const ssmi_status fits = check_launches("gated_ff_bwd", d, p, dx, dw_gate || dw_up);
  if (fits != SSMI_OK) return fits;
  return dispatch_dtype(d->dtype, [&](auto tag) -> ssmi_status {
    return gated_bwd<decltype(tag)>(d, x, w_gate, w_up, b_gate, b_up, dy, dx, dw_gate, dw_up, db_gate, db_up, ws, as_stream(stream));
  });
}

}  // extern "C"
