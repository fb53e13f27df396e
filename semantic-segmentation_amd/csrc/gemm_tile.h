// Matrix-core tile engine of the row operators: D[p][q] = sum_k P[p][k] Q[q][k] for one workgroup's tile, both operands streamed
// through LDS, float32 accumulation.  Used by the gated feed-forward unit (gated.hip).
//
// Roles.  q is the row index of the result in memory (a pixel, or an input channel of a weight gradient), p runs along its
// contiguous axis: the accumulator layout of the 32x32 instructions gives a lane one q and runs of four consecutive p, i.e. vector
// stores and epilogues that see a pixel's neighbouring channels.
// Either operand comes in one of two memory forms:
//   rows:  [index][k], k contiguous             - staged as 128-byte rows, read back with ds_read_b128
//   cols:  [k][index], index contiguous         - staged as k rows, read back transposed (ds_read_tr16_b64 for bfloat16, single words
//                                                 for float32), so Keras kernels [in][out] and weight gradients need no transposed copy
// A K step is 128 bytes of a row: 64 bfloat16 or 32 float32 values.  Four waves split the tile 2 x 2; a wave owns SP x SQ
// accumulators of 32 x 32.
// Staging: global -> LDS directly, 16 bytes a lane; the LDS image is linear in the lane order, so the swizzle against bank conflicts
// is applied to the source: slot s of a row holds piece s ^ f(row), f chosen so that one read of a wave spreads over all banks.
// Two stages: the loads of step t + 1 are issued behind the one barrier of step t and have its whole arithmetic to arrive.
// Lanes that must see zeros (past the last row, past K) pass an out-of-range offset; the buffer check returns zeros.
// Everything is addressed from a per-tile 64-bit base, so tensors may be larger than 2 GiB; a tile's own extent may not.
#pragma once
#include "common.h"

namespace ssmi {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char* lds_bytes;

static constexpr int kStepBytes = 128;

__device__ __forceinline__ unsigned spread_blocks(unsigned b, unsigned n) {      // workgroups of one XCD take consecutive tiles (a bijection of [0, n))
  const unsigned q = n >> 3, r = n & 7u, x = b & 7u;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
}

// 64 lanes x 16 bytes from buffer offsets to LDS bytes [at, at + 1024), `at` uniform.  In assembly because the compiler, which cannot
// tell the two stages apart, would wait for every such load in front of the next LDS read; nothing is returned in registers, and the
// tile loop waits for them itself (stage_wait) in front of the barrier that publishes a stage.
__device__ __forceinline__ void stage16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff, unsigned at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}
__device__ __forceinline__ void stage_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// One operand of one tile.  N: indices of the tile (p or q), COLS: memory form.
template <typename T, int N, bool COLS>
struct Operand {
  static constexpr int kElems = 16 / (int)sizeof(T);                 // values per 16-byte piece
  static constexpr int kStepK = kStepBytes / (int)sizeof(T);
  static constexpr int kBytes = N * kStepBytes;                      // LDS bytes of one stage
  static constexpr int kLoads = kBytes / 4096;                       // per lane and step
  static constexpr int kRowBytes = COLS ? N * (int)sizeof(T) : kStepBytes;
  static constexpr int kRowsPerLoad = 4096 / kRowBytes;              // LDS rows that the workgroup stages with one load per lane
  static_assert(kBytes % 4096 == 0, "whole loads");

  unsigned voff[kLoads];
  int k_in;                      // the lane's first k of a step (rows) / its k row of load 0 (cols)
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned step_bytes;           // buffer offset from one K step to the next

  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!COLS) return row & 7;
    if constexpr (sizeof(T) == 2) return kRowBytes >= 256 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
    return ((row >> 2) & 1) << 3;
  }

  // base: element (index 0 of the tile, k 0); ld: elements from one memory row to the next; count: valid indices of the tile
  __device__ __forceinline__ void init(const T* base, int64_t ld, int count) {
    rsrc = make_rsrc(base, 0x7FFFFFFFu);
    const int tid = threadIdx.x;
    constexpr int kPieces = kRowBytes / 16;
    const int row = tid / kPieces, slot = tid % kPieces;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int rj = row + j * kRowsPerLoad;
      const int piece = slot ^ swizzle(rj);
      if constexpr (COLS) {
        voff[j] = piece * kElems < count ? (unsigned)(rj * ld * (int64_t)sizeof(T)) + piece * 16u : kOOB;
        if (j == 0) k_in = rj;
      } else {
        voff[j] = rj < count ? (unsigned)(rj * ld * (int64_t)sizeof(T)) + piece * 16u : kOOB;
        if (j == 0) k_in = piece * kElems;      // the same for every load: rows advance by multiples of eight
      }
    }
    step_bytes = COLS ? (unsigned)(ld * (kStepK * (int64_t)sizeof(T))) : (unsigned)kStepBytes;
  }

  // requests K step t into the stage at `lds`; left: valid k from this step's first on; skip: bytes in front of step 0
  __device__ __forceinline__ void request(lds_bytes lds, int t, int left, unsigned skip = 0) const {
    const unsigned soff = (unsigned)t * step_bytes + skip;
    const unsigned dst = (unsigned)(uintptr_t)lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int k = COLS ? k_in + j * kRowsPerLoad : k_in;
      stage16(rsrc, k < left ? voff[j] : kOOB, soff, dst + j * 4096);
    }
  }

  // the lane's part of fragment (32 indices from 32 * s on, k piece ks of four): eight bfloat16 or four float32
  struct Reader {
    unsigned at;      // byte address inside the stage, subtile 0, ks 0
    __device__ __forceinline__ void init(int lane) {
      const int r = lane & 31, hh = lane >> 5;
      if constexpr (!COLS) {
        at = (unsigned)(r * kStepBytes + ((hh ^ (r & 7)) << 4));
      } else if constexpr (sizeof(T) == 2) {
        const int sq = (lane >> 2) & 3, sp = lane & 3, gh = (lane >> 4) & 1;
        const int row = 8 * hh + sq;
        at = (unsigned)(row * kRowBytes + (((2 * gh + (sp >> 1)) ^ swizzle(row)) << 4) + ((sp & 1) << 3));
      } else {
        at = (unsigned)(4 * hh * kRowBytes + (r * 4 ^ (hh << 7)));
      }
    }
    __device__ __forceinline__ u32x4 get(lds_bytes stage, int s, int ks) const {
      if constexpr (!COLS) {
        return *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(stage + s * 32 * kStepBytes + (at ^ (unsigned)(ks << 5)));
      } else if constexpr (sizeof(T) == 2) {
        // subtiles lie 64 bytes apart inside the swizzled 256 (128) bytes
        constexpr int kIn = kRowBytes >= 256 ? 4 : 2;
        lds_bytes p = stage + (at ^ (unsigned)((s % kIn) << 6)) + (s / kIn) * 256 + ks * 16 * kRowBytes;
        struct { s16x4 lo, hi; } pr;
        // rows four on share the swizzle of 256-byte rows ((row & 3)) and of 128-byte rows ((row >> 1) & 1)
        pr.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        pr.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * kRowBytes));
        return __builtin_bit_cast(u32x4, pr);
      } else {
        lds_bytes p = stage + (at ^ (unsigned)((s & 1) << 7)) + (s >> 1) * 256 + ks * 8 * kRowBytes;
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<__attribute__((address_space(3))) unsigned*>(p + j * kRowBytes);
        return v;
      }
    }
  };
};

template <typename T>
__device__ __forceinline__ f32x16 mfma_step(u32x4 p, u32x4 q, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
  } else {
    const f32x4 a = __builtin_bit_cast(f32x4, p), b = __builtin_bit_cast(f32x4, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
}

// The K loop of a tile.  Sides: request(stage, t) stages step t, p(stage, i, ks) / q(stage, j, ks) read fragments.  Fragments are read
// one k piece ahead of their arithmetic, also over the step boundary: the barrier sits in front of a step's LAST piece, whose
// fragments are in registers already, so the first reads of the next step run under it.
template <typename T, int SP, int SQ, typename Sides>
__device__ __forceinline__ void tile_product(const Sides& sides, lds_bytes lds, int steps, f32x16 (&acc)[SP][SQ]) {
#pragma unroll
  for (int i = 0; i < SP; ++i)
#pragma unroll
    for (int j = 0; j < SQ; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;
  if (steps <= 0) return;
  constexpr int kStage = Sides::kStage;
  u32x4 p[2][SP], q[2][SQ];
  auto read = [&](int buf, lds_bytes stage, int ks) {
#pragma unroll
    for (int i = 0; i < SP; ++i) p[buf][i] = sides.p(stage, i, ks);
#pragma unroll
    for (int j = 0; j < SQ; ++j) q[buf][j] = sides.q(stage, j, ks);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
      for (int j = 0; j < SQ; ++j) acc[i][j] = mfma_step<T>(p[buf][i], q[buf][j], acc[i][j]);
  };
  sides.request(lds, 0);
  stage_wait();
  __syncthreads();
  if (steps > 1) sides.request(lds + kStage, 1);
  read(0, lds, 0);
  for (int t = 0; t < steps; ++t) {
    lds_bytes cur = lds + (t & 1) * kStage, nxt = lds + ((t + 1) & 1) * kStage;
    read(1, cur, 1);
    multiply(0);
    read(0, cur, 2);
    multiply(1);
    read(1, cur, 3);
    multiply(0);
    stage_wait();
    __syncthreads();      // step t + 1 is there, and nobody reads step t any more
    __builtin_amdgcn_sched_barrier(0);
    if (t + 2 < steps) sides.request(cur, t + 2);
    if (t + 1 < steps) read(0, nxt, 0);
    multiply(1);
  }
}

// The accumulators of a tile as rows in LDS, for an epilogue in memory order: q rows of 2 * 32 * SP float32 values, then `body(row, q,
// col)` for every row and every fourth column under COLS, consecutive lanes on consecutive columns.  From the accumulator layout a
// store touches 32 rows for 16 bytes each, and unrolling an epilogue over 256 registers overruns the instruction cache (the gated
// unit's first form: 650 us for 65536 x 512 -> 2048, of which the products take 300).  Rows are padded by four values: the writes, one q
// a lane, then step through the banks.  128 q rows go at a time (the large tile's 256 do not fit).
// pos(i): first column of subtile i of this wave.
template <int SP, int SQ>
struct TileRows {
  static constexpr int kWidth = SP * 64, kStride = kWidth + 4, kAtOnce = SQ > 2 ? 2 : SQ, kRows = 64 * kAtOnce;
  static constexpr int kBytes = kRows * kStride * 4;
};
// Rounds go in groups of GROUP unrolled ones (`body`'s last argument counts inside a group, so it may index registers); early(first
// row, rows per round, q_of) runs in front of a pass's LDS writes, next() behind every group.
template <int SP, int SQ, int COLS, int GROUP, typename Pos, typename Early, typename Body, typename Next>
__device__ __forceinline__ void tile_rows(const f32x16 (&acc)[SP][SQ], float* lds, int wq, Pos pos, Early early, Body body, Next next) {
  typedef TileRows<SP, SQ> R;
  constexpr int kLanes = COLS / 4, kPerRound = 256 / kLanes, kRounds = R::kRows / kPerRound;
  const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5;
  const int col = (threadIdx.x % kLanes) * 4, first = threadIdx.x / kLanes;
#pragma unroll
  for (int pass = 0; pass < SQ / R::kAtOnce; ++pass) {
    auto q_of = [&](int row) { return (row / (32 * R::kAtOnce)) * (32 * SQ) + pass * (32 * R::kAtOnce) + row % (32 * R::kAtOnce); };
    early(first, kPerRound, q_of);
    if (pass) __syncthreads();
#pragma unroll
    for (int jj = 0; jj < R::kAtOnce; ++jj)
#pragma unroll
      for (int i = 0; i < SP; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f32x16& a = acc[i][pass * R::kAtOnce + jj];
          *reinterpret_cast<f32x4*>(lds + (wq * (32 * R::kAtOnce) + jj * 32 + r) * R::kStride + pos(i) + 8 * k + 4 * hh) =
              f32x4{a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]};
        }
    __syncthreads();
    static_assert(kRounds % GROUP == 0, "whole groups");
#pragma unroll 1
    for (int n = 0; n < kRounds; n += GROUP) {
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        const int row = first + (n + i) * kPerRound;
        body(lds + row * R::kStride, q_of(row), col, i);
      }
      next();
    }
  }
}

}  // namespace ssmi
