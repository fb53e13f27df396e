// Matrix-core tile engine of the row operators: D[p][q] = sum_k P[p][k] Q[q][k] for one workgroup's tile, both operands streamed
// through LDS, float32 accumulation.  Used by the gated feed-forward unit (gated.hip).
//
// Roles.  q is the row index of the result in memory (a pixel, or an input channel of a weight gradient), p runs along its
// contiguous axis: the accumulator layout of the 32x32 instructions gives a lane one q and runs of four consecutive p, i.e. vector
// stores and epilogues that see a pixel's neighbouring channels.
// Either operand comes in one of two memory forms:
//   rows:  [index][k], k contiguous             - staged as rows of STEP bytes, read back with ds_read_b128
//   cols:  [k][index], index contiguous         - staged as k rows, read back transposed (ds_read_tr16_b64 for bfloat16, single words
//                                                 for float32), so Keras kernels [in][out] and weight gradients need no transposed copy
// A K step is STEP = 128 or 64 bytes of a row: 64 or 32 bfloat16, half as many float32 values.  Four waves split the tile 2 x 2; a wave owns SP x SQ
// accumulators of 32 x 32.
// Staging: global -> LDS directly, 16 bytes a lane; the LDS image is linear in the lane order, so the swizzle against bank conflicts
// is applied to the source: slot s of a row holds piece s ^ f(row), f chosen so that one read of a wave spreads over all banks.
// kStages stages: a step's one barrier sits in front of its last fragments' arithmetic; behind it the stage is free for the loads of
// step t + kStages, which then have the arithmetic of kStages - 1 steps to arrive.
// Lanes that must see zeros (past the last row, past K) pass an out-of-range offset; the buffer check returns zeros.
// Everything is addressed from a per-tile 64-bit base, so tensors may be larger than 2 GiB; a tile's own extent may not.
#pragma once
#include "common.h"

namespace ssmi {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) unsigned char* lds_bytes;

static constexpr int64_t kMostBlocks = 1 << 24;      // of 256 threads: a launch has fewer than 2^32 of them

__device__ __forceinline__ unsigned spread_blocks(unsigned b, unsigned n) {      // workgroups of one XCD take consecutive tiles (a bijection of [0, n))
  const unsigned q = n >> 3, r = n & 7u, x = b & 7u;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
}

// Which (p, q) tile a workgroup takes.  Consecutive workgroups of an XCD walk kGroupQ row tiles under one column tile, then the
// next column tile: the workgroups of an XCD that run together share a few row tiles and column tiles through its L2
// (1, 2, 4, 8, 16 measured within 3 % of each other).
static constexpr int kGroupQ = 4;
struct TileAt { int p, q; };
__device__ __forceinline__ TileAt tile_at(unsigned v, unsigned np, unsigned nq) {
  const unsigned per = kGroupQ * np, grp = v / per, in = v - grp * per;
  const unsigned gq = min((unsigned)kGroupQ, nq - grp * kGroupQ);
  // divisions run on the vector unit: back to scalars, the tile's addresses hang on them
  return {(int)__builtin_amdgcn_readfirstlane(in / gq), (int)__builtin_amdgcn_readfirstlane(grp * kGroupQ + in % gq)};
}

// 64 lanes x 16 bytes from buffer offsets to LDS bytes [at, at + 1024), `at` uniform.  In assembly because the compiler, which cannot
// tell the two stages apart, would wait for every such load in front of the next LDS read; nothing is returned in registers, and the
// tile loop waits for them itself (stage_wait, in order) in front of the barrier that publishes a stage.  The pause covers what M0 needs and
// the five wait states of a scalar operand that a vector instruction wrote (a spilled one, read back): the compiler does not look into
// assembly for them.
__device__ __forceinline__ void stage16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned soff, unsigned at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}
template <int LEFT>
__device__ __forceinline__ void stage_wait() {      // until at most LEFT loads are on their way
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// One operand of one tile.  N: indices of the tile (p or q), COLS: memory form, STEP: bytes of a K step.
template <typename T, int N, bool COLS, int STEP>
struct Operand {
  static constexpr int kElems = 16 / (int)sizeof(T);                 // values per 16-byte piece
  static constexpr int kStepK = STEP / (int)sizeof(T);
  static constexpr int kBytes = N * STEP;                      // LDS bytes of one stage
  static constexpr int kLoads = kBytes / 4096;                       // per lane and step
  static constexpr int kRowBytes = COLS ? N * (int)sizeof(T) : STEP;
  static constexpr int kRowsPerLoad = 4096 / kRowBytes;              // LDS rows that the workgroup stages with one load per lane
  static_assert(kBytes % 4096 == 0, "whole loads");

  unsigned voff[kLoads];
  int k_in;                      // the lane's first k of a step (rows) / its k row of load 0 (cols)
  __amdgpu_buffer_rsrc_t rsrc;
  unsigned step_bytes;           // buffer offset from one K step to the next

  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!COLS) return STEP == 128 ? (row >> 1) & 7 : (row >> 2) & 3;      // sixteen rows' 16-byte reads: all of the 64 banks
    if constexpr (sizeof(T) == 2) return kRowBytes >= 256 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
    return ((row >> 2) & 1) << 3;
  }

  // base: element (index 0 of the tile, k 0); ld: elements from one memory row to the next; count: valid indices of the tile
  __device__ __forceinline__ void init(const T* base, int64_t ld, int count) {
    rsrc = make_rsrc(base, 0x7FFFFFFFu);
    const int tid = threadIdx.x;
    constexpr int kRowPieces = kRowBytes / 16;
    const int row = tid / kRowPieces, slot = tid % kRowPieces;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int rj = row + j * kRowsPerLoad;
      const int piece = slot ^ swizzle(rj);
      if constexpr (COLS) {
        voff[j] = piece * kElems < count ? (unsigned)(rj * ld * (int64_t)sizeof(T)) + piece * 16u : kOOB;
        if (j == 0) k_in = rj;
      } else {
        voff[j] = rj < count ? (unsigned)(rj * ld * (int64_t)sizeof(T)) + piece * 16u : kOOB;
        if (j == 0) k_in = piece * kElems;      // the same for every load: rows advance by multiples of sixteen
      }
    }
    step_bytes = COLS ? (unsigned)(ld * (kStepK * (int64_t)sizeof(T))) : (unsigned)STEP;
  }

  // load j of K step t into the stage at `lds`; left: valid k from this step's first on (<= 0: none, zeros arrive); skip: bytes in
  // front of step 0
  __device__ __forceinline__ void one(lds_bytes lds, int t, int j, int left, unsigned skip = 0) const {
    stage16(rsrc, (COLS ? k_in + j * kRowsPerLoad : k_in) < left ? voff[j] : kOOB, (unsigned)t * step_bytes + skip,
            (unsigned)(uintptr_t)lds + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024 + j * 4096);
  }

  // the lane's part of fragment (32 indices from 32 * s on, k piece ks of four): eight bfloat16 or four float32
  struct Reader {
    unsigned at;      // byte address inside the stage, subtile 0, ks 0
    __device__ __forceinline__ void init(int lane) {
      const int r = lane & 31, hh = lane >> 5;
      if constexpr (!COLS) {
        at = (unsigned)(r * STEP + ((hh ^ swizzle(r)) << 4));
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
        return *reinterpret_cast<__attribute__((address_space(3))) u32x4*>(stage + s * 32 * STEP + (at ^ (unsigned)(ks << 5)));
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

// The K loop of a tile.  Sides: one(stage, t, j) is load j of step t (zeros for a step past the last), p(stage, i, ks) / q(stage, j, ks)
// read fragments.  Fragments are read one k piece ahead of their arithmetic, also over the step boundary: the barrier sits in front of a
// step's LAST piece, whose fragments are in registers already.  Behind it the next step's first reads and the loads of step t + kStages
// go between that piece's matrix instructions, one load each: in a row they would leave the matrix unit idle for as long as they take
// to issue.  Every step issues the same loads, so the waits count them and the loop has no special ends.
// float32 sums over long axes (Sides::kChunks) go in chunks of kChunk k that are added up at their ends: the error of a running sum grows with
// the root of its length, that of a chunk and of the sum over chunks does not show.  Gated unit, error of y at 1024, 4096 and 16384 channels
// 4.1e-7, 4.2e-7 and 4.6e-7 of its norm; running sums 8.4e-7, 1.7e-6 and 3.4e-6, the library's float32 products 8.3e-7, 1.7e-6 and 1.6e-6.
static constexpr int kChunk = 256;
template <typename T, int SP, int SQ, typename Sides>
__device__ __forceinline__ void tile_product(const Sides& sides, lds_bytes lds, int steps, f32x16 (&acc)[SP][SQ]) {
#pragma unroll
  for (int i = 0; i < SP; ++i)
#pragma unroll
    for (int j = 0; j < SQ; ++j)
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;
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
  constexpr int kStages = Sides::kStages, kPieces = Sides::kStep / 32, kAhead = (kStages - 2) * Sides::kLoads;
  constexpr int kLoads = Sides::kLoads, kPer = (kLoads + SP * SQ - 1) / (SP * SQ);
#pragma unroll
  for (int t = 0; t < kStages; ++t)
#pragma unroll
    for (int j = 0; j < kLoads; ++j) sides.one(lds + t * kStage, t, j);
  stage_wait<(kStages - 1) * kLoads>();
  __syncthreads();
  read(0, lds, 0);
  constexpr bool kChunks = sizeof(T) == 4 && Sides::kChunks;
  constexpr int kChunkSteps = kChunk * (int)sizeof(T) / Sides::kStep;
  f32x16 sum[kChunks ? SP : 1][kChunks ? SQ : 1];
  if constexpr (kChunks) {
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
      for (int j = 0; j < SQ; ++j) sum[i][j] = acc[i][j];      // zeros
  }
  int at = 0;
  for (int t = 0; t < steps; ++t) {
    if constexpr (kChunks) {
      if (t % kChunkSteps == 0 && t) {
#pragma unroll
        for (int i = 0; i < SP; ++i)
#pragma unroll
          for (int j = 0; j < SQ; ++j) {
            sum[i][j] += acc[i][j];
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.f;
          }
      }
    }
    lds_bytes cur = lds + at * kStage;
    at = at + 1 == kStages ? 0 : at + 1;
    lds_bytes nxt = lds + at * kStage;
#pragma unroll
    for (int ks = 0; ks + 1 < kPieces; ++ks) {
      read((ks + 1) & 1, cur, ks + 1);
      multiply(ks & 1);
    }
    stage_wait<kAhead>();
    __syncthreads();      // step t + 1 is there for everyone, and nobody reads step t any more
    __builtin_amdgcn_sched_barrier(0);
    read(0, nxt, 0);
#pragma unroll
    for (int m = 0; m < SP * SQ; ++m) {
      acc[m / SQ][m % SQ] = mfma_step<T>(p[1][m / SQ], q[1][m % SQ], acc[m / SQ][m % SQ]);
#pragma unroll
      for (int j = m * kPer; j < (m + 1) * kPer && j < kLoads; ++j) sides.one(cur, t + kStages, j);
      if (m * kPer < kLoads) __builtin_amdgcn_sched_barrier(0);
    }
  }
  if constexpr (kChunks) {
#pragma unroll
    for (int i = 0; i < SP; ++i)
#pragma unroll
      for (int j = 0; j < SQ; ++j) acc[i][j] += sum[i][j];
  }
  stage_wait<0>();      // the zeros of the steps past the last: the epilogue takes the LDS over
  __syncthreads();
}

// The accumulators of a tile as rows in LDS, for an epilogue in memory order: q rows of 2 * 32 * SP float32 values; consecutive lanes
// take consecutive columns, four each, out of COLS.  From the accumulator layout a store would touch 32 rows for 16 bytes each.  Rows
// are padded by four values: the writes, one q a lane, then step through the banks.  64 * kAtOnce q rows go at a time.
//   pos(i)                     first column of subtile i of this wave
//   early(pass)                in front of a pass's LDS writes
//   round(row, qc, i)          the lane's row of LDS values and its q: first() + qc.  UNROLL = kRounds makes qc and i constants, so that
//                              an epilogue without branches keeps many rounds in flight and addresses its rows with scalars.
template <int SP, int SQ, int COLS, int AT_ONCE = (SQ > 2 ? 2 : SQ)>
struct TileRows {
  static constexpr int kWidth = SP * 64, kStride = kWidth + 4, kAtOnce = AT_ONCE, kRows = 64 * kAtOnce, kPasses = SQ / kAtOnce;
  static constexpr int kBytes = kRows * kStride * 4;
  static constexpr int kLanes = COLS / 4, kPerRound = 256 / kLanes, kRounds = kRows / kPerRound, kHalf = 32 * kAtOnce;
  static_assert(kHalf % kPerRound == 0 && COLS <= kWidth, "rounds stay inside a wave's rows");
  static __device__ __forceinline__ int first() { return (int)threadIdx.x / kLanes; }
  static __device__ __forceinline__ int col() { return (int)(threadIdx.x % kLanes) * 4; }
  static __device__ __forceinline__ constexpr int q_of(int pass, int i) {
    return (i * kPerRound / kHalf) * (32 * SQ) + pass * kHalf + i * kPerRound % kHalf;
  }
  template <int UNROLL, typename Pos, typename Early, typename Round>
  static __device__ __forceinline__ void run(const f32x16 (&acc)[SP][SQ], float* lds, int wq, Pos pos, Early early, Round round) {
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5;
    const float* const mine = lds + first() * kStride + col();
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      early(pass);
      if (pass) __syncthreads();
#pragma unroll
      for (int jj = 0; jj < kAtOnce; ++jj)
#pragma unroll
        for (int i = 0; i < SP; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const f32x16& a = acc[i][pass * kAtOnce + jj];
            *reinterpret_cast<f32x4*>(lds + (wq * kHalf + jj * 32 + r) * kStride + pos(i) + 8 * k + 4 * hh) =
                f32x4{a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]};
          }
      __syncthreads();
#pragma unroll UNROLL
      for (int i = 0; i < kRounds; ++i) {
        round(mine + i * kPerRound * kStride, q_of(pass, i), i);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // four rounds in flight: more cost registers the accumulators need
      }
    }
  }
};

// four values to memory, bfloat16 with one conversion per pair; PAST: past the caches
template <typename T, bool PAST = false>
__device__ __forceinline__ void put4(T* p, f32x4 v) {
  if constexpr (sizeof(T) == 2) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2), b = __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2);
    const u32x2 w = {__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)};
    if constexpr (PAST) __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(p));
    else *reinterpret_cast<u32x2*>(p) = w;
  } else {
    if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
    else *reinterpret_cast<f32x4*>(p) = v;
  }
}

// up to four values (n of them), in one access where `vec` allows it
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], int n, bool vec) {
  if (vec && n >= 4) {
    Act<T>::gst4(p, f32x4{v[0], v[1], v[2], v[3]});
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) Act<T>::gst(p + i, v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void fetch4(const T* p, float (&v)[4], int n, bool vec) {
  if (vec && n >= 4) {
    const f32x4 a = Act<T>::gld4(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? Act<T>::gld(p + i) : 0.f;
  }
}

// Sixteen consecutive bfloat16 columns of a row straight from the accumulator layout: the row's lower lane (hh = 0) holds columns 0-3 (`a`)
// and 8-11 (`b`), the upper one 4-7 and 12-15.  One swap of the wave's halves brings each lane eight of them: a 16-byte store, 32 bytes a
// row.
__device__ __forceinline__ void put8(bf16* row, int hh, f32x4 a, f32x4 b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  auto pair = [](float x, float y) __attribute__((always_inline)) { return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{x, y}), bf16x2)); };
  const auto p = __builtin_amdgcn_permlane32_swap(pair(a[0], a[1]), pair(b[0], b[1]), false, false);
  const auto q = __builtin_amdgcn_permlane32_swap(pair(a[2], a[3]), pair(b[2], b[3]), false, false);
  *reinterpret_cast<u32x4*>(row + 8 * hh) = u32x4{p[0], q[0], p[1], q[1]};
}
}  // namespace ssmi
