// 8-bit activation checkpoints: a tensor that waits for the backward pass in half (bfloat16) or a quarter (float32) of its bytes.
//
// Every pixel's channels are taken in groups of 32 (the last one may be shorter).  A group keeps one power of two s and its
// values as e4m3 codes q (four significant bits, largest 448):
//   s = the smallest power of two >= 2^-111 under which max |x| rounds to at most 448, i.e. max |x| <= 464 s
//   q = round to nearest even (x / s)                restored value = q * s
// so a value is off by at most half a step, |x| 2^-4 or s 2^-10, whichever is larger, and the restored value is exact in
// bfloat16 and float32 (four significant bits times a power of two).  Scales under 2^-111 are not used: every intermediate
// stays a normal float32.  A group that holds an infinity or a NaN restores as NaN.
//
// The passes move bytes and nothing else binds them: a lane owns 16 bytes of a pixel (eight bfloat16 or four float32 channels, so that a
// wave's accesses are whole lines), four or eight lanes share a group, and the group's maximum is two or three cross-lane steps on the
// integer patterns of |x| (which order as the values do and put infinities and NaN on top).
// Measured: store + restore of 1M x 64 bfloat16 pixels 77 us, 5.3 TB/s of the 407 MB that they move (a large copy: 5.2 TB/s).
#include "common.h"

namespace ssmi {

static constexpr int kGroup = 32;

template <typename T> struct Piece {
  static constexpr int kCh = 16 / (int)sizeof(T), kLanes = kGroup / kCh, kAtOnce = 256 / kLanes;      // channels a lane, lanes a group, groups a block
};

// a lane's channels as they travel; VEC: all there or all absent, and 16-byte accesses are allowed
template <typename T, bool VEC, int N>
__device__ __forceinline__ void load_piece(const T* p, int n, float (&v)[N]) {
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
      const f32x4 a = Act<T>::gld4(p + q);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[q + i] = a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? Act<T>::gld(p + i) : 0.f;
  }
}
// PAST: past the caches
template <typename T, bool VEC, bool PAST, int N>
__device__ __forceinline__ void store_piece(T* p, int n, const float (&v)[N]) {
  if constexpr (VEC) {
    u32x4 w;
    if constexpr (sizeof(T) == 2) {
      const u32x2 x = pack_bf16x4(f32x4{v[0], v[1], v[2], v[3]}), y = pack_bf16x4(f32x4{v[4], v[5], v[6], v[7]});
      w = u32x4{x[0], x[1], y[0], y[1]};
    } else {
      w = __builtin_bit_cast(u32x4, (f32x4{v[0], v[1], v[2], v[3]}));
    }
    if constexpr (PAST) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
    else *reinterpret_cast<u32x4*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) Act<T>::gst(p + i, v[i]);
  }
}
// N codes, four to a word
template <bool VEC, int N>
__device__ __forceinline__ void load_codes(const uint8_t* p, int n, unsigned (&w)[N / 4]) {
  if constexpr (VEC && N == 8) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0];
    w[1] = v[1];
  } else if constexpr (VEC) {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  } else {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) w[k] = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) w[i >> 2] |= (unsigned)p[i] << (8 * (i & 3));
  }
}
template <bool VEC, int N>
__device__ __forceinline__ void store_codes(uint8_t* p, int n, const unsigned (&w)[N / 4]) {
  if constexpr (VEC && N == 8) {
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
  } else if constexpr (VEC) {
    *reinterpret_cast<unsigned*>(p) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// How a block's lane groups lie over the tensor: `gp` groups of a pixel side by side (all of them up to a block's worth, then
// blockIdx.y counts further), `ppb` pixels at a time.  A lane keeps its channels for the whole kernel, so the parameters of its
// BatchNormalization are loaded once, and walks pixels in steps of the grid.
struct Lane {
  int64_t pix, step;      // first pixel, pixels from one step to the next
  int g, ch, n;           // group, first channel, channels (<= 0: none)
  bool lead;              // the first lane of its group
};
template <typename T>
__device__ __forceinline__ int pixels_at_once(int groups) { return Piece<T>::kAtOnce / min(groups, Piece<T>::kAtOnce); }
template <typename T>
__device__ __forceinline__ Lane lane_of(int c, int groups) {
  typedef Piece<T> P;
  const int gp = min(groups, P::kAtOnce), ppb = P::kAtOnce / gp;
  const int lg = (int)threadIdx.x / P::kLanes, part = (int)threadIdx.x % P::kLanes;
  const int p = lg / gp;
  Lane l;
  l.g = lg - p * gp + P::kAtOnce * (int)blockIdx.y;
  l.pix = (int64_t)blockIdx.x * ppb + p;
  l.step = (int64_t)gridDim.x * ppb;
  l.ch = l.g * kGroup + part * P::kCh;
  l.n = p < ppb && l.g < groups ? min(P::kCh, c - l.ch) : 0;
  l.lead = part == 0;
  return l;
}

static constexpr int kSteps = 4;      // pixels per lane and round: independent loads in flight

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void act8_store_kernel(const T* __restrict__ x, int64_t ld, int64_t npix, int c, int groups,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  typedef Piece<T> P;
  constexpr int N = P::kCh;
  const Lane l = lane_of<T>(c, groups);
  // a block's lanes stay together (the maximum crosses lanes): rounds go by its first pixel
  for (int64_t base = (int64_t)blockIdx.x * pixels_at_once<T>(groups), pix = l.pix; base < npix; base += kSteps * l.step, pix += kSteps * l.step) {
    float v[kSteps][N];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[s][i] = 0.f;
      if (l.n > 0 && pix + s * l.step < npix) load_piece<T, VEC>(x + (pix + s * l.step) * ld + l.ch, l.n, v[s]);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) top = max(top, __builtin_bit_cast(unsigned, v[s][i]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = 1; o < P::kLanes; o <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
      const bool fine = top < 0x7F800000u;
      // 464 / 256 = 1.8125: a mantissa above it carries into the exponent
      const int e = max((int)((top + 0x17FFFFu) >> 23) - 8, 16);
      const float inv = __builtin_bit_cast(float, (unsigned)(254 - (fine ? e : 127)) << 23);
      unsigned w[N / 4];
#pragma unroll
      for (int k = 0; k < N / 4; ++k) {
        const int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k] * inv, v[s][4 * k + 1] * inv, 0, false);
        w[k] = fine ? (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k + 2] * inv, v[s][4 * k + 3] * inv, q, true) : 0u;
      }
      const int64_t px = pix + s * l.step;
      if (l.n > 0 && px < npix) {
        store_codes<VEC, N>(codes + px * c + l.ch, l.n, w);
        if (l.lead) scales[px * groups + l.g] = (uint8_t)(fine ? e : 255);
      }
    }
  }
}

struct RestoreBn {
  const float *mean, *invstd, *gamma, *beta, *alpha, *drop;
  int act;
  float slope;
  int64_t hw;
};

template <int N>
__device__ __forceinline__ void decode(const unsigned (&w)[N / 4], unsigned byte, float (&v)[N]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float s = __builtin_bit_cast(float, byte == 255u ? 0x7FC00000u : byte << 23);
#pragma unroll
  for (int k = 0; k < N / 4; ++k) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
    v[4 * k] = a[0] * s;
    v[4 * k + 1] = a[1] * s;
    v[4 * k + 2] = b[0] * s;
    v[4 * k + 3] = b[1] * s;
  }
}

// BN: also the output of the BatchNormalization -> activation -> SpatialDropout behind the stored tensor, which the backward pass
// needs beside it (operand of the next weight gradient); y (nullable) the restored tensor itself
template <typename T, bool VEC, bool BN, bool PAST>
__global__ __launch_bounds__(256) void act8_restore_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t npix, int c,
                                                           int groups, T* __restrict__ y, int64_t ld_y, RestoreBn bn, T* __restrict__ out,
                                                           int64_t ld_out) {
  constexpr int N = Piece<T>::kCh;
  const Lane l = lane_of<T>(c, groups);
  if (l.n <= 0) return;
  float mean[N], invstd[N], gamma[N], beta[N], slope[N];
  if constexpr (BN) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = min(l.ch + i, c - 1);
      mean[i] = bn.mean[k];
      invstd[i] = bn.invstd[k];
      gamma[i] = bn.gamma[k];
      beta[i] = bn.beta[k];
      slope[i] = bn.act == SSMI_ACT_PRELU ? bn.alpha[k] : bn.act == SSMI_ACT_LEAKY ? bn.slope : 1.f;
    }
  }
  for (int64_t pix = l.pix; pix < npix; pix += kSteps * l.step) {
    unsigned w[kSteps][N / 4], sc[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t px = min(pix + s * l.step, npix - 1);      // past the end: the last pixel again, not stored
      load_codes<VEC, N>(codes + px * c + l.ch, l.n, w[s]);
      sc[s] = scales[px * groups + l.g];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t px = pix + s * l.step;
      if (px >= npix) break;
      float v[N];
      decode<N>(w[s], sc[s], v);
      if (!BN || y) store_piece<T, VEC, PAST>(y + px * ld_y + l.ch, l.n, v);
      if constexpr (BN) {
        float drop[N];
#pragma unroll
        for (int i = 0; i < N; ++i) drop[i] = 1.f;
        if (bn.drop) {
          const int64_t img = npix <= 0xFFFFFFFFll ? (int64_t)((unsigned)px / (unsigned)bn.hw) : px / bn.hw;      // hw <= npix
          load_piece<float, VEC>(bn.drop + img * c + l.ch, l.n, drop);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float z = gamma[i] * ((v[i] - mean[i]) * invstd[i]) + beta[i];      // the order of bn_act_fwd_kernel
          const float r = z > 0.f ? z : slope[i] * z;
          v[i] = r * drop[i];
        }
        store_piece<T, VEC, PAST>(out + px * ld_out + l.ch, l.n, v);
      }
    }
  }
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static ssmi_status check_sizes(const char* who, int64_t npix, int32_t c) {
  SSMI_REQUIRE(npix > 0 && npix < (1ll << 48) && c > 0 && c <= (1 << 20), SSMI_E_SHAPE, "%s: %lld pixels of %d channels", who, (long long)npix, c);
  return SSMI_OK;
}
// sixteen rounds of four pixels a lane at the most (the parameters are loaded once per lane), but enough blocks to fill the card
template <typename T>
static inline dim3 blocks_for(int64_t npix, int groups) {
  constexpr int at_once = Piece<T>::kAtOnce;
  const int gp = groups < at_once ? groups : at_once, ny = (groups + at_once - 1) / at_once;
  const int64_t all = ceil_div64(npix, (int64_t)(at_once / gp) * kSteps);
  int64_t nx = ceil_div64(all, 16);
  const int64_t fill = ceil_div64(4096, ny);
  if (nx < fill) nx = all < fill ? all : fill;
  if (nx > (1 << 20)) nx = 1 << 20;
  return dim3((unsigned)nx, (unsigned)ny);
}

}  // namespace ssmi

using namespace ssmi;

extern "C" {

ssmi_status ssmi_act8_store(const void* x, int64_t ld, int64_t npix, int32_t c, int32_t dtype, uint8_t* codes, uint8_t* scales, void* stream) {
  SSMI_REQUIRE(x && codes && scales, SSMI_E_INVALID_ARG, "act8_store: null pointer");
  SSMI_REQUIRE(ld >= c, SSMI_E_SHAPE, "act8_store: pixel stride %lld is less than %d channels", (long long)ld, c);
  const ssmi_status st = check_sizes("act8_store", npix, c);
  if (st != SSMI_OK) return st;
  const int groups = (c + kGroup - 1) / kGroup;
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld % 8 == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const T* xt = static_cast<const T*>(x);
    if (vec) hipLaunchKernelGGL((act8_store_kernel<T, true>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), xt, ld, npix, c, groups, codes, scales);
    else hipLaunchKernelGGL((act8_store_kernel<T, false>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), xt, ld, npix, c, groups, codes, scales);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

ssmi_status ssmi_act8_restore(const uint8_t* codes, const uint8_t* scales, int64_t npix, int32_t c, int32_t dtype, void* y, int64_t ld_y, void* stream) {
  SSMI_REQUIRE(codes && scales && y, SSMI_E_INVALID_ARG, "act8_restore: null pointer");
  SSMI_REQUIRE(ld_y >= c, SSMI_E_SHAPE, "act8_restore: pixel stride %lld is less than %d channels", (long long)ld_y, c);
  const ssmi_status st = check_sizes("act8_restore", npix, c);
  if (st != SSMI_OK) return st;
  const int groups = (c + kGroup - 1) / kGroup;
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld_y % 8 == 0 && aligned16(y) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    T* yt = static_cast<T*>(y);
    const RestoreBn none = {};
    if (vec) hipLaunchKernelGGL((act8_restore_kernel<T, true, false, false>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), codes, scales, npix, c, groups, yt, ld_y, none, (T*)nullptr, (int64_t)0);
    else hipLaunchKernelGGL((act8_restore_kernel<T, false, false, false>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), codes, scales, npix, c, groups, yt, ld_y, none, (T*)nullptr, (int64_t)0);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

ssmi_status ssmi_act8_restore_bn_act(const uint8_t* codes, const uint8_t* scales, int64_t npix, int32_t c, int32_t dtype, const ssmi_bn_params* bn,
                                     int32_t act, const float* alpha, float slope, const float* drop, int64_t hw, void* y, int64_t ld_y, void* out,
                                     int64_t ld_out, void* stream) {
  SSMI_REQUIRE(codes && scales && bn && out, SSMI_E_INVALID_ARG, "act8_restore_bn_act: null pointer");
  SSMI_REQUIRE(bn->mean && bn->invstd && bn->gamma && bn->beta, SSMI_E_INVALID_ARG, "act8_restore_bn_act: null BatchNormalization parameter");
  SSMI_REQUIRE(act >= SSMI_ACT_NONE && act <= SSMI_ACT_LEAKY, SSMI_E_INVALID_ARG, "act8_restore_bn_act: unknown activation %d", act);
  SSMI_REQUIRE(act != SSMI_ACT_PRELU || alpha, SSMI_E_INVALID_ARG, "act8_restore_bn_act: PReLU needs its slopes");
  SSMI_REQUIRE(ld_out >= c && (!y || ld_y >= c), SSMI_E_SHAPE, "act8_restore_bn_act: a pixel stride is less than %d channels", c);
  SSMI_REQUIRE(!drop || (hw > 0 && npix % hw == 0), SSMI_E_SHAPE, "act8_restore_bn_act: %lld pixels are no whole images of %lld", (long long)npix, (long long)hw);
  const ssmi_status st = check_sizes("act8_restore_bn_act", npix, c);
  if (st != SSMI_OK) return st;
  const int groups = (c + kGroup - 1) / kGroup;
  const RestoreBn p = {bn->mean, bn->invstd, bn->gamma, bn->beta, alpha, drop, act, slope, hw};
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld_out % 8 == 0 && aligned16(out) && (!y || (ld_y % 8 == 0 && aligned16(y))) && (!drop || aligned16(drop)) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    // Two results of 256 MB and more together do not stay in the memory-side cache of that size; written past the caches they take 115 us
    // instead of 131 (1M x 64 float32), with a reader behind them 264 instead of 284.  Under it the reader is faster with them there (2 x 67 MB
    // 73 us, past the caches 75); one result of any size measures the same either way.
    const bool past = npix * c * (int64_t)sizeof(T) * (y ? 2 : 1) >= (256ll << 20);
    T *yt = static_cast<T*>(y), *ot = static_cast<T*>(out);
    if (vec && past) hipLaunchKernelGGL((act8_restore_kernel<T, true, true, true>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), codes, scales, npix, c, groups, yt, ld_y, p, ot, ld_out);
    else if (vec) hipLaunchKernelGGL((act8_restore_kernel<T, true, true, false>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), codes, scales, npix, c, groups, yt, ld_y, p, ot, ld_out);
    else hipLaunchKernelGGL((act8_restore_kernel<T, false, true, false>), blocks_for<T>(npix, groups), dim3(256), 0, as_stream(stream), codes, scales, npix, c, groups, yt, ld_y, p, ot, ld_out);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

}  // extern "C"
