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
// The passes move bytes and nothing else binds them: four lanes share a group, a lane owns eight channels (16 bytes of
// bfloat16 in, 8 bytes of codes out), the group's maximum is two cross-lane steps on the integer patterns of |x| (which order as
// the values do and put infinities and NaN on top).
#include "common.h"

namespace ssmi {

static constexpr int kGroup = 32;

// rows of 8 channels as they travel; VEC: the lane's channels are all there or all absent and 16-byte accesses are allowed
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  if constexpr (VEC) {
    const f32x4 a = Act<T>::gld4(p), b = Act<T>::gld4(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Act<T>::gld(p + i) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  if constexpr (VEC) {
    const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    if constexpr (sizeof(T) == 2) {
      const u32x2 x = pack_bf16x4(a), y = pack_bf16x4(b);
      *reinterpret_cast<u32x4*>(p) = u32x4{x[0], x[1], y[0], y[1]};
    } else {
      Act<T>::gst4(p, a);
      Act<T>::gst4(p + 4, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) Act<T>::gst(p + i, v[i]);
  }
}
template <bool VEC>
__device__ __forceinline__ u32x2 load_codes(const uint8_t* p, int n) {
  if constexpr (VEC) return *reinterpret_cast<const u32x2*>(p);
  u32x2 w = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) w[i >> 2] |= (unsigned)p[i] << (8 * (i & 3));
  return w;
}

// Where a block's work starts: 64 groups a step (four lanes each).  The pixel of the block's first group costs one uniform 64-bit
// division, the lane's own place in front of it a 32-bit one.
struct GroupAt {
  int64_t pix;
  int g;
};
__device__ __forceinline__ GroupAt group_at(int64_t first, unsigned lane_group, unsigned groups) {
  const int64_t p0 = first / groups;
  const unsigned t = (unsigned)(first - p0 * groups) + lane_group;
  const unsigned dp = t / groups;
  return {p0 + dp, (int)(t - dp * groups)};
}

static constexpr int kSteps = 4;      // groups per lane: independent loads in flight

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void act8_store_kernel(const T* __restrict__ x, int64_t ld, int64_t ngroups, int c, unsigned groups,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t first = (int64_t)blockIdx.x * (64 * kSteps);
  const unsigned lg = threadIdx.x >> 2, part = threadIdx.x & 3;
  float v[kSteps][8];
  int64_t pix[kSteps];
  int ch[kSteps], n[kSteps], gi[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const GroupAt at = group_at(first, lg + 64 * s, groups);
    pix[s] = at.pix;
    gi[s] = at.g;
    ch[s] = at.g * kGroup + (int)part * 8;
    n[s] = first + lg + 64 * s < ngroups ? min(8, c - ch[s]) : 0;      // <= 0: nothing here
#pragma unroll
    for (int i = 0; i < 8; ++i) v[s][i] = 0.f;
    if (n[s] > 0) load8<T, VEC>(x + pix[s] * ld + ch[s], n[s], v[s]);
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(unsigned, v[s][i]) & 0x7FFFFFFFu);
    top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
    top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
    const bool fine = top < 0x7F800000u;
    // 464 / 256 = 1.8125: a mantissa above it carries into the exponent
    const int e = max((int)((top + 0x17FFFFu) >> 23) - 8, 16);
    const float inv = __builtin_bit_cast(float, (unsigned)(254 - (fine ? e : 127)) << 23);
    u32x2 w = {0u, 0u};
    if (fine) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k] * inv, v[s][4 * k + 1] * inv, 0, false);
        w[k] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[s][4 * k + 2] * inv, v[s][4 * k + 3] * inv, q, true);
      }
    }
    if (n[s] > 0) {
      uint8_t* const d = codes + pix[s] * c + ch[s];
      if constexpr (VEC) {
        *reinterpret_cast<u32x2*>(d) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n[s]) d[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
      }
      if (part == 0) scales[pix[s] * groups + gi[s]] = (uint8_t)(fine ? e : 255);
    }
  }
}

struct RestoreBn {
  const float *mean, *invstd, *gamma, *beta, *alpha, *drop;
  int act;
  float slope;
  int64_t hw;
};

__device__ __forceinline__ void decode8(u32x2 w, unsigned byte, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float s = __builtin_bit_cast(float, byte == 255u ? 0x7FC00000u : byte << 23);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[k], true);
    v[4 * k] = a[0] * s;
    v[4 * k + 1] = a[1] * s;
    v[4 * k + 2] = b[0] * s;
    v[4 * k + 3] = b[1] * s;
  }
}

// BN: also the output of the BatchNormalization -> activation -> SpatialDropout behind the stored tensor, which the backward pass
// needs beside it (operand of the next weight gradient); y (nullable) the restored tensor itself
template <typename T, bool VEC, bool BN>
__global__ __launch_bounds__(256) void act8_restore_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t ngroups, int c,
                                                           unsigned groups, T* __restrict__ y, int64_t ld_y, RestoreBn bn, T* __restrict__ out,
                                                           int64_t ld_out) {
  const int64_t first = (int64_t)blockIdx.x * (64 * kSteps);
  const unsigned lg = threadIdx.x >> 2, part = threadIdx.x & 3;
  u32x2 w[kSteps];
  unsigned sc[kSteps];
  int64_t pix[kSteps];
  int ch[kSteps], n[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const GroupAt at = group_at(first, lg + 64 * s, groups);
    pix[s] = at.pix;
    ch[s] = at.g * kGroup + (int)part * 8;
    n[s] = first + lg + 64 * s < ngroups ? min(8, c - ch[s]) : 0;
    w[s] = u32x2{0u, 0u};
    sc[s] = 127;
    if (n[s] > 0) {
      w[s] = load_codes<VEC>(codes + pix[s] * c + ch[s], n[s]);
      sc[s] = scales[pix[s] * groups + at.g];
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (n[s] <= 0) continue;
    float v[8];
    decode8(w[s], sc[s], v);
    if (!BN || y) store8<T, VEC>(y + pix[s] * ld_y + ch[s], n[s], v);
    if constexpr (BN) {
      const float* const drop = bn.drop ? bn.drop + (pix[s] < (1ll << 32) && bn.hw < (1ll << 32) ? (int64_t)((unsigned)pix[s] / (unsigned)bn.hw) : pix[s] / bn.hw) * c
                                        : nullptr;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = VEC ? ch[s] + i : min(ch[s] + i, c - 1);
        const float z = bn.gamma[k] * ((v[i] - bn.mean[k]) * bn.invstd[k]) + bn.beta[k];      // the order of bn_act_fwd_kernel
        const float a = bn.act == SSMI_ACT_PRELU ? bn.alpha[k] : bn.slope;
        const float r = bn.act == SSMI_ACT_NONE || z > 0.f ? z : a * z;
        v[i] = drop ? r * drop[k] : r;
      }
      store8<T, VEC>(out + pix[s] * ld_out + ch[s], n[s], v);
    }
  }
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static ssmi_status check_sizes(const char* who, int64_t npix, int32_t c, int64_t* ngroups) {
  SSMI_REQUIRE(npix > 0 && c > 0 && c <= (1 << 20), SSMI_E_SHAPE, "%s: %lld pixels of %d channels", who, (long long)npix, c);
  const int64_t g = (c + kGroup - 1) / kGroup;
  // one launch holds fewer than 2^32 work-items, four to a group, kSteps groups each
  SSMI_REQUIRE(npix <= ((1ll << 32) - 256) / g, SSMI_E_UNSUPPORTED, "%s: %lld pixels of %d channels are too many for one launch", who, (long long)npix, c);
  *ngroups = npix * g;
  return SSMI_OK;
}
static inline dim3 blocks_for(int64_t ngroups) { return dim3((unsigned)ceil_div64(ngroups, 64 * kSteps)); }

}  // namespace ssmi

using namespace ssmi;

extern "C" {

ssmi_status ssmi_act8_store(const void* x, int64_t ld, int64_t npix, int32_t c, int32_t dtype, uint8_t* codes, uint8_t* scales, void* stream) {
  SSMI_REQUIRE(x && codes && scales, SSMI_E_INVALID_ARG, "act8_store: null pointer");
  SSMI_REQUIRE(ld >= c, SSMI_E_SHAPE, "act8_store: pixel stride %lld is less than %d channels", (long long)ld, c);
  int64_t ng;
  const ssmi_status st = check_sizes("act8_store", npix, c, &ng);
  if (st != SSMI_OK) return st;
  const unsigned groups = (unsigned)((c + kGroup - 1) / kGroup);
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld % 8 == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const T* xt = static_cast<const T*>(x);
    if (vec) hipLaunchKernelGGL((act8_store_kernel<T, true>), blocks_for(ng), dim3(256), 0, as_stream(stream), xt, ld, ng, c, groups, codes, scales);
    else hipLaunchKernelGGL((act8_store_kernel<T, false>), blocks_for(ng), dim3(256), 0, as_stream(stream), xt, ld, ng, c, groups, codes, scales);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

ssmi_status ssmi_act8_restore(const uint8_t* codes, const uint8_t* scales, int64_t npix, int32_t c, int32_t dtype, void* y, int64_t ld_y, void* stream) {
  SSMI_REQUIRE(codes && scales && y, SSMI_E_INVALID_ARG, "act8_restore: null pointer");
  SSMI_REQUIRE(ld_y >= c, SSMI_E_SHAPE, "act8_restore: pixel stride %lld is less than %d channels", (long long)ld_y, c);
  int64_t ng;
  const ssmi_status st = check_sizes("act8_restore", npix, c, &ng);
  if (st != SSMI_OK) return st;
  const unsigned groups = (unsigned)((c + kGroup - 1) / kGroup);
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld_y % 8 == 0 && aligned16(y) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    T* yt = static_cast<T*>(y);
    const RestoreBn none = {};
    if (vec) hipLaunchKernelGGL((act8_restore_kernel<T, true, false>), blocks_for(ng), dim3(256), 0, as_stream(stream), codes, scales, ng, c, groups, yt, ld_y, none, (T*)nullptr, (int64_t)0);
    else hipLaunchKernelGGL((act8_restore_kernel<T, false, false>), blocks_for(ng), dim3(256), 0, as_stream(stream), codes, scales, ng, c, groups, yt, ld_y, none, (T*)nullptr, (int64_t)0);
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
  int64_t ng;
  const ssmi_status st = check_sizes("act8_restore_bn_act", npix, c, &ng);
  if (st != SSMI_OK) return st;
  const unsigned groups = (unsigned)((c + kGroup - 1) / kGroup);
  const RestoreBn p = {bn->mean, bn->invstd, bn->gamma, bn->beta, alpha, drop, act, slope, hw};
  return dispatch_dtype(dtype, [&](auto tag) -> ssmi_status {
    using T = decltype(tag);
    const bool vec = c % 8 == 0 && ld_out % 8 == 0 && aligned16(out) && (!y || (ld_y % 8 == 0 && aligned16(y))) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    T *yt = static_cast<T*>(y), *ot = static_cast<T*>(out);
    if (vec) hipLaunchKernelGGL((act8_restore_kernel<T, true, true>), blocks_for(ng), dim3(256), 0, as_stream(stream), codes, scales, ng, c, groups, yt, ld_y, p, ot, ld_out);
    else hipLaunchKernelGGL((act8_restore_kernel<T, false, true>), blocks_for(ng), dim3(256), 0, as_stream(stream), codes, scales, ng, c, groups, yt, ld_y, p, ot, ld_out);
    SSMI_LAUNCH_CHECK();
    return SSMI_OK;
  });
}

}  // extern "C"
