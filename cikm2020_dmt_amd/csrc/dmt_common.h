// Shared device/host helpers for libdmt_hip.so (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdarg.h>

#include "../../include/dmt_hip.h"

typedef unsigned short bf16_t;  // raw bfloat16 bits

void dmt_set_error(const char* fmt, ...);
extern int g_dmt_route_trace;     // dmt_route_trace(1): every successful launch notes its route label (which kernel variant ran)
void dmt_route_note(const char* what);

#define DMT_CHECK_ARG(cond, ...)            \
  do {                                      \
    if (!(cond)) {                          \
      dmt_set_error(__VA_ARGS__);           \
      return DMT_ERR_ARG;                   \
    }                                       \
  } while (0)

#define DMT_CHECK_LAUNCH(what)                                                       \
  do {                                                                               \
    hipError_t e__ = hipGetLastError();                                              \
    if (e__ != hipSuccess) {                                                         \
      dmt_set_error("%s: launch failed: %s", what, hipGetErrorString(e__));          \
      return DMT_ERR_LAUNCH;                                                         \
    }                                                                                \
    if (g_dmt_route_trace) dmt_route_note(what);                                     \
  } while (0)

__device__ __forceinline__ float bf2f(bf16_t h) { return __uint_as_float(((uint32_t)h) << 16); }
__device__ __forceinline__ bf16_t f2bf(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (bf16_t)((u >> 16) | 0x40u);  // quiet NaN
  u += 0x7fffu + ((u >> 16) & 1u);                                           // round to nearest even
  return (bf16_t)(u >> 16);
}

// two floats -> packed pair of bf16 (round to nearest even): compiles to ONE v_cvt_pk_bf16_f32 that hipcc schedules itself
// (an inline-asm cvt feeding an MFMA / LDS store needs hand-placed wait states: wrong results were seen under register pressure)
typedef __bf16 dmt_bf16x2_t __attribute__((ext_vector_type(2)));
typedef float dmt_f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned dmt_pack_bf16(float lo, float hi) {
  const dmt_f32x2_t v = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, dmt_bf16x2_t));
}

template <typename T> __device__ __forceinline__ float ldf(const T* p);
template <> __device__ __forceinline__ float ldf<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float ldf<bf16_t>(const bf16_t* p) { return bf2f(*p); }
template <typename T> __device__ __forceinline__ void stf(T* p, float v);
template <> __device__ __forceinline__ void stf<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void stf<bf16_t>(bf16_t* p, float v) { *p = f2bf(v); }

// Wavefront-wide reductions on the VALU: four DPP steps (quad_perm [1,0,3,2], quad_perm [2,3,0,1], row_half_mirror, row_mirror) leave
// every lane with the result of its 16-lane row, four v_readlane combine the rows.  (__shfl_xor is a ds_bpermute_b32: six LDS
// instructions per reduction -- the LayerNorm kernels, two reductions per 640-byte row, were bound by the LDS pipe, not by memory.)
template <int CTRL> __device__ __forceinline__ float dmt_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float dmt_lane_f(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ float wave_sum(float v) {
  v += dmt_dpp<0xB1>(v);
  v += dmt_dpp<0x4E>(v);
  v += dmt_dpp<0x141>(v);
  v += dmt_dpp<0x140>(v);
  return (dmt_lane_f(v, 0) + dmt_lane_f(v, 16)) + (dmt_lane_f(v, 32) + dmt_lane_f(v, 48));
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dmt_dpp<0xB1>(v));
  v = fmaxf(v, dmt_dpp<0x4E>(v));
  v = fmaxf(v, dmt_dpp<0x141>(v));
  v = fmaxf(v, dmt_dpp<0x140>(v));
  return fmaxf(fmaxf(dmt_lane_f(v, 0), dmt_lane_f(v, 16)), fmaxf(dmt_lane_f(v, 32), dmt_lane_f(v, 48)));
}

// cap tanh(x / cap) of a score x = scale s, in log2 units (dmt_attn_var_*, dmt_kv_attn).  With 2^a = e^(2x / cap) and r = 1 / (1 + 2^a):
//   far:   cap (1 - 2 r), exact at both ends (the power runs to infinity or zero), r and the difference off by up to 3 2^-23 of the CAP, whatever
//          the score: any number of steps of a score far below it;
//   near:  x w(a^2) where |a| < 1 (x / cap = ln 2 / 2), w = tanh(u) / u with u = a ln 2 / 2 a polynomial of minimal relative error (2^-24.7), and
//          `far` elsewhere: under 2^-20 of the value, whatever the cap.
// bf16 operands with a cap of at most 64 take `far`: its 2^-15.4 of a score is an 85th of the rounding of the weights to bf16, and no more than
// what the fp32 sum of a score of that size is off by.  fp32 operands and larger caps take `near` (bf16, 256 histories of up to 200, 4 heads of 80,
// forward and backward: 235 us with a cap of 1000, 222 with one of 20).  The derivative 1 - tanh^2 is 4 r (1 - r) in both.
struct dmt_cap {
  float c1, ck, cap2;                  // scale log2e, 2 scale log2e / cap, cap log2e (scale and cap are at most 1e38: twice cap2 is finite)
  bool near;
  __host__ __device__ __forceinline__ dmt_cap(float scale, float cap, bool bf16)
      : c1(scale * 1.44269504088896340736f), ck(cap > 0.f ? fminf(2.f * 1.44269504088896340736f * scale / cap, 3e38f) : 0.f),
        cap2(cap * 1.44269504088896340736f), near(!bf16 || cap > 64.f) {}
  __device__ __forceinline__ float r(float s) const { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(ck * s)); }
  static __device__ __forceinline__ float derivative(float r) { return 4.f * r * (1.f - r); }
  // the capped score less `b`, from s and r(s)
  template <bool NEAR> __device__ __forceinline__ float less(float s, float r, float b) const {
    const float far = __builtin_fmaf(-2.f * cap2, r, cap2 - b);
    if (!NEAR) return far;
    const float a = ck * s, t = a * a;
    const float w = __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, -8.5321815e-05f, 1.9189704e-03f), -4.003699e-02f), 1.f);
    return t < 1.f ? __builtin_fmaf(c1 * s, w, -b) : far;
  }
  __device__ __forceinline__ float operator()(float s) const { return near ? less<true>(s, r(s), 0.f) : less<false>(s, r(s), 0.f); }
};

// counter-based dropout mask shared by every kernel (and restated in oracle/dmt_oracle.py:dropout_mask)
__device__ __forceinline__ uint32_t dmt_mix32(uint32_t h) {
  h ^= h >> 16; h *= 0x85EBCA6Bu; h ^= h >> 13; h *= 0xC2B2AE35u; h ^= h >> 16;
  return h;
}
__device__ __forceinline__ bool dmt_drop_keep(uint32_t seed, uint32_t idx, uint32_t thr24) { return (dmt_mix32(idx ^ seed) >> 8) < thr24; }

static inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }
