// Rows of elements as floats, and the angles of rotary positions: shared by
// rotary.h and the cache's append (kv_append.h).
#pragma once

#include "common.h"
#include "../kargs.h"

using namespace bwpp;

namespace rotary_pos {

// N elements of T at any address aligned to T, as floats; load_once: past the caches.
template <class T, int N>
struct Vec;
template <int N>
struct Vec<float, N> {
  typedef float V __attribute__((ext_vector_type(N), aligned(4)));
  static __device__ __forceinline__ void load(const float *p, float (&o)[N]) {
    const V v = *reinterpret_cast<const V *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i];
  }
  static __device__ __forceinline__ void load_once(const float *p, float (&o)[N]) {
    const V v = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i];
  }
  static __device__ __forceinline__ void store(float *p, const float (&o)[N]) {
    V v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = o[i];
    *reinterpret_cast<V *>(p) = v;
  }
};
template <>
struct Vec<float, 1> {
  static __device__ __forceinline__ void load(const float *p, float (&o)[1]) { o[0] = *p; }
  static __device__ __forceinline__ void load_once(const float *p, float (&o)[1]) { o[0] = __builtin_nontemporal_load(p); }
  static __device__ __forceinline__ void store(float *p, const float (&o)[1]) { *p = o[0]; }
};
template <int N>
struct Vec<uint16_t, N> {
  typedef uint32_t V __attribute__((ext_vector_type(N / 2), aligned(2)));
  static __device__ __forceinline__ void load(const uint16_t *p, float (&o)[N]) {
    const V v = *reinterpret_cast<const V *>(p);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      o[2 * i] = __uint_as_float(v[i] << 16);
      o[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void load_once(const uint16_t *p, float (&o)[N]) {
    const V v = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      o[2 * i] = __uint_as_float(v[i] << 16);
      o[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(uint16_t *p, const float (&o)[N]) {
    V v;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = pack_bf16x2(o[2 * i], o[2 * i + 1]);
    *reinterpret_cast<V *>(p) = v;
  }
};
template <>
struct Vec<uint16_t, 2> {
  static __device__ __forceinline__ void load(const uint16_t *p, float (&o)[2]) {
    o[0] = bf16_bits_to_f32(p[0]);
    o[1] = bf16_bits_to_f32(p[1]);
  }
  static __device__ __forceinline__ void store(uint16_t *p, const float (&o)[2]) {
    p[0] = f32_to_bf16_bits(o[0]);
    p[1] = f32_to_bf16_bits(o[1]);
  }
};
template <>
struct Vec<uint16_t, 1> {
  static __device__ __forceinline__ void load(const uint16_t *p, float (&o)[1]) { o[0] = bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ void load_once(const uint16_t *p, float (&o)[1]) {
    o[0] = bf16_bits_to_f32(__builtin_nontemporal_load(p));
  }
  static __device__ __forceinline__ void store(uint16_t *p, const float (&o)[1]) { *p = f32_to_bf16_bits(o[0]); }
};

// N elements as they are, at any address aligned to T.
template <class T, int N>
__device__ __forceinline__ void copy_row(const T *src, T *dst) {
  if constexpr (N * sizeof(T) >= 8) {
    typedef uint32_t V __attribute__((ext_vector_type(N * sizeof(T) / 4), aligned(sizeof(T))));
    *reinterpret_cast<V *>(dst) = *reinterpret_cast<const V *>(src);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = src[i];
  }
}

// Frequency i in quarter turns per position.
__device__ __forceinline__ double quarter_turns(const BwppRotaryArgs &a, uint32_t i) {
  double f = exp2((double)i * a.log2_step);
  if (a.scaling == 1) f *= a.inv_factor;
  if (a.scaling == 2) {
    const double kept = fmin(fmax((a.turns * f - a.low) * a.inv_range, 0.0), 1.0);
    f *= kept + (1.0 - kept) * a.inv_factor;
  }
  return f * 0.63661977236758134308;  // 2 / pi
}

__device__ __forceinline__ float2 cos_sin(const BwppRotaryArgs &a, double u) {
  const double k = rint(u);
  const float z = (float)((u - k) * 1.57079632679489661923), w = z * z;
  const int q = (int)(int64_t)k & 3;
  // sin z and cos z for |z| <= pi / 4
  float s = fmaf(w, -2.50521083854417e-8f, 2.75573192239859e-6f);
  s = fmaf(w, s, -1.98412698412698e-4f);
  s = fmaf(w, s, 8.33333333333333e-3f);
  s = fmaf(w, s, -0.166666666666667f);
  s = fmaf(z * w, s, z);
  float c = fmaf(w, -2.75573192239859e-7f, 2.48015873015873e-5f);
  c = fmaf(w, c, -1.38888888888889e-3f);
  c = fmaf(w, c, 4.16666666666667e-2f);
  c = fmaf(w, c, -0.5f);
  c = fmaf(w, c, 1.0f);
  const float cs = q & 1 ? s : c, sn = q & 1 ? c : s;
  return make_float2((q == 1 || q == 2 ? -cs : cs) * a.cos_scale, (q >= 2 ? -sn : sn) * a.sin_scale);
}

}  // namespace rotary_pos
