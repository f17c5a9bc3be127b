// Element types of the row operators (layer norm, token log probabilities):
// aligned packs of elements, their conversion to and from pairs of fp32, and
// the packed fp32 arithmetic of sm_100 (two operations an instruction, each
// rounded as the scalar one).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>

namespace b200 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two 16-bit elements in a word <-> two fp32.
template <typename T>
__device__ __forceinline__ float2 word_to_pair(uint32_t u);
template <>
__device__ __forceinline__ float2 word_to_pair<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 word_to_pair<__half>(uint32_t u) {
  __half2 h;
  memcpy(&h, &u, 4);
  return __half22float2(h);
}
template <typename T>
__device__ __forceinline__ uint32_t pair_to_word(float2 v);
template <>
__device__ __forceinline__ uint32_t pair_to_word<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}
template <>
__device__ __forceinline__ uint32_t pair_to_word<__half>(float2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}

// VEC elements moved together: a 16-byte access (two for eight floats), or one element.
template <typename T, int VEC>
struct alignas(VEC * 2 < 16 ? VEC * 2 : 16) Pack {
  static_assert(sizeof(T) == 2 && VEC % 2 == 0, "16-bit packs hold pairs");
  uint32_t u[VEC / 2];
  __device__ __forceinline__ float2 pair(int i) const { return word_to_pair<T>(u[i]); }
  __device__ __forceinline__ void set_pair(int i, float2 v) { u[i] = pair_to_word<T>(v); }
};
template <int VEC>
struct alignas(VEC * 4 < 16 ? VEC * 4 : 16) Pack<float, VEC> {
  float v[VEC];
  __device__ __forceinline__ float2 pair(int i) const { return make_float2(v[2 * i], v[2 * i + 1]); }
  __device__ __forceinline__ void set_pair(int i, float2 p) {
    v[2 * i] = p.x;
    v[2 * i + 1] = p.y;
  }
};
template <typename T>
struct Pack<T, 1> {
  T v;
};
template <>
struct alignas(4) Pack<float, 1> {
  float v;
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}

// Elements of T in one 16-byte access.
template <typename T>
constexpr int kVec16 = 16 / static_cast<int>(sizeof(T));

// The elements of NV packs as fp32 pairs, in order.
template <typename T, int VEC, int NV>
__device__ __forceinline__ void unpack(const Pack<T, VEC> (&p)[NV], float2 (&f)[VEC * NV / 2]) {
  static_assert(VEC * NV % 2 == 0, "an even number of elements");
  if constexpr (VEC == 1) {
#pragma unroll
    for (int j = 0; j < NV / 2; ++j) f[j] = make_float2(to_f32(p[2 * j].v), to_f32(p[2 * j + 1].v));
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) f[j * (VEC / 2) + i] = p[j].pair(i);
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void repack(const float2 (&f)[VEC * NV / 2], Pack<T, VEC> (&p)[NV]) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int j = 0; j < NV / 2; ++j) {
      p[2 * j].v = from_f32<T>(f[j].x);
      p[2 * j + 1].v = from_f32<T>(f[j].y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) p[j].set_pair(i, f[j * (VEC / 2) + i]);
  }
}

__device__ __forceinline__ float2 pair_of(float v) { return make_float2(v, v); }

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

}  // namespace b200
