// Vectors of channels for the convolution kernels: loads and stores of V elements, and packed float32 arithmetic on them.
#pragma once
#include <initializer_list>
#include "common.cuh"

namespace mb200 {
namespace {

constexpr int kConvK = 4;

template <typename T, int V> struct alignas(sizeof(T) * V) CVec {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ CVec<T, V> cload(const T* p, bool ok) {
  CVec<T, V> r;
  if (!ok) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = Elem<T>::from_f(0.f);
  } else if constexpr (sizeof(T) * V == 16) {
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  } else if constexpr (sizeof(T) * V == 8) {
    *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = __ldg(p + i);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void cstore(T* p, const CVec<T, V>& r) {
  if constexpr (sizeof(T) * V == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else if constexpr (sizeof(T) * V == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(&r);
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = r.v[i];
  }
}

// W channels of float arithmetic in one value: W = 2 uses the packed f32x2 instructions (one issue
// slot for two channels; these kernels would otherwise be bound by instruction issue, not by HBM).
template <int W> struct Pk;
template <> struct Pk<1> {
  float v;
  __device__ __forceinline__ static Pk splat(float a) { return {a}; }
  __device__ __forceinline__ static Pk load(const float* p, int stride) { return {p[0]}; }
  __device__ __forceinline__ float sum() const { return v; }
};
template <> struct Pk<2> {
  float2 v;
  __device__ __forceinline__ static Pk splat(float a) { return {make_float2(a, a)}; }
  __device__ __forceinline__ static Pk load(const float* p, int stride) { return {make_float2(p[0], p[stride])}; }
};
__device__ __forceinline__ Pk<1> pfma(Pk<1> a, Pk<1> b, Pk<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Pk<1> pmul(Pk<1> a, Pk<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Pk<1> padd(Pk<1> a, Pk<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Pk<1> psigmoid(Pk<1> a) { return {sigmoid_fast(a.v)}; }
__device__ __forceinline__ Pk<2> pfma(Pk<2> a, Pk<2> b, Pk<2> c) { return {__ffma2_rn(a.v, b.v, c.v)}; }
__device__ __forceinline__ Pk<2> pmul(Pk<2> a, Pk<2> b) { return {__fmul2_rn(a.v, b.v)}; }
__device__ __forceinline__ Pk<2> padd(Pk<2> a, Pk<2> b) { return {__fadd2_rn(a.v, b.v)}; }
__device__ __forceinline__ Pk<2> psigmoid(Pk<2> a) {
  const float2 m = __fmul2_rn(a.v, make_float2(-kLog2e, -kLog2e));
  const float2 d = __fadd2_rn(make_float2(ex2f(m.x), ex2f(m.y)), make_float2(1.f, 1.f));
  return {make_float2(rcpf(d.x), rcpf(d.y))};
}
// V raw elements <-> V/W packs
template <typename T, int V, int W>
__device__ __forceinline__ void unpack(const CVec<T, V>& r, Pk<W> (&o)[V / W]) {
#pragma unroll
  for (int i = 0; i < V / W; ++i) {
    if constexpr (W == 1) o[i].v = Elem<T>::to_f(r.v[i]);
    else o[i].v = pair_f(&r.v[2 * i]);
  }
}
template <typename T, int V, int W>
__device__ __forceinline__ CVec<T, V> pack(const Pk<W> (&o)[V / W]) {
  CVec<T, V> r;
#pragma unroll
  for (int i = 0; i < V / W; ++i) {
    if constexpr (W == 1) r.v[i] = Elem<T>::from_f(o[i].v);
    else if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<__nv_bfloat162*>(&r.v[2 * i]) = __floats2bfloat162_rn(o[i].v.x, o[i].v.y);
    } else { r.v[2 * i] = o[i].v.x; r.v[2 * i + 1] = o[i].v.y; }
  }
  return r;
}

inline bool conv_vec_ok(int64_t ED, int kv, std::initializer_list<const void*> ptrs,
                        std::initializer_list<int64_t> strides) {
  if (ED % kv) return false;
  for (const void* p : ptrs) if (!aligned16(p)) return false;
  for (int64_t s : strides) if (s % kv) return false;
  return true;
}

}  // namespace
}  // namespace mb200
