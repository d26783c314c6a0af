// A thread's V neighbouring columns in fp32 registers.
#pragma once

#include "nsb_common.cuh"

namespace nsb {

constexpr float kLog2e = 1.4426950408889634f;

// Arithmetic on a thread's V columns, two per instruction where V allows (same roundings).
#define NSB_PAIR(x, i) (*reinterpret_cast<unsigned long long*>(&(x)[i]))
#define NSB_CPAIR(x, i) (*reinterpret_cast<const unsigned long long*>(&(x)[i]))
template <int V>
struct alignas(V >= 2 ? 8 : 4) Cols {
  float v[V];
  __device__ __forceinline__ float& operator[](int i) { return v[i]; }
  __device__ __forceinline__ const float& operator[](int i) const { return v[i]; }
};
template <int V>
__device__ __forceinline__ Cols<V> all(float c) {
  Cols<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = c;
  return r;
}
template <int V>
__device__ __forceinline__ Cols<V> fma(const Cols<V>& a, const Cols<V>& b, const Cols<V>& c) {
  Cols<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(NSB_PAIR(r.v, i))
          : "l"(NSB_CPAIR(a.v, i)), "l"(NSB_CPAIR(b.v, i)), "l"(NSB_CPAIR(c.v, i)));
  } else {
    r[0] = fmaf(a[0], b[0], c[0]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Cols<V> mul(const Cols<V>& a, const Cols<V>& b) {
  Cols<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(NSB_PAIR(r.v, i)) : "l"(NSB_CPAIR(a.v, i)), "l"(NSB_CPAIR(b.v, i)));
  } else {
    r[0] = __fmul_rn(a[0], b[0]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Cols<V> add(const Cols<V>& a, const Cols<V>& b) {
  Cols<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      asm("add.rn.f32x2 %0, %1, %2;" : "=l"(NSB_PAIR(r.v, i)) : "l"(NSB_CPAIR(a.v, i)), "l"(NSB_CPAIR(b.v, i)));
  } else {
    r[0] = __fadd_rn(a[0], b[0]);
  }
  return r;
}

// Widening and rounding of V elements, two 16-bit ones per register at a time (one by one they cost the shifts and
// permutes that take them out of their register and put them back).
template <typename T, int V>
__device__ __forceinline__ Cols<V> widen(const Vec<T, V>& v) {
  Cols<V> o;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (Elem<T>::kDtype == NSB_BF16) {
        o[i] = __uint_as_float(w[i / 2] << 16);
        o[i + 1] = __uint_as_float(w[i / 2] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
        o[i] = f.x, o[i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = Elem<T>::to_f32(v.v[i]);
  }
  return o;
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const Cols<V>& c) {
  Vec<T, V> o;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (Elem<T>::kDtype == NSB_BF16)
        *reinterpret_cast<__nv_bfloat162*>(&o.v[i]) = __floats2bfloat162_rn(c[i], c[i + 1]);
      else
        *reinterpret_cast<__half2*>(&o.v[i]) = __floats2half2_rn(c[i], c[i + 1]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) o.v[v] = Elem<T>::from_f32(c[v]);
  }
  return o;
}

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_if(bool on, const T* p) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = Elem<T>::zero();
  if (on) v = *reinterpret_cast<const Vec<T, V>*>(p);
  return v;
}

__device__ __forceinline__ float ex2(float q) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(q));
  return e;
}
__device__ __forceinline__ float rcp(float q) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(q));
  return r;
}

}  // namespace nsb
