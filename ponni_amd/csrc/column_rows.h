// Rows of a [rows, columns] array by lanes that hold a few consecutive columns
// each (norm.h, kernels_logp.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace ponni_hip {

// N consecutive elements of a row, as they are in memory; element j as a float.  (Kept packed: as an array of
// 16-bit elements the compiler gives each a register.)
template <class T, int N> struct Pack {
  typedef T Vector __attribute__((ext_vector_type(N)));
  typedef T Anywhere __attribute__((ext_vector_type(N), aligned(sizeof(T))));  // (gfx950 loads 16 bytes at any address)
  Vector v;
  __device__ float operator[](int j) const { return float(v[j]); }
  __device__ void set(int j, float x) { v[j] = T(x); }
  __device__ void put(int j, T x) { v[j] = x; }
  __device__ T raw(int j) const { return v[j]; }
  __device__ void fill(float x) {
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = T(x);
  }
  // `count` (1 .. N) elements; the rest are `rest`.
  __device__ void load(T const* p, int count, float rest) {
    if (count >= N) {
      v = *reinterpret_cast<Anywhere const*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) v[j] = j < count ? p[j] : T(rest);
    }
  }
  __device__ void store(T* p, int count) const {
    if (count >= N) {
      *reinterpret_cast<Anywhere*>(p) = v;
    } else {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (j < count) p[j] = v[j];
    }
  }
  // What was computed from it is not kept from before.
  __device__ void pin() { asm volatile("" : "+v"(v)); }
};
template <class T> struct Pack<T, 1> {
  T v;
  __device__ float operator[](int) const { return float(v); }
  __device__ void set(int, float x) { v = T(x); }
  __device__ void put(int, T x) { v = x; }
  __device__ T raw(int) const { return v; }
  __device__ void fill(float x) { v = T(x); }
  __device__ void load(T const* p, int, float) { v = *p; }
  __device__ void store(T* p, int) const { *p = v; }
  __device__ void pin() {}
};

}  // namespace ponni_hip
