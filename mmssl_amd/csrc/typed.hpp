// Element types of the operators that take fp32, bf16 and fp16 alike: 16-byte vectors of a row, read into and written from
// fp32 registers. A vector load wants no more than its elements' alignment (global dwordx4 accesses may start at any
// element on gfx950), so rows of odd width and odd pitch take the same path as aligned ones; only a row's last, partial
// vector goes element by element.
#pragma once
#include "common.hpp"

namespace mmssl {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T raw __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  typedef float f32 __attribute__((ext_vector_type(16 / sizeof(T))));
};

// `left` = elements of the row from p on; nothing at or behind p + left is touched, what is missing is 0. FULL: the caller
// knows that a row holds whole vectors only (the partial path costs registers even where it is never taken).
template <class T, bool FULL = false>
__device__ __forceinline__ typename Vec<T>::raw load_raw(const T* __restrict__ p, int left) {
  typename Vec<T>::raw v;
  if (FULL || left >= Vec<T>::N) {
    v = *reinterpret_cast<const typename Vec<T>::raw*>(p);
  } else {
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k) v[k] = k < left ? p[k] : (T)0.0f;
  }
  return v;
}

template <class T>
__device__ __forceinline__ typename Vec<T>::f32 to_f32(typename Vec<T>::raw v) {
  return __builtin_convertvector(v, typename Vec<T>::f32);
}

// one rounding, to nearest even
template <class T, bool FULL = false>
__device__ __forceinline__ void store_f32(T* __restrict__ p, int left, typename Vec<T>::f32 f) {
  const typename Vec<T>::raw v = __builtin_convertvector(f, typename Vec<T>::raw);
  if (FULL || left >= Vec<T>::N) {
    *reinterpret_cast<typename Vec<T>::raw*>(p) = v;
  } else {
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k)
      if (k < left) p[k] = v[k];
  }
}

// N fp32 values of a workspace row (4-byte aligned), N = 4 or 8
template <int N, class F, bool FULL = false>
__device__ __forceinline__ F load_part(const float* __restrict__ p, int left) {
  F f;
#pragma unroll
  for (int h = 0; h < N; h += 4) {
    const Vec<float>::raw q = load_raw<float, FULL>(p + h, left - h);
#pragma unroll
    for (int k = 0; k < 4; ++k) f[h + k] = q[k];
  }
  return f;
}
template <int N, bool FULL = false, class F>
__device__ __forceinline__ void store_part(float* __restrict__ p, int left, F f) {
#pragma unroll
  for (int h = 0; h < N; h += 4) {
    Vec<float>::f32 q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = f[h + k];
    store_f32<float, FULL>(p + h, left - h, q);
  }
}

inline bool known_dtype(int t) { return t == MMSSL_F32 || t == MMSSL_BF16 || t == MMSSL_F16; }
inline int dtype_bytes(int t) { return t == MMSSL_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// a launch counts its threads in 32 bits
inline bool launchable(int64_t blocks, int threads) { return blocks <= 0xffffffffLL / threads; }

// CALL(T) once, with the element type of code DT
#define MMSSL_BY_DTYPE(DT, CALL)        \
  do {                                  \
    if ((DT) == MMSSL_F32) {            \
      CALL(float);                      \
    } else if ((DT) == MMSSL_BF16) {    \
      CALL(bf16_t);                     \
    } else {                            \
      CALL(f16_t);                      \
    }                                   \
  } while (0)

}  // namespace mmssl
