// Element types of the recurrent-policy operators (layer_norm.hip, decay_attention.hip): fp32, fp16 and bf16 in memory, fp32 in
// registers, vectors of up to 16 bytes.  Narrowing is the hardware's round to nearest even.
#pragma once
#include "oige_common.hpp"

namespace oige {

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
struct alignas(sizeof(T)) Loose {  // a vector on any element's boundary: one access all the same
  T v[N];
};

template <typename T>
constexpr int VEC16 = 16 / (int)sizeof(T);  // elements of a 16-byte access

inline int elem_bytes(int dtype) { return dtype == OIGE_F32 ? 4 : (dtype == OIGE_F16 || dtype == OIGE_BF16 ? 2 : 0); }

// One element into a buffer whose type is a launch constant (parameters of another type than the activations).
__device__ __forceinline__ void store_elem(void* p, int64_t i, float x, int dtype) {
  if (dtype == OIGE_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == OIGE_F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<__bf16*>(p)[i] = (__bf16)x;
}

// How a row's elements are reached.  ELEMS_FULL: 16-byte accesses and every lane's piece lies inside the row.  ELEMS_WIDE: 16-byte
// accesses (the row starts on a boundary, its length is a multiple of the access width), pieces behind its end are left out.
// ELEMS_SINGLE: element by element.  ELEMS_LOOSE: accesses as wide, on any element's boundary; a run of CNT elements across the row's
// end is moved forward to end with the row (which is CNT long at least), so lanes near the end hold some elements twice.
constexpr int ELEMS_FULL = 0, ELEMS_WIDE = 1, ELEMS_SINGLE = 2, ELEMS_LOOSE = 3;
template <int CNT, int MODE>
__device__ __forceinline__ int run_start(int off, int limit) {
  return MODE == ELEMS_LOOSE && off + CNT > limit ? limit - CNT : off;
}

// All bits where `in`, none elsewhere, as a value the compiler knows nothing about: an AND with it stays one instruction, where a
// select between a loaded value and zero has become a branch around the load.
__device__ __forceinline__ uint32_t bits_if(bool in) {
  uint32_t m = in ? 0xFFFFFFFFu : 0u;
  asm("" : "+v"(m));
  return m;
}
__device__ __forceinline__ float and_bits(float x, uint32_t m) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & m); }

// CNT consecutive elements from `off` of a row of `limit`, as floats; elements behind the limit read as 0 (ELEMS_LOOSE: from
// run_start on).  A piece behind the end re-reads the row's first one (no load inside a conditional block).
template <typename T, int CNT, int MODE>
__device__ __forceinline__ void load_run(float (&out)[CNT], const T* row, int off, int limit) {
  constexpr int W = MODE == ELEMS_SINGLE ? 1 : (CNT < VEC16<T> ? CNT : VEC16<T>);
#pragma unroll
  for (int b = 0; b < CNT; b += W) {
    if (MODE == ELEMS_LOOSE) {
      const Loose<T, W> x = *reinterpret_cast<const Loose<T, W>*>(row + run_start<CNT, MODE>(off, limit) + b);
#pragma unroll
      for (int e = 0; e < W; ++e) out[b + e] = (float)x.v[e];
      continue;
    }
    const bool ok = MODE == ELEMS_FULL || off + b < limit;
    const Pack<T, W> x = *reinterpret_cast<const Pack<T, W>*>(row + (ok ? off + b : 0));
    const uint32_t in = MODE == ELEMS_FULL ? 0u : bits_if(ok);
#pragma unroll
    for (int e = 0; e < W; ++e) out[b + e] = MODE == ELEMS_FULL ? (float)x.v[e] : and_bits((float)x.v[e], in);
  }
}

// The same in two halves, the second where the values are needed: until then they stay as they are in memory, in flight.
template <typename T, int CNT, int MODE>
struct Run {
  static constexpr int W = MODE == ELEMS_SINGLE ? 1 : (CNT < VEC16<T> ? CNT : VEC16<T>);
  Pack<T, W> x[CNT / W];
  __device__ __forceinline__ void issue(const T* row, int off, int limit) {
#pragma unroll
    for (int b = 0; b < CNT / W; ++b) {
      if (MODE == ELEMS_LOOSE) x[b] = __builtin_bit_cast(Pack<T, W>, *reinterpret_cast<const Loose<T, W>*>(row + run_start<CNT, MODE>(off, limit) + b * W));
      else x[b] = *reinterpret_cast<const Pack<T, W>*>(row + (MODE == ELEMS_FULL || off + b * W < limit ? off + b * W : 0));
    }
  }
  // Nothing was asked for: the registers hold no value (without this the last one would be kept for a round that does not come).
  __device__ __forceinline__ void forget() {
    constexpr int BYTES = W * (int)sizeof(T);
    typedef uint32_t words __attribute__((ext_vector_type(BYTES < 8 ? 2 : BYTES / 4)));
#pragma unroll
    for (int b = 0; b < CNT / W; ++b) {
      if constexpr (BYTES >= 8) {
        words w;
        asm volatile("" : "=v"(w));
        x[b] = __builtin_bit_cast(Pack<T, W>, w);
      } else if constexpr (BYTES == 4) {
        uint32_t w;
        asm volatile("" : "=v"(w));
        x[b] = __builtin_bit_cast(Pack<T, W>, w);
      } else {
        uint16_t w;
        asm volatile("" : "=v"(w));
        x[b] = __builtin_bit_cast(Pack<T, W>, w);
      }
    }
  }
  __device__ __forceinline__ void take(float (&out)[CNT], int off, int limit) const {
#pragma unroll
    for (int b = 0; b < CNT / W; ++b) {
      constexpr bool WHOLE = MODE == ELEMS_FULL || MODE == ELEMS_LOOSE;
      const uint32_t in = WHOLE ? 0u : bits_if(off + b * W < limit);
#pragma unroll
      for (int e = 0; e < W; ++e) out[b * W + e] = WHOLE ? (float)x[b].v[e] : and_bits((float)x[b].v[e], in);
    }
  }
};

template <typename T, int CNT, int MODE>
__device__ __forceinline__ void store_run(const float (&in)[CNT], T* row, int off, int limit) {
  constexpr int W = MODE == ELEMS_SINGLE ? 1 : (CNT < VEC16<T> ? CNT : VEC16<T>);
#pragma unroll
  for (int b = 0; b < CNT; b += W) {
    if (MODE == ELEMS_FULL || (MODE == ELEMS_LOOSE ? off : off + b) < limit) {
      Pack<T, W> x;
#pragma unroll
      for (int e = 0; e < W; ++e) x.v[e] = (T)in[b + e];
      if (MODE == ELEMS_LOOSE) *reinterpret_cast<Loose<T, W>*>(row + run_start<CNT, MODE>(off, limit) + b) = __builtin_bit_cast(Loose<T, W>, x);
      else *reinterpret_cast<Pack<T, W>*>(row + off + b) = x;
    }
  }
}

}  // namespace oige
