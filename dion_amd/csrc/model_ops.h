// Device helpers shared by the operators of the model around the optimizer step: embedding.hip, qk_norm.hip, cross_entropy.hip.
#pragma once
#include "common.h"

constexpr int DA_WAVE = 64;

// Token ids, targets and positions come as 32- or 64-bit integers.
struct DaIndex {
  const void* p;
  int wide;   // 1: int64
};
__device__ __forceinline__ long long da_index(const DaIndex& x, long long i) {
  return x.wide ? static_cast<const long long*>(x.p)[i] : (long long)static_cast<const int*>(x.p)[i];
}

// Several of them: all requested before the first is used.
template <int N>
__device__ __forceinline__ void da_indices(const DaIndex& x, const long long (&at)[N], long long (&v)[N]) {
  if (x.wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<const long long*>(x.p)[at[i]];
  } else {
    int w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = static_cast<const int*>(x.p)[at[i]];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = w[i];
  }
}

// Division of any 32-bit number by one known on the host, in three instructions or four in place of some 25: a multiplication and a shift
// (Granlund and Montgomery, Division by invariant integers using multiplication, 1994).
struct DaDivisor {
  unsigned mul, shift, by;
  __device__ __forceinline__ unsigned quotient(unsigned n) const {
    return (unsigned)(((unsigned long long)__umulhi(n, mul) + n) >> shift);
  }
};
__host__ inline DaDivisor da_divisor(unsigned by) {
  DaDivisor d{0, 0, by};
  while ((1ull << d.shift) < by) ++d.shift;
  d.mul = (unsigned)(((1ull << 32) * ((1ull << d.shift) - by)) / by + 1);
  return d;
}

// Sum and maximum over groups of 2^log2_group neighbouring lanes, in every lane: inside 16 lanes by moves within the vector unit.
template <typename F>
__device__ __forceinline__ float da_group_reduce(float v, int log2_group, F&& join) {
#define DA_DPP(ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))
  if (log2_group > 0) v = join(v, DA_DPP(0xb1));    // lane ^ 1
  if (log2_group > 1) v = join(v, DA_DPP(0x4e));    // lane ^ 2
  if (log2_group > 2) v = join(v, DA_DPP(0x141));   // mirrored inside 8 lanes: the other four
  if (log2_group > 3) v = join(v, DA_DPP(0x140));   // mirrored inside 16 lanes: the other eight
#undef DA_DPP
  if (log2_group > 4) v = join(v, __shfl_xor(v, 16));
  if (log2_group > 5) v = join(v, __shfl_xor(v, 32));
  return v;
}
__device__ __forceinline__ float da_group_sum(float v, int log2_group = 6) {
  return da_group_reduce(v, log2_group, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float da_group_max(float v, int log2_group = 6) {
  return da_group_reduce(v, log2_group, [](float a, float b) { return fmaxf(a, b); });
}

__host__ inline size_t da_esize(int dtype) { return dtype == DA_BF16 ? 2 : 4; }
// Lanes of a row of dim elements, cols to a lane (dim up to 2^31 - 1).
__host__ inline int da_lanes(int dim, int cols) { return dim / cols + (dim % cols != 0); }
__host__ inline bool da_float_dtype(int dtype) { return dtype == DA_BF16 || dtype == DA_F32; }
__host__ inline bool da_aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// N elements of a row, kept as they lie in memory.  Addresses are aligned to the elements only: the hardware takes 16-byte accesses
// at any address, so that rows of odd width move in vectors too.
template <typename T, int N> struct DaVec;
template <int N> struct DaVec<bf16_t, N> {
  typedef unsigned raw_t __attribute__((ext_vector_type(N / 2), aligned(2)));
  raw_t raw;
  __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = __builtin_bit_cast(float, raw[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, raw[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) raw[i] = (unsigned)f2bf(v[2 * i]) | ((unsigned)f2bf(v[2 * i + 1]) << 16);
  }
};
template <int N> struct DaVec<float, N> {
  typedef float raw_t __attribute__((ext_vector_type(N), aligned(4)));
  raw_t raw;
  __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = raw[i];
  }
  __device__ __forceinline__ void set(const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = v[i];
  }
};
// A row of n >= N elements as vectors of N: lane i takes those from min(i N, n - N) on, so that every vector lies inside the row and
// none is a special case to load (a branch around each load would keep the next one waiting).  The last lane shares its first
// `skip` elements with the lane before: where both hold the same bits both store them, else the lane before does.
template <int N>
__device__ __forceinline__ int da_column(int lane, int n, int& skip) {
  const int c = lane * N < n - N ? lane * N : n - N;
  skip = lane * N - c;
  return c;
}
template <bool STREAM = false, typename T, int N>
__device__ __forceinline__ void da_load(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = ld_as_float(p);
  } else {
    const auto* src = reinterpret_cast<const typename DaVec<T, N>::raw_t*>(p);
    DaVec<T, N> w;
    if constexpr (STREAM) w.raw = __builtin_nontemporal_load(src);
    else w.raw = *src;
    w.get(v);
  }
}
template <bool STREAM = false, typename T, int N>
__device__ __forceinline__ void da_store(T* p, int skip, const float (&v)[N]) {
  if constexpr (N == 1) {
    st_from_float(p, v[0]);
  } else if (skip == 0) {
    DaVec<T, N> w;
    w.set(v);
    auto* dst = reinterpret_cast<typename DaVec<T, N>::raw_t*>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(w.raw, dst);
    else *dst = w.raw;
  } else {
#pragma unroll
    for (int i = 1; i < N; ++i)
      if (i >= skip) st_from_float(p + i, v[i]);
  }
}
