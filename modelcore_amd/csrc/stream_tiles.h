// Tiles of 32 keys of a paged bf16 cache in LDS, and the matrix cores' operands out of them: what the streaming
// kernels of few pairs (paged_stream.hip) and of trees (tree_stream.hip) share. Layouts: paged_stream.hip.
#pragma once

#include "paged_stream.h"

namespace mcamd {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <int DP>
struct Shape {
  static constexpr int CPR = DP / 8;     // 16-byte chunks of an LDS row
  static constexpr int RPI = 64 / CPR;   // rows of a load
  static constexpr int NI = KT / RPI;    // loads of a tile
  static constexpr int NV = 16 / RPI;    // of 16 keys
  static constexpr int KD = DP / 16, MD = DP / 32;
  static constexpr int TILE = KT * DP;   // elements
  // Chunk c of row r is stored at slot c ^ k_swz(r) (K), c ^ v_swz(r) (V).
  static __device__ __forceinline__ constexpr int k_swz(int r) {
    return CPR >= 16 ? r & 15 : CPR == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  }
  static __device__ __forceinline__ constexpr int v_swz(int r) {
    return CPR >= 16 ? 4 * (r & 3) + ((r >> 2) & 3) : CPR == 8 ? 4 * ((r >> 1) & 1) : 0;
  }
};

__device__ __forceinline__ uint32_t lds_addr(const void *p) {
  return uint32_t(uintptr_t((const __attribute__((address_space(3))) void *)(p)));
}

// N LDS reads and the wait for them, as one piece: the compiler would wait for the loads to LDS under way
// before any read of its own.
template <int N>
__device__ __forceinline__ void read_rows(bf16x8 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b128 %0, %8\n ds_read_b128 %1, %9\n ds_read_b128 %2, %10\n ds_read_b128 %3, %11\n"
        "ds_read_b128 %4, %12\n ds_read_b128 %5, %13\n ds_read_b128 %6, %14\n ds_read_b128 %7, %15\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b128 %0, %4\n ds_read_b128 %1, %5\n ds_read_b128 %2, %6\n ds_read_b128 %3, %7\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
        : "memory");
  else
    asm volatile("ds_read_b128 %0, %2\n ds_read_b128 %1, %3\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void read_columns(bf16x4 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n ds_read_b64_tr_b16 %1, %9\n ds_read_b64_tr_b16 %2, %10\n"
        "ds_read_b64_tr_b16 %3, %11\n ds_read_b64_tr_b16 %4, %12\n ds_read_b64_tr_b16 %5, %13\n"
        "ds_read_b64_tr_b16 %6, %14\n ds_read_b64_tr_b16 %7, %15\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n ds_read_b64_tr_b16 %1, %5\n ds_read_b64_tr_b16 %2, %6\n"
        "ds_read_b64_tr_b16 %3, %7\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
        : "memory");
  else
    asm volatile("ds_read_b64_tr_b16 %0, %2\n ds_read_b64_tr_b16 %1, %3\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1])
                 : "memory");
}

// The same from an offset on, bytes that an instruction holds (below 65536).
template <int OFF, int N>
__device__ __forceinline__ void read_rows_at(bf16x8 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  static_assert(OFF < 65536, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b128 %0, %8 offset:%16\n ds_read_b128 %1, %9 offset:%16\n ds_read_b128 %2, %10 offset:%16\n"
        "ds_read_b128 %3, %11 offset:%16\n ds_read_b128 %4, %12 offset:%16\n ds_read_b128 %5, %13 offset:%16\n"
        "ds_read_b128 %6, %14 offset:%16\n ds_read_b128 %7, %15 offset:%16\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "i"(OFF)
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b128 %0, %4 offset:%8\n ds_read_b128 %1, %5 offset:%8\n ds_read_b128 %2, %6 offset:%8\n"
        "ds_read_b128 %3, %7 offset:%8\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF)
        : "memory");
  else
    asm volatile("ds_read_b128 %0, %2 offset:%4\n ds_read_b128 %1, %3 offset:%4\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1]), "i"(OFF)
                 : "memory");
}
// Four rows (or two) from each of two offsets on.
template <int OFF, int OFF2, int N>
__device__ __forceinline__ void read_rows_two(bf16x8 (&f)[N], bf16x8 (&g)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4, "");
  static_assert(OFF2 < 65536, "");
  if constexpr (N == 4)
    asm volatile(
        "ds_read_b128 %0, %8 offset:%12\n ds_read_b128 %4, %8 offset:%13\n"
        "ds_read_b128 %1, %9 offset:%12\n ds_read_b128 %5, %9 offset:%13\n"
        "ds_read_b128 %2, %10 offset:%12\n ds_read_b128 %6, %10 offset:%13\n"
        "ds_read_b128 %3, %11 offset:%12\n ds_read_b128 %7, %11 offset:%13\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(g[0]), "=&v"(g[1]), "=&v"(g[2]), "=&v"(g[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF), "i"(OFF2)
        : "memory");
  else
    asm volatile(
        "ds_read_b128 %0, %4 offset:%6\n ds_read_b128 %2, %4 offset:%7\n"
        "ds_read_b128 %1, %5 offset:%6\n ds_read_b128 %3, %5 offset:%7\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(g[0]), "=&v"(g[1])
        : "v"(a[0]), "v"(a[1]), "i"(OFF), "i"(OFF2)
        : "memory");
}
template <int OFF, int N>
__device__ __forceinline__ void read_columns_at(bf16x4 (&f)[N], const uint32_t (&a)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  static_assert(OFF < 65536, "");
  if constexpr (N == 8)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%16\n ds_read_b64_tr_b16 %1, %9 offset:%16\n"
        "ds_read_b64_tr_b16 %2, %10 offset:%16\n ds_read_b64_tr_b16 %3, %11 offset:%16\n"
        "ds_read_b64_tr_b16 %4, %12 offset:%16\n ds_read_b64_tr_b16 %5, %13 offset:%16\n"
        "ds_read_b64_tr_b16 %6, %14 offset:%16\n ds_read_b64_tr_b16 %7, %15 offset:%16\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]),
          "=&v"(f[7])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "i"(OFF)
        : "memory");
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%8\n ds_read_b64_tr_b16 %1, %5 offset:%8\n"
        "ds_read_b64_tr_b16 %2, %6 offset:%8\n ds_read_b64_tr_b16 %3, %7 offset:%8\n s_waitcnt lgkmcnt(0)"
        : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(OFF)
        : "memory");
  else
    asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%4\n ds_read_b64_tr_b16 %1, %3 offset:%4\n s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0]), "=&v"(f[1])
                 : "v"(a[0]), "v"(a[1]), "i"(OFF)
                 : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "");
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

}  // namespace
}  // namespace mcamd
