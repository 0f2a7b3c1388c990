// What the attention kernels share: vector types, exchanges between the lanes
// that hold one query's keys, and the layout of key tiles in LDS.
#pragma once

#include "ltx_common.h"

namespace ltx {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr float kLog2e = 1.4426950408889634f;

// Max / sum of a lane's value with lane l ^ 32's (the lane holding the other
// 16 keys of the same query): one v_permlane32_swap, no LDS round trip.
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The same over the four lanes l ^ 16, l ^ 32, l ^ 48 (the pipelined kernels'
// layout: a query's keys lie in four lanes).
__device__ __forceinline__ float quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// The pipelined kernels' tile layout in LDS: rows of NC 16-byte chunks without
// padding, chunk c of row r stored at c ^ row_swizzle(r), so that the 16 rows
// that a fragment read touches (one chunk index each) fall on 16 different
// 16-byte bank groups.  K rows hold keys in the order key_of_row: LDS row bits
// (half, kbit, g1 g0, r1 r0) hold key bits (half, g1 g0, kbit, r1 r0), so that
// a lane's scores of two adjacent 16-key blocks are 8 consecutive keys.
template <int NC>
__host__ __device__ constexpr int row_swizzle(int r) { return NC == 16 ? (r & 15) : ((r >> 1) & 7); }
// chunk pairs of a token-major V tile's key rows: the 8 keys that half a
// transposing fragment read touches (two blocks of 4, 8 keys apart, one 32-byte
// chunk pair each) fall on 8 different 32-byte bank groups
template <int NC>
__host__ __device__ constexpr int key_swizzle(int r) {
  return NC == 16 ? 2 * ((r & 3) | ((r >> 1) & 4)) : 2 * (((r >> 1) & 1) | ((r >> 2) & 2));
}
__host__ __device__ constexpr int key_of_row(int r) { return (r & 35) | ((r & 12) << 1) | ((r & 16) >> 2); }

}  // namespace ltx
