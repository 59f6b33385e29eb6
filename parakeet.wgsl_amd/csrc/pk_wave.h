// pk_wave.h - reductions over a wavefront of 64 lanes with data-parallel
// primitives: each step is one VALU instruction that reads a neighbour's
// register (a shift within 16 lanes, then the broadcast of a row's last lane
// into the next), where a shuffle goes through the LDS crossbar. The result
// is lane 63's, read into a scalar register, so it is uniform, and the order
// of the sums is fixed. sync() orders what lanes exchange through LDS.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pk {
namespace wave {

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t identity, uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)identity, (int)x, CTRL, ROWS, 0xf, false);
}

// op over the 64 lanes of x; lanes without a neighbour see the identity.
template <typename Op>
__device__ __forceinline__ uint32_t reduce_bits(uint32_t x, uint32_t identity, Op op) {
  x = op(x, dpp<0x111, 0xf>(identity, x));  // row_shr:1
  x = op(x, dpp<0x112, 0xf>(identity, x));
  x = op(x, dpp<0x114, 0xf>(identity, x));
  x = op(x, dpp<0x118, 0xf>(identity, x));  // lane 15 of each row of 16 holds the row
  x = op(x, dpp<0x142, 0xa>(identity, x));  // row_bcast:15 into rows 1 and 3
  x = op(x, dpp<0x143, 0xc>(identity, x));  // row_bcast:31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

__device__ __forceinline__ float sum(float x) {
  return __uint_as_float(reduce_bits(__float_as_uint(x), 0u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// The largest lane, NaN left out; minus infinity if every lane is NaN.
__device__ __forceinline__ float max(float x) {
  return __uint_as_float(reduce_bits(__float_as_uint(x), 0xff800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}

// LDS that lanes of this wavefront wrote before is what its lanes read behind,
// and what they read before is not overwritten yet. The LDS takes a
// wavefront's accesses in their order, so this is an order for the compiler,
// which sees one lane's addresses, and no instruction.
__device__ __forceinline__ void sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace wave
}  // namespace pk
