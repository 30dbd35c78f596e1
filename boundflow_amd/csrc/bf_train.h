// Shared device helpers of the training operators (bf_train_*.hip): element types and their
// vector loads, token reads, workgroup reductions.
#pragma once

#include "bf_common.h"

#include <cstring>

namespace bf {

// Element type codes of the training entry points.
enum : int { TE_F32 = 0, TE_BF16 = 1, TE_F16 = 2 };

inline bool elem_ok(int code) { return code >= TE_F32 && code <= TE_F16; }
inline int elem_bytes(int code) { return code == TE_F32 ? 4 : 2; }

// Calls f(T()) with the element type of a code that elem_ok has passed.
template <class F>
inline int with_elem(int code, F f) {
  switch (code) {
    case TE_F32: return f(float());
    case TE_BF16: return f(__bf16());
    default: return f(_Float16());
  }
}

// N elements at any alignment of T, as fp32.  The copy is one access of up to 16 bytes (gfx950
// reads and writes global memory at any alignment), so a row of odd length or a view that
// starts anywhere takes the same path as an aligned one.
template <class T, int N>
struct Pack {
  T v[N];
};

template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <class T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// Sixteen bytes as they are.
typedef uint32_t Words __attribute__((ext_vector_type(4)));

// Zeros that the compiler does not know for constants: known ones it stores element by element where the
// address may be unaligned (eight 2-byte stores for one of 16 bytes).
__device__ __forceinline__ Words zero_words() {
  uint32_t z = 0;
  asm volatile("" : "+v"(z));
  return Words{z, z, z, z};
}

// Element `i` of a token array of 4- or 8-byte integers; a value that no vocabulary of fewer
// than 2^31 entries holds becomes the nearest 32-bit one, so its sign and its being too large stay.
__device__ __forceinline__ int load_token(const void* tokens, int bytes, int64_t i) {
  if (bytes == 4) return static_cast<const int*>(tokens)[i];
  const int64_t t = static_cast<const int64_t*>(tokens)[i];
  return t > 0x7fffffffLL ? 0x7fffffff : t < -0x7fffffffLL ? -0x7fffffff : (int)t;
}

// Max over the 64 lanes of a wave by the DPP steps of wave_sum (a lane that a step leaves unwritten
// meets its own value), returned to every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {
  const int x = __float_as_int(v);
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(x, x, CTRL, ROWS, 0xf, false)));
}

__device__ __forceinline__ float wave_max(float v) {
  v = dpp_max<0xb1, 0xf>(v);
  v = dpp_max<0x4e, 0xf>(v);
  v = dpp_max<0x141, 0xf>(v);
  v = dpp_max<0x140, 0xf>(v);
  v = dpp_max<0x142, 0xa>(v);
  v = dpp_max<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Max and sum over the 16 lanes of a row, by the first four of those steps, returned to each of them.
__device__ __forceinline__ float row16_max(float v) {
  return dpp_max<0x140, 0xf>(dpp_max<0x141, 0xf>(dpp_max<0x4e, 0xf>(dpp_max<0xb1, 0xf>(v))));
}

__device__ __forceinline__ float row16_sum(float v) {
  v += __builtin_amdgcn_update_dpp(0.f, v, 0xb1, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0.f, v, 0x4e, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0.f, v, 0x141, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0.f, v, 0x140, 0xf, 0xf, false);
  return v;
}

// Sum over a workgroup of WAVES waves, in a fixed order; `red` holds WAVES floats.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (WAVES == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += red[w];
  return s;
}

}  // namespace bf
