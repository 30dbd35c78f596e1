// Dropout with a mask that is never stored: whether element e is kept follows from a seed, a counter and e, so the
// backward pass makes the mask again.
//
//   y_e = r_e + (u_e >= border ? x_e / (1 - border / 2^16) : 0),   border = p 2^16, rounded
//
// u_e is 16 bits of the counter-based generator Philox 4x32 of ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011): its counter is (e / 8, counter), 64 bits each, its key the seed, and its
// 128 bits give eight elements.  e counts the elements of x in their order, whatever x's strides.

#include "bf_train.h"

namespace bf {

struct DropoutArgs {
  const void* x;
  const void* residual;
  void* out;
  int64_t rows, dim;            // elements e = row * dim + column
  int64_t x_ld, residual_ld;
  int64_t first, blocks;        // of eight elements: those of this launch
  uint32_t key0, key1, border;
  uint64_t counter;
  const int64_t* counter_dev;   // read instead, where given
  float scale;
};

struct Philox {
  uint32_t w[4];
};

__device__ __forceinline__ Philox philox(uint64_t block, uint64_t counter, uint32_t k0, uint32_t k1) {
  uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = (uint32_t)counter, d = (uint32_t)(counter >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t one = (uint64_t)a * 0xD2511F53u, two = (uint64_t)c * 0xCD9E8D57u;
    a = (uint32_t)(two >> 32) ^ b ^ k0;
    b = (uint32_t)two;
    c = (uint32_t)(one >> 32) ^ d ^ k1;
    d = (uint32_t)one;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{a, b, c, d}};
}

// A thread per eight elements; eight that span rows (a width that is no multiple of eight, in rows with gaps) are addressed one by
// one.  Bound by memory: 16384 x 4096 bf16 46 us (268 MB at 5.8 TB/s), with a residual 70 us (403 MB at 5.7 TB/s); rows
// with gaps, of an odd width, the same.  A small tensor takes the host's call, 8 us.
template <class T, bool FLAT>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.blocks) return;
  const int64_t block = p.first + at, e0 = block * 8, total = p.rows * p.dim;
  const uint64_t counter = p.counter_dev ? (uint64_t)*p.counter_dev : p.counter;
  const Philox u = philox(block, counter, p.key0, p.key1);
  const T* x = (const T*)p.x;
  const T* r = (const T*)p.residual;
  T* out = (T*)p.out;
  auto element = [&](int k, float xk, float rk) {
    const uint32_t drawn = (u.w[k >> 1] >> (16 * (k & 1))) & 0xffff;
    const float kept = drawn >= p.border ? xk * p.scale : 0.f;   // a dropped infinity or NaN is dropped
    return (T)(r ? kept + rk : kept);
  };
  // where x and the residual have the eight: a row's part unless they span rows or end the last one
  int64_t row = 0, col = e0;
  if constexpr (!FLAT) {
    row = div_rows(e0, p.dim, total < (1LL << 31));
    col = e0 - row * p.dim;
  }
  const int64_t width = FLAT ? total : p.dim;
  if (col + 8 <= width) {
    const Pack<T, 8> xs = load_pack<T, 8>(x + row * p.x_ld + col);
    Pack<T, 8> rs, ys;
    if (r) rs = load_pack<T, 8>(r + row * p.residual_ld + col);
#pragma unroll
    for (int k = 0; k < 8; ++k) ys.v[k] = element(k, (float)xs.v[k], r ? (float)rs.v[k] : 0.f);
    store_pack(out + e0, ys);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (e0 + k >= total) break;
    out[e0 + k] = element(k, (float)x[row * p.x_ld + col], r ? (float)r[row * p.residual_ld + col] : 0.f);
    if (!FLAT && ++col == p.dim) {
      col = 0;
      ++row;
    }
    if (FLAT) ++col;
  }
}

}  // namespace bf

using namespace bf;

extern "C" int bf_dropout(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, int elem, int64_t rows,
                          int64_t dim, double p, int64_t seed, int64_t counter, const int64_t* counter_dev, void* out,
                          hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem), "bf_dropout: element type %d", elem);
  BF_REQUIRE(rows >= 0 && dim >= 0 && x_ld >= dim && residual_ld >= (residual ? dim : 0), "bf_dropout: bad sizes");
  BF_REQUIRE(p >= 0.0 && p <= 1.0, "bf_dropout: probability %g", p);
  if (rows == 0 || dim == 0) return BF_OK;
  BF_REQUIRE(x && out, "bf_dropout: null pointer");
  if (rows > (1LL << 40) || dim > (1LL << 40) || rows > (1LL << 42) / dim) {
    set_error("bf_dropout: %lld x %lld elements are more than it takes", (long long)rows, (long long)dim);
    return BF_ERANGE;
  }
  DropoutArgs a;
  memset(&a, 0, sizeof(a));
  a.x = x;
  a.residual = residual;
  a.out = out;
  a.rows = rows;
  a.dim = dim;
  a.x_ld = x_ld;
  a.residual_ld = residual_ld;
  a.key0 = (uint32_t)seed;
  a.key1 = (uint32_t)((uint64_t)seed >> 32);
  a.border = (uint32_t)(p * 65536.0 + 0.5);
  a.scale = a.border < 65536 ? (float)(65536.0 / (65536 - a.border)) : 0.f;
  a.counter = (uint64_t)counter;
  a.counter_dev = counter_dev;
  const bool flat = (x_ld == dim || rows == 1) && (!residual || residual_ld == dim || rows == 1);
  const int64_t all = ceil_div(rows * dim, 8), most = 1LL << 31;
  for (a.first = 0; a.first < all; a.first += most) {
    a.blocks = all - a.first < most ? all - a.first : most;
    const dim3 grid((unsigned)ceil_div(a.blocks, 256));
    with_elem(elem, [&](auto t) {
      using T = decltype(t);
      if (flat) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, stream, a);
      return 0;
    });
    BF_LAUNCH_CHECK("bf_dropout");
  }
  return BF_OK;
}
