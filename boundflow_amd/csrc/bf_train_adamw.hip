// AdamW over many weight tensors in one launch, moments in fp32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Everything is computed in fp32; w is the weight, or its fp32 master copy where there is one, and is
// rounded to the weight's type once.  The moments of all tensors lie in one array each, every
// tensor from a multiple of ADAMW_BLOCK elements on.
//
// Moments in 8 bits: m and r = sqrt(v) as float8 e4m3 numbers times a scale per ADAMW_BLOCK elements
// (the block's largest magnitude over 448, e4m3's largest number).  The root halves v's range in the
// exponent, so a block's numbers reach down to 2^-17.8 of its largest.  An average that moves by less than
// half a spacing (3 to 6 per cent) a step would stay where it is if it were rounded to the nearest number, so
// a magnitude is rounded by adding a phase below one spacing and cutting: up in as many steps of many
// as it is parts of a spacing above the number below.  The phase of element i at step t is the fraction
// of i sqrt(2) + t (golden ratio): its values over the steps are as even as a sequence can have them, so
// what is lost in one step is made up within a few (random numbers would leave a random walk).
// r is rounded to at least the least number (the update divides by it); a block whose largest
// is below 2^-100 is held as zeros; a moment that is not finite is held as NaN and takes no part
// in its block's scale.
//
// Bound by memory: 150 M bf16 weights with master copies and fp32 moments 917 us for 4.2 GB = 4.6 TB/s; 300 M bf16
// weights with 8-bit moments 668 us for 3.04 GB = 4.5 TB/s, with roots and quotients rounded correctly (some 90 vector
// instructions a weight, which still fit beside the traffic).  The tensors' addresses come as launch arguments: no table
// on the device has to be kept in step with them, and a step of six small tensors is one launch of 5.4 us.

#include "bf_train.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

namespace bf {

constexpr int ADAMW_BLOCK = 128;
constexpr int ADAMW_THREADS = 256;
// Elements of a thread: with fp32 moments four, 16 bytes, so that a wave's accesses are whole lines (eight took
// 1004 us for 150 M bf16 weights with master copies, four 917: 4.6 TB/s); with 8-bit moments eight, 16 lanes a block.
constexpr int adamw_vec(bool eight) { return eight ? 8 : 4; }
constexpr int adamw_chunk(bool eight) { return ADAMW_THREADS * adamw_vec(eight); }   // elements of a workgroup
constexpr int ADAMW_MOST = 96;                                // tensors of a launch (they lie in its arguments)

struct AdamWTensors {
  void* p[ADAMW_MOST];
  const void* g[ADAMW_MOST];
  int64_t n[ADAMW_MOST];
  int64_t at[ADAMW_MOST];          // first element in the moments
  int first[ADAMW_MOST + 1];       // first workgroup
  int count;
};

struct AdamWStep {
  void *m, *v;
  float *m_scale, *v_scale, *master;
  const float* grad_scale;
  float scale, b1, w1, b2, w2, eps, keep, rate, inv_root_bc2;
  uint32_t phase;
};

constexpr float kLargest8 = 448.f, kLeastTop8 = 7.888609052210118e-31f;   // 2^-100

// Max over the 16 lanes of a row of bit patterns of magnitudes (ordered as unsigned numbers).
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));    // quad_perm [1, 0, 3, 2]
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));    // quad_perm [2, 3, 0, 1]
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));   // row_half_mirror
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));   // row_mirror
  return v;
}

// Eight values of a block held in 8 bits: their codes, and the block's scale.  u: phases of 20 bits.
template <bool ROOT>
__device__ __forceinline__ uint64_t hold8(const float (&x)[8], const uint32_t (&u)[8], float* scale) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, (uint32_t)__float_as_int(x[k]) & 0x7fffffffu);
  top = row_max(top);
  const bool odd = top >= 0x7f800000u;   // the same in the block's 16 lanes
  if (odd) {
    top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t b = (uint32_t)__float_as_int(x[k]) & 0x7fffffffu;
      top = max(top, b < 0x7f800000u ? b : 0u);
    }
    top = row_max(top);
  }
  const float largest = __int_as_float((int)top);
  const bool used = largest >= kLeastTop8;
  const float inverse = used ? 1.f / largest * kLargest8 : 0.f;
  *scale = used ? largest * (1.f / kLargest8) : 0.f;
  uint64_t codes = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float y = fminf(fabsf(x[k]) * inverse, kLargest8);
    // spacings below y in units of 2^-20, plus the phase, cut: from 2^-6 on the bit pattern counts them
    uint32_t code = y < 0.015625f ? ((uint32_t)(y * 536870912.f) + u[k]) >> 20
                                  : (((uint32_t)__float_as_int(y) + u[k]) >> 20) - (120u << 3);
    if (ROOT)
      code = y > 0.f ? max(code, 1u) : code;
    else
      code |= ((uint32_t)__float_as_int(x[k]) >> 24) & 0x80u;
    if (odd && ((uint32_t)__float_as_int(x[k]) & 0x7fffffffu) >= 0x7f800000u) code = 0x7f;
    codes |= (uint64_t)code << (8 * k);
  }
  return codes;
}

__device__ __forceinline__ void taken8(uint64_t codes, float scale, float (&x)[8]) {
  typedef float float2v __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)(codes >> (32 * h));
    const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[4 * h] = a.x * scale;
    x[4 * h + 1] = a.y * scale;
    x[4 * h + 2] = b.x * scale;
    x[4 * h + 3] = b.y * scale;
  }
}

template <class T, int VEC>
__device__ __forceinline__ void load_elems(const T* p, int64_t left, float (&x)[VEC]) {
  if (left >= VEC) {
    const Pack<T, VEC> r = load_pack<T, VEC>(p);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = (float)r.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = k < left ? (float)p[k] : 0.f;
  }
}

template <class T, int VEC>
__device__ __forceinline__ void store_elems(T* p, int64_t left, const float (&x)[VEC]) {
  if (left >= VEC) {
    Pack<T, VEC> r;
#pragma unroll
    for (int k = 0; k < VEC; ++k) r.v[k] = (T)x[k];
    store_pack(p, r);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k < left) p[k] = (T)x[k];
  }
}

template <class TP, class TG, bool EIGHT>
__global__ __launch_bounds__(ADAMW_THREADS) void adamw_kernel(AdamWTensors a, AdamWStep c) {
  constexpr int VEC = adamw_vec(EIGHT);
  // the workgroup's tensor: the last whose first workgroup is not past this one
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= (int)blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const int64_t i0 = ((int64_t)blockIdx.x - a.first[lo]) * adamw_chunk(EIGHT) + threadIdx.x * VEC;
  const int64_t left = a.n[lo] - i0, e0 = a.at[lo] + i0;
  // a block's padding is held with it
  const bool in = EIGHT ? i0 < ceil_div(a.n[lo], ADAMW_BLOCK) * ADAMW_BLOCK : left > 0;
  if (!in) return;   // in 8 bits a block's 16 lanes leave together
  TP* p = static_cast<TP*>(a.p[lo]) + i0;
  const TG* g = static_cast<const TG*>(a.g[lo]) + i0;
  float gs = c.scale;
  if (c.grad_scale) gs *= *c.grad_scale;
  float gr[VEC], w[VEC], m[VEC], v[VEC];
  load_elems(g, left, gr);
  if (c.master) load_elems(c.master + e0, left, w);
  else load_elems(static_cast<const TP*>(p), left, w);
  if constexpr (EIGHT) {
    uint64_t mc, vc;
    __builtin_memcpy(&mc, static_cast<const uint8_t*>(c.m) + e0, 8);
    __builtin_memcpy(&vc, static_cast<const uint8_t*>(c.v) + e0, 8);
    taken8(mc, c.m_scale[e0 / ADAMW_BLOCK], m);
    taken8(vc, c.v_scale[e0 / ADAMW_BLOCK], v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] *= v[k];
  } else {
    load_elems(static_cast<const float*>(c.m) + e0, left, m);
    load_elems(static_cast<const float*>(c.v) + e0, left, v);
  }
  float r[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const float x = gr[k] * gs;
    m[k] = m[k] * c.b1 + x * c.w1;
    v[k] = v[k] * c.b2 + x * x * c.w2;
    r[k] = sqrtf(v[k]);
    w[k] = w[k] * c.keep - m[k] / (r[k] * c.inv_root_bc2 + c.eps) * c.rate;
  }
  store_elems(p, left, w);
  if (c.master) store_elems(c.master + e0, left, w);
  if constexpr (EIGHT) {
    uint32_t u[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) u[k] = ((uint32_t)(e0 + k) * 0x6A09E667u + c.phase) >> 12;
    float ms, vs;
    const uint64_t mc = hold8<false>(m, u, &ms), vc = hold8<true>(r, u, &vs);
    __builtin_memcpy(static_cast<uint8_t*>(c.m) + e0, &mc, 8);
    __builtin_memcpy(static_cast<uint8_t*>(c.v) + e0, &vc, 8);
    if (e0 % ADAMW_BLOCK == 0) {
      c.m_scale[e0 / ADAMW_BLOCK] = ms;
      c.v_scale[e0 / ADAMW_BLOCK] = vs;
    }
  } else {
    store_elems(static_cast<float*>(c.m) + e0, left, m);
    store_elems(static_cast<float*>(c.v) + e0, left, v);
  }
}

// Whether no two of the arrays that a step writes share memory: two workgroups would step such elements at once, in
// whatever order.  0.02 us of the host for eight arrays, 2.3 us for 305.
struct Span {
  uintptr_t from, to;
};

static bool apart(Span* spans, int count) {
  std::sort(spans, spans + count, [](const Span& a, const Span& b) { return a.from < b.from; });
  for (int k = 1; k < count; ++k)
    if (spans[k].from < spans[k - 1].to) return false;
  return true;
}

}  // namespace bf

using namespace bf;

extern "C" {

int bf_adamw_multi(int count, void* const* p, const void* const* g, const int64_t* n, int p_elem, int g_elem, void* m,
                   void* v, float* m_scale, float* v_scale, float* master, double lr, double beta1, double beta2,
                   double eps, double weight_decay, int64_t step, float grad_scale, const float* grad_scale_dev,
                   hipStream_t stream) {
  BF_REQUIRE(elem_ok(p_elem) && elem_ok(g_elem), "bf_adamw_multi: element types %d, %d", p_elem, g_elem);
  BF_REQUIRE(count >= 0 && step >= 1, "bf_adamw_multi: %d tensors, step %lld", count, (long long)step);
  BF_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "bf_adamw_multi: betas %g, %g, eps %g",
             beta1, beta2, eps);
  BF_REQUIRE((m_scale != nullptr) == (v_scale != nullptr), "bf_adamw_multi: one moment has scales, the other none");
  if (count == 0) return BF_OK;
  BF_REQUIRE(p && g && n, "bf_adamw_multi: null pointer");
  // All checks come before the first launch: a call that is refused has stepped nothing.
  constexpr int FEW = 256, OTHERS = 5;
  Span few[FEW];
  std::unique_ptr<Span[]> many;
  if ((int64_t)count + OTHERS > FEW) {
    many.reset(new (std::nothrow) Span[(size_t)count + OTHERS]);
    BF_REQUIRE(many, "bf_adamw_multi: no host memory to check %d tensors", count);
  }
  Span* spans = many ? many.get() : few;
  int written = 0;
  int64_t total = 0;
  const int chunk = adamw_chunk(m_scale != nullptr);
  const auto writes = [&](const void* array, int64_t bytes) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(array);
    if (array && bytes) spans[written++] = Span{from, from + (uintptr_t)bytes};
  };
  for (int k = 0; k < count; ++k) {
    BF_REQUIRE(n[k] >= 0 && (n[k] == 0 || (p[k] && g[k])), "bf_adamw_multi: tensor %d", k);
    if (!launch_fits(ceil_div(n[k], chunk), ADAMW_THREADS)) {
      set_error("bf_adamw_multi: tensor %d of %lld elements is more than a launch takes", k, (long long)n[k]);
      return BF_ERANGE;
    }
    writes(p[k], n[k] * elem_bytes(p_elem));
    total += ceil_div(n[k], ADAMW_BLOCK) * ADAMW_BLOCK;
  }
  if (total == 0) return BF_OK;
  BF_REQUIRE(m && v, "bf_adamw_multi: null pointer");
  writes(m, total * (m_scale ? 1 : 4));
  writes(v, total * (m_scale ? 1 : 4));
  writes(m_scale, total / ADAMW_BLOCK * 4);
  writes(v_scale, total / ADAMW_BLOCK * 4);
  writes(master, total * 4);
  BF_REQUIRE(apart(spans, written),
             "bf_adamw_multi: two of the weights, moments and copies share memory (tied weights are listed once)");
  // scalars in double, rounded once
  AdamWStep c;
  c.m = m;
  c.v = v;
  c.m_scale = m_scale;
  c.v_scale = v_scale;
  c.master = master;
  c.grad_scale = grad_scale_dev;
  c.scale = grad_scale;
  c.b1 = (float)beta1;
  c.w1 = (float)(1.0 - beta1);
  c.b2 = (float)beta2;
  c.w2 = (float)(1.0 - beta2);
  c.eps = (float)eps;
  c.keep = (float)(1.0 - lr * weight_decay);
  c.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  c.inv_root_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  c.phase = (uint32_t)(uint64_t)step * 0x9E3779B9u;
  int64_t at = 0;
  for (int k = 0; k < count;) {
    AdamWTensors a;
    memset(&a, 0, sizeof(a));
    int64_t blocks = 0;
    for (; k < count && a.count < ADAMW_MOST; ++k) {
      if (n[k] == 0) continue;
      const int64_t more = ceil_div(n[k], chunk);
      if (!launch_fits(blocks + more, ADAMW_THREADS)) break;   // a launch takes any one tensor
      a.p[a.count] = p[k];
      a.g[a.count] = g[k];
      a.n[a.count] = n[k];
      a.at[a.count] = at;
      a.first[a.count] = (int)blocks;
      at += ceil_div(n[k], ADAMW_BLOCK) * ADAMW_BLOCK;
      blocks += more;
      ++a.count;
    }
    if (blocks == 0) continue;
    a.first[a.count] = (int)blocks;
    const int rc = with_elem(p_elem, [&](auto tp) -> int {
      using TP = decltype(tp);
      return with_elem(g_elem, [&](auto tg) -> int {
        using TG = decltype(tg);
        if (m_scale)
          hipLaunchKernelGGL((adamw_kernel<TP, TG, true>), dim3((unsigned)blocks), dim3(ADAMW_THREADS), 0, stream, a, c);
        else
          hipLaunchKernelGGL((adamw_kernel<TP, TG, false>), dim3((unsigned)blocks), dim3(ADAMW_THREADS), 0, stream, a,
                             c);
        BF_LAUNCH_CHECK("adamw_kernel");
        return BF_OK;
      });
    });
    if (rc != BF_OK) return rc;
  }
  return BF_OK;
}

}  // extern "C"
