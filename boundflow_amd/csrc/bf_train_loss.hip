// Losses of token logits, with their gradients.
//
// With z = logits / temperature, l = log sum exp z and the log-probability p_t = z[t] - l of the
// token t that a row predicts, a loss L whose derivative by p_t is g has the logit gradient
//   dL/dlogits = g / temperature * (onehot(t) - softmax(z)).
//
// Policy loss (bf_policy_loss): with r = exp(p_t - old), A the advantage, w the row's weight,
//   L = sum w (-min(r A, clip(r, 1 - lo, 1 + hi) A) + k (exp(d) - d - 1)),   d = ref - p_t.
// Preference loss (bf_preference_loss): with s = sum over a response's rows of p_t - ref,
//   L = mean over pairs of -(1 - e) log sigma(h) - e log sigma(-h),   h = beta (s_chosen - s_rejected).
//
// Exponentials are taken in base 2 of c z, c = log2(e) / temperature, against a whole number
// K >= max(c z): the argument c z - K is one fused multiply-add of the logit (rounded once), and
// moving a sum from one K to a larger one is a multiplication by a power of two, which is exact.

#include "bf_train.h"

#include <cmath>

namespace bf {

constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Logits below -2^126 (a type's lowest value in a mask, say) count in rows that have nothing else:
// those are uniform over what is not -inf, as the difference of equal logits says.  In base 2 they
// would overflow, so they have a K of their own.  A row of -inf alone has no distribution (NaN).
constexpr float kLowest = -8.507059173023462e37f;    // -2^126
constexpr float kLowK = -1.7014118346046923e38f;     // -2^127: against any other K its terms are 0

// Adds 2^(c z - K) over N logits to the sum s at K, raising K where a logit needs it.
template <int N>
__device__ __forceinline__ void add_terms(float& K, float& s, const float (&z)[N], float c) {
  float m = z[0];
#pragma unroll
  for (int k = 1; k < N; ++k) m = fmaxf(m, z[k]);
  if (m < kLowest) {
    const float K1 = m > -__builtin_inff() ? fmaxf(K, kLowK) : K;
    K = K1;   // from -inf, where s is 0 (or NaN)
#pragma unroll
    for (int k = 0; k < N; ++k) s += z[k] != z[k] ? z[k] : K == kLowK && z[k] > -__builtin_inff() ? 1.f : 0.f;
    return;
  }
  const float K1 = fmaxf(K, ceilf(m * c));
  if (K1 != K) {
    s = K > kLowK ? s * __builtin_amdgcn_exp2f(K - K1) : s != s ? s : 0.f;
    K = K1;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) s += __builtin_amdgcn_exp2f(fmaf(z[k], c, -K));
}

// s 2^from as a multiple of 2^to, to >= from; a sum of nothing (from is -inf) stays nothing
__device__ __forceinline__ float moved(float s, float from, float to) {
  return from == to ? s : s * exp2_fast(from - to);
}

// 2^(c z - K)
__device__ __forceinline__ float term(float z, float c, float K) {
  return K == kLowK ? (z > -__builtin_inff() ? 1.f : 0.f) : exp2_fast(fmaf(z, c, -K));
}

// Rows of logits: row n is logits + (n / T) ld_b + (n % T) ld_t.
struct LogitRows {
  int64_t T, ld_b, ld_t;
  int64_t V;
  __device__ __forceinline__ int64_t offset(int64_t n) const {
    const int64_t b = div_rows(n, T, n < (1LL << 31) && T < (1LL << 31));
    return b * ld_b + (n - b * T) * ld_t;
  }
};

// a row that takes part: not masked, and its token not negative
__device__ __forceinline__ bool live_row(const uint8_t* mask, const void* tokens, int token_bytes, int64_t n) {
  return (mask == nullptr || mask[n]) && load_token(tokens, token_bytes, n) >= 0;
}

constexpr int LOSS_THREADS = 256, LOSS_WAVES = LOSS_THREADS / 64;

// ---------------------------------------------------------------------------
// (K, sum of 2^(c z - K)) of a part of a row.  Workgroup = (row, part of `chunk` elements).
template <class T>
__global__ __launch_bounds__(LOSS_THREADS) void loss_partial_kernel(const T* __restrict__ logits, LogitRows rows,
                                                                    const void* __restrict__ tokens, int token_bytes,
                                                                    const uint8_t* __restrict__ mask, float c, int parts,
                                                                    int64_t chunk, float2* __restrict__ part) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float red_k[LOSS_WAVES], red_s[LOSS_WAVES];
  const int64_t n = blockIdx.x / (unsigned)parts;
  const int q = (int)(blockIdx.x % (unsigned)parts);
  if (!live_row(mask, tokens, token_bytes, n)) return;
  const T* row = logits + rows.offset(n);
  const int64_t from = q * chunk, to = min(from + chunk, rows.V);
  float K = -__builtin_inff(), s = 0.f;
  for (int64_t d = from + threadIdx.x * VEC; d < to; d += LOSS_THREADS * VEC) {
    float z[VEC];
    if (d + VEC <= to) {
      const Pack<T, VEC> x = load_pack<T, VEC>(row + d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) z[k] = (float)x.v[k];
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) z[k] = d + k < to ? (float)row[d + k] : -__builtin_inff();
    }
    add_terms(K, s, z, c);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float K2 = __shfl_xor(K, d), s2 = __shfl_xor(s, d), K1 = fmaxf(K, K2);
    s = moved(s, K, K1) + moved(s2, K2, K1);
    K = K1;
  }
  if ((threadIdx.x & 63) == 0) {
    red_k[threadIdx.x >> 6] = K;
    red_s[threadIdx.x >> 6] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < LOSS_WAVES; ++w) {
      const float K1 = fmaxf(K, red_k[w]);
      s = moved(s, K, K1) + moved(red_s[w], red_k[w], K1);
      K = K1;
    }
    part[blockIdx.x] = make_float2(K, s);
  }
}

// A row's softmax: K, s over its parts, and the log-probability of its token.
struct RowSoftmax {
  float K, s, logp;
};

template <class T>
__device__ __forceinline__ RowSoftmax row_softmax(const T* logits, const LogitRows& rows, int64_t n, int t,
                                                  const float2* part, int parts, float c) {
  RowSoftmax r;
  r.K = -__builtin_inff();
  r.s = 0.f;
  for (int q = 0; q < parts; ++q) {
    const float2 x = part[n * parts + q];
    const float K1 = fmaxf(r.K, x.x);
    r.s = moved(r.s, r.K, K1) + moved(x.y, x.x, K1);
    r.K = K1;
  }
  // a token past the vocabulary shows as NaN
  if ((int64_t)t >= rows.V) {
    r.logp = __int_as_float(0x7fc00000);
    return r;
  }
  const float z = (float)logits[rows.offset(n) + t];
  const float x = r.K == kLowK ? (z > -__builtin_inff() ? 0.f : z) : fmaf(z, c, -r.K);
  r.logp = (x - log2_fast(r.s)) * kLn2;
  return r;
}

// What the gradient of a row needs: dlogits = 2^(c z - K) * q (+ g at the token).
// A row with g = 0 gets zeros and its logits are not read.
__device__ __forceinline__ float4 row_gradient(const RowSoftmax& r, float g) {
  return make_float4(r.K, -g / r.s, g, 0.f);
}

template <class T>
__global__ __launch_bounds__(LOSS_THREADS) void loss_grad_kernel(const T* __restrict__ logits, LogitRows rows,
                                                                 const void* __restrict__ tokens, int token_bytes,
                                                                 float c, int parts, int64_t chunk,
                                                                 const float4* __restrict__ coef, T* __restrict__ grad) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t n = blockIdx.x / (unsigned)parts;
  const int q = (int)(blockIdx.x % (unsigned)parts);
  const T* row = logits + rows.offset(n);
  T* out = grad + n * rows.V;
  const float4 f = coef[n];
  const int64_t t = load_token(tokens, token_bytes, n);
  const int64_t from = q * chunk, to = min(from + chunk, rows.V);
  const bool read = f.z != 0.f;
  for (int64_t d = from + threadIdx.x * VEC; d < to; d += LOSS_THREADS * VEC) {
    if (d + VEC <= to) {
      Pack<T, VEC> x;
      if (read) {
        x = load_pack<T, VEC>(row + d);
        float y[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = term((float)x.v[k], c, f.x) * f.y;
        if (t >= d && t < d + VEC)
#pragma unroll
          for (int k = 0; k < VEC; ++k) y[k] += t == d + k ? f.z : 0.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x.v[k] = (T)y[k];
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x.v[k] = (T)0.f;
      }
      store_pack(out + d, x);
    } else {
      for (int64_t e = d; e < to; ++e)
        out[e] = (T)(read ? term((float)row[e], c, f.x) * f.y + (t == e ? f.z : 0.f) : 0.f);
    }
  }
}

// ---------------------------------------------------------------------------
// Policy loss

struct PolicyArgs {
  const void* tokens;
  const float *old_logp, *ref_logp, *advantages;
  const uint8_t* mask;
  int64_t B, T, adv_b, adv_t;
  float low, high, kl_weight, c, inv_t, grad_scale;
  int token_bytes, by_sequence;
};

constexpr int WEIGHT_THREADS = 1024, WEIGHT_WAVES = WEIGHT_THREADS / 64;

// weight[b]: 1 / live rows (of all, or with by_sequence of the sequence times the sequences that have
// any).  One workgroup, a wave per sequence.
__global__ __launch_bounds__(WEIGHT_THREADS) void policy_weights_kernel(PolicyArgs a, float* __restrict__ weight) {
  __shared__ float red[WEIGHT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float total = 0.f, some = 0.f;   // of a wave's sequences, in lane 0
  for (int64_t b = wave; b < a.B; b += WEIGHT_WAVES) {
    int live = 0;
    for (int64_t t = lane; t < a.T; t += 64) live += live_row(a.mask, a.tokens, a.token_bytes, b * a.T + t);
#pragma unroll
    for (int d = 32; d; d >>= 1) live += __shfl_xor(live, d);
    if (lane == 0) {
      weight[b] = (float)live;
      total += (float)live;
      some += live > 0 ? 1.f : 0.f;
    }
  }
  const float all = block_sum<WEIGHT_WAVES>(a.by_sequence ? some : total, red);
  __syncthreads();   // weight[] is written by the waves' first lanes
  for (int64_t b = threadIdx.x; b < a.B; b += WEIGHT_THREADS) {
    const float live = weight[b];
    weight[b] = live > 0.f ? 1.f / (a.by_sequence ? live * all : all) : 0.f;
  }
}

struct PolicyRow {
  float policy, kl, outside, g;
};

// A live row's terms and dL/dp_t, before its weight.
__device__ __forceinline__ PolicyRow policy_row(const PolicyArgs& a, int64_t n, float logp) {
  PolicyRow r;
  const int64_t b = div_rows(n, a.T, n < (1LL << 31) && a.T < (1LL << 31));
  const float A = a.advantages[b * a.adv_b + (n - b * a.T) * a.adv_t];
  const float ratio = expf(logp - a.old_logp[n]);
  const float plain = ratio * A, clipped = fminf(fmaxf(ratio, a.low), a.high) * A;
  const bool out = clipped < plain;   // the clipped side is the smaller: a constant, without a gradient
  r.policy = out ? -clipped : -plain;
  r.outside = out ? 1.f : 0.f;
  r.g = out ? 0.f : -plain;
  r.kl = 0.f;
  if (a.ref_logp) {
    const float apart = a.ref_logp[n] - logp, e = expm1f(apart);
    r.kl = e - apart;
    r.g -= a.kl_weight * e;
  }
  return r;
}

// One thread per row: its gradient's coefficients, and the workgroup's share of the sums.
template <class T>
__global__ __launch_bounds__(LOSS_THREADS) void policy_rows_kernel(const T* __restrict__ logits, LogitRows rows,
                                                                   PolicyArgs a, const float2* __restrict__ part,
                                                                   int parts, const float* __restrict__ weight,
                                                                   float* __restrict__ logp, float4* __restrict__ coef,
                                                                   float4* __restrict__ sums) {
  __shared__ float red[LOSS_WAVES];
  const int64_t n = (int64_t)blockIdx.x * LOSS_THREADS + threadIdx.x, N = a.B * a.T;
  float policy = 0.f, kl = 0.f, outside = 0.f;
  if (n < N) {
    float lp = 0.f;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live_row(a.mask, a.tokens, a.token_bytes, n)) {
      const RowSoftmax x = row_softmax(logits, rows, n, load_token(a.tokens, a.token_bytes, n), part, parts, a.c);
      const PolicyRow r = policy_row(a, n, x.logp);
      const float w = weight[div_rows(n, a.T, n < (1LL << 31) && a.T < (1LL << 31))];
      lp = x.logp;
      policy = w * r.policy;
      kl = w * r.kl;
      outside = w * r.outside;
      f = row_gradient(x, w * r.g * a.inv_t * a.grad_scale);
    }
    logp[n] = lp;
    coef[n] = f;
  }
  policy = block_sum<LOSS_WAVES>(policy, red);
  kl = block_sum<LOSS_WAVES>(kl, red);
  outside = block_sum<LOSS_WAVES>(outside, red);
  if (threadIdx.x == 0) sums[blockIdx.x] = make_float4(policy, kl, outside, 0.f);
}

// Sixteen bytes of logits as they are.  as_floats keeps the compiler from holding on to the fp32 values of a
// row between its two uses, which would take twice the registers that the row does.
typedef uint32_t Words __attribute__((ext_vector_type(4)));

template <class T, int VEC>
__device__ __forceinline__ void as_floats(Words& w, float (&z)[VEC]) {
  asm volatile("" : "+v"(w));
  Pack<T, VEC> x;
  __builtin_memcpy(&x, &w, sizeof(x));
#pragma unroll
  for (int e = 0; e < VEC; ++e) z[e] = (float)x.v[e];
}

// base: the same in the whole workgroup (scalar registers); at: the thread's bytes
__device__ __forceinline__ Words load_words(const void* base, uint32_t at) {
  Words w;
  __builtin_memcpy(&w, static_cast<const char*>(base) + at, sizeof(w));
  return w;
}

// A workgroup's row in registers: vector k * THREADS + tid of 16 bytes in x[k], and of the elements
// past the last whole vector the tid-th in `rest`.
template <class T, int THREADS, int NV>
struct HeldRow {
  static constexpr int VEC = 16 / sizeof(T), WAVES = THREADS / 64, STEP = THREADS * 16;
  Words x[NV];
  float rest;

  static __device__ __forceinline__ uint32_t at() { return threadIdx.x * 16u; }
  static __device__ __forceinline__ bool has(int k, int vecs) { return k * THREADS + (int)threadIdx.x < vecs; }

  __device__ __forceinline__ void load(int k, const T* row, int vecs) {
    if (has(k, vecs)) x[k] = load_words(reinterpret_cast<const char*>(row) + k * STEP, at());
  }
  __device__ __forceinline__ void load_rest(const T* row, int vecs, int V) {
    const int e = vecs * VEC + (int)threadIdx.x;
    if (e < V) rest = (float)row[e];
  }

  // (K, sum) of the row's softmax, the same in every thread; `red` holds WAVES pairs
  __device__ __forceinline__ float2 softmax(int vecs, int V, float c, float2* red) {
    float K = -__builtin_inff(), s = 0.f, z[VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (has(k, vecs)) {
        as_floats<T>(x[k], z);
        add_terms(K, s, z, c);
      }
    if (vecs * VEC + (int)threadIdx.x < V) {
      const float one[1] = {rest};
      add_terms(K, s, one, c);
    }
    const float Kw = wave_max(K);
    s = wave_sum(moved(s, K, Kw));
    if constexpr (WAVES == 1) return make_float2(Kw, s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(Kw, s);
    __syncthreads();
    K = red[0].x;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) K = fmaxf(K, red[w].x);
    s = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += moved(red[w].y, red[w].x, K);
    return make_float2(K, s);
  }
};

// What a workgroup writes for a row: its gradient, or zeros.
enum : int { ROW_ZEROS, ROW_TERMS, ROW_LOWEST };

// g (onehot(t) - softmax) of vector k, written; q = -g / sum.  `how` is the same in the whole workgroup.
template <class T, int THREADS, int NV>
__device__ __forceinline__ void write_gradient(HeldRow<T, THREADS, NV>& h, int k, int vecs, T* out, int how, float c,
                                               float K, float q, float g, int t) {
  constexpr int VEC = HeldRow<T, THREADS, NV>::VEC;
  if (!h.has(k, vecs)) return;
  float f[VEC];
  if (how == ROW_TERMS) {
    as_floats<T>(h.x[k], f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = exp2_fast(fmaf(f[e], c, -K)) * q;
  } else if (how == ROW_LOWEST) {
    as_floats<T>(h.x[k], f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = f[e] > -__builtin_inff() ? q : 0.f;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = 0.f;
  }
  const int d = t - (k * THREADS + (int)threadIdx.x) * VEC;
  if (d >= 0 && d < VEC)
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] += d == e ? g : 0.f;
  Pack<T, VEC> y;
#pragma unroll
  for (int e = 0; e < VEC; ++e) y.v[e] = (T)f[e];
  __builtin_memcpy(reinterpret_cast<char*>(out) + k * HeldRow<T, THREADS, NV>::STEP + h.at(), &y, sizeof(y));
}

// The whole loss of a row in one pass over its logits.  A workgroup holds a row in registers, reduces its
// softmax, forms the row's term and writes the gradient; as each vector's gradient is stored, the same
// vector of the workgroup's next row is loaded into its registers, so that loads are in flight while
// gradients are formed and stored.  Every logit is read once and every gradient written once.
template <class T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void policy_row_kernel(const T* __restrict__ logits, LogitRows rows, PolicyArgs a,
                                                             const float* __restrict__ weight,
                                                             float* __restrict__ logp, T* __restrict__ grad,
                                                             float4* __restrict__ sums) {
  using Held = HeldRow<T, THREADS, NV>;
  __shared__ float2 red[2][Held::WAVES];
  const int N = (int)(a.B * a.T), V = (int)rows.V, vecs = V / Held::VEC;
  const float c = a.c;
  Held h;
  int n = blockIdx.x;
  bool live = n < N && live_row(a.mask, a.tokens, a.token_bytes, n);
  const T* row = logits + (n < N ? rows.offset(n) : 0);
  if (live) {
#pragma unroll
    for (int k = 0; k < NV; ++k) h.load(k, row, vecs);
    h.load_rest(row, vecs, V);
  }
  float policy = 0.f, kl = 0.f, outside = 0.f;
  // two buffers, by turns of the rows that use them: before one is filled again, every wave has passed the barrier
  // of the row in between, and so has read it
  int buf = 0;
  while (n < N) {
    const int next = n + (int)gridDim.x;
    const bool next_live = next < N && live_row(a.mask, a.tokens, a.token_bytes, next);
    const T* next_row = logits + (next < N ? rows.offset(next) : 0);
    float lp = 0.f, K = 0.f, q = 0.f, g = 0.f;
    int t = -1, how = ROW_ZEROS;
    if (live) {
      t = load_token(a.tokens, a.token_bytes, n);
      const float zt = t < V ? (float)row[t] : 0.f;
      const float2 soft = h.softmax(vecs, V, c, red[buf]);
      buf ^= 1;
      K = soft.x;
      const float arg = K == kLowK ? (zt > -__builtin_inff() ? 0.f : zt) : fmaf(zt, c, -K);
      lp = t < V ? (arg - log2_fast(soft.y)) * kLn2 : __int_as_float(0x7fc00000);
      const PolicyRow r = policy_row(a, n, lp);
      const float w = weight[div_rows(n, a.T, true)];
      policy += w * r.policy;
      kl += w * r.kl;
      outside += w * r.outside;
      g = w * r.g * a.inv_t * a.grad_scale;
      q = -g / soft.y;
      how = __builtin_amdgcn_readfirstlane(g == 0.f ? ROW_ZEROS : K == kLowK ? ROW_LOWEST : ROW_TERMS);
      if (how == ROW_ZEROS) t = -1;
    }
    if (threadIdx.x == 0) logp[n] = lp;
    T* out = grad + (int64_t)n * V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (grad) write_gradient(h, k, vecs, out, how, c, K, q, g, t);
      if (next_live) h.load(k, next_row, vecs);
      // the loads stay behind the stores of their registers' old contents, in which no copy of the row is made
      __builtin_amdgcn_sched_barrier(0);
    }
    if (grad) {
      const int e = vecs * Held::VEC + (int)threadIdx.x;
      if (e < V) out[e] = (T)(how == ROW_ZEROS ? 0.f : term(h.rest, c, K) * q + (t == e ? g : 0.f));
    }
    if (next_live) h.load_rest(next_row, vecs, V);
    n = next;
    live = next_live;
    row = next_row;
  }
  if (threadIdx.x == 0) sums[blockIdx.x] = make_float4(policy, kl, outside, 0.f);
}

// stats: loss, policy term, KL, clipped share
__global__ __launch_bounds__(LOSS_THREADS) void policy_stats_kernel(const float4* __restrict__ sums, int64_t count,
                                                                    float kl_weight, float* __restrict__ stats) {
  __shared__ float red[LOSS_WAVES];
  float policy = 0.f, kl = 0.f, outside = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += LOSS_THREADS) {
    policy += sums[i].x;
    kl += sums[i].y;
    outside += sums[i].z;
  }
  policy = block_sum<LOSS_WAVES>(policy, red);
  kl = block_sum<LOSS_WAVES>(kl, red);
  outside = block_sum<LOSS_WAVES>(outside, red);
  if (threadIdx.x == 0) {
    stats[0] = policy + kl_weight * kl;
    stats[1] = policy;
    stats[2] = kl;
    stats[3] = outside;
  }
}

// ---------------------------------------------------------------------------
// Preference loss

struct PreferenceArgs {
  const void* tokens;
  const float* ref_logp;
  const int64_t* offsets;
  int64_t N, pairs;
  float beta, smoothing, grad_scale;
  int token_bytes;
};

// log sigma(x) = min(x, 0) - log(1 + exp(-|x|))
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// One workgroup per pair: the rows' log-probabilities, the responses' sums, the pair's loss, and the
// rows' gradient coefficients.
template <class T>
__global__ __launch_bounds__(LOSS_THREADS) void preference_pairs_kernel(
    const T* __restrict__ logits, LogitRows rows, PreferenceArgs a, const float2* __restrict__ part, int parts, float c,
    float* __restrict__ logp, float4* __restrict__ coef, float* __restrict__ rewards, float* __restrict__ losses) {
  __shared__ float red[LOSS_WAVES];
  const int64_t pair = blockIdx.x;
  float sum[2];
  int64_t from[2], to[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int64_t k = pair + side * a.pairs;
    // offsets are data: whatever they hold, the rows read are the batch's
    from[side] = min(max(a.offsets[k], (int64_t)0), a.N);
    to[side] = min(max(a.offsets[k + 1], from[side]), a.N);
    float s = 0.f;
    for (int64_t n = from[side] + threadIdx.x; n < to[side]; n += LOSS_THREADS) {
      const int t = load_token(a.tokens, a.token_bytes, n);
      float lp = 0.f;
      if (t >= 0) {
        const RowSoftmax x = row_softmax(logits, rows, n, t, part, parts, c);
        lp = x.logp;
        s += lp - a.ref_logp[n];
        coef[n] = make_float4(x.K, x.s, 0.f, 0.f);
      }
      logp[n] = lp;
    }
    sum[side] = block_sum<LOSS_WAVES>(s, red);
  }
  const float h = a.beta * sum[0] - a.beta * sum[1];
  const float dh = -((1.f - a.smoothing) * sigmoid(-h) - a.smoothing * sigmoid(h));
  if (threadIdx.x == 0) {
    rewards[pair] = a.beta * sum[0];
    rewards[pair + a.pairs] = a.beta * sum[1];
    losses[pair] = -((1.f - a.smoothing) * log_sigmoid(h) + a.smoothing * log_sigmoid(-h));
  }
  const float g = dh * a.beta * a.grad_scale / (float)a.pairs;
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int64_t n = from[side] + threadIdx.x; n < to[side]; n += LOSS_THREADS)
      if (load_token(a.tokens, a.token_bytes, n) >= 0) {   // coef[n]: written by this thread above
        const float4 f = coef[n];
        coef[n] = row_gradient(RowSoftmax{f.x, f.y, 0.f}, side ? -g : g);
      }
}

__global__ void preference_clear_kernel(int64_t N, float* __restrict__ logp, float4* __restrict__ coef) {
  const int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= N) return;
  logp[n] = 0.f;
  coef[n] = make_float4(0.f, 0.f, 0.f, 0.f);
}

__global__ __launch_bounds__(LOSS_THREADS) void preference_loss_kernel(const float* __restrict__ losses, int64_t pairs,
                                                                       float* __restrict__ loss) {
  __shared__ float red[LOSS_WAVES];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < pairs; i += LOSS_THREADS) s += losses[i];
  s = block_sum<LOSS_WAVES>(s, red);
  if (threadIdx.x == 0) *loss = pairs ? s / (float)pairs : 0.f;
}

// ---------------------------------------------------------------------------
// Parts of a row: enough workgroups to fill the device where there are few rows.
struct Parts {
  int count;
  int64_t chunk;
};

static Parts row_parts(int64_t N, int64_t V, int elem) {
  const int64_t step = LOSS_THREADS * (16 / elem_bytes(elem));
  int64_t want = N < 2048 ? ceil_div(2048, N > 0 ? N : 1) : 1;
  const int64_t most = ceil_div(V, step);
  if (want > most) want = most;
  if (want > 64) want = 64;
  Parts p;
  p.chunk = ceil_div(ceil_div(V, want), step) * step;
  p.count = (int)ceil_div(V, p.chunk);
  return p;
}

// The row kernel's workgroup for V logits: the smallest that holds a row, or 0 where none does
// (rows of 65536 fp32 or 131072 16-bit logits and more).
static int row_threads(int64_t V, int elem) {
  const int64_t vecs = V / (16 / elem_bytes(elem));
  return vecs <= 256 ? 64 : vecs <= 1024 ? 256 : vecs <= 4096 ? 512 : vecs <= 16384 ? 1024 : 0;
}

static bool rows_fit(int64_t N, int64_t V) { return V < (1LL << 30) && N < (1LL << 24); }

}  // namespace bf

using namespace bf;

extern "C" {

// the sums of the row kernel's workgroups, or of 256 rows each
static int64_t sum_groups(int64_t N) {
  const int64_t parts = ceil_div(N, LOSS_THREADS), groups = N < 4096 ? N : 4096;
  return parts > groups ? parts : groups;
}

// coef [N] float4, part [N * parts] float2, sums float4, weight [B]
int64_t bf_policy_loss_workspace(int64_t B, int64_t T, int64_t V, int elem) {
  if (!elem_ok(elem) || B < 0 || T < 0 || V <= 0) return 0;
  const int64_t N = B * T;
  return 4 * N + 2 * N * row_parts(N, V, elem).count + 4 * sum_groups(N) + B;
}

int bf_policy_loss(const void* logits, int elem, int64_t B, int64_t T, int64_t V, int64_t ld_b, int64_t ld_t,
                   const void* tokens, int token_bytes, const float* old_logp, const float* ref_logp,
                   const float* advantages, int64_t adv_b, int64_t adv_t, const void* mask, float clip_low,
                   float clip_high, float kl_weight, double temperature, int by_sequence, float grad_scale, float* logp,
                   float* stats, void* grad, float* workspace, hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8), "bf_policy_loss: element type %d, token bytes %d",
             elem, token_bytes);
  BF_REQUIRE(B >= 0 && T >= 0 && V > 0 && ld_b >= 0 && ld_t >= 0 && adv_b >= 0 && adv_t >= 0,
             "bf_policy_loss: bad sizes");
  BF_REQUIRE(temperature > 0.0 && clip_low >= 0.f && clip_high >= 0.f, "bf_policy_loss: temperature %g, clip %g, %g",
             temperature, clip_low, clip_high);
  BF_REQUIRE(stats, "bf_policy_loss: null pointer");
  const int64_t N = B * T;
  BF_REQUIRE(N == 0 || (logits && tokens && old_logp && advantages && logp && workspace),
             "bf_policy_loss: null pointer");
  if (!rows_fit(N, V) || B >= (1LL << 24) || T >= (1LL << 24)) {
    set_error("bf_policy_loss: %lld rows of %lld logits: rows below 2^24, logits below 2^30", (long long)N,
              (long long)V);
    return BF_ERANGE;
  }
  PolicyArgs a{tokens, old_logp, ref_logp, advantages, static_cast<const uint8_t*>(mask), B, T, adv_b, adv_t,
               1.f - clip_low, 1.f + clip_high, kl_weight, (float)(1.4426950408889634074 / temperature),
               (float)(1.0 / temperature), grad_scale, token_bytes, by_sequence};
  const LogitRows rows{T > 0 ? T : 1, ld_b, ld_t, V};
  const Parts p = row_parts(N, V, elem);
  float4* coef = reinterpret_cast<float4*>(workspace);
  float4* sums = coef + N;
  const int64_t blocks = ceil_div(N, LOSS_THREADS);
  float2* part = reinterpret_cast<float2*>(sums + sum_groups(N));
  float* weight = reinterpret_cast<float*>(part + N * p.count);
  if (N * p.count >= (1LL << 31)) {
    set_error("bf_policy_loss: %lld rows of %lld logits are too many", (long long)N, (long long)V);
    return BF_ERANGE;
  }
  if (N > 0) {
    hipLaunchKernelGGL(policy_weights_kernel, dim3(1), dim3(WEIGHT_THREADS), 0, stream, a, weight);
    BF_LAUNCH_CHECK("policy_weights_kernel");
    const int threads = row_threads(V, elem);
    if (threads && N >= 256) {
      // as many workgroups as the device holds; each goes through its rows
      const int64_t most = 256 * (threads == 64 ? 16 : threads == 256 ? 6 : threads == 512 ? 2 : 1);
      const int64_t groups = N < most ? N : most;
      const int rc = with_elem(elem, [&](auto e) -> int {
        using E = decltype(e);
        auto run = [&](auto kernel) -> int {
          hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3((unsigned)threads), 0, stream,
                             static_cast<const E*>(logits), rows, a, weight, logp, static_cast<E*>(grad), sums);
          BF_LAUNCH_CHECK("policy_row_kernel");
          return BF_OK;
        };
        return threads == 64    ? run(policy_row_kernel<E, 64, 4>)
               : threads == 256 ? run(policy_row_kernel<E, 256, 4>)
               : threads == 512 ? run(policy_row_kernel<E, 512, 8>)
                                : run(policy_row_kernel<E, 1024, 16>);
      });
      if (rc != BF_OK) return rc;
      hipLaunchKernelGGL(policy_stats_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, sums, groups, kl_weight, stats);
      BF_LAUNCH_CHECK("policy_stats_kernel");
      return BF_OK;
    }
    const int rc = with_elem(elem, [&](auto e) -> int {
      using E = decltype(e);
      const E* x = static_cast<const E*>(logits);
      hipLaunchKernelGGL(loss_partial_kernel<E>, dim3((unsigned)(N * p.count)), dim3(LOSS_THREADS), 0, stream, x, rows,
                         tokens, token_bytes, a.mask, a.c, p.count, p.chunk, part);
      BF_LAUNCH_CHECK("loss_partial_kernel");
      hipLaunchKernelGGL(policy_rows_kernel<E>, dim3((unsigned)blocks), dim3(LOSS_THREADS), 0, stream, x, rows, a, part,
                         p.count, weight, logp, coef, sums);
      BF_LAUNCH_CHECK("policy_rows_kernel");
      if (grad) {
        hipLaunchKernelGGL(loss_grad_kernel<E>, dim3((unsigned)(N * p.count)), dim3(LOSS_THREADS), 0, stream, x, rows,
                           tokens, token_bytes, a.c, p.count, p.chunk, coef, static_cast<E*>(grad));
        BF_LAUNCH_CHECK("loss_grad_kernel");
      }
      return BF_OK;
    });
    if (rc != BF_OK) return rc;
  }
  hipLaunchKernelGGL(policy_stats_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, sums, blocks, kl_weight, stats);
  BF_LAUNCH_CHECK("policy_stats_kernel");
  return BF_OK;
}

// coef [N] float4, part [N * parts] float2, losses [pairs]
int64_t bf_preference_loss_workspace(int64_t N, int64_t V, int64_t pairs, int elem) {
  if (!elem_ok(elem) || N < 0 || V <= 0 || pairs < 0) return 0;
  return 4 * N + 2 * N * row_parts(N, V, elem).count + pairs;
}

int bf_preference_loss(const void* logits, int elem, int64_t N, int64_t V, int64_t ld, const void* tokens,
                       int token_bytes, const float* ref_logp, const int64_t* offsets, int64_t pairs, float beta,
                       float smoothing, float grad_scale, float* logp, float* rewards, float* loss, void* grad,
                       float* workspace, hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8),
             "bf_preference_loss: element type %d, token bytes %d", elem, token_bytes);
  BF_REQUIRE(N >= 0 && V > 0 && ld >= 0 && pairs >= 0, "bf_preference_loss: bad sizes");
  BF_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, "bf_preference_loss: label smoothing %g", smoothing);
  BF_REQUIRE(loss && (pairs == 0 || (offsets && rewards && workspace)), "bf_preference_loss: null pointer");
  BF_REQUIRE(N == 0 || (logits && tokens && ref_logp && logp && workspace), "bf_preference_loss: null pointer");
  if (!rows_fit(N, V) || pairs >= (1LL << 24)) {
    set_error("bf_preference_loss: %lld rows of %lld logits, %lld pairs: rows and pairs below 2^24, logits below 2^30",
              (long long)N, (long long)V, (long long)pairs);
    return BF_ERANGE;
  }
  const PreferenceArgs a{tokens, ref_logp, offsets, N, pairs, beta, smoothing, grad_scale, token_bytes};
  const LogitRows rows{N > 0 ? N : 1, 0, ld, V};
  const Parts p = row_parts(N, V, elem);
  const float c = 1.4426950408889634f;
  float4* coef = reinterpret_cast<float4*>(workspace);
  float2* part = reinterpret_cast<float2*>(coef + N);
  float* losses = reinterpret_cast<float*>(part + N * p.count);
  if (N * p.count >= (1LL << 31)) {
    set_error("bf_preference_loss: %lld rows of %lld logits are too many", (long long)N, (long long)V);
    return BF_ERANGE;
  }
  const int rc = with_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    const E* x = static_cast<const E*>(logits);
    if (N > 0) {
      hipLaunchKernelGGL(preference_clear_kernel, dim3((unsigned)ceil_div(N, 256)), dim3(256), 0, stream, N, logp, coef);
      BF_LAUNCH_CHECK("preference_clear_kernel");
      hipLaunchKernelGGL(loss_partial_kernel<E>, dim3((unsigned)(N * p.count)), dim3(LOSS_THREADS), 0, stream, x, rows,
                         tokens, token_bytes, nullptr, c, p.count, p.chunk, part);
      BF_LAUNCH_CHECK("loss_partial_kernel");
    }
    if (pairs > 0) {
      hipLaunchKernelGGL(preference_pairs_kernel<E>, dim3((unsigned)pairs), dim3(LOSS_THREADS), 0, stream, x, rows, a,
                         part, p.count, c, logp, coef, rewards, losses);
      BF_LAUNCH_CHECK("preference_pairs_kernel");
    }
    if (N > 0 && grad) {
      hipLaunchKernelGGL(loss_grad_kernel<E>, dim3((unsigned)(N * p.count)), dim3(LOSS_THREADS), 0, stream, x, rows,
                         tokens, token_bytes, c, p.count, p.chunk, coef, static_cast<E*>(grad));
      BF_LAUNCH_CHECK("loss_grad_kernel");
    }
    return BF_OK;
  });
  if (rc != BF_OK) return rc;
  hipLaunchKernelGGL(preference_loss_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, losses, pairs, loss);
  BF_LAUNCH_CHECK("preference_loss_kernel");
  return BF_OK;
}

}  // extern "C"
