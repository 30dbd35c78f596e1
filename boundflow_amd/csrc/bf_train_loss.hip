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
// A softmax is held as (M, s): the largest logit M, and s = sum of 2^(c (z - M)), c = log2(e) / temperature.
// The difference of two logits is exact or rounded by a share of itself, so rows of any magnitude
// (masks of -1e9 or of the type's lowest value, which fill a whole row now and then) keep the accuracy of
// their differences; a row of -inf alone has no distribution, and a NaN or +inf makes its row NaN.

#include "bf_train.h"

#include <cmath>
#include <type_traits>

namespace bf {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kFloor = -3.4028234663852886e38f;   // M of no logits: the lowest fp32, so that -inf - M is -inf

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// 2^(c (z - M))
__device__ __forceinline__ float term(float z, float c, float M) { return exp2_fast((z - M) * c); }

// (M, s) with N more logits
template <int N>
__device__ __forceinline__ void add_terms(float& M, float& s, const float (&z)[N], float c) {
  float m = M;
#pragma unroll
  for (int k = 0; k < N; ++k) m = fmaxf(m, z[k]);
  s *= term(M, c, m);
  M = m;
#pragma unroll
  for (int k = 0; k < N; ++k) s += term(z[k], c, m);
}

// The log-probability of a logit z.  The difference is not taken through base 2, where that of a mask's value, the
// type's lowest, would pass the largest fp32.
__device__ __forceinline__ float log_prob(float z, float inv_t, float M, float s) {
  return (z - M) * inv_t - log2_fast(s) * kLn2;
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

// The elements before a row's first whole 32-bit word: one where a row of 16-bit elements starts at an odd one (every other
// row of an odd vocabulary).  Vectors start behind it: 16-byte accesses off a word's boundary take half as long
// again (8192 rows of 50001 bf16 logits, policy loss: 413 us against 347 of 50002).
template <class T>
__device__ __forceinline__ int row_lead(const T* row) {
  return sizeof(T) == 2 ? (int)(reinterpret_cast<uintptr_t>(row) >> 1 & 1) : 0;
}

// a row that takes part: not masked, and its token not negative
__device__ __forceinline__ bool live_row(const uint8_t* mask, const void* tokens, int token_bytes, int64_t n) {
  const bool shown = mask == nullptr || mask[n];
  const int t = load_token(tokens, token_bytes, n);   // both loads under way together
  return shown & (t >= 0);
}

constexpr int LOSS_THREADS = 256, LOSS_WAVES = LOSS_THREADS / 64;

// (M, s) over a workgroup of WAVES waves, the same in every thread; `red` holds WAVES pairs and is
// written before the barrier that it has, and read after it.
template <int WAVES>
__device__ __forceinline__ float2 block_softmax(float M, float s, float c, float2* red) {
  float m = wave_max(M);
  s = wave_sum(s * term(M, c, m));
  if constexpr (WAVES == 1) return make_float2(m, s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  m = red[0].x;
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, red[w].x);
  s = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += red[w].y * term(red[w].x, c, m);
  return make_float2(m, s);
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

// The rows' weights: 1 / live rows, or with by_sequence 1 / (live rows of the sequence * sequences that have any).  Up to
// COUNT_GROUPS workgroups count a share of the rows (of the sequences) each; a row's weight is formed from the counts
// where it is needed.
constexpr int COUNT_GROUPS = 64, COUNT_HELD = 2048, COUNT_THREADS = 1024;

struct PolicyCounts {
  float* share;     // [COUNT_GROUPS]: live rows, or sequences that have any, of each workgroup
  float* live;      // [B], by_sequence: live rows
  int groups;
};

// Workgroup `group` of counts.groups; `held` (LDS) holds the counts of COUNT_HELD sequences at a time.  A thread has the
// flags of eight rows under way at once.
template <int THREADS>
__device__ __forceinline__ void policy_count(const PolicyArgs& a, const PolicyCounts& counts, int group, int* held,
                                             float* red) {
  constexpr int AT_ONCE = 8;
  const unsigned T = (unsigned)a.T;
  int total = 0;
  // the group's sequences, or with the rows taken as one, its rows
  const int64_t all = a.by_sequence ? a.B : a.B * a.T, each = (all + counts.groups - 1) / counts.groups;
  const int64_t from = min(group * each, all), to = min(from + each, all);
  for (int64_t b0 = from; b0 < to;) {
    const int64_t b1 = a.by_sequence ? min(b0 + COUNT_HELD, to) : to;
    const int64_t row0 = a.by_sequence ? b0 * a.T : b0;
    const unsigned rows = (unsigned)(a.by_sequence ? (b1 - b0) * a.T : b1 - b0);
    if (a.by_sequence) {
      for (int b = threadIdx.x; b < (int)(b1 - b0); b += THREADS) held[b] = 0;
      __syncthreads();
    }
    for (unsigned i0 = threadIdx.x; i0 < rows + threadIdx.x; i0 += AT_ONCE * THREADS) {
      bool in[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const unsigned i = i0 + u * THREADS;
        in[u] = i < rows && live_row(a.mask, a.tokens, a.token_bytes, row0 + i);
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (!a.by_sequence) {
          total += in[u];
          continue;
        }
        const unsigned b = min(i0 + u * THREADS, rows - 1) / T;
        const uint64_t found = __ballot(in[u]);
        const unsigned lo = __builtin_amdgcn_readfirstlane(b), hi = __builtin_amdgcn_readlane(b, 63);
        if (lo == hi) {   // a wave's 64 rows are mostly one sequence's
          if ((threadIdx.x & 63) == 0 && found) atomicAdd(&held[lo], __popcll(found));
        } else if (in[u]) {
          atomicAdd(&held[b], 1);
        }
      }
    }
    if (a.by_sequence) {
      __syncthreads();
      for (int b = threadIdx.x; b < (int)(b1 - b0); b += THREADS) {
        counts.live[b0 + b] = (float)held[b];
        total += held[b] ? 1 : 0;
      }
      __syncthreads();
    }
    b0 = b1;
  }
  // below 2^24 rows in all: exact
  const float share = block_sum<THREADS / 64>((float)total, red);
  if (threadIdx.x == 0) counts.share[group] = share;
}

__global__ __launch_bounds__(COUNT_THREADS) void policy_count_kernel(PolicyArgs a, PolicyCounts counts) {
  __shared__ int held[COUNT_HELD];
  __shared__ float red[COUNT_THREADS / 64];
  policy_count<COUNT_THREADS>(a, counts, blockIdx.x, held, red);
}

// The sum of the shares, by a whole wave.
__device__ __forceinline__ float count_sum(const PolicyCounts& counts) {
  const int lane = threadIdx.x & 63;
  return wave_sum(lane < counts.groups ? counts.share[lane] : 0.f);
}

// A live row's weight; sum: count_sum's
__device__ __forceinline__ float row_weight(const PolicyArgs& a, const PolicyCounts& counts, unsigned b, float sum) {
  return 1.f / (a.by_sequence ? counts.live[b] * sum : sum);
}

struct PolicyRow {
  float policy, kl, outside, g;
};

// A live row's terms and dL/dp_t, before its weight.
__device__ __forceinline__ PolicyRow policy_term(float logp, float old, float ref, bool has_ref, float A, float low,
                                                 float high, float kl_weight) {
  PolicyRow r;
  // Without an advantage there is no term, where the exponential overflows too (a NaN stays one).  Asked of the exponent,
  // beside the exponential: asked of the ratio, behind it, 4088 rows of 32000 bf16 logits took 104.3 us, so 103.6.
  const float ahead = logp - old, ratio = expf(ahead);
  const float plain = A == 0.f && ahead > 88.f ? 0.f : ratio * A, clipped = fminf(fmaxf(ratio, low), high) * A;
  const bool out = clipped < plain;   // the clipped side is the smaller: a constant, without a gradient
  r.policy = out ? -clipped : -plain;
  r.outside = out ? 1.f : 0.f;
  r.g = out ? 0.f : -plain;
  r.kl = 0.f;
  if (has_ref) {
    const float apart = ref - logp, e = expm1f(apart);
    r.kl = e - apart;
    if (kl_weight != 0.f) r.g -= kl_weight * e;   // 0 * inf would be NaN where the exponential overflows
  }
  return r;
}

// stats: loss, policy term, KL, clipped share
__device__ __forceinline__ void write_stats(float policy, float kl, float outside, float kl_weight, float* stats) {
  stats[0] = kl_weight != 0.f ? policy + kl_weight * kl : policy;
  stats[1] = policy;
  stats[2] = kl;
  stats[3] = outside;
}

// Sums of three values over a workgroup, in a fixed order, in the first thread.
template <int WAVES>
__device__ __forceinline__ float3 block_sum3(float x, float y, float z, float4* red) {
  x = wave_sum(x);
  y = wave_sum(y);
  z = wave_sum(z);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float4(x, y, z, 0.f);
  __syncthreads();
  float3 r = make_float3(0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    r.x += red[w].x;
    r.y += red[w].y;
    r.z += red[w].z;
  }
  return r;
}

constexpr int STATS_THREADS = 512;

__global__ __launch_bounds__(STATS_THREADS) void policy_stats_kernel(const float4* __restrict__ sums, int64_t count,
                                                                     float kl_weight, float* __restrict__ stats) {
  __shared__ float4 red[STATS_THREADS / 64];
  float policy = 0.f, kl = 0.f, outside = 0.f;
  for (int64_t i = threadIdx.x; i < count; i += STATS_THREADS) {
    const float4 x = sums[i];
    policy += x.x;
    kl += x.y;
    outside += x.z;
  }
  const float3 r = block_sum3<STATS_THREADS / 64>(policy, kl, outside, red);
  if (threadIdx.x == 0) write_stats(r.x, r.y, r.z, kl_weight, stats);
}

// as_floats keeps the compiler from holding on to the fp32 values of a
// row between its two uses, which would take twice the registers that the row does.
template <class T, int VEC>
__device__ __forceinline__ void as_floats(Words& w, float (&z)[VEC]) {
  asm volatile("" : "+v"(w));
  Pack<T, VEC> x;
  __builtin_memcpy(&x, &w, sizeof(x));
#pragma unroll
  for (int e = 0; e < VEC; ++e) z[e] = (float)x.v[e];
}

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform(float x) { return __int_as_float(uniform(__float_as_int(x))); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return ((int64_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x);
}

// How a row of V elements lies in vectors: `lead` elements, `vecs` vectors of VEC, and the rest; those outside of the
// vectors, VEC at most, are a thread's each.
template <class T>
struct RowShape {
  static constexpr int VEC = 16 / sizeof(T);
  int lead, vecs;
  __device__ __forceinline__ RowShape(const T* row, int V) : lead(uniform(row_lead(row))), vecs((V - lead) / VEC) {}
  // the thread's element outside of the vectors, V or more if it has none
  __device__ __forceinline__ int loose() const {
    return (int)threadIdx.x < lead ? (int)threadIdx.x : vecs * VEC + (int)threadIdx.x;
  }
  // the thread that holds element t, of THREADS
  template <int THREADS>
  __device__ __forceinline__ int holder(int t) const {
    const int v = (t - lead) / VEC;
    return t < lead ? t : v < vecs ? v % THREADS : t - vecs * VEC;
  }
};

// A workgroup's row in registers: vector k * THREADS + tid of 16 bytes in x[k], and the thread's loose element in `rest`.
// The first FULL steps are whole in every row that the kernel takes.
template <class T, int THREADS, int NV, int FULL>
struct HeldRow {
  static constexpr int VEC = 16 / sizeof(T), WAVES = THREADS / 64;
  using Shape = RowShape<T>;
  Words x[NV];
  float rest;

  static __device__ __forceinline__ bool has(int k, int vecs) {
    return k < FULL || k * THREADS + (int)threadIdx.x < vecs;
  }
  // Loads are never skipped: with a branch around them the compiler waits for every access at every turn.  Threads
  // past the row's end load its last vector (element) again, and of a row that is not to be read (`read` 0) every
  // thread loads the first, one cache line.
  __device__ __forceinline__ void load(int k, const T* row, int read, Shape f) {
    const int lane = k < FULL ? (int)threadIdx.x : min((int)threadIdx.x, f.vecs - 1 - k * THREADS);
    // a step that begins past the row's end lies before it by as much: lane is negative there
    const char* at = reinterpret_cast<const char*>(row + f.lead) + read * (k * THREADS * 16);
    __builtin_memcpy(&x[k], k < FULL ? at + (uint32_t)(read * lane * 16) : at + read * lane * 16, 16);
  }
  __device__ __forceinline__ void load_rest(const T* row, int read, Shape f, int V) {
    rest = (float)row[(uint32_t)(read * min(f.loose(), V - 1))];
  }
  // (M, s) of the thread with vector k, or with its loose element
  __device__ __forceinline__ void add(int k, Shape f, float c, float& M, float& s) {
    float z[VEC];
    as_floats<T>(x[k], z);
    if (has(k, f.vecs)) add_terms(M, s, z, c);
  }
  __device__ __forceinline__ void add_rest(Shape f, int V, float c, float& M, float& s) {
    const float one[1] = {rest};
    if (f.loose() < V) add_terms(M, s, one, c);
  }
  // q 2^(c (z - M)) of vector k; zeros where `keep` is 0, whatever the vector holds (else it is ~0)
  __device__ __forceinline__ void store(int k, T* out, Shape f, float c, float M, float q, uint32_t keep) {
    float y[VEC];
    as_floats<T>(x[k], y);
    Pack<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = (T)(term(y[e], c, M) * q);
    Words w;
    __builtin_memcpy(&w, &r, 16);
    w &= keep;
    if (has(k, f.vecs))
      __builtin_memcpy(reinterpret_cast<char*>(out + f.lead) + k * THREADS * 16 + threadIdx.x * 16u, &w, 16);
  }
};

// A row of zeros.
template <class T, int THREADS>
__device__ __forceinline__ void clear_row(T* out, int V) {
  const RowShape<T> f(out, V);
  if (f.loose() < V) out[f.loose()] = (T)0.f;
  const Words zero = zero_words();
  for (int v = threadIdx.x; v < f.vecs; v += THREADS)
    __builtin_memcpy(reinterpret_cast<char*>(out + f.lead) + v * 16, &zero, 16);
}

// The loop over a row's vectors: vector k's gradient is formed and stored (GRAD), the same vector of the next row
// is loaded into its registers, and a vector that was loaded LAG steps before is added to the next row's (M, s).
template <bool GRAD, class T, int THREADS, int NV, int FULL>
__device__ __forceinline__ void row_step(HeldRow<T, THREADS, NV, FULL>& h, T* out, RowShape<T> f, const T* next_row,
                                         int next_live, RowShape<T> next, int V, float c, float Mr, float q,
                                         uint32_t keep, float& M, float& s) {
  constexpr int LAG = (NV + 1) / 2;
  if (GRAD && f.loose() < V) out[f.loose()] = (T)(keep ? term(h.rest, c, Mr) * q : 0.f);
  h.load_rest(next_row, next_live, next, V);
#pragma unroll
  for (int k = 0; k < NV + LAG; ++k) {
    if (k < NV) {
      if (GRAD) h.store(k, out, f, c, Mr, q, keep);
      h.load(k, next_row, next_live, next);
    }
    if (k >= LAG) h.add(k - LAG, next, c, M, s);
    // loads stay behind the stores of their registers' old contents: the row is held once
    __builtin_amdgcn_sched_barrier(0);
  }
  h.add_rest(next, V, c, M, s);
}

// A row's scalars, fetched a row before they are needed.
struct PolicyScalars {
  int n, t, live;
  float old, ref, A, w;
};

__device__ __forceinline__ PolicyScalars policy_scalars(const PolicyArgs& a, const PolicyCounts& counts, int n, int N) {
  PolicyScalars r;
  r.n = n;
  r.live = 0;
  r.t = -1;
  r.old = r.ref = r.A = r.w = 0.f;
  if (n < N) {
    const unsigned b = (unsigned)n / (unsigned)a.T;
    r.t = load_token(a.tokens, a.token_bytes, n);
    r.live = (a.mask == nullptr || a.mask[n]) & (r.t >= 0);
    r.old = a.old_logp[n];
    r.ref = a.ref_logp ? a.ref_logp[n] : 0.f;
    r.A = a.advantages[b * a.adv_b + (n - b * (unsigned)a.T) * a.adv_t];
    r.w = a.by_sequence ? counts.live[b] : 1.f;   // to be multiplied by the sum, and inverted
  }
  return r;
}

// The same in scalar registers, once they have arrived.
__device__ __forceinline__ PolicyScalars uniform(const PolicyScalars& x) {
  return {uniform(x.n), uniform(x.t), uniform(x.live), uniform(x.old), uniform(x.ref), uniform(x.A), uniform(x.w)};
}

// The whole loss of a row in one pass over its logits.  A workgroup holds a row in registers: its softmax is
// there when the row before has been written, the row's term follows, and row_step writes the gradient
// while it reads the next row and sums its softmax.  Loads, stores and exponentials are under way together, and
// what is left between two rows is LAG vectors, a reduction and the term.
//
// Each turn of the grid takes as many rows as it has workgroups, the workgroups moved on by `stride` from
// turn to turn: the rows that padding masks stand at the same places of every sequence, and without it a
// workgroup would meet them at every turn or at none.
//
// Bound by memory: 8184 rows of 128000 bf16 logits, a fifth of them padding, 755 us for 3.76 GB = 5.0 TB/s, 4088 of
// 32000 in 97 us = 4.8 TB/s (a large copy: 4.65).  Reading every row twice took 1192 and 166 us; held rows whose sums
// waited for the whole next row 1095; with branches around the accesses (a wait for everything before each) 1040.
template <bool GRAD, class T, int THREADS, int NV, int FULL>
__global__ __launch_bounds__(THREADS) void policy_row_kernel(const T* __restrict__ logits, LogitRows rows, PolicyArgs a,
                                                             PolicyCounts counts, float* __restrict__ logp,
                                                             T* __restrict__ grad,
                                                             float4* __restrict__ sums, unsigned stride) {
  using Held = HeldRow<T, THREADS, NV, FULL>;
  __shared__ float2 red[2][Held::WAVES];
  const int N = (int)(a.B * a.T), V = (int)rows.V;
  const float c = a.c, count = count_sum(counts);
  unsigned place = blockIdx.x, first = 0;   // of the workgroup in the turn, and the turn's first row
  const auto next_turn = [&] {
    first += gridDim.x;
    place += stride;
    if (place >= gridDim.x) place -= gridDim.x;
    return (int)(first + place);
  };
  Held h;
  // the first row from x on that takes part; those that do not get their zeros here.  The loop below goes from one
  // such row to the next, in one piece: a branch in it that leaves the row's registers alone would have the
  // compiler keep two sets of them.
  const auto settled = [&](PolicyScalars x) {
    while (x.n < N && !x.live) {
      const PolicyScalars after = policy_scalars(a, counts, next_turn(), N);
      if (threadIdx.x == 0) logp[x.n] = 0.f;
      if (GRAD) clear_row<T, THREADS>(grad + (int64_t)x.n * V, V);
      x = uniform(after);
    }
    return x;
  };
  PolicyScalars here = settled(uniform(policy_scalars(a, counts, (int)place, N)));
  PolicyScalars after = policy_scalars(a, counts, next_turn(), N);
  const T* row = logits + (here.n < N ? uniform(rows.offset(here.n)) : 0);
  float M = kFloor, s = 0.f;   // of the thread, for the row that it holds
  RowShape<T> shape(row, V);
  if (here.n < N) row_step<false>(h, grad, shape, row, 1, shape, V, c, 0.f, 0.f, 0u, M, s);
  float zt = uniform(here.n < N && here.t < V ? (float)row[here.t] : 0.f);
  float policy = 0.f, kl = 0.f, outside = 0.f;
  // two buffers, by turns: before one is filled again, every wave has passed the barrier of the row in between, and
  // so has read it
  int buf = 0;
  while (here.n < N) {
    const PolicyScalars then = settled(uniform(after));
    after = policy_scalars(a, counts, next_turn(), N);
    const T* next_row = logits + (then.n < N ? uniform(rows.offset(then.n)) : 0);
    const float zt_next = then.live && then.t < V ? (float)next_row[then.t] : 0.f;
    const float2 soft = block_softmax<Held::WAVES>(M, s, c, red[buf]);
    buf ^= 1;
    // the same in every thread, and in scalar registers for the loop
    const float Mr = uniform(soft.x);
    const float lp = here.t < V ? log_prob(zt, a.inv_t, Mr, soft.y) : __int_as_float(0x7fc00000);
    const PolicyRow r = policy_term(lp, here.old, here.ref, a.ref_logp != nullptr, here.A, a.low, a.high, a.kl_weight);
    const float w = 1.f / (here.w * count);
    policy += w * r.policy;
    kl += w * r.kl;
    outside += w * r.outside;
    const float g = w * r.g * a.inv_t * a.grad_scale, q = uniform(-g / soft.y);
    const uint32_t keep = uniform(g == 0.f ? 0 : -1);
    if (threadIdx.x == 0) logp[here.n] = lp;
    T* out = grad + (int64_t)here.n * V;
    M = kFloor;
    s = 0.f;
    const RowShape<T> next_shape(next_row, V);
    row_step<GRAD>(h, out, shape, next_row, then.live, next_shape, V, c, Mr, q, keep, M, s);
    // the token's own element, by the thread that wrote its vector
    if (GRAD && keep && here.t < V && (int)threadIdx.x == shape.template holder<THREADS>(here.t))
      out[here.t] = (T)(term(zt, c, Mr) * q + g);
    shape = next_shape;
    here = then;
    zt = uniform(zt_next);
  }
  if (threadIdx.x == 0) sums[blockIdx.x] = make_float4(policy, kl, outside, 0.f);
}

// ---------------------------------------------------------------------------
// Rows in parts: few rows, so that a workgroup each would leave the device idle, or rows that no workgroup
// holds.  One launch sums the parts' softmaxes, the next forms the rows' from them and writes the gradient.
// 45 rows of 50001 fp32 logits: 4.5 + 5.8 + 5.2 us, the latency of three launches.  The preference loss takes this way
// for batches of any size, since a row's gradient waits for the sums of its pair: 9001 rows of 50001 bf16 logits 190 us
// (4.8 TB/s) + 12 + 346 us (5.2 TB/s).  Ordering the pairs so that the second reading meets the rows in the
// memory-side cache gained nothing (a third of the traffic from there, the same time: what the XCDs exchange
// with the memory side is the limit).

// (M, s) of a part of a row.  Workgroup = (row, part of `chunk` elements).  The policy loss, whose workgroups have
// LOSS_THREADS, launches one more, which counts; the preference loss's short rows, a wave each, do without the LDS of
// the counts, which would leave a CU 19 of 32 such workgroups (65536 rows of 500 bf16 logits 70 us against 80).
template <class T, int TH>
__global__ __launch_bounds__(TH) void loss_partial_kernel(const T* __restrict__ logits, LogitRows rows, PolicyArgs a,
                                                          int64_t N, int parts, int64_t chunk,
                                                          float2* __restrict__ part, PolicyCounts counts) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float2 red[TH / 64];
  const int64_t n = blockIdx.x / (unsigned)parts;
  if constexpr (TH == LOSS_THREADS) {
    if (n == N) {
      __shared__ int held[COUNT_HELD];
      __shared__ float sum[TH / 64];
      policy_count<TH>(a, counts, 0, held, sum);
      return;
    }
  }
  const int q = (int)(blockIdx.x % (unsigned)parts);
  if (!live_row(a.mask, a.tokens, a.token_bytes, n)) return;
  const T* row = logits + rows.offset(n);
  const int64_t from = q * chunk, to = min(from + chunk, rows.V);
  float M = kFloor, s = 0.f;
  const int lead = row_lead(row + from);   // chunks are whole vectors: the same in all of them
  if (lead && threadIdx.x == TH - 1) {
    const float one[1] = {(float)row[from]};
    add_terms(M, s, one, a.c);
  }
  int64_t d = from + lead + threadIdx.x * VEC;
  for (; d + 3 * TH * VEC + VEC <= to; d += 4 * TH * VEC) {   // four loads under way
    Pack<T, VEC> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = load_pack<T, VEC>(row + d + u * TH * VEC);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float z[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) z[k] = (float)x[u].v[k];
      add_terms(M, s, z, a.c);
    }
  }
  for (; d < to; d += TH * VEC) {
    float z[VEC];
    if (d + VEC <= to) {
      const Pack<T, VEC> x = load_pack<T, VEC>(row + d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) z[k] = (float)x.v[k];
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) z[k] = d + k < to ? (float)row[d + k] : -__builtin_inff();
    }
    add_terms(M, s, z, a.c);
  }
  const float2 x = block_softmax<TH / 64>(M, s, a.c, red);
  if (threadIdx.x == 0) part[blockIdx.x] = x;
}

// A row's softmax from its parts, by 16 lanes or (ONE part) by each lane for itself, the same in each of them.
template <bool ONE>
__device__ __forceinline__ float2 row_softmax(const float2* part, int64_t n, int parts, float c) {
  if (ONE) return part[n];
  float M = kFloor, s = 0.f;
  for (int q = threadIdx.x & 15; q < parts; q += 16) {
    const float2 x = part[n * parts + q];
    const float m = fmaxf(M, x.x);
    s = s * term(M, c, m) + x.y * term(x.x, c, m);
    M = m;
  }
  const float m = row16_max(M);
  return make_float2(m, row16_sum(s * term(M, c, m)));
}

// The log-probability of a live row's token; one past the vocabulary shows as NaN.
template <class T>
__device__ __forceinline__ float token_logp(const T* logits, const LogitRows& rows, int64_t n, int t, float2 soft,
                                            float inv_t) {
  return (int64_t)t < rows.V ? log_prob((float)logits[rows.offset(n) + t], inv_t, soft.x, soft.y)
                             : __int_as_float(0x7fc00000);
}

// What the gradient of a row needs: dlogits = 2^(c (z - M)) q (+ g at the token).  A row with g = 0 gets zeros and
// its logits are not read.
__device__ __forceinline__ float4 row_gradient(float2 soft, float g) {
  return make_float4(soft.x, -g / soft.y, g, 0.f);
}

// The gradient of elements [from, to) of a row, by a workgroup.
template <int TH, class T>
__device__ __forceinline__ void write_row_gradient(const T* row, T* out, int64_t from, int64_t to, int64_t t, float c,
                                                   float4 f) {
  constexpr int VEC = 16 / sizeof(T);
  const bool read = f.z != 0.f;
  const int lead = row_lead(read ? row + from : out + from);
  if (lead && threadIdx.x == TH - 1)
    out[from] = (T)(read ? term((float)row[from], c, f.x) * f.y + (t == from ? f.z : 0.f) : 0.f);
  for (int64_t d = from + lead + threadIdx.x * VEC; d < to; d += TH * VEC) {
    if (d + VEC <= to) {
      if (read) {
        Pack<T, VEC> x = load_pack<T, VEC>(row + d);
        float y[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = term((float)x.v[k], c, f.x) * f.y;
        if (t >= d && t < d + VEC)
#pragma unroll
          for (int k = 0; k < VEC; ++k) y[k] += t == d + k ? f.z : 0.f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) x.v[k] = (T)y[k];
        store_pack(out + d, x);
      } else {
        const Words zero = zero_words();
        __builtin_memcpy(out + d, &zero, 16);
      }
    } else {
      for (int64_t e = d; e < to; ++e)
        out[e] = (T)(read ? term((float)row[e], c, f.x) * f.y + (t == e ? f.z : 0.f) : 0.f);
    }
  }
}

// A live row of the policy loss from its parts: log-probability, terms, and the gradient's coefficients.
template <bool ONE, class T>
__device__ __forceinline__ PolicyRow policy_part_row(const T* logits, const LogitRows& rows, const PolicyArgs& a,
                                                     const float2* part, int parts, int64_t n, int t, float* lp,
                                                     float2* soft) {
  const int64_t b = (unsigned)n / (unsigned)a.T;
  *soft = row_softmax<ONE>(part, n, parts, a.c);
  *lp = token_logp(logits, rows, n, t, *soft, a.inv_t);
  return policy_term(*lp, a.old_logp[n], a.ref_logp ? a.ref_logp[n] : 0.f, a.ref_logp != nullptr,
                     a.advantages[b * a.adv_b + (n - b * a.T) * a.adv_t], a.low, a.high, a.kl_weight);
}

// Workgroup = (row, part): its gradient; the last one: every row's log-probability, and the sums.
template <bool ONE, class T>
__global__ __launch_bounds__(LOSS_THREADS) void policy_part_kernel(const T* __restrict__ logits, LogitRows rows,
                                                                   PolicyArgs a, int64_t N, int parts, int64_t chunk,
                                                                   const float2* __restrict__ part, PolicyCounts counts,
                                                                   float* __restrict__ logp, float* __restrict__ stats,
                                                                   T* __restrict__ grad) {
  const float count = count_sum(counts);
  if (blockIdx.x == gridDim.x - 1) {
    constexpr int LANES = ONE ? 1 : 16, ROWS = LOSS_THREADS / LANES;   // rows at a time, and lanes of a row
    __shared__ float4 red[LOSS_WAVES];
    float policy = 0.f, kl = 0.f, outside = 0.f;
    for (int64_t n0 = 0; n0 < N; n0 += ROWS) {
      const int64_t n = n0 + threadIdx.x / LANES;
      const bool first = threadIdx.x % LANES == 0;
      if (n >= N) continue;   // 16 lanes together
      float lp = 0.f;
      if (live_row(a.mask, a.tokens, a.token_bytes, n)) {
        float2 soft;
        const PolicyRow r = policy_part_row<ONE>(logits, rows, a, part, parts, n, load_token(a.tokens, a.token_bytes, n),
                                                 &lp, &soft);
        const float w = row_weight(a, counts, (unsigned)n / (unsigned)a.T, count);
        if (first) {
          policy += w * r.policy;
          kl += w * r.kl;
          outside += w * r.outside;
        }
      }
      if (first) logp[n] = lp;
    }
    const float3 r = block_sum3<LOSS_WAVES>(policy, kl, outside, red);
    if (threadIdx.x == 0) write_stats(r.x, r.y, r.z, a.kl_weight, stats);
    return;
  }
  const int64_t n = blockIdx.x / (unsigned)parts;
  const int q = (int)(blockIdx.x % (unsigned)parts);
  const int t = load_token(a.tokens, a.token_bytes, n);
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live_row(a.mask, a.tokens, a.token_bytes, n)) {
    float lp;
    float2 soft;
    const PolicyRow r = policy_part_row<ONE>(logits, rows, a, part, parts, n, t, &lp, &soft);
    f = row_gradient(soft, row_weight(a, counts, (unsigned)n / (unsigned)a.T, count) * r.g * a.inv_t * a.grad_scale);
  }
  write_row_gradient<LOSS_THREADS>(logits + rows.offset(n), grad + n * rows.V, q * chunk, min(q * chunk + chunk, rows.V), (int64_t)t,
                     a.c, f);
}

// ---------------------------------------------------------------------------
// Short rows (a controller's few actions, a small vocabulary): LANES lanes a row, 1 or 16, which go over its
// elements twice (the second time from the caches).  ALONE: one workgroup does everything, counts and sums included, in
// one launch.
constexpr int SHORT_ONE = 16, SHORT_MOST = 512;   // the longest rows of one lane, and of sixteen

template <bool ALONE, int LANES, class T>
__global__ __launch_bounds__(ALONE ? COUNT_THREADS : LOSS_THREADS) void policy_short_kernel(
    const T* __restrict__ logits, LogitRows rows, PolicyArgs a, PolicyCounts counts, float* __restrict__ logp,
    float* __restrict__ stats, T* __restrict__ grad, float4* __restrict__ sums) {
  constexpr int THREADS = ALONE ? COUNT_THREADS : LOSS_THREADS, WAVES = THREADS / 64, VEC = LANES == 1 ? 1 : 16 / sizeof(T);
  __shared__ float4 red[WAVES];
  if constexpr (ALONE) {
    __shared__ int held[COUNT_HELD];
    __shared__ float sum[WAVES];
    policy_count<THREADS>(a, counts, 0, held, sum);
    __syncthreads();   // the counts are read by other threads of the workgroup than wrote them
  }
  const float count = count_sum(counts);
  const int N = (int)(a.B * a.T), V = (int)rows.V, lane = threadIdx.x % LANES;
  const float c = a.c;
  float policy = 0.f, kl = 0.f, outside = 0.f;
  for (int n = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; n < N; n += gridDim.x * (THREADS / LANES)) {
    const T* row = logits + rows.offset(n);
    T* out = grad + (int64_t)n * V;
    const int t = load_token(a.tokens, a.token_bytes, n);
    float lp = 0.f, g = 0.f, q = 0.f, M = kFloor, s = 0.f;
    if (live_row(a.mask, a.tokens, a.token_bytes, n)) {   // the same in a row's lanes
      const unsigned b = (unsigned)n / (unsigned)a.T;
      const float old = a.old_logp[n], ref = a.ref_logp ? a.ref_logp[n] : 0.f, w = row_weight(a, counts, b, count);
      const float A = a.advantages[b * a.adv_b + (n - b * (unsigned)a.T) * a.adv_t];
      const float zt = t < V ? (float)row[t] : 0.f;
      for (int d = lane * VEC; d < V; d += LANES * VEC) {
        float z[VEC];
        if (d + VEC <= V) {
          const Pack<T, VEC> x = load_pack<T, VEC>(row + d);
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[e] = (float)x.v[e];
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[e] = d + e < V ? (float)row[d + e] : -__builtin_inff();
        }
        add_terms(M, s, z, c);
      }
      if (LANES > 1) {
        const float m = row16_max(M);
        s = row16_sum(s * term(M, c, m));
        M = m;
      }
      lp = t < V ? log_prob(zt, a.inv_t, M, s) : __int_as_float(0x7fc00000);
      const PolicyRow r = policy_term(lp, old, ref, a.ref_logp != nullptr, A, a.low, a.high, a.kl_weight);
      if (lane == 0) {
        policy += w * r.policy;
        kl += w * r.kl;
        outside += w * r.outside;
      }
      g = w * r.g * a.inv_t * a.grad_scale;
      q = -g / s;
    }
    if (lane == 0) logp[n] = lp;
    if (grad)
      for (int d = lane * VEC; d < V; d += LANES * VEC) {
        if (d + VEC <= V) {
          Pack<T, VEC> x;
          if (g != 0.f) x = load_pack<T, VEC>(row + d);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            x.v[e] = (T)(g != 0.f ? term((float)x.v[e], c, M) * q + (t == d + e ? g : 0.f) : 0.f);
          store_pack(out + d, x);
        } else {
          for (int e = d; e < V; ++e) out[e] = (T)(g != 0.f ? term((float)row[e], c, M) * q + (t == e ? g : 0.f) : 0.f);
        }
      }
  }
  const float3 r = block_sum3<WAVES>(policy, kl, outside, red);
  if (threadIdx.x == 0) {
    if (ALONE) write_stats(r.x, r.y, r.z, a.kl_weight, stats);
    else sums[blockIdx.x] = make_float4(r.x, r.y, r.z, 0.f);
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

// Rows [from, to) of response k.  Offsets are data: whatever they hold, the rows are the batch's.
__device__ __forceinline__ int2 response_rows(const PreferenceArgs& a, int64_t k) {
  const int64_t from = min(max(a.offsets[k], (int64_t)0), a.N);
  return make_int2((int)from, (int)min(max(a.offsets[k + 1], from), a.N));
}

// The preference loss gives a row of up to this many vectors a lane to one wave instead of four: 65536 rows of 500 bf16
// logits 70 us against 154 (what four waves cost is the start of their workgroups), of 2000 177 against 188; from twice
// that on the four waves are ahead, 4000 in 305 us against 332.
constexpr int WAVE_VECTORS = 4;

constexpr int PAIR_THREADS = 1024, PAIR_WAVES = PAIR_THREADS / 64;
constexpr int64_t PAIR_GROUPS = 1 << 21;   // workgroups of a launch, one more beside them

// One workgroup per pair (of more than PAIR_GROUPS pairs, several one after another): the rows' log-probabilities,
// the responses' sums, the pair's loss, and the rows' gradient coefficients; one more clears the rows of no response.
template <bool ONE, class T>
__global__ __launch_bounds__(PAIR_THREADS) void preference_pairs_kernel(
    const T* __restrict__ logits, LogitRows rows, PreferenceArgs a, const float2* __restrict__ part, int parts, float c,
    float* __restrict__ logp, float4* __restrict__ coef, float* __restrict__ rewards, float* __restrict__ losses) {
  constexpr int LANES = ONE ? 1 : 16, ROWS = PAIR_THREADS / LANES;
  __shared__ float red[PAIR_WAVES];
  const int lane = threadIdx.x % LANES, groups = (int)gridDim.x - 1;
  if ((int)blockIdx.x == groups) {
    const int from = a.pairs ? response_rows(a, 0).x : (int)a.N;
    const int to = a.pairs ? response_rows(a, 2 * a.pairs - 1).y : (int)a.N;
    const int outside = from + (int)a.N - to;
    for (int i = threadIdx.x; i < outside; i += PAIR_THREADS) {
      const int n = i < from ? i : i - from + to;
      logp[n] = 0.f;
      coef[n] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  for (int64_t pair = blockIdx.x; pair < a.pairs; pair += groups) {
    float sum[2];
    int2 of[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      of[side] = response_rows(a, pair + side * a.pairs);
      float s = 0.f;
      for (int n = of[side].x + threadIdx.x / LANES; n < of[side].y; n += ROWS) {
        const int t = load_token(a.tokens, a.token_bytes, n);
        const float ref = a.ref_logp[n];
        float lp = 0.f;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);   // s of the row in y, until the pair's g is known
        if (t >= 0) {
          const float2 soft = row_softmax<ONE>(part, n, parts, c);
          lp = token_logp(logits, rows, n, t, soft, 1.f);
          if (lane == 0) s += lp - ref;
          f = make_float4(soft.x, soft.y, 1.f, 0.f);
        }
        if (lane == 0) {
          logp[n] = lp;
          coef[n] = f;
        }
      }
      sum[side] = block_sum<PAIR_WAVES>(s, red);
    }
    const float h = a.beta * sum[0] - a.beta * sum[1];
    const float dh = -((1.f - a.smoothing) * sigmoid(-h) - a.smoothing * sigmoid(h));
    if (threadIdx.x == 0) {
      rewards[pair] = a.beta * sum[0];
      rewards[pair + a.pairs] = a.beta * sum[1];
      // A term of weight 0 is not there: a response at -inf makes h infinite, and 0 * inf would be NaN.
      const float good = a.smoothing < 1.f ? (1.f - a.smoothing) * log_sigmoid(h) : 0.f;
      const float bad = a.smoothing > 0.f ? a.smoothing * log_sigmoid(-h) : 0.f;
      losses[pair] = -(good + bad);
    }
    const float g = dh * a.beta * a.grad_scale / (float)a.pairs;
    if (lane == 0)
#pragma unroll
      for (int side = 0; side < 2; ++side)
        for (int n = of[side].x + threadIdx.x / LANES; n < of[side].y; n += ROWS) {
          const float4 f = coef[n];   // written by this thread above
          if (f.z != 0.f) coef[n] = row_gradient(make_float2(f.x, f.y), side ? -g : g);
        }
  }
}

// Workgroup = (row, part): its gradient from the row's coefficients; the last one sums the pairs' losses.
template <class T, int TH>
__global__ __launch_bounds__(TH) void preference_grad_kernel(const T* __restrict__ logits, LogitRows rows,
                                                             PreferenceArgs a, int parts, int64_t chunk, float c,
                                                             const float4* __restrict__ coef,
                                                             const float* __restrict__ losses, float* __restrict__ loss,
                                                             T* __restrict__ grad) {
  if (blockIdx.x == gridDim.x - 1) {
    __shared__ float red[TH / 64];
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.pairs; i += TH) s += losses[i];
    s = block_sum<TH / 64>(s, red);
    if (threadIdx.x == 0) *loss = a.pairs ? s / (float)a.pairs : 0.f;
    return;
  }
  const int64_t n = blockIdx.x / (unsigned)parts;
  const int q = (int)(blockIdx.x % (unsigned)parts);
  write_row_gradient<TH>(logits + rows.offset(n), grad + n * rows.V, q * chunk, min(q * chunk + chunk, rows.V),
                     (int64_t)load_token(a.tokens, a.token_bytes, n), c, coef[n]);
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

// The row kernel's workgroup for rows of `vecs` whole vectors, handed to f as (threads, vectors a thread, steps that
// are whole in every such row) at compile time; 0 where no workgroup holds a row (131080 16-bit or 65540 fp32
// logits and more) or a row has no whole vector.
template <class F>
static int with_row_group(int64_t vecs, F f) {
  using std::integral_constant;
#define BF_ROW_GROUP(threads, nv, least) \
  if (vecs <= (threads) * (nv))          \
  return f(integral_constant<int, threads>(), integral_constant<int, nv>(), integral_constant<int, (least) / (threads)>())
  if (vecs < 1) return 0;
  BF_ROW_GROUP(64, 1, 0);
  BF_ROW_GROUP(64, 2, 64);
  BF_ROW_GROUP(64, 4, 128);
  BF_ROW_GROUP(256, 2, 256);
  BF_ROW_GROUP(256, 4, 512);
  BF_ROW_GROUP(512, 3, 1024);
  BF_ROW_GROUP(512, 4, 1536);
  BF_ROW_GROUP(512, 6, 2048);
  BF_ROW_GROUP(512, 8, 3072);
  BF_ROW_GROUP(1024, 6, 4096);
  BF_ROW_GROUP(1024, 8, 6144);
  BF_ROW_GROUP(1024, 10, 8192);
  BF_ROW_GROUP(1024, 12, 10240);
  BF_ROW_GROUP(1024, 14, 12288);
  BF_ROW_GROUP(1024, 16, 14336);
#undef BF_ROW_GROUP
  return 0;
}

// Workgroups whose sums are kept.
constexpr int64_t SUM_GROUPS = 4096;

// Short rows of the policy loss, and batches of them that one workgroup takes in four turns at most: a launch, and the
// gap before it, costs as much as two.
static bool short_rows(int64_t V, int elem) { return V <= (elem == TE_F32 ? SHORT_MOST / 2 : SHORT_MOST); }
static int short_lanes(int64_t V) { return V <= SHORT_ONE ? 1 : 16; }
static bool one_group(int64_t N, int64_t V, int elem) {
  return N == 0 || (short_rows(V, elem) && N * short_lanes(V) <= 4 * COUNT_THREADS);
}

// The longest launches have a workgroup a row and one more (rows in parts are few); counts of rows stay exact in fp32.
static bool rows_fit(int64_t N, int64_t V) { return V < (1LL << 30) && launch_fits(N + 1, LOSS_THREADS); }

}  // namespace bf

using namespace bf;

extern "C" {

// sums of the workgroups (row kernel, short rows), and part [N * parts] float2 (rows in parts), neither where one
// workgroup does everything; the counts' shares, and live rows [B]
int64_t bf_policy_loss_workspace(int64_t B, int64_t T, int64_t V, int elem) {
  if (!elem_ok(elem) || B < 0 || T < 0 || V <= 0 || B >= (1LL << 24) || T >= (1LL << 24) || !rows_fit(B * T, V)) return 0;
  const int64_t sums = one_group(B * T, V, elem) ? 0 : 4 * SUM_GROUPS + 2 * B * T * row_parts(B * T, V, elem).count;
  return sums + COUNT_GROUPS + B;
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
  BF_REQUIRE(stats && workspace, "bf_policy_loss: null pointer");
  if (B >= (1LL << 24) || T >= (1LL << 24) || !rows_fit(B * T, V)) {
    set_error("bf_policy_loss: %lld x %lld rows of %lld logits: rows below 2^24 - 1, logits below 2^30", (long long)B,
              (long long)T, (long long)V);
    return BF_ERANGE;
  }
  const int64_t N = B * T;
  BF_REQUIRE(N == 0 || (logits && tokens && old_logp && advantages && logp), "bf_policy_loss: null pointer");
  const PolicyArgs a{tokens, old_logp, ref_logp, advantages, static_cast<const uint8_t*>(mask), B, T, adv_b, adv_t,
                     1.f - clip_low, 1.f + clip_high, kl_weight, (float)(1.4426950408889634074 / temperature),
                     (float)(1.0 / temperature), grad_scale, token_bytes, by_sequence};
  const LogitRows rows{T > 0 ? T : 1, ld_b, ld_t, V};
  float4* sums = reinterpret_cast<float4*>(workspace);
  float2* part = reinterpret_cast<float2*>(sums + SUM_GROUPS);
  const Parts p = row_parts(N, V, elem);
  // the counting waits for loads: 1024 rows a workgroup, one a thread
  const int64_t turns = ceil_div(N, COUNT_THREADS), shares = by_sequence && B < turns ? B : turns;
  PolicyCounts counts;
  const bool alone = one_group(N, V, elem), shorts = short_rows(V, elem);
  const int lanes = short_lanes(V);
  counts.share = alone ? workspace : reinterpret_cast<float*>(part + N * p.count);
  counts.live = counts.share + COUNT_GROUPS;
  counts.groups = 1;
  return with_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    const E* x = static_cast<const E*>(logits);
    E* out = static_cast<E*>(grad);
    if (alone) {
      if (lanes == 1)
        hipLaunchKernelGGL((policy_short_kernel<true, 1, E>), dim3(1), dim3(COUNT_THREADS), 0, stream, x, rows, a,
                           counts, logp, stats, out, sums);
      else
        hipLaunchKernelGGL((policy_short_kernel<true, 16, E>), dim3(1), dim3(COUNT_THREADS), 0, stream, x, rows, a,
                           counts, logp, stats, out, sums);
      BF_LAUNCH_CHECK("policy_short_kernel");
      return BF_OK;
    }
    int64_t groups = 0;
    PolicyCounts shared = counts;
    shared.groups = (int)(shares < 1 ? 1 : shares < COUNT_GROUPS ? shares : COUNT_GROUPS);
    auto count = [&] {
      hipLaunchKernelGGL(policy_count_kernel, dim3(shared.groups), dim3(COUNT_THREADS), 0, stream, a, shared);
    };
    if (shorts) {
      count();
      groups = ceil_div(N * lanes, LOSS_THREADS);
      if (groups > 256 * 8) groups = 256 * 8;
      if (lanes == 1)
        hipLaunchKernelGGL((policy_short_kernel<false, 1, E>), dim3((unsigned)groups), dim3(LOSS_THREADS), 0, stream, x,
                           rows, a, shared, logp, stats, out, sums);
      else
        hipLaunchKernelGGL((policy_short_kernel<false, 16, E>), dim3((unsigned)groups), dim3(LOSS_THREADS), 0, stream, x,
                           rows, a, shared, logp, stats, out, sums);
      BF_LAUNCH_CHECK("policy_short_kernel");
    } else if (N >= 256) {
      const int rc = with_row_group(V / (16 / (int)sizeof(E)), [&](auto threads, auto nv, auto full) -> int {
        // as many workgroups as the device holds; each goes through its rows
        constexpr int TH = decltype(threads)::value, NV = decltype(nv)::value, FULL = decltype(full)::value;
        const int64_t most = 256 * (TH == 64 ? 16 : TH == 256 ? 6 : TH == 512 ? 2 : 1);
        groups = N < most ? N : most;
        count();
        auto launch = [&](auto kernel) {
          hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(TH), 0, stream, x, rows, a, shared, logp, out, sums,
                             (unsigned)(groups * 0.6180339887498949));
        };
        if (grad) launch(policy_row_kernel<true, E, TH, NV, FULL>);
        else launch(policy_row_kernel<false, E, TH, NV, FULL>);
        BF_LAUNCH_CHECK("policy_row_kernel");
        return BF_OK;
      });
      if (rc != BF_OK) return rc;
    }
    if (groups) {
      hipLaunchKernelGGL(policy_stats_kernel, dim3(1), dim3(STATS_THREADS), 0, stream, sums, groups, kl_weight, stats);
      BF_LAUNCH_CHECK("policy_stats_kernel");
      return BF_OK;
    }
    hipLaunchKernelGGL((loss_partial_kernel<E, LOSS_THREADS>), dim3((unsigned)(N * p.count + 1)), dim3(LOSS_THREADS), 0,
                       stream, x, rows, a, N, p.count, p.chunk, part, counts);
    BF_LAUNCH_CHECK("loss_partial_kernel");
    const unsigned grid = grad ? (unsigned)(N * p.count + 1) : 1u;
    if (p.count == 1)
      hipLaunchKernelGGL((policy_part_kernel<true, E>), dim3(grid), dim3(LOSS_THREADS), 0, stream, x, rows, a, N, p.count,
                         p.chunk, part, counts, logp, stats, out);
    else
      hipLaunchKernelGGL((policy_part_kernel<false, E>), dim3(grid), dim3(LOSS_THREADS), 0, stream, x, rows, a, N,
                         p.count, p.chunk, part, counts, logp, stats, out);
    BF_LAUNCH_CHECK("policy_part_kernel");
    return BF_OK;
  });
}

// coef [N] float4, part [N * parts] float2, losses [pairs]
int64_t bf_preference_loss_workspace(int64_t N, int64_t V, int64_t pairs, int elem) {
  if (!elem_ok(elem) || N < 0 || V <= 0 || pairs < 0 || !rows_fit(N, V)) return 0;
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
    set_error("bf_preference_loss: %lld rows of %lld logits, %lld pairs: rows below 2^24 - 1, pairs below 2^24, logits "
              "below 2^30", (long long)N, (long long)V, (long long)pairs);
    return BF_ERANGE;
  }
  const Parts p = row_parts(N, V, elem);
  const PreferenceArgs a{tokens, ref_logp, offsets, N, pairs, beta, smoothing, grad_scale, token_bytes};
  const LogitRows rows{N > 0 ? N : 1, 0, ld, V};
  const float c = 1.4426950408889634f;
  float4* coef = reinterpret_cast<float4*>(workspace);
  float2* part = reinterpret_cast<float2*>(coef + N);
  float* losses = reinterpret_cast<float*>(part + N * p.count);
  const bool wave = p.count == 1 && V <= WAVE_VECTORS * 64 * (16 / elem_bytes(elem));
  return with_elem(elem, [&](auto e) -> int {
    using E = decltype(e);
    const E* x = static_cast<const E*>(logits);
    if (N > 0) {
      PolicyArgs all = {};
      all.tokens = tokens;
      all.token_bytes = token_bytes;
      all.c = c;
      auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(N * p.count)), dim3(threads), 0, stream, x, rows, all, N, p.count, p.chunk,
                           part, PolicyCounts{});
      };
      if (wave) launch(loss_partial_kernel<E, 64>, 64);
      else launch(loss_partial_kernel<E, LOSS_THREADS>, LOSS_THREADS);
      BF_LAUNCH_CHECK("loss_partial_kernel");
    }
    const unsigned pair_grid = (unsigned)(pairs < PAIR_GROUPS ? pairs : PAIR_GROUPS) + 1;
    if (p.count == 1)
      hipLaunchKernelGGL((preference_pairs_kernel<true, E>), dim3(pair_grid), dim3(PAIR_THREADS), 0, stream, x,
                         rows, a, part, p.count, c, logp, coef, rewards, losses);
    else
      hipLaunchKernelGGL((preference_pairs_kernel<false, E>), dim3(pair_grid), dim3(PAIR_THREADS), 0, stream, x,
                         rows, a, part, p.count, c, logp, coef, rewards, losses);
    BF_LAUNCH_CHECK("preference_pairs_kernel");
    const unsigned grid = grad ? (unsigned)(N * p.count + 1) : 1u;
    auto launch = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, stream, x, rows, a, p.count, p.chunk, c, coef, losses, loss,
                         static_cast<E*>(grad));
    };
    if (wave) launch(preference_grad_kernel<E, 64>, 64);
    else launch(preference_grad_kernel<E, LOSS_THREADS>, LOSS_THREADS);
    BF_LAUNCH_CHECK("preference_grad_kernel");
    return BF_OK;
  });
}

}  // extern "C"
