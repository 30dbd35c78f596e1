// Softmax cross entropy of a linear head over a vocabulary, with the gradients of the hidden rows, the
// head's weight and its bias.  With z_nv = x_n . w_v + b_v over the rows that count, y_n their tokens:
//
//   logp_n = z_ny / t - log sum_v exp(z_nv / t),   loss = -mean of logp_n
//   G_nv   = exp(z_nv / t) / sum - [v = y_n],      s = grad_scale / (t rows)
//   dx_n   = s sum_v G_nv w_v,   dw_v = s sum_n G_nv x_n,   db_v = s sum_n G_nv
//
// The logits are never kept.  A first pass forms them tile by tile and leaves each row's largest logit M and
// sum of 2^(c (z - M)) per tile, c = log2(e) / t; a second one forms them again, a piece of the vocabulary at a
// time, and leaves the piece's G in the type of the matrix products (fp32: in three parts), from which
// the piece's dw and its share of dx are made.
//
// Rows that count (not masked, token not negative) are gathered first, in their order, and only they are multiplied.
// Every sum is in fp32 and in a fixed order.

#include "bf_vocab_gemm.h"

namespace bf {

typedef VocabTile<4, 2, 2, 4> VocabLarge;
typedef VocabTile<2, 2, 2, 2> VocabMid;

// ---------------------------------------------------------------------------
// Rows that count

// One workgroup: the rows that count in their order.  live[0] their number, source[i] row i's place, place[n] the
// inverse (-1: does not count), token[i] its token; logp is 0 where a row does not count.
__global__ void __launch_bounds__(1024) vocab_rows_kernel(const void* __restrict__ tokens, int token_bytes,
                                                          const uint8_t* __restrict__ mask, int N, int* __restrict__ live,
                                                          int* __restrict__ source, int* __restrict__ place,
                                                          int* __restrict__ token, float* __restrict__ logp) {
  __shared__ int sums[16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  constexpr int HELD = 4;
  int done = 0;
  for (int base = 0; base < N; base += 1024 * HELD) {
    int tok[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int n = base + 1024 * k + t;
      tok[k] = n < N && (!mask || mask[n]) ? load_token(tokens, token_bytes, n) : -1;
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int n = base + 1024 * k + t;
      const uint64_t votes = __ballot(tok[k] >= 0);
      if (lane == 0) sums[wave] = __popcll(votes);
      __syncthreads();
      int before = done, all = 0;
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
      }
      const int at = before + __popcll(votes & ((1ull << lane) - 1));
      if (n < N) {
        if (tok[k] >= 0) {
          source[at] = n;
          token[at] = tok[k];
          place[n] = at;
        } else {
          place[n] = -1;
          logp[n] = 0.f;
        }
      }
      done += all;
      __syncthreads();
    }
  }
  if (t == 0) *live = done;
}

// Eight elements of a row from column d on, zeros past the row's end.
template <class T>
__device__ __forceinline__ Pack<T, 8> row_chunk(const T* row, int d, int D) {
  if (d + 8 <= D) return load_pack<T, 8>(row + d);
  Pack<T, 8> x;
#pragma unroll
  for (int k = 0; k < 8; ++k) x.v[k] = d + k < D ? row[d + k] : (T)0.f;
  return x;
}

template <class T, class E>
__device__ __forceinline__ void pack_chunk(const Pack<T, 8>& x, E* at, int64_t part) {
  if constexpr (sizeof(T) == 2) {
    Pack<E, 8> y;
#pragma unroll
    for (int k = 0; k < 8; ++k) y.v[k] = x.v[k];
    store_pack(at, y);
  } else {
    Pack<__bf16, 8> y[VOCAB_PARTS];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      __bf16 parts[VOCAB_PARTS];
      split_parts(x.v[k], parts);
#pragma unroll
      for (int q = 0; q < VOCAB_PARTS; ++q) y[q].v[k] = parts[q];
    }
#pragma unroll
    for (int q = 0; q < VOCAB_PARTS; ++q) store_pack(at + q * part, y[q]);
  }
}

// The hidden rows that count, dense and padded with zeros to Dp columns and a multiple of 64 rows (fp32: in parts).
template <class T, class E>
__global__ void __launch_bounds__(256) vocab_pack_rows_kernel(const T* __restrict__ hidden, int64_t ld_b, int64_t ld_t,
                                                              int length, const int* __restrict__ source,
                                                              const int* __restrict__ live, int D, int Dp,
                                                              E* __restrict__ out, int64_t part) {
  const int n = blockIdx.x, rows = *live;
  if (n >= (rows + 63) / 64 * 64) return;
  const bool counts = n < rows;
  const int from = counts ? source[n] : 0;
  const T* row = hidden + (from / length) * ld_b + (from % length) * ld_t;
  for (int d = 8 * threadIdx.x; d < Dp; d += 8 * 256)
    pack_chunk<T, E>(row_chunk(row, d, counts ? D : 0), out + (int64_t)n * Dp + d, part);
}

// Rows of a weight that cannot be read as they lie, padded with zeros to Dp columns (fp32: in parts).
template <class T, class E>
__global__ void __launch_bounds__(256) vocab_pack_weight_kernel(const T* __restrict__ weight, int64_t ld, int D, int Dp,
                                                                E* __restrict__ out, int64_t part) {
  const int64_t v = blockIdx.x;
  for (int d = 8 * threadIdx.x; d < Dp; d += 8 * 256)
    pack_chunk<T, E>(row_chunk(weight + v * ld, d, D), out + v * Dp + d, part);
}

// A row's statistics from those of its tiles, its token's log-probability.  64 rows a workgroup, the tiles over 16 waves.
__global__ void __launch_bounds__(1024) vocab_rows_stats_kernel(const float2* __restrict__ part, int64_t part_ld, int tiles,
                                                                const float* __restrict__ chosen,
                                                                const int* __restrict__ token,
                                                                const int* __restrict__ source,
                                                                const int* __restrict__ live, int vocab, float c,
                                                                float inv_t, float2* __restrict__ row,
                                                                float* __restrict__ logp) {
  __shared__ float2 red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x * 64 + lane, rows = *live;
  if ((int)blockIdx.x * 64 >= rows) return;
  float top = -INFINITY, sum = 0.f;
  auto join = [&](float2 x) {
    const float held = fmaxf(top, x.x) == -INFINITY ? 0.f : fmaxf(top, x.x);
    // a share without a logit above -inf has sum 0, or NaN
    sum = sum * (top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top - held) * c)) +
          x.y * (x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((x.x - held) * c));
    top = fmaxf(top, x.x);
  };
  if (n < rows)
    for (int k = wave; k < tiles; k += 16) join(part[k * part_ld + n]);
  red[wave][lane] = make_float2(top, sum);
  __syncthreads();
  if (wave || n >= rows) return;
  for (int w = 1; w < 16; ++w) join(red[w][lane]);
  float lp = (chosen[n] - top) * inv_t - logf(sum);
  float inv = 1.f / sum;
  if (token[n] >= vocab) lp = inv = __int_as_float(0x7fc00000);   // a token past the vocabulary shows as NaN
  row[n] = make_float2(top, inv);
  logp[source[n]] = lp;
}

// The loss, by one workgroup; and where there is a gradient of the hidden rows, that: the pieces' sums joined, scaled
// and brought back to their rows, zeros in rows that do not count (workgroup 1 + n does row n).
template <class T>
__global__ void __launch_bounds__(256) vocab_finish_kernel(const float* __restrict__ logp, int N,
                                                           const int* __restrict__ live, const int* __restrict__ place,
                                                           const float* __restrict__ dx, int64_t dx_split, int64_t dx_ld,
                                                           int splits, int D, float scale, float* __restrict__ loss,
                                                           T* __restrict__ grad) {
  const int rows = max(*live, 1);
  if (blockIdx.x == 0) {
    __shared__ float red[4];
    float sum = 0.f;
    for (int n = threadIdx.x; n < N; n += 256) sum += logp[n];
    sum = block_sum<4>(sum, red);
    if (threadIdx.x == 0) *loss = *live ? -sum / (float)rows : 0.f;
    return;
  }
  const int64_t n = blockIdx.x - 1;
  const int at = place[n];
  T* out = grad + n * D;
  const float factor = scale / (float)rows;
  for (int d = 8 * threadIdx.x; d < D; d += 8 * 256) {
    Pack<T, 8> y;
    if (at < 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = (T)0.f;
    } else {
      float x[8] = {};
      for (int s = 0; s < splits; ++s) {
        const Pack<float, 8> more = load_pack<float, 8>(dx + s * dx_split + at * dx_ld + d);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] += more.v[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) y.v[k] = (T)(x[k] * factor);
    }
    if (d + 8 <= D) {
      store_pack(out + d, y);
    } else {
      for (int k = 0; d + k < D; ++k) out[d + k] = y.v[k];
    }
  }
}

// No rows: a loss of 0 and gradients of 0.
__global__ void __launch_bounds__(256) vocab_nothing_kernel(float* loss, void* dw, int64_t weights, int dw_elem, void* db,
                                                            int64_t biases, int elem) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *loss = 0.f;
  for (int k = 0; k < 16; ++k) {
    const int64_t i = ((int64_t)blockIdx.x * 16 + k) * 256 + threadIdx.x;
    if (i < weights) store_elem(dw, dw_elem, i, 0.f);
    if (i < biases) store_elem(db, elem, i, 0.f);
  }
}

// ---------------------------------------------------------------------------
// What a call of given sizes does

struct VocabPlan {
  int64_t N, D, V;
  int elem, parts;
  bool direct, grad;
  int64_t rows, Dp;          // padded
  int64_t piece;             // vocabulary of a piece
  int64_t first;             // vocabulary of a launch of the first pass
  int64_t stats_tiles;       // tiles of the vocabulary in the first pass
  int splits;
  // bytes from the workspace's start
  int64_t live, source, place, token, chosen, row, part, x, w, g, dx, bytes;
};

inline bool vocab_direct(int elem, int64_t D, const void* weight, int64_t ld) {
  return elem != TE_F32 && D % 64 == 0 && ld % 8 == 0 && (uintptr_t)weight % 16 == 0;
}

constexpr int64_t VOCAB_PIECE_BYTES = 512LL << 20;   // of a piece's G and packed weight

inline VocabPlan vocab_plan(int64_t N, int64_t D, int64_t V, int elem, const void* weight, int64_t ld, bool grad) {
  VocabPlan p;
  p.N = N;
  p.D = D;
  p.V = V;
  p.elem = elem;
  p.grad = grad;
  p.parts = elem == TE_F32 ? VOCAB_PARTS : 1;
  p.direct = vocab_direct(elem, D, weight, ld);
  p.rows = ceil_div(N, 64) * 64;
  p.Dp = ceil_div(D, 64) * 64;
  const int64_t per_token = 2 * p.parts * ((grad ? p.rows : 0) + (p.direct ? 0 : p.Dp));
  const int64_t whole = ceil_div(V, 256) * 256;
  p.piece = whole;
  if (per_token > 0) {
    p.piece = VOCAB_PIECE_BYTES / per_token / 256 * 256;
    if (p.piece < 256) p.piece = 256;
    if (p.piece > whole) p.piece = whole;
  }
  p.first = p.direct ? whole : p.piece;
  p.stats_tiles = ceil_div(V, 128);
  p.splits = 1;
  if (grad) {
    const int64_t tiles = ceil_div(N, VocabMid::BN) * ceil_div(D, VocabMid::BM);
    while (p.splits < 16 && tiles * p.splits < 256 && p.splits * 8 * 64 < p.piece) p.splits *= 2;
  }
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += ceil_div(bytes, 256) * 256;
    return from;
  };
  p.live = take(4);
  p.source = take(4 * N);
  p.place = take(4 * N);
  p.token = take(4 * N);
  p.chosen = take(4 * N);
  p.row = take(8 * N);
  p.part = take(8 * p.stats_tiles * N);
  p.x = take(2 * p.parts * p.rows * p.Dp);
  p.w = take(p.direct ? 0 : 2 * p.parts * p.piece * p.Dp);
  p.g = take(grad ? 2 * p.parts * p.rows * p.piece : 0);
  p.dx = take(grad ? 4 * p.splits * p.rows * p.Dp : 0);
  p.bytes = at;
  return p;
}

inline bool vocab_large(const VocabArgs& a) {
  return ceil_div(a.M, VocabLarge::BM) * ceil_div(a.N, VocabLarge::BN) * a.splits >= 256;
}

template <int MODE, class E, bool PARTS>
void vocab_gemm(const VocabArgs& a, hipStream_t stream) {
  if (vocab_large(a)) launch_vocab_gemm<VocabLarge, MODE, E, PARTS>(a, stream);
  else launch_vocab_gemm<VocabMid, MODE, E, PARTS>(a, stream);
}

struct VocabCall {
  const void* hidden;
  int64_t length, ld_b, ld_t;
  const void* weight;
  int64_t ld_w;
  const void* bias;
  const void* tokens;
  int token_bytes;
  const void* mask;
  double temperature;
  float grad_scale;
  float* logp;
  float* loss;
  void* grad_hidden;
  void* grad_weight;
  int grad_weight_elem;
  void* grad_bias;
  char* space;
  hipStream_t stream;
};

// T: the tensors' type, E: the matrix products'
template <class T, class E>
int vocab_run(const VocabPlan& p, const VocabCall& q) {
  constexpr bool PARTS = sizeof(T) == 4;
  hipStream_t stream = q.stream;
  const int N = (int)p.N, D = (int)p.D;
  int* live = (int*)(q.space + p.live);
  int* source = (int*)(q.space + p.source);
  int* place = (int*)(q.space + p.place);
  int* token = (int*)(q.space + p.token);
  float* chosen = (float*)(q.space + p.chosen);
  float2* row = (float2*)(q.space + p.row);
  float2* part = (float2*)(q.space + p.part);
  E* x = (E*)(q.space + p.x);
  E* w = (E*)(q.space + p.w);
  E* g = (E*)(q.space + p.g);
  float* dx = (float*)(q.space + p.dx);
  const int64_t x_part = p.rows * p.Dp, w_part = p.piece * p.Dp, g_part = p.rows * p.piece;
  const float c = (float)(1.4426950408889634 / q.temperature), inv_t = (float)(1.0 / q.temperature);
  const float scale = (float)((double)q.grad_scale / q.temperature) / (__is_same(E, _Float16) ? VOCAB_F16_SCALE : 1.f);

  hipLaunchKernelGGL(vocab_rows_kernel, dim3(1), dim3(1024), 0, stream, q.tokens, q.token_bytes, (const uint8_t*)q.mask,
                     N, live, source, place, token, q.logp);
  BF_LAUNCH_CHECK("bf_vocab_loss");
  hipLaunchKernelGGL((vocab_pack_rows_kernel<T, E>), dim3((unsigned)p.rows), dim3(256), 0, stream, (const T*)q.hidden,
                     q.ld_b, q.ld_t, (int)q.length, source, live, D, (int)p.Dp, x, x_part);
  BF_LAUNCH_CHECK("bf_vocab_loss");

  VocabArgs a;
  memset(&a, 0, sizeof(a));
  a.live = live;
  a.pairs = PARTS ? VOCAB_PAIRS : 1;
  a.elem = p.elem;
  a.tokens = token;
  a.c = c;
  a.part_ld = N;
  a.chosen = chosen;
  a.row = row;
  a.splits = 1;
  const T* weight = (const T*)q.weight;
  // the weight's rows from v0 on, as the products read them
  auto weight_rows = [&](int64_t v0, int count) {
    if (p.direct) {
      a.A = weight + v0 * q.ld_w;
      a.lda = q.ld_w;
      a.a_part = 0;
      return;
    }
    hipLaunchKernelGGL((vocab_pack_weight_kernel<T, E>), dim3((unsigned)count), dim3(256), 0, stream,
                       weight + v0 * q.ld_w, q.ld_w, D, (int)p.Dp, w, w_part);
    a.A = w;
    a.lda = p.Dp;
    a.a_part = w_part;
  };
  auto logits = [&](int64_t v0, int count) {
    weight_rows(v0, count);
    a.B = x;
    a.ldb = p.Dp;
    a.b_part = x_part;
    a.M = a.a_rows = count;
    a.N = N;
    a.b_rows = (int)p.rows;
    a.K = a.a_cols = a.b_cols = (int)p.Dp;
    a.v0 = (int)v0;
    a.bias = q.bias ? (const T*)q.bias + v0 : nullptr;
  };
  int tiles = 0;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.first) {
    const int count = (int)(p.V - v0 < p.first ? p.V - v0 : p.first);
    logits(v0, count);
    a.part = part + (int64_t)tiles * N;
    vocab_gemm<VM_STATS, E, PARTS>(a, stream);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    tiles += (int)ceil_div(count, vocab_large(a) ? VocabLarge::BM : VocabMid::BM);
  }
  hipLaunchKernelGGL(vocab_rows_stats_kernel, dim3((unsigned)ceil_div(N, 64)), dim3(1024), 0, stream, part, (int64_t)N,
                     tiles, chosen, token, source, live, (int)p.V, c, inv_t, row, q.logp);
  BF_LAUNCH_CHECK("bf_vocab_loss");

  for (int64_t v0 = 0; p.grad && v0 < p.V; v0 += p.piece) {
    const int count = (int)(p.V - v0 < p.piece ? p.V - v0 : p.piece);
    logits(v0, count);
    a.G = g;
    a.ldg = p.piece;
    a.g_part = g_part;
    a.g_rows = (int)p.rows;
    vocab_gemm<VM_GRAD, E, PARTS>(a, stream);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    // dx: the weight's rows are k
    a.B = g;
    a.ldb = p.piece;
    a.b_part = g_part;
    a.M = D;
    a.N = N;
    a.K = (int)(ceil_div(count, 64) * 64);
    a.a_rows = count;
    a.a_cols = (int)p.Dp;
    a.b_rows = (int)p.rows;
    a.splits = p.splits;
    a.dx = dx;
    a.dx_split = p.rows * p.Dp;
    a.dx_ld = p.Dp;
    a.dx_add = v0 > 0;
    vocab_gemm<VM_DX, E, PARTS>(a, stream);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    // dw: the hidden rows are k
    a.splits = 1;
    a.A = x;
    a.lda = p.Dp;
    a.a_part = x_part;
    a.a_rows = (int)p.rows;
    a.N = count;
    a.b_cols = (int)p.piece;
    a.dw = (char*)q.grad_weight + v0 * D * elem_bytes(q.grad_weight_elem);
    a.dw_ld = D;
    a.dw_elem = q.grad_weight_elem;
    a.db = q.grad_bias ? (T*)q.grad_bias + v0 : nullptr;
    a.scale = scale;
    vocab_gemm<VM_DW, E, PARTS>(a, stream);
    BF_LAUNCH_CHECK("bf_vocab_loss");
  }
  hipLaunchKernelGGL((vocab_finish_kernel<T>), dim3(p.grad ? (unsigned)(1 + N) : 1), dim3(256), 0, stream, q.logp, N, live,
                     place, dx, p.rows * p.Dp, p.Dp, p.splits, D, scale, q.loss, (T*)q.grad_hidden);
  BF_LAUNCH_CHECK("bf_vocab_loss");
  return BF_OK;
}

constexpr int64_t VOCAB_ROWS = 1LL << 23, VOCAB_DIM = 1LL << 20, VOCAB_TOKENS = 1LL << 30;

inline bool vocab_sizes_ok(int64_t N, int64_t D, int64_t V, int64_t ld_w) {
  if (!(N < VOCAB_ROWS && D <= VOCAB_DIM && V <= VOCAB_TOKENS && ld_w <= VOCAB_DIM)) return false;
  // tiles of a launch (its workgroups of 512 work-items have to stay below 2^32)
  return ceil_div(V, 128) * ceil_div(N, 128) < (1LL << 22) && ceil_div(V, 128) * ceil_div(D, 128) < (1LL << 22) &&
         ceil_div(N, 128) * ceil_div(D, 128) < (1LL << 22);
}

}  // namespace bf

using namespace bf;

extern "C" int64_t bf_vocab_loss_workspace(int64_t N, int64_t D, int64_t V, int elem, const void* weight, int64_t ld_w,
                                           int with_grad) {
  if (!elem_ok(elem) || N <= 0 || D <= 0 || V <= 0 || ld_w < D || !vocab_sizes_ok(N, D, V, ld_w)) return 0;
  return vocab_plan(N, D, V, elem, weight, ld_w, with_grad != 0).bytes / 4;
}

extern "C" int bf_vocab_loss(const void* hidden, int elem, int64_t B, int64_t T, int64_t D, int64_t ld_b, int64_t ld_t,
                             const void* weight, int64_t V, int64_t ld_w, const void* bias, const void* tokens,
                             int token_bytes, const void* mask, double temperature, float grad_scale, float* logp,
                             float* loss, void* grad_hidden, void* grad_weight, int grad_weight_elem, void* grad_bias,
                             float* workspace, hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8), "bf_vocab_loss: element type %d, token bytes %d",
             elem, token_bytes);
  BF_REQUIRE(B >= 0 && T >= 0 && D > 0 && V > 0 && ld_b >= 0 && ld_t >= 0 && ld_w >= D, "bf_vocab_loss: bad sizes");
  BF_REQUIRE(temperature > 0.0, "bf_vocab_loss: temperature %g", temperature);
  BF_REQUIRE(loss, "bf_vocab_loss: null pointer");
  const bool grad = grad_hidden || grad_weight || grad_bias;
  BF_REQUIRE(!grad || (grad_weight && (B * T == 0 || grad_hidden) && !bias == !grad_bias),
             "bf_vocab_loss: gradients of hidden rows and weight, and of the bias where there is one, come together");
  BF_REQUIRE(!grad || grad_weight_elem == elem || grad_weight_elem == TE_F32,
             "bf_vocab_loss: weight gradient of element type %d", grad_weight_elem);
  if (B > VOCAB_ROWS || T > VOCAB_ROWS || !vocab_sizes_ok(B * T, D, V, ld_w)) {
    set_error("bf_vocab_loss: %lld x %lld rows, width %lld, vocabulary %lld are more than it takes", (long long)B,
              (long long)T, (long long)D, (long long)V);
    return BF_ERANGE;
  }
  const int64_t N = B * T;
  BF_REQUIRE(weight && (N == 0 || (hidden && tokens && logp && workspace)), "bf_vocab_loss: null pointer");
  BF_REQUIRE((uintptr_t)workspace % 16 == 0, "bf_vocab_loss: workspace not aligned to 16 bytes");
  if (N == 0) {
    const int64_t weights = grad ? V * D : 0, biases = grad_bias ? V : 0;
    const int64_t blocks = ceil_div(weights > biases ? weights : biases, 256 * 16);
    hipLaunchKernelGGL(vocab_nothing_kernel, dim3(blocks ? (unsigned)blocks : 1), dim3(256), 0, stream, loss, grad_weight,
                       weights, grad_weight_elem, grad_bias, biases, elem);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    return BF_OK;
  }
  const VocabPlan p = vocab_plan(N, D, V, elem, weight, ld_w, grad);
  const VocabCall q = {hidden, T, ld_b, ld_t, weight, ld_w, bias, tokens, token_bytes, mask, temperature, grad_scale, logp,
                       loss, grad_hidden, grad_weight, grad_weight_elem, grad_bias, (char*)workspace, stream};
  switch (elem) {
    case TE_F32: return vocab_run<float, __bf16>(p, q);
    case TE_BF16: return vocab_run<__bf16, __bf16>(p, q);
    default: return vocab_run<_Float16, _Float16>(p, q);
  }
}
