// Softmax cross entropy of a linear head over a vocabulary, with the gradients of the hidden rows, the
// head's weight and its bias.  With z_nv = x_n . w_v + b_v over the rows that count, y_n their tokens:
//
//   logp_n = z_ny / t - log sum_v exp(z_nv / t),   loss = -mean of logp_n
//   G_nv   = exp(z_nv / t) / sum - [v = y_n],      s = grad_scale / (t rows)
//   dx_n   = s sum_v G_nv w_v,   dw_v = s sum_n G_nv x_n,   db_v = s sum_n G_nv
//
// The logits are not kept.  A first pass over the vocabulary (vocab_logits_kernel) leaves each row's largest logit and
// sum of exponentials per tile, and of as much of the vocabulary as the workspace has room for the exponentials in the type
// of the matrix products (fp32: in three parts).  vocab_softmax_kernel joins the tiles' statistics and makes those exponentials
// G; dx and dw follow from it (vocab_grads_kernel).  For what has no room, the logits are formed again, a
// piece at a time, with the statistics known.
//
// Rows that count (not masked, token not negative) are gathered first, in their order, and only they are multiplied.
// Every sum is in fp32 and in a fixed order.

#include "bf_vocab_gemm.h"

namespace bf {

// ---------------------------------------------------------------------------
// Rows that count

// The rows that count in their order: live[0] their number, source[i] row i's place, place[n] the inverse (-1: does not
// count), token[i] its token; logp is 0 where a row does not count.  A workgroup takes VOCAB_COUNTED rows and counts those
// before them for itself, which for many rows would be most of the work: past VOCAB_COUNTED_ROWS one workgroup takes
// all (8000 rows: 15 us by one workgroup, 8 by eight).
constexpr int VOCAB_COUNTED = 1024, VOCAB_COUNTED_ROWS = 64 * VOCAB_COUNTED;

__global__ void __launch_bounds__(1024) vocab_rows_kernel(const void* __restrict__ tokens, int token_bytes,
                                                          const uint8_t* __restrict__ mask, int N, int* __restrict__ live,
                                                          int* __restrict__ source, int* __restrict__ place,
                                                          int* __restrict__ token, float* __restrict__ logp) {
  __shared__ int sums[16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  auto token_of = [&](int n) { return n < N && (!mask || mask[n]) ? load_token(tokens, token_bytes, n) : -1; };
  const int from = blockIdx.x * VOCAB_COUNTED, to = gridDim.x == 1 ? N : min(N, from + VOCAB_COUNTED);
  int before = 0;      // of this wave's share of the rows before
#pragma unroll 8
  for (int n = t; n < from; n += 1024) before += __popcll(__ballot(token_of(n) >= 0));
  if (lane == 0) sums[wave] = before;
  __syncthreads();
  int done = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) done += sums[w];
  for (int base = from; base < to; base += 1024) {
    const int n = base + t, tok = token_of(n);
    const uint64_t votes = __ballot(tok >= 0);
    __syncthreads();
    if (lane == 0) sums[wave] = __popcll(votes);
    __syncthreads();
    int at = done + __popcll(votes & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      at += w < wave ? sums[w] : 0;
      done += sums[w];
    }
    if (n < N) {
      place[n] = tok >= 0 ? at : -1;
      if (tok >= 0) {
        source[at] = n;
        token[at] = tok;
      } else {
        logp[n] = 0.f;
      }
    }
  }
  if (blockIdx.x + 1 == gridDim.x && t == 0) *live = done;
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

// What the products read, and what rows that do not count get.  Workgroups [0, N): hidden row n to its place among
// the rows that count, dense and padded with zeros to Dp columns (fp32: in parts), or zeros to its gradient.  [N, N + 64): zeros
// behind the last row up to a multiple of 64.  The others: rows of a weight that cannot be read as it
// lies, padded and split alike.  Up to VOCAB_SCAN rows each workgroup counts for itself which rows count, which saves a launch.
// Bound by memory: 32000 x 1024 fp32 rows in three parts 52 us (330 MB at 6.3 TB/s); 50001 x 1025 fp16, which start at any two
// bytes, 37 us (211 MB at 5.7 TB/s).
constexpr int VOCAB_SCAN = 1024;

struct VocabPrepare {
  const void* hidden;
  int64_t ld_b, ld_t;
  int length;
  const void* tokens;
  int token_bytes;
  const uint8_t* mask;
  int N, D, Dp;
  int* live;
  int* source;
  int* place;
  int* token;
  float* logp;
  void* x;
  int64_t x_part;
  void* grad_hidden;        // or null
  const void* weight;       // rows to be packed, or null
  int64_t ld_w, weight_rows;
  void* w;
  int64_t w_part;
};

template <class T, class E, bool SCAN>
__global__ void __launch_bounds__(256) vocab_prepare_kernel(VocabPrepare p) {
  const int t = threadIdx.x;
  if ((int64_t)blockIdx.x >= p.N + 64) {
    const int64_t at = ((int64_t)blockIdx.x - p.N - 64) * 256 + t;
    const int chunks = p.Dp / 8;
    const int64_t v = div_rows(at, chunks, at < (1LL << 31));
    if (v >= p.weight_rows) return;
    const int d = 8 * (int)(at - v * chunks);
    pack_chunk<T, E>(row_chunk((const T*)p.weight + v * p.ld_w, d, p.D), (E*)p.w + v * p.Dp + d, p.w_part);
    return;
  }
  const int n = blockIdx.x;
  int live, at = -1;
  if constexpr (SCAN) {
    __shared__ int sums[4][2];
    int before = 0, all = 0, mine = -1;
#pragma unroll
    for (int k = 0; k < VOCAB_SCAN / 256; ++k) {
      const int i = 256 * k + t;
      const int tok = i < p.N && (!p.mask || p.mask[i]) ? load_token(p.tokens, p.token_bytes, i) : -1;
      before += __popcll(__ballot(tok >= 0 && i < n));
      all += __popcll(__ballot(tok >= 0));
      if (i == n) mine = tok;
    }
    __shared__ int own;
    if ((t & 63) == 0) {
      sums[t >> 6][0] = before;
      sums[t >> 6][1] = all;
    }
    if (t == (n & 255)) own = mine;
    __syncthreads();
    before = sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0];
    live = sums[0][1] + sums[1][1] + sums[2][1] + sums[3][1];
    if (n < p.N && own >= 0) at = before;
    if (t == 0) {
      if (n == 0) *p.live = live;
      if (at >= 0) {
        p.source[at] = n;
        p.token[at] = own;
      } else if (n < p.N) {
        p.logp[n] = 0.f;
      }
    }
  } else {
    live = *p.live;
    if (n < p.N) at = p.place[n];
  }
  E* x = (E*)p.x;
  if (n >= p.N) {      // behind the last row that counts
    at = live + n - p.N;
    if (at >= (live + 63) / 64 * 64) return;
    for (int d = 8 * t; d < p.Dp; d += 8 * 256)
      pack_chunk<T, E>(row_chunk((const T*)nullptr, d, 0), x + (int64_t)at * p.Dp + d, p.x_part);
  } else if (at >= 0) {
    const T* row = (const T*)p.hidden + (int64_t)(n / p.length) * p.ld_b + (int64_t)(n % p.length) * p.ld_t;
    for (int d = 8 * t; d < p.Dp; d += 8 * 256)
      pack_chunk<T, E>(row_chunk(row, d, p.D), x + (int64_t)at * p.Dp + d, p.x_part);
  } else if (p.grad_hidden) {
    T* row = (T*)p.grad_hidden + (int64_t)n * p.D;
    for (int d = t; d < p.D; d += 256) row[d] = (T)0.f;
  }
}

// Rows of a weight alone, for a later piece of the vocabulary.
template <class T, class E>
__global__ void __launch_bounds__(256) vocab_pack_weight_kernel(const T* __restrict__ weight, int64_t ld, int64_t rows, int D,
                                                                int Dp, E* __restrict__ out, int64_t part) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = Dp / 8;
  const int64_t v = div_rows(at, chunks, at < (1LL << 31));
  if (v >= rows) return;
  const int d = 8 * (int)(at - v * chunks);
  pack_chunk<T, E>(row_chunk(weight + v * ld, d, D), out + v * Dp + d, part);
}

// Eight numbers, G's or what G is scaled by, in its parts.
template <class E, int GP>
__device__ __forceinline__ void put_parts(float y, Pack<E, 8>* x, int e) {
  if constexpr (GP == VOCAB_PARTS) {
    __bf16 parts[VOCAB_PARTS];
    split_parts(y, parts);
#pragma unroll
    for (int q = 0; q < VOCAB_PARTS; ++q) x[q].v[e] = parts[q];
  } else {
    x[0].v[e] = (E)y;
    if constexpr (GP == 2) x[1].v[e] = (E)(__builtin_isfinite(y) ? y - (float)x[0].v[e] : 0.f);
  }
}

// Exponential e of eight as the first pass left them: fp16, or the two halves of an fp32 number.
template <class E, int GP>
__device__ __forceinline__ float held_exponential(const Pack<E, 8>* x, int e) {
  if constexpr (GP == 1) return (float)__builtin_bit_cast(_Float16, x[0].v[e]) * (1.f / VOCAB_E_SCALE);
  else
    return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, x[0].v[e]) << 16 | __builtin_bit_cast(uint16_t, x[1].v[e]));
}

template <class E>
constexpr float vocab_g_scale() { return __is_same(E, _Float16) ? VOCAB_F16_SCALE : 1.f; }

// Statistics of the rows that count, from those of their tiles, and G from the exponentials that the first pass left, in
// place.  A workgroup joins a row's tiles and takes VOCAB_CHUNK of its entries; the first one of a row writes what others
// read.  The token's entry comes from its log-probability: p - 1 from a rounded p would have no digits left where p is near 1.
// The others are rounded a second time here: they lie here with 11 bits (where G has parts, whole).
constexpr int VOCAB_CHUNK = 8192;

struct VocabSoftmax {
  const float2* part;
  int64_t part_ld;
  int tiles, tile;            // their number, and the entries of one
  const float* chosen;
  const int* token;
  const int* source;
  const int* live;
  int vocab;
  float c, inv_t;
  float2* row;
  float* logp;
  void* G;                    // or null
  int64_t ldg, g_part;
  int held;                   // entries of G
  int chunks;                 // workgroups of a row
};

template <class E, int GP>
__global__ void __launch_bounds__(256) vocab_softmax_kernel(VocabSoftmax p) {
  const int n = blockIdx.x / p.chunks, chunk = blockIdx.x - n * p.chunks;
  if (n >= *p.live) return;
  __shared__ float red[8];
  const int t = threadIdx.x, wave = t >> 6;
  const float2* part = p.part + n * p.part_ld;
  // the exponentials are on their way while the tiles are joined (3150 rows of 32000 tokens 76 us in the place of 93,
  // 5.3 TB/s; 6500 of 128000 693 in the place of 750, 4.8 TB/s)
  constexpr int PLANES = GP > 1 ? 2 : 1, COUNT = VOCAB_CHUNK / 2048;
  E* g = p.G ? (E*)p.G + n * p.ldg + chunk * VOCAB_CHUNK + 8 * t : nullptr;
  const int first = chunk * VOCAB_CHUNK + 8 * t;
  Pack<E, 8> held[COUNT][GP];
#pragma unroll
  for (int k = 0; k < COUNT; ++k)
#pragma unroll
    for (int q = 0; q < PLANES; ++q)
      if (g && first + 2048 * k < p.held) held[k][q] = load_pack<E, 8>(g + q * p.g_part + 2048 * k);
  float top = -INFINITY;
#pragma unroll 4
  for (int k = t; k < p.tiles; k += 256) top = fmaxf(top, part[k].x);
  top = wave_max(top);
  if ((t & 63) == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float sum = 0.f;
#pragma unroll 4
  for (int k = t; k < p.tiles; k += 256) {
    const float2 x = part[k];
    // a tile without a logit above -inf has sum 0, or NaN
    sum += x.x == -INFINITY ? x.y : x.y * __builtin_amdgcn_exp2f((x.x - top) * p.c);
  }
  sum = block_sum<4>(sum, red + 4);
  const int token = p.token[n];
  float lp = (p.chosen[n] - top) * p.inv_t - logf(sum);
  float inv = 1.f / sum;
  if (token >= p.vocab) lp = inv = __int_as_float(0x7fc00000);   // a token past the vocabulary shows as NaN
  if (chunk == 0 && t == 0) {
    p.row[n] = make_float2(top, inv);
    p.logp[p.source[n]] = lp;
  }
  if (!p.G) return;
  constexpr float SCALE = vocab_g_scale<E>();
  const float at_token = (expf(lp) - 1.f) * SCALE;
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int v = first + 2048 * k;
    if (v >= p.held) break;
    const float factor = __builtin_amdgcn_exp2f((part[v / p.tile].x - top) * p.c) * inv * SCALE;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      put_parts<E, GP>(v + e == token ? at_token : held_exponential<E, GP>(held[k], e) * factor, held[k], e);
#pragma unroll
    for (int q = 0; q < GP; ++q) store_pack(g + q * p.g_part + 2048 * k, held[k][q]);
  }
}

// G in place where the bias's gradient is asked for too, from statistics that vocab_softmax_kernel has left: a workgroup takes
// 2048 columns of 32 rows and leaves their sums, of what G is before it is rounded (of exponentials of 11 bits where G has
// one part, the tokens' own entries from fp32; a token's column cancels: the sums of a rounded G were up to 1.9 times as far
// from 64 bits as those of fp32).  841 rows of 50001 tokens 33 us (168 MB at 5.1 TB/s).
constexpr int VOCAB_GROUP = 32;

template <class E, int GP>
__global__ void __launch_bounds__(256) vocab_softmax_columns_kernel(VocabSoftmax p, int chunks, float* __restrict__ sums) {
  const int group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks, live = *p.live;
  const int v = 2048 * chunk + 8 * threadIdx.x;
  const int first = VOCAB_GROUP * group, last = min(first + VOCAB_GROUP, live);
  if (first >= live || v >= p.held) return;
  constexpr float SCALE = vocab_g_scale<E>();
  float sum[8] = {};
#pragma unroll 4
  for (int n = first; n < last; ++n) {
    const float2 row = p.row[n];
    const int token = p.token[n] - v;
    E* g = (E*)p.G + n * p.ldg + v;
    const float factor = __builtin_amdgcn_exp2f((p.part[n * p.part_ld + v / p.tile].x - row.x) * p.c) * row.y * SCALE;
    Pack<E, 8> x[GP];
#pragma unroll
    for (int q = 0; q < (GP > 1 ? 2 : 1); ++q) x[q] = load_pack<E, 8>(g + q * p.g_part);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = held_exponential<E, GP>(x, e) * factor;
    if (token >= 0 && token < 8) {
      const float at_token = (expf(p.logp[p.source[n]]) - 1.f) * SCALE;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = e == token ? at_token : y[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum[e] += y[e];
      put_parts<E, GP>(y[e], x, e);
    }
#pragma unroll
    for (int q = 0; q < GP; ++q) store_pack(g + q * p.g_part, x[q]);
  }
  Pack<float, 8> out;
#pragma unroll
  for (int e = 0; e < 8; ++e) out.v[e] = sum[e];
  store_pack(sums + group * p.ldg + v, out);
}

// The bias's gradient from those sums, of `group` rows each (a tile's, where the logits were formed again); what a sum rounds
// away is kept and added again.
template <class T>
__global__ void __launch_bounds__(256) vocab_bias_kernel(const float* __restrict__ sums, int64_t ld, int columns,
                                                         const int* __restrict__ live, int group, float scale,
                                                         T* __restrict__ grad) {
  const int v = blockIdx.x * 256 + threadIdx.x, groups = (*live + group - 1) / group;
  if (v >= columns) return;
  float sum = 0.f, left = 0.f;
#pragma unroll 8
  for (int k = 0; k < groups; ++k) {
    const float more = sums[k * ld + v] - left, all = sum + more;
    left = (all - sum) - more;
    sum = all;
  }
  grad[v] = (T)(sum * scale / (float)max(*live, 1));
}

// The same from logits that were summed in pieces (VM_SUMS): a row is joined by a workgroup, which holds its logits, or up to
// VOCAB_HELD_WAVE entries by one of four waves (8000 rows of 20 tokens: 5 us against 19).  It leaves the row's G, rounded once,
// and zeros in G's rows behind the last that counts.
constexpr int VOCAB_HELD = 8192, VOCAB_HELD_WAVE = 512;

struct VocabSoftmaxSums {
  VocabSoftmax s;
  const float* sums;          // [splits, rows, ld]
  int64_t split, ld;
  int splits;
  int rows;                   // of G
  const void* bias;           // or null
  int elem;
};

template <class E, int GP, bool WAVE>
__global__ void __launch_bounds__(256) vocab_softmax_sums_kernel(VocabSoftmaxSums q) {
  constexpr int THREADS = WAVE ? 64 : 256, HELD = (WAVE ? VOCAB_HELD_WAVE : VOCAB_HELD) / (8 * THREADS);
  const VocabSoftmax& p = q.s;
  const int live = *p.live, wave = threadIdx.x >> 6, t = threadIdx.x % THREADS;
  const int n = WAVE ? blockIdx.x * 4 + wave : blockIdx.x;
  E* g = p.G ? (E*)p.G + n * p.ldg : nullptr;
  if (n >= live) {
    if (!g || n >= min(q.rows, (live + 63) / 64 * 64)) return;
    for (int v = 8 * t; v < p.held; v += 8 * THREADS)
#pragma unroll
      for (int k = 0; k < GP; ++k) *(Words*)(g + k * p.g_part + v) = zero_words();
    return;
  }
  __shared__ float red[12];
  const int token = p.token[n];
  float z[HELD][8];
  float top = -INFINITY, chosen = -INFINITY;
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int v = 8 * (THREADS * k + t);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[k][e] = 0.f;
    if (v < p.vocab) {
#pragma unroll 4
      for (int s = 0; s < q.splits; ++s) {
        const Pack<float, 8> more = load_pack<float, 8>(q.sums + s * q.split + n * q.ld + v);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[k][e] += more.v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (q.bias && v + e < p.vocab) z[k][e] += load_elem(q.bias, q.elem, v + e);
      if (v + e >= p.vocab) z[k][e] = -INFINITY;
      if (v + e == token) chosen = z[k][e];
      top = fmaxf(top, z[k][e]);
    }
  }
  top = wave_max(top);
  chosen = wave_max(chosen);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) {
      red[wave] = top;
      red[4 + wave] = chosen;
    }
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    chosen = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
  }
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < HELD; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      z[k][e] = __builtin_amdgcn_exp2f((z[k][e] - top) * p.c);
      sum += z[k][e];
    }
  if constexpr (WAVE) sum = wave_sum(sum);
  else sum = block_sum<4>(sum, red + 8);
  float lp = (chosen - top) * p.inv_t - logf(sum);
  float inv = 1.f / sum;
  if (token >= p.vocab) lp = inv = __int_as_float(0x7fc00000);
  if (t == 0) {
    p.row[n] = make_float2(top, inv);
    p.logp[p.source[n]] = lp;
  }
  if (!g) return;
  constexpr float SCALE = vocab_g_scale<E>();
  const float at_token = (expf(lp) - 1.f) * SCALE;
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    const int v = 8 * (THREADS * k + t);
    if (v >= p.held) break;
    Pack<E, 8> x[GP];
#pragma unroll
    for (int e = 0; e < 8; ++e) put_parts<E, GP>(v + e == token ? at_token : z[k][e] * inv * SCALE, x, e);
#pragma unroll
    for (int m = 0; m < GP; ++m) store_pack(g + m * p.g_part + v, x[m]);
  }
}

// The loss alone.
__global__ void __launch_bounds__(256) vocab_loss_kernel(const float* __restrict__ logp, int N, const int* __restrict__ live,
                                                          float* __restrict__ loss) {
  __shared__ float red[4];
  vocab_loss<4>(logp, N, *live, loss, red);
}

// Gradients that were summed in pieces, joined and scaled: rows of the hidden rows' (brought back to their places),
// then of the weight's, then the bias's.  A thread takes eight elements.
struct VocabJoin {
  const int* live;
  const int* source;
  const float* dx;          // [dx_splits, rows, ld], or null
  int64_t dx_split;
  int dx_splits, N;
  void* grad_hidden;
  const float* dw;          // [dw_splits, V, ld], or null
  int64_t dw_split, V;
  int dw_splits;
  void* grad_weight;
  int dw_elem;
  const float* db;          // [dw_splits, V], or null
  void* grad_bias;
  int D;
  int64_t ld;
  float scale;
};

template <class T>
__device__ __forceinline__ void join_chunk(const float* from, int64_t split, int splits, int d, int D, float factor, T* out) {
  float x[8] = {};
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const Pack<float, 8> more = load_pack<float, 8>(from + s * split + d);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] += more.v[k];
  }
  Pack<T, 8> y;
#pragma unroll
  for (int k = 0; k < 8; ++k) y.v[k] = (T)(x[k] * factor);
  if (d + 8 <= D) {
    store_pack(out + d, y);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)     // unrolled: an array that is indexed by a loop lies in LDS, which took 15 us in the place of 5
      if (d + k < D) out[d + k] = y.v[k];
  }
}

template <class T>
__global__ void __launch_bounds__(256) vocab_join_kernel(VocabJoin p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = (p.D + 7) / 8, live = *p.live;
  const float factor = p.scale / (float)max(live, 1);
  int64_t row = div_rows(at, chunks, at < (1LL << 31));
  const int d = 8 * (int)(at - row * chunks);
  const int N = p.dx ? p.N : 0;
  if (row < N) {
    if (row < live)
      join_chunk(p.dx + row * p.ld, p.dx_split, p.dx_splits, d, p.D, factor, (T*)p.grad_hidden + (int64_t)p.source[row] * p.D);
    return;
  }
  row -= N;
  if (!p.dw || row >= p.V) return;
  const float* from = p.dw + row * p.ld;
  if (p.dw_elem == TE_F32) join_chunk(from, p.dw_split, p.dw_splits, d, p.D, factor, (float*)p.grad_weight + row * p.D);
  else join_chunk(from, p.dw_split, p.dw_splits, d, p.D, factor, (T*)p.grad_weight + row * p.D);
  if (p.db && d == 0) {
    float sum = 0.f;
    for (int s = 0; s < p.dw_splits; ++s) sum += p.db[s * p.V + row];
    ((T*)p.grad_bias)[row] = (T)(sum * factor);
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
  int elem, parts, g_parts;  // parts of the weight and the rows, parts of G
  bool direct, regs, grad;   // the weight is read as it lies: copied to LDS, or through registers
  int64_t rows, Dp;          // padded
  int64_t piece;             // vocabulary of a piece: what G and the packed weight have room for
  int64_t tiles;             // of the vocabulary in the first pass
  int logits_tile, grads_tile;
  bool columns;              // the bias's gradient is summed beside the softmax
  bool logits_summed;        // the logits of a row are joined by one workgroup
  int logits_splits;         // from sums over pieces of the width
  int dx_splits, dw_splits;  // of the gradients' sums
  bool dx_joined, dw_joined; // they are summed in pieces first
  // bytes from the workspace's start
  int64_t live, source, place, token, chosen, row, part, x, w, g, cols, sums, dx, dw, db, bytes;
};

inline bool vocab_direct(int elem, int64_t D, const void* weight, int64_t ld) {
  return elem != TE_F32 && D % 8 == 0 && ld % 8 == 0 && (uintptr_t)weight % 16 == 0;
}

inline int64_t vocab_tile_count(int tile, int64_t m, int64_t n, int parts) {
  switch (tile) {
    case VT_LARGE:
      return ceil_div(m, VocabLarge<1>::BM) * ceil_div(n, parts > 1 ? VocabLarge<3>::BN : VocabLarge<1>::BN);
    case VT_SLIM:
    case VT_REGS:
    case VT_THIN: return ceil_div(m, VocabSlim<1>::BM) * ceil_div(n, VocabSlim<1>::BN);
    default: return ceil_div(m, VocabMid::BM) * ceil_div(n, VocabMid::BN);
  }
}

// The same of dW, whose tiles beside Slim's dX are Wide.
inline int64_t vocab_dw_tile_count(int tile, int64_t m, int64_t n, int parts) {
  if (tile == VT_SLIM || tile == VT_REGS) return ceil_div(m, VocabWide<1>::BM) * ceil_div(n, VocabWide<1>::BN);
  return vocab_tile_count(tile, m, n, parts);
}

// Rows of X in a tile of the logits.
inline int vocab_tile_rows(int tile, int parts) {
  switch (tile) {
    case VT_LARGE: return parts > 1 ? VocabLarge<3>::BN : VocabLarge<1>::BN;
    case VT_SLIM:
    case VT_REGS:
    case VT_THIN: return VocabSlim<1>::BN;
    default: return VocabMid::BN;
  }
}

// Rows up to which a weight that cannot be copied to LDS as it lies passes through registers, where a packed copy of it would be
// most of the bytes.  fp32 (us, packed / through registers; rows of 2048 over 32000 tokens): 8 rows 399 / 262, 128 rows
// 542 / 413, 192 rows 650 / 567, scored alone 212 / 85, 261 / 148, 285 / 191.  16-bit rows of an odd width, scored: 64 rows
// of 2049 over 50001 tokens 119 / 80, 128 rows 133 / 137; with gradients, whose product along the vocabulary is read two
// bytes aside, 227 / 277.
constexpr int64_t VOCAB_REGS_FP32 = 192, VOCAB_REGS_SCORED = 64;

// The copies to LDS address G from a tile's first row by 32 bits of bytes: 256 rows of so many tokens at most.
constexpr int64_t VOCAB_PIECE = 1LL << 23;

inline VocabPlan vocab_plan(int64_t N, int64_t D, int64_t V, int elem, const void* weight, int64_t ld, bool grad,
                            bool bias, int64_t room) {
  VocabPlan p;
  p.N = N;
  p.D = D;
  p.V = V;
  p.elem = elem;
  p.grad = grad;
  p.parts = elem == TE_F32 ? VOCAB_PARTS : 1;
  p.direct = vocab_direct(elem, D, weight, ld);
  p.regs = !p.direct && (elem == TE_F32 ? N <= VOCAB_REGS_FP32 : !grad && N <= VOCAB_REGS_SCORED);
  p.rows = ceil_div(N, 64) * 64;
  p.Dp = ceil_div(D, 64) * 64;
  // by the whole vocabulary, so that the statistics have the same bits with and without gradients and whatever the room
  if (p.regs) p.logits_tile = VT_REGS;
  else if (N <= VocabSlim<1>::BN) p.logits_tile = vocab_tile_count(VT_SLIM, V, N, p.parts) > 256 ? VT_SLIM : VT_THIN;
  else if (vocab_tile_count(VT_LARGE, V, N, p.parts) >= 200) p.logits_tile = VT_LARGE;
  else p.logits_tile = p.parts == 1 && vocab_tile_count(VT_MID, V, N, p.parts) > 256 ? VT_MID : VT_DEEP;
  p.tiles = vocab_tile_count(p.logits_tile, V, 1, p.parts);
  // Few tiles are cut along the width, to some two stages at least and a workgroup for every CU at most; the joining
  // workgroup has to hold a row.  Short rows, which a wave joins, go that way cut or not.
  p.logits_splits = 1;
  p.logits_summed = false;
  if ((p.logits_tile == VT_DEEP || p.logits_tile == VT_THIN || p.logits_tile == VT_REGS) && V <= VOCAB_HELD) {
    const int64_t tiles = vocab_tile_count(p.logits_tile, V, N, p.parts);
    int64_t splits = 256 / tiles, most = p.Dp / (p.parts > 1 ? 64 : 128);
    if (splits > most) splits = most;
    if (splits > 16) splits = 16;
    if (splits > 1) p.logits_splits = (int)splits;
    p.logits_summed = splits > 1 || V <= VOCAB_HELD_WAVE;
  }
  // Rounded to one 16-bit part, G adds to the gradients' own rounding (2-norm of all errors against 64 bits over that of one
  // rounding; rows of 512 over 9000 tokens): one to eight rows 1.3 to 1.7, 65 to 8000 rows 1.12 to 1.23, bf16 and fp16, since each
  // of its errors is relative to an entry.  Two parts leave 1.00.  They are taken where they cost next to nothing, and with a
  // bias, whose columns cancel, wherever rows are joined; without one the joined ones' would take 0 to 40 % longer (us, one part /
  // two: 512 rows of 160 over 8 tokens 28 / 28, 1000 of 1024 over 1000 45 / 48, 400 of 4096 over 2000 61 / 85).
  p.g_parts = p.parts > 1 ? p.parts : grad && (N <= VocabSlim<1>::BN || (p.logits_summed && bias)) ? 2 : 1;
  p.columns = grad && bias && !p.logits_summed && p.g_parts != 2;
  const int64_t per_token = 2 * ((grad ? p.g_parts * p.rows : 0) + (p.direct || p.regs ? 0 : p.parts * p.Dp));
  const int64_t whole = ceil_div(V, 256) * 256;
  p.piece = whole;
  if (per_token > 0) {
    p.piece = room / per_token / 256 * 256;
    if (p.piece < 256) p.piece = 256;
    if (p.piece > VOCAB_PIECE) p.piece = VOCAB_PIECE;
    if (p.piece > whole) p.piece = whole;
  }
  const int64_t in_piece = p.piece < V ? p.piece : V;
  const int64_t sums_ld = ceil_div(V, 256) * 256;
  p.grads_tile = VT_SLIM;
  p.dx_splits = p.dw_splits = 1;
  p.dx_joined = p.dw_joined = false;
  if (grad) {
    if (p.regs) {
      p.grads_tile = VT_REGS;
    } else if (N <= VocabSlim<1>::BN) {
      const int64_t slim = vocab_tile_count(VT_SLIM, D, N, p.parts) + vocab_tile_count(VT_SLIM, D, in_piece, p.parts);
      p.grads_tile = slim > 256 ? VT_SLIM : VT_THIN;
    } else {
      const int64_t large = vocab_tile_count(VT_LARGE, D, N, p.parts) + vocab_tile_count(VT_LARGE, D, in_piece, p.parts);
      const int64_t mid = vocab_tile_count(VT_MID, D, N, p.parts) + vocab_tile_count(VT_MID, D, in_piece, p.parts);
      p.grads_tile = large >= 200 ? VT_LARGE : p.parts == 1 && mid > 256 ? VT_MID : VT_DEEP;
    }
    if (p.g_parts == 2 && (p.grads_tile == VT_LARGE || p.grads_tile == VT_MID)) p.grads_tile = VT_DEEP;
    // Sums are cut along k so that none of them takes longer than a good part of the whole launch, nor than it takes to
    // add one more piece's sums (some eight stages).
    const int64_t slots = p.grads_tile == VT_LARGE || p.grads_tile == VT_DEEP || p.grads_tile == VT_THIN ? 256 : 512;
    // (dw's in Slim's tiles: of work, not of workgroups)
    const int64_t dx = vocab_tile_count(p.grads_tile, D, N, p.parts), dw = vocab_tile_count(p.grads_tile, D, in_piece, p.parts);
    const int64_t dx_steps = ceil_div(in_piece, 64), dw_steps = ceil_div(N, 64);
    const int64_t most = (dx * dx_steps + dw * (dw_steps + 4)) / slots / 3;
    const int64_t least = p.parts > 1 ? 3 : 8;      // six products a step in parts
    auto cut = [&](int64_t steps, int64_t at_least, int64_t rows, int64_t limit) {
      int64_t splits = ceil_div(steps, most < at_least ? at_least : most), fits = (128LL << 20) / (4 * rows * p.Dp);
      if (splits > fits) splits = fits;
      if (splits > limit) splits = limit;
      return (int)(splits < 1 ? 1 : ceil_div(steps, ceil_div(steps, splits)));      // none without a step
    };
    p.dx_splits = cut(dx_steps, least, p.rows, 32);
    const int64_t dw_tiles = vocab_dw_tile_count(p.grads_tile, D, in_piece, p.parts);
    // dw's pieces are rows of the vocabulary each: only where it leaves CUs without a tile.  Where a piece's sums are few
    // (512 KB), shorter ones fill the CUs that dx leaves (us; rows of 512 over 100 tokens, bf16: 512 rows 29.7 / 25.2, 2000 rows
    // 37.6 / 34.1; over 500 tokens 300 rows 27 / 30, with the join that it then takes)
    const int64_t most_dw = slots / dw_tiles < 32 ? slots / dw_tiles : 32;
    p.dw_splits = p.piece < V ? 1 : cut(dw_steps, least, V, most_dw);
    if (p.piece >= V && 4 * V * p.Dp <= (512 << 10)) {
      const int64_t left = (slots - dx * p.dx_splits) / dw_tiles;
      const int shorter = cut(dw_steps, p.parts > 1 ? 2 : 3, V, left < most_dw ? left : most_dw);
      if (shorter > p.dw_splits) p.dw_splits = shorter;
    }
    p.dx_joined = p.dx_splits > 1 || p.piece < V;
    p.dw_joined = p.dw_splits > 1;
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
  p.part = take(p.logits_summed ? 0 : 8 * p.tiles * N);
  p.sums = take(p.logits_summed ? 4 * p.logits_splits * N * sums_ld : 0);
  p.x = take(2 * p.parts * p.rows * p.Dp);
  p.w = take(p.direct || p.regs ? 0 : 2 * p.parts * p.piece * p.Dp);
  p.g = take(grad ? 2 * p.g_parts * p.rows * p.piece : 0);
  p.cols = take(p.columns ? 4 * ceil_div(N, VOCAB_GROUP) * p.piece : 0);
  p.dx = take(p.dx_joined ? 4 * p.dx_splits * p.rows * p.Dp : 0);
  p.dw = take(p.dw_joined ? 4 * p.dw_splits * V * p.Dp : 0);
  p.db = take(p.dw_joined ? 4 * p.dw_splits * V : 0);
  p.bytes = at;
  return p;
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

// A rule of the plan that asks for what is not compiled is an error, not a result that is missing.
inline int vocab_no_kernel(const VocabPlan& p) {
  set_error("bf_vocab_loss: no kernel for tiles %d and %d with %d parts", p.logits_tile, p.grads_tile, p.g_parts);
  return BF_ELAUNCH;
}

// T: the tensors' type, E: the matrix products', GP: the parts of G
template <class T, class E, int GP>
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
  float* cols = (float*)(q.space + p.cols);
  float* dx = (float*)(q.space + p.dx);
  float* dw = (float*)(q.space + p.dw);
  float* db = (float*)(q.space + p.db);
  const int64_t x_part = p.rows * p.Dp, w_part = p.piece * p.Dp, g_part = p.rows * p.piece;
  const float c = (float)(1.4426950408889634 / q.temperature), inv_t = (float)(1.0 / q.temperature);
  const float scale = (float)((double)q.grad_scale / q.temperature) / (__is_same(E, _Float16) ? VOCAB_F16_SCALE : 1.f);
  const T* weight = (const T*)q.weight;
  // Without G in the way the first pass takes a weight that can be read as it lies whole; otherwise the pieces from
  // the last to the first, whose packed weight and exponentials are then there for the second pass.
  const int64_t first_piece = (p.direct || p.regs) && !p.grad ? ceil_div(p.V, 256) * 256 : p.piece;
  const int64_t pieces = ceil_div(p.V, first_piece);
  auto count_of = [&](int64_t k) { return (int)(p.V - k * first_piece < first_piece ? p.V - k * first_piece : first_piece); };

  VocabPrepare pre;
  memset(&pre, 0, sizeof(pre));
  pre.hidden = q.hidden;
  pre.ld_b = q.ld_b;
  pre.ld_t = q.ld_t;
  pre.length = (int)q.length;
  pre.tokens = q.tokens;
  pre.token_bytes = q.token_bytes;
  pre.mask = (const uint8_t*)q.mask;
  pre.N = N;
  pre.D = D;
  pre.Dp = (int)p.Dp;
  pre.live = live;
  pre.source = source;
  pre.place = place;
  pre.token = token;
  pre.logp = q.logp;
  pre.x = x;
  pre.x_part = x_part;
  pre.grad_hidden = q.grad_hidden;
  if (!p.direct && !p.regs) {
    pre.weight = weight + (pieces - 1) * first_piece * q.ld_w;
    pre.ld_w = q.ld_w;
    pre.weight_rows = count_of(pieces - 1);
    pre.w = w;
    pre.w_part = w_part;
  }
  const dim3 prepare((unsigned)(N + 64 + ceil_div(pre.weight_rows * (p.Dp / 8), 256)));
  if (N <= VOCAB_SCAN) {
    hipLaunchKernelGGL((vocab_prepare_kernel<T, E, true>), prepare, dim3(256), 0, stream, pre);
  } else {
    const dim3 counting(N > VOCAB_COUNTED_ROWS ? 1 : (unsigned)ceil_div(N, VOCAB_COUNTED));
    hipLaunchKernelGGL(vocab_rows_kernel, counting, dim3(1024), 0, stream, q.tokens, q.token_bytes, (const uint8_t*)q.mask,
                       N, live, source, place, token, q.logp);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    hipLaunchKernelGGL((vocab_prepare_kernel<T, E, false>), prepare, dim3(256), 0, stream, pre);
  }
  BF_LAUNCH_CHECK("bf_vocab_loss");

  VocabArgs a;
  memset(&a, 0, sizeof(a));
  a.live = live;
  a.elem = p.elem;
  a.splits = 1;
  a.tokens = token;
  a.c = c;
  a.part = part;
  a.part_ld = p.tiles;
  a.chosen = chosen;
  a.row = row;
  a.B = x;
  a.ldb = p.Dp;
  a.b_part = x_part;
  a.N = N;
  a.b_rows = (int)p.rows;
  a.K = (int)p.Dp;
  a.a_cols = p.direct || p.regs ? D : (int)p.Dp;
  a.ldg = p.piece;
  a.g_part = g_part;
  a.g_rows = (int)p.rows;
  // the weight's rows of a piece, as the products read them
  auto weight_rows = [&](int64_t v0, int count, bool pack) {
    a.v0 = (int)v0;
    a.M = a.a_rows = count;
    a.bias = q.bias ? (const T*)q.bias + v0 : nullptr;
    if (p.direct || p.regs) {
      a.A = weight + v0 * q.ld_w;
      a.lda = q.ld_w;
      return;
    }
    if (pack)
      hipLaunchKernelGGL((vocab_pack_weight_kernel<T, E>), dim3((unsigned)ceil_div(count * (p.Dp / 8), 256)), dim3(256), 0,
                         stream, weight + v0 * q.ld_w, q.ld_w, count, D, (int)p.Dp, w, w_part);
    a.A = w;
    a.lda = p.Dp;
    a.a_part = w_part;
  };
  for (int64_t k = pieces - 1; k >= 0; --k) {
    weight_rows(k * first_piece, count_of(k), k < pieces - 1);
    a.G = p.grad && k == 0 ? g : nullptr;
    if (p.logits_summed) {
      a.splits = p.logits_splits;
      a.sums_ld = ceil_div(p.V, 256) * 256;
      a.sums_split = N * a.sums_ld;
      a.sums = (float*)(q.space + p.sums) + k * first_piece;
    }
    const bool launched = p.logits_summed ? vocab_logits<E, PARTS ? GP : 1>(p.logits_tile, a, VM_SUMS, stream)
                                          : vocab_logits<E, GP>(p.logits_tile, a, VM_STATS, stream);
    if (!launched) return vocab_no_kernel(p);
    BF_LAUNCH_CHECK("bf_vocab_loss");
  }

  VocabSoftmax soft;
  soft.part = part;
  soft.part_ld = p.tiles;
  soft.tiles = (int)p.tiles;
  soft.tile = p.logits_tile == VT_LARGE ? VocabLarge<1>::BM : VocabMid::BM;
  soft.chosen = chosen;
  soft.token = token;
  soft.source = source;
  soft.live = live;
  soft.vocab = (int)p.V;
  soft.c = c;
  soft.inv_t = inv_t;
  soft.row = row;
  soft.logp = q.logp;
  soft.G = p.grad ? g : nullptr;
  soft.ldg = p.piece;
  soft.g_part = g_part;
  soft.held = p.grad ? (int)(ceil_div(count_of(0), 64) * 64) : 0;
  soft.chunks = p.grad ? (int)ceil_div(soft.held, VOCAB_CHUNK) : 1;
  if (p.logits_summed) {
    const VocabSoftmaxSums joined = {soft, (const float*)(q.space + p.sums), a.sums_split, a.sums_ld, p.logits_splits,
                                     (int)p.rows, q.bias, p.elem};
    if (p.V <= VOCAB_HELD_WAVE)
      hipLaunchKernelGGL((vocab_softmax_sums_kernel<E, GP, true>), dim3((unsigned)ceil_div(p.rows, 4)), dim3(256), 0, stream,
                         joined);
    else
      hipLaunchKernelGGL((vocab_softmax_sums_kernel<E, GP, false>), dim3((unsigned)p.rows), dim3(256), 0, stream, joined);
    a.splits = 1;
    a.sums = nullptr;
  } else if (p.columns) {
    VocabSoftmax stats = soft;
    stats.G = nullptr;
    stats.chunks = 1;
    hipLaunchKernelGGL((vocab_softmax_kernel<E, GP>), dim3((unsigned)N), dim3(256), 0, stream, stats);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    const int chunks = (int)ceil_div(soft.held, 2048);
    if constexpr (GP == 2) return vocab_no_kernel(p);      // two parts are summed beside dw's products
    else
      hipLaunchKernelGGL((vocab_softmax_columns_kernel<E, GP>), dim3((unsigned)(ceil_div(N, VOCAB_GROUP) * chunks)), dim3(256), 0,
                         stream, soft, chunks, cols);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    hipLaunchKernelGGL((vocab_bias_kernel<T>), dim3((unsigned)ceil_div(count_of(0), 256)), dim3(256), 0, stream, cols, p.piece,
                       count_of(0), live, VOCAB_GROUP, scale, (T*)q.grad_bias);
  } else {
    hipLaunchKernelGGL((vocab_softmax_kernel<E, GP>), dim3((unsigned)((int64_t)N * soft.chunks)), dim3(256), 0, stream, soft);
  }
  BF_LAUNCH_CHECK("bf_vocab_loss");
  if (!p.grad) {
    hipLaunchKernelGGL(vocab_loss_kernel, dim3(1), dim3(256), 0, stream, q.logp, N, live, q.loss);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    return BF_OK;
  }

  for (int64_t k = 0; k < pieces; ++k) {
    const int64_t v0 = k * first_piece;
    const int count = count_of(k);
    weight_rows(v0, count, k > 0);
    if (k > 0) {
      a.G = g;
      a.cols = p.columns ? cols : nullptr;
      if (!vocab_logits<E, GP>(p.logits_tile, a, VM_GRAD, stream)) return vocab_no_kernel(p);
      BF_LAUNCH_CHECK("bf_vocab_loss");
      if (p.columns) {
        hipLaunchKernelGGL((vocab_bias_kernel<T>), dim3((unsigned)ceil_div(count, 256)), dim3(256), 0, stream, cols, p.piece,
                           count, live, vocab_tile_rows(p.logits_tile, p.parts), scale, (T*)q.grad_bias + v0);
        BF_LAUNCH_CHECK("bf_vocab_loss");
      }
    }
    // dx: the weight's rows are k
    VocabArgs b = a;
    b.B = g;
    b.ldb = p.piece;
    b.b_part = g_part;
    b.M = D;
    b.K = (int)(ceil_div(count, 64) * 64);
    b.splits = p.dx_splits;
    b.sums = p.dx_joined ? dx : nullptr;
    b.sums_split = p.rows * p.Dp;
    b.sums_ld = p.Dp;
    b.add = k > 0;
    b.source = source;
    b.out = q.grad_hidden;
    b.out_elem = p.elem;
    b.scale = scale;
    // dw: the hidden rows are k
    VocabArgs d = b;
    d.splits = p.dw_splits;
    d.sums = p.dw_joined ? dw : nullptr;
    d.sums_split = p.V * p.Dp;
    d.db_sums = db;
    d.a_cols = (int)p.Dp;
    d.A = x;
    d.lda = p.Dp;
    d.a_part = x_part;
    d.a_rows = (int)p.rows;
    d.N = count;
    d.b_cols = (int)p.piece;
    d.out = (char*)q.grad_weight + v0 * D * elem_bytes(q.grad_weight_elem);
    d.out_elem = q.grad_weight_elem;
    d.db = q.grad_bias && !p.columns ? (T*)q.grad_bias + v0 : nullptr;
    if (!vocab_grads<E, GP>(p.grads_tile, b, d, q.logp, N, k == 0 ? q.loss : nullptr, stream)) return vocab_no_kernel(p);
    BF_LAUNCH_CHECK("bf_vocab_loss");
  }
  if (p.dx_joined || p.dw_joined) {
    VocabJoin j;
    memset(&j, 0, sizeof(j));
    j.live = live;
    j.source = source;
    if (p.dx_joined) j.dx = dx;
    j.dx_split = p.rows * p.Dp;
    j.dx_splits = p.dx_splits;
    j.N = N;
    j.grad_hidden = q.grad_hidden;
    if (p.dw_joined) j.dw = dw;
    j.dw_split = p.V * p.Dp;
    j.V = p.V;
    j.dw_splits = p.dw_splits;
    j.grad_weight = q.grad_weight;
    j.dw_elem = q.grad_weight_elem;
    if (q.grad_bias && !p.columns) j.db = db;
    j.grad_bias = q.grad_bias;
    j.D = D;
    j.ld = p.Dp;
    j.scale = scale;
    const int64_t rows = (p.dx_joined ? N : 0) + (p.dw_joined ? p.V : 0);
    hipLaunchKernelGGL((vocab_join_kernel<T>), dim3((unsigned)ceil_div(rows * ceil_div(D, 8), 256)), dim3(256), 0, stream, j);
    BF_LAUNCH_CHECK("bf_vocab_loss");
  }
  return BF_OK;
}

// Beyond, log2(e) / temperature would leave fp32's normal numbers, and 0 or infinity times the -inf of a tile's padding, or
// of a barred token, is no number.
constexpr double VOCAB_TEMPERATURE = 0x1p120;

constexpr int64_t VOCAB_ROWS = 1LL << 23, VOCAB_DIM = 1LL << 20, VOCAB_TOKENS = 1LL << 30;

inline bool vocab_sizes_ok(int64_t N, int64_t D, int64_t V, int64_t ld_w) {
  return N < VOCAB_ROWS && D <= VOCAB_DIM && V <= VOCAB_TOKENS && ld_w <= VOCAB_DIM;
}

// Every launch of a call stays below 2^32 work-items (asked before the first of them).
inline bool vocab_launches_ok(const VocabPlan& p) {
  auto products = [&](int tile, int64_t tiles) { return launch_fits(tiles + 16, tile == VT_LARGE ? 512 : 256); };
  const int64_t packed = p.direct || p.regs ? 0 : ceil_div(p.piece * (p.Dp / 8), 256);
  if (!launch_fits(p.N + 64 + packed, 256) ||
      !products(p.logits_tile, vocab_tile_count(p.logits_tile, p.V, p.N, p.parts) * p.logits_splits))
    return false;
  if (!p.grad) return true;
  const int64_t tiles = vocab_tile_count(p.grads_tile, p.D, p.N, p.parts) * p.dx_splits +
                        vocab_dw_tile_count(p.grads_tile, p.D, p.piece, p.parts) * p.dw_splits;
  const int64_t joined = (p.dx_joined ? p.N : 0) + (p.dw_joined ? p.V : 0);
  return products(p.grads_tile, tiles) && launch_fits(p.N * ceil_div(p.piece, VOCAB_CHUNK), 256) &&
         launch_fits(ceil_div(p.N, VOCAB_GROUP) * ceil_div(p.piece, 2048), 256) &&
         launch_fits(ceil_div(joined * ceil_div(p.D, 8), 256), 256);
}

}  // namespace bf

using namespace bf;

extern "C" int64_t bf_vocab_loss_workspace(int64_t N, int64_t D, int64_t V, int elem, const void* weight, int64_t ld_w,
                                           int with_grad, int with_bias, int64_t room) {
  if (!elem_ok(elem) || N <= 0 || D <= 0 || V <= 0 || ld_w < D || room < 0 || !vocab_sizes_ok(N, D, V, ld_w)) return 0;
  const VocabPlan p = vocab_plan(N, D, V, elem, weight, ld_w, with_grad != 0, with_bias != 0, room);
  return vocab_launches_ok(p) ? p.bytes / 4 : 0;
}

extern "C" int bf_vocab_loss_plan(int64_t N, int64_t D, int64_t V, int elem, const void* weight, int64_t ld_w,
                                  int with_grad, int with_bias, int64_t room, int64_t* plan) {
  BF_REQUIRE(elem_ok(elem) && N > 0 && D > 0 && V > 0 && ld_w >= D && room >= 0 && plan, "bf_vocab_loss_plan: bad arguments");
  if (!vocab_sizes_ok(N, D, V, ld_w)) {
    set_error("bf_vocab_loss_plan: more than bf_vocab_loss takes");
    return BF_ERANGE;
  }
  const VocabPlan p = vocab_plan(N, D, V, elem, weight, ld_w, with_grad != 0, with_bias != 0, room);
  plan[0] = ceil_div(V, p.piece);
  plan[1] = p.logits_tile;
  plan[2] = p.grad ? p.grads_tile : -1;
  plan[3] = p.g_parts;
  plan[4] = p.logits_summed ? p.logits_splits : 0;
  plan[5] = p.columns;
  return BF_OK;
}

extern "C" int bf_vocab_loss(const void* hidden, int elem, int64_t B, int64_t T, int64_t D, int64_t ld_b, int64_t ld_t,
                             const void* weight, int64_t V, int64_t ld_w, const void* bias, const void* tokens,
                             int token_bytes, const void* mask, double temperature, float grad_scale, float* logp,
                             float* loss, void* grad_hidden, void* grad_weight, int grad_weight_elem, void* grad_bias,
                             float* workspace, int64_t room, hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8), "bf_vocab_loss: element type %d, token bytes %d",
             elem, token_bytes);
  BF_REQUIRE(B >= 0 && T >= 0 && D > 0 && V > 0 && ld_b >= 0 && ld_t >= 0 && ld_w >= D && room >= 0,
             "bf_vocab_loss: bad sizes");
  BF_REQUIRE(temperature >= 1.0 / VOCAB_TEMPERATURE && temperature <= VOCAB_TEMPERATURE, "bf_vocab_loss: temperature %g",
             temperature);
  BF_REQUIRE(loss, "bf_vocab_loss: null pointer");
  const bool grad = grad_hidden || grad_weight || grad_bias;
  BF_REQUIRE(!grad || (grad_weight && (B * T == 0 || grad_hidden) && !bias == !grad_bias),
             "bf_vocab_loss: gradients of hidden rows and weight, and of the bias where there is one, come together");
  BF_REQUIRE(!grad || grad_weight_elem == elem || grad_weight_elem == TE_F32,
             "bf_vocab_loss: weight gradient of element type %d", grad_weight_elem);
  bool sizes = B <= VOCAB_ROWS && T <= VOCAB_ROWS && vocab_sizes_ok(B * T, D, V, ld_w);
  const int64_t cleared = sizes && grad ? ceil_div(V * D, 256 * 16) : 1;      // workgroups of a call without rows
  if (sizes && B * T == 0) sizes = launch_fits(cleared, 256);
  VocabPlan p;
  if (sizes && B * T > 0) p = vocab_plan(B * T, D, V, elem, weight, ld_w, grad, bias != nullptr, room);
  if (!sizes || (B * T > 0 && !vocab_launches_ok(p))) {
    set_error("bf_vocab_loss: %lld x %lld rows, width %lld, vocabulary %lld, weight rows %lld apart are more than it takes",
              (long long)B, (long long)T, (long long)D, (long long)V, (long long)ld_w);
    return BF_ERANGE;
  }
  const int64_t N = B * T;
  BF_REQUIRE(weight && (N == 0 || (hidden && tokens && logp && workspace)), "bf_vocab_loss: null pointer");
  BF_REQUIRE((uintptr_t)workspace % 16 == 0, "bf_vocab_loss: workspace not aligned to 16 bytes");
  if (N == 0) {
    hipLaunchKernelGGL(vocab_nothing_kernel, dim3((unsigned)cleared), dim3(256), 0, stream, loss, grad_weight, grad ? V * D : 0,
                       grad_weight_elem, grad_bias, grad_bias ? V : 0, elem);
    BF_LAUNCH_CHECK("bf_vocab_loss");
    return BF_OK;
  }
  const VocabCall q = {hidden, T, ld_b, ld_t, weight, ld_w, bias, tokens, token_bytes, mask, temperature, grad_scale, logp,
                       loss, grad_hidden, grad_weight, grad_weight_elem, grad_bias, (char*)workspace, stream};
  switch (elem) {
    case TE_F32: return vocab_run<float, __bf16, VOCAB_PARTS>(p, q);
    case TE_BF16: return p.g_parts == 2 ? vocab_run<__bf16, __bf16, 2>(p, q) : vocab_run<__bf16, __bf16, 1>(p, q);
    default: return p.g_parts == 2 ? vocab_run<_Float16, _Float16, 2>(p, q) : vocab_run<_Float16, _Float16, 1>(p, q);
  }
}
