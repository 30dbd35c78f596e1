// Token embedding of a network that trains: rows of a table by token, scaled, and the table's
// gradient.
//
//   y_i = s * table[t_i]                       (bf_embed_rows)
//   G_v = s * sum over i with t_i = v of g_i   (bf_embed_grad)
//
// The gradient is summed in fp32 over the tokens sorted by value, equal ones in their own
// order, so its bits do not depend on scheduling (adding rows with atomics, the order of the
// additions, and so the sums, would change from call to call).

#include "bf_train.h"

namespace bf {

// One thread per 16 bytes of the output.
template <class T>
__global__ void embed_rows_kernel(const T* __restrict__ table, int64_t ld, int vocab, const void* __restrict__ tokens,
                                  int token_bytes, int64_t count, int dim, int chunks, float scale,
                                  T* __restrict__ out) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t i = div_rows(at, chunks, at < (1LL << 31));
  if (i >= count) return;
  const int d0 = (int)(at - i * chunks) * VEC;
  const int t = load_token(tokens, token_bytes, i);
  T* o = out + i * (int64_t)dim + d0;
  const bool whole = d0 + VEC <= dim;
  if ((unsigned)t >= (unsigned)vocab) {
    // a negative token is padding (zeros); one past the table shows as NaN
    const T fill = (T)(t < 0 ? 0.f : __int_as_float(0x7fc00000));
    for (int k = 0; k < VEC && d0 + k < dim; ++k) o[k] = fill;
    return;
  }
  const T* row = table + (int64_t)t * ld + d0;
  if (whole) {
    Pack<T, VEC> x = load_pack<T, VEC>(row);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x.v[k] = (T)((float)x.v[k] * scale);
    store_pack(o, x);
  } else {
    for (int k = 0; d0 + k < dim; ++k) o[k] = (T)((float)row[k] * scale);
  }
}

// ---------------------------------------------------------------------------
// Sorting: a stable counting sort in one launch.  Workgroup b owns the tokens [b R, b R + R);
// it reads every token (a training batch's fit in the L2 of each XCD), counts those below its
// range, which is where its part of the order begins, and those of each of its values per wave, and
// places them.  Each of its waves reads a contiguous slice of the tokens, so equal tokens keep
// their order: slice by slice, and within 64 tokens lane by lane.
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_RANGE = 512;

inline int sort_range(int64_t vocab) {
  const int64_t r = ceil_div(vocab, 256);
  return (int)(r < SORT_RANGE ? r : SORT_RANGE);
}

__global__ __launch_bounds__(SORT_THREADS) void embed_sort_kernel(const void* __restrict__ tokens, int token_bytes,
                                                                  int count, int vocab, int range,
                                                                  int* __restrict__ start, int* __restrict__ order) {
  __shared__ int place[SORT_WAVES][SORT_RANGE];
  __shared__ int sums[SORT_WAVES], below[SORT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = blockIdx.x * range, held = min(range, vocab - v0);
  for (int k = tid; k < SORT_WAVES * SORT_RANGE; k += SORT_THREADS) (&place[0][0])[k] = 0;
  __syncthreads();
  const int slice = (int)(ceil_div(count, SORT_THREADS) * 64);
  const int from = min(wave * slice, count), to = min(from + slice, count);
  int less = 0;
  for (int i = from + lane; i < to; i += 64) {
    const int t = load_token(tokens, token_bytes, i);
    if (t >= 0 && t < v0) ++less;
    if (t >= v0 && t < v0 + held) atomicAdd(&place[wave][t - v0], 1);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) less += __shfl_xor(less, d);
  if (lane == 0) below[wave] = less;
  __syncthreads();
  // thread k < range: the number of tokens of value v0 + k, and its exclusive sum over k
  int total = 0;
  if (tid < range)
    for (int w = 0; w < SORT_WAVES; ++w) total += place[w][tid];
  int incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int base = incl - total;
  for (int w = 0; w < SORT_WAVES; ++w) {
    base += below[w];
    if (w < wave) base += sums[w];
  }
  if (tid < range) {
    if (tid < held) start[v0 + tid] = base;
    if (tid == held - 1 && v0 + held == vocab) start[vocab] = base + total;
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int n = place[w][tid];
      place[w][tid] = base;
      base += n;
    }
  }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    const int t = i < to ? load_token(tokens, token_bytes, i) : -1;
    const int k = t >= v0 && t < v0 + held ? t - v0 : -1;
    uint64_t todo = __ballot(k >= 0);
    while (todo) {   // one value of the 64 tokens at a time
      const int lead = __ffsll((unsigned long long)todo) - 1;
      const int k0 = __builtin_amdgcn_readlane(k, lead);
      const uint64_t same = __ballot(k == k0);
      if (k == k0) {
        const int at = place[wave][k0] + __popcll(same & ((1ull << lane) - 1));
        order[at] = i;
      }
      // the wave's own counter: no other wave touches it, and a wave's LDS accesses keep their order
      if (lane == lead) place[wave][k0] += __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      todo &= ~same;
    }
  }
}

// ---------------------------------------------------------------------------
// Sums.  A value that occurs at most PIECE times is summed by the workgroups of its row; a more
// frequent one is cut at the multiples of PIECE of the sorted order, every part summed by a
// workgroup of its own and the parts added in order, so a token that is half of the batch does not
// leave one workgroup with half of the work.
constexpr int PIECE = 64;
constexpr int SUM_THREADS = 256;

template <class TI, int VEC>
__device__ __forceinline__ void add_rows(float (&acc)[VEC], const TI* __restrict__ g, int64_t ld, const int* order,
                                         int from, int to, int d0, int dim) {
  if (d0 + VEC <= dim) {
    int p = from;
    for (; p + 4 <= to; p += 4) {
      Pack<TI, VEC> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = load_pack<TI, VEC>(g + order[p + u] * ld + d0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += (float)x[u].v[k];
    }
    for (; p < to; ++p) {
      const Pack<TI, VEC> x = load_pack<TI, VEC>(g + order[p] * ld + d0);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += (float)x.v[k];
    }
  } else {
    for (int p = from; p < to; ++p)
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (d0 + k < dim) acc[k] += (float)g[order[p] * ld + d0 + k];
  }
}

// `into` (fp32): the sums are added to it, and rows without a token stay as they are.
template <class TO, int VEC>
__device__ __forceinline__ void write_row(const float (&acc)[VEC], float scale, bool into, TO* __restrict__ o, int d0,
                                          int dim) {
  if (d0 + VEC <= dim) {
    Pack<TO, VEC> y;
    if (into) y = load_pack<TO, VEC>(o);
#pragma unroll
    for (int k = 0; k < VEC; ++k) y.v[k] = (TO)((into ? (float)y.v[k] : 0.f) + acc[k] * scale);
    store_pack(o, y);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (d0 + k < dim) o[k] = (TO)((into ? (float)o[k] : 0.f) + acc[k] * scale);
  }
}

// Workgroups below `row_groups`: a wave per (row, 64 VEC columns).  The others: one per piece of the
// sorted order and 256 VEC columns, for the frequent values that cross it; a piece has at most two
// (one that ends in it and one that begins in it), whose sums go to part[piece][0] and [1].
template <class TI, class TO, int VEC>
__global__ __launch_bounds__(SUM_THREADS) void embed_sum_kernel(
    const TI* __restrict__ g, int64_t ld, const void* __restrict__ tokens, int token_bytes,
    const int* __restrict__ start, const int* __restrict__ order, int vocab, int dim, int wave_chunks, int64_t row_groups,
    int group_chunks, float scale, int into, TO* __restrict__ out, float* __restrict__ part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int64_t)blockIdx.x < row_groups) {
    const int64_t at = (int64_t)blockIdx.x * (SUM_THREADS / 64) + wave;
    const int64_t v = div_rows(at, wave_chunks, at < (1LL << 31));
    if (v >= vocab) return;
    const int d0 = ((int)(at - v * wave_chunks) * 64 + lane) * VEC;
    const int from = start[v], to = start[v + 1];
    if (to - from > PIECE || (into && to == from) || d0 >= dim) return;
    float acc[VEC] = {};
    add_rows<TI, VEC>(acc, g, ld, order, from, to, d0, dim);
    write_row<TO, VEC>(acc, scale, into, out + v * dim + d0, d0, dim);
    return;
  }
  const int64_t at = (int64_t)blockIdx.x - row_groups;
  const int piece = (int)(at / group_chunks);
  const int d0 = ((int)(at % group_chunks) * SUM_THREADS + (int)threadIdx.x) * VEC;
  const int total = start[vocab], p0 = piece * PIECE, p1 = min(p0 + PIECE, total);
  if (p0 >= total || d0 >= dim) return;
  const int first = load_token(tokens, token_bytes, order[p0]), last = load_token(tokens, token_bytes, order[p1 - 1]);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int v = side ? last : first;
    const int from = start[v], to = start[v + 1];
    if (to - from <= PIECE || (side && first == last)) continue;
    float acc[VEC] = {};
    add_rows<TI, VEC>(acc, g, ld, order, max(from, p0), min(to, p1), d0, dim);
    float* o = part + ((int64_t)piece * 2 + side) * dim + d0;
    for (int k = 0; k < VEC && d0 + k < dim; ++k) o[k] = acc[k];
  }
}

// One workgroup per piece and 256 columns: where a frequent value begins in the piece, its parts
// are added in order.
template <class TO>
__global__ __launch_bounds__(SUM_THREADS) void embed_join_kernel(const void* __restrict__ tokens, int token_bytes,
                                                                 const int* __restrict__ start,
                                                                 const int* __restrict__ order, int vocab, int dim,
                                                                 int group_chunks, float scale, int into,
                                                                 TO* __restrict__ out, const float* __restrict__ part) {
  const int piece = blockIdx.x / group_chunks;
  const int d = (blockIdx.x % group_chunks) * SUM_THREADS + threadIdx.x;
  const int total = start[vocab], p0 = piece * PIECE, p1 = min(p0 + PIECE, total);
  if (p0 >= total || d >= dim) return;
  const int v = load_token(tokens, token_bytes, order[p1 - 1]);   // a value that begins here reaches its end
  const int from = start[v], to = start[v + 1];
  if (to - from <= PIECE || from < p0) return;
  const int first = load_token(tokens, token_bytes, order[p0]);
  float acc[1] = {part[((int64_t)piece * 2 + (first == v ? 0 : 1)) * dim + d]};
  for (int q = piece + 1; q * PIECE < to; ++q) acc[0] += part[(int64_t)q * 2 * dim + d];
  write_row<TO, 1>(acc, scale, into, out + (int64_t)v * dim + d, d, dim);
}

}  // namespace bf

using namespace bf;

extern "C" {

int bf_embed_rows(const void* table, int64_t table_ld, int64_t vocab, const void* tokens, int token_bytes,
                  int64_t count, int64_t dim, float scale, int elem, void* out, hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8), "bf_embed_rows: element type %d, token bytes %d",
             elem, token_bytes);
  BF_REQUIRE(vocab >= 0 && count >= 0 && dim >= 0 && table_ld >= dim, "bf_embed_rows: bad sizes");
  if (count == 0 || dim == 0) return BF_OK;
  BF_REQUIRE((table || vocab == 0) && tokens && out, "bf_embed_rows: null pointer");
  const int64_t chunks = ceil_div(dim, 16 / elem_bytes(elem)), blocks = ceil_div(count * chunks, 256);
  if (vocab >= (1LL << 31) || dim >= (1LL << 30) || blocks >= (1LL << 31)) {
    set_error("bf_embed_rows: %lld tokens of %lld columns from %lld rows are too many", (long long)count,
              (long long)dim, (long long)vocab);
    return BF_ERANGE;
  }
  return with_elem(elem, [&](auto t) -> int {
    using T = decltype(t);
    hipLaunchKernelGGL(embed_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream,
                       static_cast<const T*>(table), table_ld, (int)vocab, tokens, token_bytes, count, (int)dim,
                       (int)chunks, scale, static_cast<T*>(out));
    BF_LAUNCH_CHECK("embed_rows_kernel");
    return BF_OK;
  });
}

// start[vocab + 1], order[count], then the parts of the frequent values
int64_t bf_embed_grad_workspace(int64_t count, int64_t vocab, int64_t dim) {
  return (vocab + 1) + count + ceil_div(count, PIECE) * 2 * dim;
}

int bf_embed_grad(const void* grad, int64_t grad_ld, int elem, const void* tokens, int token_bytes, int64_t count,
                  int64_t vocab, int64_t dim, float scale, int out_elem, int accumulate, void* out, float* workspace,
                  hipStream_t stream) {
  BF_REQUIRE(elem_ok(elem) && (token_bytes == 4 || token_bytes == 8), "bf_embed_grad: element type %d, token bytes %d",
             elem, token_bytes);
  BF_REQUIRE(out_elem == elem || out_elem == TE_F32, "bf_embed_grad: a sum has the rows' type or fp32");
  BF_REQUIRE(!accumulate || out_elem == TE_F32, "bf_embed_grad: sums are added to fp32 alone");
  BF_REQUIRE(vocab >= 0 && count >= 0 && dim >= 0 && grad_ld >= dim, "bf_embed_grad: bad sizes");
  if (vocab == 0 || dim == 0 || (count == 0 && accumulate)) return BF_OK;
  BF_REQUIRE((count == 0 || (grad && tokens)) && out && workspace, "bf_embed_grad: null pointer");
  if (vocab >= (1LL << 30) || count >= (1LL << 30) || dim >= (1LL << 30)) {
    set_error("bf_embed_grad: %lld tokens, %lld values or %lld columns: each below 2^30", (long long)count,
              (long long)vocab, (long long)dim);
    return BF_ERANGE;
  }
  int* start = reinterpret_cast<int*>(workspace);
  int* order = start + vocab + 1;
  float* part = reinterpret_cast<float*>(order + count);
  const int range = sort_range(vocab);
  hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)ceil_div(vocab, range)), dim3(SORT_THREADS), 0, stream, tokens,
                     token_bytes, (int)count, (int)vocab, range, start, order);
  BF_LAUNCH_CHECK("embed_sort_kernel");
  return with_elem(elem, [&](auto ti) -> int {
    using TI = decltype(ti);
    constexpr int VEC = 16 / sizeof(TI);
    auto run = [&](auto to) -> int {
      using TO = decltype(to);
      const int64_t wave_chunks = ceil_div(dim, 64 * VEC), group_chunks = ceil_div(dim, SUM_THREADS * VEC);
      const int64_t row_groups = ceil_div(vocab * wave_chunks, SUM_THREADS / 64), pieces = ceil_div(count, PIECE);
      const int64_t join_chunks = ceil_div(dim, SUM_THREADS);
      if (row_groups + pieces * group_chunks >= (1LL << 31) || pieces * join_chunks >= (1LL << 31)) {
        set_error("bf_embed_grad: %lld rows of %lld columns are too many", (long long)vocab, (long long)dim);
        return BF_ERANGE;
      }
      hipLaunchKernelGGL((embed_sum_kernel<TI, TO, VEC>), dim3((unsigned)(row_groups + pieces * group_chunks)),
                         dim3(SUM_THREADS), 0, stream, static_cast<const TI*>(grad), grad_ld, tokens, token_bytes, start,
                         order, (int)vocab, (int)dim, (int)wave_chunks, row_groups, (int)group_chunks, scale,
                         accumulate, static_cast<TO*>(out), part);
      BF_LAUNCH_CHECK("embed_sum_kernel");
      if (count > PIECE) {
        hipLaunchKernelGGL((embed_join_kernel<TO>), dim3((unsigned)(pieces * join_chunks)), dim3(SUM_THREADS), 0,
                           stream, tokens, token_bytes, start, order, (int)vocab, (int)dim, (int)join_chunks, scale,
                           accumulate, static_cast<TO*>(out), part);
        BF_LAUNCH_CHECK("embed_join_kernel");
      }
      return BF_OK;
    };
    return out_elem == TE_F32 ? run(float()) : run(TI());
  });
}

}  // extern "C"
