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

// One thread per 16 bytes of the output.  Bound by memory: 16384 tokens of 4096 bf16 columns from 64000 rows, 42 us for
// 231 MB = 5.5 TB/s; eight tokens of 2048 columns 2.7 us, a launch.
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
// Sorting: a stable counting sort of the tokens of values [v0, v0 + held), by one workgroup.  It reads every token (a
// training batch's fit in the L2 of each XCD), counts those of each of its values per wave, and places their
// positions.  Each wave reads a contiguous slice of the tokens, so equal tokens keep their order: slice by
// slice, and within 64 tokens lane by lane.  A thread has SORT_HELD tokens under way at once; where that is all
// of them, they are read once.  Bound by latency: 16384 tokens of 32000 values 12 to 22 us by how uneven they are (the
// lanes of one value by a loop over the values took 35, loads one at a time 37).
constexpr int SORT_HELD = 16, SORT_RANGE = 512;

template <int WAVES, int RANGE>
struct SortSpace {
  int place[WAVES][RANGE];   // tokens of a value that a wave has, then where its next one goes
  int sums[WAVES], below[WAVES];
};

// f(position, i): token i's position among the range's.  begin(k, position, count): value v0 + k's part of them,
// called by one thread each; positions count from the number of tokens below v0 (BELOW) or from 0.
template <int WAVES, int RANGE, bool BELOW, class F, class G>
__device__ __forceinline__ void sort_range(const void* tokens, int token_bytes, int count, int v0, int held,
                                           SortSpace<WAVES, RANGE>& s, F f, G begin) {
  constexpr int THREADS = WAVES * 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int k = lane; k < held; k += 64) s.place[wave][k] = 0;
  __syncthreads();
  const int slice = (count + THREADS - 1) / THREADS * 64;
  const int from = min(wave * slice, count), to = min(from + slice, count);
  int t[SORT_HELD];
  const auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) {
      const int i = i0 + u * 64 + lane;
      t[u] = i < to ? load_token(tokens, token_bytes, i) : -1;
    }
  };
  int less = 0;
  for (int i0 = from; i0 < to; i0 += SORT_HELD * 64) {
    load(i0);
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) {
      if (BELOW && t[u] >= 0 && t[u] < v0) ++less;
      if (t[u] >= v0 && t[u] < v0 + held) atomicAdd(&s.place[wave][t[u] - v0], 1);
    }
  }
  if (BELOW) {
#pragma unroll
    for (int d = 32; d; d >>= 1) less += __shfl_xor(less, d);
    if (lane == 0) s.below[wave] = less;
  }
  __syncthreads();
  // thread k < RANGE: the number of tokens of value v0 + k, and its exclusive sum over k
  int total = 0;
  if (tid < held)
    for (int w = 0; w < WAVES; ++w) total += s.place[w][tid];
  int incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 63) s.sums[wave] = incl;
  __syncthreads();
  int base = incl - total;
  for (int w = 0; w < WAVES; ++w) {
    if (BELOW) base += s.below[w];
    if (w < wave) base += s.sums[w];
  }
  if (tid < held) begin(tid, base, total);
  if (tid < held)
    for (int w = 0; w < WAVES; ++w) {
      const int n = s.place[w][tid];
      s.place[w][tid] = base;
      base += n;
    }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += SORT_HELD * 64) {
    if (slice > SORT_HELD * 64) load(i0);   // else they are still held
#pragma unroll
    for (int u = 0; u < SORT_HELD; ++u) {
      const bool in = t[u] >= v0 && t[u] < v0 + held;
      uint64_t same = __ballot(in);
      if (same == 0) continue;
      // the lanes of this lane's value: those that agree with it in every bit
      const int k = in ? t[u] - v0 : 0;
      for (int b = 1; b < held; b <<= 1) {
        const uint64_t ones = __ballot(k & b);
        same &= k & b ? ones : ~ones;
      }
      // the counters are the wave's own: no other wave touches them, and a wave's LDS accesses keep their order
      if (in) {
        const int at = s.place[wave][k], before = __popcll(same & ((1ull << lane) - 1));
        f(at + before, i0 + u * 64 + lane);
        if (before == 0) s.place[wave][k] = at + __popcll(same);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

constexpr int SORT_WAVES = 16;
constexpr int64_t FILL_BYTES = 65536;   // of a workgroup

// start[v]: the first place of value v's tokens in order[], start[vocab]: the end.  The workgroups from `groups` on
// clear `fill_bytes` at `fill` meanwhile: the sort waits on the caches, and leaves the memory to them.
__global__ __launch_bounds__(SORT_WAVES * 64) void embed_sort_kernel(const void* __restrict__ tokens, int token_bytes,
                                                                    int count, int vocab, int range, int groups,
                                                                    int* __restrict__ start, int* __restrict__ order,
                                                                    char* __restrict__ fill, int64_t fill_bytes) {
  __shared__ SortSpace<SORT_WAVES, SORT_RANGE> space;
  if ((int)blockIdx.x >= groups) {
    const int64_t at = ((int64_t)blockIdx.x - groups) * FILL_BYTES + threadIdx.x * 16;
    const Words zero = zero_words();
#pragma unroll
    for (int64_t k = 0; k < FILL_BYTES; k += SORT_WAVES * 64 * 16)
      if (at + k + 16 <= fill_bytes) __builtin_memcpy(fill + at + k, &zero, 16);
    // what is left of the last 16 bytes (elements are 2 or 4)
    const int64_t rest = fill_bytes & ~(int64_t)15;
    if ((int)blockIdx.x == groups && (int64_t)threadIdx.x * 2 < fill_bytes - rest)
      reinterpret_cast<uint16_t*>(fill + rest)[threadIdx.x] = 0;
    return;
  }
  const int v0 = blockIdx.x * range, held = min(range, vocab - v0);
  sort_range<SORT_WAVES, SORT_RANGE, true>(
      tokens, token_bytes, count, v0, held, space, [&](int at, int i) { order[at] = i; },
      [&](int k, int at, int n) {
        start[v0 + k] = at;
        if (v0 + k == vocab - 1) start[vocab] = at + n;
      });
}

// ---------------------------------------------------------------------------
// Sums.

// acc[u] += rows list[first .. first + n) (lane l holds list[l]) at chunk c + u * step of 64 VEC columns, U chunks
// of TOKENS tokens under way together.  WHOLE: the chunks lie within the row; else U is 1.  What is the same in
// the wave (row, chunk) stays in scalar registers: a row of few tokens is bound by its instructions.
template <bool WHOLE, int TOKENS, int U, class TI, int VEC>
__device__ __forceinline__ void add_rows(float (&acc)[U][VEC], const TI* __restrict__ g, int64_t ld, int list, int first,
                                         int n, int c, int step, int dim) {
  const unsigned lane = threadIdx.x & 63;
  const auto load = [&](Pack<TI, VEC>(&x)[U], int p) {
    const TI* row = g + (int64_t)__builtin_amdgcn_readlane(list, first + p) * ld + c * (64 * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const TI* at = row + u * step * (64 * VEC) + lane * VEC;
      const int d = c * 64 * VEC + (int)lane * VEC;
      if (WHOLE || d + VEC <= dim) {
        x[u] = load_pack<TI, VEC>(at);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[u].v[k] = d + k < dim ? at[k] : (TI)0.f;
      }
    }
  };
  const auto add = [&](const Pack<TI, VEC>(&x)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[u][k] += (float)x[u].v[k];
  };
  int p = 0;
  for (; p + TOKENS <= n; p += TOKENS) {
    Pack<TI, VEC> x[TOKENS][U];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) load(x[i], p + i);
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) add(x[i]);
  }
  for (; p < n; ++p) {
    Pack<TI, VEC> x[U];
    load(x, p);
    add(x);
  }
}

// `into` (fp32): the sums are added to it, and rows without a token stay as they are.
template <class TO, int VEC>
__device__ __forceinline__ void write_row(const float (&acc)[VEC], float scale, bool into, TO* __restrict__ o, int left) {
  if (left >= VEC) {
    Pack<TO, VEC> y;
    if (into) y = load_pack<TO, VEC>(o);
#pragma unroll
    for (int k = 0; k < VEC; ++k) y.v[k] = (TO)((into ? (float)y.v[k] : 0.f) + acc[k] * scale);
    store_pack(o, y);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (k < left) o[k] = (TO)((into ? (float)o[k] : 0.f) + acc[k] * scale);
  }
}

// Row `row` of the table from n rows of list, chunks wave, wave + WAVES, ..., by each wave.
template <int WAVES, class TI, class TO, int VEC>
__device__ __forceinline__ void sum_row(const TI* __restrict__ g, int64_t ld, int list, int first, int n, int wave,
                                        int dim, float scale, bool into, TO* __restrict__ row) {
  constexpr int WIDTH = 64 * VEC;
  const unsigned lane = threadIdx.x & 63;
  const int whole = dim / WIDTH;   // chunks
  int c = wave;
  if (n == 0) {   // not with `into`
    const Words zero = zero_words();
    constexpr int EACH = 16 / sizeof(TO);   // elements of a store: VEC, or half of it in fp32 from 16-bit rows
    for (; c < whole; c += WAVES)
#pragma unroll
      for (int e = 0; e < VEC; e += EACH) __builtin_memcpy(row + c * WIDTH + lane * VEC + e, &zero, 16);
  } else {
    for (; c + WAVES < whole; c += 2 * WAVES) {
      float acc[2][VEC] = {};
      add_rows<true, 2, 2>(acc, g, ld, list, first, n, c, WAVES, dim);
      write_row<TO, VEC>(acc[0], scale, into, row + c * WIDTH + lane * VEC, VEC);
      write_row<TO, VEC>(acc[1], scale, into, row + (c + WAVES) * WIDTH + lane * VEC, VEC);
    }
    if (c < whole) {
      float acc[1][VEC] = {};
      add_rows<true, 4, 1>(acc, g, ld, list, first, n, c, WAVES, dim);
      write_row<TO, VEC>(acc[0], scale, into, row + c * WIDTH + lane * VEC, VEC);
      c += WAVES;
    }
  }
  if (c * WIDTH < dim) {   // the rest of the columns, by the wave whose turn it is
    const int d = c * WIDTH + (int)lane * VEC;
    float acc[1][VEC] = {};
    add_rows<false, 4, 1>(acc, g, ld, list, first, n, c, WAVES, dim);
    write_row<TO, VEC>(acc[0], scale, into, row + d, dim - d);
  }
}

// A value that occurs at most PIECE times is summed with the ROWS rows of its workgroup: the starts of both come in one
// load and the positions of all their tokens in another.  More rows a workgroup spare waits and lengthen its chain of
// rows: with 8, 4 and 2, 72, 60 and 54 us for 16384 tokens of 32000 values, 4096 bf16 columns.  A more frequent value is
// cut at the multiples of PIECE of the sorted order, every part summed by a wave of its own and the parts added in
// order, so a token that is half of the batch does not leave one wave with half of the work.
constexpr int SUM_THREADS = 256, SUM_WAVES = SUM_THREADS / 64;
constexpr int ROWS = 2, PIECE = 8;

// Workgroups below `piece_groups`: a wave per piece, for the frequent values that cross it; a piece has at most two (one
// that ends in it and one that begins in it), whose sums go to part[piece][0] and [1]; owner[piece]: the one that
// begins.  The others: one per ROWS rows.
template <class TI, class TO, int VEC>
__global__ __launch_bounds__(SUM_THREADS) void embed_sum_kernel(
    const TI* __restrict__ g, int64_t ld, const void* __restrict__ tokens, int token_bytes,
    const int* __restrict__ start, const int* __restrict__ order, int vocab, int dim, int pieces, int piece_groups, float scale, int into,
    int cleared, TO* __restrict__ out, int* __restrict__ owner, float* __restrict__ part) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x >= piece_groups) {
    const int v0 = ((int)blockIdx.x - piece_groups) * ROWS;
    const int v = min(v0 + min(lane / PIECE, ROWS - 1), vocab - 1);
    const int from = start[v], number = start[v + 1] - from;
    const int list = lane % PIECE < number ? order[from + lane % PIECE] : 0;
    for (int k = 0; k < ROWS && v0 + k < vocab; ++k) {
      const int n = __builtin_amdgcn_readlane(number, k * PIECE);
      if (n > PIECE || (cleared && n == 0)) continue;
      sum_row<SUM_WAVES, TI, TO, VEC>(g, ld, list, k * PIECE, n, wave, dim, scale, into, out + (int64_t)(v0 + k) * dim);
    }
    return;
  }
  const int piece = blockIdx.x * SUM_WAVES + wave, total = start[vocab], p0 = piece * PIECE, p1 = min(p0 + PIECE, total);
  if (piece >= pieces) return;
  if (p0 >= total) {
    if (lane == 0) owner[piece] = -1;
    return;
  }
  const int mine = p0 + lane < p1 ? order[p0 + lane] : 0;
  const int first = load_token(tokens, token_bytes, __builtin_amdgcn_readfirstlane(mine));
  const int last = load_token(tokens, token_bytes, __builtin_amdgcn_readlane(mine, p1 - 1 - p0));
  const int first_end = start[first + 1], first_all = first_end - start[first];
  const int last_from = start[last], last_all = start[last + 1] - last_from;
  if (lane == 0) owner[piece] = last_all > PIECE && last_from >= p0 ? last : -1;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if ((side ? last_all : first_all) <= PIECE || (side && first == last)) continue;
    const int from = side ? last_from - p0 : 0, to = side ? p1 - p0 : min(first_end, p1) - p0;
    sum_row<1, TI, float, VEC>(g, ld, mine, from, to - from, 0, dim, 1.f, false,
                               part + ((int64_t)piece * 2 + side) * dim);
  }
}

// Where a frequent value begins in a piece, its parts are added in order, a quarter of them by each quarter of the
// workgroup and the quarters together.  Workgroup = (`each_pieces` pieces, JOIN_COLUMNS columns, four a thread).
constexpr int JOIN_PARTS = 4, JOIN_THREADS = 1024, JOIN_COLUMNS = JOIN_THREADS / JOIN_PARTS * 4;

template <class TO>
__global__ __launch_bounds__(JOIN_THREADS) void embed_join_kernel(
    const void* __restrict__ tokens, int token_bytes, const int* __restrict__ start, const int* __restrict__ order, int dim,
    int pieces, int each_pieces, int columns, float scale, int into, const int* __restrict__ owner, TO* __restrict__ out,
    const float* __restrict__ part) {
  __shared__ float4 sums[JOIN_PARTS][JOIN_COLUMNS / 4];
  const int piece0 = blockIdx.x / (unsigned)columns * each_pieces, lane = threadIdx.x & 63;
  const int x = threadIdx.x % (JOIN_COLUMNS / 4), quarter = threadIdx.x / (JOIN_COLUMNS / 4);
  const int d = (blockIdx.x % (unsigned)columns) * JOIN_COLUMNS + x * 4;
  const int mine = lane < each_pieces && piece0 + lane < pieces ? owner[piece0 + lane] : -1;
  uint64_t todo = __ballot(mine >= 0);   // the same in every wave
  while (todo) {
    const int k = __ffsll((unsigned long long)todo) - 1, piece = piece0 + k;
    todo &= todo - 1;
    const int v = __builtin_amdgcn_readlane(mine, k);
    const int count = (start[v + 1] - 1) / PIECE - piece + 1, each = (count + JOIN_PARTS - 1) / JOIN_PARTS;
    const int end = min((quarter + 1) * each, count);
    // the value is its first piece's last, and the others' first
    const int side = load_token(tokens, token_bytes, order[piece * PIECE]) == v ? 0 : 1;
    float acc[4] = {};
    if (d < dim) {
#pragma unroll 4
      for (int q = quarter * each; q < end; ++q) {
        const float* at = part + ((int64_t)(piece + q) * 2 + (q == 0 ? side : 0)) * dim + d;
        if (d + 4 <= dim) {
          const Pack<float, 4> y = load_pack<float, 4>(at);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += y.v[e];
        } else {
          for (int e = 0; d + e < dim; ++e) acc[e] += at[e];
        }
      }
    }
    sums[quarter][x] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (quarter == 0 && d < dim) {
      float sum[4] = {};
#pragma unroll
      for (int w = 0; w < JOIN_PARTS; ++w) {
        const float4 y = sums[w][x];
        sum[0] += y.x;
        sum[1] += y.y;
        sum[2] += y.z;
        sum[3] += y.w;
      }
      write_row<TO, 4>(sum, scale, into, out + (int64_t)v * dim + d, dim - d);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Few tokens: everything in one launch.  A workgroup sorts the tokens of its rows into LDS and sums `width` columns of
// them, a wave per row; rows of more than FEW_ALONE tokens are taken by all its waves, a part each.  Bound by latency:
// 600 tokens of 1003 values, 129 fp32 columns 9.5 us (three launches: 23), and by the writing of large tables.
constexpr int FEW_TOKENS = 2048, FEW_WAVES = 8, FEW_RANGE = 128, FEW_ALONE = 8;

template <class TI, class TO, int VEC>
__global__ __launch_bounds__(FEW_WAVES * 64) void embed_few_kernel(const TI* __restrict__ g, int64_t ld,
                                                                  const void* __restrict__ tokens, int token_bytes,
                                                                  int count, int vocab, int dim, int range, int width,
                                                                  int slices, float scale, int into,
                                                                  TO* __restrict__ out) {
  __shared__ SortSpace<FEW_WAVES, FEW_RANGE> space;
  __shared__ int order[FEW_TOKENS], begin[FEW_RANGE], number[FEW_RANGE];
  __shared__ float sums[2][FEW_WAVES][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int v0 = (int)(blockIdx.x / (unsigned)slices) * range, held = min(range, vocab - v0);
  const int d0 = (int)(blockIdx.x % (unsigned)slices) * width, columns = min(width, dim - d0);
  const int chunks = (columns + 64 * VEC - 1) / (64 * VEC);
  g += d0;
  out += d0;
  sort_range<FEW_WAVES, FEW_RANGE, false>(
      tokens, token_bytes, count, v0, held, space, [&](int at, int i) { order[at] = i; },
      [&](int k, int at, int n) {
        begin[k] = at;
        number[k] = n;
      });
  __syncthreads();
  for (int k0 = 0; k0 < held; k0 += 64) {   // 64 rows' counts at a time, a lane each: one wait for all of them
    const bool mine = k0 + lane < held;
    const int n_of = mine ? number[k0 + lane] : 0, begin_of = mine ? begin[k0 + lane] : 0;
    uint64_t todo = __ballot(mine && (lane & (FEW_WAVES - 1)) == wave && n_of <= FEW_ALONE && !(into && n_of == 0));
    while (todo) {
      const int k = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      const int n = __builtin_amdgcn_readlane(n_of, k), at = __builtin_amdgcn_readlane(begin_of, k);
      const int list = lane < n ? order[at + lane] : 0;
      sum_row<1, TI, TO, VEC>(g, ld, list, 0, n, 0, columns, scale, into, out + (int64_t)(v0 + k0 + k) * dim);
    }
  }
  int buf = 0;
  uint64_t many = 0;
  for (int k0 = -64;;) {   // the frequent values, the same in the whole workgroup
    while (!many) {
      k0 += 64;
      if (k0 >= held) return;
      many = __ballot(k0 + lane < held && number[k0 + lane] > FEW_ALONE);
    }
    const int k = k0 + __ffsll((unsigned long long)many) - 1;
    many &= many - 1;
    const int n = __builtin_amdgcn_readfirstlane(number[k]);
    const int each = (n + FEW_WAVES - 1) / FEW_WAVES, q1 = min((wave + 1) * each, n);
    TO* row = out + (int64_t)(v0 + k) * dim;
    for (int c = 0; c < chunks; ++c, buf ^= 1) {
      float acc[1][VEC] = {};
      for (int q = wave * each; q < q1; q += 64) {
        const int here = min(64, q1 - q), list = lane < here ? order[begin[k] + q + lane] : 0;
        if ((c + 1) * 64 * VEC <= columns) add_rows<true, 8, 1>(acc, g, ld, list, 0, here, c, 0, columns);
        else add_rows<false, 4, 1>(acc, g, ld, list, 0, here, c, 0, columns);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[buf][wave][lane * VEC + e] = acc[0][e];
      __syncthreads();   // the other buffer is read before the barrier of the chunk that fills it again
      for (int x = threadIdx.x; x < 64 * VEC; x += FEW_WAVES * 64) {
        float sum[1] = {0.f};
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) sum[0] += sums[buf][w][x];
        const int d = c * 64 * VEC + x;
        if (d < columns) write_row<TO, 1>(sum, scale, into, row + d, 1);
      }
    }
  }
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
  if (vocab >= (1LL << 31) || dim >= (1LL << 30) || count >= (1LL << 32)) {
    set_error("bf_embed_rows: %lld tokens of %lld columns from %lld rows are too many", (long long)count,
              (long long)dim, (long long)vocab);
    return BF_ERANGE;
  }
  return with_elem(elem, [&](auto t) -> int {
    using T = decltype(t);
    // 64 GiB of rows are a launch each
    const int64_t chunks = ceil_div(dim, 16 / (int64_t)sizeof(T)), most = ((1LL << 32) - 256) / chunks;
    for (int64_t i = 0; i < count; i += most) {
      const int64_t here = count - i < most ? count - i : most;
      hipLaunchKernelGGL(embed_rows_kernel<T>, dim3((unsigned)ceil_div(here * chunks, 256)), dim3(256), 0, stream,
                         static_cast<const T*>(table), table_ld, (int)vocab,
                         static_cast<const char*>(tokens) + i * token_bytes, token_bytes, here, (int)dim, (int)chunks,
                         scale, static_cast<T*>(out) + i * dim);
      BF_LAUNCH_CHECK("embed_rows_kernel");
    }
    return BF_OK;
  });
}

// start[vocab + 1], order[count], owner and parts of the pieces; nothing for few tokens
int64_t bf_embed_grad_workspace(int64_t count, int64_t vocab, int64_t dim) {
  return count <= FEW_TOKENS ? 0 : (vocab + 1) + count + ceil_div(count, PIECE) * (1 + 2 * dim);
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
  BF_REQUIRE((count == 0 || (grad && tokens)) && out && (workspace || count <= FEW_TOKENS),
             "bf_embed_grad: null pointer");
  const int64_t pieces = ceil_div(count, PIECE), columns = ceil_div(dim, JOIN_COLUMNS);
  const auto too_many = [&] {
    set_error("bf_embed_grad: %lld tokens, %lld values or %lld columns are too many", (long long)count,
              (long long)vocab, (long long)dim);
    return BF_ERANGE;
  };
  if (vocab >= (1LL << 30) || count >= (1LL << 30) || dim >= (1LL << 30)) return too_many();
  return with_elem(elem, [&](auto ti) -> int {
    using TI = decltype(ti);
    constexpr int VEC = 16 / sizeof(TI);
    auto run = [&](auto to) -> int {
      using TO = decltype(to);
      const TI* g = static_cast<const TI*>(grad);
      TO* o = static_cast<TO*>(out);
      if (count <= FEW_TOKENS) {
        // 1024 workgroups and more where there is work for them (a CU holds three at a time with 16-bit rows and five
        // with fp32 ones: 46 and 30 KB of LDS).  The frequent values are mostly neighbours, so a
        // workgroup with all columns of its rows would be left with most of the sums: it takes a step's columns of
        // them, or more where that made more than 2048 workgroups, because every one sorts for itself.  2048
        // tokens of 32000 values, 4096 bf16 columns 75 us (all columns of 16 rows: 120), 1500 of 8000, 768 fp32 columns
        // 15 (30).
        int64_t width = 64 * VEC;
        while (width < dim && ceil_div(vocab, FEW_RANGE) * ceil_div(dim, width) > 2048) width *= 2;
        const int64_t slices = ceil_div(dim, width), r = ceil_div(vocab * slices, 1024);
        // pieces of many rows that are all written come in more workgroups: 1000 tokens of 60000 values, 3800 fp16
        // columns 124 us against 135
        const int64_t most = !accumulate && slices > 1 ? FEW_RANGE / 2 : FEW_RANGE;
        const int range = (int)(r < most ? r : most);
        const int64_t few = ceil_div(vocab, range) * slices;
        if (!launch_fits(few, FEW_WAVES * 64)) return too_many();
        hipLaunchKernelGGL((embed_few_kernel<TI, TO, VEC>), dim3((unsigned)few), dim3(FEW_WAVES * 64), 0, stream, g,
                           grad_ld, tokens, token_bytes, (int)count, (int)vocab, (int)dim, range, (int)width,
                           (int)slices, scale, accumulate, o);
        BF_LAUNCH_CHECK("embed_few_kernel");
        return BF_OK;
      }
      int* start = reinterpret_cast<int*>(workspace);
      int* order = start + vocab + 1;
      int* owner = order + count;
      float* part = reinterpret_cast<float*>(owner + pieces);
      const int64_t r = ceil_div(vocab, 256);
      const int range = (int)(r < SORT_RANGE ? r : SORT_RANGE);
      // The rows without a token are written with the others, or cleared with them while the tokens are sorted,
      // which writes the others twice: 32000 rows of 4096 bf16 columns, 16384 tokens (a third of the values), 111 us
      // against 104.
      const bool clear = !accumulate && count <= vocab;
      const int64_t groups = ceil_div(vocab, range), bytes = clear ? vocab * dim * (int64_t)sizeof(TO) : 0;
      const int64_t fills = ceil_div(bytes, FILL_BYTES);
      const int64_t piece_groups = ceil_div(pieces, SUM_WAVES);
      // narrow rows: fewer values one after another; wide ones have workgroups enough
      const int each_pieces = columns == 1 ? 2 : 8;
      const int64_t sums = piece_groups + ceil_div(vocab, ROWS), joins = ceil_div(pieces, each_pieces) * columns;
      if (!launch_fits(groups + fills, SORT_WAVES * 64) || !launch_fits(sums, SUM_THREADS) ||
          !launch_fits(joins, JOIN_THREADS))
        return too_many();
      hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)(groups + fills)), dim3(SORT_WAVES * 64), 0, stream, tokens,
                         token_bytes, (int)count, (int)vocab, range, (int)groups, start, order, static_cast<char*>(out),
                         bytes);
      BF_LAUNCH_CHECK("embed_sort_kernel");
      hipLaunchKernelGGL((embed_sum_kernel<TI, TO, VEC>), dim3((unsigned)sums), dim3(SUM_THREADS), 0, stream, g,
                         grad_ld, tokens, token_bytes, start, order, (int)vocab, (int)dim, (int)pieces,
                         (int)piece_groups, scale, accumulate, accumulate || clear, o, owner, part);
      BF_LAUNCH_CHECK("embed_sum_kernel");
      hipLaunchKernelGGL((embed_join_kernel<TO>), dim3((unsigned)joins), dim3(JOIN_THREADS), 0, stream, tokens,
                         token_bytes, start, order, (int)dim, (int)pieces, each_pieces, (int)columns, scale, accumulate, owner, o, part);
      BF_LAUNCH_CHECK("embed_join_kernel");
      return BF_OK;
    };
    return out_elem == TE_F32 ? run(float()) : run(TI());
  });
}

}  // extern "C"
