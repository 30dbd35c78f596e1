// The three products of a head's softmax cross entropy (bf_train_vocab.hip) on the 16-bit matrix cores:
//
//   z[v, n]  = W[v, :] . X[n, :]      logits, never stored: their softmax statistics, or its gradient G
//   dX[n, d] = sum over v of G[n, v] W[v, d]
//   dW[v, d] = sum over n of G[n, v] X[n, d]
//
// One kernel does them as C[M, N] = A B^T with fp32 sums in v_mfma_f32_32x32x16.  Its first index M is the one whose
// neighbours a lane holds (four in a row of C's register layout): the vocabulary for z, so that a lane owns one
// token's logits and its statistics are sums over registers, and the width d for dX and dW, so that a lane
// stores four neighbours at once.
//
// Operands lie in memory with either index contiguous.  With k contiguous (z) a lane's eight k are 16 bytes of a row;
// otherwise (W in dX, both in dW) a stage is held as rows of k and read by ds_read_b64_tr_b16, which hands a lane four
// k of its column, so that no operand is transposed in memory.
//
// fp32 values come as three bf16 parts, x = x0 + x1 + x2 (8 + 8 + 8 significant bits); a product is the sum of six
// part products, least first: x2 y0, x0 y2, x1 y1, x1 y0, x0 y1, x0 y0, one after another along k into the same
// fp32 sums.  What is left out is 2^-24 of a product.
#pragma once

#include "bf_train.h"

namespace bf {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) char lds_char;

enum : int { VM_STATS = 0, VM_GRAD = 1, VM_DX = 2, VM_DW = 3 };

constexpr int VOCAB_BK = 64;            // k of a stage
constexpr int VOCAB_PARTS = 3, VOCAB_PAIRS = 6;
// fp16 holds G times this: p - [v = y] lies within [-1, 1], and a probability below 2^-24 would be subnormal
constexpr float VOCAB_F16_SCALE = 16384.f;

struct VocabArgs {
  const void* A;
  const void* B;
  int64_t lda, ldb;          // elements between rows (of M or N with k contiguous, of k otherwise)
  int64_t a_part, b_part;    // elements between the parts of fp32 operands
  int pairs;                 // 1, or VOCAB_PAIRS for parts
  int M, N, K;               // K a multiple of VOCAB_BK
  int a_rows, b_rows;        // rows of A and B that may be read: later ones give the last one's values
  int a_cols, b_cols;        // of operands with k in their rows: elements of a row that may be read
  const int* live;           // rows of X that count, on the device
  int splits;                // VM_DX: pieces of k, each with sums of its own
  // softmax
  const void* bias;          // [M] or null, of type `elem`
  int elem;
  const int* tokens;         // [N] less v0
  int v0;
  float c;                   // log2(e) / temperature
  float2* part;              // [tiles of M, part_ld]: largest logit and sum of 2^(c (z - it)) over the tile
  int64_t part_ld;
  float* chosen;             // [N] the token's logit
  const float2* row;         // [N] largest logit, 1 / sum
  // results
  void* G;                   // [parts, rows, ldg]
  int64_t ldg, g_part;
  int g_rows;
  float* dx;                 // [splits, dx_rows, dx_ld]
  int64_t dx_split, dx_ld;
  int dx_add;                // add to what is there
  void* dw;                  // [N, dw_ld] of type dw_elem
  int64_t dw_ld;
  int dw_elem;
  void* db;                  // [N] of type `elem`, or null
  float scale;               // of dw and db, before the division by the rows that count
};

// Tiles of BM x BN, NWM x NWN waves of 32 FM x 32 FN each.
template <int FM_, int FN_, int NWM_, int NWN_>
struct VocabTile {
  static constexpr int FM = FM_, FN = FN_, NWM = NWM_, NWN = NWN_;
  static constexpr int BM = 32 * FM * NWM, BN = 32 * FN * NWN, WAVES = NWM * NWN, NT = 64 * WAVES;
  static constexpr int A_BYTES = BM * VOCAB_BK * 2, B_BYTES = BN * VOCAB_BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
};

// 16 bytes a lane from base + off to LDS at dst + 16 lane, asynchronously (vmcnt counts it)
__device__ __forceinline__ void copy16_to_lds(const void* base, uint32_t off, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory");
}

__device__ __forceinline__ floatx16 mfma16(bf16x8v a, bf16x8v b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma16(f16x8v a, f16x8v b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <class E>
struct Vec8;
template <>
struct Vec8<__bf16> {
  typedef bf16x8v type;
};
template <>
struct Vec8<_Float16> {
  typedef f16x8v type;
};

// One operand's stages: SIDE rows or columns of the tile.
//
// LDS of a stage, in slots of 16 bytes.  k contiguous: row r of 8 slots, slot s holding chunk s ^ (r % 8), so that the
// 32 lanes which read one chunk of 32 rows meet all banks.  k in rows (TR): row k of SIDE / 8 slots, slot s holding
// chunk s ^ 4 (k % 4): the four rows of k that 16 lanes read together lie 32 bytes apart.
template <bool TR, int SIDE, int WAVES>
struct VocabOperand {
  static constexpr int COPIES = SIDE * VOCAB_BK * 2 / 1024;     // of 1 KB, one wave each
  static constexpr int PER_WAVE = (COPIES + WAVES - 1) / WAVES;
  static_assert(!TR || SIDE >= 128, "the slots' permutation spans 16 of them");
  static_assert(COPIES % WAVES == 0, "every wave makes the same copies");
  uint32_t off[PER_WAVE];   // bytes from the stage's first k
  int krow[PER_WAVE];       // TR: the row of k that a lane copies

  // first: the tile's first row (k contiguous) or column (TR)
  __device__ __forceinline__ void set(int wave, int lane, int first, int rows, int cols, int64_t ld) {
#pragma unroll
    for (int j = 0; j < PER_WAVE; ++j) {
      const int copy = wave * PER_WAVE + j;
      if constexpr (TR) {
        constexpr int SLOTS = SIDE / 8;
        const int k = copy * (64 / SLOTS) + lane / SLOTS;
        int col = first + 8 * ((lane % SLOTS) ^ (4 * (k & 3)));
        if (col > cols - 8) col = cols - 8;
        krow[j] = k;
        off[j] = (uint32_t)(2 * (k * ld + col));
      } else {
        int r = first + 8 * copy + (lane >> 3);
        if (r > rows - 1) r = rows - 1;
        off[j] = (uint32_t)(2 * ((int64_t)(r - first) * ld + 8 * ((lane & 7) ^ (lane >> 3))));
      }
    }
  }

  // `base`: the stage's first k (of the tile's first row); left: rows of k from there on (TR)
  __device__ __forceinline__ void copy(const char* base, int64_t ld, int left, int wave, uint32_t dst) const {
#pragma unroll
    for (int j = 0; j < PER_WAVE; ++j) {
      uint32_t o = off[j];
      if constexpr (TR) {
        if (left < VOCAB_BK && krow[j] >= left) o -= (uint32_t)(2 * (krow[j] - (left - 1)) * ld);
      }
      copy16_to_lds(base, o, dst + (wave * PER_WAVE + j) * 1024);
    }
  }

  // the eight k 16 kk + 8 (lane / 32) .. of row or column side + lane % 32
  template <class V>
  static __device__ __forceinline__ V read(const char* stage, int side, int kk, int lane) {
    if constexpr (TR) {
      const int g = lane >> 4, i = lane & 15;
      const int k = 16 * kk + 8 * (g >> 1) + (i >> 2), col = side + 16 * (g & 1) + 4 * (i & 3);
      const int at = k * (2 * SIDE) + (((col >> 3) ^ (4 * (i >> 2))) << 4) + 2 * (col & 7);
      const lds_char* p = (const lds_char*)stage;
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + at));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + at + 4 * (2 * SIDE)));
      return __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int r = side + (lane & 31);
      return *(const V*)(stage + r * 128 + (((2 * kk + (lane >> 5)) ^ (r & 7)) << 4));
    }
  }
};

__device__ __forceinline__ float load_elem(const void* p, int elem, int64_t i) {
  switch (elem) {
    case TE_F32: return static_cast<const float*>(p)[i];
    case TE_BF16: return (float)static_cast<const __bf16*>(p)[i];
    default: return (float)static_cast<const _Float16*>(p)[i];
  }
}

__device__ __forceinline__ void store_elem(void* p, int elem, int64_t i, float x) {
  switch (elem) {
    case TE_F32: static_cast<float*>(p)[i] = x; break;
    case TE_BF16: static_cast<__bf16*>(p)[i] = (__bf16)x; break;
    default: static_cast<_Float16*>(p)[i] = (_Float16)x;
  }
}

// x in its three bf16 parts, each the nearest to what those before it leave (infinite and NaN: the first alone)
__device__ __forceinline__ void split_parts(float x, __bf16 part[VOCAB_PARTS]) {
#pragma unroll
  for (int k = 0; k < VOCAB_PARTS; ++k) {
    part[k] = (__bf16)x;
    x = __builtin_isfinite(x) ? x - (float)part[k] : 0.f;
  }
}

template <class T, int MODE, class E, bool PARTS>
__global__ void __launch_bounds__(T::NT) vocab_gemm_kernel(VocabArgs p) {
  constexpr bool A_TR = MODE >= VM_DX, B_TR = MODE == VM_DW;
  constexpr int FM = T::FM, FN = T::FN;
  typedef typename Vec8<E>::type V8;
  typedef VocabOperand<A_TR, T::BM, T::WAVES> OpA;
  typedef VocabOperand<B_TR, T::BN, T::WAVES> OpB;
  __shared__ __attribute__((aligned(1024))) char smem[2 * T::STAGE];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int live = *p.live;
  const int N = MODE == VM_DW ? p.N : min(live, p.N);

  // Tiles in the order of groups of 8 along M, a contiguous share of them to each XCD: the 32 or 64 tiles that run on
  // one XCD at a time read 8 tiles of A and 4 or 8 of B through its L2.  Only rows that count have tiles.
  const int ntm = (p.M + T::BM - 1) / T::BM, ntn = (N + T::BN - 1) / T::BN;
  const int splits = MODE == VM_DX ? p.splits : 1;
  const int tiles = ntm * ntn * splits, share = (tiles + 7) / 8;
  int tile = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || tile >= tiles) return;
  int split = 0;
  if constexpr (MODE == VM_DX) {
    split = tile / (ntm * ntn);
    tile -= split * (ntm * ntn);
  }
  const int group = tile / (8 * ntn), in_group = tile - group * (8 * ntn);
  const int width = min(8, ntm - 8 * group);
  const int tm = 8 * group + in_group % width, tn = in_group / width;
  const int m0 = tm * T::BM, n0 = tn * T::BN;

  int steps = MODE == VM_DW ? (live + VOCAB_BK - 1) / VOCAB_BK : p.K / VOCAB_BK, k_first = 0;
  if constexpr (MODE == VM_DX) {
    const int per = (steps + splits - 1) / splits;
    k_first = split * per;
    steps = max(0, min(per, steps - k_first));
  }
  const int total = PARTS ? steps * VOCAB_PAIRS : steps;

  OpA opa;
  OpB opb;
  opa.set(wave, lane, m0, p.a_rows, p.a_cols, p.lda);
  opb.set(wave, lane, n0, p.b_rows, p.b_cols, p.ldb);
  const int64_t a_step = 2 * (A_TR ? p.lda * VOCAB_BK : VOCAB_BK), b_step = 2 * (B_TR ? p.ldb * VOCAB_BK : VOCAB_BK);
  const char* a_first = (const char*)p.A + (A_TR ? 0 : 2 * (int64_t)m0 * p.lda) + k_first * a_step;
  const char* b_first = (const char*)p.B + (B_TR ? 0 : 2 * (int64_t)n0 * p.ldb) + k_first * b_step;
  const char *a_at = a_first, *b_at = b_first;
  const uint32_t lds0 = (uint32_t)(uintptr_t)((lds_char*)smem);
  int pair = 0, ks = 0;
  if constexpr (PARTS) {
    a_at = a_first + 2 * 2 * p.a_part;   // a2 b0 first
  }

  auto issue = [&](int buffer) {
    const uint32_t dst = lds0 + buffer * T::STAGE;
    opa.copy(a_at, p.lda, A_TR ? p.a_rows - (k_first + ks) * VOCAB_BK : VOCAB_BK, wave, dst);
    opb.copy(b_at, p.ldb, B_TR ? p.b_rows - (k_first + ks) * VOCAB_BK : VOCAB_BK, wave, dst + T::A_BYTES);
    a_at += a_step;
    b_at += b_step;
    if (++ks == steps) {
      ks = 0;
      ++pair;
      if constexpr (PARTS) {
        // parts of (A, B) in turn: 2 0, 0 2, 1 1, 1 0, 0 1, 0 0
        const int pa = (0b000001010010 >> (2 * pair)) & 3, pb = (0b000100011000 >> (2 * pair)) & 3;
        a_at = a_first + 2 * pa * p.a_part;
        b_at = b_first + 2 * pb * p.b_part;
      }
    }
  };

  const int wm = (wave % T::NWM) * 32 * FM, wn = (wave / T::NWM) * 32 * FN;
  floatx16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  float col_sum[FN];
  const bool sum_cols = MODE == VM_DW && p.db && tm == 0 && wave % T::NWM == 0;
#pragma unroll
  for (int j = 0; j < FN; ++j) col_sum[j] = 0.f;

  if (total > 0) issue(0);
  for (int s = 0; s < total; ++s) {
    // this wave's copies of the stage are there, then everyone's; the other buffer's readers are done
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 1 < total) issue((s + 1) & 1);
    const char* stage = smem + (s & 1) * T::STAGE;
#pragma unroll
    for (int kk = 0; kk < VOCAB_BK / 16; ++kk) {
      V8 a[FM], b[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) a[i] = OpA::template read<V8>(stage, wm + 32 * i, kk, lane);
#pragma unroll
      for (int j = 0; j < FN; ++j) b[j] = OpB::template read<V8>(stage + T::A_BYTES, wn + 32 * j, kk, lane);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma16(a[i], b[j], acc[i][j]);
      if constexpr (MODE == VM_DW) {
        // G's column sums, the bias's gradient: every part of G once, beside the first part of X
        if (sum_cols && (!PARTS || (s >= steps && s < 2 * steps) || s >= 4 * steps)) {
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) col_sum[j] += (float)b[j][e];
        }
      }
    }
  }

  // C: this lane's column n0 + wn + 32 j + lane % 32, rows m0 + wm + 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4
  const int half = lane >> 5, ln = lane & 31;
  if constexpr (MODE == VM_STATS) {
    float* red = (float*)smem;     // [NWM][BN][2]
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + 32 * j + ln;
      const int token = n < N ? p.tokens[n] - p.v0 : -1;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3);
          float z = acc[i][j][r];
          if (p.bias && m < p.M) z += load_elem(p.bias, p.elem, m);
          if (m >= p.M) z = -INFINITY;
          if (m == token) p.chosen[n] = z;
          acc[i][j][r] = z;
          top = fmaxf(top, z);
        }
      const float held = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f((acc[i][j][r] - held) * p.c);
      float2 mine = make_float2(top, sum);
      float* at = red + 2 * ((2 * (wave % T::NWM) + half) * T::BN + wn + 32 * j + ln);
      at[0] = mine.x;
      at[1] = mine.y;
    }
    __syncthreads();
    for (int col = threadIdx.x; col < T::BN; col += T::NT) {
      if (n0 + col >= N) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 2 * T::NWM; ++w) top = fmaxf(top, red[2 * (w * T::BN + col)]);
      const float held = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 2 * T::NWM; ++w) {
        const float* at = red + 2 * (w * T::BN + col);
        // a share without a logit above -inf has no sum, but one that met a NaN has
        sum += at[1] * (at[0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((at[0] - held) * p.c));
      }
      p.part[(int64_t)tm * p.part_ld + n0 + col] = make_float2(top, sum);
    }
  } else if constexpr (MODE == VM_GRAD) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + 32 * j + ln;
      if (n >= p.g_rows) continue;
      const bool counts = n < N;
      const int token = counts ? p.tokens[n] - p.v0 : -1;
      const float2 row = counts ? p.row[n] : make_float2(0.f, 0.f);
      E* g = (E*)p.G + (int64_t)n * p.ldg;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
          if (m >= p.ldg) continue;
          Pack<E, 4> out[PARTS ? VOCAB_PARTS : 1];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = 0.f;
            if (counts && m + r < p.M) {
              float z = acc[i][j][4 * q + r];
              if (p.bias) z += load_elem(p.bias, p.elem, m + r);
              x = __builtin_amdgcn_exp2f((z - row.x) * p.c) * row.y;
              if (m + r == token) x -= 1.f;
            }
            if constexpr (PARTS) {
              __bf16 part[VOCAB_PARTS];
              split_parts(x, part);
#pragma unroll
              for (int k = 0; k < VOCAB_PARTS; ++k) out[k].v[r] = part[k];
            } else {
              if constexpr (sizeof(E) == 2 && __is_same(E, _Float16)) x *= VOCAB_F16_SCALE;
              out[0].v[r] = (E)x;
            }
          }
#pragma unroll
          for (int k = 0; k < (PARTS ? VOCAB_PARTS : 1); ++k) store_pack(g + k * p.g_part + m, out[k]);
        }
    }
  } else if constexpr (MODE == VM_DX) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + 32 * j + ln;
      if (n >= N) continue;
      float* row = p.dx + split * p.dx_split + (int64_t)n * p.dx_ld;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
          if (m >= p.dx_ld) continue;
          Pack<float, 4> x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x.v[r] = acc[i][j][4 * q + r];
          if (p.dx_add) {
            const Pack<float, 4> was = load_pack<float, 4>(row + m);
#pragma unroll
            for (int r = 0; r < 4; ++r) x.v[r] += was.v[r];
          }
          store_pack(row + m, x);
        }
    }
  } else {
    const float scale = p.scale / (float)max(live, 1);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + 32 * j + ln;
      if (sum_cols) {
        const float sum = col_sum[j] + __shfl_xor(col_sum[j], 32);
        if (half == 0 && n < N) store_elem(p.db, p.elem, n, sum * scale);
      }
      if (n >= N) continue;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
          const int64_t at = (int64_t)n * p.dw_ld + m;
          if (m + 4 <= p.M) {
            if (p.dw_elem == TE_F32) {
              Pack<float, 4> x;
#pragma unroll
              for (int r = 0; r < 4; ++r) x.v[r] = acc[i][j][4 * q + r] * scale;
              store_pack((float*)p.dw + at, x);
            } else {
              Pack<E, 4> x;
#pragma unroll
              for (int r = 0; r < 4; ++r) x.v[r] = (E)(acc[i][j][4 * q + r] * scale);
              store_pack((E*)p.dw + at, x);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (m + r < p.M) store_elem(p.dw, p.dw_elem, at + r, acc[i][j][4 * q + r] * scale);
          }
        }
    }
  }
}

template <class T, int MODE, class E, bool PARTS>
inline void launch_vocab_gemm(const VocabArgs& p, hipStream_t stream) {
  const int64_t tiles = ceil_div(p.M, T::BM) * ceil_div(p.N, T::BN) * (MODE == VM_DX ? p.splits : 1);
  const int64_t blocks = 8 * ceil_div(tiles, 8);
  hipLaunchKernelGGL((vocab_gemm_kernel<T, MODE, E, PARTS>), dim3((unsigned)blocks), dim3(T::NT), 0, stream, p);
}

}  // namespace bf
