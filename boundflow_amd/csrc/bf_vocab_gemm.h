// The three products of a head's softmax cross entropy (bf_train_vocab.hip) on the 16-bit matrix cores:
//
//   z[v, n]  = W[v, :] . X[n, :]      logits, not kept: their softmax statistics and exponentials, or the softmax's gradient G
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
// Up to 64 rows, and where a bias's gradient is asked for of few tiles, G comes as two 16-bit parts: the products are not the
// time there, and a rounding of it to one adds to the results' own (vocab_plan has the figures).
//
// fp32 values come as three bf16 parts, x = x0 + x1 + x2 (8 + 8 + 8 significant bits); a product is the sum of six
// part products, least first: x0 y2, x1 y1, x2 y0, x0 y1, x1 y0, x0 y0, into the same fp32 sums.  What is left out is
// 2^-24 of a product, for values from 2^-103 up: of smaller ones what lies below 2^-126 counts as 0.  A stage holds the
// three parts of both operands, each read from LDS once for two products (the six one after another along k, a part of
// each operand in a stage: 2048 x 1024 rows over 32000 tokens 2041 us in the place of 1667, a head of eight actions 45 us
// in the place of 40).
#pragma once

#include "bf_train.h"

namespace bf {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) char lds_char;

enum : int { VM_STATS = 0, VM_GRAD = 1, VM_SUMS = 2, VM_DX = 3, VM_DW = 4 };

// z's tiles end in one of three ways.  VM_STATS: the tile's largest logit and sum of exponentials per token, and where G is
// given the exponentials themselves, 2^(c (z - the tile's largest)); vocab_softmax_kernel makes them G in place.  VM_GRAD,
// with the rows' statistics known: G.  VM_SUMS: sums over a part of k each, of a problem with so few tiles that they are
// cut along k (a CU takes 40 GB/s from memory, so few CUs take long); vocab_softmax_sums_kernel joins them.

constexpr int VOCAB_BK = 64;            // k come in multiples of this
constexpr int VOCAB_PARTS = 3;
// fp16 holds G times this: p - [v = y] lies within [-1, 1], and a probability below 2^-24 would be subnormal
constexpr float VOCAB_F16_SCALE = 16384.f;
// Exponentials, at most 1, wait for their row's statistics as fp16 times this, whichever 16-bit type G has: 11 bits down to
// 2^-29, and 0 below 2^-40.
constexpr float VOCAB_E_SCALE = 32768.f;

struct VocabArgs {
  const void* A;
  const void* B;
  int64_t lda, ldb;          // elements between rows (of M or N with k contiguous, of k otherwise)
  int64_t a_part, b_part;    // elements between the parts of fp32 operands
  int M, N, K;               // K a multiple of VOCAB_BK
  int a_rows, b_rows;        // rows of A and B that may be read: later ones give the last one's values
  int a_cols, b_cols;        // of operands with k in their rows: elements of a row that may be read
  const int* live;           // rows of X that count, on the device
  int splits;                // VM_SUMS, VM_DX, VM_DW: pieces of k, each with sums of its own
  int elem;                  // of the call's tensors
  // softmax
  const void* bias;          // [M] or null
  const int* tokens;         // [N]
  int v0;                    // the token that row 0 of A stands for
  float c;                   // log2(e) / temperature
  float2* part;              // [N, part_ld]: largest logit and sum of 2^(c (z - it)) over a tile
  int64_t part_ld;
  float* chosen;             // [N] the token's logit
  const float2* row;         // [N] largest logit, 1 / sum
  void* G;                   // [parts, g_rows, ldg], or null (VM_STATS)
  int64_t ldg, g_part;
  int g_rows;
  float* cols;               // VM_GRAD: [tiles along N, ldg] sums of G's columns over a tile's rows, or null
  // gradients
  float* sums;               // [splits, rows, sums_ld], to be joined later, or null: results are final and go to `out`
  int64_t sums_split, sums_ld;
  int add;                   // add to the sums that are there
  const int* source;         // VM_DX without sums: the row of out that row n is
  void* out;                 // dense rows of M: VM_DX of type elem, VM_DW of type out_elem
  int out_elem;
  void* db;                  // VM_DW: [N] of type elem, or null
  float* db_sums;            // [splits, N] in its place, where there are sums
  float scale;               // of out and db, before the division by the rows that count
};

// Tiles of BM x BN, NWM x NWN waves of 32 FM x 32 FN each; STAGES of LDS, OCC workgroups on a CU; parts of A and of B in a
// stage, whose products with parts i and j of i + j < max(PA, PB) are summed.
template <int FM_, int FN_, int NWM_, int NWN_, int STAGES_, int OCC_, int PA_, int PB_>
struct VocabTile {
  static constexpr int FM = FM_, FN = FN_, NWM = NWM_, NWN = NWN_, STAGES = STAGES_, OCC = OCC_, PA = PA_, PB = PB_;
  static constexpr int BK = PA == VOCAB_PARTS ? 32 : 64;   // k of a stage
  static constexpr int BM = 32 * FM * NWM, BN = 32 * FN * NWN, WAVES = NWM * NWN, NT = 64 * WAVES;
  static constexpr int A_PLANE = BM * BK * 2, B_PLANE = BN * BK * 2, A_BYTES = PA * A_PLANE;
  static constexpr int STAGE = A_BYTES + PB * B_PLANE;
  // behind the stages: the bias of the tile's rows, two floats per column from each half of a wave along M
  static constexpr int BIAS_AT = STAGES * STAGE, RED_AT = BIAS_AT + 4 * BM, LDS = RED_AT + 2 * 4 * 2 * NWM * BN;
  static constexpr int TILE = 2 * BM * BN;   // of 16-bit results
};

// 16 bytes a lane from base + off to LDS at dst + 16 lane, asynchronously (vmcnt counts it)
__device__ __forceinline__ void copy16_to_lds(const void* base, uint32_t off, uint32_t dst) {
  asm volatile(BF_COPY_TO_LDS("global_load_lds_dwordx4", "%0, %1", "%2") ::"v"(off), "s"(base), "s"(dst) : "memory", "m0");
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

// One operand's stages: SIDE rows or columns of the tile, BK k of them.
//
// LDS of a stage, in slots of 16 bytes.  k contiguous: row r of BK / 8 slots, slot s holding chunk s ^ swap(r), so that the
// 16 lanes which read one chunk of 16 rows together meet all 64 banks (r % 8 in the place of r / 2 % 8 for 64 k: half of
// them, twice; the reads of z took twice their cycles).  k in rows (TR): row k of SIDE / 8 slots, slot s holding
// chunk s ^ swap(k): 32 lanes read 64 bytes of four rows of k together, which meet all banks.
template <bool TR, int SIDE, int WAVES, int BK>
struct VocabOperand {
  static constexpr int COPIES = SIDE * BK * 2 / 1024;     // of 1 KB, one wave each
  static constexpr int PER_WAVE = (COPIES + WAVES - 1) / WAVES;
  static constexpr int SLOTS = TR ? SIDE / 8 : BK / 8, ROWS = 64 / SLOTS;   // slots of a row, rows of a copy
  static_assert(!TR || SIDE >= 64, "the slots' permutation spans 8 of them, or 16");
  static_assert(COPIES % WAVES == 0, "every wave makes the same copies");
  uint32_t off[PER_WAVE];   // bytes from the stage's first k

  static __device__ __forceinline__ int swap(int row) {
    if (TR) return SIDE >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
    return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
  }
  // the row and the chunk of eight elements of it that a lane copies
  static __device__ __forceinline__ int row(int copy, int lane) { return copy * ROWS + lane / SLOTS; }
  static __device__ __forceinline__ int chunk(int copy, int lane) { return (lane % SLOTS) ^ swap(row(copy, lane)); }

  // first: the tile's first row (k contiguous) or column (TR)
  __device__ __forceinline__ void set(int wave, int lane, int first, int rows, int cols, int64_t ld) {
#pragma unroll
    for (int j = 0; j < PER_WAVE; ++j) {
      const int copy = wave * PER_WAVE + j, r = row(copy, lane), c = 8 * chunk(copy, lane);
      if constexpr (TR) off[j] = (uint32_t)(2 * (r * ld + min(first + c, cols - 8)));
      else off[j] = (uint32_t)(2 * (min(r, rows - 1 - first) * ld + c));
    }
  }

  // `base`: the stage's first k (of the tile's first row)
  __device__ __forceinline__ void copy(const char* base, int wave, uint32_t dst) const {
#pragma unroll
    for (int j = 0; j < PER_WAVE; ++j) copy16_to_lds(base, off[j], dst + (wave * PER_WAVE + j) * 1024);
  }

  // The same of a stage that only `left` k are left for: the last row of them (TR), or the last eight of a row, stand for those
  // that are missing, whose counterparts in the other operand are zeros.
  __device__ __forceinline__ void copy_last(const char* base, int64_t ld, int left, int wave, int lane, uint32_t dst) const {
#pragma unroll
    for (int j = 0; j < PER_WAVE; ++j) {
      const int copy = wave * PER_WAVE + j;
      const int past = TR ? row(copy, lane) - (left - 1) : 8 * chunk(copy, lane) - (left - 8);
      copy16_to_lds(base, off[j] - (past > 0 ? (uint32_t)(2 * past * (TR ? ld : 1)) : 0), dst + copy * 1024);
    }
  }

  // the eight k 16 kk + 8 (lane / 32) .. of row or column side + lane % 32
  template <class V>
  static __device__ __forceinline__ V read(const char* stage, int side, int kk, int lane) {
    if constexpr (TR) {
      const int g = lane >> 4, i = lane & 15;
      const int k = 16 * kk + 8 * (g >> 1) + (i >> 2), col = side + 16 * (g & 1) + 4 * (i & 3);
      const int at = k * (2 * SIDE) + (((col >> 3) ^ swap(i >> 2)) << 4) + 2 * (col & 7);
      const lds_char* p = (const lds_char*)stage;
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + at));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + at + 4 * (2 * SIDE)));
      return __builtin_bit_cast(V, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int r = side + (lane & 31);
      return *(const V*)(stage + r * (2 * BK) + (((2 * kk + (lane >> 5)) ^ swap(lane & 31)) << 4));
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

// x in its three bf16 parts, each the nearest to what those before it leave.  The first is at most the largest bf16, past which
// it would round to infinity; the second has what that leaves, and is NaN or infinite where x is.  Parts below 2^-126 are zeros to
// the matrix cores, so x keeps all its bits from 2^-103 up.
__device__ __forceinline__ void split_parts(float x, __bf16 part[VOCAB_PARTS]) {
  constexpr float MOST = 0x1.fep127f;
  part[0] = (__bf16)__builtin_amdgcn_fmed3f(x, -MOST, MOST);
#pragma unroll
  for (int k = 1; k < VOCAB_PARTS; ++k) {
    x -= (float)part[k - 1];
    part[k] = (__bf16)x;
  }
}

// The loss, by one workgroup: minus the sum of the log-probabilities (0 in rows that do not count) over the rows that do.
// 256 threads take it, whatever the workgroup's size, so that it has the same bits with and without gradients.
template <int WAVES>
__device__ __forceinline__ void vocab_loss(const float* __restrict__ logp, int rows, int live, float* loss, float* red) {
  float sum = 0.f;
  if (threadIdx.x < 256)
#pragma unroll 8
    for (int n = threadIdx.x; n < rows; n += 256) sum += logp[n];
  sum = block_sum<WAVES>(sum, red);
  if (threadIdx.x == 0) *loss = live ? -sum / (float)live : 0.f;
}

// Waits until all but the last LEFT of this wave's copies are there.
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// Stages that pass through registers, for a weight of type S that cannot be copied as it lies (rows that do not start at 16
// bytes, fp32 that is split into parts on the way): where few rows use it, a packed copy of it would take longer than
// everything else.  The layout in LDS is VocabOperand's; what is past the end of rows or columns is zeros.
template <bool TR, int SIDE, int NT, int BK, class S>
struct VocabWeightChunks {
  typedef VocabOperand<TR, SIDE, NT / 64, BK> Op;
  static constexpr int COUNT = SIDE * BK / 8 / NT;
  Pack<S, 8> x[COUNT];

  __device__ __forceinline__ void load(const S* base, int64_t ld, int k0, int first, int rows, int cols) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int id = threadIdx.x + NT * j, along = id / Op::SLOTS, at = 8 * (id % Op::SLOTS);
      const int r = TR ? k0 + along : min(first + along, rows - 1), c = TR ? first + at : k0 + at;
      if (r < rows && c + 8 <= cols) {
        x[j] = load_pack<S, 8>(base + r * ld + c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j].v[e] = r < rows && c + e < cols ? base[r * ld + c + e] : (S)0.f;
      }
    }
  }

  template <class E>
  __device__ __forceinline__ void put(char* stage, int plane) const {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int id = threadIdx.x + NT * j, row = id / Op::SLOTS, slot = (id % Op::SLOTS) ^ Op::swap(row);
      char* to = stage + 16 * (row * Op::SLOTS + slot);
      if constexpr (sizeof(S) == 2) {
        *(Words*)to = __builtin_bit_cast(Words, x[j]);
      } else {
        Pack<__bf16, 8> y[VOCAB_PARTS];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          __bf16 parts[VOCAB_PARTS];
          split_parts(x[j].v[e], parts);
#pragma unroll
          for (int q = 0; q < VOCAB_PARTS; ++q) y[q].v[e] = parts[q];
        }
#pragma unroll
        for (int q = 0; q < VOCAB_PARTS; ++q) *(Words*)(to + q * plane) = __builtin_bit_cast(Words, y[q]);
      }
    }
  }
};

// The other operand beside it: packed rows with k contiguous.
template <int SIDE, int NT, int BK, int PLANES>
struct VocabRowChunks {
  typedef VocabOperand<false, SIDE, NT / 64, BK> Op;
  static constexpr int EACH = SIDE * BK / 8, COUNT = PLANES * EACH / NT;
  static_assert(COUNT * NT == PLANES * EACH, "whole chunks a thread");
  Words x[COUNT];

  __device__ __forceinline__ void load(const char* base, int64_t ld, int64_t part, int k0, int first, int rows) {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int id = threadIdx.x + NT * j, q = id / EACH, at = id % EACH;
      const int r = min(first + at / Op::SLOTS, rows - 1);
      x[j] = *(const Words*)(base + 2 * (q * part + r * ld + k0 + 8 * (at % Op::SLOTS)));
    }
  }
  __device__ __forceinline__ void put(char* stage) const {
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
      const int id = threadIdx.x + NT * j, q = id / EACH, at = id % EACH, row = at / Op::SLOTS;
      *(Words*)(stage + 2 * SIDE * BK * q + 16 * (row * Op::SLOTS + ((at % Op::SLOTS) ^ Op::swap(row)))) = x[j];
    }
  }
};

// One tile.  `block`: XCD block % 8 takes a share of neighbouring tiles.  GP: the parts of G.  S: the type of a weight that
// passes through registers, or void.
template <class T, int MODE, class E, int GP, class S = void>
__device__ __forceinline__ void vocab_tile(const VocabArgs& p, char* smem, uint32_t block) {
  constexpr bool A_TR = MODE >= VM_DX, B_TR = MODE == VM_DW;
  constexpr int FM = T::FM, FN = T::FN;
  typedef typename Vec8<E>::type V8;
  typedef VocabOperand<A_TR, T::BM, T::WAVES, T::BK> OpA;
  typedef VocabOperand<B_TR, T::BN, T::WAVES, T::BK> OpB;
  constexpr int BK = T::BK, PA = T::PA, PB = T::PB;
  constexpr bool PARTS = GP == VOCAB_PARTS;
  static_assert(PA == (PARTS ? VOCAB_PARTS : 1) && PB == (MODE >= VM_DX || PARTS ? GP : 1), "the operands' parts");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int live = *p.live;
  const int N = MODE == VM_DW ? p.N : min(live, p.N);

  // Tiles in the order of groups of 8 along M, a contiguous share of them to each XCD: the 32 or 64 tiles that run on
  // one XCD at a time read 8 tiles of A and 4 or 8 of B through its L2.  Only rows that count have tiles.
  const int ntm = (p.M + T::BM - 1) / T::BM, ntn = (N + T::BN - 1) / T::BN;
  const int splits = MODE >= VM_SUMS ? p.splits : 1;
  const int tiles = ntm * ntn * splits, share = (tiles + 7) / 8;
  int tile = (int)(block & 7) * share + (int)(block >> 3);
  if ((int)(block >> 3) >= share || tile >= tiles) return;
  int split = 0;
  if constexpr (MODE >= VM_SUMS) {
    split = tile / (ntm * ntn);
    tile -= split * (ntm * ntn);
  }
  const int group = tile / (8 * ntn), in_group = tile - group * (8 * ntn);
  const int width = min(8, ntm - 8 * group);
  const int tm = 8 * group + in_group % width, tn = in_group / width;
  const int m0 = tm * T::BM, n0 = tn * T::BN;

  int steps = (MODE == VM_DW ? (live + VOCAB_BK - 1) / VOCAB_BK * VOCAB_BK : p.K) / BK, k_first = 0;
  if constexpr (MODE >= VM_SUMS) {
    const int per = (steps + splits - 1) / splits;
    k_first = split * per;
    steps = max(0, min(per, steps - k_first));
  }

  OpA opa;
  OpB opb;
  opa.set(wave, lane, m0, p.a_rows, p.a_cols, p.lda);
  opb.set(wave, lane, n0, p.b_rows, p.b_cols, p.ldb);
  const int64_t a_step = 2 * (A_TR ? p.lda * BK : BK), b_step = 2 * (B_TR ? p.ldb * BK : BK);
  const char* a_at = (const char*)p.A + (A_TR ? 0 : 2 * (int64_t)m0 * p.lda) + k_first * a_step;
  const char* b_at = (const char*)p.B + (B_TR ? 0 : 2 * (int64_t)n0 * p.ldb) + k_first * b_step;
  const uint32_t lds0 = (uint32_t)(uintptr_t)((lds_char*)smem);
  int ks = 0;

  auto issue = [&](int buffer) {
    const uint32_t dst = lds0 + buffer * T::STAGE;
    // the weight's rows end where the width does and the weight where the vocabulary does; everything else has zeros up
    // to a whole stage
    int left = MODE == VM_DW ? BK : (MODE == VM_DX ? p.a_rows : p.a_cols) - (k_first + ks) * BK;
    const char* from = a_at;
    if (MODE == VM_DX && left < 1) {      // a stage past the end, in the padding of k: the last row alone
      from -= 2 * (1 - left) * p.lda;
      left = 1;
    }
#pragma unroll
    for (int part = 0; part < PA; ++part) {
      const uint32_t to = dst + part * T::A_PLANE;
      if (left < BK) opa.copy_last(from + 2 * part * p.a_part, p.lda, left, wave, lane, to);
      else opa.copy(from + 2 * part * p.a_part, wave, to);
    }
#pragma unroll
    for (int part = 0; part < PB; ++part)
      opb.copy(b_at + 2 * part * p.b_part, wave, dst + T::A_BYTES + part * T::B_PLANE);
    a_at += a_step;
    b_at += b_step;
    ++ks;
  };

  float* bias = (float*)(smem + T::BIAS_AT);
  if constexpr (MODE <= VM_GRAD) {
    // rows past the vocabulary get logits of -inf; the first barrier of the loop is before the first use
    for (int m = threadIdx.x; m < T::BM; m += T::NT)
      bias[m] = m0 + m >= p.M ? -INFINITY : p.bias ? load_elem(p.bias, p.elem, m0 + m) : 0.f;
  }

  const int wm = (wave % T::NWM) * 32 * FM, wn = (wave / T::NWM) * 32 * FN;
  floatx16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  float col_sum[FN], col_left[FN];
  const bool sum_cols = MODE == VM_DW && p.db && tm == 0 && wave % T::NWM == 0;
#pragma unroll
  for (int j = 0; j < FN; ++j) col_sum[j] = col_left[j] = 0.f;
  // G's column sums, the bias's gradient: they cancel (a token's are one less than its probability), so what a sum rounds
  // away is kept and added again
  auto column_sums = [&](const V8 (&x)[PB][FN]) {
    if (sum_cols) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        float more = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int part = PB - 1; part >= 0; --part) more += (float)x[part][j][e];
        more -= col_left[j];
        const float all = col_sum[j] + more;
        col_left[j] = (all - col_sum[j]) - more;
        col_sum[j] = all;
      }
    }
  };
  auto fragments = [&](const char* stage, int first, auto& a, auto& b) {
    constexpr int KK = sizeof(a) / sizeof(a[0]);
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int part = 0; part < (PA > PB ? PA : PB); ++part) {
        if (part < PA)
#pragma unroll
          for (int i = 0; i < FM; ++i)
            a[k][part][i] = OpA::template read<V8>(stage + part * T::A_PLANE, wm + 32 * i, first + k, lane);
        if (part < PB)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            b[k][part][j] = OpB::template read<V8>(stage + T::A_BYTES + part * T::B_PLANE, wn + 32 * j, first + k, lane);
      }
  };
  auto multiply = [&](const V8 (&a)[PA][FM], const V8 (&b)[PB][FN]) {
#pragma unroll
    for (int sum = (PA > PB ? PA : PB) - 1; sum >= 0; --sum)     // the least products first
#pragma unroll
      for (int part = 0; part <= sum; ++part) {
        if (part >= PA || sum - part >= PB) continue;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma16(a[part][i], b[sum - part][j], acc[i][j]);
      }
    if constexpr (MODE == VM_DW) column_sums(b);
  };

  if constexpr (!__is_same(S, void)) {
    static_assert(MODE != VM_DW && T::STAGES >= 2 && T::WAVES == 4, "the weight is the first operand; two buffers");
    constexpr int AHEAD = 3;      // stages under way in registers
    VocabWeightChunks<A_TR, T::BM, T::NT, BK, S> wa[AHEAD];
    VocabRowChunks<T::BN, T::NT, BK, PB> xb[AHEAD];
    auto load = [&](int s, int to) {
      const int k0 = (k_first + s) * BK;
      wa[to].load((const S*)p.A, p.lda, k0, m0, p.a_rows, p.a_cols);
      xb[to].load((const char*)p.B, p.ldb, p.b_part, k0, n0, p.b_rows);
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d)
      if (d < steps) load(d, d);
    for (int s0 = 0; s0 < steps; s0 += AHEAD) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        const int s = s0 + d;
        if (s < steps) {
          char* stage = smem + (s & 1) * T::STAGE;
          wa[d].template put<E>(stage, T::A_PLANE);
          xb[d].put(stage + T::A_BYTES);
          // everyone has read the other buffer when everyone is here
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
          if (s + AHEAD < steps) load(s + AHEAD, d);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            V8 a[1][PA][FM], b[1][PB][FN];
            fragments(stage, kk, a, b);
            multiply(a[0], b[0]);
          }
        }
      }
    }
  } else if constexpr (T::WAVES == 8) {
    // Two groups of four waves, one wave of each on a SIMD, take turns: while one multiplies what it has in registers
    // (half a stage, 16 products in 512 cycles; fp32: 24 in 768) the other reads its next half stage from LDS and starts the copies
    // of the next stage.  A buffer is written again when the second group has read its last half, and has to be there
    // three turns later.
    static_assert(T::STAGES == 2, "two buffers in turn");
    const bool second = wave >= 4;
    if (steps > 0) issue(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (second) asm volatile("s_barrier" ::: "memory");
    for (int s = 0; s < steps; ++s) {
      const char* stage = smem + (s & 1) * T::STAGE;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        constexpr int KK = BK / 32;     // 16 k each, of half a stage
        V8 a[KK][PA][FM], b[KK][PB][FN];
        fragments(stage, KK * h, a, b);
        if (h == 0 && s + 1 < steps) issue((s + 1) & 1);
        if (h == 1 && second) wait_copies<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < KK; ++k) multiply(a[k], b[k]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        if (h == 1 && !second) wait_copies<0>();
        asm volatile("s_barrier" ::: "memory");
      }
    }
    if (!second) asm volatile("s_barrier" ::: "memory");
  } else {
    // All but one of the stages are under way.
    constexpr int AHEAD = T::STAGES - 1, COPIES = PA * OpA::PER_WAVE + PB * OpB::PER_WAVE;
    if constexpr (T::STAGES == 1) {
      // for sums of one stage: the workgroups beside this one hide its copies
      if (steps > 0) issue(0);
    }
    static_assert(AHEAD * COPIES < 64 + COPIES, "what vmcnt counts");
    for (int s = 0; s < AHEAD && s < steps; ++s) issue(s);
    int from = 0, to = AHEAD;   // buffers of stage s and of the stage that is started beside it
    for (int s = 0; s < steps; ++s) {
      // this wave's copies of the stage are there, then everyone's; the readers of the buffer before it are done
      if constexpr (T::STAGES == 1) {
        if (s > 0) {
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
          issue(0);
        }
        wait_copies<0>();
      } else {
        if (s + AHEAD <= steps) wait_copies<AHEAD * COPIES - COPIES>();
        else wait_copies<0>();
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (AHEAD > 0 && s + AHEAD < steps) issue(to);
      const char* stage = smem + from * T::STAGE;
      from = from + 1 == T::STAGES ? 0 : from + 1;
      to = to + 1 == T::STAGES ? 0 : to + 1;
      // a stage's fragments are on their way together where they fit the registers, or the products would wait for LDS
      // at every 16 k
      constexpr int EACH = PA * FM + PB * FN;
      constexpr int KK = EACH * (BK / 16) <= 24 ? BK / 16 : EACH * (BK / 32) <= 24 ? BK / 32 : 1;
#pragma unroll
      for (int h = 0; h < BK / 16 / KK; ++h) {
        V8 a[KK][PA][FM], b[KK][PB][FN];
        fragments(stage, KK * h, a, b);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < KK; ++k) multiply(a[k], b[k]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // C: this lane's column n0 + wn + 32 j + lane % 32, rows m0 + wm + 32 i + 8 (r / 4) + 4 (lane / 32) + r % 4
  const int half = lane >> 5, ln = lane & 31;
  if constexpr (MODE <= VM_GRAD) {
    float* red = (float*)(smem + T::RED_AT);
    const int share_of = 2 * (wave % T::NWM) + half;      // of the 2 NWM that hold a column
    if constexpr (MODE == VM_STATS) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn + 32 * j + ln;
        const int token = n < N ? p.tokens[n] - p.v0 - m0 - wm - 4 * half : -1;   // among this lane's rows
        float top = -INFINITY, chosen = 0.f;
        bool found = false;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 b4 = *(const float4*)(bias + wm + 32 * i + 8 * q + 4 * half);
            const float add[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float z = acc[i][j][4 * q + r] + add[r];
              const bool it = token == 32 * i + 8 * q + r;
              chosen = it ? z : chosen;
              found |= it;
              acc[i][j][4 * q + r] = z;
              top = fmaxf(top, z);
            }
          }
        if (found) p.chosen[n] = chosen;
        red[share_of * T::BN + wn + 32 * j + ln] = top;
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 2 * T::NWM; ++w) top = fmaxf(top, red[w * T::BN + wn + 32 * j + ln]);
        const float held = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f((acc[i][j][r] - held) * p.c);
            acc[i][j][r] = e;
            sum += e;
          }
        red[(2 * T::NWM + share_of) * T::BN + wn + 32 * j + ln] = sum;
        if (n0 + wn + 32 * j + ln >= N) {
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        }
      }
    } else {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the stages have been read
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn + 32 * j + ln;
        const bool counts = n < N;
        const int token = counts ? p.tokens[n] - p.v0 - m0 - wm - 4 * half : -1;
        const float2 row = counts ? p.row[n] : make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 b4 = *(const float4*)(bias + wm + 32 * i + 8 * q + 4 * half);
            const float add[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float x = __builtin_amdgcn_exp2f((acc[i][j][4 * q + r] + add[r] - row.x) * p.c) * row.y;
              if (token == 32 * i + 8 * q + r) x -= 1.f;
              acc[i][j][4 * q + r] = counts ? x : 0.f;
            }
          }
      }
    }
    if (MODE == VM_GRAD && p.cols) {
      // The bias's gradient, of what G is before it is rounded: columns over this wave's rows, in lane 31 of each half.  (4096
      // rows of 2048 bf16 over 50000 tokens in pieces of 128 MB: 3.08 ms, 3.02 without a bias; 3.13 with the columns of the
      // rounded G summed beside dw's products, whose error was as large as that of the rounding of G, the same in like rows.)
      constexpr float SCALE = __is_same(E, _Float16) ? VOCAB_F16_SCALE : 1.f;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float sum = acc[i][0][r];
#pragma unroll
          for (int j = 1; j < FN; ++j) sum += acc[i][j][r];
          sum = row16_sum(sum);
          sum += __builtin_amdgcn_update_dpp(0.f, sum, 0x142, 0xa, 0xf, false);     // the row of 16 before, into the second
          if (ln == 31) red[(wave / T::NWM) * T::BM + wm + 32 * i + 8 * (r / 4) + 4 * half + r % 4] = sum * SCALE;
        }
    }
    if (MODE == VM_GRAD || p.G) {
      // The tile as rows of G: a lane has four neighbours of a row, a wave 32 rows, so it passes through LDS (slot s of
      // 16 bytes of row n at s ^ n % slots) to be written in whole lines.  In parts: one by one; exponentials, which are not
      // multiplied yet, as the upper and the lower 16 bits of an fp32 number.
      constexpr int SLOTS = T::BM / 8;
      constexpr int PLANES = GP > 1 && MODE == VM_STATS ? 2 : GP;
      static_assert(T::TILE <= T::STAGES * T::STAGE, "in the stages' memory");
#pragma unroll 1
      for (int part = 0; part < PLANES; ++part) {
        if (part) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int col = wn + 32 * j + ln;
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              Pack<E, 4> x;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float v = acc[i][j][4 * q + r];
                if constexpr (GP == 1 && MODE == VM_STATS) {
                  x.v[r] = __builtin_bit_cast(E, (_Float16)(v * VOCAB_E_SCALE));
                } else if constexpr (MODE == VM_STATS) {
                  const uint32_t bits = __float_as_uint(v);
                  x.v[r] = __builtin_bit_cast(E, (uint16_t)(part ? bits : bits >> 16));
                } else {
                  constexpr float SCALE = __is_same(E, _Float16) ? VOCAB_F16_SCALE : 1.f;
                  x.v[r] = (E)(v * SCALE);
                  if constexpr (GP > 1) acc[i][j][4 * q + r] = __builtin_isfinite(v) ? v - (float)x.v[r] * (1.f / SCALE) : 0.f;
                }
              }
              const int slot = ((wm + 32 * i) / 8 + q) ^ (col % SLOTS);
              *(Pack<E, 4>*)__builtin_assume_aligned(smem + col * (2 * T::BM) + 16 * slot + 8 * half, 8) = x;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        E* g = (E*)p.G + part * p.g_part + m0;
#pragma unroll 4
        for (int at = threadIdx.x; at < T::BN * SLOTS; at += T::NT) {
          const int col = at / SLOTS, slot = at % SLOTS;
          if (n0 + col >= p.g_rows) continue;
          E* to = g + (int64_t)(n0 + col) * p.ldg + 8 * slot;
          *(Words*)to = *(const Words*)(smem + col * (2 * T::BM) + 16 * (slot ^ (col % SLOTS)));
          // no one makes the third part of rows that do not count
          if (PARTS && MODE == VM_STATS && part == 1 && n0 + col >= N) *(Words*)(to + p.g_part) = zero_words();
        }
      }
    } else {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if constexpr (MODE == VM_STATS) {
      for (int col = threadIdx.x; col < T::BN; col += T::NT) {
        if (n0 + col >= N) continue;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 2 * T::NWM; ++w) {
          top = fmaxf(top, red[w * T::BN + col]);
          sum += red[(2 * T::NWM + w) * T::BN + col];
        }
        p.part[(n0 + col) * p.part_ld + (p.v0 + m0) / T::BM] = make_float2(top, sum);
      }
    } else if (p.cols) {
      static_assert(T::NWN * T::BM * 4 <= T::LDS - T::RED_AT, "the columns' sums in the statistics' memory");
      for (int m = threadIdx.x; m < T::BM; m += T::NT) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < T::NWN; ++w) sum += red[w * T::BM + m];
        p.cols[tn * p.ldg + m0 + m] = sum;
      }
    }
  } else if (MODE == VM_SUMS || p.sums) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = n0 + wn + 32 * j + ln;
      if (MODE == VM_DW && sum_cols) {
        const float sum = col_sum[j] + __shfl_xor(col_sum[j], 32);
        if (half == 0 && n < N) p.db_sums[(int64_t)split * N + n] = sum;
      }
      if (n >= N) continue;
      float* row = p.sums + split * p.sums_split + (int64_t)n * p.sums_ld;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
          if (m >= p.sums_ld) continue;
          Pack<float, 4> x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x.v[r] = acc[i][j][4 * q + r];
          if (p.add) {
            const Pack<float, 4> was = load_pack<float, 4>(row + m);
#pragma unroll
            for (int r = 0; r < 4; ++r) x.v[r] += was.v[r];
          }
          store_pack(row + m, x);
        }
    }
  } else {
    const float scale = p.scale / (float)max(live, 1);
    const bool wide = PARTS || p.out_elem == TE_F32;
    if (sum_cols) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn + 32 * j + ln;
        const float sum = col_sum[j] + __shfl_xor(col_sum[j], 32);
        if (half == 0 && n < N) store_elem(p.db, p.elem, n, sum * scale);
      }
    }
    // 16-bit rows pass through LDS as those of G do, fp32 ones go out four neighbours a lane
    constexpr int SLOTS = T::BM / 8;
    if (!wide) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col = wn + 32 * j + ln, n = n0 + col;
      const int64_t row = n < N ? (int64_t)(MODE == VM_DX ? p.source[n] : n) * p.M : 0;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (!wide) {
            Pack<E, 4> x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x.v[r] = (E)(acc[i][j][4 * q + r] * scale);
            const int slot = ((wm + 32 * i) / 8 + q) ^ (col % SLOTS);
            *(Pack<E, 4>*)__builtin_assume_aligned(smem + col * (2 * T::BM) + 16 * slot + 8 * half, 8) = x;
          } else if (n < N) {
            const int m = m0 + wm + 32 * i + 8 * q + 4 * half;
            float* out = (float*)p.out + row + m;
            if (m + 4 <= p.M) {
              Pack<float, 4> x;
#pragma unroll
              for (int r = 0; r < 4; ++r) x.v[r] = acc[i][j][4 * q + r] * scale;
              store_pack(out, x);
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (m + r < p.M) out[r] = acc[i][j][4 * q + r] * scale;
            }
          }
        }
    }
    if (!wide) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll 4
      for (int at = threadIdx.x; at < T::BN * SLOTS; at += T::NT) {
        const int col = at / SLOTS, slot = at % SLOTS, n = n0 + col, m = m0 + 8 * slot;
        if (n >= N || m >= p.M) continue;
        const Words x = *(const Words*)(smem + col * (2 * T::BM) + 16 * (slot ^ (col % SLOTS)));
        E* out = (E*)p.out + (int64_t)(MODE == VM_DX ? p.source[n] : n) * p.M + m;
        if (m + 8 <= p.M) {
          __builtin_memcpy(out, &x, 16);
        } else {
          const Pack<E, 8> y = __builtin_bit_cast(Pack<E, 8>, x);
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (m + r < p.M) out[r] = y.v[r];
        }
      }
    }
  }
}

template <class T, int MODE, class E, int GP, class S = void>
__global__ void __launch_bounds__(T::NT, (T::OCC * T::WAVES + 3) / 4) vocab_logits_kernel(VocabArgs p) {
  __shared__ __attribute__((aligned(1024))) char smem[T::LDS];
  vocab_tile<T, MODE, E, GP, S>(p, smem, blockIdx.x);
}

// dX (tiles T) and dW (tiles W) of a piece, in one launch: neither needs the other, and the many short tiles of dW fill the
// CUs that dX's few long ones leave.  dX's come first; the last workgroup takes the loss where `loss` is given.
template <class T, class W, class E, int GP, class S = void>
__global__ void __launch_bounds__(T::NT, (T::OCC * T::WAVES + 3) / 4)
    vocab_grads_kernel(VocabArgs dx, VocabArgs dw, uint32_t dx_blocks, const float* logp, int rows, float* loss) {
  static_assert(T::NT == W::NT, "one launch");
  constexpr int LDS = T::STAGES * T::STAGE > W::STAGES * W::STAGE ? T::STAGES * T::STAGE : W::STAGES * W::STAGE;
  static_assert(T::TILE <= LDS && W::TILE <= LDS, "tiles of results pass through the stages' memory");
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  if (loss && blockIdx.x + 1 == gridDim.x) vocab_loss<T::WAVES>(logp, rows, *dx.live, loss, (float*)smem);
  else if (blockIdx.x < dx_blocks) vocab_tile<T, VM_DX, E, GP, S>(dx, smem, blockIdx.x);
  else vocab_tile<W, VM_DW, E, GP>(dw, smem, blockIdx.x - dx_blocks);
}

// Workgroups for `tiles` tiles at most, a whole number per XCD.
inline int64_t vocab_blocks(int64_t tiles) { return 8 * ceil_div(tiles, 8); }

template <class T, class E, int GP, class S = void>
inline bool launch_vocab_logits(const VocabArgs& p, int mode, hipStream_t stream) {
  const dim3 grid((unsigned)vocab_blocks(ceil_div(p.M, T::BM) * ceil_div(p.N, T::BN) * p.splits));
  // what no call asks for is not compiled: only small grids are cut, whatever G has; few rows have G in parts, many in one
  constexpr bool FEW = T::BN == 64;
  if (mode == VM_SUMS) {
    if constexpr (GP != 2 && ((T::OCC == 1 && T::WAVES == 4) || !__is_same(S, void))) {
      hipLaunchKernelGGL((vocab_logits_kernel<T, VM_SUMS, E, GP, S>), grid, dim3(T::NT), 0, stream, p);
      return true;
    }
  } else if (mode == VM_STATS) {
    if constexpr (GP != 2 || FEW) {
      hipLaunchKernelGGL((vocab_logits_kernel<T, VM_STATS, E, GP, S>), grid, dim3(T::NT), 0, stream, p);
      return true;
    }
  } else {
    if constexpr (GP != 1 || !FEW) {
      hipLaunchKernelGGL((vocab_logits_kernel<T, VM_GRAD, E, GP, S>), grid, dim3(T::NT), 0, stream, p);
      return true;
    }
  }
  return false;
}

template <class T, class W, class E, int GP, class S = void>
inline bool launch_vocab_grads(const VocabArgs& dx, const VocabArgs& dw, const float* logp, int rows, float* loss,
                               hipStream_t stream) {
  const int64_t first = vocab_blocks(ceil_div(dx.M, T::BM) * ceil_div(dx.N, T::BN) * dx.splits);
  const int64_t all = first + vocab_blocks(ceil_div(dw.M, W::BM) * ceil_div(dw.N, W::BN) * dw.splits) + (loss ? 1 : 0);
  hipLaunchKernelGGL((vocab_grads_kernel<T, W, E, GP, S>), dim3((unsigned)all), dim3(T::NT), 0, stream, dx, dw, (uint32_t)first,
                     logp, rows, loss);
  return true;
}

// Tiles by the size of the problem; G: the parts of G (3: of everything, fp32), for the gradients PB of them.
// Large: the products' rate, 1.2 PFLOP/s over 128000 tokens of 4096 (the matrix cores busy in 68 to 72 % of the cycles, whose
// clock falls to 1.4 to 1.65 GHz meanwhile).  Mid: where Large would leave CUs without a tile.  Slim: up to 64 rows, where
// the weight's bytes are the time: 16 KB of it in a stage and two stages of two workgroups under way on a CU (44 rows
// scored over 50001 tokens of 2048: 6.3 TB/s).  Deep and Thin are these with more stages under way for grids of at most a
// workgroup per CU, whose time is the copies' latency.
constexpr int vocab_pa(int g) { return g == VOCAB_PARTS ? g : 1; }
template <int G>
using VocabLarge = VocabTile<G == 3 ? 2 : 4, 2, G == 3 ? 4 : 2, G == 3 ? 2 : 4, 2, 1, vocab_pa(G), G>;
template <int G>
using VocabDeep = VocabTile<2, 2, 2, 2, G == 1 ? 4 : 3, 1, vocab_pa(G), G>;
typedef VocabTile<1, 2, 4, 1, 6, 1, 1, 1> VocabThin;
typedef VocabTile<1, 2, 4, 1, 4, 1, 1, 2> VocabThinG;    // of G in two parts
template <int G>
using VocabSlim = VocabTile<1, 2, 4, 1, G == 1 ? 3 : 2, 2, vocab_pa(G), G>;
typedef VocabTile<2, 2, 2, 2, 2, 2, 1, 1> VocabMid;      // in parts it would be Deep
// dW beside Slim's dX: its rows are k, one stage of them, so that the tile's stores are its time
template <int G>
using VocabWide = VocabTile<1, 4, 4, 1, 1, 2, vocab_pa(G), G>;

enum : int { VT_LARGE = 0, VT_MID = 1, VT_DEEP = 2, VT_SLIM = 3, VT_THIN = 4, VT_REGS = 5 };   // REGS: Slim through registers

// Defined for each type by a file of its own (bf_vocab_*.hip).  False: there is no such kernel, and nothing was launched.
template <class E, int GP>
bool vocab_logits(int tile, const VocabArgs& p, int mode, hipStream_t stream);
template <class E, int GP>
bool vocab_grads(int tile, const VocabArgs& dx, const VocabArgs& dw, const float* logp, int rows, float* loss,
                 hipStream_t stream);

}  // namespace bf
