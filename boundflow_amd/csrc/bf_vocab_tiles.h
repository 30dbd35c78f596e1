// The tile configurations of the vocabulary loss's products, compiled for one type per file.
#pragma once

#include "bf_vocab_gemm.h"

namespace bf {

// The type of a weight that passes through registers.
template <class E, int GP>
struct WeightType {
  typedef E type;
};
template <class E>
struct WeightType<E, VOCAB_PARTS> {
  typedef float type;
};

// Of the logits' products: of 16-bit types one part of each operand, whatever G has.  fp32 rows take Large, Deep or, a few, Slim
// through registers.  False where the tile is not compiled for these parts.
template <class E, int GP>
bool vocab_logits(int tile, const VocabArgs& p, int mode, hipStream_t stream) {
  constexpr int P = vocab_pa(GP);
  constexpr bool WIDE = GP == VOCAB_PARTS;
  typedef typename WeightType<E, GP>::type S;
  switch (tile) {
    case VT_LARGE:
      if constexpr (GP != 2) return launch_vocab_logits<VocabLarge<P>, E, GP>(p, mode, stream);
      return false;
    case VT_MID:
      if constexpr (GP == 1) return launch_vocab_logits<VocabMid, E, GP>(p, mode, stream);
      return false;
    case VT_DEEP: return launch_vocab_logits<VocabDeep<P>, E, GP>(p, mode, stream);
    case VT_THIN:
      if constexpr (!WIDE) return launch_vocab_logits<VocabThin, E, GP>(p, mode, stream);
      return false;
    case VT_REGS:
      if constexpr (GP != 2) return launch_vocab_logits<VocabSlim<P>, E, GP, S>(p, mode, stream);
      return false;
    default:
      if constexpr (!WIDE) return launch_vocab_logits<VocabSlim<P>, E, GP>(p, mode, stream);
      return false;
  }
}

template <class E, int GP>
bool vocab_grads(int tile, const VocabArgs& dx, const VocabArgs& dw, const float* logp, int rows, float* loss,
                 hipStream_t stream) {
  typedef VocabLarge<GP> Large;
  typedef VocabDeep<GP> Deep;
  typedef typename WeightType<E, GP>::type S;
  switch (tile) {
    case VT_LARGE:
      if constexpr (GP != 2) return launch_vocab_grads<Large, Large, E, GP>(dx, dw, logp, rows, loss, stream);
      return false;
    case VT_MID:
      if constexpr (GP == 1) return launch_vocab_grads<VocabMid, VocabMid, E, GP>(dx, dw, logp, rows, loss, stream);
      return false;
    case VT_DEEP: return launch_vocab_grads<Deep, Deep, E, GP>(dx, dw, logp, rows, loss, stream);
    case VT_THIN:
      if constexpr (GP == 2) return launch_vocab_grads<VocabThinG, VocabThinG, E, GP>(dx, dw, logp, rows, loss, stream);
      return false;
    case VT_REGS:
      if constexpr (GP == 3)
        return launch_vocab_grads<VocabSlim<GP>, VocabWide<GP>, E, GP, S>(dx, dw, logp, rows, loss, stream);
      return false;
    default:
      if constexpr (GP == 2) return launch_vocab_grads<VocabSlim<GP>, VocabWide<GP>, E, GP>(dx, dw, logp, rows, loss, stream);
      return false;
  }
}

}  // namespace bf
