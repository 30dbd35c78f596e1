// The tile configurations of the vocabulary loss's products, compiled for one type per file.
#pragma once

#include "bf_vocab_gemm.h"

namespace bf {

template <class E, bool PARTS>
struct WeightType {
  typedef E type;
};
template <class E>
struct WeightType<E, true> {
  typedef float type;
};

template <class E, bool PARTS>
void vocab_logits(int tile, const VocabArgs& p, int mode, hipStream_t stream) {
  switch (tile) {
    case VT_LARGE: launch_vocab_logits<VocabLarge<PARTS>, E, PARTS>(p, mode, stream); break;
    case VT_MID:
      if constexpr (!PARTS) launch_vocab_logits<VocabMid, E, PARTS>(p, mode, stream);
      break;
    case VT_DEEP: launch_vocab_logits<VocabDeep<PARTS>, E, PARTS>(p, mode, stream); break;
    case VT_THIN: launch_vocab_logits<VocabThin<PARTS>, E, PARTS>(p, mode, stream); break;
    case VT_REGS:
      launch_vocab_logits<VocabSlim<PARTS>, E, PARTS, typename WeightType<E, PARTS>::type>(p, mode, stream);
      break;
    default: launch_vocab_logits<VocabSlim<PARTS>, E, PARTS>(p, mode, stream);
  }
}

template <class E, bool PARTS>
void vocab_grads(int tile, const VocabArgs& dx, const VocabArgs& dw, const float* logp, int rows, float* loss,
                 hipStream_t stream) {
  typedef VocabLarge<PARTS> Large;
  typedef VocabDeep<PARTS> Deep;
  typedef VocabThin<PARTS> Thin;
  switch (tile) {
    case VT_LARGE: launch_vocab_grads<Large, Large, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_MID:
      if constexpr (!PARTS) launch_vocab_grads<VocabMid, VocabMid, E, PARTS>(dx, dw, logp, rows, loss, stream);
      break;
    case VT_DEEP: launch_vocab_grads<Deep, Deep, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_THIN: launch_vocab_grads<Thin, Thin, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_REGS:
      launch_vocab_grads<VocabSlim<PARTS>, VocabWide<PARTS>, E, PARTS, typename WeightType<E, PARTS>::type>(
          dx, dw, logp, rows, loss, stream);
      break;
    default: launch_vocab_grads<VocabSlim<PARTS>, VocabWide<PARTS>, E, PARTS>(dx, dw, logp, rows, loss, stream);
  }
}

}  // namespace bf
