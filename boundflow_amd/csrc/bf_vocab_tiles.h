// The tile configurations of the vocabulary loss's products, compiled for one type per file.
#pragma once

#include "bf_vocab_gemm.h"

namespace bf {

template <class E, bool PARTS>
void vocab_logits(int tile, const VocabArgs& p, bool stats, hipStream_t stream) {
  switch (tile) {
    case VT_LARGE: launch_vocab_logits<VocabLarge, E, PARTS>(p, stats, stream); break;
    case VT_MID: launch_vocab_logits<VocabMid, E, PARTS>(p, stats, stream); break;
    case VT_DEEP: launch_vocab_logits<VocabDeep, E, PARTS>(p, stats, stream); break;
    case VT_THIN: launch_vocab_logits<VocabThin, E, PARTS>(p, stats, stream); break;
    default: launch_vocab_logits<VocabSlim, E, PARTS>(p, stats, stream);
  }
}

template <class E, bool PARTS>
void vocab_grads(int tile, const VocabArgs& dx, const VocabArgs& dw, const float* logp, int rows, float* loss,
                 hipStream_t stream) {
  switch (tile) {
    case VT_LARGE: launch_vocab_grads<VocabLarge, VocabLarge, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_MID: launch_vocab_grads<VocabMid, VocabMid, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_DEEP: launch_vocab_grads<VocabDeep, VocabDeep, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    case VT_THIN: launch_vocab_grads<VocabThin, VocabThin, E, PARTS>(dx, dw, logp, rows, loss, stream); break;
    default: launch_vocab_grads<VocabSlim, VocabWide, E, PARTS>(dx, dw, logp, rows, loss, stream);
  }
}

}  // namespace bf
