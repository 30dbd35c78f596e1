// The products of the vocabulary loss for fp32 in three bf16 parts.
#include "bf_vocab_tiles.h"

namespace bf {

template bool vocab_logits<__bf16, 3>(int, const VocabArgs&, int, hipStream_t);
template bool vocab_grads<__bf16, 3>(int, const VocabArgs&, const VocabArgs&, const float*, int, float*, hipStream_t);

}  // namespace bf
