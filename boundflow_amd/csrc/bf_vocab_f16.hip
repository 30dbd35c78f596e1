// The products of the vocabulary loss for f16.
#include "bf_vocab_tiles.h"

namespace bf {

template bool vocab_logits<_Float16, 1>(int, const VocabArgs&, int, hipStream_t);
template bool vocab_grads<_Float16, 1>(int, const VocabArgs&, const VocabArgs&, const float*, int, float*, hipStream_t);
template bool vocab_logits<_Float16, 2>(int, const VocabArgs&, int, hipStream_t);
template bool vocab_grads<_Float16, 2>(int, const VocabArgs&, const VocabArgs&, const float*, int, float*, hipStream_t);

}  // namespace bf
