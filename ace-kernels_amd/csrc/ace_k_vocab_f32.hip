// Vocabulary loss instantiations: f32 hidden states and weights.
#include "ace_vocab.hpp"

namespace ace {
namespace vocab {
ACE_DEFINE_VOCAB(float)
}  // namespace vocab
}  // namespace ace
