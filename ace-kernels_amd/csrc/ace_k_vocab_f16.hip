// Vocabulary loss instantiations: f16 hidden states and weights.
#include "ace_vocab.hpp"

namespace ace {
namespace vocab {
ACE_DEFINE_VOCAB(_Float16)
}  // namespace vocab
}  // namespace ace
