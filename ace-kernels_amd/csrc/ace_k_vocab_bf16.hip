// Vocabulary loss instantiations: bf16 hidden states and weights.
#include "ace_vocab.hpp"

namespace ace {
namespace vocab {
ACE_DEFINE_VOCAB(__bf16)
}  // namespace vocab
}  // namespace ace
