#include "fgms_attention_bodies.h"

namespace fgms {
template int attention_fwd<__bf16>(const AttentionArgs &);
template int attention_bwd<__bf16>(const AttentionArgs &);
}  // namespace fgms
