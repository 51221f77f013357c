#include "fgms_attention_bodies.h"

namespace fgms {
template int attention_fwd<float>(const AttentionArgs &);
template int attention_bwd<float>(const AttentionArgs &);
}  // namespace fgms
