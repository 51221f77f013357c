#include "fgms_attention_bodies.h"

namespace fgms {
template int attention_fwd<_Float16>(const AttentionArgs &);
template int attention_bwd<_Float16>(const AttentionArgs &);
}  // namespace fgms
