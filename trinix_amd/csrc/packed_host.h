// Host-only argument checks of attention over packed sequences and behind a
// shared prefix (plain C++; see host_plan.h).
#pragma once
#include "host_plan.h"
#include "trinix_attn.h"

namespace trinix {

// TRINIX_OK or the status to return; no launch.  `backward`: the gradient
// pointers and strides too.
int validate_packed(const trinix_packed_args* a, bool backward);

}  // namespace trinix
