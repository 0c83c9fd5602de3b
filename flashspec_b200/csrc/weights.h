// The weighted decode (decode attention that adds up what every cached token receives) as
// seen from the decode launchers.
#pragma once

#include <stdint.h>

#include "../../include/flashspec_b200.h"

namespace fsb {

// Where a decode leaves its scores (log2 domain, [B, Hq, stride] fp32) and its rows'
// natural-log LSEs ([B, Hq] fp32).
struct ScoreTarget {
  float* scores;
  float* lse;
  int64_t stride;
};

// weights[page, kv head, t] += sum over the kv head's queries of exp(score - LSE), for
// every live token; a row's LSE is joined from `parts` LSEs lse[part, B * Hq].
int launch_add_weights(const FsDecodeArgs* a, const ScoreTarget& t, const float* lse, int parts, float* weights,
                       void* stream);

}  // namespace fsb
