// The generic decode path (decode_generic.cu) as seen from the launchers in decode.cu.
#pragma once

#include <stddef.h>

#include "../../include/flashspec_b200.h"
#include "weights.h"

namespace fsb {

// True when the generic kernel handles these arguments (head_dim 32/64/128/256, quant
// block <= 64 tokens, page a multiple of the quant block, fp16/bf16 q, <= 8 q heads per
// kv head).
bool generic_supports(const FsDecodeArgs* a);
// Workspace bytes of a generic call (its split partials) and the split count used.
size_t generic_workspace(const FsDecodeArgs* a, int device, int* splits_out);
// w != nullptr: also store the scores, and the LSEs when one split runs.
int launch_generic_decode(const FsDecodeArgs* a, int device, void* stream, const ScoreTarget* w = nullptr);
// Where a generic call of `splits` > 1 splits leaves their LSEs, [splits, B * Hq].
const float* generic_part_lse(const FsDecodeArgs* a, int splits);

}  // namespace fsb
