// Log probabilities, entropy and top alternatives of rows of binary16 logits (logprobs.h).
#include "logprobs.h"
GD_PIPELINE_NAMED(logprobs_h, 256) { logprobs_body<ROW_F16>(a); }
