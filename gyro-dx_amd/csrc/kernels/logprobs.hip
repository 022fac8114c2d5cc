// Log probabilities, entropy and top alternatives of rows of fp32 logits (logprobs.h).
#include "logprobs.h"
GD_PIPELINE_NAMED(logprobs, 256) { logprobs_body<ROW_F32>(a); }
