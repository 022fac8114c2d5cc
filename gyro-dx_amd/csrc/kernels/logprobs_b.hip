// Log probabilities, entropy and top alternatives of rows of bf16 logits (logprobs.h).
#include "logprobs.h"
GD_PIPELINE_NAMED(logprobs_b, 256) { logprobs_body<ROW_BF16>(a); }
