// Log probabilities, entropy and top alternatives of rows of fp32 logits (logprobs.h).
#include "logprobs.h"
GD_PIPELINE_NAMED_OCC(logprobs, 256, 3) { logprobs_body<ROW_F32>(a); }
