// The residual step between two blocks, rows of up to 2048 values (block_norm.h).
#include "block_norm.h"
GD_PIPELINE_NAMED(block_norm_s, 256) { block_norm_body<1>(a); }
