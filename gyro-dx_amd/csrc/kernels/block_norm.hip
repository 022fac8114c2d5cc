// The residual step between two blocks, rows of up to 4096 values (block_norm.h).
#include "block_norm.h"
GD_PIPELINE_NAMED(block_norm, 256) { block_norm_body<2>(a); }
