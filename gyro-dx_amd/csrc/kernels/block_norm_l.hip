// The residual step between two blocks, rows of up to 16384 values (block_norm.h).
#include "block_norm.h"
GD_PIPELINE_NAMED(block_norm_l, 256) { block_norm_body<8>(a); }
