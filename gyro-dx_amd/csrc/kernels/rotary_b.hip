// Rotary positions and the cache's appending, rows of bf16 values (rotary.h).
#include "rotary.h"
GD_PIPELINE_NAMED(rotary_b, 256) { rotary_body<ROW_BF16>(a); }
