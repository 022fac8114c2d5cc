// Rotary positions and the cache's appending, rows of bf16 values (rotary.h).
#include "rotary.h"
GD_PIPELINE_NAMED_OCC(rotary_b, 256, 4) { rotary_body<ROW_BF16>(a); }
