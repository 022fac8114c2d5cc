// Rotary positions and the cache's appending, rows of binary16 values (rotary.h).
#include "rotary.h"
GD_PIPELINE_NAMED(rotary_h, 256) { rotary_body<ROW_F16>(a); }
