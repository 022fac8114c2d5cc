// Rotary positions and the cache's appending, rows of binary16 values (rotary.h).
#include "rotary.h"
GD_PIPELINE_NAMED_OCC(rotary_h, 256, 4) { rotary_body<ROW_F16>(a); }
