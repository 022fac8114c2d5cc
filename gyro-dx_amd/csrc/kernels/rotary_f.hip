// Rotary positions and the cache's appending, rows of fp32 values (rotary.h).
#include "rotary.h"
GD_PIPELINE_NAMED_OCC(rotary_f, 256, 4) { rotary_body<ROW_F32>(a); }
