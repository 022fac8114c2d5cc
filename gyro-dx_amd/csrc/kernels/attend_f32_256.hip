// Attention of fp32 rows, heads of up to 256 values (attend_f32.h).
#include "attend_f32.h"
GD_PIPELINE_NAMED(attend_f32_256, 256) { attend_f32_body<256, 4, 1>(a); }
