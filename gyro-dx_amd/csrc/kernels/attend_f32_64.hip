// Attention of fp32 rows, heads of up to 64 values (attend_f32.h).
#include "attend_f32.h"
GD_PIPELINE_NAMED(attend_f32_64, 512) { attend_f32_body<64, 8, 2>(a); }
