// Attention of fp32 rows, heads of up to 128 values (attend_f32.h).
#include "attend_f32.h"
GD_PIPELINE_NAMED(attend_f32_128, 512) { attend_f32_body<128, 8, 1>(a); }
