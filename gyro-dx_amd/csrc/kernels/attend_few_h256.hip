// Attention of few rows, binary16 heads of up to 256 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED(attend_few_h256, 256) { attend_few_body<ROW_F16, 256, 4>(a); }
