// Attention of few rows, binary16 heads of up to 128 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED_OCC(attend_few_h128, 256, 2) { attend_few_body<ROW_F16, 128, 4>(a); }
