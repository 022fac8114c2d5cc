// Attention of few rows, binary16 heads of up to 64 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED_OCC(attend_few_h64, 256, 2) { attend_few_body<ROW_F16, 64, 4>(a); }
