// Attention of few rows over short contexts, binary16 heads of up to 64 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED(attend_short_h64, 512) { attend_few_body<ROW_F16, 64, 8>(a); }
