// Attention of few rows, bf16 heads of up to 256 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED(attend_few_b256, 256) { attend_few_body<ROW_BF16, 256, 4>(a); }
