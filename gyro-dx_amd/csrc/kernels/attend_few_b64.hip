// Attention of few rows, bf16 heads of up to 64 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED_OCC(attend_few_b64, 256, 2) { attend_few_body<ROW_BF16, 64, 4>(a); }
