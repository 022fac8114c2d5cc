// Attention of few rows, bf16 heads of up to 64 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED(attend_few_b64, 256) { attend_few_body<ROW_BF16, 64>(a); }
