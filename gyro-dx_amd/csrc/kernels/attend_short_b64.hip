// Attention of few rows over short contexts, bf16 heads of up to 64 values (attend_few.h).
#include "attend_few.h"
GD_PIPELINE_NAMED(attend_short_b64, 512) { attend_few_body<ROW_BF16, 64, 8>(a); }
