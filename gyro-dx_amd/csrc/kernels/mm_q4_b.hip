// 4-bit products of many bf16 tokens, weights s (q - 8) (mm_q4.h).
#include "mm_q4.h"
GD_PIPELINE_NAMED_OCC(mm_q4_b, 256, 2) { mm_q4_body<ROW_BF16, false>(a); }
