// 4-bit products of many bf16 tokens, groups of 128 (mm_q4.h).
#include "mm_q4.h"
GD_PIPELINE_NAMED_OCC(mm_q4_b128, 256, 2) { mm_q4_body<ROW_BF16, 4>(a); }
