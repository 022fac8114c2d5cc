// 4-bit products of many binary16 tokens, groups of 32 (mm_q4.h).
#include "mm_q4.h"
GD_PIPELINE_NAMED_OCC(mm_q4_h32, 256, 2) { mm_q4_body<ROW_F16, 1>(a); }
