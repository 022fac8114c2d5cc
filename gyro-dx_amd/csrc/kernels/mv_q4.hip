// 4-bit products, four 16-row tiles per wave (mv_q4.h).
#include "mv_q4.h"
GD_PIPELINE_NAMED(mv_q4, 512) { mv_q4_body<4>(a); }
