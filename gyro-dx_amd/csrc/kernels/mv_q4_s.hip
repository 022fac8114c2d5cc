// 4-bit products of matrices with few rows, two 16-row tiles per wave (mv_q4.h).
#include "mv_q4.h"
GD_PIPELINE_NAMED(mv_q4_s, 512) { mv_q4_body<2>(a); }
