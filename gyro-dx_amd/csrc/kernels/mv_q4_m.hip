// 4-bit products, weights s q + m (mv_q4.h).
#include "mv_q4.h"
GD_PIPELINE_NAMED(mv_q4_m, 512) { mv_q4_body<2, true>(a); }
