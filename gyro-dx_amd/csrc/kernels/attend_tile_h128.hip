// Attention of many rows, binary16 heads of up to 128 values (attend_tile.h).
#include "attend_tile.h"
GD_PIPELINE_NAMED_OCC(attend_tile_h128, 256, 2) { attend_tile_body<ROW_F16, 128, 64>(a); }
