// Attention of many rows, binary16 heads of up to 256 values (attend_tile.h).
#include "attend_tile.h"
GD_PIPELINE_NAMED(attend_tile_h256, 256) { attend_tile_body<ROW_F16, 256, 32>(a); }
