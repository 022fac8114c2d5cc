// Attention of many rows, bf16 heads of up to 256 values (attend_tile.h).
#include "attend_tile.h"
GD_PIPELINE_NAMED(attend_tile_b256, 256) { attend_tile_body<ROW_BF16, 256, 32>(a); }
