// Attention of many rows, bf16 heads of up to 64 values (attend_tile.h).
#include "attend_tile.h"
GD_PIPELINE_NAMED_OCC(attend_tile_b64, 256, 2) { attend_tile_body<ROW_BF16, 64, 64>(a); }
