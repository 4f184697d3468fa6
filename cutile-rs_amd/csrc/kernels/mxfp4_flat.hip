// The MXFP4 product on wave-private stages (scaled_flat.h).
#include "scaled_flat.h"

using namespace cutile;
using namespace cutile::gemm;

SCALED_FLAT_FAMILY(linear_tile_mxfp4_entry, bf16, kScaledMxfp4, __bf16, 2, 2, 1)
SCALED_FLAT_FAMILY(linear_tile_mxfp4_entry, f32, kScaledMxfp4, float, 2, 2, 1)
