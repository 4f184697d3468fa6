// The MXFP8 and NVFP4 products on wave-private stages (scaled_flat.h).
#include "scaled_flat.h"

using namespace cutile;
using namespace cutile::gemm;

SCALED_FLAT_FAMILY(linear_tile_entry, mxfp8_bf16, kScaledMxfp8, __bf16, 2, 2, 1)
SCALED_FLAT_FAMILY(linear_tile_entry, mxfp8_f32, kScaledMxfp8, float, 2, 2, 1)
SCALED_FLAT_FAMILY(linear_tile_nvfp4_entry, bf16, kScaledNvfp4, __bf16, 2, 2, 1)
SCALED_FLAT_FAMILY(linear_tile_nvfp4_entry, f32, kScaledNvfp4, float, 2, 2, 1)
