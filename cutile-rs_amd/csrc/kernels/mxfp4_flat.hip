// The MXFP4 product on wave-private stages (scaled_flat.h), up to 64 x 64 outputs a workgroup: wider blocks are slower than the 128 x 128 tiles of
// mxfp4_gemm.hip wherever there are enough of them to fill the chip (64 x 128 blocks 200 x 14336 x 4096 24.7 us, the tiles 13.7; 512 x 4096 x 4096 14.1, 12.3).
#include "scaled_flat.h"

using namespace cutile;
using namespace cutile::gemm;

SCALED_FLAT_STRIPS(linear_tile_mxfp4_entry, bf16, kScaledMxfp4, __bf16, 2, 2, 1)
SCALED_FLAT_STRIPS(linear_tile_mxfp4_entry, f32, kScaledMxfp4, float, 2, 2, 1)
