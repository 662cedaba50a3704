// The cross entropy's products with fp32 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileFp32(HeadTile what, const HeadTileArgs& args, int slices, hipStream_t stream) {
    const dim3 grid = headGrid(args, 128, slices);
    switch (what) {
        case HeadTile::kLogSum:
            launch(&headTileFp32<HeadTile::kLogSum>, "cross entropy logits", grid, dim3(256), stream, args);
            break;
        case HeadTile::kGradLogits:
            launch(&headTileFp32<HeadTile::kGradLogits>, "cross entropy logits' gradient", grid, dim3(256), stream, args);
            break;
        case HeadTile::kGradHidden:
            launch(&headTileFp32<HeadTile::kGradHidden>, "cross entropy hidden gradient", grid, dim3(256), stream, args);
            break;
        case HeadTile::kGradWeight:
            launch(&headTileFp32<HeadTile::kGradWeight>, "cross entropy weight gradient", grid, dim3(256), stream, args);
            break;
    }
}

}  // namespace ftrain::train
