// The cross entropy's products with fp32 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileFp32(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    constexpr void (*large[4])(HeadTileArgs) = {&headTileFp32<HeadTile::kLogSum, 128>, &headTileFp32<HeadTile::kGradLogits, 128>,
                                                &headTileFp32<HeadTile::kGradHidden, 128>, &headTileFp32<HeadTile::kGradWeight, 128>};
    constexpr void (*small[3])(HeadTileArgs) = {&headTileFp32<HeadTile::kLogSum, 64>, &headTileFp32<HeadTile::kGradLogits, 64>,
                                                &headTileFp32<HeadTile::kGradHidden, 64>};
    const int i = static_cast<int>(what);
    launchHead(rows == 128 ? large[i] : small[i], kHeadNames[i], args, rows, rows, 256, slices, stream);
}

}  // namespace ftrain::train
