// The cross entropy's products with fp32 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileFp32(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    using W = HeadTile;
    constexpr void (*large[5])(HeadTileArgs) = {&headTileFp32<W::kLogSum, 128>, &headTileFp32<W::kGradLogits, 128>,
                                                &headTileFp32<W::kGradHidden, 128>, &headTileFp32<W::kGradWeight, 128>,
                                                &headTileFp32<W::kLogits, 128>};
    constexpr void (*small[5])(HeadTileArgs) = {&headTileFp32<W::kLogSum, 64>, &headTileFp32<W::kGradLogits, 64>,
                                                &headTileFp32<W::kGradHidden, 64>, nullptr, &headTileFp32<W::kLogits, 64>};
    const int i = static_cast<int>(what);
    launchHead(rows == 128 ? large[i] : small[i], kHeadNames[i], args, rows, rows, 256, slices, stream);
}

}  // namespace ftrain::train
