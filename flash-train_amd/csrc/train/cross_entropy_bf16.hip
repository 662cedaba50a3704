// The cross entropy's products with bf16 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileBf16(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    launchHeadTileHalf<true>(what, rows, args, slices, stream);
}

void launchHeadGradientsBf16(const HeadTileArgs& hidden, int slices, const HeadTileArgs& weight, hipStream_t stream) {
    launchHeadGradientsHalf<true>(hidden, slices, weight, stream);
}

}  // namespace ftrain::train
