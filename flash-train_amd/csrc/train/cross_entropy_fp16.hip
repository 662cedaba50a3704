// The cross entropy's products with fp16 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileFp16(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    launchHeadTileHalf<false>(what, rows, args, slices, stream);
}

void launchHeadGradientsFp16(const HeadTileArgs& hidden, int slices, const HeadTileArgs& weight, hipStream_t stream) {
    launchHeadGradientsHalf<false>(hidden, slices, weight, stream);
}

}  // namespace ftrain::train
