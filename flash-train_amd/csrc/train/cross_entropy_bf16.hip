// The cross entropy's products with bf16 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileBf16(HeadTile what, const HeadTileArgs& args, int slices, hipStream_t stream) {
    launchHeadTileHalf<true>(what, args, slices, stream);
}

}  // namespace ftrain::train
