// The cross entropy's products with fp16 operands.
#include "cross_entropy_tiles.hpp"

namespace ftrain::train {

void launchHeadTileFp16(HeadTile what, const HeadTileArgs& args, int slices, hipStream_t stream) {
    launchHeadTileHalf<false>(what, args, slices, stream);
}

}  // namespace ftrain::train
