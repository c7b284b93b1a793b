// attn_tile_f16.hip -- the matrix kernels of attn_tile.h for f16.
#include "attn_tile.h"

namespace tkv {

int launch_attn_tile_f16(Ctx* c, const AttnArgs& a, bool i8) {
    return attn::launch_tile<_Float16>(c, a, i8);
}

}  // namespace tkv
