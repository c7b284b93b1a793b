// attn_tile_f32.hip -- the matrix kernels of attn_tile.h for f32.
#include "attn_tile.h"

namespace tkv {

int launch_attn_tile_f32(Ctx* c, const AttnArgs& a, bool i8) {
    return attn::launch_tile<float>(c, a, i8);
}

}  // namespace tkv
