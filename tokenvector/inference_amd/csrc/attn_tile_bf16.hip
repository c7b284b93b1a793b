// attn_tile_bf16.hip -- the matrix kernels of attn_tile.h for bf16.
#include "attn_tile.h"

namespace tkv {

int launch_attn_tile_bf16(Ctx* c, const AttnArgs& a, bool i8) {
    return attn::launch_tile<__bf16>(c, a, i8);
}

}  // namespace tkv
