// attn_few_f32.hip -- the matrix kernels of attn_few.h for f32.
#include "attn_few.h"

namespace tkv {

int launch_attn_few_f32(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16) {
    return attn::launch_few<float>(c, a, i8, blocks_of_16);
}

}  // namespace tkv
