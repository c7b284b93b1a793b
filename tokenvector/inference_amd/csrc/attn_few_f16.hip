// attn_few_f16.hip -- the matrix kernels of attn_few.h for f16.
#include "attn_few.h"

namespace tkv {

int launch_attn_few_f16(Ctx* c, const AttnArgs& a, bool i8, int blocks_of_16) {
    return attn::launch_few<_Float16>(c, a, i8, blocks_of_16);
}

}  // namespace tkv
