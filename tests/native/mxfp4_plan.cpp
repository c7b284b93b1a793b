// Says which kernels products and linears of 4-bit operands take: for each line "m n k"
// of the input, on a card of 256 compute units, "kind splits takes_rows codes_few" and
// the few-row kernel's "tokens row_blocks waves splits" with coded tokens and without.
#include <cstdio>

#include "../../tokenvector/inference_amd/csrc/mxfp4_plan.h"

int main() {
    using namespace tkv::mx;
    long long m, n, k;
    while (scanf("%lld %lld %lld", &m, &n, &k) == 3) {
        const Shape p = {m, n, (int32_t)parts(k, 32), 256, true};
        const TilePlan t = tile_plan(p);
        const FewPlan c = few_plan(p, true), x = few_plan(p, false);
        printf("%d %d %d %d  %d %d %d %d  %d %d %d %d\n", t.kind, t.splits, (int)takes_rows(p), (int)codes_few(p, k), c.tokens,
               c.row_blocks, c.waves, c.splits, x.tokens, x.row_blocks, x.waves, x.splits);
    }
    return 0;
}
