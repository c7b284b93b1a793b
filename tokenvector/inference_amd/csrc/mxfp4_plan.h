// mxfp4_plan.h -- which kernel a product or linear of 4-bit operands goes to, by
// rules on its sizes and the card's compute units.  Host arithmetic alone, so that
// what each size takes can be asked without a device.
#pragma once

#include <math.h>
#include <stdint.h>

namespace tkv {
namespace mx {

// A product's sizes, `blocks` of a row, and the card: its compute units, and whether
// the context has counts for joining splits over K.
struct Shape {
    int64_t m, n;
    int32_t blocks;
    int cus;
    bool joins;
};
inline int64_t parts(int64_t all, int64_t of) { return (all + of - 1) / of; }

// ---- many rows: tiles ----------------------------------------------------------

// The kinds of tiles, and the times that choose among them, in us, as measured: of
// a slice with 1 .. `held` workgroups of a CU at work, and of a workgroup besides.
// What they stand for, 256 x 256, 128 x 128, 128 x 64, 64 x 64 and 64 x 64 with four
// stages instead of two: 8192 x 8192 of 8192 263, 331, 393, 479, 515; 8192 x 2304 of
// 768 (f32) 30, 24, 22, 25, 34; 1024 x 14336 of 4096 35, 40, 45, 55, 66; 512 x 4096
// of 4096 26, 15, 12, 12, 11; 128 x 8192 of 8192 46, 25, 21, 19, 13; 333 x 1000 of
// 2000 21, 9, 7, 5, 6.
// K is split over up to four workgroups of the last kind where its tiles leave CUs
// idle, 3.5 us for the join: 100 x 640 of 16000 20.6 -> 10.4 us (by eight 10.4), 200 x
// 1000 of 9000 13.6 -> 9.4, 128 x 4096 of 16384 (128 tiles in three) 21.1 -> 14.8 (in
// four 16.1); 300 x 300 of 3000 stays whole, 6.6 (7.2).
enum { TILE_256, TILE_128, TILE_128_64, TILE_64, TILE_64_RING, TILE_KINDS };
//   The last kind also takes the scales as they come, of up to kRowSlices slices, and lays
// them out itself, 0.5 us a workgroup more, where slabs cost a launch of 2.2 us: instead
// of either kind of 64 x 64 tiles where it is no slower for that.  333 x 8192 of 256 7.0
// us (slabs and two stages 6.7 to 7.8, by the host), 333 x 1000 of 2000 6.4 (8); 4096 x
// 4100 of 512 33.7 (21.7), 12000 x 1000 of 64 20.3 (14.7), 400 x 6000 of 4000 21.5 (18.5).
struct TilePlan {
    int kind, splits;
    bool rows;
};
constexpr int kRowSlices = 16;
inline TilePlan tile_plan(const Shape& p) {
    struct Kind {
        int64_t m, n;
        int held;
        float slice[4], rest;
    };
    static constexpr Kind kinds[TILE_KINDS] = {{256, 256, 1, {1.7f}, 8.0f},
                                               {128, 128, 2, {0.68f, 1.2f}, 3.0f},
                                               {128, 64, 3, {0.6f, 0.7f, 1.0f}, 2.5f},
                                               {64, 64, 4, {0.49f, 0.55f, 0.7f, 0.87f}, 1.0f},
                                               {64, 64, 2, {0.28f, 0.48f}, 1.0f}};
    const float slices = (float)((p.blocks + 7) >> 3);
    const auto time = [&](const Kind& k, float rest) {
        const int64_t tiles = parts(p.m, k.m) * parts(p.n, k.n), round = (int64_t)k.held * p.cus;
        const int64_t full = tiles / round, left = parts(tiles % round, p.cus);
        const float t = (float)full * (slices * k.slice[k.held - 1] + rest);
        return left ? t + slices * k.slice[left - 1] + rest : t;
    };
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < TILE_KINDS; i++) {
        const float t = time(kinds[i], kinds[i].rest);
        if (i == 0 || t < least) best = i, least = t;
    }
    const Kind& ring = kinds[TILE_64_RING];
    const int64_t tiles = parts(p.m, ring.m) * parts(p.n, ring.n);
    const int64_t splits = 3 * p.cus / 2 / tiles < 4 ? 3 * p.cus / 2 / tiles : 4;
    if (splits > 1 && p.joins) {
        const float t = ceilf(slices / (float)splits) * ring.slice[tiles * splits > p.cus] + ring.rest + 3.5f;
        if (t < least) return {TILE_64_RING, (int)splits, parts(parts(p.blocks, 8), splits) <= kRowSlices};
    }
    const bool rows = best >= TILE_64 && slices <= (float)kRowSlices && time(ring, ring.rest + 0.5f) <= least + 2.2f;
    return {best, 1, rows};
}

// ---- few rows: the weight streamed --------------------------------------------

constexpr int kFewRows = 64;
constexpr int kFewSplits = 8;

// The few-row kernel takes the scales as they come too.
inline bool takes_rows(const Shape& p) { return p.m <= kFewRows || tile_plan(p).rows; }

// Workgroups of a row block.  A CU's loads in flight bound what it reads (0.08 us for
// 256 elements of 16 rows, as long again for each 16 tokens more, and a row coded on the
// way as long for 70 blocks), so long rows of few outputs are split over the idle CUs,
// eight slabs each at least; the join costs 1.9 us.  1 x 1024 of 16384: 6.9 us, by one
// workgroup 8.9; 64 x 1024 of 8192 8.5 and 13.5; 12 x 960 of 9600, coded before, 6.0 and
// 6.3; in two 4 x 2048 of 8192 7.3 and 7.1.
inline int few_splits(const Shape& p, bool coded) {
    const int64_t rows = parts(p.n, 16), slabs = parts(p.blocks, 8);
    int64_t s = slabs / 8 < p.cus / rows ? slabs / 8 : p.cus / rows;
    if (s > kFewSplits) s = kFewSplits;
    const int64_t work = slabs * parts(p.m, 16) + (coded ? 0 : p.m * p.blocks / 70);
    return s > 1 && p.joins && work * (s - 1) >= 27 * s ? (int)s : 1;
}

// Every workgroup codes all rows (its part of them), 0.15 us for each 4096 elements
// (with several blocks of rows a workgroup 0.25), where a launch of its own costs 2.2 and
// more: 8 x 4096 of 4096 5.9 us against 6.7, 16 x 4096 7.9 and 7.1; 4 x 16384 9.2 and
// 10.6, 8 x 16384 11.0 and 11.0; one call after another, where two launches are 7.4 at least, 32 x 512 of 768 5.3 and 7.4, 12 x 4096
// of 4096 7.0 and 7.7, 24 x 7000 of 1300 8.5 and 7.5.
inline bool codes_few(const Shape& p, int64_t k) {
    const int64_t rows = parts(p.n, 16);
    if (k < 8 || p.m > (rows >= 2 * p.cus ? 16 : kFewRows)) return false;
    // (CUs with two workgroups code twice)
    const bool twice = rows >= 2 * p.cus || (p.m > 16 && rows > p.cus);
    const int64_t most = twice ? 512 : rows > p.cus || k % 8 ? 1024 : 1536;
    return p.m * p.blocks <= most * few_splits(p, false);
}

// 16-row blocks a workgroup: as many as leave a workgroup per CU, four for long rows
// or many tokens alone (16 x 16384 rows of 16384: 29.8 us, with two 34.7; of 4096 9.0
// and 8.3; 32 x 16384 of 4096 10.1 and 11.4).  Coding long rows for a block, 16 waves
// (4 x 2048 of 8192: 7.1 us, with 8 waves 8.0; 4 x 4096 of 4096 5.1 and 4.9).  Rows of
// more than 16 tokens are coded for one block and by 8 waves alone.
struct FewPlan {
    int tokens;  // in blocks of 16: 1, 2 or 4
    int row_blocks, waves, splits;
};
inline FewPlan few_plan(const Shape& p, bool coded) {
    FewPlan f = {p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4, 1, 8, few_splits(p, coded)};
    const int64_t rows = parts(p.n, 16);
    if (f.splits > 1 || (!coded && f.tokens > 1)) return f;
    if (f.tokens < 4 && rows >= 4 * p.cus && (f.tokens == 2 || p.blocks >= 256)) f.row_blocks = 4;
    else if (rows >= 2 * p.cus) f.row_blocks = 2;
    else if (!coded && p.blocks >= 256) f.waves = 16;
    return f;
}

}  // namespace mx
}  // namespace tkv
