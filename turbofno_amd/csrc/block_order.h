// Which blocks a launch has and which pieces of work they take. Plain arithmetic, so that it can be checked without a GPU.
#pragma once
#include <algorithm>

namespace tfno {

// A dimension of a launch holds fewer than 2^32 threads, so from 2^22 blocks (of up to 512) on there are several rows of them, whose last blocks have nothing to do
constexpr long kGridRow = 1L << 22;
constexpr long grid_rows(long blocks) { return blocks <= kGridRow ? 1 : (blocks + kGridRow - 1) / kGridRow; }
// Places side by side to one XCD, `run` to each of the eight: block `id` runs on XCD id % 8. Blocks behind the last place get one that is beyond all
constexpr long kNoPlace = 1L << 48;
constexpr long side_by_side(long id, long run) { return id / 8 < run ? id % 8 * run + id / 8 : kNoPlace; }

// Tiles of a product, `row_tiles` over each of `column_tiles` tiles of columns. With many columns (from 64 tiles on) those of the same columns follow one another on one XCD, whose L2 cache
// then holds them; `turns`: neighbours go to the XCDs in turns, otherwise side by side to one of them. Tiles beyond the last are those of blocks that have none
struct Tile {
    long column;
    int row;
};
constexpr bool tiles_by_xcd(long column_tiles) { return column_tiles >= 64; }
constexpr long tile_blocks(int row_tiles, long column_tiles) { return (tiles_by_xcd(column_tiles) ? (column_tiles + 7) / 8 * 8 : column_tiles) * row_tiles; }
constexpr Tile tile_of(long id, int row_tiles, long column_tiles, bool by_xcd, bool turns)
{
    const long slot = by_xcd ? id / 8 : id, nth = slot / row_tiles, among = nth * 8 + id % 8;
    return { !by_xcd ? nth : turns ? among : side_by_side(among, (column_tiles + 7) / 8), (int)(slot % row_tiles) };
}

// Persistent blocks over strips of a field (gradient of the layer norm): those of a block, of `strips` from the one `base`, are every `step`th of all, or, `together`, of an eighth of them
constexpr long kGradBlocks = 512;
struct StripTurns {
    long base, strips, run, step;
    constexpr StripTurns(long from, long all, bool together) : base(from), strips(all), run(together ? (all + 7) / 8 : 0), step(std::min(together ? run : all, together ? kGradBlocks / 8 : kGradBlocks)) { }
    constexpr long blocks() const { return run ? 8 * step : step; }
    constexpr long first(unsigned block) const { return base + (run ? block % 8 * run + block / 8 : block); }
    constexpr long last(unsigned block) const { return base + (run && (block % 8 + 1) * run < strips ? (block % 8 + 1) * run : strips); }
};
// Strips of a launch, up to 64 for each block: one sum over many more would round off as a whole, the more the larger it has grown (a constant gradient of 0.1 over 2^28 positions: in one launch
// off by 6.5e-5, so by 3.7e-6). Each launch has sums of its own
constexpr long kLaunchStrips = 64 * kGradBlocks;
constexpr long grad_launches(long strips) { return (strips + kLaunchStrips - 1) / kLaunchStrips; }
constexpr long strips_of_launch(long strips)            // whole rounds of blocks
{
    const long launches = grad_launches(strips);
    return launches ? ((strips + launches - 1) / launches + kGradBlocks - 1) / kGradBlocks * kGradBlocks : 0;
}
// blocks of all launches, at most: strips of 8 columns are the narrowest, of 32 where there are several launches
constexpr long grad_rows(long columns)
{
    const long launches = grad_launches((columns + 31) / 32);
    return launches > 1 ? launches * kGradBlocks : std::max(1l, std::min((columns + 7) / 8, kGradBlocks));
}

}  // namespace tfno
