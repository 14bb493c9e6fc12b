// Which blocks a launch has and which pieces of work they take. Plain arithmetic, so that it can be checked without a GPU.
#pragma once

namespace tfno {

// A dimension of a launch holds fewer than 2^32 threads, so from 2^22 blocks (of up to 512) on there are several rows of them, whose last blocks have nothing to do
constexpr long kGridRow = 1L << 22;
constexpr long grid_rows(long blocks) { return blocks <= kGridRow ? 1 : (blocks + kGridRow - 1) / kGridRow; }
// Places side by side to one XCD, `run` to each of the eight: block `id` runs on XCD id % 8. Blocks behind the last place get one that is beyond all
constexpr long kNoPlace = 1L << 48;
constexpr long side_by_side(long id, long run) { return id / 8 < run ? id % 8 * run + id / 8 : kNoPlace; }

}  // namespace tfno
