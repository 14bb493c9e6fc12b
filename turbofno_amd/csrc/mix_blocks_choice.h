// Which kernel of the product in 8 bits with scales by blocks (mix_blocks.hip) takes a call, and how many columns it needs: a wave or a block whose columns are not all there takes the last ones
// of the field instead. Plain arithmetic on the sizes, so that it can be checked without a GPU.
#pragma once
#include <algorithm>

namespace tfno {

enum class BlocksKernel { kOneScale, kSplitNear, kSplitFar, kTile, kDirect, kStaged };
struct BlocksChoice {
    BlocksKernel kernel;
    int nt, groups;                                     // 16 nt rows of a wave, groups of waves that divide the steps
    long window;                                        // real columns that have to be there
};
struct BlocksCall {
    bool is_complex, wide;                              // wide: results in 32 bits
    long columns, ldx, ldr, ldy;                        // in real values
    int rows, contraction;
    bool in_pieces;                                     // x and W start at multiples of 16 bytes
};

// Up to this number of real values the contraction is one step or less than half of one: the product with scales per position and row has kernels for it, whose scales
// are those of one block. bf16, 64 to 64 channels at 2^20 positions 54 us (here 59 - 70), 16 to 16 at 10^6 16 us (40); 128 to 128 at 262144 29 us (26)
constexpr int kOneBlock = 64;
// Blocks of 64 columns and 16 rows up to which their waves divide the steps: bf16, 1024 to 1024 channels at 256 positions 6.8 us (tiles 7.5), at 512 11 (7.7)
constexpr long kSplitBlocks = 256;
// Tiles of 128 rows from which they are enough for the GPU: bf16, 1024 to 1024 at 8192 positions 18.7 us (with 64 rows 21.6), at 4096 13.6 (12.8), at 2048 11.2 (8.5)
constexpr long kWholeTiles = 384;
// Tiles of 64 rows up to which there is at most one for each compute unit, so that a second group of waves takes half of the steps. Two groups and one: bf16, 4096 to 4096 channels at 256
// positions 20.5 us and 23.7, 1024 to 1024 at 2001 (staged) 10.7 and 12.1, at 1024 (direct) 7.8 and 7.6; float32 1024 to 1024 at 500 10.3 and 12.1, 512 to 512 at 1000 7.4 and 7.9
constexpr long kOneTileEach = 256;
constexpr int kBlocksStep = 128;                        // real values of a step

inline BlocksChoice blocks_choice(const BlocksCall& q)
{
    if (q.contraction * (q.is_complex ? 2 : 1) <= kOneBlock) return { BlocksKernel::kOneScale, 0, 0, 0 };
    // a lane's part of an address in 32 bits, 48 rows of the input (complex: 24) and 12 of the results
    const bool near = 48 * q.ldx < (1L << 32) - 4096 && 12 * std::max(q.ldr, q.ldy) * (q.wide ? 4 : 2) < (1L << 32) - 4096;
    const int tiles16 = (q.rows + 15) / 16;
    const long columns = (q.columns + 63) / 64;
    if (!near || q.columns < 128 || columns * tiles16 <= kSplitBlocks)
        return { near && (q.contraction + kBlocksStep) * q.ldx < (1L << 31) ? BlocksKernel::kSplitNear : BlocksKernel::kSplitFar, 1, 1, 1 };
    if (q.is_complex) return { BlocksKernel::kTile, tiles16 > 2 && (columns + 3) / 4 * ((tiles16 + 3) / 4) >= 256 ? 4 : 2, 1, 64 };
    const bool whole_tiles = (columns + 1) / 2 * ((tiles16 + 7) / 8) >= kWholeTiles;
    const bool both = (columns + 1) / 2 * ((tiles16 + 3) / 4) <= kOneTileEach && q.contraction > (q.wide ? 3 : 7) * kBlocksStep;       // bf16, 512 to 512 at 2048 5.8 us with one, 6.1 with two
    // one or two steps: 128 to 128 channels at 262144 positions 24.0 us with 64 rows, 26.1 with 128; 512 to 512 at 16384 14.6 and 12.7
    if (!q.wide && q.contraction % kBlocksStep == 0 && ((q.ldx | q.columns) & 15) == 0 && q.in_pieces)
        return whole_tiles && q.contraction > 2 * kBlocksStep ? BlocksChoice{ BlocksKernel::kDirect, 4, 1, 128 } : BlocksChoice{ BlocksKernel::kDirect, 2, both ? 2 : 1, 128 };
    const long widest = q.wide ? 256 : 128;             // columns of a tile of 128 rows, which many rows make plenty of however few columns there are
    if (whole_tiles && q.columns >= widest) return { BlocksKernel::kStaged, 4, 1, widest };
    return { BlocksKernel::kStaged, 2, both ? 2 : 1, 128 };
}

}  // namespace tfno
