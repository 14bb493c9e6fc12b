// CPU check of which blocks of a launch take which pieces of work (turbofno_amd/csrc/block_order.h). Lines on standard input, their kind first: "0 strips together" strips of a field (together:
// eight runs of strips side by side, as the layer norm launches them), "1 row_tiles column_tiles turns" tiles of a product. Prints how many pieces there are that no block takes, and how many that
// more than one does.
#include "../../turbofno_amd/csrc/block_order.h"
#include <cstdio>
#include <vector>
static long launched(long blocks) { return tfno::grid_rows(blocks) == 1 ? blocks : tfno::grid_rows(blocks) * tfno::kGridRow; }
static void print(const std::vector<unsigned char>& taken)
{
    long none = 0, twice = 0;
    for (unsigned char t : taken) none += t == 0, twice += t > 1;
    std::printf("%ld %ld\n", none, twice);
}
int main()
{
    long kind, a, b, turns;
    while (std::scanf("%ld %ld %ld", &kind, &a, &b) == 3) {
        if (kind == 0) {
            const long strips = a, run = b ? (strips + 7) / 8 : 0;
            std::vector<unsigned char> taken(strips);
            for (long id = 0; id < launched(run ? 8 * run : strips); ++id) {
                const long place = run ? tfno::side_by_side(id, run) : id;
                if (place < strips && taken[place] < 2) ++taken[place];
            }
            print(taken);
        } else {
            if (std::scanf("%ld", &turns) != 1) return 1;
            std::vector<unsigned char> taken(a * b);
            for (long id = 0; id < launched(tfno::tile_blocks((int)a, b)); ++id) {
                const tfno::Tile tile = tfno::tile_of(id, (int)a, b, tfno::tiles_by_xcd(b), turns != 0);
                if (tile.column < b && taken[tile.column * a + tile.row] < 2) ++taken[tile.column * a + tile.row];
            }
            print(taken);
        }
    }
    return 0;
}
