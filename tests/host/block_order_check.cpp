// CPU check of which blocks of a launch take which pieces of work (turbofno_amd/csrc/block_order.h). Lines on standard input, their kind first: "0 strips together" strips of a field (together:
// eight runs of strips side by side, as the layer norm launches them), "1 row_tiles column_tiles turns" tiles of a product, "2 columns lanes together" strips of the layer norm's gradient. Prints how
// many pieces there are that no block takes, how many that more than one does, and for the gradient the most strips of a block, the blocks of all launches and what the workspace has room for.
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
        } else if (kind == 2) {
            if (std::scanf("%ld", &turns) != 1) return 1;
            const long columns = a, strips = (columns + 4 * b - 1) / (4 * b), each = tfno::strips_of_launch(strips);
            std::vector<unsigned char> taken(strips);
            long blocks = 0, most = 0;
            for (long base = 0; base < strips; base += each) {
                const tfno::StripTurns part(base, std::min(each, strips - base), turns && std::min(each, strips - base) >= 64);
                for (long block = 0; block < part.blocks(); ++block) {
                    long n = 0;
                    for (long s = part.first((unsigned)block); s < part.last((unsigned)block); s += part.step, ++n)
                        if (s < base || s >= strips || s >= base + each) return 1;
                        else if (taken[s] < 2) ++taken[s];
                    most = std::max(most, n);
                }
                blocks += part.blocks();
            }
            print(taken);
            std::printf("%ld %ld %ld\n", most, blocks, tfno::grad_rows(columns));
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
