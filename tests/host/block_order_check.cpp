// CPU check of which blocks of a launch take which strips of a field (turbofno_amd/csrc/block_order.h). For "strips together" on standard input prints how many strips there are that no
// block takes, and how many that more than one does. `together`: eight runs of strips side by side, as the layer norm launches them.
#include "../../turbofno_amd/csrc/block_order.h"
#include <cstdio>
#include <vector>
int main()
{
    long strips;
    int together;
    while (std::scanf("%ld %d", &strips, &together) == 2) {
        const long run = together ? (strips + 7) / 8 : 0, blocks = together ? 8 * run : strips, rows = tfno::grid_rows(blocks);
        std::vector<unsigned char> taken(strips);
        for (long id = 0; id < (rows == 1 ? blocks : rows * tfno::kGridRow); ++id) {
            const long place = run ? tfno::side_by_side(id, run) : id;
            if (place < strips && taken[place] < 2) ++taken[place];
        }
        long none = 0, twice = 0;
        for (unsigned char t : taken) none += t == 0, twice += t > 1;
        std::printf("%ld %ld\n", none, twice);
    }
    return 0;
}
