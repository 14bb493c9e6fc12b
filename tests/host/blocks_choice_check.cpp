// CPU check of which kernel of the product in 8 bits with scales by blocks takes a call (turbofno_amd/csrc/mix_blocks_choice.h). Lines "complex wide columns rows contraction ldx ldr ldy
// in_pieces" on standard input; prints the kernel, 16 rows of its waves, groups of waves and the columns that it needs.
#include "../../turbofno_amd/csrc/mix_blocks_choice.h"
#include <cstdio>
int main()
{
    int is_complex, wide, rows, contraction, in_pieces;
    long columns, ldx, ldr, ldy;
    while (std::scanf("%d %d %ld %d %d %ld %ld %ld %d", &is_complex, &wide, &columns, &rows, &contraction, &ldx, &ldr, &ldy, &in_pieces) == 9) {
        const tfno::BlocksChoice c = tfno::blocks_choice({ is_complex != 0, wide != 0, columns, ldx, ldr, ldy, rows, contraction, in_pieces != 0 });
        std::printf("%d %d %d %ld\n", (int)c.kernel, c.nt, c.groups, c.window);
    }
    return 0;
}
