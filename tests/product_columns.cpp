/* Every count of columns that a tile may have, of either kind of operand, alone and in a pair: the instruction has a
 * shape that the tensor cores take, covers the tile, and a pair's halves meet. */
#include <cstdio>

#include "tb_product_columns.h"

int main() {
    int wrong = 0;
    for (int i8 = 0; i8 < 2; ++i8)
        for (int pair = 0; pair < 2; ++pair)
            for (int columns = 1; columns <= tb_tensor::kMostColumns; ++columns) {
                const int n = tb_tensor::issued_columns(i8, pair, columns), step = i8 && pair ? 32 : 16;
                if (n % step || n < step || n > 256 || n < columns || n - columns >= step) ++wrong, std::printf("%d %d %d: %d\n", i8, pair, columns, n);
                if (pair && 2 * tb_tensor::second_half(i8, columns) != n) ++wrong, std::printf("%d %d: halves\n", i8, columns);
            }
    return wrong != 0;
}
