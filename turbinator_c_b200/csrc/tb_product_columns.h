/*
 * How many columns a product's instruction is issued for.  With 128 rows (256
 * for a pair of CTAs) the tensor cores take any multiple of 16 up to 256 of
 * 16-bit operands; of 8-bit ones a pair takes multiples of 32: each CTA brings
 * half of the columns, and 8-bit operands come sixteen rows at a time.
 */
#ifndef TB_PRODUCT_COLUMNS_H
#define TB_PRODUCT_COLUMNS_H

#ifdef __CUDACC__
#define TB_BOTH_SIDES __host__ __device__
#else
#define TB_BOTH_SIDES
#endif

namespace tb_tensor {

constexpr int kMostColumns = 256;
/* For a tile of `columns` (1 to 256): what is past them is multiplied too, and not stored. */
TB_BOTH_SIDES constexpr int issued_columns(bool i8, bool pair, int columns) {
    return i8 && pair ? (columns + 31) / 32 * 32 : (columns + 15) / 16 * 16;
}
/* Which of a tile's columns a pair's second CTA brings: from here on as many again. */
TB_BOTH_SIDES constexpr int second_half(bool i8, int columns) { return issued_columns(i8, true, columns) / 2; }

} /* namespace tb_tensor */

#endif
