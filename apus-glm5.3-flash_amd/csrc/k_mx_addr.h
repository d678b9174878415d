/*
 * k_mx_addr.h — where the tiles of the products with MXFP4 weights (k_mx_gemm.h)
 * load from and what lies where in LDS: plain arithmetic, so that
 * tests/c/test_mx_addr.cpp follows every lane of every load on the CPU.
 *
 * A step's rows are XB bytes in LDS: 128 (128 k of MXFP8, 64 k of BF16), 64 (128 k of
 * MXFP4) or 32 (64 k of MXFP4, beside BF16), piece p of 16 bytes of row r at p ^
 * fg_rot8(r) (fg_rot4(r), bit 3 of r). A load of a wave is 1 KB, 8, 16 or 32 rows of
 * one matrix; load i of wave wv is number wv + NW * i, a whole number of rows behind
 * the wave's first one, whose swizzle it has. Dual tiles alternate the two matrices
 * load by load, for odd waves the second one. A row past the matrix lies past the buffer's span and
 * loads zeros; a piece past K is put there.
 */
#ifndef K_MX_ADDR_H
#define K_MX_ADDR_H

#include "k_ffn_addr.h"

/* Load c's row of its matrix, and its piece's byte. */
template <uint32_t XB>
FG_ADDR uint32_t mg_row(uint32_t c, uint32_t lane) {
    return XB == 128u ? 8u * c + (lane >> 3) : XB == 64u ? 16u * c + (lane >> 2) : 32u * c + (lane >> 1);
}
template <uint32_t XB>
FG_ADDR uint32_t mg_byte(uint32_t lane, uint32_t row) {
    return 16u * (XB == 128u ? (lane & 7u) ^ fg_rot8(row) : XB == 64u ? (lane & 3u) ^ fg_rot4(row)
                             : (lane & 1u) ^ ((row >> 3) & 1u));
}
/* Rows from a wave's load to its next one. */
template <uint32_t XB, uint32_t NW>
FG_ADDR uint32_t mg_rows_apart(bool dual) {
    return 1024u / XB * (dual ? NW / 2u : NW);
}
/* The offset that a lane loads from: its place, or past every buffer where its piece
 * starts `left` bytes behind the step's first or later. */
FG_ADDR uint32_t mg_cut(uint32_t off, uint32_t byte, int32_t left) {
    return (int32_t)byte >= left ? FG_OOB : off;
}

/* Byte offset of word `word` of the scales of a row; past every buffer behind the row's
 * `words`. */
FG_ADDR uint32_t mg_scale(uint32_t row, uint32_t word, uint32_t words) {
    return word < words ? row * (4u * words) + 4u * word : FG_OOB;
}
/* Where a lane reads from the scales in LDS, 16 bytes a row: quads of 16-row blocks from
 * block `first` on of the matrix that begins at unit `unit` of 64 rows. */
FG_ADDR uint32_t mg_scale_at(uint32_t unit, uint32_t first, uint32_t blocks, uint32_t lane) {
    return 1024u * unit + 16u * (16u * first + (blocks < 4u ? lane & (16u * blocks - 1u) : lane));
}

/* Operand reads, from the slot's start: x's half h of block r of 16 rows (MXFP8: k 16 g
 * and 64 + 16 g; BF16: 16 g and 16 g + 8; MXFP4, no halves: block g), with r's part a
 * constant. */
template <uint32_t XB>
FG_ADDR uint32_t mg_at_x(uint32_t first, uint32_t n, uint32_t g, uint32_t h, bool bf) {
    return first * 16u * XB + (XB == 128u ? fg_at0(n, bf ? 2u * g + h : 4u * h + g) : fg_at_codes(n, g));
}
/* W's block c of wave wc, of CB: codes [16 g, 16 g + 16) of 64 (beside BF16; there two
 * blocks of one matrix come before two of the other), or block g of 128. */
template <uint32_t WB, uint32_t CB>
FG_ADDR uint32_t mg_at_w(uint32_t ast, uint32_t wc, uint32_t n, uint32_t g, bool dual) {
    const uint32_t blk = wc * CB;
    if (WB == 64u) return ast + blk * 1024u + fg_at_codes(n, g);
    const uint32_t at = dual ? (blk >> 2) * 4u + ((blk >> 1) & 1u) : blk;
    return ast + at * 512u + n * 32u + 16u * ((g >> 1) ^ (n >> 3)) + 8u * (g & 1u);
}
template <uint32_t WB>
FG_ADDR constexpr uint32_t mg_w_step(uint32_t c, bool dual) {
    return WB == 64u ? c * 1024u : dual ? 512u * ((c & 1u) * 2u + ((c >> 1) & 1u) + (c >> 2) * 4u) : c * 512u;
}

#endif /* K_MX_ADDR_H */
