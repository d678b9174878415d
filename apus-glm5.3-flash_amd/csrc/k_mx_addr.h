/*
 * k_mx_addr.h — where the tiles of the products with MXFP4 weights (k_mx_gemm.h)
 * load from and what lies where in LDS: plain arithmetic, so that
 * tests/c/test_mx_addr.cpp follows every lane of every load on the CPU.
 *
 * A step's rows are XB bytes (128: MXFP8, 64: MXFP4) in LDS, piece p of 16 bytes of
 * row r at p ^ fg_rot8(r) (fg_rot4). A load of a wave is 1 KB, 8 or 16 rows; load i
 * of wave wv is number wv + NW * i, a whole number of rows behind the wave's first
 * one, whose swizzle it has. A row past the matrix lies past the buffer's span and
 * loads zeros; a piece past K is put there.
 */
#ifndef K_MX_ADDR_H
#define K_MX_ADDR_H

#include "k_ffn_addr.h"

/* Load c's row of the tile (of one matrix: dual tiles alternate 16 rows of two), and
 * its piece's byte. */
template <uint32_t XB>
FG_ADDR uint32_t mg_row(uint32_t c, uint32_t lane) {
    return XB == 128u ? 8u * c + (lane >> 3) : 16u * c + (lane >> 2);
}
template <uint32_t XB>
FG_ADDR uint32_t mg_byte(uint32_t lane, uint32_t row) {
    return 16u * (XB == 128u ? (lane & 7u) ^ fg_rot8(row) : (lane & 3u) ^ fg_rot4(row));
}
/* Rows from a wave's load to its next one. */
template <uint32_t XB, uint32_t NW>
FG_ADDR uint32_t mg_rows_apart(bool dual) {
    return (XB == 128u ? 8u : dual ? 8u : 16u) * NW;
}
/* The offset that a lane loads from: its place, or past every buffer where its piece
 * starts `left` bytes behind the step's first or later. */
FG_ADDR uint32_t mg_cut(uint32_t off, uint32_t byte, int32_t left) {
    return (int32_t)byte >= left ? FG_OOB : off;
}

/* Word e of a step's scales in LDS: rows of x, then of W (dual: the gate's, then the up
 * projection's). Returns W's row of the tile. */
FG_ADDR uint32_t mg_scale_row(uint32_t e, uint32_t BM, uint32_t BN, bool dual, bool &second) {
    const uint32_t c = e - BM;
    second = dual && c >= BN / 2u;
    return second ? c - BN / 2u : c;
}

/* Operand reads, from the slot's start, without the immediate part: x's piece of k
 * half h (MXFP8: k 16 g and 64 + 16 g of row n; MXFP4: block g), W's, their scales. */
template <uint32_t XB>
FG_ADDR uint32_t mg_at_x(uint32_t first, uint32_t n, uint32_t g, uint32_t h) {
    return first * 16u * XB + (XB == 128u ? fg_at0(n, 4u * h + g) : fg_at_codes(n, g));
}
FG_ADDR uint32_t mg_at_w(uint32_t ast, uint32_t first, uint32_t n, uint32_t g) {
    return ast + first * 1024u + fg_at_codes(n, g);
}
FG_ADDR uint32_t mg_at_sx(uint32_t base, uint32_t first, uint32_t n, uint32_t g) {
    return base + 4u * (16u * first + n) + g;
}
FG_ADDR uint32_t mg_at_sw(uint32_t base, uint32_t BM, uint32_t first, uint32_t n, uint32_t g, bool dual) {
    return base + 4u * (BM + (dual ? 8u : 16u) * first + n) + g;
}
/* ... and of block c behind the first. */
FG_ADDR constexpr uint32_t mg_sw_step(uint32_t c, uint32_t BN, bool dual) {
    return dual ? 64u * (c >> 1) + (c & 1u) * 2u * BN : 64u * c;
}

#endif /* K_MX_ADDR_H */
