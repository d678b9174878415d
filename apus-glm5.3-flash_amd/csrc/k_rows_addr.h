/*
 * k_rows_addr.h — where the weight-streaming kernel (k_rows_gemm.h) loads from:
 * plain arithmetic, so that tests/c/test_ffn_addr.cpp follows every lane of every
 * load on the CPU.
 *
 * A chunk is 128 bytes of 16 weight rows, in two loads of 8 rows (h 0 and 1), and
 * the same k of x's rows; a lane takes one 16-byte piece of a row. The chunk that
 * K cuts has pieces past K: they are read as the chunk's first one and put into
 * LDS as zeros, on both sides. FP8 rows of K % 16 == 8 codes end in half a piece,
 * which is read 8 bytes early, where its row has them (in the chunk before where
 * it is the chunk's first: K >= 16).
 */
#ifndef K_ROWS_ADDR_H
#define K_ROWS_ADDR_H

#include <stdint.h>

#ifdef __HIPCC__
#define RW_ADDR __host__ __device__ __forceinline__
#else
#define RW_ADDR inline
#endif

/* The piece of its row that a lane of load h takes. */
RW_ADDR uint32_t rw_piece(uint32_t lane, uint32_t h) {
    return (lane & 7u) ^ ((h ? 4u + (lane >> 4) : lane >> 4) & 7u);
}
/* Pieces of the chunk that K cuts, of weight rows and of x's; 0: none is cut. */
RW_ADDR uint32_t rw_end(uint32_t row_bytes) { return ((row_bytes & 127u) + 15u) >> 4; }
RW_ADDR uint32_t rw_xend(bool bf, uint32_t end, bool half) {
    return bf ? end : 2u * end - (half ? 1u : 0u);
}
/* Piece q, off bytes into chunk wb of the wave's rows. */
RW_ADDR const uint8_t *rw_from(const uint8_t *wb, uint32_t off, uint32_t q, bool cut, bool half,
                               uint32_t end) {
    const bool past = cut && q >= end;
    const bool early = cut && half && (past ? 0u : q) == end - 1u;
    return wb + (past ? off - 16u * q : off) - (early ? 8 : 0);
}
/* x's piece q, off bytes into a chunk. */
RW_ADDR uint32_t rw_x(uint32_t off, uint32_t q, bool cut, uint32_t xend) {
    return cut && q >= xend ? off - 16u * q : off;
}

#endif /* K_ROWS_ADDR_H */
