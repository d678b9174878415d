/*
 * k_ffn_addr.h — where the tiles of the dense feed-forward products
 * (k_ffn_gemm.h) load from and what lies where in LDS: plain arithmetic, so that
 * tests/c/test_ffn_addr.cpp follows every lane of every load on the CPU, over
 * ragged rows and k.
 *
 * A load of a wave is 1 KB: lane l's 16 bytes go to byte 16 l of it. Its offset
 * is of 32 bits from a base; FG_OOB and the 15 bytes behind it are past every
 * buffer (at most FG_SPAN bytes) and end at 2^32, so such a lane loads zeros and
 * touches no memory. The mark is not moved, but for the codes' (fg_place_codes).
 */
#ifndef K_FFN_ADDR_H
#define K_FFN_ADDR_H

#include <stdint.h>

#ifdef __HIPCC__
#define FG_ADDR __host__ __device__ __forceinline__
#else
#define FG_ADDR inline
#endif

#define FG_OOB 0xFFFFFFF0u                       /* past every buffer: loads zeros */
#define FG_SPAN 0x80000000u                      /* valid offsets are below */

/* Layout 1: what the 32-byte slots of k's row of W values are XORed with, so
 * that the 8 k rows two lane groups read from one slot lie in distinct banks. */
template <uint32_t W>
FG_ADDR uint32_t fg_swizzle(uint32_t k) {
    static_assert(W % 64u == 0, "half rounds of the banks");
    return W % 128u ? ((k >> 1) & 1u) | ((k >> 3) & 2u) : ((k & 3u) << 1) | ((k >> 4) & 1u);
}

/* Layout 0 (FP8 codes): what the 16-byte pieces of row r are XORed with. A
 * ds_read_b128 is served 16 lanes at a time, rows 0-3 and 12-15 of one lane
 * group together with rows 4-11 of the next: the rotation gives the middle rows
 * a set of values that the other group's XOR with 2 (1) maps to itself, so the
 * 16 pieces fill the 64 banks. With r >> 1 alone 49% of the LDS cycles were
 * conflicts (gated FP8 1111 x 2048 x 4096: 52 us, now 49). */
FG_ADDR uint32_t fg_rot8(uint32_t r) { return ((r >> 1) + 2u) & 7u; }
FG_ADDR uint32_t fg_rot4(uint32_t r) { return ((r >> 2) + 1u) & 3u; }

/* Byte offset of lane `lane` in load c of a bf16 stage whose operand has `live`
 * rows ld elements apart (layout 1: k rows ld apart, live of their W values).
 * kq: the stage's k that the piece starts at (layout 0; the same for every c of
 * a wave). */
template <int LAYOUT, uint32_t W>
FG_ADDR uint32_t fg_place(uint32_t c, uint32_t lane, uint32_t live, uint32_t ld, uint32_t &kq) {
    if constexpr (LAYOUT == 0) {
        const uint32_t r = 8u * c + (lane >> 3), q = (lane & 7u) ^ fg_rot8(r);
        kq = 8u * q;
        return r < live ? r * ld * 2u + 16u * q : FG_OOB;
    } else {
        const uint32_t e = c * 64u + lane, k = e / (W / 8u), s = e % (W / 8u);
        const uint32_t q = s ^ 2u * fg_swizzle<W>(k);
        return 8u * q < live ? k * ld * 2u + 16u * q : FG_OOB;
    }
}
/* Dual modes: 16 rows of the gate's and the up projection's alternate. */
FG_ADDR uint32_t fg_place_dual(uint32_t c, uint32_t lane, uint32_t live, uint32_t ld, uint32_t &kq) {
    const uint32_t r = 8u * c + (lane >> 3), q = (lane & 7u) ^ fg_rot8(r);
    const uint32_t mr = 16u * (r >> 5) + (r & 15u);
    kq = 8u * q;
    return mr < live ? mr * ld * 2u + 16u * q : FG_OOB;
}
/* FP8: load b is 16 rows of 64 codes. Rows past the matrix get a mark that fg_half
 * may move by 8 and that still ends below 2^32 (a select there instead costs up
 * to 3%). */
FG_ADDR uint32_t fg_place_codes(bool dual, uint32_t b, uint32_t lane, uint32_t live, uint32_t ld,
                                uint32_t &kq) {
    const uint32_t r = lane >> 2, q = (lane & 3u) ^ fg_rot4(r), mr = 16u * (dual ? b >> 1 : b) + r;
    kq = 16u * q;
    return mr < live ? mr * ld + 16u * q : FG_OOB - 16u;
}
/* FP8 rows of K % 16 == 8 codes end in half a piece: in the last stage, of `left`
 * codes, the base is 8 bytes early, and so is that piece; the others are not. */
FG_ADDR uint32_t fg_half(uint32_t off, uint32_t left, uint32_t kq) {
    return off + (left - kq == 8u ? 0u : 8u);
}
/* A stage that K cuts. Layout 0 drops the pieces past it, layout 1 the k rows, by
 * the buffer's end. */
FG_ADDR uint32_t fg_cut(uint32_t off, uint32_t left, uint32_t kq) { return kq >= left ? FG_OOB : off; }
template <int LAYOUT>
FG_ADDR uint32_t fg_span(uint32_t left, uint32_t ld) {
    return LAYOUT == 1 && left < 64u ? left * ld * 2u : FG_SPAN;
}

/* Where an operand lies in LDS: layout 0, 16-byte piece p of row n of a block of
 * 16 rows; FP8, codes 16 g of it; layout 1, row block blk (16 values) of k. */
FG_ADDR uint32_t fg_at0(uint32_t n, uint32_t p) { return n * 128u + 16u * (p ^ fg_rot8(n)); }
FG_ADDR uint32_t fg_at_codes(uint32_t n, uint32_t g) { return n * 64u + 16u * (g ^ fg_rot4(n)); }
template <uint32_t W>
FG_ADDR const uint8_t *fg_at1(const uint8_t *stage, uint32_t k, uint32_t blk) {
    return stage + k * (2u * W) + (blk ^ fg_swizzle<W>(k)) * 32u;
}

#endif /* K_FFN_ADDR_H */
