/*
 * k_mx_rows_addr.h — where the weight-streaming kernel of the gated products with
 * MXFP4 weights (k_mx_rows.hip) loads from, what lies where in LDS, and how a launch
 * is cut: plain arithmetic, so that tests/c/test_mx_rows_addr.cpp follows every lane of
 * every access on the CPU.
 *
 * A step is 128 k, 64 bytes of a row of W; a wave's share of k is whole lines of W, two
 * steps. A workgroup's 8 waves are 8 / KS slots of 16 weight rows (of the gate's matrix
 * and of the up projection's), k over KS waves. Codes and scales are loaded through
 * buffers of the rows that a block has in its matrix, of none past the last one, whose
 * base is a row of the matrix all the same; what a wave does not load is put past the
 * buffer (FG_OOB).
 */
#ifndef K_MX_ROWS_ADDR_H
#define K_MX_ROWS_ADDR_H

#include <stddef.h>

#include "k_ffn_addr.h"

#define MR_WAVES 8u
#define MR_LDS_MAX (160u * 1024u)

FG_ADDR uint32_t mr_least(uint32_t a, uint32_t b) { return a < b ? a : b; }

/* Steps of k, and the wave's: [from, to), whole lines but for the last step. */
FG_ADDR uint32_t mr_steps(uint32_t K) { return (K + 127u) >> 7; }
struct MrShare {
    uint32_t from, to;
};
template <uint32_t KS>
FG_ADDR MrShare mr_share(uint32_t part, uint32_t nst) {
    const uint32_t lines = (nst + 1u) >> 1;
    return {2u * (part * lines / KS), mr_least(2u * ((part + 1u) * lines / KS), nst)};
}
/* Most steps of a share. */
FG_ADDR uint32_t mr_share_most(uint32_t nst, uint32_t ks) { return 2u * (((nst + 1u) / 2u + ks - 1u) / ks); }

/* x, XR bytes of a row in a step (256 BF16, 128 MXFP8, 64 MXFP4): piece v of a wave's
 * copy is 16 bytes of row r, step t of its share, piece q. In LDS a step's rows follow
 * each other, pieces swapped so that the 16 rows that a lane group reads lie in distinct
 * banks. */
struct MrPiece {
    uint32_t r, t, q;
};
template <uint32_t XR>
FG_ADDR MrPiece mr_piece(uint32_t v, uint32_t steps) {
    const uint32_t r = v / (steps * (XR / 16u)), e = v - r * (steps * (XR / 16u));
    return {r, e / (XR / 16u), e % (XR / 16u)};
}
template <uint32_t XR>
FG_ADDR uint32_t mr_spot(uint32_t r, uint32_t q) {
    return r * XR + 16u * (XR == 256u ? q ^ (r & 15u) : XR == 128u ? q ^ fg_rot8(r) : q ^ fg_rot4(r));
}
/* Piece i of lane group g's operand: k 32 g + 8 i of BF16, 16 g and 64 + 16 g of MXFP8,
 * 32 g of MXFP4. */
template <uint32_t XR>
FG_ADDR uint32_t mr_operand(uint32_t g, uint32_t i) { return XR == 256u ? 4u * g + i : XR == 128u ? 4u * i + g : g; }

/* The rows of a block: the first one of a slot, how many there are in a matrix of N, and
 * a row that is there. */
template <uint32_t KS>
FG_ADDR uint32_t mr_first(uint32_t blk, uint32_t slot) { return (blk * (MR_WAVES / KS) + slot) * 16u; }
FG_ADDR uint32_t mr_live(uint32_t first, uint32_t N) {
    /* the difference fits 31 bits and a sign, N being under 2^31 and the stream ending a
     * few blocks behind it; a guarded subtraction that wraps is what a compiler has
     * drawn wrong conclusions from (build.py's flags) */
    const int32_t left = (int32_t)(N - first);
    return (uint32_t)(left > 16 ? 16 : left > 0 ? left : 0);
}
FG_ADDR uint32_t mr_base(uint32_t first, uint32_t N) { return mr_least(first, N - 1u); }

/* Offsets into a block's rows: row n's scales of step t; load i of the two steps from
 * `step` on, 16 bytes of row 8 i + lane / 8. `end`: the bytes of a row that the share has. */
FG_ADDR uint32_t mr_scale(uint32_t n, uint32_t t, uint32_t nst) { return t < nst ? n * (4u * nst) + 4u * t : FG_OOB; }
FG_ADDR uint32_t mr_code(uint32_t i, uint32_t lane, uint32_t step, uint32_t end, uint32_t wb) {
    const uint32_t r = 8u * i + (lane >> 3), byte = 64u * step + 16u * ((lane & 7u) ^ fg_rot8(r));
    return byte < end ? r * wb + byte : FG_OOB;
}
/* Two steps of a matrix's codes in LDS, 2 KB: as they are loaded, and as lane (n, g) reads
 * block g of step i. */
FG_ADDR uint32_t mr_code_put(uint32_t i, uint32_t lane) { return 1024u * i + 16u * lane; }
FG_ADDR uint32_t mr_code_get(uint32_t n, uint32_t g, uint32_t i) { return fg_at0(n, 4u * i + g); }

/* LDS: the block's sums (f32), each wave's codes, each wave's copy of x. */
FG_ADDR constexpr uint32_t mr_lds_codes(uint32_t wave) { return MR_WAVES * 2048u + wave * 4096u; }
FG_ADDR uint32_t mr_lds_x(uint32_t wave, uint32_t rows, uint32_t xr, uint32_t most) {
    return mr_lds_codes(MR_WAVES) + wave * (rows * xr * most);
}
/* Sums: of x's row n and weight rows 4 g + [0, 4) of matrix b, and of row m and column
 * c of slot's first wave, 512 floats from wave to wave, 16 from the gate's to the up one's. */
FG_ADDR uint32_t mr_sum_put(uint32_t wave, uint32_t n, uint32_t b, uint32_t g) {
    return (wave * 16u + n) * 32u + 16u * b + 4u * g;
}
template <uint32_t KS>
FG_ADDR uint32_t mr_sum_get(uint32_t slot, uint32_t m, uint32_t c) { return (slot * KS * 16u + m) * 32u + c; }
/* Output v of a block: slot, row of x, column of the slot. */
struct MrOut {
    uint32_t slot, m, c;
};
FG_ADDR MrOut mr_out(uint32_t v) { return {v >> 8, v >> 4 & 15u, v & 15u}; }

/* How a launch is cut: mr rows of x a tile, as many as fit beside the sums and two steps
 * of weights (up to 16, tiles of as many rows each); blocks of weight rows, `turns` of
 * them one after the other in each of `grid` workgroups, as many as the chip has room
 * for. 0 rows: k is too long. */
struct MrCut {
    uint32_t mr, tiles, lds, blocks, grid, turns, occ;
};
inline MrCut mr_cut(uint32_t M, uint32_t N, uint32_t K, uint32_t xr, uint32_t ks, uint32_t ncu) {
    const size_t row = (size_t)MR_WAVES * xr * mr_share_most(mr_steps(K), ks), rest = mr_lds_codes(MR_WAVES);
    size_t most = (MR_LDS_MAX - rest) / row;
    if (most > 16) most = 16;
    MrCut r = {0, 0, 0, 0, 0, 0, 0};
    if (most == 0) return r;
    r.tiles = (uint32_t)(((size_t)M + most - 1) / most);
    r.mr = (uint32_t)(((size_t)M + r.tiles - 1) / r.tiles);
    r.lds = (uint32_t)(rest + r.mr * row);
    const size_t cols = 16 * (MR_WAVES / ks);
    r.blocks = (uint32_t)(((size_t)N + cols - 1) / cols);
    r.occ = r.lds <= MR_LDS_MAX / 2 ? 2 : 1;
    const size_t room = ((size_t)ncu * r.occ + r.tiles - 1) / r.tiles;
    r.turns = (uint32_t)((r.blocks + room - 1) / room);
    r.grid = (r.blocks + r.turns - 1) / r.turns;
    return r;
}

#endif /* K_MX_ROWS_ADDR_H */
