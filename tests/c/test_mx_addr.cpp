/*
 * test_mx_addr.cpp — every lane of every load of the tiles with MXFP4 weights
 * (k_mx_addr.h), over ragged rows and k: each address lies inside its matrix or
 * past the buffer's span, and each operand read finds the row and k block that the
 * matrix instruction's lane stands for. Exit 0 = as expected.
 */
#include <cstdio>
#include <cstring>
#include <vector>

#include "k_mx_addr.h"

static int bad;
#define EXPECT(c, ...)                                        \
    do {                                                      \
        if (!(c)) {                                           \
            if (bad++ < 10) { printf(__VA_ARGS__); puts(""); } \
        }                                                     \
    } while (0)

/* What a 16-byte piece of LDS holds: matrix (0 x, 1 W, 2 up), row of the matrix's tile,
 * byte of the row; zeros; or nothing. */
struct Piece { int mat, row, byte; };
enum { NOTHING = -1, ZERO = -2 };

enum { BF16, MXFP8, MXFP4 };

template <int XT, bool DUAL, uint32_t WM, uint32_t WN, uint32_t RB, uint32_t CB>
static void tile(uint32_t rows, uint32_t cols, uint32_t K, uint32_t xld) {
    constexpr uint32_t NW = WM * WN, BM = 16 * RB * WM, BN = 16 * CB * WN;
    constexpr uint32_t XB = XT == MXFP4 ? 64 : 128, WB = XT == BF16 ? 32 : 64, KS = XT == BF16 ? 64 : 128;
    const uint32_t words = (K + 127) / 128, nst = (K + KS - 1) / KS, all = (nst + 1) & ~1u, wb = K / 2, xrow = XT == BF16 ? 2 * K : XT == MXFP8 ? K : wb;
    for (uint32_t j = 0; j < all; j++) {
        if (j > 2 && j + 3 < all) continue;
        std::vector<Piece> x(BM * XB / 16, Piece{NOTHING, 0, 0}), w(BN * WB / 16, Piece{NOTHING, 0, 0});
        const int64_t xleft = (int64_t)xrow - XB * j, wleft = (int64_t)wb - WB * j;
        for (uint32_t wv = 0; wv < NW; wv++)
            for (uint32_t lane = 0; lane < 64; lane++) {
                const uint32_t ar = mg_row<XB>(wv, lane), aq = mg_byte<XB>(lane, ar);
                for (uint32_t i = 0; i < BM * XB / 1024 / NW; i++) {
                    const uint32_t off = mg_cut(ar * xld + aq + i * mg_rows_apart<XB, NW>(false) * xld, aq, (int32_t)xleft);
                    const uint32_t span = rows * xld, r = ar + i * mg_rows_apart<XB, NW>(false);
                    Piece &to = x[((wv + NW * i) * 1024 + 16 * lane) / 16];
                    EXPECT(to.mat == NOTHING, "x: piece written twice");
                    if (off >= span) {
                        to = {ZERO, 0, 0};
                        EXPECT(off <= FG_OOB && (r >= rows || (int64_t)aq >= xleft), "x: row %u of %u byte %u of %lld dropped", r, rows, aq, (long long)xleft);
                    } else {
                        to = {0, (int)(off / xld), (int)(off % xld)};
                        EXPECT(r < rows && off == r * xld + aq && (int64_t)aq + 16 <= xleft, "x: row %u of %u, byte %u of %lld at %u", r, rows, aq, (long long)xleft, off);
                    }
                }
                const uint32_t br = mg_row<WB>(DUAL ? wv >> 1 : wv, lane), bq = mg_byte<WB>(lane, br);
                for (uint32_t i = 0; i < BN * WB / 1024 / NW; i++) {
                    const uint32_t off = mg_cut(br * wb + bq + i * mg_rows_apart<WB, NW>(DUAL) * wb, bq, (int32_t)wleft);
                    const uint32_t span = cols * wb, r = br + i * mg_rows_apart<WB, NW>(DUAL);
                    Piece &to = w[((wv + NW * i) * 1024 + 16 * lane) / 16];
                    EXPECT(to.mat == NOTHING, "W: piece written twice");
                    if (off >= span) {
                        to = {ZERO, 0, 0};
                        EXPECT(off <= FG_OOB && (r >= cols || (int64_t)bq >= wleft), "W: row %u of %u dropped", r, cols);
                    } else {
                        to = {DUAL && (wv & 1) ? 2 : 1, (int)(off / wb), (int)(off % wb)};
                        EXPECT(r < cols && off == r * wb + bq && (int64_t)bq + 16 <= wleft, "W: row %u of %u, byte %u", r, cols, bq);
                    }
                }
            }
        /* scales: every word of a row, none of another's, past the last row past the span;
         * each unit of 64 rows once, and each block of a wave from its rows */
        if (j == 0) {
            constexpr uint32_t OUT = BN / (DUAL ? 2 : 1), XU = XT == BF16 ? 0 : (BM + 63) / 64, WU = (OUT + 63) / 64, NU = XU + WU * (DUAL ? 2 : 1);
            std::vector<Piece> sc(64 * NU, Piece{NOTHING, 0, 0});
            for (uint32_t u = 0; u < NU; u++)
                for (uint32_t lane = 0; lane < 64; lane++) {
                    const int mat = u < XU ? 0 : u < XU + WU ? 1 : 2;
                    const uint32_t row = 64 * (mat == 0 ? u : mat == 1 ? u - XU : u - XU - WU) + lane, live = mat ? cols : rows, span = live * 4 * words;
                    sc[64 * u + lane] = row < live ? Piece{mat, (int)row, 0} : Piece{ZERO, 0, 0};
                    for (uint32_t word = 0; word < words + 4; word++) {
                        const uint32_t off = mg_scale(row, word, words);
                        if (word < words && row < live) EXPECT(off + 4 <= span && off == (row * words + word) * 4, "scale of row %u, word %u at %u", row, word, off);
                        else EXPECT(off >= span, "scale of row %u, word %u at %u of %u", row, word, off, span);
                        if (word + 4 <= words && row < live) EXPECT(off + 16 <= span, "scales of row %u, word %u at %u", row, word, off);
                    }
                }
            constexpr uint32_t WBL = DUAL ? CB / 2 : CB;
            for (uint32_t wv = 0; wv < NW; wv++)
                for (int mat = XT == BF16; mat < (DUAL ? 3 : 2); mat++)
                    for (uint32_t b = 0; b < (mat ? WBL : RB); b++)
                        for (uint32_t n = 0; n < 16; n++) {
                            const uint32_t wr = wv / WN, wc = wv % WN, first = mat ? wc * WBL : wr * RB, nb = mat ? WBL : RB, live = mat ? cols : rows;
                            const uint32_t at = mg_scale_at(mat ? XU : 0, first, nb, 16 * (b & 3) + n) + 1024 * (b / 4) + (mat == 2 ? 1024 * WU : 0);
                            const uint32_t row = 16 * (first + b) + n;
                            EXPECT(at % 16 == 0 && at < 1024 * NU, "scales read at %u", at);
                            const Piece &q = sc[at / 16];
                            if (row < live) EXPECT(q.mat == mat && q.row == (int)row, "scales of matrix %d row %u: %d, %d", mat, row, q.mat, q.row);
                            else EXPECT(q.mat == ZERO, "scales of matrix %d row %u are not zero", mat, row);
                        }
            for (uint32_t lane = 0; lane < 64; lane++)
                for (uint32_t wv = 0; wv < NW; wv++) {
                    EXPECT(mg_scale_at(0, wv / WN * RB, RB, lane) + 16 <= 1024 * NU || XT == BF16, "x's scales of lane %u", lane);
                    EXPECT(mg_scale_at(XU, wv % WN * WBL, WBL, lane) + 1024 * ((WBL - 1) / 4) + 16 <= 1024 * (XU + WU), "W's scales of lane %u", lane);
                }
        }
        /* operand reads */
        auto check = [&](const char *what, const Piece &p, int mat, uint32_t row, uint32_t live, uint32_t byte, int64_t left) {
            if (row >= live || (int64_t)byte >= left) EXPECT(p.mat == ZERO, "%s: row %u byte %u is not zero", what, row, byte);
            else EXPECT(p.mat == mat && p.row == (int)row && p.byte == (int)byte, "%s: row %u byte %u holds %d, row %d, byte %d", what, row, byte, p.mat, p.row, p.byte);
        };
        for (uint32_t wr = 0; wr < WM; wr++)
            for (uint32_t wc = 0; wc < WN; wc++)
                for (uint32_t n = 0; n < 16; n++)
                    for (uint32_t g = 0; g < 4; g++) {
                        for (uint32_t r = 0; r < RB; r++) {
                            const uint32_t row = 16 * (wr * RB + r) + n;
                            for (uint32_t h = 0; h < (XB == 128 ? 2u : 1u); h++) {
                                const uint32_t at = mg_at_x<XB>(wr * RB, n, g, h, XT == BF16) + r * 16 * XB;
                                EXPECT(at % 16 == 0 && at + 16 <= BM * XB, "x: read at %u", at);
                                check("x", x[at / 16], 0, row, rows, XT == BF16 ? 32 * g + 16 * h : XT == MXFP8 ? 64 * h + 16 * g : 16 * g, xleft);
                            }
                        }
                        for (uint32_t c = 0; c < CB; c++) {
                            const uint32_t blk = wc * CB + c, row = 16 * (DUAL ? blk >> 1 : blk) + n;
                            const uint32_t at = mg_at_w<WB, CB>(0, wc, n, g, DUAL) + mg_w_step<WB>(c, DUAL);
                            EXPECT(at % (WB / 4) == 0 && at + WB / 4 <= BN * WB, "W: read at %u", at);
                            check("W", w[at / 16], DUAL && (blk & 1) ? 2 : 1, row, cols, WB == 64 ? 16 * g : 16 * (g >> 1), wleft);
                            EXPECT(WB == 64 || at % 16 == 8 * (g & 1), "W: half %u", at % 16);
                        }
                    }
    }
}

template <int XT, bool DUAL, uint32_t WM, uint32_t WN, uint32_t RB, uint32_t CB>
static void shapes() {
    constexpr uint32_t BM = 16 * RB * WM, OUT = 16 * CB * WN / (DUAL ? 2 : 1);
    for (uint32_t K : {32u, 64u, 96u, 128u, 160u, 256u, 288u, 1120u, 4096u})
        for (uint32_t rows : {1u, 15u, BM - 1, BM})
            for (uint32_t cols : {1u, 17u, OUT - 1, OUT})
                for (uint32_t pad : {0u, 48u})
                    if (rows <= BM && cols <= OUT && (XT == BF16 || !pad))
                        tile<XT, DUAL, WM, WN, RB, CB>(rows, cols, K, XT == BF16 ? 2 * K + pad : XT == MXFP8 ? K : K / 2);
}
template <int XT, uint32_t WM, uint32_t WN, uint32_t RB, uint32_t CB>
static void both() {
    shapes<XT, false, WM, WN, RB, CB>();
    shapes<XT, true, WM, WN, RB, CB>();
}
template <uint32_t WM, uint32_t WN, uint32_t RB, uint32_t CB>
static void types() {
    both<MXFP8, WM, WN, RB, CB>();
    both<MXFP4, WM, WN, RB, CB>();
}

int main() {
    types<2, 2, 8, 8>();
    types<2, 2, 8, 4>();
    types<2, 2, 4, 4>();
    types<2, 2, 2, 4>();
    types<2, 2, 2, 2>();
    types<1, 2, 2, 2>();
    both<BF16, 1, 4, 16, 4>();
    both<BF16, 1, 4, 12, 4>();
    both<BF16, 1, 4, 8, 4>();
    both<BF16, 1, 4, 8, 2>();
    both<BF16, 1, 4, 4, 2>();
    printf(bad ? "FAIL\n" : "PASS\n");
    return bad != 0;
}
