/*
 * test_mx_rows_addr.cpp — every lane of every access of the weight-streaming kernel with
 * MXFP4 weights (k_mx_rows_addr.h), as k_mx_rows.hip makes them: each load lies inside
 * its matrix or past its buffer, whose base is a row of the matrix, each LDS access
 * inside its part of the launch's LDS; each operand read finds the row and the k block
 * that the matrix instruction's lane stands for; each output leaves once, from the sums
 * of its own row, column and waves. Exit 0 = as expected.
 */
#include <cstdio>
#include <map>
#include <set>
#include <vector>

#include "k_mx_rows_addr.h"

static int bad;
#define EXPECT(c, ...)                                        \
    do {                                                      \
        if (!(c)) {                                           \
            if (bad++ < 10) { printf(__VA_ARGS__); puts(""); } \
        }                                                     \
    } while (0)

/* 16 bytes of LDS: byte `byte` of a matrix's row `row`; zeros; or nothing. */
struct Piece { int64_t row, byte; };
enum { NOTHING = -1, ZERO = -2 };

template <uint32_t XR, uint32_t KS>
static void launch(uint32_t M, uint32_t N, uint32_t K, uint32_t xld, uint32_t ncu) {
    const MrCut cut = mr_cut(M, N, K, XR, KS, ncu);
    if (cut.mr == 0) return;
    constexpr uint32_t GPP = MR_WAVES / KS, XI = XR == 256 ? 4 : XR == 128 ? 2 : 1;
    const uint32_t nst = mr_steps(K), wb = K / 2, ld = 4 * nst, most = mr_share_most(nst, KS);
    const uint32_t xbytes = XR == 256 ? 2 * K : XR == 128 ? K : wb;
    EXPECT(cut.lds <= MR_LDS_MAX && cut.mr <= 16 && (uint64_t)cut.mr * cut.tiles >= M && (uint64_t)cut.mr * (cut.tiles - 1) < M, "tiles");
    EXPECT((uint64_t)cut.grid * cut.turns >= cut.blocks && cut.grid <= cut.blocks && (uint64_t)cut.blocks * 16 * GPP >= N, "blocks");
    EXPECT(mr_lds_x(MR_WAVES, cut.mr, XR, most) <= cut.lds, "LDS");
    std::map<uint64_t, int> outs;
    const bool every = cut.grid * cut.tiles <= 12;
    for (uint32_t by = 0; by < cut.tiles; by++) {
        if (!every && by > 0 && by + 1 < cut.tiles) continue;
        const uint32_t m0 = by * cut.mr, mrows = M - m0 < cut.mr ? M - m0 : cut.mr;
        for (uint32_t bx = 0; bx < cut.grid; bx++) {
            if (!every && bx > 0 && bx + 1 < cut.grid) continue;
            for (uint32_t wv = 0; wv < MR_WAVES; wv++) {
                const uint32_t part = wv % KS, slot = wv / KS;
                const MrShare s = mr_share<KS>(part, nst);
                EXPECT(s.from <= s.to && s.to <= nst && s.to - s.from <= most && s.from % 2 == 0, "share %u", wv);
                EXPECT(part ? s.from == mr_share<KS>(part - 1, nst).to : s.from == 0, "shares meet");
                EXPECT(part + 1 < KS || s.to == nst, "shares end");
                const uint32_t nc = s.to - s.from, nq = (nc + 3) / 4;
                if (nc == 0) continue;
                /* the copy of x */
                const uint32_t xl = mr_lds_x(wv, mrows, XR, most), xend = xl + mrows * XR * most;
                EXPECT(xl >= mr_lds_codes(MR_WAVES) && xend <= cut.lds && xl == mr_lds_x(0, mrows, XR, most) + wv * (xend - xl), "x's part");
                std::vector<Piece> x((xend - xl) / 16, Piece{NOTHING, 0});
                const uint32_t all = mrows * nc * (XR / 16);
                for (uint32_t v = 0; v < (all + 511) / 512 * 512; v++) {
                    if (v >= all) continue;
                    const MrPiece at = mr_piece<XR>(v, nc);
                    const uint32_t byte = (s.from + at.t) * XR + 16 * at.q, spot = at.t * (mrows * XR) + mr_spot<XR>(at.r, at.q);
                    EXPECT(at.r < mrows && at.t < nc && spot % 16 == 0 && xl + spot + 16 <= xend, "x's place");
                    if (byte < xbytes)
                        EXPECT((uint64_t)(m0 + at.r) * xld + byte + 16 <= (uint64_t)(M - 1) * xld + xbytes && byte + 16 <= xbytes, "x at %u", byte);
                    Piece &q = x[spot / 16];
                    EXPECT(q.row == NOTHING, "two pieces of x in one place");
                    q = byte < xbytes ? Piece{(int64_t)m0 + at.r, byte} : Piece{ZERO, 0};
                }
                const uint32_t wend = 64 * s.to < wb ? 64 * s.to : wb;
                EXPECT(mr_lds_codes(wv) + 4096 <= mr_lds_codes(MR_WAVES), "W's part");
                for (uint32_t blk = bx, turn = 0; turn <= cut.turns; turn++, blk += cut.grid) {  /* one ahead of the last */
                    const uint32_t first = mr_first<KS>(blk, slot), live = mr_live(first, N), base = mr_base(first, N);
                    EXPECT(base < N && live <= 16 && (live == 0 || (base == first && first + live <= N)), "rows %u + %u", base, live);
                    EXPECT(live == (blk < cut.blocks && first < N ? (N - first < 16 ? N - first : 16u) : 0u), "count %u", live);
                    for (uint32_t lq = 0; lq < nq; lq++) {
                        for (uint32_t lane = 0; lane < 64; lane++) {     /* scales */
                            const uint32_t n = lane & 15, t = s.from + 4 * lq + (lane >> 4), off = mr_scale(n, t, nst);
                            const bool in = off != FG_OOB && off < live * ld;
                            EXPECT(in == (n < live && t < nst), "scale %u of row %u", t, n);
                            if (in) EXPECT(off == n * ld + 4 * t && (uint64_t)base * ld + off + 4 <= (uint64_t)N * ld, "scale");
                            const uint32_t tc = t < nst - 1 ? t : nst - 1, mine = n < mrows - 1 ? n : mrows - 1;
                            EXPECT((uint64_t)(m0 + mine) * ld + 4 * tc + 4 <= (uint64_t)M * ld, "x's scale");
                        }
                        for (uint32_t h = 0; h < 2; h++) {               /* codes */
                            const uint32_t step = s.from + 4 * lq + 2 * h;
                            std::vector<Piece> w(128, Piece{NOTHING, 0});
                            for (uint32_t i = 0; i < 2; i++)
                                for (uint32_t lane = 0; lane < 64; lane++) {
                                    const uint32_t off = mr_code(i, lane, step, wend, wb), at = mr_code_put(i, lane);
                                    const bool in = off != FG_OOB && off < live * wb;
                                    EXPECT(off == FG_OOB || off < FG_SPAN, "mark");
                                    if (in) EXPECT((uint64_t)base * wb + off + 16 <= (uint64_t)N * wb && off % wb + 16 <= wend, "code at %u", off);
                                    EXPECT(at % 16 == 0 && at + 16 <= 2048 && w[at / 16].row == NOTHING, "W's place");
                                    w[at / 16] = in ? Piece{(int64_t)base + off / wb, off % wb} : Piece{ZERO, 0};
                                }
                            for (uint32_t i = 0; i < 2 && step + i < s.to && blk < cut.blocks; i++)
                                for (uint32_t lane = 0; lane < 64; lane++) {
                                    const uint32_t n = lane & 15, g = lane >> 4, t = step + i, mine = n < mrows - 1 ? n : mrows - 1;
                                    const Piece &c = w[mr_code_get(n, g, i) / 16];
                                    const bool in = n < live && 64 * t + 16 * g < wb;
                                    EXPECT(in ? c.row == first + n && c.byte == 64 * t + 16 * g : c.row == ZERO, "W's operand %u %u", n, g);
                                    for (uint32_t k = 0; k < XI; k++) {
                                        const uint32_t at = (t - s.from) * (mrows * XR) + mr_spot<XR>(mine, mr_operand<XR>(g, k));
                                        EXPECT(xl + at + 16 <= xend, "x's operand");
                                        const Piece &q = x[at / 16];
                                        const uint32_t byte = t * XR + (XR == 256 ? 64 * g + 16 * k : XR == 128 ? 16 * g + 64 * k : 16 * g);
                                        EXPECT(byte < xbytes ? q.row == m0 + mine && q.byte == byte : q.row == ZERO, "x's piece %u %u", n, g);
                                    }
                                }
                        }
                    }
                }
            }
            /* the join: what each float of the sums is */
            struct Sum { int wave, row, mat, col; };
            std::vector<Sum> red(MR_WAVES * 512, Sum{-1, 0, 0, 0});
            for (uint32_t wv = 0; wv < MR_WAVES; wv++)
                for (uint32_t b = 0; b < 2; b++)
                    for (uint32_t lane = 0; lane < 64; lane++)
                        for (uint32_t i = 0; i < 4; i++) {
                            const uint32_t n = lane & 15, g = lane >> 4, at = mr_sum_put(wv, n, b, g) + i;
                            EXPECT(at < red.size() && 4 * at + 4 <= mr_lds_codes(0) && red[at].wave < 0, "sum");
                            red[at] = Sum{(int)wv, (int)n, (int)b, (int)(4 * g + i)};
                        }
            for (uint32_t blk = bx; blk < cut.blocks; blk += cut.grid)
                for (uint32_t tid = 0; tid < 64 * MR_WAVES; tid++) {
                    const MrOut at = mr_out(tid);
                    const uint32_t o = mr_first<KS>(blk, at.slot) + at.c;
                    if (!(at.slot < GPP && at.m < mrows && o < N)) continue;
                    outs[(uint64_t)(m0 + at.m) * N + o]++;
                    for (uint32_t k = 0; k < KS; k++)
                        for (uint32_t b = 0; b < 2; b++) {
                            const Sum &s = red[mr_sum_get<KS>(at.slot, at.m, at.c) + 512 * k + 16 * b];
                            EXPECT(s.wave == (int)(at.slot * KS + k) && s.row == (int)at.m && s.mat == (int)b && s.col == (int)at.c, "join");
                        }
                }
        }
    }
    for (auto &v : outs) EXPECT(v.second == 1 && v.first < (uint64_t)M * N, "output %llu", (unsigned long long)v.first);
    if (every) EXPECT(outs.size() == (uint64_t)M * N, "%zu outputs of %u x %u", outs.size(), M, N);
}

template <uint32_t XR, uint32_t KS>
static void all() {
    const uint32_t shape[][3] = {{1, 1, 32}, {1, 15, 64}, {1, 16, 128}, {1, 17, 160}, {1, 70, 96}, {3, 300, 544}, {16, 33, 1024},
                                 {17, 129, 2080}, {40, 64, 4096}, {65, 40, 8224}, {5, 530, 6400}, {20, 20, 20000}, {3, 9000, 256},
                                 {16, 300, 4096}, {1, 12288, 4096}, {5, 12288, 4096}, {16, 4096, 12288}, {2, 48, 32768}, {192, 257, 352},
                                 {7, 31, 288}, {33, 100, 1184}, {300, 20000, 64}};
    const uint32_t unit = XR == 256 ? 2 : 1, part = XR == 64 ? 2 : 1;
    for (auto &s : shape)
        for (uint32_t ncu : {256u, 3u})
            for (uint32_t pad : {0u, 48u}) launch<XR, KS>(s[0], s[1], s[2], s[2] * unit / part + pad, ncu);
}

int main(void) {
    all<256, 8>();
    all<256, 4>();
    all<128, 8>();
    all<128, 4>();
    all<64, 8>();
    all<64, 4>();
    const uint32_t most = 0x7fffffffu;                   /* rows at the end of the range, and blocks behind them */
    EXPECT(mr_live(most - 7, most) == 7 && mr_live(most, most) == 0 && mr_live(most + 20000, most) == 0 && mr_live(0, most) == 16, "range");
    if (bad) printf("%d faults\n", bad);
    puts(bad ? "FAIL" : "PASS");
    return bad != 0;
}
