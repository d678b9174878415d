/*
 * The dense feed-forward tiles' loads on the CPU (k_ffn_addr.h), and those of the
 * weight-streaming kernel (k_rows_addr.h): every lane of every load of every
 * stage or chunk, over ragged rows and k. Each access lies inside its
 * own row of the matrix or is marked as past the buffer, with its whole 16 bytes
 * below 2^32; and what the operand reads then find in LDS is the matrix's value,
 * or zero past its end.
 */
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "k_ffn_addr.h"
#include "k_rows_addr.h"

static long g_loads, g_marked;

#define REQUIRE(ok, ...)                                                            \
    do {                                                                            \
        if (!(ok)) {                                                                \
            std::printf("FAIL %s:%d %s: ", __FILE__, __LINE__, #ok);                \
            std::printf(__VA_ARGS__);                                               \
            std::printf("\n");                                                      \
            std::exit(1);                                                           \
        }                                                                           \
    } while (0)

/* Lane's 16 bytes at 32-bit offset off of a buffer of span bytes that begins at
 * byte `base` of a matrix of `bytes` bytes: its address there, or -1 = zeros. */
static long load(long base, uint32_t off, uint32_t span, long bytes) {
    g_loads++;
    if (off >= span) {
        REQUIRE((uint64_t)off + 16u <= (uint64_t)1 << 32, "offset %#x wraps", off);
        g_marked++;
        return -1;
    }
    REQUIRE((uint64_t)off + 16u <= span, "offset %#x in a span of %#x", off, span);
    const long at = base + (long)off;
    REQUIRE(at >= 0 && at + 16 <= bytes, "byte %ld of %ld", at, bytes);
    return at;
}

/* byte i of a matrix; never 0 */
static uint8_t value(long i) { return (uint8_t)(1 + i * 7 % 251); }

static void put(std::vector<uint8_t> &lds, uint32_t to, long at) {
    for (uint32_t e = 0; e < 16; e++) lds[to + e] = at < 0 ? 0 : value(at + e);
}

/* FP8 codes [N, K]: tiles of BN rows (dual: of two matrices of the same shape, BN
 * / 2 rows each) */
static void codes(uint32_t N, uint32_t K, uint32_t BN, bool dual) {
    const uint32_t outn = dual ? BN / 2 : BN, nst = (K + 63u) / 64u;
    const bool half = K & 8u;
    const long bytes = (long)N * K;
    for (uint32_t col0 = 0; col0 < N; col0 += outn) {
        const uint32_t cols = N - col0 < outn ? N - col0 : outn;
        std::vector<uint32_t> off(BN / 16 * 64), kq(64 * 4);
        for (uint32_t wv = 0; wv < 4; wv++)
            for (uint32_t lane = 0; lane < 64; lane++)
                for (uint32_t b = wv; b < BN / 16; b += 4)
                    off[b * 64 + lane] = fg_place_codes(dual, b, lane, cols, K, kq[wv * 64 + lane]);
        for (uint32_t j = 0; j < nst; j++) {
            std::vector<uint8_t> lds(BN * 64u);
            const uint32_t left = K - 64u * j;
            long base = (long)col0 * K + 64 * j;
            if (half && j + 1 == nst) {
                base -= 8;
                for (uint32_t i = 0; i < off.size(); i++)
                    off[i] = fg_half(off[i], left, kq[(i / 64) % 4 * 64 + i % 64]);
            }
            for (uint32_t i = 0; i < off.size(); i++) {
                const uint32_t o = fg_cut(off[i], left, kq[(i / 64) % 4 * 64 + i % 64]);
                const long at = load(base, o, FG_SPAN, bytes);
                put(lds, i * 16u, at);
            }
            for (uint32_t b = 0; b < BN / 16; b++)
                for (uint32_t n = 0; n < 16; n++)
                    for (uint32_t g = 0; g < 4; g++) {
                        const uint8_t *v = &lds[b * 1024u + fg_at_codes(n, g)];
                        const bool down = half && j + 1 == nst && left - 16u * g == 8u;
                        const uint32_t mr = 16u * (dual ? b >> 1 : b) + n;
                        for (uint32_t e = 0; e < 16; e++) {
                            const uint32_t k = 64u * j + 16u * g + e;
                            const uint8_t got = !down ? v[e] : e < 8 ? v[8 + e] : 0;
                            const uint8_t want = mr < cols && k < K ? value((long)(col0 + mr) * K + k) : 0;
                            REQUIRE(got == want, "codes N %u K %u tile %u row %u k %u", N, K, BN, col0 + mr, k);
                        }
                    }
        }
    }
}

/* bf16 [R, K], rows ld apart, k fast: tiles of T rows (dual: 16 by 16 with those
 * of another matrix of the same shape) */
template <uint32_t T>
static void k_fast(uint32_t R, uint32_t K, uint32_t ld, bool dual) {
    const uint32_t outn = dual ? T / 2 : T, nst = (K + 63u) / 64u;
    const long bytes = 2 * ((long)(R - 1) * ld + K);
    for (uint32_t row0 = 0; row0 < R; row0 += outn) {
        const uint32_t live = R - row0 < outn ? R - row0 : outn;
        std::vector<uint32_t> off(T / 8 * 64), kq(64 * 4);
        for (uint32_t wv = 0; wv < 4; wv++)
            for (uint32_t lane = 0; lane < 64; lane++)
                for (uint32_t c = wv; c < T / 8; c += 4)
                    off[c * 64 + lane] = dual ? fg_place_dual(c, lane, live, ld, kq[wv * 64 + lane])
                                              : fg_place<0, T>(c, lane, live, ld, kq[wv * 64 + lane]);
        for (uint32_t j = 0; j < nst; j++) {
            std::vector<uint8_t> lds(T * 128u);
            const uint32_t left = K - 64u * j;
            const long base = 2 * ((long)row0 * ld + 64 * j);
            for (uint32_t i = 0; i < off.size(); i++) {
                const uint32_t o = fg_cut(off[i], left, kq[(i / 64) % 4 * 64 + i % 64]);
                const long at = load(base, o, fg_span<0>(left, ld), bytes);
                REQUIRE(at < 0 || at % (2l * ld) + 16 <= 2l * K, "k fast R %u K %u ld %u: past a row", R, K, ld);
                put(lds, i * 16u, at);
            }
            for (uint32_t r = 0; r < T; r++)
                for (uint32_t k = 0; k < 64; k++) {
                    const uint32_t mr = dual ? 16u * (r >> 5) + (r & 15u) : r;
                    const uint8_t *v = &lds[(r / 16) * 2048u + fg_at0(r % 16, k / 8) + 2u * (k % 8)];
                    for (uint32_t e = 0; e < 2; e++) {
                        const long at = 2 * ((long)(row0 + mr) * ld + 64 * j + k) + e;
                        REQUIRE(v[e] == (mr < live && 64 * j + k < K ? value(at) : 0), "k fast R %u K %u ld %u tile %u row %u k %u", R, K, ld,
                                T, row0 + mr, 64 * j + k);
                    }
                }
        }
    }
}

/* bf16 [K, ld], the operand's R rows along a row of it (whole vectors) */
template <uint32_t W>
static void k_slow(uint32_t R, uint32_t K, uint32_t ld) {
    const uint32_t nst = (K + 63u) / 64u, r8 = (R + 7u) & ~7u;
    const long bytes = 2 * ((long)(K - 1) * ld + r8);
    for (uint32_t row0 = 0; row0 < R; row0 += W) {
        const uint32_t live = R - row0 < W ? R - row0 : W;
        uint32_t kq = 0;
        for (uint32_t j = 0; j < nst; j++) {
            std::vector<uint8_t> lds(W * 128u);
            const uint32_t left = K - 64u * j;
            const long base = 2 * ((long)row0 + 64l * j * ld);
            for (uint32_t c = 0; c < W / 8; c++)
                for (uint32_t lane = 0; lane < 64; lane++) {
                    const uint32_t o = fg_place<1, W>(c, lane, live, ld, kq);
                    const long at = load(base, o, fg_span<1>(left, ld), bytes);
                    REQUIRE(at < 0 || at % (2l * ld) + 16 <= 2l * r8, "k slow R %u K %u ld %u: past a row", R, K, ld);
                    put(lds, c * 1024u + lane * 16u, at);
                }
            for (uint32_t k = 0; k < 64; k++)
                for (uint32_t r = 0; r < W; r++) {
                    const uint8_t *v = fg_at1<W>(lds.data(), k, r / 16) + 2u * (r % 16);
                    for (uint32_t e = 0; e < 2; e++) {
                        const long at = 2 * ((long)(row0 + r) + (64l * j + k) * ld) + e;
                        const bool in = r < ((live + 7u) & ~7u) && 64 * j + k < K;
                        REQUIRE(v[e] == (in ? value(at) : 0), "k slow R %u K %u ld %u tile %u row %u k %u", R, K, ld, W, row0 + r, 64 * j + k);
                    }
                }
        }
    }
}

template <uint32_t T>
static void tiles(uint32_t R, uint32_t K) {
    k_fast<T>(R, K, K, false);
    k_fast<T>(R, K, K + 24, false);
    k_fast<T>(R, K, K, true);
    k_slow<T>(R, K, (R + 7u) & ~7u);
    k_slow<T>(R, K + 3, ((R + 7u) & ~7u) + 16);
}

/* the weight rows [O, K] of wave groups of NT blocks of 16, chunk by chunk: FP8
 * codes, or bf16 where bf */
static void weights(uint32_t O, uint32_t K, uint32_t NT, bool bf) {
    const uint32_t KB = bf ? 2 * K : K, nch = (KB + 127u) / 128u, end = rw_end(KB);
    const bool half = !bf && (K & 8u);
    const long bytes = (long)O * KB;
    for (uint32_t row0 = 0; row0 < O; row0 += 16 * NT)
        for (uint32_t b = 0; b < NT; b++)
            for (uint32_t c = 0; c < nch; c++)
                for (uint32_t i = 0; i < 128; i++) {
                    const uint32_t lane = i % 64, h = i / 64, q = rw_piece(lane, h), r = 16 * b + 8 * h + lane / 8;
                    const uint32_t last = O - 1 - row0, row = row0 + (r < last ? r : last);
                    const bool cut = end && c == nch - 1;
                    const uint8_t *zero = nullptr;
                    const long at = rw_from(zero, (row - row0) * KB + 16 * q, q, cut, half, end) - zero + (long)row0 * KB + 128l * c;
                    g_loads++;
                    REQUIRE(at >= 0 && at + 16 <= bytes, "weights O %u K %u bf %d: byte %ld of %ld", O, K, bf, at, bytes);
                    REQUIRE(at >= (long)row * KB && at + 16 <= (long)(row + 1) * KB, "weights O %u K %u bf %d: past a row", O, K, bf);
                    if (cut && q >= end) {               /* becomes zeros */
                        g_marked++;
                        continue;
                    }
                    /* where LDS row r has the piece, it is the row's, or its last 8
                     * bytes are in the upper half */
                    const long want = (long)row * KB + 128l * c + 16l * q;
                    const bool down = cut && half && q == end - 1;
                    REQUIRE(at == want - (down ? 8 : 0), "weights O %u K %u bf %d row %u chunk %u piece %u", O, K, bf, row, c, q);
                    REQUIRE(want + (down ? 8 : 16) <= (long)(row + 1) * KB, "weights O %u K %u bf %d: a piece past K", O, K, bf);
                }
}

/* x's pieces of a chunk: those of K are kept and lie in the row, the others are
 * read inside the row */
static void inputs(uint32_t K, bool bf) {
    const uint32_t KB = bf ? 2 * K : K, nch = (KB + 127u) / 128u, end = rw_end(KB), pieces = bf ? 8 : 16;
    const uint32_t xend = rw_xend(bf, end, !bf && (K & 8u));
    for (uint32_t c = 0; c < nch; c++)
        for (uint32_t q = 0; q < pieces; q++) {
            const bool cut = end && c == nch - 1;
            const long at = (long)c * pieces * 16 + rw_x(16 * q, q, cut, xend), own = 16l * (c * pieces + q);
            g_loads++;
            REQUIRE(at >= 0 && at + 16 <= 2l * K, "x K %u bf %d: byte %ld", K, bf, at);
            REQUIRE((own + 16 <= 2l * K) == !(cut && q >= xend), "x K %u bf %d chunk %u piece %u", K, bf, c, q);
            REQUIRE((cut && q >= xend) || at == own, "x K %u bf %d chunk %u piece %u", K, bf, c, q);
        }
}

int main() {
    for (uint32_t K = 8; K <= 1032; K += 8)
        for (int bf = 0; bf < 2; bf++) {
            if (!bf && K < 16) continue;                 /* a half piece needs a whole one */
            inputs(K, bf);
            for (uint32_t O : {1u, 5u, 16u, 17u, 40u, 96u, 129u})
                for (uint32_t NT : {1u, 2u}) weights(O, K, NT, bf);
        }
    static const uint32_t rows[] = {1, 5, 33, 64, 130, 265};
    for (uint32_t R : rows) {
        for (uint32_t K : {16u, 24u, 40u, 56u, 64u, 72u, 88u, 120u, 128u, 136u, 200u, 1032u})
            for (uint32_t BN : {64u, 128u, 256u}) {
                codes(R, K, BN, false);
                codes(R, K, BN, true);
            }
        for (uint32_t K : {8u, 16u, 56u, 64u, 72u, 200u}) {
            tiles<64>(R, K);
            tiles<128>(R, K);
            tiles<192>(R, K);
            tiles<256>(R, K);
        }
    }
    std::printf("%ld loads, %ld of them past a matrix: PASS\n", g_loads, g_marked);
    return 0;
}
