/*
 * k_rows.hip — weight-streaming linear for a few activation rows (gfx950):
 * Y [M, N] = bf16(X [M, K] . W [N, K]^T) with FP8-block weights (c/gdsa.h:
 * 525-534) or BF16 ones (c/bf16.h:712-767), from one decode row over
 * speculative verifies and short prompts to a few dozen rows.
 *
 * A wave owns NT groups of 16 weight rows and, with KS waves splitting K, a
 * run of 128-byte-wide chunks of them. Per chunk it loads the weights (two
 * whole-line 16-byte loads a lane per group) and the same k range of MR rows
 * of x (1 KB loads: 4 rows of 256 bytes against FP8 codes, 8 of 128 against
 * BF16) into registers, writes both to a wave-private LDS slot and reads
 * them back in the layout of v_mfma_f32_16x16x32_bf16; NA chunks are in
 * flight. No barrier until the KS partial sums meet in LDS, added in a fixed
 * order (deterministic). Streaming x beside the weights, instead of staging
 * all of it first, takes any M x K; the weights are read once per MR rows.
 * LDS pieces are XOR-swizzled by row so the operand reads hit distinct banks.
 * Rows past M or N re-read the last row: computed, never stored.
 *
 * What bounds it: HBM for the larger weights (LM head 154880 x 4096, M = 1:
 * 180 us, 7.1 TB/s; o_proj 4096 x 16384, M = 4: 11.9 us, 5.7 TB/s), else the
 * chunk round trip of a wave (rw_cfgs' chunk times; the LDS traffic of x
 * from 16 rows on) and ~2.3 us of launch, first load and reduction.
 * Against passes of <= 4 rows over the weights: o_proj M = 4 46.7 -> 11.9 us,
 * q_a 1536 x 4096 M = 11 13.3 -> 5.1, LM head M = 1 205 -> 180, M = 8
 * 411 -> 181; and against the MFMA GEMM, q_a M = 64 14.6 -> 7.5.
 */
#include "k_rows_gemm.h"

/* a launch's row tiles (grid y) and workgroups along the weight rows (grid x:
 * under 2^32 threads); more take several launches */
#define RW_MAX_TILES ((size_t)65535)
#define RW_MAX_BLOCKS (GHIP_MAX_THREADS / (RW_NW * 64))

/* One launchable form: MR rows of x, NT groups of 16 weight rows per wave, K
 * over KS waves. chunk: measured microseconds of a wave's chunk step. */
struct RwCfg {
    uint32_t mr, nt, ks;
    float chunk;
    const void *kern;
    uint32_t lds;
    void (*launch)(dim3, uint32_t, hipStream_t, hipEvent_t, hipEvent_t, const uint8_t *,
                   const float *, const uint16_t *, uint16_t *, uint32_t, uint32_t, uint32_t,
                   const uint32_t *, uint32_t, uint32_t);
};

template <bool BF, int MR, int NT, int KS, int NA, int SL>
static void rw_run(dim3 grid, uint32_t lds, hipStream_t st, hipEvent_t e0, hipEvent_t e1,
                   const uint8_t *w, const float *s, const uint16_t *x, uint16_t *y, uint32_t M,
                   uint32_t O, uint32_t K, const uint32_t *exact, uint32_t blk0,
                   uint32_t tile0) {
    GHIP_LAUNCH(e0, e1, (k_rows_gemm<BF, MR, NT, KS, NA, SL, GHIP_EP_STORE>), grid,
                dim3(RW_NW * 64), lds, st, w, s, x, y, M, O, K, exact, blk0, tile0, RwMore{});
}

#define RW_CFG(BF, MR, NT, KS, NA, SL, T)                                                  \
    {MR, NT, KS, T, (const void *)k_rows_gemm<BF, MR, NT, KS, NA, SL, GHIP_EP_STORE>, rw_lds<BF, MR, NT, SL>(), \
     rw_run<BF, MR, NT, KS, NA, SL>}

/* Two chunks in flight up to 16 rows of x (o_proj, M = 8: 14.0 us against
 * 14.9 with one), one where x's registers and LDS slots grow past that
 * (q_a, M = 32: 7.6 against 8.0 with two). */
static const RwCfg rw_fp8[] = {
    RW_CFG(false, 4, 1, 8, 2, 2, 0.55f),  RW_CFG(false, 4, 1, 4, 2, 2, 0.55f),
    RW_CFG(false, 4, 1, 2, 2, 2, 0.56f),  RW_CFG(false, 8, 1, 8, 2, 2, 0.65f),
    RW_CFG(false, 8, 1, 4, 2, 2, 0.65f),  RW_CFG(false, 8, 1, 2, 2, 2, 0.62f),
    RW_CFG(false, 16, 1, 8, 1, 1, 0.85f), RW_CFG(false, 16, 2, 8, 2, 2, 1.30f),
    RW_CFG(false, 16, 2, 4, 2, 2, 1.30f), RW_CFG(false, 32, 1, 8, 1, 1, 1.30f),
    RW_CFG(false, 32, 2, 8, 1, 1, 1.70f), RW_CFG(false, 32, 2, 4, 1, 1, 1.70f),
    RW_CFG(false, 64, 2, 4, 1, 1, 2.20f),
};
static const RwCfg rw_bf16[] = {
    RW_CFG(true, 8, 1, 8, 2, 2, 0.50f),  RW_CFG(true, 8, 1, 4, 2, 2, 0.50f),
    RW_CFG(true, 16, 1, 8, 2, 2, 0.58f), RW_CFG(true, 16, 1, 4, 2, 2, 0.60f),
    RW_CFG(true, 16, 2, 4, 2, 2, 0.75f), RW_CFG(true, 32, 1, 8, 1, 1, 0.85f),
    RW_CFG(true, 32, 2, 8, 1, 1, 1.20f), RW_CFG(true, 32, 2, 4, 1, 1, 1.15f),
};

/* Estimated microseconds of a form: 2.3 + the larger of rounds of the chip x
 * a wave's chunks x the chunk time and the weights at 6.5 TB/s + a tenth of
 * the other (within 20% of the measured times over M = 1..192 and the shapes
 * above). Where the weights' bytes decide, the form with less LDS a workgroup
 * is the better one by a few percent (more workgroups a CU; LM head, M = 1:
 * 8 rows x 1 group 178 us, 16 x 2 184). Forms of 4 and 8 rows only take as
 * many: more row tiles would re-read the weights. */
static float rw_estimate(const RwCfg &c, bool bf, size_t M, size_t N, size_t K, uint32_t n_cu) {
    if (c.mr < 16 && M > c.mr) return 1e30f;
    const double gpp = 16.0 * c.nt * (RW_NW / c.ks);
    const double wgs = (double)(size_t)((N + gpp - 1) / gpp) * (double)((M + c.mr - 1) / c.mr);
    const double nch = (double)(bf ? 2 * K : K) / 128.0;
    const double rounds = (double)(size_t)((wgs + n_cu - 1) / n_cu);
    const double nc = (double)(size_t)((nch + c.ks - 1) / c.ks);
    const double hbm = (double)N * (double)(bf ? 2 * K : K) / 6.5e6;
    /* A round's first loads and reduction: hidden under no other workgroup by
     * the form of 64 rows (16384 x 1536: 13.4 us at M = 64 in one round, 25.4
     * at 128 in two, where the MFMA GEMM takes 21.5), and past the first round
     * of other FP8 forms with two or more blocks where a wave has few chunks
     * (32768 x 1024: M = 48 in six rounds of 16 rows 37.9 us, M = 64 in four
     * of 32 27.5, the GEMM 16.6 and 18; 16384 x 1536, M = 80, three rounds 22,
     * the GEMM 20.5). */
    const double over = c.mr > 32 ? 3.8 * rounds
                        : !bf && c.mr * c.nt >= 32 && nc < 8.0 ? 2.0 * (rounds - 1.0)
                                                         : 0.0;
    const double t = rounds * nc * c.chunk + over;
    const double lds = t < hbm ? 0.0015 * hbm * c.mr * c.nt : 0.0;
    return (float)(2.3 + (t > hbm ? t + 0.1 * hbm : hbm + 0.1 * t) + lds);
}

static const RwCfg *rw_pick(bool bf, size_t M, size_t N, size_t K, uint32_t n_cu, float *est) {
    const RwCfg *best = nullptr;
    const RwCfg *tab = bf ? rw_bf16 : rw_fp8;
    const size_t n = bf ? sizeof rw_bf16 / sizeof *rw_bf16 : sizeof rw_fp8 / sizeof *rw_fp8;
    for (size_t i = 0; i < n; i++) {
        const float c = rw_estimate(tab[i], bf, M, N, K, n_cu);
        if (!best || c < *est) {
            best = &tab[i];
            *est = c;
        }
    }
    return best;
}

/* 32-bit offsets inside a wave's rows */
extern "C" int ghip_rows_fits(int bf, size_t M, size_t N, size_t K, const void *w, const void *x) {
    return M > 0 && M <= 0x7fffffffu && N > 0 && N <= 0x7fffffffu && K > 0
        && K <= ((size_t)1 << 24) && K % (bf ? 64 : 128) == 0 && ((uintptr_t)w & 15) == 0
        && ((uintptr_t)x & 15) == 0;
}

extern "C" float ghip_rows_estimate(int bf, size_t M, size_t N, size_t K, uint32_t n_cu) {
    float est = 0.0f;
    (void)rw_pick(bf != 0, M, N, K, n_cu, &est);
    return est;
}

extern "C" uint32_t ghip_rows_form(int bf, size_t M, size_t N, size_t K, uint32_t n_cu) {
    float est = 0.0f;
    const RwCfg *c = rw_pick(bf != 0, M, N, K, n_cu, &est);
    return c->mr << 16 | c->nt << 8 | c->ks;
}

extern "C" hipError_t ghip_launch_rows(int bf, const void *w, const float *scales,
                                       const uint16_t *x, uint16_t *y, size_t M, size_t N,
                                       size_t K, const uint32_t *exact_dev, uint32_t n_cu,
                                       hipEvent_t e0, hipEvent_t e1, hipStream_t st) {
    if (!ghip_rows_fits(bf, M, N, K, w, x) || n_cu == 0) return hipErrorInvalidValue;
    float est = 0.0f;
    const RwCfg *c = rw_pick(bf != 0, M, N, K, n_cu, &est);
    const size_t gpp = 16u * c->nt * (RW_NW / c->ks), blocks = (N + gpp - 1) / gpp;
    const size_t tiles = (M + c->mr - 1) / c->mr;
    for (size_t t0 = 0; t0 < tiles; t0 += RW_MAX_TILES)
        for (size_t b0 = 0; b0 < blocks; b0 += RW_MAX_BLOCKS) {
            const size_t nt = tiles - t0 < RW_MAX_TILES ? tiles - t0 : RW_MAX_TILES;
            const size_t nb = blocks - b0 < RW_MAX_BLOCKS ? blocks - b0 : RW_MAX_BLOCKS;
            c->launch(dim3((uint32_t)nb, (uint32_t)nt), c->lds, st,
                      t0 == 0 && b0 == 0 ? e0 : nullptr,
                      t0 + nt == tiles && b0 + nb == blocks ? e1 : nullptr, (const uint8_t *)w,
                      scales, x, y, (uint32_t)M, (uint32_t)N, (uint32_t)K, exact_dev,
                      (uint32_t)b0, (uint32_t)t0);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

extern "C" hipError_t ghip_rows_init(void) {
    for (const RwCfg &c : rw_fp8) {
        hipError_t e = hipFuncSetAttribute(c.kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)c.lds);
        if (e != hipSuccess) return e;
    }
    for (const RwCfg &c : rw_bf16) {
        hipError_t e = hipFuncSetAttribute(c.kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)c.lds);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
