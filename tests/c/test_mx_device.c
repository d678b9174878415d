/*
 * test_mx_device.c — which device the entries of the norm, of microscaled values
 * and of the products with them use and leave current, and what their backward
 * passes lay out in the workspace, on a stub of the runtime with two devices: the
 * host layer's own object
 * (ghip_backend.c.o) over the few runtime calls and launchers that it needs here.
 * The backend's device is 1. Exit 0 = as expected.
 */
#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "backend_hip.h"
#include "ghip_internal.h"

static int current, launches, launched_on = -1, fail_launch, fail_malloc;
static char streams[2];                          /* a stream of each device */
#define STREAM(d) ((void *)&streams[d])

hipError_t hipGetDeviceCount(int *n) { *n = 2; return hipSuccess; }
hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) { current = d; return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int d) {
    (void)d;
    memset(p, 0, sizeof *p);
    strcpy(p->gcnArchName, "gfx950");
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t a, int d) {
    (void)a; (void)d;
    *v = 256;
    return hipSuccess;
}
hipError_t hipStreamCreate(hipStream_t *s) { *s = STREAM(1); return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d) { *d = (int)((char *)s - streams); return hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned f) { (void)f; *p = malloc(n); return hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) {
    if (fail_malloc) return hipErrorOutOfMemory;
    *p = malloc(n);
    return hipSuccess;
}
hipError_t hipMemcpy(void *d, const void *s, size_t n, hipMemcpyKind k) { (void)k; memcpy(d, s, n); return hipSuccess; }
hipError_t hipMemset(void *d, int v, size_t n) { memset(d, v, n); return hipSuccess; }
const char *hipGetErrorString(hipError_t e) { (void)e; return "an error"; }

hipError_t ghip_moe_decode_init(void) { return hipSuccess; }
hipError_t ghip_linear_init(uint32_t n) { (void)n; return hipSuccess; }
hipError_t ghip_moe_prefill_init(void) { return hipSuccess; }
hipError_t ghip_ffn_init(uint32_t n) { (void)n; return hipSuccess; }
hipError_t ghip_pf_scratch_init(int d) { (void)d; return hipSuccess; }
size_t ghip_ffn_part_bytes(size_t M, size_t N, size_t K) { (void)M; (void)N; (void)K; return 0; }
static hipError_t launch(void) {
    launches++;
    launched_on = current;
    return fail_launch ? hipErrorInvalidValue : hipSuccess;
}
hipError_t ghip_launch_ffn(int mode, const GhipProd *p, const GhipEp *ep, hipStream_t st) {
    (void)mode; (void)p; (void)ep; (void)st;
    return launch();
}
static const void *read_as_bf16[2];              /* the weights of the last dx */
hipError_t ghip_launch_ffn_grads(const GhipProd *dx, const GhipEp *edx, const GhipProd *dw, const GhipEp *edw, const GhipFfnSum *sum,
                                 hipStream_t st) {
    (void)edx; (void)edw; (void)sum; (void)st;
    if (dw) fail_launch = 1;                     /* frozen weights */
    read_as_bf16[0] = dx ? dx->b : NULL;
    read_as_bf16[1] = dx ? dx->b2 : NULL;
    return launch();
}
size_t ghip_mx_scale_ld(size_t K) { return (K + 127) / 128 * 4; }
hipError_t ghip_launch_mx_quantize(int type, const uint16_t *x, uint8_t *codes, uint8_t *scales, size_t R, size_t K, size_t ldx, hipStream_t st) {
    (void)type; (void)x; (void)codes; (void)scales; (void)R; (void)K; (void)ldx; (void)st;
    return launch();
}
static const void *written[8];
static int nwritten;
hipError_t ghip_launch_mx_dequant(int type, const uint8_t *codes, const uint8_t *scales, uint16_t *out, size_t R, size_t K, size_t ldo, hipStream_t st) {
    (void)type; (void)codes; (void)scales; (void)R; (void)K; (void)ldo; (void)st;
    written[nwritten++ & 7] = out;
    return launch();
}
hipError_t ghip_launch_rmsnorm(const GhipNorm *p, hipStream_t st) { (void)p; (void)st; return launch(); }
size_t ghip_rmsnorm_part_bytes(size_t M, size_t D) { return M * D * 4; }
hipError_t ghip_launch_rmsnorm_grad(const GhipNormGrad *p, hipStream_t st) { (void)p; (void)st; return launch(); }
hipError_t ghip_launch_mx(int mode, const GhipMxProd *p, const GhipEp *ep, hipStream_t st) {
    (void)mode; (void)p; (void)ep; (void)st;
    return launch();
}

static uint16_t buf[16384] __attribute__((aligned(16)));
static uint8_t *const codes = (uint8_t *)buf, *const ws = (uint8_t *)(buf + 4096);
#define WS (sizeof buf - 8192)

enum { ENTRIES = 8 };
static int call(int which, void *stream) {
    nwritten = 0;
    switch (which) {
    case 0: return apus_ghip_mx_quantize_dev(APUS_GHIP_MXFP4, buf, codes, codes, 4, 64, 0, stream);
    case 1: return apus_ghip_mx_dequant_dev(APUS_GHIP_MXFP8, codes, codes, buf, 4, 64, 0, stream);
    case 2: return apus_ghip_rmsnorm_dev(buf, buf, buf, buf, NULL, codes, codes, NULL, 4, 64, 0, 0, 0, 0, 1e-5f, stream);
    case 3: return apus_ghip_rmsnorm_backward_dev(buf, buf, NULL, buf, buf, buf, buf, 4, 64, 0, 0, 0, 0, 1e-5f, ws, WS, stream);
    case 4:
        return apus_ghip_mxfp4_linear_dev(codes, codes, APUS_GHIP_MXFP8, codes, codes, buf, buf, buf, 4, 8, 64, 0, 0, 0, APUS_GHIP_ACT_GELU, stream);
    case 5:
        return apus_ghip_mxfp4_gated_dev(codes, codes, codes, codes, APUS_GHIP_BF16, codes, NULL, buf, 4, 8, 64, 0, 0, APUS_GHIP_ACT_SILU, 1.0f,
                                         stream);
    case 6:
        return apus_ghip_mxfp4_linear_backward_dev(codes, codes, buf, NULL, buf, buf, buf, 4, 8, 64, 0, 0, 0, APUS_GHIP_ACT_SILU, ws, WS, stream);
    default:
        return apus_ghip_mxfp4_gated_backward_dev(codes, codes, codes, codes, buf, buf, buf, 4, 8, 64, 0, 0, 0, APUS_GHIP_ACT_SILU, 0.0f, ws, WS,
                                                  stream);
    }
}

static int bad;
static void expect(const char *what, int which, int rc, int want_rc, int was, int some) {
    const int ok = rc == want_rc && current == was && (some ? launches > 0 && launched_on == 1 : launches == 0);
    if (!ok) {
        bad = 1;
        printf("%s, entry %d: rc %d, device %d current after %d, %d launches on %d (%s)\n", what, which, rc, current, was, launches,
               launched_on, apus_ghip_last_error());
    }
    launches = 0;
    launched_on = -1;
}

int main(int argc, char **argv) {
    const int first = argc > 1 ? atoi(argv[1]) : 0;   /* the call that initialises */
    setenv("APUS_GHIP_DEVICE", "1", 1);
    current = 0;
    fail_malloc = 1;
    expect("initialisation that fails", first, call(first, NULL), 1, 0, 0);
    fail_malloc = 0;
    expect("first call", first, call(first, NULL), 0, 0, 1);
    for (int which = 0; which < ENTRIES; which++)
        for (int was = 0; was < 2; was++) {
            current = was;
            expect("null stream", which, call(which, NULL), 0, was, 1);
            expect("own stream", which, call(which, STREAM(1)), 0, was, 1);
            expect("the other device's stream", which, call(which, STREAM(0)), 1, was, 0);
            fail_launch = 1;
            expect("failed launch", which, call(which, NULL), 1, was, 1);
            fail_launch = 0;
        }
    /* the weights that dx reads are those that were laid out, whole and inside the workspace */
    for (int which = 6; which < ENTRIES; which++) {
        const int rc = call(which, NULL), n = which - 5;
        for (int k = 0; k < n; k++)
            if (rc || nwritten != n || read_as_bf16[k] != written[k] || written[k] != ws + k * 8 * 64 * 2) {
                bad = 1;
                printf("entry %d: rc %d, matrix %d of %d written at %p, read at %p\n", which, rc, k, nwritten, written[k], read_as_bf16[k]);
            }
    }
    printf(bad ? "FAIL\n" : "PASS\n");
    return bad;
}
