/*
 * test_ffn_device.c — which device the dense feed-forward entries use and leave
 * current, on a stub of the runtime with two devices: the host layer's own object
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
hipError_t ghip_launch_ffn_grads(const GhipProd *dx, const GhipEp *edx, const GhipProd *dw, const GhipEp *edw, const GhipFfnSum *sum,
                                 hipStream_t st) {
    (void)dx; (void)edx; (void)dw; (void)edw; (void)sum; (void)st;
    return launch();
}

static uint16_t buf[4096] __attribute__((aligned(16)));

static int call(int which, void *stream) {
    switch (which) {
    case 0: return apus_ghip_bf16_linear_ep_dev(buf, buf, NULL, NULL, buf, 4, 8, 16, 0, 0, 0, APUS_GHIP_ACT_SILU, stream);
    case 1:
        return apus_ghip_fp8blk_linear_ep_dev((uint8_t *)buf, (float *)buf, buf, NULL, NULL, buf, 4, 8, 16, 0, 0, 0, APUS_GHIP_ACT_NONE, 0,
                                              stream);
    case 2: return apus_ghip_bf16_gated_dev(buf, buf, buf, buf, 4, 8, 16, 0, 0, APUS_GHIP_ACT_SILU, 0.0f, stream);
    case 3:
        return apus_ghip_fp8blk_gated_dev((uint8_t *)buf, (float *)buf, (uint8_t *)buf, (float *)buf, buf, buf, 4, 8, 16, 0, 0,
                                          APUS_GHIP_ACT_SILU, 0.0f, 1, stream);
    case 4:
        return apus_ghip_bf16_linear_ep_backward_dev(buf, buf, NULL, buf, buf, buf, buf, 4, 8, 16, 0, 0, 0, APUS_GHIP_ACT_SILU, buf,
                                                     sizeof buf, stream);
    default:
        return apus_ghip_bf16_gated_backward_dev(buf, buf, buf, buf, buf, buf, buf, 4, 8, 16, 0, 0, 0, APUS_GHIP_ACT_SILU, 0.0f, buf,
                                                 sizeof buf, stream);
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
    for (int which = 0; which < 6; which++)
        for (int was = 0; was < 2; was++) {
            current = was;
            expect("null stream", which, call(which, NULL), 0, was, 1);
            expect("own stream", which, call(which, STREAM(1)), 0, was, 1);
            expect("the other device's stream", which, call(which, STREAM(0)), 1, was, 0);
            fail_launch = 1;
            expect("failed launch", which, call(which, NULL), 1, was, 1);
            fail_launch = 0;
        }
    printf(bad ? "FAIL\n" : "PASS\n");
    return bad;
}
