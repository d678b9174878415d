/*
 * k_norm.hip — the root-mean-square norm with the residual's addition, and its
 * gradient (gfx950).
 *
 *   s = bf16(x + r), y = s rstd gamma, rstd = 1 / sqrt(mean(s^2) + eps)
 *   dx = rstd gamma dy - s rstd^3 mean(gamma dy s) + ds
 *   dgamma = sum over the rows of dy s rstd
 *
 * Bound by HBM for many rows, by one chain of load, reduction and store for a
 * few. A row lies in the registers of T threads, V pieces of 8 values each, so
 * that it is read once; a wave adds by DPP, the waves of a row through LDS, in a
 * fixed order. Sums, statistics and the values in between are f32. s is rounded
 * before the norm because it is what the stream holds and what the gradient is
 * given; y is rounded once, to bf16 or, with its block's scale, to MXFP8.
 *
 * The gradient's groups of threads walk the rows a grid apart, so that dgamma's sums
 * stay in registers and 512 workgroups' worth of them goes to memory once; a second
 * launch adds these in order. The next row is loaded while one is summed. Of a few rows
 * whose rstd is given one launch makes both, dgamma from s and dy read again.
 *
 * Measured: 8192 x 4096 with a residual to s and MXFP8 44.1 us (236 MB, 5.4 TB/s); its
 * gradient with ds 53.0 + 4.9 (268 MB and 17: 5.0 TB/s; 71.5 in all with no row loaded
 * ahead); one row of 4096 3.0, a launch's time; 300 x 1536 gradient 3.5.
 */
#include <type_traits>

#include "ghip_mx.h"

typedef unsigned short nm_u16x8 __attribute__((ext_vector_type(8)));

/* The sum over a wave, in every lane: 16 lanes by DPP, the four rows in order. */
__device__ __forceinline__ float nm_wave_sum(float v) {
    auto dpp = [&](auto ctrl) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    dpp(std::integral_constant<int, 0xB1>{});    /* lane ^ 1 */
    dpp(std::integral_constant<int, 0x4E>{});    /* lane ^ 2 */
    dpp(std::integral_constant<int, 0x141>{});   /* mirrored in 8 */
    dpp(std::integral_constant<int, 0x140>{});   /* mirrored in 16 */
    const int i = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16)))
         + (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

/* N sums over the T threads of a row, in every one of them. */
template <int T, int N>
__device__ __forceinline__ void nm_sum(float (&v)[N], float *lds) {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = nm_wave_sum(v[k]);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        const uint32_t wv = threadIdx.x >> 6, base = threadIdx.x / T * W;
        __syncthreads();                         /* the row before has been read */
        if ((threadIdx.x & 63u) == 0u)
#pragma unroll
            for (int k = 0; k < N; k++) lds[k * 16 + wv] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) s += lds[k * 16 + base + w];
            v[k] = s;
        }
    }
}

/* Columns [col, col + 8) of a row, zeros past D; the device takes 16-byte accesses
 * at any alignment of 2. */
__device__ __forceinline__ nm_u16x8 nm_load(const uint16_t *row, uint32_t col, uint32_t D) {
    nm_u16x8 d = {0, 0, 0, 0, 0, 0, 0, 0};
    if (col + 8u <= D) {
        __builtin_memcpy(&d, row + col, 16);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; e++)
            if (col + e < D) d[e] = row[col + e];
    }
    return d;
}
__device__ __forceinline__ void nm_store(uint16_t *row, uint32_t col, uint32_t D, const nm_u16x8 &d) {
    if (col + 8u <= D) {
        __builtin_memcpy(row + col, &d, 16);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; e++)
            if (col + e < D) row[col + e] = d[e];
    }
}
__device__ __forceinline__ nm_u16x8 nm_pack(const float (&v)[8]) {
    nm_u16x8 d;
#pragma unroll
    for (int e = 0; e < 8; e++) d[e] = __builtin_bit_cast(unsigned short, (__bf16)v[e]);
    return d;
}

/* x + r, rounded */
__device__ __forceinline__ nm_u16x8 nm_add(const nm_u16x8 &x, const nm_u16x8 &r) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = ghip_bf16_f32(x[e]) + ghip_bf16_f32(r[e]);
    return nm_pack(v);
}

__device__ __forceinline__ float nm_rstd(float sum, uint32_t D, float eps) {
    return 1.0f / sqrtf(sum / (float)D + eps);
}

/* What a row with this rstd is multiplied by before its squares and products are added: 1,
 * or, of rows below 2^-50 and past 2^50, the power of two that keeps these sums f32
 * numbers. Exact, so the sums are the same where the row's own would have been. */
__device__ __forceinline__ float nm_up(float rstd) {
    const uint32_t low = 77u << 23, high = 177u << 23;   /* 2^-50, 2^50 */
    if (__float_as_uint(rstd) - low <= high - low) return 1.0f;
    return rstd > 1.0f ? 0x1p80f : rstd < 1.0f ? 0x1p-80f : 1.0f;
}

__device__ __forceinline__ void nm_squares(const nm_u16x8 &s, float up, float (&sum)[1]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float v = ghip_bf16_f32(s[e]) * up;
        sum[0] += v * v;
    }
}

/* y's columns [col, col + 8); rstd of the row times up */
__device__ __forceinline__ void nm_out(const GhipNorm &p, size_t row, uint32_t col, const nm_u16x8 &s,
                                       const nm_u16x8 &g, float up, float rstd) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        v[e] = ghip_bf16_f32(s[e]) * up * rstd;
        if (p.gamma) v[e] *= ghip_bf16_f32(g[e]);
    }
    if (p.y) nm_store(p.y + row * p.ldy, col, p.D, nm_pack(v));
    if (p.codes) {                               /* D % 32 == 0: whole quads */
        const uint32_t sc = mx_scale<GHIP_MXFP8>(mx_quad_max(mx_amax8(v)));
        *(ghip_u32x2 *)(p.codes + row * p.D + col) = mx_codes8<GHIP_MXFP8>(v, sc);
        if ((threadIdx.x & 3u) == 0u) {
            const uint32_t ld = (p.D + 127u) / 128u * 4u, b = col >> 5;
            uint8_t *q = p.scales + row * ld;
            q[b] = (uint8_t)sc;
            if (b == p.D / 32u - 1u)
                for (uint32_t j = b + 1u; j < ld; j++) q[j] = 0;
        }
    }
}

template <int T, int V>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rmsnorm(GhipNorm p, size_t row0) {
    __shared__ float lds[16];
    const uint32_t t = threadIdx.x % T;
    const size_t row = row0 + (size_t)blockIdx.x * (T < 256 ? 256 / T : 1) + threadIdx.x / T;
    static_assert(T == 64 || T >= 256, "a row a wave, or a workgroup");
    if (T == 64 && row >= p.M) return;
    nm_u16x8 s[V], g[V];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t col = 8u * (t + T * i);
        if (col < p.D) {
            s[i] = nm_load(p.x + row * p.ldx, col, p.D);
            if (p.r) g[i] = nm_load(p.r + row * p.ldr, col, p.D);
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t col = 8u * (t + T * i);
        if (col < p.D) {
            if (p.r) s[i] = nm_add(s[i], g[i]);
            if (p.gamma) g[i] = nm_load(p.gamma, col, p.D);
            nm_squares(s[i], 1.0f, sum);
        }
    }
    nm_sum<T, 1>(sum, lds);
    float rstd = nm_rstd(sum[0], p.D, p.eps);
    const float up = nm_up(rstd);
    if (up != 1.0f) {                            /* the whole row's threads */
        sum[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (8u * (t + T * i) < p.D) nm_squares(s[i], up, sum);
        nm_sum<T, 1>(sum, lds);
        rstd = nm_rstd(sum[0], p.D, p.eps * up * up);
    }
    if (p.rstd && t == 0u) p.rstd[row] = rstd * up;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t col = 8u * (t + T * i);
        if (col < p.D) {
            if (p.sum) nm_store(p.sum + row * p.lds, col, p.D, s[i]);
            nm_out(p, row, col, s[i], g[i], up, rstd);
        }
    }
}

/* Rows of any length: x (and r) read twice, the second time from the caches. Each
 * thread reads again only what it wrote or nobody did, so sum or y may be x or r. */
__global__ __launch_bounds__(1024) void k_rmsnorm_long(GhipNorm p, size_t row0) {
    __shared__ float lds[16];
    const size_t row = row0 + blockIdx.x;
    const uint16_t *x = p.x + row * p.ldx, *q = p.r ? p.r + row * p.ldr : nullptr;
    float sum[1] = {0.0f};
    auto value = [&](uint32_t col) {
        const nm_u16x8 d = nm_load(x, col, p.D);
        return q ? nm_add(d, nm_load(q, col, p.D)) : d;
    };
    for (uint32_t col = 8u * threadIdx.x; col < p.D; col += 8192u) nm_squares(value(col), 1.0f, sum);
    nm_sum<1024, 1>(sum, lds);
    float rstd = nm_rstd(sum[0], p.D, p.eps);
    const float up = nm_up(rstd);
    if (up != 1.0f) {
        sum[0] = 0.0f;
        for (uint32_t col = 8u * threadIdx.x; col < p.D; col += 8192u) nm_squares(value(col), up, sum);
        nm_sum<1024, 1>(sum, lds);
        rstd = nm_rstd(sum[0], p.D, p.eps * up * up);
    }
    if (p.rstd && threadIdx.x == 0u) p.rstd[row] = rstd * up;
    for (uint32_t col = 8u * threadIdx.x; col < p.D; col += 8192u) {
        const nm_u16x8 d = value(col), g = p.gamma ? nm_load(p.gamma, col, p.D) : d;
        if (p.sum) nm_store(p.sum + row * p.lds, col, p.D, d);
        nm_out(p, row, col, d, g, up, rstd);
    }
}

/* ---- gradient ------------------------------------------------------------ */

/* dx's columns [col, col + 8); a = rstd, c = rstd mean(gamma dy s). s rstd and c are of the size
 * of 1 and of dy whatever the row's is; rstd^3 leaves the f32 range for rows past 2^42. */
__device__ __forceinline__ void nm_dx(const GhipNormGrad &p, size_t row, uint32_t col, const nm_u16x8 &s,
                                      const nm_u16x8 &dy, const nm_u16x8 &g, const nm_u16x8 &ds, float a, float c) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float d = ghip_bf16_f32(dy[e]);
        if (p.gamma) d *= ghip_bf16_f32(g[e]);
        v[e] = a * (d - ghip_bf16_f32(s[e]) * a * c);
    }
    if (p.ds)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += ghip_bf16_f32(ds[e]);
    nm_store(p.dx + row * p.lddx, col, p.D, nm_pack(v));
}

/* Sums of gamma dy s and s^2 over these columns, s times up. */
__device__ __forceinline__ void nm_products(const GhipNormGrad &p, const nm_u16x8 &s, const nm_u16x8 &dy,
                                            const nm_u16x8 &g, float up, float (&sum)[2]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float d = ghip_bf16_f32(dy[e]);
        const float v = ghip_bf16_f32(s[e]) * up;
        if (p.gamma) d *= ghip_bf16_f32(g[e]);
        sum[0] += d * v;
        sum[1] += v * v;
    }
}

/* Each group of T threads walks rows a grid apart; its share of dgamma stays in
 * registers and goes to memory once, part[group][D]. */
template <int T, int V>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rmsnorm_grad(GhipNormGrad p) {
    __shared__ float lds[32];
    constexpr uint32_t PER = T < 256 ? 256 / T : 1;
    const uint32_t t = threadIdx.x % T;
    const size_t group = (size_t)blockIdx.x * PER + threadIdx.x / T, groups = (size_t)gridDim.x * PER;
    nm_u16x8 g[V];
    float acc[V][8] = {};
#pragma unroll
    for (int i = 0; i < V; i++) {
        const uint32_t col = 8u * (t + T * i);
        if (p.gamma && col < p.D) g[i] = nm_load(p.gamma, col, p.D);
    }
    /* Every group of a block makes as many rounds (the barriers of nm_sum); rows past the
     * last are read as it and come to nothing. The next row is on its way while this one
     * is summed (but for the longest rows, which fill the registers) */
    constexpr bool AHEAD = V <= 2;
    constexpr int V1 = AHEAD ? V : 1;
    nm_u16x8 s[V], dy[V], ds[V], s1[V1], dy1[V1], ds1[V1];
    float given = 0.0f, given1 = 0.0f;
    auto load = [&](size_t first, nm_u16x8 (&s)[V], nm_u16x8 (&dy)[V], nm_u16x8 (&ds)[V], float &given) {
        const size_t row = first + threadIdx.x / T, r = row < p.M ? row : p.M - 1;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = 8u * (t + T * i);
            if (col < p.D) {
                s[i] = nm_load(p.s + r * p.lds, col, p.D);
                dy[i] = nm_load(p.dy + r * p.lddy, col, p.D);
                if (p.ds && p.dx) ds[i] = nm_load(p.ds + r * p.ldds, col, p.D);
            }
        }
        if (p.rstd) given = p.rstd[r];
    };
    size_t first = (size_t)blockIdx.x * PER;
    load(first, s, dy, ds, given);
    for (;;) {
        const size_t row = first + threadIdx.x / T, next = first + groups;
        const bool more = next < p.M;
        if constexpr (AHEAD)
            if (more) load(next, s1, dy1, ds1, given1);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
            if (8u * (t + T * i) < p.D) nm_products(p, s[i], dy[i], g[i], 1.0f, sum);
        nm_sum<T, 2>(sum, lds);
        float a = p.rstd ? given : nm_rstd(sum[1], p.D, p.eps);
        float c = a * (sum[0] / (float)p.D);
        const float up = nm_up(a);
        if (up != 1.0f) {                        /* the whole row's threads */
            sum[0] = sum[1] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++)
                if (8u * (t + T * i) < p.D) nm_products(p, s[i], dy[i], g[i], up, sum);
            nm_sum<T, 2>(sum, lds);
            if (!p.rstd) a = nm_rstd(sum[1], p.D, p.eps * up * up) * up;
            c = a / up * (sum[0] / (float)p.D);
        }
        if (row < p.M) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t col = 8u * (t + T * i);
                if (col < p.D) {
                    if (p.dx) nm_dx(p, row, col, s[i], dy[i], g[i], ds[i], a, c);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[i][e] += ghip_bf16_f32(dy[i][e]) * (ghip_bf16_f32(s[i][e]) * a);
                }
            }
        }
        if (!more) break;
        first = next;
        if constexpr (AHEAD) {
            given = given1;
#pragma unroll
            for (int i = 0; i < V; i++) {
                s[i] = s1[i];
                dy[i] = dy1[i];
                ds[i] = ds1[i];
            }
        } else {
            load(first, s, dy, ds, given);
        }
    }
    if (p.part) {
        const size_t ld = (p.D + 7u) & ~7u;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = 8u * (t + T * i);
            if (col < p.D) {
                float *q = p.part + group * ld + col;
                *(ghip_f32x4 *)q = (ghip_f32x4){acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
                *(ghip_f32x4 *)(q + 4) = (ghip_f32x4){acc[i][4], acc[i][5], acc[i][6], acc[i][7]};
            }
        }
    }
}

/* A few rows whose rstd is given, in one launch: row_blocks workgroups take a row (or
 * four) each for dx, the others 32 columns each for dgamma, which read s and dy again.
 * dx may not be dy. */
template <int T, int V>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rmsnorm_grad_few(GhipNormGrad p, uint32_t row_blocks) {
    constexpr uint32_t TH = T < 256 ? 256 : T, PER = TH / T, Q = TH / 4u;
    __shared__ float lds[Q * 33u];
    if (blockIdx.x < row_blocks) {
        const uint32_t t = threadIdx.x % T;
        const size_t row = (size_t)blockIdx.x * PER + threadIdx.x / T;
        if (T == 64 && row >= p.M) return;
        nm_u16x8 s[V], dy[V], g[V], ds[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = 8u * (t + T * i);
            if (col < p.D) {
                s[i] = nm_load(p.s + row * p.lds, col, p.D);
                dy[i] = nm_load(p.dy + row * p.lddy, col, p.D);
                if (p.gamma) g[i] = nm_load(p.gamma, col, p.D);
                if (p.ds) ds[i] = nm_load(p.ds + row * p.ldds, col, p.D);
            }
        }
        const float a = p.rstd[row], up = nm_up(a);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
            if (8u * (t + T * i) < p.D) nm_products(p, s[i], dy[i], g[i], up, sum);
        nm_sum<T, 2>(sum, lds);
        const float c = a / up * (sum[0] / (float)p.D);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t col = 8u * (t + T * i);
            if (col < p.D) nm_dx(p, row, col, s[i], dy[i], g[i], ds[i], a, c);
        }
        return;
    }
    const uint32_t q = threadIdx.x >> 2, c = 8u * (threadIdx.x & 3u), first = (blockIdx.x - row_blocks) * 32u;
    float v[8] = {};
    if (first + c < p.D)
#pragma unroll 4
        for (size_t row = q; row < p.M; row += Q) {
            const nm_u16x8 s = nm_load(p.s + row * p.lds, first + c, p.D), dy = nm_load(p.dy + row * p.lddy, first + c, p.D);
            const float a = p.rstd[row];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += ghip_bf16_f32(dy[e]) * (ghip_bf16_f32(s[e]) * a);
        }
#pragma unroll
    for (int e = 0; e < 8; e++) lds[q * 33u + c + e] = v[e];
    __syncthreads();
    const uint32_t n = threadIdx.x & 31u, h = threadIdx.x >> 5;
    float s = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < 8; k++) s += lds[(8u * h + k) * 33u + n];
    __syncthreads();
    lds[h * 33u + n] = s;
    __syncthreads();
    if (threadIdx.x < 32u && first + n < p.D) {
        s = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < TH / 32u; k++) s += lds[k * 33u + n];
        p.dgamma[first + n] = (uint16_t)ghip_bf16_bits(s);
    }
}

/* Rows of any length, dx or (dx NULL) rstd to part. */
__global__ __launch_bounds__(1024) void k_rmsnorm_grad_long(GhipNormGrad p, size_t row0) {
    __shared__ float lds[32];
    const size_t row = row0 + blockIdx.x;
    const uint16_t *s = p.s + row * p.lds, *dy = p.dy + row * p.lddy;
    float sum[2] = {0.0f, 0.0f};
    auto gamma = [&](uint32_t col) { return p.gamma ? nm_load(p.gamma, col, p.D) : nm_u16x8{}; };
    float up = p.rstd ? nm_up(p.rstd[row]) : 1.0f;
    auto add = [&]() {
        sum[0] = sum[1] = 0.0f;
        for (uint32_t col = 8u * threadIdx.x; col < p.D; col += 8192u)
            nm_products(p, nm_load(s, col, p.D), nm_load(dy, col, p.D), gamma(col), up, sum);
        nm_sum<1024, 2>(sum, lds);
    };
    add();
    if (!p.rstd && (up = nm_up(nm_rstd(sum[1], p.D, p.eps))) != 1.0f) add();
    const float a = p.rstd ? p.rstd[row] : nm_rstd(sum[1], p.D, p.eps * up * up) * up;
    const float c = a / up * (sum[0] / (float)p.D);
    if (!p.dx) {
        if (threadIdx.x == 0u) p.part[row] = a;
        return;
    }
    for (uint32_t col = 8u * threadIdx.x; col < p.D; col += 8192u)
        nm_dx(p, row, col, nm_load(s, col, p.D), nm_load(dy, col, p.D), gamma(col),
              p.ds ? nm_load(p.ds + row * p.ldds, col, p.D) : nm_u16x8{}, a, c);
}

__global__ __launch_bounds__(256) void k_rmsnorm_dgamma_long(GhipNormGrad p) {
    __shared__ float lds[8][256];
    /* 32 pieces of 8 columns, 8 rows at a time */
    const uint32_t c = threadIdx.x & 31u, q = threadIdx.x >> 5, col = 8u * (blockIdx.x * 32u + c);
    float v[8] = {};
    if (col < p.D)
        for (size_t row = q; row < p.M; row += 8u) {
            const nm_u16x8 s = nm_load(p.s + row * p.lds, col, p.D), dy = nm_load(p.dy + row * p.lddy, col, p.D);
            const float a = p.rstd[row];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] += ghip_bf16_f32(dy[e]) * (ghip_bf16_f32(s[e]) * a);
        }
#pragma unroll
    for (int e = 0; e < 8; e++) lds[q][8u * c + e] = v[e];
    __syncthreads();
    const uint32_t n = blockIdx.x * 256u + threadIdx.x;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) s += lds[k][threadIdx.x];
    if (n < p.D) p.dgamma[n] = (uint16_t)ghip_bf16_bits(s);
}

/* dgamma = the groups' sums, added in order: 16 columns a workgroup, 4 a thread in
 * every 64th group, the 64 threads' sums through LDS. */
__global__ __launch_bounds__(256) void k_rmsnorm_dgamma(const float *__restrict__ part, uint32_t groups,
                                                        uint32_t D, uint16_t *__restrict__ dgamma) {
    __shared__ float lds[64][17];
    const uint32_t c = 4u * (threadIdx.x & 3u), q = threadIdx.x >> 2, col = blockIdx.x * 16u + c;
    const size_t ld = (D + 7u) & ~7u;
    ghip_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (col < ld)
#pragma unroll 4
        for (uint32_t k = q; k < groups; k += 64u) v += *(const ghip_f32x4 *)(part + k * ld + col);
#pragma unroll
    for (int e = 0; e < 4; e++) lds[q][c + e] = v[e];
    __syncthreads();
    const uint32_t n = threadIdx.x & 15u, h = threadIdx.x >> 4;
    float s = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) s += lds[4u * h + k][n];
    __syncthreads();
    lds[h][n] = s;
    __syncthreads();
    if (threadIdx.x < 16u && blockIdx.x * 16u + n < D) {
        s = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < 16; k++) s += lds[k][n];
        dgamma[blockIdx.x * 16u + n] = (uint16_t)ghip_bf16_bits(s);
    }
}

/* ---- which form ----------------------------------------------------------- */

/* By the row's length: as few threads a row as hold it in one or two pieces each, for a
 * wave needs no barrier, and more threads than pieces idle at it. Microseconds of 2^26
 * values (a residual, y in BF16; the gradient with dgamma), the next forms beside:
 *   D          norm                                      gradient
 *   512        64x1 91, 64x2 92, 256x1 143               64x2 93, 64x1 94, 256x1 318
 *   1024       64x2 98, 256x1 99, 512x1 149              64x2 93, 256x1 182, 512x1 206
 *   2048       512x1 92, 256x1 94, 1024x1 130            256x1 101, 512x1 111, 256x4 121
 *   (MXFP8     256x1 81, 512x1 94)
 *   4096       512x1 91, 1024x1 94, 256x2 98             512x1 84, 256x4 91, 256x2 93
 *   8192       1024x1 92, 512x2 98, 256x4 102            256x4 86, 1024x1 91, 512x2 110
 *   16384      1024x2 100, 512x4 105, two passes 115     512x4 103, 1024x2 132
 * A single row takes 3.3 us at 8192 by 1024x1, 4.8 by 256x4. */

/* Launches of at most this many blocks (2^32 threads along x are refused). */
#define NM_BLOCKS ((size_t)1 << 21)
#define NM_GRAD_BLOCKS ((size_t)512)

template <int T, int V>
static hipError_t norm_run(const GhipNorm *p, hipStream_t st) {
    constexpr size_t PER = T < 256 ? 256 / T : 1;
    for (size_t r = 0; r < p->M; r += NM_BLOCKS * PER) {
        const size_t left = (p->M - r + PER - 1) / PER;
        hipLaunchKernelGGL((k_rmsnorm<T, V>), dim3((uint32_t)(left < NM_BLOCKS ? left : NM_BLOCKS)),
                           dim3(T < 256 ? 256 : T), 0, st, *p, r);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" hipError_t ghip_launch_rmsnorm(const GhipNorm *p, hipStream_t st) {
    if (p->M == 0 || p->D == 0 || (p->codes && p->D % 32)) return hipErrorInvalidValue;
    if (p->D <= 512) return norm_run<64, 1>(p, st);
    if (p->D <= 1024) return norm_run<64, 2>(p, st);
    if (p->D <= 2048) return norm_run<256, 1>(p, st);
    if (p->D <= 4096) return norm_run<512, 1>(p, st);
    if (p->D <= 8192) return norm_run<1024, 1>(p, st);
    if (p->D <= 16384) return norm_run<1024, 2>(p, st);
    for (size_t r = 0; r < p->M; r += NM_BLOCKS) {
        hipLaunchKernelGGL(k_rmsnorm_long, dim3((uint32_t)(p->M - r < NM_BLOCKS ? p->M - r : NM_BLOCKS)),
                           dim3(1024), 0, st, *p, r);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

/* Blocks that walk the rows: two a CU, or as many as there are rows for. The part
 * has a row for each group of T threads. */
template <int T>
static constexpr size_t grad_per() { return T < 256 ? 256 / T : 1; }
template <int T>
static size_t grad_blocks(size_t M) {
    const size_t n = (M + grad_per<T>() - 1) / grad_per<T>();
    return n < NM_GRAD_BLOCKS ? n : NM_GRAD_BLOCKS;
}

/* Whether one launch that reads s and dy twice is taken: its columns' walk over the rows
 * grows with their number, its second reads with their size. us of M x D, one launch : two
 * (all with ds):
 *   M       1536          4096          8192          16384
 *   1       3.4 :  5.9    3.2 :  5.8    4.0 :  7.5    4.4 :  8.4
 *   300     3.5 :  7.0    3.8 :  9.4    6.5 : 16.1   16.2 : 24.4
 *   512     3.8 :  7.9    4.5 : 12.3   11.0 : 19.3   25.7 : 33.3
 *   1024    6.2 :  9.0   12.2 : 14.8   23.2 : 23.9   46.8 : 44.1
 *   2048   16.0 : 11.7   26.8 : 18.3   44.1 : 33.7   88.8 : 71.2 */
static bool grad_few(const GhipNormGrad *p) {
    return p->dgamma && p->rstd && p->dx != p->dy && p->M <= 1024 && p->M * p->D <= (size_t)1 << 23;
}

template <int T, int V>
static hipError_t grad_run(const GhipNormGrad *p, hipStream_t st) {
    const size_t blocks = grad_blocks<T>(p->M);
    if (grad_few(p)) {
        const uint32_t rows = p->dx ? (uint32_t)((p->M + grad_per<T>() - 1) / grad_per<T>()) : 0u;
        hipLaunchKernelGGL((k_rmsnorm_grad_few<T, V>), dim3(rows + (p->D + 31u) / 32u), dim3(T < 256 ? 256 : T), 0, st,
                           *p, rows);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((k_rmsnorm_grad<T, V>), dim3((uint32_t)blocks), dim3(T < 256 ? 256 : T), 0, st, *p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p->dgamma) return e;
    hipLaunchKernelGGL(k_rmsnorm_dgamma, dim3((p->D + 15u) / 16u), dim3(256), 0, st, p->part,
                       (uint32_t)(blocks * grad_per<T>()), p->D, p->dgamma);
    return hipGetLastError();
}

/* f(T, V) of the form for D columns; false for rows of any length. */
template <typename F>
static bool grad_form(size_t D, F f) {
    using std::integral_constant;
    if (D <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (D <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (D <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (D <= 4096) f(integral_constant<int, 512>{}, integral_constant<int, 1>{});
    else if (D <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else if (D <= 16384) f(integral_constant<int, 512>{}, integral_constant<int, 4>{});
    else return false;
    return true;
}

extern "C" size_t ghip_rmsnorm_part_bytes(size_t M, size_t D) {
    size_t n = M * 4;
    grad_form(D, [&](auto t, auto) {
        constexpr int T = decltype(t)::value;
        n = grad_blocks<T>(M) * grad_per<T>() * ((D + 7) & ~(size_t)7) * 4;
    });
    return n;
}

extern "C" hipError_t ghip_launch_rmsnorm_grad(const GhipNormGrad *p, hipStream_t st) {
    if (p->M == 0 || p->D == 0 || (p->dgamma && !p->part)) return hipErrorInvalidValue;
    hipError_t e = hipSuccess;
    if (grad_form(p->D, [&](auto t, auto v) { e = grad_run<decltype(t)::value, decltype(v)::value>(p, st); }))
        return e;
    /* rstd, dgamma, dx: dx may be dy */
    GhipNormGrad q = *p;
    auto rows = [&]() {
        for (size_t r = 0; r < q.M; r += NM_BLOCKS) {
            hipLaunchKernelGGL(k_rmsnorm_grad_long, dim3((uint32_t)(q.M - r < NM_BLOCKS ? q.M - r : NM_BLOCKS)),
                               dim3(1024), 0, st, q, r);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    };
    if (p->dgamma) {
        if (!p->rstd) {
            q.dx = nullptr;
            if ((e = rows()) != hipSuccess) return e;
            q.rstd = p->part;
        }
        hipLaunchKernelGGL(k_rmsnorm_dgamma_long, dim3((p->D + 255u) / 256u), dim3(256), 0, st, q);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    q.dx = p->dx;
    return p->dx ? rows() : hipSuccess;
}
