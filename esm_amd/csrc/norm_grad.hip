// LayerNorm for training: the forward pass that leaves its row statistics, and the backward pass with the reduction of
// the weight's and the bias's gradients.
//
//   h = (x - mean) rstd,  y = h gamma + beta
//   g = dy gamma,  dx = rstd (g - mean_d(g) - h mean_d(g h)),  dgamma = sum_rows dy h,  dbeta = sum_rows dy
//
// Both are bound by HBM: the forward pass has to move 2 M d elements, the backward pass 3 M d.  WPR waves share a row
// and keep all of it in registers (one read), sums run in fp32, and the next row's loads are in flight while the current
// one is reduced.  A lane owns the same columns of every row it meets, so it sums its columns of dgamma / dbeta in
// registers; each workgroup leaves one partial row, and a second kernel adds the partial rows in a fixed order (no
// atomics: the same inputs give the same bits).
#include <type_traits>

#include "common.hpp"

namespace {

constexpr int NG_MAX_D = 12288;      // 8 waves x 64 lanes x 24 elements
constexpr int NG_MAX_GROUPS = 512;   // partial rows of dgamma / dbeta

template <typename T> struct NgVec;  // 16 bytes of T
template <> struct NgVec<float> { static constexpr int N = 4; };
template <> struct NgVec<__bf16> { static constexpr int N = 8; };

// VEC elements of a row: one 16-byte load, or one element where width, stride or address rule that out
template <typename T, int VEC> struct NgRaw { u32x4 v; };
template <> struct NgRaw<float, 1> { float v; };
template <> struct NgRaw<__bf16, 1> { unsigned short v; };

template <typename T, int VEC>
__device__ __forceinline__ NgRaw<T, VEC> ng_load(const T* p) {
    NgRaw<T, VEC> r;
    r.v = *(const decltype(r.v)*)p;
    return r;
}
__device__ __forceinline__ void ng_unpack(const NgRaw<float, 4>& r, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(r.v[e]);
}
__device__ __forceinline__ void ng_unpack(const NgRaw<__bf16, 8>& r, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(r.v[e] << 16);
        f[2 * e + 1] = __uint_as_float(r.v[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ void ng_unpack(const NgRaw<float, 1>& r, float* f) { f[0] = r.v; }
__device__ __forceinline__ void ng_unpack(const NgRaw<__bf16, 1>& r, float* f) { f[0] = bf16_bits_to_f32(r.v); }
__device__ __forceinline__ void ng_store(float* p, const float (&f)[4]) { *(f32x4*)p = f32x4{f[0], f[1], f[2], f[3]}; }
__device__ __forceinline__ void ng_store(__bf16* p, const float (&f)[8]) {
    *(u32x4*)p = u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}
__device__ __forceinline__ void ng_store(float* p, const float (&f)[1]) { *p = f[0]; }
__device__ __forceinline__ void ng_store(__bf16* p, const float (&f)[1]) { *p = (__bf16)f[0]; }

// Threads of a workgroup: four waves, eight where eight waves share a row.
constexpr int ng_threads(int wpr) { return wpr == 8 ? 512 : 256; }

// Sum of (a, b) over the WPR waves of a row.  `buf` holds one pair per wave and alternates between two halves, so that
// one barrier per call is enough: a wave reaches the call after next only behind the barrier that every reader of the
// earlier half has passed.  All waves of the workgroup call it equally often.
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf, int& half) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (WPR > 1) {
        const int wave = threadIdx.x >> 6;
        float* p = buf + half * 16;
        if ((threadIdx.x & 63) == 0) { p[2 * wave] = a; p[2 * wave + 1] = b; }
        __syncthreads();
        const int w0 = wave / WPR * WPR;
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) { a += p[2 * (w0 + w)]; b += p[2 * (w0 + w) + 1]; }
        half ^= 1;
    }
}

template <typename T, int VEC, int NV, int WPR>
__global__ __launch_bounds__(ng_threads(WPR)) void norm_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ beta, T* __restrict__ y,
                                                                   float* __restrict__ stats, int M, int d, float eps) {
    constexpr int ROWS = ng_threads(WPR) / 64 / WPR;  // rows a workgroup works on at once
    __shared__ float buf[32];
    const int lane = threadIdx.x & (64 * WPR - 1), slot = threadIdx.x / (64 * WPR);
    const int nvec = d / VEC;
    const int stride = gridDim.x * ROWS;
    int half = 0;
    NgRaw<T, VEC> raw[NV];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + i * 64 * WPR < nvec) raw[i] = ng_load<T, VEC>(x + (int64_t)r * ldx + lane * VEC + i * 64 * WPR * VEC);
    };
    int first = blockIdx.x * ROWS;  // uniform over the workgroup: every wave makes the same number of turns
    if (first + slot < M) load(first + slot);
    for (; first < M; first += stride) {
        const int row = first + slot;
        const bool on = row < M;
        float v[NV][VEC], sum = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (on && lane + i * 64 * WPR < nvec) ng_unpack(raw[i], v[i]);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += v[i][e];
        }
        if (row + stride < M) load(row + stride);
        row_sum2<WPR>(sum, none, buf, half);
        const float mean = sum / (float)d;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + i * 64 * WPR < nvec)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    v[i][e] -= mean;
                    sq += v[i][e] * v[i][e];
                }
        row_sum2<WPR>(sq, none, buf, half);
        const float rstd = 1.0f / sqrtf(sq / (float)d + eps);
        if (!on) continue;
        if (lane == 0) *(f32x2*)(stats + 2 * (int64_t)row) = f32x2{mean, rstd};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane + i * 64 * WPR;
            if (c >= nvec) continue;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float b = beta ? beta[c * VEC + e] : 0.f;
                o[e] = v[i][e] * rstd * gamma[c * VEC + e] + b;
            }
            ng_store(y + (int64_t)row * d + lane * VEC + i * 64 * WPR * VEC, o);
        }
    }
}

template <typename T, int VEC, int NV, int WPR>
__global__ __launch_bounds__(ng_threads(WPR)) void norm_bwd_kernel(const T* __restrict__ dy, int64_t lddy,
                                                                   const T* __restrict__ x, int64_t ldx,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ stats, T* __restrict__ dx,
                                                                   float* __restrict__ pg, float* __restrict__ pb, int M,
                                                                   int d) {
    constexpr int ROWS = ng_threads(WPR) / 64 / WPR;
    __shared__ float buf[32];
    extern __shared__ float part[];  // [ROWS - 1][2][d]
    const int lane = threadIdx.x & (64 * WPR - 1), slot = threadIdx.x / (64 * WPR);
    const int nvec = d / VEC;
    const int stride = gridDim.x * ROWS;
    const float inv_d = 1.0f / (float)d;
    int half = 0;
    NgRaw<T, VEC> rx[NV], rg[NV];
    float mean = 0.f, rstd = 0.f;
    auto load = [&](int r) {
        const f32x2 st = *(const f32x2*)(stats + 2 * (int64_t)r);
        mean = st[0];
        rstd = st[1];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (lane + i * 64 * WPR < nvec) {
                rx[i] = ng_load<T, VEC>(x + (int64_t)r * ldx + lane * VEC + i * 64 * WPR * VEC);
                rg[i] = ng_load<T, VEC>(dy + (int64_t)r * lddy + lane * VEC + i * 64 * WPR * VEC);
            }
        }
    };
    float w[NV][VEC], ag[NV][VEC], ab[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = lane + i * 64 * WPR;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            ag[i][e] = ab[i][e] = 0.f;
            w[i][e] = c < nvec ? gamma[c * VEC + e] : 0.f;
        }
    }
    int first = blockIdx.x * ROWS;
    if (first + slot < M) load(first + slot);
    for (; first < M; first += stride) {
        const int row = first + slot;
        const bool on = row < M;
        float h[NV][VEC], g[NV][VEC], c1 = 0.f, c2 = 0.f;
        const float rs = rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (on && lane + i * 64 * WPR < nvec) {
                ng_unpack(rx[i], h[i]);
                ng_unpack(rg[i], g[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i][e] = (h[i][e] - mean) * rs;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) h[i][e] = g[i][e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                ag[i][e] += g[i][e] * h[i][e];
                ab[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                c1 += g[i][e];
                c2 += g[i][e] * h[i][e];
            }
        }
        if (row + stride < M) load(row + stride);
        row_sum2<WPR>(c1, c2, buf, half);
        if (!on) continue;
        c1 *= inv_d;
        c2 *= inv_d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane + i * 64 * WPR;
            if (c >= nvec) continue;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = (g[i][e] - c1 - h[i][e] * c2) * rs;
            ng_store(dx + (int64_t)row * d + lane * VEC + i * 64 * WPR * VEC, o);
        }
    }
    if (!pg && !pb) return;
    // the workgroup's row slots, added in order
    if (slot > 0) {
        float* p = part + (int64_t)(slot - 1) * 2 * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane + i * 64 * WPR;
            if (c < nvec)
#pragma unroll
                for (int e = 0; e < VEC; ++e) { p[c * VEC + e] = ag[i][e]; p[d + c * VEC + e] = ab[i][e]; }
        }
    }
    __syncthreads();
    if (slot == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane + i * 64 * WPR;
            if (c < nvec)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float a = ag[i][e], b = ab[i][e];
                    for (int s = 0; s < ROWS - 1; ++s) {
                        a += part[(int64_t)s * 2 * d + c * VEC + e];
                        b += part[(int64_t)s * 2 * d + d + c * VEC + e];
                    }
                    if (pg) pg[(int64_t)blockIdx.x * d + c * VEC + e] = a;
                    if (pb) pb[(int64_t)blockIdx.x * d + c * VEC + e] = b;
                }
        }
    }
}

// Column sums of the G partial rows: 32 columns x 32 groups of rows per workgroup, then the groups in order.
__global__ __launch_bounds__(1024) void norm_grad_reduce_kernel(const float* __restrict__ pg, const float* __restrict__ pb,
                                                                float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                int G, int d) {
    __shared__ float part[32][33];
    const float* src = blockIdx.y ? pb : pg;
    float* dst = blockIdx.y ? dbeta : dgamma;
    if (!dst) return;  // uniform
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    float a = 0.f;
    if (c < d)
        for (int r = grp; r < G; r += 32) a += src[(int64_t)r * d + c];
    part[grp][col] = a;
    __syncthreads();
    if (grp == 0 && c < d) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) a += part[i][col];
        dst[c] = a;
    }
}

__global__ void norm_grad_zero_kernel(float* a, float* b, int d) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < d) {
        if (a) a[i] = 0.f;
        if (b) b[i] = 0.f;
    }
}

// Waves per row: as few as keep a lane at 24 elements or less (the backward pass holds about six fp32 values of each).
int ng_waves(int d) { return d <= 1536 ? 1 : d <= 2 * 1536 ? 2 : d <= 4 * 1536 ? 4 : 8; }
int ng_rows(int wpr) { return wpr == 8 ? 1 : 4 / wpr; }
// Workgroups of the backward pass: two per CU hold enough loads in flight, and more of them only add partial rows; at
// small M a row slot sees at least four rows.
int ng_groups(int M, int d) {
    const int rows = ng_rows(ng_waves(d));
    const int want = (M + 4 * rows - 1) / (4 * rows);
    return want < NG_MAX_GROUPS ? want : NG_MAX_GROUPS;
}

// f(constant<VEC>, constant<NV>, constant<WPR>) for a row of d elements
template <typename T, int VEC, typename F>
bool ng_dispatch(int d, F f) {
    const int wpr = ng_waves(d);
    const int e = (d + 64 * wpr - 1) / (64 * wpr);
#define NG_TRY(E, W) \
    if (wpr == W && e <= E) return f(std::integral_constant<int, VEC>{}, std::integral_constant<int, (E) / VEC>{}, std::integral_constant<int, W>{})
    NG_TRY(8, 1);
    NG_TRY(16, 1);
    NG_TRY(24, 1);
    NG_TRY(16, 2);
    NG_TRY(24, 2);
    NG_TRY(16, 4);
    NG_TRY(24, 4);
    NG_TRY(16, 8);
    NG_TRY(24, 8);
#undef NG_TRY
    return false;
}

bool ng_wide(const void* p, int64_t ld, int size) { return ((uintptr_t)p & 15) == 0 && (ld * size) % 16 == 0; }

template <typename T>
int norm_fwd(const T* x, int64_t ldx, const float* gamma, const float* beta, T* y, float* stats, int M, int d, float eps,
             hipStream_t s) {
    auto go = [&](auto vec, auto nv, auto wpr) {
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value, W = decltype(wpr)::value;
        const int rows = ng_rows(W), want = (M + rows - 1) / rows;
        hipLaunchKernelGGL((norm_fwd_kernel<T, V, N, W>), dim3(want < 2048 ? want : 2048), dim3(ng_threads(W)), 0, s, x, ldx,
                           gamma, beta, y, stats, M, d, eps);
        return true;
    };
    const bool wide = ng_wide(x, ldx, sizeof(T)) && ng_wide(y, d, sizeof(T));
    if (!(wide ? ng_dispatch<T, NgVec<T>::N>(d, go) : ng_dispatch<T, 1>(d, go)))
        ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_fwd: d=%d", d);
    ESMK_CHECK_LAUNCH("esmk_layernorm_fwd");
    return ESMK_OK;
}

template <typename T>
int norm_bwd(const T* dy, int64_t lddy, const T* x, int64_t ldx, const float* gamma, const float* stats, T* dx,
             float* dgamma, float* dbeta, float* ws, int M, int d, hipStream_t s) {
    const int G = ng_groups(M, d);
    // one workgroup: its partial row is the result
    float* pg = dgamma ? (G == 1 ? dgamma : ws) : nullptr;
    float* pb = dbeta ? (G == 1 ? dbeta : ws + (int64_t)G * d) : nullptr;
    auto go = [&](auto vec, auto nv, auto wpr) {
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value, W = decltype(wpr)::value;
        const int lds = (ng_rows(W) - 1) * 2 * d * (int)sizeof(float);  // at most 3 x 2 x 1536 x 4 = 36 KiB
        hipLaunchKernelGGL((norm_bwd_kernel<T, V, N, W>), dim3(G), dim3(ng_threads(W)), lds, s, dy, lddy, x, ldx, gamma, stats,
                           dx, pg, pb, M, d);
        return true;
    };
    const bool wide = ng_wide(x, ldx, sizeof(T)) && ng_wide(dy, lddy, sizeof(T)) && ng_wide(dx, d, sizeof(T));
    if (!(wide ? ng_dispatch<T, NgVec<T>::N>(d, go) : ng_dispatch<T, 1>(d, go)))
        ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_bwd: d=%d", d);
    if (G > 1 && (dgamma || dbeta))
        hipLaunchKernelGGL(norm_grad_reduce_kernel, dim3((d + 31) / 32, 2), dim3(1024), 0, s, pg, pb, dgamma, dbeta, G, d);
    ESMK_CHECK_LAUNCH("esmk_layernorm_bwd");
    return ESMK_OK;
}

}  // namespace

extern "C" int esmk_layernorm_fwd(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, void* y,
                                  float* stats, int M, int d, float eps, esmk_stream_t stream) {
    if (M < 0 || d <= 0 || d > NG_MAX_D) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_fwd: M=%d, d=%d (1..%d)", M, d, NG_MAX_D);
    if (dtype != ESMK_F32 && dtype != ESMK_BF16) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: bad dtype %d", dtype);
    if (M == 0) return ESMK_OK;
    if (!x || !gamma || !y || !stats) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: null pointer");
    if (ldx < d) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: row stride %lld below d=%d", (long long)ldx, d);
    if ((uintptr_t)stats & 7) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: stats must be 8-byte aligned");
    if (dtype == ESMK_F32) return norm_fwd<float>((const float*)x, ldx, gamma, beta, (float*)y, stats, M, d, eps, (hipStream_t)stream);
    return norm_fwd<__bf16>((const __bf16*)x, ldx, gamma, beta, (__bf16*)y, stats, M, d, eps, (hipStream_t)stream);
}

extern "C" size_t esmk_layernorm_bwd_workspace_bytes(int M, int d) {
    if (M <= 0 || d <= 0 || d > NG_MAX_D) return 0;
    const int G = ng_groups(M, d);
    return G == 1 ? 0 : (size_t)G * 2 * d * sizeof(float);
}

extern "C" int esmk_layernorm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int dtype, const float* gamma,
                                  const float* stats, void* dx, float* dgamma, float* dbeta, void* workspace,
                                  size_t workspace_bytes, int M, int d, esmk_stream_t stream) {
    if (M < 0 || d <= 0 || d > NG_MAX_D) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_bwd: M=%d, d=%d (1..%d)", M, d, NG_MAX_D);
    if (dtype != ESMK_F32 && dtype != ESMK_BF16) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: bad dtype %d", dtype);
    if (M == 0) {  // no rows: the parameters' gradients are zero
        if (dgamma || dbeta)
            hipLaunchKernelGGL(norm_grad_zero_kernel, dim3((d + 255) / 256), dim3(256), 0, (hipStream_t)stream, dgamma, dbeta, d);
        ESMK_CHECK_LAUNCH("esmk_layernorm_bwd");
        return ESMK_OK;
    }
    if (!dy || !x || !gamma || !stats || !dx) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: null pointer");
    if (ldx < d || lddy < d) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: row stride below d=%d", d);
    if ((uintptr_t)stats & 7) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: stats must be 8-byte aligned");
    if ((dgamma || dbeta) && esmk_layernorm_bwd_workspace_bytes(M, d) > (workspace ? workspace_bytes : 0))
        ESMK_FAIL(ESMK_ERR_WORKSPACE, "esmk_layernorm_bwd: needs %zu workspace bytes", esmk_layernorm_bwd_workspace_bytes(M, d));
    if (dtype == ESMK_F32)
        return norm_bwd<float>((const float*)dy, lddy, (const float*)x, ldx, gamma, stats, (float*)dx, dgamma, dbeta,
                               (float*)workspace, M, d, (hipStream_t)stream);
    return norm_bwd<__bf16>((const __bf16*)dy, lddy, (const __bf16*)x, ldx, gamma, stats, (__bf16*)dx, dgamma, dbeta,
                            (float*)workspace, M, d, (hipStream_t)stream);
}
