// Preference loss of packed sequence pairs (paired log ratios against a frozen model), forward and backward.
//
//   l_s = sum of log softmax(z_t)[y_t] over the scored tokens of sequence s
//   m_i = beta ((l_2i - ref_2i) - (l_2i+1 - ref_2i+1))
//   L   = mean_i [(1 - eps) softplus(-m_i) + eps softplus(m_i) - alpha l_2i / max(1, scored_2i)]
//   dL/dz_t = c_t (onehot(y_t) - softmax z_t),  c_t = dL/dl of its sequence, 0 where the token is not scored
//
// A token's softmax needs its row of logits alone, a row's gradient needs both sequences of its pair: so one pass over the
// logits leaves (max, sum of exponentials, target's logit) of every token, a workgroup per pair forms the log-probabilities and
// adds them (in 64 bits: a margin is a small difference of two long sums) and leaves c_t, and the backward pass reads the logits
// once more and writes the gradient.  Sums run in a fixed order.  The first and the last pass are bound by memory (10 ragged pairs over
// 4096 bf16 entries: 20 us, 5.0 TB/s, and 31 us, 6.3 TB/s with the logits partly in the cache), the pairs by a few dependent
// reads and their logarithms (5 to 7 us).
#include <type_traits>

#include "common.hpp"

namespace {

// token state: max, sum of exp(z - max), the target's logit, c_t (until the pair is known: 1 if the token is scored, else 0).
// Its log-probability is formed from them in 64 bits (pref_pair_kernel()): one of -5 is off by 2^-22 in 32, and a margin adds up a
// thousand of those.
typedef f32x4 TokState;

template <typename T> struct PlT;
template <> struct PlT<float> { static constexpr int N = 4; };
template <> struct PlT<__bf16> { static constexpr int N = 8; };

__device__ __forceinline__ float pl_get(const float* p) { return *p; }
__device__ __forceinline__ float pl_get(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void pl_unpack(const float* p, float (&f)[4]) {
    const f32x4 v = *(const f32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = v[e];
}
__device__ __forceinline__ void pl_unpack(const __bf16* p, float (&f)[8]) {
    const u32x4 v = *(const u32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(v[e] << 16);
        f[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ void pl_store(float* p, const float (&f)[4]) { *(f32x4*)p = f32x4{f[0], f[1], f[2], f[3]}; }
__device__ __forceinline__ void pl_store(__bf16* p, const float (&f)[8]) {
    *(u32x4*)p = u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
}

constexpr float PL_LOG2E = 1.4426950408889634f, PL_LN2 = 0.6931471805599453f;
constexpr float PL_LOG2E_LOW = 1.9259629911e-8f;  // log2(e) - fp32(log2(e))

// exp(x) for x <= 0 with the product x log2(e) carried in two parts: exp2 alone would lose |x| 2^-24 of the result
__device__ __forceinline__ float pl_exp(float x) {
    const float h = x * PL_LOG2E;
    const float l = fmaf(x, PL_LOG2E, -h) + x * PL_LOG2E_LOW;
    const float r = __builtin_amdgcn_exp2f(h);
    return h < -3e38f ? 0.f : fmaf(r * PL_LN2, l, r);  // x = -inf makes l NaN; a NaN x stays one
}
// exp(x) as a term of a long sum: x log2(e) rounded once, which is off to either side.  The product with fp32(log2(e)) is off to one
// side, by 7e-8 of the sum at x = -5, and a margin adds up a thousand tokens' of it: gradients of 10 ragged pairs over 4096 fp32
// entries off by 1.7e-6, and by 1e-7 so (forward pass of the bf16 ones 21.9 and 23.4 us; with both parts of pl_exp() 27.6).
__device__ __forceinline__ float pl_exp_term(float x) { return __builtin_amdgcn_exp2f(fmaf(x, PL_LOG2E, x * PL_LOG2E_LOW)); }

// Rows start at any element: a row is covered by 16-byte pieces of memory; the first and the last may hold elements of
// the neighbouring rows, and are read and written element by element.
template <typename T>
struct Row {
    const T* base;  // 16-byte aligned, at or below the row's first element
    int lead, n_pieces, V;
    __device__ __forceinline__ Row(const T* z, int64_t row, int V_) : V(V_) {
        const T* p = z + row * V_;
        lead = (int)(((uintptr_t)p & 15) / sizeof(T));
        base = p - lead;
        n_pieces = (lead + V_ + PlT<T>::N - 1) / PlT<T>::N;
    }
    __device__ __forceinline__ int col(int piece) const { return piece * PlT<T>::N - lead; }
    __device__ __forceinline__ bool whole(int c) const { return c >= 0 && c + PlT<T>::N <= V; }
    __device__ __forceinline__ void load(int piece, float (&f)[PlT<T>::N], float fill) const {
        const int c = col(piece);
        if (whole(c)) {
            pl_unpack(base + (int64_t)piece * PlT<T>::N, f);
        } else {
#pragma unroll
            for (int e = 0; e < PlT<T>::N; ++e)
                f[e] = c + e >= 0 && c + e < V ? pl_get(base + (int64_t)piece * PlT<T>::N + e) : fill;
        }
    }
};

template <int CTRL>
__device__ __forceinline__ float pl_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
    if constexpr (LPR == 64) {
        v = fmaxf(v, __shfl_xor(v, 32));
        v = fmaxf(v, __shfl_xor(v, 16));
    }
    // within 16 lanes on the vector ALU: lane ^ 1, lane ^ 2, mirrored in 8, mirrored in 16
    v = fmaxf(v, pl_dpp<0xB1>(v));
    v = fmaxf(v, pl_dpp<0x4E>(v));
    v = fmaxf(v, pl_dpp<0x141>(v));
    return fmaxf(v, pl_dpp<0x140>(v));
}
template <int LPR>
__device__ __forceinline__ float row_add(float v) {
    if constexpr (LPR == 64) {
        v += __shfl_xor(v, 32);
        v += __shfl_xor(v, 16);
    }
    v += pl_dpp<0xB1>(v);
    v += pl_dpp<0x4E>(v);
    v += pl_dpp<0x141>(v);
    return v + pl_dpp<0x140>(v);
}

// LPR lanes per row
template <typename T, int LPR>
__global__ __launch_bounds__(256) void pref_token_kernel(const T* __restrict__ z, const int64_t* __restrict__ targets,
                                                         const int* __restrict__ cu, int n_seq, TokState* __restrict__ tok,
                                                         unsigned* __restrict__ done, int N, int V) {
    constexpr int E = PlT<T>::N, CH = 4;  // pieces in flight per lane
    if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;  // for the pair kernel behind this one
    const int sub = threadIdx.x & (LPR - 1);
    const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (row >= N) return;
    const int64_t y = targets[row];
    if (y < 0 || y >= V || row < cu[0] || row >= cu[n_seq]) {  // not scored: its logits are not looked at
        if (sub == 0) tok[row] = TokState{0.f, 0.f, 0.f, 0.f};
        return;
    }
    const Row<T> r(z, row, V);
    float m = -INFINITY, l = 0.f;
    for (int p0 = sub; p0 < r.n_pieces; p0 += LPR * CH) {
        float f[CH][E];
        float t = m;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (p0 + i * LPR < r.n_pieces) r.load(p0 + i * LPR, f[i], -INFINITY);
            else
#pragma unroll
                for (int e = 0; e < E; ++e) f[i][e] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) t = fmaxf(t, f[i][e]);
        const float base = t == -INFINITY ? 0.f : t;  // only -inf so far: exp(-inf) = 0, and not exp(-inf + inf)
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) s += pl_exp_term(f[i][e] - base);
        l = fmaf(l, pl_exp(m - base), s);
        m = t;
    }
    const float top = row_max<LPR>(m);
    l = row_add<LPR>(l * (m == -INFINITY ? 0.f : pl_exp(m - top)));
    // no finite logit: log 0, and the row's loss is not finite, as the formula has it
    if (sub == 0) tok[row] = TokState{top, l, pl_get(z + row * V + y), 1.f};
}

// One workgroup per pair: a few dependent reads long, so a thread requests up to four tokens of both sequences at once.
constexpr int PL_PAIR = 512;
__global__ __launch_bounds__(PL_PAIR) void pref_pair_kernel(TokState* __restrict__ tok, const int* __restrict__ cu,
                                                            const float* __restrict__ ref, int N, int P, double beta,
                                                            double eps, double alpha, float* __restrict__ logps,
                                                            double* __restrict__ pair_loss, unsigned* __restrict__ done,
                                                            float* __restrict__ loss) {
    constexpr int WAVES = PL_PAIR / 64, AHEAD = 4;
    __shared__ double red[2][WAVES];
    __shared__ int cnt[WAVES];
    __shared__ bool last;
    const int i = blockIdx.x, wave = threadIdx.x >> 6;
    const int at[3] = {min(max(cu[2 * i], 0), N), min(max(cu[2 * i + 1], 0), N), min(max(cu[2 * i + 2], 0), N)};
    const f32x2 r = {ref[2 * i], ref[2 * i + 1]};
    double a[2] = {0.0, 0.0};
    int n = 0;
    for (int t0 = threadIdx.x; at[0] + t0 < at[1] || at[1] + t0 < at[2]; t0 += PL_PAIR * AHEAD) {
        f32x4 v[2][AHEAD];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int t = at[s] + t0 + j * PL_PAIR;
                v[s][j] = t < at[s + 1] ? tok[t] : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (v[s][j][3] == 0.f) continue;  // not scored
                a[s] += ((double)v[s][j][2] - (double)v[s][j][0]) - log((double)v[s][j][1]);
                if (s == 0) ++n;
            }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a[0] += __shfl_xor(a[0], o);
        a[1] += __shfl_xor(a[1], o);
        n += __shfl_xor(n, o);
    }
    if ((threadIdx.x & 63) == 0) {
        red[0][wave] = a[0];
        red[1][wave] = a[1];
        cnt[wave] = n;
    }
    __syncthreads();
    double l[2] = {0.0, 0.0};
    int scored = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        l[0] += red[0][w];
        l[1] += red[1][w];
        scored += cnt[w];
    }
    scored = max(1, scored);
    const double m = beta * ((l[0] - (double)r[0]) - (l[1] - (double)r[1]));
    const double t = exp(-fabs(m)), q = 1.0 / (1.0 + t), up = m >= 0.0 ? q : t * q, down = m >= 0.0 ? t * q : q;
    const double gm = beta * (eps * up - (1.0 - eps) * down) / P;
    const float c[2] = {(float)(gm - alpha / scored / P), (float)-gm};
#pragma unroll
    for (int s = 0; s < 2; ++s)
        for (int k = at[s] + (int)threadIdx.x; k < at[s + 1]; k += PL_PAIR)
            if (tok[k][3] != 0.f) tok[k][3] = c[s];
    if (threadIdx.x == 0) {
        const double lg = log1p(t), sp = fmax(m, 0.0) + lg, sn = fmax(-m, 0.0) + lg;
        // a term whose weight is zero is left out: 0 x inf would be NaN
        double L = eps != 1.0 ? (1.0 - eps) * sn : 0.0;
        if (eps != 0.0) L += eps * sp;
        if (alpha != 0.0) L -= alpha * l[0] / scored;
        logps[2 * i] = (float)l[0];
        logps[2 * i + 1] = (float)l[1];
        // The workgroup that finishes last adds the pairs' losses, in their order: its counter says that all are written.
        __hip_atomic_store(pair_loss + i, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)P - 1u;
    }
    __syncthreads();
    if (!last) return;
    double sum = 0.0;
    for (int k = threadIdx.x; k < P; k += PL_PAIR) sum += __hip_atomic_load(pair_loss + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[0][wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += red[0][w];
        *loss = (float)(sum / P);
    }
}

template <typename T, int LPR>
__global__ __launch_bounds__(256) void pref_grad_kernel(const T* __restrict__ z, const int64_t* __restrict__ targets,
                                                        const TokState* __restrict__ tok, const float* __restrict__ grad,
                                                        T* __restrict__ dz, int N, int V) {
    constexpr int E = PlT<T>::N;
    const int sub = threadIdx.x & (LPR - 1);
    const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    if (row >= N) return;
    const TokState st = tok[row];
    const int64_t y = targets[row];
    const bool on = st[3] != 0.f;  // 0: not scored, or behind the last sequence
    const float c = on ? (grad ? st[3] * *grad : st[3]) : 0.f, minus = -c / st[1];
    const Row<T> r(z, row, V);
    T* out = dz + row * V - r.lead;
    for (int p = sub; p < r.n_pieces; p += LPR) {
        float f[E], o[E];
        const int col = r.col(p);
        if (on) {
            r.load(p, f, 0.f);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(pl_exp(f[e] - st[0]), minus, col + e == (int)y ? c : 0.f);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = 0.f;
        }
        T* q = out + (int64_t)p * E;
        if (r.whole(col)) {
            pl_store(q, o);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (col + e >= 0 && col + e < V) q[e] = (T)o[e];
        }
    }
}

// 16 lanes per row up to 256 entries (the 64-entry vocabulary is one 16-byte piece per lane), a wave above.
template <typename F>
void pl_dispatch(int V, F f) {
    if (V <= 256) f(std::integral_constant<int, 16>{});
    else f(std::integral_constant<int, 64>{});
}

template <typename T>
void pl_token(const void* z, const int64_t* y, const int* cu, int n_seq, TokState* tok, unsigned* done, int N, int V, hipStream_t s) {
    pl_dispatch(V, [&](auto lpr) {
        constexpr int LPR = decltype(lpr)::value;
        hipLaunchKernelGGL((pref_token_kernel<T, LPR>), dim3(N ? (N + 256 / LPR - 1) / (256 / LPR) : 1), dim3(256), 0, s, (const T*)z, y, cu, n_seq, tok, done, N, V);
    });
}
template <typename T>
void pl_grad(const void* z, const int64_t* y, const TokState* tok, const float* g, void* dz, int N, int V, hipStream_t s) {
    pl_dispatch(V, [&](auto lpr) {
        constexpr int LPR = decltype(lpr)::value;
        hipLaunchKernelGGL((pref_grad_kernel<T, LPR>), dim3((N + 256 / LPR - 1) / (256 / LPR)), dim3(256), 0, s, (const T*)z, y, tok, g, (T*)dz, N, V);
    });
}

int pl_check(const char* who, const void* z, int dtype, const void* targets, const void* saved, int N, int V) {
    if (N < 0 || V <= 0 || V > (1 << 30)) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: N=%d, V=%d", who, N, V);
    if (dtype != ESMK_F32 && dtype != ESMK_BF16) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: bad dtype %d", who, dtype);
    if (N >= (1 << 26)) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "%s: N=%d (at most 2^26 - 1 tokens)", who, N);  // 2^32 threads, 64 a token
    if (N > 0 && (!z || !targets || !saved)) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: null pointer", who);
    if (((uintptr_t)z | (uintptr_t)saved) & 15) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: logits and saved must be 16-byte aligned", who);
    return ESMK_OK;
}

}  // namespace

extern "C" size_t esmk_pref_loss_saved_bytes(int N, int n_pairs) {
    return N < 0 || n_pairs < 0 ? 0 : (size_t)N * sizeof(TokState) + (size_t)(n_pairs + 1) * sizeof(double);
}

extern "C" int esmk_pref_loss_fwd(const void* logits, int dtype, const int64_t* targets, const int32_t* cu_seqlens,
                                  int n_pairs, const float* ref_logps, double beta, double label_smoothing, double nll_weight,
                                  int N, int V, void* saved, size_t saved_bytes, float* logps, float* loss,
                                  esmk_stream_t stream) {
    if (int rc = pl_check("esmk_pref_loss_fwd", logits, dtype, targets, saved, N, V)) return rc;
    if (n_pairs <= 0 || n_pairs >= (1 << 23))  // a launch holds fewer than 2^32 threads, PL_PAIR a pair
        ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_pref_loss_fwd: n_pairs=%d (1..2^23 - 1)", n_pairs);
    if (!cu_seqlens || !ref_logps || !logps || !loss || !saved) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_pref_loss_fwd: null pointer");
    if (!(label_smoothing >= 0.0 && label_smoothing <= 1.0)) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_pref_loss_fwd: label_smoothing outside [0, 1]");
    if (saved_bytes < esmk_pref_loss_saved_bytes(N, n_pairs))
        ESMK_FAIL(ESMK_ERR_WORKSPACE, "esmk_pref_loss_fwd: saved needs %zu bytes", esmk_pref_loss_saved_bytes(N, n_pairs));
    hipStream_t s = (hipStream_t)stream;
    TokState* tok = (TokState*)saved;
    double* pair_loss = (double*)(tok + N);
    unsigned* done = (unsigned*)(pair_loss + n_pairs);
    if (dtype == ESMK_F32) pl_token<float>(logits, targets, cu_seqlens, 2 * n_pairs, tok, done, N, V, s);
    else pl_token<__bf16>(logits, targets, cu_seqlens, 2 * n_pairs, tok, done, N, V, s);
    hipLaunchKernelGGL(pref_pair_kernel, dim3(n_pairs), dim3(PL_PAIR), 0, s, tok, cu_seqlens, ref_logps, N, n_pairs, beta,
                       label_smoothing, nll_weight, logps, pair_loss, done, loss);
    ESMK_CHECK_LAUNCH("esmk_pref_loss_fwd");
    return ESMK_OK;
}

extern "C" int esmk_pref_loss_bwd(const void* logits, int dtype, const int64_t* targets, const void* saved,
                                  const float* grad_loss, void* dlogits, int N, int V, esmk_stream_t stream) {
    if (int rc = pl_check("esmk_pref_loss_bwd", logits, dtype, targets, saved, N, V)) return rc;
    if (N == 0) return ESMK_OK;
    if (!dlogits || ((uintptr_t)dlogits & 15)) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_pref_loss_bwd: dlogits must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == ESMK_F32) pl_grad<float>(logits, targets, (const TokState*)saved, grad_loss, dlogits, N, V, s);
    else pl_grad<__bf16>(logits, targets, (const TokState*)saved, grad_loss, dlogits, N, V, s);
    ESMK_CHECK_LAUNCH("esmk_pref_loss_bwd");
    return ESMK_OK;
}
