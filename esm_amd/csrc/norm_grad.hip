// LayerNorm for training: the forward pass that leaves its row statistics, and the backward pass with the reduction of
// the weight's and the bias's gradients.
//
//   h = (x - mean) rstd,  y = h gamma + beta
//   g = dy gamma,  dx = rstd (g - mean_d(g) - h mean_d(g h)),  dgamma = sum_rows dy h,  dbeta = sum_rows dy
//
// Both are bound by HBM: the forward pass has to move 2 M d elements, the backward pass 3 M d.  At 32768 x 1152 bf16 the
// forward pass takes 30 us (5.0 TB/s; a copy of the same size 5.0), the backward pass 39 + 5 us (5.8 TB/s).  WPR waves share a row
// and keep all of it in registers (one read), sums run in fp32, and the next row's loads are in flight while the current
// one is reduced.  A lane owns the same columns of every row it meets, so it sums its columns of dgamma / dbeta in
// registers; each workgroup leaves one partial row, and a second kernel adds the partial rows in a fixed order (no
// atomics: the same inputs give the same bits).  Few rows take the columns apart instead (norm_columns), and narrow rows share a
// wave ("narrow rows" below).
#include <type_traits>

#include "common.hpp"

namespace {

constexpr int NG_MAX_D = 12288;      // 8 waves x 64 lanes x 24 elements
constexpr int NG_MAX_M = 1 << 30;    // a row number plus the rows of a whole grid stays inside 31 bits
constexpr int NG_FWD_GROUPS = 1024;  // four workgroups per CU; 512 to 2048 measure alike
constexpr int NG_MAX_GROUPS = 512;   // of the backward pass, and so partial rows; 768 and 1024: 2 to 10 % slower

template <typename T> struct NgVec;  // 16 bytes of T
template <> struct NgVec<float> { static constexpr int N = 4; };
template <> struct NgVec<__bf16> { static constexpr int N = 8; };

// VEC elements of a row: 16 bytes, or one element where width, stride or address rule that out.  Rows go through buffer
// descriptors that end where the row ends: a lane past the end reads zeros and its stores are dropped, so neither loop has
// a branch around its loads and stores (with branches the compiler cannot count what is in flight and waits for all of it:
// the forward pass took 54 us at 32768 x 1152 bf16 that way).
template <typename T, int VEC> struct NgRaw { u32x4 v; };
template <> struct NgRaw<float, 1> { unsigned v; };
template <> struct NgRaw<__bf16, 1> { unsigned short v; };

__device__ __forceinline__ __amdgpu_buffer_rsrc_t ng_row(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000);
}
template <typename T, int VEC>
__device__ __forceinline__ NgRaw<T, VEC> ng_load(__amdgpu_buffer_rsrc_t row, int off) {
    NgRaw<T, VEC> r;
    if constexpr (VEC > 1) r.v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(row, off, 0, 0));
    else if constexpr (sizeof(T) == 4) r.v = __builtin_amdgcn_raw_buffer_load_b32(row, off, 0, 0);
    else r.v = __builtin_amdgcn_raw_buffer_load_b16(row, off, 0, 0);
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
__device__ __forceinline__ void ng_unpack(const NgRaw<float, 1>& r, float* f) { f[0] = __uint_as_float(r.v); }
__device__ __forceinline__ void ng_unpack(const NgRaw<__bf16, 1>& r, float* f) { f[0] = bf16_bits_to_f32(r.v); }
template <typename T, int VEC>
__device__ __forceinline__ void ng_store(__amdgpu_buffer_rsrc_t row, int off, const float (&f)[VEC]) {
    if constexpr (VEC == 8)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])}, row, off, 0, 0);
    else if constexpr (VEC == 4)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}, row, off, 0, 0);
    else if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(f[0]), row, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16_bits(f[0]), row, off, 0, 0);
}
// VEC fp32 parameters
template <int VEC>
__device__ __forceinline__ void ng_param(const float* p, int d, int off, float (&f)[VEC]) {
    const __amdgpu_buffer_rsrc_t r = ng_row(p, p ? d * 4 : 0);
#pragma unroll
    for (int e = 0; e < VEC; e += VEC > 1 ? 4 : 1) {
        if constexpr (VEC > 1) {
            const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (off + e) * 4, 0, 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) f[e + i] = __uint_as_float(v[i]);
        } else {
            f[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (off + e) * 4, 0, 0));
        }
    }
}

// Threads of a workgroup: four waves, eight where eight waves share a row.
constexpr int ng_threads(int wpr) { return wpr == 8 ? 512 : 256; }

// Sum over the 64 lanes, the same in all of them, on the vector ALU alone (DPP within 16 lanes, then the half-row and
// half-wave swaps): a row waits for two such sums, and through the LDS crossbar each of their six steps costs its latency.
__device__ __forceinline__ float lane_sum(float v) {
    auto step = [&](auto ctrl) { v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false)); };
    step(std::integral_constant<int, 0xB1>{});   // lane ^ 1
    step(std::integral_constant<int, 0x4E>{});   // lane ^ 2
    step(std::integral_constant<int, 0x141>{});  // mirrored in 8
    step(std::integral_constant<int, 0x140>{});  // mirrored in 16
    auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Sum of (a, b) over the WPR waves of a row.  `buf` holds one pair per wave and alternates between two halves, so that
// one barrier per call is enough: a wave reaches the call after next only behind the barrier that every reader of the
// earlier half has passed.  All waves of the workgroup call it equally often.
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf, int& half) {
    a = lane_sum(a);
    b = lane_sum(b);
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
    constexpr int STEP = 64 * WPR * VEC;              // elements between a lane's vectors
    __shared__ float buf[32];
    const int lane = threadIdx.x & (64 * WPR - 1);
    const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
    const int stride = gridDim.x * ROWS, bytes = d * (int)sizeof(T);
    const float inv_d = 1.0f / (float)d;
    int half = 0;
    NgRaw<T, VEC> raw[NV];
    auto load = [&](int r) {
        const __amdgpu_buffer_rsrc_t xr = ng_row(x + (r < M ? r : 0) * ldx, r < M ? bytes : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = ng_load<T, VEC>(xr, (lane * VEC + i * STEP) * (int)sizeof(T));
    };
    int row = blockIdx.x * ROWS + slot;
    load(row);
    __builtin_amdgcn_sched_barrier(0);  // the row first: the loop then waits for loads by count, not for stores
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ng_param<VEC>(gamma, d, lane * VEC + i * STEP, w[i]);
        ng_param<VEC>(beta, d, lane * VEC + i * STEP, b[i]);
    }
    for (; row - slot < M; row += stride) {  // the same number of turns in every wave of the workgroup
        float v[NV][VEC], sum = 0.f, none = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ng_unpack(raw[i], v[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += v[i][e];
        }
        load(row + stride < M ? row + stride : M);
        row_sum2<WPR>(sum, none, buf, half);
        const float mean = sum * inv_d;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool in = lane * VEC + i * STEP < d;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] = in ? v[i][e] - mean : 0.f;
                sq += v[i][e] * v[i][e];
            }
        }
        row_sum2<WPR>(sq, none, buf, half);
        const float rstd = 1.0f / sqrtf(sq * inv_d + eps);
        const int at = row < M ? row : 0;
        const __amdgpu_buffer_rsrc_t sr = ng_row(stats + 2 * (int64_t)at, row < M ? 8 : 0);
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(mean), __float_as_uint(rstd)}, sr, lane * 8, 0, 0);
        const __amdgpu_buffer_rsrc_t yr = ng_row(y + (int64_t)at * d, row < M ? bytes : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = v[i][e] * rstd * w[i][e] + b[i][e];
            ng_store<T, VEC>(yr, (lane * VEC + i * STEP) * (int)sizeof(T), o);
        }
    }
}

// The parameters' gradients of few rows, by workgroups of their own in the same launch: 32 columns each, all rows, x and dy read a
// second time (from the cache).  That spares the partial rows, their kernel and its launch: backward pass of 66, 512, 1000 rows of
// 1152 bf16 9.2, 9.5, 10.1 us with partial rows and 3.3, 7.0, 11.3 so (enqueued call by call 15.6 and 11.5 at all three); 512, 768
// rows of 4096 fp32 11.5, 12.9 and 10.7, 14.5.
template <typename T>
__device__ __forceinline__ void norm_columns(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                                             const float* __restrict__ stats, float* __restrict__ dgamma,
                                             float* __restrict__ dbeta, int M, int d, int block) {
    __shared__ float sums[16][2][32];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, groups = blockDim.x >> 5, c = block * 32 + col;
    float a = 0.f, b = 0.f;
    if (c < d)
#pragma unroll 8
        for (int r = grp; r < M; r += groups) {
            const float g = (float)dy[r * lddy + c];
            a += g * (((float)x[r * ldx + c] - stats[2 * r]) * stats[2 * r + 1]);
            b += g;
        }
    sums[grp][0][col] = a;
    sums[grp][1][col] = b;
    __syncthreads();
    if (grp > 0 || c >= d) return;
    for (int i = 1; i < groups; ++i) {
        a += sums[i][0][col];
        b += sums[i][1][col];
    }
    if (dgamma) dgamma[c] = a;
    if (dbeta) dbeta[c] = b;
}

// The last `cols` workgroups take columns (pg and pb are the gradients themselves), the others rows.
template <typename T, int VEC, int NV, int WPR>
__global__ __launch_bounds__(ng_threads(WPR)) void norm_bwd_kernel(const T* __restrict__ dy, int64_t lddy,
                                                                   const T* __restrict__ x, int64_t ldx,
                                                                   const float* __restrict__ gamma,
                                                                   const float* __restrict__ stats, T* __restrict__ dx,
                                                                   float* __restrict__ pg, float* __restrict__ pb, int M,
                                                                   int d, int cols) {
    const int row_groups = gridDim.x - cols;
    if ((int)blockIdx.x >= row_groups) return norm_columns(dy, lddy, x, ldx, stats, pg, pb, M, d, blockIdx.x - row_groups);
    constexpr int ROWS = ng_threads(WPR) / 64 / WPR, STEP = 64 * WPR * VEC;
    __shared__ float buf[32];
    extern __shared__ float part[];  // [ROWS - 1][2][d]
    const int lane = threadIdx.x & (64 * WPR - 1);
    const int slot = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));
    const int stride = row_groups * ROWS, bytes = d * (int)sizeof(T);
    const float inv_d = 1.0f / (float)d;
    int half = 0;
    NgRaw<T, VEC> rx[NV], rg[NV];
    float mean = 0.f, rstd = 0.f;
    auto load = [&](int r) {
        const int at = r < M ? r : 0;
        const int n = r < M ? bytes : 0;
        const __amdgpu_buffer_rsrc_t xr = ng_row(x + at * ldx, n), gr = ng_row(dy + at * lddy, n);
        mean = r < M ? stats[2 * (int64_t)at] : 0.f;
        rstd = r < M ? stats[2 * (int64_t)at + 1] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            rx[i] = ng_load<T, VEC>(xr, (lane * VEC + i * STEP) * (int)sizeof(T));
            rg[i] = ng_load<T, VEC>(gr, (lane * VEC + i * STEP) * (int)sizeof(T));
        }
    };
    int row = blockIdx.x * ROWS + slot;
    load(row);
    __builtin_amdgcn_sched_barrier(0);
    float w[NV][VEC], ag[NV][VEC], ab[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ng_param<VEC>(gamma, d, lane * VEC + i * STEP, w[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ag[i][e] = ab[i][e] = 0.f;
    }
    for (; row - slot < M; row += stride) {
        float h[NV][VEC], g[NV][VEC], c1 = 0.f, c2 = 0.f;
        const float rs = rstd;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            // past the row's end, and in a row past the last, dy reads as zero: nothing is added anywhere (h is finite there)
            ng_unpack(rx[i], h[i]);
            ng_unpack(rg[i], g[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[i][e] = (h[i][e] - mean) * rs;
                ag[i][e] += g[i][e] * h[i][e];
                ab[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                c1 += g[i][e];
                c2 += g[i][e] * h[i][e];
            }
        }
        load(row + stride < M ? row + stride : M);
        row_sum2<WPR>(c1, c2, buf, half);
        c1 *= inv_d;
        c2 *= inv_d;
        const __amdgpu_buffer_rsrc_t dr = ng_row(dx + (int64_t)(row < M ? row : 0) * d, dx && row < M ? bytes : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = (g[i][e] - c1 - h[i][e] * c2) * rs;
            ng_store<T, VEC>(dr, (lane * VEC + i * STEP) * (int)sizeof(T), o);
        }
    }
    if (cols > 0 || (!pg && !pb)) return;
    // the workgroup's row slots, added in order
    constexpr int Q = VEC > 1 ? 4 : 1;  // floats per LDS access
    typedef float fq __attribute__((ext_vector_type(Q)));
    if (slot > 0) {
        float* p = part + (slot - 1) * 2 * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = lane * VEC + i * STEP;
            if (c < d)
#pragma unroll
                for (int e = 0; e < VEC; e += Q) {
                    fq u, v;
#pragma unroll
                    for (int j = 0; j < Q; ++j) { u[j] = ag[i][e + j]; v[j] = ab[i][e + j]; }
                    *(fq*)(p + c + e) = u;
                    *(fq*)(p + d + c + e) = v;
                }
        }
    }
    __syncthreads();
    if (slot > 0) return;
    const __amdgpu_buffer_rsrc_t gr = ng_row(pg + (int64_t)blockIdx.x * d, pg ? d * 4 : 0);
    const __amdgpu_buffer_rsrc_t br = ng_row(pb + (int64_t)blockIdx.x * d, pb ? d * 4 : 0);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = lane * VEC + i * STEP;
        if (c < d)
            for (int s = 0; s < ROWS - 1; ++s)
#pragma unroll
                for (int e = 0; e < VEC; e += Q) {
                    const fq u = *(const fq*)(part + s * 2 * d + c + e), v = *(const fq*)(part + s * 2 * d + d + c + e);
#pragma unroll
                    for (int j = 0; j < Q; ++j) { ag[i][e + j] += u[j]; ab[i][e + j] += v[j]; }
                }
#pragma unroll
        for (int e = 0; e < VEC; e += Q) {
            float u[Q], v[Q];
#pragma unroll
            for (int j = 0; j < Q; ++j) { u[j] = ag[i][e + j]; v[j] = ab[i][e + j]; }
            ng_store<float, Q>(gr, (c + e) * 4, u);
            ng_store<float, Q>(br, (c + e) * 4, v);
        }
    }
}

// ---- narrow rows ----------------------------------------------------------------------------------------------------------
// Up to 256 elements: 16 lanes per row, four rows in a wave.  A wave per row spends about 150 instructions on one whatever its
// width: 32768 x 64 bf16 forward and backward 9.6, 12.2 us that way and 4.8, 7.6 this way; x 77 fp32 10.6, 15.5 and 6.6, 9.0;
// x 256 bf16 10.3, 13.4 and 7.7, 12.8.  The 16 rows of a workgroup go through one buffer descriptor; lanes past the end of a row,
// and rows past the last, are addressed out of its range.
constexpr int NG_NARROW = 256, NG_NARROW_ROWS = 16;
constexpr int NG_OUT = 0x7ffffff0;

__device__ __forceinline__ float sum16(float v) {
    auto step = [&](auto ctrl) { v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false)); };
    step(std::integral_constant<int, 0xB1>{});   // lane ^ 1
    step(std::integral_constant<int, 0x4E>{});   // lane ^ 2
    step(std::integral_constant<int, 0x141>{});  // mirrored in 8
    step(std::integral_constant<int, 0x140>{});  // mirrored in 16
    return v;
}
// the same column of a wave's four rows
__device__ __forceinline__ float sum_rows4(float v) {
    auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// Rows row0 .. row0 + 15 of a tensor, as far as they exist; a lane's elements start at its column.
template <typename T, int VEC, int NV>
struct NgRows {
    int off[NV];  // bytes from the first row
    int ld;       // bytes
    __device__ __forceinline__ NgRows(int64_t ld_, int slot, int sub, int d) : ld((int)(ld_ * (int)sizeof(T))) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (sub + i * 16) * VEC;
            off[i] = c < d ? slot * ld + c * (int)sizeof(T) : NG_OUT;
        }
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(const void* p, int row0, int M, int d) const {
        const int rows = min(M - row0, NG_NARROW_ROWS);  // below 1: none
        return ng_row((const char*)p + (int64_t)(rows > 0 ? row0 : 0) * ld, rows > 0 ? (rows - 1) * ld + d * (int)sizeof(T) : 0);
    }
};

template <typename T, int VEC, int NV>
__global__ __launch_bounds__(256) void norm_fwd_narrow_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ gamma,
                                                              const float* __restrict__ beta, T* __restrict__ y,
                                                              float* __restrict__ stats, int M, int d, float eps) {
    const int sub = threadIdx.x & 15, slot = threadIdx.x >> 4, stride = gridDim.x * NG_NARROW_ROWS;
    const float inv_d = 1.0f / (float)d;
    const NgRows<T, VEC, NV> rx(ldx, slot, sub, d), ry(d, slot, sub, d);
    NgRaw<T, VEC> raw[NV];
    auto load = [&](int row0) {
        const __amdgpu_buffer_rsrc_t r = rx.at(x, row0, M, d);
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = ng_load<T, VEC>(r, rx.off[i]);
    };
    int row0 = blockIdx.x * NG_NARROW_ROWS;
    load(row0);
    __builtin_amdgcn_sched_barrier(0);
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ng_param<VEC>(gamma, d, (sub + i * 16) * VEC, w[i]);
        ng_param<VEC>(beta, d, (sub + i * 16) * VEC, b[i]);
    }
    for (; row0 < M; row0 += stride) {
        float v[NV][VEC], sum = 0.f, sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ng_unpack(raw[i], v[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += v[i][e];
        }
        load(row0 + stride);
        const float mean = sum16(sum) * inv_d;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] = rx.off[i] != NG_OUT ? v[i][e] - mean : 0.f;
                sq += v[i][e] * v[i][e];
            }
        const float rstd = 1.0f / sqrtf(sum16(sq) * inv_d + eps);
        if (sub == 0 && row0 + slot < M) *(f32x2*)(stats + 2 * (int64_t)(row0 + slot)) = f32x2{mean, rstd};
        const __amdgpu_buffer_rsrc_t r = ry.at(y, row0, M, d);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = v[i][e] * rstd * w[i][e] + b[i][e];
            ng_store<T, VEC>(r, ry.off[i], o);
        }
    }
}

template <typename T, int VEC, int NV>
__global__ __launch_bounds__(256) void norm_bwd_narrow_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                                                              int64_t ldx, const float* __restrict__ gamma,
                                                              const float* __restrict__ stats, T* __restrict__ dx,
                                                              float* __restrict__ pg, float* __restrict__ pb, int M, int d,
                                                              int cols) {
    const int row_groups = gridDim.x - cols;
    if ((int)blockIdx.x >= row_groups) return norm_columns(dy, lddy, x, ldx, stats, pg, pb, M, d, blockIdx.x - row_groups);
    __shared__ float part[3][2][NG_NARROW];
    const int sub = threadIdx.x & 15, slot = threadIdx.x >> 4, stride = row_groups * NG_NARROW_ROWS;
    const float inv_d = 1.0f / (float)d;
    const NgRows<T, VEC, NV> rx(ldx, slot, sub, d), rg(lddy, slot, sub, d), ro(d, slot, sub, d);
    NgRaw<T, VEC> raw_x[NV], raw_g[NV];
    f32x2 st;
    auto load = [&](int row0) {
        const __amdgpu_buffer_rsrc_t a = rx.at(x, row0, M, d), b = rg.at(dy, row0, M, d);
        st = *(const f32x2*)(stats + 2 * (int64_t)min(row0 + slot, M - 1));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            raw_x[i] = ng_load<T, VEC>(a, rx.off[i]);
            raw_g[i] = ng_load<T, VEC>(b, rg.off[i]);
        }
    };
    int row0 = blockIdx.x * NG_NARROW_ROWS;
    load(row0);
    __builtin_amdgcn_sched_barrier(0);
    float w[NV][VEC], ag[NV][VEC], ab[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ng_param<VEC>(gamma, d, (sub + i * 16) * VEC, w[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ag[i][e] = ab[i][e] = 0.f;
    }
    for (; row0 < M; row0 += stride) {
        float h[NV][VEC], g[NV][VEC], c1 = 0.f, c2 = 0.f;
        const bool on = row0 + slot < M;
        const float mean = on ? st[0] : 0.f, rs = on ? st[1] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            ng_unpack(raw_x[i], h[i]);  // past the end of the row, and in a row past the last, dy reads as zero
            ng_unpack(raw_g[i], g[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[i][e] = (h[i][e] - mean) * rs;
                ag[i][e] += g[i][e] * h[i][e];
                ab[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                c1 += g[i][e];
                c2 += g[i][e] * h[i][e];
            }
        }
        load(row0 + stride);
        c1 = sum16(c1) * inv_d;
        c2 = sum16(c2) * inv_d;
        const __amdgpu_buffer_rsrc_t r = ro.at(dx, row0, dx ? M : 0, d);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = (g[i][e] - c1 - h[i][e] * c2) * rs;
            ng_store<T, VEC>(r, ro.off[i], o);
        }
    }
    if (cols > 0 || (!pg && !pb)) return;
    const int wave = threadIdx.x >> 6;
    const bool first = (threadIdx.x & 63) < 16;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            ag[i][e] = sum_rows4(ag[i][e]);
            ab[i][e] = sum_rows4(ab[i][e]);
            const int c = (sub + i * 16) * VEC + e;
            if (wave > 0 && first && c < d) {
                part[wave - 1][0][c] = ag[i][e];
                part[wave - 1][1][c] = ab[i][e];
            }
        }
    __syncthreads();
    if (wave > 0 || !first) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = (sub + i * 16) * VEC + e;
            if (c >= d) continue;
            if (pg) pg[(int64_t)blockIdx.x * d + c] = ag[i][e] + part[0][0][c] + part[1][0][c] + part[2][0][c];
            if (pb) pb[(int64_t)blockIdx.x * d + c] = ab[i][e] + part[0][1][c] + part[1][1][c] + part[2][1][c];
        }
}

// Column sums of the G partial rows: 32 columns x 32 groups of rows per workgroup, then the groups in order.  A few
// microseconds of latency: a group's rows are requested eight at a time.
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
#pragma unroll 8
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
// small M a row slot sees at least four rows (two narrow ones).
int ng_groups(int M, int d) {
    const int rows = d <= NG_NARROW ? 2 * NG_NARROW_ROWS : 4 * ng_rows(ng_waves(d));
    const int want = (M + rows - 1) / rows;
    return want < NG_MAX_GROUPS ? want : NG_MAX_GROUPS;
}
constexpr int NG_FEW = 512;  // rows up to which the parameters' gradients are taken column by column, see norm_columns()

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

// d <= NG_NARROW: f(constant<VEC>, constant<NV>)
template <int VEC, typename F>
void ng_narrow_dispatch(int d, F f) {
    if (d <= 128) f(std::integral_constant<int, VEC>{}, std::integral_constant<int, 8 / VEC>{});
    else f(std::integral_constant<int, VEC>{}, std::integral_constant<int, 16 / VEC>{});
}
// The offsets of 16 rows have to fit a buffer descriptor.
bool ng_narrow(int d, int64_t ld, int size) { return d <= NG_NARROW && ld * size < (1LL << 27); }

bool ng_wide(const void* p, int64_t ld, int size) { return ((uintptr_t)p & 15) == 0 && (ld * size) % 16 == 0; }

template <typename T>
int norm_fwd(const T* x, int64_t ldx, const float* gamma, const float* beta, T* y, float* stats, int M, int d, float eps,
             hipStream_t s) {
    auto go = [&](auto vec, auto nv, auto wpr) {
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value, W = decltype(wpr)::value;
        const int rows = ng_rows(W), want = (M + rows - 1) / rows, cap = NG_FWD_GROUPS;
        hipLaunchKernelGGL((norm_fwd_kernel<T, V, N, W>), dim3(want < cap ? want : cap), dim3(ng_threads(W)), 0, s, x, ldx,
                           gamma, beta, y, stats, M, d, eps);
        return true;
    };
    const bool wide = ng_wide(x, ldx, sizeof(T)) && ng_wide(y, d, sizeof(T));
    if (ng_narrow(d, ldx, sizeof(T))) {
        auto narrow = [&](auto vec, auto nv) {
            constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
            const int want = (M + NG_NARROW_ROWS - 1) / NG_NARROW_ROWS;
            hipLaunchKernelGGL((norm_fwd_narrow_kernel<T, V, N>), dim3(want < NG_FWD_GROUPS ? want : NG_FWD_GROUPS), dim3(256), 0, s,
                               x, ldx, gamma, beta, y, stats, M, d, eps);
        };
        if (wide) ng_narrow_dispatch<NgVec<T>::N>(d, narrow);
        else ng_narrow_dispatch<1>(d, narrow);
        ESMK_CHECK_LAUNCH("esmk_layernorm_fwd");
        return ESMK_OK;
    }
    if (!(wide ? ng_dispatch<T, NgVec<T>::N>(d, go) : ng_dispatch<T, 1>(d, go)))
        ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_fwd: d=%d", d);
    ESMK_CHECK_LAUNCH("esmk_layernorm_fwd");
    return ESMK_OK;
}

template <typename T>
int norm_bwd(const T* dy, int64_t lddy, const T* x, int64_t ldx, const float* gamma, const float* stats, T* dx,
             float* dgamma, float* dbeta, float* ws, int M, int d, hipStream_t s) {
    const bool few = M <= NG_FEW;  // the row workgroups then have one turn of rows each
    const int turn = d <= NG_NARROW ? NG_NARROW_ROWS : ng_rows(ng_waves(d));
    const int cols = few && (dgamma || dbeta) ? (d + 31) / 32 : 0;
    const int G = !few ? ng_groups(M, d) : dx ? (M + turn - 1) / turn : 0;  // few rows: the row workgroups are there for dx alone
    float* pg = dgamma ? (few ? dgamma : ws) : nullptr;
    float* pb = dbeta ? (few ? dbeta : ws + (int64_t)G * d) : nullptr;
    auto go = [&](auto vec, auto nv, auto wpr) {
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value, W = decltype(wpr)::value;
        const int lds = few ? 0 : (ng_rows(W) - 1) * 2 * d * (int)sizeof(float);  // at most 3 x 2 x 1536 x 4 = 36 KiB
        hipLaunchKernelGGL((norm_bwd_kernel<T, V, N, W>), dim3(G + cols), dim3(ng_threads(W)), lds, s, dy, lddy, x, ldx, gamma,
                           stats, dx, pg, pb, M, d, cols);
        return true;
    };
    const bool wide = ng_wide(x, ldx, sizeof(T)) && ng_wide(dy, lddy, sizeof(T)) && ng_wide(dx, d, sizeof(T));
    auto narrow = [&](auto vec, auto nv) {
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
        hipLaunchKernelGGL((norm_bwd_narrow_kernel<T, V, N>), dim3(G + cols), dim3(256), 0, s, dy, lddy, x, ldx, gamma, stats, dx, pg, pb, M, d,
                           cols);
    };
    if (ng_narrow(d, ldx, sizeof(T)) && ng_narrow(d, lddy, sizeof(T))) {
        if (wide) ng_narrow_dispatch<NgVec<T>::N>(d, narrow);
        else ng_narrow_dispatch<1>(d, narrow);
    } else if (!(wide ? ng_dispatch<T, NgVec<T>::N>(d, go) : ng_dispatch<T, 1>(d, go)))
        ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_bwd: d=%d", d);
    if (!few && (dgamma || dbeta))
        hipLaunchKernelGGL(norm_grad_reduce_kernel, dim3((d + 31) / 32, 2), dim3(1024), 0, s, pg, pb, dgamma, dbeta, G, d);
    ESMK_CHECK_LAUNCH("esmk_layernorm_bwd");
    return ESMK_OK;
}

}  // namespace

extern "C" int esmk_layernorm_fwd(const void* x, int dtype, int64_t ldx, const float* gamma, const float* beta, void* y,
                                  float* stats, int M, int d, float eps, esmk_stream_t stream) {
    if (M < 0 || M > NG_MAX_M || d <= 0 || d > NG_MAX_D) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_fwd: M=%d (0..2^30), d=%d (1..%d)", M, d, NG_MAX_D);
    if (dtype != ESMK_F32 && dtype != ESMK_BF16) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: bad dtype %d", dtype);
    if (M == 0) return ESMK_OK;
    if (!x || !gamma || !y || !stats) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: null pointer");
    if (ldx < d) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: row stride %lld below d=%d", (long long)ldx, d);
    if ((uintptr_t)stats & 7) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_fwd: stats must be 8-byte aligned");
    if (dtype == ESMK_F32) return norm_fwd<float>((const float*)x, ldx, gamma, beta, (float*)y, stats, M, d, eps, (hipStream_t)stream);
    return norm_fwd<__bf16>((const __bf16*)x, ldx, gamma, beta, (__bf16*)y, stats, M, d, eps, (hipStream_t)stream);
}

extern "C" size_t esmk_layernorm_bwd_workspace_bytes(int M, int d) {
    if (M <= 0 || M > NG_MAX_M || d <= 0 || d > NG_MAX_D) return 0;
    return M <= NG_FEW ? 0 : (size_t)ng_groups(M, d) * 2 * d * sizeof(float);
}

extern "C" int esmk_layernorm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int dtype, const float* gamma,
                                  const float* stats, void* dx, float* dgamma, float* dbeta, void* workspace,
                                  size_t workspace_bytes, int M, int d, esmk_stream_t stream) {
    if (M < 0 || M > NG_MAX_M || d <= 0 || d > NG_MAX_D) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "esmk_layernorm_bwd: M=%d (0..2^30), d=%d (1..%d)", M, d, NG_MAX_D);
    if (dtype != ESMK_F32 && dtype != ESMK_BF16) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: bad dtype %d", dtype);
    if (M == 0) {  // no rows: the parameters' gradients are zero
        if (dgamma || dbeta)
            hipLaunchKernelGGL(norm_grad_zero_kernel, dim3((d + 255) / 256), dim3(256), 0, (hipStream_t)stream, dgamma, dbeta, d);
        ESMK_CHECK_LAUNCH("esmk_layernorm_bwd");
        return ESMK_OK;
    }
    if (!dy || !x || !gamma || !stats) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: null pointer");
    if (!dx && !dgamma && !dbeta) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_layernorm_bwd: null pointer (no gradient is wanted)");
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
