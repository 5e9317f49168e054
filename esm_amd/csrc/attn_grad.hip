// Block-diagonal (varlen packed, non-causal) attention for training, head dim 64 or 128: a forward pass that leaves the
// log-sum-exp of every query row, and a backward pass that recomputes the probabilities from it.
//
//   S = scale Q K^T (masked keys: -inf),  P = exp(S - lse),  O = P V
//   delta = rowsum(dO O),  dS = P (dO V^T - delta),  dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q
//
// Query heads share key heads in groups of n_heads / n_kv_heads.  A query row without any key gets O = 0, lse = -inf and
// no gradient; tokens before the first and behind the last sequence get zeros (lse -inf).
//
// Matrix products run on v_mfma_f32_32x32x16_bf16 with fp32 accumulators.  A product's operand that lives in the lanes is
// held in registers for the whole kernel (queries in the forward and dQ kernels, keys in the dK / dV kernel); the other
// side streams through a two-slot LDS ring of 64- or 32-row tiles, filled by LDS-DMA one tile ahead.  Scores are formed with
// the resident side on the lanes and the streamed side in the registers, so the exponentiated tile converts in place (bf16,
// the second operand of the MFMA that consumes it) and softmax statistics stay in fp32.  The transposed operand of the
// second product is read from the same row-major tile with ds_read_b64_tr_b16: the LDS image's 16-byte chunks are
// XOR-swizzled by a function of the row that keeps both the row reads and the transposed reads free of bank conflicts.
//
// Calls whose blocks of 128 rows do not fill the card run smaller blocks, whose four waves share the other side ("few rows" below,
// ag_few()).
//
// The backward pass is two kernels, each with one owner for every output element (no atomics, so the same inputs give the
// same bits): dQ per query block (three products; it also forms delta), dK / dV per key block (four).
//
// Measured (forward, dQ, dK dV): 64 x 512 tokens, 18 heads of 64: 113, 170, 221 us - eight tiles per workgroup, so that a third
// of its life is the load of the first rows and the store of the last; 4 x 4096, 40 heads of 64: 691, 936, 1246 us (995, 1101,
// 1103 TFLOP/s) - matrix pipes 55 to 60 % busy at the clock the power limit leaves; a 2 TB/s share of HBM in both.
#include <math.h>

#include <type_traits>

#include "common.hpp"

namespace {

constexpr int TR = 64;       // rows of a streamed tile, where a kernel does not say 32
constexpr int AG_WAVES = 4;
constexpr float AG_LOG2E = 1.4426950408889634f, AG_LN2 = 0.6931471805599453f;

__device__ __forceinline__ int crow(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }

// A strided [token][head][D] tensor, strides in elements.
struct View {
    const __bf16* p;
    int64_t tok, head;
};
struct OutView {
    __bf16* p;
    int64_t tok, head;
};

// ---- LDS image of a tile: row r at r * 2D bytes, its 16-byte chunk c at c ^ swz(r) -----------------------------
//   row reads (32 rows, one logical chunk, ds_read_b128): 16 consecutive rows cover all 64 banks
//   transposed reads (rows 4h..4h+3, 64 bytes each, ds_read_b64_tr_b16): the four rows cover all 64 banks
template <int D>
__device__ __forceinline__ int swz(int r) {
    if constexpr (D == 64) return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1);  // bit reversal of (r >> 1) & 7
    else return (r & 3) << 2 | ((r >> 2) & 3);
}

// LDS-DMA of one tile: a wave moves pieces of 1 KiB (64 lanes x 16 bytes, LDS side linear, swizzle on the source address).
// Rows past `rows` are out of the descriptor's range and land as zeros.
template <int D, int ROWS = TR, int WAVES = AG_WAVES>
struct Stage {
    static constexpr int RB = 2 * D, CPR = D / 8, PIECES = ROWS * RB / 1024 / WAVES;
    unsigned off[PIECES];
    unsigned ldb;
    __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
        ldb = (unsigned)(ld * 2);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = (wave * PIECES + i) * (64 / CPR) + lane / CPR;
            off[i] = (unsigned)r * ldb + (unsigned)((lane & (CPR - 1)) ^ swz<D>(r)) * 16u;
        }
    }
    // Rows whose bit is clear are addressed out of range and land as zeros (a masked row may hold NaN or inf, and 0 times
    // those is NaN).
    __device__ __forceinline__ void go_masked(char* lds, const __bf16* first, int rows, int wave, int lane, unsigned long long bits) const {
        const int nrec = (int)((rows < ROWS ? rows - 1 : ROWS - 1) * ldb + RB);
        const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)first, 0, nrec, 0x00020000);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = (wave * PIECES + i) * (64 / CPR) + lane / CPR;
            const int o = (bits >> r) & 1 ? (int)off[i] : 0x7ffffff0;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(d, LDS_PTR(lds + (wave * PIECES + i) * 1024), 16, o, 0, 0, 0);
        }
    }
    // first: first row of the tile (wave-uniform), rows: rows of it that exist (>= 1)
    __device__ __forceinline__ void go(char* lds, const __bf16* first, int rows, int wave) const {
        const int nrec = (int)((rows < ROWS ? rows - 1 : ROWS - 1) * ldb + RB);
        const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)first, 0, nrec, 0x00020000);
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(d, LDS_PTR(lds + (wave * PIECES + i) * 1024), 16, (int)off[i], 0, 0, 0);
    }
};

// Transposed fragments (first operand of an MFMA over 16 tile rows) of all D / 32 column tiles, for 16-row step SP and, at
// D = 64, also SP + 1: eight ds_read_b64_tr_b16.  Fragment slot (hi, j) holds tile row 16 SP + 4 hi + (j & 3) + 8 (j >> 2),
// which is the row of accumulator register 8 (SP & 1) + j: the converted scores are the second operand as they stand.
// The wait is part of the statement: no load is in flight when the compiler sees its outputs.
template <int D>
struct TrAddr {
    unsigned a[2][D / 32];  // [rows +0 / +8][column tile], bytes inside a tile
    __device__ __forceinline__ void init(int lane) {
        const int i = lane & 15, g = (lane >> 4) & 1, hi = lane >> 5;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 4 * hi + (i >> 2) + 8 * e, ch = 2 * g + ((i & 3) >> 1);
#pragma unroll
            for (int t = 0; t < D / 32; ++t) a[e][t] = (unsigned)(r * 2 * D + (((4 * t + ch) ^ swz<D>(r)) << 4) + (i & 1) * 8);
        }
    }
};
struct TrFrag { u32x2 v[8]; };

#define AG_TR8(F, A0, A1, A2, A3, A4, A5, A6, A7, O0, O1)                                                               \
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%c16\n\tds_read_b64_tr_b16 %1, %9 offset:%c16\n\t"                    \
                 "ds_read_b64_tr_b16 %2, %10 offset:%c16\n\tds_read_b64_tr_b16 %3, %11 offset:%c16\n\t"                  \
                 "ds_read_b64_tr_b16 %4, %12 offset:%c17\n\tds_read_b64_tr_b16 %5, %13 offset:%c17\n\t"                  \
                 "ds_read_b64_tr_b16 %6, %14 offset:%c17\n\tds_read_b64_tr_b16 %7, %15 offset:%c17\n\t"                  \
                 "s_waitcnt lgkmcnt(0)"                                                                                 \
                 : "=&v"(F.v[0]), "=&v"(F.v[1]), "=&v"(F.v[2]), "=&v"(F.v[3]), "=&v"(F.v[4]), "=&v"(F.v[5]),             \
                   "=&v"(F.v[6]), "=&v"(F.v[7])                                                                         \
                 : "v"(A0), "v"(A1), "v"(A2), "v"(A3), "v"(A4), "v"(A5), "v"(A6), "v"(A7), "i"(O0), "i"(O1)              \
                 : "memory")

// D = 64: v[4 s + 2 t + e] for 16-row steps SP + s; D = 128: v[2 t + e] for step SP
template <int D, int SP>
__device__ __forceinline__ TrFrag tr_read(const TrAddr<D>& ta, unsigned tile) {
    TrFrag f;
    constexpr int O = SP * 16 * 2 * D;
    if constexpr (D == 64) {
        const unsigned a0 = tile + ta.a[0][0], a1 = tile + ta.a[1][0], a2 = tile + ta.a[0][1], a3 = tile + ta.a[1][1];
        AG_TR8(f, a0, a1, a2, a3, a0, a1, a2, a3, O, O + 16 * 2 * D);
    } else {
        AG_TR8(f, tile + ta.a[0][0], tile + ta.a[1][0], tile + ta.a[0][1], tile + ta.a[1][1], tile + ta.a[0][2],
               tile + ta.a[1][2], tile + ta.a[0][3], tile + ta.a[1][3], O, O);
    }
    return f;
}
__device__ __forceinline__ bf16x8 tr_frag(const TrFrag& f, int i) {
    return __builtin_bit_cast(bf16x8, u32x4{f.v[i].x, f.v[i].y, f.v[i + 1].x, f.v[i + 1].y});
}

// acc[t] (column tile t of D, lanes = resident rows) += X^T . B, X = tile rows 32 MT .. 32 MT + 31, b = their two 16-row steps
template <int D, int MT>
__device__ __forceinline__ void mfma_tr(f32x16 (&acc)[D / 32], const TrAddr<D>& ta, unsigned tile, const bf16x8 (&b)[2]) {
    if constexpr (D == 64) {
        const TrFrag f = tr_read<D, 2 * MT>(ta, tile);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag(f, 4 * s + 2 * t), b[s], acc[t], 0, 0, 0);
    } else {
        {
            const TrFrag f = tr_read<D, 2 * MT>(ta, tile);
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag(f, 2 * t), b[0], acc[t], 0, 0, 0);
        }
        const TrFrag f = tr_read<D, 2 * MT + 1>(ta, tile);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_frag(f, 2 * t), b[1], acc[t], 0, 0, 0);
    }
}

// init + (32 tile rows from `tile` on) . (resident rows)^T; roff: row_off() of this lane
template <int D>
__device__ __forceinline__ f32x16 mfma_rows(const char* tile, int roff, const bf16x8 (&b)[D / 16], f32x16 init) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
        init = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(tile + (roff ^ (ks << 5))), b[ks], init, 0, 0, 0);
    return init;
}
template <int D>
__device__ __forceinline__ int row_off(int l31, int hi) {  // swz() repeats every 16 rows: rows 32 further are 64 D bytes further
    return l31 * 2 * D + ((hi ^ swz<D>(l31)) << 4);
}

__device__ __forceinline__ f32x16 splat16(float v) {
    f32x16 r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v;
    return r;
}

// maximum / sum of a value over the two half-waves that share a resident row
__device__ __forceinline__ float half_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Row of D outputs from accumulators [column 32 t + crow(r, hi)][row on the lane]: a half-wave exchange leaves 16
// contiguous bytes in every lane.  All lanes take part; `on` guards the store.
template <int D>
__device__ __forceinline__ void store_row(__bf16* row, const f32x16 (&o)[D / 32], float mul, int hi, bool on) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            const unsigned ax = pack_bf16x2(o[t][4 * g] * mul, o[t][4 * g + 1] * mul);
            const unsigned ay = pack_bf16x2(o[t][4 * g + 2] * mul, o[t][4 * g + 3] * mul);
            const unsigned bx = pack_bf16x2(o[t][4 * g + 4] * mul, o[t][4 * g + 5] * mul);
            const unsigned by = pack_bf16x2(o[t][4 * g + 6] * mul, o[t][4 * g + 7] * mul);
            const auto sx = __builtin_amdgcn_permlane32_swap(ax, bx, false, false);
            const auto sy = __builtin_amdgcn_permlane32_swap(ay, by, false, false);
            if (on) *(u32x4*)(row + 32 * t + 8 * g + 8 * hi) = u32x4{sx[0], sy[0], sx[1], sy[1]};
        }
}

// ---- which rows a block owns -------------------------------------------------------------------------------------------
// The stretches of tokens are the sequences plus what lies before the first and behind the last.  Stretch e (0 .. n + 1)
// starts at B(e) and gets block numbers from B(e) / 128 + e on: at least ceil(length / 128) of them, so the grid
// N / 128 + n + 2 is known without reading cu_seqlens, and a block finds its stretch by search.  Offsets are clamped into
// [0, N]: a bad cu_seqlens cannot lead outside the buffers.
//
// Order of the blocks above 62 sequences (find_span_even() for fewer): the blocks of a head over about one sequence are a
// group, and groups (all heads of a sequence, then the next) are dealt to the eight XCDs in turn.  A group shares its keys in one
// XCD's L2, the XCDs together read whole rows of a fused qkv buffer, and sequences of unequal length load all XCDs alike.  Within
// an XCD four groups advance together: its workgroups go to its shader engines in turn, and a group's block numbers without rows
// would otherwise fall to the same engines every time (128-token sequences: every second number; forward pass 118 -> 86 us).
constexpr int AG_BLK = 128, AG_FEW_BLK = 32;  // rows a workgroup owns
struct Order {
    int n_blk, chunk, heads, grid;       // chunk: block numbers of an average sequence
    unsigned by_chunk, by_heads;         // reciprocals, see quotient()
    float per_blk;                       // stretches per block number
    bool even, by_length;                // find_span_even()
    unsigned by_eights, by_rest;         // reciprocals of heads & ~7 and heads & 7
};
struct Span {
    int64_t s0;
    int len, first;  // rows of the stretch, first row of the block
    bool dead;       // no sequence: outputs are zeros
};
// n / d with m = floor((2^32 - 1) / d): the product is at most one short
__device__ __forceinline__ int quotient(int n, int d, unsigned m) {
    const int q = (int)__umulhi((unsigned)n, m);
    return n - q * d >= d ? q + 1 : q;
}
// Up to 62 sequences, one lane per stretch: block numbers without gaps, dealt to the XCDs one by one, where groups load them
// unequally as soon as there are few.  Measured by groups and so: one sequence of 8192, 10 heads of 64: forward pass 414 and 217
// us, backward 1310 and 622; 24 of 217 to 1031, 16 : 4 heads of 128, backward 541 and 436; 60 of 512, 18 heads of 64: 107, 345 and
// 106, 344; 10 of 2048, 16 heads of 128: 355, 1166 and 378, 1228, the most it loses.  Above 62 sequences counting costs short ones
// more than gaps do (250 of 20 to 130, backward: 140 and 147).
// In a stretch the heads go round the XCDs in eights, so that the blocks of a head share its keys in one L2 (all heads at a
// time: 60 of 512, 9 heads: 59 and 69 us), and what is left of the heads block by block.  Long sequences come in the order of
// their lengths, so that the last workgroups to start are the shortest (24 of 217 to 1031 above: nearly half of what is gained;
// below 512 tokens on average it costs more than it gives): a lane adds up the blocks of the stretches that come before its own.
constexpr int EVEN_MAX = 64, EVEN_LONG = 512;
__device__ __forceinline__ int scan64(int v) {  // sum over this lane and those before it
    auto add = [&](auto ctrl, auto rows) { v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false); };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from the lane 1, 2, 4, 8 before, in 16
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // from the 16, then the 32, before
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return v;
}
template <int BLK>
__device__ __forceinline__ bool find_span_even(const Order& od, const int* __restrict__ cu, int n, int N, int& head, Span& s) {
    const int lane = threadIdx.x & 63, b = blockIdx.x;
    auto start = [&](int i) { return i <= 0 ? 0 : i >= n + 2 ? N : min(max(cu[i - 1], 0), N); };
    auto lane_of = [](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
    const int from = start(lane), len = max(start(lane + 1) - from, 0), blocks = (len + BLK - 1) / BLK;
    const bool live = lane >= 1 && lane <= n;
    int before = 0;
    if (!od.by_length || __ballot(live && len != lane_of(len, 1)) == 0) {  // all alike: nothing to order
        before = scan64(blocks) - blocks;
    } else {
        const int key = (live ? blocks : 0) * 64 + 63 - lane;
        for (int j0 = 0; j0 < n + 2; j0 += 8)
#pragma unroll
            for (int j = j0; j < j0 + 8; ++j)  // lanes past the last stretch have no blocks
                before += lane_of(key, j) > key ? lane_of(blocks, j) : 0;
    }
    before *= od.heads;
    const unsigned long long mine = __ballot(b >= before && b < before + blocks * od.heads);
    if (mine == 0) return false;
    const int o = (int)__builtin_ctzll(mine), eights = od.heads & ~7, of_eights = lane_of(blocks, o) * eights;
    int r = b - lane_of(before, o), blk;
    if (r < of_eights) {
        blk = quotient(r, eights, od.by_eights);
        head = r - blk * eights;
    } else {
        r -= of_eights;
        blk = quotient(r, od.heads & 7, od.by_rest);
        head = eights + r - blk * (od.heads & 7);
    }
    s.s0 = lane_of(from, o);
    s.len = lane_of(len, o);
    s.first = blk * BLK;
    s.dead = o == 0 || o == n + 1;
    return true;
}
// false: no such block (uniform over the workgroup).  Everything here is on the scalar side, and for sequences of about
// equal length one read of eight offsets settles it (a vector search took 4500 cycles of a 512-token block's 40000).
template <int BLK = AG_BLK>
__device__ __forceinline__ bool find_span(const Order& od, const int* __restrict__ cu, int n, int N, int& head, Span& s) {
    if (od.even) return find_span_even<BLK>(od, cu, n, N, head, s);
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;  // blocks go to the XCDs round-robin
    const int four = at >> 2, turn = quotient(four, od.chunk, od.by_chunk), group = (turn * 4 + (at & 3)) * 8 + xcd;
    const int c = quotient(group, od.heads, od.by_heads);
    head = group - c * od.heads;
    const int b = c * od.chunk + (four - turn * od.chunk);
    if (b >= od.n_blk) return false;
    auto clamp = [&](int v) { return min(max(v, 0), N); };
    auto start = [&](int e) { return e <= 0 ? 0 : e >= n + 2 ? N : clamp(cu[e - 1]); };
    int lo = -1, a = 0, z = 0;
    if (n >= 7) {  // cu has eight entries: those around where equal lengths would put the block
        int g = (int)((float)b * od.per_blk) - 4;
        g = min(max(g, 0), n - 7);
        int v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = clamp(cu[g + i]);  // B(g + 1 + i)
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            const bool in = v[i] / BLK + g + 1 + i <= b && b < v[i + 1] / BLK + g + 2 + i;
            lo = in ? g + 1 + i : lo;
            a = in ? v[i] : a;
            z = in ? v[i + 1] : z;
        }
    }
    if (lo < 0) {  // elsewhere: halving
        lo = 0;
        int hi = n + 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (start(mid) / BLK + mid <= b) lo = mid;
            else hi = mid - 1;
        }
        a = start(lo);
        z = start(lo + 1);
    }
    s.s0 = a;
    s.len = max(z - a, 0);
    const int64_t first = (int64_t)(b - a / BLK - lo) * BLK;
    s.dead = lo == 0 || lo == n + 1;
    s.first = (int)first;
    return first < s.len;
}

// Which keys of a tile take part, one bit each; `row` is this lane's key.
__device__ __forceinline__ unsigned char mask_byte(const unsigned char* mask, int64_t s0, int row, int len) {
    return row < len ? (mask ? mask[s0 + row] : 1) : 0;
}
// Accumulator start of 32 scores from a tile's row of floats in LDS (0, or -inf where the key takes no part): masking costs
// the row reads and no vector instruction.
__device__ __forceinline__ f32x16 rows16(const float* st, int mt, int hi) {
    f32x16 r;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 a = *(const f32x4*)(st + 32 * mt + 8 * g + 4 * hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[4 * g + e] = a[e];
    }
    return r;
}
__device__ __forceinline__ bf16x8 pack8(const float* f) {
    return __builtin_bit_cast(bf16x8, u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])});
}

// The key side of the forward and dQ kernels: K and V tiles through the ring, key masks, and the loop over the tiles.
// MASK instantiations take every tile through the biased path; the others only a last tile that is not full, behind the
// loop (one path inside the loop: a second one costs a copy of the accumulators per tile).  LONE: there is one tile, and it
// goes there too.
template <int D, int KT, bool MASK, bool LONE, typename F>
__device__ __forceinline__ void for_key_tiles(const View& k, const View& v, const unsigned char* mask, const Span& sp, int kvh,
                                              char* smem, float (*bias)[KT], int wave, int lane, F tile) {
    constexpr int TILE = KT * 2 * D, SLOT = 2 * TILE;
    const __bf16* kb = k.p + sp.s0 * k.tok + kvh * k.head;
    const __bf16* vb = v.p + sp.s0 * v.tok + kvh * v.head;
    Stage<D, KT> sk, sv;
    sk.init(k.tok, wave, lane);
    sv.init(v.tok, wave, lane);
    const int nt = (sp.len + KT - 1) / KT;
    auto mask_at = [&](int t) -> unsigned char { return KT == 64 || lane < KT ? mask_byte(mask, sp.s0, t * KT + lane, sp.len) : 0; };
    auto stage = [&](int slot, int kt, unsigned long long bits) {
        char* base = smem + slot;
        const __bf16 *kp = kb + (int64_t)kt * KT * k.tok, *vp = vb + (int64_t)kt * KT * v.tok;
        if constexpr (MASK) {
            sk.go_masked(base, kp, sp.len - kt * KT, wave, lane, bits);
            sv.go_masked(base + TILE, vp, sp.len - kt * KT, wave, lane, bits);
        } else {
            sk.go(base, kp, sp.len - kt * KT, wave);
            sv.go(base + TILE, vp, sp.len - kt * KT, wave);
        }
    };
    unsigned long long bits = 0;  // of tile kt
    unsigned char mb = 0;         // of tile kt + 1
    if constexpr (MASK) {
        bits = __ballot(mask_at(0) != 0);
        mb = mask_at(1);
    }
    stage(0, 0, bits);
    const int nloop = LONE ? 0 : MASK ? nt : sp.len / KT;
    for (int kt = 0; kt < nloop; ++kt) {
        const int cur = (kt & 1) * SLOT;
        if constexpr (MASK)
            if (wave == 0 && (KT == 64 || lane < KT)) bias[kt & 1][lane] = (bits >> lane) & 1 ? 0.f : -INFINITY;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // tile kt has landed for every wave, and the other slot is read by none
        __builtin_amdgcn_sched_barrier(0);
        const unsigned long long now = bits;
        if constexpr (MASK) {
            bits = __ballot(mb != 0);
            mb = mask_at(kt + 2);
        }
        if (kt + 1 < nt) stage(SLOT - cur, kt + 1, bits);
        if constexpr (MASK)
            if (now == 0) continue;  // every wave has the same bits
        tile(std::integral_constant<bool, MASK>{}, cur, bias[kt & 1]);
    }
    if ((LONE || !MASK) && nloop < nt) {  // rows past the end landed as zeros
        const int cur = (nloop & 1) * SLOT;
        const bool in = MASK ? (bits >> lane) & 1 : nloop * KT + lane < sp.len;
        if (wave == 0 && (KT == 64 || lane < KT)) bias[0][lane] = in ? 0.f : -INFINITY;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (!MASK || bits != 0) tile(std::true_type{}, cur, bias[0]);
    }
}

// A lane's row of its block.  Where it is stored it is worked out anew, from a lane number that no register has kept (own_lane(),
// which the compiler cannot see to be the same): the loops have none to spare.
__device__ __forceinline__ int own_lane() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }
struct OwnRow {
    int64_t tok;
    bool on;
    __device__ __forceinline__ OwnRow(const Span& sp, int wave, int lane) {
        const int row = sp.first + wave * 32 + (lane & 31);
        on = row < sp.len;
        tok = sp.s0 + (on ? row : sp.len - 1);
    }
};

// ---- sequences of few keys -----------------------------------------------------------------------------------------------
// dS = P (dP - delta) sums to zero over a query's keys, so where few are averaged dq and dk are small differences, and what
// rounding leaves in dS counts.  Where at most 64 keys of a sequence take part, masked ones not counted, the backward pass
//   * takes delta + rowsum(P (dP - delta)) for delta, which is free of the rounding of out, and
//   * puts dS into its products in two bf16 parts.
// dq of 2, 4 and 16 keys (among 130 tokens) is off by 4.0e-3, 3.0e-3, 2.2e-3 of its norm without the first; of 64 keys by 2.4e-3
// without the second; with both by 1.7e-3, which is the rounding of dq alone.  Backward pass of 500 sequences of 64 tokens, 18
// heads: 215 and 226 us.  The rule looks at the sequence's own keys alone: a padded row's gradients are as exact as the packed
// sequence's, whatever else is in the call.
// Of 65 to 512 keys dq and dk are off by 2.5e-3 and 2.4e-3, and with dS in two parts by 1.8e-3.  That would cost calls of many blocks
// 14 to 18 % (backward pass, 18 heads: 160 x 200 tokens 278 and 318 us, 64 x 512 354 and 420), and costs those of few blocks 3 %
// ("few rows" below; 8 x 512, 2 heads: 31.3 and 32.3), which have it.
constexpr int AG_FEW_KEYS = 64, AG_SOME_KEYS = 512;

// The keys of a sequence that take part, or any number above `most` if there are more.  Masked sequences count 512 at a time, so that
// all but very sparse masks cost one read (64 x 512 tokens with a mask, backward pass: 359 and 365 us).
__device__ __forceinline__ int live_keys(const unsigned char* mask, const Span& sp, int lane, int most) {
    if (!mask || sp.len <= AG_FEW_KEYS) return sp.len;  // of 64 tokens no more than that
    int n = 0;
    for (int r0 = 0; r0 < sp.len && n <= most; r0 += 512) {
        unsigned char m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = mask_byte(mask, sp.s0, r0 + 64 * i + lane, sp.len);
#pragma unroll
        for (int i = 0; i < 8; ++i) n += __popcll(__ballot(m[i] != 0));
    }
    return n;
}
__device__ __forceinline__ bool few_keys(const unsigned char* mask, const Span& sp, int lane) {
    return live_keys(mask, sp, lane, AG_FEW_KEYS) <= AG_FEW_KEYS;
}

// What the rounding of f to `a` leaves, rounded again: f is off by 2^-17 relative at most in the two parts together.
struct Rest { bf16x8 b[2]; };
__device__ __forceinline__ Rest rest_of(const float (&f)[16], const bf16x8 (&a)[2]) {
    float r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = f[i] - (float)a[i >> 3][i & 7];
    return Rest{{pack8(r), pack8(r + 8)}};
}
// acc += X^T . f, f in two parts, both formed before either product and one product at a time: the kernels that call this have
// no registers to spare.
template <int D, int MT>
__device__ __forceinline__ void mfma_tr_two(f32x16 (&acc)[D / 32], const TrAddr<D>& ta, unsigned tile, const float (&f)[16]) {
    __builtin_amdgcn_sched_barrier(0);
    const bf16x8 a[2] = {pack8(f), pack8(f + 8)};
    const Rest rest = rest_of(f, a);
    __builtin_amdgcn_sched_barrier(0);
    mfma_tr<D, MT>(acc, ta, tile, a);
    mfma_tr<D, MT>(acc, ta, tile, rest.b);
    __builtin_amdgcn_sched_barrier(0);
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// Key tiles of 64 rows at head dim 64 (32: 10 % slower, twice the barriers), of 32 at 128: half the score registers and LDS
// make room for a third wave per SIMD (64 x 512, 9 heads of 128: 124 -> 109 us; 24 ragged, 16 heads, masked: 172 -> 163 us).
template <int D, bool MASK>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? (MASK ? 3 : 4) : 3) void attn_fwd_lse_kernel(View q, View k, View v, OutView o,
                                                                     float* __restrict__ lse, const int* __restrict__ cu,
                                                                     int n_seg, const unsigned char* __restrict__ mask,
                                                                     int N, int group, Order od, float c) {
    constexpr int KT = D == 64 ? 64 : 32, MT = KT / 32, TILE = KT * 2 * D;
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];
    __shared__ __attribute__((aligned(16))) float bias[2][KT];
    const int lane = threadIdx.x & 63, l31 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int head;
    Span sp;
    if (!find_span(od, cu, n_seg, N, head, sp)) return;
    f32x16 acc[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] = splat16(0.f);
    // The row's place is worked out again where it is stored (the compiler cannot see that it is the same): kept, it is what
    // the loop has no registers for, and 28 bytes a lane went to memory and back (131 -> 122 us at 64 x 512).
    auto finish = [&](float mul, float stat) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int row = sp.first + wave * 32 + (tid & 31), h = (tid >> 5) & 1;
        const bool on = row < sp.len;
        const int64_t tok = sp.s0 + (on ? row : sp.len - 1);
        store_row<D>(o.p + tok * o.tok + head * o.head, acc, mul, h, on);
        if (on && h == 0) lse[(int64_t)head * N + tok] = stat;
    };
    if (sp.dead) {
        finish(0.f, -INFINITY);
        return;
    }
    bf16x8 qf[D / 16];
    {
        const int64_t tok = sp.s0 + min(sp.first + wave * 32 + l31, sp.len - 1);
        const __bf16* qp = q.p + tok * q.tok + head * q.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const bf16x8*)(qp + ks * 16);
    }
    const int koff = row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem);
    // p = exp2(c s - mc).  Any reference mc gives the same quotient, so it follows the row maximum only where it has to: it
    // is taken from the first tile with keys, and again when a tile's sum passes 2^16 (fp32 sums and bf16 probabilities have
    // the range).  That spares the maximum over every tile (1136 -> 933 us at 4 x 4096 with the masks' own kernels).
    float mc = 0.f, l = 0.f;
    bool fresh = true;  // no reference yet
    for_key_tiles<D, KT, MASK, false>(k, v, mask, sp, head / group, smem, bias, wave, lane, [&](auto biased, int cur, const float* st) {
        constexpr bool BIASED = decltype(biased)::value;
        f32x16 s[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt] = mfma_rows<D>(smem + cur + mt * 64 * D, koff, qf, BIASED ? rows16(st, mt, hi) : splat16(0.f));
        bf16x8 p[MT][2];
        float ps;
        auto probabilities = [&] {
            ps = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float e[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    e[r] = __builtin_amdgcn_exp2f(fmaf(s[mt][r], c, -mc));
                    ps += e[r];
                }
                // 2^-8 relative at most, in the product with V only; the row sum keeps fp32
                p[mt][0] = pack8(e);
                p[mt][1] = pack8(e + 8);
            }
        };
        auto largest = [&] {
            float mx = s[0][0];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
            mx = half_max(mx) * c;
            return mx == -INFINITY ? 0.f : mx;
        };
        if (fresh) {  // a tile with keys has them for every row
            mc = largest();
            fresh = false;
        }
        probabilities();
        if (__builtin_expect(__any(!(ps <= 65536.f)), 0)) {
            const float mn = fmaxf(mc, largest());
            const float a = __builtin_amdgcn_exp2f(mc - mn);
            mc = mn;
            l *= a;
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[t][r] *= a;
            probabilities();
        }
        l += ps;
        mfma_tr<D, 0>(acc, ta, lds0 + cur + TILE, p[0]);
        if constexpr (MT == 2) mfma_tr<D, 1>(acc, ta, lds0 + cur + TILE, p[1]);
    });
    l = half_sum(l);
    // no key: zeros; NaN stays
    finish(l > 0.f ? 1.0f / l : l, l == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * AG_LN2);
}

// ---- backward: dQ and delta --------------------------------------------------------------------------------------------
// A block's rows, for sequences of many keys, of few in one tile, and of few among masked ones in several tiles: the three share
// no registers, so that none spills for another.
enum Keys { MANY, FEW_ONE_TILE, FEW_SCATTERED };
template <int D, bool MASK, Keys KEYS>
__device__ __forceinline__ void dq_rows(const View& dout, const View& q, const View& k, const View& v, const View& o,
                                        const float* __restrict__ lse, float* __restrict__ delta, const OutView& dq,
                                        const unsigned char* __restrict__ mask, int N, int group, float scale, int head,
                                        const Span& sp, char* smem, float (*bias)[TR], int wave, int lane) {
    constexpr int TILE = TR * 2 * D;
    const int l31 = lane & 31, hi = lane >> 5;
    bf16x8 qf[D / 16], gf[D / 16];
    float dl = 0.f, nl;
    {
        const int64_t tok = OwnRow(sp, wave, lane).tok;
        nl = -lse[(int64_t)head * N + tok] * AG_LOG2E;  // +inf only where every tile is skipped
        const __bf16* qp = q.p + tok * q.tok + head * q.head + hi * 8;
        const __bf16* gp = dout.p + tok * dout.tok + head * dout.head + hi * 8;
        const __bf16* xp = o.p + tok * o.tok + head * o.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            qf[ks] = *(const bf16x8*)(qp + ks * 16);
            gf[ks] = *(const bf16x8*)(gp + ks * 16);
            const bf16x8 xf = *(const bf16x8*)(xp + ks * 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) dl += (float)gf[ks][j] * (float)xf[j];
        }
    }
    dl = half_sum(dl);
    const float c = scale * AG_LOG2E;
    const int koff = row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem);
    f32x16 nd = splat16(-dl);  // dP starts from -delta

    f32x16 acc[D / 32];
    auto clear = [&] {
#pragma unroll
        for (int t = 0; t < D / 32; ++t) acc[t] = splat16(0.f);
    };
    auto half = [&](auto mt_, auto biased, int cur, const float* st) {
        constexpr int mt = decltype(mt_)::value;
        const f32x16 s = mfma_rows<D>(smem + cur + mt * 64 * D, koff, qf, decltype(biased)::value ? rows16(st, mt, hi) : splat16(0.f));
        const f32x16 dp = mfma_rows<D>(smem + cur + TILE + mt * 64 * D, koff, gf, nd);
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, nl)) * dp[r];
        if constexpr (KEYS != MANY) {
            mfma_tr_two<D, mt>(acc, ta, lds0 + cur, e);
        } else {
            const bf16x8 ds[2] = {pack8(e), pack8(e + 8)};  // 2^-8 relative at most, for the product with K
            mfma_tr<D, mt>(acc, ta, lds0 + cur, ds);
        }
    };
    auto both = [&](auto biased, int cur, const float* st) {
        half(std::integral_constant<int, 0>{}, biased, cur, st);
        half(std::integral_constant<int, 1>{}, biased, cur, st);
    };
    auto more = [&](int cur, const float* st) {  // this lane's part of rowsum(P (dP - delta)) over a tile
        float m = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const f32x16 s = mfma_rows<D>(smem + cur + mt * 64 * D, koff, qf, rows16(st, mt, hi));
            const f32x16 dp = mfma_rows<D>(smem + cur + TILE + mt * 64 * D, koff, gf, nd);
#pragma unroll
            for (int r = 0; r < 16; ++r) m += __builtin_amdgcn_exp2f(fmaf(s[r], c, nl)) * dp[r];
        }
        return m;
    };
    auto tiles = [&](auto lone, auto tile) {
        for_key_tiles<D, TR, MASK, decltype(lone)::value>(k, v, mask, sp, head / group, smem, bias, wave, lane, tile);
    };
    clear();
    if constexpr (KEYS == MANY) {
        tiles(std::false_type{}, [&](auto biased, int cur, const float* st) { both(biased, cur, st); });
    } else if constexpr (KEYS == FEW_ONE_TILE) {
        tiles(std::true_type{}, [&](auto biased, int cur, const float* st) {
            nd = splat16(nd[0] - half_sum(more(cur, st)));
            both(biased, cur, st);
        });
    } else {  // delta from a pass of its own
        float m = 0.f;
        tiles(std::false_type{}, [&](auto, int cur, const float* st) { m += more(cur, st); });
        nd = splat16(nd[0] - half_sum(m));
        __syncthreads();  // the ring and the biases have been read
        clear();
        tiles(std::false_type{}, [&](auto biased, int cur, const float* st) { both(biased, cur, st); });
    }
    const int at = own_lane();
    const OwnRow r(sp, wave, at);
    if (r.on && at < 32) delta[(int64_t)head * N + r.tok] = -nd[0];
    store_row<D>(dq.p + r.tok * dq.tok + head * dq.head, acc, scale, at >> 5, r.on);
}

template <int D, bool MASK>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? 3 : 2) void attn_bwd_dq_kernel(View dout, View q, View k, View v, View o,
                                                                    const float* __restrict__ lse,
                                                                    float* __restrict__ delta, OutView dq,
                                                                    const int* __restrict__ cu, int n_seg,
                                                                    const unsigned char* __restrict__ mask, int N,
                                                                    int group, Order od, float scale) {
    constexpr int TILE = TR * 2 * D;
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];
    __shared__ __attribute__((aligned(16))) float bias[2][TR];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int head;
    Span sp;
    if (!find_span(od, cu, n_seg, N, head, sp)) return;
    if (sp.dead) {
        const OwnRow r(sp, wave, lane);
        f32x16 z[D / 32];
#pragma unroll
        for (int t = 0; t < D / 32; ++t) z[t] = splat16(0.f);
        store_row<D>(dq.p + r.tok * dq.tok + head * dq.head, z, 0.f, lane >> 5, r.on);
        return;
    }
    auto rows = [&](auto keys) {
        dq_rows<D, MASK, decltype(keys)::value>(dout, q, k, v, o, lse, delta, dq, mask, N, group, scale, head, sp, smem, bias, wave, lane);
    };
    if (sp.len <= TR) return rows(std::integral_constant<Keys, FEW_ONE_TILE>{});
    if constexpr (MASK)
        if (few_keys(mask, sp, lane)) return rows(std::integral_constant<Keys, FEW_SCATTERED>{});
    rows(std::integral_constant<Keys, MANY>{});
}

// ---- backward: dK and dV -----------------------------------------------------------------------------------------------
// At head dim 128 the accumulators take 128 registers and K's fragments 32; V's would leave one wave per SIMD, so they are
// read from LDS where they are used (LDS reads run at 256 bytes a cycle, a third of the time unused), and the ring holds
// 32-row tiles: 64 KiB a workgroup, two of them on a CU.
// Both head dims run at their register limit.  The loops over full tiles use no scratch: the lane's row is worked out again at the
// store, and the path of few keys is a body of its own that forms one product at a time (with 24 spilled registers in its loop, 500 x
// 64 tokens, 18 heads took 365 us, backward pass, instead of 226).  Head dim 64 keeps 24 bytes a lane in it around the loops.
constexpr int dkdv_rt(int D) { return D == 128 ? 32 : 64; }  // rows of a streamed tile

template <int D, bool FEW>
__device__ __forceinline__ void dkdv_rows(const View& dout, const View& q, const View& k, const View& v,
                                          const float* __restrict__ lse, const float* __restrict__ delta, const OutView& dk,
                                          const OutView& dv, int N, int group, float scale, int kvh, const Span& sp, bool live,
                                          char* smem, float (*stat)[2][dkdv_rt(D)], int wave, int lane) {
    constexpr bool VL = D == 128;
    constexpr int RT = dkdv_rt(D), TILE = RT * 2 * D, SLOT = 2 * TILE;
    const int l31 = lane & 31, hi = lane >> 5;
    f32x16 ak[D / 32], av[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) ak[t] = av[t] = splat16(0.f);
    // A key that takes no part has its own lane: its column is computed, from zero rows where its fragments are registers,
    // and not used.
    bf16x8 kf[D / 16], vf[VL ? 1 : D / 16];
    {
        const int64_t tok = OwnRow(sp, wave, lane).tok;
        const __bf16* kp = k.p + tok * k.tok + kvh * k.head + hi * 8;
        const __bf16* vp = v.p + tok * v.tok + kvh * v.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            u32x4 a = u32x4{0u, 0u, 0u, 0u}, b = a;
            if (live) {
                a = *(const u32x4*)(kp + ks * 16);
                if constexpr (!VL) b = *(const u32x4*)(vp + ks * 16);
            }
            kf[ks] = __builtin_bit_cast(bf16x8, a);
            if constexpr (!VL) vf[ks] = __builtin_bit_cast(bf16x8, b);
        }
    }
    if constexpr (VL) {  // the wave's own 32 rows, so that nothing but its own loads has to be waited for
        const int r0 = sp.first + wave * 32, rows = sp.len - r0;
        if (rows > 0) {
            const __bf16* vb = v.p + (sp.s0 + r0) * v.tok + kvh * v.head;
            const int nrec = (int)((rows < 32 ? rows - 1 : 31) * (unsigned)(v.tok * 2) + 2 * D);
            const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)vb, 0, nrec, 0x00020000);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + lane / 16;
                const unsigned off = (unsigned)r * (unsigned)(v.tok * 2) + (unsigned)((lane & 15) ^ swz<D>(r)) * 16u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(d, LDS_PTR(smem + 2 * SLOT + wave * 32 * 2 * D + i * 1024), 16, (int)off, 0, 0, 0);
            }
        }
    }
    Stage<D, RT> sq, sg;
    sq.init(q.tok, wave, lane);
    sg.init(dout.tok, wave, lane);
    const int nt = (sp.len + RT - 1) / RT;  // query tiles per head of the group
    const int total = nt * group;
    const float inv_scale = 1.0f / scale;
    float next = 0.f;
    int gq = 0, qt = 0;  // head of the group and tile that stage() takes next
    // of rows past the end; a scalar: kept per lane it was read from scratch in the loop at D 128, and waiting for that waits for the
    // tile in flight too (8 x 2048 tokens, 16 heads, backward pass 980 -> 1050 us)
    const int none = __builtin_amdgcn_readfirstlane(wave ? 0 : 0x7f800000);
    auto stage = [&](int slot) {
        const int left = sp.len - qt * RT, head = kvh * group + gq;
        const int64_t t0 = sp.s0 + (int64_t)qt * RT;
        char* base = smem + slot;
        sq.go(base, q.p + t0 * q.tok + head * q.head, left, wave);
        sg.go(base + TILE, dout.p + t0 * dout.tok + head * dout.head, left, wave);
        if (wave < 2) {  // wave 0: lse, wave 1: delta.  Rows past the end get probability 2^-inf = 0
            const float* src = (wave ? delta : lse) + (int64_t)head * N + t0;
            const float x = lane < left && lane < RT ? src[lane] : __int_as_float(none);
            next = wave ? -x : -x * inv_scale;
        }
        if (++qt == nt) { qt = 0; ++gq; }
    };
    stage(0);
    const int koff = row_off<D>(l31, hi);
    const int voff = 2 * SLOT + wave * 32 * 2 * D + row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(smem);
    const float c = scale * AG_LOG2E;

    auto dp_of = [&](auto mt_, int cur, const float* st) {  // dO V^T - delta
        constexpr int mt = decltype(mt_)::value;
        f32x16 dp = rows16(st + RT, mt, hi);
        if constexpr (VL) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(smem + cur + TILE + mt * 64 * D + (koff ^ (ks << 5))),
                                                             *(const bf16x8*)(smem + (voff ^ (ks << 5))), dp, 0, 0, 0);
        } else {
            dp = mfma_rows<D>(smem + cur + TILE + mt * 64 * D, koff, vf, dp);
        }
        return dp;
    };
    auto half = [&](auto mt_, int cur, const float* st) {
        constexpr int mt = decltype(mt_)::value;
        const f32x16 s = mfma_rows<D>(smem + cur + mt * 64 * D, koff, kf, rows16(st, mt, hi));  // Q K^T - lse / scale
        float e[16], f[16];
        if constexpr (FEW) {  // one product at a time: registers
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(s[r] * c);
            const bf16x8 p[2] = {pack8(e), pack8(e + 8)};  // 2^-8 relative at most, for the product with dO
            __builtin_amdgcn_sched_barrier(0);
            mfma_tr<D, mt>(av, ta, lds0 + cur + TILE, p);
            __builtin_amdgcn_sched_barrier(0);
            const f32x16 dp = dp_of(mt_, cur, st);
#pragma unroll
            for (int r = 0; r < 16; ++r) f[r] = e[r] * dp[r];
            mfma_tr_two<D, mt>(ak, ta, lds0 + cur, f);
        } else {
            const f32x16 dp = dp_of(mt_, cur, st);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                e[r] = __builtin_amdgcn_exp2f(s[r] * c);
                f[r] = e[r] * dp[r];
            }
            // 2^-8 relative at most, for the products with dO and Q
            const bf16x8 p[2] = {pack8(e), pack8(e + 8)}, ds[2] = {pack8(f), pack8(f + 8)};
            mfma_tr<D, mt>(av, ta, lds0 + cur + TILE, p);
            mfma_tr<D, mt>(ak, ta, lds0 + cur, ds);
        }
    };
    for (int i = 0; i < total; ++i) {
        const int cur = (i & 1) * SLOT;
        if (wave < 2 && lane < RT) stat[i & 1][wave][lane] = next;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < total) stage(SLOT - cur);
        half(std::integral_constant<int, 0>{}, cur, &stat[i & 1][0][0]);
        if constexpr (RT == 64) half(std::integral_constant<int, 1>{}, cur, &stat[i & 1][0][0]);
    }
    if (!live) {
#pragma unroll
        for (int t = 0; t < D / 32; ++t) ak[t] = av[t] = splat16(0.f);
    }
    const int at = own_lane();
    const OwnRow r(sp, wave, at);
    store_row<D>(dk.p + r.tok * dk.tok + kvh * dk.head, ak, scale, at >> 5, r.on);
    store_row<D>(dv.p + r.tok * dv.tok + kvh * dv.head, av, 1.f, at >> 5, r.on);
}

template <int D>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? 3 : 2) void attn_bwd_dkdv_kernel(View dout, View q, View k, View v,
                                                                      const float* __restrict__ lse,
                                                                      const float* __restrict__ delta, OutView dk,
                                                                      OutView dv, const int* __restrict__ cu, int n_seg,
                                                                      const unsigned char* __restrict__ mask, int N,
                                                                      int group, Order od, float scale) {
    constexpr int RT = dkdv_rt(D);
    __shared__ __attribute__((aligned(1024))) char smem[4 * RT * 2 * D + (D == 128 ? AG_BLK * 2 * D : 0)];
    __shared__ __attribute__((aligned(16))) float stat[2][2][RT];  // slot, (-lse / scale, -delta), row of the tile
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kvh;
    Span sp;
    if (!find_span(od, cu, n_seg, N, kvh, sp)) return;
    const OwnRow r(sp, wave, lane);
    const bool live = r.on && !sp.dead && (!mask || mask[r.tok]);
    const int keys = __syncthreads_count(live) / 2;  // two lanes a row
    if (keys == 0) {  // no key of the block takes part
        f32x16 z[D / 32];
#pragma unroll
        for (int t = 0; t < D / 32; ++t) z[t] = splat16(0.f);
        store_row<D>(dk.p + r.tok * dk.tok + kvh * dk.head, z, 0.f, lane >> 5, r.on);
        store_row<D>(dv.p + r.tok * dv.tok + kvh * dv.head, z, 0.f, lane >> 5, r.on);
        return;
    }
    if (keys <= AG_FEW_KEYS && few_keys(mask, sp, lane)) dkdv_rows<D, true>(dout, q, k, v, lse, delta, dk, dv, N, group, scale, kvh, sp, live, smem, stat, wave, lane);
    else dkdv_rows<D, false>(dout, q, k, v, lse, delta, dk, dv, N, group, scale, kvh, sp, live, smem, stat, wave, lane);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------
// Where the blocks of 128 rows do not fill the card, a workgroup owns 32 rows and its four waves take every fourth tile of the
// other side, each through a ring of its own and without a barrier; at the end their sums are joined in LDS, in the order of
// the waves.  Four times the workgroups, each a quarter as long; four times the tile loads.  One path for all masks.
// Forward and backward pass, blocks of 128 rows and this (us): one sequence of 4096, 4 heads of 64: 59, 169 and 40, 92; 3 of 2652, 4 : 1
// heads of 128, where only dK dV is short of blocks: backward pass 582 and 248.  ag_few() has the bounds and what was measured
// around them.

// Sum of the four waves' accumulators [column 32 t + crow(r, hi)][row on the lane], each times its `mul`, written as bf16 rows.
// All waves have to be done with `area`.
template <int D>
__device__ __forceinline__ void join_rows(float* area, const f32x16 (&acc)[D / 32], float mul, int wave, int lane, __bf16* p,
                                          int64_t tok, int rows) {
    float* mine = area + (wave * 32 + (lane & 31)) * (D + 4) + 4 * (lane >> 5);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(f32x4*)(mine + 32 * t + 8 * g) = f32x4{acc[t][4 * g] * mul, acc[t][4 * g + 1] * mul, acc[t][4 * g + 2] * mul, acc[t][4 * g + 3] * mul};
    __syncthreads();
    const int row = threadIdx.x >> 3, col = (threadIdx.x & 7) * (D / 8);
#pragma unroll
    for (int j = 0; j < D / 8; j += 8) {
        f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
        for (int w = 0; w < AG_WAVES; ++w) {
            const float* src = area + (w * 32 + row) * (D + 4) + col + j;
            a += *(const f32x4*)src;
            b += *(const f32x4*)(src + 4);
        }
        if (row < rows)
            *(u32x4*)(p + row * tok + col + j) = u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
    }
}

// Tiles wave, wave + 4, ... of 32 keys, through the wave's own ring (2 slots of K and V).
template <int D, typename F>
__device__ __forceinline__ void for_own_tiles(const View& k, const View& v, const unsigned char* mask, const Span& sp, int kvh,
                                              char* ring, float (*bias)[32], int wave, int lane, F tile) {
    constexpr int TILE = 32 * 2 * D, SLOT = 2 * TILE;
    const __bf16* kb = k.p + sp.s0 * k.tok + kvh * k.head;
    const __bf16* vb = v.p + sp.s0 * v.tok + kvh * v.head;
    Stage<D, 32, 1> sk, sv;
    sk.init(k.tok, 0, lane);
    sv.init(v.tok, 0, lane);
    const int nt = (sp.len + 31) / 32;
    auto mask_at = [&](int t) -> unsigned char { return lane < 32 ? mask_byte(mask, sp.s0, t * 32 + lane, sp.len) : 0; };
    auto stage = [&](int slot, int kt, unsigned long long bits) {
        sk.go_masked(ring + slot, kb + (int64_t)kt * 32 * k.tok, sp.len - kt * 32, 0, lane, bits);
        sv.go_masked(ring + slot + TILE, vb + (int64_t)kt * 32 * v.tok, sp.len - kt * 32, 0, lane, bits);
    };
    if (wave >= nt) return;
    unsigned long long bits = __ballot(mask_at(wave) != 0);  // of tile kt
    unsigned char mb = mask_at(wave + AG_WAVES);             // of tile kt + 4
    stage(0, wave, bits);
    for (int kt = wave, i = 0; kt < nt; kt += AG_WAVES, i ^= 1) {
        const int cur = i * SLOT;
        if (lane < 32) bias[i][lane] = (bits >> lane) & 1 ? 0.f : -INFINITY;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the tile has landed, the other slot has been read
        __builtin_amdgcn_sched_barrier(0);
        const unsigned long long now = bits;
        bits = __ballot(mb != 0);
        mb = mask_at(kt + 2 * AG_WAVES);
        if (kt + AG_WAVES < nt) stage(SLOT - cur, kt + AG_WAVES, bits);
        if (now != 0) tile(cur, bias[i]);
    }
}

template <int D>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? 2 : 1) void attn_fwd_few_kernel(View q, View k, View v, OutView o,
                                                                                      float* __restrict__ lse, const int* __restrict__ cu,
                                                                                      int n_seg, const unsigned char* __restrict__ mask,
                                                                                      int N, int group, Order od, float c) {
    constexpr int TILE = 32 * 2 * D, RING = 4 * TILE;
    __shared__ __attribute__((aligned(1024))) char smem[AG_WAVES * RING];
    __shared__ __attribute__((aligned(16))) float bias[AG_WAVES][2][32];
    __shared__ float part[AG_WAVES][2][32];  // reference and sum of each wave's rows
    const int lane = threadIdx.x & 63, l31 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int head;
    Span sp;
    if (!find_span<AG_FEW_BLK>(od, cu, n_seg, N, head, sp)) return;
    const int row = sp.first + l31;
    const bool on = row < sp.len;
    const int64_t tok = sp.s0 + (on ? row : sp.len - 1);
    f32x16 acc[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] = splat16(0.f);
    if (sp.dead) {
        if (wave == 0) {
            store_row<D>(o.p + tok * o.tok + head * o.head, acc, 0.f, hi, on);
            if (on && hi == 0) lse[(int64_t)head * N + tok] = -INFINITY;
        }
        return;
    }
    bf16x8 qf[D / 16];
    {
        const __bf16* qp = q.p + tok * q.tok + head * q.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const bf16x8*)(qp + ks * 16);
    }
    const int koff = row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    char* ring = smem + wave * RING;
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(ring);
    float mc = 0.f, l = 0.f;
    bool fresh = true;
    for_own_tiles<D>(k, v, mask, sp, head / group, ring, bias[wave], wave, lane, [&](int cur, const float* st) {
        const f32x16 s = mfma_rows<D>(ring + cur, koff, qf, rows16(st, 0, hi));
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = half_max(mx) * c;
        // the reference as in the large kernel: from the first tile with keys, and again past 2^16
        if (fresh || __any(!(mx <= mc + 16.f))) {
            const float mn = fresh ? (mx == -INFINITY ? 0.f : mx) : fmaxf(mc, mx);
            const float a = fresh ? 0.f : __builtin_amdgcn_exp2f(mc - mn);
            mc = mn;
            fresh = false;
            l *= a;
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[t][r] *= a;
        }
        float e[16], ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mc));
            ps += e[r];
        }
        l += ps;
        const bf16x8 p[2] = {pack8(e), pack8(e + 8)};  // 2^-8 relative at most, in the product with V only
        mfma_tr<D, 0>(acc, ta, lds0 + cur + TILE, p);
    });
    l = half_sum(l);
    if (hi == 0) {
        part[wave][0][l31] = mc;
        part[wave][1][l31] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < AG_WAVES; ++w) top = fmaxf(top, part[w][1][l31] == 0.f ? -INFINITY : part[w][0][l31]);
#pragma unroll
    for (int w = 0; w < AG_WAVES; ++w) sum += part[w][1][l31] == 0.f ? 0.f : part[w][1][l31] * __builtin_amdgcn_exp2f(part[w][0][l31] - top);
    const float own = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(mc - top);
    if (wave == 0 && on && hi == 0) lse[(int64_t)head * N + tok] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * AG_LN2;
    join_rows<D>((float*)smem, acc, sum > 0.f ? own / sum : sum, wave, lane, o.p + (sp.s0 + sp.first) * o.tok + head * o.head, o.tok,
                 sp.len - sp.first);
}

template <int D>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? 2 : 1) void attn_bwd_dq_few_kernel(View dout, View q, View k, View v, View o,
                                                                        const float* __restrict__ lse,
                                                                        float* __restrict__ delta, OutView dq,
                                                                        const int* __restrict__ cu, int n_seg,
                                                                        const unsigned char* __restrict__ mask, int N,
                                                                        int group, Order od, float scale) {
    constexpr int TILE = 32 * 2 * D, RING = 4 * TILE;
    __shared__ __attribute__((aligned(1024))) char smem[AG_WAVES * RING];
    __shared__ __attribute__((aligned(16))) float bias[AG_WAVES][2][32];
    __shared__ float part[AG_WAVES][32];
    const int lane = threadIdx.x & 63, l31 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int head;
    Span sp;
    if (!find_span<AG_FEW_BLK>(od, cu, n_seg, N, head, sp)) return;
    const int row = sp.first + l31;
    const bool on = row < sp.len;
    const int64_t tok = sp.s0 + (on ? row : sp.len - 1);
    f32x16 acc[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] = splat16(0.f);
    if (sp.dead) {
        if (wave == 0) store_row<D>(dq.p + tok * dq.tok + head * dq.head, acc, 0.f, hi, on);
        return;
    }
    bf16x8 qf[D / 16], gf[D / 16];
    float dl = 0.f;
    {
        const __bf16* qp = q.p + tok * q.tok + head * q.head + hi * 8;
        const __bf16* gp = dout.p + tok * dout.tok + head * dout.head + hi * 8;
        const __bf16* xp = o.p + tok * o.tok + head * o.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            qf[ks] = *(const bf16x8*)(qp + ks * 16);
            gf[ks] = *(const bf16x8*)(gp + ks * 16);
            const bf16x8 xf = *(const bf16x8*)(xp + ks * 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) dl += (float)gf[ks][j] * (float)xf[j];
        }
    }
    f32x16 nd = splat16(-half_sum(dl));
    const float c = scale * AG_LOG2E;
    const float nl = -lse[(int64_t)head * N + tok] * AG_LOG2E;
    const int koff = row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    char* ring = smem + wave * RING;
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(ring);
    float e[16];  // P (dP - delta) of a tile
    auto products = [&](int cur, const float* st) {
        const f32x16 s = mfma_rows<D>(ring + cur, koff, qf, rows16(st, 0, hi));
        const f32x16 dp = mfma_rows<D>(ring + cur + TILE, koff, gf, nd);
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, nl)) * dp[r];
    };
    const int keys = live_keys(mask, sp, lane, AG_SOME_KEYS);
    if (keys <= AG_FEW_KEYS) {  // delta without the rounding of out, as in the large kernel
        float more = 0.f;
        for_own_tiles<D>(k, v, mask, sp, head / group, ring, bias[wave], wave, lane, [&](int cur, const float* st) {
            products(cur, st);
#pragma unroll
            for (int r = 0; r < 16; ++r) more += e[r];
        });
        more = half_sum(more);
        if (hi == 0) part[wave][l31] = more;
        __syncthreads();
        more = 0.f;
#pragma unroll
        for (int w = 0; w < AG_WAVES; ++w) more += part[w][l31];
        nd = splat16(nd[0] - more);
    }
    if (wave == 0 && on && hi == 0) delta[(int64_t)head * N + tok] = -nd[0];
    for_own_tiles<D>(k, v, mask, sp, head / group, ring, bias[wave], wave, lane, [&](int cur, const float* st) {
        products(cur, st);
        const bf16x8 ds[2] = {pack8(e), pack8(e + 8)};  // 2^-8 relative at most, for the product with K
        mfma_tr<D, 0>(acc, ta, lds0 + cur, ds);
        if (keys <= AG_SOME_KEYS) mfma_tr<D, 0>(acc, ta, lds0 + cur, rest_of(e, ds).b);
    });
    __syncthreads();
    join_rows<D>((float*)smem, acc, scale, wave, lane, dq.p + (sp.s0 + sp.first) * dq.tok + head * dq.head, dq.tok, sp.len - sp.first);
}

template <int D>
__global__ __launch_bounds__(AG_WAVES * 64, D == 64 ? 2 : 1) void attn_bwd_dkdv_few_kernel(View dout, View q, View k, View v,
                                                                      const float* __restrict__ lse,
                                                                      const float* __restrict__ delta, OutView dk,
                                                                      OutView dv, const int* __restrict__ cu, int n_seg,
                                                                      const unsigned char* __restrict__ mask, int N,
                                                                      int group, Order od, float scale) {
    constexpr int TILE = 32 * 2 * D, SLOT = 2 * TILE, RING = 2 * SLOT;
    __shared__ __attribute__((aligned(1024))) char smem[AG_WAVES * RING];
    __shared__ __attribute__((aligned(16))) float stat[AG_WAVES][2][2][32];  // slot, (-lse / scale, -delta), row of the tile
    const int lane = threadIdx.x & 63, l31 = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int kvh;
    Span sp;
    if (!find_span<AG_FEW_BLK>(od, cu, n_seg, N, kvh, sp)) return;
    const int row = sp.first + l31;
    const bool on = row < sp.len;
    const int64_t tok = sp.s0 + (on ? row : sp.len - 1);
    f32x16 ak[D / 32], av[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t) ak[t] = av[t] = splat16(0.f);
    const bool live = on && !sp.dead && (!mask || mask[tok]);
    if (!__any(live)) {  // no key of the block takes part; every wave has the same rows
        if (wave == 0) {
            store_row<D>(dk.p + tok * dk.tok + kvh * dk.head, ak, 0.f, hi, on);
            store_row<D>(dv.p + tok * dv.tok + kvh * dv.head, av, 0.f, hi, on);
        }
        return;
    }
    bf16x8 kf[D / 16], vf[D / 16];  // zero rows for keys that take no part: their columns are computed and not used
    {
        const __bf16* kp = k.p + tok * k.tok + kvh * k.head + hi * 8;
        const __bf16* vp = v.p + tok * v.tok + kvh * v.head + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            u32x4 a = u32x4{0u, 0u, 0u, 0u}, b = a;
            if (live) {
                a = *(const u32x4*)(kp + ks * 16);
                b = *(const u32x4*)(vp + ks * 16);
            }
            kf[ks] = __builtin_bit_cast(bf16x8, a);
            vf[ks] = __builtin_bit_cast(bf16x8, b);
        }
    }
    Stage<D, 32, 1> sq, sg;
    sq.init(q.tok, 0, lane);
    sg.init(dout.tok, 0, lane);
    const int nt = (sp.len + 31) / 32;  // query tiles per head of the group
    const int total = nt * group;
    const float inv_scale = 1.0f / scale;
    char* ring = smem + wave * RING;
    float next = 0.f;
    int gq = 0, qt = wave;  // head of the group and tile that stage() takes next
    auto stage = [&](int slot) {
        for (; qt >= nt; qt -= nt) ++gq;
        const int left = sp.len - qt * 32, head = kvh * group + gq;
        const int64_t t0 = sp.s0 + (int64_t)qt * 32;
        sq.go(ring + slot, q.p + t0 * q.tok + head * q.head, left, 0);
        sg.go(ring + slot + TILE, dout.p + t0 * dout.tok + head * dout.head, left, 0);
        // lanes 0 .. 31: lse, 32 .. 63: delta.  Rows past the end get probability 2^-inf = 0
        const float* src = (hi ? delta : lse) + (int64_t)head * N + t0;
        const float x = l31 < left ? src[l31] : hi ? 0.f : INFINITY;
        next = hi ? -x : -x * inv_scale;
        qt += AG_WAVES;
    };
    const int koff = row_off<D>(l31, hi);
    TrAddr<D> ta;
    ta.init(lane);
    const unsigned lds0 = (unsigned)(size_t)LDS_PTR(ring);
    const float c = scale * AG_LOG2E;
    if (wave < total) stage(0);
    const bool some = live_keys(mask, sp, lane, AG_SOME_KEYS) <= AG_SOME_KEYS;
    for (int i = wave, j = 0; i < total; i += AG_WAVES, j ^= 1) {
        const int cur = j * SLOT;
        stat[wave][j][hi][l31] = next;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (i + AG_WAVES < total) stage(SLOT - cur);
        const f32x16 s = mfma_rows<D>(ring + cur, koff, kf, rows16(stat[wave][j][0], 0, hi));         // Q K^T - lse / scale
        const f32x16 dp = mfma_rows<D>(ring + cur + TILE, koff, vf, rows16(stat[wave][j][1], 0, hi));  // dO V^T - delta
        float e[16], f[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            e[r] = __builtin_amdgcn_exp2f(s[r] * c);
            f[r] = e[r] * dp[r];
        }
        const bf16x8 p[2] = {pack8(e), pack8(e + 8)};  // 2^-8 relative at most, for the product with dO
        mfma_tr<D, 0>(av, ta, lds0 + cur + TILE, p);
        const bf16x8 ds[2] = {pack8(f), pack8(f + 8)};  // the same, for the product with Q
        mfma_tr<D, 0>(ak, ta, lds0 + cur, ds);
        if (some) mfma_tr<D, 0>(ak, ta, lds0 + cur, rest_of(f, ds).b);
    }
    if (!live) {
#pragma unroll
        for (int t = 0; t < D / 32; ++t) ak[t] = av[t] = splat16(0.f);
    }
    __syncthreads();
    const int64_t first = sp.s0 + sp.first;
    join_rows<D>((float*)smem, ak, scale, wave, lane, dk.p + first * dk.tok + kvh * dk.head, dk.tok, sp.len - sp.first);
    __syncthreads();
    join_rows<D>((float*)smem, av, 1.f, wave, lane, dv.p + first * dv.tok + kvh * dv.head, dv.tok, sp.len - sp.first);
}

Order ag_order(int N, int n_seg, int heads, int blk = AG_BLK) {
    Order o;
    o.n_blk = N / blk + n_seg + 2;
    o.chunk = N / blk / (n_seg > 0 ? n_seg : 1) + 1;
    o.heads = heads;
    const int groups = (o.n_blk + o.chunk - 1) / o.chunk * heads;
    o.grid = (groups + 31) / 32 * 32 * o.chunk;
    o.by_chunk = 0xffffffffu / (unsigned)o.chunk;
    o.by_heads = 0xffffffffu / (unsigned)heads;
    o.per_blk = (float)(n_seg + 2) / (float)o.n_blk;
    o.by_eights = heads >= 8 ? 0xffffffffu / (unsigned)(heads & ~7) : 0u;
    o.by_rest = heads & 7 ? 0xffffffffu / (unsigned)(heads & 7) : 0u;
    o.even = n_seg + 2 <= EVEN_MAX;
    o.by_length = N / EVEN_LONG >= n_seg;
    if (o.even) o.grid = o.n_blk * heads;
    return o;
}
// Blocks of 32 rows where there are few of 128, block numbers without rows counted: no more than CUs at head dim 64, where a CU holds
// two workgroups of 32 rows, and 144 at 128, where their rings leave one on a CU.  A workgroup of 32 rows takes a quarter of the time
// only where each wave has several tiles, so that sequences below 512 tokens on average have to fit at once as well.
// Forward and backward pass, blocks of 128 rows and of 32 (us).  Head dim 64, blocks: one of 4096, 210: 69, 187 and 66, 153; 245: 72, 189
// and 73, 169; 280: 59, 168 and 70, 165.  12 of 300, 168 (496 workgroups of 32 rows): 10.5, 22.7 and 10.4, 19.0; 210 (620): 10.5, 24.6
// and 14.0, 33.5.  Head dim 128: one of 4096, 140: 96, 318 and 88, 239; 175: 123, 324 and 139, 359; 245: 123, 324 and 184, 477.  8 of 512,
// 84: 15.8, 51.0 and 10.9, 31.0; 126: 19.1, 52.7 and 21.0, 58.4.  One of 700, 144: 20.4, 63.7 and 23.4, 64.9; these two are what it
// loses most on.  12 of 300, 168: 11.7, 36.8 and 15.9, 45.5.
bool ag_few(int N, int n_seg, int heads, int D) {
    const int per_cu = D == 64 ? 2 : 1;
    if ((N / AG_BLK + n_seg + 2) * (long long)heads > (D == 64 ? 256 : 144)) return false;
    return N / EVEN_LONG >= n_seg || (N / AG_FEW_BLK + n_seg) * (long long)heads <= 256 * per_cu;
}

bool ag_strides(const void* p, const int64_t* st, int D) {
    // 16-byte rows; a tile's offsets (64 rows) stay inside the 31 bits of a buffer descriptor
    return ((uintptr_t)p & 15) == 0 && st[0] % 8 == 0 && st[1] % 8 == 0 && st[0] >= D && st[1] >= 0 && st[0] < (1 << 23);
}

int ag_check(const char* who, const int32_t* cu, int n_seg, int N, int H, int G, int D, float scale) {
    if (D != 64 && D != 128) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128)", who, D);
    if (N < 0 || N > (1 << 30) || n_seg < 0 || H <= 0 || G <= 0 || H % G) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: n_tokens=%d, n_segments=%d, heads=%d, kv heads=%d", who, N, n_seg, H, G);
    if (!(scale > 1e-30f && scale < 1e30f)) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: scale must be positive and finite (1e-30 .. 1e30)", who);
    if (N > 0 && !cu) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "%s: null pointer", who);
    // a launch holds fewer than 2^32 threads; the order of the blocks pads the grid to at most twice this
    if (2 * ((long long)N / AG_BLK + n_seg + 3) * (H + 32) >= (1LL << 24)) ESMK_FAIL(ESMK_ERR_UNSUPPORTED, "%s: grid too large", who);
    return ESMK_OK;
}

}  // namespace

extern "C" int esmk_attn_varlen_fwd(const void* q, const void* k, const void* v, void* out, float* lse,
                                    const int64_t* strides, const int32_t* cu_seqlens, int n_segments,
                                    const uint8_t* key_mask, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                                    float scale, esmk_stream_t stream) {
    if (int rc = ag_check("esmk_attn_varlen_fwd", cu_seqlens, n_segments, n_tokens, n_heads, n_kv_heads, head_dim, scale)) return rc;
    if (n_tokens == 0) return ESMK_OK;
    if (!q || !k || !v || !out || !lse || !strides) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_attn_varlen_fwd: null pointer");
    const void* ps[4] = {q, k, v, out};
    for (int i = 0; i < 4; ++i)
        if (!ag_strides(ps[i], strides + 2 * i, head_dim))
            ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_attn_varlen_fwd: tensor %d: address and strides must be multiples of 16 bytes, token stride >= head_dim", i);
    const View vq{(const __bf16*)q, strides[0], strides[1]}, vk{(const __bf16*)k, strides[2], strides[3]}, vv{(const __bf16*)v, strides[4], strides[5]};
    const OutView vo{(__bf16*)out, strides[6], strides[7]};
    const int group = n_heads / n_kv_heads;
    const bool few = ag_few(n_tokens, n_segments, n_heads, head_dim);
    const Order od = ag_order(n_tokens, n_segments, n_heads, few ? AG_FEW_BLK : AG_BLK);
    auto* kern = few             ? (head_dim == 64 ? attn_fwd_few_kernel<64> : attn_fwd_few_kernel<128>)
                 : head_dim == 64 ? (key_mask ? attn_fwd_lse_kernel<64, true> : attn_fwd_lse_kernel<64, false>)
                                  : (key_mask ? attn_fwd_lse_kernel<128, true> : attn_fwd_lse_kernel<128, false>);
    hipLaunchKernelGGL(kern, dim3(od.grid), dim3(AG_WAVES * 64), 0, (hipStream_t)stream, vq, vk, vv, vo, lse, cu_seqlens, n_segments,
                       key_mask, n_tokens, group, od, scale * AG_LOG2E);
    ESMK_CHECK_LAUNCH("esmk_attn_varlen_fwd");
    return ESMK_OK;
}

extern "C" size_t esmk_attn_varlen_bwd_workspace_bytes(int n_tokens, int n_heads) {
    return n_tokens <= 0 || n_heads <= 0 ? 0 : (size_t)n_tokens * n_heads * sizeof(float);
}

extern "C" int esmk_attn_varlen_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                    const float* lse, void* dq, void* dk, void* dv, const int64_t* strides,
                                    const int32_t* cu_seqlens, int n_segments, const uint8_t* key_mask, int n_tokens,
                                    int n_heads, int n_kv_heads, int head_dim, float scale, void* workspace,
                                    size_t workspace_bytes, esmk_stream_t stream) {
    if (int rc = ag_check("esmk_attn_varlen_bwd", cu_seqlens, n_segments, n_tokens, n_heads, n_kv_heads, head_dim, scale)) return rc;
    if (n_tokens == 0) return ESMK_OK;
    if (!dout || !q || !k || !v || !out || !lse || !dq || !strides) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_attn_varlen_bwd: null pointer");
    if (!dk != !dv) ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_attn_varlen_bwd: null pointer (dk and dv are wanted together or not at all)");
    const void* ps[8] = {dout, q, k, v, out, dq, dk, dv};
    for (int i = 0; i < (dk ? 8 : 6); ++i)
        if (!ag_strides(ps[i], strides + 2 * i, head_dim))
            ESMK_FAIL(ESMK_ERR_INVALID_ARG, "esmk_attn_varlen_bwd: tensor %d: address and strides must be multiples of 16 bytes, token stride >= head_dim", i);
    if (!workspace || workspace_bytes < esmk_attn_varlen_bwd_workspace_bytes(n_tokens, n_heads) || ((uintptr_t)workspace & 3))
        ESMK_FAIL(ESMK_ERR_WORKSPACE, "esmk_attn_varlen_bwd: needs %zu workspace bytes", esmk_attn_varlen_bwd_workspace_bytes(n_tokens, n_heads));
    auto in = [&](int i) { return View{(const __bf16*)ps[i], strides[2 * i], strides[2 * i + 1]}; };
    auto ov = [&](int i) { return OutView{(__bf16*)ps[i], strides[2 * i], strides[2 * i + 1]}; };
    const int group = n_heads / n_kv_heads;
    const bool few_q = ag_few(n_tokens, n_segments, n_heads, head_dim), few_k = ag_few(n_tokens, n_segments, n_kv_heads, head_dim);
    const Order oq = ag_order(n_tokens, n_segments, n_heads, few_q ? AG_FEW_BLK : AG_BLK);
    const Order ok = ag_order(n_tokens, n_segments, n_kv_heads, few_k ? AG_FEW_BLK : AG_BLK);
    float* delta = (float*)workspace;
    hipStream_t s = (hipStream_t)stream;
    auto* kq = few_q           ? (head_dim == 64 ? attn_bwd_dq_few_kernel<64> : attn_bwd_dq_few_kernel<128>)
               : head_dim == 64 ? (key_mask ? attn_bwd_dq_kernel<64, true> : attn_bwd_dq_kernel<64, false>)
                              : (key_mask ? attn_bwd_dq_kernel<128, true> : attn_bwd_dq_kernel<128, false>);
    hipLaunchKernelGGL(kq, dim3(oq.grid), dim3(AG_WAVES * 64), 0, s, in(0), in(1), in(2), in(3), in(4), lse, delta, ov(5),
                       cu_seqlens, n_segments, key_mask, n_tokens, group, oq, scale);
    if (dk) {
        auto* kk = few_k ? (head_dim == 64 ? attn_bwd_dkdv_few_kernel<64> : attn_bwd_dkdv_few_kernel<128>)
                         : (head_dim == 64 ? attn_bwd_dkdv_kernel<64> : attn_bwd_dkdv_kernel<128>);
        hipLaunchKernelGGL(kk, dim3(ok.grid), dim3(AG_WAVES * 64), 0, s, in(0), in(1), in(2), in(3), lse, delta, ov(6), ov(7),
                           cu_seqlens, n_segments, key_mask, n_tokens, group, ok, scale);
    }
    ESMK_CHECK_LAUNCH("esmk_attn_varlen_bwd");
    return ESMK_OK;
}
