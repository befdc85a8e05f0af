// gfx950 kernels of linear attention with a decay for each head:
//
//   S_t = exp(g_t) S_(t-1) + k_t v_t^T,   o_t = scale * S_t^T q_t       S [k_dim][v_dim] of a v head, in f32
//
// as the recurrence itself (single tokens, few tokens) and in chunks on the matrix cores (prompts).
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace skv {

typedef __attribute__((ext_vector_type(4))) float float4_t;

// Columns col .. col + 3 of a row of n: one load, or (unaligned rows, dims that are no multiples of four) four; 0 past the end.
__device__ __forceinline__ float4_t load_four(const float *row, int col, int n, int vec) {
    float4_t x = {0.f, 0.f, 0.f, 0.f};
    if (vec) {
        if (col < n) x = *reinterpret_cast<const float4_t *>(row + col);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < n) x[e] = row[col + e];
    }
    return x;
}
__device__ __forceinline__ void store_four(float *row, int col, int n, int vec, float4_t x) {
    if (vec) {
        if (col < n) *reinterpret_cast<float4_t *>(row + col) = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < n) row[col + e] = x[e];
    }
}

// ------------------------------------------------------------------------------------
// The recurrence. A workgroup holds COLS columns of one head's state in registers, a thread four columns of every
// (1024 / COLS)-th row, and goes through the tokens: S and the outputs' terms are its own, the outputs are summed over the
// threads of a column.
// ------------------------------------------------------------------------------------
constexpr int LINEAR_K_MAX = 256;

// One token each of up to N sequences: the state read and written once and nothing else. Bound by the bytes where there are many, by the chain of
// one launch, its loads and its stores where there are few (one of 32 heads of 128 x 128, 4.2 MB, 3.6 us; eleven of 8 of 96 x 200, 13.6 MB, 6.2); so every thread loads the q and k of its rows itself, nothing waits for a
// barrier but the outputs, and a call's arguments are no longer than its sequences ask for.
template <int COLS, int NP, int N>
__global__ __launch_bounds__(256) void linear_step_kernel(LinearRows r, LinearStates<N> s) {
    constexpr int TPR = COLS / 4; // threads of a row
    constexpr int RP = 256 / TPR; // rows at a time, NP times
    __shared__ float4_t sums[4][TPR];
    const LinearDims &d = r.d;
    const int blocks = (d.v_dim + COLS - 1) / COLS;
    const int h = blockIdx.x / blocks, seq = blockIdx.y, tid = threadIdx.x;
    const int c4 = tid % TPR, r0 = tid / TPR, col = (blockIdx.x % blocks) * COLS + c4 * 4;
    const long state_at = (long)h * d.k_dim * d.v_dim;
    const float *const before = s.before[seq];
    const float *const kp = r.k + (long)seq * r.k_stride + (long)(h / d.group) * d.k_dim, *const qp = r.q + (long)seq * r.q_stride + (long)(h / d.group) * d.k_dim;
    float4_t S[NP];
    float kk[NP], qq[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = r0 + p * RP;
        S[p] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (before && row < d.k_dim) S[p] = load_four(before + state_at + (long)row * d.v_dim, col, d.v_dim, r.vec);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = min(r0 + p * RP, d.k_dim - 1);
        kk[p] = kp[row];
        qq[p] = qp[row];
    }
    const float4_t v = load_four(r.v + (long)seq * r.v_stride + (long)h * d.v_dim, col, d.v_dim, r.vec);
    const float a = expf(r.g[(long)seq * r.g_stride + h]);
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = r0 + p * RP;
        if (row < d.k_dim) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                S[p][e] = a * S[p][e] + kk[p] * v[e];
                o[e] += qq[p] * S[p][e];
            }
            store_four(s.after[seq] + state_at + (long)row * d.v_dim, col, d.v_dim, r.vec, S[p]);
        }
    }
    // the threads of a column: along sixteen lanes, the four sixteens, the wavefronts
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const auto with = [&](auto ctrl) { o[e] += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(o[e]), decltype(ctrl)::value, 0xf, 0xf, true)); };
        if constexpr (TPR <= 4) with(std::integral_constant<int, 0x124>{});
        with(std::integral_constant<int, 0x128>{});
        o[e] = rows_sum(o[e]);
    }
    if ((tid & 63) < TPR) sums[tid >> 6][c4] = o;
    __syncthreads();
    if (tid < TPR) {
        o = (sums[0][c4] + sums[1][c4] + (sums[2][c4] + sums[3][c4])) * d.scale;
        store_four(r.out + (long)seq * d.v_heads * d.v_dim + (long)h * d.v_dim, col, d.v_dim, r.vec, o);
    }
}

// n tokens of one sequence
template <int COLS>
__global__ __launch_bounds__(256) void linear_recurrent_kernel(LinearRows r, const float *before, float *after) {
    constexpr int TPR = COLS / 4;     // threads of a row
    constexpr int RP = 256 / TPR;     // rows at a time
    constexpr int NP = LINEAR_K_MAX / RP;
    __shared__ float ks[2][LINEAR_K_MAX], qs[2][LINEAR_K_MAX];
    __shared__ float4_t sums[2][4][TPR];
    const LinearDims d = r.d;
    const int blocks = (d.v_dim + COLS - 1) / COLS;
    const int h = blockIdx.x / blocks;
    const int tid = threadIdx.x, wave = tid >> 6;
    const int c4 = tid % TPR, r0 = tid / TPR;
    const int col = (blockIdx.x % blocks) * COLS + c4 * 4;
    const long state_at = (long)h * d.k_dim * d.v_dim;
    float4_t S[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = r0 + p * RP;
        S[p] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (before && row < d.k_dim) S[p] = load_four(before + state_at + (long)row * d.v_dim, col, d.v_dim, r.vec);
    }
    for (int t = 0; t < r.n; ++t) {
        const long at = t;
        const int buf = t & 1;
        if (tid < d.k_dim) {
            ks[buf][tid] = r.k[at * r.k_stride + (long)(h / d.group) * d.k_dim + tid];
            qs[buf][tid] = r.q[at * r.q_stride + (long)(h / d.group) * d.k_dim + tid] * d.scale;
        }
        const float4_t v = load_four(r.v + at * r.v_stride + (long)h * d.v_dim, col, d.v_dim, r.vec);
        const float a = expf(r.g[at * r.g_stride + h]);
        __syncthreads();
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int row = r0 + p * RP;
            if (row < d.k_dim) {
                const float kk = ks[buf][row], qq = qs[buf][row];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    S[p][e] = a * S[p][e] + kk * v[e];
                    o[e] += qq * S[p][e];
                }
            }
        }
#pragma unroll
        for (int x = TPR; x < 64; x *= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
        if ((tid & 63) < TPR) sums[buf][wave][c4] = o;
        __syncthreads();
        if (tid < TPR) {
            o = sums[buf][0][c4];
            for (int w = 1; w < 4; ++w) o += sums[buf][w][c4];
            store_four(r.out + at * ((long)d.v_heads * d.v_dim) + (long)h * d.v_dim, col, d.v_dim, r.vec, o);
        }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int row = r0 + p * RP;
        if (row < d.k_dim) store_four(after + state_at + (long)row * d.v_dim, col, d.v_dim, r.vec, S[p]);
    }
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static int may_be_wide(const LinearRows &r) {
    return aligned16(r.q) && aligned16(r.k) && aligned16(r.v) && aligned16(r.out) && (r.q_stride | r.k_stride | r.v_stride) % 4 == 0 &&
           r.d.k_dim % 4 == 0 && r.d.v_dim % 4 == 0;
}

static unsigned blocks_of(const LinearDims &d, int cols) { return (unsigned)(d.v_heads * ((d.v_dim + cols - 1) / cols)); }

template <int COLS, int NP>
static void launch_step_as(const LinearRows &r, const LinearStates<LINEAR_SEQS> &s, int seqs, hipStream_t stream) {
    const dim3 grid(blocks_of(r.d, COLS), (unsigned)seqs);
    const auto as = [&](auto few) {
        for (int i = 0; i < seqs; ++i) few.before[i] = s.before[i], few.after[i] = s.after[i];
        return few;
    };
    if (seqs <= 2) linear_step_kernel<COLS, NP, 2><<<grid, 256, 0, stream>>>(r, as(LinearStates<2>{}));
    else if (seqs <= 16) linear_step_kernel<COLS, NP, 16><<<grid, 256, 0, stream>>>(r, as(LinearStates<16>{}));
    else linear_step_kernel<COLS, NP, LINEAR_SEQS><<<grid, 256, 0, stream>>>(r, s);
}
hipError_t launch_linear_step(const LinearRows &rows, const LinearStates<LINEAR_SEQS> &s, int seqs, hipStream_t stream) {
    LinearRows r = rows;
    r.vec = may_be_wide(r);
    for (int i = 0; i < seqs; ++i) r.vec = r.vec && aligned16(s.before[i]) && aligned16(s.after[i]);
    if (blocks_of(r.d, 32) * (unsigned)seqs <= 256) {
        if (r.d.k_dim <= 64) launch_step_as<16, 1>(r, s, seqs, stream);
        else if (r.d.k_dim <= 128) launch_step_as<16, 2>(r, s, seqs, stream);
        else launch_step_as<16, 4>(r, s, seqs, stream);
    } else {
        if (r.d.k_dim <= 64) launch_step_as<32, 2>(r, s, seqs, stream);
        else if (r.d.k_dim <= 128) launch_step_as<32, 4>(r, s, seqs, stream);
        else launch_step_as<32, 8>(r, s, seqs, stream);
    }
    return hipGetLastError();
}

hipError_t launch_linear_recurrent(const LinearRows &rows, const float *before, float *after, hipStream_t stream) {
    LinearRows r = rows;
    r.vec = may_be_wide(r) && aligned16(before) && aligned16(after);
    if (blocks_of(r.d, 32) <= 256) linear_recurrent_kernel<16><<<blocks_of(r.d, 16), 256, 0, stream>>>(r, before, after);
    else linear_recurrent_kernel<32><<<blocks_of(r.d, 32), 256, 0, stream>>>(r, before, after);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------
// Chunks of 32 tokens on the matrix cores. With b_i the sum of the chunk's decays up to token i and S the state in front of it
//
//   o_i  = e^{b_i} S^T q_i + sum_{j <= i} e^{b_i - b_j} (q_i . k_j) v_j
//   S'   = e^{b_31} S + sum_j e^{b_31 - b_j} k_j v_j^T
//
// (no exponent is above 0 while no decay is; their differences are taken in 64 bits). A workgroup goes through a part of the tokens chunk
// by chunk with the state of one head, all k dims by 64 or 128 v dims, in its wavefronts' registers as accumulators [k dims][v dims]; a wavefront's
// 16 columns of it are the operand of S^T q as they lie, which fixes the order in which every operand counts its contraction: a lane's eight
// are 4g .. 4g + 3 and 16 + 4g .. of 32, g = lane / 16.
//
// Every factor is three bf16 terms, which are it exactly (each leaves at most 2^-8 of what it stands for), and a product six: the three smallest of the
// nine are below 2^-23 together. bf16 has f32's range, so no factor has units that another one could spoil: a large v, k or row of the
// state leaves what lies beside it as exact as it was, and small factors have all their bits (a term below 2^-126 may count as 0). Two f16 terms in units of
// their group's largest, three products, held neither; they took 240 us for the outputs below and 122 for the states.
//
// OUT = false: the state alone, from part to part. Parts are independent but for the state in front of them: a first launch makes what each
// adds (the first one from the caller's state), linear_scan_kernel turns that into the states, the last launch the outputs.
//
// 16384 tokens of 16 / 32 heads of 128 dims, 0.8 GB in and out: 136 us for the states (k and v once more, 3 TB/s), 10 for the scan, 317 for the
// outputs; 2000 tokens 26, 10 and 47. In the outputs' launch the vector unit is busy for 63 % of the cycles (some 800 operations a wavefront and chunk, a third of
// them the terms), the matrix cores for 38 %, LDS for 31 %; the rest is the chain of a chunk's three barriers. Two workgroups of eight wavefronts a CU, which 79 KB of
// LDS and 128 registers allow: so q comes through LDS as terms, but the keys of the scores go straight to the two wavefronts that make them.
// With two barriers (the state before the weights' products) nine registers are spilled: 6 % slower.
// ------------------------------------------------------------------------------------
constexpr int CH = 32; // tokens of a chunk
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) short short4_t;
typedef __attribute__((ext_vector_type(4))) int int4_t;

// Rows of `dims` floats, `stride` apart, of which `n` are left (a chunk's at most: within 2^31 bytes): what lies behind them reads as 0 and is not written.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_left(const float *p, int n, long stride, int dims) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(p), 0, (int)((unsigned)(n - 1) * (unsigned)stride + (unsigned)dims) * 4, 0x00027000);
}
constexpr unsigned OUTSIDE = 0x80000000u; // an offset behind all rows, and still with a row's added
constexpr int NO_COLUMN = 1 << 20;        // behind all of a row's
// Columns col .. col + N - 1 of rows of n, from `at` bytes on
template <int N, bool VEC>
__device__ __forceinline__ auto load_cols(__amdgpu_buffer_rsrc_t rows, unsigned at, int col, int n) {
    typedef __attribute__((ext_vector_type(N))) float cols_t;
    cols_t x;
    if constexpr (VEC) {
        const unsigned from = col < n ? (unsigned)col * 4u + at : OUTSIDE + at;
        if constexpr (N == 4) x = __builtin_bit_cast(cols_t, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)from, 0, 0));
        else x = __builtin_bit_cast(cols_t, __builtin_amdgcn_raw_buffer_load_b64(rows, (int)from, 0, 0));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            x[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rows, (int)(col + e < n ? (unsigned)(col + e) * 4u + at : OUTSIDE + at), 0, 0));
    }
    return x;
}
template <bool VEC>
__device__ __forceinline__ void store_cols(__amdgpu_buffer_rsrc_t rows, unsigned at, int col, int n, float4_t x) {
    typedef __attribute__((ext_vector_type(4))) unsigned u4;
    if constexpr (VEC) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, x), rows, (int)(col < n ? (unsigned)col * 4u + at : OUTSIDE + at), 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)x[e]), rows, (int)(col + e < n ? (unsigned)(col + e) * 4u + at : OUTSIDE + at), 0, 0);
    }
}
// 2^x as m 2^n, m near 1: exact to two steps whatever x is, and no product with it leaves f32 but one that has to
struct Power {
    float m;
    int n;
};
__device__ __forceinline__ Power power_of(double x) {
    const double n = __builtin_fmax(__builtin_fmin(__builtin_rint(x), 4096.0), -4096.0); // (a NaN's is in m)
    return {__builtin_amdgcn_exp2f((float)(x - n)), (int)n};
}

// Operands: eight values (half of one: four) as three terms, in the products' order
constexpr int TERMS = 3;
struct Half {
    uint2 x[TERMS];
};
struct Operand {
    uint4 x[TERMS];
    __device__ __forceinline__ Half first() const {
        Half h;
#pragma unroll
        for (int p = 0; p < TERMS; ++p) h.x[p] = make_uint2(x[p].x, x[p].y);
        return h;
    }
};
__device__ __forceinline__ Half terms_of(float4_t v) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    Half h;
#pragma unroll
    for (int p = 0; p < TERMS; ++p) {
        uint32_t t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{v[2 * i], v[2 * i + 1]}, b2));
            v[2 * i] -= __uint_as_float(t[i] << 16);
            v[2 * i + 1] -= __uint_as_float(t[i] & 0xffff0000u);
        }
        h.x[p] = make_uint2(t[0], t[1]);
    }
    return h;
}
__device__ __forceinline__ Operand terms_of(float4_t a, float4_t b) {
    const Half l = terms_of(a), h = terms_of(b);
    Operand o;
#pragma unroll
    for (int p = 0; p < TERMS; ++p) o.x[p] = make_uint4(l.x[p].x, l.x[p].y, h.x[p].x, h.x[p].y);
    return o;
}
// f(term of a, term of b), the smallest first
template <class F>
__device__ __forceinline__ void pairs(F f) {
    f(2, 0), f(0, 2), f(1, 1), f(1, 0), f(0, 1), f(0, 0);
}
__device__ __forceinline__ float4_t products(const Operand &a, const Operand &b, float4_t acc) {
    pairs([&](int p, int q) __attribute__((always_inline)) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a.x[p]), __builtin_bit_cast(bf16x8_t, b.x[q]), acc, 0, 0, 0);
    });
    return acc;
}
// of half an operand: 16 of the 32
__device__ __forceinline__ float4_t products(const Half &a, const Half &b, float4_t acc) {
    pairs([&](int p, int q) __attribute__((always_inline)) {
        acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a.x[p]), __builtin_bit_cast(short4_t, b.x[q]), acc, 0, 0, 0);
    });
    return acc;
}

// W wavefronts, 16 v dims each.
template <int DK, int W, bool OUT>
struct LinearLds {
    static constexpr int KK = DK / 32, VB = 16 * W;
    uint4 kt[TERMS][DK / 16][64];                // e^{b_31 - b_j} k_j, rows are k dims
    uint4 vt[TERMS][W][64];                      // v_j, rows are v dims
    uint4 q[OUT ? TERMS : 0][2][KK][64];         // q_i, rows are tokens
    uint2 p[OUT ? TERMS : 0][3][64];             // weights, (keys 0, queries 0), (0, 1), (1, 1)
    alignas(16) double b[2][CH];
    float from_m[2][CH], to_m[2][CH]; // e^{b_i}, e^{b_31 - b_j}
    int from_n[2][CH], to_n[2][CH];
    Power whole[2];               // e^{b_31}
    int bad[2][VB];               // the first token whose v is not finite there (CH = none)
    int any_bad[2];
};
static_assert(2 * sizeof(LinearLds<128, 8, true>) <= 160 * 1024, "two workgroups on a CU");

struct LinearChunkArgs {
    LinearRows r;
    const float *before; // the caller's, null = zeros
    float *after;
    float *slots;  // [parts - 1][v_heads][v blocks]: states behind each part but the last, in the order of the accumulators; then the caller's
                   // old one, where its new one goes to the same place (one part's workgroups may be done before another's begin)
    Power *decays; // [parts - 1][v_heads]: what a part multiplies the state by
    int parts, part_rows, blocks;
};

// Wavefronts that a SIMD holds: what LDS allows of 8 (two workgroups, heads of up to 128 k dims) or 4 wavefronts, registers to match
constexpr int linear_occupancy(int DK, int W, bool OUT) { return DK > 128 ? (OUT && W == 4 ? 1 : 2) : W == 8 ? 4 : OUT && DK == 128 ? 2 : 3; }

template <int DK, int W, bool OUT, bool VEC>
__global__ __launch_bounds__(W * 64, linear_occupancy(DK, W, OUT)) void linear_chunk_kernel(LinearChunkArgs a) {
    using Lds = LinearLds<DK, W, OUT>;
    constexpr int KK = Lds::KK, VB = Lds::VB, DT = DK / 16;
    extern __shared__ __attribute__((aligned(16))) uint4 smem[];
    Lds &m = *reinterpret_cast<Lds *>(smem);
    const LinearRows &r = a.r;
    const LinearDims &d = r.d;
    int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups go to the eight XCDs in turn: heads that share q and k to the same one
    const int bx = (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
    const int h = bx / a.blocks, vb = bx % a.blocks, part = blockIdx.y;
    const int t0 = part * a.part_rows, t1 = min(t0 + a.part_rows, r.n);
    const float *qp = r.q + (long)(h / d.group) * d.k_dim, *kp = r.k + (long)(h / d.group) * d.k_dim, *vp = r.v + (long)h * d.v_dim;
    const int col0 = vb * VB; // first v dim of the workgroup
    const long state_at = (long)h * d.k_dim * d.v_dim;
    constexpr long SLOT = (long)DK * VB; // of a (part, head, block)
    const bool in_place = a.parts > 1 && a.before == a.after;
    const auto slot = [&](int p) { return a.slots + (((long)p * d.v_heads + h) * a.blocks + vb) * SLOT + (long)wave * 16 * DK; };

    // k dims 16 i + 4 g4 + e by v dim 16 wave + n16
    float4_t S[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) S[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    // of an element in the caller's buffers; none of it lies past the last k dim, nor (OUTSIDE) past the last v dim
    const auto state_byte = [&](int i, int e) __attribute__((always_inline)) {
        const int col = col0 + wave * 16 + n16;
        return (unsigned)((i * 16 + g4 * 4 + e) * d.v_dim) * 4u + (col < d.v_dim ? (unsigned)col * 4u : OUTSIDE);
    };
    const auto to_slot = [&](int at) __attribute__((always_inline)) {
        float4_t *p = reinterpret_cast<float4_t *>(slot(at)) + lane;
#pragma unroll
        for (int i = 0; i < DT; ++i) p[i * 64] = S[i];
    };
    // a chunk's decays, by the last wavefront (one without scores), asked for two chunks ahead: sums in 64 bits, what is below e^-1000
    // counted as that (0 in 32 bits, and nothing is lost beside it). In powers of two from here on.
    double total = 0.0; // of the part
    // Where a lane's operand of q lies: the sixteen of a line are turned against each other, by the unit's number, so that the threads of
    // one row, who write the same place of sixteen lines, meet no bank twice (k dims by columns and v, four lines: by the tile's number)
    const auto unit_of = [&](int kk) { return lane ^ ((kk * 4 + g4) & 15); };
    const auto decay = [&](int c0) { return r.g[(long)min(c0 + (lane & (CH - 1)), t1 - 1) * r.g_stride + h]; };
    float gx = 0.0f; // of the chunk after the next
    const auto decays = [&](int c0, int buf, float x) __attribute__((always_inline)) {
        const int t = c0 + (lane & (CH - 1));
        x = t >= t1 ? 0.0f : x < -1000.0f ? -1000.0f : x; // (a NaN stays one)
        double s = (double)x * 1.4426950408889634;
        // sums along sixteen lanes, then the first sixteen's to the next
        const auto along = [&](auto ctrl) __attribute__((always_inline)) {
            const uint2 v = __builtin_bit_cast(uint2, s);
            s += __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_update_dpp(0, v.x, decltype(ctrl)::value, 0xf, 0xf, false),
                                                       __builtin_amdgcn_update_dpp(0, v.y, decltype(ctrl)::value, 0xf, 0xf, false)));
        };
        along(std::integral_constant<int, 0x111>{});
        along(std::integral_constant<int, 0x112>{});
        along(std::integral_constant<int, 0x114>{});
        along(std::integral_constant<int, 0x118>{});
        const auto of_lane = [&](int l) __attribute__((always_inline)) {
            const uint2 v = __builtin_bit_cast(uint2, s);
            return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_readlane(v.x, l), __builtin_amdgcn_readlane(v.y, l)));
        };
        const double first = of_lane(15);
        s += (lane & 16) ? first : 0.0;
        const double all = of_lane(31);
        total += all;
        if (lane < CH) {
            m.b[buf][lane] = s;
            const Power from = power_of(s), to = power_of(all - s);
            m.from_m[buf][lane] = from.m, m.from_n[buf][lane] = from.n;
            m.to_m[buf][lane] = to.m, m.to_n[buf][lane] = to.n;
        }
        if (lane == 0) m.whole[buf] = power_of(all);
    };

    // Registers of the chunk on its way; what lies past the part's last token or a head's last dim is 0. Columns: eight tokens of CW dims of k (whole
    // wavefronts), then of v; with outputs and eight wavefronts the first four's. The next two, the scorers: 16 keys each, as an operand lies. The last two: eight dims
    // of tokens of q. Four wavefronts have columns and q all, the first two of them keys too.
    constexpr bool APART = OUT && W == 8;
    constexpr int CW = !OUT && W == 8 ? 2 : 4;
    typedef __attribute__((ext_vector_type(CW))) float cols_t;
    constexpr int CT = APART ? 256 : W * 64;
    constexpr int KN = DK * 4 / CW, KI = KN < 64 ? 64 : KN;
    constexpr int ITEMS = KI + VB * 4 / CW;
    constexpr int NI = (ITEMS + CT - 1) / CT;
    constexpr int UNITS = CH * DK / 8, QT = APART ? 128 : 256; // of q, and the threads that have them
    constexpr int NU = OUT ? (UNITS + QT - 1) / QT : 0;
    constexpr int C_LOADS = NI * 8, K_LOADS = OUT ? KK * 2 : 0;
    static_assert(!APART || (K_LOADS <= C_LOADS && NU * 2 <= C_LOADS));
    constexpr int K_AT = APART ? 0 : C_LOADS * CW / 4, Q_AT = APART ? 0 : K_AT + K_LOADS, HELD = APART ? C_LOADS : Q_AT + NU * 2;
    float4_t held[HELD];
    const auto column = [&](int u, int e) __attribute__((always_inline)) {
        if constexpr (CW == 4) return held[u * 8 + e];
        else return cols_t{held[u * 4 + e / 2][e % 2 * 2], held[u * 4 + e / 2][e % 2 * 2 + 1]};
    };
    const auto set_column = [&](int u, int e, cols_t x) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CW; ++c) held[(u * 8 + e) * CW / 4][(e * CW + c) & 3] = x[c];
    };
    const bool has_columns = !APART || wave < 4, has_q = OUT && (!APART || wave >= 6);
    const int jt = wave - (APART ? 4 : 0); // a scorer's keys
    const bool scorer = OUT && jt >= 0 && jt < 2;
    const auto unit = [&](int u) { return tid - (APART ? 384 : 0) + u * QT; }; // of q
    const auto item = [&](int u, bool &is_k, int &grp, int &col) __attribute__((always_inline)) {
        const int idx = tid + u * CT;
        is_k = wave * 64 + u * CT < KI; // uniform
        const int i = is_k ? idx : min(idx, ITEMS - 1) - KI; // (wavefronts without one of their own load the last one's, too)
        // sixteen lanes a row, so that its bytes are asked for together
        grp = i >> 4 & 3, col = ((i >> 6) * 16 + (i & 15)) * CW;
        const bool mine = KN >= 64 || !is_k || col < DK;
        if (!mine) col = DK - CW;
        return mine;
    };
    // One path for all: were the loads themselves under a condition, what they bring would be moved where the conditions meet, and waited for.
    // So a wavefront's part says what it reads from where in the slots that all share, in numbers: columns rows, a scorer dims, the last one (q) both.
    // What it has no use for lies behind the rows' dims and costs no access.
    const auto fetch = [&](int c0) __attribute__((always_inline)) {
        const int left = min(t1 - c0, CH);
        const auto rows_of = [&](bool v, bool q) __attribute__((always_inline)) {
            // (by masks: a choice between variables is made by their addresses, and puts them into memory)
            const long as_v = -(long)v, as_q = ~as_v & -(long)q, as_k = ~as_v & ~as_q;
            const long stride = (r.v_stride & as_v) | (r.q_stride & as_q) | (r.k_stride & as_k);
            const long from = ((long)vp & as_v) | ((long)qp & as_q) | ((long)kp & as_k);
            return rows_left(reinterpret_cast<const float *>(from) + (long)c0 * stride, left, stride, v ? d.v_dim : d.k_dim);
        };
        const unsigned q_step = (unsigned)r.q_stride * 4u, k_step = (unsigned)r.k_stride * 4u, v_step = (unsigned)r.v_stride * 4u;
        const unsigned keys_at = (unsigned)(jt * 16 + n16) * k_step;
        const int keys_col = scorer ? g4 * 4 : NO_COLUMN;
        const unsigned q_at = (unsigned)(unit(0) / (DK / 8)) * q_step, q_next = (unsigned)(QT * 8 / DK) * q_step; // (a thread's units are of the same dims)
        const int q_col = has_q && unit(0) < UNITS ? (unit(0) % (DK / 8) >> 2) * 32 + (unit(0) & 3) * 4 : NO_COLUMN;
        const unsigned per_pair = APART && has_q ? q_next : 0u;
        const int col_pair = scorer ? 32 : 0, col_half = 16;
#pragma unroll
        for (int u = 0; u < NI; ++u) {
            bool is_k;
            int grp, col;
            item(u, is_k, grp, col);
            is_k |= !has_columns;
            unsigned at = (unsigned)(grp * 4) * (is_k ? k_step : v_step);
            col += is_k ? 0 : col0;
            if constexpr (APART) {
                at = has_columns ? at : has_q ? q_at : keys_at;
                col = has_columns ? col : has_q ? q_col : keys_col;
            }
            const auto x = rows_of(!is_k, APART && has_q);
            const int dims = is_k ? d.k_dim : d.v_dim;
            const unsigned per_row = has_columns ? is_k ? k_step : v_step : 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int s = u * 8 + e;
                const unsigned add = (unsigned)((e >> 2) * 16 + (e & 3)) * per_row + (APART ? (unsigned)(s / 2) * per_pair : 0u);
                const int more = APART && !has_columns ? s / 2 * col_pair + (s & 1) * col_half : 0;
                const auto y = load_cols<CW, VEC>(x, at + add, col + more, dims);
                if constexpr (CW == 4) held[s] = y;
                else set_column(u, e, y);
            }
        }
        if constexpr (!APART && OUT) {
            const auto ks = rows_of(false, false), qs = rows_of(false, true);
#pragma unroll
            for (int s = 0; s < K_LOADS; ++s) held[K_AT + s] = load_cols<4, VEC>(ks, keys_at, keys_col + s / 2 * 32 + (s & 1) * 16, d.k_dim);
#pragma unroll
            for (int s = 0; s < NU * 2; ++s) held[Q_AT + s] = load_cols<4, VEC>(qs, q_at + (unsigned)(s / 2) * q_next, q_col + (s & 1) * 16, d.k_dim);
        }
    };
    const auto stage_columns = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NI; ++u) {
            bool is_k;
            int grp, col;
            const bool mine = item(u, is_k, grp, col);
            if (wave * 64 + u * CT >= ITEMS) continue; // (uniform)
            if (is_k) { // times their decays to the chunk's end
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4_t w = *reinterpret_cast<const float4_t *>(&m.to_m[buf][i * 16 + grp * 4]);
                    const int4_t n = *reinterpret_cast<const int4_t *>(&m.to_n[buf][i * 16 + grp * 4]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        cols_t x = column(u, i * 4 + e) * w[e];
#pragma unroll
                        for (int c = 0; c < CW; ++c) x[c] = __builtin_ldexpf(x[c], n[e]);
                        set_column(u, i * 4 + e, x);
                    }
                }
            } else {
                // a v that is not finite would reach the tokens in front of it through weights of 0: its dim is kept out of the
                // products and is NaN from that token on
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int c = 0; c < CW; ++c) top = __builtin_elementwise_maximum(top, __builtin_fabsf(column(u, e)[c]));
                if (!(top < INFINITY)) {
                    int first[CW];
#pragma unroll
                    for (int c = 0; c < CW; ++c) first[c] = CH;
#pragma unroll
                    for (int e = 7; e >= 0; --e) {
                        cols_t x = column(u, e);
#pragma unroll
                        for (int c = 0; c < CW; ++c) {
                            const bool bad = !(__builtin_fabsf(x[c]) < INFINITY);
                            first[c] = bad ? (e >> 2) * 16 + grp * 4 + (e & 3) : first[c];
                            x[c] = bad ? 0.0f : x[c];
                        }
                        set_column(u, e, x);
                    }
#pragma unroll
                    for (int c = 0; c < CW; ++c) atomicMin(&m.bad[buf][col + c], first[c]);
                    m.any_bad[buf] = 1;
                }
            }
#pragma unroll
            for (int c = 0; c < CW; ++c) {
                const Operand x = terms_of(float4_t{column(u, 0)[c], column(u, 1)[c], column(u, 2)[c], column(u, 3)[c]},
                                           float4_t{column(u, 4)[c], column(u, 5)[c], column(u, 6)[c], column(u, 7)[c]});
                const int at = grp * 16 + (((col + c) ^ (col >> 4 & 3)) & 15);
                if (KN >= 64 || mine) {
#pragma unroll
                    for (int p = 0; p < TERMS; ++p) (is_k ? m.kt[p] : m.vt[p])[(col + c) >> 4][at] = x.x[p];
                }
            }
        }
    };
    const auto stage_q = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int row = unit(u) / (DK / 8), un = unit(u) % (DK / 8);
            if (UNITS % QT == 0 || unit(u) < UNITS) {
                const Operand x = terms_of(held[Q_AT + u * 2], held[Q_AT + u * 2 + 1]);
#pragma unroll
                for (int p = 0; p < TERMS; ++p) m.q[p][row >> 4][un >> 2][(un & 3) * 16 + ((row ^ un) & 15)] = x.x[p];
            }
        }
    };
    const auto q_operand = [&](int it, int kk) __attribute__((always_inline)) {
        Operand x;
#pragma unroll
        for (int p = 0; p < TERMS; ++p) x.x[p] = m.q[p][it][kk][unit_of(kk)];
        return x;
    };

    // (everything asked for before anything is waited for: decays, the first chunk, the state)
    const int last_chunk = t0 + (t1 - 1 - t0) / CH * CH;
    const float g0 = decay(t0);
    gx = decay(t0 + CH);
    fetch(t0);
    if (part == 0 && !(OUT && in_place)) {
        if (a.before) {
            const auto rows = rows_left(a.before + state_at, d.k_dim, d.v_dim, d.v_dim);
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rows, (int)state_byte(i, e), 0, 0));
        }
        if (!OUT && in_place) to_slot(a.parts - 1);
    } else if (OUT) {
        const float4_t *p = reinterpret_cast<const float4_t *>(slot(part == 0 ? a.parts - 1 : part - 1)) + lane;
#pragma unroll
        for (int i = 0; i < DT; ++i) S[i] = p[i * 64];
    }

    if (wave == W - 1) decays(t0, 0, g0);
    if (tid < VB) m.bad[0][tid] = CH;
    if (tid < 2) m.any_bad[tid] = 0;
    if constexpr (OUT) { // (to nowhere: as many stores behind the first chunk's loads as a chunk has behind the next one's, so that the loads can be waited for without the stores)
        const auto outs = rows_left(r.out, 1, 0, d.v_dim);
        const float x = __int_as_float(tid);
#pragma unroll
        for (int it = 0; it < 2; ++it) store_cols<VEC>(outs, 0, NO_COLUMN, d.v_dim, float4_t{x, x, x, x});
    }
    __syncthreads();
    int buf = 0;
    for (int c0 = t0; c0 < t1; c0 += CH, buf ^= 1) {
        // A chunk's addresses are made anew: kept from chunk to chunk they would not find room in the registers, and reading a spilled one waits
        // for all loads on their way
        asm("" : "+v"(tid));
        lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
        if (has_q) stage_q();
        if (has_columns) stage_columns(buf);
        __syncthreads();
        // (the other workgroup's wavefronts, that bring a chunk in, fill what these leave)
        if constexpr (OUT) __builtin_amdgcn_s_setprio(2);
        if (tid < VB) m.bad[buf ^ 1][tid] = CH; // (read last in the chunk before this one, a barrier ago)
        if (tid == 0) m.any_bad[buf ^ 1] = 0;
        const bool any_bad = m.any_bad[buf] != 0;
        float4_t o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        if (wave == W - 1 && c0 + CH < t1) decays(c0 + CH, buf ^ 1, gx);
        gx = decay(c0 + 2 * CH);
        if constexpr (OUT) {
            if (scorer) { // both tiles of its keys, as weights into LDS
                float4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const Operand k = terms_of(held[K_AT + 2 * kk], held[K_AT + 2 * kk + 1]);
#pragma unroll
                    for (int it = 0; it < 2; ++it) s[it] = products(k, q_operand(it, kk), s[it]);
                }
                const double *const bj = &m.b[buf][jt * 16 + g4 * 4];
                const double b[4] = {bj[0], bj[1], bj[2], bj[3]};
#pragma unroll
                for (int it = 0; it < 2; ++it) {
                    const int i = it * 16 + n16;
                    const double bi = m.b[buf][i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Power w = power_of(bi - b[e]);
                        float f = __builtin_ldexpf(s[it][e] * (w.m * d.scale), w.n);
                        asm("" : "+v"(f)); // (not under the condition: four waits one after the other)
                        s[it][e] = jt * 16 + g4 * 4 + e <= i ? f : 0.0f;
                    }
                    const Half x = terms_of(s[it]);
                    if (it >= jt) {
#pragma unroll
                        for (int p = 0; p < TERMS; ++p) m.p[p][it + jt][lane] = x.x[p];
                    }
                }
            }
        }
        if constexpr (OUT) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const Operand x = terms_of(S[2 * kk], S[2 * kk + 1]);
#pragma unroll
                for (int it = 0; it < 2; ++it) o[it] = products(x, q_operand(it, kk), o[it]);
            }
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                o[it] *= m.from_m[buf][it * 16 + n16] * d.scale;
                const int n = m.from_n[buf][it * 16 + n16];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[it][e] = __builtin_ldexpf(o[it][e], n);
            }
        }
        fetch(min(c0 + CH, last_chunk));
        if constexpr (OUT) __syncthreads(); // the weights
        Operand v;
#pragma unroll
        for (int p = 0; p < TERMS; ++p) v.x[p] = m.vt[p][wave][lane ^ (wave & 3)];
        if constexpr (OUT) {
            const int col = wave * 16 + g4 * 4;
            const auto outs = rows_left(r.out + (long)c0 * (d.v_heads * d.v_dim) + (long)h * d.v_dim, min(t1 - c0, CH), (long)d.v_heads * d.v_dim, d.v_dim);
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int i = it * 16 + n16;
                if (it == 0) { // (sees the first 16 alone)
                    Half w;
#pragma unroll
                    for (int p = 0; p < TERMS; ++p) w.x[p] = m.p[p][0][lane];
                    o[it] += products(v.first(), w, float4_t{0.f, 0.f, 0.f, 0.f});
                } else {
                    Operand w;
#pragma unroll
                    for (int p = 0; p < TERMS; ++p) {
                        const uint2 x = m.p[p][1][lane], y = m.p[p][2][lane];
                        w.x[p] = make_uint4(x.x, x.y, y.x, y.y);
                    }
                    o[it] += products(v, w, float4_t{0.f, 0.f, 0.f, 0.f});
                }
                if (any_bad) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m.bad[buf][col + e] <= i) o[it][e] = __builtin_nanf("");
                }
                store_cols<VEC>(outs, (unsigned)(i * (d.v_heads * d.v_dim)) * 4u, col0 + col, d.v_dim, o[it]);
            }
        }
        int n = __builtin_amdgcn_readfirstlane(m.whole[buf].n);
        if (n < -120 || n > 120) { // (a factor of its own would leave f32)
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[i][e] = __builtin_ldexpf(S[i][e], n);
            n = 0;
        }
        const float f = any_bad && m.bad[buf][wave * 16 + n16] < CH ? __builtin_nanf("") : __builtin_ldexpf(m.whole[buf].m, n);
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            Operand k;
#pragma unroll
            for (int p = 0; p < TERMS; ++p) k.x[p] = m.kt[p][i][lane ^ (i & 3)];
            const float4_t add = products(k, v, float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = __builtin_fmaf(S[i][e], f, add[e]); // (one rounding a chunk: summed by the matrix instruction it was off by twice as much)
        }
        if constexpr (OUT) __builtin_amdgcn_s_setprio(0);
        __syncthreads();
    }
    if (OUT && part < a.parts - 1) return;
    if (OUT) {
        const auto rows = rows_left(a.after + state_at, d.k_dim, d.v_dim, d.v_dim);
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)S[i][e]), rows, (int)state_byte(i, e), 0, 0);
    } else {
        to_slot(part);
        if (tid == (W - 1) * 64 && vb == 0) a.decays[(long)part * d.v_heads + h] = power_of(total);
    }
}

// What the parts add, into the states behind them: state_p = decay_p * state_(p - 1) + added_p.
__global__ __launch_bounds__(256) void linear_scan_kernel(float4_t *slots, const Power *decays, int parts, int heads, long per_head, long per_part) {
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    if (at >= per_part) return;
    const int h = (int)(at / per_head);
    float4_t s = slots[at];
    for (int p = 1; p < parts; ++p) {
        const float4_t x = slots[p * per_part + at];
        const Power w = decays[(long)p * heads + h];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = __builtin_ldexpf(w.m * s[e], w.n) + x[e];
        slots[p * per_part + at] = s;
    }
}

static int k_tiles_of(int k_dim) { return k_dim <= 32 ? 32 : k_dim <= 64 ? 64 : k_dim <= 128 ? 128 : 256; }
static int v_block_of(int v_dim) { return v_dim <= 64 ? 64 : 128; }

LinearParts linear_parts(const LinearDims &d, size_t n) {
    const size_t wgs = (size_t)d.v_heads * ((d.v_dim + v_block_of(d.v_dim) - 1) / v_block_of(d.v_dim));
    size_t parts = std::max<size_t>(512 / wgs, 1);
    parts = std::min<size_t>(parts, (n + 127) / 128);
    parts = std::max<size_t>(parts, std::min<size_t>(n / 1024, 32));
    const size_t rows = ((n + parts - 1) / parts + CH - 1) / CH * CH;
    return {(int)((n + rows - 1) / rows), (int)rows};
}
size_t linear_scratch_bytes(const LinearDims &d, const LinearParts &p) {
    const size_t blocks = (d.v_dim + v_block_of(d.v_dim) - 1) / v_block_of(d.v_dim);
    return (size_t)p.parts * d.v_heads * (blocks * k_tiles_of(d.k_dim) * v_block_of(d.v_dim) + 4) * sizeof(float);
}

template <int DK, int W, bool VEC>
static hipError_t launch_chunks_as(const LinearChunkArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> out_done{0}, state_done{0};
    const dim3 grid((unsigned)(a.r.d.v_heads * a.blocks), (unsigned)a.parts);
    hipError_t e = hipSuccess;
    if (a.parts > 1) {
        e = allow_full_lds(reinterpret_cast<const void *>(linear_chunk_kernel<DK, W, false, VEC>), state_done);
        if (e != hipSuccess) return e;
        linear_chunk_kernel<DK, W, false, VEC><<<dim3(grid.x, grid.y - 1), W * 64, sizeof(LinearLds<DK, W, false>), s>>>(a);
        if (a.parts > 2) {
            const long per_head = (long)a.blocks * DK * (16 * W) / 4, per_part = per_head * a.r.d.v_heads;
            linear_scan_kernel<<<(unsigned)((per_part + 255) / 256), 256, 0, s>>>(reinterpret_cast<float4_t *>(a.slots), a.decays, a.parts - 1,
                                                                                 a.r.d.v_heads, per_head, per_part);
        }
    }
    e = allow_full_lds(reinterpret_cast<const void *>(linear_chunk_kernel<DK, W, true, VEC>), out_done);
    if (e != hipSuccess) return e;
    linear_chunk_kernel<DK, W, true, VEC><<<grid, W * 64, sizeof(LinearLds<DK, W, true>), s>>>(a);
    return hipGetLastError();
}

template <int DK, int W>
static hipError_t launch_chunks(const LinearChunkArgs &a, hipStream_t s) {
    return a.r.vec ? launch_chunks_as<DK, W, true>(a, s) : launch_chunks_as<DK, W, false>(a, s);
}

hipError_t launch_linear_chunks(const LinearRows &rows, const LinearParts &p, const float *before, float *after, void *scratch, hipStream_t s) {
    LinearChunkArgs a{};
    a.r = rows;
    a.r.vec = may_be_wide(rows);
    a.before = before;
    a.after = after;
    a.parts = p.parts;
    a.part_rows = p.part_rows;
    const LinearDims &d = rows.d;
    const int VB = v_block_of(d.v_dim), DK = k_tiles_of(d.k_dim);
    a.blocks = (d.v_dim + VB - 1) / VB;
    a.slots = static_cast<float *>(scratch);
    a.decays = reinterpret_cast<Power *>(a.slots + (size_t)p.parts * d.v_heads * a.blocks * DK * VB);
    if (VB == 64) {
        switch (DK) {
        case 32: return launch_chunks<32, 4>(a, s);
        case 64: return launch_chunks<64, 4>(a, s);
        case 128: return launch_chunks<128, 4>(a, s);
        default: return launch_chunks<256, 4>(a, s);
        }
    }
    switch (DK) {
    case 32: return launch_chunks<32, 8>(a, s);
    case 64: return launch_chunks<64, 8>(a, s);
    case 128: return launch_chunks<128, 8>(a, s);
    default: return launch_chunks<256, 8>(a, s);
    }
}

} // namespace skv
