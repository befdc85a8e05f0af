// gfx950 kernels of the 4-bit element, part 2: chunked prefill over the codes, the matrix-core-bound kernel.
#include <type_traits>

#include "chunk_pages.h"
#include "fp4_tile.h"
#include "lds_copy.h"

namespace skv {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) float float2v_t;
typedef __attribute__((ext_vector_type(4))) float float4_t;
typedef __attribute__((ext_vector_type(16))) float float16_t;
typedef __attribute__((ext_vector_type(32))) float float32_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u2;
typedef __attribute__((ext_vector_type(4))) uint32_t u4;
typedef __attribute__((ext_vector_type(6))) uint32_t u6;
typedef __attribute__((ext_vector_type(8))) int int8v_t;

namespace {

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// two values rounded to bf16 (nearest even), the first in the low half: one instruction
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v_t{x, y}, bf16x2_t)); }
// 32 values as e2m3 codes of x / scale (those of `even` and `odd` take turns in the result), and the codes' values. These conversions take several
// passes and write their results as they go: a result register that is also an operand is read back changed (seen: the scale in the first result
// register, the values after the first few wrong). The compiler does not know of that, so results are early clobbers, which no operand
// shares; nor then of the wait state that a reader of the result needs.
__device__ __forceinline__ u6 to_fp6(float16_t even, float16_t odd, float scale) {
    u6 codes;
    asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n\ts_nop 1" : "=&v"(codes) : "v"(even), "v"(odd), "v"(scale));
    return codes;
}
__device__ __forceinline__ float32_t from_fp6(u6 codes, float scale) {
    float32_t x;
    asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n\ts_nop 1" : "=&v"(x) : "v"(codes), "v"(scale));
    return x;
}

} // namespace

// ------------------------------------------------------------------------------------
// Many query rows over the codes: query slot (i, g) = new row i, head g of the kv head's group, attends positions up to q_pos0 + i through
// the layer's window.
//
// One workgroup = WAVES wavefronts of TILES tiles of 16 query slots of one kv head and a range of the pages any of them attends (split). It walks its
// pages once, in steps: K's codes go to LDS as they are (1 KiB a page of 128 dims) and into the scaled products as they are, against the
// queries as five terms of e2m3 in registers (kernels_fp4.hip); V's codes are converted to f16 once for the workgroup, a page (or part of one) a
// wavefront, in the order of the operands of v_mfma_f32_16x16x32_f16 over a pair of pages. Per pair of pages and tile the products take 160
// + 256 cycles of the matrix pipe at 128 dims (two bf16 terms of the queries against K in bf16: 256 + 256).
// Per pair: S^T of the next pair with the exponentials and the two f16 terms of this pair's probabilities between its products, then O^T of this
// pair. The softmax runs in base 2 against a base that a slot's largest score is 4 to 8 above, and that moves only when one passes that. As terms, weights are 2^4
// times that and so held to 2^-33 of the largest (f16's steps end at 2^-24); with a base further down instead, scores round in larger steps (contexts 1.5 times
// as far from 64 bits). V is 2^-8 times itself. The score accumulators start at minus the base (see prefill_tile_kernel).
// With HALVES = 2 (or 4) the wavefronts are parts that hold the same slots and take the page pairs in turn; their states join through LDS.
//
// Keys that no slot of the workgroup attends have their powers set to 1 when V is converted: 0 x NaN is NaN. A row that is NaN and that some
// slots attend and others do not (a row behind theirs) is converted as if its power were 1, and the slots that attend it get their NaN in a path
// of its own. Pages with powers that f16 does not have are converted to zeros and added in bf16, from memory, behind the pair's products.
//
// What bounds it: over long contexts the products, 512 rows over 32768 of q16/kv2/hd256 in 358 us (770 TFLOP/s of those asked for, which take
// 1.63 times their time at the bf16 rate: 1250, what a large bf16 product reaches; a bf16 layer 409). The matrix pipe is busy 55 % of the cycles: V of the
// next step is converted between a step's last products and its barrier, where both wavefronts of a SIMD stand. Over short contexts its start, at head_dim 128 3 us until the queries are
// converted, 2 until the first V is, and 3 at the end: 512 rows over 0, 1024 of q32/kv8/hd128 18.1, 30.6 (16.5, 30.3).
// ------------------------------------------------------------------------------------
template <int P, int WAVES, int HALVES>
struct Fp4Chunk {
    static constexpr int G = P / 32, NB = (P + 127) / 128, U = fp4_quad(P);
    static constexpr int PAGES = P <= 128 ? 8 : P <= 256 ? 4 : 2; // of a step
    static constexpr int GP = 2 * HALVES, SP = PAGES / GP;        // pages of a group (a pair for each part), groups of a step
    static constexpr int PARTS = WAVES / PAGES, GW = G / PARTS;   // wavefronts that convert a page of V, groups of dims of each
    static constexpr int K_PAGE = 8 * P, K_POWERS = P / 2, K_BUF = PAGES * (K_PAGE + K_POWERS), V_PAGE = 32 * P, V_BUF = PAGES * V_PAGE;
    static constexpr int V_AT = 2 * K_BUF, NAN_AT = V_AT + 2 * V_BUF;
    // of the rows that are NaN: per buffer the step that has some; per (page, part) the step, and per row a bit a group
    // of the powers that f16 does not have: per buffer the step that has some, and per (page, part)
    static constexpr int NAN_WORDS = 2 * (1 + PAGES * PARTS * 17), FAR_WORDS = 2 * (1 + PAGES * PARTS);
    static constexpr size_t LDS = NAN_AT + ((NAN_WORDS + FAR_WORDS) * 4 + 15) / 16 * 16;
    static_assert(SP >= 1 && PARTS >= 1 && G % PARTS == 0, "steps of whole groups, whole groups of dims to a wavefront");
    static_assert(LDS <= 160 * 1024, "it fits a compute unit's LDS");
    static constexpr int ROW = P < 128 ? P / 4 : 32; // units of four dims of a block of a query row
    static_assert(WAVES * 16 * ROW * 16 <= 2 * V_BUF, "a block of every wavefront's queries fits V's buffers");
};

template <int P, int TILES, int WAVES, int HALVES, bool RING>
__global__ __launch_bounds__(WAVES * 64) void fp4_chunk_kernel(DecodeArgs a, ChunkPages c) {
    using L = Fp4Chunk<P, WAVES, HALVES>;
    constexpr int G = L::G, NB = L::NB, U = L::U, NT = P / 16, PAGES = L::PAGES, GP = L::GP, SP = L::SP, PARTS = L::PARTS, GW = L::GW;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Geom g = a.g;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x, kvh = blockIdx.y;
    const int n_slots = a.n_queries * g.gqa;
    constexpr int TW = WAVES / HALVES; // wavefronts of a part
    const int half = HALVES > 1 ? wave / TW : 0, tw = HALVES > 1 ? wave % TW : wave;
    const int wg_slot0 = longest_first(n_slots, TW * TILES * 16, blockIdx.z) * (TW * TILES * 16);
    const int wg_slot1 = min(n_slots, wg_slot0 + TW * TILES * 16) - 1;
    auto limit_of = [&](int slot) { return a.q_pos0 + slot_row(g, slot); };
    auto ws_of = [&](int slot) { return a.window > 0 ? max(a.window_start, limit_of(slot) + 1 - a.window) : a.window_start; };
    const int wg_ws_lo = ws_of(wg_slot0), wg_lim_hi = limit_of(wg_slot1);
    auto entry_of = [&](int pos) {
        if (!RING) return pos >> 4;
        return pos < c.new_pos0 ? max((pos - c.first_pos) >> 4, 0) : c.n_old + ((pos - c.new_first) >> 4);
    };
    const int e_lo = entry_of(wg_ws_lo), e_hi = entry_of(wg_lim_hi) + 1;
    const unsigned span = (unsigned)(e_hi - e_lo);
    const int pb0 = e_lo + (int)(((unsigned)split * span) / (unsigned)a.splits);
    const int pb1 = e_lo + (int)(((unsigned)(split + 1) * span) / (unsigned)a.splits);
    const int n_it = pb1 - pb0, n_groups = (n_it + GP - 1) / GP, n_steps = (n_groups + SP - 1) / SP;
    auto entry = [&](int it) { return min(pb0 + it, e_hi - 1); }; // past the end: a page again, unused

    // ---- what a step brings: V of its pages, K of the pages a group further (K runs a group ahead). ids: physical pages from the step's first on, one a lane
    int ids;
    auto ask_ids = [&](int it) __attribute__((always_inline)) { ids = RING ? fp4_ring_page(a, c, entry(it + lane)) : (int)entry_place<false>(a, c, entry(it + lane)); };
    const uint32_t page_bytes = (uint32_t)g.page_elems * 2;
    const size_t codes_at = (size_t)kvh * fp4_code_bytes(P), powers_at = (size_t)g.kv_heads * fp4_code_bytes(P) + (size_t)kvh * fp4_power_bytes(P);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    auto pool_of = [&](int it, bool v) __attribute__((always_inline)) {
        const bool apart = RING && fp4_in_scratch(c, entry(it));
        return reinterpret_cast<const uint8_t *>(v ? (apart ? c.v_new : a.v_pool) : (apart ? c.k_new : a.k_pool));
    };
    // K of the pages it0 + d0 .. (as many as `pages`), whose physical pages lie in lanes d0 .. of ids, to buffer `buf`
    auto copy_k = [&](int it0, int d0, auto how_many, int buf) __attribute__((always_inline)) {
        constexpr int pages = decltype(how_many)::value;
        const uint32_t to = lds0 + (uint32_t)(buf * L::K_BUF);
        if constexpr (P >= 128) {
#pragma unroll
            for (int r = 0; r < (pages * NB + WAVES - 1) / WAVES; ++r) { // a KiB each
                const int i = wave + r * WAVES, d = i / NB, b = i % NB;
                if (pages * NB % WAVES != 0 && i >= pages * NB) continue;
                const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(ids, d0 + d);
                copy_to_lds(pool_of(it0 + d0 + d, false) + codes_at + (uint64_t)page * page_bytes + b * 1024, (uint32_t)lane * 16, to + d * L::K_PAGE + b * 1024);
            }
        } else {
            constexpr int UNITS = P / 2;
#pragma unroll
            for (int r = 0; r < (pages * UNITS + WAVES * 64 - 1) / (WAVES * 64); ++r) {
                const int i = (wave + r * WAVES) * 64;
                if (i >= pages * UNITS) continue;
                const int u = i + lane, d = min(u / UNITS, pages - 1);
                const uint32_t page = (uint32_t)__shfl(ids, d0 + d);
                if (u < pages * UNITS) gather_to_lds(pool_of(it0 + d0 + d, false) + codes_at + (uint64_t)page * page_bytes + (u - d * UNITS) * 16, to + i * 16);
            }
        }
        constexpr int WORDS = P / 8;
        static_assert(pages * WORDS <= WAVES * 64, "powers: a copy a wavefront, from the last one on");
        const int i = (WAVES - 1 - wave) * 64;
        if (i < pages * WORDS) {
            const int u = i + lane, d = min(u / WORDS, pages - 1);
            const uint32_t page = (uint32_t)__shfl(ids, d0 + d);
            if (u < pages * WORDS) gather_words_to_lds(pool_of(it0 + d0 + d, false) + powers_at + (uint64_t)page * page_bytes + (u - d * WORDS) * 4, to + PAGES * L::K_PAGE + i * 4);
        }
    };
    const int vd = wave / PARTS, vp = wave % PARTS; // the page of a step that this wavefront converts, and which groups of it
    uint32_t vc[GW], vs[GW];
    auto load_v = [&](int it0) __attribute__((always_inline)) {
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(ids, vd);
        const uint8_t *at = pool_of(it0 + vd, true) + (uint64_t)page * page_bytes;
#pragma unroll
        for (int v = 0; v < GW / U; ++v) {
            uint32_t w[U];
            load_words<U>(w, at + codes_at + ((vp * (GW / U) + v) * 64 + lane) * U * 4);
#pragma unroll
            for (int u = 0; u < U; ++u) vc[v * U + u] = w[u];
        }
        load_words<GW>(vs, at + powers_at + (j * G + vp * GW) * 4);
    };
    uint32_t *const nan_step = reinterpret_cast<uint32_t *>(lds + L::NAN_AT), *const nan_of = nan_step + 2; // [2], [2][PAGES * PARTS][1 + 16]
    uint32_t *const far_step = nan_step + L::NAN_WORDS, *const far_of = far_step + 2; // [2], [2][PAGES * PARTS]
    const Inner wg_in = inner_entries<RING>(c, pb0, pb1, wg_ws_lo, wg_lim_hi);
    // V of step `step`, loaded, to buffer step & 1: per (pair, group of dims, dims n or n + 16) a KiB, a lane's 4 keys of page a, then of b
    auto convert_v = [&](int step) __attribute__((always_inline)) {
        const int it = step * PAGES + vd, e = pb0 + it;
        if (!((e >= wg_in.o0 && e < wg_in.o1) || (RING && e >= wg_in.n0 && e < wg_in.n1))) { // uniform: at an edge of what is attended
            const int en = entry(it), pos = entry_pos<RING>(c, en) + j * 4;
            const int lo = max(wg_ws_lo, entry_lo<RING>(c, en)), hi = min(wg_lim_hi, entry_hi<RING>(c, en));
            uint32_t keep = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (it < n_it && pos + i >= lo && pos + i <= hi) keep |= 255u << (8 * i);
#pragma unroll
            for (int t = 0; t < GW; ++t) vs[t] = (vs[t] & keep) | (~keep & 0x7f7f7f7fu);
        }
        uint32_t any = 0;
#pragma unroll
        for (int t = 0; t < GW; ++t) any |= fp4_far(vs[t]);
        if (__builtin_amdgcn_ballot_w64(any != 0)) { // uniform: NaN, or powers that f16 does not have
            any = 0;
#pragma unroll
            for (int t = 0; t < GW; ++t) any |= bytes_255(vs[t]);
            if (__builtin_amdgcn_ballot_w64(any != 0)) { // rows that are NaN
                uint32_t *of = nan_of + ((step & 1) * PAGES * PARTS + wave) * 17;
                if (lane == 0) nan_step[step & 1] = of[0] = (uint32_t)step + 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int t = 0; t < GW; ++t) bits |= (bytes_255(vs[t]) >> (8 * i) & 1u) << (vp * GW + t);
                    if (n == 0) of[1 + j * 4 + i] = bits;
                }
#pragma unroll
                for (int t = 0; t < GW; ++t) vs[t] ^= bytes_255(vs[t]) & 0x80808080u;
            }
            any = 0;
#pragma unroll
            for (int t = 0; t < GW; ++t) any |= fp4_far(vs[t]);
            if (__builtin_amdgcn_ballot_w64(any != 0)) { // uniform: far_pages takes all of it, from memory
                if (lane == 0) far_step[step & 1] = far_of[(step & 1) * PAGES * PARTS + wave] = (uint32_t)step + 1;
#pragma unroll
                for (int t = 0; t < GW; ++t) vc[t] = 0, vs[t] = 0x7f7f7f7fu;
            }
        }
        uint8_t *to = lds + L::V_AT + (step & 1) * L::V_BUF + (vd >> 1) * 2 * L::V_PAGE + lane * 16 + (vd & 1) * 8;
#pragma unroll
        for (int t = 0; t < GW; ++t) {
            const uint32_t w = vc[t], e4 = vs[t] - 0x01010101u * V_SHIFT;
            const uint32_t c0 = code_pair_f16<0>(w, e4 << 23), c1 = code_pair_f16<1>(w, e4 << 15), c2 = code_pair_f16<2>(w, e4 << 7), c3 = code_pair_f16<3>(w, e4 >> 1);
            uint8_t *at = to + (vp * GW + t) * 2048;
            *reinterpret_cast<u2 *>(at) = u2{__builtin_amdgcn_perm(c1, c0, 0x05040100u), __builtin_amdgcn_perm(c3, c2, 0x05040100u)};
            *reinterpret_cast<u2 *>(at + 1024) = u2{__builtin_amdgcn_perm(c1, c0, 0x07060302u), __builtin_amdgcn_perm(c3, c2, 0x07060302u)};
        }
    };
    // everything asked for with an ordinary load has arrived (the compiler does not know of the copies: see copy_to_lds)
    auto ids_here = [&]() __attribute__((always_inline)) { asm volatile("" : "+v"(ids)); };
    ask_ids(0);
    if (tid < 2) nan_step[tid] = far_step[tid] = 0;
    if (tid < 2 * PAGES * PARTS) nan_of[tid * 17] = far_of[tid] = 0; // (LDS holds what the launch before left)

    // ---- this wavefront's query tiles: rows side by side through LDS (V's buffers), a lane (slot n, group j) then has its 32 dims
    int my_limit[TILES], my_ws[TILES], t_ws_hi[TILES], t_lim_lo[TILES];
    bool t_on[TILES];
    int8v_t q_term[TILES][NB][5];
    uint32_t q_power[TILES][NB], q_last[TILES][NB]; // a byte each for the first four terms, the last one's
    float4_t *const raw = reinterpret_cast<float4_t *>(lds + L::V_AT) + wave * 16 * L::ROW;
    constexpr int ROW = L::ROW, LANES = ROW == 24 ? 32 : ROW, AT_ONCE = 64 / LANES, QL = 16 / AT_ONCE; // lanes of a row, rows of an instruction
    const int unit = lane % LANES;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        float4_t qv[NB][QL]; // every load of the tile in front of the first conversion
        const int s0 = wg_slot0 + (tw * TILES + t) * 16;
        t_on[t] = s0 < n_slots;
        const int my_slot = min(s0 + n, n_slots - 1);
        my_limit[t] = limit_of(my_slot);
        my_ws[t] = ws_of(my_slot);
        t_lim_lo[t] = limit_of(min(s0, n_slots - 1));
        t_ws_hi[t] = ws_of(min(s0 + 15, n_slots - 1));
#pragma unroll
        for (int i = 0; i < QL; ++i) {
            const float *qrow = a.q + context_row(g, kvh, min(s0 + i * AT_ONCE + lane / LANES, n_slots - 1)) * g.head_dim;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int d = b * 128 + unit * 4;
                if (a.q_vec) {
                    qv[b][i] = *reinterpret_cast<const float4_t *>(qrow + min(d, g.head_dim - 4));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) qv[b][i][e] = qrow[min(d + e, g.head_dim - 1)];
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int d = b * 128 + unit * 4;
#pragma unroll
            for (int i = 0; i < QL; ++i) {
                const int row = i * AT_ONCE + lane / LANES;
                float4_t v = qv[b][i];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = d + e < g.head_dim ? v[e] * a.qscale : 0.0f;
                if (LANES == ROW || unit < ROW) raw[row * ROW + (unit ^ (row & 7))] = v;
            }
            float16_t even, odd;
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4_t y = raw[n * ROW + ((min(j * 8, ROW - 8) + i) ^ (n & 7))];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    even[2 * i + e] = G >= 4 || j < G ? y[2 * e] : 0.0f;
                    odd[2 * i + e] = G >= 4 || j < G ? y[2 * e + 1] : 0.0f;
                    top = max(top, max(magnitude(even[2 * i + e]), magnitude(odd[2 * i + e])));
                }
            }
            // the first term's power is the smallest with the largest value <= 7.5 of it; a term leaves at most 2^-2, then 2^-7, 2^-12, 2^-17, 2^-22 of it,
            // 2^-23.9 of the largest value
            const int power = max((int)((top + 0x0fffffu) >> 23) - 2, 23);
            constexpr int down[5] = {0, 4, 9, 14, 19};
            q_last[t][b] = top >= 0x7f800000u ? 255u : (uint32_t)(power - 19);
            q_power[t][b] = top >= 0x7f800000u ? 0xffffffffu : (uint32_t)(power | (power - 4) << 8 | (power - 9) << 16) | (uint32_t)(power - 14) << 24;
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                const float scale = __uint_as_float((uint32_t)(power - down[k]) << 23);
                const u6 codes = to_fp6(even, odd, scale);
#pragma unroll
                for (int w = 0; w < 6; ++w) q_term[t][b][k][w] = (int)codes[w];
                q_term[t][b][k][6] = q_term[t][b][k][7] = 0;
                if (k < 4) {
                    const float32_t back = from_fp6(codes, scale);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        even[e] -= back[2 * e];
                        odd[e] -= back[2 * e + 1];
                    }
                }
            }
        }
    }
    ids_here();
    copy_k(0, 0, std::integral_constant<int, GP>{}, 1); // the first group's, into the second buffer
    copy_k(0, GP, std::integral_constant<int, PAGES>{}, 0);
    load_v(0);
    __syncthreads(); // (all have read their queries from V's buffers)
    convert_v(0);

    float4_t o[TILES][NT], neg_m[TILES];
    // a score whose bits reach thr moves the base, to 4 under it: any more than 8 above the base, or, of a slot without a key so far, whatever it is
    constexpr int UNSEEN = INT32_MIN, SEEN = 0x41000001;
    float m_base[TILES], l_run[TILES];
    int thr[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int u = 0; u < NT; ++u) o[t][u] = float4_t{0.f, 0.f, 0.f, 0.f};
        neg_m[t] = float4_t{0.f, 0.f, 0.f, 0.f};
        m_base[t] = l_run[t] = 0.0f;
        thr[t] = UNSEEN;
    }
    float4_t sa[TILES], sb[TILES];
    // pairs whose keys every slot of the wavefront attends
    int in0, in1, in2, in3;
    {
        int lo = t_ws_hi[0], hi = t_lim_lo[0];
#pragma unroll
        for (int t = 1; t < TILES; ++t) {
            lo = max(lo, t_ws_hi[t]);
            hi = min(hi, t_lim_lo[t]);
        }
        const Inner r = inner_entries<RING>(c, pb0, pb1, lo, hi);
        in0 = (r.o0 - pb0 + 1) >> 1;
        in1 = (r.o1 - pb0) >> 1;
        in2 = (r.n0 - pb0 + 1) >> 1;
        in3 = (r.n1 - pb0) >> 1;
    }
    auto mask = [&](int pair) __attribute__((always_inline)) {
        if ((pair >= in0 && pair < in1) || (RING && pair >= in2 && pair < in3)) return; // uniform
        const int it = 2 * pair, ea = entry(it), eb = entry(it + 1);
        const int pos_a = entry_pos<RING>(c, ea), pos_b = entry_pos<RING>(c, eb);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int lo_a = max(my_ws[t], entry_lo<RING>(c, ea)), hi_a = min(my_limit[t], entry_hi<RING>(c, ea));
            const int lo_b = max(my_ws[t], entry_lo<RING>(c, eb)), hi_b = min(my_limit[t], entry_hi<RING>(c, eb));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int pa = pos_a + j * 4 + e, pb = pos_b + j * 4 + e;
                sa[t][e] = it < n_it && pa >= lo_a && pa <= hi_a ? sa[t][e] : -INFINITY;
                sb[t][e] = it + 1 < n_it && pb >= lo_b && pb <= hi_b ? sb[t][e] : -INFINITY;
            }
        }
    };
    // (a positive float is a positive integer, every other one zero or negative)
    auto settle = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            int mi = max(max(__float_as_int(sa[t][0]), __float_as_int(sa[t][1])), __float_as_int(sa[t][2]));
            mi = max(max(mi, __float_as_int(sa[t][3])), __float_as_int(sb[t][0]));
            mi = max(max(mi, __float_as_int(sb[t][1])), __float_as_int(sb[t][2]));
            mi = max(mi, __float_as_int(sb[t][3]));
            if (__builtin_amdgcn_ballot_w64(mi >= thr[t])) {
                const float mx = fmaxf(fmaxf(fmaxf(sa[t][0], sa[t][1]), fmaxf(sa[t][2], sa[t][3])), fmaxf(fmaxf(sb[t][0], sb[t][1]), fmaxf(sb[t][2], sb[t][3])));
                const float top = rows_max(mx); // of the slot, relative to its base
                const bool unseen = thr[t] < 0;
                const float d = top > (unseen ? -INFINITY : 8.0f) ? top - 4.0f : 0.0f;
                const float alpha = unseen ? 1.0f : fast_exp2(-d);
                m_base[t] += d;
                neg_m[t] = float4_t{-m_base[t], -m_base[t], -m_base[t], -m_base[t]};
                thr[t] = unseen && top == -INFINITY ? UNSEEN : SEEN;
                l_run[t] *= alpha;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sa[t][e] -= d;
                    sb[t][e] -= d;
                }
                if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                    for (int u = 0; u < NT; ++u) o[t][u] *= alpha;
                }
            }
        }
    };
    // probabilities of the settled scores, as two f16 terms, in steps that stand between products: step q takes the exponential of score q and
    // splits those of scores q - 2 and q - 1
    float pr[TILES][2], prev[TILES];
    uint32_t hi4[TILES][4], lo4[TILES][4];
    constexpr float RAISED = 16.0f; // of weights as terms: the largest is then 2^8 to 2^12, a rounding to f16's last step 2^-33 of it at most
    auto prob_step = [&](int q) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            if (q > 0) {
                const int e = q - 1;
                l_run[t] += prev[t];
                pr[t][e & 1] = prev[t];
                if (e & 1) {
                    f16_terms(pr[t][0] * RAISED, pr[t][1] * RAISED, hi4[t][e >> 1], lo4[t][e >> 1]);
                }
            }
            if (q < 8) prev[t] = fast_exp2(q < 4 ? sa[t][q & 3] : sb[t][q & 3]);
        }
    };
    const int jk = G < 4 ? min(j, G - 1) : j; // (narrow heads: the lanes past the last group take it again, against queries of zero)
    uint32_t kc[2][NB][4], kp[2];
    // K of group `group`'s pair of this part
    auto ask_k = [&](int buf, int pos) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int d = pos * GP + half * 2 + h;
            const uint8_t *kt = lds + buf * L::K_BUF + d * L::K_PAGE, *pp = lds + buf * L::K_BUF + PAGES * L::K_PAGE + d * L::K_POWERS;
#pragma unroll
            for (int b = 0; b < NB; ++b) load_words<4>(kc[h][b], kt + ((4 * b + jk) * 16 + n) * 16);
            if constexpr (NB == 1) kp[h] = pp[jk * 16 + n];
            else if constexpr (NB == 2) kp[h] = reinterpret_cast<const uint16_t *>(pp)[j * 16 + n];
            else kp[h] = reinterpret_cast<const uint32_t *>(pp)[j * 16 + n];
        }
    };
    // V operands are asked for AHEAD of their products
    constexpr int AHEAD = NT < 4 ? NT : 4;
    u4 vr[AHEAD];
    auto ask_v = [&](const uint8_t *vt, int u) __attribute__((always_inline)) { vr[u % AHEAD] = *reinterpret_cast<const u4 *>(vt + u * 1024 + lane * 16); };
    // scores of the pair whose K is in the registers; the settled pair's probabilities between the products, and its first V operands at the end
    auto scores = [&](auto with_probs, const uint8_t *vt) __attribute__((always_inline)) {
        constexpr bool PROBS = decltype(with_probs)::value;
        __builtin_amdgcn_s_setprio(1); // (the SIMD's other wavefront is mostly in its second window, products almost alone)
        float4_t ns[2][TILES];
        int q = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int k = 4; k >= 0; --k) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int8v_t kk = {(int)kc[h][b][0], (int)kc[h][b][1], (int)kc[h][b][2], (int)kc[h][b][3], 0, 0, 0, 0};
                    const int kpow = (int)(kp[h] >> (8 * b));
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        const float4_t from = b == 0 && k == 4 ? neg_m[t] : ns[h][t];
                        ns[h][t] = k == 4   ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, q_term[t][b][4], from, 4, 2, 0, kpow, 0, (int)q_last[t][b])
                                   : k == 3 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, q_term[t][b][3], from, 4, 2, 0, kpow, 3, (int)q_power[t][b])
                                   : k == 2 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, q_term[t][b][2], from, 4, 2, 0, kpow, 2, (int)q_power[t][b])
                                   : k == 1 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, q_term[t][b][1], from, 4, 2, 0, kpow, 1, (int)q_power[t][b])
                                            : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kk, q_term[t][b][0], from, 4, 2, 0, kpow, 0, (int)q_power[t][b]);
                    }
                }
                if (PROBS) {
                    if (b == NB - 1 && k < 4) ask_v(vt, (3 - k) % AHEAD);
                    const int until = ((b * 5 + 5 - k) * 9) / (5 * NB); // steps done by the end of this beat
#pragma unroll
                    for (int s = 0; s < 9; ++s)
                        if (s >= q && s < until) prob_step(s);
                    q = until;
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            sa[t] = ns[0][t];
            sb[t] = ns[1][t];
        }
    };
    auto accumulate = [&](const uint8_t *vt, auto next_k) __attribute__((always_inline)) {
        f16x8_t ph[TILES], pl[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            ph[t] = __builtin_bit_cast(f16x8_t, u4{hi4[t][0], hi4[t][1], hi4[t][2], hi4[t][3]});
            pl[t] = __builtin_bit_cast(f16x8_t, u4{lo4[t][0], lo4[t][1], lo4[t][2], lo4[t][3]});
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const f16x8_t v = __builtin_bit_cast(f16x8_t, vr[u % AHEAD]);
#pragma unroll
            for (int t = 0; t < TILES; ++t) o[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[t], o[t][u], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < TILES; ++t) o[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[t], o[t][u], 0, 0, 0);
            if (u + AHEAD < NT) ask_v(vt, u + AHEAD);
            else if (u + AHEAD == NT) next_k();
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // a pair's pages whose V has powers that f16 does not have (convert_v left zeros): as bf16, from memory
    auto far_pages = [&](int step, int pp) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int d = (pp * HALVES + half) * 2 + h, it = step * PAGES + d, e = entry(it);
            const int pos = entry_pos<RING>(c, e) + j * 4, lo = max(wg_ws_lo, entry_lo<RING>(c, e)), hi = min(wg_lim_hi, entry_hi<RING>(c, e));
            uint32_t keep = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (it < n_it && pos + i >= lo && pos + i <= hi) keep |= 255u << (8 * i);
            const uint8_t *at = pool_of(it, true) + (uint64_t)(uint32_t)(RING ? fp4_ring_page(a, c, e) : (int)entry_place<false>(a, c, e)) * page_bytes;
            uint32_t terms[TILES][3][2]; // of 8 bits each, which leave 2^-24 of a weight; the least first
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f16x2_t a16 = __builtin_bit_cast(f16x2_t, hi4[t][2 * h + i]), b16 = __builtin_bit_cast(f16x2_t, lo4[t][2 * h + i]);
                    float x = ((float)a16[0] + (float)b16[0]) * P_SCALE, y = ((float)a16[1] + (float)b16[1]) * P_SCALE;
#pragma unroll
                    for (int k = 2; k >= 0; --k) {
                        terms[t][k][i] = bf16_pair(x, y);
                        x -= __uint_as_float(terms[t][k][i] << 16);
                        y -= __uint_as_float(terms[t][k][i] & 0xffff0000u);
                    }
                }
            }
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                if (__builtin_amdgcn_readfirstlane((int)far_of[((step & 1) * PAGES + d) * PARTS + part]) != step + 1) continue;
#pragma unroll
                for (int g0 = 0; g0 < GW / U; ++g0) {
                    uint32_t w[U];
                    load_words<U>(w, at + codes_at + ((part * (GW / U) + g0) * 64 + lane) * U * 4);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int grp = part * GW + g0 * U + u;
                        uint32_t e4 = *reinterpret_cast<const uint32_t *>(at + powers_at + (j * G + grp) * 4);
                        const uint32_t none = ~keep | bytes_255(e4); // (NaN: see nan_rows)
                        e4 = (e4 & ~none) | (none & 0x7f7f7f7fu);
                        const uint32_t c0 = code_pair<0>(w[u], e4 << 23), c1 = code_pair<1>(w[u], e4 << 15), c2 = code_pair<2>(w[u], e4 << 7), c3 = code_pair<3>(w[u], e4 >> 1);
                        // (the other page's keys are zeros)
                        const u4 first = {__builtin_amdgcn_perm(c1, c0, 0x05040100u), __builtin_amdgcn_perm(c3, c2, 0x05040100u), 0, 0};
                        const u4 second = {__builtin_amdgcn_perm(c1, c0, 0x07060302u), __builtin_amdgcn_perm(c3, c2, 0x07060302u), 0, 0};
#pragma unroll
                        for (int t = 0; t < TILES; ++t) {
#pragma unroll
                            for (int k = 0; k < 3; ++k) {
                                const bf16x8_t x = __builtin_bit_cast(bf16x8_t, u4{terms[t][k][0], terms[t][k][1], 0, 0});
                                o[t][2 * grp] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, first), x, o[t][2 * grp], 0, 0, 0);
                                o[t][2 * grp + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, second), x, o[t][2 * grp + 1], 0, 0, 0);
                            }
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };
    // the slots that attend rows that are NaN in the step's V: NaN in those groups of dims
    auto nan_rows = [&](int step) __attribute__((always_inline)) {
        for (int w = 0; w < PAGES * PARTS; ++w) {
            const uint32_t *of = nan_of + ((step & 1) * PAGES * PARTS + w) * 17;
            if (__builtin_amdgcn_readfirstlane((int)of[0]) != step + 1) continue;
            const int d = w / PARTS, it = step * PAGES + d, e = entry(it);
            if (HALVES > 1 && d % GP / 2 != half) continue;
            const int pos = entry_pos<RING>(c, e) + j * 4;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const int lo = max(my_ws[t], entry_lo<RING>(c, e)), hi = min(my_limit[t], entry_hi<RING>(c, e));
                uint32_t bits = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (it < n_it && pos + i >= lo && pos + i <= hi) bits |= of[1 + j * 4 + i];
                bits |= (uint32_t)__shfl_xor((int)bits, 16);
                bits |= (uint32_t)__shfl_xor((int)bits, 32);
#pragma unroll
                for (int u = 0; u < NT; ++u)
                    if (bits >> (u / 2) & 1u) o[t][u] += float4_t{NAN, NAN, NAN, NAN};
            }
        }
    };

    copies_landed();
    __syncthreads();
    ask_k(1, 0);
    scores(std::false_type{}, nullptr);
    mask(half);
    settle();
    ask_ids(PAGES);
    __syncthreads(); // the second buffer of K is free

    for (int step = 0; step < n_steps; ++step) {
        const int buf = step & 1;
        const bool far = __builtin_amdgcn_readfirstlane((int)far_step[buf]) == step + 1;
        if (step + 1 < n_steps) { // uniform
            ids_here();
            copy_k((step + 1) * PAGES, GP, std::integral_constant<int, PAGES>{}, buf ^ 1);
            load_v((step + 1) * PAGES);
            ask_ids((step + 2) * PAGES);
        }
        ask_k(buf, 0);
#pragma unroll
        for (int pp = 0; pp < SP; ++pp) {
            const int group = step * SP + pp;
            if (group >= n_groups) continue; // uniform
            const uint8_t *vt = lds + L::V_AT + buf * L::V_BUF + (pp * HALVES + half) * 2 * L::V_PAGE;
            scores(std::true_type{}, vt);
            accumulate(vt, [&]() __attribute__((always_inline)) {
                if (pp + 1 < SP) ask_k(buf, pp + 1);
            });
            if (far) far_pages(step, pp); // uniform
            mask((group + 1) * HALVES + half);
            settle();
        }
        if (__builtin_amdgcn_readfirstlane((int)nan_step[buf]) == step + 1) nan_rows(step);
        if (step + 1 < n_steps) convert_v(step + 1);
        copies_landed();
        __syncthreads();
    }

    // ---- the parts join their states through LDS; the first one has the result
    if constexpr (HALVES > 1) {
        float4_t *xo = reinterpret_cast<float4_t *>(lds);
        static_assert((HALVES - 1) * TW * TILES * (NT + 1) * 1024 <= L::NAN_AT, "the states fit the page buffers");
        const auto at = [&](int part, int t, int u) { return ((((part - 1) * TW + tw) * TILES + t) * (NT + 1) + u) * 64 + lane; };
        if (half > 0) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
#pragma unroll
                for (int u = 0; u < NT; ++u) xo[at(half, t, u)] = o[t][u];
                xo[at(half, t, NT)] = float4_t{thr[t] < 0 ? -INFINITY : m_base[t], l_run[t], 0.f, 0.f};
            }
        }
        __syncthreads();
        if (half > 0) return;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float w[HALVES], mx;
            w[0] = mx = thr[t] < 0 ? -INFINITY : m_base[t];
#pragma unroll
            for (int h = 1; h < HALVES; ++h) {
                w[h] = xo[at(h, t, NT)][0];
                mx = fmaxf(mx, w[h]);
            }
            const float m_safe = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) w[h] = fast_exp2(w[h] - m_safe);
            l_run[t] *= w[0];
#pragma unroll
            for (int h = 1; h < HALVES; ++h) l_run[t] += xo[at(h, t, NT)][1] * w[h];
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                o[t][u] *= w[0];
#pragma unroll
                for (int h = 1; h < HALVES; ++h) o[t][u] += xo[at(h, t, u)] * w[h];
            }
            m_base[t] = m_safe;
            thr[t] = mx == -INFINITY ? UNSEEN : SEEN;
        }
    }

    // ---- every wavefront writes its own slots
    const bool vec_ok = (g.head_dim & 3) == 0 && (a.splits_total > 1 || (reinterpret_cast<uintptr_t>(a.out) & 15) == 0);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const float l = rows_sum(l_run[t]) * (RAISED * P_SCALE);
        const int slot = wg_slot0 + (tw * TILES + t) * 16 + n;
        if (!t_on[t] || slot >= n_slots) continue;
        float *dst;
        float scale = 1.0f;
        if (a.splits_total == 1) {
            scale = 1.0f / l;
            dst = a.out + context_row(g, kvh, slot) * g.head_dim;
        } else {
            const long pidx = ((long)kvh * a.splits_total + split) * n_slots + slot;
            dst = a.part_o + pidx * g.head_dim;
            if (j == 0) {
                a.part_m[pidx] = thr[t] < 0 ? -INFINITY : m_base[t];
                a.part_l[pidx] = l;
            }
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const int col = u * 16 + j * 4;
            const float4_t v = o[t][u] * scale;
            if (vec_ok) {
                if (col < g.head_dim) *reinterpret_cast<float4_t *>(dst + col) = v;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (col + i < g.head_dim) dst[col + i] = v[i];
            }
        }
    }
}

// Query slots of a workgroup
int fp4_chunk_slots(int P, TileShape shape) {
    if (P > 256) return 64;
    if (shape == TileShape::two_tiles && P <= 128) return 256;
    return shape == TileShape::halves ? 64 : 128;
}

template <int P, int TILES, int WAVES, int HALVES, bool RING>
static hipError_t launch_chunk_of(const DecodeArgs &a, const ChunkPages &c, dim3 grid, hipStream_t s) {
    constexpr size_t lds = Fp4Chunk<P, WAVES, HALVES>::LDS;
    static std::atomic<uint64_t> lds_ok{0}; // per instantiation
    {
        hipError_t e = allow_full_lds(reinterpret_cast<const void *>(&fp4_chunk_kernel<P, TILES, WAVES, HALVES, RING>), lds_ok);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((fp4_chunk_kernel<P, TILES, WAVES, HALVES, RING>), grid, dim3(WAVES * 64), lds, s, a, c);
    return hipGetLastError();
}
template <int P, int TILES, int HALVES, int WAVES = 8>
static hipError_t launch_chunk(const DecodeArgs &a, const ChunkPages &c, dim3 grid, hipStream_t s) {
    return c.ring_pages > 0 ? launch_chunk_of<P, TILES, WAVES, HALVES, true>(a, c, grid, s) : launch_chunk_of<P, TILES, WAVES, HALVES, false>(a, c, grid, s);
}

hipError_t launch_fp4_chunk(const DecodeArgs &a, const ChunkPages &c, TileShape shape, hipStream_t s) {
    const int n_slots = a.n_queries * a.g.gqa, per_wg = fp4_chunk_slots(a.g.P, shape);
    const dim3 grid((unsigned)a.splits, (unsigned)a.g.kv_heads, (unsigned)((n_slots + per_wg - 1) / per_wg));
    switch (a.g.P) {
    case 32: return per_wg == 64 ? launch_chunk<32, 1, 2>(a, c, grid, s) : per_wg == 128 ? launch_chunk<32, 1, 1>(a, c, grid, s) : launch_chunk<32, 2, 1>(a, c, grid, s);
    case 64: return per_wg == 64 ? launch_chunk<64, 1, 2>(a, c, grid, s) : per_wg == 128 ? launch_chunk<64, 1, 1>(a, c, grid, s) : launch_chunk<64, 2, 1>(a, c, grid, s);
    case 96: return per_wg == 64 ? launch_chunk<96, 1, 2>(a, c, grid, s) : per_wg == 128 ? launch_chunk<96, 1, 1>(a, c, grid, s) : launch_chunk<96, 2, 1>(a, c, grid, s);
    case 128: return per_wg == 64 ? launch_chunk<128, 1, 2>(a, c, grid, s) : per_wg == 128 ? launch_chunk<128, 1, 1>(a, c, grid, s) : launch_chunk<128, 2, 1>(a, c, grid, s);
    case 256: return per_wg == 64 ? launch_chunk<256, 1, 2>(a, c, grid, s) : launch_chunk<256, 1, 1>(a, c, grid, s);
    case 512: return launch_chunk<512, 1, 1, 4>(a, c, grid, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace skv
