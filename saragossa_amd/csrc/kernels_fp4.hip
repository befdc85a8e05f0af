// gfx950 kernels of the 4-bit element (fp4_tile.h): rows stored as codes, read back, and attended.
#include "append_tile.h"
#include "fp4_tile.h"
#include "lds_copy.h"
#include "pre_kv.h"

namespace skv {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) float float4_t;
typedef __attribute__((ext_vector_type(16))) float float16_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u2;
typedef __attribute__((ext_vector_type(4))) uint32_t u4;
typedef __attribute__((ext_vector_type(6))) uint32_t u6;
typedef __attribute__((ext_vector_type(8))) int int8v_t;

namespace {

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// Four digits between -16 and 16, a byte each and 16 too large, as e2m3 codes of an eighth of them, side by side in 24 bits: sign and magnitude,
// which for whole eighths up to 2 is the code's last five bits as they stand.
__device__ __forceinline__ uint32_t fp6_codes_of(uint32_t u) {
    const uint32_t half = u >> 1, up = ((u | half) & 0x10101010u) >> 4, mask = (up << 8) - up; // not negative: 255
    const uint32_t pos = (u & 0x0f0f0f0fu) | (half & 0x10101010u), neg = 0x30303030u - u;
    const uint32_t c = (pos & mask) | (neg & ~mask);
    const uint32_t two = (c & 0x003f003fu) | (c >> 2 & 0x0fc00fc0u);
    return (two & 0xfffu) | (two >> 4 & 0xfff000u);
}

} // namespace

// ------------------------------------------------------------------------------------
// Rows stored: f32 rows -> codes and powers. Eight neighbouring lanes take a group of a row, four dims each, find its largest magnitude among
// themselves and convert; the group beside it is the wavefront's other half, so that rows are read 256 bytes at a time. K: the eight's
// 16 bits are the lane's 16 bytes of the matrix operand as they stand. V: a byte holds the dims c and c + 16, which lanes four apart exchange, and a
// word the byte of four rows, which lanes eight apart exchange; a quad of rows that the batch covers is stored as words, one that it
// shares with older rows as bytes.
// A workgroup takes PER times 256 such eighths of one (page, kv head), of K and of V, all loads in front of the first conversion. SAVE: what the
// page held goes to a page of its own first, every byte by the thread that writes in its place.
// ------------------------------------------------------------------------------------
struct Fp4Unit { // of a thread: which eighth of which group of which row
    int o, i, quad, grp;
    bool real; // (an odd number of groups leaves some of the last part's idle)
    __device__ __forceinline__ Fp4Unit(int groups, int part) {
        const int rest = (int)(threadIdx.x >> 5);
        o = threadIdx.x & 7;
        i = (threadIdx.x >> 3) & 3;
        quad = rest >> 1;
        grp = part * 2 + (rest & 1);
        real = grp < groups;
    }
    __device__ __forceinline__ int row() const { return quad * 4 + i; }
    __device__ __forceinline__ int dim() const { return grp * 32 + o * 4; }
};
constexpr long FP4_WGS = 4096; // workgroups from which each takes twice as much
static int fp4_parts(int P) { return (P / 32 + 1) / 2; }

template <int PER, bool SAVE = false>
__global__ __launch_bounds__(256) void store_fp4_kernel(AppendArgs a) {
    const Geom g = a.g;
    const int groups = g.P >> 5, kvh = blockIdx.y;
    // (the page's place by a vector load, in front of the rows: see append_tile)
    int logical = a.first_page + (int)blockIdx.x;
    if (a.ring_pages > 0 && logical >= a.ring_pages) logical -= a.ring_pages;
    int at = a.table ? logical : 0;
    asm("" : "+v"(at));
    const int asked = (a.table ? a.table : reinterpret_cast<const int32_t *>(a.k_src))[at]; // (no table: some valid address)
    const int row0 = (int)blockIdx.x * 16 - a.first_row; // batch row of the page's first row
    const int r_lo = max(-row0, 0), r_hi = min(16, a.n_rows - row0); // rows of the page in the batch
    const int kv_dim = g.kv_heads * g.head_dim, lane = threadIdx.x & 63;
    float x[2][PER][4];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const Fp4Unit u(groups, (int)blockIdx.z * PER + p);
        const int row = min(max(u.row(), r_lo), r_hi - 1), d = u.dim(); // clamped: every lane takes part in the exchanges
        const long from = (long)(row0 + row) * kv_dim + kvh * g.head_dim;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const float *src = (v ? a.v_src : a.k_src) + from;
            if (a.vec) { // uniform
                const float4_t y = *reinterpret_cast<const float4_t *>(src + min(d, g.head_dim - 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[v][p][e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[v][p][e] = src[min(d + e, g.head_dim - 1)];
            }
        }
    }
    const int page = __builtin_amdgcn_readfirstlane(a.table ? asked : logical);
    uint8_t *const kp = const_cast<uint8_t *>(fp4_powers(a.k_pool, g, page, kvh)), *const vp = const_cast<uint8_t *>(fp4_powers(a.v_pool, g, page, kvh));
    uint8_t *const kc = const_cast<uint8_t *>(fp4_codes(a.k_pool, g, page, kvh)), *const vc = const_cast<uint8_t *>(fp4_codes(a.v_pool, g, page, kvh));
    uint32_t held[PER][4]; // SAVE: what is there so far, K's codes, V's, their powers
    if constexpr (SAVE) {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const Fp4Unit u(groups, (int)blockIdx.z * PER + p);
            const int grp = min(u.grp, groups - 1), d = grp * 32 + u.o * 4;
            held[p][0] = *reinterpret_cast<const uint16_t *>(kc + k4_code(u.row(), d));
            held[p][1] = *reinterpret_cast<const uint32_t *>(vc + v4_code(g.P, u.quad * 4, grp * 32 + (u.o & 3) * 4 + u.i));
            held[p][2] = kp[k4_power(g.P, u.row(), grp)];
            held[p][3] = vp[v4_power(g.P, u.row(), grp)];
        }
    }
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const Fp4Unit u(groups, (int)blockIdx.z * PER + p);
        const int r = u.row(), d = u.dim();
        const bool in = u.real && r >= r_lo && r < r_hi;
        if constexpr (SAVE) {
            if (u.real) {
                uint16_t *const pools[2] = {a.k_save, a.v_save};
                uint8_t *codes[2], *powers[2];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    codes[v] = const_cast<uint8_t *>(fp4_codes(pools[v], g, blockIdx.x, kvh));
                    powers[v] = const_cast<uint8_t *>(fp4_powers(pools[v], g, blockIdx.x, kvh));
                }
                *reinterpret_cast<uint16_t *>(codes[0] + k4_code(r, d)) = (uint16_t)held[p][0];
                if (u.o < 4) *reinterpret_cast<uint32_t *>(codes[1] + v4_code(g.P, u.quad * 4, d + u.i)) = held[p][1];
                if (u.o == 0) {
                    powers[0][k4_power(g.P, r, u.grp)] = (uint8_t)held[p][2];
                    powers[1][v4_power(g.P, r, u.grp)] = (uint8_t)held[p][3];
                }
            }
        }
        uint32_t codes[2], power[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[v][p][e] = d + e < g.head_dim ? x[v][p][e] : 0.0f;
            codes[v] = fp4_codes_of(x[v][p], power[v]);
        }
        if (in) {
            *reinterpret_cast<uint16_t *>(kc + k4_code(r, d)) = (uint16_t)codes[0];
            if (u.o == 0) {
                kp[k4_power(g.P, r, u.grp)] = (uint8_t)power[0];
                vp[v4_power(g.P, r, u.grp)] = (uint8_t)power[1];
            }
        }
        const uint32_t other = (uint32_t)__shfl_xor((int)codes[1], 4);
        const uint32_t low = u.o < 4 ? codes[1] : other, high = u.o < 4 ? other : codes[1];
        const uint32_t mine = nibbles_apart(low) | nibbles_apart(high) << 4; // dims 4 (o % 4) .. of the row, each with the one 16 further
        uint32_t word = 0; // column 4 (o % 4) + i: byte q is row q of the quad
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t of_row = (uint32_t)__shfl((int)mine, (lane & ~24) | q << 3);
            word |= (of_row >> (8 * u.i) & 255u) << (8 * q);
        }
        if (u.o >= 4 || !u.real) continue;
        uint8_t *dst = vc + v4_code(g.P, u.quad * 4, d + u.i);
        if (u.quad * 4 >= r_lo && u.quad * 4 + 4 <= r_hi) {
            *reinterpret_cast<uint32_t *>(dst) = word;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (u.quad * 4 + q >= r_lo && u.quad * 4 + q < r_hi) dst[q] = (uint8_t)(word >> (8 * q));
        }
    }
}

hipError_t launch_store_fp4(const AppendArgs &a, hipStream_t s) {
    if (a.n_rows <= 0) return hipSuccess;
    AppendArgs b = append_placed(a);
    b.vec = b.vec && ((uintptr_t)a.v_src & 15) == 0;
    const long pages = (a.first_pos + a.n_rows + 15) / 16 - a.first_pos / 16;
    const int parts = fp4_parts(a.g.P);
    const bool two = parts % 2 == 0 && pages * a.g.kv_heads * parts > FP4_WGS;
    const dim3 grid((unsigned)pages, (unsigned)a.g.kv_heads, (unsigned)(two ? parts / 2 : parts));
    if (a.k_save) hipLaunchKernelGGL((store_fp4_kernel<1, true>), dim3(grid.x, grid.y, (unsigned)parts), dim3(256), 0, s, b);
    else if (two) hipLaunchKernelGGL(store_fp4_kernel<2>, grid, dim3(256), 0, s, b);
    else hipLaunchKernelGGL(store_fp4_kernel<1>, grid, dim3(256), 0, s, b);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------
// Rows read back as bf16, which holds every value exactly: the store's steps the other way round, with the same division of the work.
// ------------------------------------------------------------------------------------
template <int PER>
__global__ __launch_bounds__(256) void load_fp4_kernel(GatherArgs a, int vec) {
    const Geom g = a.g;
    const int groups = g.P >> 5, kvh = blockIdx.y, lane = threadIdx.x & 63;
    const long pos0 = (a.first_pos / 16 + blockIdx.x) * 16;
    const int page = a.table[slot_of(pos0, g.ring_rows) >> 4];
    const uint8_t *const kc = fp4_codes(a.k_pool, g, page, kvh), *const vc = fp4_codes(a.v_pool, g, page, kvh);
    const uint8_t *const kp = fp4_powers(a.k_pool, g, page, kvh), *const vp = fp4_powers(a.v_pool, g, page, kvh);
    uint32_t codes[2][PER], power[2][PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const Fp4Unit u(groups, (int)blockIdx.z * PER + p);
        const int grp = min(u.grp, groups - 1), d = grp * 32 + u.o * 4;
        codes[0][p] = *reinterpret_cast<const uint16_t *>(kc + k4_code(u.row(), d));
        codes[1][p] = *reinterpret_cast<const uint32_t *>(vc + v4_code(g.P, u.quad * 4, grp * 32 + (u.o & 3) * 4 + u.i)); // column 4 (o % 4) + i: byte q is row q
        power[0][p] = kp[k4_power(g.P, u.row(), grp)];
        power[1][p] = vp[v4_power(g.P, u.row(), grp)];
    }
    const int kv_dim = g.kv_heads * g.head_dim;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const Fp4Unit u(groups, (int)blockIdx.z * PER + p);
        const int d = u.dim();
        uint32_t mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t col = (uint32_t)__shfl((int)codes[1][p], (lane & ~24) | k << 3);
            mine |= (col >> (8 * u.i + (u.o < 4 ? 0 : 4)) & 15u) << (4 * k);
        }
        codes[1][p] = mine;
        const long row = pos0 + u.row() - a.first_pos;
        if (!u.real || row < 0 || row >= a.n_rows || d >= g.head_dim) continue;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            uint16_t *out = v ? a.v_dst : a.k_dst;
            if (!out) continue; // uniform
            const uint32_t e4 = power[v][p] << 23, w[2] = {code_pair<0>(codes[v][p], e4), code_pair<1>(codes[v][p], e4)};
            uint16_t *dst = out + row * kv_dim + kvh * g.head_dim + d;
            if (vec) { // uniform
                __builtin_nontemporal_store(u2{w[0], w[1]}, reinterpret_cast<u2 *>(dst));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < g.head_dim) dst[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            }
        }
    }
}

hipError_t launch_load_fp4(const GatherArgs &a, hipStream_t s) {
    if (a.n_rows <= 0) return hipSuccess;
    const int vec = a.g.head_dim % 4 == 0 && (((uintptr_t)a.k_dst | (uintptr_t)a.v_dst) & 7) == 0;
    const long pages = (a.first_pos + a.n_rows + 15) / 16 - a.first_pos / 16;
    const int parts = fp4_parts(a.g.P);
    const bool two = parts % 2 == 0 && pages * a.g.kv_heads * parts > FP4_WGS;
    const dim3 grid((unsigned)pages, (unsigned)a.g.kv_heads, (unsigned)(two ? parts / 2 : parts));
    if (two) hipLaunchKernelGGL(load_fp4_kernel<2>, grid, dim3(256), 0, s, a, vec);
    else hipLaunchKernelGGL(load_fp4_kernel<1>, grid, dim3(256), 0, s, a, vec);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------
// Attention over the codes: 16 query slots (row, head of the group) of one kv head against a range of the pages, as (o, m, l) or, unsplit, the
// context. The wavefronts of a workgroup hold the same slots and walk the page pairs in turn.
//
// S^T = K . Q^T takes the codes as they lie in memory: v_mfma_scale_f32_16x16x128_f8f6f4 with K as e2m1 (a lane's 16 bytes are a row's 32 dims of
// a group, its power a byte of its own) and the queries, times log2(e) / sqrt(head_dim), as five terms in e2m3 with a power a group and term:
// digits of base 32 of the values as whole numbers of 25 bits, off by at most 2^-24 of the group's largest value (as exact as products in 32 bits, but
// where the keys are small in a dim of the queries some thirty times the others: at 100 times 2.7e-6 off, at 1000 2.3e-5). Five such products of 128
// dims take 80 cycles, two of bf16 (eight instructions of 32 dims, for queries of 16 bits) 128, and the codes would have to be converted.
// O^T += V^T . P^T sums over keys, whose powers differ, so V is converted to f16 (exact, but for powers that f16 does not have, see fp4_far) in
// registers, per page and group of dims four conversions, four scales and four byte selections for eight values a lane, and P is two f16
// terms; a pair of pages is the 32 keys of v_mfma_f32_16x16x32_f16. A pair with other powers is multiplied in bf16, P in three terms (chunks of heads to 128 dims: two).
// Contexts are 2e-7 from 64 bits (2-norm, relative), 3e-7 over 32768 rows; four terms and two bf16 ones left 2.6e-6, for 4 to 10 % less time.
//
// What bounds it: over long contexts memory, 34.8 MB of 32000 rows of q32/kv8/hd128 in 14.6 us with the merge (a bf16 layer 24.9), 69.6 of
// q16/kv8/hd256 in 20.2 (45.1); over short ones the chain of table, pages, products, states and a second launch: 600 to 2000 rows 7.6 and
// 8.9 us, 100 rows 5.3 and 6.4 (bf16, 2000 rows: 7.3 and 8.4). Six rows over 8192 of q16/kv2/hd256 15.9.
// ------------------------------------------------------------------------------------
template <int P>
struct Fp4Tile {
    static constexpr int G = P / 32, U = fp4_quad(P), NB = (P + 127) / 128, VL = G / U;
};
// LDS in bytes: the queries' terms ([NB][5 terms][64 lanes][6 words]) and powers ([NB][64]); of the new rows, per row, K codes, V codes, K
// powers, V powers; then per wavefront DEPTH pairs of pages, and in their place, when all are consumed, its state.
template <int P, int WAVES>
struct Fp4Lds {
    static constexpr int NB = Fp4Tile<P>::NB, BLOCK = (5 * 6 + 1) * 64 * 4;
    static constexpr int DEPTH = 2;
    static constexpr int PAIR = 34 * P; // codes of K a, K b, V a, V b, then their powers
    static constexpr int STATE = 16 * (P + 6) * 4; // [16 slots][P + 4], m, l
    static constexpr int WAVE = DEPTH * PAIR > STATE ? DEPTH * PAIR : STATE;
    static constexpr int NEW_ROW = P + 2 * (P / 32);
    // (heads above 256 dims: no room for the queries beside the pairs, they lie in the wavefronts' second pairs until all have read them)
    static constexpr bool SHARED = P > 256;
    static_assert(!SHARED || (NB <= WAVES && BLOCK <= PAIR && DEPTH == 2), "a block of the queries in a wavefront's second pair");
    __host__ __device__ static constexpr int pairs(int new_rows) { return (SHARED ? 0 : NB * BLOCK) + (new_rows * NEW_ROW + 15) / 16 * 16; }
    __host__ __device__ static constexpr int block(int b, int new_rows) { return SHARED ? pairs(new_rows) + b * WAVE + PAIR : b * BLOCK; }
    static constexpr size_t bytes(int new_rows) { return (size_t)pairs(new_rows) + (size_t)WAVES * WAVE; }
    static_assert((SHARED ? 0 : NB * BLOCK) + MQ_APPEND_ROWS * NEW_ROW + 16 + WAVES * WAVE <= 160 * 1024, "it all fits a compute unit's LDS");
};
// MQ: more than one query row, or more than 16 heads to a kv head: slots are (row, head) pairs, 16 to a workgroup (grid z). ROWS: the launch
// stores the chunk's rows itself, at most MQ_APPEND_ROWS of them, as a decode step's does its one. PRE: a step whose queries and new K row are
// normed and rotated here, from LDS that belongs to the wavefronts' second pairs until the first barrier behind it (the
// pairs lie by depth then, the states of the wavefronts over both behind one more barrier). A step of q32/kv8/hd128 over 2000 rows from its
// projections: 9.5 us, 14.2 with norm, rotation and append as launches of their own; of q16/kv2/hd256, gated, 12.2 and 18.1. (The
// step alone: 7.6 and 9.3. The chain load, ordered sum, rotation, digits is longer than the first pages' way.)
template <int P, int WAVES, bool MQ, bool RING, bool ROWS = false, bool PRE = false>
__device__ __forceinline__ void fp4_attention_body(const DecodeArgs &a, const ChunkPages *c, const int split, const int kvh, const int tile_z) {
    using T = Fp4Tile<P>;
    constexpr int THREADS = WAVES * 64, G = T::G, U = T::U, NB = T::NB, VL = T::VL, NT = P / 16, OSTRIDE = P + 4;
    const Geom g = a.g;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_slots = (MQ ? a.n_queries : 1) * g.gqa;
    const int tile = MQ ? longest_first(n_slots, 16, tile_z) : 0;
    const int rows = min(16, n_slots - tile * 16);
    const int my_slot = min(tile * 16 + n, n_slots - 1);
    // the slot's last position and its first
    auto limit_of = [&](int slot) { return a.q_pos0 + (MQ ? slot_row(g, slot) : 0); };
    auto start_of = [&](int slot) { return a.window > 0 ? max(a.window_start, limit_of(slot) + 1 - a.window) : a.window_start; };
    const int my_limit = limit_of(my_slot), my_ws = start_of(my_slot);
    const int lim_lo = limit_of(tile * 16), lim_hi = limit_of(tile * 16 + rows - 1);
    const int ws_lo = start_of(tile * 16), ws_hi = start_of(tile * 16 + rows - 1);

    // The pages as a list in the order of positions: entry e < n_old is table[start + e] (less ring_pages past the ring's end), whose first
    // row has position pos0 + 16 e; behind them (RING) those of the chunk's own rows. (Of a ring some lie outside the layer, see ChunkPages.)
    const int pos0 = a.page_first * 16, n_old = RING ? c->n_old : INT32_MAX;
    const int apart_lo = RING ? c->apart_lo : 0, apart_hi = RING ? c->apart_hi : 0;
    auto entry_pos = [&](int e) { return RING && e >= n_old ? c->new_first + (e - n_old) * 16 : pos0 + e * 16; };
    auto entry_of = [&](int pos) { return RING && pos >= c->new_pos0 ? n_old + ((pos - c->new_first) >> 4) : max(pos - pos0, 0) >> 4; };
    const int e_lo = entry_of(ws_lo), e_hi = entry_of(lim_hi) + 1;
    const unsigned span = (unsigned)(e_hi - e_lo);
    const int pb0 = e_lo + (int)(((unsigned)split * span) / (unsigned)a.splits);
    const int pb1 = e_lo + (int)(((unsigned)(split + 1) * span) / (unsigned)a.splits);
    // this wavefront's pairs are pb0 + 2 (wave + it * WAVES)
    const int pairs = (pb1 - pb0 + 1) >> 1, n_it = pairs > wave ? (pairs - wave + WAVES - 1) / WAVES : 0;
    // place of an entry in the table
    auto place = [&](int e) __attribute__((always_inline)) {
        int at = a.ring_base + e;
        if (at >= a.ring_t) at -= a.ring_t;
        return max(at, 0);
    };
    // physical pages of the next 32 pairs, one a lane
    int ids = 0;
    auto fetch_ids = [&](int it) __attribute__((always_inline)) {
        const int e = min(pb0 + 2 * (wave + (it + (lane >> 1)) * WAVES) + (lane & 1), e_hi - 1);
        ids = RING ? fp4_ring_page(a, *c, e) : a.table[place(e)];
    };
    fetch_ids(0);

    // ---- the rows that the launch stores. A decode step's one: the wavefront that walks its page converts it, an eighth of a group a lane.
    // A chunk's: every workgroup that walks a page of theirs converts them all, and the last tile of slots, which sees all of them, stores
    // them. The codes stay in LDS, from where a wavefront patches what it has loaded.
    using L = Fp4Lds<P, WAVES>;
    constexpr bool NEW = !MQ || ROWS;
    // (PRE: V's groups alone, behind K's)
    constexpr int BY = ROWS ? THREADS : 64, MOST = ROWS ? MQ_APPEND_ROWS : 1, FIRST = PRE ? G : 0, NU = ((MOST * 2 * G - FIRST) * 8 + BY - 1) / BY;
    const int C = ROWS ? a.n_queries : 1;
    const int p_new = a.len - C, e_new = (p_new - pos0) >> 4, e_last = (a.len - 1 - pos0) >> 4;
    const bool appends = NEW && a.k_new != nullptr && e_last >= pb0 && e_new < pb1;
    const int w_new = ((e_new - pb0) >> 1) % WAVES; // (of a step)
    const bool converts = appends && (ROWS || wave == w_new), stores = tile == (n_slots - 1) / 16;
    const int by = ROWS ? tid : lane;
    float nx[NU][4];
    int page_a = 0, page_b = 0;
    using Pre = PreKvStage<P, THREADS>;
    Pre pre;
    float k_row[Pre::NE];
    if constexpr (PRE) {
        if (appends) page_a = a.table[place(min(max(e_new, 0), e_hi - 1))]; // uniform
#pragma unroll
        for (int u = 0; u < Pre::NE; ++u) {
            k_row[u] = 0.0f;
            if (appends && tid + u * THREADS < g.head_dim) k_row[u] = a.k_new[kvh * g.head_dim + tid + u * THREADS];
        }
        pre.load(a, kvh, rows, a.q_head_stride > 0 ? a.q_head_stride : g.head_dim, tid);
    }
    if constexpr (NEW) {
        if (converts) { // uniform
            const bool vec = (g.head_dim & 3) == 0 && ((reinterpret_cast<uintptr_t>(a.k_new) | reinterpret_cast<uintptr_t>(a.v_new)) & 15) == 0;
            if (!PRE) page_a = a.table[place(min(max(e_new, 0), e_hi - 1))];
            page_b = ROWS ? a.table[place(min(max(e_last, 0), e_hi - 1))] : page_a;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int idx = FIRST + ((by + u * BY) >> 3), v = idx >= C * G, row = min((idx - v * C * G) / G, C - 1), d = (idx % G) * 32 + (tid & 7) * 4;
                const float *src = (v ? a.v_new : a.k_new) + ((long)row * g.kv_heads + kvh) * g.head_dim;
                if (vec) {
                    const float4_t x = *reinterpret_cast<const float4_t *>(src + min(d, g.head_dim - 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) nx[u][e] = x[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) nx[u][e] = src[min(d + e, g.head_dim - 1)];
                }
            }
        }
    }
    // ---- queries: four dims of a slot a thread, as eighths of a group (loads side by side: with a lane's 32 dims loaded by the lane, every lane
    // on lines of its own, such loads were 1 to 2 us of a step)
    constexpr int QU = (16 * P / 4 + THREADS - 1) / THREADS;
    float4_t x[QU];
#pragma unroll
    for (int u = 0; u < (PRE ? 0 : QU); ++u) {
        const int idx = tid + u * THREADS, slot = (idx >> 3) / G, d = (idx >> 3) % G * 32 + (tid & 7) * 4;
        x[u] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (slot < rows) {
            const float *qrow = a.q + (MQ ? context_row(g, kvh, tile * 16 + slot) : (long)(kvh * g.gqa + slot)) * g.head_dim;
            if (a.q_vec) {
                x[u] = *reinterpret_cast<const float4_t *>(qrow + min(d, g.head_dim - 4));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][e] = qrow[min(d + e, g.head_dim - 1)];
            }
        }
    }

    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    uint8_t *new_rows = lds + (L::SHARED ? 0 : NB * L::BLOCK);
    constexpr int NEW_ROW = L::NEW_ROW, AT_V = P / 2, AT_KP = P, AT_VP = P + G; // in a new row
    const int n_new = NEW ? C : 0;
    constexpr int STEP = PRE ? WAVES * L::PAIR : L::PAIR; // from one of a wavefront's pairs to the next
    const int mine_off = L::pairs(n_new) + wave * (PRE ? L::PAIR : L::WAVE);
    uint8_t *const mine = lds + mine_off; // this wavefront's pairs
    const uint32_t mine_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds + (uint32_t)mine_off;
    static_assert(!PRE || (!MQ && !L::SHARED && Pre::LDS_FLOATS * 4 <= (size_t)WAVES * L::PAIR), "norm and rotation in the second pairs' place");
    const int jk = G < 4 ? min(j, G - 1) : j; // (narrow heads: the lanes past the last group take it again, against queries of zero)

    // A pair's copies to LDS: COPIES instructions. The heads' codes are whole KiBs from 128 dims on; below, and the powers always, a lane of an instruction
    // may belong to any of the four tiles (K a, K b, V a, V b).
    constexpr int CODE_COPIES = P >= 128 ? 4 * NB : P / 32, POWER_WORDS = P / 8, POWER_COPIES = (4 * POWER_WORDS + 63) / 64;
    constexpr int COPIES = CODE_COPIES + POWER_COPIES;
    const uint32_t page_bytes = (uint32_t)g.page_elems * 2;
    const size_t codes_at = (size_t)kvh * fp4_code_bytes(P), powers_at = (size_t)g.kv_heads * fp4_code_bytes(P) + (size_t)kvh * fp4_power_bytes(P);
    // where a lane's part of an instruction lies: in page a or b, so far from the page's start, of K's pool or V's
    struct Part {
        const uint8_t *from;
        bool second, v;
    };
    auto part = [&](int u, int units, int bytes, size_t at) __attribute__((always_inline)) {
        const int t = u / units;
        const bool v = t >= 2;
        return Part{reinterpret_cast<const uint8_t *>(v ? a.v_pool : a.k_pool) + at + (u - t * units) * bytes, (t & 1) != 0, v};
    };
    Part code_part[P >= 128 ? 1 : CODE_COPIES], power_part[POWER_COPIES];
    if constexpr (P < 128) {
#pragma unroll
        for (int i = 0; i < CODE_COPIES; ++i) code_part[i] = part(i * 64 + lane, P / 2, 16, codes_at);
    }
#pragma unroll
    for (int i = 0; i < POWER_COPIES; ++i) power_part[i] = part(min(i * 64 + lane, 4 * POWER_WORDS - 1), POWER_WORDS, 4, powers_at);
    auto copy_pair = [&](int it) __attribute__((always_inline)) {
        const uint32_t pa = (uint32_t)__builtin_amdgcn_readlane(ids, (2 * it) & 63), pb = (uint32_t)__builtin_amdgcn_readlane(ids, (2 * it + 1) & 63);
        const int e0 = pb0 + 2 * (wave + it * WAVES);
        const int ea = min(e0, e_hi - 1), eb = min(e0 + 1, e_hi - 1);
        const bool apart_a = RING && ea >= apart_lo && ea < apart_hi, apart_b = RING && eb >= apart_lo && eb < apart_hi;
        const uint32_t to = mine_at + (uint32_t)((it % L::DEPTH) * STEP);
        const auto address = [&](const Part &p) __attribute__((always_inline)) {
            const uint8_t *from = p.from + (uint64_t)(p.second ? pb : pa) * page_bytes;
            if constexpr (RING) {
                if (p.second ? apart_b : apart_a) from += p.v ? (const uint8_t *)c->v_new - (const uint8_t *)a.v_pool : (const uint8_t *)c->k_new - (const uint8_t *)a.k_pool;
            }
            return from;
        };
        if constexpr (P >= 128) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const bool apart = t & 1 ? apart_b : apart_a;
                const uint16_t *pool = t >= 2 ? (apart ? c->v_new : a.v_pool) : (apart ? c->k_new : a.k_pool);
                const uint8_t *from = reinterpret_cast<const uint8_t *>(pool) + codes_at + (uint64_t)(t & 1 ? pb : pa) * page_bytes;
#pragma unroll
                for (int b = 0; b < NB; ++b) MQ ? copy_to_lds(from, (uint32_t)lane * 16, to + t * 8 * P, b) : copy_to_lds_once(from, (uint32_t)lane * 16, to + t * 8 * P, b);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CODE_COPIES; ++i) gather_to_lds(address(code_part[i]), to + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < POWER_COPIES; ++i)
            if (i * 64 + 64 <= 4 * POWER_WORDS || i * 64 + lane < 4 * POWER_WORDS) gather_words_to_lds(address(power_part[i]), to + 32 * P + i * 256);
    };
    // everything asked for so far has arrived (the compiler does not know of the copies: a wait of its own behind them would be for all of them)
    asm volatile("" : "+v"(ids), "+v"(page_a), "+v"(page_b));
    if constexpr (NEW) {
#pragma unroll
        for (int u = 0; u < NU; ++u) asm volatile("" : "+v"(nx[u][0]), "+v"(nx[u][1]), "+v"(nx[u][2]), "+v"(nx[u][3]));
    }
    if constexpr (PRE) {
#pragma unroll
        for (int u = 0; u < Pre::U; ++u) asm volatile("" : "+v"(pre.q[u]));
#pragma unroll
        for (int u = 0; u < Pre::NE; ++u) asm volatile("" : "+v"(pre.wq[u]), "+v"(pre.wk[u]), "+v"(pre.rot[u]), "+v"(k_row[u]));
    } else {
#pragma unroll
        for (int u = 0; u < QU; ++u) asm volatile("" : "+v"(x[u]));
    }
    if (0 < n_it) copy_pair(0); // uniform

    // an eighth of a group of a new row, to LDS and, from the tile that stores, to the page: K's, V's
    auto row_pool = [&](int v, int row, uint8_t *&codes, uint8_t *&powers) __attribute__((always_inline)) {
        const int e = (p_new + row - pos0) >> 4, page = e == e_new ? page_a : page_b;
        uint16_t *pool = const_cast<uint16_t *>(v ? a.v_pool : a.k_pool);
        codes = const_cast<uint8_t *>(fp4_codes(pool, g, page, kvh)), powers = const_cast<uint8_t *>(fp4_powers(pool, g, page, kvh));
        return stores && e >= pb0 && e < pb1;
    };
    auto k_eighth = [&](int row, int t, int o8, uint32_t codes, uint32_t power) __attribute__((always_inline)) {
        uint8_t *cp, *pp, *to = new_rows + row * NEW_ROW;
        const bool store = row_pool(0, row, cp, pp);
        const int r = (p_new + row) & 15;
        *reinterpret_cast<uint16_t *>(to + t * 16 + o8 * 2) = (uint16_t)codes;
        if (o8 == 0) to[AT_KP + t] = (uint8_t)power;
        if (store) {
            *reinterpret_cast<uint16_t *>(cp + k4_code(r, t * 32 + o8 * 4)) = (uint16_t)codes;
            if (o8 == 0) pp[k4_power(P, r, t)] = (uint8_t)power;
        }
    };
    auto v_eighth = [&](int row, int t, int o8, uint32_t codes, uint32_t other, uint32_t power) __attribute__((always_inline)) {
        if (o8 >= 4) return;
        uint8_t *cp, *pp, *to = new_rows + row * NEW_ROW;
        const bool store = row_pool(1, row, cp, pp);
        const int r = (p_new + row) & 15;
        const uint32_t word = nibbles_apart(codes) | nibbles_apart(other) << 4;
        *reinterpret_cast<uint32_t *>(to + AT_V + t * 16 + o8 * 4) = word;
        if (o8 == 0) to[AT_VP + t] = (uint8_t)power;
        if (store) {
#pragma unroll
            for (int k = 0; k < 4; ++k) cp[v4_code(P, r, t * 32 + o8 * 4 + k)] = (uint8_t)(word >> (8 * k));
            if (o8 == 0) pp[v4_power(P, r, t)] = (uint8_t)power;
        }
    };
    auto convert_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int idx = FIRST + ((by + u * BY) >> 3), v = idx >= C * G, row = (idx - v * C * G) / G, t = idx % G, o8 = tid & 7, d = t * 32 + o8 * 4;
            const bool real = idx < 2 * C * G;
#pragma unroll
            for (int e = 0; e < 4; ++e) nx[u][e] = real && d + e < g.head_dim ? nx[u][e] : 0.0f;
            uint32_t power;
            const uint32_t codes = fp4_codes_of(nx[u], power);
            const uint32_t other = (uint32_t)__shfl_xor((int)codes, 4);
            if (!real) continue;
            if (!v) k_eighth(row, t, o8, codes, power);
            else v_eighth(row, t, o8, codes, other, power);
        }
    };
    auto no_query = [&](int slot, int t) __attribute__((always_inline)) { // (nothing reads what becomes of it)
        reinterpret_cast<uint32_t *>(lds + L::block(t >> 2, n_new))[5 * 6 * 64 + (t & 3) * 16 + slot] = 0;
    };
    // an eighth of a group of a slot's queries, to its place among the terms
    auto query_eighth = [&](int slot, int t, int o8, float4_t y) __attribute__((always_inline)) {
        uint32_t *const to = reinterpret_cast<uint32_t *>(lds + L::block(t >> 2, n_new)); // of the block, lane (slot, t % 4)
        const int at = (t & 3) * 16 + slot;
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __uint_as_float(max(__float_as_uint(top), magnitude(y[e])));
        const uint32_t most = max_of_8(magnitude(top * a.qscale));
        // the values as whole numbers of 25 bits, at most 2^24 (a float's own bits), in digits of base 32 between -16 and 15 (the first: 16), here
        // each 16 too large
        const int power = max((int)(most >> 23), 23);
        const float scale = __uint_as_float((uint32_t)(277 - power) << 23); // (times qscale it might not be finite)
        uint32_t digits[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) digits[e] = (uint32_t)((int)__builtin_rintf(y[e] * a.qscale * scale) + 16 * (1 + 32 + 1024 + 32768 + 1048576));
#pragma unroll
        for (int k = 0; k < 5; ++k) {
            uint32_t four = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) four |= (k == 0 ? digits[e] >> 20 & 63u : digits[e] >> (20 - 5 * k) & 31u) << (8 * e);
            const uint32_t codes = fp6_codes_of(four); // 24 bits; four lanes' are three words
            const uint32_t next = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)codes, 0xf9, 0xf, 0xf, false); // of the lane after
            const int o4 = o8 & 3;
            if (o4 < 3) to[(k * 64 + at) * 6 + (o8 >> 2) * 3 + o4] = codes >> (8 * o4) | next << (24 - 8 * o4);
        }
        if (o8 == 0)
            to[5 * 6 * 64 + at] = most >= 0x7f800000u ? 0xffffffffu : (uint32_t)(power | (power - 5) << 8 | (power - 10) << 16) | (uint32_t)(power - 15) << 24;
    };
    if constexpr (PRE) {
        float *const pre_lds = reinterpret_cast<float *>(lds + L::pairs(n_new) + WAVES * L::PAIR);
        pre.stage(pre_lds, a, rows, k_row, tid);
        for (int i = rows * G + tid; i < 16 * G; i += THREADS) no_query(i / G, i % G);
        const int n_rows = rows + (appends ? 1 : 0);
        __syncthreads();
        Pre::scales(pre_lds, a, rows, n_rows, tid);
        __syncthreads();
        Pre::each(pre_lds, a, rows, n_rows, tid, [&](int r, int c4, float4_t y) __attribute__((always_inline)) {
            if (r < rows) { // (eight lanes alike)
                query_eighth(r, c4 >> 3, c4 & 7, y);
            } else {
                float z[4] = {y[0], y[1], y[2], y[3]};
                uint32_t power;
                const uint32_t codes = fp4_codes_of(z, power);
                k_eighth(0, c4 >> 3, c4 & 7, codes, power);
            }
        });
    } else {
#pragma unroll
        for (int u = 0; u < QU; ++u) {
            const int idx = tid + u * THREADS, slot = (idx >> 3) / G, t = (idx >> 3) % G, o8 = tid & 7, d = t * 32 + o8 * 4;
            if (slot >= rows) {
                if (slot < 16 && o8 == 0) no_query(slot, t);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][e] = d + e < g.head_dim ? x[u][e] : 0.0f;
            query_eighth(slot, t, o8, x[u]);
        }
    }
    if constexpr (ROWS) {
        if (converts) convert_rows(); // uniform
    }
    __syncthreads();
    if constexpr (NEW && !ROWS) {
        if (converts) convert_rows(); // uniform (for itself)
    }
    int8v_t q_term[NB][5];
    uint32_t q_power[NB], q_last[NB]; // a byte each for the first four terms, the last one's
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t *terms = reinterpret_cast<const uint32_t *>(lds + L::block(b, n_new));
        q_power[b] = G >= 4 || j < G ? terms[5 * 6 * 64 + lane] : 0;
        q_last[b] = q_power[b] == 0xffffffffu ? 255u : (uint32_t)max((int)(q_power[b] & 255u) - 20, 0);
#pragma unroll
        for (int t = 0; t < 5; ++t) {
#pragma unroll
            for (int w = 0; w < 6; ++w) q_term[b][t][w] = G >= 4 || j < G ? (int)terms[(t * 64 + lane) * 6 + w] : 0;
            q_term[b][t][6] = q_term[b][t][7] = 0;
        }
    }
    if constexpr (L::SHARED) __syncthreads();
    // (not with the first pair: a compute unit accepts requests as fast as memory answers, and no wavefront passes the barrier before its own
    // are accepted)
    if (1 < n_it) copy_pair(1);

    float4_t o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = float4_t{0.f, 0.f, 0.f, 0.f};
    float b_run = -INFINITY, l_run = 0.0f; // what weights are relative to, their sum

    // a pair whose place in LDS has been read
    auto next_pair = [&](int it) __attribute__((always_inline)) {
        if (it >= n_it) return; // uniform
        if (((it) & 31) == 0) {
            fetch_ids(it);
            asm volatile("" : "+v"(ids)); // (waited for here: where the paths join it would be for every pair's copies)
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (all of this one is read)
        copy_pair(it);
    };
    for (int it = 0; it < n_it; ++it) {
        const int e0 = pb0 + 2 * (wave + it * WAVES);
        const int ea = entry_pos(e0), eb = entry_pos(min(e0 + 1, e_hi - 1));
        // ---- the pair, from LDS: the copies behind its own may still be on their way
        if (it + L::DEPTH <= n_it) copies_left<(L::DEPTH - 1) * COPIES>(); // uniform
        else copies_landed();
        const uint8_t *const pair = mine + (it % L::DEPTH) * STEP;
        uint32_t kc[2][NB][4], kp[2], vc[2][G], vp[2][G];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int b = 0; b < NB; ++b) load_words<4>(kc[h][b], pair + h * 8 * P + ((4 * b + jk) * 16 + n) * 16);
            const uint8_t *pp = pair + 32 * P + h * (P / 2);
            if constexpr (NB == 1) kp[h] = pp[jk * 16 + n];
            else if constexpr (NB == 2) kp[h] = reinterpret_cast<const uint16_t *>(pp)[j * 16 + n];
            else kp[h] = reinterpret_cast<const uint32_t *>(pp)[j * 16 + n];
        }
        const bool patches = NEW && appends && e0 + 1 >= e_new && e0 <= e_last; // uniform: the new rows' codes, from LDS
        auto take_v = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int v = 0; v < VL; ++v) {
                    uint32_t w[U];
                    load_words<U>(w, pair + (2 + h) * 8 * P + (v * 64 + lane) * U * 4);
#pragma unroll
                    for (int u = 0; u < U; ++u) vc[h][v * U + u] = w[u];
                }
                load_words<G>(vp[h], pair + 33 * P + h * (P / 2) + j * G * 4);
            }
            if constexpr (NEW) {
                if (patches) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int from = entry_pos(e0 + h) - p_new;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int vrow = from + j * 4 + i;
                            if (vrow < 0 || vrow >= C) continue;
                            const uint8_t *to = new_rows + vrow * NEW_ROW;
                            const uint32_t keep = ~(255u << (8 * i));
#pragma unroll
                            for (int t = 0; t < G; ++t) {
                                vc[h][t] = (vc[h][t] & keep) | (uint32_t)to[AT_V + t * 16 + n] << (8 * i);
                                vp[h][t] = (vp[h][t] & keep) | (uint32_t)to[AT_VP + t] << (8 * i);
                            }
                        }
                    }
                }
            }
        };
        if constexpr (P <= 128) take_v();
        if constexpr (NEW) {
            if (patches) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int from = entry_pos(e0 + h) - p_new, row = from + n;
                    if (row >= 0 && row < C) {
                        const uint8_t *to = new_rows + row * NEW_ROW;
                        uint32_t powers = 0;
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const u2 *c2 = reinterpret_cast<const u2 *>(to + (4 * b + jk) * 16);
                            const u2 c0 = c2[0], c1 = c2[1];
                            kc[h][b][0] = c0[0], kc[h][b][1] = c0[1], kc[h][b][2] = c1[0], kc[h][b][3] = c1[1];
                            powers |= (uint32_t)to[AT_KP + 4 * b + jk] << (8 * b);
                        }
                        kp[h] = powers;
                    }
                }
            }
        }
        // ---- scores of the pair: keys 4j .. 4j + 3 of slot n, of page a, then b
        float4_t s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int8v_t k = {(int)kc[h][b][0], (int)kc[h][b][1], (int)kc[h][b][2], (int)kc[h][b][3], 0, 0, 0, 0};
                const int kpow = (int)(kp[h] >> (8 * b));
                s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q_term[b][4], s[h], 4, 2, 0, kpow, 0, (int)q_last[b]);
                s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q_term[b][3], s[h], 4, 2, 0, kpow, 3, (int)q_power[b]);
                s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q_term[b][2], s[h], 4, 2, 0, kpow, 2, (int)q_power[b]);
                s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q_term[b][1], s[h], 4, 2, 0, kpow, 1, (int)q_power[b]);
                s[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q_term[b][0], s[h], 4, 2, 0, kpow, 0, (int)q_power[b]);
            }
        }
        if constexpr (P <= 128) {
            next_pair(it + L::DEPTH);
        } else { // (no registers for V beside K)
            __builtin_amdgcn_sched_barrier(0);
            take_v();
        }
        // ---- softmax in base 2; keys outside the slot's range get no weight, and where no slot of the workgroup attends them (rows past the
        // length, before the window, of a page that is not there) V's powers are cleared as well: 0 x NaN is NaN
        const int lo_b = RING ? (e0 + 1 >= n_old ? c->new_pos0 : INT32_MIN) : INT32_MIN;
        const int lo_a = RING ? (e0 >= n_old ? c->new_pos0 : INT32_MIN) : INT32_MIN;
        const int hi_a = RING && e0 < n_old ? c->new_pos0 - 1 : INT32_MAX;
        const int hi_b = e0 + 1 >= pb1 ? INT32_MIN : RING && e0 + 1 < n_old ? c->new_pos0 - 1 : INT32_MAX;
        const bool inside = ea >= max(ws_hi, lo_a) && ea + 15 <= min(lim_lo, hi_a) && eb >= max(ws_hi, lo_b) && eb + 15 <= min(lim_lo, hi_b);
        if (!inside) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int p0 = (h ? eb : ea) + j * 4, lo = h ? lo_b : lo_a, hi = h ? hi_b : hi_a;
                uint32_t keep = 0, seen = 0; // keys that some slot attends, that this lane's does
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = p0 + i;
                    const bool here = pos >= lo && pos <= hi, mine = here && pos >= my_ws && pos <= my_limit;
                    s[h][i] = mine ? s[h][i] : -INFINITY;
                    if (mine) seen |= 255u << (8 * i);
                    if (here && pos >= ws_lo && pos <= lim_hi) keep |= 255u << (8 * i);
                }
#pragma unroll
                for (int t = 0; t < G; ++t) vp[h][t] = (vp[h][t] & keep) | (~keep & 0x7f7f7f7fu);
                if constexpr (MQ) { // a row that is NaN, attended by some slots and not by others: theirs alone
#pragma unroll
                    for (int t = 0; t < G; ++t) {
                        const uint32_t nan = bytes_255(vp[h][t]);
                        if (__builtin_amdgcn_ballot_w64(nan != 0)) {
                            const float x = rows_max((nan & seen) != 0 ? 1.0f : 0.0f) > 0.0f ? NAN : 0.0f;
                            o[2 * t] += x;
                            o[2 * t + 1] += x;
                            vp[h][t] ^= nan & 0x80808080u;
                        }
                    }
                }
            }
        }
        float m_blk = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        m_blk = rows_max(m_blk);
        // (the base lies 8 below the maximum while that difference is exact; from 2^27 on a step of f32 is 16, the difference would be 0 or 16, and 2^16
        // is more than f16 has)
        const float b_blk = fabsf(m_blk) < 0x1p27f ? m_blk - V_SHIFT : m_blk;
        const float b_new = fmaxf(b_run, b_blk), b_safe = b_new == -INFINITY ? 0.0f : b_new;
        const float alpha = fast_exp2(b_run - b_safe);
        float pr[8], psum = 0.0f; // at most 2^8
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pr[i] = fast_exp2(s[i >> 2][i & 3] - b_safe);
            psum += pr[i];
        }
        l_run = l_run * alpha + psum;
        const bool rescale = alpha != 1.0f && b_run != -INFINITY; // (a slot without a key so far holds zeros)
        b_run = b_new;
        if (__builtin_amdgcn_ballot_w64(rescale)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= alpha;
        }
        // ---- O^T += V^T . P^T
        uint32_t far = 0;
#pragma unroll
        for (int t = 0; t < G; ++t) far |= fp4_far(vp[0][t]) | fp4_far(vp[1][t]);
        // dims 32 t + n and 32 t + 16 + n of the 32 keys, from the pairs that c0 .. c3 hold of each page, with weights in terms, the least first
        auto products = [&](int t, auto of_page, auto mfma, const auto &terms) __attribute__((always_inline)) {
            u4 first, second;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u4 c = of_page(vc[h][t], vp[h][t]);
                first[2 * h] = __builtin_amdgcn_perm(c[1], c[0], 0x05040100u);
                first[2 * h + 1] = __builtin_amdgcn_perm(c[3], c[2], 0x05040100u);
                second[2 * h] = __builtin_amdgcn_perm(c[1], c[0], 0x07060302u);
                second[2 * h + 1] = __builtin_amdgcn_perm(c[3], c[2], 0x07060302u);
            }
#pragma unroll
            for (const auto &x : terms) {
                o[2 * t] = mfma(first, x, o[2 * t]);
                o[2 * t + 1] = mfma(second, x, o[2 * t + 1]);
            }
        };
        // Powers that f16 does not have, or NaN, in bf16 instead.
        // Terms of 8 bits, the least first: three leave 2^-24 of a weight. Two, which leave 2^-17, where registers are those of two workgroups on a compute
        // unit: the third's would be reloaded on every pair (128 rows over 512, 1024 on rings of q32/kv8/hd128 13.1/14.2, 16.5/18.3 us).
        constexpr int TERMS = MQ && !ROWS && P <= 128 ? 2 : 3;
        const bool any_far = __builtin_amdgcn_ballot_w64(far != 0) != 0; // uniform
        if (TERMS == 3 ? __builtin_expect(any_far, false) : any_far) { // (apart from the code around it: steps of hd128 are 0.05 us faster; with two terms it spills)
            uint32_t terms[TERMS][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                typedef __attribute__((ext_vector_type(2))) float f2;
                f2 left = {pr[2 * i] * P_SCALE, pr[2 * i + 1] * P_SCALE};
#pragma unroll
                for (int k = TERMS - 1; k >= 0; --k) {
                    terms[k][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(left, bf16x2_t));
                    left -= f2{__uint_as_float(terms[k][i] << 16), __uint_as_float(terms[k][i] & 0xffff0000u)};
                }
                pr[2 * i] = pr[2 * i + 1] = 0.0f; // (f16's products then add zeros: with a path of their own, o would be in two places)
            }
#pragma unroll
            for (int t = 0; t < G; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                products(
                    t, [](uint32_t w, uint32_t e) __attribute__((always_inline)) { return u4{code_pair<0>(w, e << 23), code_pair<1>(w, e << 15), code_pair<2>(w, e << 7), code_pair<3>(w, e >> 1)}; },
                    [](u4 v, const uint32_t(&x)[4], float4_t to) __attribute__((always_inline)) {
                        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v), __builtin_bit_cast(bf16x8_t, u4{x[0], x[1], x[2], x[3]}), to, 0, 0, 0);
                    },
                    terms);
                vc[0][t] = vc[1][t] = 0;
                vp[0][t] = vp[1][t] = 0x7f7f7f7fu;
            }
        }
        {
            uint32_t terms[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f16_terms(pr[2 * i], pr[2 * i + 1], terms[1][i], terms[0][i]);
#pragma unroll
            for (int t = 0; t < G; ++t) {
                products(
                    t, [](uint32_t w, uint32_t e) __attribute__((always_inline)) {
                        e -= 0x01010101u * V_SHIFT;
                        return u4{code_pair_f16<0>(w, e << 23), code_pair_f16<1>(w, e << 15), code_pair_f16<2>(w, e << 7), code_pair_f16<3>(w, e >> 1)};
                    },
                    [](u4 v, const uint32_t(&x)[4], float4_t to) __attribute__((always_inline)) {
                        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, v), __builtin_bit_cast(f16x8_t, u4{x[0], x[1], x[2], x[3]}), to, 0, 0, 0);
                    },
                    terms);
            }
        }
        if constexpr (P > 128) next_pair(it + L::DEPTH);
    }
    l_run = rows_sum(l_run) * P_SCALE;
    if constexpr (PRE) __syncthreads(); // (a state lies over other wavefronts' pairs)

    // ---- the wavefronts' states meet in LDS, four columns a thread
    // [WAVES] of [rows][OSTRIDE], m [rows], l [rows]
    constexpr int STATE = L::WAVE / 4; // floats from one wavefront's to the next's
    float *const x0 = reinterpret_cast<float *>(lds + L::pairs(n_new)), *const xm = x0 + rows * OSTRIDE, *const xl = xm + rows;
    if (n < rows) {
        float *dst = x0 + wave * STATE + n * OSTRIDE + j * 4;
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<float4_t *>(dst + t * 16) = o[t];
        if (j == 0) {
            xm[wave * STATE + n] = b_run;
            xl[wave * STATE + n] = l_run;
        }
    }
    __syncthreads();
    // (partials are aligned where heads are whole units; the context is the caller's, at any float's address)
    const bool vec_ok = (g.head_dim & 3) == 0 && (a.splits_total > 1 || (reinterpret_cast<uintptr_t>(a.out) & 15) == 0);
    for (int u = tid; u < rows * (P / 4); u += THREADS) {
        const int row = u / (P / 4), c4 = (u - row * (P / 4)) * 4;
        float mw[WAVES], mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            mw[w] = xm[w * STATE + row];
            mx = fmaxf(mx, mw[w]);
        }
        const float m_safe = mx == -INFINITY ? 0.0f : mx;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
        float lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float wgt = fast_exp2(mw[w] - m_safe);
            acc += wgt * *reinterpret_cast<const float4_t *>(&x0[w * STATE + row * OSTRIDE + c4]);
            lsum += wgt * xl[w * STATE + row];
        }
        if (c4 >= g.head_dim) continue;
        const int slot = tile * 16 + row;
        float *dst;
        if (a.splits_total == 1) {
            acc *= 1.0f / lsum;
            if constexpr (PRE) {
                if (a.gate) {
                    const float *gate = a.gate + (long)(kvh * g.gqa + slot) * (a.q_head_stride > 0 ? a.q_head_stride : g.head_dim) + c4;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (c4 + i < g.head_dim) acc[i] *= sigmoid_gate(gate[i]);
                }
            }
            dst = a.out + (MQ ? context_row(g, kvh, slot) : (long)(kvh * g.gqa + slot)) * g.head_dim + c4;
        } else {
            const long pidx = ((long)kvh * a.splits_total + split) * n_slots + slot;
            dst = a.part_o + pidx * g.head_dim + c4;
            if (c4 == 0) {
                a.part_m[pidx] = mx;
                a.part_l[pidx] = lsum;
            }
        }
        if (vec_ok) {
            *reinterpret_cast<float4_t *>(dst) = acc;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c4 + i < g.head_dim) dst[i] = acc[i];
        }
    }
}

template <int P, int WAVES, bool MQ, bool RING, bool ROWS, bool PRE>
// (streaming chunks of heads up to 128 dims: registers for two workgroups on a compute unit. 256 rows over 2000 of q32/kv8/hd128 29.2 us, 32.9 with
// registers for one, although at 128 dims 7 or 8 are then spilled, and a wait for one reloaded among the pages is a wait for their copies too.)
__global__ __launch_bounds__(WAVES * 64, MQ && !ROWS && P <= 128 ? 4 : 1) void fp4_attention_kernel(DecodeArgs a, ChunkPages c) {
    fp4_attention_body<P, WAVES, MQ, RING, ROWS, PRE>(a, &c, blockIdx.x, blockIdx.y, blockIdx.z);
}

// Several sequences of the same model layer: grid z is the sequence, grid x covers the largest number of splits
template <int P, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fp4_attention_batch_kernel(DecodeBatchArgs b) {
    const DecodeArgs &a = b.seq[blockIdx.z];
    if ((int)blockIdx.x >= a.splits) return;
    fp4_attention_body<P, WAVES, false, false>(a, nullptr, blockIdx.x, blockIdx.y, 0);
}

template <int P, int WAVES, bool MQ, bool RING, bool ROWS = false, bool PRE = false>
static hipError_t launch_fp4_of(const DecodeArgs &a, const ChunkPages &c, hipStream_t s) {
    static std::atomic<uint64_t> lds_ok{0}; // per instantiation
    {
        hipError_t e = allow_full_lds(reinterpret_cast<const void *>(&fp4_attention_kernel<P, WAVES, MQ, RING, ROWS, PRE>), lds_ok);
        if (e != hipSuccess) return e;
    }
    const int n_slots = a.n_queries * a.g.gqa;
    const dim3 grid((unsigned)a.splits, (unsigned)a.g.kv_heads, (unsigned)((n_slots + 15) / 16));
    const size_t lds = Fp4Lds<P, WAVES>::bytes(ROWS ? a.n_queries : MQ ? 0 : 1);
    hipLaunchKernelGGL((fp4_attention_kernel<P, WAVES, MQ, RING, ROWS, PRE>), grid, dim3(WAVES * 64), lds, s, a, c);
    return hipGetLastError();
}
template <int P, int WAVES>
static hipError_t launch_fp4(const DecodeArgs &a, const ChunkPages *c, hipStream_t s) {
    if (a.k_new && (c || a.n_queries > MQ_APPEND_ROWS)) return hipErrorInvalidValue;
    if (a.pre) {
        if constexpr (P > 256) return hipErrorInvalidValue; // the caller sends these through separate launches
        else return c || a.n_queries > 1 || a.g.gqa > 16 || !a.k_new ? hipErrorInvalidValue : launch_fp4_of<P, WAVES, false, false, false, true>(a, ChunkPages{}, s);
    }
    if (c) return launch_fp4_of<P, WAVES, true, true>(a, *c, s);
    if (a.n_queries == 1 && a.g.gqa <= 16) return launch_fp4_of<P, WAVES, false, false>(a, ChunkPages{}, s);
    return a.k_new ? launch_fp4_of<P, WAVES, true, false, true>(a, ChunkPages{}, s) : launch_fp4_of<P, WAVES, true, false>(a, ChunkPages{}, s);
}

hipError_t launch_fp4_attention(const DecodeArgs &a, const ChunkPages *c, hipStream_t s) {
    if (a.split_base != 0) return hipErrorInvalidValue;
    switch (a.g.P) {
    case 32: return launch_fp4<32, 8>(a, c, s);
    case 64: return launch_fp4<64, 8>(a, c, s);
    case 96: return launch_fp4<96, 8>(a, c, s);
    case 128: return launch_fp4<128, 8>(a, c, s);
    case 256: return launch_fp4<256, 8>(a, c, s);
    case 512: return launch_fp4<512, 4>(a, c, s);
    default: return hipErrorInvalidValue;
    }
}

template <int P, int WAVES>
static hipError_t launch_fp4_batch_of(const DecodeBatchArgs &b, int n_seq, int max_splits, hipStream_t s) {
    static std::atomic<uint64_t> lds_ok{0}; // per instantiation
    {
        hipError_t e = allow_full_lds(reinterpret_cast<const void *>(&fp4_attention_batch_kernel<P, WAVES>), lds_ok);
        if (e != hipSuccess) return e;
    }
    const Geom &g = b.seq[0].g;
    const dim3 grid((unsigned)max_splits, (unsigned)g.kv_heads, (unsigned)n_seq);
    const size_t lds = Fp4Lds<P, WAVES>::bytes(1);
    hipLaunchKernelGGL((fp4_attention_batch_kernel<P, WAVES>), grid, dim3(WAVES * 64), lds, s, b);
    return hipGetLastError();
}
// One geometry, one query row a sequence, at most 16 heads a kv head (checked by the caller)
hipError_t launch_fp4_batch(const DecodeBatchArgs &b, int n_seq, int max_splits, hipStream_t s) {
    switch (b.seq[0].g.P) {
    case 32: return launch_fp4_batch_of<32, 8>(b, n_seq, max_splits, s);
    case 64: return launch_fp4_batch_of<64, 8>(b, n_seq, max_splits, s);
    case 96: return launch_fp4_batch_of<96, 8>(b, n_seq, max_splits, s);
    case 128: return launch_fp4_batch_of<128, 8>(b, n_seq, max_splits, s);
    case 256: return launch_fp4_batch_of<256, 8>(b, n_seq, max_splits, s);
    case 512: return launch_fp4_batch_of<512, 4>(b, n_seq, max_splits, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace skv
