// gfx950 kernels of an eviction: which rows of a kv head stay (its own choice, by the weights its rows have had), and the moves that close
// the gaps.
//
// Rows that stay below `keep` stay where they are; the gaps between them, in order, take the rows from `keep` on that stay, in order. So what is
// read lies at or behind `keep`, what is written below it: no move waits for another, and no more rows move than have to.
#include <algorithm>

#include "fp4_tile.h"
#include "weights.h"

namespace skv {

// ------------------------------------------------------------------------------------
// The choice: workgroups of 1024 threads, each for a stretch of a kv head's rows, up to STRETCHES of them. The first and the last rows count as
// heavier than any weight, what lies past the last one as the lightest (and, of equal rows the highest, never stays). A radix selection over the
// rows, eleven bits of the weights' order at a time, finds the lightest weight that stays and how many of that
// weight do (fewer bits where those decide): every workgroup for itself over all rows, which its threads hold; only the first eleven
// bits, where most rows are counted, are counted once, by a launch of their own. (That is for more than 16384 rows: up to there one workgroup has
// them all and leaves the moves alone, see evict_choose_kernel.) Then with S(r) the rows below r that stay
// (each workgroup counts them up to its stretch and up to `keep`), a gap at r < keep is number r - S(r) and takes the mover of that number, a row
// r >= keep that stays is mover S(r) - S(keep).
//
// Bound by the chain of passes and by what a CU alone brings in, not by bytes: 2000 rows of two heads 6.6 us, 8000 10.3, 16000 18;
// 32768 18.5 and 4.7 for the counts, where one workgroup a head took 64. Beyond, every workgroup reads all weights anew in each pass: half of 32768 rows of two
// heads of 256 dims leave in 39 us with their moves, of 32769 in 56, of 65536 in 96, of 131072 in 210.
// ------------------------------------------------------------------------------------
static_assert(sizeof(Mover) == 3 * sizeof(int32_t), "as scratch is counted");
constexpr int SEL_THREADS = 1024, SEL_WAVES = SEL_THREADS / 64, BINS = 2048, STRETCHES = 8, STRETCH = 4096, CHOSEN = 16 * SEL_THREADS;

// Weights in the order of whole numbers; NaN below all.
__device__ __forceinline__ uint32_t order_of(float w) {
    w += 0.0f; // (-0 is 0)
    const uint32_t b = __float_as_uint(w);
    return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t order_of_row(const EvictArgs &a, float w, int r) {
    const uint32_t x = r < a.len ? order_of(w) : 0u;
    return (int)(r < a.first) | ((int)(r >= a.len - a.last) & (int)(r < a.len)) ? 0xffffffffu : x;
}
template <int CTRL>
__device__ __forceinline__ int dpp0(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false); } // (0 where there is no such lane)
// Sum of the lanes up to and with this one
__device__ __forceinline__ int sum_up_to(int x) {
    x += dpp0<0x111>(x);
    x += dpp0<0x112>(x);
    x += dpp0<0x114>(x);
    x += dpp0<0x118>(x); // along sixteen
    const int a = __builtin_amdgcn_readlane(x, 15), b = __builtin_amdgcn_readlane(x, 31), c = __builtin_amdgcn_readlane(x, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return x + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

// The first eleven bits: a stretch's counts. Four copies of the bins: weights crowd into a few of them, and lanes that meet in one wait for each other.
__global__ __launch_bounds__(SEL_THREADS) void evict_count_kernel(EvictArgs a) {
    __shared__ int bins[4][BINS];
    const int kvh = blockIdx.y, tid = threadIdx.x;
    const float *const w = a.weights + kvh * a.stride;
    for (int i = tid; i < 4 * BINS; i += SEL_THREADS) bins[0][i] = 0;
    const int lo = (int)blockIdx.x * a.per, hi = min(lo + a.per, a.len);
    __syncthreads();
    for (int r = lo + tid; r < hi; r += SEL_THREADS) atomicAdd(&bins[tid & 3][order_of_row(a, w[r], r) >> 21], 1);
    __syncthreads();
    int *const out = a.counts + ((long)kvh * gridDim.x + blockIdx.x) * BINS;
    for (int i = tid; i < BINS; i += SEL_THREADS) out[i] = bins[0][i] + bins[1][i] + bins[2][i] + bins[3][i];
}

// Where the lightest that stays lies among the bins: c0 and c1 are the rows in bins 2047 - 2 tid and the next one down.
__device__ __forceinline__ void find_bin(int c0, int c1, int want, int *sums, int *found) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, top = BINS - 1 - 2 * tid;
    const int sum = sum_up_to(c0 + c1);
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int before = sum - c0 - c1;
#pragma unroll
    for (int v = 0; v < SEL_WAVES; ++v) before += v < wave ? sums[v] : 0;
    if (before < want && want <= before + c0) {
        found[0] = top, found[1] = before, found[2] = c0;
    } else if (before + c0 < want && want <= before + c0 + c1) {
        found[0] = top - 1, found[1] = before + c0, found[2] = c1;
    }
    __syncthreads();
}

// The tile of (page, kvh) at `dst` and of its sources, for K's codes or numbers and (4-bit pages) for the powers
struct TileAt {
    long codes, powers;
    __device__ TileAt(const Geom &g, int kvh)
        : codes(g.fp4 ? (long)kvh * fp4_code_bytes(g.P) : (long)kvh * g.tile_elems * 2),
          powers((long)g.kv_heads * fp4_code_bytes(g.P) + (long)kvh * fp4_power_bytes(g.P)) {}
};
// `moves` rows from `from` to `to` (each page * 16 + row of it), by a workgroup: K's pieces of 16 bytes, or V's numbers one by one, of all rows in turn, four
// of a thread asked for before the first is written.
template <class X, class F>
__device__ __forceinline__ void move_units(char *pool, long page_bytes, int moves, int per_row, const int *from, const int *to, int tid, F at) {
    const int n = moves * per_row;
    for (int u0 = tid; u0 < n; u0 += 4 * SEL_THREADS) {
        X x[4];
        X *out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = min(u0 + i * SEL_THREADS, n - 1), m = u / per_row, unit = u - m * per_row, a = from[m], b = to[m];
            x[i] = reinterpret_cast<const X *>(pool + (long)(a >> 4) * page_bytes)[at(unit, a & 15)];
            out[i] = reinterpret_cast<X *>(pool + (long)(b >> 4) * page_bytes) + at(unit, b & 15);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (u0 + i * SEL_THREADS < n) *out[i] = x[i];
    }
}
__device__ __forceinline__ void move_rows(const EvictArgs &a, int kvh, int moves, const int *from, const int *to, int tid) {
    const Geom &g = a.g;
    const TileAt t(g, kvh);
    const long bytes = g.page_elems * 2;
    char *const k = reinterpret_cast<char *>(a.k_pool), *const v = reinterpret_cast<char *>(a.v_pool);
    move_units<uint4>(k + t.codes, bytes, moves, g.fp4 ? g.P / 32 : g.f32 ? g.P / 4 : g.P / 8, from, to, tid, [&](int u, int r) { return u * 16 + r; });
    const auto word = [&](int bw) { return [bw](int u, int r) { return ((u / bw * 4 + (r >> 2)) * bw + u % bw) * 4 + (r & 3); }; };
    if (g.fp4) {
        const int P = g.P;
        move_units<uint8_t>(k + t.powers, bytes, moves, P / 32, from, to, tid, [&](int u, int r) { return k4_power(P, r, u); });
        move_units<uint8_t>(v + t.codes, bytes, moves, P / 2, from, to, tid, word(16 * fp4_quad(P)));
        move_units<uint8_t>(v + t.powers, bytes, moves, P / 32, from, to, tid, word(P / 32));
    } else if (g.f32) {
        move_units<uint32_t>(v + t.codes, bytes, moves, g.P, from, to, tid, word(16));
    } else {
        move_units<uint16_t>(v + t.codes, bytes, moves, g.P, from, to, tid, word(32));
    }
}

// Up to 1024 ROWS: one workgroup has them all, and the movers (no more than half of the rows) in LDS, so that what it leaves needs nothing more but the moves: `from` says for
// each row below `keep` where its numbers come from (-1: it stays).
// ROWS of a thread; a wavefront's lie together. MOVES: few rows can move (few_moves), and the workgroup moves them itself.
constexpr int FEW_MOVES = 64;
template <int ROWS, bool MOVES>
__global__ __launch_bounds__(SEL_THREADS) void evict_choose_kernel(EvictArgs a) {
    constexpr int MOVERS = ROWS * SEL_THREADS / 2;
    __shared__ int bins[2][BINS];
    __shared__ int sums[SEL_WAVES], found[3], seen[4][SEL_WAVES];
    __shared__ int row_of[MOVERS], held_of[MOVERS];
    __shared__ float weight_of[MOVERS];
    __shared__ int place_of[MOVES ? FEW_MOVES : 1];
    const int kvh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float *const w = a.weights + kvh * a.stride;
    const int first = wave * (ROWS * 64) + lane;
    float x[ROWS];
    int page[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) x[i] = w[min(first + i * 64, a.len - 1)];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) page[i] = a.table[min(first + i * 64, a.len - 1) >> 4];
    for (int i = tid; i < 2 * BINS; i += SEL_THREADS) bins[0][i] = 0;
    uint32_t order[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) asm("" : "+v"(x[i]));
#pragma unroll
    for (int i = 0; i < ROWS; ++i) order[i] = order_of_row(a, x[i], first + i * 64);
    __syncthreads();
    int want = a.keep;
    uint32_t bits = 0, mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        int *const b = bins[pass & 1];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            if (first + i * 64 < a.len && (order[i] & mask) == bits) atomicAdd(&b[(order[i] >> shift) & ((1u << width) - 1)], 1);
        __syncthreads();
        const int top = BINS - 1 - 2 * tid;
        const int2 c = *reinterpret_cast<const int2 *>(&b[top - 1]);
        *reinterpret_cast<int2 *>(&b[top - 1]) = make_int2(0, 0); // (for the pass after the next)
        find_bin(c.y, c.x, want, sums, found);
        bits |= (uint32_t)found[0] << shift;
        mask |= ((1u << width) - 1) << shift;
        want -= found[1];
        if (found[2] == want) break; // (uniform) all that begin like it stay
    }
    uint64_t hb[ROWS], eb[ROWS];
    int h = 0, e = 0, hk = 0, ek = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = wave * (ROWS * 64) + i * 64;
        hb[i] = __ballot((order[i] & mask) > bits && r + lane < a.len), eb[i] = __ballot((order[i] & mask) == bits && r + lane < a.len);
        const uint64_t front = r + 64 <= a.keep ? ~0ull : r >= a.keep ? 0ull : (1ull << (a.keep - r)) - 1;
        h += (int)__popcll(hb[i]), e += (int)__popcll(eb[i]);
        hk += (int)__popcll(hb[i] & front), ek += (int)__popcll(eb[i] & front);
    }
    if (lane == 0) seen[0][wave] = h, seen[1][wave] = e, seen[2][wave] = hk, seen[3][wave] = ek;
    __syncthreads();
    h = e = hk = ek = 0;
#pragma unroll
    for (int v = 0; v < SEL_WAVES; ++v) {
        if (v < wave) h += seen[0][v], e += seen[1][v];
        hk += seen[2][v], ek += seen[3][v];
    }
    const int stay_keep = hk + min(ek, want);
    const uint64_t below = (1ull << lane) - 1;
    int gap[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = first + i * 64, e_here = e + (int)__popcll(eb[i] & below);
        const bool stays = (hb[i] >> lane & 1) || ((eb[i] >> lane & 1) && e_here < want);
        const int s = h + (int)__popcll(hb[i] & below) + min(e_here, want); // S(r)
        gap[i] = r < a.keep && !stays ? r - s : -1;
        if (r >= a.keep && r < a.len && stays) row_of[s - stay_keep] = r, held_of[s - stay_keep] = page[i] * 16 + (r & 15), weight_of[s - stay_keep] = x[i];
        h += (int)__popcll(hb[i]), e += (int)__popcll(eb[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int r = first + i * 64;
        if (r < a.keep) {
            const int g = max(gap[i], 0);
            if (a.from) a.from[(long)kvh * a.keep + r] = gap[i] >= 0 ? held_of[g] : -1;
            if (a.kept) a.kept[(long)kvh * a.keep + r] = gap[i] >= 0 ? row_of[g] : r;
            if (gap[i] >= 0) w[r] = weight_of[g];
            if (MOVES && gap[i] >= 0) place_of[g] = page[i] * 16 + (r & 15);
        } else if (r < a.len) {
            w[r] = 0.0f;
        }
    }
    if constexpr (MOVES) {
        __syncthreads();
        move_rows(a, kvh, a.keep - stay_keep, held_of, place_of, tid);
    }
}

// NI > 0: a lane holds the orders of its NI rows (row i of a wavefront's stretch of 64 NI: 64 i + lane), for up to 1024 NI rows; 0: any number
// of rows, their weights read anew each time they are gone through.
template <int NI>
__global__ __launch_bounds__(SEL_THREADS) void evict_select_kernel(EvictArgs a) {
    __shared__ int bins[BINS];
    __shared__ int sums[SEL_WAVES];
    __shared__ int found[3]; // bin, rows in the bins above it, rows in it
    __shared__ int seen[4][SEL_WAVES];
    const int kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float *const w = a.weights + kvh * a.stride;
    int want = a.keep; // stay
    const int steps = NI > 0 ? NI : (a.len + SEL_THREADS - 1) / SEL_THREADS, r0 = wave * steps * 64;
    uint32_t order[NI > 0 ? NI : 1];
    const auto weight = [&](int i) __attribute__((always_inline)) {
        const int r = r0 + i * 64 + lane;
        return order_of_row(a, w[min(r, a.len - 1)], r);
    };
    if constexpr (NI > 0) { // (all asked for first)
        float x[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = w[min(r0 + i * 64 + lane, a.len - 1)];
#pragma unroll
        for (int i = 0; i < NI; ++i) asm("" : "+v"(x[i]));
#pragma unroll
        for (int i = 0; i < NI; ++i) order[i] = order_of_row(a, x[i], r0 + i * 64 + lane);
    }
    // f(first row of 64, the lane's order) of a wavefront's share
    const auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (NI > 0) {
#pragma unroll
            for (int i = 0; i < NI; ++i) f(r0 + i * 64, order[i]);
        } else {
            for (int i = 0; i < steps && r0 + i * 64 < a.len; ++i) f(r0 + i * 64, weight(i));
        }
    };

    // of the lightest that stays, the bits under `mask` of its order are `bits`, and `want` of those that have them stay
    uint32_t bits = 0, mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
        const bool counted = pass == 0 && a.counts != nullptr;
        // from the heaviest bin down: thread t has bins 2t and 2t + 1 counted from the top
        const int top = BINS - 1 - 2 * tid;
        int c0 = 0, c1 = 0;
        if (counted) {
            const int *from = a.counts + (long)kvh * gridDim.x * BINS + top - 1;
            int2 c[STRETCHES];
#pragma unroll
            for (int g = 0; g < STRETCHES; ++g) c[g] = *reinterpret_cast<const int2 *>(from + (long)min(g, (int)gridDim.x - 1) * BINS);
#pragma unroll
            for (int g = 0; g < STRETCHES; ++g)
                if (g < (int)gridDim.x) c0 += c[g].y, c1 += c[g].x;
        } else {
            for (int i = tid; i < BINS; i += SEL_THREADS) bins[i] = 0;
            __syncthreads();
            each([&](int, uint32_t x) __attribute__((always_inline)) {
                if ((x & mask) == bits) atomicAdd(&bins[(x >> shift) & ((1u << width) - 1)], 1);
            });
            __syncthreads();
            c0 = bins[top], c1 = bins[top - 1];
        }
        find_bin(c0, c1, want, sums, found);
        bits |= (uint32_t)found[0] << shift;
        mask |= ((1u << width) - 1) << shift;
        want -= found[1];
        if (found[2] == want) break; // (uniform) all that begin like it stay
    }

    // rows that are heavier, and those like the lightest that stays, in front of the workgroup's stretch and of `keep`
    const int start = (int)blockIdx.x * a.per, end = min(start + a.per, a.len);
    int h0 = 0, e0 = 0, hk = 0, ek = 0;
    each([&](int r, uint32_t x) __attribute__((always_inline)) {
        const uint64_t h = __ballot((x & mask) > bits), e = __ballot((x & mask) == bits);
        if (r < start) h0 += (int)__popcll(h), e0 += (int)__popcll(e); // (whole 64s)
        if (r < a.keep) {
            const uint64_t front = r + 64 <= a.keep ? ~0ull : (1ull << (a.keep - r)) - 1;
            hk += (int)__popcll(h & front), ek += (int)__popcll(e & front);
        }
    });
    if (lane == 0) seen[0][wave] = h0, seen[1][wave] = e0, seen[2][wave] = hk, seen[3][wave] = ek;
    __syncthreads();
    h0 = e0 = hk = ek = 0;
#pragma unroll
    for (int v = 0; v < SEL_WAVES; ++v) h0 += seen[0][v], e0 += seen[1][v], hk += seen[2][v], ek += seen[3][v];
    const int stay_keep = hk + min(ek, want);

    int32_t *const kept = a.kept + (long)kvh * a.keep;
    Mover *const moved = a.moved + (long)kvh * (a.len - a.keep);
    const uint64_t below = (1ull << lane) - 1;
    constexpr int SEL_ROWS = 4; // of a thread, 4096 of the workgroup at a time, 256 in a row a wavefront's
    for (int base = start; base < end; base += SEL_ROWS * SEL_THREADS) {
        const int first = base + wave * (SEL_ROWS * 64) + lane;
        float x[SEL_ROWS];
        uint64_t hb[SEL_ROWS], eb[SEL_ROWS];
#pragma unroll
        for (int i = 0; i < SEL_ROWS; ++i) x[i] = w[min(first + i * 64, a.len - 1)];
        int h_wave = 0, e_wave = 0;
#pragma unroll
        for (int i = 0; i < SEL_ROWS; ++i) {
            const uint32_t o = order_of_row(a, x[i], first + i * 64) & mask;
            hb[i] = __ballot(o > bits && first + i * 64 < end), eb[i] = __ballot(o == bits && first + i * 64 < end);
            h_wave += (int)__popcll(hb[i]), e_wave += (int)__popcll(eb[i]);
        }
        __syncthreads(); // (the counts before are read)
        if (lane == 0) seen[0][wave] = h_wave, seen[1][wave] = e_wave;
        __syncthreads();
        int h = h0, e = e0;
#pragma unroll
        for (int v = 0; v < SEL_WAVES; ++v) {
            const int vh = seen[0][v], ve = seen[1][v];
            h0 += vh, e0 += ve;
            if (v < wave) h += vh, e += ve;
        }
#pragma unroll
        for (int i = 0; i < SEL_ROWS; ++i) {
            const int r = first + i * 64, e_here = e + (int)__popcll(eb[i] & below);
            const bool stays = (hb[i] >> lane & 1) || ((eb[i] >> lane & 1) && e_here < want);
            const int s = h + (int)__popcll(hb[i] & below) + min(e_here, want); // S(r)
            if (r < end) {
                if (r < a.keep) kept[r] = stays ? r : ~(r - s);
                else if (stays) moved[s - stay_keep] = Mover{r, a.table[r >> 4] * 16 + (r & 15), x[i]};
            }
            h += (int)__popcll(hb[i]), e += (int)__popcll(eb[i]);
        }
    }
}

// ------------------------------------------------------------------------------------
// The moves: a workgroup the gaps of one page of one kv head, of K or of V. Of a page's row K holds pieces of 16 bytes (8, 4 or 32 dims), one
// of each sixteen in a row; V holds its place in words of four rows, BW words of a quad of rows together:
//   bf16 [P/32][4 quads][32], f32 [P/16][4][16], codes [P/32/U][4][16 U], their powers [4][P/32]
// ------------------------------------------------------------------------------------
struct Moves {
    int row[16];     // in its page; -1 = the row stays as it is
    int place[16];   // the same, its own where it stays, at its own page (the wide moves)
    long at[16];     // the page's tile, bytes from the pool's start (as pointers they would be read through the flat path)
};

template <int T>
__device__ __forceinline__ void move_pieces(const Moves &m, const char *pool, char *to, int pieces, int tid) {
    for (int u = tid; u < pieces * 16; u += T) {
        const int r = u & 15, from = m.row[r];
        if (from >= 0) reinterpret_cast<uint4 *>(to)[u] = reinterpret_cast<const uint4 *>(pool + m.at[r])[u - r + from];
    }
}
template <class E, int T>
__device__ __forceinline__ void move_words(const Moves &m, const char *pool, char *to, int words, int bw, int tid) {
    typedef __attribute__((ext_vector_type(4))) E e4;
    for (int u = tid; u < words * 4; u += T) {
        const int blk = u / (4 * bw), quad = u / bw & 3, in = u % bw;
        E x[4];
        int from[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            from[i] = m.row[quad * 4 + i];
            x[i] = E{};
            if (from[i] >= 0) x[i] = reinterpret_cast<const E *>(pool + m.at[quad * 4 + i])[((blk * 4 + (from[i] >> 2)) * bw + in) * 4 + (from[i] & 3)];
        }
        E *const p = reinterpret_cast<E *>(to) + (long)u * 4;
        if (from[0] >= 0 && from[1] >= 0 && from[2] >= 0 && from[3] >= 0) {
            *reinterpret_cast<e4 *>(p) = e4{x[0], x[1], x[2], x[3]};
        } else { // (the word's other rows are not touched: some may be another gap's source)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (from[i] >= 0) p[i] = x[i];
        }
    }
}

// 16 bytes of words that have row s[i] of y[i] in row i
template <class E>
__device__ __forceinline__ uint4 rows_of(const uint4 (&y)[4], const int (&s)[4]) {
    const uint32_t w[4][4] = {{y[0].x, y[0].y, y[0].z, y[0].w}, {y[1].x, y[1].y, y[1].z, y[1].w}, {y[2].x, y[2].y, y[2].z, y[2].w}, {y[3].x, y[3].y, y[3].z, y[3].w}};
    uint32_t out[4];
    if constexpr (sizeof(E) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // (by bits: as conditions they become an array with an index, in LDS)
            const uint32_t odd = 0u - (uint32_t)(s[i] & 1), high = 0u - (uint32_t)(s[i] >> 1);
            const uint32_t lo = (w[i][0] & ~odd) | (w[i][1] & odd), hi = (w[i][2] & ~odd) | (w[i][3] & odd);
            out[i] = (lo & ~high) | (hi & high);
        }
    } else if constexpr (sizeof(E) == 2) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t a = __builtin_amdgcn_perm(w[2 * p][2 * k + 1], w[2 * p][2 * k], 0x0100u + 0x0202u * s[2 * p]);
                const uint32_t b = __builtin_amdgcn_perm(w[2 * p + 1][2 * k + 1], w[2 * p + 1][2 * k], 0x0100u + 0x0202u * s[2 * p + 1]);
                out[2 * k + p] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t a = __builtin_amdgcn_perm(w[1][k], w[0][k], (uint32_t)(s[0] + ((s[1] + 4) << 8))), b = __builtin_amdgcn_perm(w[3][k], w[2][k], (uint32_t)(s[2] + ((s[3] + 4) << 8)));
            out[k] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}
// One V tile's words, 16 bytes at a time: rows that stay are written back as they were, so all of the page's rows must lie below `keep`
// (nobody reads them then, and nobody else writes them). Without a branch, and short: a launch's first wavefronts fetch its code as they go, some 0.1 us
// a line of 8 instructions, and in four times as many this took 13 us of 1000 rows in place of 5.5.
template <class E, int T>
__device__ __forceinline__ void move_wide(const Moves &m, const char *pool, char *to, int words, int bw, int tid) {
    constexpr int W = 4 / (int)sizeof(E); // words of 16 bytes
    const int units = words * 4 / W, runs = bw / W;
    for (int u = tid; u < units; u += T) {
        const int run = u / runs, in = u - run * runs, quad = run & 3;
        uint4 y[4];
        int row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            row[i] = m.place[quad * 4 + i];
            y[i] = reinterpret_cast<const uint4 *>(pool + m.at[quad * 4 + i])[((run & ~3) + (row[i] >> 2)) * runs + in];
            row[i] &= 3;
        }
        reinterpret_cast<uint4 *>(to)[u] = rows_of<E>(y, row);
    }
}

// All rows of a page whose rows all lie below `keep`, those that stay as they are: whole lines are written (10 layers' halves of 32768 rows 651 -> 620 us)
template <int T>
__device__ __forceinline__ void move_pieces_wide(const Moves &m, const char *pool, char *to, int pieces, int tid) {
    for (int u = tid; u < pieces * 16; u += T) {
        const int r = u & 15;
        reinterpret_cast<uint4 *>(to)[u] = reinterpret_cast<const uint4 *>(pool + m.at[r])[u - r + m.place[r]];
    }
}
template <int T>
__device__ __forceinline__ void move_k(const Geom &g, const TileAt &t, const Moves &m, const Moves &powers, const char *pool, char *dst, bool wide, int tid) {
    const int pieces = g.fp4 ? g.P / 32 : g.f32 ? g.P / 4 : g.P / 8;
    if (wide) move_pieces_wide<T>(m, pool, dst + t.codes, pieces, tid);
    else move_pieces<T>(m, pool, dst + t.codes, pieces, tid);
    if (g.fp4)
        for (int u = tid; u < g.P / 2; u += T) {
            const int r = u & 15, grp = u >> 4, from = powers.row[r];
            if (from >= 0) dst[t.powers + k4_power(g.P, r, grp)] = pool[powers.at[r] + k4_power(g.P, from, grp)];
        }
}
template <int T>
__device__ __forceinline__ void move_v(const Geom &g, const TileAt &t, const Moves &m, const Moves &powers, const char *pool, char *dst, bool wide, int tid) {
    if (g.fp4) {
        if (wide) move_wide<uint8_t, T>(m, pool, dst + t.codes, g.P / 2, 16 * fp4_quad(g.P), tid);
        else move_words<uint8_t, T>(m, pool, dst + t.codes, g.P / 2, 16 * fp4_quad(g.P), tid);
        move_words<uint8_t, T>(powers, pool, dst + t.powers, g.P / 32, g.P / 32, tid);
    } else if (g.f32) {
        if (wide) move_wide<uint32_t, T>(m, pool, dst + t.codes, g.P, 16, tid);
        else move_words<uint32_t, T>(m, pool, dst + t.codes, g.P, 16, tid);
    } else {
        if (wide) move_wide<uint16_t, T>(m, pool, dst + t.codes, g.P, 32, tid);
        else move_words<uint16_t, T>(m, pool, dst + t.codes, g.P, 32, tid);
    }
}

// 16384 of 32768 rows of two heads of 256 dims, some 67 MB with the lines that are read and written by parts: 25 us, 2.7 TB/s.
constexpr int MOVE_THREADS = 256;
__global__ __launch_bounds__(MOVE_THREADS) void evict_move_kernel(EvictArgs a) {
    __shared__ Moves m, powers; // (4-bit pages: of the codes, of the powers)
    const Geom &g = a.g;
    // (workgroups go to the eight XCDs in turn: neighbouring pages, whose gaps take neighbouring rows, to the same one)
    const int kvh = blockIdx.y, tid = threadIdx.x, page = (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3));
    const bool is_v = blockIdx.z != 0;
    char *const pool = reinterpret_cast<char *>(is_v ? a.v_pool : a.k_pool);
    const TileAt t(g, kvh);
    float *const w = a.weights + kvh * a.stride;
    bool any = false;
    const int to_page = a.table[min(page, (a.keep - 1) >> 4)];
    if (tid < 16) {
        const int row = page * 16 + tid;
        int from = row, held = 0;
        if (row < a.keep && a.from) {
            held = a.from[(long)kvh * a.keep + row];
            from = held >= 0 ? -1 : row;
        } else if (row < a.keep) {
            int32_t *const kept = a.kept + (long)kvh * a.keep + row;
            const int gap = ~*kept; // (a gap's number; or, a row that stays or a gap whose other workgroup was here already, below 0)
            from = ~gap;
            if (gap >= 0) {
                const Mover x = a.moved[(long)kvh * (a.len - a.keep) + gap];
                from = x.row;
                held = x.held;
                if (!is_v) {
                    *kept = from;
                    w[row] = x.weight;
                }
            } else if (from != row) {
                held = a.table[from >> 4] * 16 + (from & 15);
            }
        }
        any = from != row;
        if (!any) held = to_page * 16 + tid;
        const long src = (long)(held >> 4) * g.page_elems * 2;
        m.place[tid] = held & 15;
        m.row[tid] = powers.row[tid] = any ? held & 15 : -1;
        m.at[tid] = src + t.codes;
        powers.at[tid] = src + t.powers;
    }
    if (!is_v && !a.from)
        for (long r = a.keep + (long)page * MOVE_THREADS + tid; r < a.len; r += (long)gridDim.x * MOVE_THREADS) w[r] = 0.0f;
    if (!__syncthreads_or(any)) return;
    char *const dst = pool + (long)to_page * g.page_elems * 2;
    const bool wide = (page + 1) * 16 <= a.keep;
    if (!is_v) move_k<MOVE_THREADS>(g, t, m, powers, pool, dst, wide, tid);
    else move_v<MOVE_THREADS>(g, t, m, powers, pool, dst, wide, tid);
}

// One row leaves (a cache at its budget, a token at a time): the lightest of those between, of equal ones the highest, and the last row takes its place.
// 2049 rows of eight heads of 128 dims 6.7 us, by the two launches of more rows 14.7: a chain of launch, weights, places, numbers and stores.
__global__ __launch_bounds__(SEL_THREADS) void evict_one_kernel(EvictArgs a) {
    __shared__ Moves mk, mv, pk, pv;
    __shared__ uint32_t lightest[SEL_WAVES];
    __shared__ int at[SEL_WAVES];
    const Geom &g = a.g;
    const int kvh = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float *const w = a.weights + kvh * a.stride;
    const int page_from = a.table[a.keep >> 4], hi = a.len - a.last;
    uint32_t low = 0xffffffffu;
    int row = -1;
    for (int r = a.first + tid; r < hi; r += 4 * SEL_THREADS) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = order_of(w[min(r + i * SEL_THREADS, hi - 1)]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at_i = min(r + i * SEL_THREADS, hi - 1);
            if (x[i] < low || (x[i] == low && at_i > row)) low = x[i], row = at_i;
        }
    }
    // the lowest order of a wavefront, then the highest of its rows that have it
    const auto lanes = [](auto x, auto best) __attribute__((always_inline)) {
        x = best(x, (decltype(x))__builtin_amdgcn_mov_dpp((int)x, 0xb1, 0xf, 0xf, true));
        x = best(x, (decltype(x))__builtin_amdgcn_mov_dpp((int)x, 0x4e, 0xf, 0xf, true));
        x = best(x, (decltype(x))__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xf, 0xf, true));
        x = best(x, (decltype(x))__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xf, 0xf, true));
        const auto b = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
        x = best((decltype(x))b[0], (decltype(x))b[1]);
        const auto c = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
        return best((decltype(x))c[0], (decltype(x))c[1]);
    };
    const auto lower = [](uint32_t x, uint32_t y) { return min(x, y); };
    const auto higher = [](int x, int y) { return max(x, y); };
    const uint32_t wave_low = lanes(low, lower);
    const int wave_row = lanes(low == wave_low ? row : -1, higher);
    if ((tid & 63) == 0) lightest[wave] = wave_low, at[wave] = wave_row;
    __syncthreads();
    uint32_t least = 0xffffffffu;
    int leaves = -1;
#pragma unroll
    for (int v = 0; v < SEL_WAVES; ++v) {
        const uint32_t x = lightest[v];
        const int r = at[v];
        if (r >= 0 && (x < least || (x == least && r > leaves))) least = x, leaves = r;
    }
    leaves = __builtin_amdgcn_readfirstlane(leaves);
    if (a.kept) {
        int32_t *const kept = a.kept + (long)kvh * a.keep;
        for (int r = tid; r < a.keep; r += SEL_THREADS) kept[r] = r == leaves ? a.keep : r;
    }
    const TileAt t(g, kvh);
    const int page = leaves >> 4;
    char *const k_pool = reinterpret_cast<char *>(a.k_pool), *const v_pool = reinterpret_cast<char *>(a.v_pool);
    if (tid < 16) {
        const long src = (long)page_from * g.page_elems * 2;
        const int from = leaves < a.keep && tid == (leaves & 15) ? a.keep & 15 : -1;
        mk.row[tid] = mv.row[tid] = pk.row[tid] = pv.row[tid] = from;
        mk.at[tid] = src + t.codes;
        mv.at[tid] = src + t.codes;
        pk.at[tid] = src + t.powers;
        pv.at[tid] = src + t.powers;
    }
    __syncthreads();
    if (tid == 0) {
        const float last = w[a.keep];
        if (leaves < a.keep) w[leaves] = last;
        w[a.keep] = 0.0f;
    }
    if (leaves >= a.keep) return;
    const long dst = (long)a.table[page] * g.page_elems * 2;
    if (tid < 256) move_k<256>(g, t, mk, pk, k_pool, k_pool + dst, false, tid);
    else if (tid < 512) move_v<256>(g, t, mv, pv, v_pool, v_pool + dst, false, tid - 256);
}

// Whether the workgroup that chooses moves the rows itself: no launch of 3 us more, but a row of V is a part of each line of its four rows, of which a CU
// brings in 25 bytes a nanosecond. With its read-back, us: bf16 of eight heads of 128 dims, 16 of 1024 rows 16.3 -> 14.5, 32 of them 16.4 -> 15.3, 64
// (not taken) 16.3 -> 17.9; of two heads of 256 15.5 -> 14.5, 15.7 -> 17.1 (not taken); 4-bit, 64 rows, 15.1 -> 14.1, 128 15.2 -> 16.4.
static bool few_moves(const EvictArgs &a) {
    const int moves = std::min(a.keep, a.len - a.keep), four_rows = a.g.P * (a.g.fp4 ? 2 : a.g.f32 ? 16 : 8);
    return a.stretches == 1 && moves <= FEW_MOVES && moves * four_rows <= 32768;
}

size_t plan_evict(EvictArgs &a, bool lists_kept) {
    const size_t kvh = (size_t)a.g.kv_heads, gone = (size_t)(a.len - a.keep);
    a.stretches = a.len <= CHOSEN ? 1 : std::min((a.len + STRETCH - 1) / STRETCH, STRETCHES);
    a.per = ((a.len + a.stretches - 1) / a.stretches + SEL_THREADS - 1) / SEL_THREADS * SEL_THREADS;
    a.stretches = (a.len + a.per - 1) / a.per;
    a.few = few_moves(a);
    if (gone == 1 || a.few) return 0;
    if (a.stretches == 1) return kvh * (gone > 0 ? (size_t)a.keep : 0) * sizeof(int32_t);
    return kvh * (3 * gone + (lists_kept ? 0 : (size_t)a.keep) + (size_t)a.stretches * BINS) * sizeof(int32_t);
}
void place_evict(EvictArgs &a, void *scratch) {
    if (a.len - a.keep == 1 || a.few) return;
    const size_t kvh = (size_t)a.g.kv_heads, gone = (size_t)(a.len - a.keep);
    int32_t *p = static_cast<int32_t *>(scratch);
    const auto take = [&](size_t n) {
        int32_t *const at = p;
        p += n;
        return at;
    };
    if (a.stretches == 1) {
        a.from = gone > 0 ? take(kvh * (size_t)a.keep) : nullptr;
        return;
    }
    a.counts = take(kvh * a.stretches * BINS); // (first: read by twos)
    a.moved = reinterpret_cast<Mover *>(take(kvh * gone * 3));
    if (!a.kept) a.kept = take(kvh * (size_t)a.keep);
}

template <bool MOVES>
static void choose_rows(const EvictArgs &a, hipStream_t s) {
    const unsigned heads = (unsigned)a.g.kv_heads;
    if (a.len <= 4 * SEL_THREADS) evict_choose_kernel<4, MOVES><<<heads, SEL_THREADS, 0, s>>>(a);
    else if (a.len <= 8 * SEL_THREADS) evict_choose_kernel<8, MOVES><<<heads, SEL_THREADS, 0, s>>>(a);
    else evict_choose_kernel<16, MOVES><<<heads, SEL_THREADS, 0, s>>>(a);
}

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    const unsigned heads = (unsigned)a.g.kv_heads;
    if (a.len - a.keep == 1) {
        evict_one_kernel<<<heads, SEL_THREADS, 0, s>>>(a);
        return hipGetLastError();
    }
    if (a.few) {
        choose_rows<true>(a, s);
        return hipGetLastError();
    }
    if (a.stretches == 1) {
        choose_rows<false>(a, s);
    } else {
        const dim3 grid((unsigned)a.stretches, heads);
        evict_count_kernel<<<grid, SEL_THREADS, 0, s>>>(a);
        if (a.len <= 32 * SEL_THREADS) evict_select_kernel<32><<<grid, SEL_THREADS, 0, s>>>(a);
        else evict_select_kernel<0><<<grid, SEL_THREADS, 0, s>>>(a);
    }
    if (a.keep < a.len)
        evict_move_kernel<<<dim3((unsigned)(((a.keep + 15) / 16 + 7) / 8 * 8), heads, 2), MOVE_THREADS, 0, s>>>(a);
    return hipGetLastError();
}

} // namespace skv
