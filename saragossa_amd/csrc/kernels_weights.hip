// gfx950 kernels of the weights that cached rows get from queries:
//
//   w[h][r] += sum over the slots i of kv head h (queries and heads of its group) of exp(s_i[r] - M_i) / L_i
//   s_i[r] = scale q_i . K[h][r], r up to the query's own row;  M_i = max_r s_i[r], L_i = sum_r exp(s_i[r] - M_i)
//
// A weight needs its slot's M and L, sums over all rows, before it can be added to its row's sum over all slots. Few slots (a decoded token):
// K is read once, the scores stay in memory in between (4 bytes a slot and row beside the row of K), and a second launch adds up. Many slots (a chunk): the
// scores are made twice, once down the rows and once across the slots.
//
// S^T = K . Q^T on the matrix cores, sixteen rows by sixteen slots: lane l has rows 4 (l / 16) .. + 3 of slot l % 16. The
// operand of K is the page as it lies: of bf16 pages 8 dims a lane (32 a product), of f32 pages 4 dims (16), of 4-bit pages the 32 codes of one
// group, converted to bf16 (exact), whose power the lane holds: four products count dims 8 s .. 8 s + 7 of each of four groups, and the queries'
// operands are laid out to match. Queries are two or three bf16 terms, or f32.
#include <algorithm>

#include "fp4_tile.h"
#include "weights.h"

namespace skv {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float float4_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

enum { BF16 = 0, F32 = 1, FP4 = 2 };

// Products of a tile (of f32 pages four instructions each), what a lane loads of a page, and where a product's dims are.
template <int EL, int P>
struct Tile {
    static constexpr int BLOCKS = (P + 127) / 128; // 4-bit pages: of four groups
    static constexpr int STEPS = EL == BF16 ? P / 32 : EL == F32 ? P / 16 : 4 * BLOCKS;
    static constexpr int DIMS = EL == F32 ? 4 : 8; // of a lane's share of a product
    static __device__ __forceinline__ int dim(int step, int j) {
        return EL == BF16 ? step * 32 + j * 8 : EL == F32 ? step * 16 + j * 4 : (step >> 2) * 128 + j * 32 + (step & 3) * 8;
    }
    static constexpr int LOADS = EL == FP4 ? BLOCKS : STEPS; // of 16 bytes
    struct Raw {
        u32x4_t x[LOADS];
        uint32_t power[EL == FP4 ? BLOCKS : 1];
    };
    // Unit `unit` of 64 a load (the lane that would hold it) of a page
    template <bool ONCE>
    static __device__ __forceinline__ void load(Raw &r, int i, const uint16_t *pool, const Geom &g, int page, int kvh, int unit) {
        if constexpr (EL == FP4) {
            const int grp = i * 4 + (unit >> 4), row = unit & 15, held = min(grp, P / 32 - 1); // (groups past the last: zeros, see convert)
            const u32x4_t *p = reinterpret_cast<const u32x4_t *>(fp4_codes(pool, g, page, kvh)) + held * 16 + row;
            r.x[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
            r.power[i] = fp4_powers(pool, g, page, kvh)[k4_power(P, row, held)];
        } else {
            const u32x4_t *p = reinterpret_cast<const u32x4_t *>(pool + (long)page * g.page_elems + (long)kvh * g.tile_elems) + i * 64 + unit;
            r.x[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
        }
    }
    // Operand `step` of what `load` brought
    static __device__ __forceinline__ u32x4_t operand(const Raw &r, int step, int unit) {
        if constexpr (EL == FP4) {
            const uint32_t e = r.power[step >> 2] << 23, c = r.x[step >> 2][step & 3];
            u32x4_t o = {code_pair<0>(c, e), code_pair<1>(c, e), code_pair<2>(c, e), code_pair<3>(c, e)};
            if constexpr (P % 128 != 0)
                if ((step >> 2) * 4 + (unit >> 4) >= P / 32) o = u32x4_t{0, 0, 0, 0};
            return o;
        } else {
            return r.x[step];
        }
    }
};

template <int EL>
__device__ __forceinline__ float4_t product(u32x4_t k, u32x4_t q, float4_t s) {
    if constexpr (EL == F32) {
        const float4_t x = __builtin_bit_cast(float4_t, k), y = __builtin_bit_cast(float4_t, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], s, 0, 0, 0);
        return s;
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q), s, 0, 0, 0);
    }
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight values as bf16 terms
template <int N>
__device__ __forceinline__ void bf16_terms(float (&x)[8], u32x4_t (&out)[N]) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x[2 * i], x[2 * i + 1]}, b2));
            out[p][i] = t;
            x[2 * i] -= __uint_as_float(t << 16);
            x[2 * i + 1] -= __uint_as_float(t & 0xffff0000u);
        }
}

// A lane's share of a product's queries: DIMS dims of a slot, scaled, as PLANES operands (bf16 terms; f32: one).
template <int EL, int P, int PLANES>
__device__ __forceinline__ void query_operands(const WeightsArgs &a, int kvh, int slot, int dim, u32x4_t (&out)[PLANES]) {
    using T = Tile<EL, P>;
    float x[T::DIMS];
    const bool live = slot < a.n_slots;
    const float *row = a.q + context_row(a.g, kvh, min(slot, a.n_slots - 1)) * a.g.head_dim;
    const int hd = a.g.head_dim;
    if (a.q_vec) { // (head_dim is a multiple of four)
#pragma unroll
        for (int u = 0; u < T::DIMS / 4; ++u) {
            const float4_t v = *reinterpret_cast<const float4_t *>(row + min(dim + 4 * u, hd - 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * u + e] = v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < T::DIMS; ++e) x[e] = row[min(dim + e, hd - 1)];
    }
#pragma unroll
    for (int e = 0; e < T::DIMS; ++e) x[e] = live && dim + e < hd ? x[e] * a.qscale : 0.0f;
    if constexpr (EL == F32) {
        out[0] = __builtin_bit_cast(u32x4_t, float4_t{x[0], x[1], x[2], x[3]});
    } else {
        bf16_terms(x, out);
    }
}

// Last row that a slot sees
__device__ __forceinline__ int limit_of(const WeightsArgs &a, int slot) { return a.len - a.n_queries + slot_row(a.g, slot); }

// Running maximum and sum, of this lane's rows
struct Running {
    float m = -INFINITY, l = 0.0f;
    template <int N>
    __device__ __forceinline__ void add(const float4_t (&s)[N]) {
        float top = m;
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = l * exp2_of(m - base);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += exp2_of(s[i][e] - base);
        l = sum;
        m = top;
    }
    __device__ __forceinline__ void join(float m2, float l2) {
        const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
        l = l * exp2_of(m - base) + l2 * exp2_of(m2 - base);
        m = top;
    }
    // of all four rows of lanes
    __device__ __forceinline__ void across() {
        const float top = rows_max(m), base = top == -INFINITY ? 0.0f : top;
        l = rows_sum(l * exp2_of(m - base));
        m = top;
    }
};

// ---- few slots -----------------------------------------------------------------------------
// Bound by memory where rows are many (32768 of two heads of 256 dims, 33.5 MB: 8.4 us, 4 TB/s, and 3 for the second launch), by two launches
// where they are few (1024 of eight heads of 128: 4.2 and 3.0). One launch in which a workgroup holds a head's scores is slower from 32 rows on: a
// CU alone brings in some 25 bytes a nanosecond.
// One workgroup per (split of the rows, kv head, 16 slots): its wavefronts walk the pages in turn, G at a time, the next ones on their way.
template <int EL, int P>
struct Few {
    using T = Tile<EL, P>;
    static constexpr int PLANES = EL == F32 ? 1 : 3;
    static constexpr int G = EL == FP4 ? (P <= 128 ? 4 : 2) : EL == BF16 && P <= 128 ? 2 : 1;
};
// Workgroups and their wavefronts: 10 layers of 32768 rows of two heads of 256 dims 127 us, with 512 workgroups of four 133, with 1024, twice the
// splits to join, 156; 4-bit, 8 of 30001 of eight heads, 130, 132, 148. Few pages are divided until two wavefronts have work, since a CU brings in little
// alone: 383 rows of two heads of 512 dims, 4-bit 12.4 us with work for all eight, 9.1 for four, 8.8 for two; f32 17.7, 14.3, 14.1.
constexpr int FEW_WAVES = 8;
constexpr size_t FEW_WGS = 256;

template <int EL, int P>
__global__ __launch_bounds__(FEW_WAVES * 64) void weights_scores_kernel(WeightsArgs a) {
    using T = Tile<EL, P>;
    constexpr int PLANES = Few<EL, P>::PLANES, G = Few<EL, P>::G;
    __shared__ u32x4_t q[PLANES][T::STEPS][64];
    __shared__ float join[2][FEW_WAVES][16];
    const int split = blockIdx.x, kvh = blockIdx.y, tile = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int slot = tile * 16 + n;
    const int limit = limit_of(a, min(slot, a.n_slots - 1));
    const int pages = a.rows16 / 16;
    const int pb0 = (int)((long)split * pages / a.splits), pb1 = (int)((long)(split + 1) * pages / a.splits);

    typename T::Raw k[G];
    int ids[G];
    const auto ask = [&](int pb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < G; ++i) ids[i] = a.table[min(pb + i, pb1 - 1)];
    };
    const auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int u = 0; u < T::LOADS; ++u) T::template load<true>(k[i], u, a.k_pool, a.g, ids[i], kvh, lane);
    };
    const int stride = FEW_WAVES * G;
    int pb = pb0 + wave * G;
    if (pb1 > pb0) { // (uniform; a wavefront without pages of its own asks for the last one)
        ask(pb);
        load();
        ask(pb + stride);
    }
    for (int idx = tid; idx < T::STEPS * 64; idx += FEW_WAVES * 64) {
        u32x4_t x[PLANES];
        query_operands<EL, P, PLANES>(a, kvh, tile * 16 + (idx & 15), T::dim(idx >> 6, (idx >> 4) & 3), x);
#pragma unroll
        for (int p = 0; p < PLANES; ++p) q[p][idx >> 6][idx & 63] = x[p];
    }
    __syncthreads();
    Running run;
    float *const scores = a.scores + ((long)kvh * a.n_slots + slot) * a.rows16 + j * 4;
    for (; pb < pb1; pb += stride) {
        float4_t s[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float4_t part[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int step = 0; step < T::STEPS; ++step) {
                const u32x4_t o = T::operand(k[i], step, lane);
#pragma unroll
                for (int p = 0; p < PLANES; ++p) part[(step + p) & 1] = product<EL>(o, q[p][step][lane], part[(step + p) & 1]);
            }
            s[i] = part[0] + part[1];
        }
        if (pb + stride < pb1) {
            load();
            ask(pb + 2 * stride);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int row = (pb + i) * 16 + j * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = pb + i < pb1 && row + e <= limit ? s[i][e] : -INFINITY;
            if (pb + i < pb1 && slot < a.n_slots) *reinterpret_cast<float4_t *>(scores + (long)(pb + i) * 16) = s[i];
        }
        run.add(s);
    }
    run.across();
    if (j == 0) {
        join[0][wave][n] = run.m;
        join[1][wave][n] = run.l;
    }
    __syncthreads();
    if (tid < 16 && slot < a.n_slots) {
        Running all;
        for (int w = 0; w < FEW_WAVES; ++w) all.join(join[0][w][tid], join[1][w][tid]);
        const long at = ((long)kvh * a.n_slots + slot) * a.splits + split;
        a.part_m[at] = all.m;
        a.part_l[at] = all.l;
    }
}

// Largest and sum over a wavefront, every lane receiving the result
__device__ __forceinline__ float turned(float v, int by) { // lane's neighbour `by` places on, of its sixteen
    const int x = __float_as_int(v);
    switch (by) {
    case 1: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));
    case 2: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
    case 4: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
    default: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));
    }
}
__device__ __forceinline__ float lanes16_max(float v) {
#pragma unroll
    for (int o = 1; o < 16; o *= 2) v = fmaxf(v, turned(v, o));
    return v;
}
__device__ __forceinline__ float wave_max(float v) { return rows_max(lanes16_max(v)); }
__device__ __forceinline__ float lanes16_sum(float v) {
#pragma unroll
    for (int o = 1; o < 16; o *= 2) v += turned(v, o);
    return v;
}
__device__ __forceinline__ float wave_sum(float v) { return rows_sum(lanes16_sum(v)); }

// A score's weight; 0 of a row that the query does not see, also where its sum is a NaN
__device__ __forceinline__ float weight_of(float s, float m, float r) { return s == -INFINITY ? 0.0f : exp2_of(s - m) * r; }

// The scores' weights, added to the rows': a thread a row, its first scores on their way while every workgroup joins the splits' maxima
// and sums for itself: 16 or 64 lanes a slot, AT_ONCE of them asked for before the first is joined (48 slots of 1862 rows of eight heads of 128 dims, both
// launches: 14.3 us; a wavefront a slot, one after the other, and scores one after the other, 19.1).
constexpr int FEW_SLOTS = 64, FEW_SPLITS = 256;
template <int LANES, int PER, int AT_ONCE>
__device__ __forceinline__ void join_splits(const WeightsArgs &a, int kvh, float *m, float *r) {
    constexpr int SLOTS = 256 / LANES; // side by side
    const int lane = threadIdx.x % LANES;
    for (int base = 0; base < a.n_slots; base += SLOTS * AT_ONCE) {
        const int first = base + threadIdx.x / LANES;
        float pm[AT_ONCE][PER], pl[AT_ONCE][PER];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const long at = ((long)kvh * a.n_slots + min(first + u * SLOTS, a.n_slots - 1)) * a.splits + min(lane + i * LANES, a.splits - 1);
                pm[u][i] = a.part_m[at];
                pl[u][i] = a.part_l[at];
            }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (u > 0 && base + u * SLOTS >= a.n_slots) break; // (uniform)
            float top = pm[u][0];
#pragma unroll
            for (int i = 1; i < PER; ++i) top = fmaxf(top, pm[u][i]);
            top = LANES == 64 ? wave_max(top) : lanes16_max(top);
            const float from = top == -INFINITY ? 0.0f : top;
            float l = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) l += lane + i * LANES < a.splits ? pl[u][i] * exp2_of(pm[u][i] - from) : 0.0f;
            l = LANES == 64 ? wave_sum(l) : lanes16_sum(l);
            if (lane == 0 && first + u * SLOTS < a.n_slots) {
                m[first + u * SLOTS] = top;
                r[first + u * SLOTS] = 1.0f / l;
            }
        }
    }
}

__global__ __launch_bounds__(256) void weights_add_kernel(WeightsArgs a) {
    constexpr int EARLY = 8;
    __shared__ float m[FEW_SLOTS], r[FEW_SLOTS];
    const int kvh = blockIdx.y, tid = threadIdx.x;
    const long row = min((long)blockIdx.x * 256 + tid, (long)a.len - 1);
    const float *s = a.scores + (long)kvh * a.n_slots * a.rows16 + row;
    float *const to = a.weights + kvh * a.stride + row;
    float early[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) early[i] = s[(long)min(i, a.n_slots - 1) * a.rows16];
    const float before = *to;
    if (a.splits <= 16) join_splits<16, 1, 4>(a, kvh, m, r);
    else if (a.splits <= 64) join_splits<64, 1, 4>(a, kvh, m, r);
    else join_splits<64, FEW_SPLITS / 64, 2>(a, kvh, m, r);
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
        if (i < a.n_slots) sum += weight_of(early[i], m[i], r[i]);
    for (int slot = EARLY; slot < a.n_slots; slot += EARLY) {
#pragma unroll
        for (int i = 0; i < EARLY; ++i) early[i] = s[(long)min(slot + i, a.n_slots - 1) * a.rows16];
#pragma unroll
        for (int i = 0; i < EARLY; ++i)
            if (slot + i < a.n_slots) sum += weight_of(early[i], m[slot + i], r[slot + i]);
    }
    if ((long)blockIdx.x * 256 + tid < a.len) *to = before + sum;
}

// ---- many slots ----------------------------------------------------------------------------
// Numbers of f32 pages as three bf16 terms too, and six products (what is left out is below 2^-24): 96 cycles for 32 dims where the f32
// instruction takes 256. Whoever brings a page converts it.
//
// Bound by the matrix cores and, of the wider heads, by the LDS that feeds them. 512 rows of q16/kv2/hd256 over 16896, bf16: 128 us down the rows and
// 139 across the slots, 139 GFLOP as bf16 each (1.05 PFLOP/s; a large library product reaches 1.2), with three short launches 248 a layer in turn.
// 32 of q32/kv8/hd128 over 5003 f32 rows: 12.5 and 14.7 (f32 instructions: 28 and 24), 34 in all; 63 of q8/kv2/hd512 over 32204: 119 and 125.
template <int EL, int P>
struct Many {
    static constexpr int STEPS = EL == FP4 ? 4 * ((P + 127) / 128) : P / 32; // of 32 dims
    static constexpr int KPL = EL == F32 ? 3 : 1, QPL = EL == F32 ? 3 : 2;   // terms of keys, of queries
    static constexpr int K_OPS = KPL * STEPS, OPS = QPL * STEPS;            // operands of a page, of a tile of queries
    static constexpr int TILES = EL == F32 || P <= 256 ? 2 : 1;             // a wavefront's, in weights_stats_kernel
    static constexpr int PAGES = EL == F32 ? (P <= 128 ? 2 : 1) : P <= 128 ? 4 : P <= 256 ? 2 : 1; // staged at a time there
    static constexpr int KP = K_OPS <= 8 ? 4 : K_OPS == 24 ? 1 : 2;         // pages of a wavefront in weights_sum_kernel (24: 96 us with one where two take 102; 48: 156, 125)
    static constexpr int QT = P <= 128 ? 2 : 1;                             // tiles of queries staged at a time there
    // What brings a page's operands: a unit is a lane's 16 bytes (f32: twice that, eight dims of a row), 64 a load
    static constexpr int LOADS = EL == FP4 ? STEPS / 4 : STEPS;
    struct Raw {
        u32x4_t x[EL == F32 ? 2 : 1];
        uint32_t power;
    };
    static __device__ __forceinline__ Raw load(const uint16_t *pool, const Geom &g, int page, int kvh, int load, int unit) {
        Raw r;
        if constexpr (EL == FP4) {
            const int grp = min(load * 4 + (unit >> 4), P / 32 - 1); // (groups past the last: zeros, see put)
            r.x[0] = reinterpret_cast<const u32x4_t *>(fp4_codes(pool, g, page, kvh))[grp * 16 + (unit & 15)];
            r.power = fp4_powers(pool, g, page, kvh)[k4_power(P, unit & 15, grp)];
        } else {
            const u32x4_t *const p = reinterpret_cast<const u32x4_t *>(pool + (long)page * g.page_elems + (long)kvh * g.tile_elems);
            if constexpr (EL == F32) { // dims 32 load + 8 j .. + 7: two pieces of 4 dims, 16 units apart
                const int j = unit >> 4, at = (load * 2 + (j >> 1)) * 64 + (j & 1) * 32 + (unit & 15);
                r.x[0] = p[at];
                r.x[1] = p[at + 16];
            } else {
                r.x[0] = p[load * 64 + unit];
            }
        }
        return r;
    }
    // put(operand's number, operand) of each that the load has
    template <class F>
    static __device__ __forceinline__ void put(const Raw &r, int load, int unit, F f) {
        if constexpr (EL == FP4) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint32_t e = r.power << 23, c = r.x[0][s];
                u32x4_t o = {code_pair<0>(c, e), code_pair<1>(c, e), code_pair<2>(c, e), code_pair<3>(c, e)};
                if (P % 128 != 0 && load * 4 + (unit >> 4) >= P / 32) o = u32x4_t{0, 0, 0, 0};
                f(load * 4 + s, o);
            }
        } else if constexpr (EL == F32) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(r.x[e >> 2][e & 3]);
            u32x4_t o[3];
            bf16_terms(x, o);
#pragma unroll
            for (int p = 0; p < 3; ++p) f(p * STEPS + load, o[p]);
        } else {
            f(load, r.x[0]);
        }
    }
    // s += a step's products; key(term), query(term): operands
    template <class K, class Q>
    static __device__ __forceinline__ void step(float4_t &s, K key, Q query) {
        if constexpr (EL == F32) {
            s = product<BF16>(key(2), query(0), s);
            s = product<BF16>(key(0), query(2), s);
            s = product<BF16>(key(1), query(1), s);
            s = product<BF16>(key(1), query(0), s);
            s = product<BF16>(key(0), query(1), s);
            s = product<BF16>(key(0), query(0), s);
        } else {
            s = product<BF16>(key(0), query(1), s);
            s = product<BF16>(key(0), query(0), s);
        }
    }
};

// The queries as operands, [tile][term][step][64 lanes]
template <int EL, int P>
__global__ __launch_bounds__(256) void weights_queries_kernel(WeightsArgs a) {
    using M = Many<EL, P>;
    constexpr int LAYOUT = EL == FP4 ? FP4 : BF16;
    const int kvh = blockIdx.y, tile = blockIdx.x;
    u32x4_t *const out = reinterpret_cast<u32x4_t *>(a.q_ops) + ((long)kvh * a.tiles + tile) * (M::OPS * 64);
    for (int idx = threadIdx.x; idx < M::STEPS * 64; idx += 256) {
        u32x4_t x[M::QPL];
        query_operands<LAYOUT, P, M::QPL>(a, kvh, tile * 16 + (idx & 15), Tile<LAYOUT, P>::dim(idx >> 6, (idx >> 4) & 3), x);
#pragma unroll
        for (int p = 0; p < M::QPL; ++p) out[p * M::STEPS * 64 + idx] = x[p];
    }
}

// M and L of each slot: a wavefront holds the queries of TILES tiles, the pages come through LDS for all four. A lane keeps a maximum of its own
// rows, joined at the end.
template <int EL, int P>
__global__ __launch_bounds__(256) void weights_stats_kernel(WeightsArgs a) {
    using M = Many<EL, P>;
    constexpr int NP = M::PAGES, UNITS = NP * M::LOADS * 64, LOADS = (UNITS + 255) / 256;
    extern __shared__ __attribute__((aligned(16))) u32x4_t pages[]; // [2][NP][K_OPS][64]
    const int split = blockIdx.x, kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int tile0 = (int)blockIdx.z * 4 * M::TILES;
    const int last = min((tile0 + 4 * M::TILES) * 16, a.n_slots) - 1; // slot
    const int n_pages = (limit_of(a, last) >> 4) + 1;
    const int pb0 = (int)((long)split * n_pages / a.splits), pb1 = (int)((long)(split + 1) * n_pages / a.splits);

    u32x4_t q[M::TILES][M::OPS];
    int limit[M::TILES], lowest[M::TILES];
    Running run[M::TILES];
#pragma unroll
    for (int t = 0; t < M::TILES; ++t) {
        const int tile = min(tile0 + wave * M::TILES + t, a.tiles - 1);
        const u32x4_t *p = reinterpret_cast<const u32x4_t *>(a.q_ops) + ((long)kvh * a.tiles + tile) * (M::OPS * 64) + lane;
#pragma unroll
        for (int i = 0; i < M::OPS; ++i) q[t][i] = p[i * 64];
        limit[t] = limit_of(a, min(tile * 16 + n, a.n_slots - 1));
        lowest[t] = limit_of(a, tile * 16);
    }
    // the loads of a thread: units tid, tid + 256, .. of [page][load][64]
    typename M::Raw raw[LOADS];
    const auto fetch = [&](int pb) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int idx = min(tid + u * 256, UNITS - 1), page = idx / (M::LOADS * 64);
            raw[u] = M::load(a.k_pool, a.g, a.table[min(pb + page, pb1 - 1)], kvh, idx / 64 % M::LOADS, idx & 63);
        }
    };
    const auto stage = [&](int buf) __attribute__((always_inline)) {
        u32x4_t *const to = pages + (long)buf * NP * M::K_OPS * 64;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int idx = tid + u * 256, page = idx / (M::LOADS * 64);
            if (UNITS % 256 == 0 || idx < UNITS)
                M::put(raw[u], idx / 64 % M::LOADS, idx & 63, [&](int op, u32x4_t x) __attribute__((always_inline)) { to[(page * M::K_OPS + op) * 64 + (idx & 63)] = x; });
        }
    };
    int buf = 0;
    if (pb1 > pb0) fetch(pb0);
    for (int pb = pb0; pb < pb1; pb += NP, buf ^= 1) {
        stage(buf);
        __syncthreads(); // (two buffers: a wavefront that stages the next one has read the one before this)
        if (pb + NP < pb1) fetch(pb + NP);
        const u32x4_t *const k = pages + (long)buf * NP * M::K_OPS * 64 + lane;
        float4_t s[M::TILES][NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
#pragma unroll
            for (int t = 0; t < M::TILES; ++t) s[t][i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int step = 0; step < M::STEPS; ++step) {
                u32x4_t o[M::KPL];
#pragma unroll
                for (int p = 0; p < M::KPL; ++p) o[p] = k[(i * M::K_OPS + p * M::STEPS + step) * 64];
#pragma unroll
                for (int t = 0; t < M::TILES; ++t)
                    M::step(s[t][i], [&](int p) { return o[p]; }, [&](int p) { return q[t][p * M::STEPS + step]; });
            }
        }
#pragma unroll
        for (int t = 0; t < M::TILES; ++t) {
            if ((pb + NP) * 16 > lowest[t] + 1 || pb + NP > pb1) { // (uniform)
#pragma unroll
                for (int i = 0; i < NP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = (pb + i) * 16 + j * 4 + e;
                        s[t][i][e] = pb + i < pb1 && row <= limit[t] ? s[t][i][e] : -INFINITY;
                    }
            }
            run[t].add(s[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < M::TILES; ++t) {
        run[t].across();
        const int slot = (tile0 + wave * M::TILES + t) * 16 + n;
        if (j == 0 && slot < a.n_slots) {
            const long at = ((long)kvh * a.n_slots + slot) * a.splits + split;
            a.part_m[at] = run[t].m;
            a.part_l[at] = run[t].l;
        }
    }
}

// M and 1 / L of each slot from its splits, a wavefront a slot; slots that fill the last tile get 0s.
__global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
    const int kvh = blockIdx.y, slot = (int)blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    float2 out = {0.0f, 0.0f};
    if (slot < a.n_slots) {
        Running run;
        const long at = ((long)kvh * a.n_slots + slot) * a.splits;
        for (int i = lane; i < a.splits; i += 64) run.join(a.part_m[at + i], a.part_l[at + i]);
        const float top = wave_max(run.m), base = top == -INFINITY ? 0.0f : top;
        out = make_float2(top, 1.0f / wave_sum(run.l * exp2_of(run.m - base)));
    }
    if (lane == 0) a.stats[(long)kvh * a.tiles * 16 + slot] = out;
}

// The weights of each row: a wavefront holds KP pages of keys, the queries come through LDS for all four.
template <int EL, int P>
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsArgs a) {
    using M = Many<EL, P>;
    constexpr int UNITS = (M::QT * M::OPS * 64 + 255) / 256; // of a thread
    constexpr int ALL = M::QT * M::OPS * 64;
    extern __shared__ __attribute__((aligned(16))) u32x4_t queries[]; // [2][QT][OPS][64], then the slots' M and 1 / L, [2][QT * 16]
    float2 *const stats = reinterpret_cast<float2 *>(queries + 2 * M::QT * M::OPS * 64);
    const int kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int n_pages = a.rows16 / 16, first_page = (int)blockIdx.x * 4 * M::KP, page0 = first_page + wave * M::KP;
    // tiles that see the workgroup's first row, divided among the splits
    const int t_lo = (int)((long)max(first_page * 16 - (a.len - a.n_queries), 0) * a.g.gqa / 16);
    const int span = a.tiles - t_lo;
    const int t0 = t_lo + (int)((long)blockIdx.z * span / a.sum_splits), t1 = t_lo + (int)((long)(blockIdx.z + 1) * span / a.sum_splits);

    u32x4_t k[M::KP][M::K_OPS];
    {
        typename M::Raw raw[M::KP][M::LOADS];
#pragma unroll
        for (int i = 0; i < M::KP; ++i) {
            const int id = a.table[min(page0 + i, n_pages - 1)];
#pragma unroll
            for (int u = 0; u < M::LOADS; ++u) raw[i][u] = M::load(a.k_pool, a.g, id, kvh, u, lane);
        }
#pragma unroll
        for (int i = 0; i < M::KP; ++i)
#pragma unroll
            for (int u = 0; u < M::LOADS; ++u) M::put(raw[i][u], u, lane, [&](int op, u32x4_t x) __attribute__((always_inline)) { k[i][op] = x; });
    }
    const u32x4_t *const q_ops = reinterpret_cast<const u32x4_t *>(a.q_ops) + (long)kvh * a.tiles * (M::OPS * 64);
    const float2 *const all = a.stats + (long)kvh * a.tiles * 16;
    u32x4_t on_way[UNITS];
    float2 stat = {0.0f, 0.0f};
    const auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int idx = min(tid + u * 256, ALL - 1), tile = min(t + idx / (M::OPS * 64), t1 - 1);
            on_way[u] = q_ops[(long)tile * (M::OPS * 64) + idx % (M::OPS * 64)];
        }
        if (tid < M::QT * 16) stat = all[min(t * 16 + tid, a.tiles * 16 - 1)];
    };
    float4_t sum[M::KP];
#pragma unroll
    for (int i = 0; i < M::KP; ++i) sum[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    int buf = 0;
    if (t1 > t0) fetch(t0);
    for (int t = t0; t < t1; t += M::QT, buf ^= 1) {
        u32x4_t *const to = queries + (long)buf * M::QT * M::OPS * 64;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
            if (ALL % 256 == 0 || tid + u * 256 < ALL) to[tid + u * 256] = on_way[u];
        if (tid < M::QT * 16) stats[buf * M::QT * 16 + tid] = stat;
        __syncthreads(); // (two buffers, as above)
        if (t + M::QT < t1) fetch(t + M::QT);
#pragma unroll
        for (int c = 0; c < M::QT; ++c) {
            if (t + c >= t1) break; // uniform
            const u32x4_t *const q = to + c * M::OPS * 64 + lane;
            float4_t s[M::KP];
#pragma unroll
            for (int i = 0; i < M::KP; ++i) s[i] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int step = 0; step < M::STEPS; ++step) {
                u32x4_t o[M::QPL];
#pragma unroll
                for (int p = 0; p < M::QPL; ++p) o[p] = q[(p * M::STEPS + step) * 64];
#pragma unroll
                for (int i = 0; i < M::KP; ++i) M::step(s[i], [&](int p) { return k[i][p * M::STEPS + step]; }, [&](int p) { return o[p]; });
            }
            const float2 mr = stats[(buf * M::QT + c) * 16 + n];
            const int slot = (t + c) * 16 + n;
            if ((page0 + M::KP) * 16 > limit_of(a, (t + c) * 16) + 1 || (t + c + 1) * 16 > a.n_slots) { // uniform
                const int limit = slot < a.n_slots ? limit_of(a, slot) : -1;
#pragma unroll
                for (int i = 0; i < M::KP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float w = exp2_of(s[i][e] - mr.x) * mr.y;
                        sum[i][e] += (page0 + i) * 16 + j * 4 + e <= limit ? w : 0.0f;
                    }
            } else {
#pragma unroll
                for (int i = 0; i < M::KP; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[i][e] += exp2_of(s[i][e] - mr.x) * mr.y;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < M::KP; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][e] = lanes16_sum(sum[i][e]);
        const int row = (page0 + i) * 16 + j * 4;
        if (n == 0 && page0 + i < n_pages) {
            if (a.sum_splits > 1) {
                *reinterpret_cast<float4_t *>(a.part_sum + ((long)blockIdx.z * a.g.kv_heads + kvh) * a.rows16 + row) = sum[i];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (row + e < a.len) a.weights[kvh * a.stride + row + e] += sum[i][e];
            }
        }
    }
}

__global__ __launch_bounds__(256) void weights_collect_kernel(WeightsArgs a) {
    const int kvh = blockIdx.y;
    const long row = (long)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.len) return;
    float sum = 0.0f;
    for (int z = 0; z < a.sum_splits; ++z) sum += a.part_sum[((long)z * a.g.kv_heads + kvh) * a.rows16 + row];
    a.weights[kvh * a.stride + row] += sum;
}

// ---- host side -----------------------------------------------------------------------------
static bool few_slots(const WeightsArgs &a) { return a.n_slots <= FEW_SLOTS; }

template <int EL, int P>
static size_t plan_as(WeightsArgs &a) {
    const size_t kvh = (size_t)a.g.kv_heads, pages = (size_t)a.rows16 / 16;
    a.tiles = (a.n_slots + 15) / 16;
    if (few_slots(a)) {
        const size_t wgs = kvh * a.tiles;
        a.splits = (int)std::max<size_t>(std::min<size_t>({FEW_WGS / wgs, pages / (2 * Few<EL, P>::G), FEW_SPLITS}), 1);
        return (kvh * a.n_slots * (a.rows16 + 2 * (size_t)a.splits)) * sizeof(float);
    }
    using M = Many<EL, P>;
    const size_t stat_wgs = kvh * ((a.tiles + 4 * M::TILES - 1) / (4 * M::TILES)), sum_wgs = kvh * ((pages + 4 * M::KP - 1) / (4 * M::KP));
    a.splits = (int)std::max<size_t>(std::min<size_t>(512 / stat_wgs, pages / (2 * M::PAGES)), 1);
    a.sum_splits = (int)std::max<size_t>(std::min<size_t>(512 / sum_wgs, (size_t)a.tiles / (2 * M::QT)), 1);
    const size_t ops = kvh * a.tiles * M::OPS * 64 * sizeof(uint4);
    return ops + kvh * a.tiles * 16 * sizeof(float2) + 2 * kvh * a.n_slots * a.splits * sizeof(float) +
           (a.sum_splits > 1 ? (size_t)a.sum_splits * kvh * a.rows16 * sizeof(float) : 0);
}
template <int EL, int P>
static void place_as(WeightsArgs &a, char *p) {
    const size_t kvh = (size_t)a.g.kv_heads;
    const auto take = [&](size_t bytes) {
        char *at = p;
        p += bytes;
        return at;
    };
    if (few_slots(a)) {
        a.scores = reinterpret_cast<float *>(take(kvh * a.n_slots * (size_t)a.rows16 * sizeof(float)));
    } else {
        a.q_ops = reinterpret_cast<uint4 *>(take(kvh * a.tiles * Many<EL, P>::OPS * 64 * sizeof(uint4)));
        a.stats = reinterpret_cast<float2 *>(take(kvh * a.tiles * 16 * sizeof(float2)));
        if (a.sum_splits > 1) a.part_sum = reinterpret_cast<float *>(take((size_t)a.sum_splits * kvh * a.rows16 * sizeof(float)));
    }
    a.part_m = reinterpret_cast<float *>(take(kvh * a.n_slots * (size_t)a.splits * sizeof(float)));
    a.part_l = reinterpret_cast<float *>(take(kvh * a.n_slots * (size_t)a.splits * sizeof(float)));
}
template <int EL, int P>
static hipError_t launch_as(const WeightsArgs &a, hipStream_t s) {
    const unsigned kvh = (unsigned)a.g.kv_heads, rows256 = (unsigned)((a.len + 255) / 256);
    if (few_slots(a)) {
        weights_scores_kernel<EL, P><<<dim3((unsigned)a.splits, kvh, (unsigned)a.tiles), FEW_WAVES * 64, 0, s>>>(a);
        weights_add_kernel<<<dim3(rows256, kvh), 256, 0, s>>>(a);
        return hipGetLastError();
    }
    using M = Many<EL, P>;
    static std::atomic<uint64_t> stats_done{0}, sum_done{0};
    hipError_t e = allow_full_lds(reinterpret_cast<const void *>(weights_stats_kernel<EL, P>), stats_done);
    if (e == hipSuccess) e = allow_full_lds(reinterpret_cast<const void *>(weights_sum_kernel<EL, P>), sum_done);
    if (e != hipSuccess) return e;
    weights_queries_kernel<EL, P><<<dim3((unsigned)a.tiles, kvh), 256, 0, s>>>(a);
    weights_stats_kernel<EL, P><<<dim3((unsigned)a.splits, kvh, (unsigned)((a.tiles + 4 * M::TILES - 1) / (4 * M::TILES))), 256,
                                  2 * M::PAGES * M::K_OPS * 1024, s>>>(a);
    weights_join_kernel<<<dim3((unsigned)(a.tiles * 4), kvh), 256, 0, s>>>(a);
    weights_sum_kernel<EL, P><<<dim3((unsigned)((a.rows16 / 16 + 4 * M::KP - 1) / (4 * M::KP)), kvh, (unsigned)a.sum_splits), 256,
                                2 * M::QT * (M::OPS * 1024 + 16 * sizeof(float2)), s>>>(a);
    if (a.sum_splits > 1) weights_collect_kernel<<<dim3(rows256, kvh), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int EL, int P>
static size_t at_once_as(const Geom &g, size_t before, size_t left) {
    const size_t kvh = (size_t)g.kv_heads, gqa = (size_t)g.gqa, rows16 = (before + left + 15) / 16 * 16;
    const size_t per_slot = left * gqa <= FEW_SLOTS ? kvh * rows16 * sizeof(float) : kvh * Many<EL, P>::OPS * 64;
    const size_t most = (size_t)(left * gqa <= FEW_SLOTS ? 256 : 128) << 20;
    return std::min(left, std::max<size_t>(most / (per_slot * gqa), 1));
}

// f<EL, P>(..) of the layer's element and padded head
#define SKV_WEIGHTS_OF(f, g, ...)                                                                    \
    do {                                                                                             \
        if ((g).f32) SKV_WEIGHTS_P(f, F32, (g).P, __VA_ARGS__);                                      \
        if ((g).fp4) SKV_WEIGHTS_P(f, FP4, (g).P, __VA_ARGS__);                                      \
        SKV_WEIGHTS_P(f, BF16, (g).P, __VA_ARGS__);                                                  \
    } while (0)
#define SKV_WEIGHTS_P(f, EL, p, ...)               \
    switch (p) {                                   \
    case 32: return f<EL, 32>(__VA_ARGS__);        \
    case 64: return f<EL, 64>(__VA_ARGS__);        \
    case 96: return f<EL, 96>(__VA_ARGS__);        \
    case 128: return f<EL, 128>(__VA_ARGS__);      \
    case 256: return f<EL, 256>(__VA_ARGS__);      \
    default: return f<EL, 512>(__VA_ARGS__);       \
    }

size_t weights_at_once(const Geom &g, size_t before, size_t left) { SKV_WEIGHTS_OF(at_once_as, g, g, before, left); }
size_t plan_weights(WeightsArgs &a) { SKV_WEIGHTS_OF(plan_as, a.g, a); }
void place_weights(WeightsArgs &a, void *scratch) { SKV_WEIGHTS_OF(place_as, a.g, a, static_cast<char *>(scratch)); }
hipError_t launch_weights(const WeightsArgs &args, hipStream_t s) {
    WeightsArgs a = args;
    a.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.g.head_dim % 4 == 0;
    SKV_WEIGHTS_OF(launch_as, a.g, a, s);
}

} // namespace skv
