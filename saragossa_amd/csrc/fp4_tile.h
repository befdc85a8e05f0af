// The 4-bit element's pages, shared by its kernels.
//
// A row of a head is kept in groups of 32 dims: codes of 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one power
// of two a group, as a byte e + 127. 4.25 bits a value, 3.76 times less than bf16. For a group whose largest magnitude is t
//
//   e    = the smallest with t <= 7 * 2^e, between -125 and 125
//   code = x / 2^e to the nearest, ties to the even code, above 6 to 6
//
// 7 and not 6: a value of 7 becomes 6, off by one, which is half of the step between 4 and 6 that rounding costs there anyway, and a
// smaller e halves every step of the group. The bounds of e keep every value a normal bf16 (and so f32) number: 0.5 * 2^-125 to
// 6 * 2^125. A group with an infinity or NaN has the byte 255 and reads as NaN, all of it. A value is a code of two significant bits times a power
// of two, so bf16 holds it exactly, and so the products below multiply what was stored, not a rounding of it.
//
// Codes and powers are what gfx950 converts (v_cvt_scalef32_pk_bf16_fp4: two values an instruction; it looks at the exponent field of its
// scale operand alone) and multiplies (v_mfma_scale_f32_16x16x128_f8f6f4, a power a lane's 32 codes): the layout is theirs.
//
// A page (16 rows, all kv heads) is the codes of kv head 0, 1, .., then the powers of kv head 0, 1, .. (so codes start at whole KiBs where
// head_dim is 128 or more):
//
//   K codes   [P/32 groups][16 rows][16 bytes]                dims 2i and 2i + 1 of the group in byte i: a lane's A operand
//   K powers  [4 groups of 128 dims][16 rows][P/128 blocks]
//   V codes   [P/32/U][4 row-quads][16 cols][U groups][4 rows] dims c and c + 16 of the group in a byte; U = the groups of 16 bytes, at most 4
//   V powers  [4 row-quads][P/32 groups][4 rows]
#pragma once

#include "skv_internal.h"

namespace skv {

__host__ __device__ constexpr int fp4_code_bytes(int P) { return 8 * P; }  // of one (page, kv head), K or V
__host__ __device__ constexpr int fp4_power_bytes(int P) { return P / 2; }
__host__ __device__ constexpr int fp4_quad(int P) { return P / 32 < 4 ? P / 32 : 4; } // U
// Byte of an element's code, from the start of the (page, kv head) codes, and of its power, from that of the powers
__host__ __device__ inline int k4_code(int r, int d) { return ((d >> 5) * 16 + r) * 16 + ((d & 31) >> 1); } // nibble d & 1
__host__ __device__ inline int k4_power(int P, int r, int g) { return ((g & 3) * 16 + r) * ((P + 127) / 128) + (g >> 2); }
__host__ __device__ inline int v4_code(int P, int r, int d) { // nibble (d >> 4) & 1
    const int U = fp4_quad(P), g = d >> 5;
    return (((g / U) * 64 + (r >> 2) * 16 + (d & 15)) * U + g % U) * 4 + (r & 3);
}
__host__ __device__ inline int v4_power(int P, int r, int g) { return ((r >> 2) * (P / 32) + g) * 4 + (r & 3); }

#ifdef __HIPCC__
// Where the codes and the powers of a kv head's tile start
__device__ __forceinline__ const uint8_t *fp4_codes(const uint16_t *pool, const Geom &g, long page, int kvh) {
    return reinterpret_cast<const uint8_t *>(pool) + page * g.page_elems * 2 + kvh * fp4_code_bytes(g.P);
}
__device__ __forceinline__ const uint8_t *fp4_powers(const uint16_t *pool, const Geom &g, long page, int kvh) {
    return reinterpret_cast<const uint8_t *>(pool) + page * g.page_elems * 2 + g.kv_heads * fp4_code_bytes(g.P) + kvh * fp4_power_bytes(g.P);
}
// A group's byte from the bits of its largest magnitude (as integers, NaN and infinities above all numbers): the exponent, one more where the
// leading bits pass 1.75, less two. A group of zeros has the power 1.
__device__ __forceinline__ uint32_t fp4_power_of(uint32_t top) {
    if (top >= 0x7f800000u) return 255u;
    if (top == 0) return 127u;
    const int e = (int)((top + 0x1fffffu) >> 23) - 2;
    return (uint32_t)min(max(e, 2), 252);
}
// The largest of 8 neighbouring lanes' x
__device__ __forceinline__ uint32_t max_of_8(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));  // lane ^ 1
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));  // lane ^ 2
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, false)); // the other four
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// Four dims of a group, an eighth of it (the lane's, of 8 neighbours), as 16 bits of codes; the group's byte in `power`
__device__ __forceinline__ uint32_t fp4_codes_of(const float (&x)[4], uint32_t &power) {
    const uint32_t top = max_of_8(max(max(magnitude(x[0]), magnitude(x[1])), max(magnitude(x[2]), magnitude(x[3]))));
    power = fp4_power_of(top);
    const float scale = __uint_as_float(power << 23);
    const uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1) & 0xffffu;
}
// Four codes in a byte each
__device__ __forceinline__ uint32_t nibbles_apart(uint32_t c) {
    c = (c | c << 8) & 0x00ff00ffu;
    return (c | c << 4) & 0x0f0f0f0fu;
}
// N words from p, as wide as its alignment (16 bytes of a multiple of four words, else 4 times their number) allows
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&x)[N], const uint8_t *p) {
    typedef __attribute__((ext_vector_type(2))) uint32_t u2;
    typedef __attribute__((ext_vector_type(4))) uint32_t u4;
#pragma unroll
    for (int i = 0; i + 4 <= N; i += 4) {
        const u4 v = *reinterpret_cast<const u4 *>(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i + e] = v[e];
    }
    if constexpr (N == 3) { // (12 bytes apart: words)
        typedef __attribute__((ext_vector_type(3), aligned(4))) uint32_t u3;
        const u3 v = *reinterpret_cast<const u3 *>(p);
        x[0] = v[0], x[1] = v[1], x[2] = v[2];
    } else if constexpr (N == 2) {
        const u2 v = *reinterpret_cast<const u2 *>(p);
        x[0] = v[0], x[1] = v[1];
    } else if constexpr (N == 1) {
        x[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// 255 in the bytes of w that are
__device__ __forceinline__ uint32_t bytes_255(uint32_t w) {
    const uint32_t x = ~w, zero = ~(((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x | 0x7f7f7f7fu); // the top bit of the bytes of x that are 0
    return (zero >> 7) * 255u;
}

// Byte B of two codes as two bf16 values, the low nibble's in the low half; `power` has the group's byte in its exponent field (the rest of
// it is not looked at)
template <int B>
__device__ __forceinline__ uint32_t code_pair(uint32_t codes, uint32_t power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, __uint_as_float(power), B));
}

// V as f16, at 2^-8 of its value, against probabilities at 2^8 of theirs: exact for powers of 2^-15 to 2^16 (codes are multiples of 1/2 up to 6, f16's
// steps 2^-24, its largest 65504), and two f16 terms hold a probability to 2^-22 of itself, or 2^-33 of the largest,
// where two bf16 terms hold 2^-17, three 2^-24.
// Four rows' powers, those above and below it at 255 or below 112: bits in `far`.
constexpr int V_SHIFT = 8;
constexpr float P_SCALE = 1.0f / 256.0f; // of the sums of probabilities
__device__ __forceinline__ uint32_t fp4_far(uint32_t powers) { return ((powers + 0x10101010u) ^ 0x80808080u) & 0xe0e0e0e0u; } // (bytes 112 to 143 have none)
template <int B>
__device__ __forceinline__ uint32_t code_pair_f16(uint32_t codes, uint32_t power) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, __uint_as_float(power), B));
}
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
// x and y as two terms
__device__ __forceinline__ void f16_terms(float x, float y, uint32_t &hi, uint32_t &lo) {
    typedef __attribute__((ext_vector_type(2))) float f2;
    const f16x2_t h = __builtin_convertvector(f2{x, y}, f16x2_t);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x - (float)h[0], y - (float)h[1]}, f16x2_t));
}

#endif

// Entry e of a ring chunk's list of pages (ChunkPages): whether it lies in the chunk's scratch, and its page there or in the layer's pools.
__device__ __forceinline__ bool fp4_in_scratch(const ChunkPages &c, int e) { return e >= c.apart_lo && e < c.apart_hi; }
__device__ __forceinline__ int fp4_ring_page(const DecodeArgs &a, const ChunkPages &c, int e) {
    int at = e < c.n_old ? c.start + e : c.new_start + min(e - c.n_old, c.ring_pages - 1);
    if (at >= c.ring_pages) at -= c.ring_pages;
    const int page = a.table[max(at, 0)]; // (every lane asks for some entry: no load of its own under a condition)
    return fp4_in_scratch(c, e) ? c.apart_id + e : page;
}

} // namespace skv
