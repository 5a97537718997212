// Packed blocks as integer levels: every format's weight is dl * level - ml, with an 8-bit
// level and float32 dl, ml per 32 or per 16 values. Products with Q8_0 activations (8-bit
// levels, one scale per 32 values) are then sums of exact integer dot products.
//
// Unit: 32 consecutive values of a row, aligned to 32 (one Q8_0 block of the activations).
// Lv<T>::load brings what unit j of a block needs into WORDS registers, Lv<T>::levels makes of
// them its levels as 8 words (4 levels each, value order) and dl, ml of its two halves of 16
// values; two steps, so that loads can run ahead. G16: the halves' scales differ; HASMIN: ml is
// not always zero; SIGNED: levels are int8 (else 0 .. 31). FOLD: a superblock has one scale, base, and
// integer factors sub (dl[h] = base * sub(h)) whose products with the levels stay below 2048
// (Q6_K: up to 4096). dl and ml are exact: a float16
// times a few scale bits.
#pragma once

#include "qs_kernels.h"

namespace qs {

// Global memory through the read-only path, shared memory (SM) plainly.
template <bool SM, class V>
__device__ __forceinline__ V ld_v(const V* p) {
    if constexpr (SM) return *p;
    else return __ldg(p);
}

// N words at any address, little-endian. AL: the alignment that is known; below 4 the aligned
// words that hold the bytes are loaded and shifted (none of them lies wholly outside the bytes).
template <int N, int AL, bool SM = false>
__device__ __forceinline__ void ld_words(const uint8_t* p, uint32_t* w) {
    if constexpr (AL >= 16 && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = ld_v<SM>(reinterpret_cast<const uint4*>(p) + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (AL >= 8 && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 v = ld_v<SM>(reinterpret_cast<const uint2*>(p) + i);
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else if constexpr (AL >= 4) {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = ld_v<SM>(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
        const uint32_t off = (uint32_t)(uintptr_t)p & 3, sh = 8 * off;
        const uint32_t* a = reinterpret_cast<const uint32_t*>(p - off);
        uint32_t v[N + 1];
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = ld_v<SM>(a + i);
        v[N] = off ? ld_v<SM>(a + N) : 0u;
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = __funnelshift_r(v[i], v[i + 1], sh);
    }
}
template <int AL, bool SM = false>
__device__ __forceinline__ uint32_t ld_u16(const uint8_t* p) {
    if constexpr (AL >= 2) return ld_v<SM>(reinterpret_cast<const unsigned short*>(p));
    else return (uint32_t)ld_v<SM>(p) | ((uint32_t)ld_v<SM>(p + 1) << 8);
}
__device__ __forceinline__ float h2f(uint32_t bits) { return f16_val((uint16_t)bits); }
// 4 bits -> 4 bytes of 0 / 1 (bit i -> byte i)
__device__ __forceinline__ uint32_t bits_to_bytes(uint32_t b) { return ((b & 0xFu) * 0x00204081u) & 0x01010101u; }
// bytes of w (1 .. 127) negated where the byte of m (0 / 1) is 1: no byte carries into the next
__device__ __forceinline__ uint32_t neg_bytes(uint32_t w, uint32_t m) { return (w ^ (m * 0xFFu)) + m; }
// bytes (below 128) minus the bytes of b (up to 128) as int8: bit 7 set keeps every difference from
// borrowing, and is then taken back
__device__ __forceinline__ uint32_t sub_bytes(uint32_t w, uint32_t b) { return ((w | 0x80808080u) - b) ^ 0x80808080u; }

template <int T> struct Lv;

template <> struct Lv<QS_Q4_0> {
    static constexpr int QK = 32, BB = 18, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = false;
    static constexpr int WORDS = 5;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int, uint32_t* r) {
        ld_words<4, 1, SM>(b + 2, r);
        r[4] = ld_u16<AL, SM>(b);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[4]);
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = sub_bytes(r[i] & 0x0F0F0F0Fu, 0x08080808u);
            q[4 + i] = sub_bytes((r[i] >> 4) & 0x0F0F0F0Fu, 0x08080808u);
        }
    }
};

template <> struct Lv<QS_Q4_1> {
    static constexpr int QK = 32, BB = 20, MAXAL = 4;
    static constexpr bool G16 = false, HASMIN = true, SIGNED = false, FOLD = false;
    static constexpr int WORDS = 5;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int, uint32_t* r) {
        ld_words<5, AL, SM>(b, r);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[0] & 0xFFFFu);
        ml[0] = ml[1] = -h2f(r[0] >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = r[1 + i] & 0x0F0F0F0Fu;
            q[4 + i] = (r[1 + i] >> 4) & 0x0F0F0F0Fu;
        }
    }
    // the block's minima, one per unit (per 16 values for Q2_K)
    template <int AL>
    __device__ static void minima(const uint8_t* b, float* m) { m[0] = -h2f(ld_u16<AL>(b + 2)); }
};

template <> struct Lv<QS_Q5_0> {
    static constexpr int QK = 32, BB = 22, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = false;
    static constexpr int WORDS = 6;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int, uint32_t* r) {
        ld_words<5, 1, SM>(b + 2, r);
        r[5] = ld_u16<AL, SM>(b);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[5]);
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = sub_bytes((r[1 + i] & 0x0F0F0F0Fu) | (bits_to_bytes(r[0] >> (4 * i)) << 4), 0x10101010u);
            q[4 + i] = sub_bytes(((r[1 + i] >> 4) & 0x0F0F0F0Fu) | (bits_to_bytes(r[0] >> (16 + 4 * i)) << 4), 0x10101010u);
        }
    }
};

template <> struct Lv<QS_Q5_1> {
    static constexpr int QK = 32, BB = 24, MAXAL = 8;
    static constexpr bool G16 = false, HASMIN = true, SIGNED = false, FOLD = false;
    static constexpr int WORDS = 6;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int, uint32_t* r) {
        ld_words<6, AL, SM>(b, r);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[0] & 0xFFFFu);
        ml[0] = ml[1] = -h2f(r[0] >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = (r[2 + i] & 0x0F0F0F0Fu) | (bits_to_bytes(r[1] >> (4 * i)) << 4);
            q[4 + i] = ((r[2 + i] >> 4) & 0x0F0F0F0Fu) | (bits_to_bytes(r[1] >> (16 + 4 * i)) << 4);
        }
    }
    // the block's minima, one per unit (per 16 values for Q2_K)
    template <int AL>
    __device__ static void minima(const uint8_t* b, float* m) { m[0] = -h2f(ld_u16<AL>(b + 2)); }
};

template <> struct Lv<QS_Q8_0> {
    static constexpr int QK = 32, BB = 34, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = false;
    static constexpr int WORDS = 9;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int, uint32_t* r) {
        ld_words<8, 1, SM>(b + 2, r);
        r[8] = ld_u16<AL, SM>(b);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[8]);
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = r[i];
    }
};

template <> struct Lv<QS_Q2_K> {
    static constexpr int QK = 256, BB = 84, MAXAL = 4;
    static constexpr bool G16 = true, HASMIN = true, SIGNED = false, FOLD = true;
    static constexpr int WORDS = 10;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<8, AL, SM>(b + 16 + 32 * (j / 4), r);
        ld_words<1, AL, SM>(b + 80, r + 8);
        r[9] = ld_u16<AL, SM>(b + 2 * j);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        const float dd = h2f(r[8] & 0xFFFFu), dm = h2f(r[8] >> 16);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t sc = r[9] >> (8 * h);
            dl[h] = dd * (float)(sc & 15u);
            ml[h] = dm * (float)((sc >> 4) & 15u);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = (r[i] >> (2 * (j & 3))) & 0x03030303u;
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[8] & 0xFFFFu); }
    __device__ static int sub(const uint32_t* r, int, int h) { return (int)((r[9] >> (8 * h)) & 15u); }
    template <int AL>
    __device__ static void minima(const uint8_t* b, float* m) {
        uint32_t s[4], d[1];
        ld_words<4, AL>(b, s);
        ld_words<1, AL>(b + 80, d);
        const float dm = h2f(d[0] >> 16);
#pragma unroll
        for (int i = 0; i < 16; i++) m[i] = dm * (float)((s[i / 4] >> (8 * (i & 3) + 4)) & 15u);
    }
};

template <> struct Lv<QS_Q3_K> {
    static constexpr int QK = 256, BB = 110, MAXAL = 2;
    static constexpr bool G16 = true, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 20;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<8, AL, SM>(b + 32 + 32 * (j / 4), r);
        ld_words<8, AL, SM>(b, r + 8);
        ld_words<3, 1, SM>(b + 96, r + 16);
        r[19] = ld_u16<AL, SM>(b + 108);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            dl[h] = base(r) * (float)sub(r, j, h);
            ml[h] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = sub_bytes(((r[i] >> (2 * (j & 3))) & 0x03030303u) | (((r[8 + i] >> j) & 0x01010101u) << 2), 0x04040404u);
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[19]); }
    __device__ static int sub(const uint32_t* r, int j, int h) {
        // scale g = 2 j + h: low 4 bits in nibble g / 8 of byte g % 8, high 2 bits of byte 8 + g % 4
        const int g = 2 * j + h;
        const uint32_t ls = ((g & 4 ? r[17] : r[16]) >> (8 * (g & 3) + 4 * (g >> 3))) & 15u;
        return (int)(ls | (((r[18] >> (8 * (g & 3) + 2 * (g >> 2))) & 3u) << 4)) - 32;
    }
};

// scale and minimum j of a Q4_K / Q5_K block, from its 12 scale bytes as words
__device__ __forceinline__ void k4_scale_min(const uint32_t* s, int j, float& sc, float& mn) {
    const int sh = 8 * (j & 3);
    const uint32_t a = s[0] >> sh, m = s[1] >> sh, c = s[2] >> sh;
    sc = (float)(j < 4 ? a & 63u : (c & 15u) | ((a >> 2) & 48u));
    mn = (float)(j < 4 ? m & 63u : ((c >> 4) & 15u) | ((m >> 2) & 48u));
}

template <> struct Lv<QS_Q4_K> {
    static constexpr int QK = 256, BB = 144, MAXAL = 16;
    static constexpr bool G16 = false, HASMIN = true, SIGNED = false, FOLD = true;
    static constexpr int WORDS = 12;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<4, AL, SM>(b, r + 8);
        ld_words<8, AL, SM>(b + 16 + 32 * (j / 2), r);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        float sc, mn;
        k4_scale_min(r + 9, j, sc, mn);
        dl[0] = dl[1] = h2f(r[8] & 0xFFFFu) * sc;
        ml[0] = ml[1] = h2f(r[8] >> 16) * mn;
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = (r[i] >> (4 * (j & 1))) & 0x0F0F0F0Fu;
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[8] & 0xFFFFu); }
    __device__ static int sub(const uint32_t* r, int j, int) {
        float sc, mn;
        k4_scale_min(r + 9, j, sc, mn);
        return (int)sc;
    }
    template <int AL>
    __device__ static void minima(const uint8_t* b, float* m) {
        uint32_t h[4];
        ld_words<4, AL>(b, h);
        const float dm = h2f(h[0] >> 16);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float sc, mn;
            k4_scale_min(h + 1, j, sc, mn);
            m[j] = dm * mn;
        }
    }
};

template <> struct Lv<QS_Q5_K> {
    static constexpr int QK = 256, BB = 176, MAXAL = 16;
    static constexpr bool G16 = false, HASMIN = true, SIGNED = false, FOLD = true;
    static constexpr int WORDS = 20;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<4, AL, SM>(b, r + 8);
        ld_words<8, AL, SM>(b + 16, r + 12);
        ld_words<8, AL, SM>(b + 48 + 32 * (j / 2), r);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        float sc, mn;
        k4_scale_min(r + 9, j, sc, mn);
        dl[0] = dl[1] = h2f(r[8] & 0xFFFFu) * sc;
        ml[0] = ml[1] = h2f(r[8] >> 16) * mn;
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = ((r[i] >> (4 * (j & 1))) & 0x0F0F0F0Fu) | (((r[12 + i] >> j) & 0x01010101u) << 4);
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[8] & 0xFFFFu); }
    __device__ static int sub(const uint32_t* r, int j, int) {
        float sc, mn;
        k4_scale_min(r + 9, j, sc, mn);
        return (int)sc;
    }
    template <int AL>
    __device__ static void minima(const uint8_t* b, float* m) {
        uint32_t h[4];
        ld_words<4, AL>(b, h);
        const float dm = h2f(h[0] >> 16);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float sc, mn;
            k4_scale_min(h + 1, j, sc, mn);
            m[j] = dm * mn;
        }
    }
};

template <> struct Lv<QS_Q6_K> {
    static constexpr int QK = 256, BB = 210, MAXAL = 2;
    static constexpr bool G16 = true, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 18;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<8, AL, SM>(b + 64 * (j / 4) + 32 * (j & 1), r);
        ld_words<8, AL, SM>(b + 128 + 32 * (j / 4), r + 8);
        r[16] = ld_u16<AL, SM>(b + 208);
        r[17] = ld_u16<AL, SM>(b + 192 + 2 * j);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        // unit j: half c = j / 4, low nibbles of ql at 32 (j & 1) for j & 3 < 2, high ones for the rest
        const float d = h2f(r[16]);
        dl[0] = d * (float)(int8_t)(r[17] & 0xFFu);
        dl[1] = d * (float)(int8_t)(r[17] >> 8);
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = sub_bytes(((r[i] >> (4 * ((j >> 1) & 1))) & 0x0F0F0F0Fu) | (((r[8 + i] >> (2 * (j & 3))) & 0x03030303u) << 4), 0x20202020u);
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[16]); }
    __device__ static int sub(const uint32_t* r, int, int h) { return (int)(int8_t)(r[17] >> (8 * h)); }
};

// four levels of an IQ2 code (2 bits each: 8, 25, 43) as bytes
__device__ __forceinline__ uint32_t iq2_bytes(uint32_t c) {
    // selector nibbles 0, 1, 2 pick from the byte table 08 19 2B (3 does not occur)
    const uint32_t sel = (c & 3u) | ((c & 0xCu) << 2) | ((c & 0x30u) << 4) | ((c & 0xC0u) << 6);
    return __byte_perm(0x2B2B1908u, 0u, sel);
}
// 8 signed levels of codebook entry `code` under the sign bits sg
__device__ __forceinline__ void iq2_signed(uint32_t code, uint32_t sg, uint32_t* q) {
    q[0] = neg_bytes(iq2_bytes(code & 0xFFu), bits_to_bytes(sg));
    q[1] = neg_bytes(iq2_bytes(code >> 8), bits_to_bytes(sg >> 4));
}
// 7 sign bits and their parity in bit 7
__device__ __forceinline__ uint32_t sign8(uint32_t i) { return i | ((__popc(i) & 1u) << 7); }

template <> struct Lv<QS_IQ2_XXS> {
    static constexpr int QK = 256, BB = 66, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 3;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<2, 1, SM>(b + 2 + 8 * j, r);
        r[2] = ld_u16<AL, SM>(b);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t* kgrid, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = (h2f(r[2]) * (0.5f + (float)(r[1] >> 28))) * 0.25f;
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; s++)
            iq2_signed(__ldg(kgrid + ((r[0] >> (8 * s)) & 0xFFu)), sign8((r[1] >> (7 * s)) & 127u), q + 2 * s);
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[2]) * 0.125f; }
    __device__ static int sub(const uint32_t* r, int, int) { return 1 + 2 * (int)(r[1] >> 28); }
};

template <> struct Lv<QS_IQ2_XS> {
    static constexpr int QK = 256, BB = 74, MAXAL = 2;
    static constexpr bool G16 = true, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 4;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<2, 1, SM>(b + 2 + 8 * j, r);
        r[2] = ld_u16<AL, SM>(b);
        r[3] = ld_v<SM>(b + 66 + j);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t* kgrid, uint32_t* q, float* dl, float* ml) {
        const float d = h2f(r[2]);
        dl[0] = (d * (0.5f + (float)(r[3] & 15u))) * 0.25f;
        dl[1] = (d * (0.5f + (float)(r[3] >> 4))) * 0.25f;
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const uint32_t c = (r[s / 2] >> (16 * (s & 1))) & 0xFFFFu;
            iq2_signed(__ldg(kgrid + (c & 511u)), sign8(c >> 9), q + 2 * s);
        }
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[2]) * 0.125f; }
    __device__ static int sub(const uint32_t* r, int, int h) { return 1 + 2 * (int)((r[3] >> (4 * h)) & 15u); }
};

template <> struct Lv<QS_IQ2_S> {
    static constexpr int QK = 256, BB = 82, MAXAL = 2;
    static constexpr bool G16 = true, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 5;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<1, 1, SM>(b + 2 + 4 * j, r);
        ld_words<1, 1, SM>(b + 34 + 4 * j, r + 1);
        r[2] = ld_u16<AL, SM>(b);
        r[3] = ld_v<SM>(b + 74 + j);
        r[4] = ld_v<SM>(b + 66 + j);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t* kgrid, uint32_t* q, float* dl, float* ml) {
        const float d = h2f(r[2]);
        dl[0] = (d * (0.5f + (float)(r[3] & 15u))) * 0.25f;
        dl[1] = (d * (0.5f + (float)(r[3] >> 4))) * 0.25f;
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; s++)
            iq2_signed(__ldg(kgrid + (((r[0] >> (8 * s)) & 0xFFu) | (((r[4] >> (2 * s)) & 3u) << 8))), (r[1] >> (8 * s)) & 0xFFu, q + 2 * s);
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[2]) * 0.125f; }
    __device__ static int sub(const uint32_t* r, int, int h) { return 1 + 2 * (int)((r[3] >> (4 * h)) & 15u); }
};

// four levels of an IQ3 code (3 bits each): byte table lo (levels 0..3), hi (levels 4..7)
__device__ __forceinline__ uint32_t iq3_bytes(uint32_t c, uint32_t lo, uint32_t hi) {
    return __byte_perm(lo, hi, (c & 7u) | ((c & 0x38u) << 1) | ((c & 0x1C0u) << 2) | ((c & 0xE00u) << 3));
}

template <> struct Lv<QS_IQ3_XXS> {
    static constexpr int QK = 256, BB = 98, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 4;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<2, 1, SM>(b + 2 + 8 * j, r);
        ld_words<1, 1, SM>(b + 66 + 4 * j, r + 2);
        r[3] = ld_u16<AL, SM>(b);
    }
    __device__ static void levels(const uint32_t* r, int, const uint16_t* kgrid, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = (h2f(r[3]) * (0.5f + (float)(r[2] >> 28))) * 0.5f;
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {  // levels 4, 12, ... 52, 62
            const uint32_t sg = sign8((r[2] >> (7 * (i / 2))) & 127u) >> (4 * (i & 1));
            q[i] = neg_bytes(iq3_bytes(__ldg(kgrid + ((r[i / 4] >> (8 * (i & 3))) & 0xFFu)), 0x1C140C04u, 0x3E342C24u), bits_to_bytes(sg));
        }
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[3]) * 0.25f; }
    __device__ static int sub(const uint32_t* r, int, int) { return 1 + 2 * (int)(r[2] >> 28); }
};

template <> struct Lv<QS_IQ3_S> {
    static constexpr int QK = 256, BB = 110, MAXAL = 2;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = true;
    static constexpr int WORDS = 6;
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<2, 1, SM>(b + 2 + 8 * j, r);
        ld_words<1, 1, SM>(b + 74 + 4 * j, r + 2);
        r[3] = ld_u16<AL, SM>(b);
        r[4] = ld_v<SM>(b + 66 + j);
        r[5] = ld_v<SM>(b + 106 + j / 2);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t* kgrid, uint32_t* q, float* dl, float* ml) {
        dl[0] = dl[1] = h2f(r[3]) * (float)(1u + 2u * ((r[5] >> (4 * (j & 1))) & 15u));
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)  // levels 1, 3, ... 15
            q[i] = neg_bytes(iq3_bytes(__ldg(kgrid + (((r[i / 4] >> (8 * (i & 3))) & 0xFFu) | (((r[4] >> i) & 1u) << 8))), 0x07050301u, 0x0F0D0B09u),
                             bits_to_bytes(r[2] >> (4 * i)));
    }
    __device__ static float base(const uint32_t* r) { return h2f(r[3]); }
    __device__ static int sub(const uint32_t* r, int j, int) { return 1 + 2 * (int)((r[5] >> (4 * (j & 1))) & 15u); }
};

template <> struct Lv<QS_IQ4_XS> {
    static constexpr int QK = 256, BB = 136, MAXAL = 8;
    static constexpr bool G16 = false, HASMIN = false, SIGNED = true, FOLD = false;
    static constexpr int WORDS = 6;
    // the 16 level values, 4 to a word: -127 -104 -83 -65 | -49 -35 -22 -10 | 1 13 25 38 | 53 69 89 113
    __device__ static uint32_t value4(uint32_t n) {  // 4 nibbles (one per byte) -> their bytes
        const uint32_t lo = (n & 0x07u) | ((n & 0x0700u) >> 4) | ((n & 0x070000u) >> 8) | ((n & 0x07000000u) >> 12);
        const uint32_t a = __byte_perm(0xBFAD9881u, 0xF6EADDCFu, lo), c = __byte_perm(0x26190D01u, 0x71594535u, lo);
        const uint32_t m = ((n >> 3) & 0x01010101u) * 0xFFu;
        return (a & ~m) | (c & m);
    }
    template <int AL, bool SM = false>
    __device__ static void load(const uint8_t* b, int j, uint32_t* r) {
        ld_words<2, AL, SM>(b, r + 4);
        ld_words<4, AL, SM>(b + 8 + 16 * j, r);
    }
    __device__ static void levels(const uint32_t* r, int j, const uint16_t*, uint32_t* q, float* dl, float* ml) {
        const uint32_t ls = (r[5] >> (4 * j)) & 15u, hs = (r[4] >> (16 + 2 * j)) & 3u;
        dl[0] = dl[1] = h2f(r[4] & 0xFFFFu) * (float)((int)(ls | (hs << 4)) - 32);
        ml[0] = ml[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            q[i] = value4(r[i] & 0x0F0F0F0Fu);
            q[4 + i] = value4((r[i] >> 4) & 0x0F0F0F0Fu);
        }
    }
};

}  // namespace qs
