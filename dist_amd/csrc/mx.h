// Microscaled 4-bit floating point (MXFP4): the element grid, the shared scale and the storage layout, used by mxfp4.hip, rmsnorm.hip and gemm_mx.hip.
//
// Elements are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), 32 along the quantised axis share one power of two 2^(byte - 127):
//   byte = max(floor(log2(max |x|)) + 127 - 2, 0);  code = e2m1(x / 2^(byte - 127)), nearest, ties to the even code, magnitudes above 6 -> 6.
// An infinity or a NaN in a block makes its byte 255 (the format's NaN): the block reads back, and multiplies, as NaN.
// Codes: row-major bytes, element 2i in the low half of byte i, rows padded with zeros to a whole block of 32.
// Scales: [chunk of 256 elements][row][8 bytes], byte 2 g + s of a chunk = block 4 s + g.  v_mfma_scale_f32_16x16x128_f8f6f4 takes the scale of lane group g (block
// g of its 128 elements) from a byte of that lane's register, the byte's number being part of the instruction: the two bytes of a lane group are its operands of
// two consecutive K steps, one 16-bit load each.  A chunk's scales of neighbouring rows are contiguous, so a tile of rows stages them as one run.
#pragma once
#include "common.h"

namespace mx {

constexpr int BLOCK = 32, CHUNK = 256;
typedef float f32x2_t __attribute__((ext_vector_type(2)));

DEV unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }       // ordered like |x|, with infinity and then NaN on top: maxima keep them
DEV int scale_byte(unsigned amax_bits) {
    const int e = (int)(amax_bits >> 23);
    return e == 255 ? 255 : max(e - 2, 0);
}
DEV float scale_value(int byte) { return __uint_as_float(byte == 0 ? 0x00400000u : (unsigned)byte << 23); }   // byte 255: NaN or infinity bits, never used as a divisor
// a launch takes fewer than 2^32 work items along an axis: these entry points refuse what needs more (DIST_ERR_ARG), before they launch anything
inline bool too_many(int64_t blocks, int threads) { return blocks > (int64_t)0xffffffffll / threads; }
// position of block b (of the whole row) inside the scales of `rows` rows
DEV long scale_at(long row, long rows, int b) { return ((long)(b >> 3) * rows + row) * 8 + 2 * (b & 3) + ((b >> 2) & 1); }

// eight values -> eight codes, first value in the low half of the first byte.  v_cvt_scalef32_pk_fp4_f32 divides by its scale operand and rounds to nearest even
// with saturation; checked against the definition for every bf16 value at twelve scales, the subnormal one among them.
DEV unsigned pack8(const float v[8], int byte) {
    if (byte == 255) return 0u;
    const float s = scale_value(byte);
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    return w;
}
DEV void unpack8(unsigned w, int byte, float v[8]) {
    const float s = scale_value(byte);
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
    const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
    if (byte == 255) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(0x7fc00000u);
    }
}

// Eight neighbouring elements of a row <-> fp32.  `n`: how many of them there are (the others read as zeros and are not written).  AL: rows of whole groups at 16-byte
// addresses; otherwise any address of whole elements - the vector instructions take those too, only slower, which still is far better than element by element (3001 rows
// of 1411 fp32 take the norm 9.7 us so, 12.6 by single elements).
typedef int i32x2_t __attribute__((ext_vector_type(2)));
template <typename T> struct __attribute__((packed)) Loose { T v[8]; };
template <bool AL, typename T> DEV void load8(const T* p, long n, float o[8]) {
    Frag<T> f;
    if (n >= 8) {
        if constexpr (AL) frag_load(f, p);
        else {
            const Loose<T> u = *reinterpret_cast<const Loose<T>*>(p);
            f = __builtin_bit_cast(Frag<T>, u);
        }
    } else {
        frag_zero(f);
        if constexpr (!AL) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) frag_set(f, e, to_f(p[e]));
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = frag_get(f, e);
}
// The same for loads that run ahead, from rows of eight elements at least: a partial group is read as the row's last eight elements, and settle() moves them into place
// when they are used.  (Zeros or single elements written into a load's registers under another mask wait for that load: 10630 rows of 1411 bf16 took the norm's gradient
// 64 us so, and take it 38.)
template <bool AL, typename T> struct Raw8 {
    Frag<T> f;
    DEV Raw8() { frag_zero(f); }
    DEV void load(const T* p, long n) {
        if (n <= 0) return;
        if constexpr (AL) frag_load(f, p);
        else {
            const Loose<T> u = *reinterpret_cast<const Loose<T>*>(n < 8 ? p + (n - 8) : p);
            f = __builtin_bit_cast(Frag<T>, u);
        }
    }
    DEV void settle(long n) {
        if constexpr (!AL) {
            constexpr int W = sizeof(T) == 2 ? 4 : 8, E = 8 / W;        // words, elements of a word
            struct Words { unsigned w[W]; };
            Words q = __builtin_bit_cast(Words, f);
#pragma unroll
            for (int i = 0; i < W; ++i) asm volatile("" : "+v"(q.w[i]));       // (not in front of the loads' arrival: hipcc moves it up to them)
            if (n < 8) {
                const int k = n > 0 ? 8 - (int)n : 8;                // down by k elements, zeros behind them
#pragma unroll
                for (int bit = 4; bit >= E; bit >>= 1)
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const unsigned up = i + bit / E < W ? q.w[i + bit / E] : 0u;
                        q.w[i] = k == 8 ? 0u : k & bit ? up : q.w[i];
                    }
                if constexpr (E == 2) {
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const unsigned up = i + 1 < W ? q.w[i + 1] : 0u;
                        q.w[i] = k & 1 ? q.w[i] >> 16 | up << 16 : q.w[i];
                    }
                }
            }
            f = __builtin_bit_cast(Frag<T>, q);
        }
    }
    DEV float get(int e) const { return frag_get(f, e); }
};
// stores: past the caches' keeping where rows are aligned (outputs that a later kernel reads from memory anyway)
template <bool AL, typename T> DEV void store8(T* p, long n, const float o[8]) {
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) frag_set(f, e, o[e]);
    if (n >= 8) {
        if constexpr (AL) frag_store_nt(f, p);
        else *reinterpret_cast<Loose<T>*>(p) = __builtin_bit_cast(Loose<T>, f);
    } else if constexpr (!AL) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = from_f<T>(o[e]);
    }
}

// eight floats / bf16 at a 16-byte address
DEV void load_v8(const float* p, float o[8]) {
    Frag<float> f;
    frag_load(f, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f.v[e];
}

}  // namespace mx
