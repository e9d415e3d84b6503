// act8_common.h -- the packed 8-bit form shared by act8.hip and act8_product.hip.
//
// A row of S values is cut into blocks of 128.  Block b has the exponent byte e + 127, e the smallest integer (not below -126) with
// max |value| <= Q 2^e, Q = 127 (int8) or 448 (e4m3: the largest number), and the codes value 2^-e rounded to nearest even.  A power of two
// costs an e4m3 code nothing (its relative step is the same at every scale) and an int8 code half a bit on average; in return scaling is exact
// -- codes are reproducible bit for bit by anyone, a code times its scale has no rounding -- and the scale is what the matrix instruction
// takes (one exponent byte per lane), so the product needs no arithmetic of its own for it.
// Byte 255 marks a block that held an Inf or a NaN: 255 << 23 read as a float is Inf, and int8 codes 0 or e4m3 codes NaN times Inf read NaN,
// so no reader tests for it.
// Rows of codes are padded with zero codes to whole blocks and rows of bytes with zeros to a multiple of 4: a product runs over whole blocks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "wmh_common.h"

#define ACT8_BLOCK 128

static inline __host__ __device__ size_t act8_blocks(size_t S) { return (S + ACT8_BLOCK - 1) / ACT8_BLOCK; }
static inline __host__ __device__ size_t act8_pitch(size_t S) { return act8_blocks(S) * ACT8_BLOCK; }
static inline __host__ __device__ size_t act8_scale_pitch(size_t S) { return (act8_blocks(S) + 3) & ~(size_t)3; }

// Exponent byte of a block from the largest |value| in it, taken as bits (unsigned order = order of the values, Inf and NaN above all).
// 127 = 1.984375 2^6 and 448 = 1.75 2^8: one step up where the fraction is larger than that of Q.
template <int FMT>
__device__ __forceinline__ unsigned act8_byte(unsigned amax_bits) {
    const int ex = (int)(amax_bits >> 23), fr = (int)(amax_bits & 0x7FFFFFu);
    const int b = FMT == WMH_ACT8_INT8 ? ex - 6 + (fr > 0x7E0000) : ex - 8 + (fr > 0x600000);
    return ex == 255 ? 255u : (unsigned)(b < 1 ? 1 : b);
}
__device__ __forceinline__ float act8_scale(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }                  // 2^e; 255: Inf
__device__ __forceinline__ float act8_inverse(unsigned byte) { return __builtin_bit_cast(float, (254u - (byte == 255u ? 0u : byte)) << 23); }

// Four values (times 2^-e already) to four codes, the first in the low byte.
template <int FMT>
__device__ __forceinline__ unsigned act8_encode4(float a, float b, float c, float d, bool bad) {
    if constexpr (FMT == WMH_ACT8_INT8) {
        // 1.5 2^23 + q: the addition rounds to nearest even at the units place and leaves q's two's complement in the low byte
        const float m = 12582912.f;
        const unsigned ua = __builtin_bit_cast(unsigned, a + m), ub = __builtin_bit_cast(unsigned, b + m);
        const unsigned uc = __builtin_bit_cast(unsigned, c + m), ud = __builtin_bit_cast(unsigned, d + m);
        const unsigned lo = __builtin_amdgcn_perm(ub, ua, 0x0C0C0400u), hi = __builtin_amdgcn_perm(ud, uc, 0x0C0C0400u);
        return bad ? 0u : lo | (hi << 16);
    } else {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
        return bad ? 0x7F7F7F7Fu : (unsigned)r;
    }
}
// Four codes to four values; exact.  (int8 as (u - 128) s of the biased byte u: one fma of u s and -128 s would overflow at the largest scale.)
template <int FMT>
__device__ __forceinline__ void act8_decode4(unsigned w, float s, float (&v)[4]) {
    if constexpr (FMT == WMH_ACT8_INT8) {
        const unsigned u = w ^ 0x80808080u;
        v[0] = ((float)(u & 0xFFu) - 128.f) * s; v[1] = ((float)((u >> 8) & 0xFFu) - 128.f) * s;
        v[2] = ((float)((u >> 16) & 0xFFu) - 128.f) * s; v[3] = ((float)(u >> 24) - 128.f) * s;
    } else {
        v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s; v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s;
        v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s; v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s;
    }
}

// The neighbouring code above (up) or below; the outermost stays.  e4m3 is sign and magnitude, with two zeros.
template <int FMT>
__device__ __forceinline__ unsigned act8_next(unsigned c, bool up) {
    if constexpr (FMT == WMH_ACT8_INT8) {
        const int v = (int)(int8_t)c, n = up ? v + 1 : v - 1;
        return (unsigned)(n > 127 ? 127 : n < -127 ? -127 : n) & 0xFFu;
    } else {
        const unsigned m = c & 0x7Fu, neg = c & 0x80u;
        if ((neg == 0) == up) return m < 0x7Eu ? c + 1 : c;           // away from zero
        return m ? c - 1 : (up ? 0x01u : 0x81u);
    }
}
// Largest of 32 lanes in all of them: four steps inside a row of 16, then rows against each other (gfx950's swap: even rows of one register
// against odd rows of another); no LDS crossbar.
__device__ __forceinline__ unsigned act8_lanes_max(unsigned m) {
#define ACT8_DPP_MAX(CTRL) { const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, CTRL, 0xF, 0xF, true); m = m > o ? m : o; }
    ACT8_DPP_MAX(0xB1)                // neighbours
    ACT8_DPP_MAX(0x4E)                // pairs of a quad
    ACT8_DPP_MAX(0x141)               // half row mirrored
    ACT8_DPP_MAX(0x140)               // row mirrored
#undef ACT8_DPP_MAX
    const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    return a[0] > a[1] ? a[0] : a[1];
}
// The same over the 32 even and the 32 odd lanes apart.
__device__ __forceinline__ unsigned act8_parity_max(unsigned m) {
#define ACT8_DPP_MAX(CTRL) { const unsigned o = (unsigned)__builtin_amdgcn_mov_dpp((int)m, CTRL, 0xF, 0xF, true); m = m > o ? m : o; }
    ACT8_DPP_MAX(0x4E)                // pairs of a quad
    ACT8_DPP_MAX(0x124)               // row turned by 4
    ACT8_DPP_MAX(0x128)               // row turned by 8
#undef ACT8_DPP_MAX
    const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = a[0] > a[1] ? a[0] : a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return b[0] > b[1] ? b[0] : b[1];
}
// z: voxels 2 l, 2 l + 1 of lane l at kw 0 and 1 -> four voxels 4 (l / 2) .. of kw 0 in even lanes and of kw 1 in odd ones.
__device__ __forceinline__ void act8_trade(const float (&z)[4], bool odd, float (&v)[4]) {
    const float s0 = odd ? z[0] : z[1], s1 = odd ? z[2] : z[3];
    const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, s0), 0xB1, 0xF, 0xF, true));
    const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, s1), 0xB1, 0xF, 0xF, true));
    v[0] = odd ? r0 : z[0]; v[1] = odd ? r1 : z[2];
    v[2] = odd ? z[1] : r0; v[3] = odd ? z[3] : r1;
}
__device__ __forceinline__ unsigned act8_abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7FFFFFFFu; }

// Element types of the tensors on the other side.  Four at a time where four are left: rows start at any element, and the memory path takes
// 16- and 8-byte accesses at the alignment of an element.
struct Act8F32 {
    typedef float T;
    typedef float T4 __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
struct Act8BF16 {
    typedef uint16_t T;
    typedef uint16_t T4 __attribute__((ext_vector_type(4), aligned(2)));
    static __device__ __forceinline__ float get(uint16_t x) { return __builtin_bit_cast(float, (unsigned)x << 16); }
    static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }                  // nearest even
};
struct Act8F16 {
    typedef uint16_t T;
    typedef uint16_t T4 __attribute__((ext_vector_type(4), aligned(2)));
    static __device__ __forceinline__ float get(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
// Values v .. v + 3 of a row of S; zero behind its end.
template <typename E>
__device__ __forceinline__ void act8_load4(const typename E::T* row, size_t v, size_t S, float (&z)[4]) {
    if (v + 4 <= S) {
        const typename E::T4 t = *reinterpret_cast<const typename E::T4*>(row + v);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = E::get(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = v + i < S ? E::get(row[v + i]) : 0.f;
    }
}
template <typename E>
__device__ __forceinline__ void act8_store4(typename E::T* row, size_t v, size_t S, const float (&z)[4]) {
    if (v + 4 <= S) {
        typename E::T4 t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = E::put(z[i]);
        *reinterpret_cast<typename E::T4*>(row + v) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (v + i < S) row[v + i] = E::put(z[i]);
    }
}
