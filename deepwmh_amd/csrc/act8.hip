// act8.hip -- 8-bit activation checkpoints: pack (by rows, by columns, by the taps of a transposed convolution), unpack, and the
// InstanceNorm + LeakyReLU backward pass that reads the codes.  The form itself: act8_common.h.
#include <type_traits>
#include "act8_common.h"

// Accesses that pass the caches by.  Pack reads and unpack writes this way where the tensor is too large for the 256 MB last-level cache to hand it
// from or to its neighbour (us, a pass that writes the tensor + pack, and unpack + a pass that reads it: 268 MB 152 + 203 through the caches, 132 +
// 194 past them; 134 MB 64 + 86 and 65 + 99).
template <bool FAR, typename T> __device__ __forceinline__ T act8_ld(const T* p) { if constexpr (FAR) return __builtin_nontemporal_load(p); else return *p; }
template <bool FAR, typename T> __device__ __forceinline__ void act8_st(const T& v, T* p) { if constexpr (FAR) __builtin_nontemporal_store(v, p); else *p = v; }
static inline bool act8_far(size_t bytes) { return bytes > (size_t)192 << 20; }

// ---- pack -------------------------------------------------------------------------------------------------------------------------------
// 32 lanes x 4 values = one block, so that loads and stores are contiguous over a wave and the maximum stays inside half a wave.  A half-wave takes
// U blocks (8 apart) with all their loads issued first: the pass is bound by the memory (2 x 32 x 128^3 float32: 104 us, 6.5 TB/s), and one load a
// lane in flight leaves half of it idle (203 us).
// NORM 1: the activation lrelu(x scale + shift) is packed.  NORM 2: x is, and a code whose value would fall on the other side of the LeakyReLU's kink
// than x, x scale + shift <= 0 instead of > 0 or the reverse, gives way to its neighbour on x's side (off by up to one step instead of half of one):
// a backward pass on rounded values then takes the same branch everywhere.  Without that a value's rounding of 1 % of a channel's spread would
// flip 0.3 % of the branches, which is 6 % of a gradient's norm in every layer.  (2 x 32 x 128^3 float32 to int8, replayed: plain 104 us, activated 110,
// sign kept 119.)
// FLAT: rows of fewer than 32 blocks; blocks are numbered through the rows.  Blocks that lie whole inside their rows (all but a workgroup's last,
// or all where S is a multiple of 128) take a path without a condition between the loads.
template <typename E, int FMT, int NORM, bool FLAT, bool FAR>
__global__ __launch_bounds__(256) void act8_pack_kernel(const typename E::T* __restrict__ x, size_t sn, size_t sc, const float* __restrict__ ss, float slope,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, unsigned C, unsigned rows, size_t S) {
    constexpr unsigned U = 4;
    const size_t nb = act8_blocks(S), sp = act8_scale_pitch(S), units = FLAT ? rows * nb : nb;
    const unsigned l = threadIdx.x & 31, hw = threadIdx.x >> 5;
    auto work = [&](unsigned row0, const typename E::T* x0, float a0, float b0, size_t first, auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::value;
        float z[U][4];
        unsigned row[U];
        size_t blk[U];
#pragma unroll
        for (unsigned u = 0; u < U; ++u) {
            const size_t unit = WHOLE || first + 8 * u < units ? first + 8 * u : first;
            row[u] = FLAT ? (unsigned)unit / (unsigned)nb : row0;
            blk[u] = FLAT ? (unsigned)unit - row[u] * (unsigned)nb : unit;
            const typename E::T* xr = FLAT ? x + (size_t)(row[u] / C) * sn + (size_t)(row[u] % C) * sc : x0;
            if constexpr (WHOLE) {
                const typename E::T4 t = act8_ld<FAR>(reinterpret_cast<const typename E::T4*>(xr + blk[u] * ACT8_BLOCK + 4 * l));
#pragma unroll
                for (int i = 0; i < 4; ++i) z[u][i] = E::get(t[i]);
            } else {
                act8_load4<E>(xr, blk[u] * ACT8_BLOCK + 4 * l, S, z[u]);
            }
        }
#pragma unroll
        for (unsigned u = 0; u < U; ++u) {
            if (!WHOLE && first + 8 * u >= units) break;
            const size_t v = blk[u] * ACT8_BLOCK + 4 * l;
            const float a = FLAT && NORM ? ss[2 * (size_t)row[u]] : a0, b = FLAT && NORM ? ss[2 * (size_t)row[u] + 1] : b0;
            if constexpr (NORM == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[u][i] = WHOLE || v + i < S ? wmh_lrelu(fmaf(z[u][i], a, b), slope) : 0.f;
            }
            const unsigned m0 = act8_abs_bits(z[u][0]), m1 = act8_abs_bits(z[u][1]), m2 = act8_abs_bits(z[u][2]), m3 = act8_abs_bits(z[u][3]);
            const unsigned m01 = m0 > m1 ? m0 : m1, m23 = m2 > m3 ? m2 : m3;
            const unsigned byte = act8_byte<FMT>(act8_lanes_max(m01 > m23 ? m01 : m23));
            const float inv = act8_inverse(byte);
            unsigned w = act8_encode4<FMT>(z[u][0] * inv, z[u][1] * inv, z[u][2] * inv, z[u][3] * inv, byte == 255u);
            if (!WHOLE && FMT == WMH_ACT8_E4M3 && byte == 255u)                                     // the padding stays zero
                w &= v + 4 <= S ? 0xFFFFFFFFu : v >= S ? 0u : 0xFFFFFFFFu >> (8 * (4 - (unsigned)(S - v)));
            if constexpr (NORM == 2) {
                float q[4];
                act8_decode4<FMT>(w, act8_scale(byte), q);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool pos = fmaf(z[u][i], a, b) > 0.f;
                    if ((fmaf(q[i], a, b) > 0.f) != pos && byte != 255u && (WHOLE || v + i < S))
                        w = (w & ~(0xFFu << (8 * i))) | (act8_next<FMT>((w >> (8 * i)) & 0xFFu, pos == (a > 0.f)) << (8 * i));
                }
            }
            reinterpret_cast<unsigned*>(codes + (row[u] * nb + blk[u]) * ACT8_BLOCK)[l] = w;
            if (l == 0 || (blk[u] == nb - 1 && l < sp - blk[u])) scales[row[u] * sp + blk[u] + l] = l == 0 ? (uint8_t)byte : 0;
        }
    };
    for (unsigned row = blockIdx.y; row < (FLAT ? 1u : rows); row += gridDim.y) {
        const typename E::T* xr = x + (size_t)(row / C) * sn + (size_t)(row % C) * sc;
        float a = 1.f, b = 0.f;
        if constexpr (NORM && !FLAT) { a = ss[2 * (size_t)row]; b = ss[2 * (size_t)row + 1]; }
        for (size_t f = (size_t)blockIdx.x * 8 * U; f < units; f += (size_t)gridDim.x * 8 * U) {
            if (FLAT ? S % ACT8_BLOCK == 0 && f + 8 * U <= units : (f + 8 * U) * ACT8_BLOCK <= S) work(row, xr, a, b, f + hw, std::true_type());
            else if (f + hw < units) work(row, xr, a, b, f + hw, std::false_type());
        }
    }
}

// A workgroup packs 64 columns of one block of 128 rows.  Wave w has the rows 32 w .. 32 w + 31: 16 lanes read 64 neighbouring columns of a row, four
// a lane, and each of the four groups of 16 has eight rows, so that a lane ends with eight neighbouring codes of each of its columns.  The columns'
// maxima meet in LDS, the codes are turned there, and every store writes a column's whole line of 128 bytes
// (4100 x 2048 bfloat16: 6.9 us replayed, 25 MB at 3.7 TB/s, and 10.2 a call, which is the host; one lane a column with 128 rows in its registers and
// scattered stores of 16 bytes took 38).  A workgroup has one phase of loads, two barriers and one of stores: latency is what is left.
template <typename E, int FMT>
__global__ __launch_bounds__(256) void act8_pack_columns_kernel(const typename E::T* __restrict__ x, size_t sb, size_t ld, uint8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ scales, size_t R, size_t S) {
    constexpr int LP = 136;                                     // bytes between columns in LDS
    __shared__ unsigned top[4][64];
    __shared__ __attribute__((aligned(16))) uint8_t turned[64 * LP];
    const size_t nb = act8_blocks(R), sp = act8_scale_pitch(R), r0 = (size_t)blockIdx.y * ACT8_BLOCK, s0 = (size_t)blockIdx.x * 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = 4 * (lane & 15), first = 32 * w + 8 * g;
    const typename E::T* xp = x + blockIdx.z * sb;
    float z[8][4];
    if (r0 + ACT8_BLOCK <= R && s0 + 64 <= S) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const typename E::T4 t = *reinterpret_cast<const typename E::T4*>(xp + (r0 + first + i) * ld + s0 + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[i][e] = E::get(t[e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[i][0] = z[i][1] = z[i][2] = z[i][3] = 0.f;
            if (r0 + first + i < R) act8_load4<E>(xp + (r0 + first + i) * ld, s0 + c, S, z[i]);
        }
    }
    unsigned m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m[e] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { const unsigned u = act8_abs_bits(z[i][e]); m[e] = m[e] > u ? m[e] : u; }
        const auto a = __builtin_amdgcn_permlane16_swap(m[e], m[e], false, false);
        m[e] = a[0] > a[1] ? a[0] : a[1];
        const auto b = __builtin_amdgcn_permlane32_swap(m[e], m[e], false, false);
        m[e] = b[0] > b[1] ? b[0] : b[1];
    }
    if (g == 0) *reinterpret_cast<uint4*>(&top[w][c]) = make_uint4(m[0], m[1], m[2], m[3]);
    __syncthreads();
    const size_t left = R - r0;                                 // rows of this block that exist (or more)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned m01 = top[0][c + e] > top[1][c + e] ? top[0][c + e] : top[1][c + e], m23 = top[2][c + e] > top[3][c + e] ? top[2][c + e] : top[3][c + e];
        const unsigned byte = act8_byte<FMT>(m01 > m23 ? m01 : m23);
        const float inv = act8_inverse(byte);
        unsigned q[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            q[k] = act8_encode4<FMT>(z[4 * k][e] * inv, z[4 * k + 1][e] * inv, z[4 * k + 2][e] * inv, z[4 * k + 3][e] * inv, byte == 255u);
            if (FMT == WMH_ACT8_E4M3 && byte == 255u) {         // the padding stays zero
                const size_t v = first + 4 * k;
                q[k] &= v + 4 <= left ? 0xFFFFFFFFu : v >= left ? 0u : 0xFFFFFFFFu >> (8 * (4 - (unsigned)(left - v)));
            }
        }
        *reinterpret_cast<uint2*>(turned + (c + e) * LP + first) = make_uint2(q[0], q[1]);
        if (w == 0 && g == 0 && s0 + c + e < S) {
            uint8_t* sr = scales + (blockIdx.z * S + s0 + c + e) * sp;
            sr[blockIdx.y] = (uint8_t)byte;
            if (blockIdx.y == nb - 1)
                for (size_t k = nb; k < sp; ++k) sr[k] = 0;
        }
    }
    __syncthreads();
    const int col = threadIdx.x >> 2, part = (threadIdx.x & 3) * 32;
    if (s0 + col < S) {
        uint8_t* out = codes + ((blockIdx.z * S + s0 + col) * nb + blockIdx.y) * ACT8_BLOCK + part;
        const uint2* t = reinterpret_cast<const uint2*>(turned + col * LP + part);
        const uint2 t0 = t[0], t1 = t[1], t2 = t[2], t3 = t[3];
        *reinterpret_cast<uint4*>(out) = make_uint4(t0.x, t0.y, t1.x, t1.y);
        *reinterpret_cast<uint4*>(out + 16) = make_uint4(t2.x, t2.y, t3.x, t3.y);
    }
}

#define ACT8_BY_TYPE(DT, FMT, CALL)                                                                                                            \
    switch ((DT) * 2 + (FMT)) {                                                                                                                \
        case 0: { typedef Act8F32 E; constexpr int F = 0; CALL; } break;                                                                       \
        case 1: { typedef Act8F32 E; constexpr int F = 1; CALL; } break;                                                                       \
        case 2: { typedef Act8BF16 E; constexpr int F = 0; CALL; } break;                                                                      \
        case 3: { typedef Act8BF16 E; constexpr int F = 1; CALL; } break;                                                                      \
        case 4: { typedef Act8F16 E; constexpr int F = 0; CALL; } break;                                                                       \
        default: { typedef Act8F16 E; constexpr int F = 1; CALL; } break;                                                                      \
    }
static bool bad_form(int dtype, int fmt) { return dtype < 0 || dtype > 2 || fmt < 0 || fmt > 1; }
static bool bad_codes(const void* codes, const void* scales) { return !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)scales % 4; }

extern "C" size_t wmh_act8_pitch(size_t S) { return act8_pitch(S); }
extern "C" size_t wmh_act8_scale_pitch(size_t S) { return act8_scale_pitch(S); }

extern "C" int wmh_act8_pack(const void* x, int dtype, size_t sn, size_t sc, const float* ss, int mode, float slope, int fmt, uint8_t* codes,
                             uint8_t* scales, int N, int C, size_t S, void* stream) {
    if (mode < 0 || mode > 2 || (mode != 0 && N > 0 && C > 0 && S > 0 && !ss)) return wmh_fail(WMH_EINVAL, "act8_pack: bad mode, or no scale and shift for it");
    if (bad_form(dtype, fmt) || N < 0 || C < 0) return wmh_fail(WMH_EINVAL, "act8_pack: bad type, format or size");
    if (N == 0 || C == 0 || S == 0) return WMH_OK;
    if (!x || bad_codes(codes, scales) || (uintptr_t)x % (dtype == WMH_F32 ? 4 : 2)) return wmh_fail(WMH_EINVAL, "act8_pack: null or misaligned pointer");
    const size_t rows = (size_t)N * C, nb = act8_blocks(S);
    if (rows > 0xFFFFFFFFu) return wmh_fail(WMH_EINVAL, "act8_pack: more than 2^32 rows");
    const bool flat = nb < 32 && rows * nb <= 0xFFFFFF00u;
    const size_t gx = ((flat ? rows * nb : nb) + 31) / 32;
    const dim3 grid(gx > 0x3FFFFF ? 0x3FFFFFu : (unsigned)gx, flat ? 1 : rows > 65535 ? 65535u : (unsigned)rows);
    hipStream_t st = (hipStream_t)stream;
    const bool far = !flat && act8_far(rows * S * (dtype == WMH_F32 ? 4 : 2));
#define ACT8_PACK(NORM, FLAT, FAR) \
    ACT8_BY_TYPE(dtype, fmt, hipLaunchKernelGGL((act8_pack_kernel<E, F, NORM, FLAT, FAR>), grid, dim3(256), 0, st, (const E::T*)x, sn, sc, ss, slope, codes, scales, (unsigned)C, (unsigned)rows, S))
#define ACT8_PACK_AT(NORM)                                                                                                                     \
    if (flat) { ACT8_PACK(NORM, true, false); } else if (far) { ACT8_PACK(NORM, false, true); } else { ACT8_PACK(NORM, false, false); }
    if (mode == 0) { ACT8_PACK_AT(0) } else if (mode == 1) { ACT8_PACK_AT(1) } else { ACT8_PACK_AT(2) }
#undef ACT8_PACK_AT
#undef ACT8_PACK
    return wmh_check_launch("act8_pack_kernel");
}
extern "C" int wmh_act8_pack_columns(const void* x, int dtype, size_t sb, size_t ld, int fmt, uint8_t* codes, uint8_t* scales, int B, size_t R, size_t S,
                                     void* stream) {
    if (bad_form(dtype, fmt) || B < 0 || B > 65535) return wmh_fail(WMH_EINVAL, "act8_pack_columns: bad type, format or size");
    if (B == 0 || R == 0 || S == 0) return WMH_OK;
    if (!x || bad_codes(codes, scales) || (uintptr_t)x % (dtype == WMH_F32 ? 4 : 2)) return wmh_fail(WMH_EINVAL, "act8_pack_columns: null or misaligned pointer");
    if (act8_blocks(R) > 65535 || (S + 63) / 64 > 0xFFFFFF) return wmh_fail(WMH_EINVAL, "act8_pack_columns: more than 8388480 rows or 2^30 columns");
    const dim3 grid((unsigned)((S + 63) / 64), (unsigned)act8_blocks(R), (unsigned)B);
    ACT8_BY_TYPE(dtype, fmt, hipLaunchKernelGGL((act8_pack_columns_kernel<E, F>), grid, dim3(256), 0, (hipStream_t)stream, (const E::T*)x, sb, ld, codes, scales, R, S));
    return wmh_check_launch("act8_pack_columns_kernel");
}

// ---- unpack -----------------------------------------------------------------------------------------------------------------------------
// A lane reads four codes and writes four values: the writes, four fifths of the traffic, are contiguous over a wave.  U quads a lane in flight;
// FLAT and whole quads as in pack.  2 x 32 x 128^3 to float32: 96 us, 7.0 TB/s.
template <typename E, int FMT, bool NORM, bool FLAT, bool FAR>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ ss,
                                                          float slope, typename E::T* __restrict__ y, unsigned rows, size_t S) {
    constexpr unsigned U = 4;
    const size_t nb = act8_blocks(S), sp = act8_scale_pitch(S), nq = (S + 3) / 4, units = FLAT ? rows * nq : nq;
    auto work = [&](unsigned row0, float a0, float b0, size_t first, auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::value;
        unsigned w[U], byte[U], row[U];
        size_t q[U];
#pragma unroll
        for (unsigned u = 0; u < U; ++u) {
            const size_t unit = WHOLE || first + 256 * u < units ? first + 256 * u : first;
            row[u] = FLAT ? (unsigned)unit / (unsigned)nq : row0;
            q[u] = FLAT ? (unsigned)unit - row[u] * (unsigned)nq : unit;
            w[u] = reinterpret_cast<const unsigned*>(codes + row[u] * nb * ACT8_BLOCK)[q[u]];
            byte[u] = scales[row[u] * sp + q[u] / 32];
        }
#pragma unroll
        for (unsigned u = 0; u < U; ++u) {
            if (!WHOLE && first + 256 * u >= units) break;
            float v[4];
            act8_decode4<FMT>(w[u], act8_scale(byte[u]), v);
            if constexpr (NORM) {
                const float a = FLAT ? ss[2 * (size_t)row[u]] : a0, b = FLAT ? ss[2 * (size_t)row[u] + 1] : b0;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = wmh_lrelu(fmaf(v[i], a, b), slope);
            }
            if constexpr (WHOLE) {
                typename E::T4 t;
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = E::put(v[i]);
                act8_st<FAR>(t, reinterpret_cast<typename E::T4*>(y + row[u] * S + 4 * q[u]));
            } else {
                act8_store4<E>(y + row[u] * S, 4 * q[u], S, v);
            }
        }
    };
    for (unsigned row = blockIdx.y; row < (FLAT ? 1u : rows); row += gridDim.y) {
        float a = 1.f, b = 0.f;
        if constexpr (NORM && !FLAT) { a = ss[2 * (size_t)row]; b = ss[2 * (size_t)row + 1]; }
        for (size_t f = (size_t)blockIdx.x * 256 * U; f < units; f += (size_t)gridDim.x * 256 * U) {
            if (FLAT ? S % 4 == 0 && f + 256 * U <= units : 4 * (f + 256 * U) <= S) work(row, a, b, f + threadIdx.x, std::true_type());
            else if (f + threadIdx.x < units) work(row, a, b, f + threadIdx.x, std::false_type());
        }
    }
}
extern "C" int wmh_act8_unpack(const uint8_t* codes, const uint8_t* scales, int fmt, const float* ss, float slope, void* y, int dtype, int N, int C, size_t S,
                               void* stream) {
    if (bad_form(dtype, fmt) || N < 0 || C < 0) return wmh_fail(WMH_EINVAL, "act8_unpack: bad type, format or size");
    if (N == 0 || C == 0 || S == 0) return WMH_OK;
    if (!y || bad_codes(codes, scales) || (uintptr_t)y % (dtype == WMH_F32 ? 4 : 2)) return wmh_fail(WMH_EINVAL, "act8_unpack: null or misaligned pointer");
    const size_t rows = (size_t)N * C, nq = (S + 3) / 4;
    if (rows > 0xFFFFFFFFu) return wmh_fail(WMH_EINVAL, "act8_unpack: more than 2^32 rows");
    const bool flat = nq < 1024 && rows * nq <= 0xFFFF0000u;
    const size_t gx = ((flat ? rows * nq : nq) + 1023) / 1024;
    const dim3 grid(gx > 0x3FFFFF ? 0x3FFFFFu : (unsigned)gx, flat ? 1 : rows > 65535 ? 65535u : (unsigned)rows);
    hipStream_t st = (hipStream_t)stream;
    const bool far = !flat && act8_far(rows * S * (dtype == WMH_F32 ? 4 : 2));
#define ACT8_UNPACK(NORM, FLAT, FAR) \
    ACT8_BY_TYPE(dtype, fmt, hipLaunchKernelGGL((act8_unpack_kernel<E, F, NORM, FLAT, FAR>), grid, dim3(256), 0, st, codes, scales, ss, slope, (E::T*)y, (unsigned)rows, S))
    if (ss && flat) { ACT8_UNPACK(true, true, false); } else if (ss && far) { ACT8_UNPACK(true, false, true); } else if (ss) { ACT8_UNPACK(true, false, false); }
    else if (flat) { ACT8_UNPACK(false, true, false); } else if (far) { ACT8_UNPACK(false, false, true); } else { ACT8_UNPACK(false, false, false); }
#undef ACT8_UNPACK
    return wmh_check_launch("act8_unpack_kernel");
}

// ---- InstanceNorm + LeakyReLU backward ----------------------------------------------------------------------------------------------------
// z = y scale + shift, a = lrelu(z), dA = g1 + g2 + sum_k wseg[k][c] dl[k], dz = dA lrelu'(z), xh = (y - mean) rstd with y from the codes:
//   reduce  per (n, c): sum dz, sum dz xh, sum a dl[k]
//   apply   dy = gamma rstd (dz - sum dz / S - xh sum(dz xh) / S), and sum dy
// Both passes are bound by the memory: a lane takes four voxels a step (one dword of codes, 16 bytes of every other source) and U steps with their
// loads issued together; the sources are template parameters so that no branch stands between the loads.  Four terms are added in 32 bits, the
// rest in 64, in a fixed order.  KT: classes of the head a kernel is built for (a padded class with weight 0 would make NaN of an infinite gradient).
#define ACT8_MAXK 4
struct Act8Bwd {
    const uint8_t* codes; const uint8_t* scales; const float* ss; const float* mr; const float* gamma;
    const float* g1; const float* g2; const float* dl; const float* wseg;
    float* dy; float* dgamma; float* dbeta; float* dwseg; float* dbias;
    double* psums; double* dysum;
    int N, C, K, split;
    size_t S; float slope;
};
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ double act8_block_sum(double v, double* sh) {
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0] + sh[1] + sh[2] + sh[3];
    __syncthreads();
    return v;
}
// The sources of one row, and a quad of them.
template <int FMT, int SRC, int KT>
struct Act8Row {
    const uint8_t* codes; const uint8_t* scales; const float* g1; const float* g2; const float* dl[KT ? KT : 1];
    float w[KT ? KT : 1], sc, sh, mean, rstd, slope;
    __device__ __forceinline__ Act8Row(const Act8Bwd& a, size_t nc) {
        const size_t n = nc / a.C, c = nc % a.C;
        codes = a.codes + nc * act8_pitch(a.S); scales = a.scales + nc * act8_scale_pitch(a.S);
        g1 = (SRC & 1) ? a.g1 + nc * a.S : nullptr; g2 = (SRC & 2) ? a.g2 + nc * a.S : nullptr;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            dl[k] = a.dl + (n * KT + k) * a.S;
            w[k] = a.wseg[k * a.C + c];
        }
        sc = a.ss[2 * nc]; sh = a.ss[2 * nc + 1]; mean = a.mr[2 * nc]; rstd = a.mr[2 * nc + 1]; slope = a.slope;
    }
};
template <int SRC, int KT>
struct Act8Quad { unsigned code, byte; f32x4u g1, g2, l[KT ? KT : 1]; };
template <bool FAR, int FMT, int SRC, int KT>
__device__ __forceinline__ void act8_quad_load(Act8Quad<SRC, KT>& t, const Act8Row<FMT, SRC, KT>& r, size_t q) {
    t.code = act8_ld<FAR>(reinterpret_cast<const unsigned*>(r.codes) + q);
    t.byte = r.scales[q >> 5];
    if constexpr ((SRC & 1) != 0) t.g1 = act8_ld<FAR>(reinterpret_cast<const f32x4u*>(r.g1 + 4 * q));
    if constexpr ((SRC & 2) != 0) t.g2 = act8_ld<FAR>(reinterpret_cast<const f32x4u*>(r.g2 + 4 * q));
#pragma unroll
    for (int k = 0; k < KT; ++k) t.l[k] = *reinterpret_cast<const f32x4u*>(r.dl[k] + 4 * q);
}
// The quad that passes the row's end: what lies behind it counts as a gradient of zero.
template <int FMT, int SRC, int KT>
__device__ __forceinline__ void act8_quad_load_tail(Act8Quad<SRC, KT>& t, const Act8Row<FMT, SRC, KT>& r, size_t q, size_t S) {
    t.code = reinterpret_cast<const unsigned*>(r.codes)[q];
    t.byte = r.scales[q >> 5];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = 4 * q + i < S;
        const size_t v = in ? 4 * q + i : S - 1;
        if constexpr ((SRC & 1) != 0) t.g1[i] = in ? r.g1[v] : 0.f;
        if constexpr ((SRC & 2) != 0) t.g2[i] = in ? r.g2[v] : 0.f;
#pragma unroll
        for (int k = 0; k < KT; ++k) t.l[k][i] = in ? r.dl[k][v] : 0.f;
    }
}
template <int FMT, int SRC, int KT>
__device__ __forceinline__ void act8_quad_values(const Act8Quad<SRC, KT>& t, const Act8Row<FMT, SRC, KT>& r, float (&dz)[4], float (&xh)[4], float (&z)[4]) {
    float y[4];
    act8_decode4<FMT>(t.code, act8_scale(t.byte), y);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float d = 0.f;
        if constexpr ((SRC & 1) != 0) d += t.g1[i];
        if constexpr ((SRC & 2) != 0) d += t.g2[i];
#pragma unroll
        for (int k = 0; k < KT; ++k) d = fmaf(r.w[k], t.l[k][i], d);
        z[i] = fmaf(y[i], r.sc, r.sh);
        dz[i] = z[i] > 0.f ? d : d * r.slope;
        xh[i] = (y[i] - r.mean) * r.rstd;
    }
}
template <int FMT, int SRC, int KT>
__global__ __launch_bounds__(256) void act8_bwd_reduce_kernel(const Act8Bwd a) {
    __shared__ double sh[4];
    constexpr int U = KT ? 2 : 4;
    const size_t nc = blockIdx.y, nq = a.S / 4;
    const Act8Row<FMT, SRC, KT> r(a, nc);
    double s0 = 0.0, s1 = 0.0, sk[KT ? KT : 1] = {};
    auto use = [&](const Act8Quad<SRC, KT>& t) __attribute__((always_inline)) {
        float dz[4], xh[4], z[4];
        act8_quad_values(t, r, dz, xh, z);
        s0 += (double)((dz[0] + dz[1]) + (dz[2] + dz[3]));
        s1 += (double)fmaf(dz[3], xh[3], fmaf(dz[2], xh[2], fmaf(dz[1], xh[1], dz[0] * xh[0])));
        if constexpr (KT > 0) {
            float act[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) act[i] = z[i] > 0.f ? z[i] : z[i] * r.slope;
#pragma unroll
            for (int k = 0; k < KT; ++k) sk[k] += (double)fmaf(act[3], t.l[k][3], fmaf(act[2], t.l[k][2], fmaf(act[1], t.l[k][1], act[0] * t.l[k][0])));
        }
    };
    const size_t step = (size_t)gridDim.x * 256;
    size_t q = (size_t)blockIdx.x * 256 + threadIdx.x;
    auto sweep = [&](auto far) __attribute__((always_inline)) {
        for (; q + (U - 1) * step < nq; q += U * step) {
            Act8Quad<SRC, KT> t[U];
#pragma unroll
            for (int u = 0; u < U; ++u) act8_quad_load<decltype(far)::value>(t[u], r, q + u * step);
#pragma unroll
            for (int u = 0; u < U; ++u) use(t[u]);
        }
        for (; q < nq; q += step) {
            Act8Quad<SRC, KT> t;
            act8_quad_load<decltype(far)::value>(t, r, q);
            use(t);
        }
    };
    // rows whose sources the second pass could not find in the 256 MB last-level cache are read past it: those behind them stay
    if ((gridDim.y - nc) * a.S * ((SRC & 1) * 4 + (SRC & 2) * 2 + 1) > (size_t)256 << 20) sweep(std::true_type());
    else sweep(std::false_type());
    if (q == nq && 4 * nq < a.S) {
        Act8Quad<SRC, KT> t;
        act8_quad_load_tail(t, r, q, a.S);
        use(t);
    }
    double* out = a.psums + (nc * a.split + blockIdx.x) * (2 + ACT8_MAXK);
    double t = act8_block_sum(s0, sh); if (threadIdx.x == 0) out[0] = t;
    t = act8_block_sum(s1, sh); if (threadIdx.x == 0) out[1] = t;
#pragma unroll
    for (int k = 0; k < KT; ++k) { t = act8_block_sum(sk[k], sh); if (threadIdx.x == 0) out[2 + k] = t; }
}
template <int FMT, int SRC, int KT>
__global__ __launch_bounds__(256) void act8_bwd_apply_kernel(const Act8Bwd a) {
    __shared__ double sh[4];
    constexpr int U = KT ? 2 : 4;
    const size_t nc = gridDim.y - 1 - blockIdx.y, nq = a.S / 4;
    const Act8Row<FMT, SRC, KT> r(a, nc);
    double p0 = 0.0, p1 = 0.0;
    for (int p = threadIdx.x; p < a.split; p += 256) { p0 += a.psums[(nc * a.split + p) * (2 + ACT8_MAXK)]; p1 += a.psums[(nc * a.split + p) * (2 + ACT8_MAXK) + 1]; }
    const float m1 = (float)(act8_block_sum(p0, sh) / (double)a.S), m2 = (float)(act8_block_sum(p1, sh) / (double)a.S);
    const float gr = (a.gamma ? a.gamma[nc % a.C] : 1.f) * r.rstd;
    float* out = a.dy + nc * a.S;
    double acc = 0.0;
    auto use = [&](const Act8Quad<SRC, KT>& t, float (&o)[4]) __attribute__((always_inline)) {
        float dz[4], xh[4], z[4];
        act8_quad_values(t, r, dz, xh, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = gr * (dz[i] - m1 - xh[i] * m2);
    };
    const size_t step = (size_t)gridDim.x * 256;
    size_t q = (size_t)blockIdx.x * 256 + threadIdx.x;
    for (; q + (U - 1) * step < nq; q += U * step) {
        Act8Quad<SRC, KT> t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) act8_quad_load<true>(t[u], r, q + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float o[4];
            use(t[u], o);
            acc += (double)((o[0] + o[1]) + (o[2] + o[3]));
            act8_st<true>(f32x4u{o[0], o[1], o[2], o[3]}, reinterpret_cast<f32x4u*>(out + 4 * (q + u * step)));
        }
    }
    for (; q < nq; q += step) {
        Act8Quad<SRC, KT> t;
        float o[4];
        act8_quad_load<true>(t, r, q);
        use(t, o);
        acc += (double)((o[0] + o[1]) + (o[2] + o[3]));
        *reinterpret_cast<f32x4u*>(out + 4 * q) = f32x4u{o[0], o[1], o[2], o[3]};
    }
    if (q == nq && 4 * nq < a.S) {
        Act8Quad<SRC, KT> t;
        float o[4];
        act8_quad_load_tail(t, r, q, a.S);
        use(t, o);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * q + i < a.S) { out[4 * q + i] = o[i]; acc += (double)o[i]; }
    }
    const double t = act8_block_sum(acc, sh);
    if (threadIdx.x == 0) a.dysum[nc * a.split + blockIdx.x] = t;
}
// Rows that fit a workgroup's registers: a workgroup takes a channel, keeps a row's dz and xh between the sums and their use -- its sources are read
// once -- and adds the channel's parameter gradients over the samples itself: one launch.
template <int FMT, int SRC, int KT, int Q>
__global__ __launch_bounds__(512) void act8_bwd_row_kernel(const Act8Bwd a) {
    __shared__ double sh[8];
    auto block_sum = [&](double v) {
        for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        v = ((sh[0] + sh[1]) + (sh[2] + sh[3])) + ((sh[4] + sh[5]) + (sh[6] + sh[7]));
        __syncthreads();
        return v;
    };
    const int c = blockIdx.x;
    const size_t nq = a.S / 4;
    double t0 = 0.0, t1 = 0.0, acc = 0.0, sk[KT ? KT : 1] = {};
    for (int n = 0; n < a.N; ++n) {
        const size_t nc = (size_t)n * a.C + c;
        const Act8Row<FMT, SRC, KT> r(a, nc);
        Act8Quad<SRC, KT> t[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const size_t q = threadIdx.x + 512 * k;
            if (q < nq) act8_quad_load<false>(t[k], r, q);
            else if (4 * q < a.S) act8_quad_load_tail(t[k], r, q, a.S);
        }
        float dz[Q][4], xh[Q][4];
        double s0 = 0.0, s1 = 0.0;
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            if (4 * (threadIdx.x + 512 * (size_t)k) >= a.S) continue;
            float z[4];
            act8_quad_values(t[k], r, dz[k], xh[k], z);
            s0 += (double)((dz[k][0] + dz[k][1]) + (dz[k][2] + dz[k][3]));
            s1 += (double)fmaf(dz[k][3], xh[k][3], fmaf(dz[k][2], xh[k][2], fmaf(dz[k][1], xh[k][1], dz[k][0] * xh[k][0])));
            if constexpr (KT > 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] * r.slope;
#pragma unroll
                for (int j = 0; j < KT; ++j) sk[j] += (double)fmaf(z[3], t[k].l[j][3], fmaf(z[2], t[k].l[j][2], fmaf(z[1], t[k].l[j][1], z[0] * t[k].l[j][0])));
            }
        }
        s0 = block_sum(s0); s1 = block_sum(s1);
        t0 += s0; t1 += s1;
        const float m1 = (float)(s0 / (double)a.S), m2 = (float)(s1 / (double)a.S), gr = (a.gamma ? a.gamma[c] : 1.f) * r.rstd;
        float* out = a.dy + nc * a.S;
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const size_t q = threadIdx.x + 512 * k;
            if (4 * q >= a.S) continue;
            float o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[i] = gr * (dz[k][i] - m1 - xh[k][i] * m2);
                if (q < nq || 4 * q + i < a.S) acc += (double)o[i];
            }
            act8_store4<Act8F32>(out, 4 * q, a.S, o);
        }
    }
    acc = block_sum(acc);
#pragma unroll
    for (int j = 0; j < KT; ++j) sk[j] = block_sum(sk[j]);
    if (threadIdx.x) return;
    if (a.dbeta) a.dbeta[c] = (float)t0;
    if (a.dgamma) a.dgamma[c] = (float)t1;
    if (a.dbias) a.dbias[c] = (float)acc;
    if (a.dwseg)
#pragma unroll
        for (int j = 0; j < KT; ++j) a.dwseg[j * a.C + c] = (float)sk[j];
}
// Parameter gradients: one wave per channel over the n rows and their slices.
__global__ __launch_bounds__(64) void act8_bwd_param_kernel(const Act8Bwd a) {
    const int c = blockIdx.x;
    double s[3 + ACT8_MAXK] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < a.N * a.split; i += 64) {
        const size_t at = ((size_t)(i / a.split) * a.C + c) * a.split + i % a.split;
#pragma unroll
        for (int k = 0; k < 2 + ACT8_MAXK; ++k)
            if (k < 2 + a.K) s[k] += a.psums[at * (2 + ACT8_MAXK) + k];
        s[2 + ACT8_MAXK] += a.dysum[at];
    }
#pragma unroll
    for (int k = 0; k < 3 + ACT8_MAXK; ++k)
        for (int m = 1; m < 64; m <<= 1) s[k] += __shfl_xor(s[k], m);
    if (threadIdx.x) return;
    if (a.dbeta) a.dbeta[c] = (float)s[0];
    if (a.dgamma) a.dgamma[c] = (float)s[1];
    if (a.dbias) a.dbias[c] = (float)s[2 + ACT8_MAXK];
    if (a.dwseg)
        for (int k = 0; k < a.K; ++k) a.dwseg[k * a.C + c] = (float)s[2 + k];
}
// (us of replayed graphs, two passes / rows: 2 x 320 x 64 10.1 / 6.6, 2 x 256 x 4096 12.2 / 8.1, 2 x 128 x 8192 12.3 / 9.2, 2 x 1 x 8192 9.0 / 7.9, 1 x 61 x
// 2431 10.6 / 4.8; a workgroup takes its samples in turn: 8 x 64 x 8192 17.9 / 27.3, 8 x 4 x 8192 9.5 / 23.5.)
static bool bwd_in_rows(int N, size_t S) { return S <= 8192 && N <= 2; }
static int bwd_split(int N, int C, size_t S) {
    const size_t rows = (size_t)N * C;
    size_t s = (4096 + rows - 1) / rows, most = (S + 4095) / 4096;
    return (int)(s > most ? most : s);
}
extern "C" size_t wmh_act8_in_lrelu_bwd_scratch_doubles(int N, int C, size_t S) {
    if (N < 1 || C < 1 || S < 1 || bwd_in_rows(N, S)) return 0;
    return (size_t)N * C * bwd_split(N, C, S) * (3 + ACT8_MAXK);
}
// The second pass takes the rows from the last to the first -- what the first pass read last is still in the last-level cache -- and goes past the
// caches itself, so that its own traffic does not push the rest out: 2 x 32 x 128^3 370 -> 320 us (1.88 GB, 5.9 TB/s), and faster at every size down
// to 17 MB with the passes around it (40 -> 37).  The first pass reads past the caches what the second will not find there: with the passes around
// it 680 -> 660.  (Rows a few at a time, so that the second pass would find all of the first one's sources there: 395 us
// with 32 rows at once, 412 with 8 and 479 with 4, against 370 before.)
template <int FMT, int SRC, int KT>
static void launch_bwd(const Act8Bwd& a, unsigned rows, hipStream_t st) {
    if (bwd_in_rows(a.N, a.S)) {
        if (a.S <= 2048) hipLaunchKernelGGL((act8_bwd_row_kernel<FMT, SRC, KT, 1>), dim3(a.C), dim3(512), 0, st, a);
        else hipLaunchKernelGGL((act8_bwd_row_kernel<FMT, SRC, KT, 4>), dim3(a.C), dim3(512), 0, st, a);
        return;
    }
    const dim3 grid((unsigned)a.split, rows);
    hipLaunchKernelGGL((act8_bwd_reduce_kernel<FMT, SRC, KT>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((act8_bwd_apply_kernel<FMT, SRC, KT>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL(act8_bwd_param_kernel, dim3(a.C), dim3(64), 0, st, a);
}
template <int FMT, int KT>
static void launch_bwd_sources(const Act8Bwd& a, unsigned rows, hipStream_t st) {
    switch ((a.g1 ? 1 : 0) + (a.g2 ? 2 : 0)) {
        case 0: if constexpr (KT > 0) launch_bwd<FMT, 0, KT>(a, rows, st); break;
        case 1: launch_bwd<FMT, 1, KT>(a, rows, st); break;
        case 2: launch_bwd<FMT, 2, KT>(a, rows, st); break;
        default: launch_bwd<FMT, 3, KT>(a, rows, st); break;
    }
}
template <int FMT>
static void launch_bwd_form(const Act8Bwd& a, unsigned rows, hipStream_t st) {
    switch (a.K) {
        case 0: launch_bwd_sources<FMT, 0>(a, rows, st); break;
        case 1: launch_bwd_sources<FMT, 1>(a, rows, st); break;
        case 2: launch_bwd_sources<FMT, 2>(a, rows, st); break;
        case 3: launch_bwd_sources<FMT, 3>(a, rows, st); break;
        default: launch_bwd_sources<FMT, 4>(a, rows, st); break;
    }
}
extern "C" int wmh_act8_in_lrelu_bwd(const uint8_t* codes, const uint8_t* scales, int fmt, const float* ss, const float* mean_rstd, const float* gamma,
                                     const float* g1, const float* g2, const float* dlogits, const float* wseg, int K, float* dy, float* dgamma, float* dbeta,
                                     float* dwseg, float* dbias, double* scratch, int N, int C, size_t S, float slope, void* stream) {
    if (bad_form(0, fmt) || N < 1 || C < 1 || S < 1 || (size_t)N * C > 65535) return wmh_fail(WMH_EINVAL, "act8_in_lrelu_bwd: bad format or size (1 to 65535 channels in all)");
    if (bad_codes(codes, scales) || !ss || !mean_rstd || !dy || (!scratch && wmh_act8_in_lrelu_bwd_scratch_doubles(N, C, S))) return wmh_fail(WMH_EINVAL, "act8_in_lrelu_bwd: null or misaligned pointer");
    if (!g1 && !g2 && !dlogits) return wmh_fail(WMH_EINVAL, "act8_in_lrelu_bwd: no gradient source");
    if (dlogits && (!wseg || K < 1 || K > ACT8_MAXK)) return wmh_fail(WMH_EINVAL, "act8_in_lrelu_bwd: head gradient without head weights, or not 1 to 4 classes");
    const unsigned rows = (unsigned)(N * C);
    Act8Bwd a{codes, scales, ss, mean_rstd, gamma, g1, g2, dlogits, wseg, dy, dgamma, dbeta, dlogits ? dwseg : nullptr, dbias, nullptr, nullptr,
              N, C, dlogits ? K : 0, bwd_split(N, C, S), S, slope};
    a.psums = scratch;
    a.dysum = scratch + (size_t)rows * a.split * (2 + ACT8_MAXK);
    if (fmt == WMH_ACT8_INT8) launch_bwd_form<WMH_ACT8_INT8>(a, rows, (hipStream_t)stream);
    else launch_bwd_form<WMH_ACT8_E4M3>(a, rows, (hipStream_t)stream);
    return wmh_check_launch("act8_in_lrelu_bwd kernels");
}
