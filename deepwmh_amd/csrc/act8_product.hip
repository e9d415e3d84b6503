// act8_product.hip -- the product of two packed e4m3 tensors (act8_common.h), and the weight gradient of a transposed convolution formed by it.
//
//   C[m, n] = sum over blocks of 128 k:  2^(ea[m, blk] + eb[n, blk]) sum_{k in blk} a[m, k] b[n, k]
//
// Two instructions, by the type of the result:
//  bfloat16  v_mfma_scale_f32_32x32x64_f8f6f4 on the codes themselves.  It takes one exponent byte per lane for each operand -- lane l holds row
//            l % 32 and 32 of the 64 k -- so a block of 128 is two instructions with the same bytes and the scales cost no arithmetic.  Inside it
//            eight neighbouring products are aligned to the largest and cut 2^-13 below (measured: 1 + 2^-13 stays, 1 + 2^-14 is lost; the same for
//            the unscaled fp8 instruction), which is 1.5e-5 of a sum of random terms at any length: a 250th of the result's own rounding.
//  float32   v_mfma_f32_32x32x16_bf16 on the codes widened to bfloat16 with their scale, which is exact (the type has float32's exponents; a value
//            below 2^-126 may lose bits): float32 sums, 1e-7, at half the rate.
// Accumulators are fp32 across the whole sum.
#include <type_traits>
#include "act8_common.h"

typedef float f32x4s __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

static inline unsigned cdivu(size_t a, size_t b) { return (unsigned)((a + b - 1) / b); }

struct Act8Prod {
    const uint8_t* a; const uint8_t* as; const uint8_t* b; const uint8_t* bs;
    void* c; float* slabs;
    int M, N, B;
    size_t nb, sp;                    // blocks and scale bytes per row
    int sum;                          // 1: one C for the whole batch
    int P, chunk;                     // parts of the sum and groups of 4 blocks in each
    int gm, gn;                       // tiles along M and N
};

// Eight codes to bfloat16 with their scale; exact.
__device__ __forceinline__ bf16x8 act8_widen(int lo, int hi, float s) {
    const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
    const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
    return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
// acc += b a^T over 64 k of a block for MT x NT tiles; j: the block's byte in the dwords of scales.
template <int MT, int NT, bool WIDE>
__device__ __forceinline__ void act8_tiles(const i32x8 (&fa)[MT], const i32x8 (&fb)[NT], f32x16 (&acc)[MT][NT], const unsigned (&ca)[MT], const unsigned (&cb)[NT],
                                           const int j) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int k = 0; k < NT; ++k)
                switch (j) {                                    // (a constant behind unrolling: the byte is part of the instruction)
                    case 0: acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k], fa[i], acc[i][k], 0, 0, 0, (int)cb[k], 0, (int)ca[i]); break;
                    case 1: acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k], fa[i], acc[i][k], 0, 0, 1, (int)cb[k], 1, (int)ca[i]); break;
                    case 2: acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k], fa[i], acc[i][k], 0, 0, 2, (int)cb[k], 2, (int)ca[i]); break;
                    default: acc[i][k] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[k], fa[i], acc[i][k], 0, 0, 3, (int)cb[k], 3, (int)ca[i]); break;
                }
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            bf16x8 wb[NT];
#pragma unroll
            for (int k = 0; k < NT; ++k) wb[k] = act8_widen(fb[k][2 * q], fb[k][2 * q + 1], act8_scale((cb[k] >> (8 * j)) & 0xFFu));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const bf16x8 wa = act8_widen(fa[i][2 * q], fa[i][2 * q + 1], act8_scale((ca[i] >> (8 * j)) & 0xFFu));
#pragma unroll
                for (int k = 0; k < NT; ++k) acc[i][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[k], wa, acc[i][k], 0, 0, 0);
            }
        }
    }
}
// E neighbouring values of a row, `left` of which exist; rows start at any element, and the memory path takes wide stores there.
template <int E>
__device__ __forceinline__ void act8_put(float* to, const float* v, int left) {
    if (left >= E) {
        *reinterpret_cast<f32x4s*>(to) = f32x4s{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < left) to[e] = v[e];
}
typedef uint16_t u16x8s __attribute__((ext_vector_type(8), aligned(2)));
template <int E>
__device__ __forceinline__ void act8_put(uint16_t* to, const float* v, int left) {
    if (left >= E) {
        u16x8s t;
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = Act8BF16::put(v[e]);
        *reinterpret_cast<u16x8s*>(to) = t;
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (e < left) to[e] = Act8BF16::put(v[e]);
}

// Results through LDS, a wave's 32 rows at a time, so that a store writes whole lines: straight from the registers a wave would write 16 or 32 bytes of
// 32 rows at once (8192 x 8192 float32 results: 520 us for the stores).  PARTS: the sum may have been cut (not where the tile is the largest).
template <int MT, int NT, bool WIDE, int NW, int BYTES, bool PARTS>
__device__ __forceinline__ void act8_store(const Act8Prod& p, uint8_t* lds, const f32x16 (&acc)[MT][NT], int lane, int w, int wm, int wn, int m0, int n0, int part,
                                           int item) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int r = lane & 31, h = lane >> 5;
    constexpr int LP = NT * 32 + 4;                             // row pitch in floats
    float* mine = reinterpret_cast<float*>(lds) + w * 32 * LP;
    static_assert(NW * 32 * LP * 4 <= BYTES, "the results fit the tiles' memory");
    const size_t out = ((size_t)part * (p.sum ? 1 : p.B) + item) * p.M;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<float4*>(mine + r * LP + j * 32 + 8 * q + 4 * h) =
                    make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // (only this wave's own rows)
        const int mb = m0 + (wm * MT + i) * 32, nbase = n0 + wn * NT * 32;
        if (WIDE || (PARTS && p.P > 1)) {
            constexpr int PER = NT * 8, RW = 64 / PER;          // lanes a row, rows a store
            float* c = PARTS && p.P > 1 ? p.slabs : reinterpret_cast<float*>(p.c);
#pragma unroll
            for (int q = 0; q < 32 / RW; ++q) {
                const int row = q * RW + lane / PER, col = (lane % PER) * 4;
                const float4 v = *reinterpret_cast<const float4*>(mine + row * LP + col);
                if (mb + row < p.M) act8_put<4>(c + (out + mb + row) * p.N + nbase + col, &v.x, p.N - nbase - col);
            }
        } else {
            constexpr int PER = NT * 4, RW = 64 / PER;
            uint16_t* c = reinterpret_cast<uint16_t*>(p.c);
#pragma unroll
            for (int q = 0; q < 32 / RW; ++q) {
                const int row = q * RW + lane / PER, col = (lane % PER) * 8;
                float v[8];
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(mine + row * LP + col);
                *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(mine + row * LP + col + 4);
                if (mb + row < p.M) act8_put<8>(c + (out + mb + row) * p.N + nbase + col, v, p.N - nbase - col);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// A workgroup of WM x WN waves forms TM x TN = (32 MT WM) x (32 NT WN) outputs, a wave MT x NT tiles of 32 x 32.  One step is one block of 128 k:
//  * The rows' 128 bytes come by LDS-DMA (16 bytes a lane, no registers), one step ahead of the matrix instructions, into the other of two
//    buffers; one barrier a step.  The DMA is written as asm: a builtin would make the compiler wait for it in front of the step's LDS reads.
//  * Two rows are the 64 banks' 256 bytes, and sixteen lanes a cycle read 16 bytes each of their own rows: the sixteen-byte pieces of row r are stored
//    in the order piece ^ (r / 2 % 8), so sixteen neighbouring rows hit all banks once (piece ^ (r % 8), every second bank twice, takes twice the LDS
//    cycles: 8192^3 470 us against 455).  The order is made by the addresses the DMA reads from.
//  * Scale bytes are read four blocks (a dword) at a time, a group ahead, and stay in registers; the instruction picks its byte.
//  * b is the first operand, so that a lane holds one row of C and four neighbouring columns in its registers: 8- and 16-byte stores.
// The sum may be cut into P parts of whole groups of 4 blocks, over batch items too where they are summed; the parts go to slabs that are added in
// order.
template <int WM, int WN, int MT, int NT, int KB, bool WIDE>
__global__ __launch_bounds__(64 * WM * WN, (MT * NT == 8 ? 2 : 1)) void act8_product_kernel(const Act8Prod p) {
    constexpr int NW = WM * WN, TM = 32 * MT * WM, TN = 32 * NT * WN, BLK = (TM + TN) * ACT8_BLOCK, STAGE = KB * BLK, NI = (TM + TN) / 8 / NW, NIA = TM / 8 / NW;
    static_assert(TM % (8 * NW) == 0 && TN % (8 * NW) == 0, "every wave loads whole eights of rows of a and of b");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5, wm = w % WM, wn = w / WM;
    // tiles in bands of 8 rows of tiles, an eighth of the list for each XCD (workgroups go to the XCDs in turn): what an XCD works on at a time is
    // a compact patch whose operands its L2 holds
    int t = blockIdx.x;
    {
        const int total = p.gm * p.gn, per = total / 8;
        if (t < per * 8) t = (t % 8) * per + t / 8;
    }
    const int band = t / (8 * p.gn), rows = min(8, p.gm - band * 8), in = t - band * 8 * p.gn;
    const int m0 = (band * 8 + in % rows) * TM, n0 = (in / rows) * TN;
    const int part = blockIdx.y, item = blockIdx.z;
    const int G = (int)(p.sp / 4);                              // groups of one item
    const size_t pitch = p.nb * ACT8_BLOCK;

    // This lane's piece of the rows it loads: 32-bit offsets from the tile's first row where the tile is large (a register less each; the plan
    // takes large tiles for rows below 2^24 bytes only), whole addresses where it is small.
    constexpr bool NEAR = MT * NT > 1;
    unsigned off[NI];
    const uint8_t* src[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const bool isa = i < NIA;
        const int row = (i * NW + w) * 8 + (lane >> 3) - (isa ? 0 : TM);
        const int g = isa ? min(m0 + row, p.M - 1) : min(n0 + row, p.N - 1);
        const unsigned piece = ((lane & 7) ^ ((w & 1) * 4 + (lane >> 4))) * 16;
        if constexpr (NEAR) off[i] = (unsigned)(g - (isa ? m0 : n0)) * (unsigned)pitch + piece;
        else src[i] = (isa ? p.a : p.b) + (size_t)g * pitch + piece;
    }
    const unsigned lbase = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    // blocks j0 .. j0 + KB - 1 of group g of item b into a buffer
    auto fetch = [&](int buf, int b, int g, int j0) __attribute__((always_inline)) {
        const size_t ob = (size_t)g * 512 + 128 * j0, oa = ob + (size_t)b * p.M * pitch, oc = ob + (size_t)b * p.N * pitch;
        const int left = KB > 1 ? (int)min((size_t)KB, p.nb - 4 * (size_t)g - j0) : 1;
#pragma unroll
        for (int k = 0; k < KB; ++k) {
            if (k >= left) break;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const unsigned to = lbase + buf * STAGE + k * BLK + (i * NW + w) * 1024;
                if constexpr (NEAR) {
                    const uint8_t* q = (i < NIA ? p.a + (size_t)m0 * pitch + oa : p.b + (size_t)n0 * pitch + oc) + 128 * k;
                    // (s_nop 4: the five wait states a scalar address would need had a vector instruction made it)
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off[i]), "s"(q) : "memory", "m0");
                } else {
                    const uint8_t* q = src[i] + (i < NIA ? oa : oc) + 128 * k;
                    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to), "v"(q) : "memory", "m0");
                }
            }
        }
    };
    const uint8_t* sra[MT]; const uint8_t* srb[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sra[i] = p.as + (size_t)min(m0 + (wm * MT + i) * 32 + r, p.M - 1) * p.sp;
#pragma unroll
    for (int j = 0; j < NT; ++j) srb[j] = p.bs + (size_t)min(n0 + (wn * NT + j) * 32 + r, p.N - 1) * p.sp;
    unsigned na[MT], nb[NT], ca[MT], cb[NT];
    auto scales = [&](int b, int g) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MT; ++i) na[i] = *reinterpret_cast<const unsigned*>(sra[i] + (size_t)b * p.M * p.sp + 4 * (size_t)g);
#pragma unroll
        for (int j = 0; j < NT; ++j) nb[j] = *reinterpret_cast<const unsigned*>(srb[j] + (size_t)b * p.N * p.sp + 4 * (size_t)g);
    };
    unsigned la[2][2], lb[2][2];                                // LDS addresses of the lane's pieces: half of the block, piece
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const unsigned at = r * 128 + (((4 * (u >> 1) + 2 * h + (u & 1)) ^ (r >> 1 & 7)) * 16);
        la[u >> 1][u & 1] = wm * MT * 4096 + at;
        lb[u >> 1][u & 1] = (TM + wn * NT * 32) * 128 + at;
    }
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const int g1 = min((part + 1) * p.chunk, p.sum ? p.B * G : G);
    int gi = part * p.chunk, buf = 0;
    int b = p.sum ? (G ? gi / G : 0) : item, g = p.sum ? (G ? gi % G : 0) : gi;
    if (gi < g1) {
        scales(b, g);
        fetch(0, b, g, 0);
    }
    for (; gi < g1; ++gi) {
        const int nj = (int)min((size_t)4, p.nb - 4 * (size_t)g);
        int bn = b, gn = g + 1;                                 // the group behind this one
        if (gn == G && p.sum) { gn = 0; ++bn; }
#pragma unroll
        for (int j0 = 0; j0 < 4; j0 += KB) {
            if (j0 >= nj) break;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (j0 == 0) {
#pragma unroll
                for (int i = 0; i < MT; ++i) { asm volatile("" : "+v"(na[i])); ca[i] = na[i]; }
#pragma unroll
                for (int i = 0; i < NT; ++i) { asm volatile("" : "+v"(nb[i])); cb[i] = nb[i]; }
                if (gi + 1 < g1) scales(bn, gn);
            }
            if (j0 + KB < nj) fetch(buf ^ 1, b, g, j0 + KB);
            else if (gi + 1 < g1) fetch(buf ^ 1, bn, gn, 0);
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                if (k > 0 && j0 + k >= nj) break;
                const uint8_t* s = lds + buf * STAGE + k * BLK;
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    i32x8 fa[MT], fb[NT];
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const i32x4 x = *reinterpret_cast<const i32x4*>(s + lb[t2][0] + 4096 * i), y = *reinterpret_cast<const i32x4*>(s + lb[t2][1] + 4096 * i);
                        fb[i] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const i32x4 x = *reinterpret_cast<const i32x4*>(s + la[t2][0] + 4096 * i), y = *reinterpret_cast<const i32x4*>(s + la[t2][1] + 4096 * i);
                        fa[i] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    }
                    act8_tiles<MT, NT, WIDE>(fa, fb, acc, ca, cb, j0 + k);
                }
            }
            buf ^= 1;
        }
        b = bn; g = gn;
    }

    act8_store<MT, NT, WIDE, NW, 2 * STAGE, (MT * NT < 8)>(p, lds, acc, lane, w, wm, wn, m0, n0, part, item);
}
// The large tile on the 8-bit instruction, for long sums: 256 x 256 by four waves of 128 x 128, one workgroup a CU.  A wave alone on its SIMD hides nothing
// by itself, so everything is asked for ahead of the matrix instructions and between them, in turn:
//  * Fragments are in registers twice: while one half of a block (64 k) is multiplied the other is read from LDS.
//  * Units of 64 rows x 128 bytes (whole lines) pass through 19 slots of LDS: a block's eight units that are read, the next block's eight, and three of the
//    one behind it.  A block's slots are free as soon as its second half is in registers, which is what the one barrier a block says.  Six of its sixteen
//    loads (a wave's) go out in the first half and ten in the second; sent in a burst they are slower (8192^3: 420 us against 410), and so are half blocks
//    of 64 bytes a row, which ask for every line twice (455).
//  * All loads are LDS-DMA, the scales' dwords too (the block's own, with every block), and return in order, so that s_waitcnt counts them.  Past the end
//    the last block is fetched again, so that the counts hold.
// 8192^3 402 to 410 us = 2700 TFLOP/s in a steady run (the eight waves above with their two buffers 450; the library's product of the same codes without
// block scales 329 to 340); without its memory traffic the loop takes 343, the traffic alone 277.  The clock moves under this load: of 60 launches in a row
// the tenth took 540 us and the last 406, and between other kernels 450 to 500 are usual.
__global__ __launch_bounds__(256, 1) void act8_product_deep_kernel(const Act8Prod p) {
    constexpr int UNIT = 64 * ACT8_BLOCK, NS = 19, SCALES = NS * UNIT;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];    // NS units, then two sets of 512 scale dwords
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5, wm = w & 1, wn = w >> 1;
    int t = blockIdx.x;
    {
        const int total = p.gm * p.gn, per = total / 8;
        if (t < per * 8) t = (t % 8) * per + t / 8;
    }
    const int band = t / (8 * p.gn), rows = min(8, p.gm - band * 8), in = t - band * 8 * p.gn;
    const int m0 = (band * 8 + in % rows) * 256, n0 = (in / rows) * 256;
    const int item = blockIdx.z, b = p.sum ? 0 : item, nb = (int)p.nb, T = p.sum ? p.B * nb : nb;        // T: blocks of the sum
    const size_t pitch = p.nb * ACT8_BLOCK;

    unsigned off[16], soff[2];
#pragma unroll
    for (int d = 0; d < 16; ++d) {                              // load d of a step: eight rows of unit d / 2
        const int row = (d >> 1 & 3) * 64 + ((d & 1) * 4 + w) * 8 + (lane >> 3);
        const int g = d < 8 ? min(m0 + row, p.M - 1) - m0 : min(n0 + row, p.N - 1) - n0;
        off[d] = (unsigned)g * (unsigned)pitch + ((lane & 7) ^ ((w & 1) * 4 + (lane >> 4))) * 16;
    }
    soff[0] = (unsigned)(min(m0 + w * 64 + lane, p.M - 1) - m0) * (unsigned)p.sp;
    soff[1] = (unsigned)(min(n0 + w * 64 + lane, p.N - 1) - n0) * (unsigned)p.sp;
    const unsigned lbase = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

    int fblk = 0;                                               // block of its item that is fetched
    const uint8_t* qa = p.a + ((size_t)b * p.M + m0) * pitch;
    const uint8_t* qb = p.b + ((size_t)b * p.N + n0) * pitch;
    const uint8_t* sa = p.as + ((size_t)b * p.M + m0) * p.sp;
    const uint8_t* sb = p.bs + ((size_t)b * p.N + n0) * p.sp;
    int fleft = T, fslot = 0;                                   // blocks to fetch, this one among them; slot of the next unit
    int mblk = 0;                                               // block of its item that is multiplied
    auto dma = [&](int d) __attribute__((always_inline)) {
        const unsigned to = lbase + fslot * UNIT + ((d & 1) * 4 + w) * 1024;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(off[d]), "s"(d < 8 ? qa : qb) : "memory", "m0");
        if (d & 1) fslot = fslot == NS - 1 ? 0 : fslot + 1;
    };
    auto fetch_scales = [&](int set) __attribute__((always_inline)) {
        const unsigned to = lbase + SCALES + set * 2048 + w * 256;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" :: "s"(to), "v"(soff[0]), "s"(sa + (fblk & ~3)) : "memory", "m0");
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" :: "s"(to + 1024), "v"(soff[1]), "s"(sb + (fblk & ~3)) : "memory", "m0");
    };
    auto advance = [&]() __attribute__((always_inline)) {       // (selects: the matrix instructions must stay in one block with the reads they hide)
        const bool on = --fleft > 0, wrap = on && fblk + 1 == nb;
        qa += (on ? ACT8_BLOCK : 0) + (wrap ? (size_t)(p.M - 1) * pitch : 0);
        qb += (on ? ACT8_BLOCK : 0) + (wrap ? (size_t)(p.N - 1) * pitch : 0);
        sa += wrap ? (size_t)p.M * p.sp : 0;
        sb += wrap ? (size_t)p.N * p.sp : 0;
        fblk = wrap ? 0 : fblk + (on ? 1 : 0);
    };
    unsigned at[2][2];                                          // the lane's pieces of a row: half of the block, piece
#pragma unroll
    for (int u = 0; u < 4; ++u) at[u >> 1][u & 1] = r * 128 + (((4 * (u >> 1) + 2 * h + (u & 1)) ^ (r >> 1 & 7)) * 16);
    i32x4 fa[2][4][2], fb[2][4][2];
    int rslot = 0;                                              // slot of the first unit of the step that is read
    unsigned base[4];                                           // of the wave's two units of a and two of b
    auto bases = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = rslot + (i < 2 ? 2 * wm + i : 4 + 2 * wn + i - 2);
            base[i] = (s >= NS ? s - NS : s) * UNIT;
        }
    };
    auto read = [&](int k, int q) __attribute__((always_inline)) {       // sixteen bytes q of 16 of half k of the step's fragments
        const int i = q >> 2, u = q & 1;
        if (q & 2) fa[k][i][u] = *reinterpret_cast<const i32x4*>(lds + (base[i >> 1] + at[k][u]) + 4096 * (i & 1));
        else fb[k][i][u] = *reinterpret_cast<const i32x4*>(lds + (base[2 + (i >> 1)] + at[k][u]) + 4096 * (i & 1));
    };
    unsigned ca[4], cb[4];
    auto read_scales = [&](int set) __attribute__((always_inline)) {
        const unsigned* sc = reinterpret_cast<const unsigned*>(lds + SCALES + set * 2048);
#pragma unroll
        for (int i = 0; i < 4; ++i) { ca[i] = sc[wm * 128 + 32 * i + r]; cb[i] = sc[256 + wn * 128 + 32 * i + r]; }
    };
    f32x16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    auto multiply = [&](int k, int q, const unsigned (&xa)[4], const unsigned (&xb)[4]) __attribute__((always_inline)) {
        const int i = q >> 2, j = q & 3;
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_shufflevector(fb[k][j][0], fb[k][j][1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                                    __builtin_shufflevector(fa[k][i][0], fa[k][i][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0,
                                                                    (int)xb[j], 0, (int)xa[i]);
    };

#pragma unroll
    for (int k = 0; k < 2; ++k) {
        fetch_scales(k);
#pragma unroll
        for (int d = 0; d < 16; ++d) dma(d);
        advance();
    }
    asm volatile("s_waitcnt vmcnt(18)\n\ts_barrier" ::: "memory");
    bases();
    read_scales(0);
#pragma unroll
    for (int q = 0; q < 16; ++q) read(0, q);
    for (int m = 0; m < T; ++m) {
        unsigned xa[4], xb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { xa[i] = ca[i] >> (8 * (mblk & 3)); xb[i] = cb[i] >> (8 * (mblk & 3)); }
        mblk = mblk + 1 == nb ? 0 : mblk + 1;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            read(1, q);
            multiply(0, q, xa, xb);
            if (q < 12 && q % 2 == 0) dma(q / 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        // the next step has landed (all but the six loads just asked for), and every wave has this one in registers: its slots may be written
        asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        rslot = rslot + 8 >= NS ? rslot + 8 - NS : rslot + 8;
        bases();
        read_scales((m + 1) & 1);
        fetch_scales(m & 1);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            read(0, q);
            multiply(1, q, xa, xb);
            if (q < 10) dma(6 + q);
            if (q == 10) advance();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    act8_store<4, 4, false, 4, NS * UNIT, false>(p, lds, acc, lane, w, wm, wn, m0, n0, 0, item);
}
// c[i] = sum of the P slabs of n floats: a workgroup takes 32 outputs, its 8 half-waves every eighth of the slabs each, in order, and the eight sums
// are added in order.
template <bool WIDE>
__global__ __launch_bounds__(256) void act8_product_join_kernel(const float* __restrict__ slabs, void* __restrict__ c, size_t n, int P) {
    __shared__ float sh[8][32];
    const int l = threadIdx.x & 31, k = threadIdx.x >> 5;
    for (size_t base = (size_t)blockIdx.x * 32; base < n; base += (size_t)gridDim.x * 32) {
        const size_t i = base + l < n ? base + l : n - 1;
        float s = 0.f;
#pragma unroll 8
        for (int q = k; q < P; q += 8) s += slabs[(size_t)q * n + i];
        sh[k][l] = s;
        __syncthreads();
        if (k == 0 && base + l < n) {
#pragma unroll
            for (int q = 1; q < 8; ++q) s += sh[q][l];
            if constexpr (WIDE) reinterpret_cast<float*>(c)[i] = s;
            else reinterpret_cast<uint16_t*>(c)[i] = Act8BF16::put(s);
        }
        __syncthreads();
    }
}
static void launch_join(bool wide, const float* slabs, void* c, size_t n, int P, hipStream_t st) {
    const unsigned blocks = cdivu(n, 32) > 65536u ? 65536u : cdivu(n, 32);
    if (wide) hipLaunchKernelGGL(act8_product_join_kernel<true>, dim3(blocks), dim3(256), 0, st, slabs, c, n, P);
    else hipLaunchKernelGGL(act8_product_join_kernel<false>, dim3(blocks), dim3(256), 0, st, slabs, c, n, P);
}

// Tiles and parts, by measurement (us, float32 / bfloat16 result, replayed graphs of ten calls) of one to three items.  Tiles of many small items are counted
// like those of one large matrix, whether or not they are full: 256 x (64 x 64 x 512) takes 18 / 11 us on 256 tiles of 256 x 256.
//  0  256 x 256, one workgroup a CU: from 192 tiles on (4096^3: 109 / 58, tile 1 136 / 80; with 128 tiles, 4096 x 2048 x 1024, 30 / 22 against
//     24 / 16 of tile 1).  bfloat16 results of sums from 4096 k on by four waves (8192 x 8192 x 16384 845, by eight 908; 4096^3 58 / 62; 3600 x 3900 x
//     3500 52 / 51, 3600 x 3900 x 2100 38 / 35: a longer start and end), the others by eight of 128 x 64.
//  1  128 x 128, two workgroups a CU: from 257 tiles on (the 4096 x 2048 x 1024 above: tile 2 28 / 20)
//  4  128 x 128 with two blocks a step, where every tile has a CU: 224 to 256 tiles (2048^3: 25 / 16, tile 1 27 / 18, tile 2 27 / 19; with 189
//     tiles, 300 x 8000 x 2500, 26 / 18 against 24 / 17 of tile 2)
//  2  64 x 64, five workgroups a CU: more than 256 tiles
//  3  64 x 64 with four blocks a step: up to 256 tiles, a step is a memory latency (1024^3: 7.0 / 5.8, tile 2 7.7 / 6.4)
//  5  32 x 128 for up to 32 rows (16 x 4096 x 4096: 8.3 / 7.9, tile 3 8.9 / 7.9)
// A sum is cut where the tiles leave CUs idle (half of them or more) and it is long enough to pay for the join, from 6 groups of 512 k on: 64 x
// 256 x 65536 in 64 parts 12 us, in 32 16, in 128 13; 40 x 8192 x 2048 (4 groups) 9.6 whole, 12.6 in two.
struct Act8Plan { int tile, P, chunk, gm, gn; };
static Act8Plan plan_product(int B, int M, int N, size_t K, int sum) {
    static const int tm[6] = {256, 128, 64, 64, 128, 32}, tn[6] = {256, 128, 64, 64, 128, 128};
    const size_t items = sum ? 1 : B, groups = act8_scale_pitch(K) / 4 * (sum ? B : 1);
    const bool near = act8_pitch(K) < ((size_t)1 << 24);        // 32-bit offsets inside a large tile
    Act8Plan q;
    auto tiles = [&](int i) { return (size_t)cdivu(M, tm[i]) * cdivu(N, tn[i]) * items; };
    if (M <= 32) q.tile = 5;
    else if (near && tiles(0) >= 192) q.tile = 0;
    else if (near && tiles(1) > 256) q.tile = 1;
    else if (near && tiles(1) >= 224) q.tile = 4;
    else q.tile = tiles(2) > 256 ? 2 : 3;
    q.gm = (int)cdivu(M, tm[q.tile]); q.gn = (int)cdivu(N, tn[q.tile]);
    const size_t t = tiles(q.tile), want = q.tile == 5 ? 512 : 256;
    size_t P = groups >= 6 && t <= want / 2 ? want / t : 1;
    if (P > groups) P = groups ? groups : 1;
    q.chunk = (int)((groups + P - 1) / P);
    q.P = q.chunk ? (int)((groups + q.chunk - 1) / q.chunk) : 1;
    return q;
}
extern "C" size_t wmh_act8_product_workspace_floats(int B, int M, int N, size_t K, int sum) {
    if (B < 1 || M < 1 || N < 1) return 0;
    const Act8Plan q = plan_product(B, M, N, K, sum);
    return q.P > 1 ? (size_t)q.P * (sum ? 1 : B) * M * N : 0;
}
template <int WM, int WN, int MT, int NT, int KB, bool WIDE>
static int launch_product(const Act8Prod& p, hipStream_t st) {
    constexpr int bytes = 2 * KB * (32 * MT * WM + 32 * NT * WN) * ACT8_BLOCK;
    const void* f = reinterpret_cast<const void*>(&act8_product_kernel<WM, WN, MT, NT, KB, WIDE>);
    if (bytes > 65536 && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        return wmh_fail(WMH_ELAUNCH, "act8_product: the device refuses the kernel's shared memory");
    hipLaunchKernelGGL((act8_product_kernel<WM, WN, MT, NT, KB, WIDE>), dim3(p.gm * p.gn, p.P, p.sum ? 1 : p.B), dim3(64 * WM * WN), bytes, st, p);
    return wmh_check_launch("act8_product_kernel");
}
// (The plan cuts no sum into parts where it takes the large tile.)
static int launch_product_deep(const Act8Prod& p, hipStream_t st) {
    constexpr int bytes = 19 * 64 * ACT8_BLOCK + 2 * 2048;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&act8_product_deep_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        return wmh_fail(WMH_ELAUNCH, "act8_product: the device refuses the kernel's shared memory");
    hipLaunchKernelGGL(act8_product_deep_kernel, dim3(p.gm * p.gn, 1, p.sum ? 1 : p.B), dim3(256), bytes, st, p);
    return wmh_check_launch("act8_product_deep_kernel");
}
template <bool WIDE>
static int launch_product_tile(int tile, const Act8Prod& p, hipStream_t st) {
    switch (tile) {
        case 0:
            if (!WIDE && p.nb * (p.sum ? p.B : 1) >= 32) return launch_product_deep(p, st);
            return launch_product<2, 4, 4, 2, 1, WIDE>(p, st);
        case 1: return launch_product<2, 2, 2, 2, 1, WIDE>(p, st);
        case 2: return launch_product<2, 2, 1, 1, 1, WIDE>(p, st);
        case 3: return launch_product<2, 2, 1, 1, 4, WIDE>(p, st);
        case 4: return launch_product<2, 2, 2, 2, 2, WIDE>(p, st);
        default: return launch_product<1, 4, 1, 1, 1, WIDE>(p, st);
    }
}
static int product(const uint8_t* a, const uint8_t* as, const uint8_t* b, const uint8_t* bs, void* c, int dtype, float* ws, int B, int M, int N, size_t K,
                   int sum, hipStream_t st) {
    const Act8Plan q = plan_product(B, M, N, K, sum);
    if ((size_t)q.gm * q.gn > 0x7FFFFF || q.P > 65535 || (!sum && B > 65535) || act8_scale_pitch(K) / 4 * (size_t)(sum ? B : 1) > 0x7FFFFFFF)
        return wmh_fail(WMH_EINVAL, "act8_product: more than 65535 items, 2^23 tiles or 2^31 groups of 512 k");
    const Act8Prod p{a, as, b, bs, c, ws, M, N, B, act8_blocks(K), act8_scale_pitch(K), sum, q.P, q.chunk, q.gm, q.gn};
    const int rc = dtype == WMH_F32 ? launch_product_tile<true>(q.tile, p, st) : launch_product_tile<false>(q.tile, p, st);
    if (rc != WMH_OK || q.P == 1) return rc;
    const size_t n = (size_t)(sum ? 1 : B) * M * N;
    launch_join(dtype == WMH_F32, ws, c, n, q.P, st);
    return wmh_check_launch("act8_product_join_kernel");
}
extern "C" int wmh_act8_product(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales, void* c, int dtype, float* workspace,
                                int B, int M, int N, size_t K, int sum, void* stream) {
    if (B < 0 || M < 0 || N < 0 || (dtype != WMH_F32 && dtype != WMH_BF16)) return wmh_fail(WMH_EINVAL, "act8_product: bad size or output type");
    if (M == 0 || N == 0 || (B == 0 && !sum)) return WMH_OK;
    if (!c || (uintptr_t)c % (dtype == WMH_F32 ? 4 : 2)) return wmh_fail(WMH_EINVAL, "act8_product: null or misaligned output");
    if (B > 0 && K > 0 && (!a || !b || !a_scales || !b_scales || (uintptr_t)a % 16 || (uintptr_t)b % 16 || (uintptr_t)a_scales % 4 || (uintptr_t)b_scales % 4))
        return wmh_fail(WMH_EINVAL, "act8_product: null or misaligned operand");
    if ((!workspace || (uintptr_t)workspace % 16) && wmh_act8_product_workspace_floats(B, M, N, K, sum))
        return wmh_fail(WMH_EINVAL, "act8_product: null or misaligned workspace");
    return product(a, a_scales, b, b_scales, c, dtype, workspace, B, M, N, K, sum, (hipStream_t)stream);
}

// ---- weight gradient of a transposed convolution (kernel = stride = (kt, 2, 2)) -----------------------------------------------------------
//   dW[ci, (co, t)] = sum_{n, v} q(lrelu(x[n, ci, v] sc + sh)) q(dY[n, co, 2v + t]):  a product over the voxels, which are contiguous in x.
// Two forms.  Separate: x and dY are packed (dY by taps: row (n, co, kd, kh, kw), blocks along the low-resolution voxels), then multiplied.  A wave
// packs the two kw of a block: they are neighbours in memory, a lane reads its two voxels' pairs and trades halves with its neighbour, so that even
// lanes hold four voxels of kw 0 and odd lanes of kw 1.
__global__ __launch_bounds__(256) void act8_pack_taps_kernel(const float* __restrict__ dy, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int kt,
                                                             unsigned H, unsigned W, unsigned S, unsigned units /* N Cout kt 2 blocks */) {
    constexpr unsigned U = 4;
    const unsigned nb = (unsigned)act8_blocks(S), sp = (unsigned)act8_scale_pitch(S), l = threadIdx.x & 63;
    const unsigned u0 = __builtin_amdgcn_readfirstlane((blockIdx.x * 4 + (threadIdx.x >> 6)) * U);
    const bool odd = l & 1;
    float z[U][4];
#pragma unroll
    for (unsigned u = 0; u < U; ++u) {
        const unsigned unit = u0 + u < units ? u0 + u : units - 1, pr = unit / nb, v = (unit - pr * nb) * ACT8_BLOCK + 2 * l;
        const unsigned kh = pr & 1, kd = (pr >> 1) % kt;
        const float* src = dy + (size_t)(pr / (2 * kt)) * 4 * kt * S;
#pragma unroll
        for (unsigned i = 0; i < 2; ++i) {
            const unsigned vc = v + i < S ? v + i : 0, q = vc / W, w = vc - q * W, h = q % H, d = q / H;
            const float* p = src + (((kt * d + kd) * 2 * H + 2 * h + kh) * 2 * W + 2 * w);
            z[u][2 * i] = v + i < S ? p[0] : 0.f;
            z[u][2 * i + 1] = v + i < S ? p[1] : 0.f;
        }
    }
#pragma unroll
    for (unsigned u = 0; u < U; ++u) {
        if (u0 + u >= units) break;
        const unsigned pr = (u0 + u) / nb, blk = u0 + u - pr * nb;
        float v[4];
        act8_trade(z[u], odd, v);
        const unsigned m0 = act8_abs_bits(v[0]), m1 = act8_abs_bits(v[1]), m2 = act8_abs_bits(v[2]), m3 = act8_abs_bits(v[3]);
        const unsigned ma = m0 > m1 ? m0 : m1, mb = m2 > m3 ? m2 : m3;
        const unsigned byte = act8_byte<WMH_ACT8_E4M3>(act8_parity_max(ma > mb ? ma : mb));
        const float inv = act8_inverse(byte);
        const size_t row = 2 * (size_t)pr + (l & 1);
        reinterpret_cast<unsigned*>(codes + (row * nb + blk) * ACT8_BLOCK)[l >> 1] =
            act8_encode4<WMH_ACT8_E4M3>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, byte == 255u);
        if (l < 2 || (blk == nb - 1 && (l >> 1) < sp - blk)) scales[row * sp + blk + (l >> 1)] = l < 2 ? (uint8_t)byte : 0;
    }
}
// Fused: one pass over x and dY.  A workgroup of 8 waves owns 64 ci x 256 (co, t) and a run of blocks; per block it packs 64 rows of x and
// 256 of dY into LDS (the same codes and bytes as the separate kernels) and multiplies them there.
//  * A unit is 16 bytes a lane: two rows of x, or the two kw rows of one (co, kd, kh).  QUAD: the width is even and the voxels a multiple of 4, so that
//    they are one load and all inside or all outside; else four loads, each voxel with its own place and its own end.
//  * A wave has all its 20 units of a block in flight (164 KB a CU); as soon as one is packed its register is loaded from the next block.
//  * Two LDS buffers, one barrier a block; what bounds it is the memory.
struct Act8Tu {
    const float* x; const float* ss; const float* dy; float* out;
    int N, Cin, Cout, H, W, tn, tiles, P, chunk;
    size_t S; float slope;
};
template <int KT, bool NORM, bool QUAD>
__global__ __launch_bounds__(512, 2) void act8_tu_wgrad_kernel(const Act8Tu a) {
    constexpr int T = 4 * KT, NX = 4, NY = 16, ROWS = 64 + 256, STAGE = ROWS * ACT8_BLOCK;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];
    __shared__ float lsc[2][ROWS];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, l = lane & 31;
    // the tiles of a part run side by side on one XCD (workgroups go to the XCDs in turn): they read the same blocks
    const int in8 = blockIdx.x / 8, part = (in8 / a.tiles) * 8 + blockIdx.x % 8, tile = in8 % a.tiles;
    const int m0 = (tile / a.tn) * 64, n0 = (tile % a.tn) * 256;
    const int nbs = (int)act8_blocks(a.S), total = a.N * nbs;
    const int b1 = min((part + 1) * a.chunk, total);
    int b = part * a.chunk;
    if (part >= a.P || b >= b1) return;                         // (whole workgroup)

    // Addresses are the sample's base and a 32-bit offset in bytes (the host checks the range), the lane's and the unit's: the unit's is of the
    // channel row in x, and of the channel and (kd, kh), the same for the whole wave, in dY
    unsigned xrow[NX], yu[NY];
#pragma unroll
    for (int i = 0; i < NX; ++i) xrow[i] = (unsigned)min(m0 + (w * NX + i) * 2 + half, a.Cin - 1);
#pragma unroll
    for (int i = 0; i < NY; ++i) {
        const int j = n0 / 2 + w * NY + i;                      // (co, kd, kh)
        yu[i] = 4u * ((unsigned)min(j / (2 * KT), a.Cout - 1) * T * (unsigned)a.S + ((j / 2 % KT) * 2 * a.H + j % 2) * 2 * a.W);
    }
    float z[NX + NY][4];
    float2 nrm[NX];
    // block number -> sample, first voxel; the lane's offsets into x's and dY's channels
    int n = b / nbs;
    size_t v0 = (size_t)(b % nbs) * ACT8_BLOCK;
    unsigned xoff[QUAD ? 1 : 4], yoff[QUAD ? 1 : 2];
    auto place = [&]() __attribute__((always_inline)) {
        const unsigned xv = (unsigned)v0 + 4 * l, yv = (unsigned)v0 + 2 * lane;
#pragma unroll
        for (unsigned e = 0; e < (QUAD ? 1 : 4); ++e) xoff[e] = 4 * (xv + e < a.S ? xv + e : 0);
#pragma unroll
        for (unsigned e = 0; e < (QUAD ? 1 : 2); ++e) {
            const unsigned yc = yv + e < a.S ? yv + e : 0;
            const unsigned wv = yc % a.W, q = yc / a.W, h = q % a.H, d = q / a.H;
            yoff[e] = 4 * (((KT * d) * 2 * a.H + 2 * h) * 2 * a.W + 2 * wv);
        }
    };
    auto load = [&](int u) __attribute__((always_inline)) {
        f32x4s t;
        if (u < NX) {
            const char* base = reinterpret_cast<const char*>(a.x + (size_t)n * a.Cin * a.S);
            if constexpr (QUAD) t = *reinterpret_cast<const f32x4s*>(base + (xrow[u] * 4u * (unsigned)a.S + xoff[0]));
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = *reinterpret_cast<const float*>(base + (xrow[u] * 4u * (unsigned)a.S + xoff[QUAD ? 0 : e]));
        } else {
            const char* base = reinterpret_cast<const char*>(a.dy + (size_t)n * a.Cout * T * a.S);
            if constexpr (QUAD) t = *reinterpret_cast<const f32x4s*>(base + (yu[u - NX] + yoff[0]));
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = *reinterpret_cast<const float*>(base + (yu[u - NX] + yoff[QUAD ? 0 : e / 2] + 4 * (e & 1)));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) z[u][e] = t[e];
    };
    auto norms = [&]() __attribute__((always_inline)) {
        if constexpr (NORM)
#pragma unroll
            for (int i = 0; i < NX; ++i) nrm[i] = *reinterpret_cast<const float2*>(a.ss + 2 * ((size_t)n * a.Cin + xrow[i]));
    };
    const int r = lane & 31, wm = w & 1, wn = w >> 1;
    unsigned la[2][2], lb[2][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const unsigned at = r * 128 + (((4 * (u >> 1) + 2 * half + (u & 1)) ^ (r & 7)) * 16);
        la[u >> 1][u & 1] = wm * 4096 + at;
        lb[u >> 1][u & 1] = (64 + wn * 64) * 128 + at;
    }
    f32x16 acc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[k][e] = 0.f;

    place();
#pragma unroll
    for (int u = 0; u < NX + NY; ++u) load(u);
    norms();
    float2 cur[NX];
    int buf = 0;
    auto step = [&](auto again) __attribute__((always_inline)) {
        constexpr bool more = decltype(again)::value;
        bool xin[4], yin[2];                                    // inside the row
#pragma unroll
        for (int e = 0; e < 4; ++e) xin[e] = v0 + 4 * l + (QUAD ? 0 : e) < a.S;
#pragma unroll
        for (int e = 0; e < 2; ++e) yin[e] = v0 + 2 * lane + (QUAD ? 0 : e) < a.S;
#pragma unroll
        for (int i = 0; i < NX; ++i) cur[i] = nrm[i];
        if constexpr (more) {
            v0 += ACT8_BLOCK;
            if (v0 >= a.S) { v0 = 0; ++n; norms(); }
            place();
        }
        uint8_t* st = lds + buf * STAGE;
#pragma unroll
        for (int u = 0; u < NX + NY; ++u) {
            float v[4];
            int row, dw;                                        // LDS row, and dword in it
            unsigned m;
            if (u < NX) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = z[u][e];
                    if constexpr (NORM) v[e] = wmh_lrelu(fmaf(v[e], cur[u < NX ? u : 0].x, cur[u < NX ? u : 0].y), a.slope);
                    v[e] = xin[e] ? v[e] : 0.f;
                }
                row = (w * NX + u) * 2 + half; dw = l;
            } else {
                float t[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = yin[e / 2] ? z[u][e] : 0.f;
                act8_trade(t, lane & 1, v);
                row = 64 + (w * NY + u - NX) * 2 + (lane & 1); dw = lane >> 1;
            }
            if constexpr (more) load(u);
            const unsigned m0_ = act8_abs_bits(v[0]), m1_ = act8_abs_bits(v[1]), m2_ = act8_abs_bits(v[2]), m3_ = act8_abs_bits(v[3]);
            const unsigned ma = m0_ > m1_ ? m0_ : m1_, mb = m2_ > m3_ ? m2_ : m3_;
            m = ma > mb ? ma : mb;
            m = u < NX ? act8_lanes_max(m) : act8_parity_max(m);
            const unsigned byte = act8_byte<WMH_ACT8_E4M3>(m);
            const float inv = act8_inverse(byte);
            const unsigned code = act8_encode4<WMH_ACT8_E4M3>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, byte == 255u);
            *reinterpret_cast<unsigned*>(st + row * 128 + (((dw >> 2) ^ (row & 7)) * 16) + (dw & 3) * 4) = code;
            if (dw == 0) lsc[buf][row] = act8_scale(byte);
            __builtin_amdgcn_sched_barrier(0);                  // one unit after the other: interleaved, their temporaries pass the register file
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const float sa = lsc[buf][wm * 32 + r], sb0 = lsc[buf][64 + wn * 64 + r], sb1 = lsc[buf][64 + wn * 64 + 32 + r];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            i32x4 fa[2], fb[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                fa[e] = *reinterpret_cast<const i32x4*>(st + la[t][e]);
                fb[0][e] = *reinterpret_cast<const i32x4*>(st + lb[t][e]);
                fb[1][e] = *reinterpret_cast<const i32x4*>(st + lb[t][e] + 4096);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bf16x8 wa = act8_widen(fa[e][2 * k], fa[e][2 * k + 1], sa);
                    acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(act8_widen(fb[0][e][2 * k], fb[0][e][2 * k + 1], sb0), wa, acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(act8_widen(fb[1][e][2 * k], fb[1][e][2 * k + 1], sb1), wa, acc[1], 0, 0, 0);
                }
        }
        buf ^= 1;
    };
    for (; b + 1 < b1; ++b) step(std::true_type());
    step(std::false_type());
    const int m = m0 + wm * 32 + r, NT = a.Cout * T;
    if (m >= a.Cin) return;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = n0 + wn * 64 + k * 32 + 8 * q + 4 * half;
            const float v[4] = {acc[k][4 * q], acc[k][4 * q + 1], acc[k][4 * q + 2], acc[k][4 * q + 3]};
            if (col < NT) act8_put<4>(a.out + ((size_t)part * a.Cin + m) * NT + col, v, 4);      // (T is a multiple of 4)
        }
}
// Fused where 32-bit offsets reach and x and dY are not read too often (us, fused / separate, replayed graphs): 1 tile, 2 x 64 -> 32 from 63 x 61 x 59,
// 121 / 210 (64^3: 133 / 380 before the product was faster); 4 tiles, 128 -> 64 from 31 x 33 x 27, 53 / 61; 8 tiles, 128 -> 128 from 16^3, 26 / 28, and 4 x
// 24^3, 84 / 119; 9 tiles, 160 -> 96 from 13^3, 26 / 23; 16 tiles, 256 -> 128 from 16^3, 36 / 33; 50 tiles, 320 -> 320 from 4^3, 31 / 13.  A few blocks take
// the same time on the device (40 -> 24 from 5 x 7 x 9: 12.2 / 11.7) and one launch less on the host (14.8 / 17.9).
struct Act8TuPlan { bool fused; int tn, tiles, P, chunk; };
static Act8TuPlan plan_tu(int N, int Cin, int Cout, int D, int H, int W, int kt) {
    const size_t S = (size_t)D * H * W, total = (size_t)N * act8_blocks(S);
    Act8TuPlan q;
    q.tn = (int)cdivu((size_t)Cout * 4 * kt, 256);
    q.tiles = q.tn * (int)cdivu(Cin, 64);
    q.fused = S * Cout * 4 * kt < ((size_t)1 << 30) && S * Cin < ((size_t)1 << 30) && total < ((size_t)1 << 30) && q.tiles <= 8;
    size_t P = 256 / (q.tiles < 1 ? 1 : q.tiles) / 8 * 8;
    if (P < 8) P = 8;
    q.chunk = (int)((total + P - 1) / P);
    q.P = q.chunk ? (int)((total + q.chunk - 1) / q.chunk) : 1;
    return q;
}

static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
template <int KT>
static void launch_tu(const Act8Tu& a, dim3 grid, hipStream_t st) {
    const bool quad = a.W % 2 == 0 && a.S % 4 == 0;
    if (a.ss && quad) hipLaunchKernelGGL((act8_tu_wgrad_kernel<KT, true, true>), grid, dim3(512), 0, st, a);
    else if (a.ss) hipLaunchKernelGGL((act8_tu_wgrad_kernel<KT, true, false>), grid, dim3(512), 0, st, a);
    else if (quad) hipLaunchKernelGGL((act8_tu_wgrad_kernel<KT, false, true>), grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((act8_tu_wgrad_kernel<KT, false, false>), grid, dim3(512), 0, st, a);
}
extern "C" size_t wmh_act8_convtranspose3d_wgrad_workspace_bytes(int N, int Cin, int Cout, int D, int H, int W, int kt) {
    if (N < 1 || Cin < 1 || Cout < 1 || D < 1 || H < 1 || W < 1 || (kt != 1 && kt != 2)) return 0;
    const size_t S = (size_t)D * H * W, ra = (size_t)N * Cin, rb = (size_t)N * Cout * 4 * kt;
    const Act8TuPlan q = plan_tu(N, Cin, Cout, D, H, W, kt);
    if (q.fused) return q.P > 1 ? (size_t)q.P * Cin * Cout * 4 * kt * 4 : 16;
    return (ra + rb) * act8_pitch(S) + up16(ra * act8_scale_pitch(S)) + up16(rb * act8_scale_pitch(S)) +
           4 * wmh_act8_product_workspace_floats(N, Cin, Cout * 4 * kt, S, 1);
}
extern "C" int wmh_act8_convtranspose3d_wgrad(const float* x, const float* ss, const float* dY, float* dW, void* workspace, int N, int Cin, int Cout, int D,
                                              int H, int W, int kt, float slope, void* stream) {
    if (N < 1 || Cin < 1 || Cout < 1 || D < 1 || H < 1 || W < 1 || (kt != 1 && kt != 2) || (size_t)Cout * 4 * kt > 0x7FFFFFFF)
        return wmh_fail(WMH_EINVAL, "act8_convtranspose3d_wgrad: bad size");
    if ((size_t)D * H * W * 4 * kt > 0x7FFFFFFF || (size_t)N * Cout * 2 * kt * act8_blocks((size_t)D * H * W) > 0xFFFFFF0)
        return wmh_fail(WMH_EINVAL, "act8_convtranspose3d_wgrad: more than 2^31 voxels in a channel of dY, or 2^36 in all of it");
    if (!x || !dY || !dW || !workspace || (uintptr_t)workspace % 16) return wmh_fail(WMH_EINVAL, "act8_convtranspose3d_wgrad: null or misaligned pointer");
    const size_t S = (size_t)D * H * W, ra = (size_t)N * Cin, rb = (size_t)N * Cout * 4 * kt;
    const Act8TuPlan q = plan_tu(N, Cin, Cout, D, H, W, kt);
    if (q.fused) {
        hipStream_t st = (hipStream_t)stream;
        const Act8Tu a{x, ss, dY, q.P > 1 ? (float*)workspace : dW, N, Cin, Cout, H, W, q.tn, q.tiles, q.P, q.chunk, S, slope};
        const dim3 grid((unsigned)((q.P + 7) / 8 * 8 * q.tiles));
        if (kt == 2) launch_tu<2>(a, grid, st);
        else launch_tu<1>(a, grid, st);
        const int rc = wmh_check_launch("act8_tu_wgrad_kernel");
        if (rc != WMH_OK || q.P == 1) return rc;
        const size_t n = (size_t)Cin * Cout * 4 * kt;
        launch_join(true, (const float*)workspace, dW, n, q.P, st);
        return wmh_check_launch("act8_product_join_kernel");
    }
    uint8_t* ac = (uint8_t*)workspace;
    uint8_t* bc = ac + ra * act8_pitch(S);
    uint8_t* as = bc + rb * act8_pitch(S);
    uint8_t* bs = as + up16(ra * act8_scale_pitch(S));
    float* pw = (float*)(bs + up16(rb * act8_scale_pitch(S)));
    int rc = wmh_act8_pack(x, WMH_F32, (size_t)Cin * S, S, ss, ss ? WMH_ACT8_ACTIVATE : WMH_ACT8_PLAIN, slope, WMH_ACT8_E4M3, ac, as, N, Cin, S, stream);
    if (rc != WMH_OK) return rc;
    const size_t units = rb / 2 * act8_blocks(S);
    hipLaunchKernelGGL(act8_pack_taps_kernel, dim3(cdivu(units, 16)), dim3(256), 0, (hipStream_t)stream, dY, bc, bs, kt, (unsigned)H, (unsigned)W, (unsigned)S,
                       (unsigned)units);
    rc = wmh_check_launch("act8_pack_taps_kernel");
    if (rc != WMH_OK) return rc;
    return product(ac, as, bc, bs, dW, WMH_F32, pw, N, Cin, Cout * 4 * kt, S, 1, (hipStream_t)stream);
}
