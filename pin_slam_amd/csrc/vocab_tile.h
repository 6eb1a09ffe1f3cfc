// The matrix-core tile of the label head (vocab.hip): C[a][b] = sum_k A[a][k] B[b][k] over 16-bit operands with k contiguous,
// accumulated in fp32.
//
// Operands lie in memory as [plane][row][k], rows padded with zeros to a multiple of 64 k.  A value of fp32 is two planes of fp16,
// x 2^e = h + l (11 bits each), and its product three matrix products, l h + h l + h h, accumulated in that order: l l, at
// most 2^-22 of the product, is left out.
//
// LDS: a row's 64 k of one step are 8 chunks of 16 bytes; chunk c of row r is kept at position c ^ ((r >> 1) & 7), so that the 16
// lanes that read one chunk of 16 rows touch every bank once.  The loads write LDS directly (the lane's place is fixed, so the
// permutation is in the addresses they read).
#pragma once
#include "pin_common.h"

namespace pin {

typedef _Float16 vt_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 vt_b8 __attribute__((ext_vector_type(8)));
typedef float vt_f4 __attribute__((ext_vector_type(4)));
typedef unsigned int vt_u4 __attribute__((ext_vector_type(4)));

constexpr int VT = 128;        // rows of A and of B a workgroup
constexpr int VT_K = 64;       // k of one step
constexpr int VT_SIDE = VT * VT_K * 2;     // bytes of one operand's step
constexpr int VT_LDS = 2 * 2 * VT_SIDE;    // two operands, two buffers

struct VocabOperand {
    const unsigned short* p;
    long ld;     // elements from row to row
    long plane;  // elements from plane to plane
    int rows;
};

template <bool BF>
__device__ __forceinline__ vt_f4 vt_mfma(vt_u4 a, vt_u4 b, vt_f4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vt_b8, a), __builtin_bit_cast(vt_b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vt_h8, a), __builtin_bit_cast(vt_h8, b), c, 0, 0, 0);
}

// one operand's step: 128 rows from `row0` on (rows behind the last one read the last one again: their results are not used), 64 k
__device__ __forceinline__ void vt_load(const VocabOperand& o, int plane, int row0, long k0, char* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int slot = (wave * 4 + i) * 64 + lane, r = slot >> 3, c = (slot & 7) ^ ((r >> 1) & 7);
        const unsigned short* src = o.p + plane * o.plane + (long)min(row0 + r, o.rows - 1) * o.ld + k0 + c * 8;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                         (__attribute__((address_space(3))) void*)(lds + (wave * 4 + i) * 1024), 16, 0, 0);
    }
}

// the lane's 8 k (chunk) of row r
__device__ __forceinline__ vt_u4 vt_read(const char* lds, int r, int chunk) {
    return *reinterpret_cast<const vt_u4*>(lds + r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4));
}

// acc[i][j]: 16 x 16 tiles of the wave's 64 x 64 quarter; lane (n = lane & 15, g = lane >> 4), register r holds row 16 i + 4 g + r of A's
// and row 16 j + n of B's quarter.  ONES (and `sum`, of a whole wave): also sum_k A[a][k] in `ones`, a product with ones.
template <bool BF, int SEGS, bool ONES = false>
__device__ __forceinline__ void vt_product(const VocabOperand& A, const VocabOperand& B, int a0, int b0, long k0, int steps, char* lds,
                                           vt_f4 (&acc)[4][4], vt_f4 (&ones)[ONES ? 4 : 1], bool sum = false) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wa = (wave >> 1) * 64, wb = (wave & 1) * 64;
    auto load = [&](int t) {
        const int seg = SEGS == 1 ? 0 : t / steps;
        const long k = k0 + (long)(SEGS == 1 ? t : t - seg * steps) * VT_K;
        char* at = lds + (t & 1) * 2 * VT_SIDE;
        vt_load(A, SEGS > 1 && seg == 0 ? 1 : 0, a0, k, at);
        vt_load(B, SEGS > 1 && seg == 1 ? 1 : 0, b0, k, at + VT_SIDE);
    };
    const int all = SEGS * steps;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // the last reads of an earlier product are done
    if (all > 0) load(0);
    for (int t = 0; t < all; ++t) {
        // this step's tiles have arrived and the other buffer's reads are done, for every wave
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (t + 1 < all) load(t + 1);
        const char* la = lds + (t & 1) * 2 * VT_SIDE;
        const char* lb = la + VT_SIDE;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            vt_u4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = vt_read(la, wa + 16 * i + (lane & 15), kk * 4 + (lane >> 4));
                b[i] = vt_read(lb, wb + 16 * i + (lane & 15), kk * 4 + (lane >> 4));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = vt_mfma<BF>(a[i], b[j], acc[i][j]);
            if (ONES && sum && (SEGS == 1 || t < steps || t >= 2 * steps)) {  // (of two pieces each once: segment 0 has l, segment 2 h)
                const vt_u4 one = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
#pragma unroll
                for (int i = 0; i < (ONES ? 4 : 1); ++i) ones[i] = vt_mfma<BF>(a[i], one, ones[i]);
            }
        }
    }
}

template <bool BF, int SEGS>
__device__ __forceinline__ void vt_product(const VocabOperand& A, const VocabOperand& B, int a0, int b0, long k0, int steps, char* lds,
                                           vt_f4 (&acc)[4][4]) {
    vt_f4 none[1];
    vt_product<BF, SEGS, false>(A, B, a0, b0, k0, steps, lds, acc, none);
}

}  // namespace pin
