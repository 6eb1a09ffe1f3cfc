// The label head over a large label set: x [n][d] rows, W [V][d] weights, b [V] biases.
//   s_iv = x_i . W_v + b_v        lse_i = log sum_v exp s_iv        nll_i = lse_i - s_i,label(i)
//   D_iv = g_i (exp(s_iv - lse_i) - [v = label(i)])     dx = D W     dW = D^T x     db = sum_i D
// (what Decoder.sem_label_prob, model/decoder.py:100-103, and the NLL term of Mapper.mapping, utils/mapper.py:782-800, do for a few labels:
// csrc/sem.h), without ever holding the n x V logits: the forward pass keeps a running maximum and sum a row, the gradient pass forms the
// logits again in pieces of the vocabulary.
//
// Numerics.  Logits are kept in units of log 2 (one fused multiply-add, and exp2 is the instruction).  bf16 / fp16 inputs multiply
// as they are, fp32 as two fp16 pieces of the value times a power of two per row (vocab_tile.h); sums, maxima and statistics are
// fp32.  D is kept in fp16 times 2^14 / 2^floor(log2 max |g|): 11 bits down to 2^-28 of the largest (rounded to bf16 it would
// cost as much error as the output's own rounding does), and the transposed x and W beside it in fp16 times a power of two of
// the tensor, which holds bf16 exactly down to 2^-31 of its largest value; fp32 again as two pieces each.
#include "vocab_tile.h"

namespace pin {

constexpr float V_LOG2E = 1.44269504088896340736f, V_LN2 = 0.69314718055994530942f;
constexpr float V_FLOOR = -1e30f;  // a maximum below every logit of a label that is not excluded (in units of log 2)
constexpr int V_AMAX = 512;        // workgroups (and partial maxima) of the first staging launch

struct VocabArgs {
    const void* x;
    const void* w;
    const void* bias;
    long ldx, ldw;
    int n, V, d;
    int dk, nk, Vk;          // padded to 64; Vk to 128
    const int* labels;
    const float* grad_nll;
    float* nll;
    float* lse;
    int* label_out;
    float* logprob;
    void* dx;
    void* dw;
    void* db;
    // workspace
    unsigned short *xa, *wa, *xt, *wt, *p, *pt;
    float *xs, *ws_, *b2;
    float *amax;             // [3][V_AMAX] partial maxima of |x|, |W|, |g|
    float *part_m, *part_s;  // [splits][nk]
    int* part_i;
    float *tlogit, *lse2, *gs;
    float* dxp;              // [dx_splits][nk][d]
    int splits, tiles_per_split, dx_splits, piece;
    int* status;
};

template <int D>
__device__ __forceinline__ float v_get(const void* p, long i) {
    if constexpr (D == PIN_F32) return reinterpret_cast<const float*>(p)[i];
    else if constexpr (D == PIN_BF16) return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
    else return (float)reinterpret_cast<const _Float16*>(p)[i];
}
template <int D>
__device__ __forceinline__ void v_put(void* p, long i, float x) {
    if constexpr (D == PIN_F32) reinterpret_cast<float*>(p)[i] = x;
    else if constexpr (D == PIN_BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)x;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
}
__device__ __forceinline__ unsigned short v_half(float x) { return __builtin_bit_cast(unsigned short, (_Float16)x); }
__device__ __forceinline__ float v_from_half(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
// e with |x| 2^e in [2^14, 2^15); 0 where there is nothing to scale or nothing finite
__device__ __forceinline__ int v_scale_exp(float amax) {
    const unsigned b = __float_as_uint(amax) & 0x7FFFFFFFu;
    if (b == 0 || b >= 0x7F800000u) return 0;
    int e;
    frexpf(amax, &e);
    return 15 - e;
}
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ float v_block_max(const float* part, float* sh) {  // the maximum of V_AMAX partial maxima, in every thread of 256
    float m = fmaxf(part[threadIdx.x], part[threadIdx.x + 256]);
    m = wave_max_f32(m);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
    __syncthreads();
    return m;
}

__device__ __forceinline__ bool v_takes_part(const VocabArgs& a, long row) { return a.labels[row] >= 0 && a.labels[row] < a.V; }

// Staging, first launch: one wave a row.  The largest |x|, |W|, |g|; the padded bias in units of log 2 (-inf: excluded, and behind the
// last label); COPY: the operand of the logit product (two scaled fp16 pieces of fp32; a padded copy of rows that are not aligned).
template <int D, bool COPY>
__global__ __launch_bounds__(256) void vocab_rows_kernel(VocabArgs a, int scan) {  // scan: the rows are needed at all (maxima or copies)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float mx = 0.f, mw = 0.f, mg = 0.f;
    for (long r = scan ? (long)blockIdx.x * 4 + wave : (long)a.n + a.V; r < (long)a.n + a.V; r += (long)gridDim.x * 4) {
        const bool is_x = r < a.n;
        const long row = is_x ? r : r - a.n;
        const void* src = is_x ? a.x : a.w;
        const long at = row * (is_x ? a.ldx : a.ldw);
        float m = 0.f;
        for (int k = lane; k < a.d; k += 64) m = fmaxf(m, fabsf(v_get<D>(src, at + k)));
        if constexpr (COPY) {
            unsigned short* out = (is_x ? a.xa : a.wa) + row * a.dk;
            const long plane = (long)(is_x ? a.n : a.V) * a.dk;
            if constexpr (D == PIN_F32) {
                const int e = v_scale_exp(wave_max_f32(m));
                for (int k = lane; k < a.dk; k += 64) {
                    const float v = k < a.d ? ldexpf(v_get<D>(src, at + k), e) : 0.f;
                    const unsigned short h = v_half(v);
                    out[k] = h;
                    out[plane + k] = v_half(v - v_from_half(h));
                }
                if (lane == 0) (is_x ? a.xs : a.ws_)[row] = ldexpf(is_x ? 1.f : V_LOG2E, -e);
            } else {
                for (int k = lane; k < a.dk; k += 64) out[k] = k < a.d ? reinterpret_cast<const unsigned short*>(src)[at + k] : (unsigned short)0;
            }
        }
        if (!is_x) mw = fmaxf(mw, m);
        else if (a.labels == nullptr || v_takes_part(a, row)) mx = fmaxf(mx, m);
    }
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < a.Vk; i += (long)gridDim.x * 256) {
        const float b = i >= a.V ? -INFINITY : a.bias == nullptr ? 0.f : v_get<D>(a.bias, i);
        a.b2[i] = b <= V_FLOOR ? -INFINITY : b * V_LOG2E;
    }
    if (a.grad_nll != nullptr)
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < a.n; i += (long)gridDim.x * 256)
            if (v_takes_part(a, i)) mg = fmaxf(mg, fabsf(a.grad_nll[i]));
    __shared__ float sh[3][4];
    mx = wave_max_f32(mx); mw = wave_max_f32(mw); mg = wave_max_f32(mg);
    if (lane == 0) { sh[0][wave] = mx; sh[1][wave] = mw; sh[2][wave] = mg; }
    __syncthreads();
    if (threadIdx.x < 3) {
        const float* s = sh[threadIdx.x];
        a.amax[threadIdx.x * V_AMAX + blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    }
}

// Staging, second launch: x^T [d][nk] and W^T [d][Vk] in fp16 (two pieces of fp32), times the tensor's power of two (fp16 as it is).
// 64 x 64 tiles through LDS; columns behind the last row are zero, and so are rows of x without a label (what they hold must not
// meet the zeros of D).
template <int D>
__global__ __launch_bounds__(256) void vocab_transpose_kernel(VocabArgs a, int x_tiles) {
    __shared__ float sh[4];
    __shared__ float tile[64][65];
    const bool is_x = (int)blockIdx.x < x_tiles;
    const float amax = v_block_max(a.amax + (is_x ? 0 : V_AMAX), sh);
    const int e = D == PIN_F16 ? 0 : v_scale_exp(amax);
    const int r0 = ((int)blockIdx.x - (is_x ? 0 : x_tiles)) * 64, k0 = blockIdx.y * 64;
    const int rows = is_x ? a.n : a.V, padded = is_x ? a.nk : a.Vk;
    const void* src = is_x ? a.x : a.w;
    const long ld = is_x ? a.ldx : a.ldw;
    for (int i = threadIdx.x; i < 4096; i += 256) {
        const int r = i >> 6, k = i & 63;
        tile[r][k] = r0 + r < rows && k0 + k < a.d && (!is_x || v_takes_part(a, r0 + r)) ? v_get<D>(src, (r0 + r) * ld + k0 + k) : 0.f;
    }
    __syncthreads();
    unsigned short* out = is_x ? a.xt : a.wt;
    const long plane = (long)a.d * padded;
    for (int i = threadIdx.x; i < 4096; i += 256) {
        const int k = i >> 6, r = i & 63;
        if (k0 + k >= a.d) continue;
        const float v = ldexpf(tile[r][k], e);
        const unsigned short h = v_half(v);
        const long at = (long)(k0 + k) * padded + r0 + r;
        out[at] = h;
        if constexpr (D == PIN_F32) out[plane + at] = v_half(v - v_from_half(h));
    }
}

// one logit in units of log 2: acc = W_v . x_i (times the two rows' powers of two for fp32)
template <int SEGS>
__device__ __forceinline__ float v_logit(float acc, float xs, float ws, float b2) {
    if constexpr (SEGS == 1) return fmaf(acc, V_LOG2E, b2);
    else return fmaf(acc, xs * ws, b2);
}

// the wave's 64 labels x 64 rows of logits: acc -> units of log 2
template <int SEGS>
__device__ __forceinline__ void v_logits(const VocabArgs& a, vt_f4 (&acc)[4][4], int v0, int i0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int vb = v0 + (wave >> 1) * 64 + 4 * g, ib = i0 + (wave & 1) * 64 + c;
    float xs[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) xs[j] = SEGS == 1 ? 1.f : a.xs[min(ib + 16 * j, a.n - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const vt_f4 b2 = *reinterpret_cast<const vt_f4*>(a.b2 + vb + 16 * i);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float ws = SEGS == 1 ? 1.f : a.ws_[min(vb + 16 * i + r, a.V - 1)];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j][r] = v_logit<SEGS>(acc[i][j][r], xs[j], ws, b2[r]);
        }
    }
}

__device__ __forceinline__ VocabOperand v_operand_w(const VocabArgs& a) {
    return a.wa != nullptr ? VocabOperand{a.wa, a.dk, (long)a.V * a.dk, a.V} : VocabOperand{reinterpret_cast<const unsigned short*>(a.w), a.ldw, 0, a.V};
}
__device__ __forceinline__ VocabOperand v_operand_x(const VocabArgs& a) {
    return a.xa != nullptr ? VocabOperand{a.xa, a.dk, (long)a.n * a.dk, a.n} : VocabOperand{reinterpret_cast<const unsigned short*>(a.x), a.ldx, 0, a.n};
}

// Forward: workgroup (row tile, split of the vocabulary).  A lane keeps (maximum, sum, lowest label of the maximum) of its 4 rows
// over the labels it sees; they are joined over the lanes, the waves and (vocab_finish_kernel) the splits.
template <bool BF, int SEGS, bool ARG>
__global__ __launch_bounds__(256, 2) void vocab_forward_kernel(VocabArgs a) {
    extern __shared__ __attribute__((aligned(16))) char vlds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int i0 = blockIdx.x * VT, ib = i0 + (wave & 1) * 64 + c;
    float m[4], s[4];
    int arg[4], lab[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        m[j] = V_FLOOR; s[j] = 0.f; arg[j] = 0x7FFFFFFF;
        lab[j] = !ARG && ib + 16 * j < a.n ? a.labels[ib + 16 * j] : -1;
    }
    const VocabOperand W = v_operand_w(a), X = v_operand_x(a);
    const int t0 = blockIdx.y * a.tiles_per_split, t1 = min(t0 + a.tiles_per_split, a.Vk / VT);
    for (int t = t0; t < t1; ++t) {
        const int v0 = t * VT;
        vt_f4 acc[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = vt_f4{0.f, 0.f, 0.f, 0.f};
        vt_product<BF, SEGS>(W, X, v0, i0, 0, a.dk / VT_K, vlds, acc);
        v_logits<SEGS>(a, acc, v0, i0);
        const int vb = v0 + (wave >> 1) * 64 + 4 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float top = m[j];
            if constexpr (ARG) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (acc[i][j][r] > top) { top = acc[i][j][r]; arg[j] = vb + 16 * i + r; }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
                const int at = lab[j] - (v0 + (wave >> 1) * 64);
                if (__any(lab[j] >= 0 && at >= 0 && at < 64)) {  // (the label of one of the wave's rows is among these)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (lab[j] >= 0 && lab[j] == vb + 16 * i + r) a.tlogit[ib + 16 * j] = acc[i][j][r];
                }
            }
            float sum = s[j] * exp2f(m[j] - top);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f(acc[i][j][r] - top);
            m[j] = top;
            s[j] = sum;
        }
    }
    // join: lanes g (labels 4 g ..), then the two waves of the same rows
    __syncthreads();
    float* sh = reinterpret_cast<float*>(vlds);
    auto join = [](float& m1, float& s1, int& a1, float m2, float s2, int a2) {
        const float top = fmaxf(m1, m2);
        s1 = s1 * exp2f(m1 - top) + s2 * exp2f(m2 - top);
        a1 = m1 > m2 ? a1 : m2 > m1 ? a2 : min(a1, a2);
        m1 = top;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1) {
            const float m2 = __shfl_xor(m[j], o, 64), s2 = __shfl_xor(s[j], o, 64);
            const int a2 = __shfl_xor(arg[j], o, 64);
            join(m[j], s[j], arg[j], m2, s2, a2);
        }
        if (wave >= 2 && g == 0) {
            const int at = (wave & 1) * 64 + 16 * j + c;
            sh[at] = m[j];
            sh[VT + at] = s[j];
            reinterpret_cast<int*>(sh)[2 * VT + at] = arg[j];
        }
    }
    __syncthreads();
    if (wave < 2 && g == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = wave * 64 + 16 * j + c;
            join(m[j], s[j], arg[j], sh[at], sh[VT + at], reinterpret_cast<int*>(sh)[2 * VT + at]);
            if (i0 + at < a.n) {
                const long o = (long)blockIdx.y * a.nk + i0 + at;
                a.part_m[o] = m[j];
                a.part_s[o] = s[j];
                if constexpr (ARG) a.part_i[o] = arg[j];
            }
        }
    }
}

// what the gradient pass reads of a row: lse in units of log 2 and the scaled upstream gradient (0: the row takes no part)
__device__ __forceinline__ void v_row_of_gradient(const VocabArgs& a, int i, int label, float lse, float gmax) {
    const bool none = i >= a.n || label < 0 || label >= a.V || lse == -INFINITY;
    a.lse2[i] = none ? 0.f : lse * V_LOG2E;
    a.gs[i] = none ? 0.f : isnan(lse) ? NAN : ldexpf(a.grad_nll[i], v_scale_exp(gmax));
}

template <bool ARG, bool GRAD>
__global__ __launch_bounds__(256) void vocab_finish_kernel(VocabArgs a) {
    __shared__ float sh[4];
    float gmax = 0.f;
    if constexpr (GRAD) gmax = v_block_max(a.amax + 2 * V_AMAX, sh);
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.nk) return;
    float m = V_FLOOR, s = 0.f;
    int arg = 0x7FFFFFFF;
    if (i < a.n)
        for (int p = 0; p < a.splits; ++p) {
            const float m2 = a.part_m[(long)p * a.nk + i], s2 = a.part_s[(long)p * a.nk + i], top = fmaxf(m, m2);
            s = s * exp2f(m - top) + s2 * exp2f(m2 - top);
            if constexpr (ARG) {
                const int a2 = a.part_i[(long)p * a.nk + i];
                arg = m > m2 ? arg : m2 > m ? a2 : min(arg, a2);
            }
            m = top;
        }
    if constexpr (ARG) {
        if (i < a.n) {
            const float rest = -log2f(s) * V_LN2;  // s = 1 + the others
            const bool fine = s > 0.f && s < INFINITY;
            a.label_out[i] = fine ? arg : -1;
            a.logprob[i] = s == 0.f ? -INFINITY : fine ? rest : NAN;
        }
    } else {
        const float lse = s == 0.f ? -INFINITY : (m + log2f(s)) * V_LN2;
        const int label = i < a.n ? a.labels[i] : -1;
        if (i < a.n) {
            a.lse[i] = lse;
            float nll = 0.f;
            if (label >= a.V) {
                nll = NAN;
                atomicOr(a.status, PIN_STATUS_LABEL_RANGE);
            } else if (label >= 0) {
                nll = s == 0.f ? INFINITY : (m - a.tlogit[i] + log2f(s)) * V_LN2;
            }
            a.nll[i] = nll;
        }
        if constexpr (GRAD) v_row_of_gradient(a, i, label, lse, gmax);
    }
}

__global__ __launch_bounds__(256) void vocab_prepare_kernel(VocabArgs a) {  // the gradient pass alone, with the lse of an earlier call
    __shared__ float sh[4];
    const float gmax = v_block_max(a.amax + 2 * V_AMAX, sh);
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.nk) return;
    const int label = i < a.n ? a.labels[i] : -1;
    if (label >= a.V) atomicOr(a.status, PIN_STATUS_LABEL_RANGE);
    v_row_of_gradient(a, i, label, i < a.n ? a.lse[i] : 0.f, gmax);
}

// D of one piece of the vocabulary: the logits again, D [n][piece] and D^T [piece][n] in fp16 (two pieces of fp32)
template <bool BF, int SEGS>
__global__ __launch_bounds__(256, 2) void vocab_probs_kernel(VocabArgs a, int p0) {
    extern __shared__ __attribute__((aligned(16))) char vlds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int i0 = blockIdx.x * VT, v0 = p0 + blockIdx.y * VT;
    vt_f4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = vt_f4{0.f, 0.f, 0.f, 0.f};
    vt_product<BF, SEGS>(v_operand_w(a), v_operand_x(a), v0, i0, 0, a.dk / VT_K, vlds, acc);
    v_logits<SEGS>(a, acc, v0, i0);
    const int vb = v0 + (wave >> 1) * 64 + 4 * g, ib = i0 + (wave & 1) * 64 + c;
    const long plane = (long)a.nk * a.piece;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = ib + 16 * j;
        if (row >= a.nk) continue;
        const float lse2 = a.lse2[row], gs = a.gs[row];
        const int lab = gs == 0.f ? -1 : a.labels[row];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned short h[4], l[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float p = __builtin_amdgcn_exp2f(acc[i][j][r] - lse2);
                p = (lab == vb + 16 * i + r ? p - 1.f : p) * gs;
                p = gs == 0.f ? 0.f : p;
                h[r] = v_half(p);
                l[r] = SEGS == 1 ? 0 : v_half(p - v_from_half(h[r]));
                const long at = (long)(vb + 16 * i + r - p0) * a.nk + row;
                a.pt[at] = h[r];
                if constexpr (SEGS > 1) a.pt[plane + at] = l[r];
            }
            const long at = (long)row * a.piece + vb + 16 * i - p0;
            *reinterpret_cast<uint2*>(a.p + at) = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
            if constexpr (SEGS > 1)
                *reinterpret_cast<uint2*>(a.p + plane + at) = make_uint2(l[0] | (unsigned)l[1] << 16, l[2] | (unsigned)l[3] << 16);
        }
    }
}

// dx += D W over one piece: partial sums [split][n][d], a split of the piece's labels each
template <int SEGS>
__global__ __launch_bounds__(256, 2) void vocab_dx_kernel(VocabArgs a, int p0, int width) {
    extern __shared__ __attribute__((aligned(16))) char vlds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int i0 = blockIdx.x * VT, k0 = blockIdx.y * VT;
    const int steps = width / VT_K, per = (steps + a.dx_splits - 1) / a.dx_splits, s0 = min((int)blockIdx.z * per, steps), s1 = min(s0 + per, steps);
    const VocabOperand P{a.p, a.piece, (long)a.nk * a.piece, a.nk}, WT{a.wt + p0, a.Vk, (long)a.d * a.Vk, a.d};
    vt_f4 acc[4][4];
    float* out = a.dxp + (long)blockIdx.z * a.nk * a.d;
    const int ib = i0 + (wave >> 1) * 64 + 4 * g, kb = k0 + (wave & 1) * 64 + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                acc[i][j][r] = p0 > 0 && ib + 16 * i + r < a.n && kb + 16 * j < a.d ? out[(long)(ib + 16 * i + r) * a.d + kb + 16 * j] : 0.f;
    vt_product<false, SEGS>(P, WT, i0, k0, (long)s0 * VT_K, s1 - s0, vlds, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (ib + 16 * i + r < a.n && kb + 16 * j < a.d) out[(long)(ib + 16 * i + r) * a.d + kb + 16 * j] = acc[i][j][r];
}

// dW and db of one piece
template <int D, int SEGS>
__global__ __launch_bounds__(256, 2) void vocab_dw_kernel(VocabArgs a, int p0) {
    extern __shared__ __attribute__((aligned(16))) char vlds[];
    __shared__ float sh[4];
    const float gmax = v_block_max(a.amax + 2 * V_AMAX, sh), xmax = v_block_max(a.amax, sh);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int v0 = blockIdx.x * VT, k0 = blockIdx.y * VT;
    const VocabOperand PT{a.pt, a.nk, (long)a.nk * a.piece, a.piece}, XT{a.xt, a.nk, (long)a.d * a.nk, a.d};
    vt_f4 acc[4][4], ones[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ones[i] = vt_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = vt_f4{0.f, 0.f, 0.f, 0.f};
    }
    const bool bias = a.db != nullptr && k0 == 0 && (wave & 1) == 0;
    vt_product<false, SEGS, true>(PT, XT, v0, k0, 0, a.nk / VT_K, vlds, acc, ones, bias);
    const int eg = v_scale_exp(gmax), e = eg + (D == PIN_F16 ? 0 : v_scale_exp(xmax));
    const int vb = p0 + v0 + (wave >> 1) * 64 + 4 * g, kb = k0 + (wave & 1) * 64 + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int v = vb + 16 * i + r;
            if (v >= a.V) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (kb + 16 * j < a.d) v_put<D>(a.dw, (long)v * a.d + kb + 16 * j, ldexpf(acc[i][j][r], -e));
            if (bias && c == 0) v_put<D>(a.db, v, ldexpf(ones[i][r], -eg));
        }
}

template <int D>
__global__ __launch_bounds__(256) void vocab_dx_finish_kernel(VocabArgs a) {
    __shared__ float sh[4];
    const float gmax = v_block_max(a.amax + 2 * V_AMAX, sh), wmax = v_block_max(a.amax + V_AMAX, sh);
    const int e = v_scale_exp(gmax) + (D == PIN_F16 ? 0 : v_scale_exp(wmax));
    const long all = (long)a.n * a.d;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < a.dx_splits; ++p) s += a.dxp[(long)p * a.nk * a.d + i];
        v_put<D>(a.dx, i, ldexpf(s, -e));
    }
}

template <int D>
__global__ __launch_bounds__(256) void vocab_no_rows_kernel(VocabArgs a) {  // n = 0: the gradients of W and b are zero
    const long all = (long)a.V * a.d;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) v_put<D>(a.dw, i, 0.f);
    if (a.db != nullptr)
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < a.V; i += (long)gridDim.x * 256) v_put<D>(a.db, i, 0.f);
}

int pin_warm_vocab() {
    hipFuncAttributes at;
    return hipFuncGetAttributes(&at, reinterpret_cast<const void*>(&vocab_prepare_kernel)) == hipSuccess ? 0 : -1;
}

// ---------------------------------------------------------------------------------------------------- host
enum { V_PREDICT = 0, V_NLL = 1, V_GRAD = 2, V_STEP = 3 };

struct VocabPlan {
    VocabArgs a;
    int dtype, segs;
    bool copy;
    long bytes;
};

static long v_up(long v, long m) { return (v + m - 1) / m * m; }

static VocabPlan v_plan(const pin_vocab_head* h, int mode, char* base) {
    VocabPlan p;
    memset(&p, 0, sizeof(p));
    VocabArgs& a = p.a;
    a.n = h->n; a.V = h->vocab; a.d = h->dim;
    a.x = h->x; a.w = h->weight; a.bias = h->bias; a.ldx = h->x_stride; a.ldw = h->weight_stride;
    a.dk = (int)v_up(a.d, VT_K); a.nk = (int)v_up(a.n > 0 ? a.n : 1, VT); a.Vk = (int)v_up(a.V, VT);
    p.dtype = h->dtype;
    p.segs = h->dtype == PIN_F32 ? 3 : 1;
    const int planes = p.segs == 1 ? 1 : 2;
    // 16-bit rows that begin and end on 16-byte borders are read where they are
    p.copy = p.segs > 1 || a.d % VT_K != 0 || a.ldx % 8 != 0 || a.ldw % 8 != 0 || ((uintptr_t)a.x | (uintptr_t)a.w) % 16 != 0;
    const int rows = a.nk / VT, tiles = a.Vk / VT;
    // forward: enough workgroups to fill the card twice over
    a.splits = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    if (a.splits > tiles) a.splits = tiles;
    a.tiles_per_split = (tiles + a.splits - 1) / a.splits;
    a.splits = (tiles + a.tiles_per_split - 1) / a.tiles_per_split;
    // gradient: pieces whose D and D^T take about 256 MB together
    long piece = (128l << 20) / (2l * planes * a.nk) / VT * VT;
    if (piece < VT) piece = VT;
    if (piece > a.Vk) piece = a.Vk;
    a.piece = (int)piece;
    const int dx_tiles = rows * (int)((a.d + VT - 1) / VT);
    a.dx_splits = dx_tiles >= 512 ? 1 : (512 + dx_tiles - 1) / dx_tiles;
    if (a.dx_splits > 16) a.dx_splits = 16;
    long at = 0;
    auto take = [&](long bytes) {
        char* q = base + at;
        at += v_up(bytes, 256);
        return q;
    };
    a.amax = (float*)take(3 * V_AMAX * 4);
    a.b2 = (float*)take((long)a.Vk * 4);
    if (p.copy) {
        a.xa = (unsigned short*)take((long)planes * a.n * a.dk * 2);
        a.wa = (unsigned short*)take((long)planes * a.V * a.dk * 2);
        if (p.segs > 1) {
            a.xs = (float*)take((long)a.n * 4);
            a.ws_ = (float*)take((long)a.V * 4);
        }
    }
    if (mode != V_GRAD) {
        a.part_m = (float*)take((long)a.splits * a.nk * 4);
        a.part_s = (float*)take((long)a.splits * a.nk * 4);
        if (mode == V_PREDICT) a.part_i = (int*)take((long)a.splits * a.nk * 4);
        else a.tlogit = (float*)take((long)a.nk * 4);
    }
    if (mode == V_GRAD || mode == V_STEP) {
        a.xt = (unsigned short*)take((long)planes * a.d * a.nk * 2);
        a.wt = (unsigned short*)take((long)planes * a.d * a.Vk * 2);
        a.lse2 = (float*)take((long)a.nk * 4);
        a.gs = (float*)take((long)a.nk * 4);
        a.p = (unsigned short*)take((long)planes * a.nk * a.piece * 2);
        a.pt = (unsigned short*)take((long)planes * a.nk * a.piece * 2);
        a.dxp = (float*)take((long)a.dx_splits * a.nk * a.d * 4);
    }
    p.bytes = at;
    return p;
}

static int v_check(const pin_vocab_head* h) {
    PIN_CHECK_ARG(h != nullptr, "NULL head");
    PIN_CHECK_ARG(h->n >= 0 && h->vocab >= 1 && h->dim >= 1, "n >= 0, vocab >= 1 and dim >= 1 are needed");
    PIN_CHECK_ARG(h->n <= PIN_VOCAB_MAX && h->vocab <= PIN_VOCAB_MAX && h->dim <= PIN_VOCAB_MAX_DIM, "a size is over PIN_VOCAB_MAX / PIN_VOCAB_MAX_DIM");
    PIN_CHECK_ARG(h->dtype >= PIN_F32 && h->dtype <= PIN_F16, "unknown dtype");
    PIN_CHECK_ARG(h->weight && (h->n == 0 || h->x), "NULL tensor");
    PIN_CHECK_ARG(h->weight_stride >= h->dim && (h->n == 0 || h->x_stride >= h->dim), "a row's stride is below dim");
    return 0;
}

// more than 64 KB of LDS has to be asked for, once per kernel
template <typename F>
static int v_reserve(F* kernel, int bytes) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == hipSuccess ? 0 : fail(-2, "label head: cannot reserve %d bytes of LDS: %s", bytes, hipGetErrorString(e));
}
#define V_RESERVE(kernel)                                      \
    do {                                                       \
        static const int reserved = v_reserve(kernel, VT_LDS); \
        if (reserved != 0) return reserved;                    \
    } while (0)
#define V_LAUNCH(kernel, grid, lds, ...) hipLaunchKernelGGL(kernel, grid, dim3(256), lds, s, __VA_ARGS__)

template <int D>
static void v_stage(const VocabPlan& p, bool transposed, hipStream_t s) {
    const VocabArgs& a = p.a;
    if (p.copy) V_LAUNCH((vocab_rows_kernel<D, true>), dim3(V_AMAX), 0, a, 1);
    else if constexpr (D != PIN_F32) V_LAUNCH((vocab_rows_kernel<D, false>), dim3(V_AMAX), 0, a, transposed && D == PIN_BF16 ? 1 : 0);
    if (transposed) V_LAUNCH((vocab_transpose_kernel<D>), dim3(a.nk / 64 + a.Vk / 64, a.dk / 64), 0, a, a.nk / 64);
}

template <bool BF, int SEGS>
static int v_forward(const VocabPlan& p, int mode, hipStream_t s) {
    const VocabArgs& a = p.a;
    const dim3 grid(a.nk / VT, a.splits);
    V_RESERVE((&vocab_forward_kernel<BF, SEGS, true>));
    V_RESERVE((&vocab_forward_kernel<BF, SEGS, false>));
    if (mode == V_PREDICT) V_LAUNCH((vocab_forward_kernel<BF, SEGS, true>), grid, VT_LDS, a);
    else V_LAUNCH((vocab_forward_kernel<BF, SEGS, false>), grid, VT_LDS, a);
    const dim3 fin(cdiv(a.nk, 256));
    if (mode == V_PREDICT) V_LAUNCH((vocab_finish_kernel<true, false>), fin, 0, a);
    else if (mode == V_NLL) V_LAUNCH((vocab_finish_kernel<false, false>), fin, 0, a);
    else V_LAUNCH((vocab_finish_kernel<false, true>), fin, 0, a);
    return 0;
}

template <int D, bool BF, int SEGS>
static int v_gradient(const VocabPlan& p, hipStream_t s) {
    const VocabArgs& a = p.a;
    const int kt = cdiv(a.d, VT);
    V_RESERVE((&vocab_probs_kernel<BF, SEGS>));
    V_RESERVE((&vocab_dx_kernel<SEGS>));
    V_RESERVE((&vocab_dw_kernel<D, SEGS>));
    for (int p0 = 0; p0 < a.Vk; p0 += a.piece) {
        const int width = p0 + a.piece < a.Vk ? a.piece : a.Vk - p0;
        V_LAUNCH((vocab_probs_kernel<BF, SEGS>), dim3(a.nk / VT, width / VT), VT_LDS, a, p0);
        V_LAUNCH((vocab_dx_kernel<SEGS>), dim3(a.nk / VT, kt, a.dx_splits), VT_LDS, a, p0, width);
        V_LAUNCH((vocab_dw_kernel<D, SEGS>), dim3(width / VT, kt), VT_LDS, a, p0);
    }
    const long all = (long)a.n * a.d;
    V_LAUNCH((vocab_dx_finish_kernel<D>), dim3(all < 1024 * 256 ? cdiv(all, 256) : 1024), 0, a);
    return 0;
}

static int v_run(const pin_vocab_head* h, int mode, const int32_t* labels, const float* grad_nll, float* nll, float* lse, int32_t* label_out,
                 float* logprob, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes, void* stream) {
    hipStream_t s = as_stream(stream);
    const bool grads = mode == V_GRAD || mode == V_STEP;
    VocabPlan p = v_plan(h, mode, (char*)workspace);
    VocabArgs& a = p.a;
    a.labels = labels; a.grad_nll = grads ? grad_nll : nullptr; a.nll = nll; a.lse = lse; a.label_out = label_out; a.logprob = logprob;
    a.dx = dx; a.dw = dw; a.db = db;
    if (a.n == 0) {
        if (grads) {
            if (p.dtype == PIN_F32) V_LAUNCH((vocab_no_rows_kernel<PIN_F32>), dim3(1024), 0, a);
            else if (p.dtype == PIN_BF16) V_LAUNCH((vocab_no_rows_kernel<PIN_BF16>), dim3(1024), 0, a);
            else V_LAUNCH((vocab_no_rows_kernel<PIN_F16>), dim3(1024), 0, a);
            PIN_CHECK_LAUNCH();
        }
        return 0;
    }
    PIN_CHECK_ARG(workspace != nullptr && ((uintptr_t)workspace & 255) == 0, "the workspace must begin at a multiple of 256 bytes");
    PIN_CHECK_ARG(workspace_bytes >= p.bytes, "workspace too small (pin_vocab_workspace_bytes)");
    a.status = status_word();
    if (a.status == nullptr) return fail(-2, "%s: no status word on this device", __func__);
    if (p.dtype == PIN_F32) v_stage<PIN_F32>(p, grads, s);
    else if (p.dtype == PIN_BF16) v_stage<PIN_BF16>(p, grads, s);
    else v_stage<PIN_F16>(p, grads, s);
    PIN_CHECK_LAUNCH();
    if (mode != V_GRAD) {
        const int e = p.dtype == PIN_F32 ? v_forward<false, 3>(p, mode, s) : p.dtype == PIN_BF16 ? v_forward<true, 1>(p, mode, s) : v_forward<false, 1>(p, mode, s);
        if (e != 0) return e;
    } else {
        V_LAUNCH(vocab_prepare_kernel, dim3(cdiv(a.nk, 256)), 0, a);
    }
    PIN_CHECK_LAUNCH();
    if (grads) {
        const int e = p.dtype == PIN_F32 ? v_gradient<PIN_F32, false, 3>(p, s)
                      : p.dtype == PIN_BF16 ? v_gradient<PIN_BF16, true, 1>(p, s) : v_gradient<PIN_F16, false, 1>(p, s);
        if (e != 0) return e;
        PIN_CHECK_LAUNCH();
    }
    return 0;
}
}  // namespace pin

using namespace pin;

extern "C" int64_t pin_vocab_workspace_bytes(int32_t n, int32_t vocab, int32_t dim, int32_t dtype, int32_t gradients) {
    pin_vocab_head h;
    memset(&h, 0, sizeof(h));
    h.n = n; h.vocab = vocab; h.dim = dim; h.dtype = dtype;
    h.x_stride = h.weight_stride = dim | 1;  // (the larger of the two forms: rows that have to be copied)
    if (n < 0 || vocab < 1 || dim < 1 || n > PIN_VOCAB_MAX || vocab > PIN_VOCAB_MAX || dim > PIN_VOCAB_MAX_DIM || dtype < PIN_F32 || dtype > PIN_F16) return -1;
    const long f = v_plan(&h, gradients ? V_STEP : V_PREDICT, nullptr).bytes, g = v_plan(&h, gradients ? V_STEP : V_NLL, nullptr).bytes;
    return f > g ? f : g;
}

extern "C" int pin_vocab_nll(const pin_vocab_head* h, const int32_t* labels, float* nll_out, float* lse_out, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    PIN_ENTER();
    if (int e = v_check(h)) return e;
    PIN_CHECK_ARG(h->n == 0 || (labels && nll_out && lse_out), "NULL pointer");
    return v_run(h, V_NLL, labels, nullptr, nll_out, lse_out, nullptr, nullptr, nullptr, nullptr, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int pin_vocab_nll_grad(const pin_vocab_head* h, const int32_t* labels, const float* lse, const float* grad_nll, void* dx, void* dweight,
                                  void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
    PIN_ENTER();
    if (int e = v_check(h)) return e;
    PIN_CHECK_ARG(dweight && (h->n == 0 || (labels && lse && grad_nll && dx)), "NULL pointer");
    return v_run(h, V_GRAD, labels, grad_nll, nullptr, const_cast<float*>(lse), nullptr, nullptr, dx, dweight, dbias, workspace, workspace_bytes, stream);
}

extern "C" int pin_vocab_nll_step(const pin_vocab_head* h, const int32_t* labels, const float* grad_nll, float* nll_out, float* lse_out, void* dx,
                                  void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
    PIN_ENTER();
    if (int e = v_check(h)) return e;
    PIN_CHECK_ARG(dweight && (h->n == 0 || (labels && grad_nll && nll_out && lse_out && dx)), "NULL pointer");
    return v_run(h, V_STEP, labels, grad_nll, nll_out, lse_out, nullptr, nullptr, dx, dweight, dbias, workspace, workspace_bytes, stream);
}

extern "C" int pin_vocab_predict(const pin_vocab_head* h, int32_t* label_out, float* logprob_out, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    PIN_ENTER();
    if (int e = v_check(h)) return e;
    PIN_CHECK_ARG(h->n == 0 || (label_out && logprob_out), "NULL pointer");
    return v_run(h, V_PREDICT, nullptr, nullptr, nullptr, nullptr, label_out, logprob_out, nullptr, nullptr, nullptr, workspace, workspace_bytes, stream);
}
