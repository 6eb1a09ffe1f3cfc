// One AdamW step over many tensors at once, moments in 32 or in 8 bits (pin_adamw_step).
//
//   t += 1;  m += (g - m) (1 - b1);  v = v b2 + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments' arithmetic is adam_elem's (pin_common.h), one rounding per operation: with weight decay 0 and fp32 moments a step
// is bit for bit pin_adam_step's, and an 8-bit code does not depend on which kernel variant wrote it.
//
// 8-bit moments: m as e4m3 (sign, 4 exponent, 3 fraction bits), v as e5m2, each with one power-of-two scale per 256 elements --
// m spans 2^-17.8 of its block's largest, v 2^-31.8 (its root, which is what divides, 2^-15.9), so |m| / sqrt(v) of an element
// that is small in its block stays bounded.  A moving average moves by (1 - b2) of itself a step, far less than half of a code's
// spacing: rounded to nearest it would never move.  Codes are therefore rounded up with the probability of the remainder, the
// dither being a hash of (seed, step, element): a step's result depends on nothing else, and a rerun gives the same bits.
// v > 0 never rounds to the code 0 (its root would divide m alone).
//
// Memory-bound: 28 bytes an element with fp32 p, g and moments, 16.06 with 8-bit moments, 10.06 with p and g in 16 bits.  One
// wave takes 256 elements (4 a lane: 16-byte loads of fp32, and the wave is the block of a scale, whose maximum is a reduction in
// registers), a workgroup CHUNK of them per round; one launch serves up to 64 tensors, whose addresses travel as
// kernel arguments -- no table to upload, nothing to keep alive, and the call can be captured.  The step count lives on the device
// (the clock, written by the last workgroup of the last launch): a captured step counts on when it is replayed.
#include "pin_common.h"

namespace pin {

constexpr int AW_BLOCK = PIN_ADAMW_BLOCK;   // elements that share a scale = elements of a wave
constexpr int AW_TENSORS = 64;              // tensors per launch: 64 x 40 bytes of arguments
constexpr int AW_UNROLL = 2;                // 256-element blocks of a wave in flight
constexpr int AW_CHUNK = 4 * AW_UNROLL * AW_BLOCK;
constexpr int AW_GRID = 2048;               // eight workgroups a compute unit, each walking its share

struct AwTensor {
    void* param;
    void* grad;
    long n;
    long offset;      // first element in the moments' layout
    float decay;      // 1 - lr wd is formed on the device (lr lives there)
    int first_chunk;  // of this launch
};
struct AwArgs {
    AwTensor t[AW_TENSORS];
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    double* clock;
    int n_tensors, n_chunks;
    float beta1, beta2, eps;
    unsigned seed;
    int advance, zero_grad;
};
static_assert(sizeof(AwArgs) <= 4096, "kernel arguments");

// dtype codes of the ABI: 0 fp32, 1 bf16, 2 fp16
template <int D> struct AwType;
template <> struct AwType<PIN_F32> { typedef float store; };
template <> struct AwType<PIN_BF16> { typedef unsigned short store; };
template <> struct AwType<PIN_F16> { typedef unsigned short store; };

template <int D>
__device__ __forceinline__ float aw_widen(typename AwType<D>::store s) {
    if constexpr (D == PIN_F32) return s;
    else if constexpr (D == PIN_BF16) return __uint_as_float((unsigned)s << 16);
    else return (float)__builtin_bit_cast(_Float16, s);
}
// round to nearest even; a NaN stays one (the integer form of the bf16 rounding would carry out of its fraction)
template <int D>
__device__ __forceinline__ typename AwType<D>::store aw_narrow(float x) {
    if constexpr (D == PIN_F32) return x;
    else if constexpr (D == PIN_BF16) return __builtin_bit_cast(unsigned short, (__bf16)x);
    else return __builtin_bit_cast(unsigned short, (_Float16)x);
}

template <int D, bool FULL>
__device__ __forceinline__ void aw_load(const void* base, long i, long n, float (&x)[4]) {
    typedef typename AwType<D>::store S;
    const S* p = reinterpret_cast<const S*>(base) + i;
    typedef S vec __attribute__((ext_vector_type(4)));
    if constexpr (FULL) {
        const vec a = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = aw_widen<D>(a[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = i + j < n ? aw_widen<D>(p[j]) : 0.f;
    }
}
template <int D, bool FULL>
__device__ __forceinline__ void aw_store(void* base, long i, long n, const float (&x)[4]) {
    typedef typename AwType<D>::store S;
    S* p = reinterpret_cast<S*>(base) + i;
    typedef S vec __attribute__((ext_vector_type(4)));
    if constexpr (FULL) {
        vec a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = aw_narrow<D>(x[j]);
        *reinterpret_cast<vec*>(p) = a;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) p[j] = aw_narrow<D>(x[j]);
    }
}

__device__ __forceinline__ unsigned aw_mixed(unsigned h) {  // two odd multipliers (the digits of the golden ratio and of e) between shifts
    h ^= h >> 16;
    h *= 0x9E3779B1u;
    h ^= h >> 15;
    h *= 0xB7E15163u;
    return h ^ (h >> 16);
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_mov_u32(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {  // the steps of wave_sum_f32
    v = max(v, dpp_mov_u32<0xB1>(v));
    v = max(v, dpp_mov_u32<0x4E>(v));
    v = max(v, dpp_mov_u32<0x141>(v));
    v = max(v, dpp_mov_u32<0x140>(v));
    return max(max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}

// The exponent of the smallest power of two >= 2^-100 that brings `largest` (the bits of a non-negative float) within
// 1.75 * 2^TOP, the largest number of the format.
template <int TOP>
__device__ __forceinline__ int aw_scale_exponent(unsigned largest) {
    const int e = (int)(largest >> 23) - 127 - TOP + ((largest & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, -100);
}
__device__ __forceinline__ float aw_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Code of |x| / 2^scale_exponent in a format of BITS fraction bits whose smallest normal is 2^LOW: n = floor(x / spacing + dither)
// spacings, and the code is the binade's first code plus n (n = 2^(BITS + 1) carries into the next binade by itself).
template <int BITS, int LOW>
__device__ __forceinline__ unsigned aw_encode(float size, float dither, unsigned largest_code) {
    const int e = max((int)(__float_as_uint(size) >> 23) - 127, LOW);
    const float n = floorf(size * aw_pow2(BITS - e) + dither);
    return min((unsigned)((e - LOW) << BITS) + (unsigned)n, largest_code);
}

template <int PD, int GD, bool EIGHT, bool FULL>
__device__ __forceinline__ void aw_block(const AwArgs& a, const AwTensor& t, long block, float lr, float lr_over_bc1, float inv_sqrt_bc2,
                                         unsigned key) {
    const int lane = threadIdx.x & 63;
    const long i = block * AW_BLOCK + 4 * lane, s = t.offset + i;
    float p[4], g[4], m[4], v[4];
    aw_load<PD, FULL>(t.param, i, t.n, p);
    aw_load<GD, FULL>(t.grad, i, t.n, g);
    if constexpr (EIGHT) {
        const unsigned mc = reinterpret_cast<const unsigned*>(a.m)[s >> 2], vc = reinterpret_cast<const unsigned*>(a.v)[s >> 2];
        const float ms = a.m_scale[s / AW_BLOCK], vs = a.v_scale[s / AW_BLOCK];
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, true);
        const auto v01 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, false), v23 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, true);
        m[0] = m01[0] * ms; m[1] = m01[1] * ms; m[2] = m23[0] * ms; m[3] = m23[1] * ms;
        v[0] = v01[0] * vs; v[1] = v01[1] * vs; v[2] = v23[0] * vs; v[3] = v23[1] * vs;
    } else {
        aw_load<PIN_F32, true>(a.m, s, 0, m);  // (the layout is padded to whole blocks: always 16 bytes)
        aw_load<PIN_F32, true>(a.v, s, 0, v);
    }
    const float keep = 1.f - lr * t.decay;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        p[j] *= keep;
        adam_elem(p[j], m[j], v[j], g[j], lr_over_bc1, inv_sqrt_bc2, a.beta1, a.beta2, a.eps);
    }
    aw_store<PD, FULL>(t.param, i, t.n, p);
    if (a.zero_grad) {
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        aw_store<GD, FULL>(t.grad, i, t.n, zero);
    }
    if constexpr (EIGHT) {
        unsigned mb[4], mm = 0, vm = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mb[j] = __float_as_uint(m[j]) & 0x7FFFFFFFu;
            mm = max(mm, mb[j]);
            vm = max(vm, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
        mm = wave_max_u32(mm);
        vm = wave_max_u32(vm);
        const int me = aw_scale_exponent<8>(mm), ve = aw_scale_exponent<15>(vm);
        const float down = aw_pow2(-me), vdown = aw_pow2(-ve);
        unsigned mc = 0, vc = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned h = aw_mixed((unsigned)(s + j) ^ key);
            const unsigned cm = aw_encode<3, -6>(__uint_as_float(mb[j]) * down, (float)(h & 0xFFFFu) * 0x1p-16f, 0x7Eu);
            unsigned cv = aw_encode<2, -14>(v[j] * vdown, (float)(h >> 16) * 0x1p-16f, 0x7Bu);
            cv = v[j] > 0.f && cv == 0 ? 1u : cv;
            mc |= (cm | (m[j] < 0.f ? 0x80u : 0u)) << (8 * j);
            vc |= cv << (8 * j);
        }
        reinterpret_cast<unsigned*>(a.m)[s >> 2] = mc;
        reinterpret_cast<unsigned*>(a.v)[s >> 2] = vc;
        if (lane == 0) {  // a moment that is not finite makes its block's scale NaN: seen by every later step, not silently coded away
            a.m_scale[s / AW_BLOCK] = mm >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : aw_pow2(me);
            a.v_scale[s / AW_BLOCK] = vm >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : aw_pow2(ve);
        }
    } else {
        aw_store<PIN_F32, true>(a.m, s, 0, m);
        aw_store<PIN_F32, true>(a.v, s, 0, v);
    }
}

template <int PD, int GD, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(AwArgs a) {
    __shared__ double sh[3];
    __shared__ unsigned sh_key;
    if (threadIdx.x == 0) {
        const double t = a.clock[0] + 1.0, p1 = a.clock[1] * (double)a.beta1, p2 = a.clock[2] * (double)a.beta2, lr = a.clock[3];
        sh[0] = lr;
        sh[1] = (double)(float)lr / (1.0 - p1);
        sh[2] = 1.0 / sqrt(1.0 - p2);
        sh_key = aw_mixed(aw_mixed(a.seed) ^ (unsigned)(unsigned long long)t);
        if (a.advance) {
            // every workgroup takes a ticket once it has read the clock; the one with the last ticket sets it and clears the counter
            unsigned long long* ticket = reinterpret_cast<unsigned long long*>(a.clock + PIN_ADAMW_CLOCK_TICKET);
            __threadfence();
            if (atomicAdd(ticket, 1ull) == (unsigned long long)gridDim.x - 1) {
                a.clock[0] = t;
                a.clock[1] = p1;
                a.clock[2] = p2;
                *ticket = 0;
            }
        }
    }
    __syncthreads();
    const float lr = (float)sh[0], lr_over_bc1 = (float)sh[1], inv_sqrt_bc2 = (float)sh[2];
    const unsigned key = sh_key;
    const int wave = threadIdx.x >> 6;
    int j = 0;
    for (int c = blockIdx.x; c < a.n_chunks; c += gridDim.x) {
        while (j + 1 < a.n_tensors && c >= a.t[j + 1].first_chunk) ++j;
        const AwTensor& t = a.t[j];
        const long base = (long)(c - t.first_chunk) * (AW_CHUNK / AW_BLOCK);
        const long blocks = (t.n + AW_BLOCK - 1) / AW_BLOCK;
        constexpr int ALIGN_P = PD == PIN_F32 ? 15 : 7, ALIGN_G = GD == PIN_F32 ? 15 : 7;
        const bool aligned = ((reinterpret_cast<uintptr_t>(t.param) & ALIGN_P) | (reinterpret_cast<uintptr_t>(t.grad) & ALIGN_G)) == 0;
        if (aligned && (base + AW_CHUNK / AW_BLOCK) * AW_BLOCK <= t.n) {
#pragma unroll
            for (int u = 0; u < AW_UNROLL; ++u)
                aw_block<PD, GD, EIGHT, true>(a, t, base + 4 * u + wave, lr, lr_over_bc1, inv_sqrt_bc2, key);
        } else {  // the tensor's last chunk, or a view that begins between 16-byte borders
            for (int u = 0; u < AW_UNROLL; ++u)
                if (base + 4 * u + wave < blocks)
                    aw_block<PD, GD, EIGHT, false>(a, t, base + 4 * u + wave, lr, lr_over_bc1, inv_sqrt_bc2, key);
        }
    }
}

template <int PD, int GD>
static void aw_launch(bool eight, int grid, hipStream_t s, const AwArgs& a) {
    if (eight) hipLaunchKernelGGL((adamw_kernel<PD, GD, true>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((adamw_kernel<PD, GD, false>), dim3(grid), dim3(256), 0, s, a);
}
template <int PD>
static void aw_launch_p(int gd, bool eight, int grid, hipStream_t s, const AwArgs& a) {
    if (gd == PIN_F32) aw_launch<PD, PIN_F32>(eight, grid, s, a);
    else if (gd == PIN_BF16) aw_launch<PD, PIN_BF16>(eight, grid, s, a);
    else aw_launch<PD, PIN_F16>(eight, grid, s, a);
}

int pin_warm_adamw() {
    hipFuncAttributes at;
    return hipFuncGetAttributes(&at, reinterpret_cast<const void*>(&adamw_kernel<PIN_F32, PIN_F32, false>)) == hipSuccess ? 0 : -1;
}
}  // namespace pin

using namespace pin;

extern "C" int pin_adamw_step(const pin_adamw_tensor* tensors_host, int32_t n_tensors, const pin_adamw_state* st, float beta1, float beta2,
                              float eps, uint32_t seed, void* stream) {
    PIN_ENTER();
    PIN_CHECK_ARG(n_tensors >= 0 && st != nullptr && (n_tensors == 0 || tensors_host != nullptr), "bad arguments");
    PIN_CHECK_ARG(st->state_bits == 32 || st->state_bits == 8, "state_bits must be 32 or 8");
    PIN_CHECK_ARG(beta1 >= 0.f && beta1 < 1.f && beta2 >= 0.f && beta2 < 1.f && eps >= 0.f, "betas must lie in [0, 1) and eps not below 0");
    PIN_CHECK_ARG(st->clock, "NULL clock");
    const bool eight = st->state_bits == 8;
    long any = 0;
    for (int j = 0; j < n_tensors; ++j) {
        const pin_adamw_tensor& t = tensors_host[j];
        PIN_CHECK_ARG(t.n >= 0 && t.offset >= 0 && t.offset % PIN_ADAMW_BLOCK == 0 && t.offset + (t.n + PIN_ADAMW_BLOCK - 1) / PIN_ADAMW_BLOCK * PIN_ADAMW_BLOCK <= st->total,
                      "a tensor lies outside the moments' layout");
        PIN_CHECK_ARG(t.n == 0 || (t.param && t.grad), "NULL tensor");
        PIN_CHECK_ARG(t.param_dtype >= PIN_F32 && t.param_dtype <= PIN_F16 && t.grad_dtype >= PIN_F32 && t.grad_dtype <= PIN_F16, "unknown dtype");
        any += t.n;
    }
    PIN_CHECK_ARG(any == 0 || (st->exp_avg && st->exp_avg_sq && (!eight || (st->exp_avg_scale && st->exp_avg_sq_scale))), "NULL moments");
    AwArgs a;
    memset(&a, 0, sizeof(a));
    a.m = st->exp_avg; a.v = st->exp_avg_sq; a.m_scale = st->exp_avg_scale; a.v_scale = st->exp_avg_sq_scale; a.clock = st->clock;
    a.zero_grad = st->zero_grad;
    a.beta1 = beta1; a.beta2 = beta2; a.eps = eps; a.seed = seed;
    // launches of up to AW_TENSORS tensors of one (parameter, gradient) type pair; the last one of the call sets the clock
    long left = 0;
    for (int j = 0; j < n_tensors; ++j) left += tensors_host[j].n > 0;
    hipStream_t s = as_stream(stream);
    if (left == 0) return fail(-1, "%s: no element to update", __func__);
    for (int pd = PIN_F32; pd <= PIN_F16; ++pd)
        for (int gd = PIN_F32; gd <= PIN_F16; ++gd) {
            long chunks = 0;
            for (int j = 0; j <= n_tensors; ++j) {
                const bool mine = j < n_tensors && tensors_host[j].n > 0 && tensors_host[j].param_dtype == pd && tensors_host[j].grad_dtype == gd;
                if (mine) {
                    const pin_adamw_tensor& t = tensors_host[j];
                    const long more = (t.n + AW_CHUNK - 1) / AW_CHUNK;
                    PIN_CHECK_ARG(chunks + more < (1l << 31), "too many elements");
                    a.t[a.n_tensors++] = AwTensor{t.param, t.grad, (long)t.n, (long)t.offset, t.weight_decay, (int)chunks};
                    chunks += more;
                    --left;
                }
                if (a.n_tensors == AW_TENSORS || (j == n_tensors && a.n_tensors > 0)) {
                    a.n_chunks = (int)chunks;
                    a.advance = left == 0;
                    const int grid = chunks < AW_GRID ? (int)chunks : AW_GRID;
                    if (pd == PIN_F32) aw_launch_p<PIN_F32>(gd, eight, grid, s, a);
                    else if (pd == PIN_BF16) aw_launch_p<PIN_BF16>(gd, eight, grid, s, a);
                    else aw_launch_p<PIN_F16>(gd, eight, grid, s, a);
                    PIN_CHECK_LAUNCH();
                    a.n_tensors = 0;
                    chunks = 0;
                }
            }
        }
    return 0;
}
