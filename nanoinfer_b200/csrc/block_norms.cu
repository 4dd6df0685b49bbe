// The norms between two sublayers in one pass over their rows: the norm on a sublayer's output y, its gate, a factor, the addition
// into the residual stream h (FP32), and the norm with which the next sublayer reads the sum:
//
//     h' = h + scale act(gate) * (y / sqrt(mean(y^2) + eps) * weight);      out = h' / sqrt(mean(h'^2) + next_eps) * gain
//
// (without `out` the second norm is left away)
//
// Bound by the bytes of the rows (8,192 rows of 4,096, y, gate and out in bfloat16: 89 us, 81 % of the copy rate); eight rows are bound
// by one row's chain of loads and sums, 3 us.  A block owns a row and keeps it in registers between the sums and the writes: every number comes
// from memory once, in 16-byte pieces of h, and all loads of a row are on their way before the first sum.
#include "common.cuh"

struct NormsArgs {
    const float* h;
    float* h_out;
    const void *y, *gate;
    void* out;
    const float *weight, *gain;
    long long ld_y, ld_gate, ld_out;
    int n_rows, width, y_type, out_type, act;          // act: 0 no gate, 1 the gate itself, 2 sigmoid, 3 silu
    float eps, next_eps, scale, share;
};
// One over the root mean square of a row's numbers; `share` is one over the width, rounded once on the host.  Where y is FP32, a step of Newton's
// behind the library's root: 0.6 x 2^-24 off as a root mean square with the product behind it, 0.73 without it and with a hardware's quotient
// (333 rows of 1,001 4.5 us, 4.4 so; 4.85 by a rounded quotient and root).  In 16 bits without: 8,192 rows of 4,096 89 us.
template <typename TY> __device__ __forceinline__ float bn_inverse(float sum, float share, float eps) {
    const float x = fmaf(sum, share, eps), r = rsqrtf(x);
    if constexpr (sizeof(TY) == 2) return r;
    const float better = fmaf(0.5f * r, fmaf(-x * r, r, 1.f), r);
    return better == better ? better : r;                  // (a sum of zero or beyond the numbers: as it is)
}

// In 16 bits 2^x and the reciprocal of the hardware (3 and |g| times 2^-24 off, where y and the gate were rounded to 2^-8); in FP32 the
// library's exponential, and the quotient put right by what it leaves (where that is no number as it is, below 1e-36 zero).
template <typename TY> __device__ __forceinline__ float bn_gate(float g, int act) {
    if (act == 1) return g;
    const float v = act == 2 ? 1.f : g;
    if constexpr (sizeof(TY) == 2) return __fdividef(v, 1.f + __expf(-g));
    const float d = 1.f + expf(-g);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    const float q = v * r, better = fmaf(fmaf(-d, q, v), r, q);
    return better == better ? better : q;
}

// Q neighbouring numbers of a row, four or one
template <int Q> __device__ __forceinline__ void bn_load(const float* p, float* v) {
    if constexpr (Q == 4) NiVec16<float>::load(p, v);
    else v[0] = *p;
}
template <int Q> __device__ __forceinline__ void bn_load(const __nv_bfloat16* p, float* v) {
    if constexpr (Q == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
    } else {
        v[0] = __bfloat162float(*p);
    }
}
template <int Q> __device__ __forceinline__ void bn_store(float* p, const float* v) {
    if constexpr (Q == 4) NiVec16<float>::store(p, v);
    else *p = v[0];
}
template <int Q> __device__ __forceinline__ void bn_store(__nv_bfloat16* p, const float* v) {
    if constexpr (Q == 4) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
        *p = __float2bfloat16_rn(v[0]);
    }
}

// Sum over the block's warps; two calls of one row use scratch of their own, so each takes one barrier.
__device__ __forceinline__ float bn_sum(float v, float* scratch) {
    v = ni_warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < (int)blockDim.x >> 5; ++w) t += scratch[w];
    return t;
}

// THREADS at most, so that BLOCKS rows share an SM: one row's sums run while another's numbers come.
template <typename TY, typename TO, int Q, int VPT, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) block_norms_row_kernel(const __grid_constant__ NormsArgs p) {
    __shared__ float scratch[2][32];
    const long long r = blockIdx.x;
    const TY* y = static_cast<const TY*>(p.y) + r * p.ld_y;
    const TY* gate = static_cast<const TY*>(p.gate) + r * p.ld_gate;
    TO* out = static_cast<TO*>(p.out) + r * p.ld_out;
    const float* h = p.h + r * p.width;
    float* h_out = p.h_out + r * p.width;
    float v[VPT][Q], s[VPT][Q], g[VPT][Q];
    const int step = blockDim.x * Q, at = threadIdx.x * Q;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (at + i * step < p.width) {
            bn_load<Q>(y + at + i * step, v[i]);
            bn_load<Q>(h + at + i * step, s[i]);
            if (p.act) bn_load<Q>(gate + at + i * step, g[i]);
        } else {
#pragma unroll
            for (int c = 0; c < Q; ++c) v[i][c] = s[i][c] = g[i][c] = 0.f;
        }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int c = 0; c < Q; ++c) ss = fmaf(v[i][c], v[i][c], ss);
    const float inv = bn_inverse<TY>(bn_sum(ss, scratch[0]), p.share, p.eps);
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (at + i * step < p.width) {
            float w[Q];
            bn_load<Q>(p.weight + at + i * step, w);
#pragma unroll
            for (int c = 0; c < Q; ++c) {
                float n = v[i][c] * inv * w[c];
                if (p.act) n *= bn_gate<TY>(g[i][c], p.act);
                s[i][c] = fmaf(p.scale, n, s[i][c]);
                ss = fmaf(s[i][c], s[i][c], ss);
            }
            bn_store<Q>(h_out + at + i * step, s[i]);
        }
    if (!p.out) return;
    const float next = bn_inverse<TY>(bn_sum(ss, scratch[1]), p.share, p.next_eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (at + i * step < p.width) {
            float w[Q], o[Q];
            bn_load<Q>(p.gain + at + i * step, w);
#pragma unroll
            for (int c = 0; c < Q; ++c) o[c] = s[i][c] * next * w[c];
            bn_store<Q>(out + at + i * step, o);
        }
}

// Rows too wide for that: what is written is read again.
template <typename TY, typename TO>
__global__ void __launch_bounds__(256) block_norms_kernel(const __grid_constant__ NormsArgs p) {
    __shared__ float scratch[2][16];
    const long long r = blockIdx.x;
    const TY* y = static_cast<const TY*>(p.y) + r * p.ld_y;
    const TY* gate = static_cast<const TY*>(p.gate) + r * p.ld_gate;
    TO* out = static_cast<TO*>(p.out) + r * p.ld_out;
    const float* h = p.h + r * p.width;
    float* h_out = p.h_out + r * p.width;
    float ss = 0.f;
    for (int i = threadIdx.x; i < p.width; i += 256) {
        const float v = ni_to_float(y[i]);
        ss = fmaf(v, v, ss);
    }
    const float inv = bn_inverse<TY>(bn_sum(ss, scratch[0]), p.share, p.eps);
    ss = 0.f;
    for (int i = threadIdx.x; i < p.width; i += 256) {
        float v = ni_to_float(y[i]) * inv * p.weight[i];
        if (p.act) v *= bn_gate<TY>(ni_to_float(gate[i]), p.act);
        v = fmaf(p.scale, v, h[i]);
        h_out[i] = v;
        ss = fmaf(v, v, ss);
    }
    if (!p.out) return;
    const float next = bn_inverse<TY>(bn_sum(ss, scratch[1]), p.share, p.next_eps);
    for (int i = threadIdx.x; i < p.width; i += 256) out[i] = ni_from_float<TO>(h_out[i] * next * p.gain[i]);
}

template <typename TY, typename TO> static void bn_launch(const NormsArgs& p, cudaStream_t stream) {
    auto apart = [&](const void* q, long long ld, int size) { return (reinterpret_cast<size_t>(q) & (4 * size - 1)) == 0 && (ld & 3) == 0; };
    const bool wide = p.width % 4 == 0 && p.width <= 16384 && apart(p.h, p.width, 4) && apart(p.h_out, p.width, 4) &&
                      apart(p.y, p.ld_y, sizeof(TY)) && (!p.out || (apart(p.out, p.ld_out, sizeof(TO)) && apart(p.gain, 0, 4))) && apart(p.weight, 0, 4) &&
                      (!p.act || apart(p.gate, p.ld_gate, sizeof(TY)));
    // A thread's Q VPT numbers: as few as possible for few rows, where a row's chain of loads and sums is the time (333 rows of
    // 1,001 in FP32: two 4.3 us, eight 6.5), eight for many, with three blocks of 512 threads on an SM: 8,192 rows of 4,096 gated
    // 89 us; sixteen with four blocks of 256 94, with three 104, four with two of 1,024 121.  Unaligned too: 4,000 rows of 2,999
    // 69 us; with one or two such blocks 104, sixteen with three of 256 115, four with two of 1,024 76.
#define BN_ROWS(Q, VPT, THREADS, BLOCKS)                                                                               \
    do {                                                                                                               \
        const int threads = ((p.width + Q * VPT - 1) / (Q * VPT) + 31) / 32 * 32;                                      \
        if (threads <= THREADS) {                                                                                      \
            block_norms_row_kernel<TY, TO, Q, VPT, THREADS, BLOCKS><<<p.n_rows, threads, 0, stream>>>(p);              \
            return;                                                                                                    \
        }                                                                                                              \
    } while (0)
    const bool few = p.n_rows <= 4 * ni_sm_count();
    if (wide) {
        if (few) BN_ROWS(4, 1, 1024, 1);
        BN_ROWS(4, 2, 512, 3);
        BN_ROWS(4, 4, 1024, 1);
    } else {
        if (few) BN_ROWS(1, 2, 1024, 1);
        BN_ROWS(1, 8, 512, 3);
        BN_ROWS(1, 8, 1024, 1);
    }
    block_norms_kernel<TY, TO><<<p.n_rows, 256, 0, stream>>>(p);
}

NI_EXPORT int ni_block_norms(const void* packed, cudaStream_t stream) {
    const NormsArgs p = *static_cast<const NormsArgs*>(packed);
    if (p.n_rows <= 0) return NI_OK;
    if (p.width <= 0 || p.act < 0 || p.act > 3) return NI_ERR_BAD_ARGUMENT;
    const bool yf = p.y_type == NI_DTYPE_F32, of = p.out_type == NI_DTYPE_F32;
    if (yf && of) bn_launch<float, float>(p, stream);
    else if (yf) bn_launch<float, __nv_bfloat16>(p, stream);
    else if (of) bn_launch<__nv_bfloat16, float>(p, stream);
    else bn_launch<__nv_bfloat16, __nv_bfloat16>(p, stream);
    NI_RETURN_LAUNCH_STATUS();
}
