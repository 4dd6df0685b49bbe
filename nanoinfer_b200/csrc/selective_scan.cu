// The scan of a selective state space layer.  Per request and channel d, with a state h [N] in FP32 kept from call to call:
//
//     delta = softplus(dt[t, d] + dt_bias[d])
//     h_n <- exp(delta A[d, n]) h_n + delta u[t, d] B[t, g, n]            g = d / (D / groups)
//     out[t, d] = (sum_n h_n C[t, g, n] + skip[d] u[t, d]) silu(z[t, d])
//
// A request's tokens are rows cu_q[i] .. cu_q[i + 1]; it starts from the state in row slots[i] and leaves its new one in row
// to_slots[i].  A slot outside of the state belongs to no request: zeros come from there and nothing is left there.
#include "common.cuh"

#include <atomic>

struct ScanArgs {
    const void *u, *dt, *b, *c, *z;
    const float *a, *skip, *dt_bias;
    float* state;
    const int *cu_q, *slots, *to_slots;
    void* out;
    long long ld_u, ld_dt, ld_b, ld_c, ld_z, ld_out, ld_state;
    int n_tokens, n_seqs, n_slots, channels, states, groups, u_type, dt_type, bc_type, softplus, max_q_len, stepwise;
};

typedef unsigned long long ss_pair;            // two floats side by side
__device__ __forceinline__ ss_pair ss_pack(float lo, float hi) {
    ss_pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void ss_unpack(ss_pair v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ ss_pair ss_fma2(ss_pair a, ss_pair b, ss_pair c) {
    ss_pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ ss_pair ss_add2(ss_pair a, ss_pair b) {
    ss_pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ ss_pair ss_mul2(ss_pair a, ss_pair b) {
    ss_pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ss_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// exp(delta a) - 1 from a2 = a log2(e).  ex2.approx is off by -0.26 .. -0.45 x 2^-24 on the average (0.65 of them as a root mean
// square) for arguments between 2^-8 and 1, which a state that remembers n tokens takes n times over: the argument is moved up by
// SS_SHIFT, which leaves 0.1.  Below 2^-6 three terms of the series are exact to 0.01 x 2^-24.
#define SS_LOG2E 1.44269504f
#define SS_SHIFT 3.01e-8f                    /* 0.35 x 2^-24 log2(e) */
#define SS_NEAR 0.015625f
__device__ __forceinline__ float ss_decay_less_one(float delta, float a2) {
    const float x = delta * a2;
    const float slow = fmaf(fmaf(x, 0.055504109f, 0.24022651f), x, 0.69314718f) * x;       // ln 2, its square / 2, its cube / 6
    const float fast = ss_ex2(fmaf(delta, a2, SS_SHIFT)) - 1.f;
    return fabsf(x) < SS_NEAR ? slow : fast;
}
__device__ __forceinline__ float ss_decay(float delta, float a2) {
    const float x = delta * a2;
    const float slow = fmaf(fmaf(fmaf(x, 0.055504109f, 0.24022651f), x, 0.69314718f), x, 1.f);
    const float fast = ss_ex2(fmaf(delta, a2, SS_SHIFT));
    return fabsf(x) < SS_NEAR ? slow : fast;
}

__device__ __forceinline__ ss_pair ss_decay2(ss_pair delta, ss_pair a2) {
    const ss_pair x = ss_mul2(delta, a2);
    ss_pair slow = ss_fma2(x, ss_pack(0.055504109f, 0.055504109f), ss_pack(0.24022651f, 0.24022651f));
    slow = ss_fma2(ss_fma2(slow, x, ss_pack(0.69314718f, 0.69314718f)), x, ss_pack(1.f, 1.f));
    float x0, x1, s0, s1, f0, f1;
    ss_unpack(ss_fma2(delta, a2, ss_pack(SS_SHIFT, SS_SHIFT)), f0, f1);
    ss_unpack(x, x0, x1);
    ss_unpack(slow, s0, s1);
    f0 = ss_ex2(f0);
    f1 = ss_ex2(f1);
    return ss_pack(fabsf(x0) < SS_NEAR ? s0 : f0, fabsf(x1) < SS_NEAR ? s1 : f1);
}

// max(v, 0) + log(1 + e), e = exp(-|v|): with x the rounded product -|v| log2(e), e = 2^x exp(-|v| - x ln 2), the second factor as one plus
// its small exponent (without it e is off by up to 1.2 |v| x 2^-24; what is left of that is the rounded ln 2, 0.046 |v| x 2^-24, the other way
// than 2^x errs: its low part would cost 8,192 tokens x 8,192 channels 531 us, so 519, 518 without the factor).  Below -88, where 2^x is zero,
// v counts as -88 (the exponent of an infinity would be no number); NaN stays.  log(1 + e) / e over (0, 1] as a polynomial of degree 9 (fitted
// for the smallest relative error, 0.08 x 2^-24), which leaves the unit of 2^x to the decays.  All in all 4.5 x 2^-24 at most, 0.9 .. 1.3 as a
// root mean square (measured from -60 to 1; less above).
#define SS_LN2 0.69314718f
__device__ __forceinline__ float ss_below(float v) {             // -|v|, -88 or NaN
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(-fabsf(v)), "f"(-88.f));
    return r;
}
__device__ __forceinline__ float ss_softplus(float v) {
    const float a = ss_below(v), x = a * SS_LOG2E;
    float e = ss_ex2(x);
    e = fmaf(e, fmaf(x, -SS_LN2, a), e);
    float q = fmaf(-0.00324398419f, e, 0.0198512822f);
    q = fmaf(q, e, -0.0569592081f);
    q = fmaf(q, e, 0.106036231f);
    q = fmaf(q, e, -0.153055742f);
    q = fmaf(q, e, 0.196759328f);
    q = fmaf(q, e, -0.249541327f);
    q = fmaf(q, e, 0.333299637f);
    q = fmaf(q, e, -0.499999017f);
    q = fmaf(q, e, 1.f);
    return fmaf(q, e, fmaxf(v, 0.f));
}

__device__ __forceinline__ ss_pair ss_softplus2(ss_pair v) {
    float v0, v1, x0, x1;
    ss_unpack(v, v0, v1);
    auto both = [](float c) { return ss_pack(c, c); };
    const ss_pair a = ss_pack(ss_below(v0), ss_below(v1)), x = ss_mul2(a, both(SS_LOG2E));
    ss_unpack(x, x0, x1);
    ss_pair e = ss_pack(ss_ex2(x0), ss_ex2(x1));
    e = ss_fma2(e, ss_fma2(x, both(-SS_LN2), a), e);
    ss_pair q = ss_fma2(both(-0.00324398419f), e, both(0.0198512822f));
    q = ss_fma2(q, e, both(-0.0569592081f));
    q = ss_fma2(q, e, both(0.106036231f));
    q = ss_fma2(q, e, both(-0.153055742f));
    q = ss_fma2(q, e, both(0.196759328f));
    q = ss_fma2(q, e, both(-0.249541327f));
    q = ss_fma2(q, e, both(0.333299637f));
    q = ss_fma2(q, e, both(-0.499999017f));
    q = ss_fma2(q, e, both(1.f));
    return ss_fma2(q, e, ss_pack(fmaxf(v0, 0.f), fmaxf(v1, 0.f)));
}

// silu in FP32, v / (1 + exp(-v)): the quotient by the hardware's reciprocal, put right by what it leaves, with the errors of a division
// (2,048 tokens x 4,096 channels 82 us, 87 by a division); where that is no number (infinities) as it is, below 1e-36 zero.
__device__ __forceinline__ float ss_silu_f32(float v) {
    const float d = 1.f + expf(-v);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    const float q = v * r, better = fmaf(fmaf(-d, q, v), r, q);
    return better == better ? better : q;
}
// silu: in 16 bits 2^x and the reciprocal of the hardware (3 x 2^-24 and |z| x 2^-24 off, where the result is rounded to 2^-8)
template <typename T> __device__ __forceinline__ float ss_silu(float z) { return ss_silu_f32(z); }
template <> __device__ __forceinline__ float ss_silu<__nv_bfloat16>(float z) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ss_ex2(-z * SS_LOG2E)));
    return z * r;
}

// N neighbouring numbers of a row (one or four), `count` of which are there; `vector`: the address is a multiple of their size
template <int N> __device__ __forceinline__ void ss_load(const float* p, float* v, bool vector, int count) {
    if constexpr (N == 4)
        if (vector && count >= N) {
            NiVec16<float>::load(p, v);
            return;
        }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < count ? p[i] : 0.f;
}
template <int N> __device__ __forceinline__ void ss_load(const __nv_bfloat16* p, float* v, bool vector, int count) {
    if constexpr (N == 4)
        if (vector && count >= N) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
            v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
            return;
        }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < count ? __bfloat162float(p[i]) : 0.f;
}
template <int N> __device__ __forceinline__ void ss_load_any(const void* p, int type, long long at, float* v, bool vector, int count) {
    if (type == NI_DTYPE_F32) ss_load<N>(static_cast<const float*>(p) + at, v, vector, count);
    else ss_load<N>(static_cast<const __nv_bfloat16*>(p) + at, v, vector, count);
}
// (eight, four or two)
template <int N> __device__ __forceinline__ void ss_store(float* p, const float* v, bool vector, int count) {
    if (vector && count >= N) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) NiVec16<float>::store(p + i, v + i);
            return;
        } else if constexpr (N == 2) {
            *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < count) p[i] = v[i];
}
template <int N> __device__ __forceinline__ void ss_store(__nv_bfloat16* p, const float* v, bool vector, int count) {
    if (vector && count >= N) {
        if constexpr (N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 8) NiVec16<__nv_bfloat16>::store(p + i, v + i);
            return;
        } else if constexpr (N == 4 || N == 2) {
            __nv_bfloat162 x[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) x[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            if constexpr (N == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(x);
            else *reinterpret_cast<__nv_bfloat162*>(p) = x[0];
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < count) p[i] = __float2bfloat16_rn(v[i]);
}

// N numbers on their way from memory, as they lie there: turned into FP32 only where they are used, so that the load need not have
// ended before.  WIDE: by 16 bytes (8, 4 for fewer), else one by one.
template <int N, bool WIDE> struct ScanRaw {
    uint32_t w[N];
    __device__ __forceinline__ void load(const void* p, int type, long long at, int count) {
        if constexpr (WIDE) {
            if (count < N) {
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = 0;
            } else if (type == NI_DTYPE_F32) {
                words<N>(static_cast<const float*>(p) + at);
            } else {
                words<N / 2>(static_cast<const __nv_bfloat16*>(p) + at);
            }
        } else if (type == NI_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = i < count ? static_cast<const uint32_t*>(p)[at + i] : 0;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = i < count ? static_cast<const uint16_t*>(p)[at + i] : 0;
        }
    }
    template <int W> __device__ __forceinline__ void words(const void* p) {
        if constexpr (W % 4 == 0) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint32_t*>(p) + i);
                w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
            }
        } else if constexpr (W == 2) {
            const uint2 x = *static_cast<const uint2*>(p);
            w[0] = x.x; w[1] = x.y;
        } else {
            w[0] = *static_cast<const uint32_t*>(p);
        }
    }
    __device__ __forceinline__ void get(int type, float* v) const {
        if (type == NI_DTYPE_F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
        } else if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i] << 16);
        }
    }
};

// More than 48 KB of shared memory are asked for once per kernel and device (a call of the runtime for every launch otherwise).
template <typename Kernel> static void ss_more_shared(Kernel kernel, int bytes, std::atomic<unsigned long long>& asked) {
    int device = 0;
    cudaGetDevice(&device);
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (asked.load(std::memory_order_relaxed) & bit) return;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
}

// What a wide access to columns `first`, first + 8, ... of every row needs: the address and the row's step are multiples of 16 bytes.
static bool ss_wide(const void* p, long long ld, int type, int step) {
    const int size = type == NI_DTYPE_F32 ? 4 : 2;
    return (reinterpret_cast<size_t>(p) & 15) == 0 && (ld * size) % 16 == 0 && (step * size) % 16 == 0;
}

// ---- prompt portions -------------------------------------------------------------------------------------------------
// A block owns CH channels of one request and walks its tokens in tiles of 32 through two buffers in shared memory.  Four warps per
// buffer load its tiles, turn dt into delta and delta u (each number once per channel, not per state) and B, C into FP32, and later
// gate, round and store the rows.  The others scan: LANES threads per channel with four states each in registers, groups of GROUP
// tokens in three overlapping steps - a group's 2^x, the updates of the states of the group before, and what its sums over the
// states leave (ScanBuffer) of the one before that.
//
// Bound by neither bytes nor 2^x alone (a state's step: one 2^x, four multiply-adds, a fourth of two 16-byte reads of shared memory):
// 2,048 tokens x 4,096 channels x 16 states in bfloat16 79 us (13 by its bytes, 30 by 2^x), 8,192 x 8,192 519 (103; 239).  One scanning
// warp per scheduler waits on the length of its own chain; with two the reads of B and C from shared memory fill that unit to 85 %.
// Within a tile a decay is one 2^x, off to one side by up to 0.25 x 2^-24 where it is near one; what the tile's first state is
// worth at its end is put right by the decay over the whole tile, from the sum of its deltas (the product of the tile's decays is
// kept as its difference from one, which loses nothing): thousands of decays near one keep no trace of the 2^x.
// STEPWISE: every decay as the single tokens' kernel takes it, and no tiles' sums - what a token gives then has the same bits
// however its request is cut into calls.
#define SS_TILE 32
#define SS_SPLIT 128                         /* tokens from which on a request is split */
#define SS_HELPERS 128                       /* per buffer */
// Up to four lanes a channel: their sums go to shared memory as they are and the helpers add them up (the exchange would cost the
// scanning warps 12 instructions for every four tokens: 2,048 tokens x 4,096 channels 92 us, so 82).
template <int LANES, int NS, int CH, int GROUP>
struct ScanBuffer {
    static constexpr int PAD = LANES * NS, ROW = CH + (CH == 64 ? 8 : 4), SUMS = LANES <= 4 ? LANES : 1;
    float2 step[SS_TILE][ROW];                 // delta, delta u; channels in the order of `place`
    float b[SS_TILE][PAD], c[SS_TILE][PAD];
    float y[SS_TILE + GROUP][SUMS > 1 ? ROW * SUMS : CH + 8];      // token t's sums in row t + GROUP (one group later than they are made)
};
// SPLIT: what the tokens of one block leave of a state of zeros, and the sums of their deltas
template <int SCAN, int NS> struct ScanCarry {
    float h[SCAN][NS], sum[SCAN];
};
__device__ __forceinline__ int ss_cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ int ss_cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ void ss_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ss_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A float of the same place in another block's shared memory
__device__ __forceinline__ float ss_of_rank(const float* mine, int rank) {
    unsigned there;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}

struct ScanYes { static constexpr bool value = true; };
struct ScanNo { static constexpr bool value = false; };
template <int LANES> struct ScanGroup { static constexpr int N = LANES < 4 ? LANES : 4; };

// Barriers between the two kinds of warps, one pair per buffer: full (the helpers arrive), done (the scanning warps arrive).
template <int THREADS> __device__ __forceinline__ void ss_wait(int barrier) { asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(THREADS) : "memory"); }
template <int THREADS> __device__ __forceinline__ void ss_arrive(int barrier) { asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "n"(THREADS) : "memory"); }

// GROUP numbers of each of LANES lanes -> lane j's sum of everybody's number j (with more lanes than numbers, in several places)
template <int LANES, int GROUP>
__device__ __forceinline__ float ss_exchange(float (&v)[GROUP], int lane) {
#pragma unroll
    for (int w = GROUP / 2; w > 0; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const float give = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
        }
    }
    float r = v[0];
#pragma unroll
    for (int w = GROUP; w < LANES; w <<= 1) r += __shfl_xor_sync(0xffffffffu, r, w);
    return r;
}

template <typename TU, int LANES, int CH, bool WIDE, bool STEPWISE, bool SPLIT>
__global__ void __launch_bounds__(LANES * CH + 2 * SS_HELPERS) selective_scan_kernel(const __grid_constant__ ScanArgs p, const int least) {
    if (p.cu_q[blockIdx.y + 1] - p.cu_q[blockIdx.y] < least) return;        // (another launch's; first of all: there may be many)
    constexpr int NS = 4, NP = NS / 2, SCAN = LANES * CH, THREADS = SCAN + SS_HELPERS, GROUP = ScanGroup<LANES>::N, PAD = LANES * NS;
    // a helper's numbers of a tile: PIECES pieces of PIECE neighbouring channels, ROWS rows apart
    constexpr int PIECE = CH >= 32 ? 8 : CH / 4, ROW_PIECES = CH / PIECE, ROWS = SS_HELPERS / ROW_PIECES, PIECES = SS_TILE / ROWS;
    typedef ScanBuffer<LANES, NS, CH, GROUP> Buffer;
    extern __shared__ __align__(16) unsigned char ss_shared[];
    Buffer* const buffers = reinterpret_cast<Buffer*>(ss_shared);
    const int seq = blockIdx.y, per_group = p.channels / p.groups, blocks = (per_group + CH - 1) / CH;
    const int rank = SPLIT ? ss_cluster_rank() : 0, ranks = SPLIT ? ss_cluster_size() : 1, block = blockIdx.x / ranks;
    const int group = block / blocks, in_group = (block - group * blocks) * CH, d0 = group * per_group + in_group;
    const int n_ch = min(CH, per_group - in_group);
    int first = max(0, min(p.cu_q[seq], p.n_tokens)), end = max(first, min(p.cu_q[seq + 1], p.n_tokens));
    const int chunk = SPLIT ? ((end - first + ranks * SS_TILE - 1) / (ranks * SS_TILE)) * SS_TILE : 0, request_end = end;
    const bool split = SPLIT && end - first >= SS_SPLIT;       // (a short request is the first block's alone)
    if (SPLIT && !split && rank > 0) return;
    if (split) {
        first = min(end, first + rank * chunk);
        end = min(end, first + chunk);
    }
    const int tiles = (end - first + SS_TILE - 1) / SS_TILE;
    const bool before = SPLIT && end < request_end;            // blocks behind this one wait for what its tokens leave
    ScanCarry<SCAN, NS>& carry = *reinterpret_cast<ScanCarry<SCAN, NS>*>(buffers + 2);

    if (threadIdx.x >= SCAN) {
        constexpr int U_TYPE = sizeof(TU) == 4 ? NI_DTYPE_F32 : NI_DTYPE_BF16;
        constexpr int BC_PIECES = SS_TILE * PAD / 4 / SS_HELPERS > 0 ? SS_TILE * PAD / 4 / SS_HELPERS : 1;
        const int mine = (threadIdx.x - SCAN) / SS_HELPERS, tid = (threadIdx.x - SCAN) % SS_HELPERS;       // the buffer's number
        Buffer& s = buffers[mine];
        const TU* u = static_cast<const TU*>(p.u) + d0;
        const TU* z = static_cast<const TU*>(p.z) + d0;
        TU* out = static_cast<TU*>(p.out) + d0;
        const int piece = tid % ROW_PIECES, col = piece * PIECE, row = tid / ROW_PIECES, count = n_ch - col;
        float bias[PIECE], skip[PIECE];
#pragma unroll
        for (int i = 0; i < PIECE; ++i) {
            bias[i] = p.dt_bias && i < count ? p.dt_bias[d0 + col + i] : 0.f;
            skip[i] = p.skip && i < count ? p.skip[d0 + col + i] : 0.f;
        }
        ScanRaw<PIECE, WIDE> ru[PIECES], rdt[PIECES], rz[PIECES], cu[PIECES], cz[PIECES];    // the next tile's, and what its end needs of this one
        ScanRaw<4, WIDE> rb[BC_PIECES], rc[BC_PIECES];
        auto fetch = [&](int k, bool all) {
            const int t0 = first + k * SS_TILE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const long long t = t0 + row + i * ROWS;
                const int n = t < end ? count : 0;
                ru[i].load(u, U_TYPE, t * p.ld_u + col, n);
                rdt[i].load(p.dt, p.dt_type, t * p.ld_dt + d0 + col, n);
                if (p.z && all) rz[i].load(z, U_TYPE, t * p.ld_z + col, n);
            }
#pragma unroll
            for (int i = 0; i < BC_PIECES; ++i) {
                const int at = tid + i * SS_HELPERS, n = at % (PAD / 4) * 4, r = at / (PAD / 4);
                const long long t = t0 + r;
                const int real = r < SS_TILE && t < end ? p.states - n : 0;
                rb[i].load(p.b, p.bc_type, t * p.ld_b + (long long)group * p.states + n, real);
                if (all) rc[i].load(p.c, p.bc_type, t * p.ld_c + (long long)group * p.states + n, real);
            }
        };
        auto stage = [&](int k) {
            const int n = end - first - k * SS_TILE;
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const int at = row + j * ROWS;
                float x[PIECE], v[PIECE];
                ru[j].get(U_TYPE, x);
                rdt[j].get(p.dt_type, v);
#pragma unroll
                for (int i = 0; i < PIECE; i += 2) {
                    v[i] += bias[i];
                    v[i + 1] += bias[i + 1];
                    if (p.softplus) ss_unpack(ss_softplus2(ss_pack(v[i], v[i + 1])), v[i], v[i + 1]);
                }
#pragma unroll
                for (int i = 0; i < PIECE; ++i)            // (tokens that do not exist change nothing)
                    s.step[at][i * ROW_PIECES + piece] = at < n ? make_float2(v[i], v[i] * x[i]) : make_float2(0.f, 0.f);
                cu[j] = ru[j];
                cz[j] = rz[j];
            }
#pragma unroll
            for (int i = 0; i < BC_PIECES; ++i) {
                const int at = tid + i * SS_HELPERS, m = at % (PAD / 4) * 4, r = at / (PAD / 4);
                if (r < SS_TILE) {
                    rb[i].get(p.bc_type, &s.b[r][m]);
                    rc[i].get(p.bc_type, &s.c[r][m]);
                }
            }
        };
        auto finish = [&](int k) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                float v[PIECE], x[PIECE];
                cu[j].get(U_TYPE, x);
#pragma unroll
                for (int i = 0; i < PIECE; ++i) {
                    const float* const sums = &s.y[GROUP + row + j * ROWS][(i * ROW_PIECES + piece) * Buffer::SUMS];
                    if constexpr (Buffer::SUMS == 4) {      // (in the exchange's order)
                        float part[4];
                        NiVec16<float>::load(sums, part);
                        v[i] = (part[0] + part[2]) + (part[1] + part[3]);
                    } else if constexpr (Buffer::SUMS == 2) {
                        v[i] = sums[0] + sums[1];
                    } else {
                        v[i] = sums[0];
                    }
                    if (p.skip) v[i] = fmaf(skip[i], x[i], v[i]);
                }
                if (p.z) {
                    cz[j].get(U_TYPE, x);
#pragma unroll
                    for (int i = 0; i < PIECE; ++i) v[i] *= ss_silu<TU>(x[i]);
                }
                const long long at = first + k * SS_TILE + row + j * ROWS;
                if (at < end) ss_store<PIECE>(out + at * p.ld_out + col, v, WIDE, count);
            }
        };
        auto walk = [&](bool all) {             // `all`: with z, C and what leaves
            if (mine < tiles) fetch(mine, all);
            for (int k = mine; k < tiles; k += 2) {
                stage(k);
                __threadfence_block();
                ss_arrive<THREADS>(1 + mine);
                if (k + 2 < tiles) fetch(k + 2, all);
                ss_wait<THREADS>(3 + mine);
                if (all) finish(k);
            }
        };
        if (split) {
            if (before) walk(false);
            __syncwarp();
            ss_cluster_arrive();
            ss_cluster_wait();
            ss_cluster_arrive();
        }
        walk(true);
        if (split) {
            __syncwarp();
            ss_cluster_wait();
        }
        return;
    }

    const int tid = threadIdx.x, lane = tid % LANES, place = tid / LANES, n0 = lane * NS, n_real = min(NS, p.states - n0);
    const int from = p.slots[seq], to = p.to_slots[seq];
    // neighbouring helpers write neighbouring places: channel PIECE q + i stands at place i ROW_PIECES + q
    const int ch = place % ROW_PIECES * PIECE + place / ROW_PIECES;
    const bool mine = ch < n_ch;
    const long long at = (long long)(d0 + ch) * p.states + n0;
    ss_pair a2[NP], h[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        float av[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            av[j] = mine && 2 * i + j < n_real ? p.a[at + 2 * i + j] * SS_LOG2E : 0.f;
            if (fabsf(av[j]) == INFINITY) av[j] = copysignf(3e38f, av[j]);           // (times a delta of zero: zero)
        }
        a2[i] = ss_pack(av[0], av[1]);
        h[i] = 0;
    }
    float total = 0.f;                          // SPLIT: of all tiles' deltas
    auto scan = [&](auto reads) {               // reads.value: with sums over the states for the helpers to finish
        constexpr bool READS = decltype(reads)::value;
        for (int k = 0; k < tiles; ++k) {
            Buffer& s = buffers[k & 1];
            const int groups = (min(SS_TILE, end - first - k * SS_TILE) + GROUP - 1) / GROUP;
            ss_pair start[NP], less[NP], e[GROUP][NP];       // less: the product of the tile's decays, less one
            float sum = 0.f, du[GROUP], held[GROUP];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                start[i] = h[i];
                less[i] = 0;
            }
            auto powers = [&](int t, ss_pair (&e)[GROUP][NP], float (&du)[GROUP]) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const float2 dd = s.step[t + j][place];
                    du[j] = dd.y;
                    if (!STEPWISE) sum += dd.x;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        float a0, a1;
                        ss_unpack(a2[i], a0, a1);
                        if constexpr (STEPWISE) e[j][i] = ss_decay2(ss_pack(dd.x, dd.x), a2[i]);
                        else e[j][i] = ss_pack(ss_ex2(fmaf(dd.x, a0, SS_SHIFT)), ss_ex2(fmaf(dd.x, a1, SS_SHIFT)));
                    }
                }
            };
            auto update = [&](int t, const ss_pair (&e)[GROUP][NP], const float (&du)[GROUP], float (&v)[GROUP]) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    float bv[NS], cv[NS];
                    NiVec16<float>::load(&s.b[t + j][n0], bv);
                    if (READS) NiVec16<float>::load(&s.c[t + j][n0], cv);
                    ss_pair y = 0;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        if (!STEPWISE) less[i] = ss_fma2(less[i], e[j][i], ss_add2(e[j][i], ss_pack(-1.f, -1.f)));
                        h[i] = ss_fma2(e[j][i], h[i], ss_pack(du[j] * bv[2 * i], du[j] * bv[2 * i + 1]));
                        if (!WIDE) {            // states that do not exist stay zero whatever delta u is
                            float v0, v1;
                            ss_unpack(h[i], v0, v1);
                            h[i] = ss_pack(2 * i < n_real ? v0 : 0.f, 2 * i + 1 < n_real ? v1 : 0.f);
                        }
                        if constexpr (READS) {
                            const ss_pair cc = ss_pack(cv[2 * i], cv[2 * i + 1]);
                            y = i ? ss_fma2(h[i], cc, y) : ss_mul2(h[i], cc);
                        }
                    }
                    float lo, hi;
                    ss_unpack(y, lo, hi);
                    v[j] = lo + hi;
                }
            };
            auto leave = [&](int t, float (&v)[GROUP]) {
                if constexpr (READS && Buffer::SUMS > 1) {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) s.y[t + j][place * LANES + lane] = v[j];
                } else if constexpr (READS) {
                    const float y = ss_exchange<LANES, GROUP>(v, lane);
                    if (lane < GROUP) s.y[t + lane][place] = y;
                }
            };
            ss_wait<THREADS>(1 + (k & 1));
            if (groups == SS_TILE / GROUP) {
                powers(0, e, du);
#pragma unroll
                for (int g = 0; g < SS_TILE / GROUP; ++g) {
                    ss_pair next_e[GROUP][NP];
                    float next_du[GROUP], v[GROUP];
                    if (g + 1 < SS_TILE / GROUP) powers((g + 1) * GROUP, next_e, next_du);
                    update(g * GROUP, e, du, v);
                    if (g > 0) leave(g * GROUP, held);
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        held[j] = v[j];
                        du[j] = next_du[j];
#pragma unroll
                        for (int i = 0; i < NP; ++i) e[j][i] = next_e[j][i];
                    }
                }
                leave(SS_TILE, held);
            } else {
#pragma unroll 1
                for (int g = 0; g < groups; ++g) {
                    powers(g * GROUP, e, du);
                    update(g * GROUP, e, du, held);
                    leave((g + 1) * GROUP, held);
                }
            }
            __threadfence_block();
            ss_arrive<THREADS>(3 + (k & 1));
#pragma unroll
            for (int i = 0; i < NP && !STEPWISE; ++i) {      // (where the first state has faded or is not finite, what the steps gave stands)
                float av[2], hv[2], lv[2], sv[2];
                ss_unpack(a2[i], av[0], av[1]);
                ss_unpack(h[i], hv[0], hv[1]);
                ss_unpack(less[i], lv[0], lv[1]);
                ss_unpack(start[i], sv[0], sv[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float more = ss_decay_less_one(sum, av[j]) - lv[j];
                    if (fabsf(lv[j]) < 0.5f && fabsf(sv[j]) < INFINITY) hv[j] = fmaf(more, sv[j], hv[j]);
                }
                h[i] = ss_pack(hv[0], hv[1]);
            }
            if (SPLIT && !READS) total += sum;
        }
    };
    if constexpr (SPLIT)
        if (before) {
            scan(ScanNo{});
            carry.sum[tid] = total;
#pragma unroll
            for (int i = 0; i < NP; ++i) ss_unpack(h[i], carry.h[tid][2 * i], carry.h[tid][2 * i + 1]);
        }
    if (split) {
        __syncwarp();
        ss_cluster_arrive();
        ss_cluster_wait();
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        float hv[2], av[2];
        ss_unpack(a2[i], av[0], av[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bool real = mine && 2 * i + j < n_real && from >= 0 && from < p.n_slots;
            hv[j] = real ? p.state[from * p.ld_state + at + 2 * i + j] : 0.f;
            for (int r = 0; split && first < end && r < rank; ++r) {
                // the blocks before this one, in order; zeros and infinities stay what single steps leave them
                const float decay = ss_decay(ss_of_rank(&carry.sum[tid], r), av[j]);
                if (hv[j] != 0.f && !(decay == 0.f && fabsf(hv[j]) == INFINITY)) hv[j] *= decay;
                hv[j] += ss_of_rank(&carry.h[tid][2 * i + j], r);
            }
        }
        h[i] = ss_pack(hv[0], hv[1]);
    }
    if (split) {
        __syncwarp();
        ss_cluster_arrive();
    }
    scan(ScanYes{});
    if (split) {                                // (every block has read the state, and the others' carries)
        __syncwarp();
        ss_cluster_wait();
        if (end < request_end || (first >= end && rank > 0)) return;
    }
    // (a request without tokens and of one slot writes nothing: the row may be one that a request with tokens owns)
    if (mine && to >= 0 && to < p.n_slots && (first < end || to != from)) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            float hv[2];
            ss_unpack(h[i], hv[0], hv[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (2 * i + j < n_real) p.state[to * p.ld_state + at + 2 * i + j] = hv[j];
        }
    }
}

template <typename TU, int LANES, int CH>
static void ss_scan(const ScanArgs& p, bool wide, int ranks, int least, cudaStream_t stream) {
    const int blocks = (p.channels / p.groups + CH - 1) / CH * p.groups;
    typedef ScanCarry<LANES * CH, 4> Carry;
    auto launch = [&](auto kernel, int ranks, std::atomic<unsigned long long>& asked) {
        const int bytes = 2 * sizeof(ScanBuffer<LANES, 4, CH, ScanGroup<LANES>::N>) + (ranks > 1 ? sizeof(Carry) : 0);
        ss_more_shared(kernel, bytes, asked);
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(blocks * ranks, p.n_seqs);
        config.blockDim = dim3(LANES * CH + 2 * SS_HELPERS);
        config.dynamicSmemBytes = bytes;
        config.stream = stream;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = ranks;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        config.attrs = &cluster;
        config.numAttrs = ranks > 1 ? 1 : 0;
        cudaLaunchKernelEx(&config, kernel, p, least);
    };
#define SS_LAUNCH(W, STEP, PARTS, RANKS)                                                              \
    do {                                                                                              \
        static std::atomic<unsigned long long> asked{0};                                              \
        launch(selective_scan_kernel<TU, LANES, CH, W, STEP, PARTS>, RANKS, asked);                   \
        return;                                                                                       \
    } while (0)
    constexpr bool FAST = LANES == 4 && CH > 32;              // (chosen for whole requests in 16-byte pieces only)
    if constexpr (sizeof(TU) == 4 && !FAST)
        if (p.stepwise) {
            if (wide) SS_LAUNCH(true, true, false, 1);
            else SS_LAUNCH(false, true, false, 1);
        }
    if constexpr (!FAST) {
        if (ranks > 1) {
            if (wide) SS_LAUNCH(true, false, true, ranks);
            else SS_LAUNCH(false, false, true, ranks);
        }
        if (!wide) SS_LAUNCH(false, false, false, 1);
    }
    SS_LAUNCH(true, false, false, 1);
}

// ---- single tokens ---------------------------------------------------------------------------------------------------
// Bound by the states, which come and go once.  LANES threads per channel with four neighbouring states each take GROUP requests at
// a time: lane s turns request s's dt, u and z into what all lanes need, and the sums over the states are exchanged so that lane s
// ends with request s's.  A block owns 256 / LANES channels of many requests, whose B and C it first lays down in FP32; every
// thread's states of the next SS_AHEAD groups are on their way into 16-byte places of its own in shared memory (no other thread
// reads them: nothing waits at a barrier).  At 16 states the copy rate leaves an SM 44 thread instructions per state.
// 128 requests x 8,192 channels x 16 states: 29 us, three quarters of the copy rate; 60 with states loaded where they are used.
#define SS_AHEAD 2
#define SS_TOKEN_THREADS 256
#define SS_TOKEN_FLOATS 1024                 /* of B, and of C, of a block's requests; SS_TOKEN_FLOATS / PAD requests at most */
struct ScanTokenShared {
    float4 h[SS_AHEAD][4][SS_TOKEN_THREADS];
    float b[SS_TOKEN_FLOATS], c[SS_TOKEN_FLOATS];
    int t[SS_TOKEN_FLOATS / 8 + 4], from[SS_TOKEN_FLOATS / 8 + 4], to[SS_TOKEN_FLOATS / 8 + 4];
};
__device__ __forceinline__ void ss_copy16(void* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

template <typename TU, int LANES>
__global__ void __launch_bounds__(SS_TOKEN_THREADS, 5) selective_tokens_kernel(const __grid_constant__ ScanArgs p, const int per_block) {
    constexpr int NS = 4, PAD = LANES * NS, CH = SS_TOKEN_THREADS / LANES, GROUP = ScanGroup<LANES>::N;
    constexpr int U_TYPE = sizeof(TU) == 4 ? NI_DTYPE_F32 : NI_DTYPE_BF16;
    extern __shared__ __align__(16) unsigned char ss_shared[];
    ScanTokenShared& sh = *reinterpret_cast<ScanTokenShared*>(ss_shared);
    const int tid = threadIdx.x, lane = tid % LANES, seq0 = blockIdx.y * per_block, n_seqs = min(per_block, p.n_seqs - seq0);
    const int per_group = p.channels / p.groups, blocks = (per_group + CH - 1) / CH, group = blockIdx.x / blocks;
    const int in_group = (blockIdx.x - group * blocks) * CH + tid / LANES, d = group * per_group + min(in_group, per_group - 1);
    const bool mine = in_group < per_group;
    for (int i = tid; i < n_seqs + GROUP - 1; i += SS_TOKEN_THREADS) {       // (places behind the last request: none)
        const int seq = seq0 + i;
        int t = -1, from = -1, to = -1;
        if (i < n_seqs) {
            t = p.cu_q[seq];
            from = p.slots[seq];
            to = p.to_slots[seq];
            const int length = p.cu_q[seq + 1] - t;
            if (t < 0 || length <= 0 || t >= p.n_tokens) t = -1;
            if (from < 0 || from >= p.n_slots) from = -1;
            if (to < 0 || to >= p.n_slots || (t < 0 && to == from)) to = -1;
            if (length > 1) t = from = to = -1;              // (another launch's)
        }
        sh.t[i] = t;
        sh.from[i] = from;
        sh.to[i] = to;
    }
    // (the launcher has seen that a row's step fits 31 bits: rows times steps are one instruction each)
    const int ld_state = (int)p.ld_state, ld_u = (int)p.ld_u, ld_dt = (int)p.ld_dt, ld_z = (int)p.ld_z;
    float* const state = p.state + (long long)d * p.states + lane * NS;
    float av[NS];
    ss_load<NS>(p.a + (long long)d * p.states + lane * NS, av, true, NS);
    const float skip = p.skip ? p.skip[d] : 0.f, bias = p.dt_bias ? p.dt_bias[d] : 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        av[i] *= SS_LOG2E;
        if (fabsf(av[i]) == INFINITY) av[i] = copysignf(3e38f, av[i]);        // (times a delta of zero: zero)
    }
    const ss_pair a01 = ss_pack(av[0], av[1]), a23 = ss_pack(av[2], av[3]);
    const int groups = (n_seqs + GROUP - 1) / GROUP;
    __syncthreads();
    auto ask = [&](int g) {
        if (g < groups)
#pragma unroll
            for (int s = 0; s < GROUP; ++s) {
                const int from = sh.from[g * GROUP + s];
                float4* const place = &sh.h[g % SS_AHEAD][s][tid];
                if (from >= 0) ss_copy16(place, state + (long long)from * ld_state);
                else *place = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int g = 0; g < SS_AHEAD; ++g) ask(g);
    ScanRaw<1, false> next_dt, next_u, next_z;
    auto scalars = [&](int g) {                 // a group's dt, u and z of this lane's request
        const int t = sh.t[g * GROUP + lane % GROUP];
        if (t >= 0) {
            next_dt.load(p.dt, p.dt_type, (long long)t * ld_dt + d, 1);
            next_u.load(p.u, U_TYPE, (long long)t * ld_u + d, 1);
            if (p.z) next_z.load(p.z, U_TYPE, (long long)t * ld_z + d, 1);
        }
    };
    scalars(0);
    for (int i = tid; i < groups * GROUP * LANES; i += SS_TOKEN_THREADS) {
        const int row = sh.t[i / LANES], n = group * PAD + i % LANES * NS;
        float b[NS] = {}, c[NS] = {};
        if (row >= 0) {
            ss_load_any<NS>(p.b, p.bc_type, row * p.ld_b + n, b, true, NS);
            ss_load_any<NS>(p.c, p.bc_type, row * p.ld_c + n, c, true, NS);
        }
        NiVec16<float>::store(&sh.b[i * NS], b);
        NiVec16<float>::store(&sh.c[i * NS], c);
    }
    __syncthreads();
    for (int g = 0; g < groups; ++g) {
        const int t = sh.t[g * GROUP + lane % GROUP];
        float v[GROUP], delta = 0.f, du = 0.f, u = 0.f, z = 0.f;
        if (t >= 0) {                           // (no token: a delta of zero, so a decay of exactly one, and nothing comes in)
            next_dt.get(p.dt_type, &delta);
            next_u.get(U_TYPE, &u);
            if (p.z) next_z.get(U_TYPE, &z);
            delta += bias;
            if (p.softplus) delta = ss_softplus(delta);
            du = delta * u;
        }
        if (g + 1 < groups) scalars(g + 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(SS_AHEAD - 1) : "memory");
#pragma unroll
        for (int s = 0; s < GROUP; ++s) {
            const int i = g * GROUP + s, to = sh.to[i];
            const float delta_s = __shfl_sync(0xffffffffu, delta, s, LANES), du_s = __shfl_sync(0xffffffffu, du, s, LANES);
            const ss_pair delta2 = ss_pack(delta_s, delta_s), du2 = ss_pack(du_s, du_s);
            ulonglong2 h = *reinterpret_cast<const ulonglong2*>(&sh.h[g % SS_AHEAD][s][tid]);
            const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&sh.b[i * PAD + lane * NS]);
            const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&sh.c[i * PAD + lane * NS]);
            h.x = ss_fma2(ss_decay2(delta2, a01), h.x, ss_mul2(du2, b.x));
            h.y = ss_fma2(ss_decay2(delta2, a23), h.y, ss_mul2(du2, b.y));
            if (mine && to >= 0) *reinterpret_cast<ulonglong2*>(state + (long long)to * ld_state) = h;
            float lo, hi;
            ss_unpack(ss_fma2(h.y, c.y, ss_mul2(h.x, c.x)), lo, hi);
            v[s] = lo + hi;
        }
        ask(g + SS_AHEAD);
        float y = ss_exchange<LANES, GROUP>(v, lane);
        if (t >= 0 && lane < GROUP && mine) {
            if (p.skip) y = fmaf(skip, u, y);
            if (p.z) y *= ss_silu<TU>(z);
            static_cast<TU*>(p.out)[t * p.ld_out + d] = ni_from_float<TU>(y);
        }
    }
}

// The same for numbers of states and addresses that 16-byte pieces do not fit.  Bound by its loads, number by number: 128 requests x 8,192
// channels x 5 states 21.7 us (8 by their bytes).
template <typename TU, int LANES>
__global__ void __launch_bounds__(256) selective_token_kernel(const __grid_constant__ ScanArgs p) {
    constexpr int NS = 4, GROUP = ScanGroup<LANES>::N;
    const int tid = threadIdx.x, lane = tid % LANES, mine = lane % GROUP, seq = blockIdx.y * GROUP + mine;
    const int d = blockIdx.x * (256 / LANES) + tid / LANES, n0 = lane * NS, n_real = d < p.channels ? min(NS, p.states - n0) : 0;
    const int dd = min(d, p.channels - 1);
    int t = -1, from = -1, to = -1;
    if (seq < p.n_seqs) {
        t = p.cu_q[seq];
        from = p.slots[seq];
        to = p.to_slots[seq];
        const int length = p.cu_q[seq + 1] - t;
        if (t < 0 || length <= 0 || t >= p.n_tokens) t = -1;
        if (from < 0 || from >= p.n_slots) from = -1;
        if (to < 0 || to >= p.n_slots || (t < 0 && to == from)) to = -1;
        if (length > 1) t = from = to = -1;                  // (another launch's)
    }
    const long long at = (long long)dd * p.states + n0, bc = (long long)(dd / (p.channels / p.groups)) * p.states + n0;
    float h[GROUP][NS], a[NS], b[GROUP][NS], c[GROUP][NS], v[GROUP], dt = 0.f, u = 0.f, z = 0.f;
#pragma unroll
    for (int s = 0; s < GROUP; ++s) {
        const int where = __shfl_sync(0xffffffffu, from, s, LANES);
        ss_load<NS>(p.state + max(where, 0) * p.ld_state + at, h[s], false, where >= 0 ? n_real : 0);
    }
    if (t >= 0) {
        ss_load_any<1>(p.dt, p.dt_type, t * p.ld_dt + dd, &dt, false, 1);
        ss_load<1>(static_cast<const TU*>(p.u) + t * p.ld_u + dd, &u, false, 1);
        if (p.z) ss_load<1>(static_cast<const TU*>(p.z) + t * p.ld_z + dd, &z, false, 1);
    }
    ss_load<NS>(p.a + at, a, false, n_real);
#pragma unroll
    for (int s = 0; s < GROUP; ++s) {
        const int row = __shfl_sync(0xffffffffu, t, s, LANES);
        ss_load_any<NS>(p.b, p.bc_type, max(row, 0) * p.ld_b + bc, b[s], false, row >= 0 ? n_real : 0);
        ss_load_any<NS>(p.c, p.bc_type, max(row, 0) * p.ld_c + bc, c[s], false, row >= 0 ? n_real : 0);
    }
    const float skip = p.skip ? p.skip[dd] : 0.f;
    float delta = dt + (p.dt_bias ? p.dt_bias[dd] : 0.f);
    if (p.softplus) delta = ss_softplus(delta);
    if (t < 0) delta = 0.f;                     // no token: a decay of exactly one, nothing comes in
    const float du = t < 0 ? 0.f : delta * u;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        a[i] *= SS_LOG2E;
        if (fabsf(a[i]) == INFINITY) a[i] = copysignf(3e38f, a[i]);           // (times a delta of zero: zero)
    }
#pragma unroll
    for (int s = 0; s < GROUP; ++s) {
        const float delta_s = __shfl_sync(0xffffffffu, delta, s, LANES), du_s = __shfl_sync(0xffffffffu, du, s, LANES);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float next = fmaf(ss_decay(delta_s, a[i]), h[s][i], du_s * b[s][i]);
            h[s][i] = i < n_real ? next : 0.f;          // (states that do not exist stay zero whatever delta u is)
        }
        v[s] = fmaf(h[s][2], c[s][2], h[s][0] * c[s][0]) + fmaf(h[s][3], c[s][3], h[s][1] * c[s][1]);       // (the other kernels' order)
    }
    float y = ss_exchange<LANES, GROUP>(v, lane);
    if (t >= 0 && lane < GROUP && d < p.channels) {
        if (p.skip) y = fmaf(skip, u, y);
        if (p.z) y *= ss_silu<TU>(z);
        static_cast<TU*>(p.out)[t * p.ld_out + dd] = ni_from_float<TU>(y);
    }
#pragma unroll
    for (int s = 0; s < GROUP; ++s) {
        const int where = __shfl_sync(0xffffffffu, to, s, LANES);
        if (where >= 0) ss_store<NS>(p.state + where * p.ld_state + at, h[s], false, n_real);
    }
}

// States that fill all lanes of a channel
static bool ss_fill(int states) { return states == 8 || states == 16 || states == 32 || states == 64 || states == 128; }

NI_EXPORT int ni_selective_scan_max_states() { return 128; }

// Requests of one token or none (the kernels leave longer ones alone)
template <typename TU> static void ss_tokens(const ScanArgs& p, cudaStream_t stream) {
    const int per_group = p.channels / p.groups;
    const bool wide = ss_fill(p.states) && ss_wide(p.state, p.ld_state, NI_DTYPE_F32, 4) && ss_wide(p.a, 0, NI_DTYPE_F32, 4) &&
                      ss_wide(p.b, p.ld_b, p.bc_type, 8) && ss_wide(p.c, p.ld_c, p.bc_type, 8) &&
                      (p.ld_state | p.ld_u | p.ld_dt | p.ld_z) < (1ll << 31);
#define SS_TOKEN(L)                                                                                                                  \
    do {                                                                                                                             \
        constexpr int GROUP = ScanGroup<L>::N;                                                                                       \
        const int groups = (p.n_seqs + GROUP - 1) / GROUP;                                                                           \
        if (wide) {                                                                                                                  \
            /* as many blocks as five per SM take, each with its share of the requests */                                            \
            const int columns = (per_group + 256 / L - 1) / (256 / L) * p.groups;                                                    \
            int rows = 5 * ni_sm_count() / columns;                                                                                  \
            rows = rows < 1 ? 1 : rows > groups ? groups : rows;                                                                     \
            int per_block = (groups + rows - 1) / rows * GROUP;                                                                      \
            if (per_block > SS_TOKEN_FLOATS / (4 * L)) per_block = SS_TOKEN_FLOATS / (4 * L);                                        \
            static std::atomic<unsigned long long> asked{0};                                                                         \
            ss_more_shared(selective_tokens_kernel<TU, L>, sizeof(ScanTokenShared), asked);                                          \
            selective_tokens_kernel<TU, L>                                                                                           \
                <<<dim3(columns, (p.n_seqs + per_block - 1) / per_block), 256, sizeof(ScanTokenShared), stream>>>(p, per_block);     \
        } else {                                                                                                                     \
            selective_token_kernel<TU, L><<<dim3((p.channels + 256 / L - 1) / (256 / L), groups), 256, 0, stream>>>(p);              \
        }                                                                                                                            \
    } while (0)
    if (p.states <= 8) SS_TOKEN(2);
    else if (p.states <= 16) SS_TOKEN(4);
    else if (p.states <= 32) SS_TOKEN(8);
    else if (p.states <= 64) SS_TOKEN(16);
    else SS_TOKEN(32);
}

template <typename TU> static void ss_launch(const ScanArgs& p, cudaStream_t stream) {
    const int per_group = p.channels / p.groups;
    const int channels = p.states <= 8 ? 64 : p.states <= 16 ? 32 : p.states <= 64 ? 16 : 8, columns = (per_group + channels - 1) / channels * p.groups;
    if (p.max_q_len <= 1) return ss_tokens<TU>(p, stream);
    // A portion beside many single tokens (the others have fewer than two tokens each on the average, and four blocks or more per SM):
    // the single ones by their own kernel first.  512 tokens and 63 single ones x 4,096 channels x 16 states 45 us, all in one 91; 2,048
    // and 63 94, 133; 512 and 7 27, 32; 512 and 1 26, 22.
    int least = 0, long_seqs = p.n_seqs;
    if (p.n_tokens - p.max_q_len < 2ll * (p.n_seqs - 1) && (p.n_seqs - 1ll) * columns >= 4ll * ni_sm_count()) {
        ss_tokens<TU>(p, stream);
        least = 2;
        long_seqs = (p.n_tokens + p.max_q_len - 1) / p.max_q_len;
    }
    const bool wide = per_group % 8 == 0 && ss_fill(p.states) &&
                      ss_wide(p.u, p.ld_u, p.u_type, 8) && ss_wide(p.dt, p.ld_dt, p.dt_type, 8) && ss_wide(p.out, p.ld_out, p.u_type, 8) &&
                      (!p.z || ss_wide(p.z, p.ld_z, p.u_type, 8)) && ss_wide(p.b, p.ld_b, p.bc_type, 8) && ss_wide(p.c, p.ld_c, p.bc_type, 8);
    // What a call takes, in clocks: a token costs a block with four scanning warps 80 (2 x 64, 4 x 32, 8 x 16 lanes and channels), with
    // eight 122 (4 x 64) or 145 (16 x 16, 32 x 8), a block of a split request 1.7 times as much; a block 3,000 for itself, in a cluster
    // 7,000, also where its part is empty.  An SM takes one block at a time, clusters of four 136 in all, of eight 112.  The longest
    // request's part, or all blocks in their turns.
    auto clocks = [&](int channels, int ranks, double per_token) {
        const double part = (double)p.max_q_len / ranks, blocks = (double)((per_group + channels - 1) / channels) * p.groups * long_seqs * ranks;
        const double at_once = (double)ni_sm_count() * (ranks == 8 ? 112 : ranks == 4 ? 136 : 148) / 148, own = ranks > 1 ? 7000 : 3000;
        if (ranks > 1) per_token *= 1.7;
        double turns = blocks / at_once;
        if (long_seqs == 1 || turns < 1) turns = (double)(long long)(turns + 0.9999);
        const double all = turns * (p.n_tokens * per_token / ((double)long_seqs * ranks) + own), longest = part * per_token + own;
        return all > longest ? all : longest;
    };
    const double token = p.states <= 32 ? 80 : 145;
    int ranks = 1;
    for (int r = 2; r <= 8 && !p.stepwise && p.max_q_len >= SS_SPLIT; r *= 2)
        if (clocks(channels, r, token) < clocks(channels, ranks, token)) ranks = r;
    if (p.states <= 8) ss_scan<TU, 2, 64>(p, wide, ranks, least, stream);
    else if (p.states <= 16) {
        if (wide && !p.stepwise && clocks(64, 1, 122) < clocks(32, ranks, 80)) ss_scan<TU, 4, 64>(p, wide, 1, least, stream);
        else ss_scan<TU, 4, 32>(p, wide, ranks, least, stream);
    }
    else if (p.states <= 32) ss_scan<TU, 8, 16>(p, wide, ranks, least, stream);
    else if (p.states <= 64) ss_scan<TU, 16, 16>(p, wide, ranks, least, stream);
    else ss_scan<TU, 32, 8>(p, wide, ranks, least, stream);
}

NI_EXPORT int ni_selective_scan(const void* packed, cudaStream_t stream) {
    const ScanArgs p = *static_cast<const ScanArgs*>(packed);
    if (p.n_seqs <= 0) return NI_OK;
    if (p.channels <= 0 || p.states <= 0 || p.groups <= 0 || p.channels % p.groups || p.n_tokens < 0) return NI_ERR_BAD_ARGUMENT;
    if (p.stepwise && p.u_type != NI_DTYPE_F32) return NI_ERR_BAD_ARGUMENT;
    if (p.states > 128 || p.n_seqs > 65535) return NI_ERR_UNSUPPORTED_SIZE;
    if (p.u_type == NI_DTYPE_F32) ss_launch<float>(p, stream);
    else ss_launch<__nv_bfloat16>(p, stream);
    NI_RETURN_LAUNCH_STATUS();
}
