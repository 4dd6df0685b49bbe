// A short causal convolution over time, channel by channel, with each request's last inputs kept from call to call:
//
//     out[t, d] = act(bias[d] + sum_k weight[d, k] x[t - taps + 1 + k, d])
//
// A request's tokens are rows cu_q[i] .. cu_q[i + 1] of x; what came before them lies in row slots[i] of the state as
// [taps - 1, D] in FP32, oldest first, and the last taps - 1 inputs go to row to_slots[i].  A slot outside of the state belongs to
// no request: zeros come from there and nothing is left there.
//
// Bound by the bytes of x and out.  A thread owns four neighbouring channels (one where rows or addresses do not allow that) and a
// tile of one request's tokens, its weights and the last inputs in registers; eight rows are on their way while the eight before
// are computed.  A tile reads taps - 1 rows that its neighbour reads too, and its weights: with tiles of 8 tokens the weights were a
// third of the time at 2,048 tokens x 4,096 channels (13.6 us), so a tile is as long as SC_BLOCKS blocks per SM allow: 12 us, 2.8
// TB/s, of which 4 are the launch and a block's first loads.  Seven ragged requests of 1,123 tokens in all x 1,031 channels in FP32 4.8.
#include "common.cuh"

#define SC_MAX_TAPS 8
#define SC_V 4
#define SC_ROWS 8              /* in flight; tiles are multiples of it */
#define SC_BLOCKS 4
#define SC_LONGEST 64

struct ConvArgs {
    const void* x;
    const float *weight, *bias;
    float* state;
    const int *cu_q, *slots, *to_slots;
    void* out;
    long long ld_x, ld_out, ld_state;
    int n_tokens, n_seqs, n_slots, channels, taps, type, silu, max_q_len;
};

// V neighbouring numbers of a row, as they lie in memory
template <typename T, int V> struct ConvRaw {
    uint32_t w[V * sizeof(T) / 4 > 0 ? V * sizeof(T) / 4 : 1];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
        else if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(*p);
        else w[0] = (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16;
    }
    __device__ __forceinline__ void get(float* v) const {
        if constexpr (V == 1 || sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                v[i] = __uint_as_float(w[i / 2] << 16);
                v[i + 1] = __uint_as_float(w[i / 2] & 0xffff0000u);
            }
        }
    }
};
template <typename T, int V> __device__ __forceinline__ void sc_store(T* p, const float* v) {
    if constexpr (V == 1) {
        *p = ni_from_float<T>(v[0]);
    } else if constexpr (V * sizeof(T) == 16) {
        NiVec16<T>::store(p, v);
    } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
}
// V neighbouring FP32 numbers
template <int V> __device__ __forceinline__ void sc_load_f32(const float* p, float* v) {
    if constexpr (V == 1) {
        v[0] = p[0];
    } else {
#pragma unroll
        for (int c = 0; c < V; c += 4) NiVec16<float>::load(p + c, v + c);
    }
}
template <int V> __device__ __forceinline__ void sc_store_f32(float* p, const float* v) {
    if constexpr (V == 1) {
        p[0] = v[0];
    } else {
#pragma unroll
        for (int c = 0; c < V; c += 4) NiVec16<float>::store(p + c, v + c);
    }
}
// The weights of a thread's V channels, tap by tap, and their bias.  A thread's V TAPS weights lie side by side, so a warp's loads of
// them would touch 32 lines each: the warp's weights come in whole lines and change owners in shared memory, where a thread's
// stretch is an odd number of 16-byte pieces (no two of eight threads in one bank).
template <int V, int TAPS> struct ConvWeights {
    static constexpr int PIECES = V * TAPS / 4, STRIDE = PIECES | 1;
    float4 w[V > 1 ? 4 : 1][V > 1 ? 32 * STRIDE : 1];
};
template <int V, int TAPS>
__device__ __forceinline__ void sc_weights(const ConvArgs& p, int d, ConvWeights<V, TAPS>& s, float (&w)[TAPS][V], float (&bias)[V]) {
    float flat[V * TAPS];
    if constexpr (V > 1) {
        constexpr int PIECES = ConvWeights<V, TAPS>::PIECES, STRIDE = ConvWeights<V, TAPS>::STRIDE;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const float4* from = reinterpret_cast<const float4*>(p.weight + (long long)(d - lane * V) * TAPS);
        const int there = min(32, (p.channels - (d - lane * V)) / V) * PIECES;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = i * 32 + lane;
            if (at < there) s.w[warp][at / PIECES * STRIDE + at % PIECES] = from[at];
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PIECES; ++i) *reinterpret_cast<float4*>(flat + 4 * i) = s.w[warp][lane * STRIDE + i];
    } else {
#pragma unroll
        for (int i = 0; i < TAPS; ++i) flat[i] = d < p.channels ? p.weight[(long long)d * TAPS + i] : 0.f;
    }
#pragma unroll
    for (int c = 0; c < V; ++c) bias[c] = p.bias && d < p.channels ? p.bias[d + c] : 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
        for (int k = 0; k < TAPS; ++k) w[k][c] = flat[c * TAPS + k];
}

struct ScTrue { static constexpr bool value = true; };
struct ScFalse { static constexpr bool value = false; };
typedef unsigned long long sc_pair;            // two floats side by side
__device__ __forceinline__ sc_pair sc_pack(float lo, float hi) {
    sc_pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void sc_unpack(sc_pair v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ sc_pair sc_fma2(sc_pair a, sc_pair b, sc_pair c) {
    sc_pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ sc_pair sc_mul2(sc_pair a, sc_pair b) {
    sc_pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// silu of two numbers in 16 bits: 2^x and the reciprocal of the hardware (a few 2^-24 off, where the result is rounded to 2^-8)
__device__ __forceinline__ sc_pair sc_silu2(sc_pair v) {
    float x0, x1;
    sc_unpack(sc_mul2(v, sc_pack(-1.44269504f, -1.44269504f)), x0, x1);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x1));
    sc_unpack(sc_fma2(sc_pack(x0, x1), sc_pack(1.f, 1.f), sc_pack(1.f, 1.f)), x0, x1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x1));
    return sc_mul2(v, sc_pack(x0, x1));
}

// silu in FP32, v / (1 + exp(-v)): the quotient by the hardware's reciprocal, put right by what it leaves, with the errors of a division
// (2,048 tokens x 4,096 channels 15 us, 26 by a division); where that is no number (infinities) as it is, below 1e-36 zero.
__device__ __forceinline__ float sc_silu_f32(float v) {
    const float d = 1.f + expf(-v);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    const float q = v * r, better = fmaf(fmaf(-d, q, v), r, q);
    return better == better ? better : q;
}

// One token's row: the taps' sum, its activation, the rounding.  Four channels go two by two (half the instructions).
template <typename T, int V, int TAPS>
__device__ __forceinline__ void sc_token(const ConvArgs& p, T* out, const float (&w)[TAPS][V], const float (&bias)[V], const float (&seen)[TAPS][V]) {
    float v[V];
    if constexpr (V > 1) {
#pragma unroll
        for (int c = 0; c < V; c += 2) {
            sc_pair x = sc_pack(bias[c], bias[c + 1]);
#pragma unroll
            for (int k = 0; k < TAPS; ++k) x = sc_fma2(sc_pack(w[k][c], w[k][c + 1]), sc_pack(seen[k][c], seen[k][c + 1]), x);
            if (sizeof(T) == 2 && p.silu) x = sc_silu2(x);
            sc_unpack(x, v[c], v[c + 1]);
        }
    } else {
        v[0] = bias[0];
#pragma unroll
        for (int k = 0; k < TAPS; ++k) v[0] = fmaf(w[k][0], seen[k][0], v[0]);
        if (sizeof(T) == 2 && p.silu) {
            float same;
            sc_unpack(sc_silu2(sc_pack(v[0], v[0])), v[0], same);
        }
    }
    if (sizeof(T) == 4 && p.silu)
#pragma unroll
        for (int c = 0; c < V; ++c) v[c] = sc_silu_f32(v[c]);
    sc_store<T, V>(out, v);
}

template <typename T, int V, int TAPS>
__global__ void __launch_bounds__(128) short_convolution_kernel(const __grid_constant__ ConvArgs p, const int tile_len) {
    constexpr int KEPT = TAPS - 1;
    __shared__ ConvWeights<V, TAPS> weights;
    // The request and tile behind this block's number: request i's tiles begin at cu_q[i] / tile_len + i, which leaves each of them a tile
    // or more.  Blocks below the first one's (cu_q[0] rows belong to no request) have nothing to do: they end, since a tile must be one
    // block's alone.  Every warp looks at 32 places at a time: 1,024 requests take two loads (a walk over all lengths before a block's
    // request took 2,000 requests of two tokens x 1,024 channels from 31 to 93 us, 256 x 4,096 from 17 to 21).
    int seq = 0, tile = blockIdx.x;
    for (int n = p.n_seqs; n > 1;) {
        const int step = (n + 31) / 32, i = seq + (int)(threadIdx.x & 31) * step;
        const bool there = (int)(threadIdx.x & 31) * step < n;
        const int begin = there ? max(0, min(p.cu_q[i], p.n_tokens)) / tile_len + i : 0;
        const int k = __popc(__ballot_sync(0xffffffffu, there && begin <= (int)blockIdx.x)) - 1;
        if (k < 0) return;                      // (the whole block: every warp has looked at the same places)
        tile = max((int)blockIdx.x - __shfl_sync(0xffffffffu, begin, k), 0);
        seq += k * step;
        n = min(step, n - k * step);
    }
    const int d = (blockIdx.y * 128 + threadIdx.x) * V;
    const bool mine = d < p.channels;
    const int first = max(0, min(p.cu_q[seq], p.n_tokens)), end = max(first, min(p.cu_q[seq + 1], p.n_tokens));
    const long long t0 = first + (long long)tile * tile_len;
    if (t0 >= end && tile > 0) return;
    const int n = mine ? (int)min((long long)tile_len, end - t0) : 0;
    const T* x = static_cast<const T*>(p.x) + d;
    T* out = static_cast<T*>(p.out) + d;
    const int from = p.slots[seq];
    const bool any = mine && from >= 0 && from < p.n_slots;
    const float* old = p.state + (any ? from : 0) * p.ld_state + d;
    ConvRaw<T, V> raw[SC_ROWS], next[SC_ROWS], before[KEPT > 0 ? KEPT : 1];
#pragma unroll
    for (int j = 0; j < SC_ROWS; ++j)
        if (j < n) raw[j].load(x + (t0 + j) * p.ld_x);
    float seen[TAPS][V], w[TAPS][V], bias[V];
    if (tile > 0 && mine) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) before[i].load(x + (t0 - KEPT + i) * p.ld_x);
    }
    sc_weights<V, TAPS>(p, d, weights, w, bias);
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {          // the inputs before the tile: of this call, or kept (a first tile has them all kept)
        if (tile > 0) {
            before[i].get(seen[i]);
        } else if (any) {
            sc_load_f32<V>(old + (long long)i * p.channels, seen[i]);
        } else {
#pragma unroll
            for (int c = 0; c < V; ++c) seen[i][c] = 0.f;
        }
    }
    for (int t = 0; t < n; t += SC_ROWS) {
        const int rows = n - t;
        const T* then = x + (t0 + t + SC_ROWS) * p.ld_x;
        T* here = out + (t0 + t) * p.ld_out;
#pragma unroll
        for (int j = 0; j < SC_ROWS; ++j)
            if (SC_ROWS + j < rows) next[j].load(then + j * p.ld_x);
        auto walk = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < SC_ROWS; ++j)
                if (whole.value || j < rows) {
                    raw[j].get(seen[KEPT]);
                    sc_token<T, V, TAPS>(p, here + j * p.ld_out, w, bias, seen);
#pragma unroll
                    for (int i = 0; i < KEPT; ++i)
#pragma unroll
                        for (int c = 0; c < V; ++c) seen[i][c] = seen[i + 1][c];
                }
        };
        if (rows >= SC_ROWS) walk(ScTrue{});
        else walk(ScFalse{});
#pragma unroll
        for (int j = 0; j < SC_ROWS; ++j) raw[j] = next[j];
    }
    if (tile == 0) {           // what is kept of this call: these threads alone have read the old inputs, so they may write over them
        const int to = p.to_slots[seq], length = end - first;
        if (KEPT > 0 && to >= 0 && to < p.n_slots && (length > 0 || to != from)) {
#pragma unroll
            for (int i = 0; i < KEPT; ++i) {
                const int at = length - KEPT + i;                  // in this call's tokens, or before them
                float v[V];
                if (at >= 0) {
                    ConvRaw<T, V> r;
                    r.load(x + (long long)(first + at) * p.ld_x);
                    r.get(v);
                } else if (any) {              // (row length + i: behind the rows written so far, where both are one state)
                    sc_load_f32<V>(old + (long long)(at + KEPT) * p.channels, v);
                } else {
#pragma unroll
                    for (int c = 0; c < V; ++c) v[c] = 0.f;
                }
                sc_store_f32<V>(p.state + to * p.ld_state + (long long)i * p.channels + d, v);
            }
        }
    }
}

// Requests of one token each, four channels a thread: the kept inputs move up by one.  Bound by its one chain of loads: 64 requests x
// 8,192 channels 4.3 us.
template <typename T, int V, int TAPS>
__global__ void __launch_bounds__(128) short_convolution_token_kernel(const __grid_constant__ ConvArgs p) {
    constexpr int KEPT = TAPS - 1;
    __shared__ ConvWeights<V, TAPS> weights;
    const int seq = blockIdx.x, d = (blockIdx.y * 128 + threadIdx.x) * V;
    const int t = p.cu_q[seq], next = p.cu_q[seq + 1], from = p.slots[seq], to = p.to_slots[seq];
    float seen[TAPS][V], w[TAPS][V], bias[V];
    const bool mine = d < p.channels, token = mine && t >= 0 && t < next && t < p.n_tokens, any = mine && from >= 0 && from < p.n_slots;
    ConvRaw<T, V> raw;
    if (token) raw.load(static_cast<const T*>(p.x) + t * p.ld_x + d);
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
#pragma unroll
        for (int c = 0; c < V; ++c) seen[i][c] = 0.f;
        if (any) sc_load_f32<V>(p.state + from * p.ld_state + (long long)i * p.channels + d, seen[i]);
    }
    sc_weights<V, TAPS>(p, d, weights, w, bias);
    if (token) {
        raw.get(seen[KEPT]);
        sc_token<T, V, TAPS>(p, static_cast<T*>(p.out) + t * p.ld_out + d, w, bias, seen);
    }
    if (mine && to >= 0 && to < p.n_slots && (token || to != from))
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            sc_store_f32<V>(p.state + to * p.ld_state + (long long)i * p.channels + d, seen[token ? i + 1 : i]);
}

NI_EXPORT int ni_short_convolution_max_taps() { return SC_MAX_TAPS; }

template <typename T> static int sc_launch(const ConvArgs& p, cudaStream_t stream) {
    constexpr int V = SC_V;
    auto apart16 = [](const void* q, long long bytes) { return (reinterpret_cast<size_t>(q) & 15) == 0 && bytes % 16 == 0; };
    const bool wide = p.channels % V == 0 && apart16(p.x, p.ld_x * sizeof(T)) && apart16(p.out, p.ld_out * sizeof(T)) &&
                      apart16(p.weight, 0) && (p.taps == 1 || apart16(p.state, p.ld_state * 4));
    const bool tokens = p.max_q_len <= 1;
    const int threads = wide ? p.channels / V : p.channels;
    if (threads > 65535 * 128) return NI_ERR_UNSUPPORTED_SIZE;
    const int columns = (threads + 127) / 128;
    const long long share = ((long long)p.n_tokens * columns / (SC_BLOCKS * ni_sm_count()) + SC_ROWS - 1) / SC_ROWS * SC_ROWS;
    const int tile_len = (int)(share < SC_ROWS ? SC_ROWS : share > SC_LONGEST ? SC_LONGEST : share);
    const long long tiles = tokens ? p.n_seqs : p.n_tokens / tile_len + (long long)p.n_seqs;
    const dim3 grid((unsigned)tiles, columns);
#define SC_CASE(K)                                                                                       \
    case K:                                                                                              \
        if (tokens && wide) short_convolution_token_kernel<T, V, K><<<grid, 128, 0, stream>>>(p);        \
        else if (tokens) short_convolution_token_kernel<T, 1, K><<<grid, 128, 0, stream>>>(p);           \
        else if (wide) short_convolution_kernel<T, V, K><<<grid, 128, 0, stream>>>(p, tile_len);         \
        else short_convolution_kernel<T, 1, K><<<grid, 128, 0, stream>>>(p, tile_len);                   \
        break;
    switch (p.taps) {
        SC_CASE(1) SC_CASE(2) SC_CASE(3) SC_CASE(4) SC_CASE(5) SC_CASE(6) SC_CASE(7) SC_CASE(8)
    }
    return NI_OK;
}

NI_EXPORT int ni_short_convolution(const void* packed, cudaStream_t stream) {
    const ConvArgs p = *static_cast<const ConvArgs*>(packed);
    if (p.n_seqs <= 0) return NI_OK;
    if (p.channels <= 0 || p.taps <= 0 || p.n_tokens < 0) return NI_ERR_BAD_ARGUMENT;
    if (p.taps > SC_MAX_TAPS || p.n_seqs > 65535) return NI_ERR_UNSUPPORTED_SIZE;
    const int code = p.type == NI_DTYPE_F32 ? sc_launch<float>(p, stream) : sc_launch<__nv_bfloat16>(p, stream);
    if (code != NI_OK) return code;
    NI_RETURN_LAUNCH_STATUS();
}
