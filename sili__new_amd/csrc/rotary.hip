// rotary.hip -- rotary positions of q and k, and their gradient.
//
// Pair i of a head at position p turns by the angle p * step_i, in turns of
// 2^64: the product wraps modulo one turn, so the fraction keeps its accuracy
// at any position.  Its upper 32 bits, as a signed part of half a turn, become a
// float: within 2^-25 of half a turn (9.4e-8 rad) at the largest angles, 1.5e-9 rad
// at small ones, where sines and cosines are fp32 anyway.  Bound by memory: each
// element is read and written once.  A thread owns one run of pairs of a token,
// 16 bytes, takes its sines and cosines once and walks heads with them, four in
// flight (8192 tokens of 48 bf16 heads of 128, half of each turned: 44 us, 4.6 TB/s;
// a head at a time, 51 us).
#include "block_ops.hpp"

#include <algorithm>
#include <cmath>

namespace sili {

namespace {

constexpr unsigned TPB = 256;

// Heads in flight: a thread asks for this many before it stores the first.
constexpr int HB = 4;

// A run of elements as one register value (a struct of them ends up in memory).
template <int BYTES> struct RawOf;
template <> struct RawOf<2> { typedef uint16_t type; };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<8> { typedef uint2 type; };
template <> struct RawOf<16> { typedef uint4 type; };
template <typename T, int N>
using Raw = typename RawOf<N * (int)sizeof(T)>::type;

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> get(const T *p) { return *reinterpret_cast<const Raw<T, N> *>(p); }
template <typename T, int N>
__device__ __forceinline__ void put(T *p, const Raw<T, N> &r) { *reinterpret_cast<Raw<T, N> *>(p) = r; }

// V pairs of one head turned: x1 and x2 in a run each (half), or in turn in one
// run of 2 V (interleaved; x2 unused).
template <typename T, int V, bool HALF>
__device__ __forceinline__ void turn(T *y, int rot, int i, Raw<T, HALF ? V : 2 * V> r1, Raw<T, HALF ? V : 2 * V> r2, const float (&c)[V],
                                     const float (&s)[V]) {
    constexpr int R = HALF ? V : 2 * V;
    using RawR = Raw<T, R>;
    const Pack<T, R> p = __builtin_bit_cast(Pack<T, R>, r1), q = __builtin_bit_cast(Pack<T, R>, r2);
    Pack<T, R> u, w;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float x1 = (float)(HALF ? p.v[j] : p.v[2 * j % R]), x2 = (float)(HALF ? q.v[j] : p.v[(2 * j + 1) % R]);
        // which product is fused is fixed, so that every variant gives the same bits
        const T y1 = (T)__builtin_fmaf(x1, c[j], -(x2 * s[j])), y2 = (T)__builtin_fmaf(x2, c[j], x1 * s[j]);
        if (HALF) {
            u.v[j] = y1;
            w.v[j] = y2;
        } else {
            u.v[2 * j % R] = y1;
            u.v[(2 * j + 1) % R] = y2;
        }
    }
    put<T, R>(y + (HALF ? i : 2 * i), __builtin_bit_cast(RawR, u));
    if (HALF) put<T, R>(y + rot / 2 + i, __builtin_bit_cast(RawR, w));
}

// Thread: (token, unit); units [0, rot / 2 / V) turn V pairs, the rest copy W
// channels.  blockIdx.y cuts the heads (q's, then k's) into shares.
template <typename T, int V, int W, bool HALF>
__global__ __launch_bounds__(TPB) void k_rotary(sili_rotary_args a, uint32_t units, int share) {
    const uint32_t id = blockIdx.x * TPB + threadIdx.x, t = id / units, unit = id - t * units;
    if (t >= (uint64_t)a.tokens) return;
    const int rot = (int)a.rot_dim, turning = rot / 2 / V;
    const bool turns = (int)unit < turning;
    const int i = turns ? (int)unit * V : rot + ((int)unit - turning) * W;
    const int nq = (int)a.q_heads, heads = nq + (int)a.k_heads;
    auto in = [&](int h) {
        return h < nq ? (const T *)a.q + t * a.q_token_stride + h * a.q_head_stride
                      : (const T *)a.k + t * a.k_token_stride + (h - nq) * a.k_head_stride;
    };
    auto out = [&](int h) {
        return h < nq ? (T *)a.q_out + t * a.q_out_token_stride + h * a.q_out_head_stride
                      : (T *)a.k_out + t * a.k_out_token_stride + (h - nq) * a.k_out_head_stride;
    };
    const int h1 = min((int)(blockIdx.y + 1) * share, heads);
    if (!turns) {
        for (int h = blockIdx.y * share; h < h1; h += HB) {
            Raw<T, W> p[HB];
#pragma unroll
            for (int k = 0; k < HB; ++k) p[k] = get<T, W>(in(min(h + k, h1 - 1)) + i);
#pragma unroll
            for (int k = 0; k < HB; ++k)
                if (h + k < h1) put<T, W>(out(h + k) + i, p[k]);
        }
        return;
    }
    float c[V], s[V];
    const int64_t pos = a.positions[t];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint64_t phase = (uint64_t)pos * a.phase_steps[i + j];
        sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s[j], &c[j]);
        c[j] *= a.scale;
        s[j] *= a.inverse ? -a.scale : a.scale;
    }
    for (int h = blockIdx.y * share; h < h1; h += HB) {
        constexpr int R = HALF ? V : 2 * V;
        Raw<T, R> x1[HB], x2[HB];
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            const T *x = in(min(h + k, h1 - 1));
            x1[k] = get<T, R>(x + (HALF ? i : 2 * i));
            x2[k] = HALF ? get<T, R>(x + rot / 2 + i) : x1[k];
        }
#pragma unroll
        for (int k = 0; k < HB; ++k)
            if (h + k < h1) turn<T, V, HALF>(out(h + k), rot, i, x1[k], x2[k], c, s);
    }
}

template <typename T, int V, int W, bool HALF>
void run(const sili_rotary_args &a, hipStream_t st) {
    const int64_t units = a.rot_dim / 2 / V + (a.head_dim - a.rot_dim) / W;
    const int64_t blocks = (a.tokens * units + TPB - 1) / TPB, heads = a.q_heads + a.k_heads;
    require(a.tokens * units < (int64_t(1) << 32) - TPB, "rotary: too many tokens");
    // heads a thread walks: as few as fill the GPU (2048 blocks), but the HB that
    // it has in flight, since the sines are worth about one head's traffic
    const int64_t shares = std::clamp<int64_t>(2048 / std::max<int64_t>(blocks, 1), 1, heads);
    int64_t share = (heads + shares - 1) / shares;
    if (share > 1) share = (share + HB - 1) / HB * HB;
    launch(k_rotary<T, V, W, HALF>, dim3((unsigned)blocks, (unsigned)((heads + share - 1) / share)), dim3(TPB), 0, st, a,
           (uint32_t)units, (int)share);
}

}  // namespace

void rotary(const sili_rotary_args &a, hipStream_t st) {
    require(a.tokens >= 0 && a.q_heads >= 0 && a.k_heads >= 0, "rotary: negative size");
    require(a.tokens < (int64_t(1) << 31), "rotary: too many tokens");
    require(a.q_heads <= 65535 && a.k_heads <= 65535 && a.q_heads + a.k_heads <= 65535, "rotary: too many heads");
    require(a.head_dim > 0 && a.head_dim <= 65536, "rotary: head_dim out of range");
    require(a.rot_dim >= 0 && a.rot_dim % 2 == 0 && a.rot_dim <= a.head_dim, "rotary: rot_dim is not an even number up to head_dim");
    require(a.layout == SILI_ROTARY_HALF || a.layout == SILI_ROTARY_INTERLEAVED, "rotary: unknown layout");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "rotary: unknown dtype");
    if (a.tokens == 0 || a.q_heads + a.k_heads == 0) return;
    require((a.positions && a.phase_steps) || a.rot_dim == 0, "rotary: NULL positions or phase_steps");
    require(a.q_heads == 0 || (a.q && a.q_out), "rotary: NULL q");
    require(a.k_heads == 0 || (a.k && a.k_out), "rotary: NULL k");
    // 16-byte runs need every address, stride and size to divide them
    const int64_t es = dtype_size(a.dtype), run_len = 16 / es;
    const bool half = a.layout == SILI_ROTARY_HALF;
    auto ok = [&](int64_t heads, const void *x, int64_t ts, int64_t hs) {
        return heads == 0 || (aligned(x, 16) && ts % run_len == 0 && hs % run_len == 0);
    };
    const bool fits = (half ? a.rot_dim / 2 : a.rot_dim) % run_len == 0 && (a.head_dim - a.rot_dim) % run_len == 0 &&
                      ok(a.q_heads, a.q, a.q_token_stride, a.q_head_stride) && ok(a.k_heads, a.k, a.k_token_stride, a.k_head_stride) &&
                      ok(a.q_heads, a.q_out, a.q_out_token_stride, a.q_out_head_stride) &&
                      ok(a.k_heads, a.k_out, a.k_out_token_stride, a.k_out_head_stride);
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        constexpr int N = 16 / (int)sizeof(T);
        if (half) fits ? run<T, N, N, true>(a, st) : run<T, 1, 1, true>(a, st);
        else fits ? run<T, N / 2, N, false>(a, st) : run<T, 1, 1, false>(a, st);
    });
    SILI_HIP(hipGetLastError());
}

void rotary_steps(int64_t rot_dim, double base, int scaling, double factor, double original_len, double low,
                  double high, uint64_t *steps, float *scale) {
    require(rot_dim >= 0 && rot_dim % 2 == 0, "rotary_steps: rot_dim is not an even number");
    require(base > 1.0 && std::isfinite(base), "rotary_steps: base must be above 1");
    require(scaling >= SILI_ROTARY_PLAIN && scaling <= SILI_ROTARY_BASE, "rotary_steps: unknown scaling");
    require(scaling == SILI_ROTARY_PLAIN || (factor >= 1.0 && std::isfinite(factor)), "rotary_steps: factor must be at least 1");
    require(scaling != SILI_ROTARY_BANDS || (original_len > 0.0 && low < high), "rotary_steps: bands need original_len > 0 and low < high");
    require(scaling != SILI_ROTARY_BASE || rot_dim > 2, "rotary_steps: a changed base needs rot_dim > 2");
    constexpr double TAU = 6.283185307179586476925;
    const double n = (double)rot_dim;
    if (scaling == SILI_ROTARY_BASE) base *= std::pow(factor, n / (n - 2.0));
    for (int64_t i = 0; i < rot_dim / 2; ++i) {
        double turns = std::pow(base, -2.0 * (double)i / n) / TAU;  // below 1 / TAU
        if (scaling == SILI_ROTARY_LINEAR) turns /= factor;
        else if (scaling == SILI_ROTARY_BANDS) {
            const double keep = std::clamp((turns * original_len - low) / (high - low), 0.0, 1.0);
            turns *= (1.0 - keep) / factor + keep;
        }
        steps[i] = (uint64_t)std::nearbyint(turns * 0x1p64);
    }
    *scale = scaling == SILI_ROTARY_BANDS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
}

}  // namespace sili
