// rotary.hip -- rotary positions of q and k, and their gradient.
//
// Pair i of a head at position p turns by the angle p * step_i, in turns of
// 2^64: the product wraps modulo one turn, so the fraction keeps its accuracy
// at any position (32 bits of it are used, 1.5e-9 rad).  Bound by memory: each
// element is read and written once.  A thread owns one vector of pairs of a
// token, takes its sines and cosines once and walks heads with them.
#include "block_ops.hpp"

#include <algorithm>
#include <cmath>

namespace sili {

namespace {

constexpr unsigned TPB = 256;

// V pairs (or, past the rotated channels, V copied channels) of one head.
template <typename T, int V, bool HALF>
__device__ __forceinline__ void turn(const T *x, T *y, int rot, int i, const float (&c)[V], const float (&s)[V]) {
    if (HALF) {
        float a[V], b[V], u[V], w[V];
        load_pack<T, V>(x + i, a);
        load_pack<T, V>(x + rot / 2 + i, b);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            u[j] = a[j] * c[j] - b[j] * s[j];
            w[j] = b[j] * c[j] + a[j] * s[j];
        }
        store_pack<T, V>(y + i, u);
        store_pack<T, V>(y + rot / 2 + i, w);
    } else {
        float a[2 * V], u[2 * V];
        load_pack<T, 2 * V>(x + 2 * i, a);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            u[2 * j] = a[2 * j] * c[j] - a[2 * j + 1] * s[j];
            u[2 * j + 1] = a[2 * j + 1] * c[j] + a[2 * j] * s[j];
        }
        store_pack<T, 2 * V>(y + 2 * i, u);
    }
}

// Thread: (token, unit); units [0, rot / 2 / V) turn V pairs, the rest copy V
// channels.  blockIdx.y cuts the heads (q's, then k's) into shares.
template <typename T, int V, bool HALF>
__global__ __launch_bounds__(TPB) void k_rotary(sili_rotary_args a, int units, int share) {
    const int64_t id = (int64_t)blockIdx.x * TPB + threadIdx.x;
    const int64_t t = id / units;
    const int unit = (int)(id - t * units);
    if (t >= a.tokens) return;
    const int rot = (int)a.rot_dim, turning = rot / 2 / V;
    float c[V], s[V];
    const int i = unit * V;
    if (unit < turning) {
        const int64_t p = a.positions[t];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint64_t phase = (uint64_t)p * a.phase_steps[i + j];
            const float half_turns = (float)(int32_t)(phase >> 32) * 0x1p-31f;
            sincospif(half_turns, &s[j], &c[j]);
            c[j] *= a.scale;
            s[j] *= a.inverse ? -a.scale : a.scale;
        }
    }
    const int heads = (int)(a.q_heads + a.k_heads);
    const int h0 = blockIdx.y * share, h1 = min(h0 + share, heads);
    for (int h = h0; h < h1; ++h) {
        const bool isq = h < a.q_heads;
        const int64_t g = isq ? h : h - a.q_heads;
        const T *x = isq ? (const T *)a.q + t * a.q_token_stride + g * a.q_head_stride
                         : (const T *)a.k + t * a.k_token_stride + g * a.k_head_stride;
        T *y = isq ? (T *)a.q_out + t * a.q_out_token_stride + g * a.q_out_head_stride
                   : (T *)a.k_out + t * a.k_out_token_stride + g * a.k_out_head_stride;
        if (unit < turning) turn<T, V, HALF>(x, y, rot, i, c, s);
        else {
            const int at = rot + (unit - turning) * V;
            *reinterpret_cast<Pack<T, V> *>(y + at) = *reinterpret_cast<const Pack<T, V> *>(x + at);
        }
    }
}

template <typename T, int V>
void run(const sili_rotary_args &a, hipStream_t st) {
    const int64_t units = a.rot_dim / 2 / V + (a.head_dim - a.rot_dim) / V;
    const int64_t blocks = (a.tokens * units + TPB - 1) / TPB, heads = a.q_heads + a.k_heads;
    require(blocks <= INT32_MAX, "rotary: too many tokens");
    // heads a thread walks: as few as fill the GPU (2048 blocks), since the
    // sines are worth about one head's traffic
    const int64_t shares = std::clamp<int64_t>(2048 / std::max<int64_t>(blocks, 1), 1, heads);
    const int share = (int)((heads + shares - 1) / shares);
    const dim3 grid((unsigned)blocks, (unsigned)((heads + share - 1) / share));
    if (a.layout == SILI_ROTARY_HALF) launch(k_rotary<T, V, true>, grid, dim3(TPB), 0, st, a, (int)units, share);
    else launch(k_rotary<T, V, false>, grid, dim3(TPB), 0, st, a, (int)units, share);
}

}  // namespace

void rotary(const sili_rotary_args &a, hipStream_t st) {
    require(a.tokens >= 0 && a.q_heads >= 0 && a.k_heads >= 0, "rotary: negative size");
    require(a.q_heads + a.k_heads <= 65535, "rotary: too many heads");
    require(a.head_dim > 0 && a.head_dim <= 65536, "rotary: head_dim out of range");
    require(a.rot_dim >= 0 && a.rot_dim % 2 == 0 && a.rot_dim <= a.head_dim, "rotary: rot_dim is not an even number up to head_dim");
    require(a.layout == SILI_ROTARY_HALF || a.layout == SILI_ROTARY_INTERLEAVED, "rotary: unknown layout");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "rotary: unknown dtype");
    if (a.tokens == 0 || a.q_heads + a.k_heads == 0) return;
    require((a.positions && a.phase_steps) || a.rot_dim == 0, "rotary: NULL positions or phase_steps");
    require(a.q_heads == 0 || (a.q && a.q_out), "rotary: NULL q");
    require(a.k_heads == 0 || (a.k && a.k_out), "rotary: NULL k");
    // vectors need every address and size to divide: 16 bytes of an
    // interleaved head hold half as many pairs as a run of a half layout
    const int64_t es = dtype_size(a.dtype);
    auto fits = [&](int64_t v) {
        const int64_t run = a.layout == SILI_ROTARY_HALF ? v : 2 * v;
        auto ok = [&](int64_t heads, const void *x, int64_t ts, int64_t hs) {
            return heads == 0 || (aligned(x, (size_t)(run * es)) && ts % run == 0 && hs % run == 0);
        };
        return a.rot_dim / 2 % v == 0 && a.rot_dim % run == 0 && (a.head_dim - a.rot_dim) % v == 0 &&
               ok(a.q_heads, a.q, a.q_token_stride, a.q_head_stride) && ok(a.k_heads, a.k, a.k_token_stride, a.k_head_stride) &&
               ok(a.q_heads, a.q_out, a.q_out_token_stride, a.q_out_head_stride) &&
               ok(a.k_heads, a.k_out, a.k_out_token_stride, a.k_out_head_stride);
    };
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        if (fits(4)) run<T, 4>(a, st);
        else run<T, 1>(a, st);
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
