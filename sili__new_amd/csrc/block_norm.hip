// block_norm.hip -- the norm after a block, its gate and residual scale, and
// the norm before the next block, forward and backward.
//
//   n = u r1 w1,  y = b x + a g n,  h = y r2 w2,   r = rsqrt(mean(.^2) + eps)
//   gy  = dy + r2 (w2 dh - yh mean(w2 dh yh)),     yh = y r2
//   dx  = b gy,  dn = a g gy,  dg = a n gy,  dw2 = sum dh yh,  dw1 = sum dn uh
//   du  = r1 (w1 dn - uh mean(w1 dn uh)),          uh = u r1
#include "block_ops.hpp"
#include "wave.hpp"

#include <algorithm>

namespace sili {

namespace {

constexpr unsigned TPB = 256;
constexpr int64_t WIDEST = 32768;

// ---- rows of any width ----------------------------------------------------------
// Rows of more than 8192 channels: a block a row, what is between its passes in LDS,
// the sums over tokens in the workspace.

// Sum over the block, in a fixed order.
__device__ __forceinline__ float block_sum(float v, float (&part)[TPB / 64]) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (unsigned w = 0; w < TPB / 64; ++w) s += part[w];
    return s;
}

template <typename T>
__global__ __launch_bounds__(TPB) void k_norm_fwd(sili_block_norm_args a) {
    extern __shared__ float s_row[];  // y
    __shared__ float s_part[TPB / 64];
    const int64_t t = blockIdx.x;
    const int n = (int)a.width;
    const T *u = (const T *)a.u + t * a.u_stride;
    const T *x = a.x ? (const T *)a.x + t * a.x_stride : nullptr;
    const T *gate = a.gate ? (const T *)a.gate + t * a.gate_stride : nullptr;
    float r1 = 1.0f;
    if (a.w_post) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < n; i += TPB) s += (float)u[i] * (float)u[i];
        r1 = rsqrtf(block_sum(s, s_part) / (float)n + a.eps);
        if (a.rstd_post && threadIdx.x == 0) a.rstd_post[t] = r1;
    }
    float s = 0.0f;
    for (int i = threadIdx.x; i < n; i += TPB) {
        float v = (float)u[i];
        if (a.w_post) v *= r1 * a.w_post[i];
        if (gate) v *= (float)gate[i];
        v *= a.u_scale;
        if (x) v += a.x_scale * (float)x[i];
        s_row[i] = v;
        s += v * v;
    }
    float r2 = 0.0f;
    if (a.w_pre) {
        r2 = rsqrtf(block_sum(s, s_part) / (float)n + a.eps);
        if (a.rstd_pre && threadIdx.x == 0) a.rstd_pre[t] = r2;
    }
    // y may be x and h may be u: every thread writes only elements it alone has read
    for (int i = threadIdx.x; i < n; i += TPB) {
        ((T *)a.y)[t * a.y_stride + i] = (T)s_row[i];
        if (a.w_pre) ((T *)a.h)[t * a.h_stride + i] = (T)(s_row[i] * r2 * a.w_pre[i]);
    }
}

// Rows t = blockIdx.x, + gridDim.x, ...; each thread sums its channels' weight
// and gate gradients over them into part[3][blocks][width].
template <typename T>
__global__ __launch_bounds__(TPB) void k_norm_bwd(sili_block_norm_args a, sili_block_norm_grads g) {
    extern __shared__ float s_row[];  // gy, then the three sums
    __shared__ float s_part[TPB / 64];
    const int n = (int)a.width;
    float *gy = s_row;
    float *part = (float *)g.workspace + (int64_t)blockIdx.x * n;
    const int64_t plane = (int64_t)gridDim.x * n;
    const bool shared_gate = a.gate && g.dgate && a.gate_stride == 0;
    bool begun = false;
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const T *u = (const T *)a.u + t * a.u_stride;
        const T *y = (const T *)a.y + t * a.y_stride;
        const T *gate = a.gate ? (const T *)a.gate + t * a.gate_stride : nullptr;
        const T *dy = g.dy ? (const T *)g.dy + t * g.dy_stride : nullptr;
        const T *dh = g.dh ? (const T *)g.dh + t * g.dh_stride : nullptr;
        const float r2 = dh ? a.rstd_pre[t] : 0.0f, r1 = a.w_post ? a.rstd_post[t] : 1.0f;
        float m2 = 0.0f;
        if (dh) {
            float s = 0.0f;
            for (int i = threadIdx.x; i < n; i += TPB) s += a.w_pre[i] * (float)dh[i] * ((float)y[i] * r2);
            m2 = block_sum(s, s_part) / (float)n;
        }
        float s = 0.0f;
        for (int i = threadIdx.x; i < n; i += TPB) {
            float v = dy ? (float)dy[i] : 0.0f;
            if (dh) {
                const float yh = (float)y[i] * r2;
                v += r2 * (a.w_pre[i] * (float)dh[i] - yh * m2);
                if (g.dw_pre) part[2 * plane + i] = (begun ? part[2 * plane + i] : 0.0f) + (float)dh[i] * yh;
            }
            gy[i] = v;
            if (g.dx) ((T *)g.dx)[t * g.dx_stride + i] = (T)(a.x_scale * v);
            if (a.w_post) s += a.w_post[i] * (a.u_scale * v * (gate ? (float)gate[i] : 1.0f)) * ((float)u[i] * r1);
        }
        const float m1 = a.w_post ? block_sum(s, s_part) / (float)n : 0.0f;
        for (int i = threadIdx.x; i < n; i += TPB) {
            const float v = a.u_scale * gy[i], uh = (float)u[i] * r1, w = a.w_post ? a.w_post[i] : 1.0f;
            const float dn = gate ? v * (float)gate[i] : v;
            if (gate && g.dgate) {
                if (shared_gate) part[i] = (begun ? part[i] : 0.0f) + v * uh * w;
                else ((T *)g.dgate)[t * g.dgate_stride + i] = (T)(v * uh * w);
            }
            if (a.w_post && g.dw_post) part[plane + i] = (begun ? part[plane + i] : 0.0f) + dn * uh;
            if (g.du) ((T *)g.du)[t * g.du_stride + i] = (T)(a.w_post ? r1 * (w * dn - uh * m1) : dn);
        }
        begun = true;
    }
}

// ---- rows of up to 8 channels a thread ------------------------------------------
// A block walks rows t = blockIdx.x, + gridDim.x, ... with its channels' weights
// (and, backward, their gradients' sums) in registers, so each element of a row
// crosses memory once, and asks for the next row before it reduces this one.
// Memory bounds it: 8192 rows of 5120 bf16 channels forward 79 us (4.2 TB/s),
// backward 122 (4.1; a block a row with its row in LDS took 271 and 1251).
// Thread: NV vectors of V channels, channel (k * blockDim.x + thread) * V.

// Sum over the block, in a fixed order, one barrier a sum: consecutive sums take
// the two halves of part in turn.
struct BlockSum {
    float (*part)[16];
    int turn = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = wave_sum(v);
        const int waves = blockDim.x >> 6;
        if (waves == 1) return v;
        float *p = part[turn];
        turn ^= 1;
        if ((threadIdx.x & 63u) == 0u) p[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.0f;
        for (int w = 0; w < waves; ++w) s += p[w];
        return s;
    }
};

template <typename T, int V, int NV>
struct Row {
    Pack<T, V> v[NV];
    __device__ __forceinline__ void load(const void *base, int64_t offset, int n) {
        const T *p = (const T *)base + offset;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = (k * (int)blockDim.x + (int)threadIdx.x) * V;
            if (i < n) v[k] = *reinterpret_cast<const Pack<T, V> *>(p + i);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) v[k].v[j] = (T)0.0f;
        }
    }
    __device__ __forceinline__ float at(int e) const { return (float)v[e / V].v[e % V]; }
};
// e-th channel of this thread's
template <int V>
__device__ __forceinline__ int channel(int e) {
    return (e / V * (int)blockDim.x + (int)threadIdx.x) * V + e % V;
}
template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(void *base, int64_t offset, int n, const float (&x)[V * NV]) {
    T *p = (T *)base + offset;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = (k * (int)blockDim.x + (int)threadIdx.x) * V;
        float y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = x[k * V + j];
        if (i < n) store_pack<T, V>(p + i, y);
    }
}
template <int V, int NV>
__device__ __forceinline__ void load_weights(const float *w, float fill, int n, float (&x)[V * NV]) {
#pragma unroll
    for (int e = 0; e < V * NV; ++e) {
        const int i = channel<V>(e);
        x[e] = i < n ? (w ? w[i] : fill) : 0.0f;
    }
}

template <typename T, int V, int NV>
__global__ __launch_bounds__(1024) void k_norm_fwd_rows(sili_block_norm_args a) {
    constexpr int E = V * NV;
    __shared__ float s_part[2][16];
    BlockSum sum{s_part};
    const int n = (int)a.width;
    const float inv_n = 1.0f / (float)n;
    float w1[E], w2[E];  // w1: u_scale and a shared gate folded in
    load_weights<V, NV>(a.w_post, 1.0f, n, w1);
    load_weights<V, NV>(a.w_pre, 0.0f, n, w2);
    const bool own_gate = a.gate && a.gate_stride != 0;
    Row<T, V, NV> u, x, g;
    if (a.gate && !own_gate) g.load(a.gate, 0, n);
#pragma unroll
    for (int e = 0; e < E; ++e) w1[e] *= a.u_scale * (a.gate && !own_gate ? g.at(e) : 1.0f);
    int64_t t = blockIdx.x;
    auto fetch = [&] {
        u.load(a.u, t * a.u_stride, n);
        if (a.x) x.load(a.x, t * a.x_stride, n);
        if (own_gate) g.load(a.gate, t * a.gate_stride, n);
    };
    fetch();
    while (t < a.tokens) {
        float y[E], s = 0.0f;
        float r1 = 1.0f;
        if (a.w_post) {
#pragma unroll
            for (int e = 0; e < E; ++e) s += u.at(e) * u.at(e);
            r1 = rsqrtf(sum(s) * inv_n + a.eps);
            if (a.rstd_post && threadIdx.x == 0) a.rstd_post[t] = r1;
        }
        s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            y[e] = u.at(e) * r1 * w1[e];
            if (own_gate) y[e] *= g.at(e);
            if (a.x) y[e] += a.x_scale * x.at(e);
            s += y[e] * y[e];
        }
        const int64_t row = t;
        t += gridDim.x;
        if (t < a.tokens) fetch();
        store_row<T, V, NV>(a.y, row * a.y_stride, n, y);
        if (a.w_pre) {
            const float r2 = rsqrtf(sum(s) * inv_n + a.eps);
            if (a.rstd_pre && threadIdx.x == 0) a.rstd_pre[row] = r2;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] *= r2 * w2[e];
            store_row<T, V, NV>(a.h, row * a.h_stride, n, y);
        }
    }
}

// MOST: threads a block may have; fewer leave more registers to each (with 1024
// the 8 channels a thread spill: 8192 rows of 5120 bf16 channels 124 us).
template <typename T, int V, int NV, int MOST>
__global__ __launch_bounds__(MOST) void k_norm_bwd_rows(sili_block_norm_args a, sili_block_norm_grads g) {
    constexpr int E = V * NV;
    __shared__ float s_part[2][16];
    BlockSum sum{s_part};
    const int n = (int)a.width;
    const float inv_n = 1.0f / (float)n;
    const bool own_gate = a.gate && a.gate_stride != 0, shared_gate = a.gate && !own_gate;
    float w1[E], w2[E], gs[E];  // gs: u_scale and a shared gate
    load_weights<V, NV>(a.w_post, 1.0f, n, w1);
    load_weights<V, NV>(a.w_pre, 0.0f, n, w2);
    Row<T, V, NV> u, y, dy, dh, gt;
    if (shared_gate) gt.load(a.gate, 0, n);
#pragma unroll
    for (int e = 0; e < E; ++e) gs[e] = a.u_scale * (shared_gate ? gt.at(e) : 1.0f);
    float dw2[E], dw1[E], dg[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw2[e] = dw1[e] = dg[e] = 0.0f;
    int64_t t = blockIdx.x;
    float r1 = 1.0f, r2 = 0.0f;
    auto fetch = [&] {
        if (g.dh) {
            dh.load(g.dh, t * g.dh_stride, n);
            y.load(a.y, t * a.y_stride, n);
            r2 = a.rstd_pre[t];
        }
        if (g.dy) dy.load(g.dy, t * g.dy_stride, n);
        u.load(a.u, t * a.u_stride, n);
        if (own_gate) gt.load(a.gate, t * a.gate_stride, n);
        if (a.w_post) r1 = a.rstd_post[t];
    };
    fetch();
    while (t < a.tokens) {
        float v[E], uh[E], s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = g.dy ? dy.at(e) : 0.0f;
        if (g.dh) {
            float wd[E], yh[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                yh[e] = y.at(e) * r2;
                wd[e] = w2[e] * dh.at(e);
                dw2[e] += dh.at(e) * yh[e];
                s += wd[e] * yh[e];
            }
            const float m2 = sum(s) * inv_n;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += r2 * (wd[e] - yh[e] * m2);
        }
        // v: gradient of y; then dn, the gradient of n
        float out[E], dn[E];
        s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            uh[e] = u.at(e) * r1;
            dn[e] = v[e] * gs[e] * (own_gate ? gt.at(e) : 1.0f);
            s += w1[e] * dn[e] * uh[e];
        }
        const int64_t row = t;
        const float q1 = r1;
        t += gridDim.x;
        if (t < a.tokens) fetch();
        if (g.dx) {
#pragma unroll
            for (int e = 0; e < E; ++e) out[e] = a.x_scale * v[e];
            store_row<T, V, NV>(g.dx, row * g.dx_stride, n, out);
        }
        if (a.gate && g.dgate) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                out[e] = a.u_scale * v[e] * uh[e] * w1[e];
                dg[e] += out[e];
            }
            if (own_gate) store_row<T, V, NV>(g.dgate, row * g.dgate_stride, n, out);
        }
        const float m1 = a.w_post ? sum(s) * inv_n : 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dw1[e] += dn[e] * uh[e];
            out[e] = a.w_post ? q1 * (w1[e] * dn[e] - uh[e] * m1) : dn[e];
        }
        if (g.du) store_row<T, V, NV>(g.du, row * g.du_stride, n, out);
    }
    const int64_t plane = (int64_t)gridDim.x * n;
    float *part = (float *)g.workspace + (int64_t)blockIdx.x * n;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = channel<V>(e);
        if (i >= n) continue;
        if (shared_gate && g.dgate) part[i] = dg[e];
        if (g.dw_post) part[plane + i] = dw1[e];
        if (g.dw_pre && g.dh) part[2 * plane + i] = dw2[e];
    }
}

// out[i] = the sum of part[b][i] over the blocks b, in an order of their own: 16
// runs of every 16th block, then the runs.  A block takes 64 channels.
__global__ __launch_bounds__(1024) void k_norm_sums(const float *part, int64_t plane, int blocks, int n, float *d0, float *d1,
                                                    float *d2) {
    __shared__ float s_run[16][64];
    float *out = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    if (!out) return;
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
    const float *p = part + blockIdx.y * plane + i;
    float s = 0.0f;
    if (i < n)
#pragma unroll 8
        for (int b = run; b < blocks; b += 16) s += p[(int64_t)b * n];
    s_run[run][lane] = s;
    __syncthreads();
    if (run != 0 || i >= n) return;
    s = 0.0f;
    for (int k = 0; k < 16; ++k) s += s_run[k][lane];
    out[i] = s;
}

// Blocks of the backward pass, and so runs of its sums over tokens: one of ten
// waves (5120 channels) a CU, whose sums cost 3 % of the rows' traffic (8192 rows
// of bf16: 119 + 5 us; two blocks a CU 133 + 7), more of the narrower ones while
// each still walks 16 rows.
int64_t bwd_blocks(const sili_block_norm_args &a) {
    const int64_t waves = (a.width + 511) / 512, cus = 256;
    return std::min(a.tokens, std::max(cus, std::min(cus * std::max<int64_t>(1, 12 / waves), a.tokens / 16)));
}

// Whether rows can move in vectors of v elements: every row of every operand
// begins at a multiple of their size.
bool fits(const sili_block_norm_args &a, const sili_block_norm_grads *g, int v) {
    const size_t es = (size_t)dtype_size(a.dtype);
    auto row = [&](const void *p, int64_t stride) { return !p || (aligned(p, v * es) && stride % v == 0); };
    bool ok = a.width % v == 0 && row(a.u, a.u_stride) && row(a.x, a.x_stride) && row(a.gate, a.gate_stride) &&
              row(a.y, a.y_stride) && row(a.h, a.h_stride);
    if (g) ok = ok && row(g->dy, g->dy_stride) && row(g->dh, g->dh_stride) && row(g->du, g->du_stride) && row(g->dx, g->dx_stride) &&
                (g->dgate_stride == 0 || row(g->dgate, g->dgate_stride));
    return ok;
}

// Calls f(V, NV, threads) with the vectors that fit and the least channels a
// thread that keep a row in 512 threads, up to 8; false for wider rows.
template <typename T, typename F>
bool with_shape(const sili_block_norm_args &a, const sili_block_norm_grads *g, F &&f) {
    constexpr int VEC = 16 / (int)sizeof(T);
    auto threads = [&](int64_t e) { return (unsigned)((((a.width + e - 1) / e + 63) / 64) * 64); };
    if (a.width > 8192) return false;
    if (fits(a, g, VEC)) {
        if (VEC == 8 || a.width <= 4096) f(std::integral_constant<int, VEC>{}, std::integral_constant<int, 1>{}, threads(VEC));
        else f(std::integral_constant<int, VEC>{}, std::integral_constant<int, 8 / VEC>{}, threads(8));
        return true;
    }
    using One = std::integral_constant<int, 1>;
    if (a.width <= 512) f(One{}, std::integral_constant<int, 1>{}, threads(1));
    else if (a.width <= 1024) f(One{}, std::integral_constant<int, 2>{}, threads(2));
    else if (a.width <= 2048) f(One{}, std::integral_constant<int, 4>{}, threads(4));
    else f(One{}, std::integral_constant<int, 8>{}, threads(8));
    return true;
}

enum Use { SIZES, FORWARD, BACKWARD };

void check(const sili_block_norm_args &a, const char *what, Use use) {
    const bool grad = use == BACKWARD;
    const std::string w(what);
    auto need = [&](bool ok, const char *m) {
        if (!ok) throw_error(SILI_ERR_INVALID, w + ": " + m);
    };
    need(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "unknown dtype");
    need(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "tokens out of range");
    need(a.width >= 1 && a.width <= WIDEST, "width must be 1 to 32768");
    if (a.tokens == 0 || use == SIZES) return;
    need(a.u, "u is NULL");
    need(grad || a.y, "y is NULL");
    need(!a.w_pre || (grad ? a.y && a.rstd_pre : a.h != nullptr), grad ? "y or rstd_pre is NULL" : "h is NULL");
    need(!grad || !a.w_post || a.rstd_post, "rstd_post is NULL");
}

}  // namespace

void block_norm_forward(const sili_block_norm_args &a, hipStream_t st) {
    check(a, "block_norm_forward", FORWARD);
    if (a.tokens == 0) return;
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        const bool done = with_shape<T>(a, nullptr, [&](auto v, auto nv, unsigned threads) {
            // as many blocks as run at once (2048 threads a CU)
            const int64_t blocks = std::min<int64_t>(a.tokens, 256 * std::max(1u, std::min(32u, 2048 / threads)));
            launch(k_norm_fwd_rows<T, decltype(v)::value, decltype(nv)::value>, dim3((unsigned)blocks), dim3(threads), 0, st, a);
        });
        if (!done) launch(k_norm_fwd<T>, dim3((unsigned)a.tokens), dim3(TPB), (uint32_t)(4 * a.width), st, a);
    });
    SILI_HIP(hipGetLastError());
}

size_t block_norm_workspace(const sili_block_norm_args &a) {
    check(a, "block_norm_workspace", SIZES);
    return (size_t)(3 * bwd_blocks(a) * a.width) * sizeof(float);
}

void block_norm_backward(const sili_block_norm_args &a, const sili_block_norm_grads &g, hipStream_t st) {
    check(a, "block_norm_backward", BACKWARD);
    require(!g.dh || a.w_pre, "block_norm_backward: dh without w_pre");
    require(!g.dgate || (a.gate && (a.gate_stride == 0) == (g.dgate_stride == 0)), "block_norm_backward: dgate and gate differ");
    require(!g.dw_post || a.w_post, "block_norm_backward: dw_post without w_post");
    require(!g.dw_pre || a.w_pre, "block_norm_backward: dw_pre without w_pre");
    require(a.tokens == 0 || (g.workspace && g.workspace_bytes >= block_norm_workspace(a)), "block_norm_backward: workspace too small");
    const int n = (int)a.width;
    float *dgate = a.gate_stride == 0 ? (float *)g.dgate : nullptr;
    const int64_t blocks = bwd_blocks(a);
    if (blocks == 0 && !dgate && !g.dw_post && !g.dw_pre) return;
    if (blocks > 0)
        with_dtype(a.dtype, [&](auto z) {
            using T = decltype(z);
            const bool done = with_shape<T>(a, &g, [&](auto v, auto nv, unsigned threads) {
                constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
                if (threads <= 768) launch(k_norm_bwd_rows<T, V, NV, 768>, dim3((unsigned)blocks), dim3(threads), 0, st, a, g);
                else launch(k_norm_bwd_rows<T, V, NV, 1024>, dim3((unsigned)blocks), dim3(threads), 0, st, a, g);
            });
            if (!done) launch(k_norm_bwd<T>, dim3((unsigned)blocks), dim3(TPB), (uint32_t)(4 * a.width), st, a, g);
        });
    // without dh the pre-norm's weights have no gradient, and no partial sums
    if (dgate || g.dw_post || (g.dw_pre && g.dh))
        launch(k_norm_sums, dim3((n + 63) / 64, 3), dim3(1024), 0, st, (const float *)g.workspace, blocks * n, (int)blocks, n,
               dgate, g.dw_post, g.dh ? g.dw_pre : nullptr);
    if (g.dw_pre && !g.dh)
        launch(k_norm_sums, dim3((n + 63) / 64, 3), dim3(1024), 0, st, (const float *)nullptr, (int64_t)0, 0, n, (float *)nullptr,
               (float *)nullptr, g.dw_pre);
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
