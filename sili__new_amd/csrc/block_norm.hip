// block_norm.hip -- the norm after a block, its gate and residual scale, and
// the norm before the next block, forward and backward.
//
//   n = u r1 w1,  y = b x + a g n,  h = y r2 w2,   r = rsqrt(mean(.^2) + eps)
//   gy  = dy + r2 (w2 dh - yh mean(w2 dh yh)),     yh = y r2
//   dx  = b gy,  dn = a g gy,  dg = a n gy,  dw2 = sum dh yh,  dw1 = sum dn uh
//   du  = r1 (w1 dn - uh mean(w1 dn uh)),          uh = u r1
#include "block_ops.hpp"

#include <algorithm>

namespace sili {

namespace {

constexpr unsigned TPB = 256;
constexpr int64_t WIDEST = 32768;

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

// out[i] = the sum of part[b][i] over the blocks, in their order.
__global__ __launch_bounds__(TPB) void k_norm_sums(const float *part, int64_t plane, int blocks, int n, float *d0, float *d1,
                                                   float *d2) {
    float *out = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    const int i = blockIdx.x * TPB + threadIdx.x;
    if (!out || i >= n) return;
    const float *p = part + blockIdx.y * plane + i;
    float s = 0.0f;
    for (int b = 0; b < blocks; ++b) s += p[(int64_t)b * n];
    out[i] = s;
}

int64_t bwd_blocks(const sili_block_norm_args &a) { return std::min<int64_t>(a.tokens, 512); }

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
        launch(k_norm_fwd<decltype(z)>, dim3((unsigned)a.tokens), dim3(TPB), (uint32_t)(4 * a.width), st, a);
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
            launch(k_norm_bwd<decltype(z)>, dim3((unsigned)blocks), dim3(TPB), (uint32_t)(4 * a.width), st, a, g);
        });
    // without dh the pre-norm's weights have no gradient, and no partial sums
    if (dgate || g.dw_post || (g.dw_pre && g.dh))
        launch(k_norm_sums, dim3((n + TPB - 1) / TPB, 3), dim3(TPB), 0, st, (const float *)g.workspace, blocks * n, (int)blocks, n,
               dgate, g.dw_post, g.dh ? g.dw_pre : nullptr);
    if (g.dw_pre && !g.dh)
        launch(k_norm_sums, dim3((n + TPB - 1) / TPB, 3), dim3(TPB), 0, st, (const float *)nullptr, (int64_t)0, 0, n, (float *)nullptr,
               (float *)nullptr, g.dw_pre);
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
