// fp4_linear.hip -- dense weights in 4 bits with a scale a group of inputs:
// packed, and multiplied.
#include "block_ops.hpp"
#include "mma.hpp"
#include "wave.hpp"

#include <algorithm>

namespace sili {

namespace {

// N elements at any address of an element: one load where the hardware has one
// for the size (it takes any alignment).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// ---- packing ---------------------------------------------------------------------
constexpr int PACK_TPB = 256;

template <int N>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = 1; d < N; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// A thread takes 8 inputs, group / 8 neighbours a group.
template <typename T, typename S, int G>
__global__ __launch_bounds__(PACK_TPB) void k_fp4_pack(sili_fp4_pack_args a) {
    const int64_t per_row = a.w.n_in / 8, total = a.w.n_out * per_row;
    for (int64_t i = (int64_t)blockIdx.x * PACK_TPB + threadIdx.x; i < total; i += (int64_t)gridDim.x * PACK_TPB) {
        const int64_t row = i / per_row, sub = i - row * per_row;
        const auto in = *reinterpret_cast<const Loose<T, 8> *>((const T *)a.rows + row * a.row_stride + 8 * sub);
        float x[8], top = 0.0f, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = (float)in.v[j];
            top = fmaxf(top, fabsf(x[j]));
            sum += x[j] * 0.0f;  // 0, or NaN for what is not finite
        }
        top = group_max<G / 8>(fmaxf(top, sum == 0.0f ? 0.0f : INFINITY));
        const float scale = (float)(S)(top / 6.0f);
        const bool finite = scale < INFINITY, zero = !finite || scale < 0x1p-120f;
        const float inv = zero ? 0.0f : 1.0f / scale;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= fp4_encode(x[j] * inv) << (4 * j);
        *reinterpret_cast<uint32_t *>(a.w.codes + row * a.w.codes_stride + 4 * sub) = zero ? 0u : w;
        if (sub % (G / 8) == 0)
            ((S *)a.w.scales)[row * a.w.scales_stride + sub / (G / 8)] = (S)(!finite ? __builtin_nanf("") : zero ? 0.0f : scale);
    }
}

// ---- products --------------------------------------------------------------------
// y = x W^T on the bf16 matrix cores: 16 tokens (A's rows) by 16 outputs (B's
// columns) by 32 inputs.  Codes are exact in bf16 and x enters in bf16 parts; the
// sum over a group is scaled in fp32, a lane's output having one scale.  A wave
// takes 128 inputs of 16 NT outputs a step: a lane loads 16 bytes of a row, and
// four lanes' dwords are exchanged so that each product has 32 consecutive
// inputs, whose scales are the same.  The waves of a block take steps in turn and
// are joined in LDS; blocks that share outputs (splits) through the workspace.
//
// MERGED: with 4 (fp32) or 8 (f16) tokens at most, the parts of x go to rows that
// would be empty: row r + RT k holds part k of token r.
constexpr int LINEAR_STEP = 128;

struct LinearPlan {
    int32_t waves, splits, chunk;  // of a block; chunk: steps a split
    int32_t steps, token_tiles;
    float *part;  // [splits][tokens][n_out]
};

// x, y in N parts, each the first 8 bits of what the parts before leave: all of
// the value in the end, and no part larger than it.
template <int N>
__device__ __forceinline__ void cut_bf16(float x, float y, uint32_t (&part)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
        part[k] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        x -= bf16_lo(part[k]);
        y -= bf16_hi(part[k]);
    }
}

__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b) {  // odd rows of 16 lanes of a, even rows of b
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {  // upper half of a, lower half of b
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

template <typename S, int N>
__device__ __forceinline__ void load_scales(const S *p, int have, float (&s)[N]) {
    if (have >= N) {
        const auto v = *reinterpret_cast<const Loose<S, N> *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = (float)v.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = i < have ? (float)p[i] : 0.0f;
    }
}

__device__ __forceinline__ void store_as(void *p, int dtype, int64_t at, float x) {
    if (dtype == SILI_F32) ((float *)p)[at] = x;
    else if (dtype == SILI_BF16) ((__bf16 *)p)[at] = (__bf16)x;
    else ((_Float16 *)p)[at] = (_Float16)x;
}

template <typename T, int G, int NT, bool MERGED>
__global__ __launch_bounds__(1024) void k_linear_few(sili_fp4_linear_args a, LinearPlan pl) {
    constexpr int P = q_parts<T>(), RT = MERGED ? (P == 3 ? 4 : 8) : 16, PM = MERGED ? 1 : P;
    constexpr int GS = LINEAR_STEP / G;  // groups a step
    extern __shared__ float s_sum[];
    const int wave = (int)uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
    const int tile = blockIdx.x / pl.token_tiles, t0 = (blockIdx.x - tile * pl.token_tiles) * RT, split = blockIdx.y;
    const int64_t n0 = (int64_t)tile * (16 * NT);
    const int k_end = (int)a.w.n_in;

    const int64_t token = min((int64_t)t0 + r16 % RT, a.tokens - 1);
    const T *x = (const T *)a.x + token * a.x_stride + 8 * g;
    const uint8_t *codes[NT];
    int64_t scale_row[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = min(n0 + 16 * t + r16, a.w.n_out - 1);
        codes[t] = a.w.codes + n * a.w.codes_stride + 16 * g;
        scale_row[t] = n * a.w.scales_stride;
    }
    uint32_t take[P];
#pragma unroll
    for (int k = 0; k < P; ++k) take[k] = r16 / RT == k ? ~0u : 0u;

    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    uint4 w[NT];
    float sc[NT][GS];
    Loose<T, 8> xs[4];
    auto fetch = [&](int step) {
        const int k0 = step * LINEAR_STEP, left = k_end - k0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            w[t] = make_uint4(0, 0, 0, 0);
            if (32 * g < left) w[t] = *reinterpret_cast<const uint4 *>(codes[t] + k0 / 2);
            const int64_t at = scale_row[t] + k0 / G;
            const int have = left / G;
            if (a.w.scale_dtype == SILI_F32) load_scales((const float *)a.w.scales + at, have, sc[t]);
            else if (a.w.scale_dtype == SILI_BF16) load_scales((const __bf16 *)a.w.scales + at, have, sc[t]);
            else load_scales((const _Float16 *)a.w.scales + at, have, sc[t]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (32 * s < left) {
                xs[s] = *reinterpret_cast<const Loose<T, 8> *>(x + k0 + 32 * s);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[s].v[j] = (T)0.0f;
            }
        }
    };
    const int last = min(pl.steps, (split + 1) * pl.chunk);
    int step = split * pl.chunk + wave;
    if (step < last) fetch(step);
    for (; step < last; step += pl.waves) {
        u32x4 av[4][PM];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t part[P];
                cut_bf16<P>((float)xs[s].v[2 * j], (float)xs[s].v[2 * j + 1], part);
#pragma unroll
                for (int k = 0; k < PM; ++k) av[s][k][j] = MERGED ? pick<P>(part, take) : part[k];
            }
        uint32_t ww[NT][4];
        float ss[NT][GS];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            ww[t][0] = w[t].x;
            ww[t][1] = w[t].y;
            ww[t][2] = w[t].z;
            ww[t][3] = w[t].w;
#pragma unroll
            for (int i = 0; i < GS; ++i) ss[t][i] = sc[t][i];
        }
        if (step + pl.waves < last) fetch(step + pl.waves);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            swap16(ww[t][0], ww[t][1]);
            swap16(ww[t][2], ww[t][3]);
            swap32(ww[t][0], ww[t][2]);
            swap32(ww[t][1], ww[t][3]);
#pragma unroll
            for (int i = 0; i < GS; ++i) {
                f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = i * (4 / GS); s < (i + 1) * (4 / GS); ++s) {
                    const u32x4 b = codes8(ww[t][s]);
#pragma unroll
                    for (int k = 0; k < PM; ++k) sum = mma(av[s][k], b, sum);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][j] = __builtin_fmaf(sum[j], ss[t][i], acc[t][j]);
            }
        }
    }

    // lane: output r16, rows 4 g + j of A
    if (MERGED) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (RT == 4) acc[t][j] += __shfl_xor(acc[t][j], 16, 64);
                acc[t][j] += __shfl_xor(acc[t][j], 32, 64);
            }
    }
    constexpr int W = 16 * NT;
    float *mine = s_sum + wave * (RT * W);
    if (4 * g < RT) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) mine[(4 * g + j) * W + 16 * t + r16] = acc[t][j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < RT * W; i += 64 * pl.waves) {
        const int row = i / W;
        const int64_t t = t0 + row, n = n0 + (i - row * W);
        if (t >= a.tokens || n >= a.w.n_out) continue;
        float y = 0.0f;
        for (int v = 0; v < pl.waves; ++v) y += s_sum[v * (RT * W) + i];
        if (pl.splits > 1) pl.part[((int64_t)split * a.tokens + t) * a.w.n_out + n] = y;
        else store_as(a.y, a.out_dtype, t * a.y_stride + n, y);
    }
}

constexpr int JOIN_TPB = 256;

__global__ __launch_bounds__(JOIN_TPB) void k_linear_join(sili_fp4_linear_args a, LinearPlan pl) {
    const int64_t total = a.tokens * a.w.n_out;
    for (int64_t i = (int64_t)blockIdx.x * JOIN_TPB + threadIdx.x; i < total; i += (int64_t)gridDim.x * JOIN_TPB) {
        float y = 0.0f;
        for (int s = 0; s < pl.splits; ++s) y += pl.part[s * total + i];
        const int64_t t = i / a.w.n_out;
        store_as(a.y, a.out_dtype, t * a.y_stride + (i - t * a.w.n_out), y);
    }
}

void check_weights(const sili_fp4_weights &w, const char *what) {
    const std::string name(what);
    auto need = [&](bool ok, const char *m) {
        if (!ok) throw_error(SILI_ERR_INVALID, name + ": " + m);
    };
    need(w.scale_dtype == SILI_F32 || w.scale_dtype == SILI_BF16 || w.scale_dtype == SILI_F16, "unknown scale_dtype");
    need(w.group == 32 || w.group == 64 || w.group == 128, "group is none of 32, 64, 128");
    need(w.n_out >= 0 && w.n_out <= INT32_MAX, "n_out out of range");
    need(w.n_in >= 0 && w.n_in <= (int64_t(1) << 30) && w.n_in % w.group == 0, "n_in is no multiple of group, or out of range");
    need(w.codes_stride % 16 == 0 && aligned(w.codes, 16), "codes or codes_stride is not 16-byte aligned");
    need(w.n_out == 0 || w.n_in == 0 || (w.codes && w.scales), "NULL weights");
    need(w.n_out <= 1 || (w.codes_stride >= w.n_in / 2 && w.scales_stride >= w.n_in / w.group), "rows of codes or scales overlap");
}

void check_linear(const sili_fp4_linear_args &a) {
    check_weights(a.w, "fp4_linear");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "fp4_linear: unknown dtype");
    require(a.out_dtype == SILI_F32 || a.out_dtype == SILI_BF16 || a.out_dtype == SILI_F16, "fp4_linear: unknown out_dtype");
    require(a.tokens >= 0 && a.tokens <= INT32_MAX, "fp4_linear: tokens out of range");
}

constexpr int LINEAR_NT = 4;

bool merges(const sili_fp4_linear_args &a) { return a.dtype == SILI_F32 ? a.tokens <= 4 : a.dtype == SILI_F16 && a.tokens <= 8; }

LinearPlan plan_linear(const sili_fp4_linear_args &a) {
    LinearPlan p{};
    const int64_t rt = !merges(a) ? 16 : a.dtype == SILI_F32 ? 4 : 8;
    p.token_tiles = (int32_t)((a.tokens + rt - 1) / rt);
    p.steps = (int32_t)((a.w.n_in + LINEAR_STEP - 1) / LINEAR_STEP);
    const int64_t blocks = std::max<int64_t>(1, (a.w.n_out + 16 * LINEAR_NT - 1) / (16 * LINEAR_NT) * p.token_tiles);
    p.waves = blocks >= 512 ? 4 : 8;
    const int64_t want = std::clamp<int64_t>(512 / blocks, 1, std::max<int64_t>(1, p.steps / (2 * p.waves)));
    p.chunk = (int32_t)std::max<int64_t>(1, (p.steps + want - 1) / want);
    p.splits = (int32_t)std::max<int64_t>(1, (p.steps + p.chunk - 1) / p.chunk);
    return p;
}

size_t linear_bytes(const sili_fp4_linear_args &a, const LinearPlan &p) {
    return p.splits == 1 ? 0 : (size_t)a.tokens * (size_t)a.w.n_out * (size_t)p.splits * sizeof(float);
}

template <int G, typename F>
void with_group_of(F &&f) { f(std::integral_constant<int, G>{}); }
template <typename F>
void with_group(int64_t group, F &&f) {
    if (group == 32) with_group_of<32>(f);
    else if (group == 64) with_group_of<64>(f);
    else with_group_of<128>(f);
}

}  // namespace

void fp4_pack(const sili_fp4_pack_args &a, hipStream_t st) {
    check_weights(a.w, "fp4_pack");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "fp4_pack: unknown dtype");
    if (a.w.n_out == 0 || a.w.n_in == 0) return;
    require(a.rows, "fp4_pack: NULL buffer");
    const int64_t blocks = std::min<int64_t>((a.w.n_out * (a.w.n_in / 8) + PACK_TPB - 1) / PACK_TPB, 1 << 20);
    with_dtype(a.dtype, [&](auto z) {
        with_dtype(a.w.scale_dtype, [&](auto s) {
            with_group(a.w.group, [&](auto g) {
                launch(k_fp4_pack<decltype(z), decltype(s), decltype(g)::value>, dim3((unsigned)blocks), dim3(PACK_TPB), 0, st, a);
            });
        });
    });
    SILI_HIP(hipGetLastError());
}

size_t fp4_linear_workspace(const sili_fp4_linear_args &a) {
    check_linear(a);
    return linear_bytes(a, plan_linear(a));
}

void fp4_linear(const sili_fp4_linear_args &a, hipStream_t st) {
    check_linear(a);
    if (a.tokens == 0 || a.w.n_out == 0) return;
    require(a.y && (a.x || a.w.n_in == 0), "fp4_linear: NULL buffer");
    LinearPlan p = plan_linear(a);
    const size_t need = linear_bytes(a, p);
    require(need == 0 || (a.workspace && aligned(a.workspace, 16) && a.workspace_bytes >= need),
            "fp4_linear: workspace too small or not 16-byte aligned");
    p.part = static_cast<float *>(a.workspace);
    const int64_t blocks = (a.w.n_out + 16 * LINEAR_NT - 1) / (16 * LINEAR_NT) * p.token_tiles;
    require(blocks * 64 * p.waves < (int64_t(1) << 32) && p.splits <= 65535, "fp4_linear: too many tokens or outputs");
    const dim3 grid((unsigned)blocks, (unsigned)p.splits), block(64 * p.waves);
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        with_group(a.w.group, [&](auto g) {
            constexpr int G = decltype(g)::value;
            constexpr int RT = sizeof(T) == 4 ? 4 : 8;
            const uint32_t lds = (uint32_t)(p.waves * (merges(a) ? RT : 16) * 16 * LINEAR_NT * sizeof(float));
            if constexpr (q_parts<T>() > 1) {
                if (merges(a)) {
                    launch(k_linear_few<T, G, LINEAR_NT, true>, grid, block, lds, st, a, p);
                    return;
                }
            }
            launch(k_linear_few<T, G, LINEAR_NT, false>, grid, block, lds, st, a, p);
        });
    });
    if (p.splits > 1) {
        const int64_t joins = std::min<int64_t>((a.tokens * a.w.n_out + JOIN_TPB - 1) / JOIN_TPB, 4096);
        launch(k_linear_join, dim3((unsigned)joins), dim3(JOIN_TPB), 0, st, a, p);
    }
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
