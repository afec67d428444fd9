// fp4_linear.hip -- dense weights in 4 bits with a scale a group of inputs:
// packed, and multiplied.
#include "block_ops.hpp"
#include "mma.hpp"
#include "wave.hpp"

#include <algorithm>
#include <type_traits>

namespace sili {

namespace {

// N elements at any address of an element: one load where the hardware has one
// for the size (it takes any alignment).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// Words at any address of two bytes.
template <int N>
struct __attribute__((packed, aligned(2))) LooseWords {
    uint32_t v[N];
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
// y = x W^T on the bf16 matrix cores, x the left operand (rows: tokens), W the
// right one (columns: outputs).  Codes are exact in bf16 and x enters in bf16
// parts; a group's products are summed by themselves and then scaled in fp32, a
// lane's column having one scale.  A wave takes its outputs' rows 128 inputs a
// step: a lane loads 16 or 32 consecutive bytes, and lanes of a column exchange
// dwords so that each product has consecutive inputs, of one group.
constexpr int LINEAR_STEP = 128;

struct LinearPlan {
    int32_t splits, chunk;       // chunk: steps a split
    int32_t steps, token_tiles;  // (few tokens: turns)
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
__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {  // upper half of a, lower half of b
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

__device__ __forceinline__ void store_as(void *p, int dtype, int64_t at, float x) {
    if (dtype == SILI_F32) ((float *)p)[at] = x;
    else if (dtype == SILI_BF16) ((__bf16 *)p)[at] = (__bf16)x;
    else ((_Float16 *)p)[at] = (_Float16)x;
}
// Scales are loaded as they lie and converted where they are used: a conversion
// next to its load would wait for it.
__device__ __forceinline__ float scale_of(int dtype, uint32_t raw) {
    return dtype == SILI_F32 ? __builtin_bit_cast(float, raw) : dtype == SILI_BF16 ? bf16_lo(raw) : (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
}
__device__ __forceinline__ uint32_t load_scale(const sili_fp4_weights &w, int64_t at) {
    return w.scale_dtype == SILI_F32 ? ((const uint32_t *)w.scales)[at] : ((const uint16_t *)w.scales)[at];
}

// Few tokens: rows of one product, 16 in all with their parts, row r + RT k holding
// part k of token r (RT = 16, 8, 4 for one, two, three parts).  A block cuts x once,
// in LDS; its waves then run by themselves, 16 outputs each (or a share of their
// inputs, joined in LDS), in turns of 256 inputs asked for AHEAD turns before.  Eight
// lanes load 128 bytes of a row of codes, and four its scales, so that the cache is
// asked for a line and not for a lane at a time; the wave turns them in LDS of its
// own into what a product's lanes need.  Blocks that share outputs (splits) are
// joined through the workspace.
constexpr int FEW_TURN = 2 * LINEAR_STEP;  // inputs
constexpr int FEW_ROW = FEW_TURN / 8 + 4;  // words of a row of codes in LDS: 16 rows in all banks
constexpr int FEW_WAVES = 8;
constexpr int AHEAD = 2;

struct FewLinear {
    int32_t share;      // waves that share outputs: 1, 2, 4, 8
    int32_t tiles;      // of a block's outputs; share 1: a block takes every gridDim.x-th
    int32_t row_words;  // of x in LDS, a row
};

template <typename T, int G>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_linear_few(sili_fp4_linear_args a, LinearPlan pl, FewLinear few) {
    constexpr int P = q_parts<T>(), RT = P == 1 ? 16 : P == 2 ? 8 : 4;
    constexpr int GT = FEW_TURN / G, GL = GT >= 4 ? GT / 4 : 1;  // groups a turn; scales a lane loads
    extern __shared__ __align__(16) uint32_t s_few[];
    const int wave = (int)uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
    const int split = blockIdx.y, tokens = (int)a.tokens, n_in = (int)a.w.n_in;
    const int wk = wave % few.share, wn = wave / few.share;
    const int outs = 16 * FEW_WAVES / few.share;                                 // of a block's tile
    const int first = split * pl.chunk, last = min(pl.steps, first + pl.chunk);  // turns

    const int piece = lane & 7, scale_at = GL * (lane & (GT >= 4 ? 3 : GT - 1));
    const uint8_t *codes[2];
    int64_t scale_row;
    auto aim = [&](int tile) {
        const int64_t n0 = (int64_t)tile * outs + 16 * wn;
#pragma unroll
        for (int h = 0; h < 2; ++h) codes[h] = a.w.codes + min(n0 + 8 * h + (lane >> 3), a.w.n_out - 1) * a.w.codes_stride + 16 * piece;
        scale_row = min(n0 + (lane >> 2), a.w.n_out - 1) * a.w.scales_stride + scale_at;
    };
    uint4 w[AHEAD][2];
    uint32_t sc[AHEAD][GL];  // two bytes and GL 2: both in the first
    auto load = [&](int d, int turn) {
        const int k0 = turn * FEW_TURN, left = n_in - k0;
        const int64_t s0 = scale_row + turn * GT;
        if (left >= FEW_TURN) {
#pragma unroll
            for (int h = 0; h < 2; ++h) w[d][h] = *reinterpret_cast<const uint4 *>(codes[h] + k0 / 2);
            if (a.w.scale_dtype == SILI_F32) {
                const auto v = *reinterpret_cast<const Loose<uint32_t, GL> *>((const uint32_t *)a.w.scales + s0);
#pragma unroll
                for (int i = 0; i < GL; ++i) sc[d][i] = v.v[i];
            } else if constexpr (GL == 1) {
                sc[d][0] = ((const uint16_t *)a.w.scales)[s0];
            } else {
                sc[d][0] = reinterpret_cast<const LooseWords<1> *>((const uint16_t *)a.w.scales + s0)->v[0];
            }
        } else {  // the last inputs, a multiple of 32
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[d][h] = make_uint4(0, 0, 0, 0);
                if (32 * piece < left) w[d][h] = *reinterpret_cast<const uint4 *>(codes[h] + k0 / 2);
            }
#pragma unroll
            for (int i = 0; i < GL; ++i) sc[d][i] = 0;
#pragma unroll
            for (int i = 0; i < GL; ++i) {
                if (G * (scale_at + i) >= left) continue;
                const uint32_t v = load_scale(a.w, s0 + i);
                if (a.w.scale_dtype == SILI_F32) sc[d][i] = v;
                else sc[d][0] |= v << (16 * i);
            }
        }
    };
    // what is asked for next
    int next_tile = blockIdx.x, next_turn = first + wk;
    if (first + wk >= last) next_tile = few.tiles;
    auto fetch = [&](int d) {
        if (next_tile >= few.tiles) return;
        load(d, next_turn);
        next_turn += few.share;
        if (next_turn >= last) {
            next_turn = first + wk;
            next_tile += gridDim.x;
            aim(next_tile);
        }
    };
    aim(next_tile);
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) fetch(d);

    // LDS: a wave's codes and scales, then x: zeros past the end
    constexpr int MINE = 16 * (FEW_ROW + GT);
    uint32_t *s_w = s_few + wave * MINE, *s_x = s_few + FEW_WAVES * MINE;
    float *s_s = reinterpret_cast<float *>(s_w + 16 * FEW_ROW);
    const int per_row = (last - first) * (FEW_TURN / 8);
    for (int i = threadIdx.x; i < tokens * per_row; i += 64 * FEW_WAVES) {
        const int row = i / per_row, at = i - row * per_row, k = first * FEW_TURN + 8 * at;
        Loose<T, 8> v;
        if (k < n_in) {
            v = *reinterpret_cast<const Loose<T, 8> *>((const T *)a.x + row * a.x_stride + k);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v.v[j] = (T)0.0f;
        }
        u32x4 part[P];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t c[P];
            cut_bf16<P>((float)v.v[2 * j], (float)v.v[2 * j + 1], c);
#pragma unroll
            for (int p = 0; p < P; ++p) part[p][j] = c[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<u32x4 *>(s_x + (p * tokens + row) * few.row_words + 4 * at) = part[p];
    }
    __syncthreads();
    // this lane's row of x (tokens past the last: the last again; a fourth part: the third), its column of codes
    const uint32_t *xs = s_x + (min(r16 / RT, P - 1) * tokens + min(r16 % RT, tokens - 1)) * few.row_words + 4 * g;
    const uint32_t *ws = s_w + r16 * FEW_ROW + g;

    auto store = [&](int64_t t, int64_t n, float y) {
        if (pl.splits > 1) pl.part[((int64_t)split * tokens + t) * a.w.n_out + n] = y;
        else store_as(a.y, a.out_dtype, t * a.y_stride + n, y);
    };
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto join_parts = [&] {  // lane: output r16, rows 4 g + j of A
        if (P == 1) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y = P == 3 && g == 3 ? 0.0f : acc[j];
            if (RT == 4) y += __shfl_xor(y, 16, 64);
            acc[j] = y + __shfl_xor(y, 32, 64);
        }
    };
    int tile = blockIdx.x, turn = first + wk;
    if (turn >= last) tile = few.tiles;
    while (tile < few.tiles) {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            if (tile >= few.tiles) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) *reinterpret_cast<uint4 *>(s_w + (8 * h + (lane >> 3)) * FEW_ROW + 4 * piece) = w[d][h];
#pragma unroll
            for (int i = 0; i < GL; ++i)
                s_s[(lane >> 2) * GT + scale_at + i] = scale_of(a.w.scale_dtype, a.w.scale_dtype == SILI_F32 ? sc[d][i] : sc[d][0] >> (16 * i));
            fetch(d);
            wave_lds_sync();
            float f[GT];  // the scales of this lane's column
#pragma unroll
            for (int i = 0; i < GT; ++i) f[i] = s_s[r16 * GT + i];
            const uint32_t *x = xs + (turn - first) * (FEW_TURN / 2);
            f32x4 sum;
#pragma unroll
            for (int s = 0; s < FEW_TURN / 32; ++s) {
                const u32x4 av = *reinterpret_cast<const u32x4 *>(x + 16 * s);
                if (s % (G / 32) == 0) sum = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                sum = mma(av, codes8(ws[4 * s]), sum);
                if ((s + 1) % (G / 32) == 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(sum[j], f[s / (G / 32)], acc[j]);
                }
            }
            wave_lds_sync();
            turn += few.share;
            if (turn >= last) {
                if (few.share == 1) {
                    join_parts();
                    const int64_t n = (int64_t)tile * outs + 16 * wn + r16;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (4 * g + j < min(RT, tokens) && n < a.w.n_out) store(4 * g + j, n, acc[j]);
                        acc[j] = 0.0f;
                    }
                }
                turn = first + wk;
                tile += gridDim.x;
            }
        }
    }
    if (few.share == 1 && first < last) return;

    join_parts();
    __syncthreads();
    float *s_sum = reinterpret_cast<float *>(s_few);  // [share][RT][outputs]
    if (4 * g < RT) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s_sum[(wk * RT + 4 * g + j) * outs + 16 * wn + r16] = acc[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * outs; i += 64 * FEW_WAVES) {
        const int t = i / outs;
        const int64_t n = (int64_t)blockIdx.x * outs + (i - t * outs);
        if (n >= a.w.n_out) continue;
        float y = 0.0f;
        for (int v = 0; v < few.share; ++v) y += s_sum[v * (RT * outs) + i];
        store(t, n, y);
    }
}

// More tokens: a block's four waves take WN times 64 outputs by 4 / WN times 32 MT
// tokens, in products of 32 x 32 outputs x 16 inputs.  x is cut into its parts
// once a block, in LDS (two buffers, KC inputs each: the next ones' loads are under
// this one's products), rows padded by 16 bytes so that eight lanes' 16 bytes lie
// in all banks; a wave's 64 outputs take each operand from there twice, which is
// what the LDS can give the matrix cores.
template <typename T, int G, int WN, int MT>
struct ManyLinear {
    static constexpr int P = q_parts<T>(), WM = 4 / WN, BM = 32 * MT * WM, BN = 64 * WN;
    static constexpr int KC = sizeof(T) == 4 ? 32 : 64, ROW = KC + 8;  // bf16 of a row
    static constexpr int LDS = 2 * P * BM * ROW * 2;
};

template <typename T, int G, int WN, int MT>
__global__ __launch_bounds__(256, 2) void k_linear_many(sili_fp4_linear_args a, LinearPlan pl) {
    using M = ManyLinear<T, G, WN, MT>;
    constexpr int P = M::P, BM = M::BM, KC = M::KC, ROW = M::ROW, GS = LINEAR_STEP / G;
    constexpr int TPR = KC / 8, PASS = 256 / TPR, PASSES = (BM + PASS - 1) / PASS;  // threads a row of x; rows a pass
    constexpr int SUB = LINEAR_STEP / KC, KS = KC / 16;  // chunks a step; products a chunk
    constexpr int US = (G < KC ? G : KC) / 16;           // ... of one scale
    extern __shared__ __align__(16) uint16_t s_x[];      // [2][P][BM][ROW]
    const int tid = threadIdx.x, wave = (int)uniform(tid >> 6), lane = tid & 63, hf = lane >> 5, r32 = lane & 31;
    const int wn = wave % WN, wm = wave / WN;
    const int tile = blockIdx.x / pl.token_tiles, t0 = (blockIdx.x - tile * pl.token_tiles) * BM, split = blockIdx.y;
    const int64_t n0 = (int64_t)tile * M::BN + 64 * wn;
    const int k_end = (int)a.w.n_in;

    const uint8_t *codes[2];
    int64_t scale_row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int64_t n = min(n0 + 32 * t + r32, a.w.n_out - 1);
        codes[t] = a.w.codes + n * a.w.codes_stride + 32 * hf;
        scale_row[t] = n * a.w.scales_stride;
    }
    const T *x[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int64_t token = min((int64_t)t0 + i * PASS + tid / TPR, a.tokens - 1);
        x[i] = (const T *)a.x + token * a.x_stride + 8 * (tid % TPR);
    }

    Loose<T, 8> xs[PASSES];
    auto fetch_x = [&](int k0) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            if (k0 + 8 * (tid % TPR) < k_end) {
                xs[i] = *reinterpret_cast<const Loose<T, 8> *>(x[i] + k0);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[i].v[j] = (T)0.0f;
            }
        }
    };
    auto put_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = i * PASS + tid / TPR;
            if (BM % PASS != 0 && row >= BM) continue;
            u32x4 part[P];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t c[P];
                cut_bf16<P>((float)xs[i].v[2 * j], (float)xs[i].v[2 * j + 1], c);
#pragma unroll
                for (int k = 0; k < P; ++k) part[k][j] = c[k];
            }
#pragma unroll
            for (int k = 0; k < P; ++k)
                *reinterpret_cast<u32x4 *>(s_x + ((buf * P + k) * BM + row) * ROW + 8 * (tid % TPR)) = part[k];
        }
    };
    uint4 w[2][2];
    uint32_t sc[2][GS];  // two bytes: two a word
    auto fetch_w = [&](int step) {
        const int k0 = step * LINEAR_STEP, left = k_end - k0;
        if (left >= LINEAR_STEP) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                w[t][0] = *reinterpret_cast<const uint4 *>(codes[t] + k0 / 2);
                w[t][1] = *reinterpret_cast<const uint4 *>(codes[t] + k0 / 2 + 16);
            }
            if (a.w.scale_dtype == SILI_F32) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const auto v = *reinterpret_cast<const Loose<uint32_t, GS> *>((const uint32_t *)a.w.scales + scale_row[t] + step * GS);
#pragma unroll
                    for (int i = 0; i < GS; ++i) sc[t][i] = v.v[i];
                }
            } else if constexpr (GS == 1) {
#pragma unroll
                for (int t = 0; t < 2; ++t) sc[t][0] = ((const uint16_t *)a.w.scales)[scale_row[t] + step];
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const auto v = *reinterpret_cast<const LooseWords<GS / 2> *>((const uint16_t *)a.w.scales + scale_row[t] + step * GS);
#pragma unroll
                    for (int i = 0; i < GS / 2; ++i) sc[t][i] = v.v[i];
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    w[t][i] = make_uint4(0, 0, 0, 0);
                    if (64 * hf + 32 * i < left) w[t][i] = *reinterpret_cast<const uint4 *>(codes[t] + k0 / 2 + 16 * i);
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int i = 0; i < GS; ++i) sc[t][i] = 0;
#pragma unroll
                for (int i = 0; i < GS; ++i) {
                    if (G * i >= left) continue;
                    const uint32_t v = load_scale(a.w, scale_row[t] + step * GS + i);
                    if (a.w.scale_dtype == SILI_F32 || GS == 1) sc[t][i] = v;
                    else sc[t][i / 2] |= v << (16 * (i % 2));
                }
            }
        }
    };

    f32x16 acc[2][MT];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][m][i] = 0.0f;

    const int first = split * pl.chunk, last = min(pl.steps, first + pl.chunk);
    if (first < last) {
        fetch_w(first);
        fetch_x(first * LINEAR_STEP);
        put_x(0);
    }
    int buf = 0;
    for (int step = first; step < last; ++step) {
        uint32_t ww[2][8];
        float ss[2][GS];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t d[8] = {w[t][0].x, w[t][0].y, w[t][0].z, w[t][0].w, w[t][1].x, w[t][1].y, w[t][1].z, w[t][1].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // product i has dwords 2 i (lower lanes) and 2 i + 1
                ww[t][i] = d[2 * i];
                ww[t][4 + i] = d[2 * i + 1];
                swap32(ww[t][i], ww[t][4 + i]);
            }
#pragma unroll
            for (int i = 0; i < GS; ++i)
                ss[t][i] = scale_of(a.w.scale_dtype, a.w.scale_dtype == SILI_F32 || GS == 1 ? sc[t][i] : sc[t][i / 2] >> (16 * (i % 2)));
        }
        if (step + 1 < last) fetch_w(step + 1);
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
            const bool more = sub + 1 < SUB || step + 1 < last;
            __syncthreads();
            if (more) fetch_x(step * LINEAR_STEP + (sub + 1) * KC);
            const uint16_t *base = s_x + (buf * P * BM + 32 * MT * wm + r32) * ROW + 8 * hf;
            // the inputs of a chunk that share a scale
#pragma unroll
            for (int s = 0; s < KS; s += US) {
                const int k = sub * KS + s;  // product of the step
                u32x4 b[US][2];
#pragma unroll
                for (int u = 0; u < US; ++u)
#pragma unroll
                    for (int t = 0; t < 2; ++t) b[u][t] = codes8(ww[t][k + u]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    f32x16 sum[2];
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[0][i] = sum[1][i] = 0.0f;
#pragma unroll
                    for (int u = 0; u < US; ++u)
#pragma unroll
                        for (int p = 0; p < P; ++p) {
                            const u32x4 av = *reinterpret_cast<const u32x4 *>(base + (p * BM + 32 * m) * ROW + 16 * (s + u));
#pragma unroll
                            for (int t = 0; t < 2; ++t) sum[t] = mma(av, b[u][t], sum[t]);
                        }
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[t][m][i] = __builtin_fmaf(sum[t][i], ss[t][k / (G / 16)], acc[t][m][i]);
                    // here: the compiler would keep the sums of several scales until the accumulators' next use
#pragma unroll
                    for (int t = 0; t < 2; ++t) __asm__ volatile("" : "+v"(acc[t][m]));
                }
            }
            if (more) put_x(buf ^ 1);
            buf ^= 1;
        }
    }
    // lane: output r32; result 4 i + j of a tile is token 8 i + 4 hf + j
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int64_t n = n0 + 32 * t + r32;
        if (n >= a.w.n_out) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t tok = t0 + 32 * (MT * wm + m) + 8 * (i >> 2) + 4 * hf + (i & 3);
                if (tok >= a.tokens) continue;
                if (pl.splits > 1) pl.part[((int64_t)split * a.tokens + tok) * a.w.n_out + n] = acc[t][m][i];
                else store_as(a.y, a.out_dtype, tok * a.y_stride + n, acc[t][m][i]);
            }
    }
}

constexpr int JOIN_TPB = 256;

__global__ __launch_bounds__(JOIN_TPB) void k_linear_join(sili_fp4_linear_args a, LinearPlan pl) {
    const int64_t total = a.tokens * a.w.n_out;
    for (int64_t i = (int64_t)blockIdx.x * JOIN_TPB + threadIdx.x; i < total; i += (int64_t)gridDim.x * JOIN_TPB) {
        float y = 0.0f;
#pragma unroll 8
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

// How a call is launched.
struct LinearLaunch {
    int64_t blocks = 0;
    bool few_tokens = false;
    int wn = 0, mt = 0;  // more tokens: a block's shape
    uint32_t lds = 0;
    LinearPlan plan{};
    FewLinear few{};
};

// Few tokens.  512 blocks of 8 waves fill the GPU twice over.  Fewer (outputs / 128):
// waves share outputs where x is small (up to 8 rows of 16384 inputs, which every such
// block holds whole), else blocks split the inputs and are joined.  us of a call, its
// inputs x outputs, rows of x (tokens times parts); share 1, share 2 .. 8, splits:
//     5120 x 32768, 3 rows   19.6, 18.7, 21.3      5120 x 5120, 1 row   -, 5.8, 9.0
//     5120 x 32768, 8 rows   23.0, 26.0, 23.0      5120 x 5120, 8 rows  -, 8.7, 9.3
//     5120 x 32768, 16 rows  27.5, 42.8, 26.5      32768 x 5120, 8 rows -, 31.5, 24.2
//     5120 x 1000, 3 rows    -, 4.9, 6.5           32768 x 1000, 3 rows -, 9.1, 8.3
// A block whose waves do not share goes on to other outputs with the x it holds
// (5120 x 131071, 8 rows: 78 us, 92 with blocks of one tile).
void plan_few(const sili_fp4_linear_args &a, int64_t parts, LinearLaunch &L) {
    auto tiles = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    LinearPlan &p = L.plan;
    FewLinear &f = L.few;
    L.few_tokens = true;
    p.token_tiles = 1;
    p.steps = (int32_t)tiles(a.w.n_in, FEW_TURN);
    const int64_t turns = std::max<int64_t>(1, p.steps), rows = a.tokens * parts, rt = parts == 1 ? 16 : parts == 2 ? 8 : 4;
    const int64_t base = tiles(a.w.n_out, 16 * FEW_WAVES), want = std::max<int64_t>(1, 512 / base);
    int64_t splits = 1;
    f.share = 1;
    if (rows <= 8 && turns <= 64) {
        while (f.share < 8 && f.share * 2 <= std::min(want, turns)) f.share *= 2;
    } else {
        splits = std::clamp<int64_t>(want, 1, std::max<int64_t>(1, turns / 4));
    }
    f.tiles = (int32_t)tiles(a.w.n_out, 16 * FEW_WAVES / f.share);
    // words of LDS beside x, and what x may take of 112 KiB
    const int64_t words = FEW_WAVES * 16 * (FEW_ROW + FEW_TURN / a.w.group), room = (112 << 8) - words;
    splits = std::max(splits, tiles(turns, std::max<int64_t>(1, (room / rows - 4) / (FEW_TURN / 2))));
    p.chunk = (int32_t)tiles(turns, splits);
    p.splits = (int32_t)tiles(turns, p.chunk);
    f.row_words = p.chunk * (FEW_TURN / 2) + 4;
    L.lds = (uint32_t)(4 * std::max<int64_t>(words + rows * f.row_words, rt * 16 * FEW_WAVES));
    L.blocks = f.tiles;
    if (f.share == 1 && p.steps > 0) {
        const int64_t fit = std::max<int64_t>(1, 256 * std::clamp<int64_t>((160 << 10) / L.lds, 1, 3) / p.splits);
        L.blocks = tiles(f.tiles, tiles(f.tiles, fit));
    }
}

LinearLaunch plan_linear(const sili_fp4_linear_args &a) {
    LinearLaunch L;
    LinearPlan &p = L.plan;
    auto tiles = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    const int64_t parts = a.dtype == SILI_F32 ? 3 : a.dtype == SILI_F16 ? 2 : 1;
    if (a.tokens <= (parts == 1 ? 16 : parts == 2 ? 8 : 4)) {
        plan_few(a, parts, L);
        return L;
    }
    p.steps = (int32_t)tiles(a.w.n_in, LINEAR_STEP);
    const int64_t steps = std::max<int64_t>(1, p.steps);
    L.wn = a.tokens <= 32 ? 4 : 2;
    L.mt = a.tokens <= 64 ? 1 : 2;
    p.token_tiles = (int32_t)tiles(a.tokens, 32 * L.mt * (4 / L.wn));
    L.blocks = tiles(a.w.n_out, 64 * L.wn) * p.token_tiles;
    const int64_t want = std::clamp<int64_t>(512 / std::max<int64_t>(1, L.blocks), 1, std::max<int64_t>(1, steps / 4));
    p.chunk = (int32_t)tiles(steps, want);
    p.splits = (int32_t)tiles(steps, p.chunk);
    return L;
}

size_t linear_bytes(const sili_fp4_linear_args &a, const LinearPlan &p) {
    return p.splits == 1 ? 0 : (size_t)a.tokens * (size_t)a.w.n_out * (size_t)p.splits * sizeof(float);
}

template <typename T, int G>
void run_linear(const sili_fp4_linear_args &a, const LinearLaunch &L, hipStream_t st) {
    const LinearPlan &p = L.plan;
    const dim3 grid((unsigned)L.blocks, (unsigned)p.splits);
    if (L.few_tokens) {
        launch(k_linear_few<T, G>, grid, dim3(64 * FEW_WAVES), L.lds, st, a, p, L.few);
    } else if (L.wn == 4) {
        launch(k_linear_many<T, G, 4, 1>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 4, 1>::LDS, st, a, p);
    } else if (L.mt == 1) {
        launch(k_linear_many<T, G, 2, 1>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 2, 1>::LDS, st, a, p);
    } else {
        launch(k_linear_many<T, G, 2, 2>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 2, 2>::LDS, st, a, p);
    }
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
    return linear_bytes(a, plan_linear(a).plan);
}

void fp4_linear(const sili_fp4_linear_args &a, hipStream_t st) {
    check_linear(a);
    if (a.tokens == 0 || a.w.n_out == 0) return;
    require(a.y && (a.x || a.w.n_in == 0), "fp4_linear: NULL buffer");
    LinearLaunch L = plan_linear(a);
    const size_t need = linear_bytes(a, L.plan);
    require(need == 0 || (a.workspace && aligned(a.workspace, 16) && a.workspace_bytes >= need),
            "fp4_linear: workspace too small or not 16-byte aligned");
    L.plan.part = static_cast<float *>(a.workspace);
    require(L.blocks * 1024 < (int64_t(1) << 32), "fp4_linear: too many tokens or outputs");
    with_dtype(a.dtype, [&](auto z) {
        with_group(a.w.group, [&](auto g) { run_linear<decltype(z), decltype(g)::value>(a, L, st); });
    });
    if (L.plan.splits > 1) {
        const int64_t joins = std::min<int64_t>((a.tokens * a.w.n_out + JOIN_TPB - 1) / JOIN_TPB, 4096);
        launch(k_linear_join, dim3((unsigned)joins), dim3(JOIN_TPB), 0, st, a, L.plan);
    }
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
