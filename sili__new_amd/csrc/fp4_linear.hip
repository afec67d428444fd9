// fp4_linear.hip -- dense weights in 4 bits with a scale a group of inputs:
// packed, and multiplied.
#include "block_ops.hpp"
#include "mma.hpp"
#include "wave.hpp"

#include <algorithm>
#include <type_traits>

namespace sili {

namespace {

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

// A thread takes 8 inputs, group / 8 neighbours a group.  Bound by the codec's arithmetic, 286
// vector instructions for the 8 in any type: 32768 x 5120 139 us from fp32 (5.5 TB/s), 132 from
// bf16, 128 from f16 (3.3 TB/s, floor 83); 131071 x 5120 570, 491, 493.
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
// lane's column having one scale.
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

// Few tokens, up to 16: rows of one product a part of x (PM of them), or, with
// 8 (two parts) or 4 (three) at most, of one product in all (PM 1), whose row r + RT k
// holds part k of token r.  A block cuts x once, in LDS; its waves then run by themselves, 16 outputs each (or a share of their
// inputs, joined in LDS), in turns of 256 inputs asked for AHEAD turns before.  Eight
// lanes load 128 bytes of a row of codes, and four its scales, so that the cache is
// asked for a line and not for a lane at a time; the wave turns them in LDS of its
// own into what a product's lanes need.  Blocks that share outputs (splits) are
// joined through the workspace.
constexpr int FEW_TURN = 2 * LINEAR_STEP;  // inputs
constexpr int FEW_ROW = FEW_TURN / 8 + 4;  // words of a row of codes in LDS: 16 rows in all banks
// Waves of a block, us with 4, 8 and 16: 1 fp32 token of 5120 x 32768 29.1, 21.8, 25.5; 8 bf16
// of 32768 x 5120 40.0, 23.7, 27.5; 16 fp32 of 5120 x 32768 46.9, 38.8, 36.7.  Turns ahead, us
// with 1, 2 and 3: the first of these 20.5, 21.8, 22.7 (its scales bf16) and with fp32 scales,
// which take the most loads, 26.3 with 1 and 23.0 with 2; the others 23.3, 23.7, 24.5 and 38.2,
// 38.8, 39.8.
constexpr int FEW_WAVES = 8;
constexpr int AHEAD = 2;

struct FewLinear {
    int32_t share;      // waves that share outputs: 1, 2, 4, 8
    int32_t tiles;      // of a block's outputs; share 1: a block takes every gridDim.x-th
    int32_t row_words;  // of x in LDS, a row
};

template <typename T, int G, int PM>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_linear_few(sili_fp4_linear_args a, LinearPlan pl, FewLinear few) {
    constexpr int P = q_parts<T>(), RT = P == PM ? 16 : P == 2 ? 8 : 4;
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
    const uint32_t *xs = s_x + ((P == PM ? 0 : min(r16 / RT, P - 1)) * tokens + min(r16 % RT, tokens - 1)) * few.row_words + 4 * g;
    const uint32_t *ws = s_w + r16 * FEW_ROW + g;
    const int part_words = tokens * few.row_words;

    auto store = [&](int64_t t, int64_t n, float y) {
        if (pl.splits > 1) pl.part[((int64_t)split * tokens + t) * a.w.n_out + n] = y;
        else store_as(a.y, a.out_dtype, t * a.y_stride + n, y);
    };
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto join_parts = [&] {  // lane: output r16, rows 4 g + j of A
        if (P == PM) return;
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
                if (s % (G / 32) == 0) sum = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                const u32x4 b = codes8(ws[4 * s]);
#pragma unroll
                for (int k = 0; k < PM; ++k) sum = mma(*reinterpret_cast<const u32x4 *>(x + k * part_words + 16 * s), b, sum);
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
// tokens, in products of 32 x 32 outputs x 16 inputs.  LDS holds, twice, a step's
// codes and scales and KC inputs of x cut into its parts: the next ones' loads are
// under this one's products, each a line of the cache at a time.  A lane of a product
// has eight codes of an even (lower half of the wave) or odd word of a row, so a row
// keeps its even words before its odd ones.  Rows are padded by 16 bytes: 16 lanes'
// 16 bytes lie in all banks.  A wave's 64 outputs take each operand of x twice,
// which is what LDS can give the matrix cores.  128 bf16 tokens of 5120 x 131071: 234 us,
// 0.73 PFLOP/s; the products and what turns their codes alone 134, the rest writes to LDS
// (34), loads (46) and outputs (14), which do not overlap with them.
template <typename T, int G, int WN, int MT>
struct ManyLinear {
    static constexpr int P = q_parts<T>(), WM = 4 / WN, BM = 32 * MT * WM, BN = 64 * WN;
    static constexpr int KC = sizeof(T) == 4 ? 32 : 64, ROW = KC + 8;  // bf16 of a row of x
    static constexpr int GS = LINEAR_STEP / G, C_ROW = LINEAR_STEP / 8 + 4;  // words of a row of codes
    static constexpr int X_WORDS = P * BM * ROW / 2, W_WORDS = BN * C_ROW, S_WORDS = BN * GS;
    static constexpr int LDS = 2 * 4 * (X_WORDS + W_WORDS + S_WORDS);
};

template <typename T, int G, int WN, int MT>
__global__ __launch_bounds__(256, 2) void k_linear_many(sili_fp4_linear_args a, LinearPlan pl) {
    using M = ManyLinear<T, G, WN, MT>;
    constexpr int P = M::P, BM = M::BM, BN = M::BN, KC = M::KC, ROW = M::ROW, GS = M::GS, C_ROW = M::C_ROW;
    constexpr int TPR = KC / 8, PASS = 256 / TPR, PASSES = (BM + PASS - 1) / PASS;  // threads a row of x; rows a pass
    constexpr int SUB = LINEAR_STEP / KC, KS = KC / 16;                             // chunks a step; products a chunk
    constexpr int US = (G < KC ? G : KC) / 16;                                      // ... of one scale
    static_assert(SUB % 2 == 0, "a step's chunks begin with an even one");
    constexpr bool WHOLE = P == 1 && G > KC;  // sums go on into the next chunk (more parts: their registers are dearer)
    constexpr int NW = BN * 4 / 256, NS = BN * GS / 256 > 0 ? BN * GS / 256 : 1;    // loads a thread
    extern __shared__ __align__(16) uint32_t s_many[];
    uint32_t *s_w = s_many + 2 * M::X_WORDS;
    float *s_s = reinterpret_cast<float *>(s_w + 2 * M::W_WORDS);
    uint16_t *s_x = reinterpret_cast<uint16_t *>(s_many);  // [2][P][BM][ROW]
    const int tid = threadIdx.x, wave = (int)uniform(tid >> 6), lane = tid & 63, hf = lane >> 5, r32 = lane & 31;
    const int wn = wave % WN, wm = wave / WN;
    const int tile = blockIdx.x / pl.token_tiles, t0 = (blockIdx.x - tile * pl.token_tiles) * BM, split = blockIdx.y;
    const int64_t b0 = (int64_t)tile * BN;
    const int k_end = (int)a.w.n_in;

    const T *x[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int64_t token = min((int64_t)t0 + i * PASS + tid / TPR, a.tokens - 1);
        x[i] = (const T *)a.x + token * a.x_stride;
    }
    const uint8_t *codes[NW];  // 16 bytes: inputs 32 (tid % 4) .. + 31 of a row
#pragma unroll
    for (int i = 0; i < NW; ++i) codes[i] = a.w.codes + min(b0 + 64 * i + tid / 4, a.w.n_out - 1) * a.w.codes_stride;
    int64_t scales[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) scales[i] = min(b0 + (256 * i + tid) / GS, a.w.n_out - 1) * a.w.scales_stride;

    // Every thread asks for the same number of loads whatever the step: the compiler
    // could else not tell which of them are still under way, and would wait for all.
    // What lies past the inputs asks for their last ones, and is stored as zeros.
    Loose<T, 8> xs2[2][PASSES];  // of even and odd chunks
    auto fetch_x = [&](Loose<T, 8>(&xs)[PASSES], int k0) {
        const int k = min(k0 + 8 * (tid % TPR), k_end - 8);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) xs[i] = *reinterpret_cast<const Loose<T, 8> *>(x[i] + k);
    };
    auto put_x = [&](const Loose<T, 8>(&xs)[PASSES], int k0, int buf) {
        const uint32_t keep = k0 + 8 * (tid % TPR) < k_end ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = i * PASS + tid / TPR;
            if (BM % PASS != 0 && row >= BM) continue;
            u32x4 part[P];
            if constexpr (P == 1) {
                part[0] = __builtin_bit_cast(u32x4, xs[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t c[P];
                    cut_bf16<P>((float)xs[i].v[2 * j], (float)xs[i].v[2 * j + 1], c);
#pragma unroll
                    for (int k = 0; k < P; ++k) part[k][j] = c[k];
                }
            }
#pragma unroll
            for (int k = 0; k < P; ++k) *reinterpret_cast<u32x4 *>(s_x + ((buf * P + k) * BM + row) * ROW + 8 * (tid % TPR)) = part[k] & keep;
        }
    };
    struct Weights {
        uint4 w[NW];
        uint32_t sc[NS];
    } w2[2];  // of even and odd steps
    const int groups = k_end / G;
    auto fetch_w = [&](Weights &v, int step) {
        const int k = min(step * LINEAR_STEP + 32 * (tid % 4), k_end - 32), s = min(step * GS + tid % GS, groups - 1);
#pragma unroll
        for (int i = 0; i < NW; ++i) v.w[i] = *reinterpret_cast<const uint4 *>(codes[i] + k / 2);
        if (a.w.scale_dtype == SILI_F32) {
#pragma unroll
            for (int i = 0; i < NS; ++i) v.sc[i] = ((const uint32_t *)a.w.scales)[scales[i] + s];
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) v.sc[i] = ((const uint16_t *)a.w.scales)[scales[i] + s];
        }
    };
    auto put_w = [&](const Weights &v, int step, int buf) {
        const uint32_t keep = step * LINEAR_STEP + 32 * (tid % 4) < k_end ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            uint32_t *row = s_w + buf * M::W_WORDS + (64 * i + tid / 4) * C_ROW + 2 * (tid % 4);
            *reinterpret_cast<uint2 *>(row) = make_uint2(v.w[i].x & keep, v.w[i].z & keep);
            *reinterpret_cast<uint2 *>(row + LINEAR_STEP / 16) = make_uint2(v.w[i].y & keep, v.w[i].w & keep);
        }
        if (BN * GS >= 256 || tid < BN * GS) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                s_s[buf * M::S_WORDS + 256 * i + tid] = step * GS + tid % GS < groups ? scale_of(a.w.scale_dtype, v.sc[i]) : 0.0f;
        }
    };

    f32x16 acc[2][MT], sum[2][MT];
    const f32x16 zero = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = zero;

    const int first = split * pl.chunk, last = min(pl.steps, first + pl.chunk);
    if (first < last) {
        fetch_w(w2[0], first);
        fetch_x(xs2[0], first * LINEAR_STEP);
        fetch_w(w2[1], first + 1);
        fetch_x(xs2[1], first * LINEAR_STEP + KC);
        put_w(w2[0], first, 0);
        put_x(xs2[0], first * LINEAR_STEP, 0);
    }
    // Step `step`, whose parity is `odd`: asks for the step after the next, and in each
    // chunk for the chunk after the next.
    auto run = [&](int step, auto odd) {
        constexpr int ODD = decltype(odd)::value;
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
            constexpr int wbuf = ODD;
            const int buf = sub & 1;
            __syncthreads();
            if (sub == 0) fetch_w(w2[ODD], step + 2);
            const int k0 = step * LINEAR_STEP + sub * KC;
            fetch_x(xs2[buf], k0 + 2 * KC);
            uint32_t ww[2][KS];
            const uint32_t *wr = s_w + wbuf * M::W_WORDS + (64 * wn + r32) * C_ROW + (LINEAR_STEP / 16) * hf + KS * sub;
            const float *sr = s_s + wbuf * M::S_WORDS + (64 * wn + r32) * GS;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < KS; ++k) ww[t][k] = wr[32 * t * C_ROW + k];
            float f[2][US < KS ? KS / US : 1];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < KS / US; ++i) f[t][i] = sr[32 * t * GS + (sub * KS + i * US) / (G / 16)];
            const uint16_t *base = s_x + (buf * P * BM + 32 * MT * wm + r32) * ROW + 8 * hf;
            // x's operands, FEED products before theirs: the compiler left to itself waits
            // for each read of LDS.  Two and four before theirs take the same time within 1 %
            // (128 tokens of 5120 x 131071: 239 and 237 us); four do not fit the registers of two
            // tiles beside a chunk's own sums (128 of 5120 x 32768, groups of 32: 84 and 128 us).
            constexpr int NQ = KS * P * MT, FEED = WHOLE || MT == 1 ? 4 : 2;
            u32x4 av[NQ], b[2];
#pragma unroll
            for (int q = 0; q < NQ + FEED; ++q) {
                if (q < NQ) {
                    const int s = q / (P * MT), p = q / MT % P, m = q % MT;
                    av[q] = *reinterpret_cast<const u32x4 *>(base + (p * BM + 32 * m) * ROW + 16 * s);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (q < FEED) continue;
                const int o = q - FEED, s = o / (P * MT), p = o / MT % P, m = o % MT, k = sub * KS + s;  // product of the step
                const bool begins = WHOLE ? k % (G / 16) == 0 : s % US == 0, ends = WHOLE ? (k + 1) % (G / 16) == 0 : (s + 1) % US == 0;
                if (p == 0 && m == 0) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) b[t] = codes8(ww[t][s]);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) sum[t][m] = mma(av[o], b[t], begins && p == 0 ? zero : sum[t][m]);
                if (ends && p == P - 1 && m == MT - 1) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) acc[t][i][j] = __builtin_fmaf(sum[t][i][j], f[t][s / US], acc[t][i][j]);
                            // here: the compiler would keep the sums of several scales until the accumulators' next use
                            __asm__ volatile("" : "+v"(acc[t][i]));
                        }
                }
            }
            put_x(xs2[buf ^ 1], k0 + KC, buf ^ 1);
            if (sub == SUB - 1) put_w(w2[ODD ^ 1], step + 1, wbuf ^ 1);
        }
    };
    for (int step = first; step < last; step += 2) {
        run(step, std::integral_constant<int, 0>{});
        if (step + 1 < last) run(step + 1, std::integral_constant<int, 1>{});
    }
    // lane: output r32; result 4 i + j of a tile is token 8 i + 4 hf + j
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int64_t n = b0 + 64 * wn + 32 * t + r32;
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

Rows codes_of(const sili_fp4_weights &w) { return rows_of(w.codes, w.n_out, w.n_in / 2, w.codes_stride, 1); }
Rows scales_of(const sili_fp4_weights &w) { return rows_of(w.scales, w.n_out, w.n_in / w.group, w.scales_stride, dtype_size(w.scale_dtype)); }

void check_linear(const sili_fp4_linear_args &a) {
    check_weights(a.w, "fp4_linear");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "fp4_linear: unknown dtype");
    require(a.out_dtype == SILI_F32 || a.out_dtype == SILI_BF16 || a.out_dtype == SILI_F16, "fp4_linear: unknown out_dtype");
    require(a.tokens >= 0 && a.tokens <= INT32_MAX, "fp4_linear: tokens out of range");
}

// How a call is launched.
struct LinearLaunch {
    int64_t blocks = 0;
    bool few_tokens = false, merged = false;
    int wn = 0, mt = 0;  // more tokens: a block's shape
    uint32_t lds = 0;
    int64_t most_splits = 1;  // few tokens: what plan.splits is rounded down from; no less for more tokens
    LinearPlan plan{};
    FewLinear few{};
};

// Few tokens.  512 blocks of 8 waves fill the GPU twice over.  Fewer (outputs / 128):
// waves share outputs where x is small (up to 4 rows of up to 16384 inputs, of which a
// block holds all), else blocks split the inputs and are joined.  us of a call, its
// inputs x outputs, rows of x (tokens times parts); share 1, the best share, the best
// splits:
//     5120 x 32768, 3 rows   19.6, 18.7, 21.3      5120 x 5120, 1 row   -, 5.8, 9.0
//     5120 x 32768, 8 rows   23.0, 26.0, 23.0      5120 x 5120, 8 rows  16.5, 8.7, 9.3
//     5120 x 32768, 16 rows  27.5, 42.8, 26.5      32768 x 5120, 8 rows -, 31.5, 24.2
//     5120 x 1000, 3 rows    -, 4.9, 6.5           32768 x 1000, 3 rows -, 9.1, 8.3
// (8 rows share well by 4 but not by 8, and lose by 2: they split.  Inputs that LDS does
// not hold split only: 4 rows of 16384 x 5120 14.0, shared and split 25.9, 3 rows 14.0 and
// 17.3; x 1000 8.2 and 10.6.)  A split takes four turns at least: 8 bf16 tokens, us with 2, 4
// and 8, 1024 x 5120 6.9, 5.6, -; 4096 x 1000 6.5, 8.6, 10.4, x 5120 8.6, 9.4, 11.3; 16384 x 1000
// 8.3, 8.8, 11.1; 32768 x 1000 12.3, 10.5, 11.7.  A block whose
// waves do not share goes on to other outputs with the x it holds (5120 x 131071, 8
// rows: 78 us, 92 with blocks of one tile).  More than 16 tokens' kernel took 48 us for
// 5 fp32 tokens of 5120 x 32768, this one 28.
void plan_few(const sili_fp4_linear_args &a, int64_t parts, LinearLaunch &L) {
    auto tiles = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    LinearPlan &p = L.plan;
    FewLinear &f = L.few;
    L.few_tokens = true;
    p.token_tiles = 1;
    p.steps = (int32_t)tiles(a.w.n_in, FEW_TURN);
    const int64_t turns = std::max<int64_t>(1, p.steps), rows = a.tokens * parts;
    L.merged = rows <= (parts == 3 ? 12 : 16);
    const int64_t rt = !L.merged || parts == 1 ? 16 : parts == 2 ? 8 : 4;
    const int64_t base = tiles(a.w.n_out, 16 * FEW_WAVES), want = std::max<int64_t>(1, 512 / base);
    int64_t splits = 1;
    f.share = 1;
    // words of LDS beside x, what x may take of 112 KiB, and the turns of x that it holds
    const int64_t words = FEW_WAVES * 16 * (FEW_ROW + FEW_TURN / a.w.group), room = (112 << 8) - words;
    const int64_t held = std::max<int64_t>(1, (room / rows - 4) / (FEW_TURN / 2));
    if (rows <= 4 && turns <= std::min<int64_t>(64, held)) {
        while (f.share < 8 && f.share * 2 <= std::min(want, turns)) f.share *= 2;
    } else {
        splits = std::clamp<int64_t>(want, 1, std::max<int64_t>(1, turns / 4));
    }
    f.tiles = (int32_t)tiles(a.w.n_out, 16 * FEW_WAVES / f.share);
    splits = std::max(splits, tiles(turns, held));
    L.most_splits = splits;
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
    if (a.tokens <= 16) {
        plan_few(a, parts, L);
        return L;
    }
    p.steps = (int32_t)tiles(a.w.n_in, LINEAR_STEP);
    const int64_t steps = std::max<int64_t>(1, p.steps);
    // A block's waves lie side by side over 256 outputs, or in two rows over 128 (us, inputs
    // 5120, groups of 128: 32 bf16 tokens x 32768 outputs 37 and 44, x 5120 14.3 and 16.0,
    // fp32 55 and 87; 33 tokens 52 and 45, 18.4 and 16.1, 89 and 88).  In bf16 a wave takes 64
    // tokens where tiles of 64 are filled in pairs and 8192 steps of 128 x 128 x 128 are left,
    // 32 a CU (us with one tile and two: 5120 x 131071 128 tokens 278 and 237, 65 264 and 228,
    // 192 403 and 421; x 32768 128 76.0 and 76.6, 256 140 and 117; 2048 x 65536 128 59 and 53;
    // 32768 x 5120 128 87 and 78, 256 165 and 132; and of fewer steps 8192 x 8192 128 38 and 40,
    // 2048 x 32768 33 and 41, 5120 x 5120 25.5 and 27.0, 1024 x 32768 20.8 and 31.4).  In f16 and
    // fp32 it loses at every size (128 of 5120 x 32768 110 and 138, 163 and 188).
    const int64_t pairs = tiles(a.tokens, 128);
    L.wn = a.tokens <= 32 ? 4 : 2;
    L.mt = a.dtype == SILI_BF16 && tiles(a.tokens, 64) == 2 * pairs && tiles(a.w.n_out, 128) * pairs * steps >= 8192 ? 2 : 1;
    p.token_tiles = (int32_t)tiles(a.tokens, 32 * L.mt * (4 / L.wn));
    L.blocks = tiles(a.w.n_out, 64 * L.wn) * p.token_tiles;
    // A split takes four steps at least: 64 bf16 tokens, us with 2, 4 and 8, 1024 x 1000 9.3,
    // 10.3, 12.6; 4096 x 1000 10.6, 11.0, 14.1, x 5120 17.2, 16.1, 16.5; 16384 x 1000 17.4, 14.4, 15.9.
    const int64_t want = std::clamp<int64_t>(512 / std::max<int64_t>(1, L.blocks), 1, std::max<int64_t>(1, steps / 4));
    p.chunk = (int32_t)tiles(steps, want);
    p.splits = (int32_t)tiles(steps, p.chunk);
    return L;
}

// A workspace for the call and for those of fewer tokens, which may split where it does
// not: tokens x splits at most, over the plans that plan_linear takes up to a.tokens.
// Blocks of 64 or 128 tokens and 128 outputs split into 512 / blocks at most, so those of more
// than 32 tokens need 128 x 512 / (outputs / 128) rows of sums however many they are.
size_t linear_bytes(const sili_fp4_linear_args &a, const LinearPlan &p) {
    auto tiles = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    sili_fp4_linear_args few = a;
    few.tokens = std::min<int64_t>(a.tokens, 16);
    LinearLaunch L;
    plan_few(few, a.dtype == SILI_F32 ? 3 : a.dtype == SILI_F16 ? 2 : 1, L);
    int64_t rows = L.most_splits > 1 ? few.tokens * L.most_splits : 0;
    const int64_t steps = tiles(a.w.n_in, LINEAR_STEP) / 4;
    auto more = [&](int64_t tokens, int64_t blocks, int64_t most) {
        const int64_t splits = std::min(512 / blocks, steps);
        if (splits > 1) rows = std::max(rows, std::min(tokens * splits, most));
    };
    if (a.tokens > 16) more(std::min<int64_t>(a.tokens, 32), tiles(a.w.n_out, 256), INT64_MAX);
    if (a.tokens > 32) more(a.tokens, tiles(a.w.n_out, 128), 128 * 512 / tiles(a.w.n_out, 128));
    if (p.splits > 1) rows = std::max(rows, a.tokens * p.splits);
    return (size_t)rows * (size_t)a.w.n_out * sizeof(float);
}

template <typename T, int G>
void run_linear(const sili_fp4_linear_args &a, const LinearLaunch &L, hipStream_t st) {
    const LinearPlan &p = L.plan;
    const dim3 grid((unsigned)L.blocks, (unsigned)p.splits);
    if (L.few_tokens) {
        launch(L.merged ? k_linear_few<T, G, 1> : k_linear_few<T, G, q_parts<T>()>, grid, dim3(64 * FEW_WAVES), L.lds, st, a, p, L.few);
    } else if (L.wn == 4) {
        launch(k_linear_many<T, G, 4, 1>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 4, 1>::LDS, st, a, p);
    } else if (L.mt == 1) {
        launch(k_linear_many<T, G, 2, 1>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 2, 1>::LDS, st, a, p);
    } else {
        if constexpr (__is_same(T, __bf16)) launch(k_linear_many<T, G, 2, 2>, grid, dim3(256), (uint32_t)ManyLinear<T, G, 2, 2>::LDS, st, a, p);
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
    const Rows in = rows_of(a.rows, a.w.n_out, a.w.n_in, a.row_stride, dtype_size(a.dtype)), codes = codes_of(a.w), scales = scales_of(a.w);
    require(!meet(codes, in) && !meet(scales, in) && !meet(codes, scales), "fp4_pack: outputs overlap the rows or each other");
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
    return a.tokens == 0 || a.w.n_out == 0 ? 0 : linear_bytes(a, plan_linear(a).plan);
}

void fp4_linear(const sili_fp4_linear_args &a, hipStream_t st) {
    check_linear(a);
    if (a.tokens == 0 || a.w.n_out == 0) return;
    require(a.y && (a.x || a.w.n_in == 0), "fp4_linear: NULL buffer");
    LinearLaunch L = plan_linear(a);
    const size_t need = L.plan.splits == 1 ? 0 : linear_bytes(a, L.plan);  // what other calls need is theirs
    require(need == 0 || (a.workspace && aligned(a.workspace, 16) && a.workspace_bytes >= need),
            "fp4_linear: workspace too small or not 16-byte aligned");
    L.plan.part = static_cast<float *>(a.workspace);
    require(L.blocks * 512 < (int64_t(1) << 32) && L.plan.splits <= 65535, "fp4_linear: too many tokens, outputs or inputs");
    require(apart(a.tokens, a.w.n_out, a.y_stride), "fp4_linear: rows of y overlap");
    const Rows y = rows_of(a.y, a.tokens, a.w.n_out, a.y_stride, dtype_size(a.out_dtype)), work = row(a.workspace, (int64_t)need, 1);
    for (const Rows &r : {rows_of(a.x, a.tokens, a.w.n_in, a.x_stride, dtype_size(a.dtype)), codes_of(a.w), scales_of(a.w)})
        require(!meet(y, r) && !meet(work, r), "fp4_linear: y or the workspace overlaps an input");
    require(!meet(y, work), "fp4_linear: y overlaps the workspace");
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
