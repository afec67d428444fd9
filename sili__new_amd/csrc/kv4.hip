// kv4.hip -- a paged cache of keys and values in 4 bits: rows written and read
// back, and attention over it.
//
// A stored head is scale * code[c], code an E2M1 value; its scale is amax / 6,
// so the largest element takes the largest level.
#include "block_ops.hpp"
#include "mma.hpp"
#include "wave.hpp"

#include <algorithm>
#include <cmath>
#include <utility>

namespace sili {

namespace {

__device__ __forceinline__ float wave_max(float v) {
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// ---- rows ------------------------------------------------------------------------
// 4.25 bits stored a channel beside the row's own. A thread takes
// 8 channels of a (token, kv head), k's and v's: 16 or 32 bytes a load, a dword of
// k codes, four bytes of v codes.  The bytes of 16 tokens share their 16-byte runs
// of v codes, so a block takes one head of as many tokens as its threads cover:
// their bytes meet in one L2 (a block of one token's heads, whose neighbours run on
// other XCDs, wrote 2048 tokens of 40 fp32 heads in 42 us; so, 29, and 30 read).
// Writing is bound by the codec's arithmetic (vector units 88 % busy, 526
// instructions for 16 channels; 3.3 TB/s), reading back by neither it (53 %) nor
// the bytes (3.2 TB/s): short waves that wait for their codes, then for their stores.
constexpr int ROWS_TPB = 256;

// Maximum over the aligned group of N lanes.
template <int N>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = 1; d < N; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool packed, float (&x)[8]) {
    if (packed) {
        load_pack<T, 8>(p, x);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)p[j];
    }
}

// Codes of eight channels (channel j in nibble j), and the head's scale.  The factor
// is 6 * (1 / amax), rounded twice: within 2^-23 of 6 / amax, so a code is another
// than the exact quotient's only where that lies as near to the middle of two levels
// (25 of the 122944 pairs of bf16 values within 8 octaves of amax; of 6 / amax 10).  It is
// the format's definition, so that codes are equal wherever they are computed so.
template <int N>
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], float &scale) {
    float top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(x[j]));
        sum += x[j] * 0.0f;  // 0, or NaN for what is not finite
    }
    const float bad = sum != 0.0f || sum != sum ? INFINITY : 0.0f;
    top = group_max<N>(fmaxf(top, bad));
    const bool finite = top < INFINITY, zero = !finite || top < 0x1p-120f;
    const float inv = zero ? 0.0f : 6.0f * (1.0f / top);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= fp4_encode(x[j] * inv) << (4 * j);
    scale = !finite ? __builtin_nanf("") : zero ? 0.0f : top / 6.0f;
    return zero ? 0u : w;
}

template <typename T, int D, bool WRITE>
__global__ __launch_bounds__(ROWS_TPB) void k_kv4_rows(sili_kv4_rows_args a, bool packed) {
    constexpr int N = D / 8;  // threads of a head
    const sili_kv4_cache &c = a.cache;
    const uint32_t H = (uint32_t)c.kv_heads, h = blockIdx.x % H;
    const uint32_t t = blockIdx.x / H * (ROWS_TPB / N) + threadIdx.x / N, sub = threadIdx.x % N;
    if (t >= (uint32_t)a.tokens) return;
    const int32_t slot = a.slots[t];
    const uint32_t ps = (uint32_t)c.page_size;
    const bool held = slot >= 0 && (int64_t)slot < c.n_pages * c.page_size;
    if (WRITE && !held) return;
    const uint32_t page = held ? (uint32_t)slot / ps : 0u, at = held ? (uint32_t)slot - page * ps : 0u;
    const int64_t first = ((int64_t)page * H + h) * ps;  // this head's first slot in the page
    T *k = (T *)a.k + t * a.k_token_stride + h * a.k_head_stride + 8 * sub;
    T *v = (T *)a.v + t * a.v_token_stride + h * a.v_head_stride + 8 * sub;
    uint32_t *kc = reinterpret_cast<uint32_t *>(c.k + (first + at) * (D / 2)) + sub;
    uint8_t *vc = c.v + (first + (at & ~15u)) * (D / 2) + 64 * sub + (at & 15u);  // channel pair 4 sub, key at % 16
    float *ks = c.k_scale + first + at, *vs = c.v_scale + first + at;
    if (WRITE) {
        float x[8], y[8], sk, sv;
        load8<T>(k, packed, x);
        load8<T>(v, packed, y);
        *kc = encode8<N>(x, sk);
        const uint32_t w = encode8<N>(y, sv);
#pragma unroll
        for (int j = 0; j < 4; ++j) vc[16 * j] = (uint8_t)(w >> (8 * j));
        if (sub == 0) {
            *ks = sk;
            *vs = sv;
        }
    } else {
        uint32_t w[2] = {0, 0};
        float s[2] = {0.0f, 0.0f};
        if (held) {
            w[0] = *kc;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[1] |= (uint32_t)vc[16 * j] << (8 * j);
            s[0] = *ks;
            s[1] = *vs;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            T *out = r ? v : k;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fp4_decode((w[r] >> (4 * j)) & 15u) * s[r];
            if (packed) {
                store_pack<T, 8>(out, x);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) out[j] = (T)x[j];
            }
        }
    }
}

// ---- attention -----------------------------------------------------------------
//
// Rows of a (request, kv head) are its query tokens times the group of query
// heads that share the kv head: row = token * group + head in group.  Both
// kernels take 64 keys a step on the bf16 matrix cores:
//
//   S^T = K q^T               codes x q
//   p   = exp2(c (k_scale S - m)),   l += p
//   O^T += V^T (v_scale p)^T  codes x weights
//
// E2M1 codes are exact in bf16, and the two scales of a key multiply its score
// and its weight in fp32, so the cache's values lose nothing; q and p enter in
// bf16 parts, each the nearest to what the parts before leave.  With the scores
// transposed a row is a lane's column in both products, so its statistics and
// its scaling need no exchange, and the key order is chosen so that the scores
// a lane holds are the k indices its share of the second product's right operand
// takes: no weight moves between lanes.
//
// The running maximum m is raised only when a score passes it by 2^8 (in exp2's
// argument 8): until then weights stay below 2^8 and nothing has to be rescaled.
constexpr float SLACK = 8.0f;

// Four keys of a channel pair (a dword of V) to the even and the odd channel.
__device__ __forceinline__ void codes_by_channel(uint32_t w, uint32_t (&even)[2], uint32_t (&odd)[2]) {
    const uint32_t a = codes<0>(w), b = codes<1>(w), c = codes<2>(w), d = codes<3>(w);
    even[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    odd[0] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    even[1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    odd[1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}
// x[j] *= what lane j of this row of 16 lanes holds (DPP row_newbcast, folded
// into the product).
template <int... J>
__device__ __forceinline__ void times_row(float (&x)[16], float s, std::integer_sequence<int, J...>) {
    ((x[J] *= dpp_f32<0x150 + J>(s)), ...);
}
__device__ __forceinline__ void times_scales(float (&x)[16], float s) { times_row(x, s, std::make_integer_sequence<int, 16>{}); }
__device__ __forceinline__ float lanes_max(float v) {  // over the four lanes of a row
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float lanes_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// bf16 parts of p: 24 bits for fp32, 16 for f16 and bf16.
template <typename T>
constexpr int p_parts() { return sizeof(T) == 4 ? 3 : 2; }
// Sum over the CP columns of a row, 16 / CP lanes apart in their 16.
template <int CP>
__device__ __forceinline__ float columns_sum(float v) {
    if (CP >= 2) v += dpp_f32<DPP_ROW_ROR8>(v);
    if (CP >= 4) v += dpp_f32<DPP_ROW_ROR4>(v);
    return v;
}

// How a launch cuts the work, set on the host.
struct AttendPlan {
    int32_t kv_heads, group;  // query heads a kv head
    uint32_t group_inv;       // floor(2^32 / group), at most 2^32 - 1
    int32_t n_pages, most;    // pages of the cache; keys that max_len and the table allow
    int32_t window;           // 0: none
    bool q_packed, out_packed;  // rows of q in 16-byte pieces; of out in pieces of 4 elements
    int32_t groups_per_page;  // page_size / 16
    int32_t page_shift;       // its logarithm, or -1
    int32_t splits, chunk;    // keys a split takes: a multiple of a block's step
    int32_t waves;            // of a block whose waves share rows
    int32_t join_rows;        // rows such a block joins at most
    int32_t columns;          // columns a row takes
    int32_t row_tiles;        // tiles of 16 rows a wave of the few-rows kernel takes
    int32_t many;             // the most rows of a request for the few-rows kernel; more: the other
    float c;                  // |scale| log2(e)
    bool negative;            // scale < 0: the sign goes to q
    const uint64_t *ancestors;  // trees: the new tokens that a token sees
    float *part_o;            // [tokens * q_heads][splits][D], unnormalised
    float2 *part_ml;          // [tokens * q_heads][splits]: m c, l
};

// The query token of a row: row / group (the estimate is at most one too low).
__device__ __forceinline__ int32_t token_of(const AttendPlan &pl, int32_t row) {
    const int32_t q = (int32_t)__umulhi((uint32_t)row, pl.group_inv);
    return q + (row - q * pl.group >= pl.group ? 1 : 0);
}
// Keeps a wave-uniform branch that is seldom taken a branch: the compiler would
// else turn it into selects that every step pays for, or keep its conditions.
__device__ __forceinline__ void stay_branch(int32_t &x, int32_t &y) { __asm__ volatile("" : "+v"(x), "+v"(y)); }
// Four channels of an output row.
template <typename T>
__device__ __forceinline__ void store4(T *out, const float (&x)[4], bool packed) {
    if (packed) {
        store_pack<T, 4>(out, x);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = (T)x[j];
    }
}

// A request's query tokens: the first, how many it has, and how many of them are
// computed: the launch and the join's LDS are sized for max_new and for the
// batch's tokens, which q_start may pass (it does where a step brought more tokens
// than its buffers hold).  A negative start, or an end before it: none.
struct Queries {
    int32_t first, all, n;
};
__device__ __forceinline__ Queries queries_of(const sili_kv4_attend_args &a, int req) {
    const int32_t from = a.q_start[req], upto = a.q_start[req + 1];
    Queries q;
    q.first = max(from, 0);
    q.all = from < 0 ? 0 : max(upto, from) - from;
    q.n = max(0, min(q.all, min((int32_t)a.max_new, (int32_t)a.tokens - q.first)));
    return q;
}

// Keys that query i of n sees, [begin, end), both within the keys there are
// whatever the length says.
struct KeyRange {
    int32_t base, cap, window;  // keys before the first query, keys there are
    bool causal;
    __device__ __forceinline__ KeyRange(const sili_kv4_attend_args &a, const AttendPlan &pl, const Queries &q, int req) {
        const int32_t len = max(a.kv_lens[req], 0);
        base = len - q.all;
        cap = min(len, pl.most);
        window = pl.window;
        causal = a.causal != 0;
    }
    __device__ __forceinline__ int32_t end(int32_t i) const { return causal ? max(0, min(cap, base + i + 1)) : cap; }
    __device__ __forceinline__ int32_t begin(int32_t i) const {
        const int32_t upto = base + i + 1;  // negative where the query comes before the first key
        return window > 0 && upto > window ? min(cap, upto - window) : 0;
    }
};

// What a drafted token sees: the keys [begin, context) before the request's new
// tokens, and base + j for the bits j of mask.  A window drops the earliest.
struct TreeRange {
    int32_t base, cap, window, all;
    __device__ __forceinline__ TreeRange(const KeyRange &kr, const Queries &q) : base(kr.base), cap(kr.cap), window(kr.window), all(q.all) {}
    __device__ __forceinline__ int32_t context() const { return max(0, min(base, cap)); }
    // of all of a request's tokens: no key before, none from, the keys that every one sees
    __device__ __forceinline__ int32_t first() const { return window > 0 ? max(0, context() - window) : 0; }
    __device__ __forceinline__ int32_t last() const { return min(cap, context() + SILI_TREE_MOST); }
    __device__ __forceinline__ int32_t all_first() const {
        return window > 0 ? (int32_t)max((int64_t)0, min((int64_t)cap, (int64_t)base + SILI_TREE_MOST - window)) : 0;
    }
    __device__ __forceinline__ int32_t of(uint64_t &mask) const {  // begin; cuts the mask
        mask &= all < SILI_TREE_MOST ? (uint64_t(1) << max(all, 0)) - 1 : ~uint64_t(0);
        if (window <= 0) return 0;
        int32_t n = __popcll(mask);
        const int64_t from = (int64_t)base + n - window;
        for (; n > window; --n) mask &= mask - 1;
        return (int32_t)max((int64_t)0, min((int64_t)cap, from));
    }
};
// Bit j (of 16): the row sees key at + j.
__device__ __forceinline__ uint32_t seen16(const TreeRange &tr, int32_t begin, uint64_t mask, int32_t at) {
    auto below = [](int32_t n) { return n >= 16 ? 0xFFFFu : n > 0 ? (1u << n) - 1u : 0u; };
    const int32_t off = at - tr.base;  // of the mask's bits
    const uint32_t drafted = off >= SILI_TREE_MOST || off <= -16 ? 0u : (uint32_t)(off >= 0 ? mask >> off : mask << -off);
    return ((below(tr.context() - at) & ~below(begin - at)) | drafted) & below(tr.cap - at);
}

// Registers allow this many waves on a SIMD without spilling.
template <typename T, int D, int CP, int R = 1>
constexpr int waves_per_simd() {
    if (R > 1) return 2;
    constexpr bool lean = __is_same(T, __bf16) || (CP > 1 && D < 256);  // no more than two parts in registers
    return (D == 64 ? 4 : D == 128 ? 3 : 2) - (lean ? 0 : 1);
}

// Few rows: a tile of 16 a block, whose waves take a step of keys each in turn and
// are joined in LDS; every byte of the cache goes from memory to one wave's
// registers, a step ahead.  Memory bounds it (8 kv heads of 5.1 K keys a request,
// 128 requests: 153 us, 4.6 TB/s of the 5.65 that the loads alone reach).  With
//     16x16 tile x, row of K  ->  key 16 (row / 4) + 4 x + row % 4
// a lane's results of the four score tiles are the keys 16 g .. 16 g + 15, g =
// lane / 16.  The left operands come from memory as the lane needs them: a
// quarter of a K row, and 16 keys of a V channel pair, are 16 bytes each.
//
// CP > 1: with 16 / CP rows at most, the parts of q and p go to the columns that
// would be empty instead of to products of their own: column r + (16 / CP) k
// holds part k of row r.  Scores are summed over a row's columns (rotations
// within 16 lanes), so every one of them holds the row's weights and takes its
// own part of them; the outputs are summed once, at the end.
//
// TREE: rows are drafted tokens, which see the context and their ancestors.  Steps
// before the new tokens are as without; the last one or two take a bit a key.  R
// tiles of rows share a step's turned codes.  The vector units bound it
// there (64 requests of 28 tokens x 5 heads over 5.1 K keys: 377 us, 0.47
// PFLOP/s; 69 % busy with the codes and the softmax, the matrix cores 37 %).
template <typename T, int D, int WAVES, int CP, bool TREE, int R = 1>
__global__ __launch_bounds__(64 * WAVES, (waves_per_simd<T, D, CP, R>())) void k_attend_few(sili_kv4_attend_args a, AttendPlan pl) {
    constexpr int QP = q_parts<T>(), PP = p_parts<T>();
    constexpr int KS = D / 32;   // steps of 32 channels
    constexpr int CT = D / 32;   // blocks of 32 output channels
    constexpr int RT = 16 / CP;  // rows of a tile
    constexpr int BR = R * RT;   // ... of a block
    constexpr int QM = CP > 1 ? 1 : QP, PM = CP > 1 ? 1 : PP;  // products each
    static_assert(CP == 1 || (CP >= QP && CP >= PP), "parts fit the columns");
    extern __shared__ float s_join[];
    const sili_kv4_cache &cache = a.cache;
    const int wave = (int)uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
    const int my_row = r16 % RT, my_part = r16 / RT;
    const int H = pl.kv_heads, group = pl.group;
    const int h = blockIdx.x % H, tile = blockIdx.x / H, split = blockIdx.y, req = blockIdx.z;
    const int32_t *table = a.block_table + (int64_t)req * a.table_width;
    constexpr int32_t stride = 64 * WAVES;
    // the page of the first step, asked for before the lengths are here (the
    // table has the entry whatever they say)
    int32_t key = split * pl.chunk + 64 * wave;
    auto entry = [&](int32_t k) {
        const int32_t mine = (k >> 4) + g;
        return table[pl.page_shift >= 0 ? mine >> pl.page_shift : mine / pl.groups_per_page];
    };
    int32_t page = -1;
    if (pl.window == 0 && key + 16 * g < pl.most) page = entry(key);

    const Queries qs = queries_of(a, req);
    const KeyRange kr(a, pl, qs, req);
    const int32_t n_rows = qs.n * group;
    const int32_t first = tile * BR;
    if (n_rows > pl.many || first >= n_rows) return;
    const int32_t i_first = token_of(pl, first), i_last = token_of(pl, min(first + BR - 1, n_rows - 1));
    const TreeRange tr(kr, qs);
    const int32_t lo = (TREE ? tr.first() : kr.begin(i_first)) & ~63, hi = TREE ? tr.last() : kr.end(i_last);
    // what every row sees
    const int32_t all_end = TREE ? tr.context() : kr.end(i_first), all_begin = TREE ? tr.all_first() : kr.begin(i_last);
    const int32_t c1 = lo + min(hi - lo, (split + 1) * pl.chunk);

    uint32_t take_q[QP], take_p[PP];  // CP > 1: the part this lane's column holds
#pragma unroll
    for (int k = 0; k < QP; ++k) take_q[k] = my_part == k ? ~0u : 0u;
#pragma unroll
    for (int k = 0; k < PP; ++k) take_p[k] = my_part == k ? ~0u : 0u;

    // this lane's rows, one of each tile
    uint64_t my_mask[R];
    int32_t end[R], begin[R];
    u32x4 q[R][KS][QM];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t row = min(first + r * RT + my_row, n_rows - 1), i = token_of(pl, row);
        my_mask[r] = TREE ? pl.ancestors[qs.first + i] : 0;
        end[r] = kr.end(i);
        begin[r] = TREE ? tr.of(my_mask[r]) : kr.begin(i);
        const T *src = (const T *)a.q + (int64_t)(qs.first + i) * a.q_token_stride + (h * group + (row - i * group)) * a.q_head_stride + g * (D / 4);
        float xs[KS][8];
        if (pl.q_packed) {
#pragma unroll
            for (int s = 0; s < KS; ++s) load_pack<T, 8>(src + 8 * s, xs[s]);
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) xs[s][j] = (float)src[8 * s + j];
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = pl.negative ? -xs[s][j] : xs[s][j];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t part[QP];
                split_bf16<QP>(x[2 * j], x[2 * j + 1], part);
#pragma unroll
                for (int k = 0; k < QM; ++k) q[r][s][k][j] = CP > 1 && QP > 1 ? pick<QP>(part, take_q) : part[k];
            }
        }
    }

    float m[R], l[R];  // m in units of c; l of this lane's keys only
    f32x4 o[R][CT][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) o[r][ct][0] = o[r][ct][1] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }

    // The keys of a step as this lane needs them, loaded a step ahead: a part's
    // registers take the next step's as soon as this one's are used.
    uint32_t kw[4][KS];
    float ks, vs;  // scales of key 16 g + r16: the products take them from their lane
    uint4 vw[CT];
    bool held;   // the 16 keys of this lane group are in the cache
    int32_t at;  // where they lie, in groups of 16 keys
    auto page_of = [&](int32_t k) -> int32_t { return k + 16 * g < kr.cap ? entry(k) : -1; };
    auto locate = [&](int32_t k) {
        const int32_t mine = (k >> 4) + g;
        held = page >= 0 && page < pl.n_pages && k + 16 * g < kr.cap;
        const int32_t in_page = pl.page_shift >= 0 ? mine & (pl.groups_per_page - 1) : mine % pl.groups_per_page;
        at = held ? (page * H + h) * pl.groups_per_page + in_page : h * pl.groups_per_page;
    };
    auto load_k = [&] {
        const int32_t kat = __shfl(at, (r16 >> 2) << 4, 64);
        const uint8_t *kp = cache.k + ((int64_t)kat * 16 + (r16 & 3)) * (D / 2) + g * (D / 8);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint8_t *p = kp + 4 * x * (D / 2);
            if constexpr (D == 64) {
                const uint2 w = *reinterpret_cast<const uint2 *>(p);
                kw[x][0] = w.x;
                kw[x][1] = w.y;
            } else {
#pragma unroll
                for (int s = 0; s < KS; s += 4) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(p + 4 * s);
                    kw[x][s] = w.x;
                    kw[x][s + 1] = w.y;
                    kw[x][s + 2] = w.z;
                    kw[x][s + 3] = w.w;
                }
            }
        }
    };
    auto load_v = [&] {
        ks = cache.k_scale[(int64_t)at * 16 + r16];
        vs = cache.v_scale[(int64_t)at * 16 + r16];
        const uint8_t *vp = cache.v + (int64_t)at * (16 * (D / 2)) + r16 * 16;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) vw[ct] = *reinterpret_cast<const uint4 *>(vp + ct * 256);
    };
    if (pl.window > 0) {
        key = key < hi - lo ? lo + key : c1;
        page = page_of(key);
    }
    if (key < c1) {
        locate(key);
        load_k();
        load_v();
        page = page_of(key + stride);
    }
    for (; key < c1; key += stride) {
        f32x4 sc[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[r][x] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const u32x4 kk = codes8(kw[x][s]);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < QM; ++k) sc[r][x] = mma(kk, q[r][s][k], sc[r][x]);
            }
        // wave-uniform: every row sees every key of the step
        const bool here = held, whole = key >= all_begin && key + 64 <= all_end && __all(here);
        const bool more = key + stride < c1;
        if (more) {
            locate(key + stride);
            load_k();
            page = page_of(key + 2 * stride);
        }
        u32x4 p[R][2][PM];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[16], w[16];  // scores, then weights, of keys 16 g + 0 .. 15
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                v[j] = sc[r][j >> 2][j & 3];
                if (QP > 1) v[j] = columns_sum<CP>(v[j]);
            }
            times_scales(v, ks);
            uint32_t seen = 0;
            if (!whole) {
                if constexpr (TREE) {
                    seen = here ? seen16(tr, begin[r], my_mask[r], key + 16 * g) : 0u;
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = (seen & (1u << j)) != 0 ? v[j] : -INFINITY;
                } else {
                    int32_t from = here ? begin[r] - (key + 16 * g) : 16, to = end[r] - (key + 16 * g);
                    stay_branch(from, to);
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = j >= from && j < to ? v[j] : -INFINITY;
                }
            }
            float top = v[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, v[j]);
            top *= pl.c;
            if (__any(top > m[r] + SLACK)) {
                const float up = fmaxf(m[r], lanes_max(top));
                // a row without a key so far keeps m = -inf, and factor 1 on its zeros
                const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[r] - up);
                m[r] = up;
                l[r] *= keep;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    o[r][ct][0] *= keep;
                    o[r][ct][1] *= keep;
                }
            }
            const float ref = m[r] == -INFINITY ? 0.0f : m[r];
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                w[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[j], pl.c, -ref));
                sum += w[j];
            }
            l[r] += sum;
            times_scales(w, vs);
            if (!whole) {
                // a key that this row does not see may hold anything
                if constexpr (TREE) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) w[j] = (seen & (1u << j)) != 0 ? w[j] : 0.0f;
                } else {
                    int32_t from = here ? begin[r] - (key + 16 * g) : 16, to = end[r] - (key + 16 * g);
                    stay_branch(from, to);
#pragma unroll
                    for (int j = 0; j < 16; ++j) w[j] = j >= from && j < to ? w[j] : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t part[PP];
                    split_bf16<PP>(w[8 * e + 2 * j], w[8 * e + 2 * j + 1], part);
#pragma unroll
                    for (int k = 0; k < PM; ++k) p[r][e][k][j] = CP > 1 ? pick<PP>(part, take_p) : part[k];
                }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t e0[2], o0[2], e1[2], o1[2];
                codes_by_channel(e ? vw[ct].z : vw[ct].x, e0, o0);
                codes_by_channel(e ? vw[ct].w : vw[ct].y, e1, o1);
                const u32x4 even = {e0[0], e0[1], e1[0], e1[1]}, odd = {o0[0], o0[1], o1[0], o1[1]};
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int y = 0; y < PM; ++y) {
                        o[r][ct][0] = mma(even, p[r][e][y], o[r][ct][0]);
                        o[r][ct][1] = mma(odd, p[r][e][y], o[r][ct][1]);
                    }
            }
        if (more) load_v();
    }
    // lane: row r16 of a tile, channels 32 ct + 8 g + 2 i + (even, odd)
    const int ROWS = pl.join_rows;
    float *s_o = s_join, *s_m = s_join + WAVES * ROWS * D, *s_l = s_m + WAVES * ROWS;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float all = lanes_sum(l[r]);
        f32x4 sum[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum[ct][0][i] = columns_sum<CP>(o[r][ct][0][i]);
                sum[ct][1][i] = columns_sum<CP>(o[r][ct][1][i]);
            }
        const int row = r * RT + r16;
        if (first + row < n_rows && r16 < RT) {
            float *dst = s_o + (wave * ROWS + row) * D + 8 * g;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    dst[32 * ct + 2 * i] = sum[ct][0][i];
                    dst[32 * ct + 2 * i + 1] = sum[ct][1][i];
                }
            if (g == 0) {
                s_m[wave * ROWS + row] = m[r];
                s_l[wave * ROWS + row] = all;
            }
        }
    }
    __syncthreads();
    const int rows = min(BR, n_rows - first);
    for (int at = threadIdx.x; at < rows * (D / 4); at += 64 * WAVES) {
        const int row = at / (D / 4), ch = 4 * (at - row * (D / 4));
        float f[WAVES], mm = -INFINITY, ll = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            f[w] = s_m[w * ROWS + row];
            mm = fmaxf(mm, f[w]);
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            // a wave without keys has m = -inf and zeros
            f[w] = f[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(f[w] - mm);
            ll += f[w] * s_l[w * ROWS + row];
            const float4 x = *reinterpret_cast<const float4 *>(s_o + (w * ROWS + row) * D + ch);
            acc[0] += f[w] * x.x;
            acc[1] += f[w] * x.y;
            acc[2] += f[w] * x.z;
            acc[3] += f[w] * x.w;
        }
        const int32_t i = token_of(pl, first + row);
        const int64_t token = qs.first + i, qh = h * group + (first + row - i * group);
        if (pl.splits > 1) {
            const int64_t slot = (token * a.q_heads + qh) * pl.splits + split;
            if (ll != 0.0f) *reinterpret_cast<float4 *>(pl.part_o + slot * D + ch) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (ch == 0) pl.part_ml[slot] = make_float2(mm, ll);
        } else {
            const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] *= inv;
            store4<T>((T *)a.out + token * a.out_token_stride + qh * a.out_head_stride + ch, acc, pl.out_packed);
            if (a.lse && ch == 0)
                a.lse[token * a.q_heads + qh] = ll != 0.0f ? (mm + __builtin_amdgcn_logf(ll)) * 0.69314718f : -INFINITY;
        }
    }
}

// Many rows: 128 a block, 32 a wave.  The block turns a step's codes into bf16 once,
// in LDS (two buffers: the next step's codes are asked for before this one's
// products and written after them), and each wave takes its 32x32 tiles from
// there.  With tile x of K's keys in order, a lane's 16 results are the keys
// 32 x + 8 a + 4 hf + b (a, b < 4; hf = lane / 32), so V's keys lie in LDS in the
// order 0-3, 8-11, 4-7, 12-15 of every 16: eight at 16 s + 8 hf are the lane's
// own.  Rows of LDS are padded by 16 bytes, which spreads eight lanes' 16 bytes
// over all banks.  A weight enters in one bf16 part: its rounding is as large as
// the output's own, together 1.4 times that (2 x 2047 tokens: 0.0023 of the output's
// norm off against 0.0017); a second part is half as many products again (532 us
// against 428).  The sum l takes the weights unrounded.  Half of a step's scores
// are scaled under the products of the other half, and the weights of 16 keys are
// taken under the products of the 16 before; without, the wave's vector work and
// its products take turns (2 x 2047 tokens of 40 heads under a window of 4096: 455
// us, with it 430, 0.75 PFLOP/s, at 2.38 GHz; a card that idled begins at 2.06 GHz
// and takes 500).
// Issue bounds it, with a last round of blocks that leaves half of their places empty.
constexpr int MANY_WAVES = 4, MANY_ROWS = 32 * MANY_WAVES;

constexpr int MANY_D = 128;

struct ManyLds {
    static constexpr int D = MANY_D;
    static constexpr int K_ROW = 2 * D + 16, V_ROW = 2 * 64 + 16;  // bytes
    uint8_t k[64 * K_ROW];  // [key][channel]
    uint8_t v[D * V_ROW];   // [channel][key], the even channels before the odd ones
    float ks[64], vs[64];  // ks times c
    int32_t held[4];        // the group of 16 keys is in the cache
};

__global__ __launch_bounds__(64 * MANY_WAVES, 2) void k_attend_many(sili_kv4_attend_args a, AttendPlan pl) {
    using T = __bf16;
    constexpr int D = MANY_D, KS = D / 16, CT = D / 32;
    using Lds = ManyLds;
    extern __shared__ __align__(16) uint8_t s_many[];
    Lds *lds = reinterpret_cast<Lds *>(s_many);
    const sili_kv4_cache &cache = a.cache;
    const int tid = threadIdx.x, wave = (int)uniform(tid >> 6), lane = tid & 63, hf = lane >> 5, r32 = lane & 31;
    const int H = pl.kv_heads, group = pl.group;
    const int h = blockIdx.x % H, tile = blockIdx.x / H, req = blockIdx.z;
    const int32_t *table = a.block_table + (int64_t)req * a.table_width;
    const Queries qs = queries_of(a, req);
    const KeyRange kr(a, pl, qs, req);
    const int32_t n_rows = qs.n * group;
    const int32_t block_first = tile * MANY_ROWS;
    if (n_rows <= pl.many || block_first >= n_rows) return;
    const int32_t c0 = kr.begin(token_of(pl, block_first)) & ~63, c1 = kr.end(token_of(pl, min(block_first + MANY_ROWS, n_rows) - 1));

    // this wave's rows (past the last: the last again), and this lane's
    const int32_t first = block_first + 32 * wave, row = min(first + r32, n_rows - 1), my_i = token_of(pl, row);
    const int32_t i_first = token_of(pl, min(first, n_rows - 1)), i_last = token_of(pl, min(first + 31, n_rows - 1));
    const int32_t end = kr.end(my_i), begin = kr.begin(my_i);
    const int32_t w_begin = kr.begin(i_first), w_end = first < n_rows ? kr.end(i_last) : 0;  // what any row sees
    const int32_t all_end = kr.end(i_first), all_begin = kr.begin(i_last);                   // what every row sees

    u32x4 q[KS];  // channels 16 s + 8 hf + 0 .. 7
    {
        const T *src = (const T *)a.q + (int64_t)(qs.first + my_i) * a.q_token_stride + (h * group + (row - my_i * group)) * a.q_head_stride + 8 * hf;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8];
            load8<T>(src + 16 * s, pl.q_packed, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) q[s][j] = pl.negative ? pack_bf16(-x[2 * j], -x[2 * j + 1]) : pack_bf16(x[2 * j], x[2 * j + 1]);
        }
    }

    float m = -INFINITY, l = 0.0f;  // m in units of c; l of this lane's keys only
    f32x16 o[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[ct][i] = 0.0f;

    // A step's codes: a thread turns 32 channels of a key, and 16 keys of a channel
    // pair, of the step's group of 16 keys tid / 64; consecutive threads write
    // consecutive rows of LDS.  Their pages are asked for a step before them.
    uint4 kw, vw;
    float scale = 0.0f;
    int32_t held = 0, page = -1, scale_page = -1;
    const int scale_group = (tid & 63) >> 4;
    auto entry = [&](int32_t key, int sub) {  // of group `sub` of 16 keys
        const int32_t mine = (key >> 4) + sub;
        return 16 * mine < kr.cap ? table[pl.page_shift >= 0 ? mine >> pl.page_shift : mine / pl.groups_per_page] : -1;
    };
    auto find = [&](int32_t key) {
        page = entry(key, wave);
        scale_page = entry(key, scale_group);
    };
    // where the group lies, in groups of 16 keys; of a page outside the cache: some place in it
    auto place = [&](int32_t pg, int32_t key, int sub) -> int64_t {
        const int32_t mine = (key >> 4) + sub;
        const int32_t in_page = pl.page_shift >= 0 ? mine & (pl.groups_per_page - 1) : mine % pl.groups_per_page;
        return (int64_t)((pg >= 0 && pg < pl.n_pages ? pg : 0) * H + h) * pl.groups_per_page + in_page;
    };
    auto fetch = [&](int32_t key) {
        const int64_t at = place(page, key, wave) * (8 * D);
        kw = *reinterpret_cast<const uint4 *>(cache.k + at + (lane % 16) * (D / 2) + lane / 16 * 16);
        vw = *reinterpret_cast<const uint4 *>(cache.v + at + lane * 16);
        if (tid < 128) {
            scale = (tid < 64 ? cache.k_scale : cache.v_scale)[place(scale_page, key, scale_group) * 16 + (tid & 15)];
            held = scale_page >= 0 && scale_page < pl.n_pages;
        }
    };
    auto unpack = [&](Lds &b) {
        u32x4 *kd = reinterpret_cast<u32x4 *>(b.k + (16 * wave + lane % 16) * Lds::K_ROW + lane / 16 * 64);
        kd[0] = codes8(kw.x);
        kd[1] = codes8(kw.y);
        kd[2] = codes8(kw.z);
        kd[3] = codes8(kw.w);
        uint32_t e[4][2], d[4][2];
        codes_by_channel(vw.x, e[0], d[0]);
        codes_by_channel(vw.y, e[1], d[1]);
        codes_by_channel(vw.z, e[2], d[2]);
        codes_by_channel(vw.w, e[3], d[3]);
        uint8_t *vd = b.v + lane * Lds::V_ROW + wave * 32;
        *reinterpret_cast<u32x4 *>(vd) = (u32x4){e[0][0], e[0][1], e[2][0], e[2][1]};
        *reinterpret_cast<u32x4 *>(vd + 16) = (u32x4){e[1][0], e[1][1], e[3][0], e[3][1]};
        *reinterpret_cast<u32x4 *>(vd + D / 2 * Lds::V_ROW) = (u32x4){d[0][0], d[0][1], d[2][0], d[2][1]};
        *reinterpret_cast<u32x4 *>(vd + D / 2 * Lds::V_ROW + 16) = (u32x4){d[1][0], d[1][1], d[3][0], d[3][1]};
        if (tid < 128) (tid < 64 ? b.ks : b.vs)[tid & 63] = tid < 64 ? scale * pl.c : scale;
        if (tid < 64 && (tid & 15) == 0) b.held[tid >> 4] = held;
    };

    if (c0 < c1) {
        find(c0);
        fetch(c0);
        find(c0 + 64);
        unpack(lds[0]);
    }
    int buf = 0;
    for (int32_t key = c0; key < c1; key += 64, buf ^= 1) {
        __syncthreads();
        const Lds &b = lds[buf];
        const bool more = key + 64 < c1;
        if (more) {
            fetch(key + 64);
            find(key + 128);
        }
        if (key < w_end && key + 64 > w_begin) {
            f32x16 sc[2];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[x][i] = 0.0f;
            float ref = m == -INFINITY ? 0.0f : m;
            float v[32];  // scores less ref, then weights: 16 x + 4 a + b
            // K's operands, AHEAD products before theirs: the compiler left to itself
            // waits for each read of LDS.  The first half's scores are scaled under the
            // second half's products.
            constexpr int AHEAD = 4;
            u32x4 kk[2 * KS];
            f32x4 f[8];
#pragma unroll
            for (int s = 0; s < 2 * KS + AHEAD; ++s) {
                if (s < 2 * KS) {
                    kk[s] = *reinterpret_cast<const u32x4 *>(b.k + (32 * (s / KS) + r32) * Lds::K_ROW + 32 * (s % KS) + 16 * hf);
                    if (s % 2 == 1) f[s / 2] = *reinterpret_cast<const f32x4 *>(b.ks + 8 * (s / 2) + 4 * hf);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int t = s - AHEAD;
                if (t >= 0) sc[t / KS] = mma(kk[t], q[t % KS], sc[t / KS]);
                if (t >= KS + 2) {  // the first half's last product is two before this one
                    constexpr int LEFT = KS - 2;
#pragma unroll
                    for (int j = 16 * (t - KS - 2) / LEFT; j < 16 * (t - KS - 1) / LEFT; ++j) {
                        v[j] = __builtin_fmaf(sc[0][j], f[j >> 2][j & 3], -ref);
                        __asm__ volatile("" : "+v"(v[j]));  // here, not past the next branch
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int j = 16; j < 32; ++j) v[j] = __builtin_fmaf(sc[1][j - 16], f[j >> 2][j & 3], -ref);
            // wave-uniform: every row sees every key of the step
            const int4 in = *reinterpret_cast<const int4 *>(b.held);
            const bool whole = key >= all_begin && key + 64 <= all_end && uniform(in.x & in.y & in.z & in.w) != 0;
            const int32_t there[4] = {in.x, in.y, in.z, in.w};
            // w[0 .. n) (v[at ..), j: 16 x + 4 a + b) where this row sees the key, else `other`
            auto hide = [&](float *w, int at, int n, float other) {
                int32_t from = begin - key - 4 * hf, to = end - key - 4 * hf;
                stay_branch(from, to);
#pragma unroll
                for (int j = at; j < at + n; ++j) {
                    const int32_t k = 8 * (j >> 2) + (j & 3);
                    w[j - at] = k >= from && k < to && there[j >> 3] != 0 ? w[j - at] : other;
                }
            };
            if (!whole) hide(v, 0, 32, -INFINITY);
            float top = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
            top += ref;
            if (__any(top > m + SLACK)) {
                const float up = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
                // a row without a key so far keeps m = -inf, and factor 1 on its zeros
                const float keep = up == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - up);
                m = up;
                l *= keep;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) o[ct] *= keep;
                const float less = up == -INFINITY ? 0.0f : up - ref;
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] -= less;
            }
            // Weights of 16 keys at a time, under the products of the 16 before.
            float sum = 0.0f, w[8];
            auto weigh = [&](int t) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float4 f = *reinterpret_cast<const float4 *>(b.vs + 8 * (2 * t + y) + 4 * hf);
                    const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float g = __builtin_amdgcn_exp2f(v[8 * t + 4 * y + i]);
                        sum += g;
                        w[4 * y + i] = g * fs[i];
                    }
                }
            };
            u32x4 vv[2][CT];
            auto values = [&](int t) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) vv[t & 1][ct] = *reinterpret_cast<const u32x4 *>(b.v + (32 * ct + r32) * Lds::V_ROW + 32 * t + 16 * hf);
            };
            weigh(0);
            values(0);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (!whole) hide(w, 8 * t, 8, 0.0f);  // a key that this row does not see may hold anything
                u32x4 p;
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = pack_bf16(w[2 * j], w[2 * j + 1]);
                if (t < 3) {
                    values(t + 1);
                    weigh(t + 1);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) o[ct] = mma(vv[t & 1][ct], p, o[ct]);
                if (t < 3) {  // the order: reads of LDS, the four packs; a product, two exp2, four others; ...
                    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                    }
                }
            }
            l += sum;
        }
        if (more) unpack(lds[buf ^ 1]);
    }
    l += __shfl_xor(l, 32, 64);

    // lane: row r32; result 4 a + b of tile ct is row 32 ct + 8 a + 4 hf + b of V's
    // channels in LDS, even ones in the first half of the tiles
    const int64_t token = qs.first + my_i, qh = h * group + (row - my_i * group);
    if (first + r32 >= n_rows) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    T *out = (T *)a.out + token * a.out_token_stride + qh * a.out_head_stride;
#pragma unroll
    for (int ct = 0; ct < CT / 2; ++ct)
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const int i = 4 * (y >> 1) + 2 * (y & 1), ch = 2 * (32 * ct + 8 * (y >> 1) + 4 * hf) + 4 * (y & 1);
            const float x[4] = {o[ct][i] * inv, o[ct + CT / 2][i] * inv, o[ct][i + 1] * inv, o[ct + CT / 2][i + 1] * inv};
            store4<T>(out + ch, x, pl.out_packed);
        }
    if (a.lse && hf == 0) a.lse[token * a.q_heads + qh] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.69314718f : -INFINITY;
}

// Joins the splits of a row: a block a (row, kv head, request); D / 4 threads
// share a split's channels, and the block's thread groups take every GROUPS-th
// split.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attend_join(sili_kv4_attend_args a, AttendPlan pl) {
    constexpr int GROUPS = 256 / (D / 4);
    __shared__ float4 s_acc[256];
    __shared__ float s_w[4], s_sum[GROUPS];
    const int32_t row = blockIdx.x, h = blockIdx.y, req = blockIdx.z;
    const int32_t group = pl.group;
    const Queries qs = queries_of(a, req);
    const int32_t n_rows = qs.n * group;
    if (n_rows > pl.many || row >= n_rows) return;
    const int32_t i = token_of(pl, row);
    const int64_t token = qs.first + i, qh = h * group + (row - i * group);
    const int64_t id = token * a.q_heads + qh;
    const float2 *ml = pl.part_ml + id * pl.splits;
    float m = -INFINITY;
    for (int s = threadIdx.x; s < pl.splits; s += 256) m = fmaxf(m, ml[s].x);
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_w[0], s_w[1]), fmaxf(s_w[2], s_w[3]));
    const int part = threadIdx.x / (D / 4), ch = 4 * (threadIdx.x % (D / 4));
    const float *src = pl.part_o + id * pl.splits * D + ch;
    float l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int s = part; s < pl.splits; s += GROUPS) {
        const float2 x = ml[s];
        // a split without keys has written no sums
        const float4 v = x.y != 0.0f ? *reinterpret_cast<const float4 *>(src + (int64_t)s * D) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float f = x.y != 0.0f ? __builtin_amdgcn_exp2f(x.x - m) : 0.0f;
        l += f * x.y;
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
    }
    s_acc[threadIdx.x] = acc;
    if (ch == 0) s_sum[part] = l;
    __syncthreads();
    if (part != 0) return;
    l = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < GROUPS; ++k) {
        const float4 v = s_acc[k * (D / 4) + threadIdx.x];
        l += s_sum[k];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    store4<T>((T *)a.out + token * a.out_token_stride + qh * a.out_head_stride + ch, x, pl.out_packed);
    if (a.lse && ch == 0) a.lse[id] = l != 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.69314718f : -INFINITY;
}

void check_cache(const sili_kv4_cache &c, const char *what) {
    const std::string w(what);
    auto need = [&](bool ok, const char *m) {
        if (!ok) throw_error(SILI_ERR_INVALID, w + ": " + m);
    };
    need(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "head_dim is none of 64, 128, 256");
    need(c.page_size >= 16 && c.page_size % 16 == 0 && c.page_size <= 65536, "page_size is not a multiple of 16 up to 65536");
    need(c.kv_heads >= 1 && c.kv_heads <= 65535, "kv_heads out of range");
    need(c.n_pages >= 0 && c.n_pages <= (int64_t(1) << 31) / c.page_size, "more than 2^31 slots");
    need(c.n_pages == 0 || (c.k && c.v && c.k_scale && c.v_scale), "NULL cache");
    need(aligned(c.k, 16) && aligned(c.v, 16) && aligned(c.k_scale, 16) && aligned(c.v_scale, 16), "cache is not 16-byte aligned");
}

template <bool WRITE>
void rows(const sili_kv4_rows_args &a, hipStream_t st, const char *what) {
    check_cache(a.cache, what);
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "kv4 rows: unknown dtype");
    require(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "kv4 rows: tokens out of range");
    if (a.tokens == 0) return;
    require(a.slots && a.k && a.v, "kv4 rows: NULL buffer");
    const int64_t tokens = ROWS_TPB / (a.cache.head_dim / 8);  // of a block
    const int64_t blocks = (a.tokens + tokens - 1) / tokens * a.cache.kv_heads;
    require(blocks < (int64_t(1) << 32) / ROWS_TPB, "kv4 rows: too many rows");
    auto packs = [&](const void *p, int64_t ts, int64_t hs) {
        return aligned(p, (size_t)(8 * dtype_size(a.dtype))) && ts % 8 == 0 && hs % 8 == 0;
    };
    const bool packed = packs(a.k, a.k_token_stride, a.k_head_stride) && packs(a.v, a.v_token_stride, a.v_head_stride);
    const dim3 grid((unsigned)blocks);
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        switch (a.cache.head_dim) {
            case 64: launch(k_kv4_rows<T, 64, WRITE>, grid, dim3(ROWS_TPB), 0, st, a, packed); break;
            case 128: launch(k_kv4_rows<T, 128, WRITE>, grid, dim3(ROWS_TPB), 0, st, a, packed); break;
            default: launch(k_kv4_rows<T, 256, WRITE>, grid, dim3(ROWS_TPB), 0, st, a, packed); break;
        }
    });
    SILI_HIP(hipGetLastError());
}

void check_attend(const sili_kv4_attend_args &a, bool tree) {
    check_cache(a.cache, tree ? "kv4_attend_tree" : "kv4_attend");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "kv4_attend: unknown dtype");
    require(a.requests >= 0 && a.requests <= 65535, "kv4_attend: requests out of range");
    require(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "kv4_attend: tokens out of range");
    require(a.q_heads >= 1 && a.q_heads % a.cache.kv_heads == 0, "kv4_attend: q_heads is no multiple of kv_heads");
    require(a.q_heads <= 65535 && a.tokens * a.q_heads <= INT32_MAX, "kv4_attend: too many query heads");
    require(a.cache.n_pages * (a.cache.page_size / 16) * a.cache.kv_heads <= INT32_MAX, "kv4_attend: cache too large");
    require(a.table_width >= 0 && a.max_new >= 0 && a.max_len >= 0, "kv4_attend: negative size");
    require(a.max_len <= INT32_MAX && a.max_new <= INT32_MAX && a.table_width <= INT32_MAX, "kv4_attend: bound out of range");
    require(a.window >= 0 && (a.window == 0 || a.causal), "kv4_attend: a window needs the causal mask");
    require(!tree || (a.causal && a.max_new <= SILI_TREE_MOST), "kv4_attend_tree: not causal, or max_new is past SILI_TREE_MOST");
}

}  // namespace

void kv4_append(const sili_kv4_rows_args &a, hipStream_t st) { rows<true>(a, st, "kv4_append"); }
void kv4_read(const sili_kv4_rows_args &a, hipStream_t st) { rows<false>(a, st, "kv4_read"); }

namespace {

// Waves of a CU that run the few-rows kernel at once.
int waves_of(int dtype, int64_t head_dim, int columns) {
    int n = 0;
    with_dtype(dtype, [&](auto z) {
        using T = decltype(z);
        auto of = [&](auto d) {
            constexpr int D = decltype(d)::value;
            return 4 * (columns > 1 ? waves_per_simd<T, D, 2>() : waves_per_simd<T, D, 1>());
        };
        n = head_dim == 64 ? of(std::integral_constant<int, 64>{}) : head_dim == 128 ? of(std::integral_constant<int, 128>{})
                                                                                     : of(std::integral_constant<int, 256>{});
    });
    return n;
}

constexpr int64_t LEAST_KEYS = 256;  // of a split
constexpr int64_t FILL = 256 * 4;    // blocks of 4 waves that the GPU takes at once, at most

// [tokens][heads][d] elements as rows: tokens of heads, or heads of tokens where those are
// further apart.
Rows heads_of(const void *p, int64_t tokens, int64_t heads, int64_t d, int64_t token_stride, int64_t head_stride, int64_t bytes) {
    auto size = [](__int128 v) { return v < 0 ? -v : v; };
    const __int128 ts = (__int128)token_stride * bytes, hs = (__int128)head_stride * bytes;
    const bool by_token = tokens > 1 && (heads == 1 || size(ts) >= size(hs));
    const int64_t n = by_token ? tokens : heads, inner = by_token ? heads : tokens;
    const __int128 pitch = by_token ? ts : hs, step = by_token ? hs : ts, reach = (inner - 1) * step;
    return {(const char *)p + (int64_t)std::min<__int128>(0, reach), n, size(reach) + (__int128)d * bytes, pitch};
}

// Blocks read q, masks and lengths while others write.
void check_overlap(const sili_kv4_attend_args &a, const uint64_t *ancestors, size_t work_bytes) {
    const int64_t es = dtype_size(a.dtype), d = a.cache.head_dim, heads = a.cache.n_pages * a.cache.kv_heads, ps = a.cache.page_size;
    const Rows out = heads_of(a.out, a.tokens, a.q_heads, d, a.out_token_stride, a.out_head_stride, es);
    const Rows lse = row(a.lse, a.tokens * a.q_heads, 4), work = row(a.workspace, (int64_t)work_bytes, 1);
    const bool in_place = a.q == a.out && a.q_token_stride == a.out_token_stride && a.q_head_stride == a.out_head_stride;
    const Rows q = heads_of(a.q, a.tokens, a.q_heads, d, a.q_token_stride, a.q_head_stride, es);
    const Rows read[] = {row(ancestors, a.tokens, 8),
                         row(a.q_start, a.requests + 1, 4),
                         row(a.kv_lens, a.requests, 4),
                         row(a.block_table, a.requests, a.table_width * 4),
                         rows_of(a.cache.k, heads, ps * (d / 2), ps * (d / 2), 1),
                         rows_of(a.cache.v, heads, ps * (d / 2), ps * (d / 2), 1),
                         rows_of(a.cache.k_scale, heads, ps, ps, 4),
                         rows_of(a.cache.v_scale, heads, ps, ps, 4)};
    bool ok = (in_place || !meet(out, q)) && !meet(lse, q) && !meet(work, q);
    for (const Rows &r : read) ok = ok && !meet(out, r) && !meet(lse, r) && !meet(work, r);
    require(ok, "kv4_attend_tree: out, lse or the workspace overlaps an input");
    require(!meet(out, lse) && !meet(out, work) && !meet(lse, work), "kv4_attend_tree: out, lse and the workspace overlap");
}

// How a call is launched: requests of up to plan.many rows go to the few-rows
// kernel, `tiles` row tiles a (request, kv head), those of more to the other.
struct Launch {
    int64_t rows = 0, tiles = 0, many_tiles = 0;
    AttendPlan plan{};
};

Launch plan_attend(const sili_kv4_attend_args &a, bool tree) {
    Launch L;
    AttendPlan &p = L.plan;
    const int64_t group = a.q_heads / a.cache.kv_heads, heads = a.requests * a.cache.kv_heads;
    const int64_t rows = std::min(a.max_new, a.tokens) * group;  // of the longest request at most; below 2^31 as tokens * q_heads is
    const int64_t gpp = a.cache.page_size / 16, es = dtype_size(a.dtype);
    p.kv_heads = (int32_t)a.cache.kv_heads;
    p.group = (int32_t)group;
    p.group_inv = group == 1 ? ~0u : (uint32_t)((uint64_t(1) << 32) / (uint64_t)group);
    p.n_pages = (int32_t)a.cache.n_pages;
    p.most = p.n_pages == 0 ? 0 : (int32_t)std::min({a.max_len, a.table_width * a.cache.page_size, int64_t(INT32_MAX) - (1 << 20)});
    // lengths are int32, so a window of 2^31 - 1 hides nothing (max_len says less: positions
    // count the keys past it)
    p.window = a.window < INT32_MAX ? (int32_t)a.window : 0;
    p.q_packed = aligned(a.q, (size_t)(8 * es)) && a.q_token_stride % 8 == 0 && a.q_head_stride % 8 == 0;
    p.out_packed = aligned(a.out, (size_t)(4 * es)) && a.out_token_stride % 4 == 0 && a.out_head_stride % 4 == 0;
    p.groups_per_page = (int32_t)gpp;
    p.page_shift = (gpp & (gpp - 1)) == 0 ? (int32_t)__builtin_ctzll((unsigned long long)gpp) : -1;
    // a scale of zero leaves all scores equal; c > 0 keeps hidden ones at -inf
    p.c = std::max(std::fabs(a.scale) * 1.44269504f, 0x1p-100f);
    p.negative = a.scale < 0.0f;

    // The many-rows kernel pays where its blocks fill the GPU, two a CU (bf16, 8 kv
    // heads of 5 query heads each, chunks at the end of 4096 keys more, us of it and of
    // the other: 1280 blocks 452 and 625, 768 276 and 310, 640 214 and 258, 384 146 and
    // 152, 320 204 and 197 or 151 and 128, 160 142 and 104), in bf16 and at its
    // head_dim.  For fp32 and f16 a like kernel was slower at 1280 blocks (2 x 2047
    // tokens: 1200 and 1013, 873 and 743).  For head_dim 64 and 256 one was tried at 320
    // blocks only (133 and 98, 394 and 276), where that of 128 loses too: what it would
    // do at 512 and more is not known.  192 rows of 2048 keys took 33 us in the few-rows kernel, 51 in the
    // other.
    constexpr int64_t FEW_ROWS = 256;
    const int64_t many_tiles = (rows + MANY_ROWS - 1) / MANY_ROWS;
    if (!tree && a.dtype == SILI_BF16 && a.cache.head_dim == MANY_D && rows > FEW_ROWS && heads * many_tiles >= 512) L.many_tiles = many_tiles;
    p.many = L.many_tiles ? (int32_t)FEW_ROWS : INT32_MAX;

    const int parts = a.dtype == SILI_F32 ? 4 : 2;
    p.columns = rows <= 16 / parts ? parts : 1;
    // Trees of many rows in bf16, at head_dim 128: a wave takes two tiles of rows with the
    // same turned codes where that leaves 2048 blocks of 4096 keys and more (us with one
    // and two, 8 kv heads x 5, requests x rows of keys: 64 x 160 of 8192 441 and 397, of 4096
    // 228 and 214, of 300 60 and 66; 64 x 320 of 8192 742 and 657; 64 x 105 304 and 333, half
    // of the last pair being empty; 16 x 160 131 and 139; 8 x 160 96 and 112; 4 x 320 91 and
    // 98).  At head_dim 64 it gains nothing (64 x 160 of 8192: 279 and 281); of f16 and fp32,
    // whose q takes more registers, none was built.
    const int64_t reach_most = p.window > 0 ? std::min(p.most, p.window) : p.most;
    const bool paired = tree && a.dtype == SILI_BF16 && a.cache.head_dim == 128 && rows > 128 && heads * ((rows + 31) / 32) >= 2048 &&
                        reach_most >= 4096;
    p.row_tiles = paired ? 2 : 1;
    const int64_t tile_rows = 16 / p.columns * p.row_tiles;
    L.rows = std::min<int64_t>(rows, p.many);
    L.tiles = (L.rows + tile_rows - 1) / tile_rows;
    p.join_rows = (int32_t)std::min(tile_rows, rows);
    // keys a row tile can reach: its rows' windows, aligned to 64
    int64_t reach = p.most;
    if (p.window > 0) reach = std::min<int64_t>(reach, int64_t(p.window) + (tree ? SILI_TREE_MOST : (tile_rows - 1) / group + 1) + 63);
    const int64_t blocks = std::max<int64_t>(1, heads * L.tiles);
    // few blocks: as many waves in one as a CU holds, so that fewer splits are left
    // to join (40 heads of 131071 keys, 8 blocks a split: 31 + 5 us against 31 + 7
    // with 4 waves; 320 blocks of 2048 keys: 24 us against 22.6, a second round)
    const int wide = waves_of(a.dtype, a.cache.head_dim, p.columns);
    p.waves = blocks <= 128 ? wide : 4;
    const int64_t step = 64 * p.waves;
    // splits until every SIMD has as many waves as registers allow; fp32, which the
    // vector units bound, two at most (320 blocks of 2048 keys: 22.7 us, with a
    // second split 21.4 + 4.7 to join)
    const int64_t fill = 256 * std::max(1, std::min(wide, a.dtype == SILI_F32 ? 8 : wide) / p.waves);
    // A split takes 256 keys at least; of a tree whose blocks half fill the GPU 1280, for a
    // join costs 5 us (14 rows a block, us with 256 and 1280: head_dim 64 in f16 160 blocks of
    // 700 keys 12.4 and 7.3, of 1300 14.3 and 15.6, of 2600 18.5 and 17.5, 240 14.1 and 7.8, 16.1 and
    // 16.8, 20.6 and 20.7; head_dim 128 in fp32 192 of 700 18.8 and 12.7, of 1300 22.5 and 22.4;
    // 256 in bf16 256 of 700 25.5 and 16.9, 160 of 1300 23.3 and 27.9; with 2560 keys 700 the same,
    // 1300 less, 2600 more: 11.5 and 20.6 at the first of these; below 128 blocks 64 of 2600 at
    // head_dim 64 12.6 and 14.4).
    const int64_t least = tree && blocks >= 128 ? 1280 : LEAST_KEYS;
    const int64_t want = std::clamp<int64_t>(fill / blocks, 1, std::max<int64_t>(1, (reach + least - 1) / least));
    p.chunk = (int32_t)std::max(step, ((reach + want - 1) / want + step - 1) / step * step);
    p.splits = (int32_t)std::max<int64_t>(1, (reach + p.chunk - 1) / p.chunk);
    return L;
}

size_t part_bytes(const sili_kv4_attend_args &a, const AttendPlan &p, bool tree) {
    const size_t each = (size_t)a.cache.head_dim * sizeof(float) + sizeof(float2), rows = (size_t)a.tokens * (size_t)a.q_heads;
    const size_t own = p.splits == 1 ? 0 : rows * (size_t)p.splits * each;
    if (!tree) return own;
    // Fewer requests, tokens or keys may be split where these are not.  With requests x
    // max_new tokens at most, blocks x a tile's rows are no less than the tokens' rows, and a
    // call splits into FILL / blocks pieces and into one for 256 keys: rows x splits is
    // bounded whatever the call.
    const int64_t reach = p.window > 0 ? std::min<int64_t>(p.most, int64_t(p.window) + SILI_TREE_MOST + 63) : p.most;
    if (reach <= LEAST_KEYS) return own;
    const size_t pieces = (size_t)((reach + LEAST_KEYS - 1) / LEAST_KEYS);
    return std::max(own, std::min(rows * pieces, (size_t)FILL * (16 / p.columns)) * each);
}

template <typename T, int D, bool TREE>
void run_few(const sili_kv4_attend_args &a, const Launch &L, hipStream_t st) {
    AttendPlan p = L.plan;
    constexpr int PARTS = sizeof(T) == 4 ? 4 : 2;
    constexpr int WIDE = 4 * waves_per_simd<T, D, 1>(), WIDE_P = 4 * waves_per_simd<T, D, PARTS>();
    p.part_o = static_cast<float *>(a.workspace);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + a.tokens * a.q_heads * p.splits * D);
    const dim3 grid((unsigned)(L.tiles * a.cache.kv_heads), (unsigned)p.splits, (unsigned)a.requests), block(64 * p.waves);
    const uint32_t lds = p.waves * p.join_rows * (D + 2) * sizeof(float);
    if (p.columns > 1) {
        if (p.waves == WIDE_P) launch(k_attend_few<T, D, WIDE_P, PARTS, TREE>, grid, block, lds, st, a, p);
        else launch(k_attend_few<T, D, 4, PARTS, TREE>, grid, block, lds, st, a, p);
    } else if (p.row_tiles > 1) {
        if constexpr (TREE && __is_same(T, __bf16) && D == 128) launch(k_attend_few<T, D, 4, 1, TREE, 2>, grid, block, lds, st, a, p);
    } else {
        if (p.waves == WIDE) launch(k_attend_few<T, D, WIDE, 1, TREE>, grid, block, lds, st, a, p);
        else launch(k_attend_few<T, D, 4, 1, TREE>, grid, block, lds, st, a, p);
    }
    if (p.splits > 1)
        launch(k_attend_join<T, D>, dim3((unsigned)L.rows, (unsigned)a.cache.kv_heads, (unsigned)a.requests), dim3(256), 0, st, a, p);
}

}  // namespace

size_t kv4_attend_workspace(const sili_kv4_attend_args &a) {
    check_attend(a, false);
    return part_bytes(a, plan_attend(a, false).plan, false);
}

size_t kv4_attend_tree_workspace(const sili_kv4_attend_args &a) {
    check_attend(a, true);
    return part_bytes(a, plan_attend(a, true).plan, true);
}

namespace {

template <bool TREE>
void attend(const sili_kv4_attend_args &a, const uint64_t *ancestors, hipStream_t st) {
    check_attend(a, TREE);
    if (a.tokens == 0 || a.requests == 0 || a.max_new == 0) return;
    require(a.q && a.out && a.q_start && a.kv_lens, "kv4_attend: NULL buffer");
    require(a.block_table || a.table_width == 0, "kv4_attend: NULL block_table");
    require(!TREE || ancestors, "kv4_attend_tree: NULL ancestors");
    Launch L = plan_attend(a, TREE);
    L.plan.ancestors = ancestors;
    const size_t need = L.plan.splits == 1 ? 0 : part_bytes(a, L.plan, TREE);  // what other calls need is theirs
    require(need == 0 || (a.workspace && aligned(a.workspace, 16) && a.workspace_bytes >= need),
            "kv4_attend: workspace too small or not 16-byte aligned");
    const int64_t most = (int64_t(1) << 32) - 1;  // threads of a grid's x
    require(L.tiles * a.cache.kv_heads * 64 * L.plan.waves <= most && L.many_tiles * a.cache.kv_heads * 64 * MANY_WAVES <= most &&
                L.rows * (L.plan.splits > 1 ? 256 : 1) <= most && L.plan.splits <= 65535,
            "kv4_attend: too many rows or keys");
    if (TREE) check_overlap(a, ancestors, need);
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        switch (a.cache.head_dim) {
            case 64: run_few<T, 64, TREE>(a, L, st); break;
            case 128: run_few<T, 128, TREE>(a, L, st); break;
            default: run_few<T, 256, TREE>(a, L, st); break;
        }
    });
    if (L.many_tiles) {
        launch(k_attend_many, dim3((unsigned)(L.many_tiles * a.cache.kv_heads), 1, (unsigned)a.requests), dim3(64 * MANY_WAVES),
               (uint32_t)(2 * sizeof(ManyLds)), st, a, L.plan);
    }
    SILI_HIP(hipGetLastError());
}

}  // namespace

void kv4_attend(const sili_kv4_attend_args &a, hipStream_t st) { attend<false>(a, nullptr, st); }
void kv4_attend_tree(const sili_kv4_attend_args &a, const uint64_t *ancestors, hipStream_t st) { attend<true>(a, ancestors, st); }

}  // namespace sili
