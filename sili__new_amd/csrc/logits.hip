// logits.hip -- penalties for repeated tokens, biases and masks on logits.
//
// A block holds a chunk of the vocabulary of one request: it counts the
// request's history there in LDS (low 31 bits: how often past counted_from; top
// bit: before it), and then goes over the request's rows, two or eight tokens a
// thread and load, whose biases stay in registers.  A bit a token says whether it occurs at
// all: most eights ask for no count.  A row whose own path has tokens in the chunk
// adds them to the counts and takes them off again; the others pass without a
// barrier.  Rows begin at any element (vocabularies are odd): loads of 16 bytes at any
// address.  Bound by the bytes of the rows, in short calls by the launch and the scan of
// the history.
#include "block_ops.hpp"

#include <algorithm>
#include <type_traits>

namespace sili {

namespace {

constexpr uint32_t SEEN = 0x80000000u;

struct LogitsPlan {
    int32_t chunks, row_groups;  // blocks of a request
};

// N tokens a thread.
template <typename T, int TPB, int N>
__global__ __launch_bounds__(TPB, 8) void k_logits_constrain(sili_logits_constrain_args a, LogitsPlan pl) {
    constexpr int CHUNK = N * TPB;
    __shared__ __align__(16) uint32_t s_count[CHUNK];
    __shared__ uint32_t s_any[CHUNK / 32];
    const int tid = threadIdx.x, lane = tid & 63;
    // the first chunks of all requests first: vocabularies begin with their frequent tokens,
    // which take longest to count
    const uint32_t groups = (uint32_t)(a.requests * pl.row_groups), chunk = blockIdx.x / groups, block = blockIdx.x - chunk * groups;
    const uint32_t req = block / (uint32_t)pl.row_groups, part = block - req * (uint32_t)pl.row_groups;
    const int32_t c0 = (int32_t)chunk * CHUNK, c1 = (int32_t)min((int64_t)c0 + CHUNK, a.vocab);

    int32_t first = (int32_t)req, all = 1;
    if (a.q_start) {
        const int32_t from = a.q_start[req], upto = a.q_start[req + 1];
        first = max(from, 0);
        all = from < 0 || upto < from ? 0 : upto - from;
    }
    const int32_t n = min(all, (int32_t)a.rows - first);
    if ((int32_t)part >= n) return;

    // A wave's lanes hold the masks of the block's next 64 rows: their addresses are
    // there before they are needed.
    int32_t my_allow = -1;
    uint32_t path_lo = 0, path_hi = 0;
    auto look_up = [&](int32_t i) {  // of rows i, i + row_groups, ...
        const int64_t mine = i + (int64_t)lane * pl.row_groups;
        if (mine >= n) return;
        const int32_t row = first + (int32_t)mine;
        if (a.allow) my_allow = a.allow_row ? a.allow_row[row] : row;
        if (a.ancestors) {
            path_lo = (uint32_t)a.ancestors[row];
            path_hi = (uint32_t)(a.ancestors[row] >> 32);
        }
    };
    look_up((int32_t)part);

    const int32_t at = N * tid, v0 = c0 + at;  // this thread's tokens: v0 .. v0 + N - 1
    Loose<T, N> z;
    uint32_t bits = ~0u;  // those allowed
    auto fetch = [&](int32_t row, int slot) {
        const int32_t m = (int32_t)__builtin_amdgcn_readlane((uint32_t)my_allow, slot);
        const bool masked = a.allow && m >= 0 && m < a.n_allow;
        bits = masked && v0 < c1 ? a.allow[m * a.allow_stride + (v0 >> 5)] >> (v0 & 31) : ~0u;
        const T *src = (const T *)a.logits + row * a.logits_stride + v0;
        if (v0 + N <= c1) {
            z = *reinterpret_cast<const Loose<T, N> *>(src);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (v0 + j < c1) z.v[j] = src[j];
        }
    };
    fetch(first + (int32_t)part, 0);

    const bool counts = a.history != nullptr || a.ancestors != nullptr;
    int32_t mine = -1;  // token `lane` of the request's path, where it is in this chunk
    uint64_t in_chunk = 0;
    if (counts) {
        for (int i = tid; i < CHUNK / 4; i += TPB) reinterpret_cast<uint4 *>(s_count)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < CHUNK / 32; i += TPB) s_any[i] = 0;
        if (a.ancestors && lane < min(all, (int32_t)a.rows - first)) {
            const int32_t v = a.tokens[first + lane];
            if (v >= c0 && v < c1) mine = v - c0;
        }
        in_chunk = __ballot(mine >= 0);
        __syncthreads();
        if (tid < 64 && mine >= 0) atomicOr(&s_any[mine >> 5], 1u << (mine & 31));
    }
    if (a.history) {
        const int32_t len = (int32_t)max((int64_t)0, min((int64_t)a.history_lens[req], a.history_stride));
        const int32_t since = a.counted_from ? a.counted_from[req] : 0;
        const int32_t *past = a.history + req * a.history_stride;
        // M entries from i on.  A frequent token's atomics run one after another: none where
        // nothing changes.
        auto count = [&](int32_t i, const auto &v, auto m) {
            constexpr int M = decltype(m)::value;
            uint32_t held[M], word[M];
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int32_t k = v[j] >= c0 && v[j] < c1 ? v[j] - c0 : 0;
                held[j] = __hip_atomic_load(&s_count[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                word[j] = __hip_atomic_load(&s_any[k >> 5], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (v[j] < c0 || v[j] >= c1) continue;
                const int32_t k = v[j] - c0;
                const uint32_t bit = 1u << (k & 31);
                if ((word[j] & bit) == 0) atomicOr(&s_any[k >> 5], bit);
                if (i + j >= since) atomicAdd(&s_count[k], 1u);
                else if ((held[j] & SEEN) == 0) atomicOr(&s_count[k], SEEN);
            }
        };
        const int32_t whole = len & ~3;
#pragma unroll 2
        for (int32_t i = 4 * tid; i < whole; i += 4 * TPB)
            count(i, reinterpret_cast<const Loose<int32_t, 4> *>(past + i)->v, std::integral_constant<int, 4>{});
        if (tid < len - whole) count(whole + tid, &past[whole + tid], std::integral_constant<int, 1>{});
    }
    if (counts) __syncthreads();
    const float rep = a.repetition ? a.repetition[req] : 1.0f, freq = a.frequency ? a.frequency[req] : 0.0f,
                pres = a.presence ? a.presence[req] : 0.0f;
    const uint32_t any = counts ? s_any[at >> 5] >> (at & 31) & ((1u << N) - 1u) : 0u;
    Loose<float, N> bias = {};
    if (a.bias) {
        const float *src = a.bias + req * a.bias_stride + v0;
        if (v0 + N <= c1) {
            bias = *reinterpret_cast<const Loose<float, N> *>(src);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (v0 + j < c1) bias.v[j] = src[j];
        }
    }

    int slot = 0;  // of the row among those looked up
    for (int32_t i = (int32_t)part; i < n; i += pl.row_groups) {
        const int32_t row = first + i;
        const uint32_t lo = __builtin_amdgcn_readlane(path_lo, slot), hi = __builtin_amdgcn_readlane(path_hi, slot);
        const uint64_t path = ((uint64_t)hi << 32 | lo) & in_chunk;
        const bool adds = tid < 64 && mine >= 0 && (path >> lane & 1) != 0;
        if (path != 0) {
            __syncthreads();  // waves may still be at a row before it, which has no barrier of its own
            if (adds) atomicAdd(&s_count[mine], 1u);
            __syncthreads();
        }
        float x[N];
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = (float)z.v[j];
        if (any != 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t c = s_count[at + j];
                if (c == 0) continue;
                x[j] = x[j] > 0.0f ? x[j] / rep : x[j] * rep;
                if ((c & ~SEEN) != 0) x[j] -= freq * (float)(c & ~SEEN) + pres;
            }
        }
        Loose<T, N> out;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (a.bias) x[j] += bias.v[j];
            out.v[j] = (T)((bits >> j & 1) != 0 ? x[j] : -INFINITY);
        }
        if (i + pl.row_groups < n) {
            if (++slot == 64) {
                look_up(i + pl.row_groups);
                slot = 0;
            }
            fetch(row + pl.row_groups, slot);
        }
        T *dst = (T *)a.out + row * a.out_stride + v0;
        if (v0 + N <= c1) {
            *reinterpret_cast<Loose<T, N> *>(dst) = out;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (v0 + j < c1) dst[j] = out.v[j];
        }
        if (path != 0) {
            __syncthreads();
            if (adds) atomicSub(&s_count[mine], 1u);
            __syncthreads();
        }
    }
}

}  // namespace

void logits_constrain(const sili_logits_constrain_args &a, hipStream_t st) {
    constexpr int64_t MOST = (int64_t(1) << 31) - 1, STEP = 8192;  // what a thread's next token, entry or row may lie past the last one
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "logits_constrain: unknown dtype");
    require(a.rows >= 0 && a.rows <= MOST - STEP, "logits_constrain: rows out of range");
    require(a.vocab >= 0 && a.vocab <= MOST - STEP, "logits_constrain: vocab out of range");
    require(a.requests >= 0 && a.requests <= MOST, "logits_constrain: requests out of range");
    require(!a.history || (a.history_stride >= 0 && a.history_stride <= MOST - STEP), "logits_constrain: history_stride out of range");
    require(!a.history || a.history_lens, "logits_constrain: history without history_lens");
    require(!a.ancestors == !a.tokens, "logits_constrain: tokens and ancestors go together");
    require(!a.bias || a.bias_stride == 0 || a.bias_stride >= a.vocab, "logits_constrain: bias_stride is below vocab");
    require(!a.allow || (a.n_allow >= 0 && a.allow_stride >= (a.vocab + 31) / 32), "logits_constrain: allow_stride is below vocab / 32");
    if (a.rows == 0 || a.vocab == 0 || a.requests == 0) return;
    require(a.logits && a.out, "logits_constrain: NULL buffer");
    require(a.out != a.logits || a.out_stride == a.logits_stride, "logits_constrain: in place with other strides");
    require(apart(a.rows, a.vocab, a.out_stride), "logits_constrain: rows of out overlap");
    const int64_t es = dtype_size(a.dtype), words = (a.vocab + 31) / 32;
    const Rows out = rows_of(a.out, a.rows, a.vocab, a.out_stride, es);
    const Rows read[] = {a.out == a.logits ? Rows{} : rows_of(a.logits, a.rows, a.vocab, a.logits_stride, es),
                         row(a.q_start, a.requests + 1, 4),
                         rows_of(a.history, a.requests, a.history_stride, a.history_stride, 4),
                         row(a.history_lens, a.requests, 4),
                         row(a.counted_from, a.requests, 4),
                         row(a.tokens, a.rows, 4),
                         row(a.ancestors, a.rows, 8),
                         row(a.repetition, a.requests, 4),
                         row(a.presence, a.requests, 4),
                         row(a.frequency, a.requests, 4),
                         rows_of(a.bias, a.bias_stride == 0 ? 1 : a.requests, a.vocab, a.bias_stride, 4),
                         rows_of(a.allow, a.n_allow, words, a.allow_stride, 4),
                         row(a.allow_row, a.rows, 4)};
    for (const Rows &r : read) require(!meet(out, r), "logits_constrain: out overlaps an input");
    LogitsPlan p;
    // Chunks of 8192 tokens, whose 1024 threads scan a history in few loads (64 requests
    // of 8 rows of 131071 and histories of 8192: 97 us, with chunks of 4096 and 256
    // threads 105); of 1024 where those would leave CUs without a block (one row of
    // 131071: 7.2 us, with 8192 8.4).
    const bool large = a.requests * ((a.vocab + 8191) / 8192) >= 256;
    const int64_t chunk = large ? 8192 : 1024;
    p.chunks = (int32_t)((a.vocab + chunk - 1) / chunk);
    // rows of a request share its counts; few requests: their rows go to several blocks
    const int64_t each = (a.rows + a.requests - 1) / a.requests, blocks = a.requests * p.chunks;
    p.row_groups = a.q_start ? (int32_t)std::clamp<int64_t>(1024 / blocks, 1, each) : 1;
    require(blocks * p.row_groups < (int64_t(1) << 32) / 1024, "logits_constrain: too many requests");
    const dim3 grid((unsigned)(blocks * p.row_groups));
    with_dtype(a.dtype, [&](auto z) {
        using T = decltype(z);
        if (large) launch(k_logits_constrain<T, 1024, 8>, grid, dim3(1024), 0, st, a, p);
        else launch(k_logits_constrain<T, 512, 2>, grid, dim3(512), 0, st, a, p);
    });
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
