// logits.hip -- penalties for repeated tokens, biases and masks on logits.
//
// A block holds a chunk of the vocabulary of one request: it counts the
// request's history there in LDS (low 31 bits: how often past counted_from; top
// bit: before it), and then goes over the request's rows, eight tokens a thread
// and load, whose biases stay in registers.  A bit a token says whether it occurs at
// all: most eights ask for no count.  A row whose own path has tokens in the chunk
// adds them to the counts and takes them off again; the others pass without a
// barrier.  Rows begin at any element (vocabularies are odd): loads of 16 bytes at any
// address.  Bound by the bytes of the rows, in short calls by the launch and the scan of
// the history.
#include "block_ops.hpp"

#include <algorithm>

namespace sili {

namespace {

constexpr int LOGITS_TPB = 256, LOGITS_PACK = 8;
constexpr uint32_t SEEN = 0x80000000u;

struct LogitsPlan {
    int32_t chunks, row_groups;  // blocks of a request
};

template <typename T, int CHUNK>
__global__ __launch_bounds__(LOGITS_TPB) void k_logits_constrain(sili_logits_constrain_args a, LogitsPlan pl) {
    constexpr int N = LOGITS_PACK, IT = CHUNK / (N * LOGITS_TPB) > 0 ? CHUNK / (N * LOGITS_TPB) : 1;
    __shared__ __align__(16) uint32_t s_count[CHUNK];
    __shared__ uint32_t s_any[CHUNK / 32];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t block = blockIdx.x / (uint32_t)pl.chunks, chunk = blockIdx.x - block * (uint32_t)pl.chunks;
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

    // this thread's tokens: c0 + N tid + N LOGITS_TPB k
    const int32_t at = N * tid;
    Loose<T, N> z[IT];
    auto fetch = [&](int32_t row) {
        const T *src = (const T *)a.logits + row * a.logits_stride + c0;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int32_t i = at + k * N * LOGITS_TPB;
            if (c0 + i + N <= c1) {
                z[k] = *reinterpret_cast<const Loose<T, N> *>(src + i);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (c0 + i + j < c1) z[k].v[j] = src[i + j];
            }
        }
    };
    fetch(first + (int32_t)part);

    const bool counts = a.history != nullptr || a.ancestors != nullptr;
    int32_t mine = -1;  // token `lane` of the request's path, where it is in this chunk
    uint64_t in_chunk = 0;
    if (counts) {
        for (int i = tid; i < CHUNK / 4; i += LOGITS_TPB) reinterpret_cast<uint4 *>(s_count)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < CHUNK / 32; i += LOGITS_TPB) s_any[i] = 0;
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
        auto count = [&](int32_t i, int32_t v) {
            if (v < c0 || v >= c1) return;
            atomicOr(&s_any[(v - c0) >> 5], 1u << ((v - c0) & 31));
            if (i < since) atomicOr(&s_count[v - c0], SEEN);
            else atomicAdd(&s_count[v - c0], 1u);
        };
        const int32_t whole = len & ~3;
#pragma unroll 4
        for (int32_t i = 4 * tid; i < whole; i += 4 * LOGITS_TPB) {
            const auto v = *reinterpret_cast<const Loose<int32_t, 4> *>(past + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) count(i + j, v.v[j]);
        }
        if (tid < len - whole) count(whole + tid, past[whole + tid]);
    }
    if (counts) __syncthreads();
    const float rep = a.repetition ? a.repetition[req] : 1.0f, freq = a.frequency ? a.frequency[req] : 0.0f,
                pres = a.presence ? a.presence[req] : 0.0f;
    Loose<float, N> bias[IT];
    uint32_t any[IT];
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int32_t i = at + k * N * LOGITS_TPB;
        any[k] = counts && i < CHUNK ? s_any[i >> 5] >> (i & 31) & 0xFFu : 0u;
        if (!a.bias) continue;
        const float *src = a.bias + req * a.bias_stride + c0 + i;
        if (c0 + i + N <= c1) {
            bias[k] = *reinterpret_cast<const Loose<float, N> *>(src);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (c0 + i + j < c1) bias[k].v[j] = src[j];
        }
    }

    for (int32_t i = (int32_t)part; i < n; i += pl.row_groups) {
        const int32_t row = first + i;
        const uint64_t path = a.ancestors ? a.ancestors[row] & in_chunk : 0;  // uniform
        const bool adds = tid < 64 && mine >= 0 && (path >> lane & 1) != 0;
        if (path != 0) {
            if (adds) atomicAdd(&s_count[mine], 1u);
            __syncthreads();
        }
        const int64_t m = !a.allow ? -1 : a.allow_row ? a.allow_row[row] : row;
        const uint32_t *allow = m >= 0 && m < a.n_allow ? a.allow + m * a.allow_stride : nullptr;
        T *dst = (T *)a.out + row * a.out_stride + c0;
        Loose<T, N> out[IT];
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int32_t e = at + k * N * LOGITS_TPB, v = c0 + e;
            if (v >= c1) continue;
            const uint32_t bits = allow ? allow[v >> 5] >> (v & 31) : 0xFFu;
            float x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = (float)z[k].v[j];
            if (any[k] != 0) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint32_t c = s_count[e + j];
                    if (c == 0) continue;
                    x[j] = x[j] > 0.0f ? x[j] / rep : x[j] * rep;
                    if ((c & ~SEEN) != 0) x[j] -= freq * (float)(c & ~SEEN) + pres;
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (a.bias) x[j] += bias[k].v[j];
                out[k].v[j] = (T)((bits >> j & 1) != 0 ? x[j] : -INFINITY);
            }
        }
        if (i + pl.row_groups < n) fetch(row + pl.row_groups);
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int32_t e = at + k * N * LOGITS_TPB, v = c0 + e;
            if (v + N <= c1) {
                *reinterpret_cast<Loose<T, N> *>(dst + e) = out[k];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (v + j < c1) dst[e + j] = out[k].v[j];
            }
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
    constexpr int64_t MOST = (int64_t(1) << 31) - 1;
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "logits_constrain: unknown dtype");
    require(a.rows >= 0 && a.rows <= MOST, "logits_constrain: rows out of range");
    require(a.vocab >= 0 && a.vocab <= MOST - 4096, "logits_constrain: vocab out of range");
    require(a.requests >= 0 && a.requests <= MOST, "logits_constrain: requests out of range");
    require(a.history_stride >= 0, "logits_constrain: negative history_stride");
    require(!a.history || a.history_lens, "logits_constrain: history without history_lens");
    require(!a.ancestors == !a.tokens, "logits_constrain: tokens and ancestors go together");
    require(!a.bias || a.bias_stride == 0 || a.bias_stride >= a.vocab, "logits_constrain: bias_stride is below vocab");
    require(!a.allow || (a.n_allow >= 0 && a.allow_stride >= (a.vocab + 31) / 32), "logits_constrain: allow_stride is below vocab / 32");
    if (a.rows == 0 || a.vocab == 0 || a.requests == 0) return;
    require(a.logits && a.out, "logits_constrain: NULL buffer");
    require(a.out != a.logits || a.out_stride == a.logits_stride, "logits_constrain: in place with other strides");
    LogitsPlan p;
    // small chunks where large ones would leave CUs without a block
    const int64_t chunk = a.requests * ((a.vocab + 4095) / 4096) < 256 ? 1024 : 4096;
    p.chunks = (int32_t)((a.vocab + chunk - 1) / chunk);
    // rows of a request share its counts; few requests: their rows go to several blocks
    const int64_t each = (a.rows + a.requests - 1) / a.requests, blocks = a.requests * p.chunks;
    p.row_groups = a.q_start ? (int32_t)std::clamp<int64_t>(1024 / blocks, 1, each) : 1;
    require(blocks * p.row_groups < (int64_t(1) << 32) / LOGITS_TPB, "logits_constrain: too many requests");
    const dim3 grid((unsigned)(blocks * p.row_groups));
    with_dtype(a.dtype, [&](auto z) {
        launch(chunk == 1024 ? k_logits_constrain<decltype(z), 1024> : k_logits_constrain<decltype(z), 4096>, grid, dim3(LOGITS_TPB), 0, st, a, p);
    });
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
