// logits.hip -- penalties for repeated tokens, biases and masks on logits.
//
// A block holds a chunk of the vocabulary of one request: it counts the
// request's history there in LDS (low 31 bits: how often past counted_from; top
// bit: before it), and then goes over the request's rows, adding each row's own
// path to the counts and taking it off again.  Bound by the bytes of the rows,
// in short calls by the launch and the scan of the history.
#include "block_ops.hpp"

#include <algorithm>

namespace sili {

namespace {

constexpr int LOGITS_TPB = 256, LOGITS_CHUNK = 4096;
constexpr uint32_t SEEN = 0x80000000u;

struct LogitsPlan {
    int32_t chunks, row_groups;  // blocks of a request
};

template <typename T>
__global__ __launch_bounds__(LOGITS_TPB) void k_logits_constrain(sili_logits_constrain_args a, LogitsPlan pl) {
    __shared__ uint32_t s_count[LOGITS_CHUNK];
    const int tid = threadIdx.x;
    const uint32_t block = blockIdx.x / (uint32_t)pl.chunks, chunk = blockIdx.x - block * (uint32_t)pl.chunks;
    const uint32_t req = block / (uint32_t)pl.row_groups, part = block - req * (uint32_t)pl.row_groups;
    const int32_t c0 = (int32_t)chunk * LOGITS_CHUNK, c1 = (int32_t)min((int64_t)c0 + LOGITS_CHUNK, a.vocab);

    int32_t first = (int32_t)req, all = 1;
    if (a.q_start) {
        const int32_t from = a.q_start[req], upto = a.q_start[req + 1];
        first = max(from, 0);
        all = from < 0 || upto < from ? 0 : upto - from;
    }
    const int32_t n = min(all, (int32_t)a.rows - first);
    if ((int32_t)part >= n) return;

    const bool counts = a.history != nullptr || a.ancestors != nullptr;
    if (counts) {
        for (int i = tid; i < LOGITS_CHUNK; i += LOGITS_TPB) s_count[i] = 0;
        __syncthreads();
    }
    if (a.history) {
        const int32_t len = (int32_t)max((int64_t)0, min((int64_t)a.history_lens[req], a.history_stride));
        const int32_t since = a.counted_from ? a.counted_from[req] : 0;
        const int32_t *past = a.history + req * a.history_stride;
        for (int32_t i = tid; i < len; i += LOGITS_TPB) {
            const int32_t v = past[i];
            if (v < c0 || v >= c1) continue;
            if (i < since) atomicOr(&s_count[v - c0], SEEN);
            else atomicAdd(&s_count[v - c0], 1u);
        }
        __syncthreads();
    }
    const float rep = a.repetition ? a.repetition[req] : 1.0f, freq = a.frequency ? a.frequency[req] : 0.0f,
                pres = a.presence ? a.presence[req] : 0.0f;
    const float *bias = a.bias ? a.bias + req * a.bias_stride : nullptr;

    for (int32_t i = (int32_t)part; i < n; i += pl.row_groups) {
        const int32_t row = first + i;
        int32_t mine = -1;  // a token of the row's path, in this chunk
        if (a.ancestors) {
            if (tid < min(all, min(SILI_TREE_MOST, (int32_t)a.rows - first)) && (a.ancestors[row] >> tid & 1) != 0) {
                const int32_t v = a.tokens[first + tid];
                if (v >= c0 && v < c1) mine = v - c0;
            }
            if (mine >= 0) atomicAdd(&s_count[mine], 1u);
            __syncthreads();
        }
        const int64_t m = !a.allow ? -1 : a.allow_row ? a.allow_row[row] : row;
        const uint32_t *allow = m >= 0 && m < a.n_allow ? a.allow + m * a.allow_stride : nullptr;
        const T *src = (const T *)a.logits + row * a.logits_stride;
        T *dst = (T *)a.out + row * a.out_stride;
        for (int32_t v = c0 + tid; v < c1; v += LOGITS_TPB) {
            float z = (float)src[v];
            const uint32_t c = counts ? s_count[v - c0] : 0u;
            if (c != 0) {
                z = z > 0.0f ? z / rep : z * rep;
                if ((c & ~SEEN) != 0) z -= freq * (float)(c & ~SEEN) + pres;
            }
            if (bias) z += bias[v];
            if (allow && (allow[v >> 5] >> (v & 31) & 1) == 0) z = -INFINITY;
            dst[v] = (T)z;
        }
        if (a.ancestors) {
            __syncthreads();
            if (mine >= 0) atomicSub(&s_count[mine], 1u);
            __syncthreads();
        }
    }
}

}  // namespace

void logits_constrain(const sili_logits_constrain_args &a, hipStream_t st) {
    constexpr int64_t MOST = (int64_t(1) << 31) - 1;
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "logits_constrain: unknown dtype");
    require(a.rows >= 0 && a.rows <= MOST, "logits_constrain: rows out of range");
    require(a.vocab >= 0 && a.vocab <= MOST - LOGITS_CHUNK, "logits_constrain: vocab out of range");
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
    p.chunks = (int32_t)((a.vocab + LOGITS_CHUNK - 1) / LOGITS_CHUNK);
    // rows of a request share its counts; few requests: their rows go to several blocks
    const int64_t each = (a.rows + a.requests - 1) / a.requests, blocks = a.requests * p.chunks;
    p.row_groups = a.q_start ? (int32_t)std::clamp<int64_t>(1024 / blocks, 1, each) : 1;
    require(blocks * p.row_groups < (int64_t(1) << 32) / LOGITS_TPB, "logits_constrain: too many requests");
    const dim3 grid((unsigned)(blocks * p.row_groups));
    with_dtype(a.dtype, [&](auto z) { launch(k_logits_constrain<decltype(z)>, grid, dim3(LOGITS_TPB), 0, st, a, p); });
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
