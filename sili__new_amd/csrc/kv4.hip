// kv4.hip -- a paged cache of keys and values in 4 bits: rows written and read
// back, and attention over it.
//
// A stored head is scale * code[c], code an E2M1 value; its scale is amax / 6,
// so the largest element takes the largest level.
#include "block_ops.hpp"
#include "wave.hpp"

#include <algorithm>
#include <cmath>

namespace sili {

namespace {

__device__ __forceinline__ float wave_max(float v) {
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// Byte b of a stored head (channels 2b, 2b + 1) in the k and v code arrays;
// head: index of (page, kv head).
__device__ __forceinline__ int64_t k_byte(const sili_kv4_cache &c, int64_t head, int slot, int b) {
    return (head * c.page_size + slot) * (c.head_dim / 2) + b;
}
__device__ __forceinline__ int64_t v_byte(const sili_kv4_cache &c, int64_t head, int slot, int b) {
    return ((head * (c.page_size / 16) + slot / 16) * (c.head_dim / 2) + b) * 16 + slot % 16;
}

constexpr int ROWS_TPB = 256;

// One wave a (token, kv head): k's head, then v's.
template <typename T, bool WRITE>
__global__ __launch_bounds__(ROWS_TPB) void k_kv4_rows(sili_kv4_rows_args a) {
    const int64_t id = (int64_t)blockIdx.x * (ROWS_TPB / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const sili_kv4_cache &c = a.cache;
    if (id >= a.tokens * c.kv_heads) return;
    const int64_t t = id / c.kv_heads, h = id - t * c.kv_heads;
    const int64_t slot = a.slots[t];
    const bool held = slot >= 0 && slot < c.n_pages * c.page_size;
    if (WRITE && !held) return;
    const int64_t page = held ? slot / c.page_size : 0;
    const int at = held ? (int)(slot - page * c.page_size) : 0;
    const int64_t head = page * c.kv_heads + h;
    const int pairs = (int)c.head_dim / 2;
    for (int which = 0; which < 2; ++which) {
        T *row = which ? (T *)a.v + t * a.v_token_stride + h * a.v_head_stride
                       : (T *)a.k + t * a.k_token_stride + h * a.k_head_stride;
        uint8_t *codes = which ? c.v : c.k;
        float *scales = (which ? c.v_scale : c.k_scale) + head * c.page_size + at;
        if (WRITE) {
            float top = 0.0f;
            bool bad = false;
            for (int b = lane; b < pairs; b += 64) {
                const float x = fabsf((float)row[2 * b]), y = fabsf((float)row[2 * b + 1]);
                bad |= !(x < INFINITY) || !(y < INFINITY);
                top = fmaxf(top, fmaxf(x, y));
            }
            top = wave_max(top);
            bad = __any(bad);
            const bool zero = top < 0x1p-120f || bad;
            const float inv = zero ? 0.0f : 6.0f / top;
            for (int b = lane; b < pairs; b += 64) {
                const uint32_t lo = zero ? 0u : fp4_encode((float)row[2 * b] * inv);
                const uint32_t hi = zero ? 0u : fp4_encode((float)row[2 * b + 1] * inv);
                codes[which ? v_byte(c, head, at, b) : k_byte(c, head, at, b)] = (uint8_t)(lo | hi << 4);
            }
            if (lane == 0) *scales = bad ? __builtin_nanf("") : zero ? 0.0f : top / 6.0f;
        } else {
            const float scale = held ? *scales : 0.0f;
            for (int b = lane; b < pairs; b += 64) {
                const uint32_t byte = held ? codes[which ? v_byte(c, head, at, b) : k_byte(c, head, at, b)] : 0u;
                row[2 * b] = (T)(fp4_decode(byte & 15u) * scale);
                row[2 * b + 1] = (T)(fp4_decode(byte >> 4) * scale);
            }
        }
    }
}

// The request of query token t: the last that begins at or before it.
__device__ __forceinline__ int64_t request_of(const int32_t *start, int64_t n, int64_t t) {
    int64_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One wave a (query token, query head).  Per step of 64 keys: a lane takes the
// score of one key; the running maximum and sum are updated; then a lane takes
// a channel pair of the values.
template <typename T>
__global__ __launch_bounds__(64) void k_kv4_attend(sili_kv4_attend_args a) {
    __shared__ float s_q[256], s_p[64];
    __shared__ int64_t s_v[64];
    const sili_kv4_cache &c = a.cache;
    const int lane = threadIdx.x, d = (int)c.head_dim;
    const int64_t t = blockIdx.x, qh = blockIdx.y, h = qh / (a.q_heads / c.kv_heads);
    if (t < a.q_start[0] || t >= a.q_start[a.requests]) return;
    const int64_t r = request_of(a.q_start, a.requests, t);
    const int64_t n_new = a.q_start[r + 1] - a.q_start[r], i = t - a.q_start[r];
    if (i >= a.max_new) return;
    const int64_t kv = a.kv_lens[r], last = kv - n_new + i;
    int64_t end = min(min(kv, a.max_len), a.table_width * c.page_size), begin = 0;
    if (a.causal) {
        end = min(end, last + 1);
        if (a.window > 0) begin = max((int64_t)0, last + 1 - a.window);
    }
    const T *q = (const T *)a.q + t * a.q_token_stride + qh * a.q_head_stride;
    for (int k = lane; k < d; k += 64) s_q[k] = (float)q[k] * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t base = begin; base < end; base += 64) {
        const int64_t j = base + lane;
        float s = -INFINITY, vs = 0.0f;
        int64_t vb = -1;
        if (j < end) {
            const int64_t page = a.block_table[r * a.table_width + j / c.page_size];
            const int at = (int)(j % c.page_size);
            if (page >= 0 && page < c.n_pages) {
                const int64_t head = page * c.kv_heads + h;
                const uint32_t *codes = reinterpret_cast<const uint32_t *>(c.k + k_byte(c, head, at, 0));
                float dot = 0.0f;
                for (int w = 0; w < d / 8; ++w) {
                    const uint32_t x = codes[w];
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot += fp4_decode((x >> (4 * e)) & 15u) * s_q[8 * w + e];
                }
                s = dot * c.k_scale[head * c.page_size + at];
                vs = c.v_scale[head * c.page_size + at];
                vb = v_byte(c, head, at, 0);
            }
        }
        const float m_new = fmaxf(m, wave_max(s));
        // no key seen yet: exp(-inf - -inf) would be NaN
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = __expf(m - ref), p = vb >= 0 ? __expf(s - ref) : 0.0f;
        l = l * keep + wave_sum(p);
        m = m_new;
        s_p[lane] = vb >= 0 ? p * vs : 0.0f;
        s_v[lane] = vb;
        __syncthreads();
        for (int e = 0; e < 4; ++e) o[e] *= keep;
        for (int b = lane, e = 0; b < d / 2; b += 64, e += 2)
            for (int k = 0; k < 64; ++k) {
                if (s_v[k] < 0) continue;
                const uint32_t x = c.v[s_v[k] + 16 * b];
                o[e] += s_p[k] * fp4_decode(x & 15u);
                o[e + 1] += s_p[k] * fp4_decode(x >> 4);
            }
        __syncthreads();
    }
    T *out = (T *)a.out + t * a.out_token_stride + qh * a.out_head_stride;
    for (int b = lane, e = 0; b < d / 2; b += 64, e += 2) {
        out[2 * b] = (T)(l != 0.0f ? o[e] / l : 0.0f);
        out[2 * b + 1] = (T)(l != 0.0f ? o[e + 1] / l : 0.0f);
    }
    if (a.lse && lane == 0) a.lse[t * a.q_heads + qh] = l != 0.0f ? m + __logf(l) : -INFINITY;
}

void check_cache(const sili_kv4_cache &c, const char *what) {
    const std::string w(what);
    auto need = [&](bool ok, const char *m) {
        if (!ok) throw_error(SILI_ERR_INVALID, w + ": " + m);
    };
    need(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "head_dim is none of 64, 128, 256");
    need(c.page_size >= 16 && c.page_size % 16 == 0 && c.page_size <= 65536, "page_size is not a multiple of 16 up to 65536");
    need(c.kv_heads >= 1 && c.kv_heads <= 65535, "kv_heads out of range");
    need(c.n_pages >= 0 && c.n_pages * c.page_size <= (int64_t(1) << 31), "more than 2^31 slots");
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
    const int64_t blocks = (a.tokens * a.cache.kv_heads + ROWS_TPB / 64 - 1) / (ROWS_TPB / 64);
    require(blocks <= INT32_MAX, "kv4 rows: too many rows");
    with_dtype(a.dtype, [&](auto z) {
        launch(k_kv4_rows<decltype(z), WRITE>, dim3((unsigned)blocks), dim3(ROWS_TPB), 0, st, a);
    });
    SILI_HIP(hipGetLastError());
}

void check_attend(const sili_kv4_attend_args &a) {
    check_cache(a.cache, "kv4_attend");
    require(a.dtype == SILI_F32 || a.dtype == SILI_BF16 || a.dtype == SILI_F16, "kv4_attend: unknown dtype");
    require(a.requests >= 0 && a.requests <= 65535, "kv4_attend: requests out of range");
    require(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "kv4_attend: tokens out of range");
    require(a.q_heads >= 1 && a.q_heads % a.cache.kv_heads == 0, "kv4_attend: q_heads is no multiple of kv_heads");
    require(a.q_heads <= 65535, "kv4_attend: too many query heads");
    require(a.table_width >= 0 && a.max_new >= 0 && a.max_len >= 0, "kv4_attend: negative size");
    require(a.max_len < (int64_t(1) << 31) && a.max_new < (int64_t(1) << 31), "kv4_attend: bound out of range");
    require(a.window >= 0 && (a.window == 0 || a.causal), "kv4_attend: a window needs the causal mask");
}

}  // namespace

void kv4_append(const sili_kv4_rows_args &a, hipStream_t st) { rows<true>(a, st, "kv4_append"); }
void kv4_read(const sili_kv4_rows_args &a, hipStream_t st) { rows<false>(a, st, "kv4_read"); }

size_t kv4_attend_workspace(const sili_kv4_attend_args &a) {
    check_attend(a);
    return 0;
}

void kv4_attend(const sili_kv4_attend_args &a, hipStream_t st) {
    check_attend(a);
    if (a.tokens == 0 || a.requests == 0 || a.max_new == 0) return;
    require(a.q && a.out && a.q_start && a.kv_lens, "kv4_attend: NULL buffer");
    require(a.block_table || a.table_width == 0, "kv4_attend: NULL block_table");
    with_dtype(a.dtype, [&](auto z) {
        launch(k_kv4_attend<decltype(z)>, dim3((unsigned)a.tokens, (unsigned)a.q_heads), dim3(64), 0, st, a);
    });
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
