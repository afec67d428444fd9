// slots.hip -- block tables, slot maps and positions of a step from request
// lengths.
//
// Two exclusive sums over the requests order everything: of the new tokens
// (where a request's tokens begin in the step) and of the pages it takes
// beyond those it holds, ceil((c + n) / P) - ceil(c / P).  Token t belongs to
// the last request that begins at or before t; page i of the step likewise.
#include "block_ops.hpp"
#include "wave.hpp"

#include <algorithm>

namespace sili {

namespace {

constexpr int FEW = 4096;       // requests whose sums a block holds in LDS
constexpr unsigned FEW_TPB = 512;
constexpr unsigned MANY_TPB = 1024;

struct Req {
    int32_t cached, fresh;  // tokens held, tokens new
    int32_t have, take;     // pages held, pages taken
    uint32_t flags;
};

__device__ __forceinline__ Req request(const sili_request_slots_args &a, int64_t r) {
    Req q;
    const int32_t c = a.cached_lens[r], n = a.new_lens[r];
    q.flags = (c < 0 || n < 0) ? SILI_SLOTS_BAD_LENGTH : 0u;
    q.cached = max(c, 0);
    q.fresh = max(n, 0);
    if (q.fresh > INT32_MAX - q.cached) {
        q.fresh = INT32_MAX - q.cached;
        q.flags |= SILI_SLOTS_BAD_LENGTH;
    }
    const uint32_t p = (uint32_t)a.page_size;
    q.have = (int32_t)(((uint32_t)q.cached + p - 1u) / p);
    const int32_t all = (int32_t)(((uint32_t)q.cached + (uint32_t)q.fresh + p - 1u) / p);
    q.take = all - q.have;
    if (q.fresh > 0 && all > a.table_width) q.flags |= SILI_SLOTS_TABLE_FULL;
    return q;
}

// Whether every slot of a page is representable.
__device__ __forceinline__ bool good_page(const sili_request_slots_args &a, int32_t page) {
    return page >= 0 && ((int64_t)page + 1) * a.page_size <= (int64_t)INT32_MAX + 1;
}
__device__ __forceinline__ int32_t slot_of(const sili_request_slots_args &a, int32_t page, uint32_t offset) {
    return good_page(a, page) ? page * (int32_t)a.page_size + (int32_t)offset : -1;
}

// The page that request r's first new token shares with its cached ones, when
// it is no page.
__device__ __forceinline__ uint32_t held_flags(const sili_request_slots_args &a, const Req &q, int64_t r) {
    const uint32_t p = (uint32_t)a.page_size, at = (uint32_t)q.cached / p;
    if (q.fresh == 0 || (uint32_t)q.cached % p == 0u || at >= a.table_width) return 0u;
    return good_page(a, a.block_table[r * a.table_width + at]) ? 0u : (uint32_t)SILI_SLOTS_BAD_PAGE;
}

// Exclusive sums of (x, y) over the block; the block's totals in tx, ty.
template <unsigned TPB>
__device__ __forceinline__ void block_scan(int64_t &x, int64_t &y, int64_t &tx, int64_t &ty, int64_t (&part)[2][TPB / 64]) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const int64_t x0 = x, y0 = y;
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t ux = __shfl_up(x, d, 64), uy = __shfl_up(y, d, 64);
        if ((int)lane >= d) {
            x += ux;
            y += uy;
        }
    }
    if (lane == 63u) {
        part[0][wave] = x;
        part[1][wave] = y;
    }
    __syncthreads();
    tx = ty = 0;
    int64_t bx = 0, by = 0;
    for (uint32_t w = 0; w < TPB / 64; ++w) {
        if (w == wave) {
            bx = tx;
            by = ty;
        }
        tx += part[0][w];
        ty += part[1][w];
    }
    x += bx - x0;
    y += by - y0;
    __syncthreads();  // part is written again by a next call
}

// The last r in [0, n) with start[r] <= t (start ascending, start[0] <= t).
template <typename I>
__device__ __forceinline__ int64_t owner(const int32_t *start, I n, int64_t t) {
    I lo = 0, hi = n;
    while (hi - lo > 1) {
        const I mid = (lo + hi) >> 1;
        if ((int64_t)start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Up to FEW requests: every block sums all the lengths itself (they are a few
// KB, from L2), so that one launch does the whole step; then the blocks share
// the requests, the pages and the tokens.
__global__ __launch_bounds__(FEW_TPB) void k_slots_few(sili_request_slots_args a) {
    extern __shared__ int32_t s_start[];  // tokens [R], pages [R]
    __shared__ int64_t s_part[2][FEW_TPB / 64];
    __shared__ uint32_t s_flags;
    const int R = (int)a.requests;
    int32_t *tok = s_start, *pag = s_start + R;
    const int per = (R + (int)FEW_TPB - 1) / (int)FEW_TPB;
    const int r0 = min((int)threadIdx.x * per, R), r1 = min(r0 + per, R);
    if (threadIdx.x == 0) s_flags = 0;
    int64_t nt = 0, np = 0, T, P;
    uint32_t flags = 0;
    for (int r = r0; r < r1; ++r) {
        const Req q = request(a, r);
        nt += q.fresh;
        np += q.take;
        flags |= q.flags;
        if (blockIdx.x == 0) flags |= held_flags(a, q, r);
    }
    block_scan<FEW_TPB>(nt, np, T, P, s_part);
    for (int r = r0; r < r1; ++r) {
        const Req q = request(a, r);
        tok[r] = (int32_t)min(nt, (int64_t)INT32_MAX);
        pag[r] = (int32_t)min(np, (int64_t)INT32_MAX);
        nt += q.fresh;
        np += q.take;
    }
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * FEW_TPB + threadIdx.x, step = (int64_t)gridDim.x * FEW_TPB;
    for (int64_t r = first; r <= R; r += step) {
        a.q_start[r] = r < R ? tok[r] : (int32_t)min(T, (int64_t)INT32_MAX);
        if (r < R) {
            const Req q = request(a, r);
            a.kv_lens[r] = q.cached + q.fresh;
        }
    }
    for (int64_t i = first; i < P && i < INT32_MAX; i += step) {
        const int64_t r = owner(pag, R, i);
        const int64_t at = request(a, r).have + (i - pag[r]);
        if (at < a.table_width) a.block_table[r * a.table_width + at] = i < a.n_free ? a.free_pages[i] : -1;
    }
    for (int64_t t = first; t < a.max_tokens; t += step) {
        int32_t pos = 0, slot = -1;
        if (t < T) {
            const int64_t r = owner(tok, R, t);
            const Req q = request(a, r);
            pos = q.cached + (int32_t)(t - tok[r]);
            const uint32_t at = (uint32_t)pos / (uint32_t)a.page_size;
            int32_t page = -1;
            if ((int64_t)at >= a.table_width) page = -1;
            else if ((int32_t)at < q.have) page = a.block_table[r * a.table_width + at];
            else {
                const int64_t i = (int64_t)pag[r] + ((int32_t)at - q.have);
                page = i < a.n_free ? a.free_pages[i] : -1;
            }
            slot = slot_of(a, page, (uint32_t)pos - at * (uint32_t)a.page_size);
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    if (blockIdx.x == 0) {
        const int64_t n = min(P, a.n_free);
        for (int64_t i = threadIdx.x; i < n; i += FEW_TPB)
            if (!good_page(a, a.free_pages[i])) flags |= SILI_SLOTS_BAD_PAGE;
        if (P > a.n_free) flags |= SILI_SLOTS_NO_PAGE;
        if (T > a.max_tokens) flags |= SILI_SLOTS_TOKENS_FULL;
        if (flags) atomicOr(&s_flags, flags);
        __syncthreads();
        if (threadIdx.x == 0) {
            a.status[0] = (int32_t)min(n, (int64_t)INT32_MAX);
            a.status[1] = (int32_t)s_flags;
        }
    }
}

// More requests: one block walks them in order and writes their rows, then a
// second launch takes the tokens, which find their request in q_start and
// their page in the table.
__global__ __launch_bounds__(MANY_TPB) void k_slots_rows(sili_request_slots_args a) {
    __shared__ int64_t s_part[2][MANY_TPB / 64];
    __shared__ uint32_t s_flags;
    if (threadIdx.x == 0) s_flags = 0;
    int64_t baseT = 0, baseP = 0;
    uint32_t flags = 0;
    for (int64_t c = 0; c < a.requests; c += MANY_TPB) {
        const int64_t r = c + threadIdx.x;
        Req q{};
        if (r < a.requests) q = request(a, r);
        int64_t nt = q.fresh, np = q.take, T, P;
        block_scan<MANY_TPB>(nt, np, T, P, s_part);
        if (r < a.requests) {
            flags |= q.flags | held_flags(a, q, r);
            a.q_start[r] = (int32_t)min(baseT + nt, (int64_t)INT32_MAX);
            a.kv_lens[r] = q.cached + q.fresh;
            for (int32_t j = 0; j < q.take && (int64_t)q.have + j < a.table_width; ++j) {
                const int64_t i = baseP + np + j;
                const int32_t page = i < a.n_free ? a.free_pages[i] : -1;
                if (i < a.n_free && !good_page(a, page)) flags |= SILI_SLOTS_BAD_PAGE;
                a.block_table[r * a.table_width + q.have + j] = page;
            }
        }
        baseT += T;
        baseP += P;
    }
    if (baseP > a.n_free) flags |= SILI_SLOTS_NO_PAGE;
    if (baseT > a.max_tokens) flags |= SILI_SLOTS_TOKENS_FULL;
    __syncthreads();
    if (flags) atomicOr(&s_flags, flags);
    __syncthreads();
    if (threadIdx.x == 0) {
        a.q_start[a.requests] = (int32_t)min(baseT, (int64_t)INT32_MAX);
        a.status[0] = (int32_t)min(min(baseP, a.n_free), (int64_t)INT32_MAX);
        a.status[1] = (int32_t)s_flags;
    }
}

__global__ __launch_bounds__(256) void k_slots_tokens(sili_request_slots_args a) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    int32_t pos = 0, slot = -1;
    if (t < (int64_t)a.q_start[a.requests]) {
        const int64_t r = owner(a.q_start, a.requests, t);
        pos = max(a.cached_lens[r], 0) + (int32_t)(t - a.q_start[r]);
        const uint32_t at = (uint32_t)pos / (uint32_t)a.page_size;
        if ((int64_t)at < a.table_width)
            slot = slot_of(a, a.block_table[r * a.table_width + at], (uint32_t)pos - at * (uint32_t)a.page_size);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

}  // namespace

void request_slots(const sili_request_slots_args &a, hipStream_t st) {
    constexpr int64_t MOST = (int64_t(1) << 31) - 1;
    require(a.requests >= 0 && a.requests <= MOST, "request_slots: requests out of range");
    require(a.page_size > 0 && a.page_size <= MOST, "request_slots: page_size out of range");
    require(a.n_free >= 0 && a.table_width >= 0, "request_slots: negative size");
    require(a.max_tokens >= 0 && a.max_tokens < MOST, "request_slots: max_tokens out of range");
    require(a.requests == 0 || (a.cached_lens && a.new_lens && a.kv_lens), "request_slots: NULL buffer");
    require(a.requests == 0 || a.table_width == 0 || a.block_table, "request_slots: NULL block_table");
    require(a.n_free == 0 || a.free_pages, "request_slots: NULL free_pages");
    require(a.max_tokens == 0 || (a.positions && a.slots), "request_slots: NULL buffer");
    require(a.q_start && a.status, "request_slots: NULL buffer");
    if (a.requests <= FEW) {
        // four tokens a thread, and no more blocks than the GPU runs at once
        const int64_t blocks = std::clamp<int64_t>((a.max_tokens + 4 * FEW_TPB - 1) / (4 * FEW_TPB), 1, 512);
        launch(k_slots_few, dim3((unsigned)blocks), dim3(FEW_TPB), (uint32_t)(8 * std::max<int64_t>(a.requests, 1)), st, a);
    } else {
        launch(k_slots_rows, dim3(1), dim3(MANY_TPB), 0, st, a);
        if (a.max_tokens > 0) launch(k_slots_tokens, dim3((unsigned)((a.max_tokens + 255) / 256)), dim3(256), 0, st, a);
    }
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
