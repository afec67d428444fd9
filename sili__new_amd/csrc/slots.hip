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

// The call's arguments and the division by page_size.
struct Step {
    sili_request_slots_args a;
    int32_t shift;  // page_size = 2^shift, or -1
};
__device__ __forceinline__ uint32_t page_of(const Step &s, uint32_t pos) {
    return s.shift >= 0 ? pos >> s.shift : pos / (uint32_t)s.a.page_size;
}

struct Req {
    int32_t cached, fresh;  // tokens held, tokens new
    int32_t have, take;     // pages held, pages taken
    uint32_t flags;
};

__device__ __forceinline__ Req request(const Step &s, int32_t c, int32_t n) {
    Req q;
    q.flags = (c < 0 || n < 0) ? SILI_SLOTS_BAD_LENGTH : 0u;
    q.cached = max(c, 0);
    q.fresh = max(n, 0);
    if (q.fresh > INT32_MAX - q.cached) {
        q.fresh = INT32_MAX - q.cached;
        q.flags |= SILI_SLOTS_BAD_LENGTH;
    }
    const uint32_t p = (uint32_t)s.a.page_size - 1u;
    q.have = (int32_t)page_of(s, (uint32_t)q.cached + p);
    const int32_t all = (int32_t)page_of(s, (uint32_t)q.cached + (uint32_t)q.fresh + p);
    q.take = all - q.have;
    if (q.fresh > 0 && all > s.a.table_width) q.flags |= SILI_SLOTS_TABLE_FULL;
    return q;
}

// Whether every slot of a page is representable.
__device__ __forceinline__ bool good_page(const sili_request_slots_args &a, int32_t page) {
    return page >= 0 && ((int64_t)page + 1) * a.page_size <= (int64_t)INT32_MAX + 1;
}
__device__ __forceinline__ int32_t slot_of(const sili_request_slots_args &a, int32_t page, uint32_t offset) {
    return good_page(a, page) ? page * (int32_t)a.page_size + (int32_t)offset : -1;
}

// The page that request r's first new token shares with its cached ones: whether
// there is one, and the table's entry (any other where there is none).
__device__ __forceinline__ bool shares_page(const Step &s, const Req &q) {
    const uint32_t at = page_of(s, (uint32_t)q.cached);
    return q.fresh > 0 && (int32_t)at < q.have && at < s.a.table_width;
}
__device__ __forceinline__ int32_t shared_page(const Step &s, const Req &q, int64_t r) {
    return s.a.block_table[r * s.a.table_width + min((int64_t)page_of(s, (uint32_t)q.cached), s.a.table_width - 1)];
}

// Inclusive sum over the wave of values up to 2^34: 16 low bits and the rest
// scanned by themselves, in 32 bits.
__device__ __forceinline__ int64_t wave_scan64(int64_t x) {
    const uint32_t lo = wave_incl_scan((uint32_t)x & 0xFFFFu), hi = wave_incl_scan((uint32_t)(x >> 16));
    return ((int64_t)hi << 16) + lo;
}

// Exclusive sums of (x, y) over the block; the block's totals in tx, ty.
template <unsigned TPB>
__device__ __forceinline__ void block_scan(int64_t &x, int64_t &y, int64_t &tx, int64_t &ty, int64_t (&part)[2][TPB / 64]) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const int64_t x0 = x, y0 = y;
    x = wave_scan64(x);
    y = wave_scan64(y);
    if (lane == 63u) {
        part[0][wave] = x;
        part[1][wave] = y;
    }
    __syncthreads();
    tx = ty = 0;
    int64_t bx = 0, by = 0;
#pragma unroll
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
// the requests, the pages and the tokens, all but the last, which checks (alone it
// does both; a sharing block that checks too took 15.5 us at 4096 requests).  Latency bounds it: the lengths, the
// sums, a search in LDS and a page are one chain (64 requests 4.1 us, of which a
// launch is 3.7; 4096 with 69,000 tokens 12.6).
template <int PER>
__global__ __launch_bounds__(FEW_TPB) void k_slots_few(Step s) {
    extern __shared__ int32_t s_req[];  // first token, first page taken, cached [R each]
    __shared__ int64_t s_part[2][FEW_TPB / 64];
    __shared__ uint32_t s_flags;
    const sili_request_slots_args &a = s.a;
    const int R = (int)a.requests;
    int32_t *tok = s_req, *pag = s_req + R, *old = s_req + 2 * R;
    const int r0 = (int)threadIdx.x * PER;
    const bool checks = blockIdx.x + 1 == gridDim.x;
    const uint32_t sharing = gridDim.x == 1 ? 1u : gridDim.x - 1u;
    const int mine0 = (int)((uint32_t)R * blockIdx.x / sharing), mine1 = (int)((uint32_t)R * (blockIdx.x + 1) / sharing);
    if (threadIdx.x == 0) s_flags = 0;
    int64_t nt = 0, np = 0, T, P;
    uint32_t flags = 0;
    int32_t c[PER], n[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool in = r0 + k < R;
        c[k] = in ? a.cached_lens[r0 + k] : 0;
        n[k] = in ? a.new_lens[r0 + k] : 0;
    }
    int32_t fresh[PER], take[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const Req q = request(s, c[k], n[k]);
        nt += fresh[k] = q.fresh;
        np += take[k] = q.take;
        flags |= q.flags;
        if (r0 + k < R) {
            old[r0 + k] = q.cached;
        }
    }
    if (checks && a.table_width > 0 && R > 0) {
        int32_t page[PER];  // all asked for before the first is looked at
#pragma unroll
        for (int k = 0; k < PER; ++k) page[k] = shared_page(s, request(s, c[k], n[k]), min(r0 + k, R - 1));
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (r0 + k < R && shares_page(s, request(s, c[k], n[k])) && !good_page(a, page[k])) flags |= SILI_SLOTS_BAD_PAGE;
    }
    block_scan<FEW_TPB>(nt, np, T, P, s_part);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (r0 + k < R) {
            tok[r0 + k] = (int32_t)min(nt, (int64_t)INT32_MAX);
            pag[r0 + k] = (int32_t)min(np, (int64_t)INT32_MAX);
            if (r0 + k >= mine0 && r0 + k < mine1) {
                a.q_start[r0 + k] = tok[r0 + k];
                a.kv_lens[r0 + k] = old[r0 + k] + fresh[k];
            }
        }
        nt += fresh[k];
        np += take[k];
    }
    __syncthreads();
    if (checks) {
        const int64_t n_taken = min(P, a.n_free);
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < n_taken; i += FEW_TPB)
            if (!good_page(a, a.free_pages[i])) flags |= SILI_SLOTS_BAD_PAGE;
        if (P > a.n_free) flags |= SILI_SLOTS_NO_PAGE;
        if (T > a.max_tokens) flags |= SILI_SLOTS_TOKENS_FULL;
        if (flags) atomicOr(&s_flags, flags);
        __syncthreads();
        if (threadIdx.x == 0) {
            a.status[0] = (int32_t)min(n_taken, (int64_t)INT32_MAX);
            a.status[1] = (int32_t)s_flags;
        }
        if (gridDim.x > 1) return;
    }
    const int64_t first = (int64_t)blockIdx.x * FEW_TPB + threadIdx.x, step = (int64_t)sharing * FEW_TPB;
    if (first == 0) a.q_start[R] = (int32_t)min(T, (int64_t)INT32_MAX);
    const uint32_t mask = (uint32_t)a.page_size - 1u;
    for (int64_t t = first; t < a.max_tokens; t += step) {
        int32_t pos = 0, slot = -1;
        if (t < T) {
            const int32_t r = (int32_t)owner(tok, R, t), held = old[r];
            pos = held + (int32_t)(t - tok[r]);
            const uint32_t at = page_of(s, (uint32_t)pos);
            const int32_t have = (int32_t)page_of(s, (uint32_t)held + mask);
            int32_t page = -1;
            if ((int64_t)at < a.table_width) {
                const int64_t i = (int64_t)pag[r] + ((int32_t)at - have);
                if ((int32_t)at < have) page = a.block_table[r * a.table_width + at];
                else if (i < a.n_free) page = a.free_pages[i];
            }
            slot = slot_of(a, page, (uint32_t)pos - at * (uint32_t)a.page_size);
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
    for (int64_t i = first; i < P && i < INT32_MAX; i += step) {
        const int64_t r = owner(pag, R, i);
        const int64_t at = (int64_t)page_of(s, (uint32_t)old[r] + mask) + (i - pag[r]);
        if (at < a.table_width) {
            a.block_table[r * a.table_width + at] = i < a.n_free ? a.free_pages[i] : -1;
        } else {
            // on to the next request's pages: a length past the table may ask for 2^31
            const int64_t left = (r + 1 < R ? (int64_t)pag[r + 1] : P) - i;
            i += (left - 1) / step * step;
        }
    }
    // pages whose number passes 31 bits: there are none
    if (P > INT32_MAX) {
        for (int r = mine0 + (int)threadIdx.x; r < mine1; r += FEW_TPB) {
            const Req q = request(s, a.cached_lens[r], a.new_lens[r]);
            const int64_t upto = min((int64_t)q.have + q.take, a.table_width);
            for (int64_t at = (int64_t)q.have + (INT32_MAX - pag[r]); at < upto; ++at) a.block_table[r * a.table_width + at] = -1;
        }
    }
}

// More requests: one block walks them in order and writes their rows, then a
// second launch takes the tokens, which find their request in q_start and
// their page in the table.
__global__ __launch_bounds__(MANY_TPB) void k_slots_rows(Step s) {
    const sili_request_slots_args &a = s.a;
    __shared__ int64_t s_part[2][MANY_TPB / 64];
    __shared__ uint32_t s_flags;
    if (threadIdx.x == 0) s_flags = 0;
    int64_t baseT = 0, baseP = 0;
    uint32_t flags = 0;
    for (int64_t c = 0; c < a.requests; c += MANY_TPB) {
        const int64_t r = c + threadIdx.x;
        Req q{};
        if (r < a.requests) q = request(s, a.cached_lens[r], a.new_lens[r]);
        int64_t nt = q.fresh, np = q.take, T, P;
        block_scan<MANY_TPB>(nt, np, T, P, s_part);
        if (r < a.requests) {
            flags |= q.flags;
            if (shares_page(s, q) && !good_page(a, shared_page(s, q, r))) flags |= SILI_SLOTS_BAD_PAGE;
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

__global__ __launch_bounds__(256) void k_slots_tokens(Step s) {
    const sili_request_slots_args &a = s.a;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.max_tokens) return;
    int32_t pos = 0, slot = -1;
    if (t < (int64_t)a.q_start[a.requests]) {
        const int64_t r = owner(a.q_start, a.requests, t);
        pos = max(a.cached_lens[r], 0) + (int32_t)(t - a.q_start[r]);
        const uint32_t at = page_of(s, (uint32_t)pos);
        if ((int64_t)at < a.table_width)
            slot = slot_of(a, a.block_table[r * a.table_width + at], (uint32_t)pos - at * (uint32_t)a.page_size);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

// Blocks read lengths, tables and pages while others write their results, so no
// output may lie on an input or on another output.
void check_apart(const sili_request_slots_args &a) {
    struct Range {
        uintptr_t begin, end;
    };
    auto range = [](const int32_t *p, int64_t rows, int64_t width = 1) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        const auto bytes = (unsigned __int128)rows * (unsigned __int128)width * sizeof(int32_t);
        return Range{at, at + (uintptr_t)std::min<unsigned __int128>(bytes, UINTPTR_MAX - at)};
    };
    auto meet = [](const Range &x, const Range &y) { return std::max(x.begin, y.begin) < std::min(x.end, y.end); };
    const Range written[] = {range(a.q_start, a.requests + 1), range(a.kv_lens, a.requests), range(a.positions, a.max_tokens),
                             range(a.slots, a.max_tokens), range(a.status, 2), range(a.block_table, a.requests, a.table_width)};
    const Range read[] = {range(a.cached_lens, a.requests), range(a.new_lens, a.requests), range(a.free_pages, a.n_free)};
    for (const Range &w : written) {
        for (const Range &r : read) require(!meet(w, r), "request_slots: an output overlaps an input");
        for (const Range &o : written) require(&o == &w || !meet(w, o), "request_slots: outputs overlap");
    }
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
    check_apart(a);
    Step s{a, -1};
    if ((a.page_size & (a.page_size - 1)) == 0) s.shift = __builtin_ctzll((unsigned long long)a.page_size);
    if (a.requests <= FEW) {
        // a token a thread until every CU has a block, and one to check
        int64_t blocks = std::clamp<int64_t>((a.max_tokens + FEW_TPB - 1) / FEW_TPB, 1, 255);
        if (blocks > 1) ++blocks;
        const uint32_t lds = (uint32_t)(12 * std::max<int64_t>(a.requests, 1));
        if (a.requests <= (int)FEW_TPB) launch(k_slots_few<1>, dim3((unsigned)blocks), dim3(FEW_TPB), lds, st, s);
        else launch(k_slots_few<FEW / (int)FEW_TPB>, dim3((unsigned)blocks), dim3(FEW_TPB), lds, st, s);
    } else {
        launch(k_slots_rows, dim3(1), dim3(MANY_TPB), 0, st, s);
        if (a.max_tokens > 0) launch(k_slots_tokens, dim3((unsigned)((a.max_tokens + 255) / 256)), dim3(256), 0, st, s);
    }
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
