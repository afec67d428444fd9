// draft.hip -- ancestors and positions of drafted tokens from their parents.
//
// A wave holds a request's tree, a token a lane.  In round k a token takes the
// set of its ancestor 2^k generations up, which by then has 2^k generations, and
// that ancestor's own: six rounds hold any tree of 64 tokens.  The set's size is
// the token's depth.  Bound by its launch and three dependent loads:
// 1.8 us for 8 requests, 2.6 for 1024.
#include "block_ops.hpp"
#include "wave.hpp"

namespace sili {

namespace {

constexpr int DRAFT_WAVES = 4;

__global__ __launch_bounds__(64 * DRAFT_WAVES) void k_draft_tree(sili_draft_tree_args a) {
    const int64_t r = (int64_t)blockIdx.x * DRAFT_WAVES + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (r >= a.requests) return;
    const int32_t from = a.q_start[r], upto = a.q_start[r + 1], cached = max(a.cached_lens[r], 0);
    const int32_t first = max(from, 0);
    const int32_t n = from < 0 || upto < from ? 0 : min(upto - from, min((int32_t)a.max_new, (int32_t)a.tokens - first));
    int32_t up = lane < n ? a.parents[first + lane] : -1;
    if (up < 0 || up >= lane) up = -1;
    const uint64_t mine = uint64_t(1) << lane;
    uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
#pragma unroll
    for (int round = 0; round < 6; ++round) {
        const int at = up < 0 ? lane : up;  // at the top: its own set once more
        lo |= __shfl(lo, at, 64);
        hi |= __shfl(hi, at, 64);
        const int32_t next = __shfl(up, at, 64);
        up = up < 0 ? -1 : next;
    }
    if (lane >= n) return;
    a.ancestors[first + lane] = (uint64_t)hi << 32 | lo;
    a.positions[first + lane] = (int32_t)min((int64_t)cached + __popc(lo) + __popc(hi) - 1, (int64_t)INT32_MAX);
}

}  // namespace

void draft_tree(const sili_draft_tree_args &a, hipStream_t st) {
    require(a.requests >= 0 && a.requests < (int64_t(1) << 26), "draft_tree: requests out of range");
    require(a.tokens >= 0 && a.tokens < (int64_t(1) << 31), "draft_tree: tokens out of range");
    require(a.max_new >= 0 && a.max_new <= SILI_TREE_MOST, "draft_tree: max_new is past SILI_TREE_MOST");
    if (a.requests == 0 || a.tokens == 0 || a.max_new == 0) return;
    require(a.parents && a.q_start && a.cached_lens && a.ancestors && a.positions, "draft_tree: NULL buffer");
    // waves read lengths while others write
    const Span read[] = {span(a.parents, a.tokens * 4), span(a.q_start, (a.requests + 1) * 4), span(a.cached_lens, a.requests * 4)};
    const Span written[] = {span(a.ancestors, a.tokens * 8), span(a.positions, a.tokens * 4)};
    for (const Span &w : written)
        for (const Span &i : read) require(!meet(w, i), "draft_tree: an output overlaps an input");
    require(!meet(written[0], written[1]), "draft_tree: outputs overlap");
    launch(k_draft_tree, dim3((unsigned)((a.requests + DRAFT_WAVES - 1) / DRAFT_WAVES)), dim3(64 * DRAFT_WAVES), 0, st, a);
    SILI_HIP(hipGetLastError());
}

}  // namespace sili
