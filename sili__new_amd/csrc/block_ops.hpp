// block_ops.hpp -- the operators between the layers (request slots, rotary
// positions, block norms, the 4-bit cache) and of a step over drafted tokens
// (trees, 4-bit weights, constraints on logits): launchers, element types, checks.
#pragma once

#include "../../include/sili_hip.h"
#include "common.hpp"
#include "overlap.hpp"

#include <algorithm>

namespace sili {

void request_slots(const sili_request_slots_args &a, hipStream_t st);
void rotary(const sili_rotary_args &a, hipStream_t st);
void rotary_steps(int64_t rot_dim, double base, int scaling, double factor, double original_len, double low,
                  double high, uint64_t *steps, float *scale);
void block_norm_forward(const sili_block_norm_args &a, hipStream_t st);
void block_norm_backward(const sili_block_norm_args &a, const sili_block_norm_grads &g, hipStream_t st);
size_t block_norm_workspace(const sili_block_norm_args &a);
void kv4_append(const sili_kv4_rows_args &a, hipStream_t st);
void kv4_read(const sili_kv4_rows_args &a, hipStream_t st);
void kv4_attend(const sili_kv4_attend_args &a, hipStream_t st);
size_t kv4_attend_workspace(const sili_kv4_attend_args &a);
void draft_tree(const sili_draft_tree_args &a, hipStream_t st);
void kv4_attend_tree(const sili_kv4_attend_args &a, const uint64_t *ancestors, hipStream_t st);
size_t kv4_attend_tree_workspace(const sili_kv4_attend_args &a);
void fp4_pack(const sili_fp4_pack_args &a, hipStream_t st);
void fp4_linear(const sili_fp4_linear_args &a, hipStream_t st);
size_t fp4_linear_workspace(const sili_fp4_linear_args &a);
void logits_constrain(const sili_logits_constrain_args &a, hipStream_t st);

// Raises SILI_ERR_INVALID with `what` unless ok.
inline void require(bool ok, const char *what) {
    if (!ok) throw_error(SILI_ERR_INVALID, what);
}
inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// The bytes a contiguous buffer takes, and whether two have one in common.
struct Span {
    uintptr_t begin, end;
};
inline Span span(const void *p, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return {at, at + std::min<uintptr_t>((uintptr_t)bytes, UINTPTR_MAX - at)};
}
inline bool meet(const Span &x, const Span &y) { return std::max(x.begin, y.begin) < std::min(x.end, y.end); }

// n elements of `bytes` bytes one after another, or `rows` times that.
inline Rows row(const void *p, int64_t n, int64_t bytes) { return {p, 1, (__int128)n * bytes, 0}; }
inline Rows rows_of(const void *p, int64_t rows, int64_t n, int64_t stride, int64_t bytes) {
    return {p, rows, (__int128)n * bytes, (__int128)stride * bytes};
}
// Rows of n elements, `stride` apart, of which none has a byte of another.
inline bool apart(int64_t rows, int64_t n, int64_t stride) { return rows <= 1 || stride >= n || stride <= -n; }

// Element types of activations.  The conversions of __bf16 and _Float16 round
// to nearest even and keep NaN and infinities.
inline int64_t dtype_size(int dtype) { return dtype == SILI_F32 ? 4 : 2; }

template <typename F>
void with_dtype(int dtype, F &&f) {
    switch (dtype) {
        case SILI_F32: f(float{}); break;
        case SILI_BF16: f(__bf16{}); break;
        case SILI_F16: f(_Float16{}); break;
        default: throw_error(SILI_ERR_INVALID, "dtype is none of SILI_F32, SILI_BF16, SILI_F16");
    }
}

// N consecutive elements, moved as one load or store where T* is aligned to
// their size.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
// N elements at any address of an element: one load where the hardware has one
// for the size (it takes any alignment).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void load_pack(const T *p, float (&x)[N]) {
    const Pack<T, N> k = *reinterpret_cast<const Pack<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)k.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, const float (&x)[N]) {
    Pack<T, N> k;
#pragma unroll
    for (int i = 0; i < N; ++i) k.v[i] = (T)x[i];
    *reinterpret_cast<Pack<T, N> *>(p) = k;
}

}  // namespace sili
