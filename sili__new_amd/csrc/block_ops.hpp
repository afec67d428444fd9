// block_ops.hpp -- the operators between the layers (request slots, rotary
// positions, block norms, the 4-bit cache): launchers, element types, checks.
#pragma once

#include "../../include/sili_hip.h"
#include "common.hpp"

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

// Raises SILI_ERR_INVALID with `what` unless ok.
inline void require(bool ok, const char *what) {
    if (!ok) throw_error(SILI_ERR_INVALID, what);
}
inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

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
