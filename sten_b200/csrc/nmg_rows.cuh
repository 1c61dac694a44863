// Elements of rows as they are loaded and stored together: whole 16-byte vectors, or one element where an address or a width does not
// allow more.  Shared by the operators that work on rows of hidden states.
#pragma once

#include "nmg_vocab.cuh"

namespace nmg {
#ifdef __CUDACC__
// V elements as they were loaded: unpacked later, so that many are under way in few registers
template <typename T, int V> struct Raw {
    static_assert(V == 1 || V % VEC<T> == 0, "one element or whole vectors");
    static constexpr int N = V == 1 ? 1 : V / VEC<T>;
    std::conditional_t<V == 1, T, uint4> w[N];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (V == 1) w[i] = *p;
            else w[i] = reinterpret_cast<const uint4 *>(p)[i];
        }
    }
    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (V == 1) w[i] = DT<T>::from_f32(v);
            else {
                float f[VEC<T>];
#pragma unroll
                for (int j = 0; j < VEC<T>; j++) f[j] = v;
                w[i] = pack<T>(f);
            }
        }
    }
    __device__ __forceinline__ void unpacked(float *f) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (V == 1) f[i] = DT<T>::to_f32(w[i]);
            else unpack<T>(w[i], f + i * VEC<T>);
        }
    }
};
template <typename T, int V> __device__ __forceinline__ void load_access(const T *p, float *f) {
    Raw<T, V> r;
    r.load(p);
    r.unpacked(f);
}
template <typename T, int V> __device__ __forceinline__ void store_access(T *p, const float *f) {
    if constexpr (V == 1) {
        *p = DT<T>::from_f32(f[0]);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += VEC<T>) *reinterpret_cast<uint4 *>(p + i) = pack<T>(f + i);
    }
}
template <typename T> __device__ __forceinline__ float rounded(float v) { return DT<T>::to_f32(DT<T>::from_f32(v)); }
#endif

// Whether rows `ld` elements apart from p on begin at 16-byte boundaries (p may be NULL).
inline bool whole_vectors(const void *p, int64_t ld, int dtype) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (int64_t)dtype_size(dtype) % 16 == 0; }
inline int check_elements(const void *p, int dtype, const char *what) {
    if (!p) NMG_FAIL(NMG_ERR_INVALID, "%s must be non-NULL", what);
    if (reinterpret_cast<uintptr_t>(p) % dtype_size(dtype)) NMG_FAIL(NMG_ERR_INVALID, "%s must be aligned to its elements", what);
    return NMG_OK;
}
inline int check_dtype(int dtype) {
    if (dtype != NMG_F32 && dtype != NMG_F16 && dtype != NMG_BF16) NMG_FAIL(NMG_ERR_INVALID, "dtype must be NMG_F32, NMG_F16 or NMG_BF16, got %d", dtype);
    return NMG_OK;
}

}  // namespace nmg
