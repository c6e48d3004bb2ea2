// Elements of the operators over a model's columns: dense matrices in fp32, fp16 or bf16, read and written eight
// elements at a time, computed in fp32.
#pragma once
#include "common.hpp"

namespace bm {

enum ElemType { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };
static inline size_t elem_size(int type) { return type == ELEM_F32 ? 4 : 2; }

typedef _Float16 f16_t;
typedef __bf16 bf16_t;
template <class T> struct Eight { typedef T type __attribute__((ext_vector_type(8))); };
typedef float float8_t __attribute__((ext_vector_type(8)));

// Eight consecutive elements as they lie in memory. The address has the alignment of one element only: the wide global
// loads and stores of gfx950 take any address, so an odd leading dimension needs no path of its own.
template <class T>
struct Raw8 {
    typename Eight<T>::type v;
    __device__ __forceinline__ static Raw8 load(const T* p) { Raw8 r; __builtin_memcpy(&r.v, p, 8 * sizeof(T)); return r; }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, &v, 8 * sizeof(T)); }
    __device__ __forceinline__ float8_t wide() const { return __builtin_convertvector(v, float8_t); }
    // rounds to nearest even
    __device__ __forceinline__ static Raw8 narrow(float8_t x) { return {__builtin_convertvector(x, typename Eight<T>::type)}; }
};

// Elements i .. i+7 of a column of n; those past its end are neither read nor written and count as `fill`. A short last
// part is read (and written) in pieces of four, two and one.
template <class T>
__device__ __forceinline__ Raw8<T> load_col8(const T* col, int i, int n, T fill = T(0.f)) {
    if (i + 8 <= n) return Raw8<T>::load(col + i);
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = fill;
    const int rem = n - i;
    if (rem <= 0) return r;
    typedef T Two __attribute__((ext_vector_type(2)));
    typedef T Four __attribute__((ext_vector_type(4)));
    const T* p = col + i;
    Two two;
    if (rem & 4) {
        Four four;
        __builtin_memcpy(&four, p, sizeof(four));
        r.v[0] = four[0]; r.v[1] = four[1]; r.v[2] = four[2]; r.v[3] = four[3];
        if (rem & 2) {
            __builtin_memcpy(&two, p + 4, sizeof(two));
            r.v[4] = two[0]; r.v[5] = two[1];
            if (rem & 1) r.v[6] = p[6];
        } else if (rem & 1) {
            r.v[4] = p[4];
        }
    } else if (rem & 2) {
        __builtin_memcpy(&two, p, sizeof(two));
        r.v[0] = two[0]; r.v[1] = two[1];
        if (rem & 1) r.v[2] = p[2];
    } else {
        r.v[0] = p[0];
    }
    return r;
}
// The same in two steps, so that nothing between loads waits for one of them. RAGGED: n is not a multiple of eight; a short
// last part is loaded as the column's last eight elements, and moved to its place by settle_col8 when its turn comes.
template <bool RAGGED, class T>
__device__ __forceinline__ Raw8<T> fetch_col8(const T* col, int i, int n, T fill = T(0.f)) {
    if (RAGGED) return n < 8 ? load_col8(col, i, n, fill) : Raw8<T>::load(col + min(i, n - 8));
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = fill;
    if (i < n) r = Raw8<T>::load(col + i);
    return r;
}
template <bool RAGGED, class T>
__device__ __forceinline__ Raw8<T> settle_col8(Raw8<T> r, int i, int n, T fill = T(0.f)) {
    const int s = i + 8 - n;                    // elements in front of row i
    if (!RAGGED || s <= 0 || n < 8) return r;
    typename Eight<T>::type f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = fill;
    if (s >= 8) return {f};
    if (s & 4) r.v = __builtin_shufflevector(r.v, f, 4, 5, 6, 7, 8, 9, 10, 11);
    if (s & 2) r.v = __builtin_shufflevector(r.v, f, 2, 3, 4, 5, 6, 7, 8, 9);
    if (s & 1) r.v = __builtin_shufflevector(r.v, f, 1, 2, 3, 4, 5, 6, 7, 8);
    return r;
}
template <class T>
__device__ __forceinline__ void store_col8(T* col, int i, int n, float8_t x) {
    Raw8<T> r = Raw8<T>::narrow(x);
    if (i + 8 <= n) { r.store(col + i); return; }
    const int rem = n - i;
    if (rem <= 0) return;
    T* p = col + i;
    if (rem & 4) {
        __builtin_memcpy(p, &r.v, 4 * sizeof(T));
        p += 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[j] = r.v[j + 4];
    }
    if (rem & 2) {
        __builtin_memcpy(p, &r.v, 2 * sizeof(T));
        p += 2;
        r.v[0] = r.v[2];
    }
    if (rem & 1) *p = r.v[0];
}

template <bool RAGGED, class T>
__device__ __forceinline__ void put_col8(T* col, int i, int n, float8_t x) {
    if (RAGGED) store_col8(col, i, n, x);
    else if (i < n) Raw8<T>::narrow(x).store(col + i);
}

// Largest value over aligned groups of N lanes (the steps of group_allsum); a NaN loses against any number.
template <int N>
__device__ __forceinline__ float group_allmax(float x) {
    if (N >= 2) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR1>(x));
    if (N >= 4) x = fmaxf(x, dpp_mov<DPP_QUAD_XOR2>(x));
    if (N >= 8) x = fmaxf(x, dpp_mov<DPP_ROW_HALF_MIRROR>(x));
    if (N >= 16) x = fmaxf(x, dpp_mov<DPP_ROW_MIRROR>(x));
    if (N >= 32) x = fmaxf(x, __shfl_xor(x, 16, 64));
    if (N >= 64) x = fmaxf(x, __shfl_xor(x, 32, 64));
    return x;
}

// Sum / largest value over the TPC consecutive threads that share a column; every one of them gets it. Up to 64 threads
// lie in one wave; more are whole workgroups, which meet in sh (one entry per wave; the caller gives two calls in a
// row different entries, so that one barrier per call is enough).
template <int TPC>
__device__ __forceinline__ float column_allsum(float x, float* sh) {
    if constexpr (TPC <= 64) {
        return group_allsum<TPC>(x);
    } else {
        x = group_allsum<64>(x);
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < TPC / 64; ++w) s += sh[w];
        return s;
    }
}
template <int TPC>
__device__ __forceinline__ float column_allmax(float x, float* sh) {
    if constexpr (TPC <= 64) {
        return group_allmax<TPC>(x);
    } else {
        x = group_allmax<64>(x);
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
        __syncthreads();
        float s = sh[0];
#pragma unroll
        for (int w = 1; w < TPC / 64; ++w) s = fmaxf(s, sh[w]);
        return s;
    }
}

}  // namespace bm
