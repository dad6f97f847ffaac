// Device helpers of the streaming operators (ec_norm.hip, ec_logprob.hip, ec_adamw.hip): element types, vectors of 16 bytes
// at any element's alignment, and sums over the lanes of a wave.
#pragma once
#include "ec_common.h"

namespace ecs {

using bf16 = __bf16;
using f16 = _Float16;

// N elements of T at T's own alignment: gfx950 takes global loads and stores of 16 bytes at any address, so rows of odd
// widths and views need no path of their own
template <typename T, int N>
struct vec_of {
    typedef T raw __attribute__((ext_vector_type(N)));
    typedef raw type __attribute__((aligned(sizeof(T))));
    typedef float fraw __attribute__((ext_vector_type(N)));
};

template <typename T, int N>
using raw_t = typename vec_of<T, N>::raw;

// NT: with the streaming hint, for what is read or written once (a read of 1 GB runs at 7.0 TB/s with it, 6.25 without; a copy
// at 6.4 against 6.2)
template <bool NT, typename T, int N>
__device__ __forceinline__ raw_t<T, N> load_raw(const T* p) {
    typedef typename vec_of<T, N>::type any;
    if (NT) return __builtin_nontemporal_load(reinterpret_cast<const any*>(p));
    return *reinterpret_cast<const any*>(p);
}
template <bool NT, typename T, int N>
__device__ __forceinline__ void store_raw(T* p, raw_t<T, N> v) {
    typedef typename vec_of<T, N>::type any;
    if (NT) __builtin_nontemporal_store(v, reinterpret_cast<any*>(p));
    else *reinterpret_cast<any*>(p) = v;
}
// the first n of N (n may be anything; n <= 0: nothing is touched), the others 0
template <bool NT, typename T, int N>
__device__ __forceinline__ raw_t<T, N> load_raw_upto(const T* p, int64_t n) {
    raw_t<T, N> v = {};
    if (n >= N) {
        v = load_raw<NT, T, N>(p);
    } else if (n > 0) {  // (all loads at once, the ones behind the last at its place: a branch each would be a wait each)
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = p[j < n ? j : (int)n - 1];
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = j < n ? v[j] : (T)0.0f;
    }
    return v;
}
template <typename T, int N>
__device__ __forceinline__ void widen(raw_t<T, N> v, float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; j++) f[j] = (float)v[j];
}

template <typename T, int N, bool NT = false>
__device__ __forceinline__ void load_n(const T* p, float (&f)[N]) {
    widen<T, N>(load_raw<NT, T, N>(p), f);
}
template <typename T, int N, bool NT = false>
__device__ __forceinline__ void store_n(T* p, const float (&f)[N]) {
    raw_t<T, N> v;
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = (T)f[j];
    store_raw<NT, T, N>(p, v);
}

// the same for the first n of N
template <typename T, int N, bool NT = false>
__device__ __forceinline__ void load_upto(const T* p, int64_t n, float fill, float (&f)[N]) {
    widen<T, N>(load_raw_upto<NT, T, N>(p, n), f);
    if (n < N) {
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = j < n ? f[j] : fill;
    }
}
template <typename T, int N, bool NT = false>
__device__ __forceinline__ void store_upto(T* p, int64_t n, const float (&f)[N]) {
    if (n >= N) {
        store_n<T, N, NT>(p, f);
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < n) p[j] = (T)f[j];
    }
}

// x of the lane that a DPP control word names (within a row of 16 lanes)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;

// op over groups of W lanes (W = 1, 2, 4 .. 64, a group starts at a multiple of W); every lane gets the result, and every
// lane of the wave has to take part
template <int W, typename Op>
__device__ __forceinline__ uint32_t lanes_u32(uint32_t x, Op op) {
    if (W >= 2) x = op(x, dpp<DPP_XOR1>(x));
    if (W >= 4) x = op(x, dpp<DPP_XOR2>(x));
    if (W >= 8) x = op(x, dpp<DPP_HALF_MIRROR>(x));   // the quads hold one value each: the mirrored lane is in the other quad
    if (W >= 16) x = op(x, dpp<DPP_MIRROR>(x));       // likewise for the halves of a row
    if (W >= 32) {                                    // rows 0 <-> 1, 2 <-> 3
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = op(r[0], r[1]);
    }
    if (W >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = op(r[0], r[1]);
    }
    return x;
}
__device__ __forceinline__ uint32_t fbits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float bitsf(uint32_t x) { return __builtin_bit_cast(float, x); }

template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
    return bitsf(lanes_u32<W>(fbits(x), [](uint32_t a, uint32_t b) { return fbits(bitsf(a) + bitsf(b)); }));
}
template <int W>
__device__ __forceinline__ float lanes_max(float x) {
    return bitsf(lanes_u32<W>(fbits(x), [](uint32_t a, uint32_t b) { return fbits(fmaxf(bitsf(a), bitsf(b))); }));
}
template <int W>
__device__ __forceinline__ uint32_t lanes_umax(uint32_t x) {
    return lanes_u32<W>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int dtype_size(int d) { return d == EC_F32 ? 4 : 2; }
inline bool dtype_ok(int d) { return d == EC_F32 || d == EC_BF16 || d == EC_F16; }

}  // namespace ecs
