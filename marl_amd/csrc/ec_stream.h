// Device helpers of the streaming operators (ec_norm.hip, ec_logprob.hip, ec_adamw.hip): element types, vectors of 16 bytes
// at any element's alignment, and sums over the lanes of a wave.
#pragma once
#include "ec_common.h"

namespace ecs {

// A launch takes fewer than 2^32 threads along x: blocks from the 2^22nd on stand along y, and a few may be too many
inline dim3 grid_of(int64_t blocks) {
    const int64_t most = 1 << 22;
    return blocks <= most ? dim3((unsigned)blocks) : dim3((unsigned)most, (unsigned)((blocks + most - 1) / most));
}
__device__ __forceinline__ uint32_t block_index() { return blockIdx.y << 22 | blockIdx.x; }

using bf16 = __bf16;
using f16 = _Float16;

// N elements of T at T's own alignment: gfx950 takes global loads and stores of 16 bytes at any address, so rows of odd
// widths and views need no path of their own
template <typename T, int N>
struct vec_of {
    typedef T raw __attribute__((ext_vector_type(N)));
    typedef raw type __attribute__((aligned(sizeof(T))));
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
// The first `bytes` < 16 of a vector, the others 0: in pieces of 8, 4, 2 and 1 bytes, which are all under way together (an
// element at a time, each in a branch of its own, would be a wait each, and an address each)
typedef uint64_t u64_any __attribute__((aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));
struct Words {
    uint64_t lo, hi;
};
__device__ __forceinline__ Words load_bytes(const char* p, int bytes) {
    uint64_t r8 = 0;
    uint32_t r4 = 0, r2 = 0, r1 = 0;
    if (bytes & 8) r8 = *(const u64_any*)p;
    if (bytes & 4) r4 = *(const u32_any*)(p + (bytes & 8));
    if (bytes & 2) r2 = *(const u16_any*)(p + (bytes & 12));
    if (bytes & 1) r1 = *(const uint8_t*)(p + (bytes & 14));
    const uint64_t low = (uint64_t)(r2 | ((bytes & 2) ? r1 << 16 : r1));  // the last 2 + 1 bytes
    const uint64_t rest = (bytes & 4) ? low << 32 | r4 : low;             // the last 4 + 2 + 1
    return (bytes & 8) ? Words{r8, rest} : Words{rest, 0};
}
__device__ __forceinline__ void store_bytes(char* p, int bytes, Words w) {
    if (bytes & 8) *(u64_any*)p = w.lo;
    const uint64_t rest = (bytes & 8) ? w.hi : w.lo;
    if (bytes & 4) *(u32_any*)(p + (bytes & 8)) = (uint32_t)rest;
    const uint32_t low = (bytes & 4) ? (uint32_t)(rest >> 32) : (uint32_t)rest;
    if (bytes & 2) *(u16_any*)(p + (bytes & 12)) = (uint16_t)low;
    if (bytes & 1) *(uint8_t*)(p + (bytes & 14)) = (uint8_t)((bytes & 2) ? low >> 16 : low);
}

// the first n of N (n may be anything; n <= 0: nothing is touched), the others 0
template <bool NT, typename T, int N>
__device__ __forceinline__ raw_t<T, N> load_raw_upto(const T* p, int64_t n) {
    static_assert(N * sizeof(T) <= 16, "one vector");
    raw_t<T, N> v = {};
    if (n >= N) {
        v = load_raw<NT, T, N>(p);
    } else if (n > 0) {
        const Words w = load_bytes((const char*)p, (int)n * (int)sizeof(T));
        __builtin_memcpy(&v, &w, N * sizeof(T));
    }
    return v;
}
template <bool NT, typename T, int N>
__device__ __forceinline__ void store_raw_upto(T* p, int64_t n, raw_t<T, N> v) {
    static_assert(N * sizeof(T) <= 16, "one vector");
    if (n >= N) {
        store_raw<NT, T, N>(p, v);
    } else if (n > 0) {
        Words w{0, 0};
        __builtin_memcpy(&w, &v, N * sizeof(T));
        store_bytes((char*)p, (int)n * (int)sizeof(T), w);
    }
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
template <typename T, int N>
__device__ __forceinline__ raw_t<T, N> narrow(const float (&f)[N]) {
    raw_t<T, N> v;
#pragma unroll
    for (int j = 0; j < N; j++) v[j] = (T)f[j];
    return v;
}
// the same for the first n of N, which may be several vectors of 16 bytes
template <typename T, int N, bool NT = false>
__device__ __forceinline__ void load_upto(const T* p, int64_t n, float fill, float (&f)[N]) {
    constexpr int M = N * sizeof(T) <= 16 ? N : 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < N; q += M) {
        const raw_t<T, M> v = load_raw_upto<NT, T, M>(p + q, n - q);
#pragma unroll
        for (int j = 0; j < M; j++) f[q + j] = q + j < n ? (float)v[j] : fill;
    }
}
template <typename T, int N, bool NT = false>
__device__ __forceinline__ void store_upto(T* p, int64_t n, const float (&f)[N]) {
    constexpr int M = N * sizeof(T) <= 16 ? N : 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < N; q += M) {
        raw_t<T, M> v;
#pragma unroll
        for (int j = 0; j < M; j++) v[j] = (T)f[q + j];
        store_raw_upto<NT, T, M>(p + q, n - q, v);
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
