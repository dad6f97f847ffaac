// ec_adamw.hip -- one AdamW step over many tensors of any size, with moments in fp32 or in 8 bits.
//
//   norm = sqrt(sum g^2) over all tensors;  coef = min(1, max_norm / (norm + 1e-6));  g' = coef g
//   m' = m + (g' - m)(1 - b1);  v' = v b2 + (1 - b2) g' g'
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 8 bits: each 256 consecutive elements of a tensor share two fp32 scales; m is held as q s with q in e4m3 and
// s = max |m| / 448, and v as (q s)^2, the root being what the step divides by and having half the range of v in exponents.
// q is rounded to the nearest e4m3 value (relative step 2^-3 .. 2^-4, the states' only loss: the step itself uses m' and v'
// before they are rounded), except that the q of a v' > 0 is never 0, which would turn a rounding into a step of lr m / eps.
// A NaN stays its own element's; an infinite m' or v' makes its scale infinite, and NaN of the 256 from the next step on.
//
// Bound by HBM: every operand once, 28 bytes an element in fp32 (16 with 8-bit moments), no intermediate.  A launch takes
// up to MAX_TENSORS tensors in its argument block, so nothing is copied to the device; a block finds its tensor by the
// first block of each.  The clip reads g once more: per-block sums in double, added in a fixed order by one block, so that
// the coefficient is the same every run; it stays on the device.
//
// Measured: 151 M fp32 parameters 737 us (5.7 TB/s); 201 M in bf16 with 8-bit moments 314 to 385 us (6.5 to 5.3 TB/s), the
// norm 70 us (5.7) and the coefficient 5.
#include <cmath>

#include "ec_stream.h"

namespace {

using namespace ecs;

constexpr int MAX_TENSORS = 48;          // (the argument block stays under the 4 KB a launch can carry)
constexpr int CHUNK32 = 1024, CHUNK8 = 2048;  // elements a block
constexpr int QBLOCK = 256;              // elements that share a scale
constexpr float QMAX = 448.0f, QMIN = 0.001953125f;

struct Tensor {
    void *p, *m, *v;
    const void* g;
    float *ms, *vs;
    int64_t n;
};
struct Group {
    Tensor t[MAX_TENSORS];
    uint32_t first[MAX_TENSORS + 1];     // first block of each tensor
    int count;
};
struct Hyper {
    float omb1, b2, omb2, eps;           // 1 - beta, rounded once from double
    float step_size, inv_bc2, keep;      // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
    const float* coef;                   // of the gradients, on the device, or NULL: 1
    const float* dyn;                    // {step_size, inv_bc2, keep} on the device, or NULL
};
static_assert(sizeof(Group) + sizeof(Hyper) + 64 <= 4096, "argument block");

// the tensor of a block: each lane compares one entry of `first` (a bisection would be a chain of loads)
__device__ __forceinline__ int tensor_of(const Group& a, uint32_t block) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < a.count && a.first[lane < MAX_TENSORS ? lane : 0] <= block;
    return __popcll(__ballot(at)) - 1;
}

__device__ __forceinline__ float read_hyper(Hyper& h) {
    if (h.dyn) h.step_size = h.dyn[0], h.inv_bc2 = h.dyn[1], h.keep = h.dyn[2];
    return h.coef ? *h.coef : 1.0f;
}

// sqrt to one unit in the last place, for every v >= 0 (the instruction alone takes what is below 2^-126 as 0)
__device__ __forceinline__ float root_of(float v) {
    const bool small = v < 1e-30f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 18446744073709551616.0f : v);
    return small ? r * 2.3283064365386962890625e-10f : r;
}

// m, v -> m', v' and p -> p'; root: sqrt(v').  EXACT, where m' and the root are held in 8 bits afterwards: each operation of
// the formulas rounded once, so that a value next to a border of its 8 bits falls where the plain formulas in fp32 put it.
// The quotient is a product with v_rcp's inverse (one unit in the last place):
// its error is that of the step, far below a rounding of p
template <bool EXACT>
__device__ __forceinline__ void adam(const Hyper& h, float coef, float g, float& p, float& m, float& v, float& root) {
    g *= coef;
    if (EXACT) {  // (built without contraction)
        m = m + (g - m) * h.omb1;
        v = v * h.b2 + h.omb2 * g * g;
    } else {
        m = __builtin_fmaf(g - m, h.omb1, m);
        v = __builtin_fmaf(h.omb2 * g, g, v * h.b2);
    }
    root = EXACT ? sqrtf(v) : root_of(v);
    const float inv = __builtin_amdgcn_rcpf(__builtin_fmaf(root, h.inv_bc2, h.eps));
    p = __builtin_fmaf(-h.step_size * m, inv, p * h.keep);
}

// 32 bits: a block takes CHUNK32 consecutive elements of one tensor, four a thread, all loads ahead of all stores (151 M fp32
// parameters: 737 us, with eight a thread 757; in a loop, with stores between the loads, 816.  bf16: 590 and 619)
template <typename T, bool NT, bool FULL>
__device__ __forceinline__ void adamw32(const Tensor& t, int64_t e, Hyper& h) {
    const int64_t n = FULL ? 4 : t.n - e;
    float p[4], g[4], m[4], v[4], root;
    load_upto<T, 4, NT>((const T*)t.g + e, n, 0.0f, g);
    load_upto<float, 4, NT>((const float*)t.m + e, n, 0.0f, m);
    load_upto<float, 4, NT>((const float*)t.v + e, n, 0.0f, v);
    load_upto<T, 4, NT>((const T*)t.p + e, n, 0.0f, p);
    const float coef = read_hyper(h);
#pragma unroll
    for (int j = 0; j < 4; j++) adam<false>(h, coef, g[j], p[j], m[j], v[j], root);
    store_upto<T, 4, NT>((T*)t.p + e, n, p);
    store_upto<float, 4, NT>((float*)t.m + e, n, m);
    store_upto<float, 4, NT>((float*)t.v + e, n, v);
}

template <typename T, bool NT>
__global__ void __launch_bounds__(256) k_adamw32(Group a, Hyper h) {
    const uint32_t block = block_index();  // (those behind the last tensor's end do nothing)
    const int k = tensor_of(a, block);
    const Tensor t = a.t[k];
    const int64_t b0 = (int64_t)(block - a.first[k]) * CHUNK32, e = b0 + threadIdx.x * 4;
    if (b0 + CHUNK32 <= t.n) adamw32<T, NT, true>(t, e, h);
    else adamw32<T, NT, false>(t, e, h);
}

// 8 bits: a block takes CHUNK8 elements, eight a thread: 16-bit types eight in a row, fp32 two runs of four, half a scale's
// block apart
template <typename T>
struct Take {
    static constexpr int EACH = sizeof(T) == 4 ? 4 : 8, RUNS = 8 / EACH;
};

// N e4m3 values of N bytes at any address (N = 4, 8), the first n of them; the others 0 / untouched
template <int N>
struct Bytes {
    uint32_t w[N / 4];
};
template <int N, bool NT>
__device__ __forceinline__ Bytes<N> load8(const uint8_t* q, int64_t n) {
    const auto v = load_raw_upto<NT, uint8_t, N>(q, n);
    Bytes<N> b;
    __builtin_memcpy(&b, &v, N);
    return b;
}
template <int N, bool NT>
__device__ __forceinline__ void store8(uint8_t* q, int64_t n, const Bytes<N>& b) {
    raw_t<uint8_t, N> v;
    __builtin_memcpy(&v, &b, N);
    store_raw_upto<NT, uint8_t, N>(q, n, v);
}
template <int N>
__device__ __forceinline__ void unpack8(const Bytes<N>& b, float scale, float (&f)[N]) {
#pragma unroll
    for (int k = 0; k < N / 4; k++) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.w[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.w[k], true);
        f[4 * k] = lo[0] * scale, f[4 * k + 1] = lo[1] * scale, f[4 * k + 2] = hi[0] * scale, f[4 * k + 3] = hi[1] * scale;
    }
}
template <int N>
__device__ __forceinline__ Bytes<N> pack8(const float (&f)[N]) {
    Bytes<N> b;
#pragma unroll
    for (int k = 0; k < N / 4; k++) {
        const int q = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k], f[4 * k + 1], 0, false);
        b.w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2], f[4 * k + 3], q, true);
    }
    return b;
}
// the scale of a block with this largest magnitude (NaN left out: it stays its element's), and its inverse; a block of zeros,
// or of what is too small for 1 / s, is held as zeros
__device__ __forceinline__ float scale_of(float most, float& inv) {
    float s = most * (1.0f / QMAX);
    s = s < 1.17549435e-38f ? 0.0f : s;
    inv = s != 0.0f ? 1.0f / s : 0.0f;
    return s;
}

// half a wave takes the 256 elements of a scale, the b-th of the tensor
template <typename T, bool NT, bool FULL>
__device__ __forceinline__ void adamw8(const Tensor& t, int64_t b, Hyper& h) {
    constexpr int E = Take<T>::EACH, R = Take<T>::RUNS;
    const int64_t e0 = b * QBLOCK + (threadIdx.x & 31) * E;
    const bool on = FULL || b * QBLOCK < t.n;
    float p[R][E], g[R][E], m[R][E], v[R][E];
    Bytes<E> qm[R], qv[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int64_t e = e0 + i * (QBLOCK / R), n = FULL ? E : t.n - e;
        load_upto<T, E, NT>((const T*)t.g + e, n, 0.0f, g[i]);
        qm[i] = load8<E, NT>((const uint8_t*)t.m + e, n);
        qv[i] = load8<E, NT>((const uint8_t*)t.v + e, n);
        load_upto<T, E, NT>((const T*)t.p + e, n, 0.0f, p[i]);
    }
    const float ms = on ? t.ms[b] : 0.0f, vs = on ? t.vs[b] : 0.0f;
    const float coef = read_hyper(h);
    float most_m = 0.0f, most_v = 0.0f;
#pragma unroll
    for (int i = 0; i < R; i++) {
        unpack8(qm[i], ms, m[i]);
        unpack8(qv[i], vs, v[i]);
#pragma unroll
        for (int j = 0; j < E; j++) {
            float root;
            v[i][j] *= v[i][j];
            adam<true>(h, coef, g[i][j], p[i][j], m[i][j], v[i][j], root);
            v[i][j] = root;
            most_m = fmaxf(most_m, fabsf(m[i][j]));
            most_v = fmaxf(most_v, root);
        }
    }
    float im, iv;
    const float sm = scale_of(lanes_max<32>(most_m), im), sv = scale_of(lanes_max<32>(most_v), iv);
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int64_t e = e0 + i * (QBLOCK / R), n = FULL ? E : t.n - e;
#pragma unroll
        for (int j = 0; j < E; j++) {
            m[i][j] *= im;
            const float q = v[i][j] * iv, least = q < QMIN ? QMIN : q;  // (a NaN stays one)
            v[i][j] = v[i][j] == 0.0f ? 0.0f : least;
        }
        store_upto<T, E, NT>((T*)t.p + e, n, p[i]);
        store8<E, NT>((uint8_t*)t.m + e, n, pack8(m[i]));
        store8<E, NT>((uint8_t*)t.v + e, n, pack8(v[i]));
    }
    if (on && (threadIdx.x & 31) == 0) t.ms[b] = sm, t.vs[b] = sv;
}

template <typename T, bool NT>
__global__ void __launch_bounds__(256) k_adamw8(Group a, Hyper h) {
    const uint32_t block = block_index();
    const int k = tensor_of(a, block);
    const Tensor t = a.t[k];
    const int64_t c = block - a.first[k], b = c * (CHUNK8 / QBLOCK) + threadIdx.x / 32;
    if ((c + 1) * CHUNK8 <= t.n) adamw8<T, NT, true>(t, b, h);
    else adamw8<T, NT, false>(t, b, h);
}

// partial[blockIdx.x] = sum g^2 over `chunk` elements of a tensor, in double
template <typename T>
__global__ void __launch_bounds__(256) k_sumsq(Group a, int64_t chunk, double* partial) {
    __shared__ double s[4];
    const int k = tensor_of(a, blockIdx.x);
    const T* g = (const T*)a.t[k].g;
    const int64_t e0 = (int64_t)(blockIdx.x - a.first[k]) * chunk;
    const int64_t e1 = e0 + chunk < a.t[k].n ? e0 + chunk : a.t[k].n;
    constexpr int E = 16 / sizeof(T), U = 4;
    double x = 0.0;
    for (int64_t b = e0 + threadIdx.x * E; b < e1; b += 256 * E * U) {
        float f[U][E];
        if (b - threadIdx.x * E + 256 * E * U <= e1) {
#pragma unroll
            for (int u = 0; u < U; u++) load_n(g + b + u * 256 * E, f[u]);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) load_upto(g + b + u * 256 * E, e1 - b - u * 256 * E, 0.0f, f[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < E; j++) x = fma((double)f[u][j], (double)f[u][j], x);
    }
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

// norm and coefficient from the sums of a block's 1024 threads
__device__ __forceinline__ void write_clip(double x, float max_norm, float* norm, float* coef) {
    __shared__ double s[16];
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x) return;
    x = 0.0;
    for (int w = 0; w < 16; w++) x += s[w];
    const float total = (float)sqrt(x), c = max_norm / (total + 1e-6f);
    if (norm) *norm = total;
    *coef = c < 1.0f || c != c ? c : 1.0f;  // (a NaN norm reaches every gradient, as in clip_grad_norm_)
}

// from the partial sums: one block, a fixed order
__global__ void __launch_bounds__(1024) k_clip_coef(const double* partial, int64_t n, float max_norm, float* norm, float* coef) {
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) x += partial[i];
    write_clip(x, max_norm, norm, coef);
}

// from the gradients themselves where one block is enough: a wave takes SMALL_CHUNK elements of a tensor at a time
constexpr int64_t SMALL_TOTAL = 32 << 10, SMALL_CHUNK = 1024;
template <typename T>
__global__ void __launch_bounds__(1024) k_clip_small(Group a, float max_norm, float* norm, float* coef) {
    constexpr int E = 16 / sizeof(T), U = SMALL_CHUNK / 64 / E;
    const int lane = threadIdx.x & 63;
    double x = 0.0;
    for (uint32_t c = threadIdx.x >> 6; c < a.first[a.count]; c += 16) {
        const int k = tensor_of(a, c);
        const int64_t e = (int64_t)(c - a.first[k]) * SMALL_CHUNK + lane * E, n = a.t[k].n - e;
        float f[U][E];
#pragma unroll
        for (int u = 0; u < U; u++) load_upto((const T*)a.t[k].g + e + u * 64 * E, n - u * 64 * E, 0.0f, f[u]);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < E; j++) x = fma((double)f[u][j], (double)f[u][j], x);
    }
    write_clip(x, max_norm, norm, coef);
}

// what follows from a step count (and a learning rate) on the device: dyn = {step_size, inv_bc2, keep}
__global__ void __launch_bounds__(64) k_count_step(float* step, const float* lr_dev, double lr, double b1, double b2, double wd,
                                                   float* dyn) {
    if (threadIdx.x) return;
    const double t = (double)*step + 1.0, rate = lr_dev ? (double)*lr_dev : lr;
    *step = (float)t;
    dyn[0] = (float)(rate / (1.0 - pow(b1, t)));
    dyn[1] = (float)(1.0 / sqrt(1.0 - pow(b2, t)));
    dyn[2] = (float)(1.0 - rate * wd);
}

// elements a block of k_sumsq takes: about 4096 blocks in all
int64_t norm_chunk(int64_t total) { return cdiv(cdiv(total, 4096), 8192) * 8192; }

int64_t norm_parts(int32_t count, const int64_t* numel) {
    int64_t total = 0, parts = 0;
    for (int i = 0; i < count; i++) total += numel[i];
    if (total == 0) return 0;
    const int64_t chunk = norm_chunk(total);
    for (int i = 0; i < count; i++) parts += cdiv(numel[i], chunk);
    return parts;
}

// from this many elements on nothing of one step is left in the caches for the next: the streaming hint then
constexpr int64_t NT_ELEMENTS = 8 << 20;

template <typename T>
void go_step(const Group& a, const Hyper& h, uint32_t blocks, bool q, bool far, hipStream_t st) {
    const dim3 g = grid_of(blocks), b(256);
    if (q) {
        if (far) hipLaunchKernelGGL((k_adamw8<T, true>), g, b, 0, st, a, h);
        else hipLaunchKernelGGL((k_adamw8<T, false>), g, b, 0, st, a, h);
    } else {
        if (far) hipLaunchKernelGGL((k_adamw32<T, true>), g, b, 0, st, a, h);
        else hipLaunchKernelGGL((k_adamw32<T, false>), g, b, 0, st, a, h);
    }
}

const char* bad_tensors(const char* who, int32_t count, const void* const* grads, const int64_t* numel, const int32_t* dtypes,
                        int64_t& total) {
    static thread_local char msg[160];
    total = 0;
    if (count < 0 || (count && (!grads || !numel || !dtypes))) {
        snprintf(msg, sizeof msg, "%s: null argument", who);
        return msg;
    }
    for (int i = 0; i < count; i++) {
        if (!dtype_ok(dtypes[i]) || numel[i] < 0 || numel[i] > ((int64_t)1 << 40) || (numel[i] && !grads[i])) {
            snprintf(msg, sizeof msg, "%s: tensor %d: type %d, %lld elements%s", who, i, dtypes[i], (long long)numel[i],
                     grads[i] ? "" : ", no gradient");
            return msg;
        }
        total += numel[i];
    }
    if (cdiv(total, CHUNK32) + count > INT32_MAX) {
        snprintf(msg, sizeof msg, "%s: %lld elements", who, (long long)total);
        return msg;
    }
    return nullptr;
}

// tensors of one type, up to MAX_TENSORS at a time: fill(i) makes the i-th, go(type, group, blocks) launches
template <typename Fill, typename Go>
void each_group(int32_t count, const int64_t* numel, const int32_t* dtypes, int64_t chunk, Fill fill, Go go) {
    for (int type = EC_F32; type <= EC_F16; type++) {
        Group a;
        a.count = 0;
        uint32_t blocks = 0;
        for (int i = 0; i < count; i++) {
            if (!numel[i] || dtypes[i] != type) continue;
            if (a.count == MAX_TENSORS) {
                a.first[a.count] = blocks;
                go(type, a, blocks);
                a.count = 0;
                blocks = 0;
            }
            a.t[a.count] = fill(i);
            a.first[a.count++] = blocks;
            blocks += (uint32_t)cdiv(numel[i], chunk);
        }
        if (a.count) {
            a.first[a.count] = blocks;
            go(type, a, blocks);
        }
    }
}

}  // namespace

extern "C" int64_t ec_grad_clip_workspace(int32_t count, const int64_t* numel) {
    if (count < 1 || !numel) return 0;
    for (int i = 0; i < count; i++)
        if (numel[i] < 0) return 0;
    return 8 * norm_parts(count, numel);
}

extern "C" int ec_grad_clip_coef(int32_t count, const void* const* grads, const int64_t* numel, const int32_t* dtypes,
                                 double max_norm, float* norm, float* coef, void* work, int64_t work_bytes, void* stream) {
    int64_t total;
    if (const char* m = bad_tensors("ec_grad_clip_coef", count, grads, numel, dtypes, total)) return ec::fail(EC_EINVAL, "%s", m);
    if (!coef || !(max_norm > 0)) return ec::fail(EC_EINVAL, "ec_grad_clip_coef: no output, or a largest norm of %g", max_norm);
    const int64_t need = ec_grad_clip_workspace(count, numel);
    if (work_bytes < need || (need && (!work || (uintptr_t)work % 8)))
        return ec::fail(EC_EINVAL, "ec_grad_clip_coef: workspace of %lld bytes (%lld are needed, at a multiple of 8)",
                        (long long)work_bytes, (long long)need);
    const hipStream_t st = (hipStream_t)stream;
    const auto fill = [&](int i) {
        Tensor t{};
        t.g = grads[i], t.n = numel[i];
        return t;
    };
    // few elements in tensors of one type: one launch, not two (30000 fp32 elements in 10 tensors: 13.4 us a call, by two 15.4,
    // and 4.0 against 4.6 in a graph; 65536: 13.6 and 15.5, but 6.1 against 4.8 in a graph)
    bool small = total > 0 && total <= SMALL_TOTAL && count <= MAX_TENSORS;
    for (int i = 1; i < count; i++) small = small && dtypes[i] == dtypes[0];
    if (small) {
        each_group(count, numel, dtypes, SMALL_CHUNK, fill, [&](int type, const Group& a, uint32_t) {
            const auto k = type == EC_F32 ? k_clip_small<float> : type == EC_BF16 ? k_clip_small<bf16> : k_clip_small<f16>;
            hipLaunchKernelGGL(k, dim3(1), dim3(1024), 0, st, a, (float)max_norm, norm, coef);
        });
        EC_HIP(hipGetLastError());
        return EC_OK;
    }
    const int64_t chunk = total ? norm_chunk(total) : 1;
    double* partial = (double*)work;
    each_group(count, numel, dtypes, chunk, fill,
               [&](int type, const Group& a, uint32_t blocks) {
                   if (type == EC_F32) hipLaunchKernelGGL(k_sumsq<float>, dim3(blocks), dim3(256), 0, st, a, chunk, partial);
                   if (type == EC_BF16) hipLaunchKernelGGL(k_sumsq<bf16>, dim3(blocks), dim3(256), 0, st, a, chunk, partial);
                   if (type == EC_F16) hipLaunchKernelGGL(k_sumsq<f16>, dim3(blocks), dim3(256), 0, st, a, chunk, partial);
                   partial += blocks;
               });
    hipLaunchKernelGGL(k_clip_coef, dim3(1), dim3(1024), 0, st, (const double*)work, (int64_t)(partial - (double*)work),
                       (float)max_norm, norm, coef);
    EC_HIP(hipGetLastError());
    return EC_OK;
}

extern "C" int ec_adamw_step(int32_t count, void* const* params, const void* const* grads, void* const* exp_avg,
                             void* const* exp_avg_sq, float* const* exp_avg_scale, float* const* exp_avg_sq_scale,
                             const int64_t* numel, const int32_t* dtypes, int32_t state_bits, const float* coef, double step_host,
                             float* step_dev, float* dyn, double lr, const float* lr_dev, double beta1, double beta2, double eps,
                             double weight_decay, void* stream) {
    int64_t total;
    if (const char* m = bad_tensors("ec_adamw_step", count, grads, numel, dtypes, total)) return ec::fail(EC_EINVAL, "%s", m);
    const bool q = state_bits == 8;
    if ((state_bits != 32 && !q) || (count && (!params || !exp_avg || !exp_avg_sq || (q && (!exp_avg_scale || !exp_avg_sq_scale)))))
        return ec::fail(EC_EINVAL, "ec_adamw_step: null argument, or states of %d bits (32, or 8 with scales)", state_bits);
    for (int i = 0; i < count; i++)
        if (numel[i] && (!params[i] || !exp_avg[i] || !exp_avg_sq[i] || (q && (!exp_avg_scale[i] || !exp_avg_sq_scale[i]))))
            return ec::fail(EC_EINVAL, "ec_adamw_step: tensor %d: null pointer", i);
    if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || !(weight_decay >= 0))
        return ec::fail(EC_EINVAL, "ec_adamw_step: lr %g, betas %g and %g, eps %g, weight decay %g", lr, beta1, beta2, eps, weight_decay);
    if (step_dev ? !dyn : (!(step_host >= 1.0) || lr_dev))
        return ec::fail(EC_EINVAL, "ec_adamw_step: step count %g (from 1 on, or one on the device, with scratch)", step_host);
    if (total == 0 && !step_dev) return EC_OK;
    const hipStream_t st = (hipStream_t)stream;
    Hyper h{};
    h.omb1 = (float)(1.0 - beta1), h.b2 = (float)beta2, h.omb2 = (float)(1.0 - beta2), h.eps = (float)eps;
    h.coef = coef, h.dyn = step_dev ? dyn : nullptr;
    if (step_dev) {
        hipLaunchKernelGGL(k_count_step, dim3(1), dim3(64), 0, st, step_dev, lr_dev, lr, beta1, beta2, weight_decay, dyn);
    } else {
        h.step_size = (float)(lr / (1.0 - pow(beta1, step_host)));
        h.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, step_host)));
        h.keep = (float)(1.0 - lr * weight_decay);
    }
    const bool far = total >= NT_ELEMENTS;
    each_group(count, numel, dtypes, q ? CHUNK8 : CHUNK32,
               [&](int i) {
                   return Tensor{params[i], exp_avg[i], exp_avg_sq[i], grads[i], q ? exp_avg_scale[i] : nullptr,
                                 q ? exp_avg_sq_scale[i] : nullptr, numel[i]};
               },
               [&](int type, const Group& a, uint32_t blocks) {
                   if (type == EC_F32) go_step<float>(a, h, blocks, q, far, st);
                   if (type == EC_BF16) go_step<bf16>(a, h, blocks, q, far, st);
                   if (type == EC_F16) go_step<f16>(a, h, blocks, q, far, st);
               });
    EC_HIP(hipGetLastError());
    return EC_OK;
}
