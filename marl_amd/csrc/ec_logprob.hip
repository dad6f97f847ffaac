// ec_logprob.hip -- log-probs of given tokens (actions) under softmax(logits), with the entropy and the k likeliest
// alternatives, and the gradient.
//
// Over the entries of a row that are not excluded (avail == 0 or logit == -inf):
//   m = max l,  S1 = sum e^(l - m),  S2 = sum e^(l - m) (l - m)
//   logp = (l_token - m) - log S1,  H = log S1 - S2 / S1,  alternatives: the k largest l (ties: the lowest index)
//   d l_v = g (1[v = token] - p_v) - h p_v (log p_v + H)          g = d / d logp, h = d / d H, p_v = e^(l_v - m) / S1
//
// One pass forward: every thread keeps (m, S1, S2) of what it has seen, against a maximum raised once per batch of loads.
// The alternatives ride along: a wave keeps its k best in its lanes, sorted, and only a batch that holds something larger
// than the k-th is looked at again.  m, S1, S2 and all sums are fp32; log S1 and m stay apart up to the backward pass, so
// that logits of any size lose nothing to the sum of both.
// Bound by HBM for fp32; with bf16 the 10 vector operations an element (one of them the quarter-rate exponential) are about
// as long as its 2 bytes take.
#include <cfloat>
#include <cmath>

#include "ec_stream.h"

namespace {

using namespace ecs;

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f, INF = INFINITY;
constexpr int MAX_TOP = 64;
constexpr int U = 4;  // vectors a thread loads before it looks at them

struct LpArgs {
    const void *logits, *avail;
    const int64_t* tokens;
    int64_t rows, inner, s_outer, s_inner, a_outer, a_inner;  // row r is at (r / inner) * s_outer + (r % inner) * s_inner
    int vocab, top_k, splits, per_split;                      // per_split: columns of one split
    float *lse, *logp, *entropy;                              // lse [rows][2]: m, log S1
    float* top_logp;
    int64_t* top_index;
    char* work;                                               // [rows][splits] of part_bytes(top_k)
    // backward
    const float *entropy_in, *dlogp, *dentropy;
    void* dlogits;
};

struct Stat {
    float m, s1, s2;  // s2 in units of log2
};

__host__ __device__ inline int64_t part_bytes(int k) { return 16 + 8 * (int64_t)k; }

// two sets of entries as one
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
    const float m = fmaxf(a.m, b.m);
    // (m of nothing is -FLT_MAX with s1 = s2 = 0; differences below -200 give factors of 0 all the same and would make
    // 0 * -inf of the s2 terms)
    const float ta = fmaxf((a.m - m) * LOG2E, -200.0f), tb = fmaxf((b.m - m) * LOG2E, -200.0f);
    const float fa = __builtin_amdgcn_exp2f(ta), fb = __builtin_amdgcn_exp2f(tb);
    Stat o;
    o.m = m;
    o.s1 = a.s1 * fa + b.s1 * fb;
    o.s2 = (a.s2 + a.s1 * ta) * fa + (b.s2 + b.s1 * tb) * fb;
    return o;
}

__device__ __forceinline__ Stat wave_join(Stat a) {
    Stat o;
    o.m = lanes_max<64>(a.m);
    const float t = fmaxf((a.m - o.m) * LOG2E, -200.0f), f = __builtin_amdgcn_exp2f(t);
    o.s2 = lanes_sum<64>((a.s2 + a.s1 * t) * f);
    o.s1 = lanes_sum<64>(a.s1 * f);
    return o;
}

// a float's place in the order of floats, with -0 at 0
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = fbits(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return bitsf(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~index; }

__device__ __forceinline__ uint64_t lane_u64(uint64_t x, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// the k best keys of a wave, the i-th in lane i; 0: none
struct TopList {
    uint64_t mine, least;  // least: the k-th (the same in all lanes)
    int k;
    __device__ __forceinline__ void clear(int k_) { mine = least = 0, k = k_; }
    __device__ __forceinline__ float least_value() const { return least ? value_of((uint32_t)(least >> 32)) : -INF; }
    // takes the keys of all lanes; every lane of the wave has to take part
    __device__ __forceinline__ void take(uint64_t key) {
        uint64_t left = __ballot(key > least);
        const int lane = threadIdx.x & 63;
        while (left) {
            const int from = __ffsll((unsigned long long)left) - 1;
            const uint64_t c = lane_u64(key, from);
            const int at = __popcll(__ballot(mine > c));  // (sorted: the lanes with larger keys are the first)
            const uint64_t before = __shfl_up((unsigned long long)mine, 1);
            mine = lane < at ? mine : lane == at ? c : before;
            least = lane_u64(mine, k - 1);
            left &= left - 1;
            left &= __ballot(key > least);
        }
    }
};

template <typename T>
__device__ __forceinline__ const T* row_of(const LpArgs& p, int64_t r) {
    return (const T*)p.logits + (r / p.inner) * p.s_outer + (r % p.inner) * p.s_inner;
}
// MASK 0: none, 1: bytes, 2: int32
template <int MASK>
__device__ __forceinline__ const char* mask_of(const LpArgs& p, int64_t r) {
    return (const char*)p.avail + ((r / p.inner) * p.a_outer + (r % p.inner) * p.a_inner) * (MASK == 1 ? 1 : 4);
}

// the n first of the N logits at l + c, the others and the excluded as -inf
template <typename T, int MASK, int N>
__device__ __forceinline__ void load_logits(const T* l, const char* av, int64_t c, int64_t n, float (&f)[N]) {
    load_upto(l + c, n, -INF, f);
    if (MASK == 0) return;
    if (n >= N) {
        if (MASK == 1) {
            typedef uint8_t bytes __attribute__((ext_vector_type(N)));
            typedef bytes ubytes __attribute__((aligned(1)));
            const bytes b = *reinterpret_cast<const ubytes*>(av + c);
#pragma unroll
            for (int j = 0; j < N; j++) f[j] = b[j] ? f[j] : -INF;
        } else {
            typedef int32_t ints __attribute__((ext_vector_type(4)));
            typedef ints uints __attribute__((aligned(4)));
#pragma unroll
            for (int q = 0; q < N / 4; q++) {
                const ints b = *reinterpret_cast<const uints*>(av + (c + 4 * q) * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) f[4 * q + j] = b[j] ? f[4 * q + j] : -INF;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (j < n && !(MASK == 1 ? av[c + j] != 0 : ((const int32_t*)av)[c + j] != 0)) f[j] = -INF;
    }
}

template <typename T, int MASK>
__device__ __forceinline__ float logit_at(const T* l, const char* av, int64_t c) {
    if (MASK == 1 && av[c] == 0) return -INF;
    if (MASK == 2 && ((const int32_t*)av)[c] == 0) return -INF;
    return (float)l[c];
}

// what a row's statistics say, by the lanes of one wave
template <typename T, int MASK>
__device__ __forceinline__ void finish_row(const LpArgs& p, int64_t r, const Stat& s, const TopList& top) {
    const int lane = threadIdx.x & 63;
    const bool none = s.s1 == 0.0f;  // nothing but excluded entries
    const float ln = none ? 0.0f : __builtin_amdgcn_logf(s.s1) * LN2;
    if (lane == 0) {
        if (p.lse) {
            p.lse[2 * r] = none ? -INF : s.m;
            p.lse[2 * r + 1] = ln;
        }
        if (p.entropy) p.entropy[r] = none ? 0.0f : ln - s.s2 * LN2 / s.s1;
        if (p.logp) {
            const int64_t t = p.tokens[r];
            float v = 0.0f;
            if (t >= p.vocab) {
                v = NAN;
            } else if (t >= 0) {
                const float l = logit_at<T, MASK>(row_of<T>(p, r), MASK ? mask_of<MASK>(p, r) : nullptr, t);
                v = none ? -INF : (l - s.m) - ln;
            }
            p.logp[r] = v;
        }
    }
    if (p.top_k && lane < p.top_k) {
        float v = -INF;
        int64_t at = -1;
        if (!(s.s1 < INF)) {
            v = NAN;  // a NaN or +inf among the entries
        } else if (top.mine) {
            v = (value_of((uint32_t)(top.mine >> 32)) - s.m) - ln;
            at = (int64_t)(uint32_t)~(uint32_t)top.mine;
        }
        p.top_logp[r * p.top_k + lane] = v;
        p.top_index[r * p.top_k + lane] = at;
    }
}

// a block of 256 threads per row, or per split of a row
template <typename T, int MASK, bool TOP>
__global__ void __launch_bounds__(256) k_logp_fwd(LpArgs p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ Stat s_stat[4];
    __shared__ uint64_t s_top[TOP ? 4 : 1][MAX_TOP];
    const int64_t r = blockIdx.x / p.splits;
    const int split = (int)(blockIdx.x % p.splits), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* l = row_of<T>(p, r);
    const char* av = MASK ? mask_of<MASK>(p, r) : nullptr;
    const int64_t c0 = (int64_t)split * p.per_split;
    const int64_t c1 = c0 + p.per_split < p.vocab ? c0 + p.per_split : p.vocab;
    Stat s{-FLT_MAX, 0.0f, 0.0f};
    TopList top;
    top.clear(p.top_k);
    for (int64_t b = c0; b < c1; b += 256 * V * U) {  // (the same rounds for every thread: the lists need whole waves)
        float f[U][V];
        float top_f = -INF;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t c = b + (u * 256 + (int)threadIdx.x) * V;
            load_logits<T, MASK>(l, av, c, c1 - c, f[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < V; j++) top_f = fmaxf(top_f, f[u][j]);
        const float m = fmaxf(s.m, top_f);
        {
            const float t = fmaxf((s.m - m) * LOG2E, -200.0f), g = __builtin_amdgcn_exp2f(t);
            s.s2 = (s.s2 + s.s1 * t) * g;
            s.s1 *= g;
            s.m = m;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float t = (f[u][j] - m) * LOG2E, e = __builtin_amdgcn_exp2f(t);
                s.s1 += e;
                s.s2 = __builtin_fmaf(e, fmaxf(t, -200.0f), s.s2);  // (t = -inf: 0 * -inf)
            }
        if (TOP) {
            // an entry equal to the k-th has the larger index, unless it is of this very batch: only larger ones count
            if (__ballot(top_f > top.least_value())) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const int64_t c = b + (u * 256 + (int)threadIdx.x) * V + j;
                        top.take(f[u][j] > -INF ? key_of(f[u][j], (uint32_t)c) : 0);
                    }
            }
        }
    }
    s = wave_join(s);
    if (lane == 0) s_stat[wave] = s;
    if (TOP && lane < p.top_k) s_top[wave][lane] = top.mine;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 4; w++) {
        s = join(s, s_stat[w]);
        if (TOP) top.take(lane < p.top_k ? s_top[w][lane] : 0);
    }
    if (p.splits == 1) return finish_row<T, MASK>(p, r, s, top);
    char* to = p.work + (r * p.splits + split) * part_bytes(p.top_k);
    if (lane == 0) ((float*)to)[0] = s.m, ((float*)to)[1] = s.s1, ((float*)to)[2] = s.s2;
    if (TOP && lane < p.top_k) ((uint64_t*)(to + 16))[lane] = top.mine;
}

// the splits of a row as one: a wave per row
template <typename T, int MASK>
__global__ void __launch_bounds__(64) k_logp_join(LpArgs p) {
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    const char* from = p.work + r * p.splits * part_bytes(p.top_k);
    Stat s{-FLT_MAX, 0.0f, 0.0f};
    for (int i = lane; i < p.splits; i += 64) {
        const float* f = (const float*)(from + i * part_bytes(p.top_k));
        s = join(s, Stat{f[0], f[1], f[2]});
    }
    s = wave_join(s);
    TopList top;
    top.clear(p.top_k);
    if (p.top_k)
        for (int i = 0; i < p.splits; i++)
            top.take(lane < p.top_k ? ((const uint64_t*)(from + i * part_bytes(p.top_k) + 16))[lane] : 0);
    finish_row<T, MASK>(p, r, s, top);
}

// a block per row and 256 * V * U columns of it
template <typename T, int MASK>
__global__ void __launch_bounds__(256) k_logp_bwd(LpArgs p) {
    constexpr int V = 16 / sizeof(T);
    const int64_t r = blockIdx.x / p.splits;
    const int64_t c0 = (int64_t)(blockIdx.x % p.splits) * p.per_split;
    const T* l = row_of<T>(p, r);
    const char* av = MASK ? mask_of<MASK>(p, r) : nullptr;
    T* out = (T*)p.dlogits + r * p.vocab;
    const int64_t tok = p.tokens[r];
    const float m = p.lse[2 * r], ln = p.lse[2 * r + 1], ent = p.entropy_in[r];
    const float g = !p.dlogp || tok < 0 ? 0.0f : tok >= p.vocab ? NAN : p.dlogp[r];
    const float h = p.dentropy ? p.dentropy[r] : 0.0f;
    const bool none = m == -INF;
    const float l2 = ln * LOG2E, h2 = h * LN2, base = g + h * ent;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t c = c0 + (u * 256 + (int)threadIdx.x) * V;
        if (c >= p.vocab) return;
        float f[V];
        load_logits<T, MASK>(l, av, c, p.vocab - c, f);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float t = (f[j] - m) * LOG2E - l2;  // log2 p
            float d = -__builtin_amdgcn_exp2f(t) * __builtin_fmaf(h2, fmaxf(t, -200.0f), base);
            if (c + j == tok) d += g;
            f[j] = none || f[j] == -INF ? 0.0f : d;
        }
        store_upto(out + c, p.vocab - c, f);
    }
}

const char* bad(const char* who, const LpArgs& a, int dtype, int mask_dtype) {
    static thread_local char msg[200];
    if (!dtype_ok(dtype) || mask_dtype < 0 || mask_dtype > 2)
        snprintf(msg, sizeof msg, "%s: type %d, mask type %d", who, dtype, mask_dtype);
    else if (a.rows < 0 || a.inner < 1 || a.vocab < 1)
        snprintf(msg, sizeof msg, "%s: %lld rows (%lld a group) of %d", who, (long long)a.rows, (long long)a.inner, a.vocab);
    else if (a.s_outer < 0 || a.s_inner < 0 || a.a_outer < 0 || a.a_inner < 0)
        snprintf(msg, sizeof msg, "%s: negative stride", who);
    else if (a.rows && (!a.logits || !a.tokens || !a.avail != !mask_dtype))
        snprintf(msg, sizeof msg, "%s: null argument", who);
    else
        return nullptr;
    return msg;
}

// few rows: a row is split over as many blocks as fill the GPU, at least one batch of loads each
int splits_for(int64_t rows, int64_t vocab, int dtype) {
    const int64_t batch = 256 * U * (dtype == EC_F32 ? 4 : 8);
    const int64_t most = cdiv(vocab, batch), want = cdiv(1024, rows);
    return (int)(want < most ? want : most);
}

#define EC_LP_TYPES(GO)                                   \
    if (dtype == EC_F32) { GO(float) }                    \
    if (dtype == EC_BF16) { GO(bf16) }                    \
    if (dtype == EC_F16) { GO(f16) }

}  // namespace

extern "C" int64_t ec_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t dtype, int32_t top_k) {
    if (rows < 1 || vocab < 1 || vocab > INT32_MAX || !dtype_ok(dtype) || top_k < 0 || top_k > MAX_TOP) return 0;
    const int s = splits_for(rows, vocab, dtype);
    return s > 1 ? rows * s * part_bytes(top_k) : 0;
}

extern "C" int ec_token_logprobs_fwd(const void* logits, int64_t inner, int64_t s_outer, int64_t s_inner, const int64_t* tokens,
                                     const void* avail, int32_t mask_dtype, int64_t a_outer, int64_t a_inner, int32_t dtype,
                                     int64_t rows, int64_t vocab, int32_t top_k, float* logp, float* entropy, float* lse,
                                     float* top_logp, int64_t* top_index, void* work, int64_t work_bytes, void* stream) {
    LpArgs a{};
    a.logits = logits, a.avail = avail, a.tokens = tokens, a.rows = rows, a.inner = inner, a.s_outer = s_outer;
    a.s_inner = s_inner, a.a_outer = a_outer, a.a_inner = a_inner, a.vocab = (int)(vocab > INT32_MAX || vocab < 1 ? 0 : vocab);
    if (const char* m = bad("ec_token_logprobs_fwd", a, dtype, mask_dtype)) return ec::fail(EC_EINVAL, "%s", m);
    if (top_k < 0 || top_k > MAX_TOP || (top_k && rows && (!top_logp || !top_index)))
        return ec::fail(EC_EINVAL, "ec_token_logprobs_fwd: %d alternatives (0 .. %d, with both outputs)", top_k, MAX_TOP);
    if (rows == 0) return EC_OK;
    const int64_t need = ec_token_logprobs_workspace(rows, vocab, dtype, top_k);
    if (work_bytes < need || (need && (!work || (uintptr_t)work % 8)))
        return ec::fail(EC_EINVAL, "ec_token_logprobs_fwd: workspace of %lld bytes (%lld are needed, at a multiple of 8)",
                        (long long)work_bytes, (long long)need);
    a.top_k = top_k, a.logp = logp, a.entropy = entropy, a.lse = lse, a.top_logp = top_logp, a.top_index = top_index;
    a.work = (char*)work;
    a.splits = splits_for(rows, vocab, dtype);
    const int64_t batch = 256 * U * (dtype == EC_F32 ? 4 : 8);
    a.per_split = (int)(cdiv(cdiv(vocab, a.splits), batch) * batch < INT32_MAX ? cdiv(cdiv(vocab, a.splits), batch) * batch : INT32_MAX);
    if (rows * a.splits > INT32_MAX) return ec::fail(EC_EINVAL, "ec_token_logprobs_fwd: %lld rows", (long long)rows);
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(rows * a.splits));
#define EC_GO2(T, M)                                                                               \
    {                                                                                              \
        if (top_k) hipLaunchKernelGGL((k_logp_fwd<T, M, true>), grid, dim3(256), 0, st, a);        \
        else hipLaunchKernelGGL((k_logp_fwd<T, M, false>), grid, dim3(256), 0, st, a);             \
        if (a.splits > 1) hipLaunchKernelGGL((k_logp_join<T, M>), dim3((unsigned)rows), dim3(64), 0, st, a); \
    }
#define EC_GO(T)                          \
    if (mask_dtype == 0) EC_GO2(T, 0)     \
    if (mask_dtype == 1) EC_GO2(T, 1)     \
    if (mask_dtype == 2) EC_GO2(T, 2)
    EC_LP_TYPES(EC_GO)
#undef EC_GO
#undef EC_GO2
    EC_HIP(hipGetLastError());
    return EC_OK;
}

extern "C" int ec_token_logprobs_bwd(const void* logits, int64_t inner, int64_t s_outer, int64_t s_inner, const int64_t* tokens,
                                     const void* avail, int32_t mask_dtype, int64_t a_outer, int64_t a_inner, int32_t dtype,
                                     int64_t rows, int64_t vocab, const float* lse, const float* entropy, const float* dlogp,
                                     const float* dentropy, void* dlogits, void* stream) {
    LpArgs a{};
    a.logits = logits, a.avail = avail, a.tokens = tokens, a.rows = rows, a.inner = inner, a.s_outer = s_outer;
    a.s_inner = s_inner, a.a_outer = a_outer, a.a_inner = a_inner, a.vocab = (int)(vocab > INT32_MAX || vocab < 1 ? 0 : vocab);
    if (const char* m = bad("ec_token_logprobs_bwd", a, dtype, mask_dtype)) return ec::fail(EC_EINVAL, "%s", m);
    if (rows == 0) return EC_OK;
    if (!lse || !entropy || !dlogits) return ec::fail(EC_EINVAL, "ec_token_logprobs_bwd: null argument");
    a.lse = const_cast<float*>(lse), a.entropy_in = entropy, a.dlogp = dlogp, a.dentropy = dentropy, a.dlogits = dlogits;
    a.per_split = 256 * U * (dtype == EC_F32 ? 4 : 8);
    a.splits = (int)cdiv(vocab, a.per_split);
    if (rows * a.splits > INT32_MAX) return ec::fail(EC_EINVAL, "ec_token_logprobs_bwd: %lld rows", (long long)rows);
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)(rows * a.splits));
#define EC_GO(T)                                                                                        \
    if (mask_dtype == 0) hipLaunchKernelGGL((k_logp_bwd<T, 0>), grid, dim3(256), 0, st, a);             \
    if (mask_dtype == 1) hipLaunchKernelGGL((k_logp_bwd<T, 1>), grid, dim3(256), 0, st, a);             \
    if (mask_dtype == 2) hipLaunchKernelGGL((k_logp_bwd<T, 2>), grid, dim3(256), 0, st, a);
    EC_LP_TYPES(EC_GO)
#undef EC_GO
    EC_HIP(hipGetLastError());
    return EC_OK;
}
