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
// as long as its 2 bytes take.  The gradient reads the logits again: it needs S1 of the whole row first.
//
// Measured, forward and backward: 4.1 M rows of 11 in fp32 under int32 masks 73 and 100 us (6.3 and 6.5 TB/s of 460 and 655
// MB moved); 8192 rows of 65536 in bf16 208 and 365 us (5.2 and 5.9); 1009 rows of 50021 in fp32 under a mask of bytes, with 5
// alternatives, 47 and 71 us (5.4 and 6.4).  4 rows of 131072 in bf16 with 20 alternatives: 8.5 us and 6.6 us to join the
// splits of a row, both chains of waits.  Further from the memory's rate: 600 000 rows of 60 in fp32 50 and 61 us (3.2 and 5.0
// TB/s), a load a lane in flight and then a chain of lane sums; 10000 rows of 5001 in bf16 with 20 alternatives 43 us (2.3), which
// a wave looks for again in each of the three batches of its row.
#include <cfloat>
#include <cmath>

#include "ec_stream.h"

namespace {

using namespace ecs;

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f, INF = INFINITY;
constexpr int MAX_TOP = 64, MAX_SPLITS = 60;  // (a split per lane, and 2 * 60 * 64 keys of LDS, where they are joined)
constexpr int MOST_U = 4;  // vectors a thread loads before it looks at them, at most

struct LpArgs {
    const void *logits, *avail;
    const int64_t* tokens;
    int64_t rows, inner, s_outer, s_inner, a_outer, a_inner;  // row r is at (r / inner) * s_outer + (r % inner) * s_inner
    uint32_t by_inner;                                        // i / inner = umulhi(i, by_inner) for i < 2^16; 0: inner >= 2^15
    int vocab, top_k, splits, per_split;                      // per_split: columns of one split
    float *lse, *logp, *entropy;                              // lse [rows][2]: m, log S1
    float* top_logp;
    int64_t* top_index;
    char* work;                                               // [rows][splits] of part_bytes(top_k)
    bool ahead;                                               // taken_logit
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

// the sets of W lanes as one, in all of them
template <int W>
__device__ __forceinline__ Stat lanes_join(Stat a) {
    Stat o;
    o.m = lanes_max<W>(a.m);
    const float t = fmaxf((a.m - o.m) * LOG2E, -200.0f), f = __builtin_amdgcn_exp2f(t);
    o.s2 = lanes_sum<W>((a.s2 + a.s1 * t) * f);
    o.s1 = lanes_sum<W>(a.s1 * f);
    return o;
}

// a float's place in the order of floats, with -0 at 0
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = fbits(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return bitsf(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
constexpr uint32_t ORDER_LOWEST = 0x00800000u;  // order_of(-FLT_MAX)
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~index; }

__device__ __forceinline__ uint64_t lane_u64(uint64_t x, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// LDS written and read by one wave: in order, once the compiler keeps it so
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr int POOL = 128;  // keys that a wave ranks at once

// The k best keys of a wave, the i-th in lane i; 0: none.  What a batch of loads holds above the k-th joins them in a pool in
// LDS, where every key's place is the number of larger ones (keys are distinct: the index is part of them).  Of the first
// batch only what is no less than the k-th largest of the 64 lanes' maxima can be among the k best: for any but odd data
// little more than k keys.  That bound is found bit by bit, to 18 bits (what is below it is a bound too): a comparison each,
// and a count in the scalar unit.  (Keys inserted one after the other cost 250 cycles each: 10000 rows of 5001 in bf16 with
// 20 alternatives took 185 us.)
struct TopList {
    uint64_t mine;
    float least;  // the k-th's value (the same in all lanes), -inf where there are fewer
    int k, have;
    __device__ __forceinline__ void clear(int k_) { mine = 0, least = -INF, k = k_, have = 0; }
    __device__ __forceinline__ void set_least() {
        const uint64_t last = lane_u64(mine, k - 1);
        least = last ? value_of((uint32_t)(last >> 32)) : -INF;
    }
    // the keys of all lanes, one after the other
    __device__ __forceinline__ void insert(uint64_t key) {
        const int lane = threadIdx.x & 63;
        uint64_t last = lane_u64(mine, k - 1), left = __ballot(key > last);
        while (left) {
            const int from = __ffsll((unsigned long long)left) - 1;
            const uint64_t c = lane_u64(key, from);
            const int at = __popcll(__ballot(mine > c));  // (sorted: the lanes with larger keys are the first)
            const uint64_t before = __shfl_up((unsigned long long)mine, 1);
            mine = lane < at ? mine : lane == at ? c : before;
            last = lane_u64(mine, k - 1);
            left &= left - 1;
            left &= __ballot(key > last);
        }
    }
    // a batch: f[u][j] is column c + u * step + j; top_f: the lane's largest.  Every lane of the wave has to take part
    template <int UU, int N>
    __device__ __forceinline__ void absorb(const float (&f)[UU][N], float top_f, int64_t c, int64_t step, uint64_t* pool) {
        const int lane = threadIdx.x & 63;
        uint32_t bound;
        if (have == 0) {
            const uint32_t o = order_of(top_f);
            bound = 0;
#pragma unroll
            for (int b = 31; b >= 14; b--)
                if (__popcll(__ballot(o >= (bound | (1u << b)))) >= k) bound |= 1u << b;
        } else {
            bound = order_of(least) + 1;  // an entry equal to the k-th has a larger index than it, being of a later batch
        }
        const float from = fmaxf(value_of(bound < ORDER_LOWEST ? ORDER_LOWEST : bound), -FLT_MAX);
        if (lane < have) pool[lane] = mine;
        int n = have;
#pragma unroll
        for (int u = 0; u < UU; u++)
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float x = f[u][j];
                const bool in = x >= from;  // (-inf is below -FLT_MAX)
                const uint64_t who = __ballot(in);
                if (who) {
                    const int at = n + __popcll(who & ((1ull << lane) - 1));
                    if (in && at < POOL) pool[at] = key_of(x, (uint32_t)(c + u * step + j));
                    n += __popcll(who);
                }
            }
        if (n > POOL) {  // (many equal ones)
#pragma unroll
            for (int u = 0; u < UU; u++)
#pragma unroll
                for (int j = 0; j < N; j++) insert(f[u][j] > -INF ? key_of(f[u][j], (uint32_t)(c + u * step + j)) : 0);
            have = __popcll(__ballot(lane < k && mine != 0));
        } else {
            wave_sync();
            const uint64_t a = lane < n ? pool[lane] : 0, b = lane + 64 < n ? pool[lane + 64] : 0;
            int ra = 0, rb = 0;
            for (int i = 0; i < n; i++) ra += pool[i] > a;
            if (n > 64)
                for (int i = 0; i < n; i++) rb += pool[i] > b;
            wave_sync();
            if (a && ra < k) pool[ra] = a;
            if (b && rb < k) pool[rb] = b;
            wave_sync();
            have = n < k ? n : k;
            mine = lane < have ? pool[lane] : 0;
            wave_sync();
        }
        set_least();
    }
};

// (no division where there is nothing to divide by: in 64 bits it costs as much as ten entries)
__device__ __forceinline__ int64_t row_at(int64_t r, int64_t inner, int64_t s_outer, int64_t s_inner) {
    if (inner == 1) return r * s_outer;
    int64_t q;
    if (((r | inner) >> 32) == 0) q = (uint32_t)r / (uint32_t)inner;
    else q = r / inner;
    return q * s_outer + (r - q * inner) * s_inner;
}
template <typename T>
__device__ __forceinline__ const T* row_of(const LpArgs& p, int64_t r) {
    return (const T*)p.logits + row_at(r, p.inner, p.s_outer, p.s_inner);
}
// MASK 0: none, 1: bytes, 2: int32
template <int MASK>
__device__ __forceinline__ const char* mask_of(const LpArgs& p, int64_t r) {
    return (const char*)p.avail + row_at(r, p.inner, p.a_outer, p.a_inner) * (MASK == 1 ? 1 : 4);
}

// U vectors of N logits from l + c on, `step` apart, those from column c1 on and the excluded as -inf.  FULL: all of them lie
// below c1 (the loads then stand together, with no branch between them)
template <typename T, int MASK, bool NT, bool FULL, int UU, int N>
__device__ __forceinline__ void load_logits(const T* l, const char* av, int64_t c, int64_t step, int64_t c1, float (&f)[UU][N]) {
    raw_t<T, N> raw[UU];
    raw_t<uint8_t, N> b[MASK == 1 ? UU : 1];
    raw_t<int32_t, 4> w[MASK == 2 ? UU : 1][N / 4];
#pragma unroll
    for (int u = 0; u < UU; u++) {
        const int64_t at = c + u * step, n = FULL ? N : c1 - at;
        raw[u] = load_raw_upto<NT, T, N>(l + at, n);
        if (MASK == 1) b[MASK == 1 ? u : 0] = load_raw_upto<NT, uint8_t, N>((const uint8_t*)av + at, n);
        if (MASK == 2)
#pragma unroll
            for (int q = 0; q < N / 4; q++)
                w[MASK == 2 ? u : 0][q] = load_raw_upto<NT, int32_t, 4>((const int32_t*)av + at + 4 * q, n - 4 * q);
    }
#pragma unroll
    for (int u = 0; u < UU; u++) {
        widen<T, N>(raw[u], f[u]);
        const int64_t n = FULL ? N : c1 - (c + u * step);
#pragma unroll
        for (int j = 0; j < N; j++) {
            bool on = FULL || j < n;
            if (MASK == 1) on = b[MASK == 1 ? u : 0][j] != 0;  // (behind the last: 0)
            if (MASK == 2) on = w[MASK == 2 ? u : 0][j / 4][j % 4] != 0;
            f[u][j] = on ? f[u][j] : -INF;
        }
    }
}

template <typename T, int MASK>
__device__ __forceinline__ float logit_at(const T* l, const char* av, int64_t c) {
    if (MASK == 1 && av[c] == 0) return -INF;
    if (MASK == 2 && ((const int32_t*)av)[c] == 0) return -INF;
    return (float)l[c];
}

// log p of a row's token, whose logit is l
__device__ __forceinline__ float logp_of(const LpArgs& p, int64_t token, float l, const Stat& s, float ln) {
    if (token < 0) return 0.0f;
    if (token >= p.vocab) return NAN;
    return s.s1 == 0.0f ? -INF : (l - s.m) - ln;
}
__device__ __forceinline__ float log_s1(const Stat& s) { return s.s1 == 0.0f ? 0.0f : __builtin_amdgcn_logf(s.s1) * LN2; }

// a row's lse, entropy and log-prob, by one lane (s1 = 0: nothing but excluded entries)
__device__ __forceinline__ void write_row(const LpArgs& p, int64_t r, const Stat& s, float ln, float logp) {
    const bool none = s.s1 == 0.0f;
    if (p.lse) {
        p.lse[2 * r] = none ? -INF : s.m;
        p.lse[2 * r + 1] = ln;
    }
    if (p.entropy) {
        const float h = ln - s.s2 * LN2 / s.s1;
        p.entropy[r] = none || h < 0.0f ? 0.0f : h;  // (a rounding below 0; a NaN stays one)
    }
    if (p.logp) p.logp[r] = logp;
}
__device__ __forceinline__ void write_top(const LpArgs& p, int64_t r, int i, const Stat& s, float ln, uint64_t key) {
    float v = -INF;
    int64_t at = -1;
    if (!(s.s1 < INF)) {
        v = NAN;  // a NaN or +inf among the entries
    } else if (key) {
        v = (value_of((uint32_t)(key >> 32)) - s.m) - ln;
        at = (int64_t)(uint32_t)~(uint32_t)key;
    }
    p.top_logp[r * p.top_k + i] = v;
    p.top_index[r * p.top_k + i] = at;
}

// The logit of a row's token (one that is none: 0).  The token is loaded ahead of the row, the logit, which waits for it, behind
// the row; but ahead of it too where all blocks run at once and nothing hides that wait (one row of 32000: 17.3 us, behind
// 18.0; 5000 rows of 16000: 107 us, ahead 112)
constexpr int64_t AT_ONCE = 2048;  // blocks of 256 that the GPU holds
template <typename T, int MASK>
__device__ __forceinline__ float taken_logit(const LpArgs& p, int64_t r, int64_t tok) {
    return tok >= 0 && tok < p.vocab ? logit_at<T, MASK>(row_of<T>(p, r), MASK ? mask_of<MASK>(p, r) : nullptr, tok) : 0.0f;
}

// U vectors a thread from column b on into the row's statistics and alternatives (the same rounds for every thread: the lists
// need whole waves).  FULL: all of them below c1
template <typename T, int MASK, bool TOP, int TPR, int U, bool NT, bool FULL>
__device__ __forceinline__ void logp_batch(const T* l, const char* av, int64_t b, int t, int64_t c1, Stat& s, TopList& top,
                                           uint64_t* pool) {
    constexpr int V = 16 / sizeof(T);
    float f[U][V];
    float top_f = -INF;
    load_logits<T, MASK, NT, FULL>(l, av, b + t * V, TPR * V, c1, f);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int j = 0; j < V; j++) top_f = fmaxf(top_f, f[u][j]);
    const float m = fmaxf(s.m, top_f);
    const float d0 = fmaxf((s.m - m) * LOG2E, -200.0f), g = __builtin_amdgcn_exp2f(d0);
    s.s2 = (s.s2 + s.s1 * d0) * g;
    s.s1 *= g;
    s.m = m;
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (!FULL && TPR == 256 && b + u * TPR * V >= c1) break;  // (the same for all: nothing but -inf from here on)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = (f[u][j] - m) * LOG2E, e = __builtin_amdgcn_exp2f(d);
            s.s1 += e;
            s.s2 = __builtin_fmaf(e, fmaxf(d, -200.0f), s.s2);  // (d = -inf: 0 * -inf)
        }
    }
    if (TOP)
        if (__ballot(top_f > top.least)) top.absorb(f, top_f, b + t * V, TPR * V, pool);
}

// TPR threads a row: 16 or 64 (each row once), or a block of 256 per row or split of a row
template <typename T, int MASK, bool TOP, int TPR, int U, bool NT>
__global__ void __launch_bounds__(256) k_logp_fwd(LpArgs p) {
    constexpr int V = 16 / sizeof(T), W = TPR < 64 ? TPR : 64;
    __shared__ Stat s_stat[4];
    __shared__ uint64_t s_pool[TOP ? 4 : 1][TOP ? POOL : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = threadIdx.x % TPR;
    // (every thread makes every round: a group of rows past the last reads the last and writes nothing)
    const uint32_t block = block_index();
    const int64_t r0 = TPR == 256 ? block / (uint32_t)p.splits : (int64_t)block * (256 / TPR) + threadIdx.x / TPR;
    const bool on = r0 < p.rows;
    if (TPR == 256 && !on) return;
    const int64_t r = on ? r0 : p.rows - 1;
    const int split = TPR == 256 ? (int)(block % (uint32_t)p.splits) : 0;
    const T* l = row_of<T>(p, r);
    const char* av = MASK ? mask_of<MASK>(p, r) : nullptr;
    const int64_t c0 = (int64_t)split * p.per_split;
    const int64_t c1 = c0 + p.per_split < p.vocab ? c0 + p.per_split : p.vocab;
    Stat s{-FLT_MAX, 0.0f, 0.0f};
    const int64_t tok = p.tokens[r];
    float taken = 0.0f;
    if (p.ahead && t == 0) taken = taken_logit<T, MASK>(p, r, tok);
    TopList top;
    top.clear(p.top_k);
    int64_t b = c0;
    for (; b + TPR * V * U <= c1; b += TPR * V * U) logp_batch<T, MASK, TOP, TPR, U, NT, true>(l, av, b, t, c1, s, top, s_pool[TOP ? wave : 0]);
    if (b < c1) logp_batch<T, MASK, TOP, TPR, U, NT, false>(l, av, b, t, c1, s, top, s_pool[TOP ? wave : 0]);
    s = lanes_join<W>(s);
    if (TPR < 256) {
        const float ln = log_s1(s);
        if (on && t == 0) {
            if (!p.ahead) taken = taken_logit<T, MASK>(p, r, tok);
            write_row(p, r, s, ln, logp_of(p, tok, taken, s, ln));
        }
        if (TOP && on && t < p.top_k) write_top(p, r, t, s, ln, top.mine);
        return;
    }
    if (lane == 0) s_stat[wave] = s;
    if (TOP && lane < p.top_k) s_pool[TOP ? wave : 0][lane] = top.mine;
    __syncthreads();
    s = s_stat[0];
#pragma unroll
    for (int w = 1; w < 4; w++) s = join(s, s_stat[w]);
    const float ln = log_s1(s);
    char* to = p.splits > 1 ? p.work + (r * p.splits + split) * part_bytes(p.top_k) : nullptr;
    if (threadIdx.x == 0) {
        if (p.splits > 1) {
            ((float*)to)[0] = s.m, ((float*)to)[1] = s.s1, ((float*)to)[2] = s.s2;
        } else {
            if (!p.ahead) taken = taken_logit<T, MASK>(p, r, tok);
            write_row(p, r, s, ln, logp_of(p, tok, taken, s, ln));
        }
    }
    if (TOP) {
        // a key's place among the four waves' lists: its place in its own and the number of larger ones in the others (the
        // places behind the last key, each wave its share of them, take "none")
        int have = 0, at = lane;
        for (int w = 0; w < 4; w++) {
            const uint64_t* o = s_pool[TOP ? w : 0];
            have += __popcll(__ballot(lane < p.top_k && o[lane] != 0));
            if (w != wave)
                for (int i = 0; i < p.top_k; i++) at += o[i] > top.mine;
        }
        if (lane >= p.top_k || !top.mine) at = p.top_k;
        if (wave == 0 && lane >= have && lane < p.top_k) {
            if (to) ((uint64_t*)(to + 16))[lane] = 0;
            else write_top(p, r, lane, s, ln, 0);
        }
        if (at < p.top_k) {
            if (to) ((uint64_t*)(to + 16))[at] = top.mine;
            else write_top(p, r, at, s, ln, top.mine);
        }
    }
}

// the splits of a row as one: a block per row
template <typename T, int MASK>
__global__ void __launch_bounds__(256) k_logp_join(LpArgs p) {
    extern __shared__ uint64_t s_keys[];  // [splits][top_k], then those that may be among the best
    __shared__ int s_n;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x & 63, k = p.top_k, all = p.splits * k;
    const char* from = p.work + r * p.splits * part_bytes(k);
    // (every wave joins the statistics for itself; what is loaded is loaded first: this kernel is a chain of waits)
    Stat s{-FLT_MAX, 0.0f, 0.0f};
    const int64_t tok = p.tokens[r];
    const float taken = threadIdx.x == 255 ? taken_logit<T, MASK>(p, r, tok) : 0.0f;
    if (lane < p.splits) {
        const float* f = (const float*)(from + lane * part_bytes(k));
        s = Stat{f[0], f[1], f[2]};
    }
    uint32_t first = 0, last = 0;  // order of each split's largest and k-th
    if (threadIdx.x < 64 && k && lane < p.splits) {
        const uint64_t* q = (const uint64_t*)(from + lane * part_bytes(k) + 16);
        first = (uint32_t)(q[0] >> 32), last = (uint32_t)(q[k - 1] >> 32);
    }
    for (int i = threadIdx.x; i < all; i += 256) s_keys[i] = ((const uint64_t*)(from + (i / k) * part_bytes(k) + 16))[i % k];
    s = lanes_join<64>(s);
    const float ln = log_s1(s);
    if (threadIdx.x == 255) write_row(p, r, s, ln, logp_of(p, tok, taken, s, ln));
    if (k == 0) return;
    __syncthreads();
    // nothing below the k-th of one split can be among the best, nor below the k-th largest of the splits' largest (TopList)
    if (threadIdx.x < 64) {
        uint32_t heads = 0;
#pragma unroll
        for (int b = 31; b >= 14; b--)
            if (__popcll(__ballot(first >= (heads | (1u << b)))) >= k) heads |= 1u << b;
        last = lanes_umax<64>(last);
        const uint64_t bound = (uint64_t)(heads > last ? heads : last) << 32;
        int n = 0;
        for (int b = 0; b < all; b += 64) {
            const uint64_t o = b + lane < all ? s_keys[b + lane] : 0;
            const bool in = o && o >= bound;
            const uint64_t who = __ballot(in);
            if (in) s_keys[all + n + __popcll(who & ((1ull << lane) - 1))] = o;
            n += __popcll(who);
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const int n = s_n;
    const uint64_t* some = s_keys + all;
    for (int i = threadIdx.x; i < n; i += 256) {
        const uint64_t mine = some[i];
        int at = 0;
        for (int q = 0; q < n; q++) at += some[q] > mine;
        if (at < k) write_top(p, r, at, s, ln, mine);
    }
    for (int i = n + threadIdx.x; i < k; i += 256) write_top(p, r, i, s, ln, 0);
}

// what the gradient of a row's entries needs
struct RowGrad {
    float m, l2, h2, base, g;
    int64_t tok;
    bool none;
};
__device__ __forceinline__ RowGrad row_grad(const LpArgs& p, int64_t r) {
    RowGrad o;
    o.tok = p.tokens[r];
    o.m = p.lse[2 * r];
    o.l2 = p.lse[2 * r + 1] * LOG2E;
    o.none = o.m == -INF;
    o.g = !p.dlogp || o.tok < 0 ? 0.0f : o.tok >= p.vocab ? NAN : p.dlogp[r];
    const float h = p.dentropy ? p.dentropy[r] : 0.0f;
    o.h2 = h * LN2;
    o.base = o.g + h * p.entropy_in[r];
    return o;
}
__device__ __forceinline__ float entry_grad(const RowGrad& w, float l, int64_t c) {
    const float t = (l - w.m) * LOG2E - w.l2;  // log2 p
    float d = -__builtin_amdgcn_exp2f(t) * __builtin_fmaf(w.h2, fmaxf(t, -200.0f), w.base);
    if (c == w.tok) d += w.g;
    return w.none || l == -INF ? 0.0f : d;
}

template <typename T, int MASK, int TPR, int U, bool NT, bool FULL>
__device__ __forceinline__ void grad_batch(const RowGrad& w, const T* l, const char* av, T* out, int64_t b, int t, int64_t c1) {
    constexpr int V = 16 / sizeof(T);
    float f[U][V];
    load_logits<T, MASK, NT, FULL>(l, av, b + t * V, TPR * V, c1, f);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int64_t c = b + (u * TPR + t) * V;
        if (!FULL && TPR == 256 && b + u * TPR * V >= c1) break;  // (the same for all)
#pragma unroll
        for (int j = 0; j < V; j++) f[u][j] = entry_grad(w, f[u][j], c + j);
        store_upto<T, V, NT>(out + c, FULL ? V : c1 - c, f[u]);
    }
}

// TPR threads a row: 16 or 64 for a whole row, or a block of 256 per TPR * V * U columns of a row
template <typename T, int MASK, int TPR, int U, bool NT>
__global__ void __launch_bounds__(256) k_logp_bwd(LpArgs p) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t block = block_index();
    const int64_t r = TPR == 256 ? block / (uint32_t)p.splits : (int64_t)block * (256 / TPR) + threadIdx.x / TPR;
    if (r >= p.rows) return;
    const int64_t c0 = TPR == 256 ? (int64_t)(block % (uint32_t)p.splits) * p.per_split : 0;
    const int64_t c1 = TPR == 256 && c0 + p.per_split < p.vocab ? c0 + p.per_split : p.vocab;
    const T* l = row_of<T>(p, r);
    const char* av = MASK ? mask_of<MASK>(p, r) : nullptr;
    T* out = (T*)p.dlogits + r * p.vocab;
    const RowGrad w = row_grad(p, r);
    const int t = threadIdx.x % TPR;
    int64_t b = c0;
    for (; b + TPR * V * U <= c1; b += TPR * V * U) grad_batch<T, MASK, TPR, U, NT, true>(w, l, av, out, b, t, c1);
    if (b < c1) grad_batch<T, MASK, TPR, U, NT, false>(w, l, av, out, b, t, c1);
}

// ---- few entries a row (the env's action sets): a lane per row ----
// FEW_ROWS rows are staged through LDS as fp32, excluded entries as -inf; packed rows come in and gradients leave 16 bytes a
// lane whatever the row's width.  QUADS: widths that are multiples of 4 lie there at an odd multiple of 4, and lanes walk down
// their rows four entries at a time; other widths at an odd stride, one at a time: different banks for different lanes either
// way.  (128 rows a block: 64 and 256 are 2 to 12 % slower.)  GAPS: rows that are not packed, by a kernel of their own (in one
// kernel with them packed rows take 3 % longer).
constexpr int FEW_ROWS = 128;
// up to this width (600 000 rows of 60 forward and back: bf16 89 us, with 16 lanes a row 140; fp32 139 and 125)
constexpr int FEW_16BIT = 62, FEW_FP32 = 52;

__host__ __device__ inline int few_stride(int vocab) { return vocab % 4 ? vocab | 1 : 4 * (vocab / 4 | 1); }

__device__ __forceinline__ int row_in(int i, int vocab, uint32_t by_vocab) {  // i / vocab
    return vocab == 1 ? i : (int)__umulhi((uint32_t)i, by_vocab);
}

// f(entry, column) for the entries of a row; WRITE: f may change them
template <bool QUADS, bool WRITE, typename F>
__device__ __forceinline__ void each_entry(float* l, int vocab, F f) {
    if (QUADS) {
#pragma unroll 2
        for (int j = 0; j < vocab; j += 4) {
            float4 v = *(float4*)(l + j);
            f(v.x, j), f(v.y, j + 1), f(v.z, j + 2), f(v.w, j + 3);
            if (WRITE) *(float4*)(l + j) = v;
        }
    } else {
#pragma unroll 4
        for (int j = 0; j < vocab; j++) {
            float v = l[j];
            f(v, j);
            if (WRITE) l[j] = v;
        }
    }
}

// where the rows of a tile are, from r0 on
struct Tile {
    int64_t at_l, at_a;  // of the group that r0 is in
    uint32_t rem;        // r0's place in it
    __device__ __forceinline__ Tile(const LpArgs& p, int64_t r0) {
        int64_t q = r0;
        if (p.inner != 1) q = ((r0 | p.inner) >> 32) == 0 ? (uint32_t)r0 / (uint32_t)p.inner : r0 / p.inner;
        at_l = q * p.s_outer, at_a = q * p.a_outer, rem = (uint32_t)(r0 - q * p.inner);
    }
    __device__ __forceinline__ void find(const LpArgs& p, int row, int col, int64_t& l, int64_t& a) const {
        const uint32_t x = rem + row;
        const uint32_t q = p.inner == 1 ? x : p.by_inner ? __umulhi(x, p.by_inner) : x >= p.inner;
        const uint32_t i = p.inner == 1 ? 0 : x - q * (uint32_t)p.inner;
        l = at_l + q * p.s_outer + i * p.s_inner + col;
        a = at_a + q * p.a_outer + i * p.a_inner + col;
    }
};

// V entries of a tile from its i-th on: at once where they are of one row, or of rows in ORDER and V - 1 apart from first to
// last; else one by one, with no branch between the loads.  (4.1 M rows of 11 in fp32 under int32 masks, both slices of wider
// buffers: forward and back 83 and 107 us, an element at a time 148 and 167, packed 72 and 97)
template <typename T, int MASK, bool NT, int V>
__device__ __forceinline__ void load_apart(const LpArgs& p, const Tile& t, int i, int all, uint32_t by_vocab, bool order,
                                           float (&f1)[1][V]) {
    constexpr int S = MASK == 1 ? 1 : 4;
    const T* l = (const T*)p.logits;
    const char* av = (const char*)p.avail;
    const int last = i + V <= all ? i + V - 1 : all - 1;
    int row = row_in(i, p.vocab, by_vocab), col = i - row * p.vocab;
    const int end = row_in(last, p.vocab, by_vocab);
    int64_t l0, a0, l1, a1;
    t.find(p, row, col, l0, a0);
    t.find(p, end, last - end * p.vocab, l1, a1);
    if (i + V <= all && (row == end || (order && l1 - l0 == V - 1 && (!MASK || a1 - a0 == V - 1)))) {
        load_logits<T, MASK, NT, true>(l + l0, MASK ? av + a0 * S : nullptr, 0, 0, V, f1);
    } else {
        T x[V];
        int32_t on[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            t.find(p, row, col, l0, a0);
            x[j] = l[l0];
            on[j] = MASK == 0 ? 1 : MASK == 1 ? (int32_t)av[a0] : ((const int32_t*)av)[a0];
            if (i + j < last && ++col == p.vocab) col = 0, row++;
        }
#pragma unroll
        for (int j = 0; j < V; j++) f1[0][j] = i + j <= last && on[j] ? (float)x[j] : -INF;
    }
}

template <typename T, int MASK, bool QUADS, bool NT, bool GAPS>
__device__ __forceinline__ void stage_rows(const LpArgs& p, int64_t r0, int n, int stride, uint32_t by_vocab, bool order, float* s) {
    constexpr int V = 16 / sizeof(T);
    const int all = n * p.vocab;
    const auto put = [&](int i, const float(&f)[V]) {
        if (QUADS) {  // (four entries in a row are of one row)
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                const int row = row_in(i + q, p.vocab, by_vocab), col = i + q - row * p.vocab;
                if (i + q < all) *(float4*)(s + row * stride + col) = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
            }
        } else if (stride == p.vocab) {  // (the tile lies in LDS as in memory, with room for the last vector)
#pragma unroll
            for (int q = 0; q < V; q += 4) *(float4*)(s + i + q) = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
        } else {
            int row = row_in(i, p.vocab, by_vocab), col = i - row * p.vocab;
#pragma unroll
            for (int j = 0; j < V; j++) {
                if (i + j < all) s[row * stride + col] = f[j];
                if (++col == p.vocab) col = 0, row++;
            }
        }
    };
    float f1[1][V];
    if (!GAPS) {  // the tile is one run of n * vocab elements, in logits and mask
        const T* l = (const T*)p.logits + r0 * p.vocab;
        const char* av = MASK ? (const char*)p.avail + r0 * p.vocab * (MASK == 1 ? 1 : 4) : nullptr;
        for (int i = threadIdx.x * V; i < all; i += FEW_ROWS * V) {
            if (i + V <= all) load_logits<T, MASK, NT, true>(l, av, i, 0, all, f1);
            else load_logits<T, MASK, false, false>(l, av, i, 0, all, f1);
            put(i, f1[0]);
        }
    } else {
        const Tile t(p, r0);
        for (int i = threadIdx.x * V; i < all; i += FEW_ROWS * V) {
            load_apart<T, MASK, NT, V>(p, t, i, all, by_vocab, order, f1);
            put(i, f1[0]);
        }
    }
}

template <typename T, int MASK, bool QUADS, bool NT, bool GAPS>
__global__ void __launch_bounds__(FEW_ROWS) k_logp_few_fwd(LpArgs p, uint32_t by_vocab, bool order) {
    extern __shared__ float4 s_few[];
    const int64_t r0 = (int64_t)block_index() * FEW_ROWS, r = r0 + threadIdx.x;
    if (r0 >= p.rows) return;
    const int n = (int)(p.rows - r0 < FEW_ROWS ? p.rows - r0 : FEW_ROWS), stride = few_stride(p.vocab);
    stage_rows<T, MASK, QUADS, NT, GAPS>(p, r0, n, stride, by_vocab, order, (float*)s_few);
    __syncthreads();
    if ((int)threadIdx.x >= n) return;
    float* l = (float*)s_few + threadIdx.x * stride;
    Stat s{-FLT_MAX, 0.0f, 0.0f};
    each_entry<QUADS, false>(l, p.vocab, [&](float& x, int) { s.m = fmaxf(s.m, x); });
    each_entry<QUADS, false>(l, p.vocab, [&](float& x, int) {
        const float d = (x - s.m) * LOG2E, e = __builtin_amdgcn_exp2f(d);
        s.s1 += e;
        s.s2 = __builtin_fmaf(e, fmaxf(d, -200.0f), s.s2);
    });
    const float ln = log_s1(s);
    const int64_t tok = p.tokens[r];
    write_row(p, r, s, ln, logp_of(p, tok, tok >= 0 && tok < p.vocab ? l[tok] : 0.0f, s, ln));
    for (int i = 0; i < p.top_k; i++) {  // the largest of what is left, the first of equal ones
        float best = -INF;
        int at = -1;
        each_entry<QUADS, false>(l, p.vocab, [&](float& x, int j) {
            const bool more = x > best;
            best = more ? x : best;
            at = more ? j : at;
        });
        if (at >= 0) l[at] = -INF;
        write_top(p, r, i, s, ln, at >= 0 ? key_of(best, (uint32_t)at) : 0);
    }
}

template <typename T, int MASK, bool QUADS, bool NT, bool GAPS>
__global__ void __launch_bounds__(FEW_ROWS) k_logp_few_bwd(LpArgs p, uint32_t by_vocab, bool order) {
    extern __shared__ float4 s_few[];
    constexpr int V = 16 / sizeof(T);
    float* const s_rows = (float*)s_few;
    const int64_t r0 = (int64_t)block_index() * FEW_ROWS, r = r0 + threadIdx.x;
    if (r0 >= p.rows) return;
    const int n = (int)(p.rows - r0 < FEW_ROWS ? p.rows - r0 : FEW_ROWS), stride = few_stride(p.vocab);
    stage_rows<T, MASK, QUADS, NT, GAPS>(p, r0, n, stride, by_vocab, order, s_rows);
    __syncthreads();
    if ((int)threadIdx.x < n) {
        const RowGrad w = row_grad(p, r);
        each_entry<QUADS, true>(s_rows + threadIdx.x * stride, p.vocab, [&](float& x, int j) { x = entry_grad(w, x, j); });
    }
    __syncthreads();
    T* out = (T*)p.dlogits + r0 * p.vocab;
    const int all = n * p.vocab;
    for (int i = threadIdx.x * V; i < all; i += FEW_ROWS * V) {
        float f[V];
        if (QUADS || stride == p.vocab) {
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                int at = i + q;
                if (QUADS) {
                    const int row = i + q < all ? row_in(i + q, p.vocab, by_vocab) : 0;
                    at = i + q < all ? i + q + row * (stride - p.vocab) : 0;
                }
                const float4 v = *(const float4*)(s_rows + at);
                f[q] = v.x, f[q + 1] = v.y, f[q + 2] = v.z, f[q + 3] = v.w;
            }
        } else {
            int row = row_in(i, p.vocab, by_vocab), col = i - row * p.vocab;
#pragma unroll
            for (int j = 0; j < V; j++) {
                f[j] = i + j < all ? s_rows[row * stride + col] : 0.0f;
                if (++col == p.vocab) col = 0, row++;
            }
        }
        store_upto<T, V, NT>(out + i, all - i, f);
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

// Threads that share a row (0: a lane per row): 16 or 64 where that is at most 4 loads of 16 bytes each; the alternatives take
// whole waves.  With rows for every wave of the GPU a wave takes up to 1024 vectors, loop and all: a block has four lists of
// alternatives to make and join where a wave has one (10000 rows of 5001 in bf16 with 20 of them: 43 us, 75 with a block per
// row; 5000 rows of 16000: 123 and 109)
int threads_for(int64_t rows, int64_t vocab, int dtype, bool top) {
    if (vocab <= (dtype == EC_F32 ? FEW_FP32 : FEW_16BIT)) return 0;
    const int64_t vecs = cdiv(vocab, dtype == EC_F32 ? 4 : 8);
    return vecs <= 64 && !top ? 16 : vecs <= 256 || (rows >= 4096 && vecs <= 1024) ? 64 : 256;
}
// vectors a thread then takes at once: as few as hold the row (what is loaded past it is computed with all the same)
int vectors_for(int64_t vocab, int dtype, int tpr) {
    const int64_t each = cdiv(cdiv(vocab, dtype == EC_F32 ? 4 : 8), tpr);
    return each <= 1 ? 1 : each <= 2 ? 2 : MOST_U;
}
// how rows of few entries lie in memory, logits and mask: one behind the other; in order, with gaps; anyhow (a mask for all)
enum Layout { PACKED, APART, ANYHOW };

// (APART takes rows in order that do not overlap: what lies V - 1 apart is then V in a row)
Layout layout_of(const LpArgs& a) {
    const auto one = [&](int64_t outer, int64_t inner) {
        const bool packed = outer == a.inner * a.vocab && (a.inner == 1 || inner == a.vocab);
        if (packed || a.rows == 1) return PACKED;
        if (a.inner == 1) return outer >= a.vocab ? APART : ANYHOW;
        return inner >= a.vocab && (a.inner >= a.rows || outer >= (a.inner - 1) * inner + a.vocab) ? APART : ANYHOW;
    };
    const Layout l = one(a.s_outer, a.s_inner), m = a.avail ? one(a.a_outer, a.a_inner) : PACKED;
    return l > m ? l : m;
}
// i / vocab = umulhi(i, by_vocab) for i < 2^16 and 2 <= vocab < 2^16: the excess over 2^32 / vocab is below 1
uint32_t by_vocab(int vocab) { return (uint32_t)((((uint64_t)1 << 32) + vocab - 1) / vocab); }

// Few rows: a row is split over as many blocks as fill the GPU, at least one batch of loads each, and a second launch joins them.
// Not where a block is through in few batches: the second launch is 4 us of the host's time, and of the GPU's 1 us or, with
// alternatives to join, 5 (one row of 32000 in bf16, 4 batches: 17.4 us a call split, 13.1 whole, both 4.7 in a graph; with 20
// alternatives 21.0 and 16.6, but 11.0 and 15.5 in a graph; 2 batches: 20.9 and 16.5, 9.7 and 9.2).
int per_split(int64_t rows, int64_t vocab, int dtype, bool top) {
    if (threads_for(rows, vocab, dtype, true) != 256) return INT32_MAX;
    const int64_t batch = 256 * MOST_U * (dtype == EC_F32 ? 4 : 8), batches = cdiv(vocab, batch);
    // (to the nearest: 900 rows of 65536 45.9 us by two blocks each, 40.7 by one; 600 of 200000 71.6 and 89.4)
    const int64_t want = batches <= (top ? 2 : 4) || rows > 1024 ? 1 : (1024 + rows / 2) / rows;
    const int64_t splits = want < batches ? (want < MAX_SPLITS ? want : MAX_SPLITS) : (batches < MAX_SPLITS ? batches : MAX_SPLITS);
    const int64_t each = cdiv(batches, splits) * batch;
    return (int)(each < INT32_MAX ? each : INT32_MAX);
}
int splits_for(int64_t rows, int64_t vocab, int dtype, bool top) { return (int)cdiv(vocab, per_split(rows, vocab, dtype, top)); }

// The streaming hint for what the caches do not hold from one pass to the next.  (4.1 M rows of 11 under int32 masks 207 us
// without it, 170 with; 8192 x 65536 in bf16 553 and 505; 3200 x 10000 44 and 47.  Not for 16 and 64 threads a row, which
// share cache lines between rows: 600 000 rows of 100 146 us without, 161 with.)
bool is_far(const LpArgs& a, int dtype, int mask) {
    return a.rows * a.vocab * (dtype_size(dtype) + (mask == 1 ? 1 : mask == 2 ? 4 : 0)) >= (int64_t)96 << 20;
}

int few_lds(int vocab) { return (FEW_ROWS * few_stride(vocab) + 8) * 4; }  // (the last vector of a tile may be a partial one)

template <typename T, int MASK>
auto few_fwd(bool quads, bool far, bool gaps) {
    if (gaps)
        return quads ? far ? k_logp_few_fwd<T, MASK, true, true, true> : k_logp_few_fwd<T, MASK, true, false, true>
                     : far ? k_logp_few_fwd<T, MASK, false, true, true> : k_logp_few_fwd<T, MASK, false, false, true>;
    return quads ? far ? k_logp_few_fwd<T, MASK, true, true, false> : k_logp_few_fwd<T, MASK, true, false, false>
                 : far ? k_logp_few_fwd<T, MASK, false, true, false> : k_logp_few_fwd<T, MASK, false, false, false>;
}

template <typename T, int MASK>
void go_fwd(LpArgs a, int dtype, hipStream_t st) {
    const int tpr = threads_for(a.rows, a.vocab, dtype, a.top_k > 0), u = tpr ? vectors_for(a.vocab, dtype, tpr) : 0;
    const bool far = is_far(a, dtype, MASK);
    const Layout layout = layout_of(a);
    const auto blocks = [&](int rows) { return grid_of(cdiv(a.rows, rows)); };
    const dim3 b(256);
    a.ahead = a.splits == 1 && cdiv(a.rows, tpr ? 256 / tpr : 1) <= AT_ONCE;
    if (tpr == 0) {
        const auto few = few_fwd<T, MASK>(a.vocab % 4 == 0, far, layout != PACKED);
        hipLaunchKernelGGL(few, blocks(FEW_ROWS), dim3(FEW_ROWS), few_lds(a.vocab), st, a, by_vocab(a.vocab), layout == APART);
    } else if (tpr == 16) {
        if (u == 1) hipLaunchKernelGGL((k_logp_fwd<T, MASK, false, 16, 1, false>), blocks(16), b, 0, st, a);
        else if (u == 2) hipLaunchKernelGGL((k_logp_fwd<T, MASK, false, 16, 2, false>), blocks(16), b, 0, st, a);
        else hipLaunchKernelGGL((k_logp_fwd<T, MASK, false, 16, 4, false>), blocks(16), b, 0, st, a);
    } else if (tpr == 64 && a.top_k) {
        if (u == 1) hipLaunchKernelGGL((k_logp_fwd<T, MASK, true, 64, 1, false>), blocks(4), b, 0, st, a);
        else if (u == 2) hipLaunchKernelGGL((k_logp_fwd<T, MASK, true, 64, 2, false>), blocks(4), b, 0, st, a);
        else hipLaunchKernelGGL((k_logp_fwd<T, MASK, true, 64, 4, false>), blocks(4), b, 0, st, a);
    } else if (tpr == 64) {
        if (u == 2) hipLaunchKernelGGL((k_logp_fwd<T, MASK, false, 64, 2, false>), blocks(4), b, 0, st, a);
        else hipLaunchKernelGGL((k_logp_fwd<T, MASK, false, 64, 4, false>), blocks(4), b, 0, st, a);
    } else {
        const dim3 grid = grid_of(a.rows * a.splits);
        const auto k = a.top_k ? far ? k_logp_fwd<T, MASK, true, 256, MOST_U, true> : k_logp_fwd<T, MASK, true, 256, MOST_U, false>
                               : far ? k_logp_fwd<T, MASK, false, 256, MOST_U, true> : k_logp_fwd<T, MASK, false, 256, MOST_U, false>;
        hipLaunchKernelGGL(k, grid, b, 0, st, a);
        if (a.splits > 1) hipLaunchKernelGGL((k_logp_join<T, MASK>), dim3((unsigned)a.rows), b, 2 * 8 * a.splits * a.top_k, st, a);
    }
}

template <typename T, int MASK>
auto few_bwd(bool quads, bool far, bool gaps) {
    if (gaps)
        return quads ? far ? k_logp_few_bwd<T, MASK, true, true, true> : k_logp_few_bwd<T, MASK, true, false, true>
                     : far ? k_logp_few_bwd<T, MASK, false, true, true> : k_logp_few_bwd<T, MASK, false, false, true>;
    return quads ? far ? k_logp_few_bwd<T, MASK, true, true, false> : k_logp_few_bwd<T, MASK, true, false, false>
                 : far ? k_logp_few_bwd<T, MASK, false, true, false> : k_logp_few_bwd<T, MASK, false, false, false>;
}

template <typename T, int MASK>
void go_bwd(const LpArgs& a, int dtype, hipStream_t st) {
    const int tpr = threads_for(a.rows, a.vocab, dtype, false), u = tpr ? vectors_for(a.vocab, dtype, tpr) : 0;
    const bool far = is_far(a, dtype, MASK);
    const Layout layout = layout_of(a);
    const auto blocks = [&](int rows) { return grid_of(cdiv(a.rows, rows)); };
    const dim3 b(256);
    const auto few = few_bwd<T, MASK>(a.vocab % 4 == 0, far, layout != PACKED);
    if (tpr == 0)
        hipLaunchKernelGGL(few, blocks(FEW_ROWS), dim3(FEW_ROWS), few_lds(a.vocab), st, a, by_vocab(a.vocab), layout == APART);
    else if (tpr == 16 && u == 1)
        hipLaunchKernelGGL((k_logp_bwd<T, MASK, 16, 1, false>), blocks(16), b, 0, st, a);
    else if (tpr == 16 && u == 2)
        hipLaunchKernelGGL((k_logp_bwd<T, MASK, 16, 2, false>), blocks(16), b, 0, st, a);
    else if (tpr == 16)
        hipLaunchKernelGGL((k_logp_bwd<T, MASK, 16, 4, false>), blocks(16), b, 0, st, a);
    else if (tpr == 64 && u == 2)
        hipLaunchKernelGGL((k_logp_bwd<T, MASK, 64, 2, false>), blocks(4), b, 0, st, a);
    else if (tpr == 64)
        hipLaunchKernelGGL((k_logp_bwd<T, MASK, 64, 4, false>), blocks(4), b, 0, st, a);
    else
        hipLaunchKernelGGL((far ? k_logp_bwd<T, MASK, 256, MOST_U, true> : k_logp_bwd<T, MASK, 256, MOST_U, false>),
                           grid_of(a.rows * a.splits), b, 0, st, a);
}

#define EC_LP_GO(GO, T)                                  \
    {                                                    \
        if (mask_dtype == 0) GO<T, 0>(a, dtype, st);     \
        if (mask_dtype == 1) GO<T, 1>(a, dtype, st);     \
        if (mask_dtype == 2) GO<T, 2>(a, dtype, st);     \
    }
#define EC_LP_TYPES(GO)                       \
    if (dtype == EC_F32) EC_LP_GO(GO, float)  \
    if (dtype == EC_BF16) EC_LP_GO(GO, bf16)  \
    if (dtype == EC_F16) EC_LP_GO(GO, f16)

}  // namespace

extern "C" int64_t ec_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t dtype, int32_t top_k) {
    if (rows < 1 || vocab < 1 || vocab > INT32_MAX || !dtype_ok(dtype) || top_k < 0 || top_k > MAX_TOP) return 0;
    const int s = splits_for(rows, vocab, dtype, top_k > 0);
    return s > 1 ? rows * s * part_bytes(top_k) : 0;
}

extern "C" int ec_token_logprobs_fwd(const void* logits, int64_t inner, int64_t s_outer, int64_t s_inner, const int64_t* tokens,
                                     const void* avail, int32_t mask_dtype, int64_t a_outer, int64_t a_inner, int32_t dtype,
                                     int64_t rows, int64_t vocab, int32_t top_k, float* logp, float* entropy, float* lse,
                                     float* top_logp, int64_t* top_index, void* work, int64_t work_bytes, void* stream) {
    LpArgs a{};
    a.logits = logits, a.avail = avail, a.tokens = tokens, a.rows = rows, a.inner = inner, a.s_outer = s_outer;
    a.s_inner = s_inner, a.a_outer = a_outer, a.a_inner = a_inner, a.vocab = (int)(vocab > INT32_MAX || vocab < 1 ? 0 : vocab);
    a.by_inner = inner >= 2 && inner < 1 << 15 ? by_vocab((int)inner) : 0;
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
    a.splits = splits_for(rows, vocab, dtype, top_k > 0);
    a.per_split = per_split(rows, vocab, dtype, top_k > 0);
    if (rows * a.splits > INT32_MAX) return ec::fail(EC_EINVAL, "ec_token_logprobs_fwd: %lld rows", (long long)rows);
    const hipStream_t st = (hipStream_t)stream;
    EC_LP_TYPES(go_fwd)
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
    a.by_inner = inner >= 2 && inner < 1 << 15 ? by_vocab((int)inner) : 0;
    if (const char* m = bad("ec_token_logprobs_bwd", a, dtype, mask_dtype)) return ec::fail(EC_EINVAL, "%s", m);
    if (rows == 0) return EC_OK;
    if (!lse || !entropy || !dlogits) return ec::fail(EC_EINVAL, "ec_token_logprobs_bwd: null argument");
    a.lse = const_cast<float*>(lse), a.entropy_in = entropy, a.dlogp = dlogp, a.dentropy = dentropy, a.dlogits = dlogits;
    a.per_split = 256 * MOST_U * (dtype == EC_F32 ? 4 : 8);
    a.splits = threads_for(rows, vocab, dtype, false) == 256 ? (int)cdiv(vocab, a.per_split) : 1;
    if (rows * a.splits > INT32_MAX) return ec::fail(EC_EINVAL, "ec_token_logprobs_bwd: %lld rows", (long long)rows);
    const hipStream_t st = (hipStream_t)stream;
    EC_LP_TYPES(go_bwd)
    EC_HIP(hipGetLastError());
    return EC_OK;
}
