// ec_norm.hip -- layer norm over the last dimension, forward and backward, for rows of fp32 / bf16 / fp16.
//
//   mean = sum x / C;  var = sum (x - mean)^2 / C;  rstd = 1 / sqrt(var + eps);  xhat = (x - mean) rstd;  y = xhat w + b
//   dx = rstd (dy w - mean_c(dy w) - xhat mean_c(dy w xhat));  dw = sum_r dy xhat;  db = sum_r dy
//
// Bound by HBM: 8 and 14 operations an element against 2 and 3 elements moved.  So up to 16384 columns every element is read
// once: a row stays in the registers of the TPR threads that share it (16 bytes a thread and load, NV loads), which makes the
// variance an exact second pass over (x - mean) at no traffic; a thread keeps its columns from row to row, so that weight, bias and
// the sums of dw and db stay in registers over all rows of a block.  dw and db leave as one partial row per block, added
// up in a fixed order by a second kernel (no atomics: the same bits every run).  All sums are fp32.
//
// Measured (a copy runs at 6.4 TB/s at best): 4.1 M rows of 64 in fp32 388 us forward (5.5 TB/s) and 543 us backward (5.9);
// 16384 rows of 4096 in bf16 48 us (5.6) and 77 us (5.2), dw and db of which 5 us more.  Rows that just miss a power of two
// of vectors leave threads idle: 16384 rows of 2053 in fp16 43 us, of 4096 48.  (Not faster: as many waves as a row needs, a
// number known at run time, 119 -> 145 us for 30000 rows of 1601; three vectors a thread instead of twice the threads, 43 ->
// 44 us; idle vectors skipped by a branch, 43 -> 42 us there, but 126 -> 150 us where there are none.)  Narrow rows that end
// inside a vector: 4 M of 11 in fp32 99 us (3.9 TB/s) and 127 us (4.4).  Long ones: 4096 rows of 16384 in fp32 98 us (5.5) and
// 212 us (3.8: spills, see k_ln_bwd), 8192 of 10240 118 us (5.7) and 533 us (1.9), 8192 of 16384 in bf16 98 us (5.5) and 160 us (5.0).
#include "ec_stream.h"

namespace {

using namespace ecs;

constexpr int NUM_CU = 256;

struct NormArgs {
    const void *x, *dy, *w, *b;
    int64_t x_stride, dy_stride, rows;
    int cols, wdtype;   // wdtype: EC_F32, or the rows' type
    float eps;
    float *mean, *rstd;  // forward: written unless NULL; backward: read
    void* out;           // y or dx [rows, cols]; dx may be NULL
    float* partials;     // [gridDim.x][2][cols] or NULL
};

template <typename T, int V>
__device__ __forceinline__ void load_weight(const void* w, int wdtype, int c, int cols, float fill, float (&f)[V]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < V; j++) f[j] = fill;
    } else if (wdtype == EC_F32) {
        load_upto((const float*)w + c, (int64_t)cols - c, 0.0f, f);
    } else {
        load_upto((const T*)w + c, (int64_t)cols - c, 0.0f, f);
    }
}

constexpr int block_threads(int tpr) { return tpr < 256 ? 256 : tpr; }

// the wave of this thread's row whose value this lane picks up: each of a row's TPR / 64 waves by some lane of a group
template <int TPR>
__device__ __forceinline__ int wave_slot() {
    return ((threadIdx.x >> 6) & ~(TPR / 64 - 1)) | (threadIdx.x & (TPR / 64 - 1));
}

// 1 / sqrt(v) to one unit in the last place, for every v >= 0 (the instruction alone takes what is below 2^-126 as 0)
__device__ __forceinline__ float inverse_root(float v) {
    const bool small = v < 1e-30f;
    const float q = __builtin_amdgcn_rsqf(small ? v * 18446744073709551616.0f : v);
    return small ? q * 4294967296.0f : q;
}

// sum of (a, b) over the threads of a row.  TPR <= 64: in the wave; else through LDS, one barrier: `slot` alternates from
// call to call, so that the reads of one call are over before the call after the next writes
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*s)[16], int slot) {
    a = lanes_sum<(TPR < 64 ? TPR : 64)>(a);
    b = lanes_sum<(TPR < 64 ? TPR : 64)>(b);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) s[slot][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        const float2 v = s[slot][wave_slot<TPR>()];
        a = lanes_sum<TPR / 64>(v.x);
        b = lanes_sum<TPR / 64>(v.y);
    }
}

// How a thread reads its vectors of a row: always, from an address inside the tensor, with no branch, and what does not
// belong to the row is masked afterwards.  A row's last vector is read whole (it then holds the start of the next row, or
// padding); at the end of the tensor it is read as much further in front as it sticks out, and shifted; a thread with no
// columns reads the row's first.  (Read element by element, or under a condition, each would be a wait of its own.)
template <typename T, int V, int TPR, int NV, bool NT>
struct RowReader {
    const T* base;
    int64_t stride, rows, end;  // end: the tensor's last element plus one, at least V
    int cols;
    bool exact;                 // all of it belongs to the row, for every thread
    __device__ __forceinline__ RowReader(const void* b, int64_t stride_, int64_t rows_, int cols_)
        : base((const T*)b), stride(stride_), rows(rows_), end((rows_ - 1) * stride_ + cols_), cols(cols_), exact(cols_ == TPR * NV * V) {}
    __device__ __forceinline__ int64_t row(int64_t r) const { return (r < rows ? r : rows - 1) * stride; }
    __device__ __forceinline__ void load(int64_t r, int t, raw_t<T, V> (&v)[NV]) const {
        const int64_t off = row(r);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + t) * V;
            const int64_t at = off + (c < cols ? c : 0);
            v[i] = load_raw<NT, T, V>(base + (at + V <= end ? at : end - V));
        }
    }
    // the words of a vector's first n elements
    __device__ __forceinline__ static Words first(int n) {
        const int keep = n * (int)sizeof(T) * 8;
        return Words{keep >= 64 ? ~0ull : keep <= 0 ? 0ull : (1ull << keep) - 1, keep >= 128 ? ~0ull : keep <= 64 ? 0ull : (1ull << (keep - 64)) - 1};
    }
    __device__ __forceinline__ void masks(int t, Words (&m)[NV]) const {
#pragma unroll
        for (int i = 0; i < NV; i++) m[i] = first(cols - (i * TPR + t) * V);
    }
    __device__ __forceinline__ void mask(int64_t r, int t, const Words (&m)[NV], raw_t<T, V> (&v)[NV]) const {
        if (exact) return;
        const int64_t past = row(r) + V - end;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + t) * V;
            Words w;
            __builtin_memcpy(&w, &v[i], 16);
            if (c < cols && past + c > 0) {  // (the tensor's last vector: read past + c elements early)
                const int bits = (int)(past + c) * (int)sizeof(T) * 8;
                w = bits >= 64 ? Words{w.hi >> (bits - 64), 0} : Words{w.lo >> bits | w.hi << (64 - bits), w.hi >> bits};
            }
            w.lo &= m[i].lo;
            w.hi &= m[i].hi;
            __builtin_memcpy(&v[i], &w, 16);
        }
    }
};

// v, of which the compiler from here on knows nothing.  What was made from it before is made again, not kept; and a load of
// it is waited for here (by itself the compiler waits for the next row only behind this row's stores, and so for these too)
template <typename T, int V, int NV>
__device__ __forceinline__ void afresh(raw_t<T, V> (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
        uint32_t u[4];
        __builtin_memcpy(u, &v[i], 16);
        asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3]));
        __builtin_memcpy(&v[i], u, 16);
    }
}

template <typename T, int TPR, int NV, bool NT>
__global__ void __launch_bounds__(block_threads(TPR)) k_ln_fwd(NormArgs p) {
    constexpr int V = 16 / sizeof(T), RPB = block_threads(TPR) / TPR;
    __shared__ float4 s_red[2][block_threads(TPR) / 64];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        load_weight<T, V>(p.w, p.wdtype, (i * TPR + t) * V, p.cols, 1.0f, w[i]);
        load_weight<T, V>(p.b, p.wdtype, (i * TPR + t) * V, p.cols, 0.0f, b[i]);
    }
    const float inv_c = 1.0f / (float)p.cols;
    // columns that this thread's wave holds (TPR > 64), as the sum of squares is first taken about the wave's own mean
    float n_wave = 0.0f, inv_wave = 0.0f;
    if (TPR > 64) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int left = p.cols - (i * TPR + (t & ~63)) * V;
            n_wave += (float)(left <= 0 ? 0 : left < 64 * V ? left : 64 * V);
        }
        inv_wave = n_wave > 0.0f ? 1.0f / n_wave : 0.0f;
    }
    int slot = 0;
    // (every thread of a block makes every round: the lane sums and barriers are for all; rows behind the last are read
    // as the last and not written)
    const RowReader<T, V, TPR, NV, NT> in(p.x, p.x_stride, p.rows, p.cols);
    raw_t<T, V> x[NV], next[NV];
    Words own[NV];
    in.masks(t, own);
    in.load((int64_t)blockIdx.x * RPB + g, t, x);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB, slot ^= 1) {
        const int64_t r = r0 + g;
        const bool on = r < p.rows, more = r0 + (int64_t)gridDim.x * RPB < p.rows;
        in.mask(r, t, own, x);
        if (more) in.load(r + (int64_t)gridDim.x * RPB, t, next);  // (while this row is worked on)
        float f[NV][V];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) widen<T, V>(x[i], f[i]);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < V; j++) sum += f[i][j];
        sum = lanes_sum<(TPR < 64 ? TPR : 64)>(sum);
        // squares about the mean of the row (TPR <= 64) or of the wave's part of it, then moved to the row's mean
        const float about = sum * (TPR <= 64 ? inv_c : inv_wave);
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + t) * V;
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = c + j < p.cols ? f[i][j] - about : 0.0f;
                sq = __builtin_fmaf(d, d, sq);
            }
        }
        sq = lanes_sum<(TPR < 64 ? TPR : 64)>(sq);
        float mean = about;
        if (TPR > 64) {
            if ((threadIdx.x & 63) == 0) s_red[slot][threadIdx.x >> 6] = make_float4(sum, about, sq, n_wave);
            __syncthreads();
            const float4 v = s_red[slot][wave_slot<(TPR > 64 ? TPR : 64)>()];
            mean = lanes_sum<TPR / 64>(v.x) * inv_c;
            sq = lanes_sum<TPR / 64>(v.z + v.w * (v.y - mean) * (v.y - mean));
        }
        const float rstd = inverse_root(sq * inv_c + p.eps);
        raw_t<T, V> y[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int j = 0; j < V; j++) f[i][j] = __builtin_fmaf((f[i][j] - mean) * rstd, w[i][j], b[i][j]);
            y[i] = narrow<T, V>(f[i]);
        }
        if (more) {
            afresh<T, V, NV>(next);
#pragma unroll
            for (int i = 0; i < NV; i++) x[i] = next[i];
        }
        if (on) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * TPR + t) * V;
                store_raw_upto<NT, T, V>((T*)p.out + r * p.cols + c, p.cols - c, y[i]);
            }
            if (t == 0) {
                if (p.mean) p.mean[r] = mean;
                if (p.rstd) p.rstd[r] = rstd;
            }
        }
    }
}

template <typename T, int TPR, int NV, bool NT>
__global__ void __launch_bounds__(block_threads(TPR)) k_ln_bwd(NormArgs p) {
    constexpr int V = 16 / sizeof(T), RPB = block_threads(TPR) / TPR;
    __shared__ float2 s_red[2][16];
    __shared__ float s_part[2][RPB > 1 ? V : 1][RPB > 1 ? 256 : 1];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        load_weight<T, V>(p.w, p.wdtype, (i * TPR + t) * V, p.cols, 1.0f, w[i]);
#pragma unroll
        for (int j = 0; j < V; j++) dw[i][j] = db[i][j] = 0.0f;
    }
    const float inv_c = 1.0f / (float)p.cols;
    int slot = 0;
    const RowReader<T, V, TPR, NV, NT> in_x(p.x, p.x_stride, p.rows, p.cols), in_dy(p.dy, p.dy_stride, p.rows, p.cols);
    // (a block of 1024 threads has 128 registers a thread: no room for the next row with two vectors or more; the row then
    // stays as it was read, and xhat and dy w are made from it twice.  Weights, both sums and the row are more than 128 even
    // so: 99 registers a thread go to scratch in fp32, 16 to 18 in 16 bits)
    constexpr bool AHEAD = TPR < 1024 || NV == 1;
    raw_t<T, V> x[NV], dy[NV], next_x[NV], next_dy[NV];
    float mean = 0.0f, rstd = 0.0f, next_mean = 0.0f, next_rstd = 0.0f;
    Words own[NV];
    in_x.masks(t, own);
    const auto load = [&](int64_t r, raw_t<T, V>(&a)[NV], raw_t<T, V>(&b)[NV], float& m, float& s) {
        in_x.load(r, t, a);
        in_dy.load(r, t, b);
        m = p.mean[r < p.rows ? r : p.rows - 1], s = p.rstd[r < p.rows ? r : p.rows - 1];
    };
    load((int64_t)blockIdx.x * RPB + g, x, dy, mean, rstd);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB, slot ^= 1) {
        const int64_t r = r0 + g, r_next = r + (int64_t)gridDim.x * RPB;
        const bool on = r < p.rows, more = r0 + (int64_t)gridDim.x * RPB < p.rows;
        in_x.mask(r, t, own, x);
        in_dy.mask(r, t, own, dy);
        if (AHEAD && more) load(r_next, next_x, next_dy, next_mean, next_rstd);  // (while this row is worked on)
        if (RPB > 1 && !on) {  // a row behind the last adds nothing to dw and db
#pragma unroll
            for (int i = 0; i < NV; i++) dy[i] = raw_t<T, V>{};
        }
        float s1 = 0.0f, s2 = 0.0f, hs[AHEAD ? NV : 1][V], as[AHEAD ? NV : 1][V];
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float h = ((float)x[i][j] - mean) * rstd, d = (float)dy[i][j], a = d * w[i][j];
                // (columns behind the last: d is 0 there, and w 0 or 1)
                dw[i][j] = __builtin_fmaf(d, h, dw[i][j]);
                db[i][j] += d;
                s1 += a;
                s2 = __builtin_fmaf(a, h, s2);
                if (AHEAD) hs[AHEAD ? i : 0][j] = h, as[AHEAD ? i : 0][j] = a;
            }
            if (!AHEAD) __builtin_amdgcn_sched_barrier(0);  // (vectors one after the other: interleaved they need more registers)
        }
        row_sum2<TPR>(s1, s2, s_red, slot);
        s1 *= inv_c;
        s2 *= inv_c;
        if (!AHEAD) {
            afresh<T, V, NV>(x);
            afresh<T, V, NV>(dy);
        }
        raw_t<T, V> dx[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float o[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float h = AHEAD ? hs[AHEAD ? i : 0][j] : ((float)x[i][j] - mean) * rstd;
                const float a = AHEAD ? as[AHEAD ? i : 0][j] : (float)dy[i][j] * w[i][j];
                o[j] = rstd * (a - s1 - h * s2);
            }
            dx[i] = narrow<T, V>(o);
            if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
        if (AHEAD && more) {
            afresh<T, V, NV>(next_x);
            afresh<T, V, NV>(next_dy);
#pragma unroll
            for (int i = 0; i < NV; i++) x[i] = next_x[i], dy[i] = next_dy[i];
            mean = next_mean, rstd = next_rstd;
        }
        if (on && p.out) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * TPR + t) * V;
                store_raw_upto<NT, T, V>((T*)p.out + r * p.cols + c, p.cols - c, dx[i]);
            }
        }
        if (!AHEAD && more) load(r_next, x, dy, mean, rstd);
    }
    if (!p.partials) return;
    float* part = p.partials + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * TPR + t) * V;
        if (RPB > 1) {  // the row groups of a wave, then the waves, in a fixed order
            constexpr int APART = TPR < 64 ? 64 : TPR;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; j++) {
#pragma unroll
                for (int o = TPR; o < 64; o *= 2) {
                    dw[i][j] += __shfl_xor(dw[i][j], o);
                    db[i][j] += __shfl_xor(db[i][j], o);
                }
                s_part[0][j][threadIdx.x] = dw[i][j];
                s_part[1][j][threadIdx.x] = db[i][j];
            }
            __syncthreads();
            if ((int)threadIdx.x < TPR)
#pragma unroll
                for (int k = APART; k < 256; k += APART)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        dw[i][j] += s_part[0][j][k + t];
                        db[i][j] += s_part[1][j][k + t];
                    }
        }
        if ((int)threadIdx.x < TPR) {
            store_upto(part + c, (int64_t)p.cols - c, dw[i]);
            store_upto(part + p.cols + c, (int64_t)p.cols - c, db[i]);
        }
    }
}

// dw / db [cols] = sum over the partial rows: 64 columns a block, 16 threads a column, added in a fixed order
template <typename W>
__global__ void __launch_bounds__(1024) k_ln_wgrad(const float* partials, int n, int cols, W* dw, W* db) {
    __shared__ float s[16][64];
    W* out = blockIdx.y ? db : dw;
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), l = threadIdx.x >> 6;
    float a = 0.0f;
    if (c < cols && out)
        for (int k = l; k < n; k += 16 * 8) {
            float f[8];  // (eight loads in flight: this kernel is nothing but their latency)
#pragma unroll
            for (int u = 0; u < 8; u++) f[u] = k + 16 * u < n ? partials[((int64_t)(k + 16 * u) * 2 + blockIdx.y) * cols + c] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; u++) a += f[u];
        }
    s[l][threadIdx.x & 63] = a;
    __syncthreads();
    if (l == 0 && c < cols && out) {
        for (int k = 1; k < 16; k++) a += s[k][threadIdx.x];
        out[c] = (W)a;
    }
}

// ---- rows too long for the registers of a block: a block of 1024 threads reads its row again for each pass, three times
// forward, x and dy twice for dx and once more for dw and db (2048 rows of 32768 in bf16: 84 us forward, 105 + 57 + 5 back,
// against 42 and 63 for each element moved once at 6.4 TB/s; 1024 in fp32: 84 and 101 + 49 + 5) ----
constexpr int WIDE = 1024;

template <typename T>
__global__ void __launch_bounds__(WIDE) k_ln_fwd_wide(NormArgs p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float2 s_red[2][16];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = (const T*)p.x + r * p.x_stride;
        T* y = (T*)p.out + r * p.cols;
        float a = 0.0f, b = 0.0f, f[V];
        for (int64_t c = threadIdx.x * V; c < p.cols; c += WIDE * V) {
            load_upto(x + c, p.cols - c, 0.0f, f);
#pragma unroll
            for (int j = 0; j < V; j++) a += f[j];
        }
        row_sum2<WIDE>(a, b, s_red, 0);
        const float mean = a / (float)p.cols;
        float sq = 0.0f;
        b = 0.0f;
        for (int64_t c = threadIdx.x * V; c < p.cols; c += WIDE * V) {
            load_upto(x + c, p.cols - c, mean, f);
#pragma unroll
            for (int j = 0; j < V; j++) sq = __builtin_fmaf(f[j] - mean, f[j] - mean, sq);
        }
        row_sum2<WIDE>(sq, b, s_red, 1);
        const float rstd = inverse_root(sq / (float)p.cols + p.eps);
        for (int64_t c = threadIdx.x * V; c < p.cols; c += WIDE * V) {
            float w[V], bb[V];
            load_upto(x + c, p.cols - c, 0.0f, f);
            load_weight<T, V>(p.w, p.wdtype, (int)c, p.cols, 1.0f, w);
            load_weight<T, V>(p.b, p.wdtype, (int)c, p.cols, 0.0f, bb);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = __builtin_fmaf((f[j] - mean) * rstd, w[j], bb[j]);
            store_upto(y + c, p.cols - c, f);
        }
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(WIDE) k_ln_dx_wide(NormArgs p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float2 s_red[2][16];
    int slot = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x, slot ^= 1) {
        const T *x = (const T*)p.x + r * p.x_stride, *dy = (const T*)p.dy + r * p.dy_stride;
        T* dx = (T*)p.out + r * p.cols;
        const float mean = p.mean[r], rstd = p.rstd[r];
        float s1 = 0.0f, s2 = 0.0f, f[V], d[V], w[V];
        for (int64_t c = threadIdx.x * V; c < p.cols; c += WIDE * V) {
            load_upto(x + c, p.cols - c, 0.0f, f);
            load_upto(dy + c, p.cols - c, 0.0f, d);
            load_weight<T, V>(p.w, p.wdtype, (int)c, p.cols, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; j++) {
                s1 = __builtin_fmaf(d[j], w[j], s1);
                s2 = __builtin_fmaf(d[j] * w[j], (f[j] - mean) * rstd, s2);
            }
        }
        row_sum2<WIDE>(s1, s2, s_red, slot);
        s1 /= (float)p.cols;
        s2 /= (float)p.cols;
        for (int64_t c = threadIdx.x * V; c < p.cols; c += WIDE * V) {
            load_upto(x + c, p.cols - c, 0.0f, f);
            load_upto(dy + c, p.cols - c, 0.0f, d);
            load_weight<T, V>(p.w, p.wdtype, (int)c, p.cols, 1.0f, w);
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = rstd * (d[j] * w[j] - s1 - (f[j] - mean) * rstd * s2);
            store_upto(dx + c, p.cols - c, f);
        }
    }
}

// dw / db partials: a wave per strip of 64 x V columns (blockIdx.x), every gridDim.y-th row from blockIdx.y on
template <typename T>
__global__ void __launch_bounds__(64) k_ln_dw_wide(NormArgs p) {
    constexpr int V = 16 / sizeof(T);
    const int64_t c = ((int64_t)blockIdx.x * 64 + threadIdx.x) * V;
    float dw[V], db[V], f[V], d[V];
#pragma unroll
    for (int j = 0; j < V; j++) dw[j] = db[j] = 0.0f;
    for (int64_t r = blockIdx.y; r < p.rows; r += gridDim.y) {
        load_upto((const T*)p.x + r * p.x_stride + c, p.cols - c, 0.0f, f);
        load_upto((const T*)p.dy + r * p.dy_stride + c, p.cols - c, 0.0f, d);
        const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
        for (int j = 0; j < V; j++) {
            dw[j] = __builtin_fmaf(d[j], (f[j] - mean) * rstd, dw[j]);
            db[j] += d[j];
        }
    }
    float* part = p.partials + (int64_t)blockIdx.y * 2 * p.cols;
    store_upto(part + c, p.cols - c, dw);
    store_upto(part + p.cols + c, p.cols - c, db);
}

// ---- which variant: one vector a thread up to a wave, then as many elements a thread as registers allow before more threads:
// the sums over a row's threads cost about 100 operations a thread and row, as much as four elements do (16384 rows of 4096 in
// bf16, forward: 512 threads with 8 each 59 us, 256 with 16 each 50 us).  Backward, where a thread also holds its sums of dw and
// db, 16 elements leave two waves a SIMD, which is enough up to 2048 columns of 16 bits and not beyond (4096 columns: 81 us,
// with 512 threads of 8 each 72) ----
struct Shape {
    int tpr, nv, rpb;  // tpr 0: the wide kernels
};
Shape shape_for(int64_t rows, int64_t cols, int dtype, bool bwd) {
    const bool f32 = dtype == EC_F32;
    const int64_t vecs = cdiv(cols, f32 ? 4 : 8);
    if (rows * cols < (f32 ? 4 : 8)) return {0, 0, 1};  // (less than a vector: RowReader)
    for (int tpr : {2, 4, 8, 16, 32, 64})
        if (vecs <= tpr) return {tpr, 1, 256 / tpr};
    if (vecs <= 128) return {64, 2, 4};
    const int most = f32 ? 4 : 2;
    for (int tpr : {64, 128, 256, 512, 1024}) {
        const int nv = bwd && !f32 && tpr >= 256 ? 1 : most;
        if (vecs <= tpr * nv) return {tpr, nv, block_threads(tpr) / tpr};
    }
    if (vecs <= (f32 ? 4096 : 2048)) return {1024, f32 ? 4 : 2, 1};
    return {0, 0, 1};
}

// Waves a CU, as swept (1 to 16 blocks a CU over widths from 11 to 16384): what fills the memory's queue, and no more than
// the registers keep resident; blocks beyond that run behind each other and read their weights again.  4.1 M rows of 64 in
// fp32: forward 16 waves 967 us, 32 waves 994; backward 12 waves 964 us, 16 waves 997, 8 waves 988 (forward and back each).
int blocks_for(const Shape& s, int64_t rows, int dtype, bool bwd) {
    const int elements = s.nv * (dtype == EC_F32 ? 4 : 8);
    int waves = 16;
    if (!bwd) waves = s.tpr <= 8 ? 32 : elements > 8 && dtype == EC_F32 ? 12 : 16;
    else if (s.tpr < 1024 && s.tpr > 8) waves = s.nv > 1 ? 8 : s.tpr < 512 ? 12 : 16;
    const int64_t want = cdiv(rows, s.rpb), each = waves * 64 / block_threads(s.tpr), most = NUM_CU * (each < 1 ? 1 : each);
    return (int)(want < most ? want : most);
}
int wide_parts(int64_t rows) { return (int)(rows < 32 ? rows : 32); }

// from this many elements on nothing of a tensor is left in the caches for who reads it next: the streaming hint then
constexpr int64_t NT_ELEMENTS = 32 << 20;

template <typename T, bool BWD, int TPR, int NV>
void go(const NormArgs& a, unsigned blocks, hipStream_t st) {
    const dim3 g(blocks), b(block_threads(TPR));
    const bool far = a.rows * a.cols >= NT_ELEMENTS;
    if constexpr (BWD) {
        if (far) hipLaunchKernelGGL((k_ln_bwd<T, TPR, NV, true>), g, b, 0, st, a);
        else hipLaunchKernelGGL((k_ln_bwd<T, TPR, NV, false>), g, b, 0, st, a);
    } else {
        if (far) hipLaunchKernelGGL((k_ln_fwd<T, TPR, NV, true>), g, b, 0, st, a);
        else hipLaunchKernelGGL((k_ln_fwd<T, TPR, NV, false>), g, b, 0, st, a);
    }
}

template <typename T, bool BWD>
void dispatch(const NormArgs& a, const Shape& s, unsigned blocks, hipStream_t st) {
#define EC_LN(TPR, NV) \
    if (s.tpr == TPR && s.nv == NV) return go<T, BWD, TPR, NV>(a, blocks, st);
    EC_LN(2, 1) EC_LN(4, 1) EC_LN(8, 1) EC_LN(16, 1) EC_LN(32, 1) EC_LN(64, 1) EC_LN(64, 2)
    if constexpr (sizeof(T) == 4) {
        EC_LN(64, 4) EC_LN(128, 4) EC_LN(256, 4) EC_LN(512, 4) EC_LN(1024, 4)
    } else if constexpr (BWD) {
        EC_LN(128, 2) EC_LN(512, 1) EC_LN(1024, 1) EC_LN(1024, 2)
    } else {
        EC_LN(128, 2) EC_LN(256, 2) EC_LN(512, 2) EC_LN(1024, 2)
    }
#undef EC_LN
}

const char* bad_args(const char* who, const void* x, int64_t x_stride, int32_t dtype, int32_t wdtype, int64_t rows,
                     int64_t cols) {
    static thread_local char msg[160];
    if (!dtype_ok(dtype) || (wdtype != EC_F32 && wdtype != dtype))
        snprintf(msg, sizeof msg, "%s: type %d with weights of type %d", who, dtype, wdtype);
    else if (rows < 0 || cols < 1 || cols > (1 << 24))
        snprintf(msg, sizeof msg, "%s: %lld rows of %lld columns (1 .. 2^24)", who, (long long)rows, (long long)cols);
    else if (rows && !x)
        snprintf(msg, sizeof msg, "%s: no input", who);
    else if (x_stride < 0 || (rows > 1 && x_stride < cols))
        snprintf(msg, sizeof msg, "%s: rows of %lld columns %lld apart", who, (long long)cols, (long long)x_stride);
    else
        return nullptr;
    return msg;
}

}  // namespace

extern "C" int ec_layer_norm_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias, int32_t dtype,
                                 int32_t wdtype, int64_t rows, int64_t cols, double eps, void* y, float* mean, float* rstd,
                                 void* stream) {
    if (const char* m = bad_args("ec_layer_norm_fwd", x, x_stride, dtype, wdtype, rows, cols)) return ec::fail(EC_EINVAL, "%s", m);
    if (rows == 0) return EC_OK;
    if (!y || !(eps >= 0)) return ec::fail(EC_EINVAL, "ec_layer_norm_fwd: no output, or eps below 0");
    NormArgs a{};
    a.x = x, a.w = weight, a.b = bias, a.x_stride = x_stride, a.rows = rows, a.cols = (int)cols, a.wdtype = wdtype;
    a.eps = (float)eps, a.mean = mean, a.rstd = rstd, a.out = y;
    const hipStream_t st = (hipStream_t)stream;
    const Shape s = shape_for(rows, cols, dtype, false);
    if (s.tpr == 0) {
        const dim3 grid((unsigned)(rows < 1024 ? rows : 1024));
        if (dtype == EC_F32) hipLaunchKernelGGL(k_ln_fwd_wide<float>, grid, dim3(WIDE), 0, st, a);
        if (dtype == EC_BF16) hipLaunchKernelGGL(k_ln_fwd_wide<bf16>, grid, dim3(WIDE), 0, st, a);
        if (dtype == EC_F16) hipLaunchKernelGGL(k_ln_fwd_wide<f16>, grid, dim3(WIDE), 0, st, a);
    } else {
        const unsigned blocks = (unsigned)blocks_for(s, rows, dtype, false);
        if (dtype == EC_F32) dispatch<float, false>(a, s, blocks, st);
        if (dtype == EC_BF16) dispatch<bf16, false>(a, s, blocks, st);
        if (dtype == EC_F16) dispatch<f16, false>(a, s, blocks, st);
    }
    EC_HIP(hipGetLastError());
    return EC_OK;
}

extern "C" int64_t ec_layer_norm_bwd_partials(int64_t rows, int64_t cols, int32_t dtype) {
    if (rows < 1 || cols < 1 || cols > (1 << 24) || !dtype_ok(dtype)) return 0;
    const Shape s = shape_for(rows, cols, dtype, true);
    return s.tpr ? blocks_for(s, rows, dtype, true) : wide_parts(rows);
}

extern "C" int ec_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                                 const float* rstd, const void* weight, int32_t dtype, int32_t wdtype, int64_t rows,
                                 int64_t cols, void* dx, float* partials, int64_t n_partials, void* dweight, void* dbias,
                                 void* stream) {
    if (const char* m = bad_args("ec_layer_norm_bwd", x, x_stride, dtype, wdtype, rows, cols)) return ec::fail(EC_EINVAL, "%s", m);
    if (rows < 1) return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: no rows");
    const bool want_w = dweight || dbias;
    if (!dy || !mean || !rstd) return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: null argument");
    if (dy_stride < 0 || (rows > 1 && dy_stride < cols))
        return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: rows of %lld columns %lld apart", (long long)cols, (long long)dy_stride);
    const int64_t need = ec_layer_norm_bwd_partials(rows, cols, dtype);
    if (want_w && (!partials || n_partials != need))
        return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: %lld partial rows (%lld are needed)", (long long)(partials ? n_partials : 0),
                        (long long)need);
    if (!want_w && !dx) return EC_OK;
    NormArgs a{};
    a.x = x, a.dy = dy, a.w = weight, a.x_stride = x_stride, a.dy_stride = dy_stride, a.rows = rows, a.cols = (int)cols;
    a.wdtype = wdtype, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.out = dx;
    a.partials = want_w ? partials : nullptr;
    const hipStream_t st = (hipStream_t)stream;
    const Shape s = shape_for(rows, cols, dtype, true);
    if (s.tpr == 0) {
        if (dx) {
            const dim3 grid((unsigned)(rows < 1024 ? rows : 1024));
            if (dtype == EC_F32) hipLaunchKernelGGL(k_ln_dx_wide<float>, grid, dim3(WIDE), 0, st, a);
            if (dtype == EC_BF16) hipLaunchKernelGGL(k_ln_dx_wide<bf16>, grid, dim3(WIDE), 0, st, a);
            if (dtype == EC_F16) hipLaunchKernelGGL(k_ln_dx_wide<f16>, grid, dim3(WIDE), 0, st, a);
        }
        if (want_w) {
            const dim3 grid((unsigned)cdiv(cols, 64 * (dtype == EC_F32 ? 4 : 8)), (unsigned)need);
            if (dtype == EC_F32) hipLaunchKernelGGL(k_ln_dw_wide<float>, grid, dim3(64), 0, st, a);
            if (dtype == EC_BF16) hipLaunchKernelGGL(k_ln_dw_wide<bf16>, grid, dim3(64), 0, st, a);
            if (dtype == EC_F16) hipLaunchKernelGGL(k_ln_dw_wide<f16>, grid, dim3(64), 0, st, a);
        }
    } else {
        const unsigned blocks = (unsigned)need;
        if (dtype == EC_F32) dispatch<float, true>(a, s, blocks, st);
        if (dtype == EC_BF16) dispatch<bf16, true>(a, s, blocks, st);
        if (dtype == EC_F16) dispatch<f16, true>(a, s, blocks, st);
    }
    EC_HIP(hipGetLastError());
    if (want_w) {
        const dim3 grid((unsigned)cdiv(cols, 64), 2);
        const int n = (int)need, c = (int)cols;
        if (wdtype == EC_F32)
            hipLaunchKernelGGL(k_ln_wgrad<float>, grid, dim3(1024), 0, st, partials, n, c, (float*)dweight, (float*)dbias);
        if (wdtype == EC_BF16)
            hipLaunchKernelGGL(k_ln_wgrad<bf16>, grid, dim3(1024), 0, st, partials, n, c, (bf16*)dweight, (bf16*)dbias);
        if (wdtype == EC_F16)
            hipLaunchKernelGGL(k_ln_wgrad<f16>, grid, dim3(1024), 0, st, partials, n, c, (f16*)dweight, (f16*)dbias);
        EC_HIP(hipGetLastError());
    }
    return EC_OK;
}
