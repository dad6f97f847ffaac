// ec_norm.hip -- layer norm over the last dimension, forward and backward, for rows of fp32 / bf16 / fp16.
//
//   mean = sum x / C;  var = sum (x - mean)^2 / C;  rstd = 1 / sqrt(var + eps);  xhat = (x - mean) rstd;  y = xhat w + b
//   dx = rstd (dy w - mean_c(dy w) - xhat mean_c(dy w xhat));  dw = sum_r dy xhat;  db = sum_r dy
//
// Bound by HBM: 8 and 14 operations an element against 2 and 3 elements moved.  So every element is read once: a row stays
// in the registers of the TPR threads that share it (16 bytes a thread and load, NV loads), which makes the variance an
// exact second pass over (x - mean) at no traffic; a thread keeps its columns from row to row, so that weight, bias and
// the sums of dw and db stay in registers over all rows of a block.  dw and db leave as one partial row per block, added
// up in a fixed order by a second kernel (no atomics: the same bits every run).  All sums are fp32.
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

// sum of (a, b) over the threads of a row.  TPR <= 64: in the wave; else through LDS, one barrier: `slot` alternates from
// call to call, so that the reads of one call are over before the call after the next writes
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*s)[16], int slot) {
    a = lanes_sum<(TPR < 64 ? TPR : 64)>(a);
    b = lanes_sum<(TPR < 64 ? TPR : 64)>(b);
    if (TPR > 64) {
        if ((threadIdx.x & 63) == 0) s[slot][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        const float2 v = s[slot][threadIdx.x & (TPR / 64 - 1)];  // (a wave's value in each lane of a group)
        a = lanes_sum<TPR / 64>(v.x);
        b = lanes_sum<TPR / 64>(v.y);
    }
}

// Vectors of a row, and what of them belongs to it.  A row's last vector is read whole where that stays inside the tensor
// (it then holds the start of the next row, or padding) and masked: reading it element by element would cost every row a
// wait of its own.
template <typename T, int V>
struct Mask {
    uint32_t w[4];
    __device__ __forceinline__ void set(int n) {  // the first n
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int left = (n - k * (V / 4)) * (int)sizeof(T) * 8;  // bits of this word
            w[k] = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
        }
    }
    __device__ __forceinline__ raw_t<T, V> of(raw_t<T, V> v) const {
        uint32_t u[4];
        __builtin_memcpy(u, &v, 16);
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] &= w[k];
        __builtin_memcpy(&v, u, 16);
        return v;
    }
};
// v, of which the compiler from here on knows nothing: what was made from it before is made again, not kept
template <typename T, int V>
__device__ __forceinline__ raw_t<T, V> afresh(raw_t<T, V> v) {
    uint32_t u[4];
    __builtin_memcpy(u, &v, 16);
    asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3]));
    __builtin_memcpy(&v, u, 16);
    return v;
}
// the vector of column c < cols of a row at `off`; end: the tensor's last element plus one
template <bool NT, typename T, int V>
__device__ __forceinline__ raw_t<T, V> row_vector(const T* base, int64_t off, int c, int cols, int64_t end) {
    if (off + c + V <= end) return load_raw<NT, T, V>(base + off + c);
    return load_raw_upto<NT, T, V>(base + off + c, cols - c);
}

template <typename T, int TPR, int NV, bool NT>
__global__ void __launch_bounds__(block_threads(TPR)) k_ln_fwd(NormArgs p) {
    constexpr int V = 16 / sizeof(T), RPB = block_threads(TPR) / TPR;
    __shared__ float4 s_red[2][TPR > 64 ? TPR / 64 : 1];
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
    const bool ragged = p.cols % V != 0;
    Mask<T, V> mask[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) mask[i].set(p.cols - (i * TPR + t) * V);
    const int64_t end = (p.rows - 1) * p.x_stride + p.cols;
    raw_t<T, V> next[NV];
    const auto fetch = [&](int64_t r0) {
        const int64_t off = (r0 + g < p.rows ? r0 + g : p.rows - 1) * p.x_stride;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + t) * V;
            next[i] = raw_t<T, V>{};
            if (c < p.cols) next[i] = row_vector<NT, T, V>((const T*)p.x, off, c, p.cols, end);
        }
    };
    fetch((int64_t)blockIdx.x * RPB);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB, slot ^= 1) {
        const bool on = r0 + g < p.rows;
        const int64_t r = r0 + g;
        float f[NV][V];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) widen<T, V>(ragged ? mask[i].of(next[i]) : next[i], f[i]);
        if (r0 + (int64_t)gridDim.x * RPB < p.rows) fetch(r0 + (int64_t)gridDim.x * RPB);  // (while this row is worked on)
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
            const float4 v = s_red[slot][threadIdx.x & (TPR / 64 - 1)];
            mean = lanes_sum<TPR / 64>(v.x) * inv_c;
            sq = lanes_sum<TPR / 64>(v.z + v.w * (v.y - mean) * (v.y - mean));
        }
        const float rstd = 1.0f / sqrtf(sq * inv_c + p.eps);
        if (on) {
            T* y = (T*)p.out + r * p.cols;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * TPR + t) * V;
#pragma unroll
                for (int j = 0; j < V; j++) f[i][j] = __builtin_fmaf((f[i][j] - mean) * rstd, w[i][j], b[i][j]);
                store_upto<T, V, NT>(y + c, p.cols - c, f[i]);
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
    const bool ragged = p.cols % V != 0;
    Mask<T, V> mask[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) mask[i].set(p.cols - (i * TPR + t) * V);
    const int64_t end_x = (p.rows - 1) * p.x_stride + p.cols, end_dy = (p.rows - 1) * p.dy_stride + p.cols;
    raw_t<T, V> next_x[NV], next_dy[NV];
    float next_mean, next_rstd;
    const auto fetch = [&](int64_t r0) {
        const bool on = r0 + g < p.rows;
        const int64_t r = on ? r0 + g : p.rows - 1;
        // a row behind the last adds nothing to dw and db: its dy is taken as 0
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * TPR + t) * V;
            next_x[i] = next_dy[i] = raw_t<T, V>{};
            if (c < p.cols) {
                next_x[i] = row_vector<NT, T, V>((const T*)p.x, r * p.x_stride, c, p.cols, end_x);
                if (on) next_dy[i] = row_vector<NT, T, V>((const T*)p.dy, r * p.dy_stride, c, p.cols, end_dy);
            }
        }
        next_mean = p.mean[r], next_rstd = p.rstd[r];
    };
    // (a block of 1024 threads has 128 registers a thread: no room for the next row with two vectors or more)
    constexpr bool AHEAD = TPR < 1024 || NV == 1;
    if (AHEAD) fetch((int64_t)blockIdx.x * RPB);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < p.rows; r0 += (int64_t)gridDim.x * RPB, slot ^= 1) {
        const bool on = r0 + g < p.rows;
        const int64_t r = r0 + g;
        // (without room for the next row the row stays as it was read, and xhat is made from it twice: half the registers)
        raw_t<T, V> x[NV], dy[NV];
        if (!AHEAD) fetch(r0);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            x[i] = ragged ? mask[i].of(next_x[i]) : next_x[i];
            dy[i] = ragged ? mask[i].of(next_dy[i]) : next_dy[i];
        }
        const float mean = next_mean, rstd = next_rstd;
        if (AHEAD && r0 + (int64_t)gridDim.x * RPB < p.rows) fetch(r0 + (int64_t)gridDim.x * RPB);  // (while this row is worked on)
        float s1 = 0.0f, s2 = 0.0f;
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
            }
            if (!AHEAD) __builtin_amdgcn_sched_barrier(0);  // (vectors one after the other: interleaved they need more registers)
        }
        row_sum2<TPR>(s1, s2, s_red, slot);
        s1 *= inv_c;
        s2 *= inv_c;
        if (on && p.out) {
            T* dx = (T*)p.out + r * p.cols;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * TPR + t) * V;
                const raw_t<T, V> x2 = AHEAD ? x[i] : afresh<T, V>(x[i]), dy2 = AHEAD ? dy[i] : afresh<T, V>(dy[i]);
                float o[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float h = ((float)x2[j] - mean) * rstd;
                    o[j] = rstd * (__builtin_fmaf((float)dy2[j], w[i][j], -s1) - h * s2);
                }
                store_upto<T, V, NT>(dx + c, p.cols - c, o);
                if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (!p.partials) return;
    float* part = p.partials + (int64_t)blockIdx.x * 2 * p.cols;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * TPR + t) * V;
        if (RPB > 1) {  // the row groups of a wave, then the waves, in a fixed order
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
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
            if (wave == 0 && lane < TPR)
#pragma unroll
                for (int k = 1; k < 4; k++)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        dw[i][j] += s_part[0][j][k * 64 + t];
                        db[i][j] += s_part[1][j][k * 64 + t];
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

// ---- rows too long for the registers of a block: a block of 1024 threads reads its row again for each pass (from L2) ----
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
        const float rstd = 1.0f / sqrtf(sq / (float)p.cols + p.eps);
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

// ---- which variant: the fewest threads per row that hold it in one vector each; two or four beyond 1024 threads ----
struct Shape {
    int tpr, nv, rpb;  // tpr 0: the wide kernels
};
Shape shape_for(int64_t cols, int dtype) {
    const int64_t vecs = cdiv(cols, dtype == EC_F32 ? 4 : 8);
    for (int tpr : {2, 4, 8, 16, 32, 64, 128, 256, 512, 1024})
        if (vecs <= tpr) return tpr == 128 ? Shape{64, 2, 4} : Shape{tpr, 1, block_threads(tpr) / tpr};
    if (vecs <= 2048) return {1024, 2, 1};
    if (vecs <= 4096 && dtype == EC_F32) return {1024, 4, 1};
    return {0, 0, 1};
}

int bwd_blocks(const Shape& s, int64_t rows) {
    const int64_t want = cdiv(rows, s.rpb), most = NUM_CU * (s.tpr <= 256 ? 4 : s.tpr == 512 ? 2 : 1);
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
    EC_LN(2, 1) EC_LN(4, 1) EC_LN(8, 1) EC_LN(16, 1) EC_LN(32, 1) EC_LN(64, 1) EC_LN(64, 2) EC_LN(256, 1) EC_LN(512, 1) EC_LN(1024, 1) EC_LN(1024, 2)
    if constexpr (sizeof(T) == 4) { EC_LN(1024, 4) }
#undef EC_LN
}

const char* bad_args(const char* who, const void* x, int64_t x_stride, int32_t dtype, int32_t wdtype, int64_t rows,
                     int64_t cols) {
    static thread_local char msg[160];
    if (!dtype_ok(dtype) || (wdtype != EC_F32 && wdtype != dtype))
        snprintf(msg, sizeof msg, "%s: type %d with weights of type %d", who, dtype, wdtype);
    else if (rows < 0 || cols < 1 || cols > (1 << 24))
        snprintf(msg, sizeof msg, "%s: %lld rows of %lld columns (1 .. 2^24)", who, (long long)rows, (long long)cols);
    else if (rows && (!x || x_stride < 0))
        snprintf(msg, sizeof msg, "%s: no input, or a negative row stride", who);
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
    const Shape s = shape_for(cols, dtype);
    if (s.tpr == 0) {
        const dim3 grid((unsigned)(rows < 1024 ? rows : 1024));
        if (dtype == EC_F32) hipLaunchKernelGGL(k_ln_fwd_wide<float>, grid, dim3(WIDE), 0, st, a);
        if (dtype == EC_BF16) hipLaunchKernelGGL(k_ln_fwd_wide<bf16>, grid, dim3(WIDE), 0, st, a);
        if (dtype == EC_F16) hipLaunchKernelGGL(k_ln_fwd_wide<f16>, grid, dim3(WIDE), 0, st, a);
    } else {
        const int64_t want = cdiv(rows, s.rpb), most = NUM_CU * (s.tpr <= 256 ? 8 : s.tpr == 512 ? 4 : 2);
        const unsigned blocks = (unsigned)(want < most ? want : most);
        if (dtype == EC_F32) dispatch<float, false>(a, s, blocks, st);
        if (dtype == EC_BF16) dispatch<bf16, false>(a, s, blocks, st);
        if (dtype == EC_F16) dispatch<f16, false>(a, s, blocks, st);
    }
    EC_HIP(hipGetLastError());
    return EC_OK;
}

extern "C" int64_t ec_layer_norm_bwd_partials(int64_t rows, int64_t cols, int32_t dtype) {
    if (rows < 1 || cols < 1 || cols > (1 << 24) || !dtype_ok(dtype)) return 0;
    const Shape s = shape_for(cols, dtype);
    return s.tpr ? bwd_blocks(s, rows) : wide_parts(rows);
}

extern "C" int ec_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                                 const float* rstd, const void* weight, int32_t dtype, int32_t wdtype, int64_t rows,
                                 int64_t cols, void* dx, float* partials, int64_t n_partials, void* dweight, void* dbias,
                                 void* stream) {
    if (const char* m = bad_args("ec_layer_norm_bwd", x, x_stride, dtype, wdtype, rows, cols)) return ec::fail(EC_EINVAL, "%s", m);
    if (rows < 1) return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: no rows");
    const bool want_w = dweight || dbias;
    if (!dy || dy_stride < 0 || !mean || !rstd) return ec::fail(EC_EINVAL, "ec_layer_norm_bwd: null argument");
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
    const Shape s = shape_for(cols, dtype);
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
