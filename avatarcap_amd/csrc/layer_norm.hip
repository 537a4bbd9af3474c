// Layer norm of rows, forward and backward (include/avcap.h avc_layer_norm, avc_layer_norm_backward).  Bound by HBM: every kernel reads its inputs once and writes its outputs once.
//
//   y  = (x - mean) rstd g + b,   mean and biased variance over the row, rstd = 1 / sqrt(var + eps)
//   dx = rstd (t - mean(t) - xh mean(t xh)),   t = g dy,  xh = (x - mean) rstd
//   dg = sum_rows dy xh,  db = sum_rows dy
//
// A row is held in the registers of `tpr` lanes (a part of a wave, a wave, 256 or 1024 threads), V adjacent values (16 bytes) per lane and chunk, so the variance is taken from
// the centred values in a second pass over registers, not from a difference of sums.  Rows longer than the registers of 1024 threads take kernels that read the row again.
// The backward kernels walk rows with a fixed set of workgroups; a lane keeps the gradients of ITS columns in registers over all of its rows, the workgroups leave them in
// part[workgroup][2 C] and launch_colsum2 adds those in order: no atomics, the same bits every time.
// 262144 x 256 bf16: forward 62 us (4.3 TB/s), backward 78 us (5.2 TB/s); 16384 x 8192 f16 forward 118 us (4.6 TB/s); a large copy reaches 4.9.
#include <algorithm>
#include "avcap_internal.h"
#include "linear.h"

namespace avc { namespace lin {

namespace {

template <typename T> struct Width { static constexpr int V = 16 / sizeof(T); };

// A lane's run of V adjacent columns.  The run that the row ends in, and those past the end, are moved back to end with the row, so that every lane loads whole runs of any
// alignment without a branch (a branch around a load makes each load wait for the one before); `first` is where the lane's own columns begin in it, V if it has none.  C >= V.
template <int V> struct Run {
    int64_t at;
    int first;
    __device__ __forceinline__ Run(int64_t col, int64_t C) : at(min(col, C - V)), first((int)min(col - min(col, C - V), (int64_t)V)) {}
};

template <int V, typename T> __device__ __forceinline__ void load_run(const T *row, int64_t at, float *out)
{
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef vec loose __attribute__((aligned(sizeof(T))));               // one load, whatever the alignment
    const vec v = *reinterpret_cast<const loose *>(row + at);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = (float)v[j];
}

template <int V, typename T> __device__ __forceinline__ void store_run(T *row, const Run<V> &run, const float *in)
{
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    vec v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)in[j];
    if (run.first == 0) *reinterpret_cast<loose *>(row + run.at) = v;
    else
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (j >= run.first) row[run.at + j] = v[j];
}

// sum over the tpr threads of a row; TPR = 0: a runtime power of two up to the wave
template <int TPR> __device__ __forceinline__ float row_sum(float v, int tpr, float *red)
{
    if constexpr (TPR == 0) {
        for (int o = tpr >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
        return v;
    } else {
        for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
        __syncthreads();                                                 // the last use of `red` is over
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) s += red[w];
        return s;
    }
}

// R rows at a time per set of lanes, so that a lane has several loads in flight
template <typename T, int V, int TPR, int NCH, int R>
__global__ __launch_bounds__(TPR ? TPR : 256) void norm_kernel(const T *__restrict__ x, int64_t ldx, const T *__restrict__ g, const T *__restrict__ b, float eps, int64_t M, int64_t C, int tpr_log,
                                                              T *y, int64_t ldy, float *mean_out, float *rstd_out)
{
    __shared__ float red[16];
    const int tpr = TPR ? TPR : 1 << tpr_log, lane = threadIdx.x & (tpr - 1), rows = TPR ? 1 : 256 >> tpr_log, sub = TPR ? 0 : threadIdx.x >> tpr_log;
    const float count = (float)C;                                        // divided by, not multiplied with 1 / C: a row of equal values has that value as its mean
    for (int64_t m0 = (int64_t)blockIdx.x * rows * R; m0 < M; m0 += (int64_t)gridDim.x * rows * R) {
        float v[R][NCH][V], mean[R], rstd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {                                    // rows past the end repeat the last one: the other lanes of the wave still need the shuffles
            const T *row = x + min(m0 + r * rows + sub, M - 1) * ldx;
#pragma unroll
            for (int c = 0; c < NCH; ++c) load_run<V>(row, Run<V>(((int64_t)c * tpr + lane) * V, C).at, v[r][c]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int first = Run<V>(((int64_t)c * tpr + lane) * V, C).first;
#pragma unroll
                for (int j = 0; j < V; ++j) s += j >= first ? v[r][c][j] : 0.f;
            }
            mean[r] = row_sum<TPR>(s, tpr, red) / count;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int first = Run<V>(((int64_t)c * tpr + lane) * V, C).first;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    v[r][c][j] -= mean[r];
                    s += j >= first ? v[r][c][j] * v[r][c][j] : 0.f;
                }
            }
            rstd[r] = 1.f / sqrtf(row_sum<TPR>(s, tpr, red) / count + eps);
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const Run<V> run(((int64_t)c * tpr + lane) * V, C);
            float gg[V], bb[V];
            if (g) load_run<V>(g, run.at, gg);
            if (b) load_run<V>(b, run.at, bb);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t m = m0 + r * rows + sub;
                if (m >= M) continue;
#pragma unroll
                for (int j = 0; j < V; ++j) v[r][c][j] = v[r][c][j] * rstd[r] * (g ? gg[j] : 1.f) + (b ? bb[j] : 0.f);
                store_run<V>(y + m * ldy, run, v[r][c]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t m = m0 + r * rows + sub;
            if (mean_out && lane == 0 && m < M) { mean_out[m] = mean[r]; rstd_out[m] = rstd[r]; }
        }
    }
}

// rows longer than 1024 threads' registers: three passes over the row, the second and third from the caches
template <typename T>
__global__ __launch_bounds__(1024) void norm_long_kernel(const T *__restrict__ x, int64_t ldx, const T *__restrict__ g, const T *__restrict__ b, float eps, int64_t M, int64_t C, T *y, int64_t ldy,
                                                         float *mean_out, float *rstd_out)
{
    constexpr int V = Width<T>::V;
    __shared__ float red[16];
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const T *row = x + m * ldx;
        float v[V], s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            const Run<V> run(c, C);
            load_run<V>(row, run.at, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += j >= run.first ? v[j] : 0.f;
        }
        const float mean = row_sum<1024>(s, 1024, red) / (float)C;
        s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            const Run<V> run(c, C);
            load_run<V>(row, run.at, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += j >= run.first ? (v[j] - mean) * (v[j] - mean) : 0.f;
        }
        const float rstd = 1.f / sqrtf(row_sum<1024>(s, 1024, red) / (float)C + eps);
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            float gg[V], bb[V];
            const Run<V> run(c, C);
            load_run<V>(row, run.at, v);
            if (g) load_run<V>(g, run.at, gg);
            if (b) load_run<V>(b, run.at, bb);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * (g ? gg[j] : 1.f) + (b ? bb[j] : 0.f);
            store_run<V>(y + m * ldy, run, v);
        }
        if (mean_out && threadIdx.x == 0) { mean_out[m] = mean; rstd_out[m] = rstd; }
    }
}

template <typename T, int V, int TPR, int NCH>
__global__ __launch_bounds__(TPR ? TPR : 256) void norm_backward_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, const T *__restrict__ g,
                                                                       const float *__restrict__ mean_in, const float *__restrict__ rstd_in, int64_t M, int64_t C, int tpr_log, T *dx, int64_t lddx,
                                                                       float *part, T *dg_out, T *db_out)
{
    __shared__ float red[TPR ? 16 : 256 * (V + 1)];
    const int tpr = TPR ? TPR : 1 << tpr_log, lane = threadIdx.x & (tpr - 1), rows = TPR ? 1 : 256 >> tpr_log, sub = TPR ? 0 : threadIdx.x >> tpr_log;
    const float inv = 1.f / (float)C;
    float gg[NCH][V], dg[NCH][V], db[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        if (g) load_run<V>(g, Run<V>(((int64_t)c * tpr + lane) * V, C).at, gg[c]);
#pragma unroll
        for (int j = 0; j < V; ++j) { dg[c][j] = db[c][j] = 0.f; if (!g) gg[c][j] = 1.f; }
    }
    for (int64_t m0 = (int64_t)blockIdx.x * rows; m0 < M; m0 += (int64_t)gridDim.x * rows) {
        const bool in = m0 + sub < M;
        const int64_t m = in ? m0 + sub : 0;
        float xv[NCH][V], t[NCH][V];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int64_t at = Run<V>(((int64_t)c * tpr + lane) * V, C).at;
            load_run<V>(x + m * ldx, at, xv[c]);
            load_run<V>(dy + m * lddy, at, t[c]);
        }
        const float mean = mean_in[m], rstd = rstd_in[m];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int first = Run<V>(((int64_t)c * tpr + lane) * V, C).first;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = (xv[c][j] - mean) * rstd;
                if (in) { dg[c][j] += t[c][j] * xh; db[c][j] += t[c][j]; }
                t[c][j] *= gg[c][j];
                xv[c][j] = xh;
                s1 += j >= first ? t[c][j] : 0.f;
                s2 += j >= first ? t[c][j] * xh : 0.f;
            }
        }
        if (!dx) continue;
        s1 = row_sum<TPR>(s1, tpr, red) * inv;
        s2 = row_sum<TPR>(s2, tpr, red) * inv;
        if (!in) continue;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
            for (int j = 0; j < V; ++j) t[c][j] = rstd * (t[c][j] - s1 - xv[c][j] * s2);
            store_run<V>(dx + m * lddx, Run<V>(((int64_t)c * tpr + lane) * V, C), t[c]);
        }
    }
    if (!dg_out && !db_out) return;
    float *out = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const Run<V> run(((int64_t)c * tpr + lane) * V, C);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&v)[V] = which ? db[c] : dg[c];
            if constexpr (TPR == 0) {                                    // the workgroup's rows meet in LDS
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) red[threadIdx.x * (V + 1) + j] = v[j];
                __syncthreads();
                if (sub == 0)
                    for (int r = 1; r < rows; ++r)
#pragma unroll
                        for (int j = 0; j < V; ++j) v[j] += red[(r * tpr + lane) * (V + 1) + j];
            }
            if (sub == 0)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j >= run.first) {
                        if (gridDim.x > 1) out[which * C + run.at + j] = v[j];
                        else if (T *to = which ? db_out : dg_out) to[run.at + j] = (T)v[j];       // a single workgroup's sums are the gradients themselves
                    }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, const T *__restrict__ g,
                                                                  const float *__restrict__ mean_in, const float *__restrict__ rstd_in, int64_t M, int64_t C, T *dx, int64_t lddx)
{
    constexpr int V = Width<T>::V;
    __shared__ float red[16];
    for (int64_t m = blockIdx.x; m < M; m += gridDim.x) {
        const float mean = mean_in[m], rstd = rstd_in[m];
        float xv[V], t[V], gg[V], s1 = 0.f, s2 = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            const Run<V> run(c, C);
            load_run<V>(x + m * ldx, run.at, xv);
            load_run<V>(dy + m * lddy, run.at, t);
            if (g) load_run<V>(g, run.at, gg);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = t[j] * (g ? gg[j] : 1.f);
                s1 += j >= run.first ? u : 0.f;
                s2 += j >= run.first ? u * ((xv[j] - mean) * rstd) : 0.f;
            }
        }
        s1 = row_sum<1024>(s1, 1024, red) / (float)C;
        s2 = row_sum<1024>(s2, 1024, red) / (float)C;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            const Run<V> run(c, C);
            load_run<V>(x + m * ldx, run.at, xv);
            load_run<V>(dy + m * lddy, run.at, t);
            if (g) load_run<V>(g, run.at, gg);
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = rstd * (t[j] * (g ? gg[j] : 1.f) - s1 - (xv[j] - mean) * rstd * s2);
            store_run<V>(dx + m * lddx, run, t);
        }
    }
}

// column sums for the long rows: 256 threads x V columns, a strip of rows per workgroup
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, const float *__restrict__ mean_in,
                                                           const float *__restrict__ rstd_in, int64_t M, int64_t C, int64_t rows_per, float *part)
{
    constexpr int V = Width<T>::V;
    const int64_t col = ((int64_t)blockIdx.y * 256 + threadIdx.x) * V, m1 = min(M, ((int64_t)blockIdx.x + 1) * rows_per);
    if (col >= C) return;
    const Run<V> run(col, C);
    float dg[V] = {}, db[V] = {}, xv[V], t[V];
    for (int64_t m = (int64_t)blockIdx.x * rows_per; m < m1; ++m) {
        load_run<V>(x + m * ldx, run.at, xv);
        load_run<V>(dy + m * lddy, run.at, t);
        const float mean = mean_in[m], rstd = rstd_in[m];
#pragma unroll
        for (int j = 0; j < V; ++j) { dg[j] += t[j] * ((xv[j] - mean) * rstd); db[j] += t[j]; }
    }
    float *out = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j >= run.first) { out[run.at + j] = dg[j]; out[C + run.at + j] = db[j]; }
}

constexpr int64_t MAX_GRID = 1 << 20;                                   // the kernels walk rows beyond it
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a row of C values is spread: the smallest set of threads whose registers (up to four chunks each) hold it.
struct Spread { int tpr, nch, tpr_log; bool narrow; };                   // tpr = 0: too long; narrow: rows shorter than a run, one value per lane
Spread spread_of(int64_t C, int dtype)
{
    const int V = dtype == AVC_F32 ? 4 : 8;
    const int64_t runs = cdiv(C, V);
    if (C < V) return Spread{8, 1, 3, true};
    if (runs <= 128) {
        int lg = 3;
        while (lg < 6 && (1 << lg) < runs) ++lg;
        return Spread{1 << lg, runs > 64 ? 2 : 1, lg, false};
    }
    if (runs <= 1024) return Spread{256, runs > 512 ? 4 : runs > 256 ? 2 : 1, 8, false};
    if (runs <= 2048) return Spread{1024, 2, 10, false};
    return Spread{0, 0, 0, false};
}

// workgroups of the backward pass (strips of the column sums)
int64_t backward_blocks(int64_t M, int64_t C, int dtype)
{
    const Spread s = spread_of(C, dtype);
    if (s.tpr == 0) return std::max<int64_t>(1, std::min<int64_t>(cdiv(M, 16), 64));
    if (M <= 4 * std::max(1, 256 / s.tpr)) return 1;
    if (s.tpr <= 64) return std::min<int64_t>(cdiv(M, 256 / s.tpr), 1024);
    return std::min<int64_t>(M, s.tpr == 256 ? 1024 : 512);
}

template <typename T> int norm_forward(const void *x, int64_t ldx, const void *g, const void *b, float eps, int64_t M, int64_t C, int dtype, void *y, int64_t ldy, float *mean, float *rstd,
                                       hipStream_t s)
{
    constexpr int W = Width<T>::V;
    const Spread sp = spread_of(C, dtype);
#define AVC_NORM(V, TPR, NCH, R, BLOCK)                                                                                                                             \
    hipLaunchKernelGGL((norm_kernel<T, V, TPR, NCH, R>), dim3((unsigned)std::min<int64_t>(cdiv(M, (R) * (TPR ? 1 : 256 / sp.tpr)), MAX_GRID)), dim3(BLOCK), 0, s, (const T *)x, ldx,                \
                       (const T *)g, (const T *)b, eps, M, C, sp.tpr_log, (T *)y, ldy, mean, rstd)
    if (sp.narrow) AVC_NORM(1, 0, 1, 1, 256);
    else if (sp.tpr == 0)
        hipLaunchKernelGGL(norm_long_kernel<T>, dim3((unsigned)std::min<int64_t>(M, MAX_GRID)), dim3(1024), 0, s, (const T *)x, ldx, (const T *)g, (const T *)b, eps, M, C, (T *)y, ldy, mean, rstd);
    else if (sp.tpr <= 64) {
        if (M < 8192) { if (sp.nch == 1) AVC_NORM(W, 0, 1, 1, 256); else AVC_NORM(W, 0, 2, 1, 256); }
        else { if (sp.nch == 1) AVC_NORM(W, 0, 1, 4, 256); else AVC_NORM(W, 0, 2, 2, 256); }
    } else if (sp.tpr == 256) {
        if (sp.nch == 1) AVC_NORM(W, 256, 1, 1, 256); else if (sp.nch == 2) AVC_NORM(W, 256, 2, 1, 256); else AVC_NORM(W, 256, 4, 1, 256);
    } else AVC_NORM(W, 1024, 2, 1, 1024);
#undef AVC_NORM
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

template <typename T> int norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *g, const float *mean, const float *rstd, int64_t M, int64_t C, int dtype, void *dx,
                                        int64_t lddx, void *dg, void *db, float *part, hipStream_t s)
{
    const Spread sp = spread_of(C, dtype);
    const int64_t blocks = backward_blocks(M, C, dtype);
    const bool sums = dg || db;
    float *p = part;
    constexpr int W = Width<T>::V;
#define AVC_NORM(V, TPR, NCH, BLOCK)                                                                                                                                \
    hipLaunchKernelGGL((norm_backward_kernel<T, V, TPR, NCH>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, (const T *)dy, lddy, (const T *)x, ldx, (const T *)g, mean, rstd, M, C, sp.tpr_log,       \
                       (T *)dx, lddx, p, (T *)dg, (T *)db)
    if (sp.narrow) AVC_NORM(1, 0, 1, 256);
    else if (sp.tpr == 0) {
        if (dx && M) hipLaunchKernelGGL(norm_backward_long_kernel<T>, dim3((unsigned)std::min<int64_t>(M, MAX_GRID)), dim3(1024), 0, s, (const T *)dy, lddy, (const T *)x, ldx, (const T *)g, mean, rstd, M, C, (T *)dx, lddx);
        if (sums)
            hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((unsigned)blocks, (unsigned)cdiv(C, 256 * Width<T>::V)), dim3(256), 0, s, (const T *)dy, lddy, (const T *)x, ldx, mean, rstd, M, C,
                               cdiv(M, blocks), p);
    } else if (sp.tpr <= 64) {
        if (sp.nch == 1) AVC_NORM(W, 0, 1, 256); else AVC_NORM(W, 0, 2, 256);
    } else if (sp.tpr == 256) {
        if (sp.nch == 1) AVC_NORM(W, 256, 1, 256); else if (sp.nch == 2) AVC_NORM(W, 256, 2, 256); else AVC_NORM(W, 256, 4, 256);
    } else AVC_NORM(W, 1024, 2, 1024);
#undef AVC_NORM
    AVC_HIP(hipGetLastError());
    if (sums && (blocks > 1 || sp.tpr == 0)) return launch_colsum2(p, (int)blocks, C, dtype, dg, db, s);
    return AVC_OK;
}

}  // namespace

int layer_norm(const void *x, int64_t ldx, const void *g, const void *b, float eps, int64_t M, int64_t C, int dtype, void *y, int64_t ldy, float *mean, float *rstd, hipStream_t s)
{
    if (dtype == AVC_F32) return norm_forward<float>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
    if (dtype == AVC_BF16) return norm_forward<__bf16>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
    return norm_forward<_Float16>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
}

size_t layer_norm_backward_workspace(int64_t M, int64_t C, int dtype)
{
    const int64_t blocks = backward_blocks(M, C, dtype);
    return blocks == 1 && spread_of(C, dtype).tpr ? 0 : sizeof(float) * 2 * (size_t)blocks * (size_t)C;   // a single workgroup writes the gradients itself
}

int layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *g, const float *mean, const float *rstd, int64_t M, int64_t C, int dtype, void *dx, int64_t lddx,
                        void *dg, void *db, float *part, hipStream_t s)
{
    if (dtype == AVC_F32) return norm_backward<float>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
    if (dtype == AVC_BF16) return norm_backward<__bf16>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
    return norm_backward<_Float16>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
}

}}  // namespace avc::lin
