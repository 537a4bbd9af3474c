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
#include <algorithm>
#include "avcap_internal.h"
#include "linear.h"

namespace avc { namespace lin {

namespace {

template <typename T> struct Width { static constexpr int V = 16 / sizeof(T); };

// V values of a row from column c on, zeros past the end.  Any alignment.
template <typename T> __device__ __forceinline__ void load_run(const T *row, int64_t c, int64_t C, float *out)
{
    constexpr int V = Width<T>::V;
    T v[V];
    if (c + V <= C) __builtin_memcpy(v, row + c, sizeof v);
    else
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = c + j < C ? row[c + j] : (T)0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = (float)v[j];
}

template <typename T> __device__ __forceinline__ void store_run(T *row, int64_t c, int64_t C, const float *in)
{
    constexpr int V = Width<T>::V;
    T v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)in[j];
    if (c + V <= C) __builtin_memcpy(row + c, v, sizeof v);
    else
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < C) row[c + j] = v[j];
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

template <typename T, int TPR, int NCH>
__global__ __launch_bounds__(TPR ? TPR : 256) void norm_kernel(const T *__restrict__ x, int64_t ldx, const T *__restrict__ g, const T *__restrict__ b, float eps, int64_t M, int64_t C, int tpr_log,
                                                              T *y, int64_t ldy, float *mean_out, float *rstd_out)
{
    constexpr int V = Width<T>::V;
    __shared__ float red[16];
    const int tpr = TPR ? TPR : 1 << tpr_log, lane = threadIdx.x & (tpr - 1), rows = TPR ? 1 : 256 >> tpr_log, sub = TPR ? 0 : threadIdx.x >> tpr_log;
    for (int64_t m0 = (int64_t)blockIdx.x * rows; m0 < M; m0 += (int64_t)gridDim.x * rows) {
        const int64_t m = m0 + sub;
        const bool in = m < M;                                               // TPR = 0 only: the other lanes of the wave still need the shuffles
        const T *row = x + (in ? m : 0) * ldx;
        float v[NCH][V], s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            load_run(row, ((int64_t)c * tpr + lane) * V, C, v[c]);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[c][j];
        }
        const float inv = 1.f / (float)C, mean = row_sum<TPR>(s, tpr, red) * inv;
        s = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] -= mean;
                if (((int64_t)c * tpr + lane) * V + j < C) s += v[c][j] * v[c][j];
            }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, tpr, red) * inv + eps);
        if (!in) continue;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int64_t col = ((int64_t)c * tpr + lane) * V;
            if (col >= C) continue;
            float gg[V], bb[V];
            if (g) load_run(g, col, C, gg);
            if (b) load_run(b, col, C, bb);
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] = v[c][j] * rstd * (g ? gg[j] : 1.f) + (b ? bb[j] : 0.f);
            store_run(y + m * ldy, col, C, v[c]);
        }
        if (mean_out && lane == 0) { mean_out[m] = mean; rstd_out[m] = rstd; }
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
            load_run(row, c, C, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[j];
        }
        const float mean = row_sum<1024>(s, 1024, red) / (float)C;
        s = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            load_run(row, c, C, v);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < C) s += (v[j] - mean) * (v[j] - mean);
        }
        const float rstd = 1.f / sqrtf(row_sum<1024>(s, 1024, red) / (float)C + eps);
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            float gg[V], bb[V];
            load_run(row, c, C, v);
            if (g) load_run(g, c, C, gg);
            if (b) load_run(b, c, C, bb);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (v[j] - mean) * rstd * (g ? gg[j] : 1.f) + (b ? bb[j] : 0.f);
            store_run(y + m * ldy, c, C, v);
        }
        if (mean_out && threadIdx.x == 0) { mean_out[m] = mean; rstd_out[m] = rstd; }
    }
}

template <typename T, int TPR, int NCH>
__global__ __launch_bounds__(TPR ? TPR : 256) void norm_backward_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, const T *__restrict__ g,
                                                                       const float *__restrict__ mean_in, const float *__restrict__ rstd_in, int64_t M, int64_t C, int tpr_log, T *dx, int64_t lddx,
                                                                       float *part)
{
    constexpr int V = Width<T>::V, E = NCH * V;
    __shared__ float red[TPR ? 16 : 256 * (V + 1)];
    const int tpr = TPR ? TPR : 1 << tpr_log, lane = threadIdx.x & (tpr - 1), rows = TPR ? 1 : 256 >> tpr_log, sub = TPR ? 0 : threadIdx.x >> tpr_log;
    const float inv = 1.f / (float)C;
    float gg[NCH][V], dg[NCH][V], db[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int64_t col = ((int64_t)c * tpr + lane) * V;
        if (g) load_run(g, col, C, gg[c]);
#pragma unroll
        for (int j = 0; j < V; ++j) { dg[c][j] = db[c][j] = 0.f; if (!g) gg[c][j] = 1.f; }
    }
    for (int64_t m0 = (int64_t)blockIdx.x * rows; m0 < M; m0 += (int64_t)gridDim.x * rows) {
        const bool in = m0 + sub < M;
        const int64_t m = in ? m0 + sub : 0;
        float xv[NCH][V], t[NCH][V];
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int64_t col = ((int64_t)c * tpr + lane) * V;
            load_run(x + m * ldx, col, C, xv[c]);
            load_run(dy + m * lddy, col, C, t[c]);
        }
        const float mean = mean_in[m], rstd = rstd_in[m];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {                                // past the row's end dy is zero, and with it every sum
                const float xh = (xv[c][j] - mean) * rstd;
                if (in) { dg[c][j] += t[c][j] * xh; db[c][j] += t[c][j]; }
                t[c][j] *= gg[c][j];
                xv[c][j] = xh;
                s1 += t[c][j];
                s2 += t[c][j] * xh;
            }
        if (!dx) continue;
        s1 = row_sum<TPR>(s1, tpr, red) * inv;
        s2 = row_sum<TPR>(s2, tpr, red) * inv;
        if (!in) continue;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int64_t col = ((int64_t)c * tpr + lane) * V;
            if (col >= C) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) t[c][j] = rstd * (t[c][j] - s1 - xv[c][j] * s2);
            store_run(dx + m * lddx, col, C, t[c]);
        }
    }
    if (!part) return;
    float *out = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int64_t col = ((int64_t)c * tpr + lane) * V;
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
                    if (col + j < C) out[which * C + col + j] = v[j];
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
            load_run(x + m * ldx, c, C, xv);
            load_run(dy + m * lddy, c, C, t);
            if (g) load_run(g, c, C, gg);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = t[j] * (g ? gg[j] : 1.f);
                s1 += u;
                s2 += u * ((xv[j] - mean) * rstd);
            }
        }
        s1 = row_sum<1024>(s1, 1024, red) / (float)C;
        s2 = row_sum<1024>(s2, 1024, red) / (float)C;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
            load_run(x + m * ldx, c, C, xv);
            load_run(dy + m * lddy, c, C, t);
            if (g) load_run(g, c, C, gg);
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = rstd * (t[j] * (g ? gg[j] : 1.f) - s1 - (xv[j] - mean) * rstd * s2);
            store_run(dx + m * lddx, c, C, t);
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
    float dg[V] = {}, db[V] = {}, xv[V], t[V];
    for (int64_t m = (int64_t)blockIdx.x * rows_per; m < m1; ++m) {
        load_run(x + m * ldx, col, C, xv);
        load_run(dy + m * lddy, col, C, t);
        const float mean = mean_in[m], rstd = rstd_in[m];
#pragma unroll
        for (int j = 0; j < V; ++j) { dg[j] += t[j] * ((xv[j] - mean) * rstd); db[j] += t[j]; }
    }
    float *out = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (col + j < C) { out[col + j] = dg[j]; out[C + col + j] = db[j]; }
}

constexpr int64_t MAX_GRID = 1 << 20;                                   // the kernels walk rows beyond it
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a row of C values is spread: the smallest set of threads whose registers (two chunks each) hold it.
struct Spread { int tpr, nch, tpr_log; };                                // tpr = 0: too long
Spread spread_of(int64_t C, int dtype)
{
    const int V = dtype == AVC_F32 ? 4 : 8;
    const int64_t runs = cdiv(C, V);
    if (runs <= 128) {
        int lg = 3;
        while (lg < 6 && (1 << lg) < runs) ++lg;
        return Spread{1 << lg, runs > 64 ? 2 : 1, lg};
    }
    if (runs <= 512) return Spread{256, runs > 256 ? 2 : 1, 8};
    if (runs <= 2048) return Spread{1024, runs > 1024 ? 2 : 1, 10};
    return Spread{0, 0, 0};
}

// workgroups of the backward pass (strips of the column sums)
int64_t backward_blocks(int64_t M, int64_t C, int dtype)
{
    const Spread s = spread_of(C, dtype);
    if (s.tpr == 0) return std::max<int64_t>(1, std::min<int64_t>(cdiv(M, 16), 64));
    if (s.tpr <= 64) return std::max<int64_t>(1, std::min<int64_t>(cdiv(M, 256 / s.tpr), 1024));
    return std::max<int64_t>(1, std::min<int64_t>(M, s.tpr == 256 ? 1024 : 512));
}

template <typename T> int norm_forward(const void *x, int64_t ldx, const void *g, const void *b, float eps, int64_t M, int64_t C, int dtype, void *y, int64_t ldy, float *mean, float *rstd,
                                       hipStream_t s)
{
    const Spread sp = spread_of(C, dtype);
#define AVC_NORM(TPR, NCH, GRID, BLOCK)                                                                                                                          \
    hipLaunchKernelGGL((norm_kernel<T, TPR, NCH>), dim3((unsigned)std::min<int64_t>(GRID, MAX_GRID)), dim3(BLOCK), 0, s, (const T *)x, ldx, (const T *)g, (const T *)b, eps, M, C, sp.tpr_log, (T *)y, ldy, mean, rstd)
    if (sp.tpr == 0)
        hipLaunchKernelGGL(norm_long_kernel<T>, dim3((unsigned)std::min<int64_t>(M, MAX_GRID)), dim3(1024), 0, s, (const T *)x, ldx, (const T *)g, (const T *)b, eps, M, C, (T *)y, ldy, mean, rstd);
    else if (sp.tpr <= 64) {
        const int64_t grid = cdiv(M, 256 / sp.tpr);
        if (sp.nch == 1) AVC_NORM(0, 1, grid, 256); else AVC_NORM(0, 2, grid, 256);
    } else if (sp.tpr == 256) {
        if (sp.nch == 1) AVC_NORM(256, 1, M, 256); else AVC_NORM(256, 2, M, 256);
    } else {
        if (sp.nch == 1) AVC_NORM(1024, 1, M, 1024); else AVC_NORM(1024, 2, M, 1024);
    }
#undef AVC_NORM
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

template <typename T> int norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *g, const float *mean, const float *rstd, int64_t M, int64_t C, int dtype, void *dx,
                                        int64_t lddx, void *dg, void *db, float *part, hipStream_t s)
{
    const Spread sp = spread_of(C, dtype);
    const int64_t blocks = backward_blocks(M, C, dtype);
    float *p = dg || db ? part : nullptr;
#define AVC_NORM(TPR, NCH, BLOCK)                                                                                                                                \
    hipLaunchKernelGGL((norm_backward_kernel<T, TPR, NCH>), dim3((unsigned)blocks), dim3(BLOCK), 0, s, (const T *)dy, lddy, (const T *)x, ldx, (const T *)g, mean, rstd, M, C, sp.tpr_log,       \
                       (T *)dx, lddx, p)
    if (sp.tpr == 0) {
        if (dx && M) hipLaunchKernelGGL(norm_backward_long_kernel<T>, dim3((unsigned)std::min<int64_t>(M, MAX_GRID)), dim3(1024), 0, s, (const T *)dy, lddy, (const T *)x, ldx, (const T *)g, mean, rstd, M, C, (T *)dx, lddx);
        if (p)
            hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((unsigned)blocks, (unsigned)cdiv(C, 256 * Width<T>::V)), dim3(256), 0, s, (const T *)dy, lddy, (const T *)x, ldx, mean, rstd, M, C,
                               cdiv(M, blocks), p);
    } else if (sp.tpr <= 64) {
        if (sp.nch == 1) AVC_NORM(0, 1, 256); else AVC_NORM(0, 2, 256);
    } else if (sp.tpr == 256) {
        if (sp.nch == 1) AVC_NORM(256, 1, 256); else AVC_NORM(256, 2, 256);
    } else {
        if (sp.nch == 1) AVC_NORM(1024, 1, 1024); else AVC_NORM(1024, 2, 1024);
    }
#undef AVC_NORM
    AVC_HIP(hipGetLastError());
    if (p) return launch_colsum2(p, (int)blocks, C, dtype, dg, db, s);
    return AVC_OK;
}

}  // namespace

int layer_norm(const void *x, int64_t ldx, const void *g, const void *b, float eps, int64_t M, int64_t C, int dtype, void *y, int64_t ldy, float *mean, float *rstd, hipStream_t s)
{
    if (dtype == AVC_F32) return norm_forward<float>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
    if (dtype == AVC_BF16) return norm_forward<__bf16>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
    return norm_forward<_Float16>(x, ldx, g, b, eps, M, C, dtype, y, ldy, mean, rstd, s);
}

size_t layer_norm_backward_workspace(int64_t M, int64_t C, int dtype) { return sizeof(float) * 2 * (size_t)backward_blocks(M, C, dtype) * (size_t)C; }

int layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *g, const float *mean, const float *rstd, int64_t M, int64_t C, int dtype, void *dx, int64_t lddx,
                        void *dg, void *db, float *part, hipStream_t s)
{
    if (dtype == AVC_F32) return norm_backward<float>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
    if (dtype == AVC_BF16) return norm_backward<__bf16>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
    return norm_backward<_Float16>(dy, lddy, x, ldx, g, mean, rstd, M, C, dtype, dx, lddx, dg, db, part, s);
}

}}  // namespace avc::lin
