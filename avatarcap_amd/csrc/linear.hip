// The dense layer y = act(x W^T + b) + r and its gradients (include/avcap.h avc_linear, avc_linear_backward): which kernel serves which sizes, and the kernels around the
// tiled product (linear_tile.hip): few rows, few columns of channel-first points, sums of the splits, the activation's gradient with the bias gradient.
#include <algorithm>
#include "avcap_internal.h"
#include "linear.h"

namespace avc { namespace lin {

namespace {

// ---- one stored value with the epilogue applied ---------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void finish(float v, int64_t m, int64_t n, const Epilogue &e, T *out, int64_t ldo)
{
    if (e.bias) v += (float)((const T *)e.bias)[n];
    if (e.z) ((T *)e.z)[m * e.ldz + n] = keep_z<T>(v, e.act);
    float a[1] = {v};
    act_run<sizeof(T) == 2, 1>(a, e.act, e.slope);
    v = a[0];
    if (e.res) v += (float)((const T *)e.res)[m * e.ldr + n];
    out[m * ldo + n] = (T)v;
}

// ---- few rows: out(f, s) = sum_k F(f, k) S(s, k) with at most 16 * FB rows f against a long operand S that is read once -------------------------------------------
// A wave takes 16 rows of S and all rows of F on 16-row matrix instructions; the k axis is dealt in chunks of 128 bytes per row to the workgroup's waves, whose sums meet in
// LDS.  Lane (row l, quarter q) loads 32 adjacent bytes of its row, so a row's chunk is one 128-byte line.  One row of 1024 -> 4096 bf16: 5 us; 13 rows of 4096 -> 1024: 10 us.  float32 uses the f32 matrix instruction: the call is bound by the
// read of S, not by products.
template <typename T> struct FewArgs { const T *S; int64_t lds; const T *F; int64_t ldf; int64_t ns; int nf; int64_t K; int rows_are_f; Epilogue ep; T *out; int64_t ldo; int kw; };

template <typename T> struct Chunk { static constexpr int LANE = 32 / sizeof(T), K = 4 * LANE; typedef T vec __attribute__((ext_vector_type(LANE))); vec v; };

template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T *row, int64_t k)
{
    Chunk<T> c;
    __builtin_memcpy(&c.v, row + k, sizeof c.v);
    return c;
}
// the chunk that K ends in: values past the end are zero
template <typename T> __device__ __forceinline__ Chunk<T> load_tail(const T *row, int64_t k, int64_t K)
{
    Chunk<T> c;
#pragma unroll
    for (int j = 0; j < Chunk<T>::LANE; ++j) c.v[j] = row[min(k + j, K - 1)];
#pragma unroll
    for (int j = 0; j < Chunk<T>::LANE; ++j)
        if (k + j >= K) c.v[j] = (T)0.f;
    return c;
}

__device__ __forceinline__ f32x4 chunk_mfma(const Chunk<float> &a, const Chunk<float> &b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 chunk_mfma(const Chunk<__bf16> &a, const Chunk<__bf16> &b, f32x4 c)
{
    typedef bf16x8 h;
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(h(a.v.lo), h(b.v.lo), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(h(a.v.hi), h(b.v.hi), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 chunk_mfma(const Chunk<_Float16> &a, const Chunk<_Float16> &b, f32x4 c)
{
    typedef f16x8 h;
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(h(a.v.lo), h(b.v.lo), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(h(a.v.hi), h(b.v.hi), c, 0, 0, 0);
}

template <typename T, int FB> __global__ __launch_bounds__(1024) void few_kernel(const FewArgs<T> a)
{
    __shared__ f32x4 sums[16][FB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kslot = wave % a.kw, group = wave / a.kw, groups = (blockDim.x >> 6) / a.kw;
    const int l16 = lane & 15, q = lane >> 4;
    const int64_t s0 = ((int64_t)blockIdx.x * groups + group) * 16;
    // rows past the end repeat the last one: their results are not stored
    const T *srow = a.S + min(s0 + l16, a.ns - 1) * a.lds;
    const T *frow[FB];
#pragma unroll
    for (int b = 0; b < FB; ++b) frow[b] = a.F + (int64_t)min(16 * b + l16, a.nf - 1) * a.ldf;
    f32x4 acc[FB];
#pragma unroll
    for (int b = 0; b < FB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int CK = Chunk<T>::K, U = 4 / FB;
    const int64_t stride = (int64_t)a.kw * CK, qk = q * Chunk<T>::LANE;
    int64_t k = (int64_t)kslot * CK;
    for (; k + (U - 1) * stride + CK <= a.K; k += U * stride) {        // U chunks of both operands on their way before the first is used
        Chunk<T> s[U], f[U][FB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = load_chunk(srow, k + u * stride + qk);
#pragma unroll
            for (int b = 0; b < FB; ++b) f[u][b] = load_chunk(frow[b], k + u * stride + qk);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int b = 0; b < FB; ++b) acc[b] = chunk_mfma(s[u], f[u][b], acc[b]);
    }
    for (; k + CK <= a.K; k += stride) {
        const Chunk<T> s = load_chunk(srow, k + qk);
#pragma unroll
        for (int b = 0; b < FB; ++b) acc[b] = chunk_mfma(s, load_chunk(frow[b], k + qk), acc[b]);
    }
    if (k < a.K) {
        const Chunk<T> s = load_tail(srow, k + qk, a.K);
#pragma unroll
        for (int b = 0; b < FB; ++b) acc[b] = chunk_mfma(s, load_tail(frow[b], k + qk, a.K), acc[b]);
    }
    if (a.kw > 1) {
#pragma unroll
        for (int b = 0; b < FB; ++b) sums[wave][b][lane] = acc[b];
        __syncthreads();
        if (kslot) return;
#pragma unroll
        for (int b = 0; b < FB; ++b)
            for (int w = 1; w < a.kw; ++w) acc[b] += sums[wave + w][b][lane];
    }
#pragma unroll
    for (int b = 0; b < FB; ++b) {
        const int f = min(16 * b + l16, a.nf - 1);
        float bias[4], res[4], v[4];
        int64_t m[4], n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {                                   // every load before the first store: the outputs may lie on the residual
            const int64_t s = min(s0 + 4 * q + j, a.ns - 1);
            m[j] = a.rows_are_f ? f : s;
            n[j] = a.rows_are_f ? s : f;
            bias[j] = a.ep.bias ? (float)((const T *)a.ep.bias)[n[j]] : 0.f;
            res[j] = a.ep.res ? (float)((const T *)a.ep.res)[m[j] * a.ep.ldr + n[j]] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = acc[b][j] + bias[j];
        const bool mine = 16 * b + l16 < a.nf;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (a.ep.z && mine && s0 + 4 * q + j < a.ns) ((T *)a.ep.z)[m[j] * a.ep.ldz + n[j]] = keep_z<T>(v[j], a.ep.act);
        act_run<sizeof(T) == 2, 4>(v, a.ep.act, a.ep.slope);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (mine && s0 + 4 * q + j < a.ns) a.out[m[j] * a.ldo + n[j]] = (T)(a.ep.res ? v[j] + res[j] : v[j]);
    }
}

// ---- few output columns of channel-first points: y(m, n) = act(sum_k x[k][m] w[n][k] + b) with the points contiguous, N <= NB -------------------------------------
// Bound by the read of x: lanes take adjacent points, the workgroup's four waves a quarter of k each, the weights come through LDS.  262144 x 128 float32 -> 1: 22 us, 6.1 TB/s.
template <typename T, int NB> __global__ __launch_bounds__(256) void narrow_kernel(const T *__restrict__ x, int64_t ldx, const T *__restrict__ w, int64_t ldw, int64_t M, int N, int64_t K,
                                                                                   const Epilogue e, T *out, int64_t ldo)
{
    constexpr int V = 4, KT = 256;                                       // points per lane, k per pass
    __shared__ float wk[KT][NB];
    __shared__ float part[3][64][V * NB + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m = ((int64_t)blockIdx.x * 64 + lane) * V;
    int64_t at[V];                                                      // M < V: one by one
#pragma unroll
    for (int j = 0; j < V; ++j) at[j] = min(m + j, M - 1);
    const bool full = M % V == 0;                                       // uniform
    const int64_t mc = min(m, M - V);
    float acc[NB][V] = {};
    for (int64_t kb = 0; kb < K; kb += KT) {
        const int kt = (int)min((int64_t)KT, K - kb);
        __syncthreads();
        for (int i = threadIdx.x; i < NB * KT; i += 256) {
            const int n = i / KT, k = i % KT;
            wk[k][n] = n < N && k < kt ? (float)w[n * ldw + kb + k] : 0.f;
        }
        __syncthreads();
        if (full) {
#pragma unroll 8
            for (int k = wave; k < kt; k += 4) {
                T v[V];
                __builtin_memcpy(v, x + (kb + k) * ldx + mc, sizeof v);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[n][j] = fmaf((float)v[j], wk[k][n], acc[n][j]);
            }
        } else {
#pragma unroll 4
            for (int k = wave; k < kt; k += 4) {
                const T *src = x + (kb + k) * ldx;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int j = 0; j < V; ++j) acc[n][j] = fmaf((float)src[at[j]], wk[k][n], acc[n][j]);
            }
        }
    }
    if (wave) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int j = 0; j < V; ++j) part[wave - 1][lane][n * V + j] = acc[n][j];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float v = (acc[n][j] + part[0][lane][n * V + j]) + (part[1][lane][n * V + j] + part[2][lane][n * V + j]);
            if (n < N && m + j < M) finish<T>(v, m + j, n, e, out, ldo);
        }
}

// ---- runs of 16 bytes, whatever the alignment and the row's length -----------------------------------------------------------------------------------------------
// The V values from column c on, zeros past the row's end.  A run that would pass the end is read further back, to end with the row, and shifted down: no lane branches
// around a load.  Rows shorter than a run (SHORT) are read value by value.
template <typename T> struct Run16 { static constexpr int V = 16 / sizeof(T); typedef T vec __attribute__((ext_vector_type(V))); };
template <typename T, bool SHORT> __device__ __forceinline__ typename Run16<T>::vec read_run(const T *row, int64_t c, int64_t C)
{
    constexpr int V = Run16<T>::V;
    typename Run16<T>::vec v;
    if constexpr (SHORT) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = row[min(c + j, C - 1)];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j >= C) v[j] = (T)0.f;
    } else {
        const int64_t at = min(c, C - V);
        __builtin_memcpy(&v, row + at, sizeof v);
        shift_down(v, (int)min(c - at, (int64_t)V));
    }
    return v;
}

// ---- the activation's gradient dz = dy act'(z), and the column sums of dz in the same pass -------------------------------------------------------------------------
// Lanes take V adjacent columns, `tx` lanes a row, 256 / tx rows at a time; every workgroup walks a strip of rows and leaves its column sums in part[strip][N] (float32, a
// fixed order), which colsum_kernel adds (a single strip's sums are the bias gradient itself).  dz is rounded to the element type: it is the operand of two matrix products in
// that type.  Its rows are padded with zeros to whole runs, so that the products read it in aligned pieces.  Bound by HBM: 4.9 TB/s at 65536 x 256 float32 (36 us).
template <typename T, bool SHORT> __global__ __launch_bounds__(256) void dact_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ z, int64_t ldz, int act, float slope, int64_t M,
                                                                                    int64_t N, int64_t rows_per, int tx, T *__restrict__ dz, int64_t lddz, float *__restrict__ part,
                                                                                    T *__restrict__ db)
{
    constexpr int V = Run16<T>::V;
    typedef typename Run16<T>::vec vec;
    const int lx = threadIdx.x % tx, ly = threadIdx.x / tx, ty = 256 / tx;
    const int64_t n = ((int64_t)blockIdx.y * tx + lx) * V, m1 = min(M, ((int64_t)blockIdx.x + 1) * rows_per);
    float sum[V] = {};
    if (n < N) {
#pragma unroll 2
        for (int64_t m = blockIdx.x * rows_per + ly; m < m1; m += ty) {
            const vec g = read_run<T, SHORT>(dy + m * lddy, n, N);
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (float)g[j];
            if (z) {
                const vec s = read_run<T, SHORT>(z + m * ldz, n, N);
                float zs[V], sl[V];
                kept_z<T, V>(s, zs, act);
                slope_run<sizeof(T) == 2, V>(zs, sl, act, slope);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] *= sl[j];
            }
            if (dz) {
                vec o;
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = (T)v[j];
                *reinterpret_cast<vec *>(dz + m * lddz + n) = o;
                if (V < 8 && n + V >= N && n + V < lddz) *reinterpret_cast<vec *>(dz + m * lddz + n + V) = vec(0);      // float32: rows of 8, runs of 4
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += v[j];
        }
    }
    if (!part && !db) return;
    __shared__ float red[256][V + 1];
#pragma unroll
    for (int j = 0; j < V; ++j) red[threadIdx.x][j] = sum[j];
    __syncthreads();
    if (ly || n >= N) return;
    for (int y = 1; y < ty; ++y)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += red[y * tx + lx][j];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (n + j >= N) continue;
        if (db) db[n + j] = (T)sum[j];
        else part[(int64_t)blockIdx.x * N + n + j] = sum[j];
    }
}

// ---- rows copied to 16-byte aligned ones, zeros behind their ends ----------------------------------------------------------------------------------------------------
template <typename T, bool SHORT> __global__ __launch_bounds__(256) void pad_kernel(const T *__restrict__ src, int64_t ld, int64_t R, int64_t C, T *__restrict__ dst, int64_t ldd)
{
    constexpr int V = Run16<T>::V;
    const unsigned runs = (unsigned)(ldd / V);                          // below 2^22
    const int64_t total = R * runs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / runs, c = i % runs * V;
        *reinterpret_cast<typename Run16<T>::vec *>(dst + r * ldd + c) = read_run<T, SHORT>(src + r * ld, c, C);
    }
}

}  // namespace

// out(n) = sum over the strips of part[strip][n]: 32 columns and 32 runs of strips per workgroup, the runs' sums added in order.  Columns past N1 belong to the second output.
// A few hundred strips of a few hundred columns are too few bytes to matter; what counts is the chain of dependent loads, so 1024 threads share it (8 runs took 38 - 74 us for
// 1024 - 2048 strips).
template <typename T> __device__ __forceinline__ void column_sums(const float *__restrict__ part, int strips, int64_t N, int64_t N1, T *out, T *out2, unsigned block)
{
    __shared__ float red[32][33];
    const int lx = threadIdx.x & 31, ly = threadIdx.x >> 5;
    const int64_t n = (int64_t)block * 32 + lx;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int i = ly; i < strips; i += 32) s += part[(int64_t)i * N + n];
    }
    red[ly][lx] = s;
    __syncthreads();
    if (ly || n >= N) return;
#pragma unroll
    for (int y = 1; y < 32; ++y) s += red[y][lx];
    if (n < N1) { if (out) out[n] = (T)s; }
    else if (out2) out2[n - N1] = (T)s;
}
template <typename T> __global__ __launch_bounds__(1024) void colsum_kernel(const float *__restrict__ part, int strips, int64_t N, int64_t N1, T *out, T *out2)
{
    column_sums<T>(part, strips, N, N1, out, out2, blockIdx.x);
}

// ---- sums of the splits, added in order: four adjacent outputs per thread where there are many (24 -> 12 us for 2 x 2048 x 2048), one where there are few (128 x 256 x 256: 11 us,
// 23 us with four).  The workgroups past `blocks` take the bias gradient's column sums along, a launch saved.
constexpr int64_t SMALL_REDUCE = 1 << 20;
template <typename T> __global__ __launch_bounds__(1024) void reduce_kernel(const float *__restrict__ part, int splits, int64_t M, int64_t N, T *out, int64_t ldo, const Epilogue e, unsigned blocks,
                                                                            const float *__restrict__ strip_part, int strips, int64_t columns, T *sums)
{
    if (blockIdx.x >= blocks) {
        column_sums<T>(strip_part, strips, columns, columns, sums, (T *)nullptr, blockIdx.x - blocks);
        return;
    }
    const int64_t total = M * N, stride = (int64_t)blocks * 1024;
    if (total < SMALL_REDUCE || N % 4) {
        for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < total; i += stride) {
            float v = 0.f;
#pragma unroll 8
            for (int s = 0; s < splits; ++s) v += part[s * total + i];
            finish<T>(v, i / N, i % N, e, out, ldo);
        }
        return;
    }
    const bool small = total <= 0xffffffffll;                           // uniform; a 64-bit division costs more than the loads
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    for (int64_t i = 4 * ((int64_t)blockIdx.x * 1024 + threadIdx.x); i < total; i += 4 * stride) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int s = 0; s < splits; ++s) a += *reinterpret_cast<const f32x4 *>(part + s * total + i);
        const int64_t m = small ? (int64_t)((unsigned)i / (unsigned)N) : i / N, n = i - m * N;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j] + (e.bias ? (float)((const T *)e.bias)[n + j] : 0.f);
        vec o;
        if (e.z) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = keep_z<T>(v[j], e.act);
            *reinterpret_cast<loose *>((T *)e.z + m * e.ldz + n) = o;
        }
        act_run<sizeof(T) == 2, 4>(v, e.act, e.slope);
        if (e.res) {
            const vec r = *reinterpret_cast<const loose *>((const T *)e.res + m * e.ldr + n);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += (float)r[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (T)v[j];
        *reinterpret_cast<loose *>(out + m * ldo + n) = o;
    }
}

static int launch_columns(const float *part, int strips, int64_t N, int64_t N1, int dtype, void *out, void *out2, hipStream_t s)
{
    const dim3 grid((unsigned)((N + 31) / 32));
    if (dtype == AVC_F32) hipLaunchKernelGGL(colsum_kernel<float>, grid, dim3(1024), 0, s, part, strips, N, N1, (float *)out, (float *)out2);
    else if (dtype == AVC_BF16) hipLaunchKernelGGL(colsum_kernel<__bf16>, grid, dim3(1024), 0, s, part, strips, N, N1, (__bf16 *)out, (__bf16 *)out2);
    else hipLaunchKernelGGL(colsum_kernel<_Float16>, grid, dim3(1024), 0, s, part, strips, N, N1, (_Float16 *)out, (_Float16 *)out2);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}
int launch_colsum2(const float *part, int strips, int64_t C, int dtype, void *out, void *out2, hipStream_t s) { return launch_columns(part, strips, 2 * C, C, dtype, out, out2, s); }

namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int esize(int dtype) { return dtype == AVC_F32 ? 4 : 2; }
inline int64_t ceil8(int64_t n) { return (n + 7) & ~(int64_t)7; }

// ---- which tile, how many splits: from the sizes alone, so that the workspace can be asked for in advance -----------------------------------------------------------
// The time of a launch is estimated for every tile shape and a ladder of splits, and the least taken.  With W workgroups on the fullest CU, `occ` of them at a time, and S steps of
// k each:   launch + max(ceil(W / occ) (S lone_step + lone), W (S step + rest)) + the splits' sums written, read and reduced.
// `lone_*` is a workgroup's own latency, `step` / `rest` its share of a busy CU (matrix rate; writing the tile out).  Constants in us, fitted to 1020 timed launches of 17 shapes
// (64 .. 262144 rows, 64 .. 4096 columns and k, all three products): the choice came out 2 % slower than the best of all tiles and splits in the mean, 44 % at worst (2048 x 2048
// -> 512 bf16, 19 us for 13).
struct TileCost { int occ; double lone_step, lone, step, rest; };
constexpr TileCost COST_16[3] = {{1, 1.28, 8.3, 0.91, 0.0}, {2, 0.76, 2.8, 0.43, 3.0}, {5, 0.52, 0.0, 0.18, 1.0}};
constexpr TileCost COST_F32[3] = {{1, 2.74, 4.3, 0.00, 10.9}, {3, 2.82, 2.4, 1.60, 2.5}, {3, 0.90, 1.7, 0.57, 1.0}};
constexpr int SPLITS[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};

struct Plan { int tile, tiles_m, tiles_n, splits; int64_t kper; double us; };

Plan plan_tiles(int64_t M, int64_t N, int64_t K, int dtype)
{
    const int bk = tile_bk(dtype);
    Plan best{};
    double least = 0;
    for (int tile = TILE_BIG; tile <= TILE_SMALL; ++tile) {
        const int64_t tm = cdiv(M, tile_bm(dtype, tile)), tn = cdiv(N, tile_bn(dtype, tile));
        const TileCost &c = (dtype == AVC_F32 ? COST_F32 : COST_16)[tile];
        for (int want : SPLITS) {
            if (want > 1 && (K < (int64_t)want * 2 * bk || (double)want * M * N > 1e8)) break;
            const int64_t kper = std::max<int64_t>(bk, cdiv(cdiv(K, want), bk) * bk), splits = std::max<int64_t>(1, cdiv(K, kper)), W = cdiv(tm * tn * splits, 256);
            const double S = (double)cdiv(std::min(kper, K), bk);
            double us = std::max((double)cdiv(W, c.occ) * (S * c.lone_step + c.lone), (double)W * (S * c.step + c.rest));
            if (splits > 1) us += 3 + 8e-6 / 5 * (double)splits * M * N;
            if (!best.splits || us < least) {
                least = us;
                best = Plan{tile, (int)tm, (int)tn, (int)splits, kper, us};
            }
        }
    }
    return best;
}
size_t partial_bytes(const Plan &p, int64_t M, int64_t N) { return p.splits > 1 ? sizeof(float) * (size_t)p.splits * (size_t)M * (size_t)N : 0; }

// A large product is cut where whole tiles or whole rounds of tiles end, if a main part of (rows, cols) and the strips below and to the right of it, each with the tile and splits
// that suit it, come out cheaper than one launch whose last round or last row and column of tiles is mostly empty: 65537 rows of 545 -> 256 float32 values need 514 tiles, three
// rounds of 256 for two rounds' work (171 us; cut at 65536, 138 us).
struct Cut { int64_t rows, cols; Plan main, below, right; };
Cut plan_cut(int64_t M, int64_t N, int64_t K, int dtype)
{
    Cut best{M, N, plan_tiles(M, N, K, dtype), Plan{}, Plan{}};
    double least = best.main.us;
    const int64_t bm = tile_bm(dtype, TILE_BIG), bn = tile_bn(dtype, TILE_BIG);
    if (least < 40) return best;                                        // the strips are launches of their own
    for (int64_t cols : {N, N / bn * bn}) {
        if (cols < 1) continue;
        const int64_t tn = cdiv(cols, bn), rounds = M / bm * tn / 256;
        for (int64_t rows : {M, M / bm * bm, rounds >= 1 && rounds <= 16 ? rounds * 256 / tn * bm : (int64_t)0}) {
            if (rows < 1 || rows > M || (rows == M && cols == N)) continue;
            Cut c{rows, cols, plan_tiles(rows, cols, K, dtype), Plan{}, Plan{}};
            if (c.main.splits > 1) continue;
            double us = c.main.us;
            if (rows < M) us += (c.below = plan_tiles(M - rows, cols, K, dtype)).us + 3;
            if (cols < N) us += (c.right = plan_tiles(M, N - cols, K, dtype)).us + 3;
            if (us < least) {
                least = us;
                best = c;
            }
        }
    }
    return best;
}
constexpr int64_t MOST_ROWS = (int64_t)1 << 26;                          // per launch; products of more rows are cut into blocks of this many
size_t product_bytes(int64_t M, int64_t N, int64_t K, int dtype)
{
    if (M > MOST_ROWS) return std::max(product_bytes(MOST_ROWS, N, K, dtype), M % MOST_ROWS ? product_bytes(M % MOST_ROWS, N, K, dtype) : 0);
    const Cut c = plan_cut(M, N, K, dtype);
    return std::max(partial_bytes(c.main, c.rows, c.cols),
                    std::max(c.rows < M ? partial_bytes(c.below, M - c.rows, c.cols) : 0, c.cols < N ? partial_bytes(c.right, M, N - c.cols) : 0));
}

// lanes that share a row in the activation-gradient pass
int lanes_for(int64_t N, int v)
{
    int tx = 1;
    while (tx < 256 && (int64_t)tx * v < N) tx *= 2;
    return tx;
}
// its strips of rows: eight rows per lane, and no more strips than fill the chip
int64_t strips_for(int64_t M, int64_t N, int dtype)
{
    const int v = 16 / esize(dtype), tx = lanes_for(N, v);
    return std::max<int64_t>(1, std::min<int64_t>(cdiv(M, 8 * (256 / tx)), std::max<int64_t>(1, 2048 / cdiv(N, (int64_t)tx * v))));
}

inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
// column sums that wait for a launch to join: out = NULL once they have
struct Sums { const float *part; int strips; int64_t N; void *out; };

template <typename T> int launch_reduce(const float *part, int splits, int64_t M, int64_t N, void *out, int64_t ldo, const Epilogue &e, Sums *sums, hipStream_t s)
{
    const unsigned blocks = (unsigned)std::min<int64_t>(cdiv(M * N, M * N < SMALL_REDUCE || N % 4 ? 1024 : 4096), 8192), more = sums && sums->out ? (unsigned)cdiv(sums->N, 32) : 0;
    hipLaunchKernelGGL(reduce_kernel<T>, dim3(blocks + more), dim3(1024), 0, s, part, splits, M, N, (T *)out, ldo, e, blocks, more ? sums->part : nullptr, more ? sums->strips : 0,
                       more ? sums->N : 0, more ? (T *)sums->out : nullptr);
    AVC_HIP(hipGetLastError());
    if (more) sums->out = nullptr;
    return AVC_OK;
}

int product_part(const Operand &P, const Operand &Q, int64_t M, int64_t N, int64_t K, int dtype, const Epilogue &e, void *out, int64_t ldo, void *ws, const Plan &p, hipStream_t s,
                 Sums *sums = nullptr)
{
    AVC_REQUIRE((int64_t)p.tiles_m * p.tiles_n * p.splits < (1 << 22), AVC_ERR_ARG, "avc_linear: %lld x %lld outputs are more than one launch covers", (long long)M, (long long)N);
    TileArgs a{P, Q, M, N, K, out, ldo, e, (float *)ws, p.kper, p.tiles_m, p.tiles_n, p.splits};
    const int rc = dtype == AVC_F32 ? launch_tile_f32(a, p.tile, s) : dtype == AVC_BF16 ? launch_tile_bf16(a, p.tile, s) : launch_tile_f16(a, p.tile, s);
    if (rc != AVC_OK || p.splits == 1) return rc;
    if (dtype == AVC_F32) return launch_reduce<float>(a.partial, p.splits, M, N, out, ldo, e, sums, s);
    if (dtype == AVC_BF16) return launch_reduce<__bf16>(a.partial, p.splits, M, N, out, ldo, e, sums, s);
    return launch_reduce<_Float16>(a.partial, p.splits, M, N, out, ldo, e, sums, s);
}

inline const void *ahead(const void *p, int64_t elements, int dtype) { return p ? (const char *)p + elements * esize(dtype) : nullptr; }

// the operand, and the epilogue, from row m / column n of the output on
Operand from(const Operand &o, int64_t row, int dtype) { return Operand{ahead(o.p, o.kc ? row * o.ld : row, dtype), o.ld, o.kc, o.padded}; }
Epilogue from(const Epilogue &e, int64_t m, int64_t n, int dtype)
{
    return Epilogue{ahead(e.bias, n, dtype), ahead(e.res, m * e.ldr + n, dtype), e.ldr, (void *)ahead(e.z, m * e.ldz + n, dtype), e.ldz, e.act, e.slope};
}

int product(const Operand &P, const Operand &Q, int64_t M, int64_t N, int64_t K, int dtype, const Epilogue &e, void *out, int64_t ldo, void *ws, hipStream_t s, Sums *sums = nullptr)
{
    if (M > MOST_ROWS) {
        for (int64_t m = 0; m < M; m += MOST_ROWS) {
            const int rc = product(from(P, m, dtype), Q, std::min(MOST_ROWS, M - m), N, K, dtype, from(e, m, 0, dtype), (void *)ahead(out, m * ldo, dtype), ldo, ws, s);
            if (rc != AVC_OK) return rc;
        }
        return AVC_OK;
    }
    const Cut c = plan_cut(M, N, K, dtype);
    if (c.rows < M) {
        const int rc = product_part(from(P, c.rows, dtype), Q, M - c.rows, c.cols, K, dtype, from(e, c.rows, 0, dtype), (void *)ahead(out, c.rows * ldo, dtype), ldo, ws, c.below, s);
        if (rc != AVC_OK) return rc;
    }
    if (c.cols < N) {
        const int rc = product_part(P, from(Q, c.cols, dtype), M, N - c.cols, K, dtype, from(e, 0, c.cols, dtype), (void *)ahead(out, c.cols, dtype), ldo, ws, c.right, s);
        if (rc != AVC_OK) return rc;
    }
    return product_part(P, Q, c.rows, c.cols, K, dtype, e, out, ldo, ws, c.main, s, sums);
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------------------------------------------
constexpr int FEW = 32;
template <typename T> int launch_few(const void *S, int64_t lds, int64_t ns, const void *F, int64_t ldf, int nf, int64_t K, int rows_are_f, const Epilogue &e, void *out, int64_t ldo, hipStream_t s)
{
    FewArgs<T> a{(const T *)S, lds, (const T *)F, ldf, ns, nf, K, rows_are_f, e, (T *)out, ldo, 1};
    const int64_t groups = cdiv(ns, 16), chunks = cdiv(K, Chunk<T>::K);
    // waves that share a group's k axis: as many as bring the launch to ~4096 waves, no more than there are chunks
    while (a.kw < 16 && groups * a.kw < 4096 && a.kw * 2 <= chunks) a.kw *= 2;
    const int waves = std::max(4, a.kw), per = waves / a.kw;
    AVC_REQUIRE(cdiv(groups, per) <= (1 << 22), AVC_ERR_ARG, "avc_linear: %lld rows are more than one launch covers", (long long)ns);
    const dim3 grid((unsigned)cdiv(groups, per)), block(64 * waves);
    if (nf <= 16) hipLaunchKernelGGL((few_kernel<T, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((few_kernel<T, 2>), grid, block, 0, s, a);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

template <typename T> int launch_narrow(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t M, int N, int64_t K, const Epilogue &e, void *out, int64_t ldo, hipStream_t s)
{
    const dim3 grid((unsigned)cdiv(M, 256));
    if (N == 1) hipLaunchKernelGGL((narrow_kernel<T, 1>), grid, dim3(256), 0, s, (const T *)x, ldx, (const T *)w, ldw, M, N, K, e, (T *)out, ldo);
    else hipLaunchKernelGGL((narrow_kernel<T, 4>), grid, dim3(256), 0, s, (const T *)x, ldx, (const T *)w, ldw, M, N, K, e, (T *)out, ldo);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

#define AVC_BY_TYPE(dtype, call)                                         \
    ((dtype) == AVC_F32 ? call<float> : (dtype) == AVC_BF16 ? call<__bf16> : call<_Float16>)

enum Route { ROUTE_TILE, ROUTE_FEW_ROWS, ROUTE_FEW_COLS, ROUTE_NARROW };
Route route(int64_t M, int64_t N, bool x_kc)
{
    if (x_kc && M <= FEW) return ROUTE_FEW_ROWS;
    if (x_kc && N <= 16) return ROUTE_FEW_COLS;
    if (!x_kc && N <= 4) return ROUTE_NARROW;
    return ROUTE_TILE;
}

template <typename T> int launch_dact(const void *dy, int64_t lddy, const void *z, int64_t ldz, int act, float slope, int64_t M, int64_t N, void *dz, int64_t lddz, float *part, void *db,
                                      int64_t strips, hipStream_t s)
{
    constexpr int V = Run16<T>::V;
    const int tx = lanes_for(N, V);
    const dim3 grid((unsigned)strips, (unsigned)cdiv(N, (int64_t)tx * V));
    const int64_t rows = cdiv(M, strips);
    if (N >= V) hipLaunchKernelGGL((dact_kernel<T, false>), grid, dim3(256), 0, s, (const T *)dy, lddy, (const T *)z, ldz, act, slope, M, N, rows, tx, (T *)dz, lddz, part, (T *)db);
    else hipLaunchKernelGGL((dact_kernel<T, true>), grid, dim3(256), 0, s, (const T *)dy, lddy, (const T *)z, ldz, act, slope, M, N, rows, tx, (T *)dz, lddz, part, (T *)db);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

// rows (R, C) copied to `dst` with rows of ceil8(C)
template <typename T> int launch_pad_as(const Operand &o, int64_t R, int64_t C, void *dst, hipStream_t s)
{
    constexpr int V = Run16<T>::V;
    const int64_t ldd = ceil8(C), blocks = std::min<int64_t>(cdiv(R * (ldd / V), 256), 1 << 16);
    if (C >= V) hipLaunchKernelGGL((pad_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)o.p, o.ld, R, C, (T *)dst, ldd);
    else hipLaunchKernelGGL((pad_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)o.p, o.ld, R, C, (T *)dst, ldd);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}
int launch_pad(const Operand &o, int64_t R, int64_t C, int dtype, void *dst, hipStream_t s)          // 16 bits are copied as bits, whichever type they are
{
    return dtype == AVC_F32 ? launch_pad_as<float>(o, R, C, dst, s) : launch_pad_as<__bf16>(o, R, C, dst, s);
}

// 16-bit products whose operands' contiguous axes are no multiple of 8 cannot be read in direct pieces; staged through registers they take about twice as long (three times the weight
// gradient).  Where copying the operands to padded rows costs less than 0.6 of the product, they are copied: 8191 x 2047 -> 2047 bf16, forward 120 -> 89 us, weight gradient
// 292 -> 118 us.  Not for short calls (`least`, us): a host that cannot run ahead pays for every launch (16387 x 319 -> 256 float16 training: 126 us without copies, 132 with).
// float32 is staged in any case, but the workgroups at a ragged edge of rows that lie contiguously shift every piece they read and hold up the rest: worth 0.3 of the product there.
// `elements` are those copied, `copies` the launches.
bool worth_padding(double product_us, double least, int64_t elements, int copies, int dtype)
{
    return elements && product_us >= least && (double)elements * 2 * esize(dtype) / 4.5e6 + 3.0 * copies < (dtype == AVC_F32 ? 0.3 : 0.6) * product_us;
}

struct ForwardPad { bool x, w; size_t xb, wb, total; };
ForwardPad forward_pad(int64_t M, int64_t N, int64_t K, int dtype, bool x_kc)
{
    ForwardPad f{};
    f.x = x_kc ? dtype != AVC_F32 && K % 8 != 0 : M % 8 != 0;
    f.w = dtype != AVC_F32 && K % 8 != 0;
    const int64_t xe = x_kc ? M * ceil8(K) : K * ceil8(M), we = N * ceil8(K);
    if (!worth_padding(plan_cut(M, N, K, dtype).main.us, 30, (f.x ? xe : 0) + (f.w ? we : 0), f.x + f.w, dtype)) return ForwardPad{};
    f.xb = f.x ? align256((size_t)xe * esize(dtype)) : 0;
    f.wb = f.w ? align256((size_t)we * esize(dtype)) : 0;
    f.total = f.xb + f.wb;
    return f;
}

}  // namespace

size_t forward_workspace(int64_t M, int64_t N, int64_t K, int dtype, bool x_kc)
{
    return M && route(M, N, x_kc) == ROUTE_TILE ? forward_pad(M, N, K, dtype, x_kc).total + product_bytes(M, N, K, dtype) : 0;
}

// Layers whose gradients are no more tiles than the chip has CUs, with sums of at most eight steps: the launches cost more than the work (20.6 us of host time and three launches
// against 13.2 us and one for 16 x 24 -> 7), so one launch does it all, without workspace.  Longer sums are faster split over several workgroups (float32 gradients of 128 x 1024
// -> 1024 rows: 33 us here, 11 us split).
static bool small_backward(int64_t M, int64_t N, int64_t K, int dtype)
{
    const int64_t longest = 8 * tile_bk(dtype);
    return M >= 1 && M <= longest && N <= longest && cdiv(N, 64) * cdiv(K, 64) <= 256 && cdiv(M, 64) * cdiv(K, 64) <= 256;
}

// The backward pass's workspace: dz (padded rows), the strips' column sums, padded copies of x and w, the splits' sums.  pad_dy: dy has no activation to pass and is copied as dz.
struct BackwardSpace { size_t dz, strips, x, w, partial, total; bool pad_dy, pad_x, pad_w; };
static BackwardSpace backward_space(int64_t M, int64_t N, int64_t K, int dtype)
{
    BackwardSpace w{};
    if (small_backward(M, N, K, dtype)) return w;
    const int64_t lddz = ceil8(N);
    w.dz = align256((size_t)M * lddz * esize(dtype));
    w.strips = align256(sizeof(float) * (size_t)strips_for(M, N, dtype) * N);
    w.partial = product_bytes(N, K, M, dtype);
    if (M) w.partial = std::max(w.partial, product_bytes(M, K, N, dtype));
    if (M) {
        const double us = plan_cut(M, K, N, dtype).main.us + 2 * plan_cut(N, K, M, dtype).main.us;
        w.pad_dy = N % 8 != 0;
        w.pad_x = w.pad_w = K % 8 != 0;                                 // (channel-first x is padded along M; the larger of the two is reserved)
        const int64_t xe = std::max(M * ceil8(K), K * ceil8(M)), we = N * ceil8(K);
        if (!worth_padding(us, 60, (w.pad_dy ? M * ceil8(N) : 0) + (w.pad_x ? xe + we : 0), w.pad_dy + 2 * w.pad_x, dtype)) w.pad_dy = w.pad_x = w.pad_w = false;
        if (w.pad_x) { w.x = align256((size_t)xe * esize(dtype)); w.w = align256((size_t)we * esize(dtype)); }
    }
    w.total = w.dz + w.strips + w.x + w.w + w.partial;
    return w;
}
size_t backward_workspace(int64_t M, int64_t N, int64_t K, int dtype) { return backward_space(M, N, K, dtype).total; }

int forward(const Operand &x, const void *w, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype, const Epilogue &e, void *y, int64_t ldy, void *ws, hipStream_t s)
{
    switch (route(M, N, x.kc)) {
    case ROUTE_FEW_ROWS: return AVC_BY_TYPE(dtype, launch_few)(w, ldw, N, x.p, x.ld, (int)M, K, 1, e, y, ldy, s);
    case ROUTE_FEW_COLS: return AVC_BY_TYPE(dtype, launch_few)(x.p, x.ld, M, w, ldw, (int)N, K, 0, e, y, ldy, s);
    case ROUTE_NARROW: return AVC_BY_TYPE(dtype, launch_narrow)(x.p, x.ld, w, ldw, M, (int)N, K, e, y, ldy, s);
    default: break;
    }
    Operand P = x, Q{w, ldw, 1};
    const ForwardPad f = forward_pad(M, N, K, dtype, x.kc);
    char *space = (char *)ws;
    if (f.x) {
        const int rc = x.kc ? launch_pad(x, M, K, dtype, space, s) : launch_pad(x, K, M, dtype, space, s);
        if (rc != AVC_OK) return rc;
        P = Operand{space, x.kc ? ceil8(K) : ceil8(M), x.kc, 1};
    }
    if (f.w) {
        const int rc = launch_pad(Q, N, K, dtype, space + f.xb, s);
        if (rc != AVC_OK) return rc;
        Q = Operand{space + f.xb, ceil8(K), 1, 1};
    }
    return product(P, Q, M, N, K, dtype, e, y, ldy, space + f.total, s);
}

int backward(const void *dy, int64_t lddy, const Operand &x, const void *w, int64_t ldw, const void *z, int64_t ldz, int act, float slope, int64_t M, int64_t N, int64_t K, int dtype,
             void *dx, void *dw, void *db, void *ws, hipStream_t s)
{
    const Epilogue none{nullptr, nullptr, 0, nullptr, 0, AVC_ACT_NONE, 0.f};
    if (small_backward(M, N, K, dtype)) {
        SmallArgs a{};
        auto tiles = [](TileArgs &t, const Operand &P, const Operand &Q, int64_t m, int64_t n, int64_t k, void *out) {
            t = TileArgs{P, Q, m, n, k, out, n, Epilogue{nullptr, nullptr, 0, nullptr, 0, AVC_ACT_NONE, 0.f}, nullptr, k, (int)cdiv(m, 64), (int)cdiv(n, 64), 1};
        };
        if (dx) tiles(a.dx, Operand{dy, lddy, 1}, Operand{w, ldw, 0}, M, K, N, dx);
        if (dw) tiles(a.dw, Operand{dy, lddy, 0}, Operand{x.p, x.ld, x.kc ? 0 : 1}, N, K, M, dw);
        a.dy = dy; a.lddy = lddy; a.saved = z; a.ld_saved = ldz; a.act = act; a.slope = slope; a.M = M; a.N = N; a.db = db;
        const int64_t blocks = (int64_t)a.dx.tiles_m * a.dx.tiles_n + (int64_t)a.dw.tiles_m * a.dw.tiles_n + (db ? cdiv(N, 16) : 0);
        if (!blocks) return AVC_OK;
        return dtype == AVC_F32 ? launch_small_f32(a, (unsigned)blocks, x.kc, s) : dtype == AVC_BF16 ? launch_small_bf16(a, (unsigned)blocks, x.kc, s) : launch_small_f16(a, (unsigned)blocks, x.kc, s);
    }
    const BackwardSpace sp = backward_space(M, N, K, dtype);
    char *dz_buf = (char *)ws, *strips_buf = dz_buf + sp.dz, *x_buf = strips_buf + sp.strips, *w_buf = x_buf + sp.x, *part = w_buf + sp.w;
    const bool active = act != AVC_ACT_NONE, through = active || sp.pad_dy;      // dz is dy itself, or goes through the pass below
    const int64_t lddz = through ? ceil8(N) : lddy;
    Sums sums{};
    if (through || db) {
        const int64_t strips = strips_for(M, N, dtype);
        const int rc = AVC_BY_TYPE(dtype, launch_dact)(dy, lddy, active ? z : nullptr, ldz, act, slope, M, N, through ? dz_buf : nullptr, lddz, db && strips > 1 ? (float *)strips_buf : nullptr,
                                                       strips == 1 ? db : nullptr, strips, s);
        if (rc != AVC_OK) return rc;
        if (db && strips > 1) sums = Sums{(const float *)strips_buf, (int)strips, N, db};
    }
    const void *dz = through ? dz_buf : dy;
    if (dx && M) {
        Operand Q{w, ldw, 0};
        if (sp.pad_w) {
            const int rc = launch_pad(Q, N, K, dtype, w_buf, s);
            if (rc != AVC_OK) return rc;
            Q = Operand{w_buf, ceil8(K), 0, 1};
        }
        const int rc = product(Operand{dz, lddz, 1, through}, Q, M, K, N, dtype, none, dx, K, part, s);
        if (rc != AVC_OK) return rc;
    }
    if (dw) {
        Operand Q{x.p, x.ld, x.kc ? 0 : 1};
        if (sp.pad_x && (x.kc || M % 8)) {
            const int rc = x.kc ? launch_pad(x, M, K, dtype, x_buf, s) : launch_pad(x, K, M, dtype, x_buf, s);
            if (rc != AVC_OK) return rc;
            Q = Operand{x_buf, x.kc ? ceil8(K) : ceil8(M), x.kc ? 0 : 1, 1};
        }
        const int rc = product(Operand{dz, lddz, 0, through}, Q, N, K, M, dtype, none, dw, K, part, s, &sums);
        if (rc != AVC_OK) return rc;
    }
    if (sums.out) return launch_columns(sums.part, sums.strips, N, N, dtype, db, nullptr, s);
    return AVC_OK;
}

}}  // namespace avc::lin
