// Shared declarations of the dense-layer and layer-norm kernels (linear_tile.hip, linear.hip, layer_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/avcap.h"

namespace avc { namespace lin {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };
template <> struct Vec8<float> { typedef f32x8 type; };

// One operand of a product out(i, j) = sum_k P(i, k) Q(j, k).  `kc`: k is the contiguous axis and ld the distance of two rows; otherwise the rows are contiguous and ld is
// the distance of two k.  Elements, not bytes.  `padded`: 16-byte aligned rows whose last piece of 8 is there in full, zeros behind the end.
struct Operand { const void *p; int64_t ld; int kc; int padded = 0; };

struct Epilogue {
    const void *bias;                  // (N) or NULL
    const void *res; int64_t ldr;      // added after the activation, or NULL
    void *z; int64_t ldz;              // the value before the activation, or NULL
    int act; float slope;
};

struct TileArgs {
    Operand P, Q;
    int64_t M, N, K;
    void *out; int64_t ldo;
    Epilogue ep;
    float *partial;                    // splits > 1: (splits, M, N) float sums; reduce_kernel finishes
    int64_t kper;                      // k per split, a multiple of the k step
    int tiles_m, tiles_n, splits;
};

// tile shapes of tile_kernel
enum { TILE_BIG = 0, TILE_MID = 1, TILE_SMALL = 2 };
inline int tile_bm(int dtype, int tile) { return tile == TILE_BIG ? 256 : tile == TILE_MID ? 128 : 64; }
inline int tile_bn(int dtype, int tile) { return tile == TILE_BIG ? (dtype == AVC_F32 ? 128 : 256) : tile == TILE_MID ? 128 : 64; }
inline int tile_bk(int dtype) { return dtype == AVC_F32 ? 32 : 64; }

// the backward pass of a small layer in one launch: products of 64 x 64 tiles without splits (P of both is dy), and the column sums; tiles_m = 0 or db = NULL: not asked for
struct SmallArgs {
    TileArgs dx, dw;
    const void *dy; int64_t lddy;
    const void *saved; int64_t ld_saved;
    int act; float slope;
    int64_t M, N;
    void *db;
};
int launch_small_f32(const SmallArgs &a, unsigned blocks, bool x_kc, hipStream_t s);
int launch_small_bf16(const SmallArgs &a, unsigned blocks, bool x_kc, hipStream_t s);
int launch_small_f16(const SmallArgs &a, unsigned blocks, bool x_kc, hipStream_t s);

int launch_tile_f32(const TileArgs &a, int tile, hipStream_t s);
int launch_tile_bf16(const TileArgs &a, int tile, hipStream_t s);
int launch_tile_f16(const TileArgs &a, int tile, hipStream_t s);

// linear.hip
size_t forward_workspace(int64_t M, int64_t N, int64_t K, int dtype, bool x_kc);
size_t backward_workspace(int64_t M, int64_t N, int64_t K, int dtype);
int forward(const Operand &x, const void *w, int64_t ldw, int64_t M, int64_t N, int64_t K, int dtype, const Epilogue &e, void *y, int64_t ldy, void *ws, hipStream_t s);
int backward(const void *dy, int64_t lddy, const Operand &x, const void *w, int64_t ldw, const void *z, int64_t ldz, int act, float slope, int64_t M, int64_t N, int64_t K, int dtype,
             void *dx, void *dw, void *db, void *ws, hipStream_t s);
// out(c) and out2(c) = the sums over the strips of part[strip][2 C]
int launch_colsum2(const float *part, int strips, int64_t C, int dtype, void *out, void *out2, hipStream_t s);
// layer_norm.hip
int layer_norm(const void *x, int64_t ldx, const void *g, const void *b, float eps, int64_t M, int64_t C, int dtype, void *y, int64_t ldy, float *mean, float *rstd, hipStream_t s);
size_t layer_norm_backward_workspace(int64_t M, int64_t C, int dtype);
int layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *g, const float *mean, const float *rstd, int64_t M, int64_t C, int dtype, void *dx, int64_t lddx,
                        void *dg, void *db, float *part, hipStream_t s);

// x[j] <- x[j + s], zeros from the top; s = 0 .. 8
__device__ __forceinline__ void shift_down(f32x8 &x, int s)
{
#pragma unroll
    for (int b = 8; b >= 1; b >>= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s & b ? (j + b < 8 ? x[j + b < 8 ? j + b : j] : 0.f) : x[j];
}
__device__ __forceinline__ void shift_down(f32x4 &x, int s)                              // s = 0 .. 4
{
#pragma unroll
    for (int b = 4; b >= 1; b >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s & b ? (j + b < 4 ? x[j + b < 4 ? j + b : j] : 0.f) : x[j];
}
template <typename X> __device__ __forceinline__ void shift_down(X &v, int s)             // 8 elements of 16 bits, two to a word
{
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 x = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int b = 4; b >= 1; b >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s & (2 * b) ? (j + b < 4 ? x[j + b < 4 ? j + b : j] : 0u) : x[j];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = s & 1 ? (j < 3 ? __builtin_amdgcn_alignbit(x[j < 3 ? j + 1 : 3], x[j], 16) : x[j] >> 16) : x[j];
    v = __builtin_bit_cast(X, x);
}

// ---- activations ------------------------------------------------------------------------------------------------------------------------------------------
// float32 throughout, from v_exp_f32 / v_rcp_f32: branch-free, so that an epilogue of tens of values per lane stays small.  For float32 tensors a few ulp each; for 16-bit ones
// (HALF) within 1e-6 of the value's scale, a hundredth of their rounding, in two thirds of the instructions (gelu on 16384 x 8192 outputs: 40 us of 980).
// e^x = 2^h 2^l with h = fl(x log2 e) and l what h misses (plus the constant's own tail): the argument's rounding would cost |x| 2^-24
__device__ __forceinline__ float exp_acc(float x)
{
    constexpr float L = 1.44269502162933349609375f, LT = 1.925963033500011e-8f;
    const float h = x * L, l = fmaf(x, L, -h) + x * LT;
    const float e = __builtin_amdgcn_exp2f(h);
    return fabsf(h) < 200.f ? fmaf(e, l * 0.69314718055994531f, e) : e;     // beyond, e is 0 or inf and l may be NaN
}
__device__ __forceinline__ float rcp(float x) { return __builtin_amdgcn_rcpf(x); }

template <bool HALF> __device__ __forceinline__ float exp_of(float x) { return HALF ? __builtin_amdgcn_exp2f(x * 1.44269504f) : exp_acc(x); }

// log(1 + t), t in [0, 1]: 2 atanh(s), s = t / (2 + t) <= 1/3, seven terms of the odd series (the next is below 2^-25 of the sum)
__device__ __forceinline__ float log1p_unit(float t)
{
    const float s = t * rcp(2.f + t), q = s * s;
    float p = 1.f / 13.f;
    p = fmaf(p, q, 1.f / 11.f); p = fmaf(p, q, 1.f / 9.f); p = fmaf(p, q, 1.f / 7.f); p = fmaf(p, q, 1.f / 5.f); p = fmaf(p, q, 1.f / 3.f);
    return 2.f * fmaf(s * q, p, s);
}

// 1 - Phi(|z|) = erfc(|z| / sqrt 2) / 2 = e^(-z^2/2) t P(t), t = 1 / (1 + u / 2), u = |z| / sqrt 2.  P: least-maximum fit of erfc(u) e^(u^2) / (2 t) on 0 <= u <= 10 (relative error
// 4e-8, 3e-7 as evaluated in float32; HALF: two degrees less, 1.4e-6).  `e` receives e^(-z^2/2).
template <bool HALF> __device__ __forceinline__ float normal_tail(float z, float &e)
{
    const float t = rcp(fmaf(fabsf(z), 0.35355339059327379f, 1.f));
    if constexpr (HALF) {
        e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
        float p = 0.04411286488f;
        p = fmaf(p, t, -0.1784067303f); p = fmaf(p, t, 0.1946648061f); p = fmaf(p, t, 0.0189083051f); p = fmaf(p, t, 0.1407656819f); p = fmaf(p, t, 0.1387885064f);
        p = fmaf(p, t, 0.1411658973f);
        return e * t * p;
    }
    // the exponent in two parts, as exp_acc takes it, with what the square's rounding misses: rounded to one part it would cost z^2 / 2 steps
    constexpr float L = -0.721347510814666748046875f, LT = -9.62981516750005e-9f;
    const float q = z * z, h = q * L, l = fmaf(q, L, -h) + fmaf(q, LT, fmaf(z, z, -q) * L), x = __builtin_amdgcn_exp2f(h);
    e = q < 200.f ? fmaf(x, l * 0.69314718055994531f, x) : 0.f;             // below float32's range from 175 on
    float p = -0.0295328330f;
    p = fmaf(p, t, 0.1422793418f); p = fmaf(p, t, -0.2435828894f); p = fmaf(p, t, 0.1390137970f); p = fmaf(p, t, -0.0132990004f);
    p = fmaf(p, t, 0.1013374850f); p = fmaf(p, t, 0.1215534136f); p = fmaf(p, t, 0.1411874443f); p = fmaf(p, t, 0.1410432160f);
    return e * t * p;
}

template <bool HALF> __device__ __forceinline__ float tanh_of(float z)
{
    const float a = fabsf(z), t = exp_of<HALF>(-2.f * a), far = (1.f - t) * rcp(1.f + t), q = z * z;
    float p = -1382.f / 155925.f;                                            // the odd series where 1 - t would cancel
    p = fmaf(p, q, 62.f / 2835.f); p = fmaf(p, q, -17.f / 315.f); p = fmaf(p, q, 2.f / 15.f); p = fmaf(p, q, -1.f / 3.f);
    return a < 0.3f ? fmaf(z * q, p, z) : copysignf(far, z);
}

template <bool HALF> __device__ __forceinline__ float softplus_of(float z) { return z > 20.f ? z : fmaxf(z, 0.f) + log1p_unit(exp_of<HALF>(-fabsf(z))); }
// 1 / (1 + e^-z) and its complement, both without cancellation
template <bool HALF> __device__ __forceinline__ float sigmoid_of(float z, float &rest)
{
    const float e = exp_of<HALF>(-fabsf(z)), r = rcp(1.f + e);
    rest = z >= 0.f ? e * r : r;
    return z >= 0.f ? r : (z < 0.f ? e * r : z);
}

// v[j] = act(v[j]); the choice is uniform over the launch
template <bool HALF, int V> __device__ __forceinline__ void act_run(float (&v)[V], int act, float slope)
{
#define AVC_RUN(expr)                                                       \
    {                                                                       \
        _Pragma("unroll") for (int j = 0; j < V; ++j) { const float z = v[j]; float u; (void)u; v[j] = (expr); } \
        break;                                                              \
    }
    switch (act) {
    case AVC_ACT_RELU: AVC_RUN(z < 0.f ? 0.f : z)
    case AVC_ACT_LEAKY_RELU: AVC_RUN(z > 0.f ? z : slope * z)
    case AVC_ACT_SOFTPLUS: AVC_RUN(softplus_of<HALF>(z))
    case AVC_ACT_SIGMOID: AVC_RUN(sigmoid_of<HALF>(z, u))
    case AVC_ACT_TANH: AVC_RUN(tanh_of<HALF>(z))
    case AVC_ACT_GELU: AVC_RUN((u = normal_tail<HALF>(z, u), z * (z >= 0.f ? 1.f - u : u)))
    case AVC_ACT_SILU: AVC_RUN(z * sigmoid_of<HALF>(z, u))
    default: break;
    }
}

// +-infinity as a large finite value, for slopes that multiply z with what has long become 0: a float16 z beyond 65504 is stored as infinity while its y and gradient are finite
__device__ __forceinline__ float finite(float z) { return fabsf(z) == __builtin_inff() ? copysignf(1e15f, z) : z; }

// A kept z has the element type's size.  In bf16 calls it is float16, of the same size, where the slope depends on more than z's sign: |act''| z 2^-9 would reach the rounding that
// dz has anyway, 2^-12 does not (root mean square errors of dx, in those of an output rounded once: tanh 1.55 -> 1.41, silu 1.45 -> 1.41, the square root of 2 that two roundings
// make).  Below 2^-24 z counts as 0 and past 65504 as infinite, where no slope changes.
template <typename T> struct KeptZ { static __device__ __forceinline__ bool finer(int) { return false; } };
template <> struct KeptZ<__bf16> { static __device__ __forceinline__ bool finer(int act) { return act > AVC_ACT_LEAKY_RELU; } };
template <typename T> __device__ __forceinline__ T keep_z(float v, int act)
{
    if constexpr (sizeof(T) == 2)
        if (KeptZ<T>::finer(act)) return __builtin_bit_cast(T, (_Float16)v);
    return (T)v;
}
template <typename T, int V, typename Run> __device__ __forceinline__ void kept_z(const Run &s, float (&z)[V], int act)
{
    if constexpr (sizeof(T) == 2)
        if (KeptZ<T>::finer(act)) {
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = (float)__builtin_bit_cast(_Float16, (T)s[j]);
            return;
        }
#pragma unroll
    for (int j = 0; j < V; ++j) z[j] = (float)s[j];
}

// v[j] = act'(z[j]).  For the two piecewise linear ones the sign is all that counts, so that z may be the activation's value.
template <bool HALF, int V> __device__ __forceinline__ void slope_run(const float (&zs)[V], float (&v)[V], int act, float slope)
{
#undef AVC_RUN
#define AVC_RUN(expr)                                                       \
    {                                                                       \
        _Pragma("unroll") for (int j = 0; j < V; ++j) { const float z = zs[j]; float u, e; (void)u; (void)e; v[j] = (expr); } \
        break;                                                              \
    }
    switch (act) {
    case AVC_ACT_RELU: AVC_RUN(z <= 0.f ? 0.f : 1.f)
    case AVC_ACT_LEAKY_RELU: AVC_RUN(z > 0.f ? 1.f : slope)
    case AVC_ACT_SOFTPLUS: AVC_RUN(z > 20.f ? 1.f : sigmoid_of<HALF>(z, u))
    case AVC_ACT_SIGMOID: AVC_RUN((e = sigmoid_of<HALF>(z, u), e * u))
    case AVC_ACT_TANH: AVC_RUN((e = sigmoid_of<HALF>(2.f * z, u), 4.f * e * u))
    case AVC_ACT_GELU: AVC_RUN((u = normal_tail<HALF>(z, e), fmaf(finite(z) * 0.3989422804014327f, e, z >= 0.f ? 1.f - u : u)))
    case AVC_ACT_SILU: AVC_RUN((e = sigmoid_of<HALF>(z, u), e * fmaf(finite(z), u, 1.f)))
    default: AVC_RUN(1.f)
    }
#undef AVC_RUN
}

}}  // namespace avc::lin
