// The dense layer's products (include/avcap.h avc_linear): out(i, j) = sum_k P(i, k) Q(j, k), either operand with k or its rows contiguous, bias / activation / residual in
// the epilogue.  Built once per element type (-DAVC_LIN_F32 / _BF16 / _F16).
//
//   forward        y  = x W^T      P = x  (k contiguous, or the points when x is channel-first)   Q = W   (k contiguous)
//   input gradient dx = dz W       P = dz (k contiguous)                                          Q = W   (rows contiguous)
//   weight gradient dW = dz^T x    P = dz (rows contiguous)                                       Q = x   (rows contiguous, or k when x is channel-first)
//
// One workgroup computes a BM x BN tile; every wave a (BM / WM) x (BN / WN) part of it in v_mfma_f32_16x16x32 accumulators.  Q's rows are the matrix instruction's rows, so a
// lane holds runs of 4 adjacent columns of one output row.  The epilogue passes them through the wave's own part of LDS, two fragment rows at a time: lanes then take 16 bytes of
// a row each, adjacent lanes adjacent pieces, and one copy of the activation code serves all of the tile.  bf16: 4096^3 in 105 us (1.3 PFLOP/s, where the board's power limit
// sets the clock); 65536 x 256 -> 256 in 22 us, bound by HBM.
//
// float32 runs on the same bf16 matrix instructions: x = h + m + l, three bf16 of 8 significant bits each (rounded to nearest, so the three hold all 24 bits exactly), and
// x w = hh + (hm + mh) + (hl + mm + lh) + terms below 2^-23 |x w| that float32's own products would round away.  Six products at the bf16 rate are faster than one at the f32
// matrix rate (4096^3: 672 us, 204 TFLOP/s; the f32 rate's own peak is 157).  The head is clamped to bf16's largest finite value, so that a value beyond it (and an infinity, which then travels in the tail) does not become inf - inf.
#include <atomic>
#include <type_traits>
#include "avcap_internal.h"
#include "linear.h"

namespace avc { namespace lin {

#if defined(AVC_LIN_F32)
typedef float elem_t;
#define AVC_LAUNCH launch_tile_f32
#define AVC_LAUNCH_SMALL launch_small_f32
#elif defined(AVC_LIN_F16)
typedef _Float16 elem_t;
#define AVC_LAUNCH launch_tile_f16
#define AVC_LAUNCH_SMALL launch_small_f16
#else
typedef __bf16 elem_t;
#define AVC_LAUNCH launch_tile_bf16
#define AVC_LAUNCH_SMALL launch_small_bf16
#endif

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr bool IS_F32 = std::is_same<elem_t, float>::value;
constexpr bool IS_F16 = std::is_same<elem_t, _Float16>::value;
constexpr int NP = IS_F32 ? 3 : 1;                 // 16-bit planes per operand in LDS
constexpr int BK = IS_F32 ? 32 : 64;               // k step
typedef typename Vec8<elem_t>::type elem8;
typedef typename std::conditional<IS_F16, f16x8, bf16x8>::type half8;        // what the matrix instruction takes

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c)
{
    if constexpr (IS_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// ---- LDS layout of one operand's BR x BK tile (16-bit elements, pieces of 16 bytes) ---------------------------------------------------------------------------
// k contiguous: row r holds its BK values in BK / 8 pieces; rows contiguous: row k holds the BR values of one k in BR / 8 pieces.  The pieces of a row are permuted by an XOR
// with a function of the row so that the lanes of a fragment read fall on different banks; the permutation is applied to the global address, because a direct load writes
// LDS in lane order.
template <int BR, bool KC> struct Tile {
    static constexpr int ROW_BYTES = KC ? BK * 2 : BR * 2;
    static constexpr int PIECES = ROW_BYTES / 16;                       // per row
    static constexpr int ROWS = KC ? BR : BK;
    static constexpr int BYTES = ROWS * ROW_BYTES;
    __device__ static __forceinline__ int swizzle(int row)
    {
        if constexpr (KC) {
            if (BK == 64) return (row >> 1) & 7;
            // 64-byte rows: a 16-byte read is served 16 lanes at a time, rows 0 - 3 and 12 - 15 of one quarter with rows 4 - 11 of the next, so four groups of four rows at two
            // pieces have to differ: 0 2 3 1 by group (0 1 2 3 met itself: 39 % of the LDS cycles were conflicts)
            const int g = (row >> 2) & 3, x = g ^ (g >> 1);
            return ((x & 1) << 1) | (x >> 1);
        }
        else return (((row & 3) | (((row >> 3) & 1) << 2)) << 1) & (PIECES - 1);
    }
    // byte of piece p of row `row`
    __device__ static __forceinline__ int at(int row, int p) { return row * ROW_BYTES + ((p ^ swizzle(row)) << 4); }

    // A wave's reads: fragment t holds the rows r0 + 16 t .., the lane's 8 values of k step ks.  Offsets are two numbers per lane and an XOR with constants; `x` is to be passed
    // through fresh() once per step, or the compiler keeps every fragment's address in a register of its own through the loop (and spills).
    struct Reader { unsigned row, x; };
    __device__ static __forceinline__ Reader reader(int r0, int lane)
    {
        const int l16 = lane & 15, q = lane >> 4;
        if constexpr (KC) return Reader{(unsigned)((r0 + l16) * ROW_BYTES), (unsigned)((q ^ swizzle(l16)) << 4)};
        // ds_read_b64_tr_b16: within 16 lanes, lane 4 a + c supplies the address of 4 adjacent values of k row a, and lane i receives the 4 k values of column i
        const int a = l16 >> 2, c = l16 & 3, k = 8 * q + a;             // (the swizzle does not look at bit 2 of k)
        return Reader{(unsigned)(k * ROW_BYTES + ((c & 1) << 3)), (unsigned)(((r0 >> 3) + (c >> 1)) ^ swizzle(k)) << 4};
    }
    __device__ static __forceinline__ Reader fresh(Reader r)
    {
        asm volatile("" : "+v"(r.x));
        return r;
    }
    __device__ static __forceinline__ half8 fragment(const char *base, const Reader &r, int t, int ks)
    {
        if constexpr (KC) {
            return *reinterpret_cast<const half8 *>(base + ((r.x ^ (unsigned)(ks * 64)) + r.row) + t * 16 * ROW_BYTES);
        } else {
            const char *p = base + ((r.x ^ (unsigned)(t * 32)) + r.row) + ks * 32 * ROW_BYTES;
            const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p), v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * ROW_BYTES));
            const s16x8 w = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
            return __builtin_bit_cast(half8, w);
        }
    }
};

// ---- global -> LDS ------------------------------------------------------------------------------------------------------------------------------------------
// (a) direct: 16-byte pieces straight into LDS.  The host has checked that every piece lies wholly inside or outside of the operand (or of its padding) and is 16-byte aligned; pieces outside get an
//     offset past the buffer's end, for which the hardware writes zeros.
constexpr unsigned OUTSIDE = 0x80000000u;

template <int BR, bool KC, int NW> struct Direct {
    typedef Tile<BR, KC> L;
    static constexpr int N = L::BYTES / 1024 / NW;                      // loads per wave
    static constexpr int RPL = 1024 / L::ROW_BYTES;                     // rows per load
    static_assert(N >= 1 && L::BYTES % (1024 * NW) == 0 && RPL >= 1, "tile does not divide into the waves' loads");
    unsigned voff[N];
    const char *base;
    int64_t step_bytes, ld_bytes, left;                                 // bytes from `base` to the operand's end
    __device__ __forceinline__ void init(const Operand &o, int64_t row0, int64_t rows, int64_t k0, int64_t K, int wave, int lane)
    {
        ld_bytes = o.ld * 2;
        // (the contiguous axis is a multiple of 8, or padded to one)
        const int64_t first = KC ? row0 * o.ld + k0 : k0 * o.ld + row0, last = KC ? (rows - 1) * o.ld + ((K + 7) & ~(int64_t)7) : (K - 1) * o.ld + ((rows + 7) & ~(int64_t)7);
        base = (const char *)o.p + first * 2;
        left = (last - first) * 2;
        step_bytes = KC ? BK * 2 : BK * ld_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (i * NW + wave) * RPL + lane / L::PIECES, p = (lane % L::PIECES) ^ L::swizzle(r);
            voff[i] = (unsigned)(r * ld_bytes + p * 16);
            if (KC ? row0 + r >= rows : row0 + p * 8 >= rows) voff[i] = OUTSIDE;
        }
    }
    // the pieces of a whole step that starts at the current base
    __device__ __forceinline__ void issue_whole(char *lds, int wave)
    {
        __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)min(left, (int64_t)0x7fffffff), 0x00020000);
#pragma unroll
        for (int i = 0; i < N; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(lds + (i * NW + wave) * 1024), 16, (int)voff[i], 0, 0, 0);
        base += step_bytes;
        left -= step_bytes;
    }
    // the same where `kleft` values of k may end the step
    __device__ __forceinline__ void issue(char *lds, int64_t kleft, int wave, int lane)
    {
        __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)min(left, (int64_t)0x7fffffff), 0x00020000);
        if (kleft >= BK) {
#pragma unroll
            for (int i = 0; i < N; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(lds + (i * NW + wave) * 1024), 16, (int)voff[i], 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (i * NW + wave) * RPL + lane / L::PIECES, p = (lane % L::PIECES) ^ L::swizzle(r);
                const unsigned v = (KC ? p * 8 >= (int)kleft : r >= (int)kleft) ? OUTSIDE : voff[i];
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(lds + (i * NW + wave) * 1024), 16, (int)v, 0, 0, 0);
            }
        }
        base += step_bytes;
        left -= step_bytes;
    }
};

// (b) through registers: any alignment, any row length; float32 is split into its three planes on the way into LDS.
template <typename X> __device__ __forceinline__ void split3(const X &x, bf16x8 out[3])                  // X: f32x8
{
    constexpr float TOP = 3.3895313892515355e38f;                       // bf16's largest finite value
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const __bf16 h = (__bf16)__builtin_amdgcn_fmed3f((float)x[j], -TOP, TOP);
        const float r = (float)x[j] - (float)h;
        const __bf16 m = (__bf16)__builtin_amdgcn_fmed3f(r, -TOP, TOP);
        out[0][j] = h;
        out[1][j] = m;
        out[2][j] = (__bf16)(r - (float)m);
    }
}

template <int BR, bool KC, int NT> struct Staged {
    typedef Tile<BR, KC> L;
    static constexpr int N = (L::BYTES / 16 + NT - 1) / NT;             // pieces of 8 values per thread
    static constexpr bool FULL = L::BYTES / 16 % NT == 0;
    elem8 v[N];
    unsigned off[N];                                                    // bytes from `base` to the thread's pieces (the host keeps the strides small enough)
    const char *base;                                                   // element (row0, k0), the same for all threads
    int64_t ld, rows, axis;                                             // bytes; rows left from row0 on; length of the contiguous axis
    __device__ __forceinline__ void init(const Operand &o, int64_t row0, int64_t nrows, int64_t k0, int64_t K, int tid)
    {
        if (!KC && o.padded) nrows = (nrows + 7) & ~(int64_t)7;         // the padding is read as rows of zeros
        axis = KC ? K : nrows;
        ld = o.ld * (int64_t)sizeof(elem_t);
        rows = nrows - row0;
        base = (const char *)o.p + (KC ? row0 * ld + k0 * (int64_t)sizeof(elem_t) : k0 * ld + row0 * (int64_t)sizeof(elem_t));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * NT + tid, r = id / L::PIECES, p = id % L::PIECES;
            // rows past the end repeat the last one: their outputs are not stored
            const unsigned row = KC ? (unsigned)min((int64_t)r, rows - 1) : (unsigned)(FULL ? r : min(r, BK - 1));
            off[i] = row * (unsigned)ld + p * 8 * (unsigned)sizeof(elem_t);
        }
    }
    // No branch depends on a lane: a branch around a load would make every load wait for the one before it.  Where a step or a tile ends inside the contiguous axis, the pieces
    // that would pass its end are read further back, to end with it, and shifted down, zeros behind.  Only axes of fewer than 8 values in all are read one by one.
    __device__ __forceinline__ void load(int64_t kleft, int tid)
    {
        const bool whole = KC ? kleft >= BK : (kleft >= BK && rows >= BR);
        if (whole) {
#pragma unroll
            for (int i = 0; i < N; ++i) __builtin_memcpy(&v[i], base + off[i], sizeof v[i]);
        } else {
            const int inner = (int)min(KC ? kleft : rows, (int64_t)BR + BK), outer = (int)min(KC ? rows : kleft, (int64_t)BR + BK);      // both >= 1
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int id = i * NT + tid, r = id / L::PIECES, p = id % L::PIECES * 8;
                const char *row = base + (unsigned)min(r, outer - 1) * (unsigned)ld;
                int s = 0;
                if (axis >= 8) {
                    const int start = min(p, inner - 8);
                    s = r < outer ? min(p - start, 8) : 8;
                    __builtin_memcpy(&v[i], row + start * (int)sizeof(elem_t), sizeof v[i]);
                    shift_down(v[i], s);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    typedef typename std::conditional<IS_F32, unsigned, unsigned short>::type bits_t;
                    unsigned raw[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        raw[j] = *reinterpret_cast<const bits_t *>(row + min(p + j, inner - 1) * (int)sizeof(elem_t));
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        asm volatile("" : "+v"(raw[j]));                // the load stays outside of the choice, or it becomes a branch
                        if (p + j >= inner || r >= outer) raw[j] = 0;
                        v[i][j] = __builtin_bit_cast(elem_t, (bits_t)raw[j]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        base += KC ? (int64_t)BK * (int64_t)sizeof(elem_t) : BK * ld;
    }
    __device__ static __forceinline__ void put(char *lds, int id, const elem8 &x)
    {
        if (!FULL && id >= L::BYTES / 16) return;
        char *dst = lds + L::at(id / L::PIECES, id % L::PIECES);
        if constexpr (IS_F32) {
            bf16x8 s[3];
            split3(x, s);
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8 *>(dst + k * L::BYTES) = s[k];
        } else {
            *reinterpret_cast<elem8 *>(dst) = x;
        }
    }
    __device__ __forceinline__ void store(char *lds, int tid) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            put(lds, i * NT + tid, v[i]);
            if (NP > 1) __builtin_amdgcn_sched_barrier(0);             // one piece's planes at a time
        }
    }
};

// the same for dz = dy act'(z), rounded to the element type as the separate pass does it
template <int BR, bool KC, int NT> struct StagedSlope {
    typedef Staged<BR, KC, NT> S;
    S g, z;
    int act;
    float slope;
    __device__ __forceinline__ void init(const Operand &dy, const Operand &saved, int act_, float slope_, int64_t row0, int64_t nrows, int64_t k0, int64_t K, int tid)
    {
        act = act_;
        slope = slope_;
        g.init(dy, row0, nrows, k0, K, tid);
        if (act != AVC_ACT_NONE) z.init(saved, row0, nrows, k0, K, tid);
    }
    __device__ __forceinline__ void load(int64_t kleft, int tid)
    {
        g.load(kleft, tid);
        if (act != AVC_ACT_NONE) z.load(kleft, tid);
    }
    __device__ __forceinline__ void store(char *lds, int tid) const
    {
#pragma unroll
        for (int i = 0; i < S::N; ++i) {
            elem8 x = g.v[i];
            if (act != AVC_ACT_NONE) {
                float zs[8], sl[8];
                kept_z<elem_t, 8>(z.v[i], zs, act);
                slope_run<!IS_F32, 8>(zs, sl, act, slope);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = (elem_t)((float)x[j] * sl[j]);
            }
            S::put(lds, i * NT + tid, x);
        }
    }
};

// ---- the tile's products ------------------------------------------------------------------------------------------------------------------------------------
template <int FM, int FN, typename LP, typename LQ>
__device__ __forceinline__ void compute(const char *P, const char *Q, typename LP::Reader rp, typename LQ::Reader rq, f32x4 (&acc)[FM][FN])
{
    rp = LP::fresh(rp);
    rq = LQ::fresh(rq);
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
#pragma unroll
        for (int a = 0; a < NP; ++a) {                                  // plane of Q: h with h m l, m with h m, l with h
            half8 q[FN];
#pragma unroll
            for (int t = 0; t < FN; ++t) q[t] = LQ::fragment(Q + a * LQ::BYTES, rq, t, ks);
#pragma unroll
            for (int b = 0; b < NP - a; ++b) {
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const half8 p = LP::fragment(P + b * LP::BYTES, rp, i, ks);
#pragma unroll
                    for (int t = 0; t < FN; ++t) acc[i][t] = mfma(q[t], p, acc[i][t]);
                }
                if (NP > 1) __builtin_amdgcn_sched_barrier(0);         // or the reads of all nine plane pairs are hoisted and their registers spill
            }
        }
    }
}

template <int F, typename L> __device__ __forceinline__ void read_fragments(half8 (&f)[F], const char *base, typename L::Reader r, int ks)
{
    r = L::fresh(r);
#pragma unroll
    for (int t = 0; t < F; ++t) f[t] = L::fragment(base, r, t, ks);
}
template <int FM, int FN> __device__ __forceinline__ void multiply(const half8 (&p)[FM], const half8 (&q)[FN], f32x4 (&acc)[FM][FN])
{
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int t = 0; t < FN; ++t) acc[i][t] = mfma(q[t], p[i], acc[i][t]);
}
// deals READS LDS reads, and behind them LOADS loads into LDS, evenly among MFMAS matrix instructions of the surrounding block
template <int READS, int MFMAS, int LOADS> __device__ __forceinline__ void interleave()
{
    constexpr int PER = (MFMAS - LOADS) / READS > 0 ? (MFMAS - LOADS) / READS : 1;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
}

// 16 bytes of a row, of any alignment; what passes the row's end is left out.  (One store of a vector type: of a copy from an array the compiler makes several.)
template <int VEC, typename T> __device__ __forceinline__ void store_run(T *dst, const float *v, int64_t left)
{
    typedef T vec __attribute__((ext_vector_type(VEC)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    vec o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = (T)v[j];
    if (left >= VEC) *reinterpret_cast<loose *>(dst) = o;
    else
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < left) dst[j] = o[j];
}

// Steps of LDS.  float32's middle tile keeps one (48 KB), so that three workgroups share a CU and fill each other's waits; everything else two.
constexpr int stages(int BM) { return IS_F32 && BM == 128 ? 1 : 2; }

// DZ: P is dy, and what is multiplied is dy act'(saved)
struct Slope { Operand saved; int act; float slope; };

template <int BM, int BN, int WM, int WN, bool PKC, bool QKC, bool DMA, bool DZ>
__device__ __forceinline__ void tile_body(const TileArgs &a, const Slope &dz, unsigned id, unsigned total, char *smem)
{
    constexpr int NW = WM * WN, NT = NW * 64, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Tile<BM, PKC> LP;
    typedef Tile<BN, QKC> LQ;
    constexpr int STAGE = NP * (LP::BYTES + LQ::BYTES), STAGES = stages(BM);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // Workgroups go to the 8 XCDs in turn; give every XCD a contiguous run of tiles, walked in bands of 8 tile rows, so that its L2 sees the same rows and columns again.
    {
        const unsigned per = total >> 3, rem = total & 7, x = id & 7;
        id = x * per + min(x, rem) + (id >> 3);
    }
    const unsigned tiles = (unsigned)a.tiles_m * (unsigned)a.tiles_n, split = id / tiles, t = id % tiles;
    const unsigned band = t / (8u * (unsigned)a.tiles_n), in_band = t % (8u * (unsigned)a.tiles_n), band_rows = min(8u, (unsigned)a.tiles_m - band * 8u);
    const int64_t m0 = (int64_t)(band * 8u + in_band % band_rows) * BM, n0 = (int64_t)(in_band / band_rows) * BN;
    const int64_t k0 = (int64_t)split * a.kper, kend = min(a.K, k0 + a.kper);
    const int steps = (int)((kend - k0 + BK - 1) / BK);
    const int pr0 = (wave / WN) * (BM / WM), qr0 = (wave % WN) * (BN / WN);

    const typename LP::Reader rp = LP::reader(pr0, lane);
    const typename LQ::Reader rq = LQ::reader(qr0, lane);

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    if constexpr (DMA) {
        Direct<BM, PKC, NW> dp;
        Direct<BN, QKC, NW> dq;
        dp.init(a.P, m0, a.M, k0, a.K, wave, lane);
        dq.init(a.Q, n0, a.N, k0, a.K, wave, lane);
        // Software pipeline: while the matrix instructions of one half of a step (32 k) run, the fragments of the next half are read from LDS, and the pieces of the step after
        // next are on their way.  One barrier per step, between its halves: there every wave has read all of step s (so its buffer takes step s + 2) and every wave's pieces of
        // step s + 1, asked for a whole step ago, have arrived.
        static_assert(NP == 1 && BK == 64, "two halves of 32 k");
        constexpr int READS = FM * (PKC ? 1 : 2) + FN * (QKC ? 1 : 2);
        if (steps > 0) {
            dp.issue(smem, kend - k0, wave, lane);
            dq.issue(smem + LP::BYTES, kend - k0, wave, lane);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (steps > 1) {
                dp.issue(smem + STAGE, kend - k0 - BK, wave, lane);
                dq.issue(smem + STAGE + LP::BYTES, kend - k0 - BK, wave, lane);
            }
            half8 p0[FM], q0[FN], p1[FM], q1[FN];
            read_fragments<FN, LQ>(q0, smem + LP::BYTES, rq, 0);
            read_fragments<FM, LP>(p0, smem, rp, 0);
            // WHOLE: step s + 2 exists and is whole, so that its loads need no branch and can be dealt among the matrix instructions like the LDS reads
            auto step = [&](int s, auto whole) {
                constexpr bool WHOLE = decltype(whole)::value;
                char *cur = smem + (s & 1) * STAGE, *nxt = smem + ((s + 1) & 1) * STAGE;
                read_fragments<FN, LQ>(q1, cur + LP::BYTES, rq, 1);
                read_fragments<FM, LP>(p1, cur, rp, 1);
                multiply(p0, q0, acc);
                interleave<READS, FM * FN, 0>();
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (!WHOLE && s + 2 < steps) {
                    const int64_t kleft = kend - k0 - (int64_t)(s + 2) * BK;
                    dp.issue(cur, kleft, wave, lane);
                    dq.issue(cur + LP::BYTES, kleft, wave, lane);
                }
                // (the last step reads what the other buffer holds and uses none of it)
                read_fragments<FN, LQ>(q0, nxt + LP::BYTES, rq, 0);
                read_fragments<FM, LP>(p0, nxt, rp, 0);
                if constexpr (WHOLE) {
                    dp.issue_whole(cur, wave);
                    dq.issue_whole(cur + LP::BYTES, wave);
                }
                multiply(p1, q1, acc);
                interleave<READS, FM * FN, WHOLE ? Direct<BM, PKC, NW>::N + Direct<BN, QKC, NW>::N : 0>();
                __builtin_amdgcn_sched_barrier(0);
            };
            const int whole = (int)((kend - k0) / BK) - 2;
            int s = 0;
            for (; s < whole; ++s) step(s, std::true_type{});
            for (; s < steps; ++s) step(s, std::false_type{});
        }
    } else {
        typename std::conditional<DZ, StagedSlope<BM, PKC, NT>, Staged<BM, PKC, NT>>::type sp;
        Staged<BN, QKC, NT> sq;
        if constexpr (DZ) sp.init(a.P, dz.saved, dz.act, dz.slope, m0, a.M, k0, a.K, tid);
        else sp.init(a.P, m0, a.M, k0, a.K, tid);
        sq.init(a.Q, n0, a.N, k0, a.K, tid);
        if (steps > 0) {
            sp.load(kend - k0, tid);
            sq.load(kend - k0, tid);
        }
        for (int s = 0; s < steps; ++s) {
            char *cur = smem + (STAGES == 2 ? (s & 1) * STAGE : 0);
            if (STAGES == 1 && s) __syncthreads();
            sp.store(cur, tid);
            sq.store(cur + NP * LP::BYTES, tid);
            __syncthreads();
            if (s + 1 < steps) {
                const int64_t kleft = kend - k0 - (int64_t)(s + 1) * BK;
                sp.load(kleft, tid);
                sq.load(kleft, tid);
            }
            compute<FM, FN, LP, LQ>(cur, cur + NP * LP::BYTES, rp, rq, acc);
        }
    }

    // ---- epilogue
    const int64_t mw = m0 + pr0, nw = n0 + qr0;                         // the wave's corner
    if (a.splits > 1) {
        typedef f32x4 loose4 __attribute__((aligned(4)));
        float *part = a.partial + (int64_t)split * a.M * a.N;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t m = mw + 16 * i + (lane & 15);
            if (m >= a.M) continue;
#pragma unroll
            for (int f = 0; f < FN; ++f) {
                const int64_t n = nw + 16 * f + 4 * (lane >> 4);
                float *dst = part + m * a.N + n;
                if (n + 4 <= a.N) *reinterpret_cast<loose4 *>(dst) = acc[i][f];
                else
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < a.N) dst[j] = acc[i][f][j];
            }
        }
        return;
    }
    constexpr int VEC = 16 / sizeof(elem_t), WCOLS = BN / WN, PITCH = WCOLS * 4 + 16, LPR = WCOLS / VEC, RPI = 64 / LPR, ITER = 32 / RPI;
    static_assert(NW * 32 * PITCH <= STAGES * STAGE, "the epilogue's rows do not fit LDS");
    typedef elem_t run_t __attribute__((ext_vector_type(VEC)));
    typedef run_t loose_t __attribute__((aligned(sizeof(elem_t))));
    const Epilogue &e = a.ep;
    const int col = lane % LPR * VEC;
    const int64_t n = nw + col, left = a.N - n;
    float bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) bias[j] = e.bias && j < left ? (float)((const elem_t *)e.bias)[n + j] : 0.f;
    __syncthreads();                                                    // the last step's reads of LDS are over
    char *own = smem + wave * 32 * PITCH;
#pragma unroll 1
    for (int h = 0; h < FM / 2; ++h) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if (i / 2 == h) {
#pragma unroll
                for (int f = 0; f < FN; ++f) *reinterpret_cast<f32x4 *>(own + (16 * (i & 1) + (lane & 15)) * PITCH + (16 * f + 4 * (lane >> 4)) * 4) = acc[i][f];
            }
        __builtin_amdgcn_wave_barrier();
        run_t res[ITER];
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int64_t m = mw + 32 * h + it * RPI + lane / LPR;
            res[it] = run_t(0);
            if (e.res && m < a.M && left > 0) {
                const elem_t *r = (const elem_t *)e.res + m * e.ldr + n;
                if (left >= VEC) res[it] = *reinterpret_cast<const loose_t *>(r);
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (j < left) res[it][j] = r[j];
            }
        }
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int row = it * RPI + lane / LPR;
            const int64_t m = mw + 32 * h + row;
            float v[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(own + row * PITCH + (col + j) * 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[j + k] = x[k] + bias[j + k];
            }
            if (m >= a.M || left <= 0) continue;
            if (e.z) {
                if (KeptZ<elem_t>::finer(e.act)) store_run<VEC>((_Float16 *)e.z + m * e.ldz + n, v, left);
                else store_run<VEC>((elem_t *)e.z + m * e.ldz + n, v, left);
            }
            act_run<!IS_F32, VEC>(v, e.act, e.slope);
            if (e.res)
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] += (float)res[it][j];
            store_run<VEC>((elem_t *)a.out + m * a.ldo + n, v, left);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int WM, int WN, bool PKC, bool QKC, bool DMA>
__global__ __launch_bounds__(WM * WN * 64, IS_F32 && BM == 128 ? 3 : 2) void tile_kernel(const TileArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    tile_body<BM, BN, WM, WN, PKC, QKC, DMA, false>(a, Slope{}, blockIdx.x, gridDim.x, smem);
}

// The whole backward pass of a small layer in one launch: workgroups for the tiles of dx, then for those of dw, then for 16 columns of db each.  The three read dy and z for
// themselves and form dz on the way into LDS.
template <bool XKC> __global__ __launch_bounds__(256, 2) void small_backward_kernel(const SmallArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const unsigned id = blockIdx.x, ndx = (unsigned)a.dx.tiles_m * (unsigned)a.dx.tiles_n, ndw = (unsigned)a.dw.tiles_m * (unsigned)a.dw.tiles_n;
    if (id < ndx) {
        tile_body<64, 64, 2, 2, true, false, false, true>(a.dx, Slope{Operand{a.saved, a.ld_saved, 1}, a.act, a.slope}, id, ndx, smem);
    } else if (id < ndx + ndw) {
        tile_body<64, 64, 2, 2, false, !XKC, false, true>(a.dw, Slope{Operand{a.saved, a.ld_saved, 0}, a.act, a.slope}, id - ndx, ndw, smem);
    } else {
        float(*red)[17] = reinterpret_cast<float(*)[17]>(smem);
        const int lx = threadIdx.x & 15, ly = threadIdx.x >> 4;
        const int64_t n = (int64_t)(id - ndx - ndw) * 16 + lx, nc = min(n, a.N - 1);
        const elem_t *dy = (const elem_t *)a.dy + nc, *z = (const elem_t *)a.saved + nc;
        float s = 0.f;
        for (int64_t m = ly; m < a.M; m += 16 * 4) {
            float g[4], zs[4], sl[4];
            elem_t kept[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t r = min(m + 16 * j, a.M - 1);
                g[j] = (float)dy[r * a.lddy];
                kept[j] = a.act != AVC_ACT_NONE ? z[r * a.ld_saved] : (elem_t)0.f;
            }
            kept_z<elem_t, 4>(kept, zs, a.act);
            slope_run<!IS_F32, 4>(zs, sl, a.act, a.slope);
#pragma unroll
            for (int j = 0; j < 4; ++j) s += m + 16 * j < a.M ? g[j] * sl[j] : 0.f;
        }
        red[ly][lx] = s;
        __syncthreads();
        if (ly || n >= a.N) return;
#pragma unroll
        for (int y = 1; y < 16; ++y) s += red[y][lx];
        ((elem_t *)a.db)[n] = (elem_t)s;
    }
}

template <int BM, int BN, int WM, int WN, bool PKC, bool QKC, bool DMA> int launch_one(const TileArgs &a, hipStream_t s)
{
    constexpr int LDS = stages(BM) * NP * (Tile<BM, PKC>::BYTES + Tile<BN, QKC>::BYTES);
    static_assert(LDS <= 160 * 1024, "tile does not fit LDS");
    auto k = tile_kernel<BM, BN, WM, WN, PKC, QKC, DMA>;
    if (LDS > 64 * 1024) {                                              // once per device
        static std::atomic<uint64_t> allowed{0};
        int device = 0;
        AVC_HIP(hipGetDevice(&device));
        const uint64_t bit = 1ull << (device & 63);
        if (device > 63 || !(allowed.load(std::memory_order_acquire) & bit)) {
            AVC_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
            allowed.fetch_or(bit, std::memory_order_release);
        }
    }
    hipLaunchKernelGGL(k, dim3((unsigned)((int64_t)a.tiles_m * a.tiles_n * a.splits)), dim3(WM * WN * 64), LDS, s, a);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

template <int BM, int BN, int WM, int WN, bool DMA> int launch_layout(const TileArgs &a, hipStream_t s)
{
    if (a.P.kc) return a.Q.kc ? launch_one<BM, BN, WM, WN, true, true, DMA>(a, s) : launch_one<BM, BN, WM, WN, true, false, DMA>(a, s);
    return a.Q.kc ? launch_one<BM, BN, WM, WN, false, true, DMA>(a, s) : launch_one<BM, BN, WM, WN, false, false, DMA>(a, s);
}

template <bool DMA> int launch_shape(const TileArgs &a, int tile, hipStream_t s)
{
    if (tile == TILE_BIG) {
        if constexpr (IS_F32) return launch_layout<256, 128, 4, 2, DMA>(a, s);
        else return launch_layout<256, 256, 2, 4, DMA>(a, s);
    }
    if (tile == TILE_MID) return launch_layout<128, 128, 2, 2, DMA>(a, s);
    return launch_layout<64, 64, 2, 2, DMA>(a, s);
}

template <bool XKC> int launch_small(const SmallArgs &a, unsigned blocks, hipStream_t s)
{
    constexpr int A = Tile<64, true>::BYTES + Tile<64, false>::BYTES, B = Tile<64, false>::BYTES + Tile<64, !XKC>::BYTES, LDS = 2 * NP * (A > B ? A : B);
    static_assert(LDS <= 64 * 1024, "within the default limit");
    hipLaunchKernelGGL(small_backward_kernel<XKC>, dim3(blocks), dim3(256), LDS, s, a);
    AVC_HIP(hipGetLastError());
    return AVC_OK;
}

// the direct loads' conditions: whole 16-byte pieces, aligned, and a tile's offsets within 31 bits
bool direct_ok(const Operand &o, int64_t rows, int64_t K)
{
    const int64_t inner = o.kc ? K : rows;
    return ((uintptr_t)o.p & 15) == 0 && o.ld % 8 == 0 && (o.padded || inner % 8 == 0) && o.ld < (int64_t)1 << 21;
}

}  // namespace

int AVC_LAUNCH_SMALL(const SmallArgs &a, unsigned blocks, bool x_kc, hipStream_t s)
{
    return x_kc ? launch_small<true>(a, blocks, s) : launch_small<false>(a, blocks, s);
}

int AVC_LAUNCH(const TileArgs &a, int tile, hipStream_t s)
{
    if constexpr (!IS_F32)
        if (direct_ok(a.P, a.M, a.K) && direct_ok(a.Q, a.N, a.K)) return launch_shape<true>(a, tile, s);
    return launch_shape<false>(a, tile, s);
}

}}  // namespace avc::lin
