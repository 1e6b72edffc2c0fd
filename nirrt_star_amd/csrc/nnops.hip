// nnops.hip - the dense operators of the guidance network's layers and of its training step (C ABI: include/nirrt_nnops.h).
//
//   linear          y = act(x w^T + b) + r, and its gradients
//   cross entropy   softmax cross entropy of the scores x w^T + b without keeping them, and its gradients
//   norm / scale    2-norm of many tensors, and the clipping by it
//
// All products run through one tile loop (class-free: mainloop below) on v_mfma_f32_32x32x*: a workgroup of 4 waves owns a tile
// C[i, j] = sum_k A[i, k] B[j, k], K-steps of 128 bytes per row.  An operand is stored either with k contiguous ("KC": x, w in the forward
// product) or with i contiguous ("RC": w in dx = dz w, dz and x in dw = dz^T x); an RC operand is transposed in registers on its way
// into the LDS, so both look alike there: rows of eight 16-byte chunks along k, chunk c of row r at place c ^ sw(r).  A lane's 16-byte
// read is one operand of a 16-bit MFMA (8 k) or four of a 32-bit one (4 x 1 k); the order of k inside a step is the same in A and B, so
// the sum is the same whatever it is.  Accumulators and partial sums are fp32.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/nirrt_nnops.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr int ROW_BYTES = 128;          // bytes of k per row and step
constexpr int CHUNKS = ROW_BYTES / 16;

template <class T> struct Elem { static constexpr int PER_CHUNK = 16 / sizeof(T), STEP = ROW_BYTES / sizeof(T); };

__device__ __forceinline__ int sw(int row) { return (row ^ (row >> 3)) & 7; }   // 8 lanes on 8 neighbouring (or every 4th) rows: 8 places

__device__ __forceinline__ f32x16 mma(bf16_t, u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16_t, u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(float, u32x4 a, u32x4 b, f32x16 c)
{
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
}

// one operand: element (r, k) at p[r * ld + k] (KC) or p[k * ld + r] (RC); vec: whole 16-byte chunks (KC) / 4 elements (RC) are aligned.
// skip (RC, or null): row k of the operand counts as zeros where skip[k] == 0, whatever it holds
template <class T> struct Operand {
    const T *p;
    int64_t ld;
    int rows;
    int vec;
    const float *skip;
};

// a thread's share of one K-step of R rows: global memory -> registers -> LDS
template <class T, int R, int NT, bool RC> struct Stage {
    static constexpr int N = R * CHUNKS / NT, CE = Elem<T>::PER_CHUNK, VR = N % 4 == 0 ? 4 : 2;   // VR: rows of a transposed block
    static_assert(N % 2 == 0 && R % 4 == 0, "whole blocks per thread");
    u32x4 v[N];

    __device__ __forceinline__ void load(const Operand<T> &o, int r0, int k0, int k1, int tid)
    {
        if constexpr (!RC) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int c = tid + i * NT, row = r0 + (c >> 3), k = k0 + (c & 7) * CE;
                const T *q = o.p + (int64_t)row * o.ld + k;
                u32x4 x = {0, 0, 0, 0};
                if (row < o.rows && k < k1) {
                    if (o.vec && k + CE <= k1) x = *(const u32x4 *)q;
                    else {
                        T e[CE];
#pragma unroll
                        for (int j = 0; j < CE; j++) e[j] = k + j < k1 ? q[j] : (T)0.f;
                        __builtin_memcpy(&x, e, 16);
                    }
                }
                v[i] = x;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / VR; i++) {
                const int blk = tid + i * NT, row = r0 + (blk % (R / VR)) * VR, k = k0 + (blk / (R / VR)) * CE;
                T e[VR][CE];
#pragma unroll
                for (int j = 0; j < CE; j++) {
                    const T *q = o.p + (int64_t)(k + j) * o.ld + row;
                    T f[VR];
#pragma unroll
                    for (int s = 0; s < VR; s++) f[s] = (T)0.f;
                    if (k + j < k1 && row < o.rows && !(o.skip && o.skip[k + j] == 0.f)) {
                        if (o.vec && row + VR <= o.rows) __builtin_memcpy(f, __builtin_assume_aligned(q, VR * sizeof(T)), VR * sizeof(T));
                        else {
#pragma unroll
                            for (int s = 0; s < VR; s++)
                                if (row + s < o.rows) f[s] = q[s];
                        }
                    }
#pragma unroll
                    for (int s = 0; s < VR; s++) e[s][j] = f[s];
                }
#pragma unroll
                for (int s = 0; s < VR; s++) __builtin_memcpy(&v[VR * i + s], e[s], 16);
            }
        }
    }
    __device__ __forceinline__ void store(u32x4 *lds, int tid) const
    {
        if constexpr (!RC) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int c = tid + i * NT, r = c >> 3;
                lds[r * CHUNKS + ((c & 7) ^ sw(r))] = v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / VR; i++) {
                const int blk = tid + i * NT, r = (blk % (R / VR)) * VR, ch = blk / (R / VR);
#pragma unroll
                for (int s = 0; s < VR; s++) lds[(r + s) * CHUNKS + (ch ^ sw(r + s))] = v[VR * i + s];
            }
        }
    }
};

// the tile of C that a wave holds: MI x NI blocks of 32 x 32; block register e of a lane is row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
template <class T, int BM, int BN, int WM, int WN, bool RCA, bool RCB> struct Tile {
    static constexpr int NT = 64 * WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
    static constexpr int LDS_CHUNKS = (BM + BN) * CHUNKS;
    f32x16 acc[MI][NI];

    static __device__ __forceinline__ int row(int wave, int lane, int mi, int e) { return (wave / WN) * (BM / WM) + mi * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }
    static __device__ __forceinline__ int col(int wave, int lane, int ni) { return (wave % WN) * (BN / WN) + ni * 32 + (lane & 31); }

    // acc = sum over k in [k0, k1) of A[i0 + ., k] B[j0 + ., k]
    __device__ __forceinline__ void mainloop(const Operand<T> &a, const Operand<T> &b, int i0, int j0, int k0, int k1, u32x4 *lds)
    {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        u32x4 *la = lds, *lb = lds + BM * CHUNKS;
#pragma unroll
        for (int mi = 0; mi < MI; mi++)
#pragma unroll
            for (int ni = 0; ni < NI; ni++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[mi][ni][e] = 0.f;
        if (k0 >= k1) return;
        Stage<T, BM, NT, RCA> sa;
        Stage<T, BN, NT, RCB> sb;
        sa.load(a, i0, k0, k1, tid);
        sb.load(b, j0, k0, k1, tid);
        for (int k = k0; k < k1; k += Elem<T>::STEP) {
            __syncthreads();                 // (the previous step has been read)
            sa.store(la, tid);
            sb.store(lb, tid);
            __syncthreads();
            if (k + Elem<T>::STEP < k1) {    // the next step travels while this one is multiplied
                sa.load(a, i0, k + Elem<T>::STEP, k1, tid);
                sb.load(b, j0, k + Elem<T>::STEP, k1, tid);
            }
            const int r = lane & 31, half = lane >> 5, ra = (wave / WN) * (BM / WM) + r, rb = (wave % WN) * (BN / WN) + r;
#pragma unroll
            for (int s = 0; s < CHUNKS / 2; s++) {
                u32x4 fa[MI], fb[NI];
#pragma unroll
                for (int mi = 0; mi < MI; mi++) fa[mi] = la[(ra + 32 * mi) * CHUNKS + ((2 * s + half) ^ sw(ra + 32 * mi))];
#pragma unroll
                for (int ni = 0; ni < NI; ni++) fb[ni] = lb[(rb + 32 * ni) * CHUNKS + ((2 * s + half) ^ sw(rb + 32 * ni))];
#pragma unroll
                for (int mi = 0; mi < MI; mi++)
#pragma unroll
                    for (int ni = 0; ni < NI; ni++) acc[mi][ni] = mma((T)0.f, fa[mi], fb[ni], acc[mi][ni]);
            }
        }
    }
};

// workgroup -> tile.  Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own: XCD x gets a contiguous share of
// the tiles, walked in groups of 8 tile rows, so that what its workgroups read at one time overlaps.
__device__ __forceinline__ void tile_of(int id, int count, int tiles_i, int tiles_j, int &ti, int &tj)
{
    const int x = id & 7, q = count >> 3, rem = count & 7;
    const int t = x * q + (x < rem ? x : rem) + (id >> 3);
    const int width = 8 * tiles_j, group = t / width, first = group * 8, rows = tiles_i - first < 8 ? tiles_i - first : 8, in = t - group * width;
    ti = first + in % rows;
    tj = in / rows;
}

// ---- activations ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float act_value(int act, float z)
{
    switch (act) {
    case NIRRT_NN_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);          // (NaN stays)
    case NIRRT_NN_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678118654752f);
    case NIRRT_NN_ACT_SILU: return z / (1.f + __expf(-z));
    default: return z;
    }
}
__device__ __forceinline__ float act_slope(int act, float z)
{
    switch (act) {
    case NIRRT_NN_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case NIRRT_NN_ACT_GELU: return 0.5f * erfcf(z * -0.70710678118654752f) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
    case NIRRT_NN_ACT_SILU: { const float s = 1.f / (1.f + __expf(-z)); return s * (1.f + z * (1.f - s)); }
    default: return 1.f;
    }
}

// ---- what a product does with an element of C ------------------------------------------------------------------------------------
// y = act(C + b[j]) + r, and z
template <class T> struct EpiLinear {
    const T *b, *r;
    T *y, *z;
    int64_t ldr, ldy;
    int act, n;
    __device__ __forceinline__ float column(int j) const { return b ? (float)b[j] : 0.f; }
    __device__ __forceinline__ void put(float c, float col, int i, int j) const
    {
        const float v = c + col;
        if (z) z[(int64_t)i * n + j] = (T)v;
        float o = act_value(act, v);
        if (r) o += (float)r[(int64_t)i * ldr + j];
        y[(int64_t)i * ldy + j] = (T)o;
    }
};
// out = scale C (contiguous rows of n); scale on the device or 1
template <class T> struct EpiPlain {
    T *out;
    const float *scale;
    float factor;
    int n;
    __device__ __forceinline__ float column(int) const { return scale ? *scale * factor : factor; }
    __device__ __forceinline__ void put(float c, float col, int i, int j) const { out[(int64_t)i * n + j] = (T)(c * col); }
};
// acc (+)= C in fp32: the sum over pieces of the reduction that are multiplied one after the other
struct EpiAccumulate {
    float *out;
    int n, first;
    __device__ __forceinline__ float column(int) const { return 0.f; }
    __device__ __forceinline__ void put(float c, float, int i, int j) const
    {
        float *q = out + (int64_t)i * n + j;
        *q = first ? c : *q + c;
    }
};

// BM x BN tiles, the reduction cut into gridDim.y parts of `part`; with more than one, the parts go to `partial` (part, i, j) for k_join
template <class T, int BM, int BN, int WM, int WN, bool RCA, bool RCB, class Epi>
__global__ __launch_bounds__(64 * WM * WN) void k_gemm(Operand<T> a, Operand<T> b, int m, int n, int k, int part, float *partial, Epi epi)
{
    typedef Tile<T, BM, BN, WM, WN, RCA, RCB> Tl;
    __shared__ u32x4 lds[Tl::LDS_CHUNKS];
    Tl t;
    int ti, tj;
    tile_of(blockIdx.x, gridDim.x, (m + BM - 1) / BM, (n + BN - 1) / BN, ti, tj);
    const int k0 = blockIdx.y * part, k1 = k - k0 < part ? k : k0 + part;
    t.mainloop(a, b, ti * BM, tj * BN, k0, k1, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *pp = partial + (gridDim.y > 1 ? (int64_t)blockIdx.y * m * n : 0);
#pragma unroll
    for (int ni = 0; ni < Tl::NI; ni++) {
        const int j = tj * BN + Tl::col(wave, lane, ni);
        if (j >= n) continue;
        const float col = epi.column(j);
#pragma unroll
        for (int mi = 0; mi < Tl::MI; mi++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int i = ti * BM + Tl::row(wave, lane, mi, e);
                if (i >= m) continue;
                if (gridDim.y > 1) pp[(int64_t)i * n + j] = t.acc[mi][ni][e];
                else epi.put(t.acc[mi][ni][e], col, i, j);
            }
    }
}
// the parts of a cut reduction, added in their order
template <class Epi> __global__ __launch_bounds__(256) void k_join(const float *partial, int parts, int m, int n, Epi epi)
{
    const int64_t size = (int64_t)m * n;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < size; at += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        for (int p = 0; p < parts; p++) s += partial[p * size + at];
        const int i = (int)(at / n), j = (int)(at - (int64_t)i * n);
        epi.put(s, epi.column(j), i, j);
    }
}

// ---- dz = dy act'(z) and its column sums -------------------------------------------------------------------------------------------
// grid (column blocks of 256, row chunks): a thread walks its column of the chunk
template <class T>
__global__ __launch_bounds__(256) void k_dz(const T *z, const T *dy, int64_t lddy, T *dz, float *sums, int m, int n, int chunk, int act)
{
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= n) return;
    const int i0 = blockIdx.y * chunk, i1 = m - i0 < chunk ? m : i0 + chunk;
    float s = 0.f;
    for (int i = i0; i < i1; i++) {
        float d = (float)dy[(int64_t)i * lddy + j];
        if (act != NIRRT_NN_ACT_NONE) {
            d *= act_slope(act, (float)z[(int64_t)i * n + j]);
            if (dz) dz[(int64_t)i * n + j] = (T)d;
        }
        s += d;
    }
    if (sums) sums[(int64_t)blockIdx.y * n + j] = s;
}
template <class T> __global__ __launch_bounds__(256) void k_column_join(const float *sums, int parts, T *out, int n)
{
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= n) return;
    float s = 0.f;
    for (int p = 0; p < parts; p++) s += sums[(int64_t)p * n + j];
    out[j] = (T)s;
}

// ---- cross entropy -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float row_weight(const float *cw, int64_t t, int64_t ignore, int classes)
{
    if (t == ignore) return 0.f;
    if (t < 0 || t >= classes) return __builtin_nanf("");
    return cw ? cw[t] : 1.f;
}

// C[v, r] = w_v . x_r: a lane holds scores of NI rows r (its columns), so the running maximum and sum over the classes stay in the
// lane; the two halves of a wave and the waves above one another meet once, at the end.  grid (row tiles, parts of the classes).
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_ce_stats(Operand<T> w, Operand<T> x, const T *b, const int64_t *target, int rows, int classes,
                                                           int k, int part, float2 *stats, float *target_score)
{
    typedef Tile<T, BM, BN, WM, WN, false, false> Tl;
    __shared__ u32x4 lds[Tl::LDS_CHUNKS];
    __shared__ float2 meet[2 * WM][BN];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r0 = blockIdx.x * BN;
    float m[Tl::NI], s[Tl::NI];
    int64_t tg[Tl::NI];
#pragma unroll
    for (int ni = 0; ni < Tl::NI; ni++) {
        m[ni] = -__builtin_inff();
        s[ni] = 0.f;
        const int r = r0 + Tl::col(wave, lane, ni);
        tg[ni] = r < rows ? target[r] : -1;
    }
    const int v_end = classes - (int)blockIdx.y * part < part ? classes : ((int)blockIdx.y + 1) * part;
    for (int v0 = blockIdx.y * part; v0 < v_end; v0 += BM) {
        Tl t;
        t.mainloop(w, x, v0, r0, 0, k, lds);
#pragma unroll
        for (int mi = 0; mi < Tl::MI; mi++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int v = v0 + Tl::row(wave, lane, mi, e);
                const float add = v < v_end ? (b ? (float)b[v] : 0.f) : -__builtin_inff();
#pragma unroll
                for (int ni = 0; ni < Tl::NI; ni++) t.acc[mi][ni][e] = v < v_end ? t.acc[mi][ni][e] + add : add;
            }
#pragma unroll
        for (int ni = 0; ni < Tl::NI; ni++) {
            float top = m[ni];
            const int64_t want = tg[ni] - v0;
#pragma unroll
            for (int mi = 0; mi < Tl::MI; mi++)
#pragma unroll
                for (int e = 0; e < 16; e++) top = fmaxf(top, t.acc[mi][ni][e]);
            float sum = 0.f;
            const float ref = top == -__builtin_inff() ? 0.f : top;   // (nothing but -inf so far: exp(-inf) adds zeros)
#pragma unroll
            for (int mi = 0; mi < Tl::MI; mi++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    sum += __expf(t.acc[mi][ni][e] - ref);
                    if (want == Tl::row(wave, lane, mi, e) && want < v_end - v0) target_score[r0 + Tl::col(wave, lane, ni)] = t.acc[mi][ni][e];
                }
            s[ni] = s[ni] * __expf(m[ni] - ref) + sum;
            m[ni] = top;
        }
    }
#pragma unroll
    for (int ni = 0; ni < Tl::NI; ni++) meet[2 * (wave / WN) + (lane >> 5)][Tl::col(wave, lane, ni)] = make_float2(m[ni], s[ni]);
    __syncthreads();
    for (int c = threadIdx.x; c < BN; c += Tl::NT) {
        float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (int p = 0; p < 2 * WM; p++) top = fmaxf(top, meet[p][c].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int p = 0; p < 2 * WM; p++) sum += meet[p][c].y * __expf(meet[p][c].x - ref);
        if (r0 + c < rows) stats[(int64_t)blockIdx.y * rows + r0 + c] = make_float2(top, sum);
    }
}
// parts of a row's statistics -> lse, weighted loss; the block's sums of loss and weight (in double) for k_ce_total
__global__ __launch_bounds__(256) void k_ce_rows(const float2 *stats, int parts, const float *target_score, const int64_t *target, const float *cw,
                                                 int64_t ignore, int rows, int classes, float *lse, float *nll, double *sums)
{
    __shared__ double part[2][4];
    const int r = blockIdx.x * 256 + threadIdx.x;
    double a = 0., b = 0.;
    if (r < rows) {
        float top = -__builtin_inff(), sum = 0.f;
        for (int p = 0; p < parts; p++) top = fmaxf(top, stats[(int64_t)p * rows + r].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
        for (int p = 0; p < parts; p++) { const float2 q = stats[(int64_t)p * rows + r]; sum += q.y * __expf(q.x - ref); }
        const float l = top + logf(sum);
        const int64_t t = target[r];
        const float wt = row_weight(cw, t, ignore, classes);
        const float loss = t == ignore ? 0.f : (wt == wt ? wt * (l - target_score[r]) : wt);
        lse[r] = l;
        nll[r] = loss;
        a = loss;
        b = wt;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) { a += __shfl_down(a, d); b += __shfl_down(b, d); }
    if ((threadIdx.x & 63) == 0) { part[0][threadIdx.x >> 6] = a; part[1][threadIdx.x >> 6] = b; }
    __syncthreads();
    if (threadIdx.x < 2) sums[2 * blockIdx.x + threadIdx.x] = (part[threadIdx.x][0] + part[threadIdx.x][1]) + (part[threadIdx.x][2] + part[threadIdx.x][3]);
}
// sums of pairs in a fixed order, one workgroup
__global__ __launch_bounds__(256) void k_ce_total(const double *sums, int blocks, float *total)
{
    __shared__ double part[2][4];
    double a = 0., b = 0.;
    for (int i = threadIdx.x; i < blocks; i += 256) { a += sums[2 * i]; b += sums[2 * i + 1]; }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) { a += __shfl_down(a, d); b += __shfl_down(b, d); }
    if ((threadIdx.x & 63) == 0) { part[0][threadIdx.x >> 6] = a; part[1][threadIdx.x >> 6] = b; }
    __syncthreads();
    if (threadIdx.x == 0) {
        a = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
        b = (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]);
        total[0] = (float)a;
        total[1] = (float)b;
        total[2] = (float)(a / b);          // (no row counts: 0 / 0)
    }
}
// c_r = dloss_r weight_r (/ total weight): rel[r] = c_r / max |c|, scale[0] = max |c|; one workgroup
__global__ __launch_bounds__(1024) void k_ce_coefficients(const float *dloss, int stride, const float *total, const int64_t *target, const float *cw,
                                                          int64_t ignore, int rows, int classes, float *rel, float *scale)
{
    __shared__ float part[16];
    const float div = total ? 1.f / total[1] : 1.f;
    float top = 0.f;
    bool bad = false;
    for (int r = threadIdx.x; r < rows; r += 1024) {
        const int64_t t = target[r];
        const float c = t == ignore ? 0.f : dloss[stride ? r : 0] * row_weight(cw, t, ignore, classes) * div;
        rel[r] = c;
        bad = bad || c != c;
        top = fmaxf(top, fabsf(c));
    }
    if (bad) top = __builtin_inff();            // (a NaN row: the scale says so below)
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    top = part[0];
#pragma unroll
    for (int p = 1; p < 16; p++) top = fmaxf(top, part[p]);
    // no row counts, or something is not finite: rel keeps the coefficients themselves
    const bool usable = top > 0.f && top < __builtin_inff();
    if (usable)
        for (int r = threadIdx.x; r < rows; r += 1024) rel[r] = rel[r] / top;
    if (threadIdx.x == 0) scale[0] = usable ? top : 1.f;
}
// g' = rel_r (exp(l - lse_r) - [v = target]) FACTOR in the element type, stored (v, r): the product C[v, r] again.  16-bit products need
// 16-bit operands; rel <= 1 keeps the range, and FACTOR 4096 in f16 lifts probabilities of large vocabularies (1e-5) out of its
// subnormals.  Relative error of a rounding: 2^-9 (bf16), 2^-12 (f16) of the element, like the rounding of dz in the linear layer.
template <class T> struct Factor { static constexpr float VALUE = 1.f; };
template <> struct Factor<f16_t> { static constexpr float VALUE = 4096.f; };
template <class T> struct EpiSoftmaxGrad {
    T *g;
    int64_t ldg;
    const T *b;
    const float *lse, *rel;
    const int64_t *target;
    int64_t v0;
    __device__ __forceinline__ float column(int) const { return 0.f; }
    __device__ __forceinline__ void put(float c, float, int i, int j) const
    {
        const float coef = rel[j];
        float p = __expf(c + (b ? (float)b[v0 + i] : 0.f) - lse[j]);
        if (target[j] == v0 + i) p -= 1.f;
        g[(int64_t)i * ldg + j] = coef == 0.f ? (T)0.f : (T)(p * coef * Factor<T>::VALUE);
    }
};
// db[v] = scale / FACTOR sum_r g'[v, r]: a wave per class
template <class T> __global__ __launch_bounds__(256) void k_ce_bias(const T *g, int64_t ldg, int rows, int classes, const float *scale, T *db)
{
    const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (v >= classes) return;
    float s = 0.f;
    for (int r = threadIdx.x & 63; r < rows; r += 64) s += (float)g[(int64_t)v * ldg + r];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) db[v] = (T)(s * *scale * (1.f / Factor<T>::VALUE));
}
template <class T> __global__ __launch_bounds__(256) void k_cast(const float *in, const float *scale, float factor, T *out, int64_t n)
{
    const float f = *scale * factor;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (T)(in[i] * f);
}

// ---- norm and clipping of many tensors -------------------------------------------------------------------------------------------------
constexpr int TABLE = 128;                // tensors per launch: the table travels in the kernel's arguments (2.9 KB), no copy to wait for
constexpr int BLOCK_ELEMS = 16384;        // elements per workgroup
struct TensorTable {
    const void *in[TABLE];
    void *out[TABLE];
    int64_t n[TABLE];
    int first[TABLE];                     // first workgroup of the tensor
    uint8_t dtype[TABLE], out_dtype[TABLE];
    int count;
};
__device__ __forceinline__ int tensor_of(const TensorTable &t, int block)
{
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ float elem(const void *p, int dtype, int64_t i)
{
    return dtype == NIRRT_NN_F32 ? ((const float *)p)[i] : dtype == NIRRT_NN_BF16 ? (float)((const bf16_t *)p)[i] : (float)((const f16_t *)p)[i];
}
__global__ __launch_bounds__(256) void k_norm_parts(TensorTable t, double *parts)
{
    __shared__ double part[4];
    const int e = tensor_of(t, blockIdx.x);
    const int64_t i0 = (int64_t)(blockIdx.x - t.first[e]) * BLOCK_ELEMS, i1 = t.n[e] - i0 < BLOCK_ELEMS ? t.n[e] : i0 + BLOCK_ELEMS;
    double s = 0.;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) { const double v = elem(t.in[e], t.dtype[e], i); s += v * v; }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}
__global__ __launch_bounds__(256) void k_norm_total(const double *parts, int64_t n, float *norm)
{
    __shared__ double part[4];
    double s = 0.;
    for (int64_t i = threadIdx.x; i < n; i += 256) s += parts[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) *norm = (float)sqrt((part[0] + part[1]) + (part[2] + part[3]));
}
__global__ __launch_bounds__(256) void k_scale(TensorTable t, const float *norm, float max_norm)
{
    const int e = tensor_of(t, blockIdx.x);
    const float q = max_norm / (*norm + 1e-6f), f = q < 1.f ? q : (q == q ? 1.f : q);
    if (f == 1.f && t.in[e] == t.out[e]) return;
    const int64_t i0 = (int64_t)(blockIdx.x - t.first[e]) * BLOCK_ELEMS, i1 = t.n[e] - i0 < BLOCK_ELEMS ? t.n[e] : i0 + BLOCK_ELEMS;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) {
        const float v = elem(t.in[e], t.dtype[e], i) * f;
        if (t.out_dtype[e] == NIRRT_NN_F32) ((float *)t.out[e])[i] = v;
        else if (t.out_dtype[e] == NIRRT_NN_BF16) ((bf16_t *)t.out[e])[i] = (bf16_t)v;
        else ((f16_t *)t.out[e])[i] = (f16_t)v;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
constexpr int64_t DIM_MAX = 0x7fffffffll;
int64_t round256(int64_t b) { return (b + 255) & ~255ll; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int status() { return hipGetLastError() == hipSuccess ? 0 : -2; }
int elem_size(int dtype) { return dtype == NIRRT_NN_F32 ? 4 : 2; }
bool good_type(int dtype) { return dtype == NIRRT_NN_F32 || dtype == NIRRT_NN_BF16 || dtype == NIRRT_NN_F16; }

template <class T> Operand<T> kc(const T *p, int64_t ld, int64_t rows)
{
    return {p, ld, (int)rows, ((uintptr_t)p % 16 == 0 && ld * (int64_t)sizeof(T) % 16 == 0) ? 1 : 0, nullptr};
}
template <class T> Operand<T> rc(const T *p, int64_t ld, int64_t rows, const float *skip = nullptr)
{
    return {p, ld, (int)rows, ((uintptr_t)p % (4 * sizeof(T)) == 0 && ld % 4 == 0) ? 1 : 0, skip};
}

// tile edge and parts of the reduction.  A GPU of 256 CUs wants some 500 workgroups of four waves: 128 x 128 tiles where that many exist,
// else 64 x 64; where even these are fewer and the reduction is long, it is cut (at least four steps per part, at most 32 parts).
struct Plan { int edge, parts, part; };
Plan plan(int dtype, int64_t m, int64_t n, int64_t k)
{
    Plan p;
    const int64_t big = ceil_div(m, 128) * ceil_div(n, 128), step = ROW_BYTES / elem_size(dtype), steps = ceil_div(k, step);
    p.edge = big >= 256 ? 128 : 64;
    const int64_t tiles = ceil_div(m, p.edge) * ceil_div(n, p.edge);      // (0 for an empty result)
    int64_t parts = tiles >= 256 || tiles == 0 ? 1 : 512 / tiles;
    if (parts > steps / 4) parts = steps / 4;
    if (parts > 32) parts = 32;
    if (parts < 1) parts = 1;
    const int64_t per = ceil_div(steps, parts);
    p.part = (int)(per * step < DIM_MAX ? (per > 0 ? per * step : step) : DIM_MAX);
    p.parts = (int)(steps > 0 ? ceil_div(steps, per) : 1);
    return p;
}
int64_t plan_bytes(const Plan &p, int64_t m, int64_t n) { return p.parts > 1 ? round256(4 * m * n * p.parts) : 0; }

template <class T, bool RCA, bool RCB, class Epi>
int gemm(const Operand<T> &a, const Operand<T> &b, int64_t m, int64_t n, int64_t k, const Plan &p, float *partial, const Epi &epi, hipStream_t st)
{
    const int64_t tiles = ceil_div(m, p.edge) * ceil_div(n, p.edge);
    if (tiles > DIM_MAX) return -1;
    const dim3 grid((unsigned)tiles, (unsigned)p.parts);
    if (p.edge == 128)
        hipLaunchKernelGGL((k_gemm<T, 128, 128, 2, 2, RCA, RCB, Epi>), grid, dim3(256), 0, st, a, b, (int)m, (int)n, (int)k, p.part, partial, epi);
    else
        hipLaunchKernelGGL((k_gemm<T, 64, 64, 2, 2, RCA, RCB, Epi>), grid, dim3(256), 0, st, a, b, (int)m, (int)n, (int)k, p.part, partial, epi);
    if (p.parts > 1) {
        const int64_t blocks = ceil_div(m * n, 256);
        hipLaunchKernelGGL((k_join<Epi>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, partial, p.parts, (int)m, (int)n, epi);
    }
    return status();
}

bool good_dims(int64_t a, int64_t b, int64_t c) { return a >= 0 && b >= 0 && c >= 0 && a <= DIM_MAX - 256 && b <= DIM_MAX - 256 && c <= DIM_MAX - 256; }

constexpr int COLUMN_PARTS = 256;
int column_chunk(int64_t m) { const int64_t c = ceil_div(m, COLUMN_PARTS); return (int)(c > 32 ? c : 32); }

struct LinearBackward { Plan px, pw; int64_t dz, sums, part, total; };
LinearBackward linear_backward_layout(int dtype, int act, int64_t m, int64_t n, int64_t k)
{
    LinearBackward l;
    l.px = plan(dtype, m, k, n);
    l.pw = plan(dtype, n, k, m);
    l.dz = act == NIRRT_NN_ACT_NONE ? 0 : round256(m * n * elem_size(dtype));
    l.sums = round256(4 * n * ceil_div(m, column_chunk(m)));
    const int64_t bx = plan_bytes(l.px, m, k), bw = plan_bytes(l.pw, n, k);
    l.part = bx > bw ? bx : bw;
    l.total = l.dz + l.sums + l.part;
    return l;
}

template <class T>
int linear_t(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const void *r, int64_t ldr, void *y,
             int64_t ldy, void *z, int64_t m, int64_t n, int64_t k, void *ws, hipStream_t st)
{
    const EpiLinear<T> epi = {(const T *)b, (const T *)r, (T *)y, (T *)z, ldr, ldy, act, (int)n};
    return gemm<T, false, false>(kc((const T *)x, ldx, m), kc((const T *)w, ldw, n), m, n, k, plan(dtype, m, n, k), (float *)ws, epi, st);
}

template <class T>
int linear_backward_t(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *z, const void *dy, int64_t lddy,
                      void *dx, void *dw, void *db, int64_t m, int64_t n, int64_t k, char *ws, hipStream_t st)
{
    const LinearBackward l = linear_backward_layout(dtype, act, m, n, k);
    T *dz = (T *)ws;
    float *sums = (float *)(ws + l.dz), *part = (float *)(ws + l.dz + l.sums);
    const bool own_dz = act != NIRRT_NN_ACT_NONE;
    if (own_dz || db) {
        const int chunk = column_chunk(m), parts = (int)ceil_div(m, chunk);
        if (m > 0) {
            hipLaunchKernelGGL((k_dz<T>), dim3((unsigned)ceil_div(n, 256), (unsigned)parts), dim3(256), 0, st, (const T *)z, (const T *)dy, lddy,
                               own_dz && (dx || dw) ? dz : (T *)nullptr, db ? sums : nullptr, (int)m, (int)n, chunk, act);
        }
        if (db) hipLaunchKernelGGL((k_column_join<T>), dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st, sums, m > 0 ? parts : 0, (T *)db, (int)n);
        if (int rc_ = status()) return rc_;
    }
    const T *d = own_dz ? dz : (const T *)dy;
    const int64_t ldd = own_dz ? n : lddy;
    if (dx && m > 0 && k > 0) {
        const EpiPlain<T> epi = {(T *)dx, nullptr, 1.f, (int)k};
        if (int rc_ = gemm<T, false, true>(kc(d, ldd, m), rc((const T *)w, ldw, k), m, k, n, l.px, part, epi, st)) return rc_;
    }
    if (dw && n > 0 && k > 0) {
        const EpiPlain<T> epi = {(T *)dw, nullptr, 1.f, (int)k};
        if (int rc_ = gemm<T, true, true>(rc(d, ldd, n), rc((const T *)x, ldx, k), n, k, m, l.pw, part, epi, st)) return rc_;
    }
    return 0;
}

// cross entropy: parts of the classes, so that row tiles x parts fill the GPU
struct CeForward { int edge, parts, part; int64_t stats, score, sums, total; };
CeForward ce_layout(int64_t rows, int64_t classes)
{
    CeForward f;
    f.edge = ceil_div(rows, 128) * ceil_div(classes, 128) >= 256 ? 128 : 64;
    const int64_t row_tiles = ceil_div(rows, f.edge), class_tiles = ceil_div(classes, f.edge);
    int64_t parts = ceil_div(512, row_tiles > 0 ? row_tiles : 1);
    if (parts > class_tiles) parts = class_tiles;
    if (parts < 1) parts = 1;
    const int64_t per = ceil_div(class_tiles, parts);
    f.part = (int)(per * f.edge < DIM_MAX ? per * f.edge : DIM_MAX);
    f.parts = (int)(class_tiles > 0 ? ceil_div(class_tiles, per) : 1);
    f.stats = round256(8 * rows * f.parts);
    f.score = round256(4 * rows);
    f.sums = round256(16 * ceil_div(rows, 256));
    f.total = f.stats + f.score + f.sums;
    return f;
}
template <class T>
int ce_forward_t(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target, const float *cw, int64_t ignore,
                 float *lse, float *nll, float *total, int64_t rows, int64_t classes, int64_t k, char *ws, hipStream_t st)
{
    const CeForward f = ce_layout(rows, classes);
    float2 *stats = (float2 *)ws;
    float *score = (float *)(ws + f.stats);
    double *sums = (double *)(ws + f.stats + f.score);
    const int64_t row_tiles = ceil_div(rows, f.edge), blocks = ceil_div(rows, 256);
    if (rows > 0) {
        const dim3 grid((unsigned)row_tiles, (unsigned)f.parts);
        const Operand<T> ow = kc((const T *)w, ldw, classes), ox = kc((const T *)x, ldx, rows);
        if (f.edge == 128)
            hipLaunchKernelGGL((k_ce_stats<T, 128, 128, 2, 2>), grid, dim3(256), 0, st, ow, ox, (const T *)b, target, (int)rows, (int)classes, (int)k,
                               f.part, stats, score);
        else
            hipLaunchKernelGGL((k_ce_stats<T, 64, 64, 2, 2>), grid, dim3(256), 0, st, ow, ox, (const T *)b, target, (int)rows, (int)classes, (int)k,
                               f.part, stats, score);
        hipLaunchKernelGGL(k_ce_rows, dim3((unsigned)blocks), dim3(256), 0, st, stats, f.parts, score, target, cw, ignore, (int)rows, (int)classes,
                           lse, nll, sums);
    }
    hipLaunchKernelGGL(k_ce_total, dim3(1), dim3(256), 0, st, sums, (int)blocks, total);
    return status();
}

constexpr int64_t G_ELEMS = 1ll << 27;    // of g' at a time: pieces of the classes
struct CeBackward { int64_t piece, ldg; Plan px, pw; int64_t g, rel, acc, part, total; };
CeBackward ce_backward_layout(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    CeBackward l;
    l.ldg = (rows + 7) / 8 * 8;
    l.piece = l.ldg > 0 ? G_ELEMS / l.ldg / 128 * 128 : classes;
    if (l.piece < 128) l.piece = 128;
    if (l.piece > classes) l.piece = classes;
    l.px = plan(dtype, rows, k, l.piece);
    l.pw = plan(dtype, l.piece, k, rows);
    l.g = round256(l.ldg * l.piece * elem_size(dtype));
    l.rel = round256(4 * rows) + 256;
    l.acc = l.piece < classes ? round256(4 * rows * k) : 0;
    const int64_t bx = plan_bytes(l.px, rows, k), bw = plan_bytes(l.pw, l.piece, k);
    l.part = bx > bw ? bx : bw;
    l.total = l.g + l.rel + l.acc + l.part;
    return l;
}
template <class T>
int ce_backward_t(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target, const float *cw,
                  int64_t ignore, const float *lse, const float *dloss, int stride, const float *total, void *dx, void *dw, void *db, int64_t rows,
                  int64_t classes, int64_t k, char *ws, hipStream_t st)
{
    const CeBackward l = ce_backward_layout(dtype, rows, classes, k);
    T *g = (T *)ws;
    float *scale = (float *)(ws + l.g), *rel = scale + 64, *acc = (float *)(ws + l.g + l.rel), *part = (float *)(ws + l.g + l.rel + l.acc);
    hipLaunchKernelGGL(k_ce_coefficients, dim3(1), dim3(1024), 0, st, dloss, stride, total, target, cw, ignore, (int)rows, (int)classes, rel, scale);
    const float unlift = 1.f / Factor<T>::VALUE;
    for (int64_t v0 = 0; v0 < classes; v0 += l.piece) {
        const int64_t nv = classes - v0 < l.piece ? classes - v0 : l.piece;
        const T *wp = (const T *)w + v0 * ldw;
        if (rows > 0) {
            const EpiSoftmaxGrad<T> eg = {g, l.ldg, (const T *)b, lse, rel, target, v0};
            Plan pg = plan(dtype, nv, rows, k);
            pg.parts = 1;                    // (the scores are not cut: the softmax needs whole ones)
            pg.part = (int)(k > 0 ? k : 1);
            if (int rc_ = gemm<T, false, false>(kc(wp, ldw, nv), kc((const T *)x, ldx, rows), nv, rows, k, pg, nullptr, eg, st)) return rc_;
        }
        if (db) hipLaunchKernelGGL((k_ce_bias<T>), dim3((unsigned)ceil_div(nv, 4)), dim3(256), 0, st, (const T *)g, l.ldg, (int)rows, (int)nv, scale, (T *)db + v0);
        if (dx && rows > 0 && k > 0) {
            const Operand<T> og = rc((const T *)g, l.ldg, rows), ow = rc(wp, ldw, k);
            int rc_;
            if (l.acc) rc_ = gemm<T, true, true>(og, ow, rows, k, nv, l.px, part, EpiAccumulate{acc, (int)k, v0 == 0}, st);
            else rc_ = gemm<T, true, true>(og, ow, rows, k, nv, l.px, part, EpiPlain<T>{(T *)dx, scale, unlift, (int)k}, st);
            if (rc_) return rc_;
        }
        if (dw && k > 0) {
            const EpiPlain<T> ep = {(T *)dw + v0 * k, scale, unlift, (int)k};
            if (int rc_ = gemm<T, false, true>(kc((const T *)g, l.ldg, nv), rc((const T *)x, ldx, k, rel), nv, k, rows, l.pw, part, ep, st)) return rc_;
        }
    }
    if (dx && l.acc && rows > 0 && k > 0) {
        const int64_t blocks = ceil_div(rows * k, 256);
        hipLaunchKernelGGL((k_cast<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, acc, scale, unlift, (T *)dx, rows * k);
    }
    return status();
}

#define BY_TYPE(dtype, call)                                                                  \
    ((dtype) == NIRRT_NN_F32 ? call(float) : (dtype) == NIRRT_NN_BF16 ? call(bf16_t) : call(f16_t))

bool good_tensors(const nirrt_nn_tensor *t, int32_t count, bool out)
{
    if (count < 0 || (count > 0 && !t)) return false;
    for (int32_t i = 0; i < count; i++)
        if (t[i].n < 0 || !good_type(t[i].dtype) || (t[i].n > 0 && !t[i].data) || (out && (!good_type(t[i].out_dtype) || (t[i].n > 0 && !t[i].out))))
            return false;
    return true;
}
// calls launch(table, first workgroup, workgroups) for every TABLE tensors that hold something; the total of workgroups, < 0 on error
template <class F> int64_t for_tables(const nirrt_nn_tensor *t, int32_t count, F launch)
{
    int64_t done = 0;
    TensorTable tab;
    tab.count = 0;
    int64_t blocks = 0;
    for (int32_t i = 0; i <= count; i++) {
        if (i < count && t[i].n == 0) continue;
        const int64_t b = i < count ? ceil_div(t[i].n, BLOCK_ELEMS) : 0;
        if (b > DIM_MAX / 2) return -1;
        if (tab.count == TABLE || (i == count && tab.count > 0) || (tab.count > 0 && blocks + b > DIM_MAX / 2)) {
            if (launch(tab, done, blocks)) return -2;
            done += blocks;
            blocks = 0;
            tab.count = 0;
        }
        if (i == count) break;
        const int c = tab.count++;
        tab.in[c] = t[i].data;
        tab.out[c] = t[i].out;
        tab.n[c] = t[i].n;
        tab.first[c] = (int)blocks;
        tab.dtype[c] = (uint8_t)t[i].dtype;
        tab.out_dtype[c] = (uint8_t)t[i].out_dtype;
        blocks += b;
    }
    return done;
}

}   // namespace

extern "C" int64_t nirrt_nn_linear_workspace(int dtype, int64_t m, int64_t n, int64_t k)
{
    if (!good_type(dtype) || !good_dims(m, n, k)) return -1;
    return plan_bytes(plan(dtype, m, n, k), m, n);
}

extern "C" int nirrt_nn_linear(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const void *r, int64_t ldr,
                               void *y, int64_t ldy, void *z, int64_t m, int64_t n, int64_t k, void *workspace, void *stream)
{
    if (!good_type(dtype) || act < 0 || act > NIRRT_NN_ACT_SILU || !good_dims(m, n, k)) return -1;
    if (m == 0 || n == 0) return 0;
    if (!y || (k > 0 && (!x || !w)) || ldx < k || ldw < k || ldy < n || (r && ldr < n)) return -1;
    if (nirrt_nn_linear_workspace(dtype, m, n, k) > 0 && !workspace) return -1;
#define CALL(T) linear_t<T>(dtype, act, x, ldx, w, ldw, b, r, ldr, y, ldy, z, m, n, k, workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_linear_backward_workspace(int dtype, int act, int64_t m, int64_t n, int64_t k)
{
    if (!good_type(dtype) || act < 0 || act > NIRRT_NN_ACT_SILU || !good_dims(m, n, k)) return -1;
    return linear_backward_layout(dtype, act, m, n, k).total;
}

extern "C" int nirrt_nn_linear_backward(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *z, const void *dy,
                                        int64_t lddy, void *dx, void *dw, void *db, int64_t m, int64_t n, int64_t k, void *workspace, void *stream)
{
    if (!good_type(dtype) || act < 0 || act > NIRRT_NN_ACT_SILU || !good_dims(m, n, k)) return -1;
    if (m > 0 && n > 0 && (!dy || lddy < n || (act != NIRRT_NN_ACT_NONE && !z))) return -1;
    if (((dx || dw) && (ldx < k || ldw < k)) || (dx && m > 0 && n > 0 && k > 0 && !w) || (dw && m > 0 && n > 0 && k > 0 && !x)) return -1;
    if (!workspace && linear_backward_layout(dtype, act, m, n, k).total > 0) return -1;
#define CALL(T) linear_backward_t<T>(dtype, act, x, ldx, w, ldw, z, dy, lddy, dx, dw, db, m, n, k, (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_cross_entropy_workspace(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    if (!good_type(dtype) || !good_dims(rows, classes, k) || classes < 1) return -1;
    return ce_layout(rows, classes).total;
}

extern "C" int nirrt_nn_cross_entropy(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target,
                                      const float *class_weight, int64_t ignore_index, float *lse, float *nll, float *total, int64_t rows,
                                      int64_t classes, int64_t k, void *workspace, void *stream)
{
    if (!good_type(dtype) || !good_dims(rows, classes, k) || classes < 1 || !total || ldx < k || ldw < k) return -1;
    if (rows > 0 && (!target || !lse || !nll || !workspace || (k > 0 && (!x || !w)))) return -1;
#define CALL(T) ce_forward_t<T>(x, ldx, w, ldw, b, target, class_weight, ignore_index, lse, nll, total, rows, classes, k, (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_cross_entropy_backward_workspace(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    if (!good_type(dtype) || !good_dims(rows, classes, k) || classes < 1) return -1;
    return ce_backward_layout(dtype, rows, classes, k).total;
}

extern "C" int nirrt_nn_cross_entropy_backward(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b,
                                               const int64_t *target, const float *class_weight, int64_t ignore_index, const float *lse,
                                               const float *dloss, int dloss_stride, const float *total, void *dx, void *dw, void *db,
                                               int64_t rows, int64_t classes, int64_t k, void *workspace, void *stream)
{
    if (!good_type(dtype) || !good_dims(rows, classes, k) || classes < 1 || ldx < k || ldw < k || !workspace) return -1;
    if (dloss_stride != 0 && dloss_stride != 1) return -1;
    if (rows > 0 && (!target || !lse || !dloss || (k > 0 && (!x || !w)))) return -1;
#define CALL(T)                                                                                                                                  \
    ce_backward_t<T>(dtype, x, ldx, w, ldw, b, target, class_weight, ignore_index, lse, dloss, dloss_stride, total, dx, dw, db, rows, classes, k, \
                     (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_norm_workspace(const nirrt_nn_tensor *tensors, int32_t count)
{
    if (!good_tensors(tensors, count, false)) return -1;
    int64_t blocks = 0;
    for (int32_t i = 0; i < count; i++) blocks += ceil_div(tensors[i].n, BLOCK_ELEMS);
    return round256(8 * blocks);
}

extern "C" int nirrt_nn_norm(const nirrt_nn_tensor *tensors, int32_t count, float *norm, void *workspace, void *stream)
{
    if (!good_tensors(tensors, count, false) || !norm) return -1;
    if (!workspace && nirrt_nn_norm_workspace(tensors, count) > 0) return -1;
    hipStream_t st = (hipStream_t)stream;
    double *parts = (double *)workspace;
    const int64_t blocks = for_tables(tensors, count, [&](const TensorTable &t, int64_t first, int64_t n) {
        hipLaunchKernelGGL(k_norm_parts, dim3((unsigned)n), dim3(256), 0, st, t, parts + first);
        return status();
    });
    if (blocks < 0) return (int)blocks;
    hipLaunchKernelGGL(k_norm_total, dim3(1), dim3(256), 0, st, parts, blocks, norm);
    return status();
}

extern "C" int nirrt_nn_scale_by_norm(const nirrt_nn_tensor *tensors, int32_t count, const float *norm, float max_norm, void *stream)
{
    if (!good_tensors(tensors, count, true) || !norm || !(max_norm >= 0.f)) return -1;
    hipStream_t st = (hipStream_t)stream;
    const int64_t blocks = for_tables(tensors, count, [&](const TensorTable &t, int64_t, int64_t n) {
        hipLaunchKernelGGL(k_scale, dim3((unsigned)n), dim3(256), 0, st, t, norm, max_norm);
        return status();
    });
    return blocks < 0 ? (int)blocks : 0;
}
