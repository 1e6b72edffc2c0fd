// nnops.hip - the dense operators of the guidance network's layers and of its training step (C ABI: include/nirrt_nnops.h).
//
//   linear          y = act(x w^T + b) + r, and its gradients
//   cross entropy   softmax cross entropy of the scores x w^T + b without keeping them, and its gradients
//   norm / scale    2-norm of many tensors, and the clipping by it
//
// Products of more than 32 rows run on MFMA (16 x 16 x 32 or 32 x 32 x 16 for 16-bit, 32 x 32 x 2 for 32-bit operands): a workgroup of 4 or 8 waves owns a tile C[i, j] = sum_k A[i, k] B[j, k].  An operand is
// stored either with k contiguous ("KC": x, w in the forward product) or with i contiguous ("RC": w in dx = dz w, dz and x in dw = dz^T x).
// Two tile loops: DirectTile for operands of whole aligned 16-byte chunks (memory -> LDS, a ring of four stages), Tile for all others
// (memory -> registers -> LDS).  A lane's 16 bytes are one operand of a 16-bit MFMA (8 k) or four of a 32-bit one (4 x 1 k); the order of k
// inside a step is the same in A and B, so the sum is the same whatever it is.  Accumulators and partial sums are fp32.
//
// Times are those of an MI355X that copies at 5.1 TB/s; its library's products reach 1135 - 1290 TFLOP/s (bf16) and 131 (fp32).  For 16384 x 4096 x
// 4096 in bf16: 585 us forward with z, r and y in the epilogue, 506 dx, 476 dw (1155 TFLOP/s; the library 425 - 480 for the product); under
// these kernels the clock falls to 1.5 GHz (power).
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

// 8 lanes on 8 neighbouring (or every 4th) rows: 8 places; rows 32 apart: the same (their addresses differ by a constant)
__device__ __forceinline__ int sw(int row) { return (row ^ ((row >> 3) & 3)) & 7; }

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

typedef float f32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4_t mma16(bf16_t, u32x4 a, u32x4 b, f32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma16(f16_t, u32x4 a, u32x4 b, f32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma16(float, u32x4 a, u32x4 b, f32x4_t c)
{
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
}

// one operand: element (r, k) at p[r * ld + k] (KC) or p[k * ld + r] (RC); an RC operand counts as zeros from k = depth on
template <class T> struct Operand {
    const T *p;
    int64_t ld;
    int rows, depth;
};

// N elements from any address of their type (the hardware takes vector loads off their alignment)
template <class T, int N> struct Pack { T e[N]; };
template <class T, int N> __device__ __forceinline__ Pack<T, N> load_pack(const T *p)
{
    Pack<T, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class T, int N> __device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &v) { __builtin_memcpy(p, &v, sizeof(v)); }
// the first n of them only (zeros behind)
template <class T, int N> __device__ __forceinline__ Pack<T, N> load_some(const T *p, int n)
{
    if (n >= N) return load_pack<T, N>(p);
    Pack<T, N> v;
#pragma unroll
    for (int e = 0; e < N; e++) v.e[e] = e < n ? p[e] : (T)0.f;
    return v;
}
template <class T, int N> __device__ __forceinline__ void store_some(T *p, const Pack<T, N> &v, int n)
{
    if (n >= N) { store_pack(p, v); return; }
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e < n) p[e] = v.e[e];
}

// a thread's share of one K-step (128 bytes per row) of R rows: global memory -> registers -> LDS.  There both kinds look alike: rows of
// eight 16-byte chunks along k, chunk c of row r at place c ^ sw(r); an RC operand is transposed in registers on its way.
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
                    if (k + CE <= k1) __builtin_memcpy(&x, q, 16);
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
                    if (k + j < k1 && k + j < o.depth && row < o.rows) {
                        if (row + VR <= o.rows) __builtin_memcpy(f, q, VR * sizeof(T));
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

// The tile of C that a wave holds: MI x NI blocks of 32 x 32, 16 registers of a lane each.  SUB = 1, one 32 x 32 MFMA: register e is row 8 (e / 4) +
// 4 (lane / 32) + e % 4, column lane % 32.  SUB = 2, four 16 x 16 ones: row 16 (e / 8) + 4 (lane / 16) + e % 4, column 16 (e / 4 % 2) + lane % 16.
template <int SUB> __device__ __forceinline__ int block_row(int lane, int e) { return SUB == 2 ? 16 * (e >> 3) + 4 * (lane >> 4) + (e & 3) : 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }
template <int SUB> __device__ __forceinline__ int block_col(int lane, int e) { return SUB == 2 ? 16 * ((e >> 2) & 1) + (lane & 15) : lane & 31; }
template <class T, int BM, int BN, int WM, int WN, bool RCA, bool RCB> struct Tile {
    static constexpr int NT = 64 * WM * WN, WAVES_M = WM, WAVES_N = WN, MI = BM / WM / 32, NI = BN / WN / 32;
    static constexpr int LDS_CHUNKS = (BM + BN) * CHUNKS, SUB = 1;
    f32x16 acc[MI][NI];
    __device__ __forceinline__ float get(int mi, int ni, int e) const { return acc[mi][ni][e]; }

    static __device__ __forceinline__ int first_row(int wave) { return (wave / WN) * (BM / WM); }
    static __device__ __forceinline__ int first_col(int wave) { return (wave % WN) * (BN / WN); }

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

// ---- the same tile with operands that go from global memory to the LDS directly ---------------------------------------------------
// For operands whose 16-byte chunks are aligned and whole (see direct()): buffer loads write the LDS without passing through registers,
// out-of-range offsets give zeros.  The LDS place of a lane's chunk is fixed (base + 16 lane), so the swizzle is applied to the global
// address.  A KC operand lies as in Tile; an RC operand lies as it is, STEP rows of k with R elements each, and is transposed on its way
// out: 16-bit by the transposing LDS read (4 k x 16 rows per 16 lanes), 32-bit because an MFMA operand is one element per lane anyway.
// Four stages of 64 bytes of k per row, in a ring: one is multiplied, the next has arrived (its first operands are read during the last
// products of this one), two are on their way - a stage's loads have two steps of products to arrive in, and the barrier between steps finds
// every wave's products still running.  (Two stages of 128 bytes, each waited for whole: 58 % of the MFMA cycles busy, 600 us for
// 16384 x 4096 x 4096 in bf16.)
constexpr int STAGES = 4, RING_BYTES = 64, RING_CHUNKS = RING_BYTES / 16;
__device__ __forceinline__ int ring_sw(int row) { return (row >> 2) & 3; }   // 16 lanes on 16 rows: 16 places of 16 bytes
constexpr unsigned NOWHERE = 0x7ffffff0u;   // an offset beyond every buffer (direct() keeps them below)

// 16 bytes per lane from buffer + offset to lds + 16 lane.  Written out, because the compiler does not know which part of the LDS a load of its
// own writes, and would wait for all of them before every read.  It has no result register; the waits are arrive() below, which every use of
// the LDS stands behind.  m0 is a reserved register: the compiler keeps no value in it and writes it right before a use of its own, of which
// these kernels have none (naming it as clobbered is answered with a warning and changes nothing).
__device__ __forceinline__ void load_to_lds(u32x4 buffer, const u32x4 *lds, unsigned offset)
{
#ifdef __HIP_DEVICE_COMPILE__
    const unsigned where = (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void *)lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(where), "v"(offset), "s"(buffer) : "memory");
#endif
}

template <class T, int R, int NT, bool RC> struct DirectOperand {
    static constexpr int CE = Elem<T>::PER_CHUNK, STEP = RING_BYTES / sizeof(T), N = R * RING_CHUNKS / NT, PER_K = R / CE;
    const char *base;          // of the step to load next
    int64_t bytes, advance;    // valid bytes from base on, per step
    unsigned at[N];            // a lane's offset in a step
    int first;                 // KC: the first k of its chunk (the same in all N: rows NT / 4 apart have the same swizzle)

    // 16-byte blocks of an RC row are moved by whole bank groups: 64 bytes by k mod 4 and 32 by k / 8 (16-bit: a transposing read takes 4 k x 32
    // bytes per 16 lanes, their neighbours the k 8 on), 128 bytes by k / 4 (32-bit: the halves of a wave read k 4 apart)
    static __device__ __forceinline__ int turn(int k) { return sizeof(T) == 2 ? ((R >= 128 ? k & 3 : k & 1) << 2) | ((k >> 3) & 1) << 1 : ((k >> 2) & 1) << 3; }

    __device__ __forceinline__ void start(const Operand<T> &o, int r0, int k0, int k1, int tid)
    {
        const int64_t row_bytes = o.ld * (int64_t)sizeof(T);
        if constexpr (!RC) {
            const int rows = o.rows - r0 < R ? o.rows - r0 : R;
            base = (const char *)(o.p + (int64_t)r0 * o.ld + k0);
            bytes = (rows - 1) * row_bytes + (int64_t)(k1 - k0) * sizeof(T);
            advance = RING_BYTES;
        } else {
            base = (const char *)(o.p + (int64_t)k0 * o.ld + r0);
            // (whole 4-byte words count as in or out of range: the last one belongs to the row even if only half of it does)
            bytes = ((int64_t)((k1 < o.depth ? k1 : o.depth) - k0 - 1) * row_bytes + (int64_t)(o.rows - r0) * sizeof(T) + 3) & ~3ll;
            advance = STEP * row_bytes;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int p = i * NT + tid;
            if constexpr (!RC) {
                const int r = p / RING_CHUNKS, c = (p % RING_CHUNKS) ^ ring_sw(r);
                at[i] = (unsigned)(r * row_bytes + c * 16);
                first = c * CE;
            } else {
                const int k = p / PER_K, c = (p % PER_K) ^ turn(k);
                at[i] = (unsigned)(k * row_bytes + c * 16);
                first = 0;
            }
        }
    }
    // one of the N loads of a step (left: k still to come, this step's included); next() moves on
    __device__ __forceinline__ void load(const u32x4 *lds, int i, int left, int wave) const
    {
        const int64_t lim = bytes < (int64_t)NOWHERE ? bytes : (int64_t)NOWHERE;      // (below zero behind the end: an empty buffer)
        const u32x4 buffer = {(unsigned)(uintptr_t)base, (unsigned)((uintptr_t)base >> 32) & 0xffffu, (unsigned)(lim > 0 ? lim : 0), 0x00020000u};
        load_to_lds(buffer, lds + i * NT + wave * 64, RC || first < left ? at[i] : NOWHERE);
    }
    __device__ __forceinline__ void next()
    {
        base += advance;
        bytes -= advance;
    }
};

// Reads MFMA operands from an operand's part of a stage: the lane's byte offsets are kept, so that everything else is a constant in the
// instruction.  16-bit: a stage is one MFMA's k, M is counted in blocks of 16 rows (s = 0).  32-bit: two groups s of 32 bytes of k, M blocks of 32 rows.
template <class T, int R, bool RC, int M> struct Reader {
    static constexpr bool HALF = sizeof(T) == 2;
    int at[RC ? M : HALF ? 1 : 2];

    __device__ __forceinline__ void start(int row0, int lane, int where)
    {
        typedef DirectOperand<T, R, 64, true> Op;
        const int i = lane & 15;
        if constexpr (!RC && HALF) {
            const int r = row0 + i;
            at[0] = where + r * RING_BYTES + ((lane >> 4) ^ ring_sw(r)) * 16;
        } else if constexpr (!RC) {
            const int r = row0 + (lane & 31), c = (lane >> 5) ^ ring_sw(r);
#pragma unroll
            for (int s = 0; s < 2; s++) at[s] = where + r * RING_BYTES + (c ^ (2 * s)) * 16;
        } else {
            const int k = HALF ? 8 * (lane >> 4) + (i >> 2) : 4 * (lane >> 5), row = row0 + (HALF ? 4 * (i & 3) : lane & 31);
#pragma unroll
            for (int m = 0; m < M; m++) at[m] = where + k * (R * (int)sizeof(T)) + (((row + (HALF ? 16 : 32) * m) * (int)sizeof(T)) ^ (Op::turn(k) * 16));
        }
    }
    __device__ __forceinline__ u32x4 read(const u32x4 *lds, int stage, int m, int s) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        const __attribute__((address_space(3))) char *p = (const __attribute__((address_space(3))) char *)lds + stage;
        if constexpr (!RC) {
            return *(const __attribute__((address_space(3))) u32x4 *)(p + at[HALF ? 0 : s] + m * (HALF ? 16 : 32) * RING_BYTES);
        } else if constexpr (HALF) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            s16x4 q[2];
#pragma unroll
            for (int h = 0; h < 2; h++) q[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p + at[m] + 4 * h * (R * 2)));
            u32x4 v;
            __builtin_memcpy(&v, q, 16);
            return v;
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = *(const __attribute__((address_space(3))) unsigned *)(p + at[m] + (8 * s + j) * (R * 4));
            return v;
        }
#else
        return u32x4{};
#endif
    }
};

// all but the newest `left` loads of every wave of the workgroup have arrived
template <int left> __device__ __forceinline__ void arrive()
{
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(left) : "memory");
#endif
}

template <class T, int BM, int BN, int WM, int WN, bool RCA, bool RCB> struct DirectTile {
    static constexpr int NT = 64 * WM * WN, WAVES_M = WM, WAVES_N = WN, MI = BM / WM / 32, NI = BN / WN / 32;
    static constexpr int STAGE = (BM + BN) * RING_CHUNKS, LDS_CHUNKS = STAGES * STAGE, STEP = RING_BYTES / sizeof(T);
    // 16-bit: 16 x 16 x 32 MFMA, FA x FB blocks.  Half the accumulator traffic of 32 x 32 x 16, which is what the clock allows under power:
    // 2090 against 1860 TFLOP/s for nothing but MFMA of normal numbers, 1484 -> 1455 us for a training step of 16384 x 4096 x 4096.
    static constexpr int SUB = sizeof(T) == 2 ? 2 : 1, FA = MI * SUB, FB = NI * SUB;
    f32x16 acc[SUB == 1 ? MI : 1][SUB == 1 ? NI : 1];
    f32x4_t acc4[SUB == 2 ? FA : 1][SUB == 2 ? FB : 1];
    __device__ __forceinline__ float get(int mi, int ni, int e) const
    {
        if constexpr (SUB == 2) return acc4[2 * mi + (e >> 3)][2 * ni + ((e >> 2) & 1)][e & 3];
        else return acc[mi][ni][e];
    }

    static __device__ __forceinline__ int first_row(int wave) { return (wave / WN) * (BM / WM); }
    static __device__ __forceinline__ int first_col(int wave) { return (wave % WN) * (BN / WN); }

    typedef DirectOperand<T, BM, NT, RCA> OpA;
    typedef DirectOperand<T, BN, NT, RCB> OpB;
    static constexpr int LOADS = OpA::N + OpB::N;      // per wave and stage
    static __device__ __forceinline__ void load(const OpA &oa, const OpB &ob, u32x4 *stage, int i, int left, int wave)
    {
        if (i < OpA::N) oa.load(stage, i, left, wave);
        else ob.load(stage + BM * RING_CHUNKS, i - OpA::N, left, wave);
    }

    // a step of 16-bit products: a row of FB blocks at a time.  In between, the A operand two rows on, the B operands of the next stage and the
    // loads of three stages on (the memory pipe takes a load of a wave in 16 cycles: all of a step's at once hold up the products behind them)
    template <int P> __device__ __forceinline__ void step(const OpA &oa, const OpB &ob, const Reader<T, BM, RCA, FA> &xa, const Reader<T, BN, RCB, FB> &xb,
                                                          u32x4 (&fa)[4], u32x4 (&fb)[2][FB], u32x4 *lds, int now, int next, int free, int left, int wave)
    {
        constexpr int AT = FA % 4 ? FA * P : 0;          // where the stage's A operands begin in the ring of four registers
#pragma unroll
        for (int i = 0; i < FA; i++) {
            fa[(AT + i + 2) & 3] = xa.read(lds, (i + 2 < FA ? now : next) * 16, (i + 2) % FA, 0);
#pragma unroll
            for (int j = 0; j < FB; j++)
                if (j * FA / FB == i) fb[1 - P][j] = xb.read(lds, next * 16, j, 0);
#pragma unroll
            for (int l = 0; l < LOADS; l++)
                if (l * FA / LOADS == i) load(oa, ob, lds + free, l, left, wave);
            __builtin_amdgcn_sched_barrier(0);           // (left alone, the compiler reads behind the products and waits)
#pragma unroll
            for (int j = 0; j < FB; j++) acc4[i][j] = mma16((T)0.f, fa[(AT + i) & 3], fb[P][j], acc4[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // a step of 32-bit products: two groups of 16 bytes of k per half wave
    __device__ __forceinline__ void step(const OpA &oa, const OpB &ob, const Reader<T, BM, RCA, FA> &xa, const Reader<T, BN, RCB, FB> &xb, u32x4 (&fa)[2][MI],
                                         u32x4 (&fb)[2][NI], u32x4 *lds, int now, int next, int free, int left, int wave)
    {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int mi = 0; mi < MI; mi++) {
                fa[1 - s][mi] = xa.read(lds, (s ? next : now) * 16, mi, 1 - s);
#pragma unroll
                for (int ni = 0; ni < NI; ni++)
                    if (ni * MI / NI == mi) fb[1 - s][ni] = xb.read(lds, (s ? next : now) * 16, ni, 1 - s);
#pragma unroll
                for (int i = 0; i < LOADS; i++)
                    if (i * 2 * MI / LOADS == s * MI + mi) load(oa, ob, lds + free, i, left, wave);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ni = 0; ni < NI; ni++) acc[mi][ni] = mma((T)0.f, fa[s][mi], fb[s][ni], acc[mi][ni]);
                __builtin_amdgcn_sched_barrier(0);
            }
    }

    __device__ __forceinline__ void mainloop(const Operand<T> &a, const Operand<T> &b, int i0, int j0, int k0, int k1, u32x4 *lds)
    {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        if constexpr (SUB == 2) {
#pragma unroll
            for (int i = 0; i < FA; i++)
#pragma unroll
                for (int j = 0; j < FB; j++) acc4[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int mi = 0; mi < MI; mi++)
#pragma unroll
                for (int ni = 0; ni < NI; ni++)
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[mi][ni][e] = 0.f;
        }
        if (k0 >= k1) return;
        OpA oa;
        OpB ob;
        oa.start(a, i0, k0, k1, tid);
        ob.start(b, j0, k0, k1, tid);
        Reader<T, BM, RCA, FA> xa;
        Reader<T, BN, RCB, FB> xb;
        xa.start(first_row(wave), lane, 0);
        xb.start(first_col(wave), lane, BM * RING_BYTES);
        __syncthreads();                     // (a tile before this one has been read)
        int left = k1 - k0;                  // k that have not been asked for; behind the end the loads give zeros, the count stays even
#pragma unroll
        for (int p = 0; p < STAGES - 1; p++) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) load(oa, ob, lds + p * STAGE, i, left, wave);
            oa.next();
            ob.next();
            left -= STEP;
        }
        arrive<LOADS>();
        int now = 0, next, free;             // this stage's place in the ring, in chunks; the next one's; the one that has been read
        const auto turn = [&] {
            next = now + STAGE == LDS_CHUNKS ? 0 : now + STAGE;
            free = now == 0 ? LDS_CHUNKS - STAGE : now - STAGE;
        };
        const auto done = [&] {
            oa.next();
            ob.next();
            left -= STEP;
            arrive<LOADS>();
            now = next;
        };
        if constexpr (SUB == 2) {
            u32x4 fa[4], fb[2][FB];
            fa[0] = xa.read(lds, 0, 0, 0);
            fa[1] = xa.read(lds, 0, 1, 0);
#pragma unroll
            for (int j = 0; j < FB; j++) fb[0][j] = xb.read(lds, 0, j, 0);
            int k = k0;
            for (; k + STEP < k1; k += 2 * STEP) {
                turn();
                step<0>(oa, ob, xa, xb, fa, fb, lds, now, next, free, left, wave);
                done();
                turn();
                step<1>(oa, ob, xa, xb, fa, fb, lds, now, next, free, left, wave);
                done();
            }
            if (k < k1) {
                turn();
                step<0>(oa, ob, xa, xb, fa, fb, lds, now, next, free, left, wave);
            }
        } else {
            u32x4 fa[2][MI], fb[2][NI];
#pragma unroll
            for (int mi = 0; mi < MI; mi++) fa[0][mi] = xa.read(lds, 0, mi, 0);
#pragma unroll
            for (int ni = 0; ni < NI; ni++) fb[0][ni] = xb.read(lds, 0, ni, 0);
            for (int k = k0; k < k1; k += STEP) {
                turn();
                step(oa, ob, xa, xb, fa, fb, lds, now, next, free, left, wave);
                done();
            }
        }
        arrive<0>();                         // (the loads behind the end)
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
// Phi(z) and e = exp(-z^2 / 2) (its density is 0.3989 e): Phi(-|z|) = 1/2 erfcx(|z| / sqrt 2) e, erfcx as a polynomial of degree 9 in
// t = 1 / (1 + 0.3 x) (weighted least squares on x in [0, 14]: relative error 6.5e-8; behind it e is 0).  A sixth of erfcf's instructions.
__device__ __forceinline__ float normal_cdf(float z, float &e)
{
    const float a = __builtin_fabsf(z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.21213203435596426f, a, 1.f));
    float q = -0.12661783397197723f;
    q = __builtin_fmaf(q, t, 0.471831738948822f);
    q = __builtin_fmaf(q, t, -0.4847019910812378f);
    q = __builtin_fmaf(q, t, 0.5170591473579407f);
    q = __builtin_fmaf(q, t, -0.07405535876750946f);
    q = __builtin_fmaf(q, t, 0.206387460231781f);
    q = __builtin_fmaf(q, t, 0.1504683643579483f);
    q = __builtin_fmaf(q, t, 0.17042377591133118f);
    q = __builtin_fmaf(q, t, 0.16920475661754608f);
    e = __expf(-0.5f * z * z);
    const float tail = 0.5f * q * t * e;
    return z > 0.f ? 1.f - tail : tail;
}
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float act_value(int act, float z)
{
    float e;
    switch (act) {
    case NIRRT_NN_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);          // (NaN stays)
    case NIRRT_NN_ACT_GELU: return z * normal_cdf(z, e);
    case NIRRT_NN_ACT_SILU: return z * logistic(z);
    default: return z;
    }
}
__device__ __forceinline__ float act_slope(int act, float z)
{
    float e;
    switch (act) {
    case NIRRT_NN_ACT_RELU: return z > 0.f ? 1.f : (z == z ? 0.f : z);        // (NaN stays)
    case NIRRT_NN_ACT_GELU: { const float c = normal_cdf(z, e); return __builtin_fmaf(z * 0.39894228040143268f, e, c); }
    case NIRRT_NN_ACT_SILU: { const float s = logistic(z); return s * (1.f + z * (1.f - s)); }
    default: return 1.f;
    }
}

// ---- what a product does with four neighbouring elements C[i, j ..] of Q rows (row q: i + q step; rows of them exist, n columns) ---------
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <class T> __device__ __forceinline__ f32x4 load4(const T *p, int n)
{
    const Pack<T, 4> q = load_some<T, 4>(p, n);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)q.e[e];
    return v;
}
template <class T> __device__ __forceinline__ void store4(T *p, f32x4 v, int n)
{
    Pack<T, 4> q;
#pragma unroll
    for (int e = 0; e < 4; e++) q.e[e] = (T)v[e];
    store_some(p, q, n);
}
// y = act(C + b[j]) + r, and z in the element type, as y is: half the bytes for 16-bit types, and gradients that move by 6e-4 of themselves in
// bf16 (2-norms, 4097 x 321 x 515 and 4096 x 4096 x 4096), where the rounding of a result is 1.7e-3
template <class T> struct EpiLinear {
    const T *b, *r;
    T *y, *z;
    int64_t ldr, ldy;
    int act, n;
    template <int Q> __device__ __forceinline__ void put(f32x4 (&c)[Q], int i, int step, int rows, int j, int cnt) const
    {
        if (b) {
            const f32x4 add = load4(b + j, cnt);
#pragma unroll
            for (int q = 0; q < Q; q++) c[q] += add;
        }
        if (z) {
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (q < rows) store4(z + (int64_t)(i + q * step) * n + j, c[q], cnt);
        }
        if (act != NIRRT_NN_ACT_NONE) {
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int e = 0; e < 4; e++) c[q][e] = act_value(act, c[q][e]);
        }
        if (r) {
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (q < rows) c[q] += load4(r + (int64_t)(i + q * step) * ldr + j, cnt);
        }
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q < rows) store4(y + (int64_t)(i + q * step) * ldy + j, c[q], cnt);
    }
};
// out = scale C (contiguous rows of n); scale on the device or 1
template <class T> struct EpiPlain {
    T *out;
    const float *scale;
    float factor;
    int n;
    template <int Q> __device__ __forceinline__ void put(f32x4 (&c)[Q], int i, int step, int rows, int j, int cnt) const
    {
        const float f = scale ? *scale * factor : factor;
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q < rows) store4(out + (int64_t)(i + q * step) * n + j, c[q] * f, cnt);
    }
};
// acc (+)= C in fp32: the sum over pieces of the reduction that are multiplied one after the other
template <class T> struct EpiAccumulate {
    float *out;
    int n, first;
    template <int Q> __device__ __forceinline__ void put(f32x4 (&c)[Q], int i, int step, int rows, int j, int cnt) const
    {
        if (!first) {
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (q < rows) c[q] += load4(out + (int64_t)(i + q * step) * n + j, cnt);
        }
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q < rows) store4(out + (int64_t)(i + q * step) * n + j, c[q], cnt);
    }
};
// a part of a cut reduction: part p at out + p m n
struct EpiPart {
    float *out;
    int n;
    template <int Q> __device__ __forceinline__ void put(f32x4 (&c)[Q], int i, int step, int rows, int j, int cnt) const
    {
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q < rows) store4(out + (int64_t)(i + q * step) * n + j, c[q], cnt);
    }
};

// BM x BN tiles, the reduction cut into gridDim.y parts of `part`; with more than one, the parts go to `partial` (part, i, j) for k_join.
// A wave hands its accumulators to the epilogue through the LDS, 32 rows at a time: an MFMA block has a row's elements in 32 lanes, the
// epilogue wants four of a row in one (16-byte accesses, and code once instead of once per accumulator register).
template <class T, int BM, int BN, class Tl, class Epi>
__global__ __launch_bounds__(Tl::NT) void k_gemm(Operand<T> a, Operand<T> b, int m, int n, int k, int part, float *partial, Epi epi)
{
    constexpr int COLS = Tl::NI * 32, LD = COLS + 4, SLAB = 32 * LD / 4;      // (4 more: rows 4 apart start in other banks)
    __shared__ u32x4 lds[Tl::LDS_CHUNKS > SLAB * (Tl::NT / 64) ? Tl::LDS_CHUNKS : SLAB * (Tl::NT / 64)];
    Tl t;
    int ti, tj;
    tile_of(blockIdx.x, gridDim.x, (m + BM - 1) / BM, (n + BN - 1) / BN, ti, tj);
    const int k0 = blockIdx.y * part, k1 = k - k0 < part ? k : k0 + part;
    t.mainloop(a, b, ti * BM, tj * BN, k0, k1, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i0 = ti * BM + Tl::first_row(wave), j0 = tj * BN + Tl::first_col(wave);
    float *slab = (float *)(lds + wave * SLAB);
    constexpr int PER_ROW = COLS / 4, STEP = 64 / PER_ROW, Q = 32 / STEP;     // lanes per row, rows per pass, passes
    const int r = lane / PER_ROW, c = lane % PER_ROW * 4, j = j0 + c, cnt = n - j < 4 ? n - j : 4;
    const EpiPart part_out = {partial + (int64_t)blockIdx.y * m * n, n};
    __syncthreads();                        // (the last step has been read)
#pragma unroll
    for (int mi = 0; mi < Tl::MI; mi++) {
#pragma unroll
        for (int ni = 0; ni < Tl::NI; ni++)
#pragma unroll
            for (int e = 0; e < 16; e++) slab[block_row<Tl::SUB>(lane, e) * LD + ni * 32 + block_col<Tl::SUB>(lane, e)] = t.get(mi, ni, e);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f32x4 v[Q];
#pragma unroll
        for (int q = 0; q < Q; q++) v[q] = *(const f32x4 *)(slab + (q * STEP + r) * LD + c);
        const int i = i0 + 32 * mi + r, left = m - i, rows = left <= 0 || cnt <= 0 ? 0 : (left - 1) / STEP + 1;
        if (gridDim.y > 1) part_out.put(v, i, STEP, rows, j, cnt);
        else if (rows >= Q && cnt == 4) epi.put(v, i, STEP, Q, j, 4);         // (nothing to check)
        else if (rows > 0) epi.put(v, i, STEP, rows, j, cnt);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}
// ---- few rows (m <= 32): every weight is read for a handful of rows, so what bounds the product is reading w ---------------------------------
// A workgroup of eight waves owns 16 columns; each wave takes every eighth step of 64 bytes per row of w, eight steps in flight (8 KB per
// wave: some 64 KB per CU cover the latency), multiplies them on 16 x 16 MFMA with the rows of x straight from memory, and the waves' sums
// meet in the LDS.  One launch, nothing cut, no workspace.  7 x 4096 x 4096 in fp16: 9.8 us, 3.4 TB/s of w (a cut 64-wide tile and its join: 9 + 4 us).
template <class T> __device__ __forceinline__ u32x4 chunk_of(const T *row, int at, int k)
{
    constexpr int P = 16 / sizeof(T);
    Pack<T, P> v = {};
    if (at < k) v = load_some<T, P>(row + at, k - at);
    return __builtin_bit_cast(u32x4, v);
}
template <class T, int MT, class Epi>
__global__ __launch_bounds__(512) void k_few_rows(const T *x, int64_t ldx, const T *w, int64_t ldw, int m, int n, int k, Epi epi)
{
    constexpr int P = 16 / sizeof(T), STEP = 4 * P, DEPTH = 8, ROUND = 8 * STEP;     // elements: a wave's step, all waves' steps
    __shared__ f32x4_t meet[8][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, c = wave * STEP + (lane >> 4) * P, j0 = blockIdx.x * 16;
    // (rows behind the last are the last once more: their results go nowhere)
    const T *wr = w + (int64_t)(j0 + r < n ? j0 + r : n - 1) * ldw + c, *xr[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) xr[t] = x + (int64_t)(16 * t + r < m ? 16 * t + r : m - 1) * ldx + c;
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    int k0 = 0;
    for (; k0 + DEPTH * ROUND <= k; k0 += DEPTH * ROUND) {       // whole steps of all waves: nothing to check
        u32x4 a[MT][DEPTH], b[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; d++) b[d] = __builtin_bit_cast(u32x4, load_pack<T, P>(wr + k0 + d * ROUND));
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int d = 0; d < DEPTH; d++) a[t][d] = __builtin_bit_cast(u32x4, load_pack<T, P>(xr[t] + k0 + d * ROUND));
#pragma unroll
        for (int d = 0; d < DEPTH; d++)
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = mma16((T)0.f, a[t][d], b[d], acc[t]);
    }
    for (; k0 < k; k0 += ROUND) {
        const u32x4 b = chunk_of(wr, k0, k - c);
#pragma unroll
        for (int t = 0; t < MT; t++) acc[t] = mma16((T)0.f, chunk_of(xr[t], k0, k - c), b, acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; t++) meet[wave][t][lane] = acc[t];
    __syncthreads();
    // element (row, column) of a 16 x 16 block: register row % 4 of lane 16 (row / 4) + column
    if (threadIdx.x < 64 * MT) {
        const int t = threadIdx.x >> 6, row = (threadIdx.x & 63) >> 2, cc = (threadIdx.x & 3) * 4, i = 16 * t + row, j = j0 + cc;
        f32x4 v[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int p = 0; p < 8; p++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[0][e] += meet[p][t][16 * (row >> 2) + cc + e][row & 3];
        if (i < m && j < n) epi.put(v, i, 0, 1, j, n - j < 4 ? n - j : 4);
    }
}
// the parts of a cut reduction, added in their order
template <class Epi> __global__ __launch_bounds__(256) void k_join(const float *partial, int parts, int m, int n, Epi epi)
{
    const int64_t size = (int64_t)m * n, quads = (n + 3) / 4, all = m * quads;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
        const int i = (int)(at / quads), j = (int)(at - i * quads) * 4, cnt = n - j < 4 ? n - j : 4;
        const float *p = partial + (int64_t)i * n + j;
        f32x4 s[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
        for (int q = 0; q < parts; q++) s[0] += load4(p + q * size, cnt);
        epi.put(s, i, 0, 1, j, cnt);
    }
}

// ---- dz = dy act'(z) and its column sums -------------------------------------------------------------------------------------------
// grid (column blocks, row chunks).  A row's 16-byte packs lie on `lanes` (a power of two) neighbouring lanes, 256 / lanes rows at a time;
// a lane keeps the sums of its columns over the chunk, the rows' lanes meet in the LDS: sums (chunk, column), joined by k_column_join.  The sums take
// dz in 32 bits; what is stored is rounded to the element type, which is what 16-bit MFMA multiplies: dx and dw are 2.4e-3 off in bf16 (2-norm,
// sizes as above; 1.7e-3 is the rounding of the result alone), and in f16 a dy above 65504 / 1.13 may become infinite.  Bound by
// memory: 16384 x 4096 in bf16 93 us (4.3 TB/s; 106 with one row's loads at a time).
template <class T>
__global__ __launch_bounds__(256) void k_dz(const T *z, const T *dy, int64_t lddy, T *dz, int64_t lddz, float *sums, int m, int n, int chunk, int lanes, int act)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ float meet[256 * V];
    const int l = threadIdx.x & (lanes - 1), rr = threadIdx.x / lanes, step = 256 / lanes, j = (blockIdx.x * lanes + l) * V;
    const int i0 = blockIdx.y * chunk, i1 = m - i0 < chunk ? m : i0 + chunk, cnt = n - j < V ? n - j : V;
    float s[V];
#pragma unroll
    for (int e = 0; e < V; e++) s[e] = 0.f;
    const auto one = [&](Pack<T, V> d, const Pack<T, V> &q, int i) {
        if (act != NIRRT_NN_ACT_NONE) {
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float v = (float)d.e[e] * act_slope(act, (float)q.e[e]);
                s[e] += v;
                d.e[e] = (T)v;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) s[e] += (float)d.e[e];
        }
        if (dz) store_pack(dz + (int64_t)i * lddz + j, d);                   // (rows of whole packs, zeros behind column n)
    };
    int i = i0 + rr;
    if (cnt >= V)                                                            // whole packs: four rows' loads on their way at once
        for (; i + 3 * step < i1; i += 4 * step) {
            Pack<T, V> d[4], q[4];
#pragma unroll
            for (int g = 0; g < 4; g++) d[g] = load_pack<T, V>(dy + (int64_t)(i + g * step) * lddy + j);
#pragma unroll
            for (int g = 0; g < 4; g++) q[g] = act != NIRRT_NN_ACT_NONE ? load_pack<T, V>(z + (int64_t)(i + g * step) * n + j) : d[g];
#pragma unroll
            for (int g = 0; g < 4; g++) one(d[g], q[g], i + g * step);
        }
    if (cnt > 0)
        for (; i < i1; i += step) {
            const Pack<T, V> d = load_some<T, V>(dy + (int64_t)i * lddy + j, cnt);
            one(d, act != NIRRT_NN_ACT_NONE ? load_some<T, V>(z + (int64_t)i * n + j, cnt) : d, i);
        }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < V; e++) meet[threadIdx.x * V + e] = s[e];
    __syncthreads();
    for (int c = threadIdx.x; c < lanes * V; c += 256) {
        float a = 0.f;
        for (int r = 0; r < step; r++) a += meet[r * lanes * V + c];
        const int col = blockIdx.x * lanes * V + c;
        if (col < n) sums[(int64_t)blockIdx.y * n + col] = a;
    }
}
// out[j] = sum over parts of sums[p, j] for j < n, tail[j - n] for the n_tail columns behind them, in a fixed order: 64 columns x 4 shares of
// the parts per workgroup
template <class T> __global__ __launch_bounds__(256) void k_column_join(const float *sums, int parts, T *out, int64_t n, T *tail, int64_t n_tail)
{
    __shared__ float meet[4][64];
    const int64_t j = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    float s = 0.f;
    if (j < n + n_tail)
#pragma unroll 8
        for (int p = threadIdx.x >> 6; p < parts; p += 4) s += sums[p * (n + n_tail) + j];
    meet[threadIdx.x >> 6][threadIdx.x & 63] = s;
    __syncthreads();
    if (threadIdx.x < 64 && j < n + n_tail) {
        T *to = j < n ? out + j : tail + (j - n);
        if (j < n ? out : tail) *to = (T)((meet[0][threadIdx.x] + meet[1][threadIdx.x]) + (meet[2][threadIdx.x] + meet[3][threadIdx.x]));
    }
}

// x with the rows that do not count set to zero (whatever they hold: 0 x NaN must not reach dw), padded with zeros to ld columns and
// rows_out rows, so that whole aligned chunks can be read; one pass over x, a small part of the products behind it
template <class T>
__global__ __launch_bounds__(256) void k_rows_copy(const T *x, int64_t ldx, const float *coef, T *out, int64_t ld, int rows, int rows_out, int k)
{
    constexpr int V = 16 / sizeof(T);
    const int64_t per = ld / V, all = rows_out * per;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
        const int64_t r = at / per;
        const int c = (int)(at - r * per) * V;
        Pack<T, V> v = {};
        if (r < rows && (!coef || coef[r] != 0.f)) v = load_some<T, V>(x + r * ldx + c, k - c);
        store_pack(out + r * ld + c, v);
    }
}

// ---- cross entropy -----------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float row_weight(const float *cw, int64_t t, int64_t ignore, int classes)
{
    if (t == ignore) return 0.f;
    if (t < 0 || t >= classes) return __builtin_nanf("");
    return cw ? cw[t] : 1.f;
}

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
// exp(a - b) for a <= b: the difference first, so that scores of any size (a mask of the type's lowest value) stay finite
__device__ __forceinline__ float exp_less(float a, float b) { return __builtin_amdgcn_exp2f((a - b) * LOG2E); }

// C[v, r] = w_v . x_r: a lane holds scores of NI rows r (its columns), so the running maximum and sum over the classes stay in the
// lane; the two halves of a wave and the waves above one another meet once, at the end.  grid (row tiles, parts of the classes).  Bound by the
// products: 8192 x 1024 x 32003 in bf16 537 us (1000 TFLOP/s; the library's product alone, scores written: 499).
template <class T, int BM, int BN, class Tl>
__global__ __launch_bounds__(Tl::NT) void k_ce_stats(Operand<T> w, Operand<T> x, const T *b, const int64_t *target, int rows, int classes,
                                                           int k, int part, float2 *stats, float *target_score)
{
    constexpr int WM = Tl::WAVES_M, WN = Tl::WAVES_N, SUB = Tl::SUB, NC = Tl::NI * SUB, WIDE = 32 / SUB, GROUPS = 64 / WIDE;   // NC: a lane's columns
    __shared__ u32x4 lds[Tl::LDS_CHUNKS];
    __shared__ float2 meet[GROUPS * WM][BN];
    __shared__ __attribute__((aligned(16))) float add[BM];   // b of the tile's classes, -inf behind the last
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r0 = blockIdx.x * BN, top_row = Tl::first_row(wave) + block_row<SUB>(lane, 0);
    const int col0 = Tl::first_col(wave) + (lane & (WIDE - 1));
    float m[NC], s[NC], mine[NC];
    int tg[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        m[c] = -__builtin_inff();
        s[c] = mine[c] = 0.f;
        const int r = r0 + col0 + c * WIDE;
        const int64_t t = r < rows ? target[r] : -1;
        tg[c] = t >= 0 && t < classes ? (int)t : -1;
    }
    const int v_end = classes - (int)blockIdx.y * part < part ? classes : ((int)blockIdx.y + 1) * part;
    for (int v0 = blockIdx.y * part; v0 < v_end; v0 += BM) {
        Tl t;
        __syncthreads();                                     // (the tile before has been added)
        for (int c = threadIdx.x; c < BM; c += Tl::NT) add[c] = v0 + c < v_end ? (b ? (float)b[v0 + c] : 0.f) : -__builtin_inff();
        t.mainloop(w, x, v0, r0, 0, k, lds);
        if (k == 0) __syncthreads();                         // (otherwise the products' barriers stand between)
#pragma unroll
        for (int c = 0; c < NC; c++) {
            // the lane's scores of the column: four classes at a time
            float l[Tl::MI * 16 / SUB];
#pragma unroll
            for (int mi = 0; mi < Tl::MI; mi++)
#pragma unroll
                for (int q = 0; q < 4 / SUB; q++) {
                    const int e0 = SUB == 2 ? 8 * q + 4 * (c & 1) : 4 * q;
                    const f32x4 bb = *(const f32x4 *)(add + top_row + mi * 32 + block_row<SUB>(0, e0));
#pragma unroll
                    for (int e = 0; e < 4; e++) l[(mi * 4 / SUB + q) * 4 + e] = t.get(mi, c / SUB, e0 + e) + bb[e];
                }
            float top = m[c];
#pragma unroll
            for (int e = 0; e < Tl::MI * 16 / SUB; e++) top = fmaxf(top, l[e]);
            const float ref = top == -__builtin_inff() ? 0.f : top;   // (nothing but -inf so far: exp(-inf) adds zeros)
            const int want = tg[c] - v0 - top_row;
            if (__ballot(tg[c] >= v0 && tg[c] < v0 + BM)) {           // a row of this wave has its target in the tile
#pragma unroll
                for (int e = 0; e < Tl::MI * 16 / SUB; e++) mine[c] = want == 8 * SUB * (e >> 2) + (e & 3) ? l[e] : mine[c];
            }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < Tl::MI * 16 / SUB; e++) sum[e & 3] += exp_less(l[e], ref);
            s[c] = s[c] * exp_less(m[c], ref) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            m[c] = top;
        }
    }
    // the lane that met a row's target leaves its score: its share of the classes holds 4-row groups 8 SUB apart from its own row on
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int in = tg[c] - (int)blockIdx.y * part;
        if (tg[c] >= 0 && in >= 0 && tg[c] < v_end) {
            const int at = in % BM - top_row;
            if (at >= 0 && at < Tl::MI * 32 && (at & (8 * SUB - 1)) < 4) target_score[r0 + col0 + c * WIDE] = mine[c];
        }
    }
#pragma unroll
    for (int c = 0; c < NC; c++) meet[GROUPS * (wave / WN) + lane / WIDE][col0 + c * WIDE] = make_float2(m[c], s[c]);
    __syncthreads();
    for (int c = threadIdx.x; c < BN; c += Tl::NT) {
        float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (int p = 0; p < GROUPS * WM; p++) top = fmaxf(top, meet[p][c].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int p = 0; p < GROUPS * WM; p++) sum += meet[p][c].y * exp_less(meet[p][c].x, ref);
        if (r0 + c < rows) stats[(int64_t)blockIdx.y * rows + r0 + c] = make_float2(top, sum);
    }
}
// parts of a row's statistics (eight lanes per row) -> lse = (largest score, log of the sum of exp(l - it)), weighted loss; the block's sums of loss and weight (in double) for k_ce_total
constexpr int CE_ROWS = 32;
__global__ __launch_bounds__(256) void k_ce_rows(const float2 *stats, int parts, const float *target_score, const int64_t *target, const float *cw,
                                                 int64_t ignore, int rows, int classes, float2 *lse, float *nll, double *sums)
{
    __shared__ double part[2][4];
    const int r = blockIdx.x * CE_ROWS + threadIdx.x / 8, p0 = threadIdx.x & 7;
    double a = 0., b = 0.;
    float top = -__builtin_inff(), sum = 0.f;
    if (r < rows)
        for (int p = p0; p < parts; p += 8) {
            const float2 q = stats[(int64_t)p * rows + r];
            const float hi = fmaxf(top, q.x), ref = hi == -__builtin_inff() ? 0.f : hi;
            sum = sum * exp_less(top, ref) + q.y * exp_less(q.x, ref);
            top = hi;
        }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        const float t2 = __shfl_xor(top, d), s2 = __shfl_xor(sum, d), hi = fmaxf(top, t2), ref = hi == -__builtin_inff() ? 0.f : hi;
        sum = sum * exp_less(top, ref) + s2 * exp_less(t2, ref);
        top = hi;
    }
    if (r < rows && p0 == 0) {
        const float l = __builtin_amdgcn_logf(sum) * LN2;
        const int64_t t = target[r];
        const float wt = row_weight(cw, t, ignore, classes);
        const float loss = t == ignore ? 0.f : (wt == wt ? wt * ((top - target_score[r]) + l) : wt);
        lse[r] = make_float2(top, l);
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
// c_r = dloss_r weight_r (/ total weight), 0 where ignored
__device__ __forceinline__ float row_coefficient(const float *dloss, int stride, const float *total, const int64_t *target, const float *cw,
                                                 int64_t ignore, int classes, int64_t r)
{
    const int64_t t = target[r];
    if (t == ignore) return 0.f;
    const float c = dloss[stride ? r : 0] * row_weight(cw, t, ignore, classes);
    return total ? c / total[1] : c;
}
__device__ __forceinline__ float block_max(float v, float *part)   // 256 threads
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
}
__global__ __launch_bounds__(256) void k_ce_coefficients(const float *dloss, int stride, const float *total, const int64_t *target, const float *cw,
                                                         int64_t ignore, int rows, int classes, float *coef, float *tops)
{
    __shared__ float part[4];
    const int r = blockIdx.x * 256 + threadIdx.x;
    const float c = r < rows ? row_coefficient(dloss, stride, total, target, cw, ignore, classes, r) : 0.f;
    if (r < rows) coef[r] = c;
    const float top = block_max(fabsf(c), part);      // (a NaN does not count here: it is in coef)
    if (threadIdx.x == 0) tops[blockIdx.x] = top;
}
// scale = the largest |c| (1 if no row counts or it is infinite): {scale, 1 / scale}
__global__ __launch_bounds__(256) void k_ce_scale(const float *tops, int blocks, float *scale)
{
    __shared__ float part[4];
    float top = 0.f;
    for (int i = threadIdx.x; i < blocks; i += 256) top = fmaxf(top, tops[i]);
    top = block_max(top, part);
    if (threadIdx.x == 0) {
        const bool usable = top > 1e-30f && top < __builtin_inff();
        scale[0] = usable ? top : 1.f;
        scale[1] = usable ? 1.f / top : 1.f;
    }
}
// g' = c_r / scale (exp(l - lse_r) - [v = target]), lse in its two parts, FACTOR in the element type, stored (v, r): the product C[v, r] again.  16-bit products
// need 16-bit operands; c / scale <= 1 keeps the range, and FACTOR 4096 in f16 lifts probabilities of large vocabularies (1e-5) out of
// its subnormals.  A rounding is off by 2^-8 (bf16), 2^-11 (f16) of the element at most, like the rounding of dz in the linear layer; db is the
// sum of the rounded g'.  The scores are multiplied out again rather than kept between the passes, where rows x classes in 32 bits would
// lie; g' itself is whole up to G_ELEMS elements at a time.  That is no saving of time: at 1024 inputs in bf16 it costs 2 ps per score, writing
// and reading them 1.6, and in fp32 15 fs per input and score (991 x 1703 x 1320: 290 us against 232 of the elementary form, for 5 MB).
template <class T> struct Factor { static constexpr float VALUE = 1.f; };
template <> struct Factor<f16_t> { static constexpr float VALUE = 4096.f; };
template <class T> struct EpiSoftmaxGrad {
    T *g;
    int64_t ldg;
    const T *b;
    const float2 *lse;
    const float *coef, *scale;
    const int64_t *target;
    int64_t v0;
    int rows;
    template <int Q> __device__ __forceinline__ void put(f32x4 (&c)[Q], int i, int step, int rows_here, int j, int cnt) const
    {
        const float lift = scale[1] * Factor<T>::VALUE;
        const int real = rows - j < cnt ? rows - j : cnt;        // (columns behind the last row of x pad g with zeros)
        const float *rows_lse = (const float *)(lse + j);
        const f32x4 la = load4(rows_lse, 2 * real < 4 ? 2 * real : 4), lb = load4(rows_lse + 4, 2 * real - 4), w = load4(coef + j, real);
        const float top[4] = {la[0], la[2], lb[0], lb[2]}, rest[4] = {la[1], la[3], lb[1], lb[3]};
        int64_t t[4];
#pragma unroll
        for (int e = 0; e < 4; e++) t[e] = e < real ? target[j + e] - v0 - i : -1;
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q < rows_here) {
                const float add = b ? (float)b[v0 + i + q * step] : 0.f;
                f32x4 o;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float p = __expf((c[q][e] + add - top[e]) - rest[e]);
                    if (t[e] == q * step) p -= 1.f;
                    o[e] = w[e] == 0.f ? 0.f : p * (w[e] * lift);
                }
                store4(g + (int64_t)(i + q * step) * ldg + j, o, cnt);
            }
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
// ---- cross entropy of few classes (V <= 8): one pass over x forward, one backward ------------------------------------------------------
// Two classes and 128 inputs are what the guidance network's head has: a tile of 64 classes would be empty but for two, and what bounds the
// operator is reading x (forward) and reading x and writing dx (backward).  A row's 16-byte packs lie on G neighbouring lanes (64 / G rows
// per wave, NC packs per lane), the scores are summed over the G lanes with shuffles, everything in fp32; backward, a lane keeps dw of its
// columns over all rows of the workgroup, and the workgroups' shares are joined in a fixed order.  32768 x 128 in fp32, two classes: 13 us
// forward, 20 + 7 backward, 140 a call with torch's autograd (on the tiles of many classes 317); at the copy's rate it is 3 and 7.
template <class T, int V, int NC> struct FewRow {
    static constexpr int P = 16 / sizeof(T);
    float x[NC * P];
    __device__ __forceinline__ void load(const T *row, int k, int g, int G, bool on)
    {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int at = (c * G + g) * P;
            Pack<T, P> v = {};
            if (on && at < k) v = load_some<T, P>(row + at, k - at);
#pragma unroll
            for (int e = 0; e < P; e++) x[c * P + e] = (float)v.e[e];
        }
    }
    // scores of the classes below `classes` (the others -inf), in all G lanes; w (class, padded k) in the LDS
    __device__ __forceinline__ void scores(const float *w, const float *bias, int kp, int classes, int g, int G, float *l) const
    {
#pragma unroll
        for (int v = 0; v < V; v++) {
            float s = 0.f;
            if (v < classes)
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int e = 0; e < P; e += 4) {
                        const f32x4 q = *(const f32x4 *)(w + v * kp + (c * G + g) * P + e);
#pragma unroll
                        for (int d = 0; d < 4; d++) s = __builtin_fmaf(x[c * P + e + d], q[d], s);
                    }
            l[v] = s;
        }
        for (int d = 1; d < G; d <<= 1)
#pragma unroll
            for (int v = 0; v < V; v++) l[v] += __shfl_xor(l[v], d);
#pragma unroll
        for (int v = 0; v < V; v++) l[v] = v < classes ? l[v] + bias[v] : -__builtin_inff();
    }
};
template <class T> __device__ __forceinline__ void few_weights(const T *w, int64_t ldw, const T *b, int classes, int k, int kp, float *lw, float *lb)
{
    for (int at = threadIdx.x; at < classes * kp; at += 256) {
        const int v = at / kp, c = at - v * kp;
        lw[at] = c < k ? (float)w[v * ldw + c] : 0.f;
    }
    if (threadIdx.x < (unsigned)classes) lb[threadIdx.x] = b ? (float)b[threadIdx.x] : 0.f;
    __syncthreads();
}
template <class T, int V, int NC>
__global__ __launch_bounds__(256) void k_ce_few(const T *x, int64_t ldx, const T *w, int64_t ldw, const T *b, const int64_t *target, const float *cw,
                                                int64_t ignore, int rows, int classes, int k, int G, float2 *lse, float *nll, double *sums)
{
    extern __shared__ float few[];           // classes x kp weights, V biases
    __shared__ double part[2][4];
    const int kp = NC * G * FewRow<T, V, NC>::P, lane = threadIdx.x & 63, g = lane & (G - 1), per = 256 / G;
    float *lb = few + classes * kp;
    few_weights(w, ldw, b, classes, k, kp, few, lb);
    double a = 0., n = 0.;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < rows; r0 += gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / G;
        FewRow<T, V, NC> q;
        float l[V];
        q.load(x + r * ldx, k, g, G, r < rows);
        q.scores(few, lb, kp, classes, g, G, l);
        if (r < rows && g == 0) {
            float top = -__builtin_inff(), sum = 0.f, mine = 0.f;
            const int64_t t = target[r];
#pragma unroll
            for (int v = 0; v < V; v++) top = fmaxf(top, l[v]);
            const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
            for (int v = 0; v < V; v++) {
                sum += v < classes ? __expf(l[v] - ref) : 0.f;
                if (t == v) mine = l[v];
            }
            const float z = logf(sum), wt = row_weight(cw, t, ignore, classes);
            const float loss = t == ignore ? 0.f : (wt == wt ? wt * ((top - mine) + z) : wt);
            lse[r] = make_float2(top, z);
            nll[r] = loss;
            a += loss;
            n += wt;
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) { a += __shfl_down(a, d); n += __shfl_down(n, d); }
    if (lane == 0) { part[0][threadIdx.x >> 6] = a; part[1][threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x < 2) sums[2 * blockIdx.x + threadIdx.x] = (part[threadIdx.x][0] + part[threadIdx.x][1]) + (part[threadIdx.x][2] + part[threadIdx.x][3]);
}
// sums: per workgroup its share (class, k) of dw and behind it (class) of db, fp32; dx written whole
template <class T, int V, int NC>
__global__ __launch_bounds__(256) void k_ce_few_backward(const T *x, int64_t ldx, const T *w, int64_t ldw, const T *b, const int64_t *target,
                                                         const float *cw, int64_t ignore, const float2 *lse, const float *dloss, int stride,
                                                         const float *total, T *dx, float *sums, int rows, int classes, int k, int G)
{
    constexpr int P = FewRow<T, V, NC>::P;
    extern __shared__ float few[];           // classes x kp weights, V biases; later 256 / G x kp shares of one class
    const int kp = NC * G * P, lane = threadIdx.x & 63, g = lane & (G - 1), per = 256 / G;
    float *lb = few + classes * kp;
    few_weights(w, ldw, b, classes, k, kp, few, lb);
    float aw[V][NC * P], ab[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        ab[v] = 0.f;
#pragma unroll
        for (int e = 0; e < NC * P; e++) aw[v][e] = 0.f;
    }
    struct Ahead { FewRow<T, V, NC> q; float c; float2 z; int64_t t; } next;          // the next row travels while this one is worked on
    const auto fetch = [&](int64_t r) {
        next.q.load(x + r * ldx, k, g, G, r < rows);
        next.c = r < rows ? row_coefficient(dloss, stride, total, target, cw, ignore, classes, (int)r) : 0.f;
        next.z = r < rows ? lse[r] : make_float2(0.f, 0.f);
        next.t = r < rows ? target[r] : -1;
    };
    fetch((int64_t)blockIdx.x * per + threadIdx.x / G);
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < rows; r0 += gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / G;
        FewRow<T, V, NC> q = next.q;
        const float c = next.c;
        const float2 z = next.z;
        const int64_t t = next.t;
        float l[V], out[NC * P];
        fetch(r + (int64_t)gridDim.x * per);
#pragma unroll
        for (int e = 0; e < NC * P; e++) q.x[e] = c != 0.f ? q.x[e] : 0.f;      // (a row that does not count is zeros, whatever it holds)
        q.scores(few, lb, kp, classes, g, G, l);
#pragma unroll
        for (int e = 0; e < NC * P; e++) out[e] = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v < classes) {
                const float p = __expf((l[v] - z.x) - z.y) - (t == v ? 1.f : 0.f), gr = c == 0.f ? 0.f : p * c;
                ab[v] += gr;
#pragma unroll
                for (int m = 0; m < NC; m++)
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        aw[v][m * P + e] = __builtin_fmaf(gr, q.x[m * P + e], aw[v][m * P + e]);
                        out[m * P + e] = __builtin_fmaf(gr, few[v * kp + (m * G + g) * P + e], out[m * P + e]);
                    }
            }
        if (dx && r < rows) {
#pragma unroll
            for (int m = 0; m < NC; m++) {
                const int at = (m * G + g) * P;
                T *o = dx + r * k + at;
                Pack<T, P> v;
#pragma unroll
                for (int e = 0; e < P; e++) v.e[e] = (T)out[m * P + e];
                store_some(o, v, k - at);
            }
        }
    }
    // the workgroup's rows meet class by class
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (v >= classes) break;
        __syncthreads();
#pragma unroll
        for (int m = 0; m < NC; m++)
#pragma unroll
            for (int e = 0; e < P; e++) few[(threadIdx.x / G) * kp + (m * G + g) * P + e] = aw[v][m * P + e];
        __syncthreads();
        for (int c = threadIdx.x; c < k; c += 256) {
            float s = 0.f;
            for (int q = 0; q < per; q++) s += few[q * kp + c];
            sums[((int64_t)blockIdx.x * (k + 1)) * classes + (int64_t)v * k + c] = s;
        }
        __syncthreads();
        if (g == 0) few[threadIdx.x / G] = ab[v];
        __syncthreads();
        if (threadIdx.x == 0) {
            float s = 0.f;
            for (int q = 0; q < per; q++) s += few[q];
            sums[((int64_t)blockIdx.x * (k + 1) + k) * classes + v] = s;
        }
    }
}

template <class T> __global__ __launch_bounds__(256) void k_cast(const float *in, const float *scale, float factor, T *out, int64_t n)
{
    const float f = *scale * factor;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (T)(in[i] * f);
}

// ---- norm and clipping of many tensors -------------------------------------------------------------------------------------------------
constexpr int TABLE = 160;                // tensors per launch: the table travels in the kernel's arguments (3.7 KB), no copy to wait for
constexpr int BLOCK_ELEMS = 16384;        // elements per workgroup
struct TensorTable {
    const void *in[TABLE];
    void *out[TABLE];
    int first[TABLE + 1];                 // first workgroup of the tensor; the last one's end
    uint16_t last[TABLE];                 // elements of the tensor's last workgroup - 1
    uint8_t types[TABLE];                 // dtype | out_dtype << 4
    int count;
};
// the tensor of a workgroup, its element range in it: the lanes look at all first workgroups at once (one trip to memory; a search by halves
// is eight of them, as long as the workgroup's data takes)
__device__ __forceinline__ int tensor_of(const TensorTable &t, int block, int64_t &i0, int &n)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
#pragma unroll
    for (int q = 0; q < (TABLE + 63) / 64; q++) {
        const int i = q * 64 + lane;
        before += __popcll(__ballot(i < t.count && t.first[i < TABLE ? i : 0] <= block));
    }
    const int e = __builtin_amdgcn_readfirstlane(before - 1);
    i0 = (int64_t)(block - t.first[e]) * BLOCK_ELEMS;
    n = block + 1 == t.first[e + 1] ? t.last[e] + 1 : BLOCK_ELEMS;
    return e;
}
// f(P elements as fp32, how many of them exist, index) over the range, neighbouring packs on neighbouring lanes; eight packs of a thread are
// on their way at once (one after the other behind their bounds checks: 2.9 TB/s of a norm's reads where 4.4 are possible)
template <int P, class T, class F> __device__ __forceinline__ void for_packs(const T *p, int n, F f)
{
    constexpr int G = 8, STRIDE = 256 * P;
    int i = threadIdx.x * P;
    const auto some = [&](const Pack<T, P> &q, int cnt, int at) {
        float v[P];
#pragma unroll
        for (int e = 0; e < P; e++) v[e] = (float)q.e[e];
        f(v, cnt, at);
    };
    for (; i + (G - 1) * STRIDE + P <= n; i += G * STRIDE) {
        Pack<T, P> q[G];
#pragma unroll
        for (int g = 0; g < G; g++) q[g] = load_pack<T, P>(p + i + g * STRIDE);
#pragma unroll
        for (int g = 0; g < G; g++) some(q[g], P, i + g * STRIDE);
    }
    for (; i < n; i += STRIDE) {
        const int cnt = n - i < P ? n - i : P;
        some(load_some<T, P>(p + i, cnt), cnt, i);
    }
}
template <int P, class F> __device__ __forceinline__ void for_packs_of(const void *p, int dtype, int64_t i0, int n, F f)
{
    if (dtype == NIRRT_NN_F32) for_packs<4>((const float *)p + i0, n, f);
    else if (dtype == NIRRT_NN_BF16) for_packs<P>((const bf16_t *)p + i0, n, f);
    else for_packs<P>((const f16_t *)p + i0, n, f);
}
// squares are summed in double: no overflow below the largest element squared, and the order does not matter to the last bits of the norm.
// 260 M bf16 elements: 134 us (3.9 TB/s); scaled into fp32: 286 us (5.4 TB/s, the last 256 MB read from the cache)
__global__ __launch_bounds__(256) void k_norm_parts(TensorTable t, double *parts)
{
    __shared__ double part[4];
    int64_t i0;
    int n;
    const int e = tensor_of(t, blockIdx.x, i0, n);
    double s = 0.;
    for_packs_of<8>(t.in[e], t.types[e] & 15, i0, n, [&](const auto &v, int, int) {
        constexpr int P = sizeof(v) / sizeof(float);
        double a = 0.;
#pragma unroll
        for (int q = 0; q < P; q++) a = __builtin_fma((double)v[q], (double)v[q], a);
        s += a;
    });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}
__global__ __launch_bounds__(1024) void k_norm_total(const double *parts, int64_t n, float *norm)
{
    __shared__ double part[16];
    double s = 0.;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += parts[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.;
#pragma unroll
        for (int q = 0; q < 16; q++) s += part[q];
        *norm = (float)sqrt(s);
    }
}
template <class T, int P> __device__ __forceinline__ void put_pack(T *o, const float (&v)[P], float f, int cnt)
{
    Pack<T, P> q;
#pragma unroll
    for (int e = 0; e < P; e++) q.e[e] = (T)(v[e] * f);
    store_some(o, q, cnt);
}
__global__ __launch_bounds__(256) void k_scale(TensorTable t, const float *norm, float max_norm)
{
    int64_t i0;
    int n;
    const int e = tensor_of(t, blockIdx.x, i0, n), to = t.types[e] >> 4;
    const float q = max_norm / (*norm + 1e-6f), f = q < 1.f ? q : (q == q ? 1.f : q);
    if (f == 1.f && t.in[e] == t.out[e]) return;
    // (four elements per lane: both sides of a 16-bit -> 32-bit scaling are whole lines per instruction)
    void *out = t.out[e];
    for_packs_of<4>(t.in[e], t.types[e] & 15, i0, n, [&](const auto &v, int cnt, int i) {
        if (to == NIRRT_NN_F32) put_pack((float *)out + i0 + i, v, f, cnt);
        else if (to == NIRRT_NN_BF16) put_pack((bf16_t *)out + i0 + i, v, f, cnt);
        else put_pack((f16_t *)out + i0 + i, v, f, cnt);
    });
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
constexpr int64_t DIM_MAX = 0x7fffffffll;
constexpr int64_t MOST = DIM_MAX - 4095;  // of a dimension: kernels look up to 2048 elements past an index in 32 bits (k_few_rows; k_dz 1024)
int64_t round256(int64_t b) { return (b + 255) & ~255ll; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int status() { return hipGetLastError() == hipSuccess ? 0 : -2; }
int elem_size(int dtype) { return dtype == NIRRT_NN_F32 ? 4 : 2; }
bool good_type(int dtype) { return dtype == NIRRT_NN_F32 || dtype == NIRRT_NN_BF16 || dtype == NIRRT_NN_F16; }

template <class T> Operand<T> op(const T *p, int64_t ld, int64_t rows, int64_t depth = DIM_MAX) { return {p, ld, (int)rows, (int)depth}; }

// Tile edge and parts of the reduction, by the time they are expected to take.  A step is 64 bytes of k; a CU with q tiles of a kind to do takes
// max(lat ceil(q / fit), q work) us per step (fit: tiles resident at once), 0.3 ns per element for the epilogue, and parts are joined at 4 bytes
// per element, part and way.  Measured on one box, us per step, 256 CUs with 1 / 2 / 4 tiles each (x w^T): 16-bit 256: 0.94 2.0 4.4, 128: 0.39
// 0.67 1.33, 64: 0.28 0.33 0.62; 32-bit 256: 4.2, 128: 1.07, 64: 0.31 per tile.  slow = 1 + the number of RC operands: operands that are no whole
// aligned chunks take the register-staged tile (4097 x 321 x 515 in bf16, edge 64: 14 us with none, 22 with one, 37 with two); 0: they are.
struct Plan { int edge, parts, part; double us; };
struct TileCost { int edge, fit; double lat, work; };
Plan plan(int dtype, int64_t m, int64_t n, int64_t k, int slow = 0, int64_t most_parts = 32)
{
    static const TileCost fast16[] = {{256, 1, 0.94, 1.03}, {128, 2, 0.38, 0.33}, {64, 5, 0.28, 0.155}};
    static const TileCost fast32[] = {{256, 1, 3.7, 4.2}, {128, 2, 1.05, 1.07}, {64, 5, 0.36, 0.31}};
    static const TileCost slow16[] = {{128, 3, 1.0, 0.6}, {64, 6, 0.5, 0.25}};
    static const TileCost slow32[] = {{128, 3, 1.5, 1.25}, {64, 6, 0.6, 0.36}};
    const bool f32 = dtype == NIRRT_NN_F32;
    const TileCost *cost = slow ? (f32 ? slow32 : slow16) : (f32 ? fast32 : fast16);
    const double rc = slow <= 1 ? 1. : f32 ? (slow == 2 ? 1.2 : 1.5) : (slow == 2 ? 1.7 : 3.);
    const int64_t step = 64 / elem_size(dtype), steps = ceil_div(k, step);
    Plan best = {64, 1, (int)(steps > 0 ? steps * step : step), 0.};
    if (m <= 0 || n <= 0 || k <= 0) return best;
    best.us = 1e30;
    for (int c = slow ? 1 : 2; c >= 0; c--) {
        const double tiles = (double)ceil_div(m, cost[c].edge) * (double)ceil_div(n, cost[c].edge), elems = (double)cost[c].edge * cost[c].edge;
        for (int64_t parts = 1; parts <= most_parts && parts * 8 <= steps + 7; parts++) {
            const int64_t per = ceil_div(steps, parts);
            if (parts > 1 && ceil_div(steps, per) != parts) continue;
            const double q = ceil(tiles * parts / 256.), waves = ceil(q / cost[c].fit);
            const double run = (cost[c].lat * waves > q * cost[c].work ? cost[c].lat * waves : q * cost[c].work) * rc * per;
            const double us = run + 2. * waves + q * elems * 3e-4 + (parts > 1 ? 5. + (double)m * n * 4. * (2 * parts + 1) / 4e6 : 0.);
            if (us < best.us) best = {cost[c].edge, (int)parts, (int)(per * step), us};
        }
    }
    return best;
}
int64_t plan_bytes(const Plan &p, int64_t m, int64_t n) { return p.parts > 1 ? round256(4 * m * n * p.parts) : 0; }
// the time that copying rows into whole chunks takes: 3 TB/s and a launch
double copy_us(int dtype, int64_t rows, int64_t k) { return 4. + (double)rows * k * 2 * elem_size(dtype) / 3e6; }
int64_t padded(int dtype, int64_t k) { const int64_t c = 16 / elem_size(dtype); return (k + c - 1) / c * c; }
bool whole_rows(int dtype, const void *p, int64_t ld, int64_t k) { return (uintptr_t)p % 16 == 0 && ld * elem_size(dtype) % 16 == 0 && k == padded(dtype, k); }
// ... and no further apart than direct() takes as rows of a KC operand (the last token of every sequence lies a sequence apart)
constexpr int64_t KC_ROW_BYTES = 1 << 22;
bool near_whole_rows(int dtype, const void *p, int64_t ld, int64_t k) { return whole_rows(dtype, p, ld, k) && ld * elem_size(dtype) <= KC_ROW_BYTES; }
bool aligned_rows(int dtype, const void *p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld * elem_size(dtype) % 16 == 0; }
template <class T>
void copy_rows(const void *x, int64_t ldx, const float *coef, T *out, int64_t ld, int64_t rows, int64_t rows_out, int64_t k, hipStream_t st)
{
    const int64_t blocks = ceil_div(rows_out * (ld * (int64_t)sizeof(T) / 16), 256);
    if (blocks > 0)
        hipLaunchKernelGGL((k_rows_copy<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, (const T *)x, ldx, coef, out, ld,
                           (int)rows, (int)rows_out, (int)k);
}

// whole aligned chunks (see DirectOperand): rows and base on 16 bytes, for KC a reduction of whole chunks, offsets inside a step below 2^31
template <class T, bool RC> bool direct(const Operand<T> &o, int64_t k)
{
    const int64_t row_bytes = o.ld * (int64_t)sizeof(T);
    if ((uintptr_t)o.p % 16 || row_bytes % 16) return false;
    return RC ? row_bytes <= (1 << 24) : k % Elem<T>::PER_CHUNK == 0 && row_bytes <= KC_ROW_BYTES;
}

constexpr int64_t MOST_WORKGROUPS = (1ll << 32) / 512 - 1;      // of 512 threads: a launch has less than 2^32 of them

template <class Epi> constexpr bool always_whole = false;                        // its operands are always whole aligned chunks, its reduction in one part
template <class T> constexpr bool always_whole<EpiSoftmaxGrad<T>> = true;
template <class T, bool RCA, bool RCB, class Epi>
int gemm(const Operand<T> &a, const Operand<T> &b, int64_t m, int64_t n, int64_t k, const Plan &p, float *partial, const Epi &epi, hipStream_t st)
{
    const bool fast = direct<T, RCA>(a, k) && direct<T, RCB>(b, k);
    int edge = fast || p.edge < 256 ? p.edge : 128;         // (a plan for whole chunks, and operands beyond direct()'s row length)
    if (edge == 64 && ceil_div(m, 64) * ceil_div(n, 64) > MOST_WORKGROUPS) edge = 128;     // (a quarter of them)
    const int64_t tiles = ceil_div(m, edge) * ceil_div(n, edge);
    if (tiles > 2 * MOST_WORKGROUPS) return -1;
    const dim3 grid((unsigned)tiles, (unsigned)p.parts);
#define LAUNCH(TILE, EDGE, WM, WN)                                                                                                               \
    hipLaunchKernelGGL((k_gemm<T, EDGE, EDGE, TILE<T, EDGE, EDGE, WM, WN, RCA, RCB>, Epi>), grid, dim3(64 * WM * WN), 0, st, a, b, (int)m, (int)n, \
                       (int)k, p.part, partial, epi)
    if constexpr (always_whole<Epi>) {
        if (!fast || p.parts > 1) return -1;
    }
    if (edge == 256) LAUNCH(DirectTile, 256, 2, 4);
    else if (fast) { if (edge == 128) LAUNCH(DirectTile, 128, 2, 2); else LAUNCH(DirectTile, 64, 2, 2); }
    if constexpr (!always_whole<Epi>) {
        if (!fast) { if (edge == 128) LAUNCH(Tile, 128, 2, 2); else LAUNCH(Tile, 64, 2, 2); }
        if (p.parts > 1) {
            const int64_t blocks = ceil_div(m * ceil_div(n, 4), 256);
            hipLaunchKernelGGL((k_join<Epi>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, partial, p.parts, (int)m, (int)n, epi);
        }
    }
#undef LAUNCH
    return status();
}

bool good_dims(int64_t a, int64_t b, int64_t c) { return a >= 0 && b >= 0 && c >= 0 && a <= MOST && b <= MOST && c <= MOST; }

// k_dz: lanes per row, rows per workgroup and chunks so that some 2000 workgroups share a large matrix and a chunk is no shorter than 4 passes
struct Columns { int lanes, blocks, chunk, parts; };
Columns columns(int dtype, int64_t m, int64_t n)
{
    Columns c;
    const int64_t packs = ceil_div(n, 16 / elem_size(dtype));
    c.lanes = 1;
    while (c.lanes < 64 && c.lanes < packs) c.lanes *= 2;
    c.blocks = (int)ceil_div(packs, c.lanes);
    const int64_t step = 256 / c.lanes;
    int64_t parts = ceil_div(2048, c.blocks > 0 ? c.blocks : 1), most = ceil_div(m, 4 * step);
    if (parts > most) parts = most;
    if (parts > 512) parts = 512;
    if (parts < 1) parts = 1;
    c.chunk = (int)(m > 0 ? ceil_div(m, parts) : 1);
    c.parts = (int)ceil_div(m, c.chunk);
    return c;
}

// x w^T: few rows go to k_few_rows; operands that are no whole aligned chunks are copied into such where that is expected to pay
struct Linear { bool few, copy_x, copy_w; Plan p; int64_t kp, xs, ws, part, total; };
Linear linear_layout(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t m, int64_t n, int64_t k)
{
    Linear l = {};
    l.few = m <= 32 && ceil_div(n, 16) <= MOST_WORKGROUPS;
    l.kp = k;
    if (l.few) return l;
    l.copy_x = !whole_rows(dtype, x, ldx, k);
    l.copy_w = !whole_rows(dtype, w, ldw, k);
    if (l.copy_x || l.copy_w) {
        const Plan slow = plan(dtype, m, n, k, 1), fast = plan(dtype, m, n, padded(dtype, k));
        if (fast.us + (l.copy_x ? copy_us(dtype, m, k) : 0.) + (l.copy_w ? copy_us(dtype, n, k) : 0.) >= slow.us) {
            l.copy_x = l.copy_w = false;
            l.p = slow;
        } else {
            l.p = fast;
            l.kp = padded(dtype, k);
        }
    } else l.p = plan(dtype, m, n, k);
    l.xs = l.copy_x ? round256(m * l.kp * elem_size(dtype)) : 0;
    l.ws = l.copy_w ? round256(n * l.kp * elem_size(dtype)) : 0;
    l.part = plan_bytes(l.p, m, n);
    l.total = l.xs + l.ws + l.part;
    return l;
}
template <class T>
int linear_t(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const void *r, int64_t ldr, void *y,
             int64_t ldy, void *z, int64_t m, int64_t n, int64_t k, char *ws, hipStream_t st)
{
    const Linear l = linear_layout(dtype, x, ldx, w, ldw, m, n, k);
    const EpiLinear<T> epi = {(const T *)b, (const T *)r, (T *)y, (T *)z, ldr, ldy, act, (int)n};
    if (l.few) {
        const dim3 grid((unsigned)ceil_div(n, 16));
        if (m <= 16) hipLaunchKernelGGL((k_few_rows<T, 1, EpiLinear<T>>), grid, dim3(512), 0, st, (const T *)x, ldx, (const T *)w, ldw, (int)m, (int)n, (int)k, epi);
        else hipLaunchKernelGGL((k_few_rows<T, 2, EpiLinear<T>>), grid, dim3(512), 0, st, (const T *)x, ldx, (const T *)w, ldw, (int)m, (int)n, (int)k, epi);
        return status();
    }
    T *xs = (T *)ws, *wsp = (T *)(ws + l.xs);
    if (l.copy_x) { copy_rows(x, ldx, nullptr, xs, l.kp, m, m, k, st); x = xs; ldx = l.kp; }
    if (l.copy_w) { copy_rows(w, ldw, nullptr, wsp, l.kp, n, n, k, st); w = wsp; ldw = l.kp; }
    return gemm<T, false, false>(op((const T *)x, ldx, m), op((const T *)w, ldw, n), m, n, l.kp, l.p, (float *)(ws + l.xs + l.ws), epi, st);
}

// dx = dz w (m, k; reduction n), dw = dz^T x (n, k; reduction m).  dz is written in rows of whole chunks (also for ACT_NONE where dy's are not); w
// and x are copied into such where that is expected to pay.
struct LinearBackward { bool own_dz, copy_x, copy_w; Plan px, pw; int64_t np, kp, dz, xs, ws, sums, part, total; };
LinearBackward linear_backward_layout(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *dy, int64_t lddy, int64_t m,
                                      int64_t n, int64_t k, bool dx, bool dw)
{
    LinearBackward l = {};
    const int e = elem_size(dtype);
    l.np = padded(dtype, n);
    l.kp = padded(dtype, k);
    l.px = plan(dtype, m, k, l.np);
    l.pw = plan(dtype, n, k, m);
    l.copy_w = dx && !aligned_rows(dtype, w, ldw);
    l.copy_x = dw && !aligned_rows(dtype, x, ldx);
    const double relay_dy = act == NIRRT_NN_ACT_NONE && (dx || dw) && !whole_rows(dtype, dy, lddy, n) ? copy_us(dtype, m, n) : 0.;
    const Plan sx = plan(dtype, m, k, n, 2), sw_ = plan(dtype, n, k, m, 3);
    const bool slow_x = dx && (l.copy_w || relay_dy > 0.) && l.px.us + (l.copy_w ? copy_us(dtype, n, k) : 0.) + relay_dy / 2 >= sx.us;
    const bool slow_w = dw && (l.copy_x || relay_dy > 0.) && l.pw.us + (l.copy_x ? copy_us(dtype, m, k) : 0.) + relay_dy / 2 >= sw_.us;
    if (slow_x) { l.px = sx; l.copy_w = false; }
    if (slow_w) { l.pw = sw_; l.copy_x = false; }
    l.own_dz = act != NIRRT_NN_ACT_NONE || (relay_dy > 0. && ((dx && !slow_x) || (dw && !slow_w)));
    l.dz = l.own_dz && (dx || dw) ? round256(m * l.np * e) : 0;
    l.xs = l.copy_x ? round256(m * l.kp * e) : 0;
    l.ws = l.copy_w ? round256(n * l.kp * e) : 0;
    l.sums = round256(4 * n * columns(dtype, m, n).parts);
    const int64_t bx = dx ? plan_bytes(l.px, m, k) : 0, bw = dw ? plan_bytes(l.pw, n, k) : 0;
    l.part = bx > bw ? bx : bw;
    l.total = l.dz + l.xs + l.ws + l.sums + l.part;
    return l;
}
template <class T>
int linear_backward_t(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *z, const void *dy, int64_t lddy,
                      void *dx, void *dw, void *db, int64_t m, int64_t n, int64_t k, char *ws, hipStream_t st)
{
    const LinearBackward l = linear_backward_layout(dtype, act, x, ldx, w, ldw, dy, lddy, m, n, k, dx != nullptr, dw != nullptr);
    T *dz = (T *)ws, *xs = (T *)(ws + l.dz), *wsp = (T *)((char *)xs + l.xs);
    float *sums = (float *)((char *)wsp + l.ws), *part = (float *)((char *)sums + l.sums);
    if (n > 0 && (l.own_dz || db)) {                  // (no columns: no dz and no db, and dx is zero)
        const Columns c = columns(dtype, m, n);
        if (m > 0)
            hipLaunchKernelGGL((k_dz<T>), dim3((unsigned)c.blocks, (unsigned)c.parts), dim3(256), 0, st, (const T *)z, (const T *)dy, lddy,
                               l.dz ? dz : (T *)nullptr, l.np, db ? sums : nullptr, (int)m, (int)n, c.chunk, c.lanes, act);
        if (db)
            hipLaunchKernelGGL((k_column_join<T>), dim3((unsigned)ceil_div(n, 64)), dim3(256), 0, st, sums, c.parts, (T *)db, n, (T *)nullptr, (int64_t)0);
        if (int rc_ = status()) return rc_;
    }
    const T *d = l.dz ? dz : (const T *)dy;
    const int64_t ldd = l.dz ? l.np : lddy;
    if (dx && m > 0 && k > 0) {
        const EpiPlain<T> epi = {(T *)dx, nullptr, 1.f, (int)k};
        const T *wp = (const T *)w;
        int64_t ld = ldw;
        if (l.copy_w) { copy_rows(w, ldw, nullptr, wsp, l.kp, n, n, k, st); wp = wsp; ld = l.kp; }
        // (own dz: a reduction of whole chunks, zeros behind n)
        if (int rc_ = gemm<T, false, true>(op(d, ldd, m), op(wp, ld, k, n), m, k, l.dz ? l.np : n, l.px, part, epi, st)) return rc_;
    }
    if (dw && n > 0 && k > 0) {
        const EpiPlain<T> epi = {(T *)dw, nullptr, 1.f, (int)k};
        const T *xp = (const T *)x;
        int64_t ld = ldx;
        if (l.copy_x) { copy_rows(x, ldx, nullptr, xs, l.kp, m, m, k, st); xp = xs; ld = l.kp; }
        if (int rc_ = gemm<T, true, true>(op(d, ldd, n), op(xp, ld, k), n, k, m, l.pw, part, epi, st)) return rc_;
    }
    return 0;
}

// few classes (k_ce_few): up to 8, and a row on at most 64 lanes x 4 packs
struct Few { int lanes, packs, classes, blocks_forward, blocks, lds, lds_backward; };
constexpr int FEW_BLOCKS = 2048;
bool few_layout(int dtype, int64_t rows, int64_t classes, int64_t k, Few &f)
{
    const int p = 16 / elem_size(dtype);
    const int64_t packs = ceil_div(k > 0 ? k : 1, p);
    if (classes > 8 || packs > 256) return false;
    f.lanes = 1;
    while (f.lanes < 64 && f.lanes < packs) f.lanes *= 2;
    const int64_t per_lane = ceil_div(packs, f.lanes);
    f.packs = per_lane <= 1 ? 1 : per_lane <= 2 ? 2 : 4;
    f.classes = classes <= 2 ? 2 : classes <= 4 ? 4 : 8;
    if (f.classes * f.packs * p > 128) return false;      // registers of dw
    const int kp = f.packs * f.lanes * p, per = 256 / f.lanes;
    // forward eight workgroups per CU, so that enough rows are on their way; backward two, because each leaves a share of dw behind (and asks for
    // its next rows ahead instead): at least two and four rows per lane group
    const int64_t forward = ceil_div(rows, 2 * per), blocks = ceil_div(rows, 4 * per);
    f.blocks_forward = (int)(forward < FEW_BLOCKS ? (forward > 0 ? forward : 1) : FEW_BLOCKS);
    f.blocks = (int)(blocks < 512 ? (blocks > 0 ? blocks : 1) : 512);
    f.lds = (int)(4 * (classes * kp + 8));
    f.lds_backward = f.lds > 4 * per * kp ? f.lds : 4 * per * kp;
    return true;
}
#define FEW_LAUNCH(KERNEL, BLOCKS, LDS, ...)                                                                                     \
    do {                                                                                                                 \
        if (f.classes == 2) { if (f.packs == 1) FEW_ONE(KERNEL, 2, 1, BLOCKS, LDS, __VA_ARGS__); else if (f.packs == 2) FEW_ONE(KERNEL, 2, 2, BLOCKS, LDS, __VA_ARGS__); else FEW_ONE(KERNEL, 2, 4, BLOCKS, LDS, __VA_ARGS__); } \
        else if (f.classes == 4) { if (f.packs == 1) FEW_ONE(KERNEL, 4, 1, BLOCKS, LDS, __VA_ARGS__); else if (f.packs == 2) FEW_ONE(KERNEL, 4, 2, BLOCKS, LDS, __VA_ARGS__); else FEW_ONE(KERNEL, 4, 4, BLOCKS, LDS, __VA_ARGS__); } \
        else { if (f.packs == 1) FEW_ONE(KERNEL, 8, 1, BLOCKS, LDS, __VA_ARGS__); else if (f.packs == 2) FEW_ONE(KERNEL, 8, 2, BLOCKS, LDS, __VA_ARGS__); else FEW_ONE(KERNEL, 8, 4, BLOCKS, LDS, __VA_ARGS__); } \
    } while (0)
#define FEW_ONE(KERNEL, V, NC, BLOCKS, LDS, ...) hipLaunchKernelGGL((KERNEL<T, V, NC>), dim3((unsigned)BLOCKS), dim3(256), LDS, st, __VA_ARGS__)

// cross entropy: tile edge by the number of 128 x 128 tiles, and parts of the classes so that row tiles x parts fill the GPU.  us of the forward
// pass at edge 64 / 128 / 256, 1024 inputs, bf16: 128 tiles 20.8 / 24.2 / 32.9, 256 tiles 32.0 / 26.3 / 34.7, 512 tiles 49.4 / 32.0 / 35.1, 1024
// tiles 88.8 / 51.7 / 40.0, 4096 tiles 331 / 176 / 129; fp32: 53.8 / 77.5 / 247, 98.2 / 80.6 / 245, 170 / 138 / 246, 331 / 264 / 251, 1296 / 1028 / 975.
// x and w whose rows are no whole aligned chunks
// or lie far apart are copied into such that are not (k_rows_copy): the products read them many times
// (the copies lie behind everything else, so that a caller whose operands need none may leave their bytes out)
struct CeForward { int edge, parts, part; int64_t stats, score, sums, xs, ws, total; };
CeForward ce_layout(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    CeForward f = {};
    Few few;
    f.sums = round256(16 * (ceil_div(rows, CE_ROWS) + FEW_BLOCKS));
    f.total = f.sums;
    if (few_layout(dtype, rows, classes, k, few)) return f;
    const int64_t big = ceil_div(rows, 128) * ceil_div(classes, 128);
    f.edge = big >= 1024 ? 256 : big >= 256 ? 128 : 64;
    const int64_t row_tiles = ceil_div(rows, f.edge), class_tiles = ceil_div(classes, f.edge);
    int64_t parts = ceil_div(f.edge == 256 ? 256 : 512, row_tiles > 0 ? row_tiles : 1);
    if (parts > class_tiles) parts = class_tiles;
    if (parts < 1) parts = 1;
    const int64_t per = ceil_div(class_tiles, parts);
    f.part = (int)(per * f.edge < DIM_MAX ? per * f.edge : DIM_MAX);
    f.parts = (int)(class_tiles > 0 ? ceil_div(class_tiles, per) : 1);
    f.stats = round256(8 * rows * f.parts);
    f.score = round256(4 * rows);
    f.xs = round256(rows * padded(dtype, k) * elem_size(dtype));
    f.ws = round256(classes * padded(dtype, k) * elem_size(dtype));
    f.total = f.stats + f.score + f.sums + f.xs + f.ws;
    return f;
}
template <class T>
int ce_forward_t(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target, const float *cw, int64_t ignore,
                 float2 *lse, float *nll, float *total, int64_t rows, int64_t classes, int64_t k, char *ws, hipStream_t st)
{
    const CeForward l = ce_layout(dtype, rows, classes, k);
    double *sums = (double *)ws;
    float *score = (float *)(ws + l.sums);
    float2 *stats = (float2 *)(ws + l.sums + l.score);
    const bool copy_x = !near_whole_rows(dtype, x, ldx, k), copy_w = !near_whole_rows(dtype, w, ldw, k);
    T *xs = (T *)(ws + l.sums + l.score + l.stats), *wsp = (T *)((char *)xs + (copy_x ? l.xs : 0));
    int64_t blocks = 0;
    Few f;
    if (rows > 0 && few_layout(dtype, rows, classes, k, f)) {
        blocks = f.blocks_forward;
        FEW_LAUNCH(k_ce_few, f.blocks_forward, f.lds, (const T *)x, ldx, (const T *)w, ldw, (const T *)b, target, cw, ignore, (int)rows, (int)classes, (int)k, f.lanes, lse,
                   nll, sums);
    } else if (rows > 0) {
        blocks = ceil_div(rows, CE_ROWS);
        const int64_t kp = padded(dtype, k), row_tiles = ceil_div(rows, l.edge);
        if (copy_x) { copy_rows(x, ldx, nullptr, xs, kp, rows, rows, k, st); x = xs; ldx = kp; }
        if (copy_w) { copy_rows(w, ldw, nullptr, wsp, kp, classes, classes, k, st); w = wsp; ldw = kp; }
        const dim3 grid((unsigned)row_tiles, (unsigned)l.parts);
        const Operand<T> ow = op((const T *)w, ldw, classes), ox = op((const T *)x, ldx, rows);
#define LAUNCH(EDGE, WM, WN)                                                                                                                \
    hipLaunchKernelGGL((k_ce_stats<T, EDGE, EDGE, DirectTile<T, EDGE, EDGE, WM, WN, false, false>>), grid, dim3(64 * WM * WN), 0, st, ow, ox, \
                       (const T *)b, target, (int)rows, (int)classes, (int)kp, l.part, stats, score)
        if (l.edge == 256) LAUNCH(256, 2, 4); else if (l.edge == 128) LAUNCH(128, 2, 2); else LAUNCH(64, 2, 2);
#undef LAUNCH
        hipLaunchKernelGGL(k_ce_rows, dim3((unsigned)blocks), dim3(256), 0, st, stats, l.parts, score, target, cw, ignore, (int)rows, (int)classes,
                           lse, nll, sums);
    }
    hipLaunchKernelGGL(k_ce_total, dim3(1), dim3(256), 0, st, sums, (int)blocks, total);
    return status();
}

constexpr int64_t G_ELEMS = 1ll << 27;    // of g' at a time: pieces of the classes
struct CeBackward { int64_t piece, ldg; Plan pg, px, pw; int64_t coef, tops, xs, ws, g, acc, part, total; };
CeBackward ce_backward_layout(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    CeBackward l;
    Few f;
    if (few_layout(dtype, rows, classes, k, f)) {
        l = CeBackward{};
        l.part = round256(4 * (k + 1) * classes * f.blocks);
        l.total = l.part;
        return l;
    }
    const int64_t e = elem_size(dtype);
    l.ldg = padded(dtype, rows);
    l.piece = l.ldg > 0 ? G_ELEMS / l.ldg / 256 * 256 : classes;
    if (l.piece < 256) l.piece = 256;
    if (l.piece > classes) l.piece = classes;
    l.pg = plan(dtype, l.piece, l.ldg, padded(dtype, k), 0, 1);     // (the scores are not cut: the softmax needs whole ones)
    l.px = plan(dtype, rows, k, l.piece);
    l.pw = plan(dtype, l.piece, k, l.ldg);
    l.coef = round256(4 * rows) + 256;
    l.tops = round256(4 * ceil_div(rows, 256));
    l.xs = round256(l.ldg * padded(dtype, k) * e);
    l.ws = round256(classes * padded(dtype, k) * e);
    l.g = round256(l.ldg * l.piece * e);
    l.acc = l.piece < classes ? round256(4 * rows * k) : 0;
    const int64_t bx = plan_bytes(l.px, rows, k), bw = plan_bytes(l.pw, l.piece, k);
    l.part = bx > bw ? bx : bw;
    l.total = l.coef + l.tops + l.xs + l.ws + l.g + l.acc + l.part;
    return l;
}
template <class T>
int ce_backward_t(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target, const float *cw,
                  int64_t ignore, const float2 *lse, const float *dloss, int stride, const float *total, void *dx, void *dw, void *db, int64_t rows,
                  int64_t classes, int64_t k, char *ws, hipStream_t st)
{
    const CeBackward l = ce_backward_layout(dtype, rows, classes, k);
    Few f;
    if (few_layout(dtype, rows, classes, k, f)) {
        float *sums = (float *)ws;
        FEW_LAUNCH(k_ce_few_backward, f.blocks, f.lds_backward, (const T *)x, ldx, (const T *)w, ldw, (const T *)b, target, cw, ignore, lse, dloss, stride, total, (T *)dx,
                   sums, (int)rows, (int)classes, (int)k, f.lanes);
        if (dw || db)
            hipLaunchKernelGGL((k_column_join<T>), dim3((unsigned)ceil_div(classes * (k + 1), 64)), dim3(256), 0, st, sums, f.blocks, (T *)dw, classes * k,
                               (T *)db, classes);
        return status();
    }
    float *scale = (float *)ws, *coef = scale + 64, *tops = (float *)(ws + l.coef);
    T *xs = (T *)(ws + l.coef + l.tops), *g = (T *)((char *)xs + l.xs);
    float *acc = (float *)((char *)g + l.g), *part = (float *)((char *)acc + l.acc);
    T *wsp = (T *)((char *)part + l.part);            // (last: see ce_layout)
    const int64_t kp = padded(dtype, k), blocks = ceil_div(rows, 256);
    if (blocks > 0)
        hipLaunchKernelGGL(k_ce_coefficients, dim3((unsigned)blocks), dim3(256), 0, st, dloss, stride, total, target, cw, ignore, (int)rows, (int)classes, coef, tops);
    hipLaunchKernelGGL(k_ce_scale, dim3(1), dim3(256), 0, st, tops, (int)blocks, scale);
    copy_rows(x, ldx, coef, xs, kp, rows, l.ldg, k, st);
    if (!near_whole_rows(dtype, w, ldw, k)) { copy_rows(w, ldw, nullptr, wsp, kp, classes, classes, k, st); w = wsp; ldw = kp; }
    const float unlift = 1.f / Factor<T>::VALUE;
    for (int64_t v0 = 0; v0 < classes; v0 += l.piece) {
        const int64_t nv = classes - v0 < l.piece ? classes - v0 : l.piece;
        const T *wp = (const T *)w + v0 * ldw;
        if (rows > 0) {
            const EpiSoftmaxGrad<T> eg = {g, l.ldg, (const T *)b, lse, coef, scale, target, v0, (int)rows};
            if (int rc = gemm<T, false, false>(op(wp, ldw, nv), op((const T *)xs, kp, l.ldg), nv, l.ldg, kp, l.pg, nullptr, eg, st)) return rc;
        }
        if (db) hipLaunchKernelGGL((k_ce_bias<T>), dim3((unsigned)ceil_div(nv, 4)), dim3(256), 0, st, (const T *)g, l.ldg, (int)rows, (int)nv, scale, (T *)db + v0);
        if (dx && rows > 0 && k > 0) {
            const Operand<T> og = op((const T *)g, l.ldg, rows), ow = op(wp, ldw, k);
            int rc;
            if (l.acc) rc = gemm<T, true, true>(og, ow, rows, k, nv, l.px, part, EpiAccumulate<T>{acc, (int)k, v0 == 0}, st);
            else rc = gemm<T, true, true>(og, ow, rows, k, nv, l.px, part, EpiPlain<T>{(T *)dx, scale, unlift, (int)k}, st);
            if (rc) return rc;
        }
        if (dw && k > 0) {
            const EpiPlain<T> ep = {(T *)dw + v0 * k, scale, unlift, (int)k};
            if (int rc = gemm<T, false, true>(op((const T *)g, l.ldg, nv), op((const T *)xs, kp, k), nv, k, l.ldg, l.pw, part, ep, st)) return rc;
        }
    }
    if (dx && l.acc && rows > 0 && k > 0) {
        const int64_t cast = ceil_div(rows * k, 256);
        hipLaunchKernelGGL((k_cast<T>), dim3((unsigned)(cast < 8192 ? cast : 8192)), dim3(256), 0, st, acc, scale, unlift, (T *)dx, rows * k);
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
// calls launch(table, first workgroup, workgroups) for every TABLE tensors that hold something, from the first or from the last on; the total
// of workgroups, < 0 on error
template <class F> int64_t for_tables(const nirrt_nn_tensor *t, int32_t count, bool backward, F launch)
{
    int64_t done = 0;
    TensorTable tab;
    tab.count = 0;
    int64_t blocks = 0;
    for (int32_t q = 0; q <= count; q++) {
        const int32_t i = q == count ? count : backward ? count - 1 - q : q;
        if (i < count && t[i].n == 0) continue;
        const int64_t b = i < count ? ceil_div(t[i].n, BLOCK_ELEMS) : 0;
        if (b > DIM_MAX / 2) return -1;
        if (tab.count == TABLE || (i == count && tab.count > 0) || (tab.count > 0 && blocks + b > DIM_MAX / 2)) {
            tab.first[tab.count] = (int)blocks;
            if (launch(tab, done, blocks)) return -2;
            done += blocks;
            blocks = 0;
            tab.count = 0;
        }
        if (i == count) break;
        const int c = tab.count++;
        tab.in[c] = t[i].data;
        tab.out[c] = t[i].out;
        tab.first[c] = (int)blocks;
        tab.last[c] = (uint16_t)((t[i].n - 1) % BLOCK_ELEMS);
        tab.types[c] = (uint8_t)(t[i].dtype | t[i].out_dtype << 4);
        blocks += b;
    }
    return done;
}

}   // namespace

static bool good_linear(int dtype, int act, int64_t ldx, int64_t ldw, int64_t m, int64_t n, int64_t k)
{
    return good_type(dtype) && act >= 0 && act <= NIRRT_NN_ACT_SILU && good_dims(m, n, k) && ldx >= k && ldw >= k;
}

extern "C" int64_t nirrt_nn_linear_workspace(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t m, int64_t n, int64_t k)
{
    if (!good_linear(dtype, 0, ldx, ldw, m, n, k)) return -1;
    return linear_layout(dtype, x, ldx, w, ldw, m, n, k).total;
}

extern "C" int nirrt_nn_linear(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const void *r, int64_t ldr,
                               void *y, int64_t ldy, void *z, int64_t m, int64_t n, int64_t k, void *workspace, void *stream)
{
    if (!good_linear(dtype, act, ldx, ldw, m, n, k)) return -1;
    if (m == 0 || n == 0) return 0;
    if (!y || (k > 0 && (!x || !w)) || ldy < n || (r && ldr < n)) return -1;
    if (!workspace && nirrt_nn_linear_workspace(dtype, x, ldx, w, ldw, m, n, k) > 0) return -1;
#define CALL(T) linear_t<T>(dtype, act, x, ldx, w, ldw, b, r, ldr, y, ldy, z, m, n, k, (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_linear_backward_workspace(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *dy,
                                                      int64_t lddy, int64_t m, int64_t n, int64_t k)
{
    if (!good_linear(dtype, act, ldx, ldw, m, n, k) || lddy < n) return -1;
    int64_t most = 0;                       // of what a call may leave out
    for (int want = 0; want < 4; want++) {
        const int64_t t = linear_backward_layout(dtype, act, x, ldx, w, ldw, dy, lddy, m, n, k, want & 1, want & 2).total;
        most = t > most ? t : most;
    }
    return most;
}

extern "C" int nirrt_nn_linear_backward(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *z, const void *dy,
                                        int64_t lddy, void *dx, void *dw, void *db, int64_t m, int64_t n, int64_t k, void *workspace, void *stream)
{
    if (!good_linear(dtype, act, ldx, ldw, m, n, k) || lddy < n) return -1;
    if (m > 0 && n > 0 && (!dy || (act != NIRRT_NN_ACT_NONE && !z))) return -1;
    if ((dx && m > 0 && n > 0 && k > 0 && !w) || (dw && m > 0 && n > 0 && k > 0 && !x)) return -1;
    if (!workspace && linear_backward_layout(dtype, act, x, ldx, w, ldw, dy, lddy, m, n, k, dx != nullptr, dw != nullptr).total > 0) return -1;
#define CALL(T) linear_backward_t<T>(dtype, act, x, ldx, w, ldw, z, dy, lddy, dx, dw, db, m, n, k, (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

static bool good_cross_entropy(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    return good_type(dtype) && good_dims(rows, classes, k) && classes >= 1 && padded(dtype, k) * elem_size(dtype) <= KC_ROW_BYTES &&
           (classes <= 8 || rows < 1 << 29);          // (k_ce_rows: eight lanes per row, 2^32 in a launch)
}

extern "C" int64_t nirrt_nn_cross_entropy_workspace(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    if (!good_cross_entropy(dtype, rows, classes, k)) return -1;
    return ce_layout(dtype, rows, classes, k).total;
}

extern "C" int nirrt_nn_cross_entropy(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target,
                                      const float *class_weight, int64_t ignore_index, float *lse, float *nll, float *total, int64_t rows,
                                      int64_t classes, int64_t k, void *workspace, void *stream)
{
    if (!good_cross_entropy(dtype, rows, classes, k) || !total || ldx < k || ldw < k) return -1;
    if (rows > 0 && (!target || !lse || !nll || !workspace || (k > 0 && (!x || !w)))) return -1;
#define CALL(T) ce_forward_t<T>(dtype, x, ldx, w, ldw, b, target, class_weight, ignore_index, (float2 *)lse, nll, total, rows, classes, k, (char *)workspace, (hipStream_t)stream)
    return BY_TYPE(dtype, CALL);
#undef CALL
}

extern "C" int64_t nirrt_nn_cross_entropy_backward_workspace(int dtype, int64_t rows, int64_t classes, int64_t k)
{
    if (!good_cross_entropy(dtype, rows, classes, k)) return -1;
    return ce_backward_layout(dtype, rows, classes, k).total;
}

extern "C" int nirrt_nn_cross_entropy_backward(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b,
                                               const int64_t *target, const float *class_weight, int64_t ignore_index, const float *lse,
                                               const float *dloss, int dloss_stride, const float *total, void *dx, void *dw, void *db,
                                               int64_t rows, int64_t classes, int64_t k, void *workspace, void *stream)
{
    if (!good_cross_entropy(dtype, rows, classes, k) || ldx < k || ldw < k || !workspace) return -1;
    if (dloss_stride != 0 && dloss_stride != 1) return -1;
    if (rows > 0 && (!target || !lse || !dloss || (k > 0 && (!x || !w)))) return -1;
#define CALL(T)                                                                                                                                  \
    ce_backward_t<T>(dtype, x, ldx, w, ldw, b, target, class_weight, ignore_index, (const float2 *)lse, dloss, dloss_stride, total, dx, dw, db, rows, classes, k, \
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
    const int64_t blocks = for_tables(tensors, count, false, [&](const TensorTable &t, int64_t first, int64_t n) {
        hipLaunchKernelGGL(k_norm_parts, dim3((unsigned)n), dim3(256), 0, st, t, parts + first);
        return status();
    });
    if (blocks < 0) return (int)blocks;
    hipLaunchKernelGGL(k_norm_total, dim3(1), dim3(1024), 0, st, parts, blocks, norm);
    return status();
}

extern "C" int nirrt_nn_scale_by_norm(const nirrt_nn_tensor *tensors, int32_t count, const float *norm, float max_norm, void *stream)
{
    if (!good_tensors(tensors, count, true) || !norm || !(max_norm >= 0.f)) return -1;
    hipStream_t st = (hipStream_t)stream;
    // (from the last tensor on: what the norm read last is still in the 256 MB cache)
    const int64_t blocks = for_tables(tensors, count, true, [&](const TensorTable &t, int64_t, int64_t n) {
        hipLaunchKernelGGL(k_scale, dim3((unsigned)n), dim3(256), 0, st, t, norm, max_norm);
        return status();
    });
    return blocks < 0 ? (int)blocks : 0;
}
