// tlk_gau.hpp -- device side of the gated attention unit's core (tlk_gau_attention_fwd / _bwd), one template for float16, bfloat16 and float32.
//
//   S_ij = scale * q_i . k_j + bias[clip(j - (i + start), -D, D)]      (bias: the learned table, expanded over distances)
//   W    = relu(S)^2  or  softmax_j(S);   O = W v;   out = gate * O
//
// Tiles are 16 x 16 MFMA tiles with 32 products each (16-bit: one v_mfma_f32_16x16x32; float32: eight v_mfma_f32_16x16x4 over the same eight values
// a lane holds).  Every product is formed TRANSPOSED so that the row statistics live in one lane: S^T = K Q^T puts a query in a lane's column, four
// consecutive keys in its registers, and those registers -- converted -- are already the B operand of O^T = V^T W^T: which 32 keys a lane's eight
// operand slots name is free as long as both operands agree, so the weights never pass through shared memory.  V^T comes from the row-major V tile
// by the transposing LDS read (ds_read_b64_tr_b16).  The backward kernels use the same scheme: dQ with a query, dK / dV with a key in the column.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "tlk_lanes.hpp"

// the launch bounds below are meant for the registers; workgroups of one or two waves, and wide tiles, reach fewer waves for their LDS
#pragma clang diagnostic ignored "-Wpass-failed"

namespace tlk {
namespace gau {

enum { RELU2 = 0, SOFTMAX = 1 };

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG = -3.402823466e38f;         // running maximum before the first key: the lowest finite number, so no score lies below it

struct Args {
    const void *q, *k, *v, *gate;
    const void *table;                          // (num_buckets, heads)
    const int *bucket_of, *lens, *q_start;
    long long qs[3], ks[3], vs[3], gs[3];       // batch, row, head strides in elements
    int B, Lq, Lk, H, Hk, dk, dv, nb, D, q0, causal, table_f32;
    float scale;
    // forward
    void *out, *o;
    float *lse;                                 // (B, Lq, H, 2): the row's largest x = S log2 e, and log2 of its sum of 2^(x - largest), +inf for a row without keys
    float *part, *ml;                           // split keys: (split, B, Lq, H, dv) sums and (split, B, Lq, H, 2) maximum and sum
    int nsplit, split_keys, nchunk, nrow, fold, nparts, snake;
    // backward
    const void *dO;                             // (B, Lq, H, dv) contiguous: the gradient behind the gate
    const void *dO_low;                         // the same shape: what dO's rounding left (16-bit types with a gate and a table)
    const float *dO_exp;                        // (B, Lq, H): dO stands at 2^-dO_exp of its row (float16 with a gate; null: as it is)
    const float *delta, *delta_q;               // (B, Lq, H): sum_d dO o (softmax), at dO's scale; dq's with both parts of dO
    void *dq, *dk_, *dv_;
    float *dq_part, *dk_part, *dv_part;         // (chunk, B, Lq, H, dk); (chunk x part, B, Lk, Hk, dk), (part, B, Lk, Hk, dv): sums of several blocks, joined afterwards
    float *db_part;                             // (heads, B * chunk * nrow * waves, 2 D + 1)
};

template <class T> struct Ty;
template <> struct Ty<_Float16> {
    using V4 = h4;
    using V8 = h8;
    static constexpr bool scaled = true;        // relu^2 weights and score gradients pass float16's range: held with a running power of two
    static __device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Ty<__bf16> {
    using V4 = b4;
    using V8 = b8;
    static constexpr bool scaled = false;
    static __device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Ty<float> {
    using V4 = f4;
    using V8 = f8;
    static constexpr bool scaled = false;
    static __device__ __forceinline__ f4 mma(f8 a, f8 b, f4 c)
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// o as it is kept for the backward pass: float16 relu^2 weights are no shares of one, and o may pass 65504 where the gate brings the result back
template <class T, int KIND> using Kept = std::conditional_t<KIND == RELU2 && Ty<T>::scaled, float, T>;
template <class O> __device__ __forceinline__ void keep4(void *o, long long at, f4 x)
{
    typename Ty<O>::V4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = (O)x[r];
    *reinterpret_cast<typename Ty<O>::V4 *>(reinterpret_cast<O *>(o) + at) = y;
}

template <class T> __device__ __forceinline__ typename Ty<T>::V8 zero8()
{
    typename Ty<T>::V8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)0.f;
    return r;
}

// eight consecutive values of a row in global memory, `left` of them within its width (which is a multiple of 16 bytes); the others zero and not read
template <class T> __device__ __forceinline__ typename Ty<T>::V8 ld8(const T *p, int left)
{
    typename Ty<T>::V8 r = zero8<T>();
    if constexpr (sizeof(T) == 2) {
        if (left > 0) r = *reinterpret_cast<const typename Ty<T>::V8 *>(p);
    } else {
        f4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
        if (left > 0) a = *reinterpret_cast<const f4 *>(p);
        if (left > 4) b = *reinterpret_cast<const f4 *>(p + 4);
        r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return r;
}

// A ROWS x COLS tile in LDS, filled by direct-to-LDS loads: 64 lanes x 16 bytes land in 1024 consecutive bytes, so the tile has no padding; instead the
// 16-byte chunk c of row r stands at c ^ twist(r), which spreads the 16 rows of a fragment read and of a transposing read over all banks.  The loads go
// through a buffer descriptor: rows behind the end and columns behind the width get an offset out of its range and arrive as zeros.
template <class T, int ROWS, int COLS, int NW> struct Tile {
    static constexpr int VN = 16 / sizeof(T), C = COLS / VN, ROWB = COLS * sizeof(T), BYTES = ROWS * ROWB, N = (ROWS * C / 64 + NW - 1) / NW;
    static constexpr unsigned OOB = 0x80000000u;
    static_assert(C >= 8 && (C & (C - 1)) == 0 && ROWS * C % 64 == 0, "whole wave loads of rows of at least 128 bytes");
    static __device__ __forceinline__ int twist(int r) { return C >= 16 ? ((r << 1) & 15) | ((r >> 3) & 1) : (r >> 1) & 7; }
    unsigned off[N];
    int wave;
    __device__ __forceinline__ void init(int w, int lane, long long rs, int cend)
    {
        wave = w;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (i * NW + w) * 64 + lane, row = at / C, c = (at % C) ^ twist(row);
            off[i] = c * VN < cend ? (unsigned)(row * (int)rs * (int)sizeof(T) + c * 16) : OOB;
        }
    }
    // the buffer descriptor of the tile whose first row `base` is, with `rows` rows left (uniform): it ends with the last of them, so that the loads of the
    // rows behind it return zeros by themselves (row strides are not below the width: host check)
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_at(const T *base, int rows, long long rs)
    {
        const int n = rows < 0 ? 0 : (rows < ROWS ? rows : ROWS);
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, n * (int)rs * (int)sizeof(T), 0x00020000);
    }
    // the i-th of the wave's N loads
    __device__ __forceinline__ void load(const __amdgpu_buffer_rsrc_t &rsrc, char *lds, int i) const
    {
        const int inst = i * NW + wave;
        if (ROWS * C / 64 % NW != 0 && inst >= ROWS * C / 64) return;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void *)(lds + inst * 1024), 16, (int)off[i], 0, 0, 0);
    }
    __device__ __forceinline__ void issue(const T *base, int rows, long long rs, char *lds) const
    {
        const __amdgpu_buffer_rsrc_t rsrc = tile_at(base, rows, rs);
#pragma unroll
        for (int i = 0; i < N; ++i) load(rsrc, lds, i);
    }
    // Fragment reads.  A lane's place in the first fragment (row_at, col_at) is made once per tile and hidden from the optimiser; the place in any other is
    // one exclusive or with a constant (rows begin at multiples of the twisted field) plus a constant.  Left visible, all places of a tile are kept in
    // registers across the loop -- up to 24 of them, where the accumulators leave none.  (One step from the buffer's start to the address: after a few
    // steps the compiler loses track of which object a pointer came from, and waits for loads it need not wait for.)
    static constexpr int M = (C < 16 ? C : 16) - 1;
    static __device__ __forceinline__ int chunk(int c) { return c / (M + 1) * ((M + 1) * 16); }
    static __device__ __forceinline__ int row_at(int at, int g, int l)
    {
        int o = at + l * ROWB + (((sizeof(T) == 2 ? g : 2 * g) ^ twist(l)) << 4);
        asm volatile("" : "+v"(o));
        return o;
    }
    // values 32 ks + 8 g .. + 7 of row 16 n + l
    static __device__ __forceinline__ typename Ty<T>::V8 row8(const char *buf, int place, int n, int ks)
    {
        const int c = ks * 32 / VN, o = (place ^ ((c & M) << 4)) + chunk(c) + n * 16 * ROWB;
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const typename Ty<T>::V8 *>(buf + o);
        } else {
            const int o1 = (place ^ ((c & M) << 4) ^ 16) + chunk(c) + n * 16 * ROWB;
            const f4 a = *reinterpret_cast<const f4 *>(buf + o);
            const f4 b = *reinterpret_cast<const f4 *>(buf + o1);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    struct Col { int o[sizeof(T) == 2 ? 1 : 4]; };
    static __device__ __forceinline__ Col col_at(int at, int g, int l)
    {
        Col p;
#pragma unroll
        for (int i = 0; i < (sizeof(T) == 2 ? 1 : 4); ++i) {
            const int r = g * 4 + (sizeof(T) == 2 ? l >> 2 : i);
            p.o[i] = sizeof(T) == 2 ? at + r * ROWB + ((((l >> 1) & 1) ^ twist(r)) << 4) + (l & 1) * 8 : at + r * ROWB + (((l >> 2) ^ twist(r)) << 4) + (l & 3) * 4;
            asm volatile("" : "+v"(p.o[i]));
        }
        return p;
    }
    // rows r0 + 4 g + 0..3 of column 16 n + l (r0 a multiple of 16)
    static __device__ __forceinline__ typename Ty<T>::V4 col4(const char *buf, const Col &place, int r0, int n)
    {
        const int c = n * 16 / VN;
        if constexpr (sizeof(T) == 2) {
            const int o = (place.o[0] ^ ((c & M) << 4)) + chunk(c) + r0 * ROWB;
            return __builtin_bit_cast(typename Ty<T>::V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(buf + o)));
        } else {
            typename Ty<T>::V4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int o = (place.o[i] ^ ((c & M) << 4)) + chunk(c) + r0 * ROWB;
                v[i] = *reinterpret_cast<const float *>(buf + o);
            }
            return v;
        }
    }
    static __device__ __forceinline__ typename Ty<T>::V8 col8(const char *buf, const Col &place, int r0, int n)      // rows r0 + 4 g + 0..3 and r0 + 16 + 4 g + 0..3
    {
        return __builtin_shufflevector(col4(buf, place, r0, n), col4(buf, place, r0 + 16, n), 0, 1, 2, 3, 4, 5, 6, 7);
    }
};
// every load of this wave has landed in LDS and every read has returned; then the same for the workgroup
__device__ __forceinline__ void tiles_ready()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70);               // vmcnt(0) lgkmcnt(0), as a builtin: the compiler then knows that nothing is in flight into this tile
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <class T> __device__ __forceinline__ typename Ty<T>::V8 pack8(f4 a, f4 b)
{
    typename Ty<T>::V8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (T)a[i];
        r[4 + i] = (T)b[i];
    }
    return r;
}

// widths come in steps of 32 (64, 96, 128 for q and k), rows of a tile in powers of two
constexpr int tile_width(int dk) { return dk == 96 ? 128 : dk; }
// fragments in flight: 4, or the 3 that divide a count of 6
constexpr int batch(int n) { return n % 4 == 0 ? 4 : (n % 3 == 0 ? 3 : (n % 2 == 0 ? 2 : 1)); }
// N fragments from LDS, each used by a few matrix instructions: B of them are read while the B before are multiplied.  (An LDS read takes longer than
// the two instructions that one fragment feeds; left to itself the compiler keeps one or two reads in flight and every fragment waits.)
// `first`: the first B fragments, read by fragments() earlier, behind other work.
template <int B, class V8, class Load> __device__ __forceinline__ void fragments(V8 (&f)[B], int from, Load load)
{
#pragma unroll
    for (int i = 0; i < B; ++i) f[i] = load(from + i);
}
template <int N, int B, class V8, class Load, class Use> __device__ __forceinline__ void stream(V8 (&first)[B], Load load, Use use)
{
    static_assert(N % B == 0, "whole batches");
    V8 f[2][B];
#pragma unroll
    for (int i = 0; i < B; ++i) f[0][i] = first[i];
#pragma unroll
    for (int s = 0; s < N / B; ++s) {
        if (s + 1 < N / B) fragments(f[(s + 1) & 1], (s + 1) * B, load);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < B; ++i) use(s * B + i, f[s & 1][i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// The learned table over distances of head h, in LDS: -D .. D with MARGIN more entries of the end values on both sides, so that a tile that reaches
// across +-D is looked up without clipping (a wave's tile spans fewer than MARGIN distances).  Softmax works in powers of two, so its bias carries
// log2 e; beyond 1e38 the factor is 0.8, so that finite values stay finite and in order (two that differ there differ by 1e31 and more).
constexpr int MARGIN = 128;
__host__ __device__ __forceinline__ int table_width(int D) { return 2 * D + 1 + 2 * MARGIN; }
template <class T, int KIND> __device__ __forceinline__ void expand_bias(const Args &p, int h, float *dst, int nth)
{
    const int TW = table_width(p.D);
    for (int t = threadIdx.x; t < TW; t += nth) {
        int b = p.bucket_of[min(max(t - MARGIN, 0), 2 * p.D)];
        b = b < 0 ? 0 : (b >= p.nb ? p.nb - 1 : b);
        const long long at = (long long)b * p.H + h;
        float x = p.table_f32 ? reinterpret_cast<const float *>(p.table)[at] : (float)reinterpret_cast<const T *>(p.table)[at];
        if (KIND == SOFTMAX) {
            const float a = fabsf(x);
            x = a > 1.0e38f && a < INFINITY ? copysignf(1.0e38f * LOG2E + (a - 1.0e38f) * 0.8f, x) : x * LOG2E;
        }
        dst[t] = x;
    }
}

// the row tile of the n-th place: the longest causal walks first, from place `snake` on the shortest first
__device__ __forceinline__ int row_tile(const Args &p, int n) { return n < p.snake ? p.nrow - 1 - n : n - p.snake; }
__device__ __forceinline__ int key_end(const Args &p, int b) { const int n = p.lens ? p.lens[b] : p.Lk; return n < 0 ? 0 : (n > p.Lk ? p.Lk : n); }
__device__ __forceinline__ int row_start(const Args &p, int b)
{
    const int lim = 1 << 29, s = p.q_start ? p.q_start[b] : p.q0;
    return s < -lim ? -lim : (s > lim ? lim : s);
}

__device__ __forceinline__ float over_groups_max(float x) { return lanes_32<LaneMax>(lanes_16<LaneMax>(x)); }
__device__ __forceinline__ float over_groups_sum(float x) { return lanes_32<LaneAdd>(lanes_16<LaneAdd>(x)); }
__device__ __forceinline__ int wave_min_i(int x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ int wave_max_i(int x)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float relu_(float x) { return __builtin_elementwise_maximum(x, 0.f); }      // (v_maximum3: NaN stays NaN)
__device__ __forceinline__ float pow2_(float x) { return __builtin_amdgcn_exp2f(x); }                  // (one instruction, 1 ulp; below 2^-126: zero)

// running power of two of a column's float16 operands: values times 2^-e stay below 2^7; `t` = largest magnitude of this tile's column.
// Returns the factor for what has been summed so far (1 where nothing changes).
__device__ __forceinline__ float raise_exponent(int &e, float t)
{
    if (!(ldexpf(t, -e) > 128.f)) return 1.f;
    int n;
    (void)frexpf(t, &n);                          // t in [2^(n-1), 2^n)
    if (!(t < 1.3e36f)) n = 120;
    const float f = ldexpf(1.f, e - n < -150 ? -150 : e - n);
    e = n;
    return f;
}
constexpr int E_NONE = -120;                      // exponent before the first non-zero value

// four scores of a lane: scale and bias.  `near`: the table at the first one's distance, STEP entries further with every row; where
// the whole tile lies beyond +-D (or there is no bias) one value does for all (uniform over the wave).
template <int STEP> __device__ __forceinline__ void add_bias(f4 &s, float sc, bool is_near, const float *near, float far)
{
    if (is_near) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(s[r], sc, near[STEP * r]);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(s[r], sc, far);
    }
}

// The statistics of a softmax row.  Two numbers: next to a largest score of 10^4 and more, log2 of the sum is rounded away in one (float32, all keys of a row at a
// bias of -10^9: every weight 1 in the backward pass where it is one share of n).
__device__ __forceinline__ void keep_sum(float *lse, long long row, float m, float sum)
{
    lse[2 * row] = m;
    lse[2 * row + 1] = sum == 0.f ? INFINITY : log2f(sum);
}

// ------------------------------------------------------------------------------------------------------------------------------------ forward
// WM x WN waves; a wave owns MT x 16 rows and NT x 16 columns of the output.  Rows of a block are (head of the group, query) pairs when p.fold
// (few queries: the heads that share keys and values are answered in one pass over them).
// Block order, here and in the backward kernels: sequences, key heads and chunks of dv vary fastest, so that the blocks that walk the same keys land on
// one XCD (workgroups go to the 8 XCDs in turn) and share its L2; row tiles vary slowest, the longest causal walks first.
// Bound by: matrix cores where rows are many (4 x 8192 causal bf16 tokens, dk 128, dv 1024: 372 us, 826 TFLOP/s with S counted once; it is formed for each of
// four chunks of dv), HBM where they are few (32 x 1 token over 16384 keys, 16 heads on 4, bf16: 156 us, 4.6 TB/s; 2400 x 17 tokens f16, dv 512: 39 us, 3.7 TB/s).
template <class T, int KIND, int DK, int MT, int NT, int WM, int WN, int KT, bool ONE>
__global__ void __launch_bounds__(64 * WM * WN, WN > 1 && sizeof(T) == 2 ? (MT * NT <= 4 ? 4 : (MT * NT <= 8 ? 3 : 2)) : 2) fwd_kernel(const Args p)
{
    using V8 = typename Ty<T>::V8;
    constexpr int NTH = 64 * WM * WN, BM = WM * MT * 16, DVB = WN * NT * 16, NS = KT / 16;
    using TK = Tile<T, KT, tile_width(DK), WM * WN>;
    using TV = Tile<T, KT, DVB, WM * WN>;
    constexpr int BUF = TK::BYTES + TV::BYTES;
    // (two objects and a loop that names them in turn, not one with an offset: the compiler then knows that a transposing read of one cannot see the loads
    // in flight into the other; with one object it drains them before the first such read.  ONE: all keys are one tile, one buffer.)
    __shared__ __attribute__((aligned(1024))) char buf0[BUF], buf1[ONE ? 16 : BUF];
    extern __shared__ __attribute__((aligned(16))) float tab[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w / WN, wn = w - wm * WN, g = lane >> 4, l = lane & 15;
    const int G = p.H / p.Hk, GB = p.fold ? G : 1, HB = p.H / GB, rows = p.Lq * GB, TW = table_width(p.D);
    int id = blockIdx.x;
    const int b = id % p.B; id /= p.B;
    const int hk = id % p.Hk; id /= p.Hk;
    const int ch = id % p.nchunk; id /= p.nchunk;
    const int sp = id % p.nsplit; id /= p.nsplit;
    const int hg = id % (HB / p.Hk), rt = row_tile(p, id / (HB / p.Hk)), h0 = hk * G + hg;
    const int kend_all = key_end(p, b), q0 = row_start(p, b);
    const int c0 = ch * DVB, cend = p.dv - c0;
    const T *Q = reinterpret_cast<const T *>(p.q) + b * p.qs[0];
    const T *K = reinterpret_cast<const T *>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T *V = reinterpret_cast<const T *>(p.v) + b * p.vs[0] + hk * p.vs[2] + c0;
    // keys of this block: its split, below the length, and not beyond its last row's position
    int kb = sp * p.split_keys, ke = min(kend_all, p.nsplit > 1 ? kb + p.split_keys : kend_all);
    if (p.causal) {
        const int r0 = rt * BM, r1 = min(rows, r0 + BM) - 1;
        const int last = (r0 / p.Lq == r1 / p.Lq) ? r1 % p.Lq : p.Lq - 1;
        ke = min(ke, last + q0 + 1);
    }
    TK tk;
    TV tv;
    tk.init(w, lane, p.ks[1], p.dk);
    tv.init(w, lane, p.vs[1], cend);
    K += kb * p.ks[1];
    V += kb * p.vs[1];
    const long long kstep = KT * p.ks[1], vstep = KT * p.vs[1];
    if (kb < ke) {
        tk.issue(K, ke - kb, p.ks[1], buf0);
        tv.issue(V, ke - kb, p.vs[1], buf0 + TK::BYTES);
    }
    if (p.table)
        for (int i = 0; i < GB; ++i) expand_bias<T, KIND>(p, h0 + i, tab + i * TW, NTH);
    int qi[MT], qh[MT], pos[MT];
    bool ok[MT];
    V8 qf[MT][DK / 32];
    int pmin = 0x7fffffff, pmax = -0x7fffffff;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int r = rt * BM + (wm * MT + mt) * 16 + l;
        ok[mt] = r < rows;
        const int rr = ok[mt] ? r : 0, hi = rr / p.Lq;
        qi[mt] = rr - hi * p.Lq;
        qh[mt] = hi;
        pos[mt] = qi[mt] + q0;
        if (ok[mt]) { pmin = min(pmin, pos[mt]); pmax = max(pmax, pos[mt]); }
        const T *src = Q + (long long)qi[mt] * p.qs[1] + (h0 + hi) * p.qs[2] + g * 8;
#pragma unroll
        for (int ks = 0; ks < DK / 32; ++ks) qf[mt][ks] = ld8(src + ks * 32, ok[mt] ? p.dk - ks * 32 - g * 8 : 0);
    }
    // Few rows: a block has one or two tiles to walk, and what surrounds them is what it costs.  The results go through LDS, 16 rows at a time, so that
    // gate, o and out move as whole rows, 16 bytes a lane (from the accumulators a lane has 8 bytes of each of 16 rows: eight times as many lines to
    // touch; 2400 crops of 17 x 512 f16: 45 -> 40 us), and the gate is fetched along with everything else.
    constexpr bool EARLY = WN > 1;
    constexpr int VN = 16 / sizeof(T), RC = DVB / VN, CH = (16 * RC + NTH - 1) / NTH, LDE = DVB + 4;
    static_assert(!EARLY || 16 * LDE * 4 <= BUF, "16 rows of results fit a tile's buffer");
    u4 early[EARLY ? MT * CH : 1];
    const auto piece = [&](int mt, int i, int &er, int &ec, int &eq, int &eh) __attribute__((always_inline)) {       // this lane's i-th 16 bytes of 16 rows
        const int at = i * NTH + tid, r = (er = at / RC, rt * BM + mt * 16 + er);
        ec = (at - er * RC) * VN;
        if (at >= 16 * RC || r >= rows || ec >= cend) return false;
        eh = r / p.Lq;
        eq = r - eh * p.Lq;
        return true;
    };
    if (EARLY && p.gate && p.nsplit == 1) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                int er, ec, eq, eh;
                if (piece(mt, i, er, ec, eq, eh))
                    early[mt * CH + i] = *reinterpret_cast<const u4 *>(reinterpret_cast<const T *>(p.gate) + b * p.gs[0] + (long long)eq * p.gs[1] + (h0 + eh) * p.gs[2] + c0 + ec);
            }
    }
    pmin = __builtin_amdgcn_readfirstlane(wave_min_i(pmin));
    pmax = __builtin_amdgcn_readfirstlane(wave_max_i(pmax));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        if (!ok[mt]) pos[mt] = pmax;                               // (lanes without a row stay within the wave's distances)
    f4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[n][mt] = f4{0, 0, 0, 0};
    float m[MT], lsum[MT];
    int ex[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) { m[mt] = NEG; lsum[mt] = 0.f; ex[mt] = E_NONE; }
    const float sc = KIND == SOFTMAX ? p.scale * LOG2E : p.scale;
    float flo[MT], fhi[MT];                                        // the bias beyond +-D
    if (p.table) __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        flo[mt] = p.table ? tab[qh[mt] * TW] : 0.f;
        fhi[mt] = p.table ? tab[qh[mt] * TW + TW - 1] : 0.f;
    }    const auto step = [&](const char *cur, char *next, int j0) __attribute__((always_inline)) {
        tiles_ready();                                             // this tile has landed, and the other buffer is free
        K += kstep;
        V += vstep;
        if (!ONE) {                                                // the next tile's loads (behind the last tile they fetch nothing)
            tk.issue(K, ke - j0 - KT, p.ks[1], next);
            tv.issue(V, ke - j0 - KT, p.vs[1], next + TK::BYTES);
        }
        if (pmin > pmax || (p.causal && j0 > pmax)) return;        // no row of this wave, or none that sees this tile (uniform over the wave)
        f4 s[MT][NS];
        constexpr int KS = DK / 32, BK = batch(NS * KS), BV = batch(NT);
        const int krow = TK::row_at(0, g, l);
        const typename TV::Col vcol = TV::col_at(TK::BYTES, g, l);
        const auto key = [&](int i) __attribute__((always_inline)) { return TK::row8(cur, krow, i / KS, i % KS); };
        const auto val = [&](int i) __attribute__((always_inline)) { return TV::col8(cur, vcol, i / NT * 32, wn * NT + i % NT); };
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][n] = f4{0, 0, 0, 0};
        V8 kf[BK], vf[BV];
        fragments(kf, 0, key);
        stream<NS * KS, BK>(kf, key, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][i / KS] = Ty<T>::mma(a, qf[mt][i % KS], s[mt][i / KS]);
        });
        fragments(vf, 0, val);
        __builtin_amdgcn_sched_barrier(0);
        // scores: scale, bias, mask; most tiles lie beyond +-D of all rows and are seen by all of them
        const bool full = j0 + KT <= ke && (!p.causal || j0 + KT - 1 <= pmin);
        const int where = !p.table || j0 - pmax >= p.D ? 1 : (j0 + KT - 1 - pmin <= -p.D ? 2 : 3);
        if (full && where != 3) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float far = where == 1 ? fhi[mt] : flo[mt];
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[mt][n][r] = __builtin_fmaf(s[mt][n][r], sc, far);
            }
        } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int last = p.causal ? min(ke - 1, pos[mt]) : ke - 1;
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    add_bias<1>(s[mt][n], sc, where == 3, tab + qh[mt] * TW + (p.D + MARGIN + j0 + n * 16 + g * 4 - pos[mt]), where == 1 ? fhi[mt] : flo[mt]);
                    if (!full)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j0 + n * 16 + g * 4 + r > last) s[mt][n][r] = KIND == SOFTMAX ? -INFINITY : 0.f;
                }
            }
        }
        // weights
        float fac[MT];
        bool any = false;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            fac[mt] = 1.f;
            float down = 1.f;
            if (KIND == SOFTMAX || Ty<T>::scaled) {
                float t = s[mt][0][0];
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) t = fmaxf(t, s[mt][n][r]);
                t = over_groups_max(t);
                if (KIND == SOFTMAX) {
                    const float mn = fmaxf(m[mt], t);
                    fac[mt] = pow2_(m[mt] - mn);
                    m[mt] = mn;
                    lsum[mt] *= fac[mt];
                } else {
                    const float f = raise_exponent(ex[mt], t);
                    fac[mt] = f * f;
                    down = ldexpf(1.f, -ex[mt]);
                }
                any |= fac[mt] != 1.f;
            }
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = s[mt][n][r];
                    if (KIND == SOFTMAX) {
                        x = pow2_(x - m[mt]);
                        lsum[mt] += x;
                    } else {
                        x = relu_(x);
                        if (Ty<T>::scaled) x *= down;
                        x = x * x;
                    }
                    s[mt][n][r] = x;
                }
        }
        if ((KIND == SOFTMAX || Ty<T>::scaled) && __any(any)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[n][mt] *= fac[mt];
        }
        V8 pb[NS / 2][MT];
#pragma unroll
        for (int kk = 0; kk < NS / 2; ++kk)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) pb[kk][mt] = pack8<T>(s[mt][2 * kk], s[mt][2 * kk + 1]);
        stream<NS / 2 * NT, BV>(vf, val, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[i % NT][mt] = Ty<T>::mma(a, pb[i / NT][mt], acc[i % NT][mt]);
        });
    };
    if constexpr (ONE) {
        if (kb < ke) step(buf0, buf1, kb);
    } else {
        for (int j0 = kb; j0 < ke; j0 += 2 * KT) {
            step(buf0, buf1, j0);
            if (j0 + KT < ke) step(buf1, buf0, j0 + KT);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);                        // (vmcnt(0): nothing is on its way to LDS when the workgroup ends)
    }
    if (EARLY && p.nsplit == 1) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float fin = 1.f;
            if (KIND == SOFTMAX) {
                lsum[mt] = over_groups_sum(lsum[mt]);
                fin = lsum[mt] == 0.f ? 0.f : 1.f / lsum[mt];
                if (p.lse && ok[mt] && c0 == 0 && wn == 0 && g == 0) keep_sum(p.lse, ((long long)b * p.Lq + qi[mt]) * p.H + h0 + qh[mt], m[mt], lsum[mt]);
            } else if (Ty<T>::scaled) {
                fin = ex[mt] == E_NONE ? 0.f : ldexpf(1.f, ex[mt]);
            }
            float *res = reinterpret_cast<float *>(buf0);
            __syncthreads();                                        // the tiles, or the 16 rows before, are no longer read
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                f4 x = acc[n][mt] * fin;
                if (KIND == RELU2 && Ty<T>::scaled) x *= fin;       // (twice: see below)
                *reinterpret_cast<f4 *>(res + l * LDE + (wn * NT + n) * 16 + g * 4) = x;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                int er, ec, eq, eh;
                if (!piece(mt, i, er, ec, eq, eh)) continue;
                const long long at = (((long long)b * p.Lq + eq) * p.H + h0 + eh) * p.dv + c0 + ec;
                T y[VN], u[VN];
                __builtin_memcpy(u, &early[mt * CH + i], 16);
                float x[VN];
#pragma unroll
                for (int e = 0; e < VN; e += 4) *reinterpret_cast<f4 *>(x + e) = *reinterpret_cast<const f4 *>(res + er * LDE + ec + e);
                u4 raw;
                if (p.o) {
                    if constexpr (std::is_same_v<Kept<T, KIND>, T>) {
#pragma unroll
                        for (int e = 0; e < VN; ++e) y[e] = (T)x[e];
                        __builtin_memcpy(&raw, y, 16);
                        *reinterpret_cast<u4 *>(reinterpret_cast<T *>(p.o) + at) = raw;
                    } else {
#pragma unroll
                        for (int e = 0; e < VN; e += 4) *reinterpret_cast<f4 *>(reinterpret_cast<float *>(p.o) + at + e) = *reinterpret_cast<const f4 *>(x + e);
                    }
                }
#pragma unroll
                for (int e = 0; e < VN; ++e) y[e] = (T)(p.gate ? x[e] * (float)u[e] : x[e]);
                __builtin_memcpy(&raw, y, 16);
                *reinterpret_cast<u4 *>(reinterpret_cast<T *>(p.out) + at) = raw;
            }
        }
        return;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (KIND == SOFTMAX) lsum[mt] = over_groups_sum(lsum[mt]);
        if (!ok[mt]) continue;
        const long long row = ((long long)b * p.Lq + qi[mt]) * p.H + h0 + qh[mt];
        float fin = 1.f;
        if (KIND == SOFTMAX) fin = p.nsplit > 1 ? 1.f : (lsum[mt] == 0.f ? 0.f : 1.f / lsum[mt]);
        else if (Ty<T>::scaled) fin = ex[mt] == E_NONE ? 0.f : ldexpf(1.f, ex[mt]);      // applied twice: the square may pass float32 where the product does not
        constexpr bool TWICE = KIND == RELU2 && Ty<T>::scaled;
        const int cw = c0 + wn * NT * 16;
        if (p.nsplit > 1) {
            const long long at = (long long)sp * p.B * p.Lq * p.H + row;
            if (KIND == SOFTMAX && c0 == 0 && wn == 0 && g == 0) { p.ml[2 * at] = m[mt]; p.ml[2 * at + 1] = lsum[mt]; }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int c = cw + n * 16 + g * 4;
                f4 x = acc[n][mt] * fin;
                if (TWICE) x *= fin;
                if (c < p.dv) *reinterpret_cast<f4 *>(p.part + at * p.dv + c) = x;
            }
            continue;
        }
        if (p.lse && c0 == 0 && wn == 0 && g == 0) keep_sum(p.lse, row, m[mt], lsum[mt]);
        const T *gp = p.gate ? reinterpret_cast<const T *>(p.gate) + b * p.gs[0] + (long long)qi[mt] * p.gs[1] + (h0 + qh[mt]) * p.gs[2] : nullptr;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c = cw + n * 16 + g * 4;
            if (c >= p.dv) continue;
            f4 x = acc[n][mt] * fin;
            if (TWICE) x *= fin;
            typename Ty<T>::V4 y;
            if (p.o) keep4<Kept<T, KIND>>(p.o, row * p.dv + c, x);
            if (gp) {
                const typename Ty<T>::V4 u = *reinterpret_cast<const typename Ty<T>::V4 *>(gp + c);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] *= (float)u[r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = (T)x[r];
            *reinterpret_cast<typename Ty<T>::V4 *>(reinterpret_cast<T *>(p.out) + row * p.dv + c) = y;
        }
    }
}

// joins the key splits: a wave per row and 64 columns; 16 lanes hold the columns, four groups of lanes every fourth split each
// (512 rows of 128 in 16 splits: 6 us, a launch's own time; a lane for four columns and all splits took 14)
template <class T, int KIND> __global__ void __launch_bounds__(64) join_kernel(const Args p)
{
    const int cg = (p.dv + 63) / 64, lane = threadIdx.x, g = lane >> 4;
    const long long row = blockIdx.x / cg, nrow = (long long)p.B * p.Lq * p.H;
    const int c = (int)(blockIdx.x % cg) * 64 + (lane & 15) * 4;
    const bool in = c < p.dv;
    f4 x = {0, 0, 0, 0};
    float m = NEG, s = 0.f;
    if (KIND == SOFTMAX) {
#pragma unroll 8
        for (int i = g; i < p.nsplit; i += 4) m = fmaxf(m, p.ml[2 * (i * nrow + row)]);
        m = over_groups_max(m);
    }
#pragma unroll 8
    for (int i = g; i < p.nsplit; i += 4) {
        f4 y = {0, 0, 0, 0};
        if (in) y = *reinterpret_cast<const f4 *>(p.part + (i * nrow + row) * p.dv + c);
        if (KIND == SOFTMAX) {
            const float f = pow2_(p.ml[2 * (i * nrow + row)] - m);
            s += f * p.ml[2 * (i * nrow + row) + 1];
            x += y * f;
        } else {
            x += y;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = over_groups_sum(x[r]);
    if (KIND == SOFTMAX) {
        s = over_groups_sum(s);
        x *= s == 0.f ? 0.f : 1.f / s;
        if (p.lse && c == 0 && lane == 0) keep_sum(p.lse, row, m, s);
    }
    if (!in || g) return;
    const int h = (int)(row % p.H);
    const long long bi = row / p.H;
    typename Ty<T>::V4 y;
    if (p.o) keep4<Kept<T, KIND>>(p.o, row * p.dv + c, x);
    if (p.gate) {
        const typename Ty<T>::V4 u = *reinterpret_cast<const typename Ty<T>::V4 *>(reinterpret_cast<const T *>(p.gate) + (bi / p.Lq) * p.gs[0] + (bi % p.Lq) * p.gs[1] + h * p.gs[2] + c);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] *= (float)u[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = (T)x[r];
    *reinterpret_cast<typename Ty<T>::V4 *>(reinterpret_cast<T *>(p.out) + row * p.dv + c) = y;
}

// ----------------------------------------------------------------------------------------------------------------------------------- backward
// behind the gate: dO = dout * gate, dgate = dout * O, delta = sum_d dO * O.  LANES lanes a row; bound by HBM (4 x 4096 rows of 1024 bf16: 34 us, 6 tensors of 34 MB, which the caches hold in part).
// float16: dO stands at a power of two of its row, which puts the largest magnitude at 2^14 .. 2^15 -- the product of two float16 values reaches from 2^-48 to 2^32.
// low: what rounding dO left; the product of two 16-bit values is dO + low exactly (16 bits of bfloat16, 22 of float16).  Each kernel is given the delta of the dO that it multiplies: where
// a row sees one key, dW - delta is nothing, and one with low and one without would leave low . o of it.
template <class T> struct GateArgs {
    const T *dout, *gate;
    const void *o;
    long long gs[3];
    T *dO, *low, *dgate;
    float *delta, *delta_q, *dO_exp;
    long long rows;
    int Lq, H, dv;
};
template <class T, class O, int LANES> __global__ void __launch_bounds__(256) gate_bwd_kernel(const GateArgs<T> p)
{
    using V4 = typename Ty<T>::V4;
    const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    if (row >= p.rows) return;
    const long long bi = row / p.H;
    const T *gp = p.gate ? p.gate + (bi / p.Lq) * p.gs[0] + (bi % p.Lq) * p.gs[1] + (row % p.H) * p.gs[2] : nullptr;
    float d = 0.f, d_low = 0.f, scale = 1.f;
    if constexpr (Ty<T>::scaled)
        if (gp) {
            float top = 0.f;
            for (int c = lane * 4; c < p.dv; c += LANES * 4) {
                const V4 du = *reinterpret_cast<const V4 *>(p.dout + row * p.dv + c), u = *reinterpret_cast<const V4 *>(gp + c);
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf((float)du[r] * (float)u[r]));
            }
            top = lanes_all<LaneMax, LANES>(top);
            int e = 0;                                            // (infinite: as it is)
            if (top < INFINITY) (void)frexpf(top, &e), e -= 15;
            scale = ldexpf(1.f, -e);
            if (lane == 0) p.dO_exp[row] = (float)e;
        }
    for (int c = lane * 4; c < p.dv; c += LANES * 4) {
        const V4 du = *reinterpret_cast<const V4 *>(p.dout + row * p.dv + c);
        const auto o = *reinterpret_cast<const typename Ty<O>::V4 *>(reinterpret_cast<const O *>(p.o) + row * p.dv + c);
        V4 a, b, rest;
        if (gp) {
            const V4 u = *reinterpret_cast<const V4 *>(gp + c);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = (float)du[r] * (float)u[r] * scale;
                a[r] = (T)x;
                rest[r] = (T)(x - (float)a[r]);
                b[r] = (T)((float)du[r] * (float)o[r]);
                d += (float)a[r] * (float)o[r];
                d_low += (float)rest[r] * (float)o[r];
            }
            *reinterpret_cast<V4 *>(p.dO + row * p.dv + c) = a;
            if (p.low) *reinterpret_cast<V4 *>(p.low + row * p.dv + c) = rest;
            *reinterpret_cast<V4 *>(p.dgate + row * p.dv + c) = b;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) d += (float)du[r] * (float)o[r];
        }
    }
    d = lanes_all<LaneAdd, LANES>(d);
    if (p.delta && lane == 0) p.delta[row] = d;
    if (!p.low || !p.delta) return;                               // (uniform over the launch)
    d_low = lanes_all<LaneAdd, LANES>(d_low);
    if (lane == 0) p.delta_q[row] = d + d_low;
}

// dS of one pair from its score x (scaled, biased, masked: -inf; softmax in powers of two), dW and the row's statistics; w returns the weight.  Where dO, and dW
// with it, stand at 2^-e of their row, the weight takes 2^e: lsum is given e lower (and delta as dW), or two = 2 * 2^e -- w is then twice the weight.
template <int KIND, bool SCALED> __device__ __forceinline__ float dscore(float x, float dw, float top, float lsum, float delta, float two, float &w)
{
    if (KIND == SOFTMAX) {
        w = pow2_(x - top - lsum);
        return w * (dw - delta);
    }
    const float s = relu_(x);
    if (SCALED) {
        w = s * (s * two);
        return s * two * dw;
    }
    w = s * s;
    return 2.f * s * dw;
}

// a wave's column tile as float16 operands: divides by the running power of two (see raise_exponent), returns what rescales the sums so far
template <class T, int NS> __device__ __forceinline__ float hold(f4 (&x)[NS], int &e)
{
    if constexpr (!Ty<T>::scaled) return 1.f;
    float t = 0.f;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) t = fmaxf(t, fabsf(x[n][r]));
    const float f = raise_exponent(e, over_groups_max(t)), down = ldexpf(1.f, -e);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[n][r] *= down;
    return f;
}
template <class T> __device__ __forceinline__ float unhold(int e) { return !Ty<T>::scaled ? 1.f : (e == E_NONE ? 0.f : ldexpf(1.f, e)); }

// dQ and the bias gradient: W waves, MT x 16 queries each; walks the keys.  dS^T has a query in the column: its registers are the B operand of
// dQ^T = K^T dS^T.  The bias gradient needs sums along diagonals: a tile that lies beyond +-D of all its queries is one sum in registers, one near
// the diagonal goes through a wave's own (KT x BM) LDS tile and each lane sums two diagonals -- no atomics, the order is fixed.
// Softmax: the score gradients of a row sum to zero, but with delta = dO . o from rounded weights and the rounded o they sum to eta = dO . (W v - o), and an entry
// that most pairs share takes it up over all rows: against sums that cancel by nature it was 1e-2 of the gradient (1137 bf16 tokens, D 16), and the whole of
// it where all distances but one share an entry.  What the row really sums to is known at the end of its walk: eta times the row's weights goes off the sums, beyond +-D as
// one product (the weights are summed on the way), within them in a second walk over the tiles near the diagonal, which forms S and W again and nothing else.
// Bound by the vector work between three products per score tile: 4 x 4096 causal bf16 tokens, dk 128, dv 1024, relu^2: 250 us with two parts of dO, 176 with one; 4 x 2048 tokens, 16 heads of 64,
// softmax, causal: 134 us (of it 38 for eta and 5 for the second statistic of a row).
// LOW: dO comes in two parts.  Rounded once, dO is off by the same amounts for all keys of its row; a bucket's sum over many pairs, which cancel, keeps that (bf16, 4 x 1024
// tokens, relu^2: up to 1e-2 of the bias gradient).  One more product a tile, and its fragments: at 256 columns one wave a SIMD has the registers for them.
template <class T, int KIND, int DK, int DVC, int MT, int W, bool ONE, bool LOW>
__global__ void __launch_bounds__(64 * W, LOW && DVC == 256 ? 1 : 2) dq_kernel(const Args p)
{
    using V8 = typename Ty<T>::V8;
    constexpr int KT = 32, NTH = 64 * W, BM = W * MT * 16, NS = 2, LT = MT * 16 + 1;
    static_assert(KT == 32 && MT <= 2, "the 32 + 31 diagonals of a wave's tile are two per lane of a half wave");
    using TK = Tile<T, KT, tile_width(DK), W>;
    using TV = Tile<T, KT, DVC, W>;
    constexpr int BUF = TK::BYTES + TV::BYTES;
    __shared__ __attribute__((aligned(1024))) char buf0[BUF], buf1[ONE ? 16 : BUF];     // (two objects: see fwd_kernel)
    extern __shared__ __attribute__((aligned(16))) float tab[];
    const int TW = p.table ? table_width(p.D) : 0, NB = p.table ? 2 * p.D + 1 : 0;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, l = lane & 15;
    float *dbw = tab + TW + w * NB, *tile = tab + TW + W * NB + w * KT * LT;         // this wave's distance sums and its dS tile
    int id = blockIdx.x;
    const int b = id % p.B; id /= p.B;
    const int hk = id % p.Hk; id /= p.Hk;
    const int ch = id % p.nchunk; id /= p.nchunk;
    const int G = p.H / p.Hk, h = hk * G + id % G, rt = row_tile(p, id / G);
    const int q0 = row_start(p, b), c0 = ch * DVC, cend = p.dv - c0;
    int ke = key_end(p, b);
    if (p.causal) ke = min(ke, min(p.Lq, rt * BM + BM) - 1 + q0 + 1);
    const T *Q = reinterpret_cast<const T *>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T *K = reinterpret_cast<const T *>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T *V = reinterpret_cast<const T *>(p.v) + b * p.vs[0] + hk * p.vs[2] + c0;
    TK tk;
    TV tv;
    tk.init(w, lane, p.ks[1], p.dk);
    tv.init(w, lane, p.vs[1], cend);
    const long long kstep = KT * p.ks[1], vstep = KT * p.vs[1];
    if (0 < ke) {
        tk.issue(K, ke, p.ks[1], buf0);
        tv.issue(V, ke, p.vs[1], buf0 + TK::BYTES);
    }
    if (p.table) {
        expand_bias<T, KIND>(p, h, tab, NTH);
        for (int t = lane; t < NB; t += 64) dbw[t] = 0.f;
    }
    const int i0 = rt * BM + w * MT * 16;                                             // the wave's first query
    V8 qf[MT][DK / 32], df[MT][DVC / 32], dl[LOW ? MT : 1][LOW ? DVC / 32 : 1];
    float top[MT], lsum[MT], del[MT], up[Ty<T>::scaled ? MT : 1];                               // (up: what dO is to be multiplied by)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int i = i0 + mt * 16 + l;
        const bool ok = i < p.Lq;
        const long long row = ((long long)b * p.Lq + (ok ? i : 0)) * p.H + h;
        const T *src = Q + (long long)(ok ? i : 0) * p.qs[1] + g * 8;
#pragma unroll
        for (int ks = 0; ks < DK / 32; ++ks) qf[mt][ks] = ld8(src + ks * 32, ok ? p.dk - ks * 32 - g * 8 : 0);
        const T *dsrc = reinterpret_cast<const T *>(p.dO) + row * p.dv + c0 + g * 8;
#pragma unroll
        for (int ks = 0; ks < DVC / 32; ++ks) df[mt][ks] = ld8(dsrc + ks * 32, ok ? cend - ks * 32 - g * 8 : 0);
        if constexpr (LOW) {
            const T *lsrc = reinterpret_cast<const T *>(p.dO_low) + row * p.dv + c0 + g * 8;
#pragma unroll
            for (int ks = 0; ks < DVC / 32; ++ks) dl[mt][ks] = ld8(lsrc + ks * 32, ok ? cend - ks * 32 - g * 8 : 0);
        }
        top[mt] = KIND == SOFTMAX && ok ? p.lse[2 * row] : 0.f;
        lsum[mt] = KIND == SOFTMAX ? (ok ? p.lse[2 * row + 1] : INFINITY) : 0.f;
        del[mt] = KIND == SOFTMAX && ok && ch == 0 ? p.delta_q[row] : 0.f;              // (dW comes in chunks of dv: the subtraction belongs to one of them)
        if constexpr (Ty<T>::scaled) {
            const float e = p.dO_exp && ok ? p.dO_exp[row] : 0.f;
            up[mt] = ldexpf(1.f, (int)e);
            lsum[mt] -= e;
        }
    }
    const int pmin = i0 + q0, pmax = min(p.Lq, i0 + MT * 16) - 1 + q0;
    f4 acc[DK / 16][MT];
#pragma unroll
    for (int n = 0; n < DK / 16; ++n)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[n][mt] = f4{0, 0, 0, 0};
    int ex[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) ex[mt] = E_NONE;
    float lo = 0.f, hi = 0.f, eta[MT], mlo[MT], mhi[MT];                              // (eta, and the weight beyond -D and +D, of the lane's query)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) eta[mt] = mlo[mt] = mhi[mt] = 0.f;
    const float sc = KIND == SOFTMAX ? p.scale * LOG2E : p.scale;
    if (p.table) __syncthreads();
    const float flo = p.table ? tab[0] : 0.f, fhi = p.table ? tab[TW - 1] : 0.f;          // the bias beyond +-D
    const auto place = [&](int j0) __attribute__((always_inline)) { return !p.table || j0 - pmax >= p.D ? 1 : (j0 + KT - 1 - pmin <= -p.D ? 2 : 3); };
    const auto whole = [&](int j0) __attribute__((always_inline)) { return j0 + KT <= ke && (!p.causal || j0 + KT - 1 <= pmin) && i0 + MT * 16 <= p.Lq; };
    // scale, bias and mask of a tile's scores
    const auto scores = [&](f4 (&s)[MT][NS], int j0, bool full, int where) __attribute__((always_inline)) {
        const float far = where == 1 ? fhi : flo;
        if (full && where != 3) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[mt][n][r] = __builtin_fmaf(s[mt][n][r], sc, far);
        } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int i = i0 + mt * 16 + l, last = i >= p.Lq ? -1 : (p.causal ? min(ke - 1, i + q0) : ke - 1);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    add_bias<1>(s[mt][n], sc, where == 3, tab + (p.D + MARGIN + j0 + n * 16 + g * 4 - i - q0), far);
                    if (!full)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j0 + n * 16 + g * 4 + r > last) s[mt][n][r] = -INFINITY;
                }
            }
        }
    };
    // sums of the wave's tile along its diagonals, into the distance sums
    const auto diagonals = [&](int j0) __attribute__((always_inline)) {
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                    // lane n of each half walks half of the queries down the diagonal that begins n keys ahead; past the last key it goes on at the first, on the
                    // diagonal 32 keys behind: all lanes read at every step, and the 63 diagonals are two sums a lane
                    const int n = lane & 31, h0 = lane >> 5;
                    float ahead = 0.f, behind = 0.f;
        #pragma unroll 8
                    for (int i = 0; i < MT * 8; ++i) {
                        const int c = h0 * MT * 8 + i, r = c + n;
                        const float x = tile[(r & 31) * LT + c];
                        ahead += r < KT ? x : 0.f;
                        behind += r < KT ? 0.f : x;
                    }
                    ahead = lanes_32<LaneAdd>(ahead);
                    behind = lanes_32<LaneAdd>(behind);
                    const int e = h0 ? n - KT : n, d = e + j0 - i0 - q0;                        // key - query within the tile, and between positions
                    const float sum = h0 ? behind : ahead;
                    hi += d >= p.D ? sum : 0.f;
                    lo += d < p.D && d <= -p.D ? sum : 0.f;
                    if (d < p.D && d > -p.D) dbw[d + p.D] += sum;
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
    };
    const auto step = [&](const char *cur, char *next, int j0) __attribute__((always_inline)) {
        tiles_ready();
        K += kstep;
        V += vstep;
        if (!ONE) {
            tk.issue(K, ke - j0 - KT, p.ks[1], next);
            tv.issue(V, ke - j0 - KT, p.vs[1], next + TK::BYTES);
        }
        if (i0 >= p.Lq || (p.causal && j0 > pmax)) return;
        const bool full = whole(j0);
        const int where = place(j0);
        f4 s[MT][NS], dp[MT][NS];
        constexpr bool TIGHT = LOW ? DK > 64 && DVC == 128 : DK + DVC > 256;            // (fragments in flight: what the registers leave)
        constexpr int KS = DK / 32, VS = DVC / 32, BK = TIGHT ? 2 : batch(NS * KS), B = TIGHT ? 2 : 4, BC = TIGHT ? 2 : batch(DK / 16);
        const int krow = TK::row_at(0, g, l), vrow = TV::row_at(TK::BYTES, g, l);
        const typename TK::Col kplace = TK::col_at(0, g, l);
        const auto key = [&](int i) __attribute__((always_inline)) { return TK::row8(cur, krow, i / KS, i % KS); };
        const auto val = [&](int i) __attribute__((always_inline)) { return TV::row8(cur, vrow, i / VS, i % VS); };
        const auto kcol = [&](int i) __attribute__((always_inline)) { return TK::col8(cur, kplace, 0, i); };
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NS; ++n) { s[mt][n] = f4{0, 0, 0, 0}; dp[mt][n] = f4{0, 0, 0, 0}; }
        V8 kf[BK], vf[B], cf[BC];
        fragments(kf, 0, key);
        stream<NS * KS, BK>(kf, key, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][i / KS] = Ty<T>::mma(a, qf[mt][i % KS], s[mt][i / KS]);
        });
        fragments(vf, 0, val);
        stream<NS * VS, B>(vf, val, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                dp[mt][i / VS] = Ty<T>::mma(a, df[mt][i % VS], dp[mt][i / VS]);
                if constexpr (LOW) dp[mt][i / VS] = Ty<T>::mma(a, dl[mt][i % VS], dp[mt][i / VS]);
            }
        });
        fragments(cf, 0, kcol);
        __builtin_amdgcn_sched_barrier(0);
        scores(s, j0, full, where);
        int right = where == 1 ? -1 : 0;                           // (opaque: of a choice between two sums the compiler makes an address, and memory of the registers)
        asm volatile("" : "+v"(right));
        const auto masked = [](float x, int m) __attribute__((always_inline)) { return __builtin_bit_cast(float, __builtin_bit_cast(int, x) & m); };
        const auto gradients = [&](auto near) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float all = 0.f, mass = 0.f;
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float wgt;
                        const float x = s[mt][n][r] = dscore<KIND, Ty<T>::scaled>(s[mt][n][r], dp[mt][n][r], top[mt], lsum[mt], del[mt], Ty<T>::scaled ? 2.f * up[mt] : 2.f, wgt);
                        all += x;
                        if constexpr (decltype(near)::value) {
                            tile[(n * 16 + g * 4 + r) * LT + mt * 16 + l] = x;
                        } else {
                            mass += wgt;
                        }
                    }
                if (KIND == SOFTMAX) eta[mt] += all;
                if constexpr (!decltype(near)::value) {
                    hi += masked(all, right);
                    lo += masked(all, ~right);
                    if (KIND == SOFTMAX) {
                        mhi[mt] += masked(mass, right);
                        mlo[mt] += masked(mass, ~right);
                    }
                }
            }
        };
        if (where == 3) gradients(std::true_type());
        else gradients(std::false_type());
        if (where == 3) diagonals(j0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float f = hold<T, NS>(s[mt], ex[mt]);
            if (Ty<T>::scaled && __any(f != 1.f))
#pragma unroll
                for (int n = 0; n < DK / 16; ++n) acc[n][mt] *= f;
        }
        V8 pb[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) pb[mt] = pack8<T>(s[mt][0], s[mt][1]);
        stream<DK / 16, BC>(cf, kcol, [&](int n, V8 a) __attribute__((always_inline)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[n][mt] = Ty<T>::mma(a, pb[mt], acc[n][mt]);
        });
    };
    if constexpr (ONE) {
        if (0 < ke) step(buf0, buf1, 0);
    } else {
        for (int j0 = 0; j0 < ke; j0 += 2 * KT) {
            step(buf0, buf1, j0);
            if (j0 + KT < ke) step(buf1, buf0, j0 + KT);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);                        // (vmcnt(0): nothing is on its way to LDS when the workgroup ends)
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int i = i0 + mt * 16 + l;
        if (i >= p.Lq) continue;
        const long long row = ((long long)b * p.Lq + i) * p.H + h;
        const float fin = p.scale * unhold<T>(ex[mt]);
#pragma unroll
        for (int n = 0; n < DK / 16; ++n) {
            const int c = n * 16 + g * 4;
            if (c >= p.dk) continue;
            const f4 x = acc[n][mt] * fin;
            if (p.nchunk > 1) {
                *reinterpret_cast<f4 *>(p.dq_part + ((long long)ch * p.B * p.Lq * p.H + row) * p.dk + c) = x;
            } else {
                typename Ty<T>::V4 y;
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = (T)x[r];
                *reinterpret_cast<typename Ty<T>::V4 *>(reinterpret_cast<T *>(p.dq) + row * p.dk + c) = y;
            }
        }
    }
    if (p.table) {
        if constexpr (KIND == SOFTMAX) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                eta[mt] = over_groups_sum(eta[mt]);
                if constexpr (Ty<T>::scaled) eta[mt] /= up[mt];    // (the weights carry it)
                // (a chunk of dv has its part of eta: the parts' corrections add up as the entries do)
                lo -= eta[mt] * mlo[mt];
                hi -= eta[mt] * mhi[mt];
            }
            const auto again = [&](const char *cur, char *next, int j0) __attribute__((always_inline)) {
                if (!ONE) {
                    tiles_ready();
                    K += kstep;
                    tk.issue(K, ke - j0 - KT, p.ks[1], next);
                }
                if (i0 >= p.Lq || (p.causal && j0 > pmax) || place(j0) != 3) return;
                f4 s[MT][NS];
                const int krow = TK::row_at(0, g, l);
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int ks = 0; ks < DK / 32; ++ks) {
                        const V8 a = TK::row8(cur, krow, n, ks);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][n] = Ty<T>::mma(a, qf[mt][ks], ks ? s[mt][n] : f4{0, 0, 0, 0});
                    }
                scores(s, j0, whole(j0), 3);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) tile[(n * 16 + g * 4 + r) * LT + mt * 16 + l] = -eta[mt] * pow2_(s[mt][n][r] - top[mt] - lsum[mt]);
                diagonals(j0);
            };
            if constexpr (ONE) {
                if (0 < ke) again(buf0, buf1, 0);                  // (its keys are still there)
            } else {
                // the tiles that hold a distance within +-D of any of the workgroup's queries
                const int first = max(0, rt * BM + q0 - p.D - KT + 2) / KT * KT, end = min(ke, min(p.Lq, rt * BM + BM) - 1 + q0 + p.D);
                __syncthreads();                                   // the first walk's tiles are no longer read
                if (first < end) {
                    K = reinterpret_cast<const T *>(p.k) + b * p.ks[0] + hk * p.ks[2] + first * p.ks[1];
                    tk.issue(K, ke - first, p.ks[1], buf0);
                }
                for (int j0 = first; j0 < end; j0 += 2 * KT) {
                    again(buf0, buf1, j0);
                    if (j0 + KT < end) again(buf1, buf0, j0 + KT);
                }
                __builtin_amdgcn_s_waitcnt(0x0f70);
            }
        }
        lo = lanes_all<LaneAdd, 64>(lo);
        hi = lanes_all<LaneAdd, 64>(hi);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const long long nr = (long long)p.B * p.nchunk * p.nrow * W, at = (((long long)b * p.nchunk + ch) * p.nrow + rt) * W + w;
        float *dst = p.db_part + ((long long)h * nr + at) * NB;
        for (int t = lane; t < NB; t += 64) dst[t] = t == 0 ? lo + (p.D == 0 ? hi : 0.f) : (t == NB - 1 ? hi : dbw[t]);
    }
}

// dK and dV: W waves, MT x 16 keys each; walks the queries of every head that shares the keys.  S has a key in the column: W and dS in registers
// are the B operands of dV^T = dO^T W and dK^T = Q^T dS.  Bound as dq, with four products and twice the accumulators: 251 and 111 us at its two sizes.
template <class T, int KIND, int DK, int DVC, int MT, int W, bool ONE>
__global__ void __launch_bounds__(64 * W, DK + DVC > 256 || (Ty<T>::scaled && DK + DVC == 256) ? 1 : 2) dkv_kernel(const Args p)
{
    using V8 = typename Ty<T>::V8;
    // float16 softmax: weights are at most 1, so one fixed power of two does for them: 2^14 higher none above 2^-28 is subnormal.  It comes with the row's sum, for
    // nothing; the score gradients carry it too.  Behind a gate a weight takes 2^e of its row's dO, and rows that differ in it meet in a key: an exponent for every
    // key, as the squares have (6 x 1021 tokens, 8 heads, 72 and 104 columns: 133 us, one power of two a workgroup 118, which lost keys that small rows alone see).
    constexpr bool SOFT16 = KIND == SOFTMAX && Ty<T>::scaled;
    constexpr float HIGH = 14.f;
    constexpr int QT = 32, NTH = 64 * W, BN = W * MT * 16, NS = 2;
    using TQ = Tile<T, QT, tile_width(DK), W>;
    using TO = Tile<T, QT, DVC, W>;
    constexpr int BUF = TQ::BYTES + TO::BYTES;
    __shared__ __attribute__((aligned(1024))) char buf0[BUF], buf1[ONE ? 16 : BUF];     // (two objects: see fwd_kernel)
    __shared__ __attribute__((aligned(16))) float stats0[3 * QT], stats1[3 * QT];       // the tiles' delta (float16 relu^2: 2 * 2^e), maximum, log2 of the sum
    extern __shared__ __attribute__((aligned(16))) float tab[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, l = lane & 15, G = p.H / p.Hk, TW = table_width(p.D);
    int id = blockIdx.x;
    const int b = id % p.B; id /= p.B;
    const int hk = id % p.Hk; id /= p.Hk;
    const int ch = id % p.nchunk; id /= p.nchunk;
    const int part = id % p.nparts, rt = id / p.nparts;
    const int q0 = row_start(p, b), ke = key_end(p, b), c0 = ch * DVC, cend = p.dv - c0;
    const int j0 = rt * BN + w * MT * 16;                                               // the wave's first key
    V8 kf[MT][DK / 32], vf[MT][DVC / 32];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int j = j0 + mt * 16 + l;
        const bool ok = j < ke;
        const T *kp = reinterpret_cast<const T *>(p.k) + b * p.ks[0] + (long long)(ok ? j : 0) * p.ks[1] + hk * p.ks[2] + g * 8;
        const T *vp = reinterpret_cast<const T *>(p.v) + b * p.vs[0] + (long long)(ok ? j : 0) * p.vs[1] + hk * p.vs[2] + c0 + g * 8;
#pragma unroll
        for (int ks = 0; ks < DK / 32; ++ks) kf[mt][ks] = ld8(kp + ks * 32, ok ? p.dk - ks * 32 - g * 8 : 0);
#pragma unroll
        for (int ks = 0; ks < DVC / 32; ++ks) vf[mt][ks] = ld8(vp + ks * 32, ok ? cend - ks * 32 - g * 8 : 0);
    }
    f4 av[DVC / 16][MT], ak[DK / 16][MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int n = 0; n < DVC / 16; ++n) av[n][mt] = f4{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < DK / 16; ++n) ak[n][mt] = f4{0, 0, 0, 0};
    }
    int ev[MT], ek[MT];
    const float high = SOFT16 && !p.dO_exp ? HIGH : 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) ev[mt] = ek[mt] = E_NONE;
    const float sc = KIND == SOFTMAX ? p.scale * LOG2E : p.scale;
    const int jmin = j0, jmax = min(ke, j0 + MT * 16) - 1;
    // queries from the first that sees a key of this block
    int ib = 0;
    if (p.causal) ib = max(0, (rt * BN - q0) / QT * QT);
    if (rt * BN >= ke) ib = p.Lq;                                                       // keys behind the length only: zeros
    TQ tq;
    TO to;
    tq.init(w, lane, p.qs[1], p.dk);
    to.init(w, lane, (long long)p.H * p.dv, cend);
    for (int hg = part * G / p.nparts; hg < (part + 1) * G / p.nparts; ++hg) {             // (a part of the heads that share the keys)
        const int h = hk * G + hg;
        const long long qstep = QT * p.qs[1], ostep = (long long)QT * p.H * p.dv;
        const T *Q = reinterpret_cast<const T *>(p.q) + b * p.qs[0] + h * p.qs[2] + ib * p.qs[1];              // (the tiles in turn: Q and dO move along)
        const T *dO = reinterpret_cast<const T *>(p.dO) + (((long long)b * p.Lq + ib) * p.H + h) * p.dv + c0;
        float tp0 = 0.f, ls0 = INFINITY, dl0 = 0.f, e0 = 0.f;
        const auto issue = [&](int i, char *buf) __attribute__((always_inline)) {
            if (buf) {
                tq.issue(Q, p.Lq - i, p.qs[1], buf);
                to.issue(dO, p.Lq - i, (long long)p.H * p.dv, buf + TQ::BYTES);
            }
            if ((KIND == SOFTMAX || Ty<T>::scaled) && tid < QT) {
                const long long row = ((long long)b * p.Lq + i + tid) * p.H + h;
                const bool ok = i + tid < p.Lq;
                if (Ty<T>::scaled) e0 = p.dO_exp && ok ? p.dO_exp[row] : 0.f;
                if (KIND == SOFTMAX) {
                    tp0 = ok ? p.lse[2 * row] : 0.f;
                    ls0 = ok ? p.lse[2 * row + 1] - e0 : INFINITY;
                    dl0 = ok && ch == 0 ? p.delta[row] : 0.f;
                }
            }
        };
        const auto keep = [&](float *st) __attribute__((always_inline)) {
            if (KIND == SOFTMAX && tid < QT) { st[tid] = dl0; st[QT + tid] = tp0; st[2 * QT + tid] = ls0 - high; }
            if (KIND == RELU2 && Ty<T>::scaled && tid < QT) st[tid] = ldexpf(2.f, (int)e0);
        };
        __syncthreads();                                                                  // the previous head's tiles and table are no longer read
        if (ib < p.Lq) {
            issue(ib, buf0);
            if (p.table) {
                expand_bias<T, KIND>(p, h, tab, NTH);
                __syncthreads();
            }
        }
        const float flo = p.table && ib < p.Lq ? tab[0] : 0.f, fhi = p.table && ib < p.Lq ? tab[TW - 1] : 0.f;          // the bias beyond +-D
        const auto step = [&](const char *cur, float *st, char *next, int i0) __attribute__((always_inline)) {
            keep(st);
            tiles_ready();
            if (!ONE) issue(i0 + QT, nullptr);                     // (the statistics of the next tile)
            Q += qstep;
            dO += ostep;
            if (!ONE) {
                tq.issue(Q, p.Lq - i0 - QT, p.qs[1], next);
                to.issue(dO, p.Lq - i0 - QT, (long long)p.H * p.dv, next + TQ::BYTES);
            }
            const int pmin = i0 + q0, pmax = min(p.Lq, i0 + QT) - 1 + q0;
            if (jmax < jmin || (p.causal && jmin > pmax)) return;
            const bool full = i0 + QT <= p.Lq && j0 + MT * 16 <= ke && (!p.causal || j0 + MT * 16 - 1 <= pmin);
            const int where = !p.table || jmin - pmax >= p.D ? 1 : (jmax - pmin <= -p.D ? 2 : 3);
            const float far = where == 1 ? fhi : flo;
            f4 s[MT][NS], wt[MT][NS];                              // (wt: dW first, then the weights)
            // (float16 with its exponents passes the registers of two waves at 192 columns and more: shorter batches spill less)
            constexpr bool TIGHT = Ty<T>::scaled && DK + DVC > 160 && DK + DVC < 256;
            constexpr int KS = DK / 32, VS = DVC / 32, BK = TIGHT ? 2 : batch(NS * KS), BQ = TIGHT ? 2 : batch(DK / 16), BO = TIGHT ? 2 : 4;
            const int qplace = TQ::row_at(0, g, l), oplace = TO::row_at(TQ::BYTES, g, l);
            const typename TQ::Col qcplace = TQ::col_at(0, g, l);
            const typename TO::Col ocplace = TO::col_at(TQ::BYTES, g, l);
            const auto qrow = [&](int i) __attribute__((always_inline)) { return TQ::row8(cur, qplace, i / KS, i % KS); };
            const auto orow = [&](int i) __attribute__((always_inline)) { return TO::row8(cur, oplace, i / VS, i % VS); };
            const auto ocol = [&](int i) __attribute__((always_inline)) { return TO::col8(cur, ocplace, 0, i); };
            const auto qcol = [&](int i) __attribute__((always_inline)) { return TQ::col8(cur, qcplace, 0, i); };
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NS; ++n) { s[mt][n] = f4{0, 0, 0, 0}; wt[mt][n] = f4{0, 0, 0, 0}; }
            V8 qb[BK], ob[BO];
            fragments(qb, 0, qrow);
            stream<NS * KS, BK>(qb, qrow, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][i / KS] = Ty<T>::mma(a, kf[mt][i % KS], s[mt][i / KS]);
            });
            fragments(ob, 0, orow);
            stream<NS * VS, BO>(ob, orow, [&](int i, V8 a) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) wt[mt][i / VS] = Ty<T>::mma(a, vf[mt][i % VS], wt[mt][i / VS]);
            });
            fragments(ob, 0, ocol);
            __builtin_amdgcn_sched_barrier(0);
            if (full && where != 3) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int n = 0; n < NS; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[mt][n][r] = __builtin_fmaf(s[mt][n][r], sc, far);
            } else {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int j = j0 + mt * 16 + l, first = j >= ke ? p.Lq : (p.causal ? j - q0 : 0);             // the first query that sees this lane's key
#pragma unroll
                    for (int n = 0; n < NS; ++n) {
                        add_bias<-1>(s[mt][n], sc, where == 3, tab + (p.D + MARGIN + j - (i0 + n * 16 + g * 4 + q0)), far);
                        if (!full)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (i0 + n * 16 + g * 4 + r < first || i0 + n * 16 + g * 4 + r >= p.Lq) s[mt][n][r] = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                f4 tp = {0, 0, 0, 0}, ls = {0, 0, 0, 0}, dl = {0, 0, 0, 0};
                if (KIND == SOFTMAX || Ty<T>::scaled) dl = *reinterpret_cast<const f4 *>(st + n * 16 + g * 4);
                if (KIND == SOFTMAX) {
                    tp = *reinterpret_cast<const f4 *>(st + QT + n * 16 + g * 4);
                    ls = *reinterpret_cast<const f4 *>(st + 2 * QT + n * 16 + g * 4);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float wgt;
                        s[mt][n][r] = dscore<KIND, Ty<T>::scaled>(s[mt][n][r], wt[mt][n][r], tp[r], ls[r], dl[r], dl[r], wgt);
                        wt[mt][n][r] = wgt;
                    }
            }
            V8 wb[MT], db[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float fv = high != 0.f ? 1.f : hold<T, NS>(wt[mt], ev[mt]), fk = hold<T, NS>(s[mt], ek[mt]);
                if (Ty<T>::scaled && __any(fv != 1.f))
#pragma unroll
                    for (int n = 0; n < DVC / 16; ++n) av[n][mt] *= fv;
                if (Ty<T>::scaled && __any(fk != 1.f))
#pragma unroll
                    for (int n = 0; n < DK / 16; ++n) ak[n][mt] *= fk;
                wb[mt] = pack8<T>(wt[mt][0], wt[mt][1]);
                db[mt] = pack8<T>(s[mt][0], s[mt][1]);
            }
            stream<DVC / 16, BO>(ob, ocol, [&](int n, V8 a) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) av[n][mt] = Ty<T>::mma(a, wb[mt], av[n][mt]);
            });
            V8 cb[BQ];
            fragments(cb, 0, qcol);
            stream<DK / 16, BQ>(cb, qcol, [&](int n, V8 a) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) ak[n][mt] = Ty<T>::mma(a, db[mt], ak[n][mt]);
            });
        };
        if constexpr (ONE) {
            if (ib < p.Lq) step(buf0, stats0, buf1, ib);
        } else {
            for (int i0 = ib; i0 < p.Lq; i0 += 2 * QT) {
                step(buf0, stats0, buf1, i0);
                if (i0 + QT < p.Lq) step(buf1, stats1, buf0, i0 + QT);
            }
            __builtin_amdgcn_s_waitcnt(0x0f70);
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int j = j0 + mt * 16 + l;
        if (j >= p.Lk) continue;
        const long long row = ((long long)b * p.Lk + j) * p.Hk + hk;
        const float down = ldexpf(1.f, -(int)high), finv = high != 0.f ? down : unhold<T>(ev[mt]) * (Ty<T>::scaled && KIND == RELU2 ? 0.5f : 1.f),
                    fink = p.scale * unhold<T>(ek[mt]) * down;
        typename Ty<T>::V4 y;
#pragma unroll
        for (int n = 0; n < DVC / 16; ++n) {
            const int c = n * 16 + g * 4;
            if (c >= cend) continue;
            if (p.nparts > 1) {
                *reinterpret_cast<f4 *>(p.dv_part + ((long long)part * p.B * p.Lk * p.Hk + row) * p.dv + c0 + c) = av[n][mt] * finv;
                continue;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = (T)(av[n][mt][r] * finv);
            *reinterpret_cast<typename Ty<T>::V4 *>(reinterpret_cast<T *>(p.dv_) + row * p.dv + c0 + c) = y;
        }
#pragma unroll
        for (int n = 0; n < DK / 16; ++n) {
            const int c = n * 16 + g * 4;
            if (c >= p.dk) continue;
            const f4 x = ak[n][mt] * fink;
            if (p.nchunk * p.nparts > 1) {
                *reinterpret_cast<f4 *>(p.dk_part + ((long long)(ch * p.nparts + part) * p.B * p.Lk * p.Hk + row) * p.dk + c) = x;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = (T)x[r];
                *reinterpret_cast<typename Ty<T>::V4 *>(reinterpret_cast<T *>(p.dk_) + row * p.dk + c) = y;
            }
        }
    }
}

// y = sum over the blocks' float32 partial sums, rounded once
template <class T> __global__ void __launch_bounds__(256) sum_parts_kernel(const float *part, T *y, long long n, int parts)
{
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f4 x = *reinterpret_cast<const f4 *>(part + i);
    for (int c = 1; c < parts; ++c) x += *reinterpret_cast<const f4 *>(part + c * n + i);
    typename Ty<T>::V4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (T)x[r];
    *reinterpret_cast<typename Ty<T>::V4 *>(y + i) = v;
}

// host side, one instantiation per element type and direction (tlk_gau_{f16,bf16,f32}{,_bwd}.hip)
struct BwdIo {
    const void *dout, *o;
    void *dq, *dk, *dv, *dgate, *dtable;
    void *ws;
};
template <class T> int forward(Args a, int kind, void *ws, hipStream_t st);
template <class T> int backward(Args a, const BwdIo &io, int kind, hipStream_t st);

}  // namespace gau
}  // namespace tlk
