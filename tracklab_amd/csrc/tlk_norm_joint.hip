// tlk_norm_joint.hip -- the joint of two blocks in one pass over its rows (tlk_norm_gate_residual_fwd / _bwd):
//     y = res_scale * x + gate * N1(h),   z = N2(y)
// with N one of: ScaleNorm v g / max(|v| / sqrt d, eps), RMS norm v w / sqrt(mean v^2 + eps), layer norm, or nothing.
//
// Bound by HBM: every tensor is read or written once.  LPR lanes hold one row in registers (16-byte loads; odd widths and row strides: one value
// at a time), statistics are reduced across those lanes in fp32, and y goes from the first norm to the second unrounded.  The backward pass keeps
// nothing of the forward pass: it forms N1(h), y and both statistics again from the rows it has to read anyway.  Column sums (gradients of weights,
// biases, res_scale and of a shared gate) stay in registers over all rows of a workgroup, are joined over its row slots through LDS, and a second
// launch adds the workgroups' sums in a fixed order: no atomics, equal bits on every run.
// Measured: 40800 rows of 256 f16, two tensors read and two written: 17.5 us (4.8 TB/s, a copy reaches 5.1); 16384 rows of 4096 bf16 forward 122 us
// (5.5 TB/s, part of it from the caches), backward 258 us (five tensors read and three written around four sums over each row: 4.2 TB/s).
#include <initializer_list>

#include "tlk_lanes.hpp"

using namespace tlk;

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

enum { NONE = TLK_NORM_NONE, SCALE = TLK_NORM_SCALE, RMS = TLK_NORM_RMS, LAYER = TLK_NORM_LAYER };
enum { A_RS, A_W1, A_W2, A_GATE, A_B1, A_B2, N_ACC };        // (the first three: every kind of norm)

struct NormArgs {
    const void *h, *x, *gate, *rs, *w1, *b1, *w2, *b2, *dy, *dz;
    void *y, *z, *dh, *dx, *dgate;
    long long hs, xs, gs;            // row strides
    long long rows, per_gate;        // rows that share a gate row (1: one each)
    int d, n1, n2;
    float eps1, eps2;
    float *part;                     // (workgroup, array, d)
    int groups, per_group;           // workgroups: `per_group` for each of `groups` runs of rows_in_group rows
    long long rows_in_group;
    int slot[N_ACC], scalar[N_ACC], nacc;           // which arrays are kept, and where; which are one sum over all columns
};

// E = NV * V values a lane; value e of lane t sits in column (e / V * LPR + t) * V + e % V
template <class T, int LPR, int NV, int V> struct Row {
    static constexpr int E = NV * V, W = V;
    static __device__ __forceinline__ int col(int e, int t) { return ((e / V) * LPR + t) * V + e % V; }
    // as it stands in memory (zero behind the row), and widened
    struct Raw {
        struct __attribute__((aligned(V == 1 ? sizeof(T) : 16))) { T el[V]; } v[NV];
    };
    static __device__ __forceinline__ void fetch(const void *base, long long off, int d, int t, Raw &r)
    {
        const T *p = reinterpret_cast<const T *>(base) + off;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * LPR + t) * V;
            if constexpr (V == 1) {
                r.v[v].el[0] = c < d ? p[c] : (T)0.f;
            } else {
                u4 raw = {0, 0, 0, 0};
                if (c < d) raw = *reinterpret_cast<const u4 *>(p + c);
                __builtin_memcpy(&r.v[v], &raw, 16);
            }
        }
    }
    static __device__ __forceinline__ void widen(const Raw &r, float (&x)[E])
    {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = (float)r.v[e / V].el[e % V];
    }
    static __device__ __forceinline__ void load(const void *base, long long off, int d, int t, float (&x)[E])
    {
        Raw r;
        fetch(base, off, d, t, r);
        widen(r, x);
    }
    static __device__ __forceinline__ void store(void *base, long long off, int d, int t, const float (&r)[E])
    {
        T *p = reinterpret_cast<T *>(base) + off;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * LPR + t) * V;
            if (c >= d) continue;
            if constexpr (V == 1) {
                p[c] = (T)r[v];
            } else {
                T el[V];
#pragma unroll
                for (int i = 0; i < V; ++i) el[i] = (T)r[v * V + i];
                u4 raw;
                __builtin_memcpy(&raw, el, 16);
                *reinterpret_cast<u4 *>(p + c) = raw;
            }
        }
    }
};

// sum over the LPR lanes of a row; LPR = 256: four waves through LDS (two buffers in turn, so one barrier is enough)
template <int LPR> struct Sum {
    float *s;                        // [2][rows of the workgroup * 4]
    int flip = 0;
    __device__ __forceinline__ float operator()(float v)
    {
        v = lanes_all<LaneAdd, (LPR < 64 ? LPR : 64)>(v);
        if constexpr (LPR > 64) {
            const int w = threadIdx.x >> 6, n = blockDim.x >> 6, first = w / (LPR / 64) * (LPR / 64);
            if ((threadIdx.x & 63) == 0) s[flip * n + w] = v;
            lds_barrier();
            v = 0.f;
#pragma unroll
            for (int i = 0; i < LPR / 64; ++i) v += s[flip * n + first + i];
            flip ^= 1;
        }
        return v;
    }
};

// v -> hat (the normalised row before weight and bias), returns 1 / its norm; `live`: what of it follows the row (0 below ScaleNorm's floor)
template <int E, class S> __device__ __forceinline__ float normalise(int kind, const float (&v)[E], float (&hat)[E], const bool (&in)[E], int d, float eps, S &sum, float &live)
{
    if (kind == NONE) {
#pragma unroll
        for (int e = 0; e < E; ++e) hat[e] = v[e];
        live = 1.f;
        return 1.f;
    }
    float mean = 0.f;
    if (kind == LAYER) {
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) t += v[e];
        mean = sum(t) / (float)d;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        hat[e] = in[e] ? v[e] - mean : 0.f;
        q = __builtin_fmaf(hat[e], hat[e], q);
    }
    q = sum(q) / (float)d;
    float inv;
    if (kind == SCALE) {
        const float n = sqrtf(q);
        inv = 1.f / (n < eps ? eps : n);
        live = n < eps ? 0.f : inv;
    } else {
        inv = live = 1.f / sqrtf(q + eps);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) hat[e] *= inv;
    return inv;
}

// gradient of the row through `hat`: t = gradient of the weighted row times the weight, in place
template <int E, class S> __device__ __forceinline__ void normalise_bwd(int kind, float (&t)[E], const float (&hat)[E], const bool (&in)[E], int d, float inv, float live, S &sum)
{
    if (kind == NONE) return;
    float a = 0.f, m = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        a = __builtin_fmaf(t[e], hat[e], a);
        m += t[e];
    }
    a = sum(a) / (float)d;
    m = kind == LAYER ? sum(m) / (float)d : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = in[e] ? (t[e] - m) * inv - hat[e] * live * a : 0.f;
}

// a weight as it stands in memory (ScaleNorm: its one value everywhere; none: ones), for use row after row
template <class R, class T> __device__ __forceinline__ void fetch_weight(int kind, const void *w, int d, int t, typename R::Raw &r)
{
    if (kind == RMS || kind == LAYER) {
        R::fetch(w, 0, d, t, r);
        return;
    }
    const T g = kind == SCALE ? *reinterpret_cast<const T *>(w) : (T)1.f;
#pragma unroll
    for (int e = 0; e < R::E; ++e) r.v[e / R::W].el[e % R::W] = g;
}
template <class R, class T> __device__ __forceinline__ void load_weight(int kind, const void *w, int d, int t, float (&r)[R::E])
{
    if (kind == NONE || !w) {
#pragma unroll
        for (int e = 0; e < R::E; ++e) r[e] = 1.f;
    } else if (kind == SCALE) {
        const float g = (float)*reinterpret_cast<const T *>(w);
#pragma unroll
        for (int e = 0; e < R::E; ++e) r[e] = g;
    } else {
        R::load(w, 0, d, t, r);
    }
}

template <class T, int LPR, int NV, int V> __global__ void __launch_bounds__(256) joint_fwd_kernel(const NormArgs p)
{
    using R = Row<T, LPR, NV, V>;
    constexpr int E = R::E;
    __shared__ float s[2 * 4];
    const long long row0 = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int t = threadIdx.x % LPR;
    const bool live_row = row0 < p.rows;
    const long long row = live_row ? row0 : p.rows - 1;                  // (lanes without a row take part in the reductions)
    Sum<LPR> sum{s};
    bool in[E];
#pragma unroll
    for (int e = 0; e < E; ++e) in[e] = R::col(e, t) < p.d;
    float v[E], y[E], u[E];
    R::load(p.h, row * p.hs, p.d, t, v);
    if (p.x) R::load(p.x, row * p.xs, p.d, t, u);
    float unused;
    (void)normalise<E>(p.n1, v, y, in, p.d, p.eps1, sum, unused);
    if (p.n1 != NONE) {
        float w[E];
        load_weight<R, T>(p.n1, p.w1, p.d, t, w);
        if (p.b1) {
            float b[E];
            R::load(p.b1, 0, p.d, t, b);
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = __builtin_fmaf(y[e], w[e], b[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] *= w[e];
        }
    }
    if (p.gate) {
        float gt[E];
        R::load(p.gate, row / p.per_gate * p.gs, p.d, t, gt);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] *= gt[e];
    }
    if (p.x) {
        if (p.rs) {
            float r[E];
            R::load(p.rs, 0, p.d, t, r);
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = __builtin_fmaf(u[e], r[e], y[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += u[e];
        }
    }
    if (live_row) R::store(p.y, row * p.d, p.d, t, y);
    if (!p.z) return;                                                    // (uniform over the launch)
    (void)normalise<E>(p.n2, y, v, in, p.d, p.eps2, sum, unused);
    float w[E];
    load_weight<R, T>(p.n2, p.w2, p.d, t, w);
    if (p.b2) {
        float b[E];
        R::load(p.b2, 0, p.d, t, b);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = __builtin_fmaf(v[e], w[e], b[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= w[e];
    }
    if (live_row) R::store(p.z, row * p.d, p.d, t, v);
}

// One backward workgroup of 512 threads per CU walks rows in turn, 512 / LPR of them at a time.  The next rows' five tensors are fetched while the present
// ones pass their four reductions: a lane holds 8 values of a row, so that its sums and two rows' data fit the registers.  Rows of more than 4096 columns put 16 in a lane, and
// what does not fit goes to memory: 8192 x 8192 bf16 500 us lean and 1218 with all six arrays (192 and 384 bytes of scratch a lane), float32 1323 and 1661 (452 and 644).
constexpr int BT = 512;

// LEAN: no layer norm and no shared gate, so only res_scale and the two weights have column sums -- half the registers of a lane's sums, which is what
// lets the rows' loads stay in flight (16384 rows of 4096 bf16: 240 us, with all six arrays 320)
template <class T, int LPR, int NV, int V, bool LEAN> __global__ void __attribute__((amdgpu_flat_work_group_size(BT, BT), amdgpu_waves_per_eu(2, 2))) joint_bwd_kernel(const NormArgs p)
{
    using R = Row<T, LPR, NV, V>;
    constexpr int E = R::E, SLOTS = BT / LPR;
    extern __shared__ float lds[];
    __shared__ float s[2 * (BT / 64)];
    const int t = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const long long grp = blockIdx.x / p.per_group, first = grp * p.rows_in_group, in_grp = blockIdx.x % p.per_group;
    Sum<LPR> sum{s};
    bool in[E];
#pragma unroll
    for (int e = 0; e < E; ++e) in[e] = R::col(e, t) < p.d;
    constexpr int NA = LEAN ? 3 : N_ACC;
    float acc[NA][E];
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[a][e] = 0.f;
    const long long step = (long long)p.per_group * SLOTS;
    typename R::Raw fh, fx, fg, fy, fz;
    const auto fetch = [&](long long r0) __attribute__((always_inline)) {
        const long long row = first + (r0 + slot < p.rows_in_group ? r0 + slot : r0);
        R::fetch(p.h, row * p.hs, p.d, t, fh);
        if (p.x) R::fetch(p.x, row * p.xs, p.d, t, fx);
        if (p.gate) R::fetch(p.gate, row / p.per_gate * p.gs, p.d, t, fg);
        if (p.dy) R::fetch(p.dy, row * p.d, p.d, t, fy);
        if (p.dz) R::fetch(p.dz, row * p.d, p.d, t, fz);
    };
    // weights first: loads return in order, and one behind the next rows' would wait for them
    typename R::Raw rw1, rw2, rb1, rrs;
    fetch_weight<R, T>(p.n1, p.w1, p.d, t, rw1);
    fetch_weight<R, T>(p.n2, p.w2, p.d, t, rw2);
    fetch_weight<R, T>(p.x && p.rs ? RMS : NONE, p.rs, p.d, t, rrs);
    if (p.b1) R::fetch(p.b1, 0, p.d, t, rb1);
    if (in_grp * SLOTS < p.rows_in_group) fetch(in_grp * SLOTS);
    for (long long r0 = in_grp * SLOTS; r0 < p.rows_in_group; r0 += step) {            // (uniform over the workgroup: the reductions hold barriers)
        const bool live = r0 + slot < p.rows_in_group;
        const long long row = first + (live ? r0 + slot : r0);
        float h[E], x[E], gt[E], dy[E], dz[E], w[E];
        R::widen(fh, h);
        if (p.x) R::widen(fx, x);
        if (p.gate) R::widen(fg, gt);
        if (p.dy) R::widen(fy, dy);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) dy[e] = 0.f;
        if (p.dz) R::widen(fz, dz);
        if (r0 + step < p.rows_in_group) fetch(r0 + step);
        float hat1[E], n1[E], live1, live2, inv2 = 1.f;
        const float inv1 = normalise<E>(p.n1, h, hat1, in, p.d, p.eps1, sum, live1);
        R::widen(rw1, w);
#pragma unroll
        for (int e = 0; e < E; ++e) n1[e] = hat1[e] * w[e];
        if (p.b1) {
            float b[E];
            R::widen(rb1, b);
#pragma unroll
            for (int e = 0; e < E; ++e) n1[e] += b[e];
        }
        float rs[E];
        R::widen(rrs, rs);
        if (p.dz) {
            float hat2[E], y[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[e] = p.gate ? n1[e] * gt[e] : n1[e];
                if (p.x) y[e] = __builtin_fmaf(x[e], rs[e], y[e]);
            }
            inv2 = normalise<E>(p.n2, y, hat2, in, p.d, p.eps2, sum, live2);
            if (live) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    acc[A_W2][e] = __builtin_fmaf(dz[e], hat2[e], acc[A_W2][e]);
                    if constexpr (!LEAN) acc[A_B2][e] += dz[e];
                }
            }
            float w2[E];
            R::widen(rw2, w2);
#pragma unroll
            for (int e = 0; e < E; ++e) dz[e] *= w2[e];
            normalise_bwd<E>(p.n2, dz, hat2, in, p.d, inv2, live2, sum);
#pragma unroll
            for (int e = 0; e < E; ++e) dy[e] += dz[e];
        }
        if (p.x) {
            if (live) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[A_RS][e] = __builtin_fmaf(dy[e], x[e], acc[A_RS][e]);
            }
            if (p.dx) {
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = dy[e] * rs[e];
                if (live) R::store(p.dx, row * p.d, p.d, t, x);
            }
        }
        if (p.gate) {
            float dg[E];
#pragma unroll
            for (int e = 0; e < E; ++e) dg[e] = dy[e] * n1[e];
            if (p.per_gate == 1) {
                if (live && p.dgate) R::store(p.dgate, row * p.d, p.d, t, dg);
            } else if (live) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if constexpr (!LEAN) acc[A_GATE][e] += dg[e];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) dy[e] *= gt[e];
        }
        if (live) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                acc[A_W1][e] = __builtin_fmaf(dy[e], hat1[e], acc[A_W1][e]);
                if constexpr (!LEAN) acc[A_B1][e] += dy[e];
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) dy[e] *= w[e];
        normalise_bwd<E>(p.n1, dy, hat1, in, p.d, inv1, live1, sum);
        if (live && p.dh) R::store(p.dh, row * p.d, p.d, t, dy);
    }
    // the workgroup's column sums: its row slots joined in LDS, one array after the other
    const int CW = LPR * E;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
        if (p.slot[a] < 0) continue;
        float *dst = p.part + ((long long)blockIdx.x * p.nacc + p.slot[a]) * p.d;
        __syncthreads();
        if (p.scalar[a]) {                                               // ScaleNorm's one weight: over the columns as well
            float v = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) v += acc[a][e];
            v = lanes_all<LaneAdd, 64>(v);
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
            __syncthreads();
            if (threadIdx.x == 0) {
                v = 0.f;
                for (int i = 0; i < BT / 64; ++i) v += lds[i];
                dst[0] = v;
            }
            continue;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) lds[slot * CW + R::col(e, t)] = acc[a][e];
        __syncthreads();
        for (int c = threadIdx.x; c < p.d; c += BT) {
            float v = 0.f;
            for (int i = 0; i < SLOTS; ++i) v += lds[i * CW + c];
            dst[c] = v;
        }
    }
}

struct ColArgs {
    const float *part;               // (workgroups, nacc, d)
    void *out[N_ACC];
    int slot[N_ACC], scalar[N_ACC], d, nacc, groups, per_group;
};
// adds the workgroups' column sums in a fixed order: 64 columns x 16 runs of workgroups a block
constexpr int CR = 16;
template <class T> __global__ void __launch_bounds__(64 * CR) joint_cols_kernel(const ColArgs p)
{
    __shared__ float s[CR][64];
    const int a = blockIdx.y, cg = threadIdx.x & 63, rg = threadIdx.x >> 6;
    if (p.slot[a] < 0 || (p.scalar[a] && blockIdx.x > 0)) return;
    const bool per_gate = a == A_GATE;
    const int ng = per_gate ? p.groups : 1, nb = per_gate ? p.per_group : p.groups * p.per_group;
    if ((int)blockIdx.z >= ng) return;
    const int first = blockIdx.z * nb, share = (nb + CR - 1) / CR, b0 = rg * share, b1 = min(nb, b0 + share), c = blockIdx.x * 64 + cg, cols = p.scalar[a] ? 1 : p.d;
    float v = 0.f;
    if (c < cols) {
        const float *src = p.part + ((long long)first * p.nacc + p.slot[a]) * p.d + c;
        const long long bs = (long long)p.nacc * p.d;
#pragma unroll 8
        for (int b = b0; b < b1; ++b) v += src[b * bs];
    }
    s[rg][cg] = v;
    __syncthreads();
    if (rg || c >= cols) return;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < CR; ++i) v += s[i][cg];
    reinterpret_cast<T *>(p.out[a])[(long long)blockIdx.z * p.d + c] = (T)v;
}

template <class T, int LPR, int NV, int V> int fwd_launch(const NormArgs &a, hipStream_t st)
{
    const long long blocks = (a.rows + 256 / LPR - 1) / (256 / LPR);
    if (blocks > 0x7fffffffLL) return fail(TLK_EINVAL, "tlk_norm_gate_residual: more than 2^31 - 1 workgroups");
    hipLaunchKernelGGL((joint_fwd_kernel<T, LPR, NV, V>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    TLK_HIP(hipGetLastError());
    return TLK_OK;
}
template <class T, int LPR, int NV, int V> int bwd_launch(const NormArgs &a, hipStream_t st)
{
    static_assert(BT * NV * V * sizeof(float) <= 48 * 1024, "dynamic LDS that needs no attribute");
    const size_t smem = (size_t)BT * NV * V * sizeof(float);
    const bool lean = a.slot[A_GATE] < 0 && a.slot[A_B1] < 0 && a.slot[A_B2] < 0;
    const auto kernel = lean ? joint_bwd_kernel<T, LPR, NV, V, true> : joint_bwd_kernel<T, LPR, NV, V, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.groups * a.per_group)), dim3(BT), smem, st, a);
    TLK_HIP(hipGetLastError());
    return TLK_OK;
}

// lanes a row: forward at most 16 values a lane (beyond 4096 columns: 32), backward 8 (16)
template <class T> int pick_fwd(const NormArgs &a, bool vec, hipStream_t st)
{
    constexpr int V = 16 / sizeof(T);
    if (vec) {
        const int v = (a.d + V - 1) / V;                                   // 16-byte vectors of a row
        if (v <= 32) return fwd_launch<T, 32, 1, V>(a, st);
        if (v <= 64) return fwd_launch<T, 64, 1, V>(a, st);
        if (v <= 128) return fwd_launch<T, 64, 2, V>(a, st);
        if (v <= 256) return fwd_launch<T, 256, 1, V>(a, st);
        if (v <= 512) return fwd_launch<T, 256, 2, V>(a, st);
        if (v <= 1024) return fwd_launch<T, 256, 4, V>(a, st);
        if constexpr (V == 4) return fwd_launch<T, 256, 8, V>(a, st);
        return fail(TLK_EINVAL, "tlk_norm_gate_residual: more than 8192 columns");
    }
    if (a.d <= 256) return fwd_launch<T, 64, 4, 1>(a, st);
    if (a.d <= 1024) return fwd_launch<T, 64, 16, 1>(a, st);
    if (a.d <= 4096) return fwd_launch<T, 256, 16, 1>(a, st);
    return fwd_launch<T, 256, 32, 1>(a, st);
}
template <class T> int pick_bwd(const NormArgs &a, bool vec, hipStream_t st)
{
    constexpr int V = 16 / sizeof(T);
    if (vec) {
        const int v = (a.d + V - 1) / V;
        if (v <= 32) return bwd_launch<T, 32, 1, V>(a, st);
        if (v <= 64) return bwd_launch<T, 64, 1, V>(a, st);
        if (v <= 128) return bwd_launch<T, 128, 1, V>(a, st);
        if (v <= 256) return bwd_launch<T, 256, 1, V>(a, st);
        if (v <= 512) return bwd_launch<T, 512, 1, V>(a, st);
        if (v <= 1024) return bwd_launch<T, 512, 2, V>(a, st);
        if constexpr (V == 4) return bwd_launch<T, 512, 4, V>(a, st);
        return fail(TLK_EINVAL, "tlk_norm_gate_residual: more than 8192 columns");
    }
    if (a.d <= 256) return bwd_launch<T, 64, 4, 1>(a, st);
    if (a.d <= 1024) return bwd_launch<T, 128, 8, 1>(a, st);
    if (a.d <= 4096) return bwd_launch<T, 512, 8, 1>(a, st);
    return bwd_launch<T, 512, 16, 1>(a, st);
}

// 256 workgroups walk the rows (one per CU); a shared gate's gradient is kept per run of rows, so every run gets workgroups of its own
void cut(const tlk_norm_args *a, NormArgs &n)
{
    const long long groups = a->gate && a->gate_rows > 1 ? (a->rows + a->gate_rows - 1) / a->gate_rows : 1;
    n.groups = (int)(groups < 1 ? 1 : groups);
    n.rows_in_group = a->rows / n.groups;
    const int slots = a->dim <= 512 ? 8 : (a->dim <= 2048 ? 2 : 1);
    long long per = n.groups < 256 ? 256 / n.groups : 1, most = (n.rows_in_group + slots - 1) / slots;
    n.per_group = (int)(per < most ? per : (most < 1 ? 1 : most));
}
int arrays(const tlk_norm_args *a, int (&slot)[N_ACC])
{
    int n = 0;
    slot[A_RS] = a->res_scale ? n++ : -1;
    slot[A_GATE] = a->gate && a->gate_rows > 1 ? n++ : -1;
    slot[A_W1] = a->norm != TLK_NORM_NONE ? n++ : -1;
    slot[A_B1] = a->norm == TLK_NORM_LAYER && a->bias ? n++ : -1;
    slot[A_W2] = a->next_norm != TLK_NORM_NONE ? n++ : -1;
    slot[A_B2] = a->next_norm == TLK_NORM_LAYER && a->next_bias ? n++ : -1;
    return n;
}

int check(const tlk_norm_args *a, const char *fn)
{
    const std::string f(fn);
    if (!a) return fail(TLK_EINVAL, f + ": null arguments");
    if (a->dtype != TLK_F32 && a->dtype != TLK_F16 && a->dtype != TLK_BF16) return fail(TLK_EINVAL, f + ": dtype must be TLK_F32, TLK_F16 or TLK_BF16");
    if (a->norm < 0 || a->norm > TLK_NORM_LAYER || a->next_norm < 0 || a->next_norm > TLK_NORM_LAYER) return fail(TLK_EINVAL, f + ": unknown norm");
    if (a->rows < 0 || a->dim < 1 || a->dim > 8192) return fail(TLK_EINVAL, f + ": rows must be >= 0 and 1 <= dim <= 8192");
    if (!(a->eps >= 0.f) || !(a->next_eps >= 0.f)) return fail(TLK_EINVAL, f + ": eps must not be negative");
    if (a->rows > 0 && !a->h) return fail(TLK_EINVAL, f + ": null input");
    if ((a->norm != TLK_NORM_NONE && !a->weight) || (a->next_norm != TLK_NORM_NONE && !a->next_weight)) return fail(TLK_EINVAL, f + ": a norm needs its weight");
    if ((a->norm != TLK_NORM_LAYER && a->bias) || (a->next_norm != TLK_NORM_LAYER && a->next_bias)) return fail(TLK_EINVAL, f + ": only the layer norm takes a bias");
    if (a->res_scale && !a->x) return fail(TLK_EINVAL, f + ": res_scale without a residual");
    if (a->h_stride < a->dim || (a->x && a->x_stride < a->dim) || (a->gate && a->gate_stride < a->dim)) return fail(TLK_EINVAL, f + ": row strides must be >= dim");
    if (a->gate && (a->gate_rows < 1 || (a->rows > 0 && a->rows % a->gate_rows != 0))) return fail(TLK_EINVAL, f + ": rows must be a multiple of gate_rows");
    if (a->gate && a->gate_rows > 1 && a->rows / a->gate_rows > 65535) return fail(TLK_EINVAL, f + ": more than 65535 shared gate rows");
    return TLK_OK;
}

bool vector_rows(const tlk_norm_args *a, std::initializer_list<const void *> more)
{
    const int size = a->dtype == TLK_F32 ? 4 : 2, v = 16 / size;
    uintptr_t bits = (uintptr_t)a->h | (uintptr_t)a->x | (uintptr_t)a->gate | (uintptr_t)a->res_scale | (uintptr_t)a->bias | (uintptr_t)a->next_bias;
    if (a->norm == TLK_NORM_RMS || a->norm == TLK_NORM_LAYER) bits |= (uintptr_t)a->weight;
    if (a->next_norm == TLK_NORM_RMS || a->next_norm == TLK_NORM_LAYER) bits |= (uintptr_t)a->next_weight;
    for (const void *p : more) bits |= (uintptr_t)p;
    return (bits & 15) == 0 && a->dim % v == 0 && a->h_stride % v == 0 && (!a->x || a->x_stride % v == 0) && (!a->gate || a->gate_stride % v == 0);
}

NormArgs common(const tlk_norm_args *a)
{
    NormArgs n;
    memset(&n, 0, sizeof(n));
    n.h = a->h; n.x = a->x; n.gate = a->gate; n.rs = a->res_scale;
    n.w1 = a->weight; n.b1 = a->bias; n.w2 = a->next_weight; n.b2 = a->next_bias;
    n.hs = a->h_stride; n.xs = a->x_stride; n.gs = a->gate_stride;
    n.rows = a->rows; n.per_gate = a->gate ? a->gate_rows : 1;
    n.d = a->dim; n.n1 = a->norm; n.n2 = a->next_norm; n.eps1 = a->eps; n.eps2 = a->next_eps;
    return n;
}

}  // namespace

extern "C" int tlk_norm_gate_residual_fwd(const tlk_norm_args *a, void *y_dev, void *z_dev, void *hip_stream)
{
    const int rc = check(a, "tlk_norm_gate_residual_fwd");
    if (rc != TLK_OK) return rc;
    if (a->rows == 0) return TLK_OK;
    if ((a->next_norm != TLK_NORM_NONE) != (z_dev != nullptr)) return fail(TLK_EINVAL, "tlk_norm_gate_residual_fwd: z goes with the next norm");
    if (!y_dev) return fail(TLK_EINVAL, "tlk_norm_gate_residual_fwd: null output");
    NormArgs n = common(a);
    n.y = y_dev; n.z = z_dev;
    const bool vec = vector_rows(a, {y_dev, z_dev});
    hipStream_t st = (hipStream_t)hip_stream;
    if (a->dtype == TLK_F32) return pick_fwd<float>(n, vec, st);
    return a->dtype == TLK_F16 ? pick_fwd<_Float16>(n, vec, st) : pick_fwd<__bf16>(n, vec, st);
}

extern "C" long long tlk_norm_gate_residual_workspace(const tlk_norm_args *a)
{
    const int rc = check(a, "tlk_norm_gate_residual_workspace");
    if (rc != TLK_OK) return rc;
    if (a->rows == 0) return 0;
    NormArgs n = common(a);
    cut(a, n);
    int slot[N_ACC];
    return (long long)n.groups * n.per_group * arrays(a, slot) * a->dim * (long long)sizeof(float);
}

extern "C" int tlk_norm_gate_residual_bwd(const tlk_norm_args *a, const void *dy_dev, const void *dz_dev, const tlk_norm_grads *g, void *workspace_dev,
                                          long long workspace_bytes, void *hip_stream)
{
    const int rc = check(a, "tlk_norm_gate_residual_bwd");
    if (rc != TLK_OK) return rc;
    if (!g) return fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: null gradients");
    if (dz_dev && a->next_norm == TLK_NORM_NONE) return fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: a gradient of z without the next norm");
    int slot[N_ACC];
    const int nacc = arrays(a, slot);
    void *out[N_ACC];
    out[A_RS] = g->dres_scale; out[A_GATE] = g->dgate; out[A_W1] = g->dweight; out[A_B1] = g->dbias; out[A_W2] = g->dnext_weight; out[A_B2] = g->dnext_bias;
    for (int i = 0; i < N_ACC; ++i)
        if (slot[i] >= 0 && !out[i]) return fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: a parameter's gradient has no place");
    if (a->rows > 0 && (!g->dh || (a->x && !g->dx) || (a->gate && !g->dgate))) return fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: a gradient has no place");
    if (a->rows == 0) return nacc ? fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: no rows") : TLK_OK;
    NormArgs n = common(a);
    cut(a, n);
    if (nacc && (!workspace_dev || workspace_bytes < (long long)n.groups * n.per_group * nacc * a->dim * (long long)sizeof(float)))
        return fail(TLK_EINVAL, "tlk_norm_gate_residual_bwd: workspace too small (tlk_norm_gate_residual_workspace)");
    n.dy = dy_dev; n.dz = dz_dev; n.dh = g->dh; n.dx = g->dx; n.dgate = a->gate && a->gate_rows == 1 ? g->dgate : nullptr;
    n.part = reinterpret_cast<float *>(workspace_dev);
    n.nacc = nacc;
    memcpy(n.slot, slot, sizeof(slot));
    n.scalar[A_W1] = a->norm == TLK_NORM_SCALE;
    n.scalar[A_W2] = a->next_norm == TLK_NORM_SCALE;
    const bool vec = vector_rows(a, {dy_dev, dz_dev, g->dh, g->dx, n.dgate});
    hipStream_t st = (hipStream_t)hip_stream;
    const int rb = a->dtype == TLK_F32 ? pick_bwd<float>(n, vec, st) : (a->dtype == TLK_F16 ? pick_bwd<_Float16>(n, vec, st) : pick_bwd<__bf16>(n, vec, st));
    if (rb != TLK_OK || !nacc) return rb;
    ColArgs c;
    c.part = n.part; c.d = n.d; c.nacc = nacc; c.groups = n.groups; c.per_group = n.per_group;
    for (int i = 0; i < N_ACC; ++i) { c.out[i] = out[i]; c.slot[i] = slot[i]; c.scalar[i] = n.scalar[i]; }
    const dim3 grid((unsigned)((n.d + 63) / 64), N_ACC, (unsigned)(slot[A_GATE] >= 0 ? n.groups : 1));
    if (a->dtype == TLK_F32) hipLaunchKernelGGL(joint_cols_kernel<float>, grid, dim3(64 * CR), 0, st, c);
    else if (a->dtype == TLK_F16) hipLaunchKernelGGL(joint_cols_kernel<_Float16>, grid, dim3(64 * CR), 0, st, c);
    else hipLaunchKernelGGL(joint_cols_kernel<__bf16>, grid, dim3(64 * CR), 0, st, c);
    TLK_HIP(hipGetLastError());
    return TLK_OK;
}
