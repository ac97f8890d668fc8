// tlk_gau_host.hpp -- launches of the gated attention unit's kernels for one element type (included by tlk_gau_{f16,bf16,f32}{,_bwd}.hip).
#pragma once
#include <type_traits>

#include "tlk_gau.hpp"

namespace tlk {
namespace gau {

inline long long align_up(long long x) { return (x + 255) & ~255LL; }
inline int div_up(int a, int b) { return (a + b - 1) / b; }

// how the forward call of these sizes is cut; shared by the launch and the workspace query
struct FwdPlan {
    bool few;                // one tile of rows, waves side by side along dv; else waves below each other
    int fold, mt, dvb, bm, nrow, nchunk, nsplit, split_keys, heads;
};
inline FwdPlan plan_forward(const Args &a, int elem)
{
    FwdPlan f;
    const int G = a.H / a.Hk;
    f.fold = G > 1 && a.Lq <= 32 && (long long)G * table_width(a.D) <= 8192;
    const long long rows = (long long)a.Lq * (f.fold ? G : 1);
    f.few = rows <= 32;
    f.mt = f.few && rows <= 16 ? 1 : 2;
    f.bm = f.few ? f.mt * 16 : 128;
    f.dvb = a.dv <= 64 ? 64 : (a.dv <= 128 ? 128 : (a.dv <= 256 || !f.few || elem == 4 ? 256 : 512));
    f.nrow = (int)((rows + f.bm - 1) / f.bm);
    f.nchunk = div_up(a.dv, f.dvb);
    f.heads = f.fold ? a.Hk : a.H;
    const long long blocks = (long long)a.B * f.heads * f.nchunk * f.nrow;
    f.nsplit = 1;
    f.split_keys = a.Lk;
    // Few workgroups over many keys: the keys are split.  One tile of rows is read at the rate of HBM, which takes many workgroups: 2048, of 256 keys at least.
    // More rows are matrix products: two workgroups a CU, of 512 keys at least, and no split from half a workgroup a CU on or where the sums of the splits
    // move more than they save (bf16, dv 128, one head: 128 rows x 4096 keys 97 -> 21 us, 4 x 1024 x 4096 98 -> 32; 16 x 1024 rows x 1024 keys would go
    // 32 -> 37, x 4096 keys 100 -> 61; 192 workgroups 55 -> 70).
    const int full = f.few ? 2048 : 512, least = f.few ? 256 : 512;
    if (a.Lk > 512 && blocks > 0 && (f.few ? blocks < 2048 : blocks <= 128 && a.Lk >= 16 * blocks)) {
        const int want = (int)(f.few ? (full + blocks - 1) / blocks : full / blocks), most = div_up(a.Lk, least);
        f.nsplit = want < most ? want : most;
        f.split_keys = div_up(div_up(a.Lk, f.nsplit), 64) * 64;
        f.nsplit = div_up(a.Lk, f.split_keys);
    }
    return f;
}

struct BwdPlan {
    int dvc, nchunk, w_q, w_k, rows_q, rows_k, nrow_q, nrow_k, nparts;
    long long nr;            // distance-sum rows per head
};
inline BwdPlan plan_backward(const Args &a, int elem)
{
    BwdPlan f;
    f.dvc = a.dv <= 64 ? 64 : (a.dv <= 128 ? 128 : 256);
    f.nchunk = div_up(a.dv, f.dvc);
    const int per = elem == 4 ? 16 : 32;                            // rows (keys) of a wave: float32 operands take twice the registers
    f.w_q = a.Lq <= 2 * per ? (a.Lq <= per ? 1 : 2) : 4;
    f.w_k = a.Lk <= 2 * per ? (a.Lk <= per ? 1 : 2) : 4;
    // (a wide table leaves less LDS for the waves' own sums)
    const auto lds = [&](int w) { return 2LL * elem * 32 * ((a.dk <= 64 ? 64 : 128) + f.dvc) + 4LL * (table_width(a.D) + w * (2 * a.D + 1 + 32 * (per + 1))); };
    while (a.table && f.w_q > 1 && lds(f.w_q) + 1024 > 160 * 1024) f.w_q /= 2;
    f.rows_q = per * f.w_q;
    f.rows_k = per * f.w_k;
    f.nrow_q = div_up(a.Lq, f.rows_q);
    f.nrow_k = div_up(a.Lk, f.rows_k);
    // heads that share keys are walked by one block in turn; in parts where that leaves CUs without work
    const long long blocks = (long long)a.B * a.Hk * f.nchunk * f.nrow_k;
    const int G = a.H / a.Hk;
    f.nparts = blocks >= 1024 || blocks == 0 ? 1 : (int)(1024 / blocks < G ? 1024 / blocks : G);
    f.nr = (long long)a.B * f.nchunk * f.nrow_q * f.w_q;
    return f;
}
constexpr int DB_SPLITS = 64;

struct BwdWs {
    long long dO, low, exp, delta, delta_q, dq, dk, dv, db, db2, total;
};
inline BwdWs layout_backward(const Args &a, int kind, int elem, const BwdPlan &f)
{
    BwdWs w;
    long long at = 0;
    const long long rows = (long long)a.B * a.Lq * a.H, keys = (long long)a.B * a.Lk * a.Hk;
    const auto take = [&](long long bytes) { const long long r = at; at += align_up(bytes); return r; };
    w.dO = take(a.gate ? rows * a.dv * elem : 0);
    w.low = take(a.gate && a.table && elem == 2 ? rows * a.dv * elem : 0);
    w.exp = take(a.gate && elem == 2 ? rows * 4 : 0);
    w.delta = take(kind == SOFTMAX ? rows * 4 : 0);
    w.delta_q = take(kind == SOFTMAX && a.gate && a.table && elem == 2 ? rows * 4 : 0);
    w.dq = take(f.nchunk > 1 ? rows * a.dk * f.nchunk * 4 : 0);
    w.dk = take(f.nchunk * f.nparts > 1 ? keys * a.dk * f.nchunk * f.nparts * 4 : 0);
    w.dv = take(f.nparts > 1 ? keys * a.dv * f.nparts * 4 : 0);
    w.db = take(a.table ? f.nr * a.H * (2 * a.D + 1) * 4 : 0);
    w.db2 = take(a.table ? (long long)DB_SPLITS * a.H * (2 * a.D + 1) * 4 : 0);
    w.total = at;
    return w;
}

// sums of the waves' distance rows in a fixed order: (H, R, TW) -> (H, S, TW) -> bucket by bucket (num_buckets, H)
static __global__ void __launch_bounds__(256) db_rows_kernel(const float *part, float *out, long long R, int TW)
{
    const int h = blockIdx.x / DB_SPLITS, s = blockIdx.x % DB_SPLITS;
    const long long per = (R + DB_SPLITS - 1) / DB_SPLITS, r0 = s * per, r1 = r0 + per < R ? r0 + per : R;
    for (int t = threadIdx.x; t < TW; t += 256) {
        float x = 0.f;
#pragma unroll 8
        for (long long r = r0; r < r1; ++r) x += part[(h * R + r) * TW + t];
        out[(long long)blockIdx.x * TW + t] = x;
    }
}
template <class T> __global__ void __launch_bounds__(1024) db_buckets_kernel(const float *part, const int *bucket_of, void *dtable, int H, int TW, int nb, int f32)
{
    extern __shared__ float sums[];
    __shared__ float quarter[4][256];
    int *bk = reinterpret_cast<int *>(sums + TW);
    const int h = blockIdx.x, lane = threadIdx.x & 255, q = threadIdx.x >> 8;
    for (int t0 = 0; t0 < TW; t0 += 256) {
        const int t = t0 + lane;
        float x = 0.f;
        if (t < TW)
#pragma unroll
            for (int s = 0; s < DB_SPLITS / 4; ++s) x += part[((long long)h * DB_SPLITS + q * (DB_SPLITS / 4) + s) * TW + t];
        quarter[q][lane] = x;
        __syncthreads();
        if (q == 0 && t < TW) {
            sums[t] = quarter[0][lane] + quarter[1][lane] + quarter[2][lane] + quarter[3][lane];
            const int b = bucket_of[t];
            bk[t] = b < 0 ? 0 : (b >= nb ? nb - 1 : b);
        }
        __syncthreads();
    }
    for (int b0 = 0; b0 < nb; b0 += 64) {                             // 16 lanes a bucket
        const int b = b0 + (threadIdx.x >> 4);
        float x = 0.f;
#pragma unroll 4
        for (int t = threadIdx.x & 15; t < TW; t += 16) x += bk[t] == b ? sums[t] : 0.f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) x += __shfl_xor(x, o);
        if (b < nb && (threadIdx.x & 15) == 0) {
            if (f32) reinterpret_cast<float *>(dtable)[(long long)b * H + h] = x;
            else reinterpret_cast<T *>(dtable)[(long long)b * H + h] = (T)x;
        }
    }
}

// `fixed`: the kernel's static LDS, `smem`: the bias table and sums behind it
template <class K> int launch(K kernel, long long blocks, int threads, size_t fixed, size_t smem, const Args &a, hipStream_t st)
{
    if (blocks <= 0) return TLK_OK;
    if (blocks > 0x7fffffffLL) return fail(TLK_EINVAL, "tlk_gau_attention: more than 2^31 - 1 workgroups");
    if (fixed + smem + 1024 > 160 * 1024) return fail(TLK_EINVAL, "tlk_gau_attention: max_distance beyond the LDS tile");
    if (fixed + smem > 64 * 1024 && smem > 0) TLK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), smem, st, a);
    TLK_HIP(hipGetLastError());
    return TLK_OK;
}

template <class T, int KIND, int DK, int MT, int NT, int WM, int WN> int launch_fwd(const Args &a, const FwdPlan &f, hipStream_t st)
{
    constexpr int KT = WN == 1 && sizeof(T) == 2 && NT <= 8 ? 64 : 32;          // (two buffers of 64 keys leave two workgroups a CU up to 128 columns)
    const size_t fixed = sizeof(T) * KT * (tile_width(DK) + WN * NT * 16), smem = a.table ? sizeof(float) * (f.fold ? a.H / a.Hk : 1) * table_width(a.D) : 0;
    const long long blocks = (long long)a.B * f.heads * f.nsplit * f.nchunk * f.nrow;
    if constexpr (WN > 1)                                           // (one tile of keys: a second buffer would only keep other workgroups off the CU)
        if (a.Lk <= KT) return launch(fwd_kernel<T, KIND, DK, MT, NT, WM, WN, KT, true>, blocks, 64 * WM * WN, fixed, smem, a, st);
    return launch(fwd_kernel<T, KIND, DK, MT, NT, WM, WN, KT, false>, blocks, 64 * WM * WN, 2 * fixed, smem, a, st);
}
// Causal walks differ in length.  Between one and two workgroups a CU, all are resident at once, and the CU that holds the i-th of the first 256 is taken to
// hold the i-th behind them: those come shortest first, so that the longest walk shares its CU with the shortest.
inline int snake_from(const Args &a, long long walks, int nrow)
{
    return a.causal && walks * nrow > 256 && walks * nrow <= 512 && 256 % walks == 0 ? (int)(256 / walks) : nrow;
}
template <class T, int KIND, int DK> int pick_fwd(const Args &a, const FwdPlan &f, hipStream_t st)
{
    if (!f.few) {
        if (f.dvb == 64) return launch_fwd<T, KIND, DK, 2, 4, 4, 1>(a, f, st);
        if (f.dvb == 128) return launch_fwd<T, KIND, DK, 2, 8, 4, 1>(a, f, st);
        return launch_fwd<T, KIND, DK, 2, 16, 4, 1>(a, f, st);
    }
    if (f.mt == 1) {
        if (f.dvb == 64) return launch_fwd<T, KIND, DK, 1, 1, 1, 4>(a, f, st);
        if (f.dvb == 128) return launch_fwd<T, KIND, DK, 1, 2, 1, 4>(a, f, st);
        if constexpr (sizeof(T) == 2)
            if (f.dvb == 512) return launch_fwd<T, KIND, DK, 1, 8, 1, 4>(a, f, st);
        return launch_fwd<T, KIND, DK, 1, 4, 1, 4>(a, f, st);
    }
    if (f.dvb == 64) return launch_fwd<T, KIND, DK, 2, 1, 1, 4>(a, f, st);
    if (f.dvb == 128) return launch_fwd<T, KIND, DK, 2, 2, 1, 4>(a, f, st);
    if constexpr (sizeof(T) == 2)
        if (f.dvb == 512) return launch_fwd<T, KIND, DK, 2, 8, 1, 4>(a, f, st);
    return launch_fwd<T, KIND, DK, 2, 4, 1, 4>(a, f, st);
}
template <class T> int forward(Args a, int kind, void *ws, hipStream_t st)
{
    const FwdPlan f = plan_forward(a, sizeof(T));
    a.fold = f.fold; a.nrow = f.nrow; a.nchunk = f.nchunk; a.nsplit = f.nsplit; a.split_keys = f.split_keys;
    a.snake = snake_from(a, (long long)a.B * f.heads * f.nchunk * f.nsplit, f.nrow);
    const long long rows = (long long)a.B * a.Lq * a.H;
    a.part = reinterpret_cast<float *>(ws);
    a.ml = a.part + (f.nsplit > 1 ? rows * a.dv * f.nsplit : 0);
    int rc;
    if (kind == SOFTMAX) rc = a.dk <= 64 ? pick_fwd<T, SOFTMAX, 64>(a, f, st) : (a.dk <= 96 ? pick_fwd<T, SOFTMAX, 96>(a, f, st) : pick_fwd<T, SOFTMAX, 128>(a, f, st));
    else rc = a.dk <= 64 ? pick_fwd<T, RELU2, 64>(a, f, st) : (a.dk <= 96 ? pick_fwd<T, RELU2, 96>(a, f, st) : pick_fwd<T, RELU2, 128>(a, f, st));
    if (rc != TLK_OK || f.nsplit == 1) return rc;
    const long long blocks = rows * ((a.dv + 63) / 64);
    return kind == SOFTMAX ? launch(join_kernel<T, SOFTMAX>, blocks, 64, 0, 0, a, st) : launch(join_kernel<T, RELU2>, blocks, 64, 0, 0, a, st);
}

template <class T, int KIND, int DK, int DVC, int W, bool LOW> int launch_dq(const Args &a, const BwdPlan &f, hipStream_t st)
{
    constexpr int MT = sizeof(T) == 4 ? 1 : 2;
    const size_t fixed = sizeof(T) * 32 * (tile_width(DK) + DVC), smem = a.table ? sizeof(float) * (table_width(a.D) + W * (2 * a.D + 1) + W * 32 * (MT * 16 + 1)) : 0;
    const long long blocks = (long long)a.B * a.H * f.nchunk * f.nrow_q;
    if constexpr (W < 4)
        if (a.Lk <= 32) return launch(dq_kernel<T, KIND, DK, DVC, MT, W, true, LOW>, blocks, 64 * W, fixed, smem, a, st);
    return launch(dq_kernel<T, KIND, DK, DVC, MT, W, false, LOW>, blocks, 64 * W, 2 * fixed, smem, a, st);
}
template <class T, int KIND, int DK, int DVC, bool LOW> int pick_dq(const Args &a, const BwdPlan &f, hipStream_t st)
{
    if (f.w_q == 1) return launch_dq<T, KIND, DK, DVC, 1, LOW>(a, f, st);
    return f.w_q == 2 ? launch_dq<T, KIND, DK, DVC, 2, LOW>(a, f, st) : launch_dq<T, KIND, DK, DVC, 4, LOW>(a, f, st);
}
template <class T, int KIND, int DK, int DVC, int W> int launch_dkv(const Args &a, const BwdPlan &f, hipStream_t st)
{
    constexpr int MT = sizeof(T) == 4 ? 1 : 2;
    const size_t fixed = sizeof(T) * 32 * (tile_width(DK) + DVC), smem = a.table ? sizeof(float) * table_width(a.D) : 0;
    const long long blocks = (long long)a.B * a.Hk * f.nchunk * f.nparts * f.nrow_k;
    if constexpr (W < 4)
        if (a.Lq <= 32) return launch(dkv_kernel<T, KIND, DK, DVC, MT, W, true>, blocks, 64 * W, fixed + 768, smem, a, st);
    return launch(dkv_kernel<T, KIND, DK, DVC, MT, W, false>, blocks, 64 * W, 2 * fixed + 768, smem, a, st);
}
template <class T, int KIND, int DK, int DVC> int pick_bwd(Args a, const BwdPlan &f, hipStream_t st)
{
    a.nchunk = f.nchunk;
    a.nparts = f.nparts;
    a.nrow = f.nrow_q;
    // (two parts of dO at 256 columns: one workgroup a CU, so the longest walks first do by themselves; 4 x 4096 causal tokens, dv 1024: 298 us in the order for two, 250 so)
    a.snake = a.dO_low && DVC == 256 ? f.nrow_q : snake_from(a, (long long)a.B * a.H * f.nchunk, f.nrow_q);
    int rc;
    if constexpr (sizeof(T) == 2) rc = a.dO_low ? pick_dq<T, KIND, DK, DVC, true>(a, f, st) : pick_dq<T, KIND, DK, DVC, false>(a, f, st);
    else rc = pick_dq<T, KIND, DK, DVC, false>(a, f, st);
    if (rc != TLK_OK) return rc;
    a.nrow = f.nrow_k;
    if (f.w_k == 1) return launch_dkv<T, KIND, DK, DVC, 1>(a, f, st);
    if (f.w_k == 2) return launch_dkv<T, KIND, DK, DVC, 2>(a, f, st);
    return launch_dkv<T, KIND, DK, DVC, 4>(a, f, st);
}
template <class T, int KIND> int pick_bwd_sizes(const Args &a, const BwdPlan &f, hipStream_t st)
{
    const auto widths = [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        return f.dvc == 64 ? pick_bwd<T, KIND, DK, 64>(a, f, st) : (f.dvc == 128 ? pick_bwd<T, KIND, DK, 128>(a, f, st) : pick_bwd<T, KIND, DK, 256>(a, f, st));
    };
    if (a.dk <= 64) return widths(std::integral_constant<int, 64>());
    return a.dk <= 96 ? widths(std::integral_constant<int, 96>()) : widths(std::integral_constant<int, 128>());
}
template <class T> int backward(Args a, const BwdIo &io, int kind, hipStream_t st)
{
    const BwdPlan f = plan_backward(a, sizeof(T));
    const BwdWs w = layout_backward(a, kind, sizeof(T), f);
    char *ws = reinterpret_cast<char *>(io.ws);
    const long long rows = (long long)a.B * a.Lq * a.H, keys = (long long)a.B * a.Lk * a.Hk;
    a.dO = io.dout;
    if ((a.gate || kind == SOFTMAX) && rows > 0) {
        GateArgs<T> ga;
        ga.dout = reinterpret_cast<const T *>(io.dout); ga.gate = reinterpret_cast<const T *>(a.gate); ga.o = io.o;
        for (int i = 0; i < 3; ++i) ga.gs[i] = a.gs[i];
        ga.dO = a.gate ? reinterpret_cast<T *>(ws + w.dO) : nullptr;
        ga.low = a.gate && a.table && sizeof(T) == 2 ? reinterpret_cast<T *>(ws + w.low) : nullptr;
        ga.dO_exp = a.gate && Ty<T>::scaled ? reinterpret_cast<float *>(ws + w.exp) : nullptr;
        ga.dgate = reinterpret_cast<T *>(io.dgate);
        ga.delta = kind == SOFTMAX ? reinterpret_cast<float *>(ws + w.delta) : nullptr;
        ga.delta_q = kind == SOFTMAX && ga.low ? reinterpret_cast<float *>(ws + w.delta_q) : ga.delta;
        ga.rows = rows; ga.Lq = a.Lq; ga.H = a.H; ga.dv = a.dv;
        const int lanes = a.dv <= 64 ? 16 : (a.dv <= 128 ? 32 : 64);
        const long long blocks = (rows + 256 / lanes - 1) / (256 / lanes);
        if (blocks > 0x7fffffffLL) return fail(TLK_EINVAL, "tlk_gau_attention: more than 2^31 - 1 workgroups");
        const auto by_lanes = [&](auto o) { using O = decltype(o); return lanes == 16 ? gate_bwd_kernel<T, O, 16> : (lanes == 32 ? gate_bwd_kernel<T, O, 32> : gate_bwd_kernel<T, O, 64>); };
        const auto kernel = kind == RELU2 ? by_lanes(Kept<T, RELU2>()) : by_lanes(Kept<T, SOFTMAX>());
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, ga);
        TLK_HIP(hipGetLastError());
        if (a.gate) a.dO = ws + w.dO;
        a.delta = ga.delta;
        a.delta_q = ga.delta_q;
        a.dO_low = ga.low;
        a.dO_exp = ga.dO_exp;
    }
    a.dq = io.dq; a.dk_ = io.dk; a.dv_ = io.dv;
    a.dq_part = reinterpret_cast<float *>(ws + w.dq);
    a.dk_part = reinterpret_cast<float *>(ws + w.dk);
    a.dv_part = reinterpret_cast<float *>(ws + w.dv);
    a.db_part = reinterpret_cast<float *>(ws + w.db);
    int rc = kind == SOFTMAX ? pick_bwd_sizes<T, SOFTMAX>(a, f, st) : pick_bwd_sizes<T, RELU2>(a, f, st);
    if (rc != TLK_OK) return rc;
    const auto join = [&](const float *part, void *y, long long n, int parts) -> int {
        if (parts <= 1 || n <= 0) return TLK_OK;
        if ((n / 4 + 255) / 256 > 0x7fffffffLL) return fail(TLK_EINVAL, "tlk_gau_attention: more than 2^31 - 1 workgroups");
        hipLaunchKernelGGL(sum_parts_kernel<T>, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, part, reinterpret_cast<T *>(y), n, parts);
        TLK_HIP(hipGetLastError());
        return TLK_OK;
    };
    if ((rc = join(a.dq_part, a.dq, rows * a.dk, f.nchunk)) != TLK_OK) return rc;
    if ((rc = join(a.dk_part, a.dk_, keys * a.dk, f.nchunk * f.nparts)) != TLK_OK) return rc;
    if ((rc = join(a.dv_part, a.dv_, keys * a.dv, f.nparts)) != TLK_OK) return rc;
    if (a.table) {
        const int TW = 2 * a.D + 1;
        float *p2 = reinterpret_cast<float *>(ws + w.db2);
        hipLaunchKernelGGL(db_rows_kernel, dim3((unsigned)(a.H * DB_SPLITS)), dim3(256), 0, st, a.db_part, p2, f.nr, TW);
        hipLaunchKernelGGL(db_buckets_kernel<T>, dim3((unsigned)a.H), dim3(1024), (size_t)TW * 8, st, p2, a.bucket_of, io.dtable, a.H, TW, a.nb, a.table_f32);
        TLK_HIP(hipGetLastError());
    }
    return TLK_OK;
}

}  // namespace gau
}  // namespace tlk
