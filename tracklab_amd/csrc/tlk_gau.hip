// tlk_gau.hip -- C entries of the gated attention unit's core: argument checks, workspace, dispatch on the element type (kernels: tlk_gau.hpp).
#include "tlk_gau_host.hpp"

using namespace tlk;

namespace tlk {
namespace gau {
extern template int forward<_Float16>(Args, int, void *, hipStream_t);
extern template int forward<__bf16>(Args, int, void *, hipStream_t);
extern template int forward<float>(Args, int, void *, hipStream_t);
extern template int backward<_Float16>(Args, const BwdIo &, int, hipStream_t);
extern template int backward<__bf16>(Args, const BwdIo &, int, hipStream_t);
extern template int backward<float>(Args, const BwdIo &, int, hipStream_t);
}  // namespace gau
}  // namespace tlk

namespace {

int fill(const tlk_gau_args *a, gau::Args &p, const char *fn)
{
    const std::string f(fn);
    if (!a) return fail(TLK_EINVAL, f + ": null arguments");
    if (a->dtype != TLK_F32 && a->dtype != TLK_F16 && a->dtype != TLK_BF16) return fail(TLK_EINVAL, f + ": dtype must be TLK_F32, TLK_F16 or TLK_BF16");
    if (a->kind != TLK_GAU_RELU2 && a->kind != TLK_GAU_SOFTMAX) return fail(TLK_EINVAL, f + ": kind must be TLK_GAU_RELU2 or TLK_GAU_SOFTMAX");
    const int vn = a->dtype == TLK_F32 ? 4 : 8, big = 1 << 28;
    if (a->batch < 0 || a->len_q < 0 || a->len_k < 0 || a->len_q > big || a->len_k > big) return fail(TLK_EINVAL, f + ": batch and lengths must lie in 0..2^28");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535) return fail(TLK_EINVAL, f + ": heads must be a positive multiple of kv_heads");
    if (a->dim_k < vn || a->dim_k % vn != 0 || a->dim_k > 128) return fail(TLK_EINVAL, f + ": dim_k must be a multiple of 16 bytes of elements, at most 128");
    if (a->dim_v < vn || a->dim_v % vn != 0 || a->dim_v > 65536 || (long long)a->heads * a->dim_v > 1 << 22) return fail(TLK_EINVAL, f + ": dim_v must be a positive multiple of 16 bytes of elements, heads * dim_v at most 2^22");
    if (a->num_buckets < 0 || a->max_distance < 0 || a->max_distance > 2048) return fail(TLK_EINVAL, f + ": max_distance must lie in 0..2048");
    if ((a->num_buckets > 0) != (a->table != nullptr) || (a->num_buckets > 0) != (a->bucket_of != nullptr)) return fail(TLK_EINVAL, f + ": a bias needs num_buckets, table and bucket_of");
    const long long rows = (long long)a->batch * a->len_q, keys = (long long)a->batch * a->len_k;
    if (rows > 0 && !a->q) return fail(TLK_EINVAL, f + ": null q");
    if (keys > 0 && (!a->k || !a->v)) return fail(TLK_EINVAL, f + ": null k or v");
    if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->gate) & 15) return fail(TLK_EINVAL, f + ": q, k, v and gate must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
        if (a->q_stride[i] < 0 || a->k_stride[i] < 0 || a->v_stride[i] < 0 || (a->gate && a->gate_stride[i] < 0)) return fail(TLK_EINVAL, f + ": strides must not be negative");
        if (a->q_stride[i] % vn || a->k_stride[i] % vn || a->v_stride[i] % vn || (a->gate && a->gate_stride[i] % vn))
            return fail(TLK_EINVAL, f + ": strides must be multiples of 16 bytes");
        if (i == 1 && (a->q_stride[i] > 1 << 22 || a->k_stride[i] > 1 << 22 || a->v_stride[i] > 1 << 22)) return fail(TLK_EINVAL, f + ": row strides of q, k and v must not pass 2^22 elements");
        if (i == 1 && ((a->len_q > 1 && a->q_stride[i] < a->dim_k) || (a->len_k > 1 && (a->k_stride[i] < a->dim_k || a->v_stride[i] < a->dim_v))))
            return fail(TLK_EINVAL, f + ": row strides of q, k and v must not be below their widths");
    }
    memset(&p, 0, sizeof(p));
    p.q = a->q; p.k = a->k; p.v = a->v; p.gate = a->gate;
    p.table = a->num_buckets > 0 ? a->table : nullptr;
    p.bucket_of = a->bucket_of; p.lens = a->lens; p.q_start = a->q_start_dev;
    for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.gs[i] = a->gate_stride[i]; }
    if (a->len_q == 1) p.qs[1] = a->dim_k;                          // (the stride of a single row says nothing)
    if (a->len_k == 1) { p.ks[1] = a->dim_k; p.vs[1] = a->dim_v; }
    p.B = a->batch; p.Lq = a->len_q; p.Lk = a->len_k; p.H = a->heads; p.Hk = a->kv_heads; p.dk = a->dim_k; p.dv = a->dim_v;
    p.nb = a->num_buckets; p.D = a->num_buckets > 0 ? a->max_distance : 0; p.q0 = a->q_start; p.causal = a->causal != 0; p.table_f32 = a->table_f32 || a->dtype == TLK_F32;
    p.scale = a->scale;
    return TLK_OK;
}
int elem(int dtype) { return dtype == TLK_F32 ? 4 : 2; }
int kind_of(const tlk_gau_args *a) { return a->kind == TLK_GAU_SOFTMAX ? gau::SOFTMAX : gau::RELU2; }

long long workspace(const gau::Args &p, int kind, int size, bool backward)
{
    if (!backward) {
        const gau::FwdPlan f = gau::plan_forward(p, size);
        return f.nsplit > 1 ? (long long)p.B * p.Lq * p.H * (p.dv + 2) * f.nsplit * 4 : 0;
    }
    return gau::layout_backward(p, kind, size, gau::plan_backward(p, size)).total;
}

}  // namespace

extern "C" long long tlk_gau_attention_workspace(const tlk_gau_args *args, int backward)
{
    gau::Args p;
    const int rc = fill(args, p, "tlk_gau_attention_workspace");
    return rc != TLK_OK ? rc : workspace(p, kind_of(args), elem(args->dtype), backward != 0);
}

extern "C" int tlk_gau_attention_fwd(const tlk_gau_args *args, void *out_dev, void *o_raw_dev, float *lse_dev, void *workspace_dev, long long workspace_bytes,
                                     void *hip_stream)
{
    gau::Args p;
    const int rc = fill(args, p, "tlk_gau_attention_fwd");
    if (rc != TLK_OK) return rc;
    if ((long long)p.B * p.Lq == 0) return TLK_OK;
    if (!out_dev || (((uintptr_t)out_dev | (uintptr_t)o_raw_dev) & 15)) return fail(TLK_EINVAL, "tlk_gau_attention_fwd: out must be given, out and o_raw 16-byte aligned");
    const long long need = workspace(p, kind_of(args), elem(args->dtype), false);
    if (need > 0 && (!workspace_dev || workspace_bytes < need || ((uintptr_t)workspace_dev & 15)))
        return fail(TLK_EINVAL, "tlk_gau_attention_fwd: workspace too small or not 16-byte aligned (tlk_gau_attention_workspace)");
    p.out = out_dev; p.o = o_raw_dev; p.lse = args->kind == TLK_GAU_SOFTMAX ? lse_dev : nullptr;
    hipStream_t st = (hipStream_t)hip_stream;
    if (args->dtype == TLK_F32) return gau::forward<float>(p, kind_of(args), workspace_dev, st);
    return args->dtype == TLK_F16 ? gau::forward<_Float16>(p, kind_of(args), workspace_dev, st) : gau::forward<__bf16>(p, kind_of(args), workspace_dev, st);
}

extern "C" int tlk_gau_attention_bwd(const tlk_gau_args *args, const void *dout_dev, const void *o_raw_dev, const float *lse_dev, void *dq_dev, void *dk_dev,
                                     void *dv_dev, void *dgate_dev, void *dtable_dev, void *workspace_dev, long long workspace_bytes, void *hip_stream)
{
    gau::Args p;
    const int rc = fill(args, p, "tlk_gau_attention_bwd");
    if (rc != TLK_OK) return rc;
    const bool softmax = args->kind == TLK_GAU_SOFTMAX, rows = (long long)p.B * p.Lq > 0, keys = (long long)p.B * p.Lk > 0;
    if (rows && (!dout_dev || !dq_dev)) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: null dout or dq");
    if (keys && (!dk_dev || !dv_dev)) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: null dk or dv");
    if (rows && (softmax || p.gate) && !o_raw_dev) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: o_raw of the forward call is needed");
    if (rows && softmax && !lse_dev) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: lse of the forward call is needed");
    if ((rows && p.gate && !dgate_dev) || (p.table && !dtable_dev)) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: a gradient has no place");
    if (((uintptr_t)dout_dev | (uintptr_t)o_raw_dev | (uintptr_t)dq_dev | (uintptr_t)dk_dev | (uintptr_t)dv_dev | (uintptr_t)dgate_dev | (uintptr_t)workspace_dev) & 15)
        return fail(TLK_EINVAL, "tlk_gau_attention_bwd: tensors must be 16-byte aligned");
    const long long need = workspace(p, kind_of(args), elem(args->dtype), true);
    if (need > 0 && (!workspace_dev || workspace_bytes < need)) return fail(TLK_EINVAL, "tlk_gau_attention_bwd: workspace too small (tlk_gau_attention_workspace)");
    p.lse = const_cast<float *>(lse_dev);
    gau::BwdIo io = {dout_dev, o_raw_dev, dq_dev, dk_dev, dv_dev, dgate_dev, dtable_dev, workspace_dev};
    hipStream_t st = (hipStream_t)hip_stream;
    if (args->dtype == TLK_F32) return gau::backward<float>(p, io, kind_of(args), st);
    return args->dtype == TLK_F16 ? gau::backward<_Float16>(p, io, kind_of(args), st) : gau::backward<__bf16>(p, io, kind_of(args), st);
}
