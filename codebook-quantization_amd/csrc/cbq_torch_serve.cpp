// torch.ops.cbq's operators of batched serving (include/cbq_serve.h): checks of
// the tensors, outputs and workspaces from torch's caching allocator, torch's
// current HIP stream.  Host code only, as cbq_torch_ops.cpp.
//
//   paged_append(q, k, v, cos, sin, positions, slots, k_pages, v_pages, norm,
//                q_weight, k_weight, eps) -> q                    cbq_paged_append
//   prefix_attention_decode(q, k_pages, v_pages, prefix_table, prefix, tables,
//                           lengths, scale) -> out                cbq_prefix_attn_decode
//   prefix_attention_prompt(q, q_start, k_pages, v_pages, prefix_table, prefix,
//                           tables, lengths, scale) -> out        cbq_prefix_attn_prompt
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>

#include "../../include/cbq_hip.h"
#include "../../include/cbq_serve.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

int dtype_of(const at::Tensor &t, const char *op, const char *name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return CBQ_F32;
    case at::kBFloat16: return CBQ_BF16;
    case at::kHalf: return CBQ_F16;
    default: TORCH_CHECK(false, op, ": ", name, " must be float32, bfloat16 or float16");
    }
}

void check_on(const at::Tensor &t, const at::Tensor &ref, const char *op, const char *name)
{
    TORCH_CHECK(t.device() == ref.device(), op, ": ", name, " is on ", t.device(), ", expected ",
                ref.device());
}

void check_index(const at::Tensor &t, const at::Tensor &ref, at::ScalarType type, int64_t dim,
                 const char *op, const char *name)
{
    check_on(t, ref, op, name);
    TORCH_CHECK(t.scalar_type() == type && t.dim() == dim, op, ": ", name, " must be a ", dim,
                "-D ", type, " tensor");
}

// k_pages and v_pages [n_pages, n_kv, page, hd] in any strides with hd contiguous
cbq_paged_kv pool(const at::Tensor &k, const at::Tensor &v, const at::Tensor &ref, const char *op)
{
    check_on(k, ref, op, "k_pages");
    check_on(v, ref, op, "v_pages");
    TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(), op,
                ": k_pages and v_pages must be [n_pages, n_kv, page, hd] of one shape");
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), op,
                ": k_pages and v_pages must be of one type");
    TORCH_CHECK(k.numel() > 0, op, ": the pool is empty");
    TORCH_CHECK(k.stride(3) == 1 && v.stride(3) == 1, op,
                ": the pages' last dimension must be contiguous");
    TORCH_CHECK(k.size(0) < (1ll << 31) && k.size(1) < (1ll << 20) && k.size(2) <= 65536 &&
                    k.size(3) <= 256 && k.size(0) * k.size(2) < (1ll << 31),
                op, ": pages of at most 65536 rows of at most 256 values, fewer than 2^31 rows");
    cbq_paged_kv c;
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    for (int i = 0; i < 3; i++) {
        c.k_stride[i] = k.stride(i);
        c.v_stride[i] = v.stride(i);
    }
    c.n_pages = k.size(0);
    c.n_kv = (int32_t)k.size(1);
    c.page = (int32_t)k.size(2);
    c.hd = (int32_t)k.size(3);
    c.dtype = dtype_of(k, op, "k_pages");
    return c;
}

void check_rows(const at::Tensor &t, int64_t tokens, int64_t heads, int64_t hd,
                const at::Tensor &ref, const char *op, const char *name)
{
    check_on(t, ref, op, name);
    TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == hd, op,
                ": ", name, " must be [", tokens, ", ", heads, ", ", hd, "], got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == ref.scalar_type(), op, ": ", name, " must be of q's type");
}

// the last dimension contiguous (a copy of the few new rows where it is not)
at::Tensor rows_of(const at::Tensor &t)
{
    return t.stride(2) == 1 ? t : t.contiguous();
}

void check_done(int rc, const char *what)
{
    TORCH_CHECK(rc == CK_SUCCESS, what, " returned ", rc, " (", ck_error_string(rc), ")");
}

hipStream_t stream_of(const at::Tensor &t)
{
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

const float *weight_of(const OptTensor &w, bool norm, const at::Tensor &q, const char *op,
                       const char *name)
{
    if (!w.has_value() || !w->defined()) return nullptr;
    TORCH_CHECK(norm, op, ": ", name, " without the norm");
    check_on(*w, q, op, name);
    TORCH_CHECK(w->scalar_type() == at::kFloat && w->dim() == 1 && w->size(0) == q.size(2) &&
                    w->is_contiguous(),
                op, ": ", name, " must be a contiguous float32 [", q.size(2), "]");
    return w->data_ptr<float>();
}

at::Tensor paged_append(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                        const at::Tensor &cos, const at::Tensor &sin, const at::Tensor &positions,
                        const at::Tensor &slots, at::Tensor &k_pages, at::Tensor &v_pages,
                        bool norm, const OptTensor &q_weight, const OptTensor &k_weight, double eps)
{
    const char *op = "cbq::paged_append";
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, op, ": q must be a [N, n_q, hd] device tensor");
    const cbq_paged_kv c = pool(k_pages, v_pages, q, op);
    const int64_t N = q.size(0), n_q = q.size(1);
    TORCH_CHECK(n_q >= 1 && n_q < (1ll << 20) && N < (1ll << 31) &&
                    N * (n_q + 2 * c.n_kv) < (1ll << 31),
                op, ": fewer than 2^31 head rows");
    TORCH_CHECK(c.hd % 2 == 0 && c.hd >= 2, op, ": hd must be even");
    const int x_dtype = dtype_of(q, op, "q");
    check_rows(q, N, n_q, c.hd, q, op, "q");
    check_rows(k, N, c.n_kv, c.hd, q, op, "k");
    check_rows(v, N, c.n_kv, c.hd, q, op, "v");
    TORCH_CHECK(x_dtype == CBQ_F32 || x_dtype == c.dtype, op,
                ": 16-bit q, k and v go into pages of their own type");
    for (const auto &t : {std::make_pair(&cos, "cos"), std::make_pair(&sin, "sin")}) {
        check_on(*t.first, q, op, t.second);
        TORCH_CHECK(t.first->scalar_type() == at::kFloat && t.first->dim() == 2 &&
                        t.first->is_contiguous() && t.first->sizes() == cos.sizes(),
                    op, ": cos and sin must be contiguous float32 [positions, rot] of one shape");
    }
    const int64_t rot = cos.size(1);
    TORCH_CHECK(cos.size(0) >= 1 && rot >= 2 && rot % 2 == 0 && rot <= c.hd, op,
                ": the tables need a row, and an even width of at most hd");
    for (const auto &t : {std::make_pair(&positions, "positions"), std::make_pair(&slots, "slots")}) {
        check_index(*t.first, q, at::kLong, 1, op, t.second);
        TORCH_CHECK(t.first->size(0) == N && t.first->is_contiguous(), op, ": ", t.second,
                    " must be contiguous, one a token");
    }
    TORCH_CHECK(!norm || (std::isfinite(eps) && eps >= 0), op, ": eps must be finite and not below 0");
    const float *qw = weight_of(q_weight, norm, q, op, "q_weight"),
                *kw = weight_of(k_weight, norm, q, op, "k_weight");
    c10::DeviceGuard guard(q.device());
    at::Tensor out = at::empty({N, n_q, c.hd}, k_pages.options());
    if (N == 0) return out;
    const at::Tensor x = rows_of(q), y = rows_of(k), z = rows_of(v);
    const int64_t xs[2] = {x.stride(0), x.stride(1)}, ys[2] = {y.stride(0), y.stride(1)},
                  zs[2] = {z.stride(0), z.stride(1)};
    check_done(cbq_paged_append(x.data_ptr(), y.data_ptr(), z.data_ptr(), x_dtype, xs, ys, zs,
                                cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), (int)rot,
                                positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), norm, qw,
                                kw, (float)eps, out.data_ptr(), &c, N, (int)n_q, stream_of(q)),
               "cbq_paged_append");
    return out;
}

at::Tensor attend(const at::Tensor &q, const at::Tensor *q_start, const at::Tensor &k_pages,
                  const at::Tensor &v_pages, const at::Tensor &prefix_table, int64_t prefix,
                  const at::Tensor &tables, const at::Tensor &lengths, double scale, const char *op)
{
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, op, ": q must be a [N, n_q, hd] device tensor");
    const cbq_paged_kv c = pool(k_pages, v_pages, q, op);
    const int64_t N = q.size(0), n_q = q.size(1);
    TORCH_CHECK(c.hd == 64 || c.hd == 128 || c.hd == 256, op, ": hd must be 64, 128 or 256");
    TORCH_CHECK(dtype_of(q, op, "q") == c.dtype, op, ": q must be of the pages' type");
    TORCH_CHECK(q.size(2) == c.hd && n_q >= 1 && n_q % c.n_kv == 0, op, ": q is ", q.sizes(),
                ", the pages hold ", c.n_kv, " heads of ", c.hd);
    check_index(tables, q, at::kInt, 2, op, "tables");
    check_index(lengths, q, at::kInt, 1, op, "lengths");
    check_index(prefix_table, q, at::kInt, 1, op, "prefix_table");
    const int64_t batch = lengths.size(0), width = tables.size(1);
    TORCH_CHECK(tables.size(0) == batch && lengths.is_contiguous() &&
                    (width <= 1 || tables.stride(1) == 1) && prefix_table.is_contiguous(),
                op, ": tables [batch, pages], lengths [batch] and prefix_table must be contiguous "
                "in their last dimension");
    TORCH_CHECK(prefix >= 0 && prefix_table.size(0) < (1ll << 31) &&
                    prefix <= prefix_table.size(0) * c.page,
                op, ": prefix_table names ", prefix_table.size(0), " pages of ", c.page,
                " rows for ", prefix, " keys");
    TORCH_CHECK(width < (1ll << 31) && prefix + width * c.page <= (1ll << 31) - 65536, op,
                ": too many keys");
    TORCH_CHECK(N < (1ll << 31) && batch < (1ll << 30) && n_q < (1ll << 20) && N * n_q < (1ll << 31),
                op, ": too many rows");
    if (q_start) {
        check_index(*q_start, q, at::kInt, 1, op, "q_start");
        TORCH_CHECK(q_start->size(0) == batch + 1 && q_start->is_contiguous(), op,
                    ": q_start must be contiguous, [batch + 1]");
    } else {
        TORCH_CHECK(N == batch, op, ": one token a sequence, got ", N, " for ", batch);
    }
    TORCH_CHECK(std::abs(scale) <= 3.0e38, op, ": scale must be finite");
    const int64_t e = q.element_size();
    for (const at::Tensor *t : {&k_pages, &v_pages}) {
        bool ok = (uintptr_t)t->data_ptr() % 16 == 0;
        for (int i = 0; i < 3; i++) ok = ok && t->stride(i) * e % 16 == 0;
        TORCH_CHECK(ok, op, ": the pages must be 16-byte aligned, strides included");
    }
    c10::DeviceGuard guard(q.device());
    at::Tensor out = at::empty({N, n_q, c.hd}, q.options());
    if (N == 0) return out;
    if (batch == 0) return out.zero_();                 // tokens of no run
    at::Tensor x = rows_of(q);
    if ((uintptr_t)x.data_ptr() % 16 || x.stride(0) * e % 16 || x.stride(1) * e % 16)
        x = x.clone(at::MemoryFormat::Contiguous);
    const int64_t xs[2] = {x.stride(0), x.stride(1)};
    const size_t nws = q_start ? cbq_prefix_attn_prompt_workspace(&c, prefix, (int)width, (int)batch,
                                                                  N, (int)n_q)
                               : cbq_prefix_attn_decode_workspace(&c, prefix, (int)width, (int)batch,
                                                                  (int)n_q);
    at::Tensor ws;
    if (nws) ws = at::empty({(int64_t)nws}, q.options().dtype(at::kByte));
    void *wp = nws ? ws.data_ptr() : nullptr;
    if (q_start)
        check_done(cbq_prefix_attn_prompt(x.data_ptr(), xs, q_start->data_ptr<int32_t>(), &c,
                                          prefix_table.data_ptr<int32_t>(), prefix,
                                          tables.data_ptr<int32_t>(), tables.stride(0), (int)width,
                                          lengths.data_ptr<int32_t>(), (int)batch, N, (int)n_q,
                                          (float)scale, out.data_ptr(), wp, nws, stream_of(q)),
                   "cbq_prefix_attn_prompt");
    else
        check_done(cbq_prefix_attn_decode(x.data_ptr(), xs, &c, prefix_table.data_ptr<int32_t>(),
                                          prefix, tables.data_ptr<int32_t>(), tables.stride(0),
                                          (int)width, lengths.data_ptr<int32_t>(), (int)batch,
                                          (int)n_q, (float)scale, out.data_ptr(), wp, nws,
                                          stream_of(q)),
                   "cbq_prefix_attn_decode");
    return out;
}

at::Tensor prefix_attention_decode(const at::Tensor &q, const at::Tensor &k_pages,
                                   const at::Tensor &v_pages, const at::Tensor &prefix_table,
                                   int64_t prefix, const at::Tensor &tables,
                                   const at::Tensor &lengths, double scale)
{
    return attend(q, nullptr, k_pages, v_pages, prefix_table, prefix, tables, lengths, scale,
                  "cbq::prefix_attention_decode");
}

at::Tensor prefix_attention_prompt(const at::Tensor &q, const at::Tensor &q_start,
                                   const at::Tensor &k_pages, const at::Tensor &v_pages,
                                   const at::Tensor &prefix_table, int64_t prefix,
                                   const at::Tensor &tables, const at::Tensor &lengths,
                                   double scale)
{
    return attend(q, &q_start, k_pages, v_pages, prefix_table, prefix, tables, lengths, scale,
                  "cbq::prefix_attention_prompt");
}

// Shape functions for tracing (meta tensors): same output shapes and dtypes.
at::Tensor paged_append_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &,
                             const at::Tensor &, const at::Tensor &, const at::Tensor &,
                             const at::Tensor &, at::Tensor &k_pages, at::Tensor &, bool,
                             const OptTensor &, const OptTensor &, double)
{
    return at::empty(q.sizes(), k_pages.options());
}

at::Tensor decode_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &,
                       const at::Tensor &, int64_t, const at::Tensor &, const at::Tensor &, double)
{
    return at::empty(q.sizes(), q.options());
}

at::Tensor prompt_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &,
                       const at::Tensor &, const at::Tensor &, int64_t, const at::Tensor &,
                       const at::Tensor &, double)
{
    return at::empty(q.sizes(), q.options());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cbq, m)
{
    m.def("paged_append(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor positions, "
          "Tensor slots, Tensor(a!) k_pages, Tensor(b!) v_pages, bool norm, Tensor? q_weight, "
          "Tensor? k_weight, float eps) -> Tensor");
    m.def("prefix_attention_decode(Tensor q, Tensor k_pages, Tensor v_pages, Tensor prefix_table, "
          "int prefix, Tensor tables, Tensor lengths, float scale) -> Tensor");
    m.def("prefix_attention_prompt(Tensor q, Tensor q_start, Tensor k_pages, Tensor v_pages, "
          "Tensor prefix_table, int prefix, Tensor tables, Tensor lengths, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(cbq, CUDA, m)
{
    m.impl("paged_append", &paged_append);
    m.impl("prefix_attention_decode", &prefix_attention_decode);
    m.impl("prefix_attention_prompt", &prefix_attention_prompt);
}

TORCH_LIBRARY_IMPL(cbq, Meta, m)
{
    m.impl("paged_append", &paged_append_meta);
    m.impl("prefix_attention_decode", &decode_meta);
    m.impl("prefix_attention_prompt", &prompt_meta);
}
