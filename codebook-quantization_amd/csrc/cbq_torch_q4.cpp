// torch.ops.cbq's operators over the 4-bit paged cache (include/cbq_serve_q4.h) and
// the verification of drafted tokens (include/cbq_serve.h): checks of the tensors,
// outputs and workspaces from torch's caching allocator, torch's current HIP stream.
// Host code only, as cbq_torch_ops.cpp.
//
//   paged_append_q4(q, k, v, cos, sin, positions, slots, k_codes, k_scales, v_codes,
//                   v_scales, norm, q_weight, k_weight, eps) -> q
//   paged_read_q4(k_codes, k_scales, v_codes, v_scales, slots, dtype) -> (k, v)
//   prefix_attention_decode_q4(q, k_codes, k_scales, v_codes, v_scales, prefix_table,
//                              prefix, tables, lengths, scale) -> out
//   verify_drafts(probs, drafts, draft_probs, n_drafts, uniforms) -> (tokens, counts)
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>

#include "../../include/cbq_hip.h"
#include "../../include/cbq_serve_q4.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

int code_of(at::ScalarType t, const char *op, const char *name)
{
    switch (t) {
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

// codes [n_pages, n_kv, page, hd / 2] and scales [n_pages, n_kv, page, hd / 64, 2] of
// keys and values, which lie alike
cbq_paged_q4 pool(const at::Tensor &k_codes, const at::Tensor &k_scales, const at::Tensor &v_codes,
                  const at::Tensor &v_scales, const at::Tensor &ref, const char *op)
{
    check_on(k_codes, ref, op, "k_codes");
    check_on(k_scales, ref, op, "k_scales");
    check_on(v_codes, ref, op, "v_codes");
    check_on(v_scales, ref, op, "v_scales");
    TORCH_CHECK(k_codes.scalar_type() == at::kByte && v_codes.scalar_type() == at::kByte &&
                    k_codes.dim() == 4 && k_codes.sizes() == v_codes.sizes() &&
                    k_codes.strides() == v_codes.strides(),
                op, ": k_codes and v_codes must be uint8 [n_pages, n_kv, page, hd / 2], of one shape and "
                "one layout");
    TORCH_CHECK(k_scales.scalar_type() == at::kBFloat16 && v_scales.scalar_type() == at::kBFloat16 &&
                    k_scales.dim() == 5 && k_scales.sizes() == v_scales.sizes() &&
                    k_scales.strides() == v_scales.strides(),
                op, ": k_scales and v_scales must be bfloat16 [n_pages, n_kv, page, hd / 64, 2], of one "
                "shape and one layout");
    const int64_t hd = 2 * k_codes.size(3);
    TORCH_CHECK(hd == 64 || hd == 128 || hd == 256, op, ": hd must be 64, 128 or 256");
    TORCH_CHECK(k_codes.numel() > 0, op, ": the pool is empty");
    for (int i = 0; i < 3; i++)
        TORCH_CHECK(k_codes.size(i) == k_scales.size(i), op, ": codes are ", k_codes.sizes(),
                    ", scales ", k_scales.sizes());
    TORCH_CHECK(k_scales.size(3) == hd / 64 && k_scales.size(4) == 2, op, ": rows of ", hd,
                " values have ", hd / 64, " pairs of scale and mid");
    TORCH_CHECK(k_codes.stride(3) == 1 && k_scales.stride(4) == 1 &&
                    (hd == 64 || k_scales.stride(3) == 2),
                op, ": a row's codes and its pairs must be contiguous");
    TORCH_CHECK(k_codes.size(0) < (1ll << 31) && k_codes.size(1) < (1ll << 20) &&
                    k_codes.size(2) <= 65536 && k_codes.size(0) * k_codes.size(2) < (1ll << 31),
                op, ": pages of at most 65536 rows, fewer than 2^31 rows");
    cbq_paged_q4 c;
    c.k_codes = k_codes.data_ptr();
    c.v_codes = v_codes.data_ptr();
    c.k_scales = k_scales.data_ptr();
    c.v_scales = v_scales.data_ptr();
    bool aligned = ((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) % 16 == 0 &&
                   ((uintptr_t)c.k_scales | (uintptr_t)c.v_scales) % 4 == 0;
    double codes = 0, scales = 0;
    for (int i = 0; i < 3; i++) {
        c.code_stride[i] = k_codes.stride(i);
        c.scale_stride[i] = k_scales.stride(i);
        aligned = aligned && k_codes.stride(i) % 16 == 0 && k_scales.stride(i) % 2 == 0;
        codes += (double)k_codes.size(i) * (double)k_codes.stride(i);
        scales += (double)k_scales.size(i) * (double)k_scales.stride(i);
    }
    TORCH_CHECK(aligned, op, ": codes must be 16-byte and pairs 4-byte aligned, strides included");
    TORCH_CHECK(codes < 4294967295.0 * 16 && scales < 4294967295.0 * 2, op,
                ": offsets of 64 GiB of codes and 16 GiB of scales at most");
    c.n_pages = k_codes.size(0);
    c.n_kv = (int32_t)k_codes.size(1);
    c.page = (int32_t)k_codes.size(2);
    c.hd = (int32_t)hd;
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

at::Tensor paged_append_q4(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                           const at::Tensor &cos, const at::Tensor &sin, const at::Tensor &positions,
                           const at::Tensor &slots, at::Tensor &k_codes, at::Tensor &k_scales,
                           at::Tensor &v_codes, at::Tensor &v_scales, bool norm,
                           const OptTensor &q_weight, const OptTensor &k_weight, double eps)
{
    const char *op = "cbq::paged_append_q4";
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, op, ": q must be a [N, n_q, hd] device tensor");
    const cbq_paged_q4 c = pool(k_codes, k_scales, v_codes, v_scales, q, op);
    const int64_t N = q.size(0), n_q = q.size(1);
    TORCH_CHECK(n_q >= 1 && n_q < (1ll << 20) && N < (1ll << 31) &&
                    N * (n_q + 2 * c.n_kv) < (1ll << 31),
                op, ": fewer than 2^31 head rows");
    const int x_dtype = code_of(q.scalar_type(), op, "q");
    check_rows(q, N, n_q, c.hd, q, op, "q");
    check_rows(k, N, c.n_kv, c.hd, q, op, "k");
    check_rows(v, N, c.n_kv, c.hd, q, op, "v");
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
    TORCH_CHECK(!norm || (eps >= 0 && eps <= 3.0e38), op, ": eps must be finite and not below 0");
    const float *qw = weight_of(q_weight, norm, q, op, "q_weight"),
                *kw = weight_of(k_weight, norm, q, op, "k_weight");
    c10::DeviceGuard guard(q.device());
    at::Tensor out = at::empty({N, n_q, c.hd}, q.options());
    if (N == 0) return out;
    const at::Tensor x = rows_of(q), y = rows_of(k), z = rows_of(v);
    const int64_t xs[2] = {x.stride(0), x.stride(1)}, ys[2] = {y.stride(0), y.stride(1)},
                  zs[2] = {z.stride(0), z.stride(1)};
    check_done(cbq_paged_append_q4(x.data_ptr(), y.data_ptr(), z.data_ptr(), x_dtype, xs, ys, zs,
                                   cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), (int)rot,
                                   positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), norm, qw,
                                   kw, (float)eps, out.data_ptr(), &c, N, (int)n_q, stream_of(q)),
               "cbq_paged_append_q4");
    return out;
}

std::tuple<at::Tensor, at::Tensor> paged_read_q4(const at::Tensor &k_codes, const at::Tensor &k_scales,
                                                 const at::Tensor &v_codes, const at::Tensor &v_scales,
                                                 const at::Tensor &slots, at::ScalarType dtype)
{
    const char *op = "cbq::paged_read_q4";
    TORCH_CHECK(slots.is_cuda(), op, ": slots must be a device tensor");
    const cbq_paged_q4 c = pool(k_codes, k_scales, v_codes, v_scales, slots, op);
    check_index(slots, slots, at::kLong, 1, op, "slots");
    TORCH_CHECK(slots.is_contiguous(), op, ": slots must be contiguous");
    const int type = code_of(dtype, op, "dtype");
    const int64_t N = slots.size(0);
    TORCH_CHECK((double)N * c.n_kv * c.hd < 549755813888.0, op, ": fewer than 2^39 values");
    c10::DeviceGuard guard(slots.device());
    at::Tensor k = at::empty({N, c.n_kv, c.hd}, slots.options().dtype(dtype)), v = at::empty_like(k);
    if (N == 0) return {k, v};
    check_done(cbq_paged_read_q4(&c, slots.data_ptr<int64_t>(), N, type, k.data_ptr(), v.data_ptr(),
                                 stream_of(slots)),
               "cbq_paged_read_q4");
    return {k, v};
}

at::Tensor prefix_attention_decode_q4(const at::Tensor &q, const at::Tensor &k_codes,
                                      const at::Tensor &k_scales, const at::Tensor &v_codes,
                                      const at::Tensor &v_scales, const at::Tensor &prefix_table,
                                      int64_t prefix, const at::Tensor &tables,
                                      const at::Tensor &lengths, double scale)
{
    const char *op = "cbq::prefix_attention_decode_q4";
    TORCH_CHECK(q.is_cuda() && q.dim() == 3, op, ": q must be a [batch * tokens, n_q, hd] device tensor");
    const cbq_paged_q4 c = pool(k_codes, k_scales, v_codes, v_scales, q, op);
    const int64_t N = q.size(0), n_q = q.size(1);
    const int type = code_of(q.scalar_type(), op, "q");
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
    TORCH_CHECK(batch ? N % batch == 0 : N == 0, op, ": as many tokens for every sequence, got ", N,
                " for ", batch);
    TORCH_CHECK(prefix >= 0 && prefix_table.size(0) < (1ll << 31) &&
                    prefix <= prefix_table.size(0) * c.page,
                op, ": prefix_table names ", prefix_table.size(0), " pages of ", c.page,
                " rows for ", prefix, " keys");
    TORCH_CHECK(width < (1ll << 30) && prefix + width * c.page <= (1ll << 31) - 65536 &&
                    (prefix + c.page - 1) / c.page < (1ll << 30),
                op, ": too many keys");
    TORCH_CHECK(N < (1ll << 31) && batch < (1ll << 30) && n_q < (1ll << 20) &&
                    N * n_q <= (1ll << 31) - 65536,
                op, ": too many rows");
    TORCH_CHECK(std::abs(scale) <= 3.0e38, op, ": scale must be finite");
    c10::DeviceGuard guard(q.device());
    at::Tensor out = at::empty({N, n_q, c.hd}, q.options());
    if (N == 0) return out;
    const int64_t e = q.element_size();
    at::Tensor x = rows_of(q);
    if ((uintptr_t)x.data_ptr() % 16 || x.stride(0) * e % 16 || x.stride(1) * e % 16)
        x = x.clone(at::MemoryFormat::Contiguous);
    const int64_t xs[2] = {x.stride(0), x.stride(1)};
    const int tokens = (int)(N / batch);
    const size_t nws = cbq_prefix_attn_decode_q4_workspace(&c, prefix, (int)width, (int)batch, tokens,
                                                           (int)n_q, type);
    at::Tensor ws;
    if (nws) ws = at::empty({(int64_t)nws}, q.options().dtype(at::kByte));
    check_done(cbq_prefix_attn_decode_q4(x.data_ptr(), xs, type, &c, prefix_table.data_ptr<int32_t>(),
                                         prefix, tables.data_ptr<int32_t>(), tables.stride(0),
                                         (int)width, lengths.data_ptr<int32_t>(), (int)batch, tokens,
                                         (int)n_q, (float)scale, out.data_ptr(),
                                         nws ? ws.data_ptr() : nullptr, nws, stream_of(q)),
               "cbq_prefix_attn_decode_q4");
    return out;
}

std::tuple<at::Tensor, at::Tensor> verify_drafts(const at::Tensor &probs, const at::Tensor &drafts,
                                                 const OptTensor &draft_probs,
                                                 const OptTensor &n_drafts, const at::Tensor &uniforms)
{
    const char *op = "cbq::verify_drafts";
    TORCH_CHECK(probs.is_cuda() && probs.dim() == 3, op,
                ": probs must be a [batch, drafts + 1, vocab] device tensor");
    const int type = code_of(probs.scalar_type(), op, "probs");
    const int64_t batch = probs.size(0), n = probs.size(1) - 1, vocab = probs.size(2);
    TORCH_CHECK(n >= 0 && n < (1ll << 20) && batch < (1ll << 24) && batch * n < (1ll << 30) &&
                    vocab >= 1 && vocab < (1ll << 31),
                op, ": probs is ", probs.sizes(), ": a row a sequence and a token a row at least, and fewer "
                "than 2^24 sequences, 2^20 drafts, 2^30 of both and 2^31 tokens");
    check_index(drafts, probs, at::kLong, 2, op, "drafts");
    TORCH_CHECK(drafts.size(0) == batch && drafts.size(1) == n, op, ": drafts is ", drafts.sizes(),
                ", probs ", probs.sizes());
    check_index(uniforms, probs, at::kFloat, 2, op, "uniforms");
    TORCH_CHECK(uniforms.size(0) == batch && uniforms.size(1) == n + 1, op, ": uniforms is ",
                uniforms.sizes(), ", probs ", probs.sizes());
    const bool given = draft_probs.has_value() && draft_probs->defined();
    if (given) {
        check_on(*draft_probs, probs, op, "draft_probs");
        TORCH_CHECK(draft_probs->scalar_type() == probs.scalar_type() && draft_probs->dim() == 3 &&
                        draft_probs->size(0) == batch && draft_probs->size(1) == n &&
                        draft_probs->size(2) == vocab,
                    op, ": draft_probs must be [", batch, ", ", n, ", ", vocab, "] of probs' type, got ",
                    draft_probs->sizes());
    }
    const bool some = n_drafts.has_value() && n_drafts->defined();
    if (some) {
        check_index(*n_drafts, probs, at::kInt, 1, op, "n_drafts");
        TORCH_CHECK(n_drafts->size(0) == batch && n_drafts->is_contiguous(), op,
                    ": n_drafts must be contiguous, one a sequence");
    }
    c10::DeviceGuard guard(probs.device());
    at::Tensor tokens = at::empty({batch, n + 1}, drafts.options()),
               counts = at::empty({batch}, drafts.options().dtype(at::kInt));
    if (batch == 0) return {tokens, counts};
    // rows in any strides with the vocabulary contiguous; the small tensors whole
    auto rows = [](const at::Tensor &t) { return t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous(); };
    const at::Tensor p = rows(probs), q = given ? rows(*draft_probs) : at::Tensor(),
                     d = drafts.contiguous(), u = uniforms.contiguous();
    const int64_t ps[2] = {p.stride(0), p.stride(1)},
                  qs[2] = {given ? q.stride(0) : 0, given ? q.stride(1) : 0};
    const size_t nws = cbq_verify_drafts_workspace((int)batch, vocab);
    at::Tensor ws = at::empty({(int64_t)nws}, drafts.options().dtype(at::kByte));
    check_done(cbq_verify_drafts(p.data_ptr(), ps, d.data_ptr<int64_t>(), given ? q.data_ptr() : nullptr,
                                 qs, type, some ? n_drafts->data_ptr<int32_t>() : nullptr,
                                 u.data_ptr<float>(), (int)batch, (int)n, vocab,
                                 tokens.data_ptr<int64_t>(), counts.data_ptr<int32_t>(), ws.data_ptr(),
                                 nws, stream_of(probs)),
               "cbq_verify_drafts");
    return {tokens, counts};
}

// Shape functions for tracing (meta tensors): same output shapes and dtypes.
at::Tensor append_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                       const at::Tensor &, const at::Tensor &, const at::Tensor &, at::Tensor &,
                       at::Tensor &, at::Tensor &, at::Tensor &, bool, const OptTensor &,
                       const OptTensor &, double)
{
    return at::empty(q.sizes(), q.options());
}

std::tuple<at::Tensor, at::Tensor> read_meta(const at::Tensor &k_codes, const at::Tensor &,
                                             const at::Tensor &, const at::Tensor &,
                                             const at::Tensor &slots, at::ScalarType dtype)
{
    at::Tensor k = at::empty({slots.size(0), k_codes.size(1), 2 * k_codes.size(3)},
                             slots.options().dtype(dtype));
    return {k, at::empty_like(k)};
}

at::Tensor decode_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                       const at::Tensor &, const at::Tensor &, int64_t, const at::Tensor &,
                       const at::Tensor &, double)
{
    return at::empty(q.sizes(), q.options());
}

std::tuple<at::Tensor, at::Tensor> verify_meta(const at::Tensor &probs, const at::Tensor &drafts,
                                               const OptTensor &, const OptTensor &, const at::Tensor &)
{
    return {at::empty({probs.size(0), probs.size(1)}, drafts.options()),
            at::empty({probs.size(0)}, drafts.options().dtype(at::kInt))};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(cbq, m)
{
    m.def("paged_append_q4(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor positions, "
          "Tensor slots, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, "
          "Tensor(d!) v_scales, bool norm, Tensor? q_weight, Tensor? k_weight, float eps) -> Tensor");
    m.def("paged_read_q4(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, "
          "Tensor slots, ScalarType dtype) -> (Tensor, Tensor)");
    m.def("prefix_attention_decode_q4(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, "
          "Tensor v_scales, Tensor prefix_table, int prefix, Tensor tables, Tensor lengths, "
          "float scale) -> Tensor");
    m.def("verify_drafts(Tensor probs, Tensor drafts, Tensor? draft_probs, Tensor? n_drafts, "
          "Tensor uniforms) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(cbq, CUDA, m)
{
    m.impl("paged_append_q4", &paged_append_q4);
    m.impl("paged_read_q4", &paged_read_q4);
    m.impl("prefix_attention_decode_q4", &prefix_attention_decode_q4);
    m.impl("verify_drafts", &verify_drafts);
}

TORCH_LIBRARY_IMPL(cbq, Meta, m)
{
    m.impl("paged_append_q4", &append_meta);
    m.impl("paged_read_q4", &read_meta);
    m.impl("prefix_attention_decode_q4", &decode_meta);
    m.impl("verify_drafts", &verify_meta);
}
