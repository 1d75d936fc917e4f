// C entry points of the attention over a paged cache (include/cbq_serve.h):
// argument checks, launch plans, dispatch by type.
#include <cmath>
#include <initializer_list>

#include "cbq_prefix_attn.h"

using namespace cbq_attn;

namespace {

// Largest joint axis: a tile's or a look-ahead's indexes past it stay below 2^31.
constexpr int64_t kMaxKeys = (1ll << 31) - 65536;

int elem_bytes(int dtype) { return dtype == CBQ_F32 ? 4 : 2; }

bool sizes_ok(const cbq_paged_kv *c, int64_t prefix, int64_t width, int64_t batch, int64_t N,
              int64_t n_q)
{
    return c && c->dtype >= CBQ_F32 && c->dtype <= CBQ_F16 &&
           (c->hd == 64 || c->hd == 128 || c->hd == 256) && c->n_kv >= 1 && n_q >= 1 &&
           n_q < (1 << 20) && n_q % c->n_kv == 0 && c->page >= 1 && c->page <= 65536 &&
           c->n_pages >= 1 && c->n_pages < (1ll << 31) &&
           c->n_pages * c->page < (1ll << 31) && prefix >= 0 && prefix <= kMaxKeys && width >= 0 &&
           width * c->page <= kMaxKeys && prefix + width * c->page <= kMaxKeys && batch >= 0 &&
           batch < (1 << 30) && N >= 0 && N * n_q < (1ll << 31);
}

bool make_plan(const cbq_paged_kv *c, int64_t prefix, int64_t width, int64_t batch, int64_t N,
               int64_t n_q, bool prompt, Plan &p)
{
    const int row = c->hd * elem_bytes(c->dtype), rep = (int)(n_q / c->n_kv);
    p = prompt ? plan_prompt(row, c->hd, c->n_kv, rep, prefix, width * c->page, batch, N)
               : plan_decode(row, c->hd, c->n_kv, rep, prefix, width * c->page, batch);
    return plan_fits(p);
}

int attend(const void *q, const int64_t *q_stride, const int32_t *q_start,
           const cbq_paged_kv *cache, const int32_t *prefix_table, int64_t prefix,
           const int32_t *tables, int64_t table_stride, int width, const int32_t *lengths,
           int64_t batch, int64_t N, int64_t n_q, float scale, void *out, void *workspace,
           size_t workspace_bytes, bool prompt, hipStream_t stream)
{
    if (!sizes_ok(cache, prefix, width, batch, N, n_q)) return CK_ERR_ARG;
    if (N == 0) return CK_SUCCESS;
    if (!q || !q_stride || !cache->k || !cache->v || !out || !lengths ||
        (prefix > 0 && !prefix_table) || (width > 0 && !tables) || (prompt && !q_start) ||
        batch < 1 || !(scale >= -3.0e38f && scale <= 3.0e38f))
        return CK_ERR_ARG;
    const int64_t e = elem_bytes(cache->dtype);
    bool aligned = (((uintptr_t)q | (uintptr_t)cache->k | (uintptr_t)cache->v | (uintptr_t)out) &
                    15) == 0;
    for (int i = 0; i < 2; i++) aligned = aligned && q_stride[i] * e % 16 == 0;
    for (int i = 0; i < 3; i++)
        aligned = aligned && cache->k_stride[i] * e % 16 == 0 && cache->v_stride[i] * e % 16 == 0;
    if (!aligned) return CK_ERR_ARG;
    // rows as 32-bit offsets in the strides' common power of two: 512 GiB with
    // strides of whole 128 bytes
    uint64_t bits = 4096;
    for (int i = 0; i < 3; i += 2) bits |= (uint64_t)(cache->k_stride[i] * e | cache->v_stride[i] * e);
    const int64_t unit = (int64_t)(bits & (~bits + 1));
    for (const int64_t *st : {cache->k_stride, cache->v_stride})
        if (st[0] < 0 || st[2] < 0 || st[0] >= (1ll << 40) || st[2] >= (1ll << 40) ||
            ((double)cache->n_pages * (double)st[0] + (double)cache->page * (double)st[2]) * (double)e >=
                4294967295.0 * (double)unit)
            return CK_ERR_ARG;
    Plan p;
    if (!make_plan(cache, prefix, width, batch, N, n_q, prompt, p)) return CK_ERR_ARG;
    if (p.bytes && (!workspace || workspace_bytes < (size_t)p.bytes ||
                    ((uintptr_t)workspace & 15) != 0))
        return CK_ERR_ARG;
    AttnArgs a = {};
    a.q = q;
    a.q_st[0] = q_stride[0];
    a.q_st[1] = q_stride[1];
    a.kv = *cache;
    a.unit = (uint32_t)unit;
    a.k_page = (uint32_t)(cache->k_stride[0] * e / unit);
    a.k_row = (uint32_t)(cache->k_stride[2] * e / unit);
    a.v_page = (uint32_t)(cache->v_stride[0] * e / unit);
    a.v_row = (uint32_t)(cache->v_stride[2] * e / unit);
    a.one_stride = cache->k_stride[0] == cache->v_stride[0] &&
                   cache->k_stride[2] == cache->v_stride[2];
    a.prefix_table = prefix_table; a.tables = tables; a.lengths = lengths; a.q_start = q_start;
    a.table_st = table_stride;
    a.capacity = (int64_t)width * cache->page;
    a.out = out;
    a.part_o = (float *)workspace;
    a.part_ml = (float2 *)((float *)workspace + (p.parts > 1 ? p.parts * N * n_q * cache->hd : 0));
    a.page = cbq_div_make((uint32_t)cache->page);
    a.prefix = (int32_t)prefix; a.batch = (int32_t)batch; a.N = (int32_t)N;
    a.n_q = (int32_t)n_q; a.rep = (int32_t)(n_q / cache->n_kv);
    // The running maximum needs a factor above 0: the queries take scale's sign,
    // exactly, and a scale of 0 makes every score 0, as does one below fp32's smallest
    // step, 2^-149, whose scores of finite products are below 2^-20.
    // c below the exact factor and c_low above 0 (denormal numbers count: kernels are
    // built with them), so that a hidden key's -inf stays -inf times either.
    const float mag = scale < 0.f ? -scale : scale;
    const double exact = (double)mag * 1.4426950408889634074;
    a.c = (float)exact;
    if ((double)a.c >= exact) a.c = std::nextafter(a.c, 0.0f);
    a.c_low = std::fmax((float)(exact - (double)a.c), 0x1p-149f);
    const bool zero = !(a.c > 0.f);
    if (zero) a.c = 1.0f, a.c_low = 1.0e-9f;
    a.q_mul = zero ? 0.0f : scale < 0.f ? -1.0f : 1.0f;
    a.plan = p;
    if (cache->dtype == CBQ_F32) return launch_f32(a, p, prompt, stream);
    if (cache->dtype == CBQ_BF16) return launch_bf16(a, p, prompt, stream);
    return launch_f16(a, p, prompt, stream);
}

size_t workspace_of(const cbq_paged_kv *cache, int64_t prefix, int width, int64_t batch, int64_t N,
                    int64_t n_q, bool prompt)
{
    Plan p;
    if (!sizes_ok(cache, prefix, width, batch, N, n_q) || N == 0 || batch < 1 ||
        !make_plan(cache, prefix, width, batch, N, n_q, prompt, p))
        return 0;
    return (size_t)p.bytes;
}

}  // namespace

extern "C" size_t cbq_prefix_attn_decode_workspace(const cbq_paged_kv *cache, int64_t prefix,
                                                   int width, int batch, int n_q)
{
    return workspace_of(cache, prefix, width, batch, batch, n_q, false);
}

extern "C" int cbq_prefix_attn_decode(const void *q, const int64_t *q_stride,
                                      const cbq_paged_kv *cache, const int32_t *prefix_table,
                                      int64_t prefix, const int32_t *tables, int64_t table_stride,
                                      int width, const int32_t *lengths, int batch, int n_q,
                                      float scale, void *out, void *workspace,
                                      size_t workspace_bytes, hipStream_t stream)
{
    return attend(q, q_stride, nullptr, cache, prefix_table, prefix, tables, table_stride, width,
                  lengths, batch, batch, n_q, scale, out, workspace, workspace_bytes, false, stream);
}

extern "C" size_t cbq_prefix_attn_prompt_workspace(const cbq_paged_kv *cache, int64_t prefix,
                                                   int width, int batch, int64_t N, int n_q)
{
    return workspace_of(cache, prefix, width, batch, N, n_q, true);
}

extern "C" int cbq_prefix_attn_prompt(const void *q, const int64_t *q_stride,
                                      const int32_t *q_start, const cbq_paged_kv *cache,
                                      const int32_t *prefix_table, int64_t prefix,
                                      const int32_t *tables, int64_t table_stride, int width,
                                      const int32_t *lengths, int batch, int64_t N, int n_q,
                                      float scale, void *out, void *workspace,
                                      size_t workspace_bytes, hipStream_t stream)
{
    return attend(q, q_stride, q_start, cache, prefix_table, prefix, tables, table_stride, width,
                  lengths, batch, N, n_q, scale, out, workspace, workspace_bytes, true, stream);
}
