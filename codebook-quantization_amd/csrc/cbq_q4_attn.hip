// C entry points of the attention over the 4-bit paged cache
// (include/cbq_serve_q4.h): argument checks, launch plans, dispatch by type.
#include <cmath>

#include "cbq_q4_attn.h"

using namespace cbq_q4;

namespace {

// Largest joint axis and count of rows: a tile's indexes past either stay below 2^31.
constexpr int64_t kMaxKeys = (1ll << 31) - 65536;
// Entries of a table: their bytes are a 32-bit offset.
constexpr int64_t kMaxEntries = 1ll << 30;

bool sizes_ok(const cbq_paged_q4 *c, int64_t prefix, int64_t width, int64_t batch, int64_t tokens,
              int64_t n_q)
{
    return c && (c->hd == 64 || c->hd == 128 || c->hd == 256) && c->n_kv >= 1 && n_q >= 1 &&
           n_q < (1 << 20) && n_q % c->n_kv == 0 && c->page >= 1 && c->page <= 65536 &&
           prefix >= 0 && prefix <= kMaxKeys && width >= 0 && width * c->page <= kMaxKeys &&
           width < kMaxEntries && cbq_ceil(prefix, c->page) < kMaxEntries &&
           prefix + width * c->page <= kMaxKeys && batch >= 0 && batch < (1 << 30) && tokens >= 1 &&
           batch * tokens <= kMaxKeys && batch * tokens * n_q <= kMaxKeys;
}

bool make_plan(const cbq_paged_q4 *c, int dtype, int64_t prefix, int64_t width, int64_t batch,
               int64_t tokens, int64_t n_q, Plan &p)
{
    p = plan(c->hd, dtype == CBQ_BF16, c->n_kv, tokens * (n_q / c->n_kv), prefix, width * c->page, batch);
    return plan_fits(p);
}

}  // namespace

extern "C" size_t cbq_prefix_attn_decode_q4_workspace(const cbq_paged_q4 *cache, int64_t prefix,
                                                      int width, int batch, int tokens, int n_q,
                                                      int dtype)
{
    Plan p;
    if (!sizes_ok(cache, prefix, width, batch, tokens, n_q) || batch < 1 ||
        !make_plan(cache, dtype, prefix, width, batch, tokens, n_q, p))
        return 0;
    return (size_t)p.bytes;
}

extern "C" int cbq_prefix_attn_decode_q4(const void *q, const int64_t *q_stride, int dtype,
                                         const cbq_paged_q4 *cache, const int32_t *prefix_table,
                                         int64_t prefix, const int32_t *tables,
                                         int64_t table_stride, int width, const int32_t *lengths,
                                         int batch, int tokens, int n_q, float scale, void *out,
                                         void *workspace, size_t workspace_bytes,
                                         hipStream_t stream)
{
    if (!pool_ok(cache) || !sizes_ok(cache, prefix, width, batch, tokens, n_q) || dtype < CBQ_F32 ||
        dtype > CBQ_F16)
        return CK_ERR_ARG;
    if (batch == 0) return CK_SUCCESS;
    if (!q || !q_stride || !out || !lengths || (prefix > 0 && !prefix_table) ||
        (width > 0 && !tables) || !(scale >= -3.0e38f && scale <= 3.0e38f))
        return CK_ERR_ARG;
    const int64_t e = dtype == CBQ_F32 ? 4 : 2;
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || q_stride[0] * e % 16 || q_stride[1] * e % 16)
        return CK_ERR_ARG;
    AttnArgs a = {};
    if (!make_plan(cache, dtype, prefix, width, batch, tokens, n_q, a.plan)) return CK_ERR_ARG;
    if (a.plan.bytes && (!workspace || workspace_bytes < (size_t)a.plan.bytes ||
                         ((uintptr_t)workspace & 15) != 0))
        return CK_ERR_ARG;
    const int64_t rows = (int64_t)batch * tokens * n_q;
    a.q = q;
    a.q_st[0] = q_stride[0];
    a.q_st[1] = q_stride[1];
    a.pool = make_pool(*cache);
    a.prefix_table = prefix_table; a.tables = tables; a.lengths = lengths;
    a.table_st = table_stride;
    a.capacity = (int64_t)width * cache->page;
    a.out = out;
    a.part_o = (float *)workspace;
    a.part_ml = (float2 *)((float *)workspace + (a.plan.parts > 1 ? a.plan.parts * rows * cache->hd : 0));
    a.rep = cbq_div_make((uint32_t)(n_q / cache->n_kv));
    // pages of whole tiles, whose rows a 32-bit offset from the tile's first reaches
    a.whole = cache->page % kTile == 0 && cache->code_stride[2] < (1 << 24) && cache->scale_stride[2] < (1 << 24);
    a.tiles_a_page = cbq_div_make(a.whole ? (uint32_t)cache->page / kTile : 1);
    a.code_row = a.whole ? (uint32_t)cache->code_stride[2] : 0;
    a.pair_row = a.whole ? (uint32_t)cache->scale_stride[2] * 2 : 0;
    a.prefix = (int32_t)prefix; a.batch = batch; a.tokens = tokens; a.n_q = n_q;
    a.n_kv = cache->n_kv;
    // The running maximum needs a factor above 0: the queries take scale's sign,
    // exactly, and a scale of 0 makes every score 0, as does one below fp32's smallest
    // step, whose scores of finite products are below 2^-20.  c below the exact
    // factor and c_low above 0, so that a hidden key's -inf stays -inf times either.
    const float mag = scale < 0.f ? -scale : scale;
    const double exact = (double)mag * 1.4426950408889634074;
    a.c = (float)exact;
    if ((double)a.c >= exact) a.c = std::nextafter(a.c, 0.0f);
    a.c_low = std::fmax((float)(exact - (double)a.c), 0x1p-149f);
    const bool zero = !(a.c > 0.f);
    if (zero) a.c = 1.0f, a.c_low = 1.0e-9f;
    a.q_mul = zero ? 0.0f : scale < 0.f ? -1.0f : 1.0f;
    if (dtype == CBQ_F32) return launch_f32(a, cache->hd, stream);
    if (dtype == CBQ_BF16) return launch_bf16(a, cache->hd, stream);
    return launch_f16(a, cache->hd, stream);
}
