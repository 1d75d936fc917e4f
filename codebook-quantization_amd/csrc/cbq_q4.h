// The 4-bit paged cache (include/cbq_serve_q4.h): checks of a pool's description
// and the format's arithmetic, shared by its kernels.
#pragma once

#include "cbq_device.h"
#include "cbq_paged.h"
#include "../../include/cbq_serve_q4.h"

namespace cbq_q4 {

constexpr int kGroup = CBQ_Q4_GROUP;

// Offsets count in 16 bytes (codes) and 4 bytes (pairs), so that one 32-bit number
// holds any: 64 and 16 GiB.
constexpr int kCodeUnit = 16, kPairUnit = 4;

static inline bool pool_ok(const cbq_paged_q4 *c)
{
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales ||
        (c->hd != 64 && c->hd != 128 && c->hd != 256) || c->n_kv < 1 || c->page < 1 ||
        c->page > 65536 || c->n_pages < 1 || c->n_pages >= (1ll << 31) ||
        c->n_pages * c->page >= (1ll << 31))
        return false;
    if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & (kCodeUnit - 1) ||
        ((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & (kPairUnit - 1))
        return false;
    const double size[3] = {(double)c->n_pages, (double)c->n_kv, (double)c->page};
    double codes = 0, scales = 0;
    for (int i = 0; i < 3; i++) {
        const int64_t cs = c->code_stride[i], ss = c->scale_stride[i];
        if (cs < 0 || ss < 0 || cs % kCodeUnit || ss % 2 || cs >= (1ll << 40) || ss >= (1ll << 40))
            return false;
        codes += size[i] * (double)cs;
        scales += size[i] * (double)ss;
    }
    return codes < 4294967295.0 * kCodeUnit && scales < 4294967295.0 * kPairUnit / 2;
}

// A pool as the kernels take it: strides in units
struct Pool {
    char *codes[2];                         // keys, values
    uint32_t *pairs[2];
    uint32_t code_st[3], pair_st[3];
    int64_t n_pages;
    CbqDiv page;
};

static inline Pool make_pool(const cbq_paged_q4 &c)
{
    Pool p;
    p.codes[0] = (char *)c.k_codes;
    p.codes[1] = (char *)c.v_codes;
    p.pairs[0] = (uint32_t *)c.k_scales;
    p.pairs[1] = (uint32_t *)c.v_scales;
    for (int i = 0; i < 3; i++) {
        p.code_st[i] = (uint32_t)(c.code_stride[i] / kCodeUnit);
        p.pair_st[i] = (uint32_t)(c.scale_stride[i] * 2 / kPairUnit);
    }
    p.n_pages = c.n_pages;
    p.page = cbq_div_make((uint32_t)c.page);
    return p;
}

// Offsets of a row in units, of a page id and a row in it that are inside the pool
__device__ __forceinline__ uint32_t code_at(const Pool &p, uint32_t id, uint32_t row)
{
    return id * p.code_st[0] + row * p.code_st[2];
}
__device__ __forceinline__ uint32_t pair_at(const Pool &p, uint32_t id, uint32_t row)
{
    return id * p.pair_st[0] + row * p.pair_st[2];
}

__device__ __forceinline__ float pair_scale(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float pair_mid(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

}  // namespace cbq_q4
