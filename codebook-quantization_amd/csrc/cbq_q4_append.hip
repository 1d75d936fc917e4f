// New tokens into the 4-bit paged cache, and its rows as values
// (include/cbq_serve_q4.h).
//
// Append.  A head's row x becomes y as in paged_append (norm, rotation), and a key's
// or value's y, 64 values a group, a scale, a mid and codes.  The codes are steps:
// a sum in another order, or a rounding on the way, would move a value next to a
// border to the next code.  So keys are normed, turned and cut in 64 bits, whose
// rate here is fp32's, and the quotient (y - m) / s, which only a true division
// places right at a border, is estimated by a reciprocal and settled by its exact
// remainder.  Queries go in fp32.
//
// Sixteen lanes hold a row, four neighbouring values of each group a lane, which are
// neighbours in the row's codes too; a group's range takes four exchanges.  The values
// that a rotation pairs with a lane's are read as well (cache hits).
#include "cbq_q4.h"

namespace {

using namespace cbq_q4;

constexpr int kThreads = 256;
constexpr int kLanes = 16, kRows = kThreads / kLanes;    // lanes a row, rows a block

struct AppendArgs {
    const void *x[3];                       // queries, keys, values
    int64_t st[3][2];
    const float *cos_t, *sin_t, *w[2];
    const int64_t *positions, *slots;
    void *q_out;
    Pool pool;
    int64_t n_pos, n_slots, rows[3];
    uint32_t first[3];                      // first block of each
    CbqDiv heads[3];
    int rot, norm;
    float eps;
};

template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T e[V];
};

// 4 values, as A
template <typename T, typename A, bool VEC>
__device__ __forceinline__ void load4(const T *p, A (&x)[4])
{
    if constexpr (VEC) {
        const Pack<T, 4> a = *(const Pack<T, 4> *)p;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (A)(float)a.e[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (A)(float)p[i];
    }
}

// A lane's values of a row, [group][4] from d0 on, normed and turned.  VEC: aligned
// fours, and rot / 2 in whole fours, so that all of one turn alike.
template <typename T, typename A, int HD, bool VEC>
__device__ __forceinline__ void turned(const AppendArgs &a, const T *x, const float *w, int64_t pos,
                                       int d0, A (&y)[HD / kGroup][4])
{
    constexpr int G = HD / kGroup;
#pragma unroll
    for (int g = 0; g < G; g++) load4<T, A, VEC>(x + g * kGroup + d0, y[g]);
    A r = (A)1;
    if (a.norm) {
        A s = (A)0;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) s += y[g][i] * y[g][i];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, kLanes);
        r = (A)1 / sqrt(s / (A)HD + (A)a.eps);
    }
    const bool scaled = a.norm && w;
    const int half = a.rot / 2;
    const float *ct = a.cos_t + pos * a.rot, *st = a.sin_t + pos * a.rot;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int d = g * kGroup + d0;
        A wt[4] = {r, r, r, r};
        if (scaled) {
            load4<float, A, VEC>(w + d, wt);
#pragma unroll
            for (int i = 0; i < 4; i++) wt[i] *= r;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) y[g][i] *= wt[i];
        if constexpr (VEC) {
            if (d >= a.rot) continue;
            const int at = d < half ? d : d - half, from = d < half ? d + half : d - half;
            A c[4], s[4], other[4], ow[4] = {r, r, r, r};
            load4<float, A, true>(ct + at, c);
            load4<float, A, true>(st + at, s);
            load4<T, A, true>(x + from, other);
            if (scaled) {
                load4<float, A, true>(w + from, ow);
#pragma unroll
                for (int i = 0; i < 4; i++) ow[i] *= r;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const A o = other[i] * ow[i];
                y[g][i] = d < half ? y[g][i] * c[i] - o * s[i] : y[g][i] * c[i] + o * s[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = d + i;
                if (e >= a.rot) continue;
                const int at = e < half ? e : e - half, from = e < half ? e + half : e - half;
                const A o = (A)(float)x[from] * (scaled ? r * (A)w[from] : r);
                const A cs = (A)ct[at], sn = (A)st[at];
                y[g][i] = e < half ? y[g][i] * cs - o * sn : y[g][i] * cs + o * sn;
            }
        }
    }
}

// A group's pair and this lane's four codes of it
__device__ __forceinline__ void quantise(const double (&y)[4], uint32_t &pair, uint32_t &codes)
{
    double top = y[0], low = y[0], odd = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        top = fmax(top, y[i]);
        low = fmin(low, y[i]);
        odd += y[i] - y[i];                 // NaN once a value is not finite
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) {
        top = fmax(top, __shfl_xor(top, o));
        low = fmin(low, __shfl_xor(low, o));
        odd += __shfl_xor(odd, o);
    }
    const __bf16 mb = (__bf16)(float)((top + low) / 2);
    const double m = (double)(float)mb;
    const __bf16 sb = (__bf16)(float)(fmax(top - m, m - low) / 7.5);
    const double s = (double)(float)sb;
    const uint32_t mid = __builtin_bit_cast(uint16_t, mb), scale = __builtin_bit_cast(uint16_t, sb);
    codes = 0x8888u;
    if (!(odd == 0) || (mid & 0x7f80) == 0x7f80 || (scale & 0x7f80) == 0x7f80) {
        pair = 0x7fc00000u;
        return;
    }
    pair = scale | mid << 16;
    if (!(s > 0)) return;
    const double inv = 1 / s;
    codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double d = y[i] - m;
        double n = floor(d * inv);
        const double left = fma(-n, s, d);  // exact: n has four bits, s eight
        n += left < 0 ? -1 : left >= s ? 1 : 0;
        const int c = (int)fmin(fmax(n, -8.0), 7.0) + 8;
        codes |= (uint32_t)c << (4 * i);
    }
}

template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a)
{
    constexpr int G = HD / kGroup;
    const uint32_t block = cbq_block(blockIdx.x, blockIdx.y);
    const int kind = block >= a.first[2] ? 2 : block >= a.first[1] ? 1 : 0;
    const int64_t row = (int64_t)(block - a.first[kind]) * kRows + threadIdx.x / kLanes;
    if (row >= a.rows[kind]) return;        // whole rows: no lane waits on a left one
    const uint32_t t = cbq_div((uint32_t)row, a.heads[kind]), j = (uint32_t)row - t * a.heads[kind].d;
    const int lane = threadIdx.x % kLanes, d0 = 4 * lane;
    const T *x = (const T *)a.x[kind] + t * a.st[kind][0] + j * a.st[kind][1];
    const int64_t p = a.positions[t];
    const bool placed = p >= 0 && p < a.n_pos;
    if (kind == 0) {
        float y[G][4];
        turned<T, float, HD, VEC>(a, x, a.w[0], placed ? p : 0, d0, y);
        T *out = (T *)a.q_out + row * HD + d0;
#pragma unroll
        for (int g = 0; g < G; g++) {
            Pack<T, 4> o;
#pragma unroll
            for (int e = 0; e < 4; e++) o.e[e] = (T)y[g][e];
            *(Pack<T, 4> *)(out + g * kGroup) = o;
        }
        return;
    }
    const int64_t slot = a.slots[t];
    if (!placed || slot < 0 || slot >= a.n_slots) return;       // uniform over the row's lanes
    double y[G][4];
    if (kind == 1) {
        turned<T, double, HD, VEC>(a, x, a.w[1], p, d0, y);
    } else {
#pragma unroll
        for (int g = 0; g < G; g++) load4<T, double, VEC>(x + g * kGroup + d0, y[g]);
    }
    Pack<uint16_t, G> codes;
    uint32_t pair[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        uint32_t c;
        quantise(y[g], pair[g], c);
        codes.e[g] = (uint16_t)c;
    }
    const uint32_t id = cbq_div((uint32_t)slot, a.pool.page), r = (uint32_t)slot - id * a.pool.page.d;
    const uint32_t at = code_at(a.pool, id, r) + j * a.pool.code_st[1];
    *(Pack<uint16_t, G> *)(a.pool.codes[kind - 1] + (uint64_t)at * kCodeUnit + lane * 2 * G) = codes;
    uint32_t *to = a.pool.pairs[kind - 1] + (uint64_t)(pair_at(a.pool, id, r) + j * a.pool.pair_st[1]);
#pragma unroll
    for (int g = 0; g < G; g++)
        if (lane == g) to[g] = pair[g];
}

template <typename T, int HD> int launch_append(AppendArgs &a, bool vec, hipStream_t stream)
{
    int64_t blocks = 0;
    for (int i = 0; i < 3; i++) {
        a.first[i] = (uint32_t)blocks;
        blocks += cbq_ceil(a.rows[i], kRows);
    }
    const CbqGrid grid = cbq_grid(blocks);
    if (vec) append_kernel<T, HD, true><<<dim3(grid.x, grid.y), kThreads, 0, stream>>>(a);
    else append_kernel<T, HD, false><<<dim3(grid.x, grid.y), kThreads, 0, stream>>>(a);
    return cbq_launch_status("cbq_paged_append_q4");
}

template <typename T> int launch_append_hd(AppendArgs &a, int hd, bool vec, hipStream_t stream)
{
    if (hd == 64) return launch_append<T, 64>(a, vec, stream);
    if (hd == 128) return launch_append<T, 128>(a, vec, stream);
    return launch_append<T, 256>(a, vec, stream);
}

// ---- rows as values --------------------------------------------------------------------------
struct ReadArgs {
    Pool pool;
    const int64_t *slots;
    void *out[2];
    int64_t rows, n_slots;                  // rows (token, kv head) of either output
    uint32_t n_kv;
};

template <typename T, int HD> __global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a)
{
    constexpr int G = HD / kGroup;
    const int64_t at = (int64_t)cbq_block(blockIdx.x, blockIdx.y) * kRows + threadIdx.x / kLanes;
    if (at >= 2 * a.rows) return;
    const int kind = at >= a.rows, lane = threadIdx.x % kLanes;
    const int64_t row = at - (kind ? a.rows : 0), t = row / a.n_kv;
    const uint32_t h = (uint32_t)(row - t * a.n_kv);
    const int64_t slot = a.slots[t];
    T *out = (T *)a.out[kind] + row * HD + 4 * lane;
    Pack<uint16_t, G> codes = {};
    uint32_t pair[G] = {};
    if (slot >= 0 && slot < a.n_slots) {
        const uint32_t id = cbq_div((uint32_t)slot, a.pool.page), r = (uint32_t)slot - id * a.pool.page.d;
        const uint32_t c = code_at(a.pool, id, r) + h * a.pool.code_st[1];
        codes = *(const Pack<uint16_t, G> *)(a.pool.codes[kind] + (uint64_t)c * kCodeUnit + lane * 2 * G);
        const uint32_t *from = a.pool.pairs[kind] + (uint64_t)(pair_at(a.pool, id, r) + h * a.pool.pair_st[1]);
#pragma unroll
        for (int g = 0; g < G; g++) pair[g] = from[g];
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
        Pack<T, 4> o;
#pragma unroll
        for (int i = 0; i < 4; i++)         // s (c - 7.5) is exact: one rounding in fp32
            o.e[i] = (T)fmaf(pair_scale(pair[g]), (float)(codes.e[g] >> (4 * i) & 15) - 7.5f, pair_mid(pair[g]));
        *(Pack<T, 4> *)(out + g * kGroup) = o;
    }
}

template <typename T> int launch_read(const ReadArgs &a, int hd, hipStream_t stream)
{
    const CbqGrid grid = cbq_grid(cbq_ceil(2 * a.rows, kRows));
    const dim3 blocks(grid.x, grid.y);
    if (hd == 64) read_kernel<T, 64><<<blocks, kThreads, 0, stream>>>(a);
    else if (hd == 128) read_kernel<T, 128><<<blocks, kThreads, 0, stream>>>(a);
    else read_kernel<T, 256><<<blocks, kThreads, 0, stream>>>(a);
    return cbq_launch_status("cbq_paged_read_q4");
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int cbq_paged_append_q4(const void *q, const void *k, const void *v, int x_dtype,
                                   const int64_t *q_stride, const int64_t *k_stride,
                                   const int64_t *v_stride, const float *cos_table,
                                   const float *sin_table, int64_t n_pos, int rot,
                                   const int64_t *positions, const int64_t *slots, int norm,
                                   const float *q_weight, const float *k_weight, float eps,
                                   void *q_out, const cbq_paged_q4 *cache, int64_t N, int n_q,
                                   hipStream_t stream)
{
    if (!pool_ok(cache) || x_dtype < CBQ_F32 || x_dtype > CBQ_F16) return CK_ERR_ARG;
    if (N < 0 || N >= (1ll << 31) || n_q < 1 || rot < 2 || rot > cache->hd || rot % 2 || n_pos < 1)
        return CK_ERR_ARG;
    const int64_t heads = (int64_t)n_q + 2ll * cache->n_kv;
    if (heads >= (1ll << 31) || N * heads >= (1ll << 31)) return CK_ERR_ARG;
    if (N == 0) return CK_SUCCESS;
    if (!q || !k || !v || !q_stride || !k_stride || !v_stride || !cos_table || !sin_table ||
        !positions || !slots || !q_out || !aligned16(q_out) || (norm && !(eps >= 0.f && eps <= 3.0e38f)))
        return CK_ERR_ARG;
    AppendArgs a;
    const void *x[3] = {q, k, v};
    const int64_t *st[3] = {q_stride, k_stride, v_stride};
    const int64_t e = x_dtype == CBQ_F32 ? 4 : 2;
    // four values at once where every address allows it, else one at a time
    bool vec = aligned16(cos_table) && aligned16(sin_table) && aligned16(q_weight) &&
               aligned16(k_weight) && rot % 8 == 0;
    for (int i = 0; i < 3; i++) {
        a.x[i] = x[i];
        a.st[i][0] = st[i][0];
        a.st[i][1] = st[i][1];
        vec = vec && (uintptr_t)x[i] % (4 * e) == 0 && st[i][0] % 4 == 0 && st[i][1] % 4 == 0;
        const int n = i == 0 ? n_q : cache->n_kv;
        a.heads[i] = cbq_div_make((uint32_t)n);
        a.rows[i] = N * n;
    }
    a.cos_t = cos_table; a.sin_t = sin_table; a.w[0] = q_weight; a.w[1] = k_weight;
    a.positions = positions; a.slots = slots; a.q_out = q_out;
    a.pool = make_pool(*cache);
    a.n_pos = n_pos;
    a.n_slots = cache->n_pages * cache->page;
    a.rot = rot; a.norm = norm; a.eps = eps;
    if (x_dtype == CBQ_F32) return launch_append_hd<float>(a, cache->hd, vec, stream);
    if (x_dtype == CBQ_BF16) return launch_append_hd<__bf16>(a, cache->hd, vec, stream);
    return launch_append_hd<_Float16>(a, cache->hd, vec, stream);
}

extern "C" int cbq_paged_read_q4(const cbq_paged_q4 *cache, const int64_t *slots, int64_t N, int dtype,
                                 void *k_out, void *v_out, hipStream_t stream)
{
    if (!pool_ok(cache) || dtype < CBQ_F32 || dtype > CBQ_F16 || N < 0 || N >= (1ll << 39) ||
        (double)N * cache->n_kv * cache->hd >= 549755813888.0)
        return CK_ERR_ARG;
    if (N == 0) return CK_SUCCESS;
    if (!slots || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) return CK_ERR_ARG;
    ReadArgs a;
    a.pool = make_pool(*cache);
    a.slots = slots;
    a.out[0] = k_out;
    a.out[1] = v_out;
    a.rows = N * cache->n_kv;
    a.n_slots = cache->n_pages * cache->page;
    a.n_kv = (uint32_t)cache->n_kv;
    if (dtype == CBQ_F32) return launch_read<float>(a, cache->hd, stream);
    if (dtype == CBQ_BF16) return launch_read<__bf16>(a, cache->hd, stream);
    return launch_read<_Float16>(a, cache->hd, stream);
}
