// New tokens into a paged key/value cache (include/cbq_serve.h): head norm and
// rotation of queries and keys, keys and values into their pages, one launch.
//
// A head's row x of hd values becomes, with r = rsqrt(mean(x^2) + eps) (or 1)
// and the angle t_d of its position, for d < rot/2:
//   y[d]         = x[d] r w[d] cos t_d - x[d + rot/2] r w[d + rot/2] sin t_d
//   y[d + rot/2] = x[d + rot/2] r w[d + rot/2] cos t_d + x[d] r w[d] sin t_d
// and y[d] = x[d] r w[d] from rot on.  Everything is read once and written
// once, so HBM bounds it; one token is bound by the launch.
//
// A thread holds both members of its pairs: 8 values from the row's rotated
// half and the 8 that they turn with (two 16-byte loads of 16-bit types), so
// hd / 16 neighbouring threads hold a row, read and write it in contiguous
// 128-byte pieces at hd = 128, and add its squares by shuffles.
#include "cbq_device.h"
#include "cbq_paged.h"
#include "../../include/cbq_serve.h"

namespace {

constexpr int64_t kFourThreads = 4 * 256 * 4 * 64;    // four waves a SIMD of 256 CUs

struct AppendArgs {
    const void *q, *k, *v;
    int64_t q_st[2], k_st[2], v_st[2];
    const float *cos_t, *sin_t, *q_w, *k_w;
    const int64_t *positions, *slots;
    void *q_out;
    cbq_paged_kv cache;
    int64_t n_pos, n_slots;
    CbqDiv heads, page;                 // thread groups a token; rows of a page
    uint32_t rows;                      // N (n_q + 2 n_kv)
    int n_q, n_kv, hd, rot, norm;
    float eps;
};

template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T e[V];
};

template <typename T, int V> __device__ __forceinline__ void load_vec(const T *p, float (&x)[V])
{
    const Pack<T, V> a = *(const Pack<T, V> *)p;
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = (float)a.e[i];
}

template <typename T, int V> __device__ __forceinline__ void store_vec(T *p, const float (&x)[V])
{
    Pack<T, V> a;
#pragma unroll
    for (int i = 0; i < V; i++) a.e[i] = (T)x[i];
    *(Pack<T, V> *)p = a;
}

// V values a side; U pairs of sides a thread; L lanes a row; R neighbouring heads
// of one token a thread, all of them queries, keys or values, which share what
// the thread reads of the tables and weights.
template <typename TX, typename TC, int V, int U, int L, int R>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    const uint32_t unit = cbq_block(blockIdx.x, blockIdx.y) * (256u / L) + threadIdx.x / L;
    const int lane = threadIdx.x % L;
    if (unit >= a.rows / R) return;                     // whole rows: no lane waits on a left one
    const int64_t t = cbq_div(unit, a.heads);           // heads: groups of R of a token
    const int i = (int)(unit - (uint32_t)t * a.heads.d) * R;
    const bool is_q = i < a.n_q, is_k = !is_q && i < a.n_q + a.n_kv;
    const int j = is_q ? i : is_k ? i - a.n_q : i - a.n_q - a.n_kv;
    const int64_t *st = is_q ? a.q_st : is_k ? a.k_st : a.v_st;
    const TX *x = (const TX *)(is_q ? a.q : is_k ? a.k : a.v) + t * st[0] + j * st[1];
    const int64_t p = a.positions[t], slot = a.slots[t];
    const int half = a.rot / 2, units = a.hd / (2 * V), turned = half / V;
    float lo[R][U][V], hi[R][U][V];
    int at_lo[U], at_hi[U];
#pragma unroll
    for (int n = 0; n < U; n++) {
        const int u = lane + n * L, w = u - turned;
        at_lo[n] = u < turned ? u * V : a.rot + 2 * w * V;
        at_hi[n] = u < turned ? u * V + half : at_lo[n] + V;
        if (u < units) {
#pragma unroll
            for (int h = 0; h < R; h++) {
                load_vec<TX, V>(x + h * st[1] + at_lo[n], lo[h][n]);
                load_vec<TX, V>(x + h * st[1] + at_hi[n], hi[h][n]);
            }
        }
    }
    const bool placed = p >= 0 && p < a.n_pos;
    TC *y;
    int64_t y_step;                                     // to the next head
    if (is_q) {
        y = (TC *)a.q_out + (t * a.n_q + j) * a.hd;
        y_step = a.hd;
    } else {
        if (!placed || slot < 0 || slot >= a.n_slots) return;       // uniform over the row's lanes
        const uint32_t id = cbq_div((uint32_t)slot, a.page);
        const int64_t r = (int64_t)((uint32_t)slot - id * a.page.d);
        const int64_t *ps = is_k ? a.cache.k_stride : a.cache.v_stride;
        y = (TC *)(is_k ? a.cache.k : a.cache.v) + id * ps[0] + j * ps[1] + r * ps[2];
        y_step = ps[1];
    }
    if (is_q || is_k) {
        if (a.norm) {
            const float *w = is_q ? a.q_w : a.k_w;
            float r[R];
#pragma unroll
            for (int h = 0; h < R; h++) {
                float s = 0.f;
#pragma unroll
                for (int n = 0; n < U; n++)
                    if (lane + n * L < units)
#pragma unroll
                        for (int e = 0; e < V; e++)
                            s += lo[h][n][e] * lo[h][n][e] + hi[h][n][e] * hi[h][n][e];
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, L);
                r[h] = 1.0f / sqrtf(s / (float)a.hd + a.eps);
            }
#pragma unroll
            for (int n = 0; n < U; n++)
                if (lane + n * L < units)
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const float wl = w ? w[at_lo[n] + e] : 1.0f, wh = w ? w[at_hi[n] + e] : 1.0f;
#pragma unroll
                        for (int h = 0; h < R; h++) {
                            lo[h][n][e] *= r[h] * wl;
                            hi[h][n][e] *= r[h] * wh;
                        }
                    }
        }
        const int64_t angle = (placed ? p : 0) * a.rot;
#pragma unroll
        for (int n = 0; n < U; n++)
            if (lane + n * L < turned) {
                float c[V], s[V];
                load_vec<float, V>(a.cos_t + angle + at_lo[n], c);
                load_vec<float, V>(a.sin_t + angle + at_lo[n], s);
#pragma unroll
                for (int h = 0; h < R; h++)
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const float b = lo[h][n][e], d = hi[h][n][e];
                        lo[h][n][e] = b * c[e] - d * s[e];
                        hi[h][n][e] = d * c[e] + b * s[e];
                    }
            }
    }
#pragma unroll
    for (int n = 0; n < U; n++)
        if (lane + n * L < units) {
#pragma unroll
            for (int h = 0; h < R; h++) {
                store_vec<TC, V>(y + h * y_step + at_lo[n], lo[h][n]);
                store_vec<TC, V>(y + h * y_step + at_hi[n], hi[h][n]);
            }
        }
}

template <typename TX, typename TC, int V, int U, int L>
void launch_rows(AppendArgs &a, hipStream_t stream)
{
    // Four heads a thread where four waves a SIMD are left: 8 KiB of tables and
    // weights a token instead of 32 (12500 bf16 tokens, 48 heads of 128: 98 -> 65
    // us, 4.7 TB/s, a copy's rate; 900 tokens: 7.0 us with one head, 8.0 with four).
    const bool four = V > 1 && a.n_q % 4 == 0 && a.n_kv % 4 == 0 &&
                      (int64_t)a.rows * L / 4 >= kFourThreads;
    const int R = four ? 4 : 1;
    a.heads = cbq_div_make((uint32_t)(a.n_q + 2 * a.n_kv) / R);
    const CbqGrid grid = cbq_grid(cbq_ceil(a.rows / R, 256 / L));
    const dim3 blocks(grid.x, grid.y), threads(256);
    if (four) paged_append_kernel<TX, TC, V, U, L, V == 1 ? 1 : 4><<<blocks, threads, 0, stream>>>(a);
    else paged_append_kernel<TX, TC, V, U, L, 1><<<blocks, threads, 0, stream>>>(a);
}

template <typename TX, typename TC> int launch(AppendArgs &a, bool wide, hipStream_t stream)
{
    // 16-byte pieces where hd is one of the decoders' and every address allows
    // it; else one value at a time, a wave a row (128 pairs at most).
    if (wide && a.hd == 64) launch_rows<TX, TC, 8, 1, 4>(a, stream);
    else if (wide && a.hd == 128) launch_rows<TX, TC, 8, 1, 8>(a, stream);
    else if (wide && a.hd == 256) launch_rows<TX, TC, 8, 1, 16>(a, stream);
    else launch_rows<TX, TC, 1, 2, 64>(a, stream);
    return cbq_launch_status("cbq_paged_append");
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int cbq_paged_append(const void *q, const void *k, const void *v, int x_dtype,
                                const int64_t *q_stride, const int64_t *k_stride,
                                const int64_t *v_stride, const float *cos_table,
                                const float *sin_table, int64_t n_pos, int rot,
                                const int64_t *positions, const int64_t *slots, int norm,
                                const float *q_weight, const float *k_weight, float eps,
                                void *q_out, const cbq_paged_kv *cache, int64_t N, int n_q,
                                hipStream_t stream)
{
    if (!q || !k || !v || !q_stride || !k_stride || !v_stride || !cos_table || !sin_table ||
        !positions || !slots || !q_out || !cache || !cache->k || !cache->v)
        return CK_ERR_ARG;
    const int hd = cache->hd, n_kv = cache->n_kv, c_dtype = cache->dtype;
    if (x_dtype < CBQ_F32 || x_dtype > CBQ_F16 || c_dtype < CBQ_F32 || c_dtype > CBQ_F16 ||
        (x_dtype != CBQ_F32 && c_dtype != x_dtype))
        return CK_ERR_ARG;
    if (N < 0 || n_q < 1 || n_kv < 1 || hd < 2 || hd > 256 || hd % 2 || rot < 2 || rot > hd ||
        rot % 2 || n_pos < 1 || cache->n_pages < 1 || cache->page < 1 || cache->page > 65536 ||
        cache->n_pages >= (1ll << 31) || cache->n_pages * cache->page >= (1ll << 31))
        return CK_ERR_ARG;
    // N bounded first, so that the products below stay within 64 bits
    const int64_t heads = (int64_t)n_q + 2ll * n_kv;
    if (N >= (1ll << 31) || heads >= (1ll << 31) || N * heads >= (1ll << 31)) return CK_ERR_ARG;
    if (N == 0) return CK_SUCCESS;
    AppendArgs a;
    a.q = q; a.k = k; a.v = v;
    const int64_t e = x_dtype == CBQ_F32 ? 4 : 2, ec = c_dtype == CBQ_F32 ? 4 : 2;
    bool wide = aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                aligned16(cache->k) && aligned16(cache->v) && aligned16(cos_table) &&
                aligned16(sin_table) && rot % 16 == 0;
    for (int i = 0; i < 2; i++) {
        a.q_st[i] = q_stride[i];
        a.k_st[i] = k_stride[i];
        a.v_st[i] = v_stride[i];
        wide = wide && q_stride[i] * e % 16 == 0 && k_stride[i] * e % 16 == 0 &&
               v_stride[i] * e % 16 == 0;
    }
    for (int i = 0; i < 3; i++)
        wide = wide && cache->k_stride[i] * ec % 16 == 0 && cache->v_stride[i] * ec % 16 == 0;
    a.cos_t = cos_table; a.sin_t = sin_table; a.q_w = q_weight; a.k_w = k_weight;
    a.positions = positions; a.slots = slots; a.q_out = q_out;
    a.cache = *cache;
    a.n_pos = n_pos;
    a.n_slots = cache->n_pages * cache->page;
    a.page = cbq_div_make((uint32_t)cache->page);
    a.rows = (uint32_t)(N * heads);
    a.n_q = n_q; a.n_kv = n_kv; a.hd = hd; a.rot = rot; a.norm = norm;
    a.eps = eps;
    if (x_dtype == CBQ_BF16) return launch<__bf16, __bf16>(a, wide, stream);
    if (x_dtype == CBQ_F16) return launch<_Float16, _Float16>(a, wide, stream);
    if (c_dtype == CBQ_BF16) return launch<float, __bf16>(a, wide, stream);
    if (c_dtype == CBQ_F16) return launch<float, _Float16>(a, wide, stream);
    return launch<float, float>(a, wide, stream);
}
