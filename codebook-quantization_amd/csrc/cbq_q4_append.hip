// New tokens into the 4-bit paged cache, and its rows as values
// (include/cbq_serve_q4.h).
//
// Append.  A head's row x becomes y as in paged_append (norm, rotation), and a key's
// or value's y, 64 values a group, a scale, a mid and codes.  The codes are steps:
// a sum in another order, or a rounding on the way, would move a value next to a
// border to the next code.  So keys are normed, turned and cut in 64 bits, whose
// rate here is fp32's, and a code is the nearest border by a fast quotient and one exact
// comparison with it.  Queries go in fp32, values stay in theirs.
//
// Sixteen lanes hold a row, four neighbouring values of each group a lane, which are
// neighbours in the row's codes too; a row's sum and a group's range take four
// exchanges among neighbours, by row rotations.  Where half the rotated part is whole
// groups, or half a group, the values that turn together are the lane's own, or those of
// the lane eight away; else the others' are read too (cache hits).  A thread has
// neighbouring heads of a token, all queries, keys or values, which share what is
// read of the tables and weights, and asks for all of them before it uses one.
//
// Bound by bytes where prompts are long: 12416 tokens of 32 + 8 + 8 heads of 128 in bf16,
// 268 MB, in 60 us, 4.5 TB/s where a copy of 1 GiB reaches 5.3.  (Heads asked for one by
// one and every code settled by the remainder of a 64-bit quotient: 98 us.)  By latency
// where few: one token takes 4 us.
#include "cbq_q4.h"

namespace {

using namespace cbq_q4;

constexpr int kThreads = 256;
// Four heads a thread where that leaves four waves a SIMD of 256 CUs, else one.  32 + 8 + 8
// heads of 128 in bf16, with their read, one and four: 100 tokens 6.2 and 8.4 us, 700 10.9 and
// 11.3, 3000 26.1 and 25.3, 12000 104 and 73.  Head counts that four does not divide have one:
// of 12000 tokens 14 + 2 + 2 heads go at 3.5 TB/s, 6 + 6 + 6 at 2.7 (12 + 4 + 4 and 8 + 8 + 8 by
// four at 3.6 and 3.2).
constexpr int64_t kFourThreads = 4 * 256 * 4 * 64;
constexpr int kLanes = 16, kRows = kThreads / kLanes;    // lanes a row, rows a block

struct AppendArgs {
    const void *x[3];                       // queries, keys, values
    int64_t st[3][2];
    const float *cos_t, *sin_t, *w[2];
    const int64_t *positions, *slots;
    void *q_out;
    Pool pool;
    int64_t N, n_pos, n_slots, units[3];    // units: of heads that a thread has, of each kind
    uint32_t first[3];                      // first block of each
    CbqDiv heads[3];                        // units a token
    int n_q, n_kv, rot, norm;
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

// A lane's values of a row as they lie in memory, [group][4] from d0 on
template <typename T, int HD, bool VEC> struct Row {
    Pack<T, 4> e[HD / kGroup];

    __device__ __forceinline__ void load(const T *x, int d0)
    {
#pragma unroll
        for (int g = 0; g < HD / kGroup; g++) {
            const T *from = x + g * kGroup + d0;
            if constexpr (VEC) e[g] = *(const Pack<T, 4> *)from;
            else
#pragma unroll
                for (int i = 0; i < 4; i++) e[g].e[i] = from[i];
        }
    }
};

// x of the lane `by` further on (cyclically) in its sixteen
template <int BY> __device__ __forceinline__ float rotated(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 | BY, 0xf, 0xf, true));
}
template <int BY> __device__ __forceinline__ double rotated(double x)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(x), 0x120 | BY, 0xf, 0xf, true),
                            __builtin_amdgcn_update_dpp(0, __double2loint(x), 0x120 | BY, 0xf, 0xf, true));
}
// f over the sixteen lanes of a row, in all of them
template <typename A, typename F> __device__ __forceinline__ A over_row(A x, F f)
{
    x = f(x, rotated<8>(x));
    x = f(x, rotated<4>(x));
    x = f(x, rotated<2>(x));
    return f(x, rotated<1>(x));
}

// How a lane's values meet those that they turn with
enum { kWhole1 = 1, kWhole2 = 2, kHalf = 0, kRead = -1, kSingle = -2 };
// kWholeN: half the rotated part is N groups, kHalf: half a group; kRead: whole fours,
// read; kSingle: one value at a time (any address, any even rot)

template <int HD, int MODE> struct Angles {
    static constexpr int kN = MODE > 0 ? MODE : MODE == kHalf ? 1 : HD / kGroup;   // tables' fours a lane
    float c[kN][4], s[kN][4];

    __device__ __forceinline__ void load(const AppendArgs &a, int64_t pos, int d0)
    {
        if constexpr (MODE == kSingle) return;
        const float *ct = a.cos_t + pos * a.rot, *st = a.sin_t + pos * a.rot;
        const int half = a.rot / 2;
#pragma unroll
        for (int g = 0; g < kN; g++) {
            int d = g * kGroup + d0;
            if (MODE == kHalf) d &= 31;
            if (MODE == kRead) d = d >= a.rot ? 0 : d < half ? d : d - half;
            load4<float, float, true>(ct + d, c[g]);
            load4<float, float, true>(st + d, s[g]);
        }
    }
};

// Its weights of a norm
template <int HD, bool VEC> struct Weights {
    float e[HD / kGroup][4];

    __device__ __forceinline__ void load(const float *w, int d0)
    {
#pragma unroll
        for (int g = 0; g < HD / kGroup; g++) load4<float, float, VEC>(w + g * kGroup + d0, e[g]);
    }
};

// 1 / sqrt(x): for a double two Newton steps behind an estimate of 20 bits at least; the
// steps make NaN of infinity's 0
__device__ __forceinline__ float inv_root(float x) { return 1.f / sqrtf(x); }
__device__ __forceinline__ double inv_root(double x)
{
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; i++) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
    return x == HUGE_VAL ? 0 : y;
}

// A lane's values of a row, normed and turned.  x, w: the row and the weights, for values
// that turn with those of neither this lane nor its neighbour.
template <typename T, typename A, int HD, int MODE>
__device__ __forceinline__ void turned(const AppendArgs &a, const Row<T, HD, (MODE != kSingle)> &row,
                                       const Weights<HD, (MODE != kSingle)> &weights, const T *x,
                                       const float *w, int64_t pos, int d0, const Angles<HD, MODE> &t,
                                       A (&y)[HD / kGroup][4])
{
    constexpr int G = HD / kGroup;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[g][i] = (A)(float)row.e[g].e[i];
    A r = (A)1;
    if (a.norm) {
        A s = (A)0;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) s += y[g][i] * y[g][i];
        s = over_row(s, [](A p, A q) { return p + q; });
        r = inv_root(s / (A)HD + (A)a.eps);
    }
    const bool scaled = a.norm && w;
#pragma unroll
    for (int g = 0; g < G; g++) {
        if (scaled)
#pragma unroll
            for (int i = 0; i < 4; i++) y[g][i] *= (A)weights.e[g][i];
        if (a.norm)
#pragma unroll
            for (int i = 0; i < 4; i++) y[g][i] *= r;
    }
    if constexpr (MODE > 0) {
#pragma unroll
        for (int g = 0; g < MODE; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const A lo = y[g][i], hi = y[g + MODE][i], c = (A)t.c[g][i], s = (A)t.s[g][i];
                y[g][i] = lo * c - hi * s;
                y[g + MODE][i] = hi * c + lo * s;
            }
    } else if constexpr (MODE == kHalf) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const A mine = y[0][i], o = rotated<8>(mine), c = (A)t.c[0][i], s = (A)t.s[0][i];
            y[0][i] = d0 < 32 ? mine * c - o * s : mine * c + o * s;
        }
    } else {
        const int half = a.rot / 2;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int d = g * kGroup + d0;
            if constexpr (MODE == kRead) {
                if (d >= a.rot) continue;
                const int from = d < half ? d + half : d - half;
                A other[4], ow[4] = {1, 1, 1, 1};
                load4<T, A, true>(x + from, other);
                if (scaled) load4<float, A, true>(w + from, ow);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const A o = other[i] * ow[i] * r, c = (A)t.c[g][i], s = (A)t.s[g][i];
                    y[g][i] = d < half ? y[g][i] * c - o * s : y[g][i] * c + o * s;
                }
            } else {
                const float *ct = a.cos_t + pos * a.rot, *st = a.sin_t + pos * a.rot;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = d + i;
                    if (e >= a.rot) continue;
                    const int at = e < half ? e : e - half, from = e < half ? e + half : e - half;
                    const A o = (A)(float)x[from] * (scaled ? (A)w[from] : (A)1) * r;
                    const A c = (A)ct[at], s = (A)st[at];
                    y[g][i] = e < half ? y[g][i] * c - o * s : y[g][i] * c + o * s;
                }
            }
        }
    }
}

// fp32 first, then bf16: the compiler makes one rounding of the two otherwise, which
// differs where the first ends halfway between two numbers of the second
__device__ __forceinline__ __bf16 twice_rounded(double x)
{
    float y = (float)x;
    asm("" : "+v"(y));
    return (__bf16)y;
}

// A group's scale and mid from its largest and smallest value
__device__ __forceinline__ void group_pair(double high, double deep, __bf16 &scale, __bf16 &mid)
{
    mid = twice_rounded((high + deep) / 2);
    const double m = (double)(float)mid;
    // 1 / 7.5: its last place is 2^-29 of the number it is rounded to first
    scale = twice_rounded(fmax(high - m, m - deep) * (1 / 7.5));
}

// A group's pair and this lane's four codes of it, for any values.  A: the type that
// holds y exactly.
template <typename A> __device__ __forceinline__ void quantise(const A (&y)[4], uint32_t &pair, uint32_t &codes)
{
    A top = y[0], low = y[0], odd = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        top = fmax(top, y[i]);
        low = fmin(low, y[i]);
        odd += y[i] - y[i];                 // NaN once a value is not finite
    }
    // the sixteen lanes' answers stand side by side in the wave's
    const uint64_t bad = __ballot(!(odd == 0));
    const bool sound = !(bad >> (threadIdx.x & 48) & 0xffff);
    __bf16 mb, sb;
    group_pair((double)over_row(top, [](A p, A q) { return fmax(p, q); }),
               (double)over_row(low, [](A p, A q) { return fmin(p, q); }), sb, mb);
    const double m = (double)(float)mb;
    const float s = (float)sb;
    const uint32_t mid = __builtin_bit_cast(uint16_t, mb), scale = __builtin_bit_cast(uint16_t, sb);
    codes = 0x8888u;
    pair = 0x7fc00000u;
    if (!sound || (mid & 0x7f80) == 0x7f80 || (scale & 0x7f80) == 0x7f80) return;
    pair = scale | mid << 16;
    if (!(s > 0)) return;
    const double step = (double)s;
    const double inv = ldexp((double)__builtin_amdgcn_rcpf(__builtin_amdgcn_frexp_mantf(s)),
                             -__builtin_amdgcn_frexp_expf(s));
    codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double d = (double)y[i] - m;
        const float n = floorf((float)(d * inv));           // off by one at most
        const double left = fma(-(double)n, step, d);       // exact: n has four bits, s eight
        const int c = (int)n + 8 + (left < 0 ? -1 : left >= step ? 1 : 0);
        codes |= (uint32_t)min(max(c, 0), 15) << (4 * i);
    }
}

// The same for ordinary groups, or false (for all lanes of the row): values finite and a
// scale that is an ordinary number, and then |y - m| < 7.6 s.  So k = rint((y - m) / s) is
// the nearest border whatever the estimate's roundings, and the code is k + 8, less one
// where y lies below m + k s.  With y of 32 bits the border has to be a number of 24 bits:
// m = 0 or exponents of s and m at most 12 apart (of values that scatter about one group
// in a thousand is not, and of 16-bit ones hardly any).  With y of 64 bits y - m - k s is exact.
__device__ __forceinline__ bool quick(const float (&y)[4], uint32_t &pair, uint32_t &codes)
{
    // the maximum that a NaN passes through
    auto most = [](float p, float q) { return __builtin_elementwise_maximum(p, q); };
    auto least = [](float p, float q) { return __builtin_elementwise_minimum(p, q); };
    const float top = most(most(most(y[0], y[1]), y[2]), y[3]), low = least(least(least(y[0], y[1]), y[2]), y[3]);
    __bf16 mb, sb;
    group_pair((double)over_row(top, most), (double)over_row(low, least), sb, mb);
    const uint32_t mid = __builtin_bit_cast(uint16_t, mb), scale = __builtin_bit_cast(uint16_t, sb);
    const int em = mid >> 7 & 255, es = scale >> 7 & 255;
    const bool easy = es - 2u <= 248u && ((mid & 0x7fff) == 0 || (em > 0 && em - es + 12u <= 24u));
    pair = scale | mid << 16;
    const float m = (float)mb, s = (float)sb, inv = __builtin_amdgcn_rcpf(s);
    constexpr float kWhole = 12582912.f + 8.f;      // the integer that is added to stands in the last bits
    codes = 0;
#pragma unroll
    for (int i = 3; i >= 0; i--) {
        const float u = fmaf(y[i] - m, inv, kWhole);
        codes = (codes << 4) + (__float_as_uint(u) - (y[i] < fmaf(u - kWhole, s, m)));
    }
    return easy;
}
__device__ __forceinline__ bool quick(const double (&y)[4], uint32_t &pair, uint32_t &codes)
{
    auto most = [](double p, double q) { return fmax(p, q); };
    auto least = [](double p, double q) { return fmin(p, q); };
    const double top = most(most(y[0], y[1]), most(y[2], y[3])), low = least(least(y[0], y[1]), least(y[2], y[3]));
    const double all = (y[0] + y[1]) + (y[2] + y[3]);
    const uint64_t bad = __ballot(!(fabs(all) < HUGE_VAL));
    __bf16 mb, sb;
    group_pair(over_row(top, most), over_row(low, least), sb, mb);
    const uint32_t mid = __builtin_bit_cast(uint16_t, mb), scale = __builtin_bit_cast(uint16_t, sb);
    const bool easy = (scale >> 7 & 255) - 2u <= 248u && (mid >> 7 & 255) < 255 && !(bad >> (threadIdx.x & 48) & 0xffff);
    pair = scale | mid << 16;
    const float s = (float)sb, inv = __builtin_amdgcn_rcpf(s);
    const double m = (double)(float)mb, step = (double)s;
    constexpr float kWhole = 12582912.f + 8.f;
    codes = 0;
#pragma unroll
    for (int i = 3; i >= 0; i--) {
        const double d = y[i] - m;
        const float u = fmaf((float)d, inv, kWhole);
        codes = (codes << 4) + (__float_as_uint(u) - (fma((double)(kWhole - u), step, d) < 0));
    }
    return easy;
}

template <typename T, int HD, int MODE, int R>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a)
{
    constexpr int G = HD / kGroup;
    constexpr bool kVec = MODE != kSingle;
    const uint32_t block = cbq_block(blockIdx.x, blockIdx.y);
    const int kind = block >= a.first[2] ? 2 : block >= a.first[1] ? 1 : 0;
    const int64_t unit = (int64_t)(block - a.first[kind]) * kRows + threadIdx.x / kLanes;
    if (unit >= a.units[kind]) return;      // whole rows: no lane waits on a left one
    const uint32_t t = cbq_div((uint32_t)unit, a.heads[kind]), j = ((uint32_t)unit - t * a.heads[kind].d) * R;
    const int lane = threadIdx.x % kLanes, d0 = 4 * lane;
    const int64_t st = a.st[kind][1];
    const T *x = (const T *)a.x[kind] + t * a.st[kind][0] + j * st;
    // everything is asked for before the first use
    Row<T, HD, kVec> rows[R];
#pragma unroll
    for (int h = 0; h < R; h++) rows[h].load(x + h * st, d0);
    const int64_t p = a.positions[t], slot = kind ? a.slots[t] : 0;
    const bool placed = p >= 0 && p < a.n_pos;
    Angles<HD, MODE> angles;
    Weights<HD, kVec> weights;
    const float *w = kind < 2 ? a.w[kind] : nullptr;
    if (a.norm && w) weights.load(w, d0);
    if (kind < 2) angles.load(a, placed ? p : 0, d0);
    if (kind == 0) {
        T *out = (T *)a.q_out + ((int64_t)t * a.n_q + j) * HD + d0;
#pragma unroll
        for (int h = 0; h < R; h++) {
            float y[G][4];
            turned<T, float, HD, MODE>(a, rows[h], weights, x + h * st, w, placed ? p : 0, d0, angles, y);
#pragma unroll
            for (int g = 0; g < G; g++) {
                Pack<T, 4> o;
#pragma unroll
                for (int e = 0; e < 4; e++) o.e[e] = (T)y[g][e];
                *(Pack<T, 4> *)(out + h * HD + g * kGroup) = o;
            }
        }
        return;
    }
    if (!placed || slot < 0 || slot >= a.n_slots) return;       // uniform over the row's lanes
    const uint32_t id = cbq_div((uint32_t)slot, a.pool.page), r = (uint32_t)slot - id * a.pool.page.d;
    const uint32_t code0 = code_at(a.pool, id, r) + j * a.pool.code_st[1],
                   pair0 = pair_at(a.pool, id, r) + j * a.pool.pair_st[1];
    auto store = [&](int h, const uint32_t (&pair)[G], const uint32_t (&c)[G]) {
        Pack<uint16_t, G> codes;
#pragma unroll
        for (int g = 0; g < G; g++) codes.e[g] = (uint16_t)c[g];
        *(Pack<uint16_t, G> *)(a.pool.codes[kind - 1] + (uint64_t)(code0 + h * a.pool.code_st[1]) * kCodeUnit +
                               lane * 2 * G) = codes;
        uint32_t *to = a.pool.pairs[kind - 1] + (uint64_t)(pair0 + h * a.pool.pair_st[1]);
#pragma unroll
        for (int g = 0; g < G; g++)
            if (lane == g) to[g] = pair[g];
    };
    uint32_t pair[G], c[G], odd = 0;        // odd: heads with a group that is no ordinary one
    if (kind == 1) {
#pragma unroll
        for (int h = 0; h < R; h++) {
            double y[G][4];
            turned<T, double, HD, MODE>(a, rows[h], weights, x + h * st, w, p, d0, angles, y);
            bool easy = true;
#pragma unroll
            for (int g = 0; g < G; g++) easy = quick(y[g], pair[g], c[g]) && easy;
            if (easy) store(h, pair, c);
            else odd |= 1u << h;
        }
        for (; odd; odd &= odd - 1) {
            const int h = __builtin_ctz(odd);
            double y[G][4];
            rows[0].load(x + h * st, d0);
            turned<T, double, HD, MODE>(a, rows[0], weights, x + h * st, w, p, d0, angles, y);
#pragma unroll
            for (int g = 0; g < G; g++) quantise(y[g], pair[g], c[g]);
            store(h, pair, c);
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < R; h++) {
        bool easy = true;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float y[4] = {(float)rows[h].e[g].e[0], (float)rows[h].e[g].e[1], (float)rows[h].e[g].e[2],
                                (float)rows[h].e[g].e[3]};
            easy = quick(y, pair[g], c[g]) && easy;
        }
        if (easy) store(h, pair, c);
        else odd |= 1u << h;
    }
    for (; odd; odd &= odd - 1) {
        const int h = __builtin_ctz(odd);
        rows[0].load(x + h * st, d0);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float y[4] = {(float)rows[0].e[g].e[0], (float)rows[0].e[g].e[1], (float)rows[0].e[g].e[2],
                                (float)rows[0].e[g].e[3]};
            quantise(y, pair[g], c[g]);
        }
        store(h, pair, c);
    }
}

template <typename T, int HD, int MODE, int R> int launch_units(AppendArgs &a, hipStream_t stream)
{
    int64_t blocks = 0;
    for (int i = 0; i < 3; i++) {
        const int n = (i == 0 ? a.n_q : a.n_kv) / R;
        a.heads[i] = cbq_div_make((uint32_t)n);
        a.units[i] = a.N * n;
        a.first[i] = (uint32_t)blocks;
        blocks += cbq_ceil(a.units[i], kRows);
    }
    const CbqGrid grid = cbq_grid(blocks);
    append_kernel<T, HD, MODE, R><<<dim3(grid.x, grid.y), kThreads, 0, stream>>>(a);
    return cbq_launch_status("cbq_paged_append_q4");
}

template <typename T, int HD, int MODE> int launch_mode(AppendArgs &a, hipStream_t stream)
{
    if constexpr (MODE != kSingle) {
        const bool four = a.n_q % 4 == 0 && a.n_kv % 4 == 0 && a.N * (a.n_q + 2ll * a.n_kv) * kLanes / 4 >= kFourThreads;
        if (four) return launch_units<T, HD, MODE, 4>(a, stream);
    }
    return launch_units<T, HD, MODE, 1>(a, stream);
}

template <typename T, int HD> int launch_append(AppendArgs &a, bool vec, hipStream_t stream)
{
    if (!vec) return launch_mode<T, HD, kSingle>(a, stream);
    if (a.rot == 64) return launch_mode<T, HD, kHalf>(a, stream);
    if constexpr (HD >= 128)
        if (a.rot == 128) return launch_mode<T, HD, kWhole1>(a, stream);
    if constexpr (HD == 256)
        if (a.rot == 256) return launch_mode<T, HD, kWhole2>(a, stream);
    return launch_mode<T, HD, kRead>(a, stream);
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

// Bound by its bytes: 30011 rows of 8 heads of 128, 35 MB to 123 MB of bf16, in 32 us, 4.9
// TB/s where a copy of 1 GiB reaches 5.3.  The values are stored past the caches: with
// lines kept there for them the same rows take 47 us when the calls before have filled
// them; 384 rows take 7 us either way.
template <typename T, int HD> __global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a)
{
    constexpr int G = HD / kGroup;
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T))));     // of four values
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
        __builtin_nontemporal_store(__builtin_bit_cast(Words, o), (Words *)(out + g * kGroup));
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
    }
    a.cos_t = cos_table; a.sin_t = sin_table; a.w[0] = q_weight; a.w[1] = k_weight;
    a.positions = positions; a.slots = slots; a.q_out = q_out;
    a.pool = make_pool(*cache);
    a.n_pos = n_pos;
    a.n_slots = cache->n_pages * cache->page;
    a.N = N; a.n_q = n_q; a.n_kv = cache->n_kv;
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
