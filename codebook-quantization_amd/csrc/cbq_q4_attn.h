// Attention of a batch's newest tokens over the 4-bit paged cache with a shared
// prefix (include/cbq_serve_q4.h): the kernels, as templates on the queries' type and
// the head size; cbq_q4_attn_{f32,bf16,f16}.hip hold one type each.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - max), in one pass over the
// keys with a running maximum.  With k_jd = m + s (c - 7.5) in a group g of 64 values,
//   q.k_j = sum_g s_jg A_jg + (m_jg - 23.5 s_jg) Q_g,   A_jg = sum_d q_d (c_jd + 16),
//   sum_j p_j v_jd = B_d - 23.5 C_g + sum_j p_j m_jg,   B_d = sum_j (p_j s_jg) (c_jd + 16),
// Q_g the group's sum of q and C_g that of p_j s_jg: the codes go to the matrix cores
// as they are.  c + 16 is one bf16 number, the code in its mantissa's upper bits under
// a constant exponent: a shift and a masked or make two of them.  No value is
// rounded on the way; q and p_j s_jg are cut into as many bf16 parts as their type
// has bits for (bf16: one, fp16: two, fp32: three), and C_g sums the same parts.
//
// Rows are the query heads of a kv head beside the tokens, 16 a tile: row r of a
// sequence is token r / rep, head r % rep.  Of a prefix the rows are the whole
// batch's.
//
// Products, with the keys in the left operand: S^T = K Q^T (16 keys x 16 rows) leaves
// a lane with one row and four keys; two such tiles are the right operand of O^T =
// V^T P^T, so weights never leave their lane.  A lane's eight keys there are eight
// neighbouring ones, and the codes' order in a row (four of each group side by side)
// gives it of each key one word, whose nibble n belongs to output tile n: no
// transpose, no LDS for the codes.
#pragma once

#include <type_traits>

#include "cbq_q4.h"
#include "cbq_q4_plan.h"

namespace cbq_q4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = kAttnWaves * CBQ_WAVE;

// The running maximum stands this far (in exp2's domain) above the scores of its last
// move, so that it moves seldom and no weight passes 1: a weight keeps all its bits.
constexpr float kSlack = 8.0f;

struct AttnArgs {
    const void *q;
    int64_t q_st[2];
    Pool pool;
    const int32_t *prefix_table, *tables, *lengths;
    int64_t table_st, capacity;             // own keys that a table row can name
    void *out;
    float *part_o;                          // [part][token][n_q][hd]
    float2 *part_ml;                        // [part][token][n_q]: running maximum, sum
    CbqDiv rep;
    int32_t prefix, batch, tokens, n_q, n_kv;
    float c, q_mul;                         // exp2(c * (q_mul q) . k); q_mul folds scale's sign
    float c_low;                            // what c's rounding left, for fp32
    Plan plan;
};

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;

// max / sum over the four lanes that hold one row (lane, lane ^ 16, ^ 32, ^ 48)
__device__ __forceinline__ float groups_max(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float x)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// x = the sum of N bf16 parts (up to x's own bits); part n is taken off x
template <int N> __device__ __forceinline__ void cut(float a, float b, uint32_t (&part)[N])
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        part[n] = pack2(a, b);
        if (n + 1 < N) {
            a -= __uint_as_float(part[n] << 16);
            b -= __uint_as_float(part[n] & 0xffff0000u);
        }
    }
}

// Two codes, at bits 3..6 of either half, as the bf16 numbers c + 16
__device__ __forceinline__ uint32_t code_pair(uint32_t x) { return (x & 0x00780078u) | 0x41804180u; }

// Eight codes (low nibble first) as c + 16, in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ u32x4 eight_codes(uint32_t w)
{
    return u32x4{code_pair(w << 3), code_pair(w >> 1), code_pair(w >> 5), code_pair(w >> 9)};
}

template <int HD> struct Geo {
    static constexpr int kG = HD / kGroup;              // groups of a row
    static constexpr int kKw = HD / 32;                 // words of codes of a key a lane holds
    static constexpr int kPairs = (kG + 1) / 2;         // pairs a lane loads, of keys and of values
    static constexpr int kScales = 4 * kG * kTile;      // floats of a wave's tile in LDS
    static constexpr int kWide = HD < 128 ? HD : 128;   // values of a row joined at once
};

// The codes of one tile, in registers: of two keys for S^T and eight values for O^T
template <int HD> struct Codes {
    using G = Geo<HD>;
    uint32_t k[2][G::kKw];                  // HD / 8 bytes of a key: a quarter of its row
    uint32_t v[8][HD == 256 ? 2 : 1];       // HD / 32 bytes of a value: four codes a group
    uint32_t kp[G::kPairs], vp[G::kPairs];  // pairs: of key lane % 32, group lane / 32 (+ 2)
    uint32_t there;                         // keys of the tile that are there

    __device__ __forceinline__ void load(const AttnArgs &a, int h, int32_t id, uint32_t row)
    {
        const int lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
        // an id outside the pool (or no key) reads page 0, row 0 and is hidden
        const bool in = id >= 0 && id < a.pool.n_pages;
        there = (uint32_t)__ballot(in);
        const uint32_t p = in ? id : 0, at = in ? row : 0;
        const uint32_t co = code_at(a.pool, p, at) + h * a.pool.code_st[1];
        const uint64_t po = pair_at(a.pool, p, at) + h * a.pool.pair_st[1];
#pragma unroll
        for (int i = 0; i < G::kPairs; i++) {
            const int g = G::kG == 1 ? 0 : (lane >> 5) + 2 * i;
            kp[i] = a.pool.pairs[0][po + g];
            vp[i] = a.pool.pairs[1][po + g];
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint64_t o = (uint64_t)__shfl(co, 8 * (r >> 2) + (r & 3) + 4 * t) * kCodeUnit;
            const char *from = a.pool.codes[0] + o + g4 * (HD / 8);
            if constexpr (HD == 64) *(u32x2 *)k[t] = *(const u32x2 *)from;
            else
#pragma unroll
                for (int i = 0; i < G::kKw / 4; i++)
                    *(u32x4 *)(k[t] + 4 * i) = *(const u32x4 *)(from + 16 * i);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint64_t o = (uint64_t)__shfl(co, 8 * g4 + i) * kCodeUnit;
            const char *from = a.pool.codes[1] + o + r * (HD / 32);
            if constexpr (HD == 64) v[i][0] = *(const uint16_t *)from;
            else if constexpr (HD == 128) v[i][0] = *(const uint32_t *)from;
            else *(u32x2 *)v[i] = *(const u32x2 *)from;
        }
    }
    // The tile's pairs as floats: scales and mids - 23.5 scales of the keys, scales and
    // mids of the values, each [group][key]; 0 for a key that is not there.
    __device__ __forceinline__ void spread(float *lds) const
    {
        const int lane = threadIdx.x & 63, key = lane & 31;
        const bool in = there >> key & 1;
        if (G::kG == 1 && lane >= 32) return;
#pragma unroll
        for (int i = 0; i < G::kPairs; i++) {
            float *to = lds + ((lane >> 5) + 2 * i) * kTile + key;
            const float s = pair_scale(kp[i]), m = pair_mid(kp[i]);
            to[0] = in ? s : 0.f;
            to[G::kG * kTile] = in ? fmaf(-23.5f, s, m) : 0.f;
            to[2 * G::kG * kTile] = in ? pair_scale(vp[i]) : 0.f;
            to[3 * G::kG * kTile] = in ? pair_mid(vp[i]) : 0.f;
        }
    }
    // Eight codes of group g, the lane's half hf, of key tile t
    __device__ __forceinline__ uint32_t key_codes(int t, int g, int hf) const
    {
        if constexpr (HD == 64) return k[t][hf];
        const int stride = HD / 128;        // words of four values of every group
        return __builtin_amdgcn_perm(k[t][(2 * hf + 1) * stride + g / 2], k[t][2 * hf * stride + g / 2],
                                     g & 1 ? 0x07060302u : 0x05040100u);
    }
};

// ---- a wave's state over 16 RT rows -----------------------------------------------------------
template <typename T, int HD, int RT> struct Rows {
    using G = Geo<HD>;
    static constexpr int N = kParts<T>;
    u32x4 q[RT][N][HD / 32];
    float qsum[RT][G::kG];
    f32x4 o[RT][HD / 16], ps[RT][G::kG];    // B, and C in every element
    float mids[RT][G::kG];                  // this lane's keys' part of sum p m
    float m[RT], l[RT];                     // running maximum (exp2's domain); this lane's part of sum p

    // Row `row` of 16 from row0 on (zeros from n on): of query token token0 + row / rep,
    // head h * rep + row % rep.
    __device__ __forceinline__ void start(const AttnArgs &a, int h, int64_t token0, int row0, int n)
    {
        const int lane = threadIdx.x & 63, g4 = lane >> 4;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int row = row0 + 16 * t + (lane & 15);
            const bool in = row < n;
            const uint32_t token = cbq_div(in ? row : 0, a.rep), head = (in ? row : 0) - token * a.rep.d;
            const T *x = (const T *)a.q + (token0 + token) * a.q_st[0] + ((int64_t)h * a.rep.d + head) * a.q_st[1];
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                float sum = 0.f;
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    struct alignas(16) Eight { T e[8]; };
                    const Eight e = *(const Eight *)(x + 64 * g + 16 * g4 + 8 * hf);
                    float f[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        f[i] = in ? (float)e.e[i] * a.q_mul : 0.f;
                        sum += f[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t part[N];
                        cut<N>(f[i], f[i + 4], part);
#pragma unroll
                        for (int p = 0; p < N; p++) q[t][p][2 * g + hf][i] = part[p];
                    }
                }
                qsum[t][g] = groups_sum(sum);
                ps[t][g] = f32x4{0, 0, 0, 0};
                mids[t][g] = 0.f;
            }
#pragma unroll
            for (int d = 0; d < HD / 16; d++) o[t][d] = f32x4{0, 0, 0, 0};
            m[t] = -INFINITY;
            l[t] = 0.f;
        }
    }

    // One tile.  MASKED: bits[t] holds the keys that the lane's row of tile t sees.
    template <bool MASKED>
    __device__ __forceinline__ void tile(const AttnArgs &a, const Codes<HD> &c, const float *lds,
                                         const uint32_t (&bits)[RT])
    {
        const int lane = threadIdx.x & 63, g4 = lane >> 4;
        const float *mine = lds + 8 * g4;               // this lane's eight keys
        auto four = [&](int which, int g, int t) {
            return *(const f32x4 *)(mine + (which * G::kG + g) * kTile + 4 * t);
        };
        f32x4 s[RT][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                const f32x4 off = four(1, g, t);
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[r][t][i] = g == 0 ? off[i] * qsum[r][g] : fmaf(off[i], qsum[r][g], s[r][t][i]);
            }
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                f32x4 acc[RT];
#pragma unroll
                for (int r = 0; r < RT; r++) acc[r] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const u32x4 k = eight_codes(c.key_codes(t, g, hf));
#pragma unroll
                    for (int r = 0; r < RT; r++)
#pragma unroll
                        for (int p = 0; p < N; p++) acc[r] = mma(k, q[r][p][2 * g + hf], acc[r]);
                }
                const f32x4 scale = four(0, g, t);
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[r][t][i] = fmaf(scale[i], acc[r][i], s[r][t][i]);
            }
        }
        float p[RT][8];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const uint32_t seen = MASKED ? bits[r] >> (8 * g4) : ~0u;
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (MASKED) s[r][i / 4][i % 4] = seen >> i & 1 ? s[r][i / 4][i % 4] : -INFINITY;
                top = fmaxf(top, s[r][i / 4][i % 4]);
            }
            top = groups_max(top) * a.c;
            if (__ballot(top > m[r])) {
                const float to = top > m[r] ? top + kSlack : m[r];
                const float f = top > m[r] ? __builtin_amdgcn_exp2f(m[r] - to) : 1.0f;
                m[r] = to;
                l[r] *= f;
#pragma unroll
                for (int g = 0; g < G::kG; g++) {
                    mids[r][g] *= f;
                    ps[r][g] *= f;
                }
#pragma unroll
                for (int d = 0; d < HD / 16; d++) o[r][d] *= f;
            }
            const float base = m[r] == -INFINITY ? 0.f : -m[r];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float e = fmaf(a.c, s[r][i / 4][i % 4], base);
                if (sizeof(T) == 4) e = fmaf(a.c_low, s[r][i / 4][i % 4], e);
                p[r][i] = __builtin_amdgcn_exp2f(e);
                l[r] += p[r][i];
            }
        }
#pragma unroll
        for (int g = 0; g < G::kG; g++) {
            u32x4 w[RT][N];                 // p s, in parts
#pragma unroll
            for (int r = 0; r < RT; r++) {
                const uint32_t seen = MASKED ? bits[r] >> (8 * g4) : ~0u;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    f32x4 scale = four(2, g, t), mid = four(3, g, t);
                    if (MASKED)             // what a hidden key holds may be NaN
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (!(seen >> (4 * t + i) & 1)) scale[i] = mid[i] = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; i++) mids[r][g] = fmaf(p[r][4 * t + i], mid[i], mids[r][g]);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint32_t part[N];
                        cut<N>(p[r][4 * t + 2 * i] * scale[2 * i], p[r][4 * t + 2 * i + 1] * scale[2 * i + 1], part);
#pragma unroll
                        for (int n = 0; n < N; n++) w[r][n][2 * t + i] = part[n];
                    }
                }
#pragma unroll
                for (int n = 0; n < N; n++)
                    ps[r][g] = mma(u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}, w[r][n], ps[r][g]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                // nibble 4 g + j of a value's words: byte (4 g + j) / 2, its upper half if odd
                const int nib = 4 * g + j, word = nib / 8, byte = nib % 8 / 2;
                const uint32_t sel = (uint32_t)(byte + 4) << 16 | (uint32_t)byte;
                u32x4 x;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t e = c.v[2 * i][word], f = c.v[2 * i + 1][word];
                    x[i] = code_pair(j & 1 ? __builtin_amdgcn_perm(f >> 1, e >> 1, sel)
                                           : __builtin_amdgcn_perm(f << 3, e << 3, sel));
                }
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int n = 0; n < N; n++) o[r][nib] = mma(x, w[r][n], o[r][nib]);
            }
        }
    }

    // Sums over the lanes of a row, and the values that B, C and the mids make
    __device__ __forceinline__ void finish()
    {
#pragma unroll
        for (int r = 0; r < RT; r++) {
            l[r] = groups_sum(l[r]);
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                const float add = groups_sum(mids[r][g]);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        o[r][4 * g + j][i] = fmaf(-23.5f, ps[r][g][i], o[r][4 * g + j][i]) + add;
            }
        }
    }
};

// Four values of a row from d on: a part's, or the output
template <typename T, int HD>
__device__ __forceinline__ void put_values(const AttnArgs &a, int part, int64_t token, int head, int d,
                                           f32x4 x, float sum)
{
    const int64_t row = token * a.n_q + head;
    if (part >= 0) {
        *(f32x4 *)(a.part_o + ((int64_t)part * a.batch * a.tokens * a.n_q + row) * HD + d) = x;
        return;
    }
    const float f = sum == 0.f ? 0.f : 1.0f / sum;
    struct alignas(4 * sizeof(T)) Four { T e[4]; } y;
#pragma unroll
    for (int i = 0; i < 4; i++) y.e[i] = (T)(x[i] * f);
    *(Four *)((T *)a.out + row * HD + d) = y;
}

// The four waves' states of rows row0 .. (n rows in all) joined in LDS and written.
template <typename T, int HD, int RT>
__device__ __forceinline__ void join_waves(const AttnArgs &a, Rows<T, HD, RT> &w, char *lds, int h,
                                           int64_t token0, int row0, int n, int part)
{
    constexpr int kWide = Geo<HD>::kWide;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g4 = lane >> 4;
    float *O = (float *)lds;                            // [wave][16][kWide]
    float2 *ML = (float2 *)(O + kAttnWaves * 16 * kWide);   // [wave][16]
    float *total = (float *)(ML + kAttnWaves * 16);     // [16]
#pragma unroll
    for (int t = 0; t < RT; t++) {
        if (row0 + 16 * t >= n) break;                  // uniform over the block
        __syncthreads();                                // LDS is free
        if (lane < 16) ML[wave * 16 + r] = make_float2(w.m[t], w.l[t]);
        __syncthreads();
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < kAttnWaves; i++) top = fmaxf(top, ML[i * 16 + r].x);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < kAttnWaves; i++)
            sum += __builtin_amdgcn_exp2f(ML[i * 16 + r].x - base) * ML[i * 16 + r].y;
        const float f = __builtin_amdgcn_exp2f(w.m[t] - base);
        if (wave == 0 && lane < 16) total[r] = sum;
        const int rows = n - row0 - 16 * t < 16 ? n - row0 - 16 * t : 16;
        if (part >= 0 && wave == 0 && lane < rows) {
            const uint32_t row = row0 + 16 * t + r, token = cbq_div(row, a.rep);
            a.part_ml[((int64_t)part * a.batch * a.tokens + token0 + token) * a.n_q +
                      (int64_t)h * a.rep.d + row - token * a.rep.d] = make_float2(top, sum);
        }
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += kWide) {
            if (d0) __syncthreads();
            // row r's pieces at (piece ^ r): 16 rows of one piece would share their banks
#pragma unroll
            for (int g = d0 / kGroup; g < (d0 + kWide) / kGroup; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f32x4 x = {w.o[t][4 * g][i], w.o[t][4 * g + 1][i], w.o[t][4 * g + 2][i],
                                     w.o[t][4 * g + 3][i]};
                    const int piece = (g - d0 / kGroup) * 16 + 4 * g4 + i;
                    *(f32x4 *)(O + (wave * 16 + r) * kWide + (piece ^ r) * 4) = x * f;
                }
            __syncthreads();
            for (int e = tid; e < rows * (kWide / 4); e += kBlock) {
                const int rr = e / (kWide / 4), piece = e % (kWide / 4);
                f32x4 x = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < kAttnWaves; i++)
                    x += *(const f32x4 *)(O + (i * 16 + rr) * kWide + (piece ^ rr) * 4);
                const uint32_t row = row0 + 16 * t + rr, token = cbq_div(row, a.rep);
                put_values<T, HD>(a, part, token0 + token, h * a.rep.d + row - token * a.rep.d,
                                  d0 + piece * 4, x, total[rr]);
            }
        }
    }
}

template <int HD> constexpr int attn_lds()
{
    constexpr int tiles = kAttnWaves * Geo<HD>::kScales * 4;
    constexpr int join = kAttnWaves * 16 * Geo<HD>::kWide * 4 + kAttnWaves * 16 * 8 + 16 * 4;
    return tiles > join ? tiles : join;
}

// Rows row0 .. (of n) against the key tiles [first, end); seq -1: prefix rows of the
// whole batch.
template <typename T, int HD, int RT>
__device__ __forceinline__ void walk(const AttnArgs &a, char *lds, const Work &w, int row0, int n, int to)
{
    using G = Geo<HD>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t pre_tiles = (a.prefix + kTile - 1) / kTile;
    int32_t length = 0, end = w.end;
    const int32_t *own = nullptr;
    if (w.seq >= 0) {
        length = cbq_clamp_length(a.lengths[w.seq], a.capacity);
        own = a.tables + w.seq * a.table_st;
        end = (int32_t)cbq_min(end, (int64_t)pre_tiles + cbq_ceil(length, kTile));
        if (w.first >= end && a.plan.parts > 1) return;     // the merge counts own parts by the length
    }
    const int64_t token0 = w.seq >= 0 ? (int64_t)w.seq * a.tokens : 0;
    float *scales = (float *)lds + wave * G::kScales;
    Rows<T, HD, RT> rows;
    rows.start(a, w.h, token0, row0, n);
    // own keys that the lane's row of each tile sees
    int32_t sees[RT];
#pragma unroll
    for (int t = 0; t < RT; t++)
        sees[t] = length - a.tokens + 1 + (int32_t)cbq_div(row0 + 16 * t + (lane & 15), a.rep);
    int32_t id = -1;
    uint32_t row = 0;
    auto look = [&](int32_t tile) {                     // this lane's key's page
        id = -1;
        if (tile >= end) return;
        const int32_t j = tile_key(tile, pre_tiles, a.prefix, length, lane & 31);
        if (j < 0) return;
        const uint32_t entry = cbq_div((uint32_t)j, a.pool.page);
        row = (uint32_t)j - entry * a.pool.page.d;
        id = (tile < pre_tiles ? a.prefix_table : own)[entry];
    };
    int32_t tile = w.first + wave;
    Codes<HD> next;
    look(tile);
    if (tile < end) next.load(a, w.h, id, row);
    look(tile + kAttnWaves);
    for (; tile < end; tile += kAttnWaves) {
        const Codes<HD> now = next;
        if (tile + kAttnWaves < end) next.load(a, w.h, id, row);
        look(tile + 2 * kAttnWaves);
        now.spread(scales);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int32_t key0 = (tile - pre_tiles) * kTile;
        uint32_t bits[RT];
        bool whole = now.there == ~0u;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            bits[t] = now.there;
            if (tile >= pre_tiles) {
                const int32_t left = sees[t] - key0;
                if (left < kTile) bits[t] &= left <= 0 ? 0u : (1u << left) - 1;
            }
            whole = whole && bits[t] == ~0u;
        }
        if (__all(whole)) rows.template tile<false>(a, now, scales, bits);
        else rows.template tile<true>(a, now, scales, bits);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    rows.finish();
    join_waves<T, HD, RT>(a, rows, lds, w.h, token0, row0, n, to);
}

template <typename T, int HD, int RT> __global__ __launch_bounds__(kBlock, 2) void q4_kernel(AttnArgs a)
{
    __shared__ __attribute__((aligned(16))) char lds[attn_lds<HD>()];
    const int32_t pre_tiles = (a.prefix + kTile - 1) / kTile,
                  cap_tiles = (int32_t)((a.capacity + kTile - 1) / kTile);
    const uint32_t block = cbq_block(blockIdx.x, blockIdx.y);
    if (block >= a.plan.blocks) return;
    const Work w = work_of(a.plan, block, a.n_kv, a.batch, pre_tiles, cap_tiles);
    const int to = a.plan.parts > 1 ? w.part : -1, rows = a.tokens * (int)a.rep.d;
    if (w.seq < 0) walk<T, HD, RT>(a, lds, w, w.tile * 16 * RT, a.batch * rows, to);
    else walk<T, HD, 1>(a, lds, w, w.tile * 16, rows, to);
}

// ---- merge of the parts: a block a (token, head) -------------------------------------------------
template <typename T, int HD> __global__ __launch_bounds__(kBlock) void q4_merge_kernel(AttnArgs a)
{
    constexpr int kLanes = HD / 4, kGroups = kBlock / kLanes;
    __shared__ __attribute__((aligned(16))) float sums[kGroups][HD];
    __shared__ float totals[kGroups];
    const int tid = threadIdx.x, lane = tid & 63, group = tid / kLanes, d = tid % kLanes * 4;
    const int64_t rows = (int64_t)a.batch * a.tokens * a.n_q, row = cbq_block(blockIdx.x, blockIdx.y);
    if (row >= rows) return;
    const int64_t token = row / a.n_q;
    const int32_t length = cbq_clamp_length(a.lengths[token / a.tokens], a.capacity);
    const int parts = a.plan.pre_parts + (int)cbq_ceil(cbq_ceil(length, kTile), a.plan.own_chunk);
    float top = -INFINITY;
    for (int p = lane; p < parts; p += CBQ_WAVE) top = fmaxf(top, a.part_ml[p * rows + row].x);
    for (int i = 32; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 x = {0, 0, 0, 0};
    float sum = 0.f;
    for (int p = group; p < parts; p += kGroups) {
        const float2 ml = a.part_ml[p * rows + row];
        const f32x4 o = *(const f32x4 *)(a.part_o + (p * rows + row) * HD + d);
        const float w = __builtin_amdgcn_exp2f(ml.x - base);
        sum += w * ml.y;                    // 0 of an empty part; a NaN stays
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = w == 0.f ? x[e] : fmaf(w, o[e], x[e]);
    }
    *(f32x4 *)&sums[group][d] = x;
    if (d == 0) totals[group] = sum;
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int i = 1; i < kGroups; i++) {
        x += *(const f32x4 *)&sums[i][d];
        sum += totals[i];
    }
    put_values<T, HD>(a, -1, token, (int)(row - token * a.n_q), d, x, sum);
}

// ---- launches of one type -------------------------------------------------------------------------
template <typename T, int HD> int launch(const AttnArgs &a, hipStream_t stream)
{
    CbqGrid grid = cbq_grid(a.plan.blocks);
    q4_kernel<T, HD, 1><<<dim3(grid.x, grid.y), kBlock, 0, stream>>>(a);
    int rc = cbq_launch_status("cbq_prefix_attn_decode_q4");
    if (rc != CK_SUCCESS || a.plan.parts == 1) return rc;
    grid = cbq_grid((int64_t)a.batch * a.tokens * a.n_q);
    q4_merge_kernel<T, HD><<<dim3(grid.x, grid.y), kBlock, 0, stream>>>(a);
    return cbq_launch_status("cbq_prefix_attn_decode_q4 merge");
}

template <typename T> int launch_hd(const AttnArgs &a, int hd, hipStream_t stream)
{
    if (hd == 64) return launch<T, 64>(a, stream);
    if (hd == 128) return launch<T, 128>(a, stream);
    return launch<T, 256>(a, stream);
}

int launch_f32(const AttnArgs &a, int hd, hipStream_t stream);
int launch_bf16(const AttnArgs &a, int hd, hipStream_t stream);
int launch_f16(const AttnArgs &a, int hd, hipStream_t stream);

}  // namespace cbq_q4
