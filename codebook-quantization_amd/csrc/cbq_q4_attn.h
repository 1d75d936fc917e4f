// Attention of a batch's newest tokens over the 4-bit paged cache with a shared
// prefix (include/cbq_serve_q4.h): the kernels, as templates on the queries' type and
// the head size; cbq_q4_attn_{f32,bf16,f16}.hip hold one type each.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - max), in one pass over the
// keys with a running maximum.  With k_jd = m + s (c - 7.5) in a group g of 64 values,
//   q.k_j = sum_g s_jg A_jg + m_jg Q_g,              A_jg = sum_d q_d (c_jd + z) - R_g,
//   sum_j p_j v_jd = B_d - (z + 7.5) C_g + sum_j p_j m_jg,   B_d = sum_j (p_j s_jg) (c_jd + z),
// Q_g the group's sum of q, R_g that of (z + 7.5) q, with which the products begin, and C_g
// that of p_j s_jg: the codes go to the matrix cores as they are, and no dequantised value
// is rounded.  c + z is one fp16 number, the code in its mantissa under a constant
// exponent: z is 16, 64 or 256 where the code's lowest bit is bit 6, 4 or 2, so a
// masked or makes two of them, and a shift serves four.  A large z costs the sums bits:
// 256 for half the keys' codes of 16-bit queries (2^-18 of a score), 64 for half the
// values' of bf16 ones, else 16; fp32 queries pay a packed addition for c - 7.5, z none.
// (The code's bits alone, a subnormal number, need no or; but the products add those
// without their leading zeros: ten bits of every sum.)
//
// The other operands have to fit fp16.  A query row is scaled to a largest value in
// [2^14, 2^15), fp32 cut into two parts.  p_j s_jg is taken against 2^E, E the largest
// exponent of the scales of the values that the wave has met: its 11 bits hold down to
// 2^-26 of the largest scale, the 22 of fp32's two parts to 2^-15; below that it is off by
// 2^-37 of that scale.
//
// Rows are the query heads of a kv head beside the tokens, 16 a tile: row r of a
// sequence is token r / rep, head r % rep.  Of a prefix the rows are the whole
// batch's.
//
// Products, with the keys in the left operand: S^T = K Q^T (16 keys x 16 rows) leaves
// a lane with one row and four keys; two such tiles are the right operand of O^T =
// V^T P^T, so weights never leave their lane.  The codes' order in a row (four of each
// group side by side) gives a lane there of each of its eight keys one word, whose
// nibble n belongs to output tile n: no transpose.
//
// A wave walks tiles of 32 keys of its own.  Codes, pairs and page ids go from memory
// straight to LDS, kDepth - 1 tiles ahead, without registers on the way and without a
// wait but for the tile that is due.
//
// 24 sequences of 4000 to 32000 keys, 32 heads on 8 of 128, bf16: 110 us, 4.6 TB/s of the
// cache, where a copy of 1 GiB moves 5.3; the vector units bound it, 1300 cycles a tile
// and wave, three waves a SIMD.  One sequence of 384 keys: 10 us, two launches and the
// chain of their loads (ids, pages, parts).  Ids, queries and the length are asked for at
// once: one after the other, 16 sequences of 4 tokens behind 1000 keys took 18.5 us
// instead of 14.6, and the long ones 114.  fp32 queries take twice the products and
// an addition a pair of codes: the long ones 148 us in a captured graph, bf16 there 120.
#pragma once

#include <atomic>
#include <type_traits>

#include "cbq_q4.h"
#include "cbq_q4_plan.h"

namespace cbq_q4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = kAttnWaves * CBQ_WAVE;

// The running maximum stands this far (in exp2's domain) above the scores of its last
// move, so that it moves seldom and no weight passes 1.
constexpr float kSlack = 2.0f;

// p s 2^(kUp - E) < 2^14, and p 2^kUp <= 2^14: fp16 has room for them, and 2^-14 is its
// smallest whole number
constexpr int kUp = 14, kNone = -1000;      // kNone: no scale yet

struct AttnArgs {
    const void *q;
    int64_t q_st[2];
    Pool pool;
    const int32_t *prefix_table, *tables, *lengths;
    int64_t table_st, capacity;             // own keys that a table row can name
    void *out;
    float *part_o;                          // [part][token][n_q][hd]
    float2 *part_ml;                        // [part][token][n_q]: running maximum, sum
    CbqDiv rep, tiles_a_page;               // of pages of whole tiles
    uint32_t code_row, pair_row;            // bytes from row to row, of such pages
    int32_t whole;                          // every tile lies in one page
    int32_t prefix, batch, tokens, n_q, n_kv;
    float c, q_mul;                         // exp2(c * (q_mul q) . k); q_mul folds scale's sign
    float c_low;                            // what c's rounding left, for fp32
    Plan plan;
};

template <typename T> constexpr int kParts = sizeof(T) == 4 ? 2 : 1;

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

// Nothing is moved over this: operands unpacked or read ahead of their turn cost
// registers, and with them waves
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// x, computed in this branch and not before it
__device__ __forceinline__ uint32_t here(uint32_t x)
{
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// a and b as N fp16 parts each.  What is taken off them is the part that was made, its bits:
// a product under way to a and to fp16 would round to either of two neighbours.
template <int N> __device__ __forceinline__ void cut(float a, float b, uint32_t (&part)[N])
{
#pragma unroll
    for (int n = 0; n < N; n++) {
        part[n] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
        if (n + 1 < N) {
            asm("" : "+v"(part[n]));
            const f16x2 x = __builtin_bit_cast(f16x2, part[n]);
            a -= (float)x[0];
            b -= (float)x[1];
        }
    }
}

// a x and b y as N fp16 parts each: products rounded once, by one operation each where
// one part is asked for
template <int N> __device__ __forceinline__ void cut_products(float a, float x, float b, float y, uint32_t (&part)[N])
{
    if constexpr (N == 1) {                 // (a sum with 0 keeps the product and its rounding in one)
        const f16x2 z = {(_Float16)fmaf(a, x, 0.f), (_Float16)fmaf(b, y, 0.f)};
        part[0] = __builtin_bit_cast(uint32_t, z);
    } else {
        cut<N>(a * x, b * y, part);
    }
}

// Two codes of a word, at bits FROM .. FROM + 3 of either half, as the fp16 numbers c + z.
// The constants stay in registers, a scalar and a vector one: an operation of three
// operands takes no literal.
template <int FROM> struct Pair {
    uint32_t mask, magic;
    __device__ __forceinline__ Pair()
    {
        constexpr uint32_t bits = 0x000f000fu << FROM, exponent = (uint32_t)(25 - FROM) << 10;
        asm("s_mov_b32 %0, %1" : "=s"(mask) : "i"(bits));
        asm("v_mov_b32 %0, %1" : "=v"(magic) : "i"(exponent << 16 | exponent));
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (x & mask) | magic; }
};

// z + 7.5 of a key's codes (even and odd ones) and of a value's (lower and upper ones)
template <typename T> struct Zeros {
    static constexpr bool kNone = sizeof(T) == 4;
    static constexpr float kEven = kNone ? 0 : 263.5f, kOdd = kNone ? 0 : 23.5f;
    static constexpr float kLow = kNone ? 0 : 23.5f, kHigh = kNone ? 0 : std::is_same_v<T, __bf16> ? 71.5f : 23.5f;
};

template <typename T> struct Unpack {
    Pair<6> six;
    Pair<4> four;
    Pair<2> two;

    // Eight codes of a key (low nibble first) in the order 0 4 1 5 2 6 3 7
    __device__ __forceinline__ u32x4 key(uint32_t w) const
    {
        if constexpr (Zeros<T>::kNone) {
            return u32x4{bare(w << 6), bare(w << 2), bare(w >> 2), bare(w >> 6)};
        } else {
            const uint32_t x = w << 2, y = w >> 6;
            return u32x4{two(x), six(x), two(y), six(y)};
        }
    }
    // The lower and upper codes of two values' bytes (bits 0..7 of either half)
    __device__ __forceinline__ uint32_t low(uint32_t x) const
    {
        if constexpr (Zeros<T>::kNone) return bare(x << 6);
        else return six(x << 6);
    }
    __device__ __forceinline__ uint32_t high(uint32_t x) const
    {
        if constexpr (Zeros<T>::kNone) return bare(x << 2);
        else if constexpr (Zeros<T>::kHigh == 71.5f) return four(x);
        else return six(x << 2);
    }
    // c - 7.5, exactly
    __device__ __forceinline__ uint32_t bare(uint32_t x) const
    {
        const f16x2 off = {(_Float16)-23.5f, (_Float16)-23.5f};
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, six(x)) + off);
    }
};

template <int HD> struct Geo {
    static constexpr int kG = HD / kGroup;              // groups of a row
    static constexpr int kRow = HD / 2, kPieces = HD / 32;      // bytes of a row's codes, 16 of them a piece
    static constexpr int kRows = CBQ_WAVE / kPieces;    // rows that a copy takes
    static constexpr int kCopies = kTile / kRows;       // copies of a tile's keys (and values)
    static constexpr int kPairCopies = (kG + 1) / 2;    // of their pairs: 64 a copy
    static constexpr int kOps = 2 * kCopies + 2 * kPairCopies + 1;      // of a tile, its ids among them
    // a wave's LDS: a ring of tiles, one of page ids, scales and mids of the tile at hand
    static constexpr int kDepth = HD == 256 ? 3 : 2;
    static constexpr int kCodes = kTile * kRow, kPairs = kPairCopies * 256;
    static constexpr int kSlot = 2 * kCodes + 2 * kPairs;
    static constexpr int kIds = kDepth * kSlot, kScales = kIds + kDepth * 256;
    static constexpr int kWave = kScales + 4 * kG * kTile * 4;
    static constexpr int kWide = HD < 128 ? HD : 128;   // values of a row joined at once
    // Piece p of row r lies at p ^ mix(r): the pieces that sixteen rows are read at
    // together fall on 64 different banks.
    static __device__ __forceinline__ int mix(int row) { return row / (512 / HD) & (kPieces - 1); }
};

// ---- tiles on their way to LDS ------------------------------------------------------------------
// Written as asm, so that the compiler neither waits for a copy before an LDS read nor
// counts it: arrived() does.  A copy takes 16 (4) bytes a lane to its place in the
// wave's next 1024 (256) bytes at `lds`; M0 holds that address, with a wait state between
// its write and the load.  The LDS reads before it are done.
__device__ __forceinline__ void copy16(uint32_t lds, const char *base, uint32_t offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void copy16(uint32_t lds, const char *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds), "v"(from) : "m0", "memory");
}
__device__ __forceinline__ void copy4(uint32_t lds, const char *base, uint32_t offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :: "s"(lds), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void copy4(uint32_t lds, const char *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :: "s"(lds), "v"(from) : "m0", "memory");
}
// All but the last N of this wave's copies have arrived
template <int N> __device__ __forceinline__ void arrived()
{
    static_assert(N >= 0 && N < 64, "a six-bit counter");
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

// A wave's tiles `first`, `first` + kAttnWaves, .. below `end`, numbered 0, 1, ..
template <int HD> struct Tiles {
    using G = Geo<HD>;
    const AttnArgs &a;
    const int32_t *own;
    int32_t pre_tiles, length, first, end, h;
    char *lds;                              // this wave's
    uint32_t at;                            // its address
    uint32_t there[G::kDepth - 1];          // of the tiles on their way, in turn: keys that are there

    __device__ __forceinline__ int32_t tile(int n) const { return first + n * kAttnWaves; }
    // Place of the tile's key `key` in its table's order; the last one's past their end
    __device__ __forceinline__ int32_t place(int32_t tile, int key, bool &in) const
    {
        const bool shared = tile < pre_tiles;
        const int32_t j = (shared ? tile : tile - pre_tiles) * kTile + key, n = shared ? a.prefix : length;
        in = j < n;
        return in ? j : n - 1;
    }
    // Page ids of tile n's keys (of one that is there, where n is past the end)
    __device__ __forceinline__ void ask_ids(int n) const
    {
        bool in;
        const int32_t t = tile(n) < end ? tile(n) : tile(0);
        const int32_t j = place(t, threadIdx.x & 31, in);
        const char *table = (const char *)(t < pre_tiles ? a.prefix_table : own);
        copy4(at + G::kIds + n % G::kDepth * 256, table, 4 * cbq_div((uint32_t)j, a.pool.page));
    }
    // Tile n into slot n % kDepth, its ids there; and the ids of tile n + kDepth - 1.
    // What is not there is read from page 0, row 0.  Returns the keys that are.
    __device__ __forceinline__ uint32_t ask(int n) const
    {
        uint32_t in_pool;
        const int lane = threadIdx.x & 63;
        const int32_t t = tile(n);
        const int32_t *ids = (const int32_t *)(lds + G::kIds + n % G::kDepth * 256);
        const uint32_t to = at + n % G::kDepth * G::kSlot;
        const char *kc = a.pool.codes[0], *vc = a.pool.codes[1];
        const char *kp = (const char *)a.pool.pairs[0], *vp = (const char *)a.pool.pairs[1];
        const int sub = lane / G::kPieces, piece = lane % G::kPieces;
        if (a.whole) {                      // the tile lies in one page
            bool in;
            const uint32_t j = (t < pre_tiles ? t : t - pre_tiles), left = (t < pre_tiles ? a.prefix : length) - j * kTile;
            const int32_t id = __builtin_amdgcn_readfirstlane(ids[0]);
            in = id >= 0 && id < a.pool.n_pages;
            const uint32_t page = in ? id : 0, row = (j - cbq_div(j, a.tiles_a_page) * a.tiles_a_page.d) * kTile;
            const uint64_t co = (uint64_t)(code_at(a.pool, page, row) + h * a.pool.code_st[1]) * kCodeUnit,
                           po = (uint64_t)(pair_at(a.pool, page, row) + h * a.pool.pair_st[1]) * kPairUnit;
            in_pool = !in ? 0 : left >= kTile ? ~0u : (1u << left) - 1;
#pragma unroll
            for (int i = 0; i < G::kPairCopies; i++) {
                const uint32_t o = (lane & 31) * a.pair_row + (G::kG == 1 ? 0 : (lane >> 5) + 2 * i) * kPairUnit;
                copy4(to + 2 * G::kCodes + i * 256, kp + po, o);
                copy4(to + 2 * G::kCodes + G::kPairs + i * 256, vp + po, o);
            }
#pragma unroll
            for (int i = 0; i < G::kCopies; i++) {
                const int r = i * G::kRows + sub;
                const uint32_t o = r * a.code_row + (piece ^ G::mix(r)) * 16;
                copy16(to + i * 1024, kc + co, o);
                copy16(to + G::kCodes + i * 1024, vc + co, o);
            }
        } else {
            auto row_of = [&](int key, uint32_t &page, uint32_t &row) {
                bool in;
                const uint32_t j = (uint32_t)place(t, key, in);
                const int32_t id = ids[key];
                in = in && id >= 0 && id < a.pool.n_pages;
                page = in ? id : 0;
                row = in ? j - cbq_div(j, a.pool.page) * a.pool.page.d : 0;
                return in;
            };
            uint32_t page, row;
            in_pool = (uint32_t)__ballot(row_of(lane & 31, page, row));
            const uint64_t po = (uint64_t)(pair_at(a.pool, page, row) + h * a.pool.pair_st[1]) * kPairUnit;
#pragma unroll
            for (int i = 0; i < G::kPairCopies; i++) {
                const uint64_t o = po + (G::kG == 1 ? 0 : (lane >> 5) + 2 * i) * kPairUnit;
                copy4(to + 2 * G::kCodes + i * 256, kp + o);
                copy4(to + 2 * G::kCodes + G::kPairs + i * 256, vp + o);
            }
#pragma unroll
            for (int i = 0; i < G::kCopies; i++) {
                const int r = i * G::kRows + sub;
                row_of(r, page, row);
                const uint64_t o = (uint64_t)(code_at(a.pool, page, row) + h * a.pool.code_st[1]) * kCodeUnit +
                                   (piece ^ G::mix(r)) * 16;
                copy16(to + i * 1024, kc + o);
                copy16(to + G::kCodes + i * 1024, vc + o);
            }
        }
        ask_ids(n + G::kDepth - 1);
        return in_pool;
    }
    // The first tiles' page ids, asked for before the length is known: of the tiles below
    // `upto`, where the tables end.
    __device__ __forceinline__ void look(int32_t upto)
    {
        at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
        at = __builtin_amdgcn_readfirstlane(at);
        if (tile(0) >= upto) return;
#pragma unroll
        for (int n = 0; n < G::kDepth - 1; n++) {
            const int32_t t = tile(n) < upto ? tile(n) : tile(0);
            const bool shared = t < pre_tiles;
            const uint32_t j = (uint32_t)(shared ? t : t - pre_tiles) * kTile + (threadIdx.x & 31),
                           last = (shared ? (uint32_t)a.prefix : (uint32_t)a.capacity) - 1;
            copy4(at + G::kIds + n * 256, (const char *)(shared ? a.prefix_table : own),
                  4 * cbq_div(j < last ? j : last, a.pool.page));
        }
    }
    // The first tiles, whose ids are there
    __device__ __forceinline__ void begin()
    {
#pragma unroll
        for (int n = 0; n < G::kDepth - 1; n++)
            there[n] = tile(n) < end ? ask(n) : 0;
    }
    // Tile n has arrived, and the tile behind those under way is asked for: the keys of n
    // that are there.
    __device__ __forceinline__ uint32_t next(int n)
    {
        const uint32_t now = there[0];
#pragma unroll
        for (int i = 0; i + 2 < G::kDepth; i++) there[i] = there[i + 1];
        if (tile(n + G::kDepth - 2) < end) arrived<(G::kDepth - 2) * G::kOps>();
        else arrived<0>();
        if (tile(n + G::kDepth - 1) < end) there[G::kDepth - 2] = ask(n + G::kDepth - 1);
        return now;
    }
};

// A tile in LDS.  Key 16 t + 4 i + g of it is number 4 t + i of lane group g (lane / 16):
// four neighbouring rows a read.
template <int HD> struct Slot {
    using G = Geo<HD>;
    const char *lds;

    // The pairs of key lane % 32, group lane / 32 + 2 i, of keys (0) and values (1)
    __device__ __forceinline__ uint32_t pair(int which, int i) const
    {
        return *(const uint32_t *)(lds + 2 * G::kCodes + which * G::kPairs + i * 256 + (threadIdx.x & 63) * 4);
    }
    // The largest exponent of the lane's value scales; kNone where none counts
    __device__ __forceinline__ int exponent(uint32_t there) const
    {
        const bool in = there >> (threadIdx.x & 31) & 1;
        int e = kNone;
#pragma unroll
        for (int i = 0; i < G::kPairCopies; i++) {
            const float s = pair_scale(pair(1, i));
            if (in && s > 0.f && s < INFINITY) e = max(e, __builtin_amdgcn_frexp_expf(s));
        }
        return e;
    }
    // The tile's pairs as floats: scales and mids of the keys, scales (times 2^(kUp - E)) and
    // mids of the values, each [group][lane group][eight keys]; 0 for a key that is not
    // there.
    __device__ __forceinline__ void spread(float *to, uint32_t there, int E) const
    {
        const int lane = threadIdx.x & 63, key = lane & 31;
        const bool in = there >> key & 1;
        if (G::kG == 1 && lane >= 32) return;
        to += (lane >> 5) * kTile + (key & 3) * 8 + (key >> 2);
#pragma unroll
        for (int i = 0; i < G::kPairCopies; i++) {
            const uint32_t k = pair(0, i), v = pair(1, i);
            const float s = pair_scale(k), m = pair_mid(k);
            float vs = pair_scale(v), vm = pair_mid(v);
            // a scale that is not finite makes the mid so: p = 0 keeps it out by the mid alone
            if (!(vs >= 0.f && vs < INFINITY)) vs = 0.f, vm = __builtin_nanf("");
            to[2 * i * kTile] = in ? s : 0.f;
            to[(G::kG + 2 * i) * kTile] = in ? m : 0.f;
            to[(2 * G::kG + 2 * i) * kTile] = in ? __builtin_amdgcn_ldexpf(vs, kUp - E) : 0.f;
            to[(3 * G::kG + 2 * i) * kTile] = in ? vm : 0.f;
        }
    }
    // This lane's quarter of a key's codes: row lane % 16 of S^T's tile t
    __device__ __forceinline__ void keys(int t, uint32_t (&k)[HD / 32]) const
    {
        const int x = threadIdx.x & 15, g4 = threadIdx.x >> 4 & 3, row = 16 * t + 4 * (x & 3) + (x >> 2);
        const char *from = lds + row * G::kRow;
        if constexpr (HD == 64) *(u32x2 *)k = *(const u32x2 *)(from + ((g4 >> 1) ^ G::mix(row)) * 16 + (g4 & 1) * 8);
        else
#pragma unroll
            for (int i = 0; i < HD / 128; i++)
                *(u32x4 *)(k + 4 * i) = *(const u32x4 *)(from + ((g4 * (HD / 128) + i) ^ G::mix(row)) * 16);
    }
    // Eight codes of group g, the quarter's half hf
    static __device__ __forceinline__ uint32_t key_codes(const uint32_t (&k)[HD / 32], int g, int hf)
    {
        if constexpr (HD == 64) return k[hf];
        const int stride = HD / 128;        // words of four values of every group
        return __builtin_amdgcn_perm(k[(2 * hf + 1) * stride + g / 2], k[2 * hf * stride + g / 2],
                                     g & 1 ? 0x07060302u : 0x05040100u);
    }
    // Four codes of each group, 4 (lane % 16) .., of this lane's value number n
    __device__ __forceinline__ void value(int n, uint32_t (&v)[HD == 256 ? 2 : 1]) const
    {
        const int x = threadIdx.x & 15, g4 = threadIdx.x >> 4 & 3, row = 4 * n + g4;
        constexpr int kEach = HD / 32, kIn = 16 / kEach;        // bytes a lane, lanes a piece
        const char *from = lds + G::kCodes + row * G::kRow + ((x / kIn) ^ G::mix(row)) * 16 + x % kIn * kEach;
        if constexpr (HD == 64) v[0] = *(const uint16_t *)from;
        else if constexpr (HD == 128) v[0] = *(const uint32_t *)from;
        else *(u32x2 *)v = *(const u32x2 *)from;
    }
};

// ---- a wave's state over 16 rows --------------------------------------------------------------
template <typename T, int HD> struct Rows {
    using G = Geo<HD>;
    static constexpr int N = kParts<T>;
    static constexpr bool kCentred = Zeros<T>::kNone;       // nothing to take off the sums
    u32x4 q[N][HD / 32];
    float qsum[G::kG];
    f32x4 less[G::kG];                      // -R in every element, which the products begin with
    Unpack<T> unpack;
    f32x4 o[HD / 16], ps[G::kG];            // B, and C in every element
    float mids[G::kG];                      // this lane's keys' part of sum p m
    float m, l;                             // running maximum (exp2's domain); this lane's part of sum p
    float c, c_low;                         // exp2's factors, the row's scaling taken back
    int E;                                  // p s is times 2^(kUp - E)

    // This lane's quarter of a row's values, eight at a time
    struct Queries {
        u32x4 e[G::kG][2][sizeof(T) / 2];
    };
    // Row `row` of 16 from row0 on (the first for those from n on): of query token token0 +
    // row / rep, head h * rep + row % rep.
    static __device__ __forceinline__ void load(const AttnArgs &a, int h, int64_t token0, int row0, int n, Queries &x)
    {
        const int lane = threadIdx.x & 63, g4 = lane >> 4, row = row0 + (lane & 15);
        const uint32_t token = cbq_div(row < n ? row : 0, a.rep), head = (row < n ? row : 0) - token * a.rep.d;
        const T *from = (const T *)a.q + (token0 + token) * a.q_st[0] + ((int64_t)h * a.rep.d + head) * a.q_st[1];
#pragma unroll
        for (int g = 0; g < G::kG; g++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; i++)
                    x.e[g][hf][i] = *(const u32x4 *)((const char *)(from + 64 * g + 16 * g4 + 8 * hf) + 16 * i);
    }
    // They are there: the compiler waits for them here, and not behind what is asked for next
    static __device__ __forceinline__ void loaded(Queries &x)
    {
#pragma unroll
        for (int g = 0; g < G::kG; g++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; i++) asm volatile("" : "+v"(x.e[g][hf][i]));
    }
    // Zeros for rows from n on
    __device__ __forceinline__ void start(const AttnArgs &a, int row0, int n, const Queries &x)
    {
        const int lane = threadIdx.x & 63;
        E = kNone;
        const bool in = row0 + (lane & 15) < n;
        float f[G::kG][2][8], top = 0.f;
#pragma unroll
        for (int g = 0; g < G::kG; g++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                struct Eight { T e[8]; };
                struct Words { u32x4 e[sizeof(T) / 2]; } words;
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; i++) words.e[i] = x.e[g][hf][i];
                const Eight e = __builtin_bit_cast(Eight, words);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    f[g][hf][i] = in ? (float)e.e[i] * a.q_mul : 0.f;
                    top = fmaxf(top, fabsf(f[g][hf][i]));
                }
            }
        top = groups_max(top);
        const int up = 15 - __builtin_amdgcn_frexp_expf(top);       // top 2^up in [2^14, 2^15)
        // factors that are not 0 (a hidden key's -inf times 0 is none) and finite
        c = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.c, -up), 0x1p-149f), 3.0e38f);
        c_low = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.c_low, -up), 0x1p-149f), 3.0e38f);
#pragma unroll
        for (int g = 0; g < G::kG; g++) {
            float even = 0.f, odd = 0.f;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    f[g][hf][i] = __builtin_amdgcn_ldexpf(f[g][hf][i], up);
                    (i & 1 ? odd : even) += f[g][hf][i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t part[N];
                    cut<N>(f[g][hf][i], f[g][hf][i + 4], part);
#pragma unroll
                    for (int p = 0; p < N; p++) q[p][2 * g + hf][i] = part[p];
                }
            }
            even = groups_sum(even);
            odd = groups_sum(odd);
            qsum[g] = even + odd;
            const float r = kCentred ? 0.f : -Zeros<T>::kEven * even - Zeros<T>::kOdd * odd;
            less[g] = f32x4{r, r, r, r};
            ps[g] = f32x4{0, 0, 0, 0};
            mids[g] = 0.f;
        }
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[d] = f32x4{0, 0, 0, 0};
        m = -INFINITY;
        l = 0.f;
    }

    // A tile whose scales' largest exponent is e, over the wave
    __device__ __forceinline__ void follow(int e)
    {
        if (!__ballot(e > E)) return;
        for (int i = 32; i > 0; i >>= 1) e = max(e, __shfl_xor(e, i));
        e = __builtin_amdgcn_readfirstlane(e) + 1;          // one bit of room
        const int down = E == kNone ? 0 : E - e;
        E = e;
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[d][i] = __builtin_amdgcn_ldexpf(o[d][i], down);
        if (!kCentred)
#pragma unroll
            for (int g = 0; g < G::kG; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) ps[g][i] = __builtin_amdgcn_ldexpf(ps[g][i], down);
    }

    // One tile.  bits holds the keys that the lane's row sees; hidden: some row does not see all.
    __device__ __forceinline__ void tile(const Slot<HD> &slot, const float *lds, uint32_t bits, bool hidden)
    {
        const int lane = threadIdx.x & 63, g4 = lane >> 4;
        const float *mine = lds + 8 * g4;               // this lane's eight keys
        auto four = [&](int which, int g, int t) {
            return *(const f32x4 *)(mine + (which * G::kG + g) * kTile + 4 * t);
        };
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            phase();
            uint32_t codes[HD / 32];
            slot.keys(t, codes);
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                const f32x4 off = four(1, g, t);
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][i] = g == 0 ? off[i] * qsum[g] : fmaf(off[i], qsum[g], s[t][i]);
            }
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                f32x4 acc = kCentred ? f32x4{0, 0, 0, 0} : less[g];
                const u32x4 k[2] = {unpack.key(slot.key_codes(codes, g, 0)), unpack.key(slot.key_codes(codes, g, 1))};
#pragma unroll
                for (int p = 0; p < N; p++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) acc = mma(k[hf], q[p][2 * g + hf], acc);
                const f32x4 scale = four(0, g, t);
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][i] = fmaf(scale[i], acc[i], s[t][i]);
            }
        }
        phase();
        if (hidden) {
            const uint32_t seen = here(bits >> g4);
#pragma unroll
            for (int i = 0; i < 8; i++) s[i / 4][i % 4] = seen >> (4 * i) & 1 ? s[i / 4][i % 4] : -INFINITY;
        }
        float p[8], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, s[i / 4][i % 4]);
        // the row's maximum is found where one of its lanes passes it
        if (__ballot(top * c > m)) {
            top = groups_max(top) * c;
            const float to = top > m ? top + kSlack : m;
            const float f = top > m ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
            m = to;
            l *= f;
#pragma unroll
            for (int g = 0; g < G::kG; g++) {
                mids[g] *= f;
                if (!kCentred) ps[g] *= f;
            }
#pragma unroll
            for (int d = 0; d < HD / 16; d++) o[d] *= f;
        }
        const float base = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float e = fmaf(c, s[i / 4][i % 4], base);
            if (sizeof(T) == 4) e = fmaf(c_low, s[i / 4][i % 4], e);
            p[i] = __builtin_amdgcn_exp2f(e);
            l += p[i];
        }
        uint32_t codes[8][HD == 256 ? 2 : 1];
#pragma unroll
        for (int i = 0; i < 8; i++) slot.value(i, codes[i]);
#pragma unroll
        for (int g = 0; g < G::kG; g++) {
            phase();
            u32x4 w[N];                     // p s, in parts
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f32x4 scale = four(2, g, t);
                f32x4 mid = four(3, g, t);
                if (hidden) {               // what a hidden key holds may be NaN
                    const uint32_t seen = here(bits >> (16 * t + g4));
#pragma unroll
                    for (int i = 0; i < 4; i++) mid[i] = seen >> (4 * i) & 1 ? mid[i] : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mids[g] = fmaf(p[4 * t + i], mid[i], mids[g]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t part[N];
                    cut_products<N>(p[4 * t + 2 * i], scale[2 * i], p[4 * t + 2 * i + 1], scale[2 * i + 1], part);
#pragma unroll
                    for (int n = 0; n < N; n++) w[n][2 * t + i] = part[n];
                }
            }
            const u32x4 ones = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
            if (!kCentred)
#pragma unroll
                for (int n = 0; n < N; n++) ps[g] = mma(ones, w[n], ps[g]);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                // nibbles 4 g + j, 4 g + j + 1 of the values' words: one byte
                const int nib = 4 * g + j, word = nib / 8, byte = nib % 8 / 2;
                u32x4 x;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x[i] = __builtin_amdgcn_perm(codes[2 * i + 1][word], codes[2 * i][word],
                                                 0x0c000c00u | (uint32_t)(byte + 4) << 16 | (uint32_t)byte);
                u32x4 low, high;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    low[i] = unpack.low(x[i]);
                    high[i] = unpack.high(x[i]);
                }
#pragma unroll
                for (int n = 0; n < N; n++) {
                    o[nib] = mma(low, w[n], o[nib]);
                    o[nib + 1] = mma(high, w[n], o[nib + 1]);
                }
            }
        }
    }

    // Sums over the lanes of a row, and the values that B, C and the mids make
    __device__ __forceinline__ void finish()
    {
        const int up = E == kNone ? 0 : E - kUp;
        l = groups_sum(l);
#pragma unroll
        for (int g = 0; g < G::kG; g++) {
            const float add = groups_sum(mids[g]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float b = o[4 * g + j][i];
                    const float z = j & 1 ? Zeros<T>::kHigh : Zeros<T>::kLow;
                    o[4 * g + j][i] = add + __builtin_amdgcn_ldexpf(kCentred ? b : fmaf(-z, ps[g][i], b), up);
                }
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
template <typename T, int HD>
__device__ __forceinline__ void join_waves(const AttnArgs &a, Rows<T, HD> &w, char *lds, int h,
                                           int64_t token0, int row0, int n, int part)
{
    constexpr int kWide = Geo<HD>::kWide;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g4 = lane >> 4;
    float *O = (float *)lds;                            // [wave][16][kWide]
    float2 *ML = (float2 *)(O + kAttnWaves * 16 * kWide);   // [wave][16]
    float *total = (float *)(ML + kAttnWaves * 16);     // [16]
    __syncthreads();                                // LDS is free
    if (lane < 16) ML[wave * 16 + r] = make_float2(w.m, w.l);
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kAttnWaves; i++) top = fmaxf(top, ML[i * 16 + r].x);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < kAttnWaves; i++)
        sum += __builtin_amdgcn_exp2f(ML[i * 16 + r].x - base) * ML[i * 16 + r].y;
    const float f = __builtin_amdgcn_exp2f(w.m - base);
    if (wave == 0 && lane < 16) total[r] = sum;
    const int rows = n - row0 < 16 ? n - row0 : 16;
    if (part >= 0 && wave == 0 && lane < rows) {
        const uint32_t row = row0 + r, token = cbq_div(row, a.rep);
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
                const f32x4 x = {w.o[4 * g][i], w.o[4 * g + 1][i], w.o[4 * g + 2][i],
                                 w.o[4 * g + 3][i]};
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
            const uint32_t row = row0 + rr, token = cbq_div(row, a.rep);
            put_values<T, HD>(a, part, token0 + token, h * a.rep.d + row - token * a.rep.d,
                              d0 + piece * 4, x, total[rr]);
        }
    }
}

// ---- a shared prefix against many rows ------------------------------------------------------------
// 64 RT rows a block of one kv head, 16 RT a wave, for bf16 queries: with that many rows
// a tile's values are worth making once, as fp16 numbers in LDS for all four waves, and
// the scales' products with every row fall away.  Keys and values are taken against
// the largest exponents of the block's keys, found in a first pass over their pairs:
// (c - 8) s + (m + s / 2) in two packed operations.  The second addend is rounded to fp16
// and the sum again: each an eighth of a bf16 query's and output's own rounding, and s, of
// eight bits, not at all: so for 8 s down to 2^-27 of the largest 8 s or |m|, below that the
// roundings are to fp16's smallest number.
//
// A slot of 16 bytes holds eight values in the order 0 4 1 5 2 6 3 7 that the codes'
// masks give them; queries are read in that order, and outputs put back.
//
// 64 sequences of 32 heads of 128 behind 30011 keys, 200 to 1500 own ones: 77 us, of which
// the products would take 26.  A wave's chain from tile to tile bounds it (products,
// softmax, products: 2.3 us a tile of 64 keys, one such wave a SIMD beside those of own
// keys).  In a captured graph, where it takes 78 to 83: 64 rows a block, one to three blocks
// a CU, 95 to 101, 128 rows and two blocks 92, every wave's own tiles 110.  When it took 80,
// 256 rows a block took 123, and a launch for the prefix alone, without the own keys' blocks
// beside it, 104.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int HD> struct Made {
    static constexpr int kKeys = HD == 256 ? 32 : 64;               // of a tile
    static constexpr int kSlots = HD / 8, kRow = HD * 2;            // slots and bytes of a row
    static constexpr int kLanes = kBlock / 2 / kKeys;               // threads a row of keys, or of values
    static constexpr int kPiece = HD / 2 / kLanes;                  // bytes of codes a thread takes
    static constexpr int kSide = kKeys * kRow;                      // bytes of the keys, or the values
    static constexpr int kThere = 4 * kSide;                        // two buffers, then flags and sums
    static constexpr int kLds = kThere + 2 * kKeys * 4 + kAttnWaves * 8;
    static_assert(kPiece == 16 || kPiece == 32, "whole loads");
    // Slot s of a row lies at s ^ mix(row): 16 rows' equal slots, and the neighbouring two that
    // the transpose reads of the values take of eight rows, fall on different banks.
    static __device__ __forceinline__ constexpr int mix(int row)
    {
        if (kSlots == 8) return (row >> 1 & 3) << 1 ^ (row >> 3 & 1) * 5;   // rows of half the banks
        return (row & 7) << 1 ^ (row >> 3 & 1) * 9;
    }
};

// The largest exponent of a group's values: of max(8 s, |m|), which half of none exceeds
__device__ __forceinline__ int pair_exponent(uint32_t p)
{
    const float x = fmaxf(8.f * pair_scale(p), fabsf(pair_mid(p)));
    return x > 0.f && x < INFINITY ? __builtin_amdgcn_frexp_expf(x) : kNone;
}

// One thread's codes and pairs of a tile: a piece of one row, of the keys (the block's
// first half) or the values
template <int HD> struct Raw {
    using M = Made<HD>;
    static constexpr int kG = HD / kGroup, kWords = M::kPiece / 4;
    uint32_t w[kWords], pair[kG];
    int32_t id;                             // page of the next tile's row
    uint32_t at;
    bool in;

    static __device__ __forceinline__ int side() { return threadIdx.x / (kBlock / 2); }
    // neighbouring lanes have neighbouring rows, whose slots they write to different banks
    static __device__ __forceinline__ int row() { return threadIdx.x % M::kKeys; }
    static __device__ __forceinline__ int piece() { return threadIdx.x % (kBlock / 2) / M::kKeys; }

    __device__ __forceinline__ void look(const AttnArgs &a, int32_t key0, int32_t end)
    {
        const int32_t j = key0 + row();
        id = -1;
        if (j >= end) return;
        const uint32_t entry = cbq_div((uint32_t)j, a.pool.page);
        at = (uint32_t)j - entry * a.pool.page.d;
        id = a.prefix_table[entry];
    }
    // The tile that look() has found the pages of; no key, or an id outside the pool: zeros
    __device__ __forceinline__ void load(const AttnArgs &a, int h)
    {
        in = id >= 0 && id < a.pool.n_pages;
        const uint32_t p = in ? id : 0, r = in ? at : 0;
        const char *codes = (side() ? a.pool.codes[1] : a.pool.codes[0]) +
                            (uint64_t)(code_at(a.pool, p, r) + h * a.pool.code_st[1]) * kCodeUnit + piece() * M::kPiece;
        const uint32_t *pairs = (side() ? a.pool.pairs[1] : a.pool.pairs[0]) +
                                (uint64_t)(pair_at(a.pool, p, r) + h * a.pool.pair_st[1]);
#pragma unroll
        for (int i = 0; i < kWords / 4; i++) *(u32x4 *)(w + 4 * i) = *(const u32x4 *)(codes + 16 * i);
#pragma unroll
        for (int g = 0; g < kG; g++) pair[g] = pairs[g];
    }
    // The values of the piece, times 2^up, slot by slot into a tile whose keys begin at `tile`
    static constexpr int kMine = kWords;    // slots a thread
    f16x2 off[kG], step[kG];                // m + s / 2 and s, twice

    __device__ __forceinline__ void begin(float *there, int up)
    {
#pragma unroll
        for (int g = 0; g < kG; g++) {
            float s = __builtin_amdgcn_ldexpf(pair_scale(pair[g]), up), m = __builtin_amdgcn_ldexpf(pair_mid(pair[g]), up);
            if (!(s >= 0.f && s < INFINITY)) s = 0.f, m = __builtin_nanf("");
            if (!in) s = m = 0.f;
            const _Float16 b = (_Float16)fmaf(0.5f, s, m), one = (_Float16)s;
            off[g] = f16x2{b, b};
            step[g] = f16x2{one, one};
        }
        if (threadIdx.x < kBlock / 2 && piece() == 0) there[row()] = in ? 0.f : -INFINITY;
    }
    __device__ __forceinline__ void slot(char *tile, int i) const
    {
        const int g = i % kG, n = i / kG;
        // the words of four values of every group, twice: eight of group g
        uint32_t x;
        if constexpr (HD == 64) x = w[n];
        else x = __builtin_amdgcn_perm(w[(2 * n + 1) * (kG / 2) + g / 2], w[2 * n * (kG / 2) + g / 2],
                                       g & 1 ? 0x07060302u : 0x05040100u);
        // c - 8, exactly: the upper codes' 16 (c - 8) a sixteenth
        const f16x2 eight = {(_Float16)-1032.f, (_Float16)-1032.f}, more = {(_Float16)-72.f, (_Float16)-72.f},
                    part = {(_Float16)0.0625f, (_Float16)0.0625f};
        constexpr uint32_t kLower = 0x000f000fu, kUpper = 0x00f000f0u;      // 1024 + c, 1024 + 16 c
        auto half = [](uint32_t y, uint32_t mask) { return __builtin_bit_cast(f16x2, (y & mask) | 0x64006400u); };
        const f16x2 x0 = (half(x, kLower) + eight) * step[g] + off[g], x1 = (half(x, kUpper) * part + more) * step[g] + off[g],
                    x2 = (half(x >> 8, kLower) + eight) * step[g] + off[g],
                    x3 = (half(x >> 8, kUpper) * part + more) * step[g] + off[g];
        const int at = 8 * g + piece() * (8 / M::kLanes) + n;
        *(u32x4 *)(tile + side() * M::kSide + row() * M::kRow + (at ^ M::mix(row())) * 16) =
            u32x4{__builtin_bit_cast(uint32_t, x0), __builtin_bit_cast(uint32_t, x1),
                  __builtin_bit_cast(uint32_t, x2), __builtin_bit_cast(uint32_t, x3)};
    }
};

template <typename T, int HD, int RT>
__device__ __forceinline__ void shared_rows(const AttnArgs &a, char *lds, const Work &w, int row0, int n, int part)
{
    using M = Made<HD>;
    constexpr int kC = HD / 32, kD = HD / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15,
              g4 = lane >> 4;
    const int32_t first = w.first * kTile, end = (int32_t)cbq_min((int64_t)w.end * kTile, a.prefix);
    float *there = (float *)(lds + M::kThere);
    int2 *tops = (int2 *)(lds + M::kThere + 2 * M::kKeys * 4);
    Raw<HD> raw;
    raw.look(a, first, end);
    // the queries: rows row0 + 16 (RT wave + t) + lane % 16
    u32x4 q[RT][kC];
    f32x4 o[RT][kD];
    float m[RT], l[RT], c[RT];
    const int mine = row0 + 16 * RT * wave;
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int row = mine + 16 * t + r;
        const bool in = row < n;
        const uint32_t token = cbq_div(in ? row : 0, a.rep), head = (in ? row : 0) - token * a.rep.d;
        const T *x = (const T *)a.q + token * a.q_st[0] + ((int64_t)w.h * a.rep.d + head) * a.q_st[1];
        float f[kC][8], top = 0.f;
#pragma unroll
        for (int d = 0; d < kC; d++) {
            struct alignas(16) Eight { T e[8]; };
            const Eight e = *(const Eight *)(x + 32 * d + 8 * g4);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[d][i] = in ? (float)e.e[i] * a.q_mul : 0.f;
                top = fmaxf(top, fabsf(f[d][i]));
            }
        }
        const int up = 15 - __builtin_amdgcn_frexp_expf(groups_max(top));
        c[t] = __builtin_amdgcn_ldexpf(a.c, -up);
#pragma unroll
        for (int d = 0; d < kC; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t one[1];
                cut<1>(__builtin_amdgcn_ldexpf(f[d][i], up), __builtin_amdgcn_ldexpf(f[d][i + 4], up), one);
                q[t][d][i] = one[0];
            }
#pragma unroll
        for (int d = 0; d < kD; d++) o[t][d] = f32x4{0, 0, 0, 0};
        m[t] = -INFINITY;
        l[t] = 0.f;
    }
    // largest exponents of the part's keys and values, eight keys' pairs under way at once
    int2 top = {kNone, kNone};
    constexpr int kAhead = 8;
    for (int32_t j0 = first + tid; j0 < end; j0 += kAhead * kBlock) {
        uint64_t po[kAhead];
        bool in[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int32_t j = j0 + i * kBlock;
            const uint32_t entry = cbq_div((uint32_t)(j < end ? j : j0), a.pool.page);
            const uint32_t row = (uint32_t)(j < end ? j : j0) - entry * a.pool.page.d;
            const int32_t id = a.prefix_table[entry];
            in[i] = j < end && id >= 0 && id < a.pool.n_pages;
            po[i] = pair_at(a.pool, in[i] ? id : 0, in[i] ? row : 0) + w.h * a.pool.pair_st[1];
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++)
#pragma unroll
            for (int g = 0; g < HD / kGroup; g++) {
                const int x = pair_exponent(a.pool.pairs[0][po[i] + g]), y = pair_exponent(a.pool.pairs[1][po[i] + g]);
                top.x = max(top.x, in[i] ? x : kNone);
                top.y = max(top.y, in[i] ? y : kNone);
            }
    }
    for (int i = 32; i > 0; i >>= 1) {
        top.x = max(top.x, __shfl_xor(top.x, i));
        top.y = max(top.y, __shfl_xor(top.y, i));
    }
    if (lane == 0) tops[wave] = top;
    raw.load(a, w.h);
    raw.look(a, first + M::kKeys, end);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAttnWaves; i++) {
        top.x = max(top.x, tops[i].x);
        top.y = max(top.y, tops[i].y);
    }
    // a value is below 2^(top + 1): 2^15 of it is left
    const int k_up = top.x == kNone ? 0 : 14 - __builtin_amdgcn_readfirstlane(top.x),
              v_up = top.y == kNone ? 0 : 14 - __builtin_amdgcn_readfirstlane(top.y);
#pragma unroll
    for (int t = 0; t < RT; t++) c[t] = fminf(fmaxf(__builtin_amdgcn_ldexpf(c[t], -k_up), 0x1p-149f), 3.0e38f);
    int buffer = 0;
    const int up = Raw<HD>::side() ? v_up : k_up;
    raw.begin(there, up);
#pragma unroll
    for (int i = 0; i < Raw<HD>::kMine; i++) raw.slot(lds, i);
    for (int32_t key = first; key < end; key += M::kKeys) {
        __syncthreads();                                // the tile is there
        raw.load(a, w.h);                               // the next one (past the end: zeros)
        raw.look(a, key + 2 * M::kKeys, end);
        const char *K = lds + buffer * 2 * M::kSide, *V = K + M::kSide;
        const float *bias = there + buffer * M::kKeys;
        const bool hidden = __ballot(lane < M::kKeys && bias[lane < M::kKeys ? lane : 0] != 0.f);
        constexpr int kT = M::kKeys / 16;
        f32x4 s[RT][kT];
#pragma unroll
        for (int t = 0; t < kT; t++) {
#pragma unroll
            for (int x = 0; x < RT; x++) s[x][t] = f32x4{0, 0, 0, 0};
            const int row = 16 * t + r;
#pragma unroll
            for (int d = 0; d < kC; d++) {
                const u32x4 e = *(const u32x4 *)(K + row * M::kRow + ((4 * d + g4) ^ M::mix(row)) * 16);
#pragma unroll
                for (int x = 0; x < RT; x++) s[x][t] = mma(e, q[x][d], s[x][t]);
            }
        }
        if (hidden)
#pragma unroll
            for (int t = 0; t < kT; t++) {
                const f32x4 b = *(const f32x4 *)(bias + 16 * t + 4 * g4);
#pragma unroll
                for (int x = 0; x < RT; x++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[x][t][i] = b[i] == 0.f ? s[x][t][i] : -INFINITY;
            }
        u32x4 p[RT][kT / 2];
#pragma unroll
        for (int x = 0; x < RT; x++) {
            float high = -INFINITY;
#pragma unroll
            for (int t = 0; t < kT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) high = fmaxf(high, s[x][t][i]);
            if (__ballot(high * c[x] > m[x])) {
                high = groups_max(high) * c[x];
                const float to = high > m[x] ? high + kSlack : m[x];
                const float f = high > m[x] ? __builtin_amdgcn_exp2f(m[x] - to) : 1.0f;
                m[x] = to;
                l[x] *= f;
#pragma unroll
                for (int d = 0; d < kD; d++) o[x][d] *= f;
            }
            // weights times 2^kUp, in sums and products alike: the largest is below 2^14, and
            // fp16's 11 bits hold down to 2^-28 of it
            const float base = m[x] == -INFINITY ? 0.f : (float)kUp - m[x];
#pragma unroll
            for (int t = 0; t < kT; t++) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = __builtin_amdgcn_exp2f(fmaf(c[x], s[x][t][i], base));
                    l[x] += e[i];
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t one[1];
                    cut<1>(e[2 * i], e[2 * i + 1], one);
                    p[x][t / 2][t % 2 * 2 + i] = one[0];
                }
            }
        }
        // The values' products, a slot of the next tile made beside every second: lane (g4, r)
        // points the transpose read at key 4 g4 + r / 4, values 4 (r % 4) .. of sixteen, and
        // gets keys 4 g4 .. + 3 of value r.
        buffer ^= 1;
        char *next = lds + buffer * 2 * M::kSide;
        raw.begin(there + buffer * M::kKeys, up);
        constexpr int kSteps = kT / 2 * kD, kEvery = kSteps / Raw<HD>::kMine;
#pragma unroll
        for (int step = 0; step < kSteps; step++) {
            const int d = step % kD, k0 = step / kD * 32;
            u32x4 e;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int row = k0 + 16 * t + 4 * g4 + (r >> 2);
                const char *from = V + row * M::kRow + ((2 * d + (r >> 1 & 1)) ^ M::mix(row)) * 16 + (r & 1) * 8;
                const u32x2 four = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(s16x4 *)from));
                e[2 * t] = four[0];
                e[2 * t + 1] = four[1];
            }
#pragma unroll
            for (int x = 0; x < RT; x++) o[x][d] = mma(e, p[x][k0 / 32], o[x][d]);
            if (step % kEvery == 0) raw.slot(next, step / kEvery);
        }
    }
    // a wave's rows through its part of LDS, in the values' order
    __syncthreads();
    float *out = (float *)(lds + wave * 16 * HD * 4);
    constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int from = mine + 16 * t;
        if (from >= n) break;
        const float total = __builtin_amdgcn_ldexpf(groups_sum(l[t]), -kUp);
#pragma unroll
        for (int d = 0; d < kD; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = d * 16 + 8 * (g4 >> 1) + (g4 & 1 ? kOrder[4 + i] : kOrder[i]);
                out[r * HD + (at ^ (r & 7) << 2)] = __builtin_amdgcn_ldexpf(o[t][d][i], -v_up - kUp);
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int rows = n - from < 16 ? n - from : 16;
        for (int e = lane; e < 16 * (HD / 4); e += CBQ_WAVE) {
            const int rr = e / (HD / 4), piece = e % (HD / 4);
            const float sum = __shfl(total, rr);
            const f32x4 x = *(const f32x4 *)(out + rr * HD + (piece ^ (rr & 7)) * 4);
            const uint32_t row = from + rr, token = cbq_div(row, a.rep);
            if (rr < rows) put_values<T, HD>(a, part, token, w.h * a.rep.d + row - token * a.rep.d, piece * 4, x, sum);
        }
        if (part >= 0 && lane < rows) {
            const uint32_t row = from + r, token = cbq_div(row, a.rep);
            a.part_ml[((int64_t)part * a.batch * a.tokens + token) * a.n_q + (int64_t)w.h * a.rep.d + row -
                      token * a.rep.d] = make_float2(m[t], total);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <int HD, int RT> constexpr int attn_lds()
{
    constexpr int made = RT ? Made<HD>::kLds : 0;
    constexpr int tiles = kAttnWaves * Geo<HD>::kWave;
    constexpr int join = kAttnWaves * 16 * Geo<HD>::kWide * 4 + kAttnWaves * 16 * 8 + 16 * 4;
    constexpr int both = tiles > join ? tiles : join;
    return both > made ? both : made;
}

// Rows row0 .. (of n) against the key tiles [first, end); seq -1: prefix rows of the
// whole batch.
template <typename T, int HD>
__device__ __forceinline__ void walk(const AttnArgs &a, char *lds, const Work &w, int row0, int n, int to)
{
    using G = Geo<HD>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t pre_tiles = (a.prefix + kTile - 1) / kTile;
    const int64_t token0 = w.seq >= 0 ? (int64_t)w.seq * a.tokens : 0;
    char *mine = lds + wave * G::kWave;
    float *scales = (float *)(mine + G::kScales);
    // page ids, queries and the length under way at once, then the tiles
    Tiles<HD> tiles = {a, w.seq >= 0 ? a.tables + w.seq * a.table_st : nullptr, pre_tiles, 0, w.first + wave, w.end, w.h,
                       mine};
    tiles.look(w.end);
    typename Rows<T, HD>::Queries queries;
    Rows<T, HD>::load(a, w.h, token0, row0, n, queries);
    int32_t length = 0, end = w.end;
    if (w.seq >= 0) {
        length = cbq_clamp_length(a.lengths[w.seq], a.capacity);
        end = (int32_t)cbq_min(end, (int64_t)pre_tiles + cbq_ceil(length, kTile));
    }
    arrived<0>();
    Rows<T, HD>::loaded(queries);
    if (w.first >= end && a.plan.parts > 1) return;         // the merge counts own parts by the length
    tiles.length = length;
    tiles.end = end;
    tiles.begin();
    Rows<T, HD> rows;
    rows.start(a, row0, n, queries);
    // own keys that the lane's row sees
    const int32_t sees = length - a.tokens + 1 + (int32_t)cbq_div(row0 + (lane & 15), a.rep);
    for (int i = 0; tiles.tile(i) < end; i++) {
        const uint32_t there = tiles.next(i);
        const int32_t tile = tiles.tile(i);
        const Slot<HD> slot = {mine + i % G::kDepth * G::kSlot};
        rows.follow(slot.exponent(there));
        slot.spread(scales, there, rows.E);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // the first token sees the fewest own keys
        const int32_t key0 = (tile - pre_tiles) * kTile;
        const bool own_end = tile >= pre_tiles && key0 + kTile > length - a.tokens + 1;
        const int32_t left = own_end ? sees - key0 : kTile;
        uint32_t bits = ~0u;
        if (there != ~0u || own_end) bits = there & (left >= kTile ? ~0u : left <= 0 ? 0u : (1u << left) - 1);
        rows.tile(slot, scales, bits, there != ~0u || own_end);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    rows.finish();
    join_waves<T, HD>(a, rows, lds, w.h, token0, row0, n, to);
}

// Waves a SIMD: their registers, and tiles two (or, of one wave, three) deep in LDS, leave
// room for so many.  24 sequences of 4000 to 32000 keys, bf16, hd 128, in a captured graph:
// three waves two tiles deep 120 us, two waves three deep 143, four waves (which spill) two
// deep 275.
constexpr int simd_waves(int hd, int rt) { return hd == 256 ? 1 : rt ? 2 : 3; }

// RT: 64 RT rows a block of the prefix; 0: 16, as the own keys'.
template <typename T, int HD, int RT>
__global__ __launch_bounds__(kBlock, simd_waves(HD, RT)) void q4_kernel(AttnArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int32_t pre_tiles = (a.prefix + kTile - 1) / kTile,
                  cap_tiles = (int32_t)((a.capacity + kTile - 1) / kTile);
    const uint32_t block = cbq_block(blockIdx.x, blockIdx.y);
    if (block >= a.plan.blocks) return;
    const Work w = work_of(a.plan, block, a.n_kv, a.batch, pre_tiles, cap_tiles);
    const int to = a.plan.parts > 1 ? w.part : -1, rows = a.tokens * (int)a.rep.d;
    if constexpr (RT > 0) {
        if (w.seq < 0) {
            shared_rows<T, HD, RT>(a, lds, w, w.tile * 64 * RT, a.batch * rows, to);
            return;
        }
    }
    walk<T, HD>(a, lds, w, w.tile * 16, w.seq < 0 ? a.batch * rows : rows, to);
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
// More than 64 KiB of LDS is asked for once a kernel and device.
template <auto K> bool lds_allowed(int lds)
{
    static std::atomic<uint64_t> asked{0};
    if (lds <= 65536) return true;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev <= 63 && asked.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute((const void *)K, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return false;
    asked.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

template <typename T, int HD, int RT> int launch_rows(const AttnArgs &a, hipStream_t stream)
{
    const char *what = "cbq_prefix_attn_decode_q4";
    const CbqGrid grid = cbq_grid(a.plan.blocks);
    constexpr int lds = attn_lds<HD, RT>();
    if (!lds_allowed<q4_kernel<T, HD, RT>>(lds)) return cbq_launch_status(what);
    q4_kernel<T, HD, RT><<<dim3(grid.x, grid.y), kBlock, lds, stream>>>(a);
    return cbq_launch_status(what);
}

template <typename T, int HD> int launch(const AttnArgs &a, hipStream_t stream)
{
    constexpr int wide = std::is_same_v<T, __bf16> ? widest(HD) : 0;
    int rc;
    if (a.plan.rt == 0) rc = launch_rows<T, HD, 0>(a, stream);
    else if (a.plan.rt == 1) rc = launch_rows<T, HD, wide ? 1 : 0>(a, stream);
    else rc = launch_rows<T, HD, wide>(a, stream);
    if (rc != CK_SUCCESS || a.plan.parts == 1) return rc;
    const CbqGrid grid = cbq_grid((int64_t)a.batch * a.tokens * a.n_q);
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
