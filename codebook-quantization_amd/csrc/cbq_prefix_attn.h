// Attention of a batch over a paged key/value cache with a shared prefix
// (include/cbq_serve.h): the kernels, as templates on the cache's type and the
// head size; cbq_prefix_attn_{f32,bf16,f16}.hip hold one type each.
//
// out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s), s_j = scale q.k_j,
// in one pass over the keys: a running maximum m, sum l and weighted values o
// of each query row, o and l scaled by exp(m_old - m_new) when m grows.
//
// Rows.  The n_q / n_kv query heads that read one kv head are rows beside the
// tokens: row r of kv head h is token r / rep, head h * rep + r % rep, so the
// heads of a group share each key read.  Of a shared prefix, the rows are the
// whole batch's.
//
// Products.  Both are matrix-core products with the keys in the left operand:
// S^T = K Q^T (16 keys x 16 rows a tile) leaves a lane with one row (lane % 16)
// and four keys (4 * (lane / 16) + i), which is, for two tiles side by side, the
// right operand of O^T = V^T P^T up to an order of the keys that V's loads
// follow.  So weights never leave their lane, a row's maximum needs two
// exchanges between lane groups, and m, l and the rescaling are one value a lane.
// V^T comes out of row-major V by the LDS transpose read (16-bit types); fp32
// uses the 16x16x4 fp32 products, whose operand is one element a lane.
//
// Tiles of keys go to LDS, straight (a block's) or through registers (a wave's
// own), the loads of a tile being under way while the one before is computed;
// 16-byte slots of a row are stored at slot ^ mix(row), which spreads both
// operands' reads over the banks.
//
// What bounds it (MI355X; heads 32 on 8 of 128 unless said): of long bf16 prompts
// nothing alone: 8192 tokens 565 to 603 us by card (925 to 970 TFLOP/s; the
// framework's large product runs at 1.2 PFLOP/s), the matrix units busy 44 % of the
// cycles, the clock at 2.1 GHz and lower the fewer cycles are needed, and LDS copies
// and reads in the way (eight waves a block 529); one-token steps HBM: 64 sequences of
// 200..1500 own keys 58 us without a prefix and 85 behind 30011 shared keys (3.8 and
// 4.2 TB/s, launches and merge included); few keys two launches of 4 to 5 us and a
// chain of three dependent loads (length, page id, key).
#pragma once

#include <atomic>
#include <type_traits>

#include "cbq_device.h"
#include "cbq_paged.h"
#include "../../include/cbq_serve.h"

namespace cbq_attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kWaves = kAttnWaves, kThreads = kWaves * CBQ_WAVE;

// The running maximum follows the scores once they pass it by kSlack (in exp2's
// domain).  So that no weight passes 1 all the same, and sums of values near the end
// of their range stay inside it, a bf16 row's m stands kSlack above the largest score
// of its last move (the shift costs a weight 2^-21, far below bf16's step), and fp32
// weights are multiplied by 2^-kSlack, exactly.  fp16 weights keep the bits: 2^kSlack
// times its largest value, 65504, leaves 2^104 of fp32's range.
constexpr float kSlack = 8.0f;
template <typename T> constexpr float kAbove = std::is_same_v<T, __bf16> ? kSlack : 0.0f;
template <typename T> constexpr float kOver = kSlack - kAbove<T>;
template <typename T> constexpr float kDown = sizeof(T) == 4 ? 1.0f / 256 : 1.0f;

struct AttnArgs {
    const void *q;
    int64_t q_st[2];
    cbq_paged_kv kv;
    const int32_t *prefix_table, *tables, *lengths, *q_start;
    int64_t table_st, capacity;             // own keys that a table row can name
    void *out;
    float *part_o;                          // [part][token][n_q][hd]
    float2 *part_ml;                        // [part][token][n_q]: running maximum, sum
    CbqDiv page;
    int32_t prefix, batch, N, n_q, rep;
    // Page and row strides in `unit` bytes, a power of two that divides them all:
    // a row's offset in the pool is one 32-bit number (the host has checked).
    uint32_t unit, k_page, k_row, v_page, v_row;
    int32_t one_stride;                     // keys and values lie alike
    float c, q_mul;                         // exp2(c * (q_mul q) . k); q_mul folds scale's sign
    float c_low;                            // what c's rounding left, for fp32's weights
    Plan plan;
};

// ---- the matrix products of one type ---------------------------------------------
template <typename T> struct Mma;
template <> struct Mma<__bf16> {
    static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 pv16(u32x2 a, u32x2 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                         __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 pv16(u32x2 a, u32x2 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                                     __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {
    static __device__ __forceinline__ f32x4 qk(u32x4 a, u32x4 b, f32x4 c)
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]),
                                                     c, 0, 0, 0);
        return c;
    }
};

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, t2{(T)a, (T)b});
}

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

// ---- geometry of a type and head size ---------------------------------------------
template <typename T, int HD> struct Geo {
    static constexpr int kEl = 16 / (int)sizeof(T);         // elements of a 16-byte slot
    static constexpr int kSlots = HD / kEl;                 // slots of a row
    // Slot s of a row lies at s ^ mix(row): 16 rows' equal slots in 16 places (of
    // rows of 128 bytes: 8, two rows a bank cycle), for the reads of K; and of
    // 16-bit types, four rows' equal quads of slots in four places, for the
    // transpose reads of V.  Bits are only moved, so mix(a | b) = mix(a) ^ mix(b)
    // for a & b = 0.
    static __device__ __forceinline__ constexpr int mix(int row)
    {
        if (sizeof(T) == 4) return row & 15;
        if (kSlots == 8) return (row >> 1 & 1) << 2 | (row >> 3 & 1) << 1 | (row >> 2 & 1);
        return (row & 3) << 2 | (row >> 2 & 3);
    }
    static constexpr int kQ = kSlots / 4;                   // slots of a query row a lane holds
    static constexpr int kD = HD / 16;                      // 16-value pieces of a row
    // keys of a block's tile (K and V, two buffers: 64 KiB at most) and of a
    // wave's own tile (K and V, one buffer: 16 KiB, 32 KiB for fp32 rows of 256)
    static constexpr int kBlockKeys = block_keys(HD * (int)sizeof(T));
    static constexpr int kWaveKeys = wave_keys(HD * (int)sizeof(T));
};

// ---- a tile of keys and values: global -> registers -> LDS --------------------------
// A wave moves KEYS rows of K and of V (64 at most).  A row's slots are read by
// neighbouring lanes; its address is found once, by one lane, and comes to the others
// by a shuffle: page arithmetic in every lane cost more than the products (a prompt
// of 8192 tokens 771 us with it, 700 without).  A key's
// table entry and row in its page advance with the tiles by additions, and the entry
// of the next tile is under way while a tile is.
template <typename T, int HD, int KEYS> struct Stage {
    using G = Geo<T, HD>;
    static constexpr int kWide = CBQ_WAVE / G::kSlots, kPer = KEYS / kWide;     // rows a pass, passes
    static_assert(kWide * kPer == KEYS && KEYS <= CBQ_WAVE, "whole passes, a key a lane");
    u32x4 k[kPer], v[kPer];
    uint64_t there;                         // the loaded tile's keys that are there
    int32_t key, entry, row, id;            // this lane's key: of the next tile
    int32_t step, step_entry, step_row;

    // The walk starts at `first` and goes on in steps of `by` keys.
    __device__ __forceinline__ void start(const AttnArgs &a, const CbqKeys &keys, int32_t first,
                                          int32_t by)
    {
        const int lane = threadIdx.x & 63;
        step = by;
        step_entry = (int32_t)cbq_div((uint32_t)by, a.page);
        step_row = by - step_entry * (int32_t)a.page.d;
        key = lane < KEYS ? first + lane : -1;
        cbq_key_place(keys, a.page, key, entry, row);
        look(keys);
    }
    // keys.end may be larger than the length, until load(): a look waits for no length
    __device__ __forceinline__ void look(const CbqKeys &keys)
    {
        id = -1;
        if (key >= 0 && key < keys.end) id = (key < keys.prefix ? keys.shared : keys.own)[entry];
    }
    // Loads the tile and moves on to the next one's table entries.
    __device__ __forceinline__ void load(const AttnArgs &a, const CbqKeys &keys, int h)
    {
        const int lane = threadIdx.x & 63, from = lane / G::kSlots;
        const int64_t slot = lane % G::kSlots * G::kEl;
        const T *kp = (const T *)a.kv.k + h * a.kv.k_stride[1] + slot;
        const T *vp = (const T *)a.kv.v + h * a.kv.v_stride[1] + slot;
        // an id outside the pool (or no key) reads page 0, row 0 and becomes zeros
        const bool in = id >= 0 && id < a.kv.n_pages && key < keys.end;
        there = __ballot(in);
        const uint32_t p = in ? id : 0, r = in ? row : 0, ko = p * a.k_page + r * a.k_row;
        uint32_t o[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            o[i] = __shfl(ko, i * kWide + from);
            k[i] = *(const u32x4 *)((const char *)kp + (uint64_t)o[i] * a.unit);
        }
        if (!a.one_stride) {
            const uint32_t vo = p * a.v_page + r * a.v_row;
#pragma unroll
            for (int i = 0; i < kPer; i++) o[i] = __shfl(vo, i * kWide + from);
        }
#pragma unroll
        for (int i = 0; i < kPer; i++)
            v[i] = *(const u32x4 *)((const char *)vp + (uint64_t)o[i] * a.unit);
        if (key >= 0) cbq_key_advance(keys, a.page, step, step_entry, step_row, key, entry, row);
        look(keys);
    }
    static constexpr uint64_t kEvery = KEYS == 64 ? ~0ull : (1ull << (KEYS & 63)) - 1;
    __device__ __forceinline__ bool missing() const { return there != kEvery; }
    // place[key]: its place on the joint axis, INT32_MAX for a key that is not there
    __device__ __forceinline__ void store(u32x4 *K, u32x4 *V, int32_t *place, int32_t key0)
    {
        const int lane = threadIdx.x & 63, slot = lane % G::kSlots, sub = lane / G::kSlots;
        if (missing()) {
#pragma unroll
            for (int i = 0; i < kPer; i++)
                if (!(there >> (i * kWide + sub) & 1)) k[i] = v[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int r = i * kWide + sub;
            K[r * G::kSlots + (slot ^ G::mix(r))] = k[i];
            V[r * G::kSlots + (slot ^ G::mix(r))] = v[i];
        }
        if (lane < KEYS) place[lane] = there >> lane & 1 ? key0 + lane : INT32_MAX;
    }
};

// The same for a block's tile, straight into LDS: no registers (with them 700 us,
// without and with the values read ahead of their products 573) and no stores.  A
// lane's 16 bytes land at its place in the wave's 1 KiB, so the slot ^ mix(row)
// order of the tile is made by the lane's choice of global slot; rows that are not
// there come from a slot of zeros.
static __device__ const u32x4 kZeroSlot = {0, 0, 0, 0};

// Written as asm so that the compiler orders no LDS read behind it: stage_wait's
// barriers do.  M0 holds the LDS address; a wait state is needed between its
// write and the load.
__device__ __forceinline__ void copy_slots(uint32_t lds, const void *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(from) : "m0");
}

// Every copy and load of this wave, and its LDS accesses, are done; then all waves'.
__device__ __forceinline__ void stage_wait()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// This wave's number in its stream of four
__device__ __forceinline__ int stream_wave() { return threadIdx.x >> 6 & (kWaves - 1); }

// The same among one stream's four waves: each counts itself in, and waits until four
// times `passed` have.  Its waves pass equally often, so every wait ends.
__device__ __forceinline__ void stream_wait(uint32_t *count, uint32_t &passed)
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if ((threadIdx.x & 63) == 0)
        __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    passed += kWaves;
    while ((uint32_t)__builtin_amdgcn_readfirstlane(__hip_atomic_load(
               count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) < passed)
        __builtin_amdgcn_s_sleep(1);
    asm volatile("" ::: "memory");
}

template <typename T, int HD, int KEYS> struct Copies {
    using G = Geo<T, HD>;
    static constexpr int kRows = kThreads / G::kSlots, kPer = KEYS / kRows;
    static constexpr int kWide = CBQ_WAVE / G::kSlots, kMine = kPer * kWide;
    static_assert(kRows * kPer == KEYS && kMine <= CBQ_WAVE, "whole passes, a key a lane");
    const char *v[kPer];                    // this lane's slots of the values of the tile whose
                                            // keys were asked for last
    int32_t key, entry, row, id;            // this lane's key: of the next tile
    int32_t step_entry, step_row;
    int at;

    __device__ __forceinline__ void start(const AttnArgs &a, const CbqKeys &keys, int32_t first)
    {
        const int lane = threadIdx.x & 63, wave = stream_wave();
        at = lane < kMine ? lane / kWide * kRows + wave * kWide + lane % kWide : -1;
        step_entry = (int32_t)cbq_div((uint32_t)KEYS, a.page);
        step_row = KEYS - step_entry * (int32_t)a.page.d;
        key = at < 0 ? -1 : first + at;
        cbq_key_place(keys, a.page, key, entry, row);
        look(keys);
    }
    __device__ __forceinline__ void look(const CbqKeys &keys)
    {
        id = -1;
        if (key >= 0 && key < keys.end) id = (key < keys.prefix ? keys.shared : keys.own)[entry];
    }
    // Asks for the next tile's keys and writes their places (as Stage) and this wave's
    // flag of one that is not there.
    __device__ __forceinline__ void keys_to(const AttnArgs &a, const CbqKeys &keys, int h, uint32_t lds,
                                            int32_t *place, int32_t *flags)
    {
        const int lane = threadIdx.x & 63, wave = stream_wave(), sub = lane / G::kSlots;
        const bool in = id >= 0 && id < a.kv.n_pages;
        const uint64_t there = __ballot(in);
        constexpr uint64_t every = kMine == 64 ? ~0ull : (1ull << (kMine & 63)) - 1;
        const uint32_t p = in ? id : 0, r = in ? row : 0, ko = p * a.k_page + r * a.k_row;
        const T *kp = (const T *)a.kv.k + h * a.kv.k_stride[1];
        const T *vp = (const T *)a.kv.v + h * a.kv.v_stride[1];
        const int swz = (lane % G::kSlots) ^ G::mix(wave * kWide + sub);
        const char *k[kPer];
        uint32_t o[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            o[i] = __shfl(ko, i * kWide + sub);
            k[i] = (const char *)(kp + (swz ^ G::mix(i * kRows)) * G::kEl) + (uint64_t)o[i] * a.unit;
        }
        if (!a.one_stride) {
            const uint32_t vo = p * a.v_page + r * a.v_row;
#pragma unroll
            for (int i = 0; i < kPer; i++) o[i] = __shfl(vo, i * kWide + sub);
        }
#pragma unroll
        for (int i = 0; i < kPer; i++)
            v[i] = (const char *)(vp + (swz ^ G::mix(i * kRows)) * G::kEl) + (uint64_t)o[i] * a.unit;
        if (there != every) {
#pragma unroll
            for (int i = 0; i < kPer; i++)
                if (!(there >> (i * kWide + sub) & 1)) k[i] = v[i] = (const char *)&kZeroSlot;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) copy_slots(lds + offset(i, wave), k[i]);
        if (at >= 0) place[at] = in ? key : INT32_MAX;
        if (lane == 0) flags[wave] = there != every;
        if (at >= 0)
            cbq_key_advance(keys, a.page, KEYS, step_entry, step_row, key, entry, row);
        look(keys);
    }
    // Asks for the values of the tile whose keys keys_to() asked for last.
    __device__ __forceinline__ void values_to(uint32_t lds)
    {
#pragma unroll
        for (int i = 0; i < kPer; i++) copy_slots(lds + offset(i, stream_wave()), v[i]);
    }
    static __device__ __forceinline__ uint32_t offset(int i, int wave)
    {
        return (uint32_t)((i * kRows + wave * kWide) * G::kSlots * 16);
    }
};

// Whether a tile of values holds one that is not finite; uniform over the wave.
template <typename T, int HD, int KEYS> __device__ __forceinline__ bool odd_tile(const u32x4 *V)
{
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const int lane = threadIdx.x & 63;
    constexpr int kTimes = KEYS * Geo<T, HD>::kSlots / CBQ_WAVE;
    if constexpr (sizeof(T) == 4) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kTimes; i++) {
            const u32x4 w = V[i * CBQ_WAVE + lane];
#pragma unroll
            for (int j = 0; j < 4; j++) top = max(top, w[j] & 0x7fffffffu);
        }
        return __any(top >= 0x7f800000u);
    } else {
        u16x2 top = {0, 0};
#pragma unroll
        for (int i = 0; i < kTimes; i++) {
            const u32x4 w = V[i * CBQ_WAVE + lane];
#pragma unroll
            for (int j = 0; j < 4; j++)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu));
        }
        constexpr uint16_t inf = std::is_same_v<T, __bf16> ? 0x7f80 : 0x7c00;
        return __any(top[0] >= inf || top[1] >= inf);
    }
}

// The order of a stretch of code, for the compiler's scheduler: the first AHEAD
// LDS reads, then GROUPS times matrix instructions and one more read.
template <int GROUPS, int AHEAD, int MFMA> __device__ __forceinline__ void read_ahead()
{
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, MFMA, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
}

// Four values of a row, at hd position d: into the output (part < 0, with the
// row's sum) or a part's sums.
template <typename T, int HD>
__device__ __forceinline__ void put_values(const AttnArgs &a, int part, int64_t token, int head, int d,
                                           f32x4 x, float sum)
{
    const int64_t row = token * a.n_q + head;
    if (part >= 0) {
        *(f32x4 *)(a.part_o + ((int64_t)part * a.N * a.n_q + row) * HD + d) = x;
        return;
    }
    const float f = sum == 0.f ? 0.f : 1.0f / sum;
    x *= f;
    T *y = (T *)a.out + row * HD + d;
    if constexpr (sizeof(T) == 4) *(f32x4 *)y = x;
    else *(u32x2 *)y = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

__device__ __forceinline__ void put_stats(const AttnArgs &a, int part, int64_t token, int head,
                                          float m, float l)
{
    if (part >= 0) a.part_ml[((int64_t)part * a.N + token) * a.n_q + head] = make_float2(m, l);
}

// Keys that the run's token i sees: the prefix, and its own ones up to the token's
__device__ __forceinline__ int32_t row_sees(int32_t prefix, int32_t past, int32_t i)
{
    return prefix + (past + i + 1 > 0 ? past + i + 1 : 0);
}

// Two states of a row to one: m, l and the factors of their values
__device__ __forceinline__ void join(float &m, float &l, float2 other, float &f, float &g)
{
    const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
    f = __builtin_amdgcn_exp2f(m - base);
    g = __builtin_amdgcn_exp2f(other.x - base);
    l = l * f + other.y * g;
    m = top;
}

// 16 bytes of a query (zeros where the row is none), times scale's sign
template <typename T> __device__ __forceinline__ u32x4 query_slot(const AttnArgs &a, const T *x, bool in)
{
    u32x4 w = {0, 0, 0, 0};
    if (in) w = *(const u32x4 *)x;
    if (a.q_mul != 1.0f) {
        union { u32x4 u; T e[16 / sizeof(T)]; } y = {w};
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); i++) y.e[i] = (T)((float)y.e[i] * a.q_mul);
        w = y.u;
    }
    return w;
}

// A score's weight
template <typename T> __device__ __forceinline__ float weight(float s, float c, float c_low, float base)
{
    return __builtin_amdgcn_exp2f(fmaf(s, c, sizeof(T) == 4 ? fmaf(s, c_low, -base) : -base)) * kDown<T>;
}

// ---- RT x 16 query rows of one wave --------------------------------------------------
template <typename T, int HD, int RT> struct Rows {
    using G = Geo<T, HD>;
    u32x4 q[RT][G::kQ];
    f32x4 o[RT][G::kD];
    // m, base (m, or 0 where no key was seen) in exp2's domain; l: this lane's keys only
    float m[RT], base[RT], l[RT];
    int32_t sees[RT];                       // keys of the joint axis that the row sees
    template <int KEYS> using Scores = f32x4[RT][KEYS / 16];

    // Rows first .. first + 16 RT - 1 of n; token0 is the token of row 0.
    __device__ __forceinline__ void load(const AttnArgs &a, int h, int64_t token0, int first, int n)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = first + t * 16 + (lane & 15);
            const int token = r / a.rep;
            const T *x = (const T *)a.q + (token0 + token) * a.q_st[0] +
                         (int64_t)(h * a.rep + r - token * a.rep) * a.q_st[1];
#pragma unroll
            for (int c = 0; c < G::kQ; c++) {
                q[t][c] = query_slot(a, x + (c * 4 + g) * G::kEl, r < n);
            }
#pragma unroll
            for (int d = 0; d < G::kD; d++) o[t][d] = f32x4{0, 0, 0, 0};
            m[t] = -INFINITY;
            base[t] = l[t] = 0.f;
            sees[t] = INT32_MAX;
        }
    }

    // S^T of NK * 16 keys
    template <int NK>
    __device__ __forceinline__ void scores(const u32x4 *K, f32x4 (&s)[RT][NK])
    {
        const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int k = 0; k < NK; k++) {
#pragma unroll
            for (int t = 0; t < RT; t++) s[t][k] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < G::kQ; d++) {
                const u32x4 w = K[(k * 16 + r) * G::kSlots + ((d * 4 + g) ^ G::mix(r))];
#pragma unroll
                for (int t = 0; t < RT; t++) s[t][k] = Mma<T>::qk(w, q[t][d], s[t][k]);
            }
        }
        read_ahead<NK * G::kQ, 4, RT * (sizeof(T) == 4 ? 4 : 1)>();
    }

    // Keys that are not there or that a row does not see: -inf
    template <int NK>
    __device__ __forceinline__ void hide(f32x4 (&s)[RT][NK], const int32_t *place)
    {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const i32x4 at = *(const i32x4 *)(place + k * 16 + 4 * g);
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][k][i] = at[i] < sees[t] ? s[t][k][i] : -INFINITY;
        }
    }

    // Until the scores pass the running maximum by kSlack nothing is rescaled.
    template <int NK> __device__ __forceinline__ void raise(const f32x4 (&s)[RT][NK], float c)
    {
        float x[RT];
        bool over = false;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            x[t] = s[t][0][0];
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[t] = fmaxf(x[t], s[t][k][i]);
            x[t] = groups_max(x[t]) * c;
            over = over || x[t] > m[t] + kOver<T>;
        }
        if (!__any(over)) return;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const float now = fmaxf(m[t], x[t] + kAbove<T>);
            base[t] = now == -INFINITY ? 0.f : now;         // a row that has seen no key
            const float f = __builtin_amdgcn_exp2f(m[t] - base[t]);
            l[t] *= f;
#pragma unroll
            for (int d = 0; d < G::kD; d++) o[t][d] *= f;
            m[t] = now;
        }
    }

    // Row r sees the prefix and the own keys up to its token's
    __device__ __forceinline__ void see(const AttnArgs &a, int32_t prefix, int32_t past, int first)
    {
#pragma unroll
        for (int t = 0; t < RT; t++)
            sees[t] = row_sees(prefix, past, (first + t * 16 + (int)(threadIdx.x & 15)) / a.rep);
    }

    __device__ __forceinline__ void put(const AttnArgs &a, int part, int h, int64_t token0, int first,
                                        int n)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = first + t * 16 + (lane & 15);
            const float total = groups_sum(l[t]);
            if (r >= n) continue;
            const int64_t token = token0 + r / a.rep;
            const int head = h * a.rep + r % a.rep;
#pragma unroll
            for (int d = 0; d < G::kD; d++)
                put_values<T, HD>(a, part, token, head, d * 16 + 4 * (lane >> 4), o[t][d], total);
            if (lane < 16) put_stats(a, part, token, head, m[t], total);
        }
    }

    // The state to LDS, and another wave's of the same rows, given there by the same
    // lane, into this one
    static constexpr int kGiven = RT * G::kD;
    __device__ __forceinline__ void give(f32x4 *x, float2 *ml) const
    {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            ml[t * kThreads] = make_float2(m[t], l[t]);
#pragma unroll
            for (int d = 0; d < G::kD; d++) x[(t * G::kD + d) * kThreads] = o[t][d];
        }
    }
    __device__ __forceinline__ void take(const f32x4 *x, const float2 *ml)
    {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            float f, g;
            join(m[t], l[t], ml[t * kThreads], f, g);
#pragma unroll
            for (int d = 0; d < G::kD; d++) o[t][d] = o[t][d] * f + x[(t * G::kD + d) * kThreads] * g;
        }
    }

    // Four scores to weights, added to the row's sum
    __device__ __forceinline__ f32x4 weigh(int t, f32x4 s, float c, float c_low)
    {
        f32x4 p;
#pragma unroll
        for (int i = 0; i < 4; i++)
            p[i] = weight<T>(s[i], c, c_low, base[t]);
        l[t] += (p[0] + p[1]) + (p[2] + p[3]);
        return p;
    }

    // Weights of the tile, and the values under them
    template <int NK>
    __device__ __forceinline__ void values(const u32x4 *V, const f32x4 (&s)[RT][NK], float c, float c_low)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
        if constexpr (sizeof(T) == 4) {
            const float *F = (const float *)V;
#pragma unroll
            for (int k = 0; k < NK; k++) {
                f32x4 p[RT];
#pragma unroll
                for (int t = 0; t < RT; t++) p[t] = weigh(t, s[t][k], c, c_low);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int key = k * 16 + 4 * g + i;
#pragma unroll
                    for (int d = 0; d < G::kD; d++) {
                        const float w = F[(key * G::kSlots + ((d * 4 + (r >> 2)) ^ G::mix(key)))
                                          * 4 + (r & 3)];
#pragma unroll
                        for (int t = 0; t < RT; t++)
                            o[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, p[t][i], o[t][d], 0, 0,
                                                                           0);
                    }
                }
            }
        } else {
            // lane (g, r) points the transpose read at key 4g + r / 4, values
            // 4 (r % 4) .. + 3 and gets keys 4g .. 4g + 3 of value r
            const int key = 4 * g + (r >> 2), half = r & 1, sub = (r & 3) >> 1;
            auto piece = [&](int k, int d) {
                const int row = k * 16 + key;
                const u32x4 *p = V + row * G::kSlots + ((d * 2 + sub) ^ G::mix(row));
                return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4 *)((const u32x2 *)p + half)));
            };
            if constexpr (NK % 2 == 0) {
                // Two 16-key tiles side by side are one product's keys.  Four pieces
                // of hd are read while the four before them are in the products, and
                // the weights of the next two tiles are made beside them.
                constexpr int kParts = G::kD / 4, kAll = NK / 2 * kParts, kUnits = 2 * RT / kParts;
                u32x2 v[2][4][2];
                u32x4 p[2][RT];
                auto read = [&](int j) {
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        v[j & 1][d][0] = piece(j / kParts * 2, j % kParts * 4 + d);
                        v[j & 1][d][1] = piece(j / kParts * 2 + 1, j % kParts * 4 + d);
                    }
                };
                auto weights = [&](int pair, int u) {       // unit u of the pair: 4 scores a lane
                    const int t = u / 2, k = u % 2;
                    const f32x4 x = weigh(t, s[t][pair * 2 + k], c, c_low);
                    p[pair & 1][t][k * 2] = pack2<T>(x[0], x[1]);
                    p[pair & 1][t][k * 2 + 1] = pack2<T>(x[2], x[3]);
                };
                read(0);
#pragma unroll
                for (int u = 0; u < 2 * RT; u++) weights(0, u);
#pragma unroll
                for (int j = 0; j < kAll; j++) {
                    const int pair = j / kParts;
                    if (j + 1 < kAll) read(j + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        const u32x2 x = v[j & 1][d][0], y = v[j & 1][d][1];
                        const u32x4 w = {x[0], x[1], y[0], y[1]};
#pragma unroll
                        for (int t = 0; t < RT; t++)
                            o[t][j % kParts * 4 + d] = Mma<T>::qk(w, p[pair & 1][t],
                                                                  o[t][j % kParts * 4 + d]);
                    }
                    if (pair + 1 < NK / 2) {
#pragma unroll
                        for (int u = 0; u < kUnits; u++) weights(pair + 1, j % kParts * kUnits + u);
#pragma unroll
                        for (int i = 0; i < 4 * RT; i++) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, (10 * kUnits + 4 * RT - 1) / (4 * RT), 0);
                            __builtin_amdgcn_sched_group_barrier(0x400, (4 * kUnits + 4 * RT - 1) / (4 * RT), 0);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                static_assert(NK == 1, "one 16-key piece");
                u32x2 p[RT];
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const f32x4 x = weigh(t, s[t][0], c, c_low);
                    p[t] = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
                }
#pragma unroll
                for (int d = 0; d < G::kD; d++) {
                    const u32x2 w = piece(0, d);
#pragma unroll
                    for (int t = 0; t < RT; t++) o[t][d] = Mma<T>::pv16(w, p[t], o[t][d]);
                }
            }
        }
    }
};

// ---- 32 query rows of one wave, 16-bit types --------------------------------------------
// Rows for 32 rows on the 32x32x16 products: half the matrix instructions, one row
// a lane (lane % 32), and the vector unit overlaps them better (with four additions
// a 16 cycles of product, 18 % less time a product than 16x16x32).  A lane has keys
// 8 (i / 4) + 4 (lane / 32) + i % 4 of a 32-key tile, i < 16; eight of them are the
// right operand of a 16-key value product.
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c, __bf16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c, _Float16)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <typename T, int HD> struct Rows32 {
    using G = Geo<T, HD>;
    static constexpr int kC = HD / 16, kO = HD / 32;
    u32x4 q[kC];
    f32x16 o[kO];
    float m, base, l;                       // as Rows; l: this lane's keys only
    int32_t sees;
    template <int KEYS> using Scores = f32x16[KEYS / 32];

    __device__ __forceinline__ void load(const AttnArgs &a, int h, int64_t token0, int first, int n)
    {
        const int lane = threadIdx.x & 63, r = first + (lane & 31), token = r / a.rep;
        const T *x = (const T *)a.q + (token0 + token) * a.q_st[0] +
                     (int64_t)(h * a.rep + r - token * a.rep) * a.q_st[1];
#pragma unroll
        for (int c = 0; c < kC; c++) q[c] = query_slot(a, x + (c * 2 + (lane >> 5)) * G::kEl, r < n);
#pragma unroll
        for (int d = 0; d < kO; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.f;
        m = -INFINITY;
        base = l = 0.f;
        sees = INT32_MAX;
    }

    template <int NK> __device__ __forceinline__ void scores(const u32x4 *K, f32x16 (&s)[NK])
    {
        const int lane = threadIdx.x & 63, r = lane & 31;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[k][i] = 0.f;
#pragma unroll
        for (int c = 0; c < kC; c++)
#pragma unroll
            for (int k = 0; k < NK; k++)
                s[k] = mma32(K[(k * 32 + r) * G::kSlots + ((c * 2 + (lane >> 5)) ^ G::mix(r))], q[c],
                             s[k], T());
        read_ahead<NK * kC, 4, 1>();
    }

    template <int NK> __device__ __forceinline__ void hide(f32x16 (&s)[NK], const int32_t *place)
    {
        const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const i32x4 at = *(const i32x4 *)(place + k * 32 + 8 * j + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    s[k][4 * j + i] = at[i] < sees ? s[k][4 * j + i] : -INFINITY;
            }
    }

    template <int NK> __device__ __forceinline__ void raise(const f32x16 (&s)[NK], float c)
    {
        float x = s[0][0];
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int i = 0; i < 16; i++) x = fmaxf(x, s[k][i]);
        auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1])) * c;
        if (!__any(x > m + kOver<T>)) return;
        x = fmaxf(m, x + kAbove<T>);
        base = x == -INFINITY ? 0.f : x;
        const float f = __builtin_amdgcn_exp2f(m - base);
        l *= f;
#pragma unroll
        for (int d = 0; d < kO; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= f;
        m = x;
    }

    __device__ __forceinline__ void see(const AttnArgs &a, int32_t prefix, int32_t past, int first)
    {
        sees = row_sees(prefix, past, (first + (int)(threadIdx.x & 31)) / a.rep);
    }

    __device__ __forceinline__ void put(const AttnArgs &a, int part, int h, int64_t token0, int first,
                                        int n)
    {
        const int lane = threadIdx.x & 63, r = first + (lane & 31);
        auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        const float total = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        if (r >= n) return;
        const int64_t token = token0 + r / a.rep;
        const int head = h * a.rep + r % a.rep;
#pragma unroll
        for (int d = 0; d < kO; d++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                put_values<T, HD>(a, part, token, head, d * 32 + 8 * j + 4 * (lane >> 5),
                                  f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]},
                                  total);
        if (lane < 32) put_stats(a, part, token, head, m, total);
    }

    static constexpr int kGiven = HD / 8;
    __device__ __forceinline__ void give(f32x4 *x, float2 *ml) const
    {
        *ml = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < kO; d++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[(d * 4 + j) * kThreads] = f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2],
                                                  o[d][4 * j + 3]};
    }
    __device__ __forceinline__ void take(const f32x4 *x, const float2 *ml)
    {
        float f, g;
        join(m, l, *ml, f, g);
#pragma unroll
        for (int d = 0; d < kO; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4 y = x[(d * 4 + j) * kThreads];
#pragma unroll
                for (int i = 0; i < 4; i++) o[d][4 * j + i] = o[d][4 * j + i] * f + y[i] * g;
            }
    }

    // Weights of the tile, and the values under them: 16 keys' values are read while
    // the 16 before them are in the products, beside which the 16 keys' weights after
    // them are made.
    template <int NK>
    __device__ __forceinline__ void values(const u32x4 *V, const f32x16 (&s)[NK], float c, float)
    {
        const int lane = threadIdx.x & 63, r = lane & 15;
        const int key = 4 * (lane >> 5) + (r >> 2), sub = (lane >> 4 & 1) * 2 + ((r & 3) >> 1);
        auto piece = [&](int row0, int d) {
            const int row = row0 + key;
            const u32x4 *p = V + row * G::kSlots + ((d * 4 + sub) ^ G::mix(row));
            return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4 *)((const u32x2 *)p + (r & 1))));
        };
        u32x2 v[2][kO][2];
        u32x4 p[2];
        auto read = [&](int j) {
#pragma unroll
            for (int d = 0; d < kO; d++) {
                v[j & 1][d][0] = piece(j * 16, d);
                v[j & 1][d][1] = piece(j * 16 + 8, d);
            }
        };
        auto weigh = [&](int j) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = weight<T>(s[j / 2][j % 2 * 8 + i], c, 0.f, base);
            l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            p[j & 1] = u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                             pack2<T>(x[6], x[7])};
        };
        read(0);
        weigh(0);
#pragma unroll
        for (int j = 0; j < 2 * NK; j++) {
            if (j + 1 < 2 * NK) read(j + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < kO; d++) {
                const u32x2 x = v[j & 1][d][0], y = v[j & 1][d][1];
                o[d] = mma32(u32x4{x[0], x[1], y[0], y[1]}, p[j & 1], o[d], T());
            }
            if (j + 1 < 2 * NK) {
                weigh(j + 1);
#pragma unroll
                for (int i = 0; i < kO; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 20 / kO, 0);
                    __builtin_amdgcn_sched_group_barrier(0x400, 8 / kO, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// ---- rows key by key --------------------------------------------------------------------
// A weight of 0 times an infinite value is no number, so in a matrix product a key
// that only some of the rows see would reach the others too.  Blocks whose causal
// masks cut a tile with such a value leave their products and do their rows `row0`
// .. `row0 + m - 1` here, a wave a row, a lane a key, where a hidden key's value is
// never touched.
template <typename T, int HD>
__device__ __forceinline__ void plain_rows(const AttnArgs &a, int h, int64_t token0, int row0, int m,
                                           int n, const CbqKeys &keys, int32_t first, int32_t past,
                                           int part)
{
    using G = Geo<T, HD>;
    constexpr int kLane = HD / CBQ_WAVE;
    const int lane = threadIdx.x & 63;
    const int stop = row0 + m < n ? row0 + m : n;
    for (int r = row0 + (int)(threadIdx.x >> 6); r < stop; r += blockDim.x >> 6) {
        const int token = r / a.rep, head = h * a.rep + r - token * a.rep;
        const T *x = (const T *)a.q + (token0 + token) * a.q_st[0] + head * a.q_st[1];
        const int32_t sees = row_sees(keys.prefix, past, token), end = sees < keys.end ? sees : keys.end;
        float top = -INFINITY, l = 0.f, o[kLane] = {};
        for (int32_t key0 = first; key0 < end; key0 += CBQ_WAVE) {
            const int32_t key = key0 + lane;
            int32_t entry, row, id = -1;
            cbq_key_place(keys, a.page, key, entry, row);
            if (key < end) id = (key < keys.prefix ? keys.shared : keys.own)[entry];
            const bool in = id >= 0 && id < a.kv.n_pages;
            const int64_t p = in ? id : 0, at = in ? row : 0;
            const T *k = (const T *)a.kv.k + p * a.kv.k_stride[0] + h * a.kv.k_stride[1] +
                         at * a.kv.k_stride[2];
            const int64_t vo = p * a.kv.v_stride[0] + at * a.kv.v_stride[2];
            float s = 0.f;
            for (int c = 0; c < G::kSlots; c++) {
                union { u32x4 u; T e[G::kEl]; } kw = {*(const u32x4 *)(k + c * G::kEl)},
                                                qw = {query_slot(a, x + c * G::kEl, true)};
                for (int i = 0; i < G::kEl; i++) s = fmaf((float)kw.e[i], (float)qw.e[i], s);
            }
            float now = in ? s : -INFINITY;
            for (int i = 32; i > 0; i >>= 1) now = fmaxf(now, __shfl_xor(now, i));
            now = fmaxf(top, now * a.c + kAbove<T>);
            const float base = now == -INFINITY ? 0.f : now, f = __builtin_amdgcn_exp2f(top - base);
            const float w = in ? weight<T>(s, a.c, a.c_low, base) : 0.f;
            top = now;
            l = l * f + w;
            for (int i = 0; i < kLane; i++) o[i] *= f;
            for (uint64_t b = __ballot(in); b; b &= b - 1) {
                const int at = __builtin_ctzll(b);
                const float wk = __shfl(w, at);
                const T *v = (const T *)a.kv.v + h * a.kv.v_stride[1] + lane * kLane +
                             ((int64_t)__shfl((int)(vo >> 32), at) << 32 |
                              (uint32_t)__shfl((int)(uint32_t)vo, at));
                for (int i = 0; i < kLane; i++) o[i] = fmaf(wk, (float)v[i], o[i]);
            }
        }
        for (int i = 32; i > 0; i >>= 1) l += __shfl_xor(l, i);
        const int64_t at = (token0 + token) * a.n_q + head;
        for (int i = 0; i < kLane; i++) {
            if (part >= 0) a.part_o[((int64_t)part * a.N * a.n_q + at) * HD + lane * kLane + i] = o[i];
            else ((T *)a.out)[at * HD + lane * kLane + i] = (T)(l == 0.f ? 0.f : o[i] / l);
        }
        if (lane == 0) put_stats(a, part, token0 + token, head, top, l);
    }
}

template <typename T, int HD> constexpr int block_lds()
{
    using G = Geo<T, HD>;
    return 4 * G::kBlockKeys * G::kSlots * 16 + 2 * G::kBlockKeys * 4 + 2 * kWaves * 4;
}

// ---- 64 RT rows of a block against keys [first, end), tiles shared by the waves ----------
// 64 keys of K and V (rows of 256 bytes) in two buffers of 32 KiB, so that two blocks
// share a CU.  32 rows a wave: 16 take 772 us instead of 560 for 8192 tokens (LDS
// reads double).  Blocks of eight waves take 529 there, but 297 instead of 286 for
// 16 ragged prompts and 366 instead of 327 at hd 64; deeper rings of tiles gain
// nothing, and 32 rows of 512 bytes, which leave one wave a SIMD, lose (67 us
// instead of 48 for two chunks against 20000 keys).
//
// With STREAMS 2 eight waves are two such groups, each with a half of the keys,
// tiles and buffers of its own, in no step with the other (waits of all eight: 53 us
// instead of 48 for two chunks against 20000 keys); their states are joined in LDS
// at the end.  For grids of a block a CU, where four waves leave a SIMD one: bf16, 32
// heads on 8 of 128, 512 tokens behind 1500 shared keys 37 us instead of 45, 1024 56
// instead of 65; with more blocks two of four waves do as well (8192 tokens).
template <typename T, int HD, int RT, bool CAUSAL, int STREAMS = 1>
__device__ __forceinline__ void block_rows(const AttnArgs &a, char *lds, int h, int64_t token0,
                                           int row0, int n, const CbqKeys &whole, int32_t from,
                                           int32_t past, int part)
{
    using G = Geo<T, HD>;
    constexpr int KEYS = G::kBlockKeys, kTile = KEYS * G::kSlots;
    constexpr uint32_t kBytes = kTile * 16;
    const int all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = STREAMS > 1 ? all_wave & (kWaves - 1) : all_wave;
    const int stream = STREAMS > 1 ? all_wave / kWaves : 0;
    CbqKeys keys = whole;
    int32_t first = from;
    if (STREAMS > 1) stream_keys(from, whole.end, KEYS, STREAMS, stream, first, keys.end);
    char *mem = lds + stream * block_lds<T, HD>();
    u32x4 *K = (u32x4 *)mem, *V = K + 2 * kTile;
    int32_t *place = (int32_t *)(V + 2 * kTile), *flags = place + 2 * KEYS;
    const uint32_t lds_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)mem,
                   lds_v = lds_k + 2 * kBytes;
    const int mine = row0 + wave * 16 * RT;
    std::conditional_t<RT == 2 && sizeof(T) == 2, Rows32<T, HD>, Rows<T, HD, RT>> w;
    Copies<T, HD, KEYS> st;
    st.start(a, keys, first);
    w.load(a, h, token0, mine, n);
    int32_t all = INT32_MAX;                    // keys that every row of the block sees
    if (CAUSAL) {
        all = row_sees(keys.prefix, past, row0 / a.rep);
        w.see(a, keys.prefix, past, mine);
    }
    const int tiles = keys.end > first ? (keys.end - first + KEYS - 1) / KEYS : 0;
    uint32_t *counts = (uint32_t *)(lds + STREAMS * block_lds<T, HD>()), passed = 0;
    if (STREAMS > 1) {
        if (threadIdx.x < STREAMS) counts[threadIdx.x] = 0;
        __syncthreads();
    }
    auto wait = [&]() {
        if (STREAMS > 1) stream_wait(counts + stream, passed);
        else stage_wait();
    };
    auto step = [&](int i, int b) -> bool {                 // false: a value that is not finite
        if (i + 1 < tiles) {
            st.keys_to(a, keys, h, lds_k + (b ^ 1) * kBytes, place + (b ^ 1) * KEYS,
                       flags + (b ^ 1) * kWaves);
            st.values_to(lds_v + (b ^ 1) * kBytes);
        }
        const int32_t key0 = first + i * KEYS;
        if (CAUSAL && key0 + KEYS > all && odd_tile<T, HD, KEYS>(V + b * kTile)) return false;
        const int4 miss = *(const int4 *)(flags + b * kWaves);
        typename decltype(w)::template Scores<KEYS> s;
        __builtin_amdgcn_sched_barrier(0);
        w.scores(K + b * kTile, s);
        if (key0 + KEYS > all || __builtin_amdgcn_readfirstlane(miss.x | miss.y | miss.z | miss.w))
            w.hide(s, place + b * KEYS);
        w.raise(s, a.c);
        w.values(V + b * kTile, s, a.c, a.c_low);
        wait();
        return true;
    };
    bool fine = true;                           // every wave looks at all of a tile: uniform
    if (tiles > 0) {
        st.keys_to(a, keys, h, lds_k, place, flags);
        st.values_to(lds_v);
        wait();
        for (int i = 0;; i += 2) {
            fine = step(i, 0);
            if (!fine || i + 1 >= tiles) break;
            fine = step(i + 1, 1);
            if (!fine || i + 2 >= tiles) break;
        }
    }
    if (CAUSAL && !fine) wait();                // no copy is under way when the block ends
    bool odd = CAUSAL && !fine;
    if (STREAMS > 1) odd = __syncthreads_or(odd);
    if (CAUSAL && odd) {
        plain_rows<T, HD>(a, h, token0, row0, 16 * RT * kWaves, n, whole, from, past, part);
        return;
    }
    if constexpr (STREAMS > 1) {
        static_assert(kThreads * (decltype(w)::kGiven * 16 + RT * 8) <= STREAMS * block_lds<T, HD>(),
                      "a stream's state");
        f32x4 *x = (f32x4 *)lds + (threadIdx.x & (kThreads - 1));
        float2 *ml = (float2 *)((f32x4 *)lds + decltype(w)::kGiven * kThreads) +
                     (threadIdx.x & (kThreads - 1));
        if (stream) w.give(x, ml);
        __syncthreads();
        if (stream) return;
        w.take(x, ml);
    }
    w.put(a, part, h, token0, mine, n);
}

// ---- 16 rows of a block, the keys [first, end) dealt to its waves ------------------------
// For few rows: each wave walks tiles of its own (8 KiB of K and of V) through its
// own LDS without a barrier, and the four running states are merged at the end.  A
// decoder's rows of one sequence fill a quarter of a 16-row product or less; the
// bytes bound them, and two blocks a CU keep 128 KiB under way.  200 fp32 prompt
// tokens take 14 us this way, 23 with 64 rows a block.
template <typename T, int HD, bool CAUSAL>
__device__ __forceinline__ void wave_rows(const AttnArgs &a, char *lds, int h, int64_t token0,
                                          int row0, int n, CbqKeys keys, int32_t first,
                                          int32_t past, int part, const int32_t *length = nullptr,
                                          bool always = false)
{
    using G = Geo<T, HD>;
    constexpr int KEYS = G::kWaveKeys, kTile = KEYS * G::kSlots;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, r = lane & 15;
    u32x4 *K = (u32x4 *)lds + wave * 2 * kTile, *V = K + kTile;
    int32_t *place = (int32_t *)((u32x4 *)lds + kWaves * 2 * kTile) + wave * KEYS;
    Rows<T, HD, 1> w;
    Stage<T, HD, KEYS> st;
    st.start(a, keys, first + wave * KEYS, kWaves * KEYS);
    w.load(a, h, token0, row0, n);
    int32_t all = INT32_MAX;
    if (CAUSAL) {
        all = row_sees(keys.prefix, past, row0 / a.rep);
        w.see(a, keys.prefix, past, row0);
    }
    if (length) {                               // decode: the own keys end there
        const int32_t end = keys.prefix + cbq_clamp_length(*length, a.capacity);
        if (first >= end && !always) return;    // the merge counts own parts by the length
        if (end < keys.end) keys.end = end;
    }
    const int32_t begin = first + wave * KEYS, step = kWaves * KEYS;
    int odd = 0;                                // a value that is not finite
    if (begin < keys.end) st.load(a, keys, h);
    for (int32_t key0 = begin; key0 < keys.end; key0 += step) {
        const bool missing = st.missing();
        st.store(K, V, place, key0);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (key0 + step < keys.end) st.load(a, keys, h);
        if (CAUSAL && key0 + KEYS > all && odd_tile<T, HD, KEYS>(V)) {
            odd = 1;
            break;
        }
        f32x4 s[1][KEYS / 16];
        w.scores(K, s);
        if (missing || key0 + KEYS > all) w.hide(s, place);
        w.raise(s, a.c);
        w.values(V, s, a.c, a.c_low);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // merge: statistics first, then the weighted values, each wave's scaled to
    // the common maximum
    if (CAUSAL) {
        if (__syncthreads_or(odd)) {
            plain_rows<T, HD>(a, h, token0, row0, 16, n, keys, first, past, part);
            return;
        }
    } else {
        __syncthreads();                        // every wave is past its tiles
    }
    float *O = (float *)lds, *ML = O + kWaves * 16 * HD;
    const float l = groups_sum(w.l[0]);
    if (lane < 16) {
        ML[(wave * 16 + r) * 2] = w.m[0];
        ML[(wave * 16 + r) * 2 + 1] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; i++) top = fmaxf(top, ML[(i * 16 + r) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < kWaves; i++)
        sum += __builtin_amdgcn_exp2f(ML[(i * 16 + r) * 2] - base) * ML[(i * 16 + r) * 2 + 1];
    const float f = __builtin_amdgcn_exp2f(w.m[0] - base);
    // row r's pieces at (piece ^ r): 16 rows of one piece would share their banks
#pragma unroll
    for (int d = 0; d < G::kD; d++)
        *(f32x4 *)(O + (wave * 16 + r) * HD + (((d * 4 + g) ^ r) & (HD / 4 - 1)) * 4) = w.o[0][d] * f;
    if (wave == 0 && lane < 16) ML[kWaves * 32 + r] = sum;
    __syncthreads();
    const int rows = n - row0 < 16 ? n - row0 : 16;
    for (int e = tid; e < rows * (HD / 4); e += kThreads) {
        const int rr = e / (HD / 4), d = e % (HD / 4);
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kWaves; i++)
            x += *(const f32x4 *)(O + (i * 16 + rr) * HD + ((d ^ rr) & (HD / 4 - 1)) * 4);
        const int token = (row0 + rr) / a.rep;
        put_values<T, HD>(a, part, token0 + token, h * a.rep + row0 + rr - token * a.rep, d * 4, x,
                          ML[kWaves * 32 + rr]);
    }
    if (wave == 0 && lane < rows) {
        const int token = (row0 + r) / a.rep;
        put_stats(a, part, token0 + token, h * a.rep + row0 + r - token * a.rep, top, sum);
    }
}

// Waves a SIMD, and so blocks a CU, whose loads, products and exponentials overlap
// (one: 1627 us instead of 771 for 8192 tokens); rows of 1024 bytes need a wave's
// whole register file.
constexpr int simd_waves(int row_bytes) { return row_bytes <= 512 ? 2 : 1; }

template <typename T, int HD> constexpr int wave_lds()
{
    using G = Geo<T, HD>;
    constexpr int tiles = kWaves * (2 * G::kWaveKeys * G::kSlots * 16 + G::kWaveKeys * 4);
    constexpr int merge = kWaves * 16 * HD * 4 + kWaves * 16 * 8 + 16 * 4;
    return tiles > merge ? tiles : merge;
}

// ---- decode: parts of the prefix for all sequences, parts of each one's own keys ------------
// PT: 64 PT prefix rows a block; 0: the prefix rows are 16 at most and go as the
// own ones do.
template <typename T, int HD, int PT>
__global__ __launch_bounds__(kThreads, simd_waves(HD * (int)sizeof(T))) void decode_kernel(AttnArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const DecodeWork w = decode_work(a.plan, cbq_block(blockIdx.x, blockIdx.y), a.kv.n_kv, a.batch, a.prefix,
                                     a.capacity);
    if (w.part >= a.plan.parts) return;             // past the plan's last block
    const int to = a.plan.parts > 1 ? w.part : -1;
    if (w.seq < 0) {
        const CbqKeys keys = {a.prefix_table, nullptr, a.prefix, w.end};
        const int rows = a.batch * a.rep;
        if constexpr (PT > 0)
            block_rows<T, HD, PT, false>(a, lds, w.h, 0, w.tile * 64 * PT, rows, keys, w.first, 0, to);
        else
            wave_rows<T, HD, false>(a, lds, w.h, 0, w.tile * 16, rows, keys, w.first, 0, to);
        return;
    }
    const CbqKeys keys = {a.prefix_table, a.tables + w.seq * a.table_st, a.plan.joint ? a.prefix : 0,
                          w.end};
    wave_rows<T, HD, false>(a, lds, w.h, w.seq, w.tile * 16, a.rep, keys, w.first, 0, to,
                            a.lengths + w.seq, a.plan.parts == 1);
}

// ---- prompt: tiles of each run's rows against the keys they see -----------------------------
// RT: 64 RT rows a block; 0: 16 rows.
template <typename T, int HD, int RT, int STREAMS = 1>
__global__ __launch_bounds__(STREAMS * kThreads, simd_waves(HD * (int)sizeof(T))) void prompt_kernel(AttnArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int M = RT ? 64 * RT : 16;
    const int lane = threadIdx.x & 63, n_kv = a.kv.n_kv;
    const uint32_t block = cbq_block(blockIdx.x, blockIdx.y);
    uint32_t i = block;
    const int h = i % n_kv;
    i /= n_kv;
    const int part = i % a.plan.parts;
    // later tiles of a run see more keys: they start first
    int32_t want = a.plan.tiles - 1 - (int32_t)(i / a.plan.parts);
    if (block == 0) {                               // tokens of no run
        const int64_t lo = cbq_clamp_length(a.q_start[0], a.N),
                      hi = cbq_max(cbq_clamp_length(a.q_start[a.batch], a.N), lo);
        T *out = (T *)a.out;
        const int64_t w = (int64_t)a.n_q * HD;
        for (int64_t e = threadIdx.x; e < (lo + a.N - hi) * w; e += STREAMS * kThreads)
            out[e < lo * w ? e : e + (hi - lo) * w] = (T)0.f;
    }
    // the run that holds tile `want`: its count of tiles, summed over the runs (none
    // past the plan's last block)
    int32_t before = 0, run = -1, tile = 0, first_token = 0, count = 0, length = 0;
    for (int b0 = want < 0 ? a.batch : 0; b0 < a.batch && run < 0; b0 += CBQ_WAVE) {
        int32_t f = 0, n = 0, len = 0;
        if (b0 + lane < a.batch) {
            cbq_run(a.q_start, b0 + lane, a.N, f, n);
            len = a.lengths[b0 + lane];
        }
        const int32_t mine = (int32_t)(((int64_t)n * a.rep + M - 1) / M);
        int32_t upto = mine;
        for (int o = 1; o < CBQ_WAVE; o <<= 1) {
            const int32_t x = __shfl_up(upto, o);
            if (lane >= o) upto += x;
        }
        const uint64_t over = __ballot(before + upto > want);
        if (over) {
            const int at = __builtin_ctzll(over);
            run = b0 + at;
            tile = want - before - __shfl(upto - mine, at);
            first_token = __shfl(f, at);
            count = __shfl(n, at);
            length = __shfl(len, at);
        } else {
            before += __shfl(upto, CBQ_WAVE - 1);
        }
    }
    run = __builtin_amdgcn_readfirstlane(run);
    if (run < 0) return;                            // fewer tiles than the grid allows for
    tile = __builtin_amdgcn_readfirstlane(tile);
    first_token = __builtin_amdgcn_readfirstlane(first_token);
    count = __builtin_amdgcn_readfirstlane(count);
    const int32_t len = cbq_clamp_length(__builtin_amdgcn_readfirstlane(length), a.capacity),
                  past = len - count;
    const int rows = count * a.rep, row0 = tile * M;
    const int last = (row0 + M < rows ? row0 + M : rows) - 1;
    const int32_t sees = row_sees(a.prefix, past, last / a.rep);        // of the tile's last row
    int32_t first = 0, end = sees;
    if (a.plan.parts > 1)
        prompt_keys(sees, a.plan.parts, part,
                    RT ? Geo<T, HD>::kBlockKeys : Geo<T, HD>::kWaveKeys, first, end);
    const CbqKeys keys = {a.prefix_table, a.tables + run * a.table_st, a.prefix, end};
    if constexpr (RT > 0)
        block_rows<T, HD, RT, true, STREAMS>(a, lds, h, first_token, row0, rows, keys, first, past,
                                             a.plan.parts > 1 ? part : -1);
    else
        wave_rows<T, HD, true>(a, lds, h, first_token, row0, rows, keys, first, past,
                               a.plan.parts > 1 ? part : -1);
}

// ---- merge of the parts: W waves a (token, head) -----------------------------------------------
// HD / 4 lanes take a part's values, so a row has 256 W / HD parts under way at
// once; the first of them are requested before the common maximum is known.  A
// whole block a row for few rows and many parts (a wave a row that walks 40 parts
// took 14 us, a block 5), a wave a row for many (9888 rows of 6 parts: 41 us with
// the prompt, 30).
template <typename T, int HD, int W> __global__ __launch_bounds__(kThreads) void merge_kernel(AttnArgs a)
{
    constexpr int kLanes = HD / 4, kGroups = W * CBQ_WAVE / kLanes, kAhead = 4;
    __shared__ __attribute__((aligned(16))) float sums[kThreads / kLanes][HD];
    __shared__ float totals[kThreads / kLanes];
    const int tid = threadIdx.x, lane = tid & 63, all = tid / kLanes, d = tid % kLanes * 4;
    const int group = all % kGroups;
    const int64_t rows = (int64_t)a.N * a.n_q, block = cbq_block(blockIdx.x, blockIdx.y),
                  row = block * (kWaves / W) + all / kGroups, token = row / a.n_q;
    if (row >= rows) return;                        // whole waves; the barrier counts the rest
    // The first parts' loads wait for no length: what a part that was not written
    // holds is dropped.
    const int most = a.plan.parts;
    f32x4 o[kAhead];
    float2 ml[kAhead];
    auto part = [&](int p, f32x4 &x, float2 &s) {
        x = f32x4{0, 0, 0, 0};
        s = make_float2(-INFINITY, 0.f);
        if (p < most) {
            x = *(const f32x4 *)(a.part_o + (p * rows + row) * HD + d);
            s = a.part_ml[p * rows + row];
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++) part(group + i * kGroups, o[i], ml[i]);
    float m0 = lane < most ? a.part_ml[lane * rows + row].x : -INFINITY;
    int parts = most;
    if (a.plan.own_chunk > 0) {                     // decode: as many own parts as the length has
        const int32_t len = cbq_clamp_length(a.lengths[token], a.capacity);
        parts = a.plan.pre_parts + (int)cbq_ceil(len, a.plan.own_chunk);
    } else {                                        // prompt: a token of no run keeps its zeros
        if (token < a.q_start[0] || token >= a.q_start[a.batch]) return;
    }
    float top = lane < parts ? m0 : -INFINITY;
    for (int p = lane + CBQ_WAVE; p < parts; p += CBQ_WAVE)
        top = fmaxf(top, a.part_ml[p * rows + row].x);
    for (int i = 32; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 x = {0, 0, 0, 0};
    float sum = 0.f;
    for (int p0 = group;; p0 += kAhead * kGroups) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const bool in = p0 + i * kGroups < parts;
            const float w = in ? __builtin_amdgcn_exp2f(ml[i].x - base) : 0.f;
            sum += in ? w * ml[i].y : 0.f;          // 0 of an empty part; a NaN stays
            // the values of a part that saw no key are not written
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = w == 0.f ? x[e] : fmaf(w, o[i][e], x[e]);
        }
        if (p0 + kAhead * kGroups >= parts) break;
#pragma unroll
        for (int i = 0; i < kAhead; i++)
            part(p0 + (kAhead + i) * kGroups, o[i], ml[i]);
    }
    if constexpr (kGroups > 1) {
        *(f32x4 *)&sums[all][d] = x;
        if (tid % kLanes == 0) totals[all] = sum;
        if constexpr (W > 1) {
            __syncthreads();
        } else {                                    // the wave's own
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        if (group > 0) return;
#pragma unroll
        for (int i = 1; i < kGroups; i++) {
            x += *(const f32x4 *)&sums[all + i][d];
            sum += totals[all + i];
        }
    }
    put_values<T, HD>(a, -1, token, (int)(row - token * a.n_q), d, x, sum);
}

// Rows from which a wave each fills the CUs, however many parts: bf16 decode of 8192
// rows, hd 128, 28 parts 167 us (a block a row 194), 13 parts 100 (112), 5 parts 55
// (66); fp16, hd 256, 4096 rows of 52 parts 185 (197)
constexpr int64_t kMergeRows = 4096;

// ---- launches of one type -------------------------------------------------------------------
// More than 64 KiB of LDS is asked for once a kernel and device.
template <auto K, int STREAMS = 1> int run_kernel(int64_t blocks, int lds, const AttnArgs &a, hipStream_t stream,
                                 const char *what)
{
    static std::atomic<uint64_t> asked{0};
    if (lds > 65536) {
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess) return cbq_launch_status(what);
        const uint64_t bit = 1ull << (dev & 63);
        if (dev > 63 || !(asked.load(std::memory_order_relaxed) & bit)) {
            if (hipFuncSetAttribute((const void *)K, hipFuncAttributeMaxDynamicSharedMemorySize,
                                    lds) != hipSuccess)
                return cbq_launch_status(what);
            asked.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const CbqGrid grid = cbq_grid(blocks);
    K<<<dim3(grid.x, grid.y), dim3(STREAMS * kThreads), lds, stream>>>(a);
    return cbq_launch_status(what);
}

template <typename T, int HD> int launch(const AttnArgs &a, const Plan &p, bool prompt,
                                         hipStream_t stream)
{
    constexpr int wl = wave_lds<T, HD>(), bl = block_lds<T, HD>(), both = wl > bl ? wl : bl;
    constexpr int wide = widest(HD * (int)sizeof(T));
    int rc;
    if (prompt) {
        const char *what = "cbq_prefix_attn_prompt";
        // two streams where a wave leaves room for another on its SIMD
        constexpr int two = simd_waves(HD * (int)sizeof(T));
        if (p.rt == 0) rc = run_kernel<prompt_kernel<T, HD, 0>>(p.blocks, wl, a, stream, what);
        else if (p.rt == 1 && p.streams == 1)
            rc = run_kernel<prompt_kernel<T, HD, 1>>(p.blocks, bl, a, stream, what);
        else if (p.rt == 1)
            rc = run_kernel<prompt_kernel<T, HD, 1, two>, two>(p.blocks, two * (bl + 8), a, stream, what);
        else if (p.streams == 1)
            rc = run_kernel<prompt_kernel<T, HD, wide>>(p.blocks, bl, a, stream, what);
        else
            rc = run_kernel<prompt_kernel<T, HD, wide, two>, two>(p.blocks, two * (bl + 8), a, stream, what);
    } else {
        const char *what = "cbq_prefix_attn_decode";
        if (p.rt == 0 || !p.pre_parts)
            rc = run_kernel<decode_kernel<T, HD, 0>>(p.blocks, wl, a, stream, what);
        else if (p.rt == 1) rc = run_kernel<decode_kernel<T, HD, 1>>(p.blocks, both, a, stream, what);
        else rc = run_kernel<decode_kernel<T, HD, wide>>(p.blocks, both, a, stream, what);
    }
    if (rc != CK_SUCCESS || p.parts == 1) return rc;
    const char *what = "cbq_prefix_attn merge";
    const int64_t rows = (int64_t)a.N * a.n_q;
    if (rows >= kMergeRows)
        return run_kernel<merge_kernel<T, HD, 1>>(cbq_ceil(rows, kWaves), 0, a, stream, what);
    return run_kernel<merge_kernel<T, HD, kWaves>>(rows, 0, a, stream, what);
}

template <typename T> int launch_hd(const AttnArgs &a, const Plan &p, bool prompt,
                                    hipStream_t stream)
{
    switch (a.kv.hd) {
    case 64: return launch<T, 64>(a, p, prompt, stream);
    case 128: return launch<T, 128>(a, p, prompt, stream);
    default: return launch<T, 256>(a, p, prompt, stream);
    }
}

int launch_f32(const AttnArgs &a, const Plan &p, bool prompt, hipStream_t stream);
int launch_bf16(const AttnArgs &a, const Plan &p, bool prompt, hipStream_t stream);
int launch_f16(const AttnArgs &a, const Plan &p, bool prompt, hipStream_t stream);

}  // namespace cbq_attn
