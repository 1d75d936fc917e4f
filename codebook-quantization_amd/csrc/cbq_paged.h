// Addresses of a paged key/value cache and the launch plans of the attention
// over it: plain C++ that the kernels, the host entry points and the CPU test
// of them (tests/native/cbq_paged_host.cpp) share.
#pragma once

#include <stdint.h>

#include <algorithm>

#ifdef __HIPCC__
#define CBQ_PAGED_FN __host__ __device__ __forceinline__
#else
#define CBQ_PAGED_FN static inline
#endif

// n / d for 0 <= n < 2^31 by one 64-bit product: with 2^(s-1) < d <= 2^s and
// mul = ceil(2^(31+s) / d), mul * d - 2^(31+s) < d <= 2^s, so the product's
// error n * (mul * d - 2^(31+s)) / (d * 2^(31+s)) is below 1 / d: too small to
// reach the next integer.
struct CbqDiv {
    uint32_t d, mul, shift;
};

CBQ_PAGED_FN CbqDiv cbq_div_make(uint32_t d)
{
    uint32_t s = 0;
    while ((1ull << s) < d) s++;
    return CbqDiv{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}

CBQ_PAGED_FN uint32_t cbq_div(uint32_t n, const CbqDiv &q)
{
    return (uint32_t)(((uint64_t)n * q.mul) >> q.shift);
}

// The keys that a block walks: `prefix` shared ones, then own ones up to `end`
// (an index on the joint axis).
struct CbqKeys {
    const int32_t *shared, *own;
    int32_t prefix, end;
};

// Key j's entry in the table of its kind and its row in that page; 0, 0 for a
// key outside [0, end).
CBQ_PAGED_FN void cbq_key_place(const CbqKeys &a, const CbqDiv &page, int32_t j, int32_t &entry,
                                int32_t &row)
{
    const bool in = j >= 0 && j < a.end;
    const uint32_t i = in ? (uint32_t)(j < a.prefix ? j : j - a.prefix) : 0;
    entry = (int32_t)cbq_div(i, page);
    row = (int32_t)(i - (uint32_t)entry * page.d);
}

// From key j >= 0 to key j + step, step = step_entry * page + step_row; j, entry
// and row stay where they are at the end or past it.
CBQ_PAGED_FN void cbq_key_advance(const CbqKeys &a, const CbqDiv &page, int32_t step,
                                  int32_t step_entry, int32_t step_row, int32_t &j, int32_t &entry,
                                  int32_t &row)
{
    if (j >= a.end) return;
    const bool shared = j < a.prefix;
    j += step;
    if (shared && j >= a.prefix) {              // from the prefix's table to the own one
        cbq_key_place(a, page, j, entry, row);
        return;
    }
    entry += step_entry;
    row += step_row;
    if (row >= (int32_t)page.d) {
        row -= (int32_t)page.d;
        entry++;
    }
}

CBQ_PAGED_FN int32_t cbq_clamp_length(int32_t n, int64_t capacity)
{
    return n < 0 ? 0 : n > capacity ? (int32_t)capacity : n;
}

// Run b of a prompt batch: its first token and its length, inside [0, N).
CBQ_PAGED_FN void cbq_run(const int32_t *q_start, int b, int32_t N, int32_t &first, int32_t &count)
{
    const int32_t lo = cbq_clamp_length(q_start[b], N), hi = cbq_clamp_length(q_start[b + 1], N);
    first = lo;
    count = hi > lo ? hi - lo : 0;
}

CBQ_PAGED_FN int64_t cbq_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
CBQ_PAGED_FN int64_t cbq_min(int64_t a, int64_t b) { return a < b ? a : b; }
CBQ_PAGED_FN int64_t cbq_max(int64_t a, int64_t b) { return a > b ? a : b; }

// A launch holds fewer than 2^32 threads in a dimension (more are dropped without an
// error): of more than 2^22 blocks, of up to 512 threads, block b is (b % 2^22, b / 2^22).
// A grid of two dimensions is filled up with blocks past the last, which do nothing.
constexpr int kCbqGridBits = 22;
struct CbqGrid {
    uint32_t x, y;
};

static inline CbqGrid cbq_grid(int64_t blocks)
{
    const int64_t x = cbq_min(blocks, 1ll << kCbqGridBits);
    return CbqGrid{(uint32_t)x, (uint32_t)cbq_ceil(blocks, x)};
}

CBQ_PAGED_FN uint32_t cbq_block(uint32_t x, uint32_t y) { return y << kCbqGridBits | x; }

namespace cbq_attn {

// ---- launch plans ---------------------------------------------------------------------------
struct Plan {
    int rt;                                 // 64 rt rows a block, or 0: 16
    int32_t tiles;                          // row tiles: of the prefix rows; of a prompt, at most
    int32_t pre_parts, pre_chunk;           // decode: parts of the prefix and their keys
    int32_t own_parts, own_chunk, own_tiles;    // decode: parts of the own keys, 16-row tiles
    int32_t parts;                          // decode: all of them; prompt: key parts of a tile
    int32_t streams;                        // prompt: halves of a block's keys, walked side by side
    int32_t joint;                          // decode: a sequence's one part walks the prefix too
    int64_t blocks, bytes;
};

constexpr int64_t kCus = 256;                // of an MI355X
constexpr int kAttnWaves = 4;                // of a block
constexpr int64_t kMaxBlocks = (1ll << 31) - 1, kMaxParts = 1 << 20;    // of a plan

// Keys of a block's tile (K and V, two buffers: 64 KiB at most) and of a
// wave's own (K and V, one buffer: 16 KiB, 32 KiB for rows of 1024 bytes).
constexpr int block_keys(int row_bytes) { return row_bytes <= 256 ? 64 : 16384 / row_bytes; }
constexpr int wave_keys(int row_bytes) { return row_bytes <= 512 ? 8192 / row_bytes : 16; }

// 128 rows a block where a wave's 32 fit its registers beside a tile under way
constexpr int widest(int row_bytes) { return row_bytes <= 256 ? 2 : 1; }

inline int64_t part_bytes(int64_t parts, int64_t N, int n_q, int hd)
{
    return parts > 1 ? parts * N * n_q * (hd + 2) * 4 : 0;
}

// A prompt's block of 16, 64 or 128 rows (rt 0, 1, 2) takes this many us for 1000
// keys, alone on its CU and beside another block (rows of 1024 bytes: there is
// none), measured over 2000 to 4000 keys.
inline void walk_us(int row_bytes, int hd, int rt, double &alone, double &paired)
{
    static const float us[2][3][3][2] = {
        {{{5.4f, 8.2f}, {15, 17}, {17.5f, 20}},             // 16-bit types: hd 64, 128, 256
         {{10.4f, 14.8f}, {20, 25}, {24, 32}},
         {{22.5f, 31}, {38, 46}, {0, 0}}},
        {{{17, 27}, {46, 68}, {75, 116}},                   // fp32
         {{33, 50}, {84, 126}, {0, 0}},
         {{96, 96}, {182, 182}, {0, 0}}}};
    const float *u = us[row_bytes == 4 * hd][hd == 64 ? 0 : hd == 128 ? 1 : 2][rt];
    alone = u[0];
    paired = u[1];
}

inline Plan plan_decode(int row_bytes, int hd, int n_kv, int rep, int64_t prefix, int64_t capacity,
                        int64_t batch)
{
    Plan p = {};
    const int64_t rows = batch * rep, bk = block_keys(row_bytes), wk = kAttnWaves * wave_keys(row_bytes);
    p.rt = rows <= 16 ? 0 : rows <= 64 ? 1 : widest(row_bytes);
    int64_t tiles = cbq_ceil(rows, p.rt ? 64 * p.rt : 16), pre_parts = 0, pre_chunk = 1;
    if (prefix > 0) {
        // One block a CU, beside one of own keys: more parts cost their fp32 sums,
        // written and read once, fewer leave CUs without products (64 sequences of 32
        // heads behind 30011 keys: 133, 92, 98 and 107 us with 128, 256, 384 and 512).
        const int64_t least = p.rt ? 2 * bk : wk, want = cbq_max(1, kCus / (tiles * n_kv));
        const int64_t unit = p.rt ? bk : wk;
        pre_chunk = cbq_max(least, cbq_ceil(cbq_ceil(prefix, want), unit) * unit);
        pre_parts = cbq_ceil(prefix, pre_chunk);
    } else {
        tiles = 0;
    }
    const int64_t own_tiles = cbq_ceil(rep, 16);
    // About two blocks a CU of the full capacity, a tile a wave at least and eight at
    // most (33 sequences of 24 heads, up to 2900 keys: 17.6 us; with half and twice the
    // blocks 20).
    const int64_t share = cbq_ceil(capacity * batch * n_kv * own_tiles, 2 * kCus);
    int64_t own_chunk = cbq_min(cbq_max(cbq_ceil(share, wk), 1), 8) * wk;
    // more of a wider table than its parts and blocks are counted for
    const int64_t most = cbq_min(kMaxParts / 2, (kMaxBlocks - n_kv * tiles * pre_parts) / (n_kv * batch * own_tiles));
    if (most > 0) own_chunk = cbq_max(own_chunk, cbq_ceil(cbq_ceil(capacity, most), wk) * wk);
    const int64_t own_parts = cbq_max(cbq_ceil(capacity, own_chunk), pre_parts ? 0 : 1);
    p.blocks = n_kv * (tiles * pre_parts + batch * own_tiles * own_parts);
    p.bytes = part_bytes(pre_parts + own_parts, batch, n_kv * rep, hd);
    p.tiles = (int32_t)tiles;
    p.pre_parts = (int32_t)pre_parts;
    p.pre_chunk = (int32_t)pre_chunk;
    p.own_parts = (int32_t)own_parts;
    p.own_chunk = (int32_t)own_chunk;
    p.own_tiles = (int32_t)own_tiles;
    p.parts = (int32_t)(pre_parts + own_parts);
    if (prefix + capacity > 4 * wk) return p;
    // Few keys, four tiles a wave at most: one block a sequence and kv head can walk
    // prefix and own ones without a merge (3 us and its sums), where that is less than
    // the tiles it adds to the blocks' turns.  bf16, 8 kv heads of 128 of 4 queries, in
    // one block and in parts: 2 sequences of 3..18 keys, room for 300, 7.2 and 9.7 us;
    // 128 sequences behind 460 keys 22.5 and 19.9, 1024 of them 140 and 97; one query a
    // kv head of 64, 1024 behind 921 143 and 75.  The lengths are device data: 0.4 of
    // the room is taken for them.  Over sizes of 1 to 512 sequences the estimate's
    // choice takes 0.5 % more than the shorter of both where lengths fill up to the
    // room (2616 of them; one block everywhere 4.6 %, parts 24 %), 1.1 % where 256 keys
    // of room are left (3360; 2.3 and 35 %).
    const int64_t own = (2 * capacity + 4) / 5;
    const double one = (double)(n_kv * batch * own_tiles) / (row_bytes <= 512 ? 2 * kCus : kCus);
    const double tile = row_bytes > 512 ? 5 : row_bytes == 4 * hd ? 1.8 : 1.2;      // us of a wave's
    double alone, paired, split = 0;
    walk_us(row_bytes, hd, p.rt, alone, paired);
    if (own > 0) split = tile * std::max(1.0, one * cbq_ceil(own, wk));
    split += (double)tiles * n_kv * prefix * 0.001 * alone / kCus;
    split = std::max(split, (double)cbq_min(pre_chunk, prefix) * 0.001 * alone);            // a prefix block
    if (p.parts > 1) split += 3 + (double)p.parts * batch * n_kv * rep * hd * 8 / 5e6;
    const bool alike = !pre_parts && p.parts == 1;          // one part of own keys either way
    if (!alike && tile * std::max(1.0, one) * cbq_ceil(prefix + own, wk) > split) return p;
    p = Plan{};
    p.joint = 1;
    p.own_parts = p.parts = 1;
    p.own_chunk = (int32_t)cbq_max(prefix + capacity, 1);
    p.own_tiles = (int32_t)own_tiles;
    p.blocks = n_kv * batch * own_tiles;
    return p;
}

inline Plan plan_prompt(int row_bytes, int hd, int n_kv, int rep, int64_t prefix, int64_t capacity,
                        int64_t batch, int64_t N)
{
    // Rows a block, parts of the keys, and streams a block, by the least time: few
    // rows a block spread over the CUs, many read the keys fewer times; parts shorten
    // the walk and cost their fp32 sums, written and read, and a launch (4 us); two
    // streams halve it for a whole CU and a join in LDS.  bf16, 32 heads on 8 of 128:
    // 256 tokens 9.2 us (16 rows, one part) against 17 (128 rows, two parts), 512 15
    // (64 rows, two streams) against 28 (128, three parts) and 16 (64, one stream), 1024
    // 29 against 43 (128, two parts), 2048 57 (128, two streams) against 70 (64); behind
    // 1500 shared keys 48 18 (64 rows, seven parts) against 21 (16, one part), 1024 56
    // (128, two streams) against 65 (64, one).
    // The lengths are device data: a sequence's own keys are taken halfway between
    // the new tokens and the table's room, and no more than 1024 short of that.
    const int64_t rows = N * rep, runs = cbq_max(cbq_min(batch, N), 1);
    const int64_t own = cbq_max((capacity + N / runs) / 2, capacity - 1024);
    const int64_t keys = cbq_max(prefix + own, 1);
    const int64_t slots = row_bytes <= 512 ? 2 * kCus : kCus;
    // Bytes a us of the parts' sums, written and read.  Drawn prompts of 16 to 3000
    // tokens with 5e6 against 2.5e6 (geometric means): 90 16-bit ones of hd 256 0.6 %
    // less, 40 of 16 bits and hd 128 0.1 % more, 30 of hd 64 0.2 % more; fp32 of hd 256
    // 0.2 % less (but four times the parts of 17 tokens in wide tables), of hd 128 3.2 %
    // more, of hd 64 2.1 % more.
    const double rate = row_bytes == 512 && hd == 256 ? 5e6 : 2.5e6;
    double best = -1;
    int best_rt = 0;
    int64_t best_parts = 1, best_streams = 1;
    for (int rt = 0; rt <= widest(row_bytes); rt++) {
        const int64_t m = rt ? 64 * rt : 16;
        // two tiles of keys a part: from four the few rows over 500 to 3000 keys took
        // 1.1 to 1.3 times as long
        const int64_t least = 2 * (rt ? block_keys(row_bytes) : kAttnWaves * wave_keys(row_bytes));
        // of the runs' last tiles, half are taken to be there beside the whole ones
        const int64_t likely = n_kv * cbq_max(runs == 1 ? cbq_ceil(rows, m) : rows / m + cbq_ceil(runs, 2),
                                              runs);
        double alone, paired;
        walk_us(row_bytes, hd, rt, alone, paired);
        for (int way = 0; way < 5; way++) {
            // one stream of keys a block: one part, parts to a block a CU, to two; two
            // streams, which are two blocks' waves as one: one part, parts to a block a CU
            const int streams = way < 3 ? 1 : 2;
            if (streams == 2 && (rt == 0 || slots == kCus)) break;
            const int64_t room = streams == 2 ? kCus : slots;
            // two streams fill a CU: one block too many is a turn more
            const int64_t blocks0 = streams == 2 ? n_kv * (runs == 1 ? cbq_ceil(rows, m) : rows / m + runs)
                                                 : likely;
            const int64_t parts = way % 3 == 0 ? 1 : cbq_min((way == 2 ? slots : kCus) / blocks0,
                                                             keys / (streams * least));
            if (parts < 1 || (way % 3 && parts == 1)) continue;
            const double most = 0.001 * keys / parts;               // thousands of keys, the last tile's
            const double mean = cbq_max(keys - N / runs / 2, 1) * 0.001 / parts;
            const double fewest = 2 * mean > most ? 2 * mean - most : 0;
            const double blocks = (double)blocks0 * parts, both = streams == 2 ? 0.55 * paired : paired;
            double us;
            if (streams == 2)
                us = both * most + 3;                               // and the join
            else                // the block of the most keys shares its CU with one of few
                us = alone * most + (blocks > kCus ? (paired - alone) * fewest : 0);
            if (blocks > room) {
                // more turns than one, the last as long as its blocks where all are alike;
                // each block begins with 3 us of dependent loads
                const int64_t whole = cbq_ceil(blocks0 * parts, room);
                const double turns = blocks / room,
                             all = both * (turns * mean + (whole - turns) * fewest) + 3 * (turns - 1);
                us = us > all ? us : all;
            }
            if (parts > 1) us += 4 + (double)parts * N * n_kv * rep * hd * 8 / rate;
            if (best < 0 || us < best) {
                best = us;
                best_rt = rt;
                best_parts = parts;
                best_streams = streams;
            }
        }
    }
    Plan p = {};
    p.rt = best_rt;
    p.streams = (int32_t)best_streams;
    // a run's last tile may be part full: one more a run than the rows need
    const int64_t tiles = rows / (p.rt ? 64 * p.rt : 16) + runs;
    p.blocks = tiles * n_kv * best_parts;
    p.bytes = part_bytes(best_parts, N, n_kv * rep, hd);
    p.tiles = (int32_t)tiles;
    p.parts = (int32_t)best_parts;
    return p;
}

inline bool plan_fits(const Plan &p)
{
    return p.blocks > 0 && p.blocks <= kMaxBlocks && p.parts <= kMaxParts;
}

// ---- what a block does ------------------------------------------------------------------------
// Decode: blocks of the prefix's parts first (they compute), then own parts
// (they read), so that both kinds share the CUs.
struct DecodeWork {
    int h, tile, part, seq;                 // seq -1: the prefix
    int32_t first, end;                     // keys (own ones: as the capacity has them;
                                            // joint: of both)
};

CBQ_PAGED_FN DecodeWork decode_work(const Plan &p, uint32_t block, int n_kv, int batch,
                                    int32_t prefix, int64_t capacity)
{
    DecodeWork w;
    uint32_t i = block;
    const uint32_t pre = (uint32_t)p.tiles * p.pre_parts * n_kv;
    const bool shared = i < pre;
    if (!shared) i -= pre;
    w.h = (int)(i % n_kv);
    i /= n_kv;
    if (shared) {
        w.tile = (int)(i % p.tiles);
        w.part = (int)(i / p.tiles);
        w.seq = -1;
        w.first = w.part * p.pre_chunk;
        w.end = (int32_t)cbq_min((int64_t)w.first + p.pre_chunk, prefix);
        return w;
    }
    w.tile = (int)(i % p.own_tiles);
    i /= p.own_tiles;
    w.seq = (int)(i % batch);
    const int chunk = (int)(i / batch);
    const int64_t most = (p.joint ? prefix : 0) + capacity;
    w.part = p.pre_parts + chunk;
    w.first = (int32_t)cbq_min((int64_t)chunk * p.own_chunk, most);
    w.end = (int32_t)cbq_min((int64_t)w.first + p.own_chunk, most);
    return w;
}

// Prompt: the keys of part `part` of a tile whose rows see `sees` keys at most.
CBQ_PAGED_FN void prompt_keys(int32_t sees, int parts, int part, int unit, int32_t &first,
                              int32_t &end)
{
    const int64_t share = cbq_ceil(cbq_ceil(sees, parts), unit) * unit;
    first = (int32_t)cbq_min(part * share, sees);
    end = (int32_t)cbq_min(first + share, sees);
}

// The keys [first, end) of one of a block's streams: whole tiles to the streams in
// turn, the first ones' share the larger.
CBQ_PAGED_FN void stream_keys(int32_t from, int32_t upto, int unit, int streams, int stream,
                              int32_t &first, int32_t &end)
{
    const int64_t keys = upto > from ? upto - from : 0;
    const int64_t share = cbq_ceil(cbq_ceil(keys, unit), streams) * unit;
    first = (int32_t)(from + cbq_min(stream * share, keys));
    end = (int32_t)(from + cbq_min((stream + 1) * share, keys));
}

}  // namespace cbq_attn
