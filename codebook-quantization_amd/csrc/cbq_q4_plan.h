// Launch plans of the attention over the 4-bit paged cache and what a block of them
// does: plain C++ that the kernels, the host entry points and the CPU test of them
// (tests/native/cbq_q4_host.cpp) share.
#pragma once

#include "cbq_paged.h"

namespace cbq_q4 {

constexpr int kTile = 32;                   // keys of a wave's tile
constexpr int kAttnWaves = 4;               // waves a block, whose tiles take turns
// (16 rows, tile, kv head) products of a prefix from which on its tiles are made into values
// in LDS for all of a block's rows; with fewer the rounds of barriers cost more than they
// save.  64 sequences of 32 heads behind 30011 keys, in a captured graph as below: 83 us, and
// 110 with every wave's own.
constexpr int64_t kManyTiles = 16 * 1024;
constexpr int64_t kMaxBlocks = (1ll << 31) - 1, kMaxParts = 1 << 20, kAttnCus = 256;
constexpr int64_t kMaxBytes = 1ll << 30;      // of the own parts' sums, where there are several

struct Plan {
    int32_t rt;                             // 64 rt rows a block of the prefix, or 0: 16
    int32_t tiles;                          // row tiles of the prefix, of all sequences
    int32_t pre_parts, pre_chunk;           // parts of the prefix and their key tiles
    int32_t own_parts, own_chunk, own_tiles;    // parts of the own keys; 16-row tiles of a sequence
    int32_t parts;                          // all of them
    int32_t joint;                          // one part: a sequence's own blocks walk the prefix too
    int64_t blocks, bytes;
};

// 64 widest rows of the prefix a block, as many as a wave's registers hold
constexpr int widest(int hd) { return hd == 256 ? 1 : 2; }

inline int64_t part_bytes(int64_t parts, int64_t rows, int hd)
{
    return parts > 1 ? parts * rows * (hd + 2) * 4 : 0;
}

// rows: query rows of a sequence and kv head (tokens times query heads a kv head)
inline Plan plan(int hd, bool bf16, int n_kv, int64_t rows, int64_t prefix, int64_t capacity, int64_t batch)
{
    Plan p = {};
    const int64_t pre_tiles = cbq_ceil(prefix, kTile), cap_tiles = cbq_ceil(capacity, kTile);
    const int64_t own_tiles = cbq_ceil(rows, 16);
    const int64_t all = batch * rows;
    const bool many = bf16 && all > 16 && cbq_ceil(all, 16) * pre_tiles * n_kv >= kManyTiles;
    p.rt = many ? (int32_t)cbq_min(all > 64 ? 2 : 1, widest(hd)) : 0;
    p.own_tiles = (int32_t)own_tiles;
    // One block for all keys of a row tile, no parts to join: of few tiles a wave the join
    // costs as much as it saves, and where every CU has two such blocks parts bring no more
    // of them.  64 sequences of 32 heads, 900 to 1900 keys: 32 us against 38 in parts, but one
    // of 1200 keys 18 against 10; 300 to 3800 keys 54 against 47: lengths this uneven.
    // But every such block walks the prefix for itself, which parts read for 16 rows of all
    // sequences: 1 ns more a tile of 128 values, against 4 us and 10 ns a 1000 values of the
    // parts' sums, written, read and joined.  100 own keys and 32 heads on 8 of 128, bf16, in one
    // block and in parts: 64 sequences behind 100 keys 11 and 16 us, behind 460 17 both, behind
    // 2900 50 and 28; 1024 behind 100 93 and 123, behind 2900 549 and 183.  Over 4340 sizes of 1
    // to 1500 sequences the choice takes 1.1 % more than the shorter of both (3.6 % and five
    // times at worst without the prefix's part of it; one block everywhere 18 %, parts 15 %).
    const int64_t alone = n_kv * batch * own_tiles;
    const double again = 1e-3 * hd / 128 * (double)(alone - n_kv * cbq_ceil(all, 16)) * (double)pre_tiles,
                 sums = 4 + 1e-5 * hd * (double)(all * n_kv);
    if (pre_tiles + cap_tiles <= (alone >= 2 * kAttnCus ? 24 : 4) * kAttnWaves && again <= sums) {
        p.joint = 1;
        p.rt = 0;
        p.own_parts = p.parts = 1;
        p.own_chunk = (int32_t)cbq_max(pre_tiles + cap_tiles, 1);
        p.blocks = alone;
        return p;
    }
    int64_t tiles = cbq_ceil(all, p.rt ? 64 * p.rt : 16), pre_parts = 0, pre_chunk = 1;
    // Blocks a CU: two for the prefix (four: 33 sequences of 3 tokens behind 5000 keys take 36
    // us instead of 34), four for the own keys, 4 to 64 tiles each (two: 35.5 us, there).  One
    // for each with hd 256, of which a CU holds one block (two and four: one sequence of 9000
    // keys 26 us instead of 18, 50 of 2 tokens behind 2000 keys 52 instead of 49); one for
    // a prefix whose tiles are shared (two: 92 us instead of 83, then).
    const int64_t pre_blocks = (p.rt || hd == 256 ? 1 : 2) * kAttnCus, own_blocks = (hd == 256 ? 1 : 4) * kAttnCus;
    if (pre_tiles) {
        const int64_t want = cbq_max(1, pre_blocks / (tiles * n_kv)), unit = p.rt ? 2 : kAttnWaves;
        pre_chunk = cbq_max(p.rt ? 4 : 2 * kAttnWaves, cbq_ceil(cbq_ceil(pre_tiles, want), unit) * unit);
        pre_parts = cbq_ceil(pre_tiles, pre_chunk);
    } else {
        tiles = 0;
    }
    const int64_t share = cbq_ceil(cap_tiles * batch * n_kv * own_tiles, own_blocks);
    int64_t own_chunk = cbq_min(cbq_max(cbq_ceil(share, kAttnWaves), 1), 16) * kAttnWaves;
    // more of a wider table than its parts and blocks are counted for, or than a workspace of
    // 1 GiB holds (of rows so many that their blocks are plenty)
    const int64_t most = cbq_min(cbq_min(kMaxParts / 2, cbq_max(1, kMaxBytes / part_bytes(2, batch * rows * n_kv, hd) * 2)),
                                 (kMaxBlocks - n_kv * tiles * pre_parts) / (n_kv * batch * own_tiles));
    if (most > 0) own_chunk = cbq_max(own_chunk, cbq_ceil(cbq_ceil(cap_tiles, most), kAttnWaves) * kAttnWaves);
    const int64_t own_parts = cbq_max(cbq_ceil(cap_tiles, own_chunk), pre_parts ? 0 : 1);
    p.tiles = (int32_t)tiles;
    p.pre_parts = (int32_t)pre_parts;
    p.pre_chunk = (int32_t)pre_chunk;
    p.own_parts = (int32_t)own_parts;
    p.own_chunk = (int32_t)own_chunk;
    p.parts = (int32_t)(pre_parts + own_parts);
    p.blocks = n_kv * (tiles * pre_parts + batch * own_tiles * own_parts);
    p.bytes = part_bytes(pre_parts + own_parts, batch * rows * n_kv, hd);
    return p;
}

inline bool plan_fits(const Plan &p)
{
    return p.blocks > 0 && p.blocks <= kMaxBlocks && p.parts <= kMaxParts;
}

// A block's rows and its key tiles [first, end): of the prefix from 0 on, then (own
// parts, or all where joint) of the own keys from pre_tiles on.
struct Work {
    int h, tile, part, seq;                 // seq -1: prefix rows, of the whole batch
    int32_t first, end;                     // as the capacity has them
};

CBQ_PAGED_FN Work work_of(const Plan &p, uint32_t block, int n_kv, int batch, int32_t pre_tiles,
                          int32_t cap_tiles)
{
    Work w;
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
        w.end = (int32_t)cbq_min((int64_t)w.first + p.pre_chunk, pre_tiles);
        return w;
    }
    w.tile = (int)(i % p.own_tiles);
    i /= p.own_tiles;
    w.seq = (int)(i % batch);
    const int chunk = (int)(i / batch);
    const int64_t from = p.joint ? 0 : pre_tiles, upto = (int64_t)pre_tiles + cap_tiles;
    w.part = p.pre_parts + chunk;
    w.first = (int32_t)cbq_min(from + (int64_t)chunk * p.own_chunk, upto);
    w.end = (int32_t)cbq_min((int64_t)w.first + p.own_chunk, upto);
    return w;
}

}  // namespace cbq_q4
