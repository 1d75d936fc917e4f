// The launch plans of the attention over the 4-bit cache (csrc/cbq_q4_plan.h, the code
// that the kernels run) on the CPU, under address and undefined-behaviour sanitizers:
// every (row, key) visited once by the blocks of a plan, parts inside the workspace and
// those that the merge adds up written.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "../../codebook-quantization_amd/csrc/cbq_q4_plan.h"

using namespace cbq_q4;

static std::mt19937 rng(7);
static int64_t pick(int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); }

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)

static int kinds[4];                        // plans seen: joint, parts alone, with a shared prefix of 64 and 128 rows

static void one(int hd, bool bf16, int n_kv, int rows, int prefix, int64_t capacity, int batch)
{
    std::vector<int32_t> lengths(batch);
    for (auto &x : lengths) x = pick(0, 5) ? pick(0, capacity) : pick(0, 1) ? -5 : 1 << 30;
    const Plan p = plan(hd, bf16, n_kv, rows, prefix, capacity, batch);
    CHECK(plan_fits(p));
    kinds[p.joint ? 0 : p.rt == 0 ? 1 : p.rt == 1 ? 2 : 3]++;
    CHECK(p.rt <= widest(hd) && (bf16 || p.rt == 0));
    CHECK(p.parts == p.pre_parts + p.own_parts);
    CHECK(p.bytes == (p.parts > 1 ? (int64_t)p.parts * batch * rows * n_kv * (hd + 2) * 4 : 0));
    const int32_t pre_tiles = (prefix + kTile - 1) / kTile, cap_tiles = (int32_t)((capacity + kTile - 1) / kTile);
    // rows x tiles counted by kv head 0's blocks alone where there are several
    std::vector<uint8_t> shared((size_t)batch * rows * pre_tiles), own((size_t)batch * rows * cap_tiles);
    std::vector<uint8_t> written((size_t)p.parts * batch * rows);
    std::vector<int> heads(n_kv);
    for (int64_t block = 0; block < p.blocks; block++) {
        const Work w = work_of(p, (uint32_t)block, n_kv, batch, pre_tiles, cap_tiles);
        CHECK(w.h >= 0 && w.h < n_kv && w.part >= 0 && w.part < p.parts && w.seq < batch);
        heads[w.h]++;
        if (w.h) continue;
        if (w.seq < 0) {
            const int wide = p.rt ? 64 * p.rt : 16;
            CHECK(w.first < w.end && w.end <= pre_tiles && w.part < p.pre_parts);
            for (int r = w.tile * wide; r < (w.tile + 1) * wide && r < batch * rows; r++) {
                written[(size_t)w.part * batch * rows + r]++;
                for (int t = w.first; t < w.end; t++) shared[(size_t)r * pre_tiles + t]++;
            }
            continue;
        }
        const int32_t length = cbq_clamp_length(lengths[w.seq], capacity);
        const int32_t end = (int32_t)cbq_min(w.end, (int64_t)pre_tiles + cbq_ceil(length, kTile));
        if (w.first >= end && p.parts > 1) continue;
        for (int r = w.tile * 16; r < w.tile * 16 + 16 && r < rows; r++) {
            const size_t row = (size_t)w.seq * rows + r;
            written[(size_t)w.part * batch * rows + row]++;
            for (int t = w.first; t < end; t++) {
                if (t < pre_tiles) shared[row * pre_tiles + t]++;
                else own[row * cap_tiles + t - pre_tiles]++;
            }
        }
    }
    for (int h = 1; h < n_kv; h++) CHECK(heads[h] == heads[0]);
    for (uint8_t x : shared) CHECK(x == 1);
    for (int b = 0; b < batch; b++) {
        const int32_t length = cbq_clamp_length(lengths[b], capacity);
        const int64_t parts = p.parts == 1 ? 1 : p.pre_parts + cbq_ceil(cbq_ceil(length, kTile), p.own_chunk);
        CHECK(parts <= p.parts);
        for (int r = 0; r < rows; r++) {
            const size_t row = (size_t)b * rows + r;
            for (int t = 0; t < cap_tiles; t++) CHECK(own[row * cap_tiles + t] == (t < cbq_ceil(length, kTile)));
            for (int i = 0; i < p.parts; i++)
                CHECK(written[(size_t)i * batch * rows + row] == (i < parts));
        }
    }
}

int main()
{
    const int hds[] = {64, 128, 256};
    for (int n = 0; n < 3000; n++) {
        one(hds[pick(0, 2)], pick(0, 1), pick(1, 3), pick(1, 70), pick(0, 2) ? pick(1, 3000) : 0, pick(0, 2000),
            pick(1, 12));
    }
    for (int n = 0; n < 40; n++)            // long prefixes of many rows
        one(hds[pick(0, 2)], true, pick(2, 8), pick(2, 24), pick(2900, 20000), pick(0, 256), pick(8, 30));
    one(256, true, 8, 40, 12000, 128, 20);
    one(128, true, 8, 3, 30000, 128, 20);
    for (int i = 0; i < 4; i++) CHECK(kinds[i] > 0);
    // many rows against wide tables: the own parts' sums stay below 1 GiB
    for (int64_t rows : {1ll, 4ll, 300ll, 100000ll})
        for (int64_t batch : {1ll, 60ll, 3000ll}) {
            const Plan p = plan(128, false, 8, rows, 0, 1 << 24, batch);
            CHECK(plan_fits(p) && (p.own_parts <= 2 || p.bytes <= kMaxBytes));
        }
    // the largest tables and batches that the entry points allow
    for (int64_t batch : {1ll, 1ll << 20, (1ll << 30) - 1})
        for (int64_t capacity : {0ll, 1000ll, (1ll << 31) - 65536})
            for (int64_t prefix : {0ll, 5ll, 100000ll}) {
                if (prefix + capacity > (1ll << 31) - 65536) continue;
                const Plan p = plan(128, true, 1, 1, prefix, capacity, batch);
                if (plan_fits(p)) CHECK(p.bytes >= 0 && p.own_chunk >= 1);
            }
    printf("plans: joint %d, parts %d, shared by 64 rows %d, by 128 %d\nall cases passed\n", kinds[0], kinds[1],
           kinds[2], kinds[3]);
    return 0;
}
