// The paged cache's addresses and the attention's launch plans
// (csrc/cbq_paged.h, the code that the kernels run) on the CPU, under address
// and undefined-behaviour sanitizers: division, table entries of every key a
// block walks (tables allocated to the entry), every (row, key) visited once,
// parts inside the workspace, lengths, runs and page ids that are out of range.
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <random>
#include <string>
#include <vector>

#include "../../codebook-quantization_amd/csrc/cbq_paged.h"

using namespace cbq_attn;

static std::mt19937 rng(7);
static int64_t pick(int64_t lo, int64_t hi) { return lo + (int64_t)(rng() % (uint64_t)(hi - lo + 1)); }

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); exit(1); } } while (0)

static void divisions()
{
    for (uint32_t d = 1; d <= 65536; d = d < 300 ? d + 1 : d + 1 + rng() % 257) {
        const CbqDiv q = cbq_div_make(d);
        const uint32_t near[] = {0, 1, d - 1, d, d + 1, 0x7fffffffu, 0x7fffffffu / d * d,
                                 0x7fffffffu / d * d - 1, 0x7ffffffeu};
        for (uint32_t n : near)
            if (n < 0x80000000u) CHECK(cbq_div(n, q) == n / d);
        for (int i = 0; i < 200; i++) {
            const uint32_t n = rng() & 0x7fffffffu;
            CHECK(cbq_div(n, q) == n / d);
        }
    }
    for (uint32_t d : {65537u, 1000003u, 0x7fffffffu, 0x40000000u, 0x40000001u}) {
        const CbqDiv q = cbq_div_make(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 0x7fffffffu, 0x7ffffffeu})
            if (n < 0x80000000u) CHECK(cbq_div(n, q) == n / d);
    }
}

// The keys that a block's walks touch, `step` of them side by side: those inside
// are counted, and a walk that looks past the end names no entry.
static void walk(const CbqKeys &keys, const CbqDiv &page, int32_t first, int step,
                 const std::vector<int32_t> &prefix_table, const int32_t *own, int width,
                 std::vector<int> &seen)
{
    const int32_t step_entry = (int32_t)cbq_div(step, page), step_row = step - step_entry * (int32_t)page.d;
    for (int lane = 0; lane < step; lane++) {
        int32_t key = first + lane, entry, row;
        cbq_key_place(keys, page, key, entry, row);
        for (int64_t j = key; j < (int64_t)keys.end + 3 * step; j += step) {
            if (key >= 0 && key < keys.end) {
                const int64_t i = j < keys.prefix ? j : j - keys.prefix;
                CHECK(key == j && entry == i / page.d && row == i % page.d);
                CHECK(entry < (j < keys.prefix ? (int64_t)prefix_table.size() : width));
                volatile int32_t id = (j < keys.prefix ? keys.shared : keys.own)[entry];
                (void)id;
                seen[j]++;
            } else {
                CHECK(j >= keys.end);
            }
            cbq_key_advance(keys, page, step, step_entry, step_row, key, entry, row);
        }
    }
}

static void decode()
{
    const int hds[] = {64, 128, 256}, pages[] = {1, 3, 16, 17, 64, 256};
    const int hd = hds[pick(0, 2)], size = pick(0, 1) ? 2 : 4, page = pages[pick(0, 5)];
    const int n_kv = pick(1, 3), rep = pick(1, 40), batch = pick(1, 40), width = pick(0, 3000 / page);
    const int prefix = pick(0, 2) ? pick(1, 4000) : 0;
    const int64_t capacity = (int64_t)width * page;
    std::vector<int32_t> prefix_table(cbq_ceil(prefix, page)), tables((size_t)batch * width),
        lengths(batch);
    for (auto &x : lengths) x = pick(0, 5) ? pick(0, capacity) : pick(0, 1) ? -5 : 1 << 30;
    const Plan p = plan_decode(hd * size, hd, n_kv, rep, prefix, capacity, batch);
    CHECK(plan_fits(p));
    CHECK(p.bytes == (p.parts > 1 ? (int64_t)p.parts * batch * n_kv * rep * (hd + 2) * 4 : 0));
    const CbqDiv pg = cbq_div_make(page);
    const int pre = p.joint ? prefix : 0;           // walked by each sequence itself
    // [kv head][row tile of 16 or 64 rt rows][key] for the prefix and each sequence
    std::map<std::vector<int>, std::vector<int>> seen;
    std::map<std::vector<int>, int> parts;
    const int m = p.rt ? 64 * p.rt : 16, step = p.rt ? block_keys(hd * size) : wave_keys(hd * size) * kAttnWaves;
    for (int64_t i = 0; i < p.blocks; i++) {
        const DecodeWork w = decode_work(p, (uint32_t)i, n_kv, batch, prefix, capacity);
        CHECK(w.h >= 0 && w.h < n_kv);
        if (w.seq < 0) {
            CHECK(w.tile >= 0 && w.tile * m < batch * rep && w.part >= 0 && w.part < p.pre_parts);
            auto &s = seen[{w.h, -1, w.tile}];
            s.resize(prefix);
            walk({prefix_table.data(), nullptr, prefix, w.end}, pg, w.first, step, prefix_table, nullptr, 0, s);
        } else {
            CHECK(w.seq < batch && w.tile * 16 < rep);
            // as the kernel: first table entries by the capacity, then the length
            int32_t entry, row;
            for (int lane = 0; lane < 64; lane++) {
                const int32_t j = w.first + lane;
                cbq_key_place({prefix_table.data(), tables.data() + (size_t)w.seq * width, pre, w.end}, pg, j, entry, row);
                CHECK(j >= w.end || entry < (j < pre ? (int)prefix_table.size() : width));
            }
            const int32_t len = cbq_clamp_length(lengths[w.seq], capacity);
            if (w.first >= pre + len && p.parts > 1) continue;
            CHECK(w.part >= p.pre_parts && w.part < p.parts);
            const int32_t *own = tables.data() + (size_t)w.seq * width;
            auto &s = seen[{w.h, w.seq, w.tile}];
            s.resize(pre + capacity);
            walk({prefix_table.data(), own, pre, (int32_t)cbq_min(w.end, pre + len)}, pg, w.first, step, prefix_table,
                 own, width, s);
            parts[{w.h, w.seq, w.tile}]++;
        }
    }
    for (int h = 0; h < n_kv; h++) {
        for (int t = 0; prefix && !p.joint && t * m < batch * rep; t++)
            for (int x : seen[{h, -1, t}]) CHECK(x == 1);
        for (int b = 0; b < batch; b++)
            for (int t = 0; t * 16 < rep; t++) {
                const int32_t len = cbq_clamp_length(lengths[b], capacity);
                auto &s = seen[{h, b, t}];
                for (int j = 0; j < (int)s.size(); j++) CHECK(s[j] == (j < pre + len));
                CHECK(pre + len == 0 || (int)s.size() == pre + capacity);
                // what the merge counts (a lone part always writes the output)
                const int want = p.parts == 1 ? (p.pre_parts ? 0 : 1) : (int)cbq_ceil(len, p.own_chunk);
                CHECK((parts[{h, b, t}]) == want);
            }
    }
}

static void prompt()
{
    const int hds[] = {64, 128, 256};
    const int hd = hds[pick(0, 2)], size = pick(0, 1) ? 2 : 4, n_kv = pick(1, 4), rep = pick(1, 40);
    const int batch = pick(1, 70), width = pick(0, 300), page = 16;
    const int prefix = pick(0, 1) ? pick(1, 4000) : 0;
    std::vector<int32_t> q_start(batch + 1);
    for (int b = 0; b < batch; b++) q_start[b + 1] = q_start[b] + (pick(0, 4) ? pick(0, 90) : 0);
    const int N = q_start[batch] + 1;
    const Plan p = plan_prompt(hd * size, hd, n_kv, rep, prefix, (int64_t)width * page, batch, N);
    CHECK(plan_fits(p));
    // parts only where CUs are left, and none shorter than two tiles
    CHECK(p.parts == 1 || (int64_t)p.parts * n_kv * std::min(batch, N) <= 2 * kCus);
    CHECK(p.parts == 1 || (int64_t)p.parts * 2 * (p.rt ? block_keys(hd * size) : kAttnWaves * wave_keys(hd * size)) <=
                              prefix + std::max<int64_t>((int64_t)width * page, N));
    const int m = p.rt ? 64 * p.rt : 16;
    int64_t tiles = 0;
    for (int b = 0; b < batch; b++) {
        int32_t f, n;
        cbq_run(q_start.data(), b, N, f, n);
        CHECK(f == q_start[b] && n == q_start[b + 1] - q_start[b]);
        tiles += cbq_ceil((int64_t)n * rep, m);
    }
    CHECK(tiles <= p.tiles && p.blocks == (int64_t)p.tiles * n_kv * p.parts);
    for (int sees : {0, 1, 63, 64, 65, 1000, prefix + width * page}) {
        int32_t at = 0;
        for (int i = 0; i < p.parts; i++) {
            int32_t first, end;
            prompt_keys(sees, p.parts, i, p.rt ? block_keys(hd * size) : wave_keys(hd * size), first, end);
            CHECK(first == at && end >= first && end <= sees);
            // a block's streams: whole tiles, one after the other, the first's the more
            int32_t then = first, more = 0;
            for (int j = 0; j < p.streams; j++) {
                int32_t f, e;
                stream_keys(first, end, block_keys(hd * size), p.streams, j, f, e);
                CHECK(f == then && e >= f && (e == end || (e - first) % block_keys(hd * size) == 0));
                CHECK(j == 0 || e - f <= more);
                then = e;
                more = e - f;
            }
            CHECK(then == end);
            CHECK(p.streams == 1 || (p.rt > 0 && hd * size <= 512));
            at = end;
        }
        CHECK(at == sees);
    }
    // a run's keys: the prefix, then its own
    std::vector<int32_t> prefix_table(cbq_ceil(prefix, page)), own(width);
    const int32_t sees = prefix + (width ? (int32_t)pick(1, width * page) : 0);
    std::vector<int> seen(sees);
    const int unit = p.rt ? block_keys(hd * size) : wave_keys(hd * size) * kAttnWaves;
    for (int i = 0; i < p.parts; i++) {
        int32_t first, end;
        prompt_keys(sees, p.parts, i, p.rt ? unit : wave_keys(hd * size), first, end);
        walk({prefix_table.data(), own.data(), prefix, end}, cbq_div_make(page), first, unit, prefix_table,
             own.data(), width, seen);
    }
    for (int x : seen) CHECK(x == 1);
    // starts in no order and out of range stay inside the tokens
    for (auto &x : q_start) x = (int32_t)rng();
    for (int b = 0; b < batch; b++) {
        int32_t f, n;
        cbq_run(q_start.data(), b, N, f, n);
        CHECK(f >= 0 && n >= 0 && f + n <= N);
    }
}

static void far()
{
    // the largest axis: indexes near 2^31, and a look-ahead past the end
    const int64_t most = (1ll << 31) - 65536;
    const CbqDiv page = cbq_div_make(65536);
    std::vector<int32_t> t(cbq_ceil(most, 65536));
    const CbqKeys keys = {nullptr, t.data(), 0, (int32_t)most};
    int32_t key = (int32_t)(most - 300), entry, row;
    cbq_key_place(keys, page, key, entry, row);
    for (int i = 0; i < 5; i++) {
        if (key < keys.end) CHECK(entry == key / 65536 && row == key % 65536 && entry < (int)t.size());
        cbq_key_advance(keys, page, 256, 0, 256, key, entry, row);
    }
    CHECK(key == most - 300 + 512);
    const Plan p = plan_decode(256, 128, 8, 4, most / 2, most / 2, 1);
    CHECK(p.pre_parts > 0 && p.pre_chunk > 0 && (int64_t)p.pre_parts * p.pre_chunk >= most / 2);
    int32_t first, end;
    prompt_keys((int32_t)most, 1000, 999, 64, first, end);
    CHECK(end == most && first < end);
}

// The shapes whose two streams of keys a block the GPU tests count on
static void streams()
{
    for (int hd : {64, 128, 256})
        for (int size : {2, 4}) {
            const bool room = hd * size <= 512;
            const Plan p = plan_prompt(hd * size, hd, 8, 8, 500, 384, 1, 191);
            CHECK(!room || (p.rt == 1 && p.streams == 2));
            const Plan r = plan_prompt(hd * size, hd, 8, 16, 1900, 119, 3, 151);
            CHECK(hd * size > 256 || size == 4 || (r.rt == 2 && r.streams == 2));
        }
    const Plan few = plan_prompt(256, 128, 8, 4, 0, 64, 1, 40);
    CHECK(few.streams == 1);
}

// Grids of any number of blocks: threads of a dimension below 2^32, every block there
static void grids()
{
    for (int64_t n : {1ll, 2ll, 4194303ll, 4194304ll, 4194305ll, 16777216ll, 33554432ll, 33554433ll, 2147483647ll}) {
        const CbqGrid g = cbq_grid(n);
        CHECK(g.x > 0 && (int64_t)g.x * 512 < 1ll << 32 && g.y > 0 && g.y < 65536);
        CHECK((int64_t)g.x * g.y >= n && (int64_t)g.x * (g.y - 1) < n);
        CHECK(g.y == 1 || g.x == 1u << kCbqGridBits);           // so that indexes follow on
        CHECK(cbq_block(0, 0) == 0 && cbq_block(g.x - 1, g.y - 1) == (int64_t)g.x * g.y - 1);
        if (g.y > 1) CHECK(cbq_block(g.x - 1, 0) + 1 == cbq_block(0, 1));
    }
}

// Tables of any width: own parts and blocks within their bounds cover the capacity
static void wide()
{
    const int64_t most = (1ll << 31) - 65536;
    for (int hd : {64, 128, 256})
        for (int size : {2, 4})
            for (int n_kv : {1, 8, 32})
                for (int rep : {1, 17})
                    for (int64_t batch : {1, 512, 4096})
                        for (int64_t capacity : {(int64_t)1 << 20, (int64_t)1 << 30, most - 100})
                            for (int64_t prefix : {0, 100}) {
                                const Plan p = plan_decode(hd * size, hd, n_kv, rep, prefix, capacity, batch);
                                CHECK(plan_fits(p) && !p.joint);
                                CHECK((int64_t)p.own_parts * p.own_chunk >= capacity);
                                CHECK((int64_t)(p.own_parts - 1) * p.own_chunk < capacity);
                                const DecodeWork w = decode_work(p, (uint32_t)(p.blocks - 1), n_kv, (int)batch,
                                                                 (int32_t)prefix, capacity);
                                CHECK(w.seq == batch - 1 && w.part == p.parts - 1 && w.end == capacity);
                                const CbqGrid g = cbq_grid(p.blocks);       // those that fill the grid up
                                for (int64_t i : {p.blocks, (int64_t)g.x * g.y - 1})
                                    CHECK(i < p.blocks || decode_work(p, (uint32_t)i, n_kv, (int)batch, (int32_t)prefix,
                                                                      capacity).part >= p.parts);
                                CHECK(p.bytes == (int64_t)p.parts * batch * n_kv * rep * (hd + 2) * 4);
                            }
}

// "decode ROW_BYTES HD N_KV REP PREFIX CAPACITY BATCH" or "prompt ... N": the plan
static int show(int argc, char **argv)
{
    const std::string kind = argv[1];
    int64_t a[8] = {};
    for (int i = 2; i < argc && i < 10; i++) a[i - 2] = atoll(argv[i]);
    if (kind == "decode" && argc == 9) {
        const Plan p = plan_decode(a[0], a[1], a[2], a[3], a[4], a[5], a[6]);
        printf("joint %d rt %d pre_parts %d own_parts %d\n", p.joint, p.rt, p.pre_parts, p.own_parts);
        return 0;
    }
    if (kind == "prompt" && argc == 10) {
        const Plan p = plan_prompt(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7]);
        printf("rt %d streams %d parts %d\n", p.rt, p.streams, p.parts);
        return 0;
    }
    return 2;
}

int main(int argc, char **argv)
{
    if (argc > 1) return show(argc, argv);
    divisions();
    far();
    grids();
    wide();
    for (int i = 0; i < 150; i++) decode();
    for (int i = 0; i < 400; i++) prompt();
    streams();
    printf("all cases passed\n");
    return 0;
}
