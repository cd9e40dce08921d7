// How the attention of a shared prefix is cut: host and device arithmetic, no GPU needed.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define LCU_HD __host__ __device__
#else
#define LCU_HD
#endif

namespace lcu {

constexpr int PF_ROWS = 256, PF_TILE = 128;  // query rows of a row tile (two MMA tiles), positions of a key tile

// The units (KV head, row tile, key tile) in this order are dealt to the CTAs in contiguous ranges of equal cost; what a CTA does of one
// (KV head, row tile) is a piece with a partial result of its own.  A unit costs 1, or, where a KV head's last row tile fills one MMA tile
// and the others two, 2 there and 3 elsewhere (16 x 5 drafted tokens,
// 320 rows a KV head: 45.5 us with equal costs, 39.9 so).  CTA c's piece of pair p has number c + p: both only grow along the
// units, and each piece begins a new CTA or a new pair, so no two pieces share a number.
struct PrefixPlan {
    int rows;        // query rows of a KV head: tokens x heads of its group
    int row_tiles, key_tiles;
    int pairs, units, per;        // (KV head, row tile); all units; cost of a CTA
    int ctas, cost, cost_last;    // of a unit; of one in a KV head's last row tile
    int slot_rows;   // rows of a piece's slot
    // Parts of a row's own slots, at most, that the (KV head, token) blocks leave for a kernel of its own, which adds up with a warp per row.  0: the
    // blocks add up themselves, one row after another.
    int own_parts;

    LCU_HD int head_cost() const { return ((row_tiles - 1) * cost + cost_last) * key_tiles; }
    // Cost of all units ahead of one; a CTA's units are those where this lies in its range.
    LCU_HD int ahead(int pair, int tile) const {
        const int h = pair / row_tiles, r = pair - h * row_tiles;
        return h * head_cost() + r * cost * key_tiles + tile * (r + 1 < row_tiles ? cost : cost_last);
    }
    LCU_HD int unit_at(unsigned at) const {  // the first with that much ahead of it, or more
        const int h = (int)(at / (unsigned)head_cost()), left = (int)(at - (unsigned)h * (unsigned)head_cost()), full = (row_tiles - 1) * key_tiles;
        if (h >= pairs / row_tiles) return units;
        const int u = h * row_tiles * key_tiles + (left <= full * cost ? (left + cost - 1) / cost : full + (left - full * cost + cost_last - 1) / cost_last);
        return u < units ? u : units;
    }
    LCU_HD int first_cta(int pair) const { return ahead(pair, 0) / per; }
    LCU_HD int last_cta(int pair) const { return ahead(pair, key_tiles - 1) / per; }
    LCU_HD int slots() const { return ctas + pairs; }
};

// Number of (KV head, row tile) pairs of n tokens, `group` query heads per KV head; parts of a row's own slots.
inline long long prefix_pairs(int n, int group, int nkvh) { return (long long)nkvh * ((n * group + PF_ROWS - 1) / PF_ROWS); }
inline int prefix_own_parts(int n, int nkvh, int sms) {
    const long long blocks = (long long)n * nkvh, parts = blocks >= 3LL * sms ? 1 : 3LL * sms / blocks;
    return parts < 8 ? (int)parts : 8;
}

// CTAs that share a (KV head, token)'s slots and add up their parts as a cluster: up to 8 where blocks are few, 64 slots and more each.
inline int own_splits(long long blocks, long long slots, int sms) {
    int splits = 1;
    while (splits < 8 && blocks * splits <= sms && slots > (long long)splits * 64) splits *= 2;
    return splits;
}

// A prefix that the blocks of the own slots read themselves, once per token, instead of the tensor cores once per 256 rows: one launch instead
// of two or three.  Estimates in microseconds, of heads of 128 (and of 64): a warp's 16 slots 0.75 (0.55), an SM 60 KB of keys and values from L2, clusters
// beyond what runs at once their rows' sums; for the tensor cores 4.6 to begin, end and add up, 0.5 more where a third kernel adds up, 2.4 (1.8) a
// round of key tiles.  Measured with 32 heads over 8 of 128, 1 / 8 / 33 tokens: prefix of 16 5.5 / 6.1 / 7.2 us against 10.1 / 10.8 / 14.3; of 600 7.6 /
// 10.6 / 21.8 against 10.5 / 11.1 / 15.3; of 2000 12.1 / 18.9 / 55 against 12.9 / 16.1 / 19.2; of 4000 18 / 31 / 101 against 15 / 18 / 23.
inline bool prefix_walk(int n, int group, int nkvh, uint32_t prefix_len, long long own_slots, int sms, int dh) {
    const long long blocks = (long long)n * nkvh;
    const int splits = own_splits(blocks, own_slots + prefix_len, sms);
    const double steps = (double)prefix_len / (32.0 * splits) * (0.35 + 0.4 * dh / 128), bytes = (double)blocks * prefix_len * dh * 4 / (60e3 * sms);
    const double tiles = (double)prefix_pairs(n, group, nkvh) * ((prefix_len + PF_TILE - 1) / PF_TILE) / sms * (1.2 + 1.2 * dh / 128);
    const double crowd = blocks * splits > sms && splits > 1 ? 0.06 * group * splits : 0;
    return (steps > bytes ? steps : bytes) + crowd < 4.6 + (blocks > sms ? 0.5 : 0) + tiles;
}

// Costs and units are counted in 32 bits, which is more than two seconds of work.
inline bool prefix_fits(int n, int group, int nkvh, uint32_t prefix_len) {
    return prefix_pairs(n, group, nkvh) <= 0x10000000 && prefix_pairs(n, group, nkvh) * ((prefix_len + (long long)PF_TILE - 1) / PF_TILE) <= 0x10000000;
}

// A prefix of prefix_len > 0 positions (that prefix_fits), at most `sms` CTAs; own_slots: what the sequences' own tables have room for.
// One CTA of the prefix fills an SM.  The own slots' blocks get the SMs that it leaves, and all of them behind it: fewer CTAs of the prefix
// with more key tiles each make it longer and the rest shorter.  Estimates in microseconds: 8 to begin and end, a key tile 1.2 to 2.4 (heads
// of 0 to 128), 7 from a piece to the next, own slots (half of what there is room for) at 30 KB per SM.
inline PrefixPlan prefix_plan(int n, int group, int nkvh, uint32_t prefix_len, int sms, int dh, long long own_slots, int n_seq = 0x7fffffff) {
    PrefixPlan p;
    p.rows = n * group;
    p.row_tiles = (p.rows + PF_ROWS - 1) / PF_ROWS;
    p.key_tiles = (int)((prefix_len + PF_TILE - 1) / PF_TILE);
    p.pairs = (int)prefix_pairs(n, group, nkvh);
    p.units = p.pairs * p.key_tiles;
    p.slot_rows = p.rows < PF_ROWS ? p.rows : PF_ROWS;
    const int last = p.rows - (p.row_tiles - 1) * PF_ROWS;  // rows of the last row tile
    const bool uneven = p.row_tiles > 1 && last <= 128;
    p.cost = uneven ? 3 : 1;
    p.cost_last = uneven ? 2 : 1;
    const int total = nkvh * p.head_cost();
    const long long pair_cost = (long long)p.key_tiles * p.cost;
    const double tile = (1.2 + 1.2 * dh / 128) * (p.row_tiles == 1 && last <= 128 ? 0.7 : 1) / p.cost, own = (double)nkvh * own_slots * dh * 4 * 0.5 / 30e3;  // the latter in SM microseconds
    const long long fair = ((long long)total + sms - 1) / sms, least = fair < p.cost ? p.cost : fair;  // no range without a unit
    // More blocks than SMs do not add up: they would wait for the prefix and hold their places from those that have not begun.  Nor do blocks of
    // many rows and parts: a warp takes every second row, and eight parts of it, in a microsecond, where the third kernel costs 2.5 (64 heads over
    // 8, 2 x 5 drafted tokens behind 1391 26.5 us and 14.6 with it, 16 over 1, 3 x 5 behind 9000 64 and 25; 32 over 8, 3 tokens behind 8000, 6 rounds, 22.8
    // and 25.2).
    const long long each = ((long long)n + n_seq - 1) / n_seq, tokens = each < 16 / group ? each : 16 / group;  // of a block, about
    const long long rounds = (pair_cost / least + 9) / 8 * ((tokens * group + 1) / 2);
    p.own_parts = (long long)n * nkvh > sms || rounds > 6 ? prefix_own_parts(n, nkvh, sms) : 0;
    double best = 0;
    for (long long per = least; per <= 8 * least && (per == least || per <= total); ++per) {
        const long long ctas = (total - p.cost_last) / per + 1;
        const long long pieces = per >= pair_cost ? (per + pair_cost - 1) / pair_cost : pair_cost % per ? 2 : 1;
        const double prefix = 1 + 7 * pieces + tile * per, left = p.own_parts ? own - (double)(sms - ctas) * (prefix - 8) : 0;
        const double t = prefix + (left > 0 ? left / sms + (left < 4.0 * sms ? left * 1.5 / sms : 6) : 0);
        if (per == least || t < best) {
            best = t;
            p.per = (int)per;
            p.ctas = (int)ctas;
        }
        if (!p.own_parts || per > least + 64 * p.cost) break;
    }
    return p;
}

// Workspace: (maximum, sum) of each row of every slot, then of the own parts, [part][KV head][row]; then their unnormalised outputs.
inline size_t prefix_own_row(const PrefixPlan &p) { return (size_t)p.slots() * p.slot_rows; }
inline size_t prefix_part_rows(const PrefixPlan &p, int nkvh) { return prefix_own_row(p) + (size_t)p.own_parts * nkvh * p.rows; }
inline size_t prefix_ml_bytes(const PrefixPlan &p, int nkvh) { return (prefix_part_rows(p, nkvh) * 8 + 255) / 256 * 256; }
// ... at most, whatever the plan
inline size_t prefix_bytes(int n, int group, int nkvh, uint32_t prefix_len, int sms, int dh) {
    PrefixPlan p = prefix_plan(n, group, nkvh, prefix_len, sms, dh, 0);
    p.ctas = sms;
    p.own_parts = prefix_own_parts(n, nkvh, sms);
    return prefix_ml_bytes(p, nkvh) + prefix_part_rows(p, nkvh) * dh * 4;
}

}  // namespace lcu
