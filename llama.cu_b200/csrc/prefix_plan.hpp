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

// The units (KV head, row tile, key tile) in this order are dealt to the CTAs in equal contiguous ranges; what a CTA does of one
// (KV head, row tile) is a piece with a partial result of its own.  CTA c's piece of pair p has number c + p: both only grow along the
// units, and each piece begins a new CTA or a new pair, so no two pieces share a number.
struct PrefixPlan {
    int rows;        // query rows of a KV head: tokens x heads of its group
    int row_tiles, key_tiles;
    long long pairs, units, per;  // (KV head, row tile); all units; units of a CTA
    int ctas;
    int slot_rows;   // rows of a piece's slot
    // More (KV head, token) blocks for the own slots than SMs: they leave their parts too, at most so many of a row, and a kernel of its
    // own adds up.  (A block that adds up waits for the prefix, and would hold its place beside it from the blocks that have not begun.)
    int own_parts;

    LCU_HD long long first_cta(long long pair) const { return pair * key_tiles / per; }
    LCU_HD long long last_cta(long long pair) const { return ((pair + 1) * key_tiles - 1) / per; }
    LCU_HD long long slots() const { return ctas + pairs; }
};

// n tokens, `group` query heads per KV head, a prefix of prefix_len > 0 positions, at most `sms` CTAs
inline PrefixPlan prefix_plan(int n, int group, int nkvh, uint32_t prefix_len, int sms) {
    PrefixPlan p;
    p.rows = n * group;
    p.row_tiles = (p.rows + PF_ROWS - 1) / PF_ROWS;
    p.key_tiles = (int)((prefix_len + PF_TILE - 1) / PF_TILE);
    p.pairs = (long long)nkvh * p.row_tiles;
    p.units = p.pairs * p.key_tiles;
    p.per = (p.units + sms - 1) / sms;
    p.ctas = (int)((p.units + p.per - 1) / p.per);
    p.slot_rows = p.rows < PF_ROWS ? p.rows : PF_ROWS;
    const long long blocks = (long long)n * nkvh;
    p.own_parts = blocks <= sms ? 0 : blocks >= 6LL * sms ? 1 : (int)(6LL * sms / blocks);
    return p;
}

// Workspace, in rows: those of every slot, then those of the own parts, [part][KV head][row].  (maximum, sum) of each, then their unnormalised outputs.
inline size_t prefix_own_row(const PrefixPlan &p) { return (size_t)p.slots() * p.slot_rows; }
inline size_t prefix_part_rows(const PrefixPlan &p, int nkvh) { return prefix_own_row(p) + (size_t)p.own_parts * nkvh * p.rows; }
inline size_t prefix_ml_bytes(const PrefixPlan &p, int nkvh) { return (prefix_part_rows(p, nkvh) * 8 + 255) / 256 * 256; }
inline size_t prefix_bytes(const PrefixPlan &p, int nkvh, int dh) { return prefix_ml_bytes(p, nkvh) + prefix_part_rows(p, nkvh) * dh * 4; }

}  // namespace lcu
