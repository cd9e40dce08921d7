// Attention of a batch whose sequences share a prefix, on a caller's pages (no counterpart in the reference, whose sessions share nothing on the
// device): one softmax over the prefix and the token's own slots,
//
//   o = sum_j exp(scale q k_j - m) v_j / sum_j exp(scale q k_j - m),   j in the prefix, then in the token's own slots
//
// cut where the keys are: partial sums relative to a maximum of their own, (m, l, O), add up as O 2^(m - M), l 2^(m - M).
//
//  - prefix_tc_kernel: the prefix, for all tokens at once, on the 5th-generation tensor cores.  The query rows (token, head of the group) of
//    a KV head fill tiles of 256 rows, so the prefix is read once per 256 rows instead of once per token; the roles, tensor memory and
//    arithmetic are those of attention_tc.cu.  The units (KV head, row tile, key tile) are dealt to one CTA per SM in
//    contiguous ranges of equal cost; a CTA leaves one partial result per (KV head, row tile) that it meets.
//  - own_kernel: each token's own slots.  A CTA owns a KV head and up to 16 query rows of one sequence's consecutive tokens (drafted tokens
//    share their keys); its two warps take 16 keys each in turns, with a softmax of their own and both products in registers (mma.sync),
//    and meet once at the end.  It is launched as a programmatic dependent: its blocks run on the SMs that the prefix leaves, then on all.
//  - The sum of all parts: at the end of own_kernel where its blocks, their rows and the parts are few, else in own_sum_kernel.
//  - A prefix that is short next to the number of tokens is read by own_kernel too, ahead of the token's own slots, and the call is one launch.
//
// Measured on a B200 (calls in a graph), heads of 128: 256 tokens of 64 heads over 8 behind 32000 positions 293 us (0.92 PFLOP/s; exponentials and products
// take turns, half of the time each) and 324 in long runs at 1000 W; 16 x 5 drafted tokens of 32 over 8 behind 8001 35.4 us: prefix 22 (15 of units, 7 to
// begin, end and leave parts), own slots 9, sum 4.  A unit there is a chain: scores, maximum, accumulator, exponentials, products, one warp to a scheduler
// and tile; tensor cores, exponentials and issue slots are each busy a quarter of the time.
//
// f32 scores and softmax, sums in f32 over the weights as they are, weights rounded to the activation type ahead of the second product (its
// operands are 16-bit), one rounding of the output.  (Sums over the rounded weights, as attention.cu takes them, are no closer to the
// softmax where many weights count and cost 4 % of the prefix in conversions; a weight that stands alone is a power of two and is not rounded.)
// The largest weight of a part is 1, but 2^14 in f16: f16 ends at 2^-24, and below a 1 thousands of keys 2^-25 of it each would be in the sum and
// not in the product.  The power of two is in the maximum that a part is relative to, so the sum of parts knows nothing of it.
#include "attention_tc.cuh"
#include "paged.cuh"
#include "prefix_plan.hpp"

#include <type_traits>

namespace lcu {

template <class T> constexpr float PF_TOP = 0.f;  // the largest weight is 2^PF_TOP
template <> constexpr float PF_TOP<__half> = 14.f;
// what weights are relative to, of the largest scaled score (rounded up: no weight is above the largest, however large the scores)
template <class T> __device__ __forceinline__ float pf_reference(float n) {
    if constexpr (PF_TOP<T> != 0.f) return __fsub_ru(n, PF_TOP<T>);
    return n;
}

struct PrefixArgs {
    void *o;
    const void *q;
    int sto, sho, stq, shq;
    lcu_kv_pages pages;
    const int32_t *prefix_table, *table, *tok_seq;
    const uint32_t *tok_ctx;
    uint32_t prefix_len;  // of the parts in the workspace
    uint32_t walk_len;    // or of what own_kernel reads itself, ahead of the token's own slots
    int table_stride, n_seq, page_shift, n, nh, nkvh;
    float scale2;  // scores in powers of two
    PrefixPlan plan;
    float2 *part_ml;  // [slot][row], then own parts [part][KV head][row]
    float *part_o;    // ... [dh]
    size_t own_row;   // where the latter begin
};

// ------------------------------------------------------------------ the prefix

constexpr int PF_THREADS = 320;
constexpr int PF_MAX_STAGES = 4;

struct PfShared {
    unsigned long long k_full[PF_MAX_STAGES], k_empty[PF_MAX_STAGES], v_full[PF_MAX_STAGES], v_empty[PF_MAX_STAGES];
    unsigned long long q_full[2], s_full[2], p_ready[2][2], pv_done[2], drain;
    volatile int unit0, unit1;  // of the CTA (read where they are needed: registers are short)
    uint32_t tmem_base;
    int abort_flag;
};

template <int DH> constexpr int pf_stages() { return DH == 64 ? 4 : 2; }
template <int DH> constexpr size_t pf_smem() { return 1024 + (size_t)(DH / 64) * AT_BOX * (2 + 2 * pf_stages<DH>()) + sizeof(PfShared); }

__device__ __forceinline__ void pf_tma_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n}"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
// four products of K = 16, weights in tensor memory (8 columns each), values in shared memory (2 KB each): one election for all
__device__ __forceinline__ void pf_mma_ts4(uint32_t d, uint32_t w, uint64_t v, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred e, p, q;\n .reg .b32 a;\n .reg .b64 b;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 q, 0, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n add.u32 a, %1, 8;\n add.u64 b, %2, 128;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n add.u32 a, %1, 16;\n add.u64 b, %2, 256;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n add.u32 a, %1, 24;\n add.u64 b, %2, 384;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, q;\n}"
                 ::"r"(d), "r"(w), "l"(v), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pf_st8(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void pf_arrive(uint32_t bar, int lane) {  // of a warp, behind its accesses to tensor or shared memory
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pf_st32(float *p, const uint32_t *r) {  // 32 bytes at once: a row per lane, so each store is a sector of its own
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

// what a CTA does of one (KV head, row tile)
struct PfPiece {
    int unit, pair;  // first unit
    int hkv, row0, rows, j0, j1;
    bool two;
};
__device__ __forceinline__ PfPiece pf_piece(const PrefixPlan &pl, int unit, int end) {  // end: first unit behind the CTA's range
    PfPiece p;
    p.unit = unit;
    p.pair = unit / pl.key_tiles;
    p.j0 = unit - p.pair * pl.key_tiles;
    p.j1 = min(pl.key_tiles, p.j0 + (end - unit));
    p.hkv = p.pair / pl.row_tiles;
    p.row0 = (p.pair - p.hkv * pl.row_tiles) * PF_ROWS;
    p.rows = min(PF_ROWS, pl.rows - p.row0);
    p.two = p.rows > 128;
    return p;
}
__device__ __forceinline__ PfPiece pf_next(const PrefixPlan &pl, const PfPiece &p, int end) { return pf_piece(pl, p.unit + (p.j1 - p.j0), end); }

template <class T, int DH>
__global__ void __launch_bounds__(PF_THREADS, 1)
prefix_tc_kernel(const PrefixArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, uint32_t fmt) {
    constexpr int NB = DH / 64, TILE = NB * AT_BOX, ST = pf_stages<DH>();
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (tc_smem(smem_raw) & 1023u)) & 1023u);
    unsigned char *Qs = smem, *Ks = Qs + 2 * TILE, *Vs = Ks + ST * TILE;
    PfShared *sh = reinterpret_cast<PfShared *>(Vs + ST * TILE);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    grid_dep_launch();
    const int ppt = 128 >> a.page_shift, n_prefix_pages = (int)((a.prefix_len + a.pages.page_tokens - 1) >> a.page_shift);  // pages of a tile, of all

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            tc_mbar_init(tc_smem(&sh->k_full[i]), 1);
            tc_mbar_init(tc_smem(&sh->k_empty[i]), 1);
            tc_mbar_init(tc_smem(&sh->v_full[i]), 1);
            tc_mbar_init(tc_smem(&sh->v_empty[i]), 1);
        }
        tc_mbar_init(tc_smem(&sh->drain), 1);
        for (int t = 0; t < 2; ++t) {
            tc_mbar_init(tc_smem(&sh->q_full[t]), 4);
            tc_mbar_init(tc_smem(&sh->s_full[t]), 1);
            tc_mbar_init(tc_smem(&sh->p_ready[t][0]), 4);
            tc_mbar_init(tc_smem(&sh->p_ready[t][1]), 4);
            tc_mbar_init(tc_smem(&sh->pv_done[t]), 1);
        }
        sh->abort_flag = 0;
        sh->unit0 = a.plan.unit_at(blockIdx.x * (unsigned)a.plan.per);
        sh->unit1 = a.plan.unit_at((blockIdx.x + 1) * (unsigned)a.plan.per);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&sh->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh->tmem_base, tmem_o = tmem + 256;  // S_t in columns 128 t .., O_t behind them
    int k_issued = 0, v_issued = 0;  // stages that warp 0 has requested

    if (warp == 0) {
        // ---------------- TMA producer: the ring runs on through all pieces
        const uint32_t kf = tc_smem(&sh->k_full[0]), ke = tc_smem(&sh->k_empty[0]), vf = tc_smem(&sh->v_full[0]), ve = tc_smem(&sh->v_empty[0]);
        const int pt = a.pages.page_tokens;
        const int u0 = sh->unit0, u1 = sh->unit1;
        auto page_of = [&](int tile) {  // lane i: page i of the tile; an id that names no page is one behind the map, which reads zeros
            const int i = tile * ppt + lane;
            const int id = lane < ppt && i < n_prefix_pages ? a.prefix_table[i] : 0;
            return id < 0 || id >= a.pages.n_pages ? a.pages.n_pages : id;
        };
        int slot = 0, hkv = u0 / a.plan.key_tiles / a.plan.row_tiles, j = u0 % a.plan.key_tiles;
        int pair = u0 / a.plan.key_tiles;
        int id = page_of(j);
        auto load = [&](uint32_t dst, const CUtensorMap *map, uint32_t bar, int n) {
            tc_warp_expect_tx(bar, (uint32_t)(n * pt * 128 * NB));
            for (int i = 0; i < n; ++i) {
                const int page = __shfl_sync(0xffffffffu, id, i);
                for (int b = 0; b < NB; ++b) pf_tma_4d(dst + (uint32_t)(b * AT_BOX + i * pt * 128), map, 64 * b, 0, hkv, page, bar);
            }
        };
        uint32_t phase = 1;
        bool ok = true;
        for (int u = u0; u < u1; ++u) {
            const int n = min(ppt, n_prefix_pages - j * ppt);
            ok = tc_warp_wait(ke + 8 * slot, phase, &sh->abort_flag);
            if (!ok) break;
            load(tc_smem(Ks) + (uint32_t)(slot * TILE), &map_k, kf + 8 * slot, n);
            ++k_issued;
            ok = tc_warp_wait(ve + 8 * slot, phase, &sh->abort_flag);
            if (!ok) break;
            load(tc_smem(Vs) + (uint32_t)(slot * TILE), &map_v, vf + 8 * slot, n);
            ++v_issued;
            if (++j == a.plan.key_tiles) {
                j = 0;
                ++pair;
                hkv = pair / a.plan.row_tiles;
            }
            if (u + 1 < u1) id = page_of(j);
            if (++slot == ST) { slot = 0; phase ^= 1u; }
        }
        if (!ok) sh->abort_flag = 1;
    } else if (warp == 1) {
        // ---------------- MMA issuer
        const uint32_t id_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        const uint32_t id_o = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)(DH >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        const uint64_t q0 = tc_desc(tc_smem(Qs)), k0 = tc_desc(tc_smem(Ks)), v0 = at_desc_mn(tc_smem(Vs));
        const uint32_t kf = tc_smem(&sh->k_full[0]), ke = tc_smem(&sh->k_empty[0]), vf = tc_smem(&sh->v_full[0]), ve = tc_smem(&sh->v_empty[0]);
        const uint32_t sf = tc_smem(&sh->s_full[0]), pr = tc_smem(&sh->p_ready[0][0]), pd = tc_smem(&sh->pv_done[0]), qf = tc_smem(&sh->q_full[0]);
        auto scores = [&](int t, int slot) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
                tc_warp_mma4(tmem + 128 * t, q0 + (uint64_t)((t * TILE + b * AT_BOX) >> 4), k0 + (uint64_t)((slot * TILE + b * AT_BOX) >> 4), id_s, b > 0);
            tc_warp_commit(sf + 8 * t);
        };
        int slot = 0;
        uint32_t phase = 0, p_phase = 0, q_phase = 0, seen = 0;  // bit t of the last three: tile t's; whether it has had products
        bool ok = true;
        for (PfPiece p = pf_piece(a.plan, sh->unit0, sh->unit1); ok && p.unit < sh->unit1; p = pf_next(a.plan, p, sh->unit1)) {
            const int nt = p.two ? 2 : 1;
            for (int t = 0; t < nt && ok; ++t) {
                ok = tc_warp_wait(qf + 8 * t, q_phase >> t & 1u, &sh->abort_flag);
                q_phase ^= 1u << t;
            }
            ok = ok && tc_warp_wait(kf + 8 * slot, phase, &sh->abort_flag);
            for (int t = 0; t < nt && ok; ++t)
                if (seen >> t & 1u) ok = tc_warp_wait(pd + 8 * t, (p_phase >> t & 1u) ^ 1u, &sh->abort_flag);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            seen |= nt == 2 ? 3u : 1u;
            for (int t = 0; t < nt; ++t) scores(t, slot);
            tc_warp_commit(ke + 8 * slot);
            for (int j = p.j0; j < p.j1 && ok; ++j) {
                const int next = slot + 1 == ST ? 0 : slot + 1;
                const uint32_t next_phase = slot + 1 == ST ? phase ^ 1u : phase;
                const bool more = j + 1 < p.j1;
                ok = tc_warp_wait(vf + 8 * slot, phase, &sh->abort_flag);
                if (ok && more) ok = tc_warp_wait(kf + 8 * next, next_phase, &sh->abort_flag);
                for (int t = 0; t < nt && ok; ++t) {
                    for (int h = 0; h < 2 && ok; ++h) {  // weights of 64 positions at a time
                        ok = tc_warp_wait(pr + 16 * t + 8 * h, p_phase >> t & 1u, &sh->abort_flag);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        pf_mma_ts4(tmem_o + DH * t, tmem + 128 * t + 32 * h, v0 + (uint64_t)((slot * TILE + h * 8192) >> 4), id_o, j > p.j0 || h > 0);
                    }
                    if (!ok) break;
                    tc_warp_commit(pd + 8 * t);
                    if (t == nt - 1) tc_warp_commit(ve + 8 * slot);
                    if (more) {
                        // The next scores go over the columns of these weights.  Products of unlike shapes or accumulators are not ordered
                        // among themselves, so the ones that read the weights have to have ended (1 % of the time).
                        ok = tc_warp_wait(pd + 8 * t, p_phase >> t & 1u, &sh->abort_flag);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        scores(t, next);
                        if (t == nt - 1) tc_warp_commit(ke + 8 * next);
                    }
                    p_phase ^= 1u << t;
                }
                slot = next;
                phase = next_phase;
            }
        }
        if (!ok) sh->abort_flag = 1;
    } else {
        // ---------------- queries, softmax and partial output of one tile: a row per thread
        const int t = (warp - 2) >> 2, q = warp & 3, row = q * 32 + lane;  // a warp may only touch TMEM lanes [32 q, 32 q + 32)
        const int group = a.nh / a.nkvh;
        const uint32_t ts = tmem + ((uint32_t)(q * 32) << 16) + 128 * t, to = tmem_o + ((uint32_t)(q * 32) << 16) + DH * t;
        // 16 bytes per thread and step, as the 128-byte swizzle has them; zeros behind the last row.  A short loop of asynchronous copies: unrolled,
        // with the rows in registers, it was the longest part of a cold start (4 of 5 us).
        auto load_q = [&](const PfPiece &p) {
            constexpr int CH = DH / 8, STEP = 128 / CH;  // rows a step
            const int i = tid - 64 - 128 * t, c = i % CH, r0 = i / CH, left = p.rows - 128 * t;
            int tok = (p.row0 + 128 * t + r0) / group, g = p.row0 + 128 * t + r0 - tok * group;
            const int tok_step = STEP / group, g_step = STEP - tok_step * group;
            uint32_t dst = tc_smem(Qs) + (uint32_t)(t * TILE + (c >> 3) * AT_BOX + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4));
#pragma unroll 1
            for (int r = r0; r < 128; r += STEP) {
                const bool valid = r < left;
                const T *src = reinterpret_cast<const T *>(a.q) + (valid ? (size_t)tok * a.stq + (size_t)(p.hkv * group + g) * a.shq + 8 * c : 0);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
                dst += STEP * 128;
                tok += tok_step;
                g += g_step;
                if (g >= group) {
                    g -= group;
                    ++tok;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            pf_arrive(tc_smem(&sh->q_full[t]), lane);
        };
        auto bad_pages = [&](int tile) {  // bit i: page i of the tile names no page
            const int i = tile * ppt + lane;
            const int id = lane < ppt && i < n_prefix_pages ? a.prefix_table[i] : 0;
            return __ballot_sync(0xffffffffu, id < 0 || id >= a.pages.n_pages);
        };
        const uint32_t pr = tc_smem(&sh->p_ready[t][0]);
        int it = 0;          // units of the CTA so far
        uint32_t mine = 0;   // ... that had this tile
        bool ok = true;
        PfPiece p = pf_piece(a.plan, sh->unit0, sh->unit1);
        if (t == 0 || p.two) load_q(p);
        while (p.unit < sh->unit1) {
            const bool active = t == 0 || p.two, some = active && 128 * t + q * 32 < p.rows;  // ... of this warp's rows
            float top = -INFINITY, ref = -INFINITY, l = 0.f;  // the largest score; what weights are relative to; their sum
            bool far = true;                                  // of the warp: a ref is so large that its rounding counts, or there is none yet
            if (active) {
                unsigned bad = bad_pages(p.j0);
                for (int j = p.j0; j < p.j1; ++j, ++mine) {
                    const int p0 = j * 128, left = (int)min((long long)a.prefix_len - p0, 128ll);
                    if (t == 0 && left < 128) {  // V rows behind the prefix: whatever a page holds there has weight zero
                        const int u = it + (j - p.j0), slot = u % ST;
                        ok = tc_mbar_wait(tc_smem(&sh->v_full[slot]), (uint32_t)(u / ST) & 1u, &sh->abort_flag);
                        uint4 *v = reinterpret_cast<uint4 *>(Vs + (size_t)slot * TILE);
                        for (int i = left * 8 + (tid - 64); ok && i < 128 * 8; i += 128)
#pragma unroll
                            for (int b = 0; b < NB; ++b) v[b * (AT_BOX / 16) + i] = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    ok = ok && tc_mbar_wait(tc_smem(&sh->s_full[t]), mine & 1u, &sh->abort_flag);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    const unsigned hide = bad;
                    if (j + 1 < p.j1) bad = bad_pages(j + 1);
                    if (some) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        uint32_t s[128];
#pragma unroll
                        for (int c = 0; c < 128; c += 32) at_ld32(ts + c, s + c);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (left < 128 || hide) {
#pragma unroll
                            for (int c = 0; c < 128; ++c)
                                if (c >= left || (hide >> (c >> a.page_shift) & 1u)) s[c] = 0xff800000u;
                        }
                        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 128; c += 8)
#pragma unroll
                            for (int i = 0; i < 4; ++i) m4[i] = at_max3(m4[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 4 + i]));
                        const float most = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), m = pf_reference<T>(most * a.scale2);
                        if (__any_sync(0xffffffffu, m > ref) || far) {
                            const float mn = fmaxf(ref, m), corr = ref == -INFINITY ? 0.f : at_exp2(ref - mn);
                            l *= corr;
                            ref = mn;
                            top = fmaxf(top, most);
                            if (j > p.j0) {
#pragma unroll 1
                                for (int c = 0; c < DH; c += 16) {
                                    uint32_t o[16];
                                    tc_ld16(to + c, o);
                                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                                    at_st16(to + c, o);
                                }
                            }
                            far = __any_sync(0xffffffffu, fabsf(ref) >= 4096.f);
                        }
                        const unsigned long long mul = at_pair(a.scale2, a.scale2);
                        unsigned long long l2[2] = {0ull, 0ull};
                        auto weights = [&](auto difference_first, float sub, float plus) {
                            const unsigned long long off = at_pair(-sub, -sub), off2 = at_pair(plus, plus);
#pragma unroll
                            for (int h = 0; h < 8; ++h) {
                                uint32_t w[8];
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const int c = 16 * h + 2 * i;
                                    const unsigned long long v = at_pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                                    const float2 x = at_unpair(difference_first ? at_fma2(at_add2(v, off), mul, off2) : at_fma2(v, mul, off));
                                    const float y0 = at_exp2(x.x), y1 = at_exp2(x.y);
                                    w[i] = Act<T>::pack(y0, y1);
                                    l2[i & 1] = at_add2(l2[i & 1], at_pair(y0, y1));
                                }
                                pf_st8(ts + 8 * h, w);
                                if (h == 3) {
                                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                                    pf_arrive(pr, lane);
                                }
                            }
                        };
                        // ref is rounded and the product inside the FMA is not: a row's weights are all off by the same factor, 2^(half a step of ref).
                        // Steps of 2^-12 and less are nothing; beyond, the difference to the largest score comes first, so that weights end where they should.
                        // (Two copies cost 1 %; one, with scores that a branch may have changed, 3 to 4.)
                        if (far) {
                            const bool none = top == -INFINITY;  // a row whose scores are all -inf keeps zero weights
                            weights(std::true_type{}, none ? 0.f : top, none ? 0.f : __fmul_rn(top, a.scale2) - ref);
                        } else weights(std::false_type{}, ref, 0.f);
                        const float2 la = at_unpair(at_add2(l2[0], l2[1]));
                        l += la.x + la.y;
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    } else {
                        pf_arrive(pr, lane);
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    pf_arrive(pr + 8, lane);
                }
                if (!ok) break;
            }
            it += p.j1 - p.j0;
            const PfPiece next = pf_next(a.plan, p, sh->unit1);
            // the products of this tile's scores have ended (their last commit was waited for): its queries may be replaced
            if (next.unit < sh->unit1 && (t == 0 || next.two)) load_q(next);
            if (active) {
                ok = tc_mbar_wait(tc_smem(&sh->pv_done[t]), (mine - 1) & 1u, &sh->abort_flag);  // (those before it had ended when the last scores were issued)
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const size_t at = (size_t)(blockIdx.x + p.pair) * a.plan.slot_rows + 128 * t + row;
                const bool valid = 128 * t + row < p.rows;
                if (valid) a.part_ml[at] = make_float2(ref, l);
                if (some) {
#pragma unroll
                    for (int c = 0; c < DH; c += 32) {
                        uint32_t o[32];
                        at_ld32(to + c, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        if (!valid) continue;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) pf_st32(a.part_o + at * DH + c + i, o + i);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
            p = next;
        }
        if (!ok) sh->abort_flag = 1;
    }
    __syncthreads();
    if (sh->abort_flag) {  // a wait has run out: what still writes to the CTA's memory ends first, and the rows it had become NaN
        if (warp == 0) {
            tc_warp_drain_ring(tc_smem(&sh->k_full[0]), k_issued, ST);
            tc_warp_drain_ring(tc_smem(&sh->v_full[0]), v_issued, ST);
        }
        if (warp == 1) {
            tc_warp_commit(tc_smem(&sh->drain));
            tc_warp_drain(tc_smem(&sh->drain), 0u);
        }
        for (PfPiece p = pf_piece(a.plan, sh->unit0, sh->unit1); p.unit < sh->unit1; p = pf_next(a.plan, p, sh->unit1))
            for (int r = tid; r < p.rows; r += PF_THREADS) a.part_ml[(size_t)(blockIdx.x + p.pair) * a.plan.slot_rows + r] = make_float2(0.f, __int_as_float(0x7fc00000));
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ------------------------------------------------------------------ own slots, and the sum

constexpr int OW_KEYS = 16, OW_WARPS = 2, OW_THREADS = 32 * OW_WARPS;
// A warp's tiles: keys and values of the chunk that it works on and, where blocks are few, of the next (eight blocks of a ring of one on an SM, five
// of a ring of two: 264 blocks that read 4000 slots each take 101 us with two and 122 with one, 800 blocks and 1000 slots 68 and 56).
template <int DH> constexpr size_t ow_tile_bytes() { return (size_t)OW_KEYS * (DH + 8) * 2; }
constexpr int ow_tiles(int depth) { return OW_WARPS * 2 * depth; }
template <int DH> constexpr size_t ow_smem(int depth) { return (ow_tiles(depth) + 1) * ow_tile_bytes<DH>(); }  // and the queries; later the warps' parts: 16 rows of DH f32 each
static_assert(ow_smem<64>(1) >= OW_WARPS * 16 * 64 * 4 && ow_smem<128>(1) >= OW_WARPS * 16 * 128 * 4, "parts of the warps");
template <int DH> constexpr size_t ow_part_bytes() { return (size_t)16 * DH * 4 + 16 * 8; }  // a CTA's part in the first one's memory (clusters)

__device__ __forceinline__ void ow_cp16(void *dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ow_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ow_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}
__device__ __forceinline__ void ow_ldm4(uint32_t r[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}
__device__ __forceinline__ void ow_ldm4t(uint32_t r[4], const void *p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)) : "memory");
}
__device__ __forceinline__ float ow_quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float ow_quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// factor of a part (m, l, O) in a sum relative to M: a part without a maximum has l = 0 and O = 0, or NaN, which stays
__device__ __forceinline__ float ow_factor(float m, float M) { return m == -INFINITY ? 1.f : at_exp2(m - M); }

// a row's part, spread over a warp: PD values per lane
template <int PD> struct OwPart {
    float m, l, o[PD];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < PD; ++i) o[i] = 0.f;
    }
    __device__ __forceinline__ void add(float pm, float pl, const float *v) {
        const float M = fmaxf(m, pm), f = ow_factor(m, M), g = ow_factor(pm, M);
        m = M;
        l = l * f + pl * g;
#pragma unroll
        for (int i = 0; i < PD; ++i) o[i] = o[i] * f + v[i] * g;
    }
};

// Adds the prefix's parts of row `row` of a KV head, and `own` parts of its own slots in the workspace; normalises and stores.  Eight parts at a
// time, all of whose loads are in flight together: rows are few next to what the memory can hold in flight, and each trip costs a microsecond.
template <class T, int DH>
__device__ __forceinline__ void ow_finish(const PrefixArgs &a, OwPart<DH / 32> &p, int hkv, int row, int own, int lane) {
    constexpr int PD = DH / 32, AHEAD = 8;
    const int group = a.nh / a.nkvh, tok = row / group;
    if (a.prefix_len) {
        const int pair = hkv * a.plan.row_tiles + row / PF_ROWS, first = a.plan.first_cta(pair);
        const int shared = a.plan.last_cta(pair) - first + 1, parts = shared + own;
        const size_t at0 = (size_t)(first + pair) * a.plan.slot_rows + row % PF_ROWS, at1 = a.own_row + (size_t)hkv * a.plan.rows + row;
        const size_t apart1 = (size_t)a.nkvh * a.plan.rows;
        auto at = [&](int s) { return s < shared ? at0 + (size_t)s * a.plan.slot_rows : at1 + (size_t)(s - shared) * apart1; };
#pragma unroll 1
        for (int s0 = 0; s0 < parts; s0 += AHEAD) {
            float v[AHEAD][PD];
            const float2 x = lane < AHEAD && s0 + lane < parts ? __ldcg(a.part_ml + at(s0 + lane)) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (s0 + i >= parts) break;
                const float *src = a.part_o + at(s0 + i) * DH;
                if constexpr (PD == 4) {
                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(src) + lane);
                    v[i][0] = y.x; v[i][1] = y.y; v[i][2] = y.z; v[i][3] = y.w;
                } else {
                    const float2 y = __ldcg(reinterpret_cast<const float2 *>(src) + lane);
                    v[i][0] = y.x; v[i][1] = y.y;
                }
            }
            const float M = fmaxf(p.m, warp_max(x.x)), f = ow_factor(p.m, M), g = ow_factor(x.x, M);
            p.m = M;
            p.l = p.l * f + warp_sum(x.y * g);
#pragma unroll
            for (int d = 0; d < PD; ++d) p.o[d] *= f;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const float w = __shfl_sync(0xffffffffu, g, i);
                if (s0 + i < parts)
#pragma unroll
                    for (int d = 0; d < PD; ++d) p.o[d] = fmaf(v[i][d], w, p.o[d]);
            }
        }
    }
    const float inv = p.l == 0.f ? 0.f : 1.f / p.l;
    T *dst = reinterpret_cast<T *>(a.o) + (size_t)tok * a.sto + (size_t)(hkv * group + row % group) * a.sho + lane * PD;
#pragma unroll
    for (int i = 0; i < PD; i += 2) *reinterpret_cast<uint32_t *>(dst + i) = Act<T>::pack(p.o[i] * inv, p.o[i + 1] * inv);
}

// grid (splits, KV heads, tokens); the splits of a token are a cluster where own_kernel adds up.
// Bound by the chain of instructions of a step (16 keys: 404 instructions, 3.6 cycles each with one warp on a scheduler; loads are 0.1 of these), and
// where blocks fill the SMs by L2 at 60 KB per SM and microsecond.  Hence two chains of products for the scores, and no branch around masks or copies:
// with branches the step has 280 instructions and takes 20 % longer.
template <class T, int DH, int DEPTH>
__global__ void __launch_bounds__(OW_THREADS, DEPTH == 1 ? 8 : 5) own_kernel(const PrefixArgs a, int tokens_per, int splits) {
    constexpr int ROW = DH + 8, KS = DH / 16, PD = DH / 32, CH = DH / 8;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float ml[OW_WARPS][16][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, t4 = lane & 3;
    const int hkv = blockIdx.y, t = blockIdx.z, split = blockIdx.x, group = a.nh / a.nkvh;
    const bool first_block = (blockIdx.x | blockIdx.y | blockIdx.z) == 0;
    grid_dep_launch();
    const bool leave = a.prefix_len && a.plan.own_parts, cluster = splits > 1 && !leave;
    if (cluster) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for ahead of stores to the first CTA
    // consecutive tokens of one sequence, cut at multiples of tokens_per
    // (of all tokens that may be among them, in one round trip)
    const int before = t % tokens_per, most = min(tokens_per - before, a.n - t);
    const int lane_seq = a.tok_seq[t + min(lane, most - 1)], last_seq = before ? a.tok_seq[t - 1] : -1;
    const uint32_t lane_ctx = a.tok_ctx[t + min(lane, most - 1)];
    const int seq = __shfl_sync(0xffffffffu, lane_seq, 0);
    const bool mine = seq >= 0 && seq < a.n_seq && (before == 0 || last_seq != seq);
    if (!mine) {
        if (cluster) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (first_block) grid_dep_wait();  // the grid ends behind the prefix, whatever its blocks have to do
        return;
    }
    const unsigned same = __ballot_sync(0xffffffffu, lane < most && lane_seq == seq);
    const int n_tok = __ffs(~same) - 1, rows = n_tok * group;  // most <= 16: there is a zero
    const uint32_t cap = (uint32_t)a.table_stride << a.page_shift;
    uint32_t ctx = 0;  // of the longest
    if (lane < n_tok) ctx = min(lane_ctx, cap);
    const int r0 = gid, r1 = gid + 8;  // this thread's rows
    const uint32_t lim0 = __shfl_sync(0xffffffffu, ctx, r0 / group), lim1 = __shfl_sync(0xffffffffu, ctx, r1 / group);  // 0 behind the last row
    const uint32_t lim_min = __reduce_min_sync(0xffffffffu, lane < n_tok ? ctx : 0xffffffffu);
    ctx = __reduce_max_sync(0xffffffffu, ctx);
    const int walked = (int)((a.walk_len + OW_KEYS - 1) / OW_KEYS), chunks = walked + (int)((ctx + OW_KEYS - 1) / OW_KEYS);  // chunks of the prefix, of all keys

    T *const qs = reinterpret_cast<T *>(smem + ow_tiles(DEPTH) * ow_tile_bytes<DH>());  // [16][ROW], rows behind the last are zero
    for (int i = tid; i < 16 * CH; i += OW_THREADS) {
        const int r = i / CH, c = 8 * (i % CH);
        const bool valid = r < rows;
        ow_cp16(qs + r * ROW + c, reinterpret_cast<const T *>(a.q) + (valid ? (size_t)(t + r / group) * a.stq + (size_t)(hkv * group + r % group) * a.shq + c : 0), valid);
    }
    ow_commit();
    T *const k_tiles = reinterpret_cast<T *>(smem + (size_t)warp * 2 * DEPTH * ow_tile_bytes<DH>());  // [DEPTH] tiles of keys, then of values
    const int step = splits * OW_WARPS;
    // lane i: key i of a chunk.  The id of its page is loaded a step ahead of its use.
    auto page_of = [&](int chunk) {
        const bool shared = chunk < walked;
        const uint32_t key = (uint32_t)(shared ? chunk : chunk - walked) * OW_KEYS + (lane & 15);
        if (chunk >= chunks || key >= (shared ? a.walk_len : ctx)) return -1;
        return shared ? a.prefix_table[key >> a.page_shift] : a.table[(size_t)seq * a.table_stride + (key >> a.page_shift)];
    };
    auto request = [&](int chunk, int page, int tile) {  // its keys and values, zeros where there are none; which there are
        const uint32_t key = (uint32_t)(chunk < walked ? chunk : chunk - walked) * OW_KEYS + (lane & 15);
        const bool valid = page >= 0 && page < a.pages.n_pages;
        const long long at = valid ? (long long)page * a.pages.stride_page + (long long)(key & ((1u << a.page_shift) - 1)) * a.pages.stride_tok + (long long)hkv * a.pages.stride_head : 0;
        const unsigned some = __ballot_sync(0xffffffffu, valid);
        if (chunk < chunks) {
            T *const kd = k_tiles + tile * OW_KEYS * ROW + lane / CH * ROW + 8 * (lane % CH), *const vd = kd + DEPTH * OW_KEYS * ROW;
#pragma unroll
            for (int i = 0; i < OW_KEYS * CH / 32; ++i) {
                const int k = lane / CH + i * (32 / CH);
                const long long off = __shfl_sync(0xffffffffu, at, k) + 8 * (lane % CH);
                const bool is = some >> k & 1u;
                ow_cp16(kd + i * (32 / CH) * ROW, reinterpret_cast<const T *>(a.pages.k) + off, is);
                ow_cp16(vd + i * (32 / CH) * ROW, reinterpret_cast<const T *>(a.pages.v) + off, is);
            }
        }
        ow_commit();
        return some & 0xffffu;
    };
    float o[DH / 8][4];
#pragma unroll
    for (int i = 0; i < DH / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // Keys and values of DEPTH chunks in flight, and the page ids of the one behind them.
    const int c0 = split * OW_WARPS + warp;
    unsigned there[DEPTH];  // which keys of each there are
    {
        int page[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) page[i] = page_of(c0 + i * step);
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) there[i] = request(c0 + i * step, page[i], i);
    }
    int page_next = page_of(c0 + DEPTH * step);
    ow_wait<DEPTH>();
    __syncthreads();  // the queries are there
    int tile = 0;
    for (int c = c0; c < chunks; c += step) {
        const unsigned here = there[0];
        T *const ks = k_tiles + tile * OW_KEYS * ROW, *const vs = ks + DEPTH * OW_KEYS * ROW;
        ow_wait<DEPTH - 1>();
        const uint32_t first = (uint32_t)(c < walked ? 0 : c - walked) * OW_KEYS;  // of the token's own slots
        const uint32_t see0 = c < walked ? 0xffffffffu : lim0, see1 = c < walked ? 0xffffffffu : lim1;
        float s[2][4] = {}, s2[2][4] = {};  // two chains of products each
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
            uint32_t qa[4], b[4];
            ow_ldm4(qa, qs + (lane & 15) * ROW + 16 * k + (lane >> 4) * 8);
            ow_ldm4(b, ks + ((lane & 7) + (lane >> 4) * 8) * ROW + 16 * k + (lane >> 3 & 1) * 8);
            mma16816<T>(s[0], qa[0], qa[1], qa[2], qa[3], b[0], b[1]);
            mma16816<T>(s[1], qa[0], qa[1], qa[2], qa[3], b[2], b[3]);
            ow_ldm4(qa, qs + (lane & 15) * ROW + 16 * k + 16 + (lane >> 4) * 8);
            ow_ldm4(b, ks + ((lane & 7) + (lane >> 4) * 8) * ROW + 16 * k + 16 + (lane >> 3 & 1) * 8);
            mma16816<T>(s2[0], qa[0], qa[1], qa[2], qa[3], b[0], b[1]);
            mma16816<T>(s2[1], qa[0], qa[1], qa[2], qa[3], b[2], b[3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[h][e] += s2[h][e];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = 8 * h + 2 * t4 + e;
                const uint32_t key = first + i;
                const bool seen = here >> i & 1u;
                s[h][e] = seen && key < see0 ? s[h][e] * a.scale2 : -INFINITY;
                s[h][2 + e] = seen && key < see1 ? s[h][2 + e] * a.scale2 : -INFINITY;
            }
        const float n0 = fmaxf(m0, pf_reference<T>(ow_quad_max(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])))));
        const float n1 = fmaxf(m1, pf_reference<T>(ow_quad_max(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])))));
        const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
        const float f0 = m0 == -INFINITY ? 1.f : at_exp2(m0 - b0), f1 = m1 == -INFINITY ? 1.f : at_exp2(m1 - b1);  // (a row that has seen nothing has nothing to scale)
        m0 = n0;
        m1 = n1;
        uint32_t pa[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float x0 = at_exp2(s[h][0] - b0), x1 = at_exp2(s[h][1] - b0), y0 = at_exp2(s[h][2] - b1), y1 = at_exp2(s[h][3] - b1);
            l0 = (h ? l0 : l0 * f0) + (x0 + x1);
            l1 = (h ? l1 : l1 * f1) + (y0 + y1);
            pa[2 * h] = Act<T>::pack(x0, x1);
            pa[2 * h + 1] = Act<T>::pack(y0, y1);
        }
        if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
            for (int i = 0; i < DH / 8; ++i) {
                o[i][0] *= f0;
                o[i][1] *= f0;
                o[i][2] *= f1;
                o[i][3] *= f1;
            }
        }
        // Keys that one token of the group sees and another does not: a weight of zero times a value that is not finite would be NaN.
        bool odd = false;
        if (c >= walked && first + OW_KEYS > lim_min && lim_min < ctx)
            for (int i = lane; i < OW_KEYS * DH / 2; i += 32) {
                const float2 v = Act<T>::to_f2(*reinterpret_cast<const uint32_t *>(vs + i / (DH / 2) * ROW + i % (DH / 2) * 2));
                odd = odd || !(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY);
            }
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
            for (int i = 0; i < OW_KEYS; ++i) {
                const int from = (lane & ~3) | (i & 7) >> 1;  // the lane that has the weights of key i
                const float2 u0 = Act<T>::to_f2(__shfl_sync(0xffffffffu, i < 8 ? pa[0] : pa[2], from)), u1 = Act<T>::to_f2(__shfl_sync(0xffffffffu, i < 8 ? pa[1] : pa[3], from));
                const float x0 = i & 1 ? u0.y : u0.x, x1 = i & 1 ? u1.y : u1.x;
                const uint32_t key = first + i;
                const bool seen = here >> i & 1u;
#pragma unroll
                for (int d = 0; d < DH / 8; ++d) {
                    const float2 v = Act<T>::to_f2(*reinterpret_cast<const uint32_t *>(vs + i * ROW + 8 * d + 2 * t4));
                    if (seen && key < lim0) {
                        o[d][0] = fmaf(x0, v.x, o[d][0]);
                        o[d][1] = fmaf(x0, v.y, o[d][1]);
                    }
                    if (seen && key < lim1) {
                        o[d][2] = fmaf(x1, v.x, o[d][2]);
                        o[d][3] = fmaf(x1, v.y, o[d][3]);
                    }
                }
            }
        } else
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) {
            uint32_t b[4];
            ow_ldm4t(b, vs + (lane & 15) * ROW + 16 * i + (lane >> 4) * 8);
            mma16816<T>(o[2 * i], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
            mma16816<T>(o[2 * i + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
        }
        __syncwarp();  // this tile of keys and of values may be replaced
#pragma unroll
        for (int i = 0; i + 1 < DEPTH; ++i) there[i] = there[i + 1];
        there[DEPTH - 1] = request(c + DEPTH * step, page_next, tile);
        page_next = page_of(c + (DEPTH + 1) * step);
        if (++tile == DEPTH) tile = 0;
    }
    ow_wait<0>();
    l0 = ow_quad_sum(l0);
    l1 = ow_quad_sum(l1);
    __syncthreads();  // the tiles are done with: the warps' parts go there
    float *parts = reinterpret_cast<float *>(smem);  // [warp][16][DH]
    if (t4 == 0) {
        ml[warp][gid][0] = m0;
        ml[warp][gid][1] = l0;
        ml[warp][gid + 8][0] = m1;
        ml[warp][gid + 8][1] = l1;
    }
#pragma unroll
    for (int i = 0; i < DH / 8; ++i) {
        float *d = parts + ((size_t)warp * 16 + gid) * DH + 8 * i + 2 * t4;
        *reinterpret_cast<float2 *>(d) = make_float2(o[i][0], o[i][1]);
        *reinterpret_cast<float2 *>(d + 8 * DH) = make_float2(o[i][2], o[i][3]);
    }
    __syncthreads();
    // a warp per row from here on
    auto both = [&](int r) {  // the two warps' parts of a row
        OwPart<PD> p;
        p.clear();
#pragma unroll
        for (int w = 0; w < OW_WARPS; ++w) p.add(ml[w][r][0], ml[w][r][1], parts + ((size_t)w * 16 + r) * DH + lane * PD);
        return p;
    };
    if (cluster) {
        float *const cluster_o = reinterpret_cast<float *>(smem + ow_smem<DH>(DEPTH));  // in the first CTA: [split][16][DH], then (m, l) [split][16]
        float *const cluster_ml = cluster_o + (size_t)splits * 16 * DH;
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
#pragma unroll 1
        for (int r = warp; r < rows; r += OW_WARPS) {
            const OwPart<PD> p = both(r);
            uint32_t peer;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"((uint32_t)__cvta_generic_to_shared(cluster_o + ((size_t)split * 16 + r) * DH + lane * PD)), "r"(0));
#pragma unroll
            for (int i = 0; i < PD; ++i) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(peer + 4 * i), "f"(p.o[i]) : "memory");
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"((uint32_t)__cvta_generic_to_shared(cluster_ml + ((size_t)split * 16 + r) * 2)), "r"(0));
            if (lane == 0) asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer), "f"(p.m), "f"(p.l) : "memory");
            __syncwarp();
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (split != 0) return;
        grid_dep_wait();
#pragma unroll 1
        for (int r = warp; r < rows; r += OW_WARPS) {
            OwPart<PD> p;
            p.clear();
            for (int s = 0; s < splits; ++s) p.add(cluster_ml[(s * 16 + r) * 2], cluster_ml[(s * 16 + r) * 2 + 1], cluster_o + ((size_t)s * 16 + r) * DH + lane * PD);
            ow_finish<T, DH>(a, p, hkv, t * group + r, 0, lane);
        }
        return;
    }
    if (leave) {  // own_sum_kernel adds up
#pragma unroll 1
        for (int r = warp; r < rows; r += OW_WARPS) {
            const OwPart<PD> p = both(r);
            const size_t at = a.own_row + ((size_t)split * a.nkvh + hkv) * a.plan.rows + t * group + r;
            if (lane == 0) a.part_ml[at] = make_float2(p.m, p.l);
#pragma unroll
            for (int i = 0; i < PD; i += 2) *reinterpret_cast<float2 *>(a.part_o + at * DH + lane * PD + i) = make_float2(p.o[i], p.o[i + 1]);
        }
        if (first_block) grid_dep_wait();
        return;
    }
    grid_dep_wait();  // the parts of the prefix
#pragma unroll 1
    for (int r = warp; r < rows; r += OW_WARPS) {
        OwPart<PD> p = both(r);
        ow_finish<T, DH>(a, p, hkv, t * group + r, 0, lane);
    }
}

// Sum of a row's own part and the prefix's: a warp per row, behind own_kernel (which ends behind the prefix).  3 to 4 us, of which parts eight at a
// time are a round trip each.
template <class T, int DH>
__global__ void __launch_bounds__(256, 4) own_sum_kernel(const PrefixArgs a, int splits) {
    constexpr int PD = DH / 32;
    const int lane = threadIdx.x & 31, hkv = blockIdx.y, row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= a.plan.rows) return;
    const int seq = a.tok_seq[row / (a.nh / a.nkvh)];
    grid_dep_wait();  // (rows of padding too: the call ends behind its kernels, which still write to the workspace)
    if (seq < 0 || seq >= a.n_seq) return;
    OwPart<PD> p;
    p.clear();
    ow_finish<T, DH>(a, p, hkv, row, splits, lane);
}

// ------------------------------------------------------------------ host side

static int pf_map(CUtensorMap *m, int dt, const void *base, const lcu_kv_pages &p, int dh, int nkvh) {
    const cuuint64_t dims[4] = {(cuuint64_t)dh, (cuuint64_t)p.page_tokens, (cuuint64_t)nkvh, (cuuint64_t)p.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.stride_tok * 2, (cuuint64_t)p.stride_head * 2, (cuuint64_t)p.stride_page * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.page_tokens, 1, 1}, es[4] = {1, 1, 1, 1};
    LCU_REQUIRE(tc_encode_fn(), "attention_prefix: no cuTensorMapEncodeTiled");
    const CUresult r = tc_encode_fn()(m, dt == LCU_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base), dims, strides,
                                      box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LCU_REQUIRE(r == CUDA_SUCCESS, "attention_prefix: cuTensorMapEncodeTiled failed with %d", (int)r);
    return LCU_OK;
}

template <class T, int DH, int DEPTH>
static int own_run(const PrefixArgs &a, int splits, bool cluster, cudaStream_t s) {
    static OncePerDevice once;
    const int set = once.run([]() -> int {
        LCU_CHECK_CUDA(cudaFuncSetAttribute(own_kernel<T, DH, DEPTH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(ow_smem<DH>(DEPTH) + 8 * ow_part_bytes<DH>())));
        return LCU_OK;
    });
    if (set) return set;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.nkvh, a.n);
    cfg.blockDim = dim3(OW_THREADS);
    cfg.dynamicSmemBytes = ow_smem<DH>(DEPTH) + (cluster ? splits * ow_part_bytes<DH>() : 0);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n_attr = 0;
    if (cluster) {
        attr[n_attr].id = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = splits;
        attr[n_attr].val.clusterDim.y = attr[n_attr].val.clusterDim.z = 1;
        ++n_attr;
    }
    if (a.prefix_len) {
        attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
        ++n_attr;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n_attr;
    LCU_CHECK_CUDA(cudaLaunchKernelEx(&cfg, own_kernel<T, DH, DEPTH>, a, 16 / (a.nh / a.nkvh), splits));
    return LCU_OK;
}

template <class T, int DH>
static int prefix_run(const PrefixArgs &a, int dt, cudaStream_t s) {
    if (a.prefix_len) {
        static OncePerDevice once;
        const int set = once.run([]() -> int {
            LCU_CHECK_CUDA(cudaFuncSetAttribute(prefix_tc_kernel<T, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pf_smem<DH>()));
            return LCU_OK;
        });
        if (set) return set;
        CUtensorMap mk, mv;
        int rc = pf_map(&mk, dt, a.pages.k, a.pages, DH, a.nkvh);
        if (!rc) rc = pf_map(&mv, dt, a.pages.v, a.pages, DH, a.nkvh);
        if (rc) return rc;
        LCU_CHECK_CUDA(launch_kernel(prefix_tc_kernel<T, DH>, dim3(a.plan.ctas), dim3(PF_THREADS), pf_smem<DH>(), s, false, a, mk, mv, dt == LCU_BF16 ? 1u : 0u));
    }
    // keys of long contexts: over a cluster where blocks are few, over blocks that leave a part each where there are more
    const long long cap = a.walk_len + ((long long)a.table_stride << a.page_shift), blocks = (long long)a.nkvh * a.n;
    const bool leave = a.prefix_len && a.plan.own_parts;
    int splits;
    if (leave) splits = (int)(cap < 64LL * a.plan.own_parts ? (cap + 63) / 64 > 0 ? (cap + 63) / 64 : 1 : a.plan.own_parts);
    else splits = own_splits(blocks, cap, sm_count());
    const bool cluster = splits > 1 && !leave;
    const int rc = blocks * splits <= 5LL * sm_count() ? own_run<T, DH, 2>(a, splits, cluster, s) : own_run<T, DH, 1>(a, splits, cluster, s);
    if (rc) return rc;
    if (leave) LCU_CHECK_CUDA(launch_kernel(own_sum_kernel<T, DH>, dim3((a.plan.rows + 7) / 8, a.nkvh), dim3(256), 0, s, true, a, splits));
    return LCU_OK;
}

}  // namespace lcu

using namespace lcu;

extern "C" size_t lcu_attention_prefix_workspace_size(int n, int nh, int nkvh, int dh, uint32_t prefix_len) {
    if (n <= 0 || n > 65535 || nkvh <= 0 || nkvh > 65535 || nh < nkvh || nh % nkvh || nh / nkvh > 16 || dh <= 0 || !prefix_len || !prefix_fits(n, nh / nkvh, nkvh, prefix_len)) return 0;  // (the call refuses these)
    return prefix_bytes(n, nh / nkvh, nkvh, prefix_len, sm_count(), dh);
}

extern "C" int lcu_op_attention_prefix(void *o, int sto, int sho, const void *q, int stq, int shq, const lcu_kv_pages *pages, const int32_t *prefix_table,
                                       uint32_t prefix_len, const int32_t *table, int table_stride, int n_seq, const int32_t *tok_seq,
                                       const uint32_t *tok_ctx, int n, int nh, int nkvh, int dh, float scale, int dt, void *workspace,
                                       size_t workspace_len, lcu_stream_t s) {
    PrefixArgs a{};
    int rc = kv_pages_take(&a.pages, pages, nkvh, "attention_prefix");
    if (rc) return rc;
    LCU_REQUIRE(dt == LCU_F16 || dt == LCU_BF16, "attention_prefix: dtype %d unsupported", dt);
    LCU_REQUIRE(dh == 64 || dh == 128, "attention_prefix: dh = %d unsupported (64, 128)", dh);
    LCU_REQUIRE(n >= 0 && n <= 65535 && nkvh >= 1 && nkvh <= 65535 && nh >= nkvh && nh % nkvh == 0 && nh / nkvh <= 16,
                "attention_prefix: %d tokens, %d query heads over %d", n, nh, nkvh);
    const float scale2 = scale * 1.4426950408889634f;  // finite too: a score of 0 stays one
    LCU_REQUIRE(scale > 0.f && scale2 < INFINITY, "attention_prefix: scale %g", (double)scale);
    LCU_REQUIRE(prefix_len <= 0x7fffffffu && table_stride >= 0 && (long long)table_stride * pages->page_tokens <= 0x7fffffffll && n_seq >= 1,
                "attention_prefix: prefix of %u, %d sequences of %d pages", prefix_len, n_seq, table_stride);
    if (n == 0) return LCU_OK;
    LCU_REQUIRE(!prefix_len || prefix_fits(n, nh / nkvh, nkvh, prefix_len), "attention_prefix: prefix of %u for %d tokens of %d heads: more than a call takes", prefix_len, n, nh);
    LCU_REQUIRE(o && q && tok_seq && tok_ctx && (prefix_table || !prefix_len) && (table || !table_stride), "attention_prefix: null argument");
    LCU_REQUIRE((((uintptr_t)o | (uintptr_t)q | (uintptr_t)pages->k | (uintptr_t)pages->v) % 16) == 0 && (sto | sho | stq | shq) % 8 == 0 &&
                    pages->stride_page % 8 == 0 && pages->stride_tok % 8 == 0 && a.pages.stride_head % 8 == 0,
                "attention_prefix: rows of q, o and the pages start on 16 bytes");
    const size_t need = lcu_attention_prefix_workspace_size(n, nh, nkvh, dh, prefix_len);
    LCU_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_len >= need), "attention_prefix: workspace of %zu bytes, %zu needed (256-byte aligned)",
                workspace_len, need);
    a.o = o; a.sto = sto; a.sho = sho; a.q = q; a.stq = stq; a.shq = shq;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.table = table; a.table_stride = table_stride; a.n_seq = n_seq; a.tok_seq = tok_seq; a.tok_ctx = tok_ctx;
    while ((1 << a.page_shift) < pages->page_tokens) ++a.page_shift;
    a.n = n; a.nh = nh; a.nkvh = nkvh; a.scale2 = scale2;
    if (prefix_len && prefix_walk(n, nh / nkvh, nkvh, prefix_len, (long long)table_stride * pages->page_tokens, sm_count(), dh)) {
        a.walk_len = prefix_len;
        a.prefix_len = 0;
    } else if (prefix_len) {
        a.plan = prefix_plan(n, nh / nkvh, nkvh, prefix_len, sm_count(), dh, (long long)(n_seq < n ? n_seq : n) * table_stride * pages->page_tokens, n_seq);
        a.part_ml = reinterpret_cast<float2 *>(workspace);
        a.part_o = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(workspace) + prefix_ml_bytes(a.plan, nkvh));
        a.own_row = prefix_own_row(a.plan);
    }
    if (dt == LCU_F16) return dh == 64 ? prefix_run<__half, 64>(a, dt, as_stream(s)) : prefix_run<__half, 128>(a, dt, as_stream(s));
    return dh == 64 ? prefix_run<__nv_bfloat16, 64>(a, dt, as_stream(s)) : prefix_run<__nv_bfloat16, 128>(a, dt, as_stream(s));
}
