"""Attention of a batch that shares a prefix, on a caller's pages (needs a B200)."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import serve_ref as R
from serve_ref import DEV, DT, HALF

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences of (own slots, new tokens) behind a prefix; tokens in the order given, padding at `pad` places behind them."""

    def __init__(self, seed, seqs, prefix, nh, nkvh, dh, dt, page, pad=0, layout="own", capacity=None, std=1.0, pages=None):
        r = np.random.default_rng(seed)
        self.dims = nh, nkvh, dh, dt, page
        self.prefix = prefix
        self.per = capacity if capacity is not None else max([-(-s // page) for s, _ in seqs], default=0)
        self.n_seq = max(len(seqs), 1)
        shared = -(-prefix // page)
        need = shared + self.n_seq * self.per
        self.n_pages = pages or need + 2
        ids = r.permutation(self.n_pages)[:need]
        self.prefix_ids, self.ids = ids[:shared].astype(np.int32), ids[shared:].reshape(self.n_seq, self.per).astype(np.int32)
        shape = (self.n_pages, 2, nkvh, page, dh) if layout == "own" else (2, self.n_pages, page, nkvh, dh)
        self.pool = R.rng_normal(seed, shape, dt, std)
        self.layout = layout
        self.tok_seq = np.concatenate([np.repeat(np.arange(len(seqs)), [m for _, m in seqs]), np.full(pad, -1)]).astype(np.int32)
        self.ctx = np.concatenate([np.arange(s - m + 1, s + 1) for s, m in seqs] + [np.full(pad, 3)]).astype(np.int64)
        self.n = len(self.tok_seq)
        self.q = R.rng_normal(seed + 1, (self.n, nh, dh), dt, 1.5)
        self.scale = dh ** -0.5
        self.o = torch.full((self.n, nh, dh), 7.0, dtype=DT[dt], device=DEV)

    def pages_args(self):
        p, page = self.pool, self.dims[4]
        if self.layout == "own":
            return p.data_ptr(), p[:, 1].data_ptr(), p.stride(0), p.stride(3), p.stride(2), self.n_pages, page
        return p[0].data_ptr(), p[1].data_ptr(), p.stride(1), p.stride(2), p.stride(3), self.n_pages, page

    def run(self, L, workspace=None):
        nh, nkvh, dh, dt, page = self.dims
        lib = L.load_library()
        self.dev = [R.i32(self.prefix_ids), R.i32(self.ids), R.i32(self.tok_seq), R.i32(self.ctx.astype(np.uint32).view(np.int32))]
        need = lib.lcu_attention_prefix_workspace_size(self.n, nh, nkvh, dh, self.prefix)
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV) if workspace is None else workspace  # NaN all over
        L.check(lib.lcu_op_attention_prefix(self.o.data_ptr(), self.o.stride(0), self.o.stride(1), self.q.data_ptr(), self.q.stride(0), self.q.stride(1),
                                            L.KvPages(*self.pages_args()), self.dev[0].data_ptr(), self.prefix, self.dev[1].data_ptr() if self.per else None, self.per,
                                            self.n_seq, self.dev[2].data_ptr(), self.dev[3].data_ptr(), self.n, nh, nkvh, dh, self.scale, dt, ws.data_ptr(), ws.numel(),
                                            R.stream()))
        self.ws = ws
        return self.o

    def rows(self, ids, count):
        """Keys and values [positions, nkvh, dh] of the first `count` slots; those on pages that are none are left out."""
        page = self.dims[4]
        pos = np.arange(min(count, len(ids) * page))
        at = np.asarray(ids, dtype=np.int64)[pos // page] if len(pos) else pos
        pos, at = pos[(at >= 0) & (at < self.n_pages)], at[(at >= 0) & (at < self.n_pages)]
        at, slot = torch.as_tensor(at, device=DEV), torch.as_tensor(pos % page, device=DEV)
        if self.layout == "own":
            return self.pool[at, 0, :, slot], self.pool[at, 1, :, slot]
        return self.pool[0, at, slot], self.pool[1, at, slot]

    def check(self):
        """Against 64 bits.  Scores: products exact, 32-bit sums of dh <= 128 terms (chains of at most 128 roundings of 2^-24, truncation counted
        double, on sum |q k| scale <= `mag`), so weights are off by 2^-16 mag + 2^-19 (exponentials, sums, merges) relatively, each weight is
        rounded to the type (half a step), and so is the result."""
        nh, nkvh, dh, dt, _ = self.dims
        shared = self.rows(self.prefix_ids, self.prefix)
        for t in range(self.n):
            if not 0 <= self.tok_seq[t] < self.n_seq:
                assert (self.o[t] == 7).all(), f"token {t} is none"
                continue
            own = self.rows(self.ids[self.tok_seq[t]], int(self.ctx[t]))
            want, mag = R.attention(self.q[t], *shared, *own, self.scale)
            keys = torch.cat([shared[0], own[0]]).double().abs()
            g = nh // nkvh
            most = torch.einsum("hgd,phd->hgp", self.q[t].double().abs().view(nkvh, g, dh), keys).amax().item() * self.scale if keys.numel() else 0.0
            tol = HALF[dt] * want.abs() + 2 * (HALF[dt] + 2.0 ** -16 * most + 2.0 ** -19) * mag + 2.0 ** -24
            off = (self.o[t].double() - want).abs()
            assert not self.o[t].isnan().any() and (off <= tol).all(), f"token {t}: {float(off.max())} off, {float((off / tol).max())} of what is allowed"


@pytest.mark.parametrize("dt", [0, 1])
@pytest.mark.parametrize("nh,nkvh,dh,page,prefix,seqs,pad", [
    (32, 8, 128, 64, 100, [(1, 1)], 0),                                  # one token behind a short prefix
    (32, 8, 64, 16, 1, [(5, 1), (70, 1), (1, 1)], 2),                    # a prefix of one, padding
    (4, 4, 64, 8, 0, [(33, 1), (0, 0), (129, 4)], 0),                    # no prefix, a sequence without tokens
    (12, 4, 128, 32, 127, [(9, 3), (65, 5), (2, 2), (64, 1)], 1),        # three heads a group, drafted tokens
    (20, 4, 64, 128, 128, [(200, 1), (128, 2), (1, 1)], 0),              # pages of a whole tile
    (16, 1, 128, 16, 129, [(17, 7), (300, 1)], 3),                       # sixteen heads a group
    (7, 7, 64, 64, 515, [(10, 1)] * 30, 0),
    (64, 8, 128, 64, 1000, [(i % 90 + 1, 1) for i in range(70)], 5),     # several tiles of query rows
    (8, 1, 128, 32, 4100, [(40, 8), (600, 2)], 0),                       # one KV head: the prefix in many splits
    (32, 8, 128, 64, 2000, [(30, 1), (1500, 1), (700, 3), (4, 4)], 0),   # long contexts of their own
])
def test_batches(L, dt, nh, nkvh, dh, page, prefix, seqs, pad):
    b = Batch(nh + prefix, seqs, prefix, nh, nkvh, dh, dt, page, pad)
    b.run(L)
    b.check()


@pytest.mark.parametrize("prefix", [2, 63, 64, 65, 255, 256, 257, 384, 1023, 9001])
def test_lengths_of_the_prefix(L, prefix):
    b = Batch(prefix, [(3, 1), (20, 2)], prefix, 8, 2, 64, 1, 16)
    b.run(L)
    b.check()


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("prefix", [0, 70])
def test_lengths_of_own_contexts(L, dh, prefix):
    b = Batch(dh, [(s, 1) for s in (1, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 400)], prefix, 6, 2, dh, 0, 8)
    b.run(L)
    b.check()


def test_nothing_to_see_and_pages_of_others(L):
    """A token without any key gets zeros; what lies behind a context, in the rest of its page, on pages of others, may be anything."""
    for prefix in (0, 37):
        b = Batch(prefix + 3, [(5, 1), (40, 2), (17, 1)], prefix, 8, 2, 128, 1, 16, capacity=5)
        b.ctx[0] = 0
        seen = torch.zeros(b.pool.shape, dtype=torch.bool, device=DEV)
        for ids, count in [(b.prefix_ids, prefix), (b.ids[1], 40), (b.ids[2], 17)]:
            for p in range(count):
                seen[int(ids[p // 16]), :, :, p % 16] = True
        filth = torch.where(torch.rand(b.pool.shape, device=DEV) < 0.5, torch.nan, torch.inf).to(b.pool.dtype)
        b.pool = torch.where(seen, b.pool, filth)
        b.run(L)
        b.check()
        if not prefix:
            assert (b.o[0] == 0).all()


def test_no_pages_of_their_own(L):
    b = Batch(4, [(0, 0), (0, 0)], 300, 8, 2, 64, 0, 32, capacity=0)
    b.tok_seq, b.ctx, b.n = np.array([0, 1, 1, 0], np.int32), np.array([0, 5, 0, 9], np.int64), 4
    b.q, b.o = R.rng_normal(5, (4, 8, 64), 0), torch.full((4, 8, 64), 7.0, dtype=DT[0], device=DEV)
    b.run(L)
    b.check()


@pytest.mark.parametrize("page", [8, 64, 128])
def test_page_ids_that_name_no_page(L, page):
    """In the prefix, at its end, and in own tables: their positions are not seen; a prefix of nothing else is none; contexts end with the table."""
    b = Batch(page, [(page * 3 + 1, 1), (page * 4, 2), (page, 1)], page * 20 + 3, 8, 2, 128, 0, page, capacity=4)
    b.prefix_ids[[0, 7, 20]] = -1, b.n_pages, 2 ** 31 - 1
    b.ids[0, 1], b.ids[1, 3], b.ids[2, 0] = -5, b.n_pages + 7, -2 ** 31
    b.ctx[1], b.ctx[2] = 2 ** 32 - 1, page * 4 + 1
    b.run(L)
    b.check()
    b.prefix_ids[:] = -1
    b.o[:] = 7
    b.run(L)
    b.check()
    assert (b.o[3] == 0).all()


@pytest.mark.parametrize("layout", ["own", "token"])
def test_strides(L, layout):
    """Queries cut out of a fused projection's rows, outputs into wider rows, the cache by tokens instead of heads."""
    b = Batch(8, [(50, 1), (9, 4), (77, 1)], 333, 12, 4, 64, 1, 16, 2, layout)
    qkv = R.rng_normal(9, (b.n, 20 * 64 + 8), 1, 1.5)
    b.q = qkv[:, 8:8 + 12 * 64].unflatten(1, (12, 64))
    wide = torch.full((b.n, 12 * 72), 7.0, dtype=DT[1], device=DEV)
    b.o = wide.unflatten(1, (12, 72))[..., :64]
    b.run(L)
    b.check()
    assert (wide.unflatten(1, (12, 72))[..., 64:] == 7).all()


def test_pages_behind_32_bits(L):
    b = Batch(11, [(20, 1), (3, 1)], 200, 8, 8, 128, 1, 64, pages=2 ** 32 // (2 * 8 * 64 * 128) + 9, std=0.0)
    fresh = R.rng_normal(12, (4, 2, 8, 64, 128), 1)
    b.prefix_ids = np.array([b.n_pages - 1, 0, 5, b.n_pages - 2], np.int32)
    for i, p in enumerate(b.prefix_ids):
        b.pool[int(p)] = fresh[i]
    b.run(L)
    b.check()


def test_scores_far_apart(L):
    """One key carries all weight, from tile to tile another; scores of hundreds; a scale that is not 1 / sqrt(dh)."""
    b = Batch(13, [(90, 1), (5, 2)], 700, 8, 2, 64, 0, 16, std=3.0)
    b.scale = 1.0
    b.run(L)
    b.check()


def test_values_that_are_not_finite_stay_with_their_rows(L):
    """NaN in one token's query, in one KV head of one sequence: nobody else's rows change."""
    a, b = (Batch(14, [(20, 1), (33, 1), (8, 1)], 150, 8, 2, 64, 1, 16) for _ in range(2))
    b.q[0] = torch.nan
    b.pool[int(b.ids[1, 0]), 1, 1, 3] = torch.nan
    a.run(L)
    b.run(L)
    assert b.o[0].isnan().all() and b.o[1, 4:].isnan().all()
    assert torch.equal(a.o[1, :4], b.o[1, :4]) and torch.equal(a.o[2], b.o[2])


@pytest.mark.parametrize("filth", [math.nan, math.inf])
def test_values_that_only_later_drafts_see(L, filth):
    """Drafted tokens share their keys' tiles: what the last one alone sees is not finite, and the others' rows stay as they were."""
    a, b = (Batch(17, [(20, 4), (16, 3), (49, 2)], 40, 8, 2, 128, 0, 16) for _ in range(2))
    for seq, slot in ((0, 19), (1, 15), (2, 48)):
        b.pool[int(b.ids[seq, slot // 16]), 1, :, slot % 16] = filth
    a.run(L)
    b.run(L)
    last = [3, 6, 8]
    others = [t for t in range(9) if t not in last]
    assert not b.o[last].isfinite().any()
    for t in others:
        assert (a.o[t].double() - b.o[t].double()).abs().max() <= 2.0 ** -10 * a.o[t].abs().max().item()  # (sums in another order)
    b.pool = a.pool
    b.o = b.o[others].clone()
    b.tok_seq, b.ctx, b.q, b.n = b.tok_seq[others], b.ctx[others], b.q[others], len(others)
    b.check()


def test_the_same_answer_twice_and_on_another_stream(L):
    """No atomics: the same bits in every run; two calls at once with workspaces of their own."""
    b = [Batch(15 + i, [(100, 2)] * 9, 3000, 32, 8, 128, 0, 64) for i in range(2)]
    want = []
    for x in b:
        want.append(x.run(L).clone())
        x.check()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in b]
    for _ in range(10):
        for x, s in zip(b, streams):
            with torch.cuda.stream(s):
                x.o.zero_()
                x.run(L, x.ws)
    torch.cuda.synchronize()
    for x, w in zip(b, want):
        assert torch.equal(x.o, w)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("nh,tokens", [(8, 1), (8, 40), (32, 33), (32, 40), (32, 100)])
def test_slow_memory(L, dh, nh, tokens):
    """Caches flushed ahead of each run, so that tiles of keys come late and out of step with the products: the same bits in every run.  Row tiles
    of both kinds, prefixes that end inside a tile, several pieces of work per CTA."""
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=DEV)
    for prefix in (8001, 30011):
        b = Batch(prefix + tokens, [(7, 1)] * tokens, prefix, nh, 8, dh, 1, 32)
        first = b.run(L).clone()
        b.check() if tokens <= 33 else None
        for _ in range(8):
            flush.zero_()
            b.o.zero_()
            b.run(L, torch.full_like(b.ws, 255))
            assert torch.equal(b.o, first)


def test_matches_a_contexts_own_cache(L):
    """The pages that rounds of lcu_step filled, read through lcu_kv_layer_pages and lcu_seq_pages."""
    from dataclasses import replace
    cfg = replace(L.CONFIGS["tiny"], act_dtype=L.BF16, nctx=512)
    ctx = L.load_model(cfg, L.synth_weights_torch(cfg, 0, DEV), kv_bytes=1 << 24)
    seqs = [ctx.seq_create() for _ in range(3)]
    lens = [77, 5, 130]
    for s, n in zip(seqs, lens):
        out = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
        ctx.seq_resize(s, n)
        ctx.step([(s, 0, n)], np.arange(n, dtype=np.uint32) + 3, out)
    torch.cuda.synchronize()
    page, layer = ctx.page_tokens, 1
    pages = ctx.layer_pages(layer)
    ids = [ctx.seq_pages(s) for s in seqs]
    assert [len(i) for i in ids] == [-(-n // page) for n in lens] and pages.n_pages == ctx.pages_total and pages.page_tokens == page
    # the third sequence's cache as the prefix of tokens of the other two
    b = Batch(16, [(77, 1), (5, 1)], 130, cfg.nh, cfg.nkvh, cfg.dh, L.BF16, page)
    b.n_pages, b.prefix_ids = pages.n_pages, ids[2]
    b.ids = np.full((2, b.per), -1, np.int32)
    for i in (0, 1):
        b.ids[i, :len(ids[i])] = ids[i]
    shape = (pages.n_pages, cfg.n_layers, 2, cfg.nkvh, page, cfg.dh)
    raw = L._view(pages.k - layer * 2 * pages.stride_head * cfg.nkvh * 2, int(np.prod(shape)), L.BF16, 0).view(shape)
    b.pool = raw[:, layer]
    assert b.pool.data_ptr() == pages.k and b.pool[:, 1].data_ptr() == pages.v and b.pool.stride(0) == pages.stride_page
    b.run(L)
    b.check()
    with pytest.raises(L.LcuError):
        ctx.layer_pages(cfg.n_layers)
    with pytest.raises(L.LcuError):
        ctx.seq_pages(99)


def speculative_round(L, state):
    """append -> attention -> head -> probabilities -> verification, as a host would chain them."""
    lib, s = L.load_library(), R.stream()
    nh, nkvh, dh, dt, n, vocab = (state[x] for x in ("nh", "nkvh", "dh", "dt", "n", "vocab"))
    qkv, st = state["qkv"], state["qkv"].stride(0)
    q, k, v = (qkv[:, i * dh:].data_ptr() for i in (0, nh, nh + nkvh))
    L.check(lib.lcu_op_kv_append(state["pages"], state["table"].data_ptr(), state["per"], state["seqs"], state["tok_seq"].data_ptr(), state["slot"].data_ptr(), k, st, dh, v, st,
                                 dh, state["q"].data_ptr(), nh * dh, dh, q, st, dh, state["pos"].data_ptr(), state["prep"], n, nh, nkvh, dh, dt, s))
    L.check(lib.lcu_op_attention_prefix(state["o"].data_ptr(), nh * dh, dh, state["q"].data_ptr(), nh * dh, dh, state["pages"], state["prefix_table"].data_ptr(), state["prefix"],
                                        state["table"].data_ptr(), state["per"], state["seqs"], state["tok_seq"].data_ptr(), state["ctx"].data_ptr(), n, nh, nkvh, dh,
                                        dh ** -0.5, dt, state["ws"].data_ptr(), state["ws"].numel(), s))
    L.check(lib.lcu_op_linear(state["logits"].data_ptr(), vocab, state["o"].data_ptr(), nh * dh, state["head"].data_ptr(), dt, None, 0, n, nh * dh, vocab, dt, s))
    L.check(lib.lcu_op_softmax_rows(state["probs"].data_ptr(), vocab, state["logits"].data_ptr(), vocab, state["t"].data_ptr(), n, vocab, dt, s))
    L.check(lib.lcu_op_verify_drafts(state["accepted"].data_ptr(), state["tokens"].data_ptr(), state["probs"].data_ptr(), vocab, None, 0, state["drafted"].data_ptr(), None,
                                     state["u"].data_ptr(), state["seqs"], state["k"], vocab, L.F32, s))


def test_a_speculative_round_eager_and_captured(L):
    """All operators in a row, then the same captured and replayed with other inputs, slots and contexts."""
    nh, nkvh, dh, dt, page, seqs, k, prefix, vocab, per = 8, 2, 64, 1, 16, 5, 3, 210, 1000, 6
    n, r = seqs * (k + 1), np.random.default_rng(1)
    ids = r.permutation(14 + seqs * per).astype(np.int32)
    pool = R.rng_normal(1, (len(ids), 2, nkvh, page, dh), dt)
    lib = L.load_library()
    sin, cos = R.tables(prefix + per * page, dh)
    w = R.rng_normal(2, (dh,), dt)
    S = dict(nh=nh, nkvh=nkvh, dh=dh, dt=dt, n=n, vocab=vocab, seqs=seqs, k=k, prefix=prefix, per=per, sin=sin, cos=cos, w=w,
             prep=L.QkPrep(w.data_ptr(), w.data_ptr(), sin.data_ptr(), cos.data_ptr(), dt, 1e-6, sin.shape[0], dh, 1),
             pages=L.KvPages(pool.data_ptr(), pool[:, 1].data_ptr(), pool.stride(0), pool.stride(3), pool.stride(2), len(ids), page),
             prefix_table=R.i32(ids[:14]), table=R.i32(ids[14:].reshape(seqs, per)), tok_seq=R.i32(np.repeat(np.arange(seqs), k + 1)),
             q=torch.zeros(n, nh, dh, dtype=DT[dt], device=DEV), o=torch.zeros(n, nh, dh, dtype=DT[dt], device=DEV), head=R.rng_normal(3, (vocab, nh * dh), dt, 0.2),
             logits=torch.zeros(n, vocab, dtype=DT[dt], device=DEV), probs=torch.zeros(n, vocab, device=DEV), t=torch.full((n,), 0.9, device=DEV),
             accepted=torch.zeros(seqs, dtype=torch.int32, device=DEV), tokens=torch.zeros(seqs, k + 1, dtype=torch.int32, device=DEV),
             ws=torch.empty(lib.lcu_attention_prefix_workspace_size(n, nh, nkvh, dh, prefix), dtype=torch.uint8, device=DEV),
             qkv=torch.zeros(n, (nh + 2 * nkvh) * dh, dtype=DT[dt], device=DEV), slot=torch.zeros(n, dtype=torch.int32, device=DEV), pos=torch.zeros(n, dtype=torch.int32, device=DEV),
             ctx=torch.zeros(n, dtype=torch.int32, device=DEV), drafted=torch.zeros(seqs, k, dtype=torch.int32, device=DEV), u=torch.zeros(seqs, k + 1, device=DEV))

    def fill(seed):
        past = np.random.default_rng(seed).integers(0, per * page - k, seqs)
        slot = (past[:, None] + np.arange(k + 1)).reshape(-1)
        S["slot"].copy_(R.i32(slot)), S["pos"].copy_(R.i32(slot + prefix)), S["ctx"].copy_(R.i32(slot + 1))
        S["qkv"].copy_(R.rng_normal(seed, S["qkv"].shape, dt))
        S["u"].copy_(torch.as_tensor(np.random.default_rng(seed).random((seqs, k + 1), dtype=np.float32)))

    def check(before):
        """Every step against 64 bits, from what the step before it left."""
        x = S["qkv"].unflatten(1, (nh + 2 * nkvh, dh))
        at = S["table"][S["tok_seq"].long(), (S["slot"] // page).long()].long(), (S["slot"] % page).long()
        turned, mag = R.turn(x[:, :nh + nkvh], w, 1e-6, S["pos"], sin, cos, dh, True)
        got = torch.cat([S["q"], pool[at[0], 0, :, at[1]]], 1)
        assert ((got.double() - turned).abs() <= HALF[dt] * turned.abs() + 16 * 2.0 ** -24 * mag).all()
        assert torch.equal(pool[at[0], 1, :, at[1]], x[:, nh + nkvh:])
        before[at[0], :, :, at[1]] = pool[at[0], :, :, at[1]]
        assert torch.equal(pool, before)  # nothing else moved
        b = Batch(1, [(1, 1)] * seqs, prefix, nh, nkvh, dh, dt, page)
        b.pool, b.n_pages, b.prefix_ids, b.ids, b.n = pool, len(ids), ids[:14], ids[14:].reshape(seqs, per), n
        b.tok_seq, b.ctx, b.q, b.o = S["tok_seq"].cpu().numpy(), S["ctx"].cpu().numpy(), S["q"], S["o"]
        b.check()
        lg = S["o"].view(n, -1).double() @ S["head"].double().T
        assert ((S["logits"].double() - lg).abs() <= HALF[dt] * lg.abs() + 512 * 2.0 ** -24 * (S["o"].view(n, -1).double().abs() @ S["head"].double().abs().T)).all()
        p = R.softmax_rows(S["logits"], S["t"])
        assert (S["probs"].double() - p).abs().max() < 2.0 ** -17
        want = R.verify(S["probs"].view(seqs, k + 1, vocab).cpu().numpy(), None, S["drafted"].cpu().numpy(), None, S["u"].cpu().numpy())
        assert np.array_equal(S["accepted"].cpu().numpy(), want[0]) and np.array_equal(S["tokens"].cpu().numpy(), want[1])

    fill(1)
    before = pool.clone()
    speculative_round(L, S)
    # drafts that the target likes: its own largest tokens
    S["drafted"].copy_(S["probs"].view(seqs, k + 1, vocab)[:, :k].argmax(-1).int())
    speculative_round(L, S)
    check(before)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        speculative_round(L, S)
    for seed in (2, 3):
        fill(seed)
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        check(before)
    assert math.isfinite(float(S["probs"].sum()))


@pytest.mark.parametrize("tokens", [2, 40])
def test_a_call_of_padding_alone_ends_behind_its_kernels(L, tokens):
    """What is queued behind the call finds the workspace at rest."""
    b = Batch(77, [], 9000, 32, 8, 128, 0, 64, pad=tokens)
    b.run(L)
    b.ws.zero_()
    torch.cuda.synchronize()
    assert (b.o == 7).all() and (b.ws == 0).all()


# Behind thousands of tokens (padding but for a few) the prefix is on the tensor cores however short it is; behind a few, the blocks of the own slots read it.
@pytest.mark.parametrize("dt,dh", [(0, 128), (1, 64)])
@pytest.mark.parametrize("prefix,pad", [(8, 30000), (9, 30000), (63, 1500), (64, 1500), (65, 1500), (127, 1000), (129, 1000), (255, 500), (257, 500)])
def test_short_prefixes_of_many_tokens(L, dt, dh, prefix, pad):
    b = Batch(prefix + dh, [(3, 1), (40, 2), (0 + 1, 1)], prefix, 32, 8, dh, dt, 16, pad=pad, std=2.0)
    few = Batch(prefix + dh, [(3, 1), (40, 2), (0 + 1, 1)], prefix, 32, 8, dh, dt, 16, pad=2, std=2.0)
    few.q, few.pool, few.prefix_ids, few.ids = b.q[:few.n].clone(), b.pool, b.prefix_ids, b.ids
    b.run(L)
    few.run(L)
    few.check()
    assert (b.o[4:] == 7).all()
    b.n, b.tok_seq, b.ctx = 4, b.tok_seq[:4], b.ctx[:4]
    b.check()


@pytest.mark.parametrize("page", [8, 16, 64, 128])
@pytest.mark.parametrize("pad", [0, 900])
def test_prefix_pages_that_name_no_page(L, page, pad):
    """Few tokens and many: the slots of such pages are not seen, whoever reads the prefix."""
    b = Batch(page, [(20, 1), (page + 3, 3)], 300, 32, 8, 128, 1, page, pad=pad)
    b.prefix_ids[1], b.prefix_ids[-1] = -1, b.n_pages
    if len(b.prefix_ids) > 4:
        b.prefix_ids[3] = 2 ** 31 - 1
    b.ids[1, 0] = -7
    b.run(L)
    b.n, b.tok_seq, b.ctx = 4, b.tok_seq[:4], b.ctx[:4]
    b.check()


@pytest.mark.parametrize("pad", [0, 900])
@pytest.mark.parametrize("filth", [math.nan, math.inf])
def test_filth_behind_a_prefix_and_behind_contexts(L, pad, filth):
    """Slots that nobody sees: of the prefix's last page, of the sequences', of pages of others."""
    b = Batch(31, [(5, 1), (37, 3), (1, 1)], 201, 32, 8, 128, 0, 32, pad=pad)
    keep = torch.zeros(b.pool.shape[0], 32, dtype=torch.bool)
    for ids, count in [(b.prefix_ids, 201), (b.ids[0], 5), (b.ids[1], 37), (b.ids[2], 1)]:
        for s in range(count):
            keep[ids[s // 32], s % 32] = True
    b.pool.masked_fill_(~keep.to(DEV)[:, None, None, :, None], filth)
    b.run(L)
    b.n, b.tok_seq, b.ctx = 5, b.tok_seq[:5], b.ctx[:5]
    b.check()


@pytest.mark.parametrize("dh,nh,nkvh", [(128, 32, 32), (64, 24, 8), (128, 64, 4), (64, 5, 5)])
@pytest.mark.parametrize("tokens,own", [(1, 3000), (20, 700), (300, 90)])
def test_own_contexts_of_few_and_many_blocks(L, dh, nh, nkvh, tokens, own):
    b = Batch(dh + tokens, [(1 + (own * (i + 1)) // tokens, 1) for i in range(tokens)], 0 if tokens > 20 else 70, nh, nkvh, dh, 1, 16)
    b.run(L)
    b.check()


FIRST = """
import sys
sys.path[:0] = sys.argv[1:3]
import torch
import llama_cu_b200 as L
import serve_ref as R
import test_prefix_gpu as P
lib = L.load_library()
few, many = P.Batch(1, [(5, 1), (40, 2)], 100, 32, 8, 128, 0, 16), P.Batch(2, [(30, 1)] * 40, 3000, 32, 8, 128, 1, 64)
x = R.rng_normal(3, (400, 20001), 2)
probs = torch.zeros_like(x)
u = torch.rand(100, 4, device="cuda")
drafted = torch.zeros(100, 3, dtype=torch.int32, device="cuda")
accepted, tokens = torch.zeros(100, dtype=torch.int32, device="cuda"), torch.zeros(100, 4, dtype=torch.int32, device="cuda")
q = R.rng_normal(4, (50, 8, 128), 0)
out, pos = torch.zeros_like(q), torch.arange(50, dtype=torch.int32, device="cuda")
sin, cos = R.tables(50, 64)
prep = L.QkPrep(None, None, sin.data_ptr(), cos.data_ptr(), 0, 1e-6, 50, 64, 1)
slots = torch.arange(50, dtype=torch.int32, device="cuda")
seq, table = torch.zeros_like(slots), torch.arange(4, dtype=torch.int32, device="cuda")
pool = torch.zeros(4, 2, 8, 16, 128, dtype=torch.float16, device="cuda")
pages = L.KvPages(pool.data_ptr(), pool[:, 1].data_ptr(), pool.stride(0), pool.stride(3), pool.stride(2), 4, 16)
for b in (few, many):
    b.dev = [R.i32(b.prefix_ids), R.i32(b.ids), R.i32(b.tok_seq), R.i32(b.ctx)]
    b.ws = torch.zeros(lib.lcu_attention_prefix_workspace_size(b.n, 32, 8, 128, b.prefix), dtype=torch.uint8, device="cuda")

def calls():
    s = R.stream()
    L.check(lib.lcu_op_qk_norm_rope(out.data_ptr(), 1024, 128, q.data_ptr(), 1024, 128, None, 0, 0, None, 0, 0, pos.data_ptr(), prep, 50, 8, 0, 128, 0, s))
    L.check(lib.lcu_op_kv_append(pages, table.data_ptr(), 4, 1, seq.data_ptr(), slots.data_ptr(), q.data_ptr(), 1024, 128, out.data_ptr(), 1024, 128, None, 0, 0, None, 0, 0,
                                 None, None, 50, 0, 8, 128, 0, s))
    for b in (few, many):
        L.check(lib.lcu_op_attention_prefix(b.o.data_ptr(), b.o.stride(0), 128, b.q.data_ptr(), b.q.stride(0), 128, L.KvPages(*b.pages_args()), b.dev[0].data_ptr(), b.prefix,
                                            b.dev[1].data_ptr(), b.per, b.n_seq, b.dev[2].data_ptr(), b.dev[3].data_ptr(), b.n, 32, 8, 128, b.scale, b.dims[3],
                                            b.ws.data_ptr(), b.ws.numel(), s))
    L.check(lib.lcu_op_softmax_rows(probs.data_ptr(), 20001, x.data_ptr(), 20001, None, 400, 20001, 2, s))
    L.check(lib.lcu_op_verify_drafts(accepted.data_ptr(), tokens.data_ptr(), probs.data_ptr(), 20001, None, 0, drafted.data_ptr(), None, u.data_ptr(), 100, 3, 20001, 2, s))

torch.cuda.synchronize()
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=side):
    calls()  # nothing of the library has run before
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (out, pool, few.o, many.o, probs, accepted, tokens)]
few.check(), many.check()
for t in (out, pool, few.o, many.o, probs, accepted, tokens):
    t.zero_()
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (out, pool, few.o, many.o, probs, accepted, tokens))) and got[1].any()
print("captured")
"""


def test_first_calls_of_a_process_may_be_captured(L):
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(here), here], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
