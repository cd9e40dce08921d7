"""Queries and keys normed and rotated in one pass, keys and values appended to pages (needs a B200)."""
import numpy as np
import pytest
import torch

import serve_ref as R
from serve_ref import DEV, DT, HALF

pytestmark = pytest.mark.gpu


def close(got, want, mag, dt):
    """One rounding of the result (half a step), and 32-bit arithmetic ahead of it: the sum of up to 256 squares in chains of 8 values and
    5 exchanges, the root, two products and the rotation are below 16 roundings of 2^-24 on the values that enter; subnormals of f16."""
    tol = HALF[dt] * want.abs() + 16 * 2.0 ** -24 * mag + (2.0 ** -25 if dt == 0 else 0)
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} values off, worst {(got.double() - want).abs().max()}"


def prep(L, q_w, k_w, w_dt, sin, cos, rot, halves, eps=1e-6):
    return L.QkPrep(R.addr(q_w), R.addr(k_w), R.addr(sin), R.addr(cos), w_dt, eps, 0 if sin is None else sin.shape[0], rot, int(halves))


def rows(seed, n, heads, dh, dt, form):
    """[n, heads, dh] views: 'whole' contiguous, 'cut' out of wider rows (16-byte pieces), 'odd' off every alignment."""
    if form == "whole":
        return R.rng_normal(seed, (n, heads, dh), dt)
    pad = 8 if form == "cut" else 3
    wide = R.rng_normal(seed, (n, heads * (dh + pad) + pad), dt)
    return wide[:, pad:].unflatten(1, (heads, dh + pad))[..., :dh]


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("n,nh,nkvh,dh,rot,halves,norm,form", [
    (1, 32, 8, 128, 128, True, "own", "whole"), (7, 4, 4, 64, 64, False, "f32", "whole"), (33, 7, 1, 80, 40, False, "own", "cut"),
    (5, 3, 3, 96, 48, True, None, "cut"), (301, 20, 4, 256, 256, True, "own", "whole"), (2, 5, 0, 192, 64, False, "f32", "whole"),
    (9, 0, 2, 32, 32, True, "own", "cut"), (3, 2, 1, 1, 0, False, "own", "odd"), (4, 3, 1, 66, 22, True, "f32", "odd"),
    (130, 4, 2, 37, 36, False, "own", "odd"), (6, 4, 2, 128, 0, False, "own", "whole"), (2500, 4, 1, 64, 32, False, None, "whole"),
    (3, 2, 2, 128, 120, True, "own", "whole"), (3, 2, 2, 128, 12, False, "own", "whole")])
def test_norm_and_rotation(L, dt, n, nh, nkvh, dh, rot, halves, norm, form):
    lib = L.load_library()
    w_dt = L.F32 if norm == "f32" else dt
    q, k = rows(1, n, nh, dh, dt, form), rows(2, n, nkvh, dh, dt, form)
    q_w, k_w = (R.rng_normal(s, (dh,), w_dt) if norm else None for s in (3, 4))
    sin, cos = R.tables(n + 5, rot) if rot else (None, None)
    pos = torch.randperm(n + 5, generator=torch.Generator().manual_seed(n))[:n].int().to(DEV)
    qo, ko = torch.full((n, nh, dh), 7.0, dtype=DT[dt], device=DEV), torch.full((n, nkvh, dh), 7.0, dtype=DT[dt], device=DEV)
    p = prep(L, q_w, k_w, w_dt, sin, cos, rot, halves)
    L.check(lib.lcu_op_qk_norm_rope(qo.data_ptr(), nh * dh, dh, q.data_ptr(), q.stride(0), q.stride(1), ko.data_ptr(), nkvh * dh, dh, k.data_ptr(), k.stride(0),
                                    k.stride(1), R.addr(pos) if rot else None, p, n, nh, nkvh, dh, dt, R.stream()))
    for x, w, got in ((q, q_w, qo), (k, k_w, ko)):
        close(got, *R.turn(x, w, 1e-6, pos, sin, cos, rot, halves), dt)


@pytest.mark.parametrize("dh,rot,halves", [(128, 128, True), (64, 32, False), (66, 66, True)])
def test_in_place_and_positions_behind_the_tables(L, dh, rot, halves):
    lib, dt, n, nh, nkvh = L.load_library(), 1, 40, 6, 2
    qkv = R.rng_normal(5, (n, (nh + nkvh) * dh), dt)
    before = qkv.clone()
    sin, cos = R.tables(30, rot)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)  # ten of them have no row
    pos[3] = -1
    q_w = R.rng_normal(6, (dh,), dt)
    st = qkv.stride(0)
    L.check(lib.lcu_op_qk_norm_rope(qkv.data_ptr(), st, dh, qkv.data_ptr(), st, dh, qkv[:, nh * dh:].data_ptr(), st, dh, qkv[:, nh * dh:].data_ptr(), st, dh, pos.data_ptr(),
                                    prep(L, q_w, None, dt, sin, cos, rot, halves), n, nh, nkvh, dh, dt, R.stream()))
    fine = torch.tensor([i < 30 and i != 3 for i in range(n)], device=DEV)
    assert torch.equal(qkv[~fine], before[~fine])
    x = before[fine].unflatten(1, (nh + nkvh, dh))
    got = qkv[fine].unflatten(1, (nh + nkvh, dh))
    close(got[:, :nh], *R.turn(x[:, :nh], q_w, 1e-6, pos[fine], sin, cos, rot, halves), dt)
    close(got[:, nh:], *R.turn(x[:, nh:], None, 1e-6, pos[fine], sin, cos, rot, halves), dt)


def test_rows_of_zeros_and_of_the_largest_values(L):
    """A row of zeros stays zero (eps carries it); squares beyond 32 bits leave a factor of zero, as in 32-bit arithmetic."""
    lib, dt, dh = L.load_library(), 1, 64
    q = torch.zeros(3, 1, dh, dtype=DT[dt], device=DEV)
    q[1] = 3e38
    q[2] = torch.nan
    o = torch.ones_like(q)
    w = torch.ones(dh, dtype=DT[dt], device=DEV)
    L.check(lib.lcu_op_qk_norm_rope(o.data_ptr(), dh, dh, q.data_ptr(), dh, dh, None, 0, 0, None, 0, 0, None, prep(L, w, None, dt, None, None, 0, 0), 3, 1, 0, dh, dt, R.stream()))
    assert (o[:2] == 0).all() and o[2].isnan().all()


def pool_of(pages, page, nkvh, dh, dt, layout, fill=7.0):
    """(tensor, KvPages arguments): 'own' is the framework's [page][k|v][head][token][dh], 'token' [k|v][page][token][head][dh]."""
    if layout == "own":
        t = torch.full((pages, 2, nkvh, page, dh), fill, dtype=DT[dt], device=DEV)
        return t, (t.data_ptr(), t[:, 1].data_ptr(), t.stride(0), t.stride(3), t.stride(2), pages, page)
    t = torch.full((2, pages, page, nkvh, dh), fill, dtype=DT[dt], device=DEV)
    return t, (t[0].data_ptr(), t[1].data_ptr(), t.stride(1), t.stride(2), t.stride(3), pages, page)


def place(pool, layout, page, slot, kv):
    return pool[page, kv, :, slot] if layout == "own" else pool[kv, page, slot]


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("nh,nkvh,dh,rot,halves,norm,page,layout", [
    (32, 8, 128, 128, False, False, 64, "own"), (4, 2, 64, 64, True, True, 8, "token"), (0, 3, 80, 80, False, True, 16, "own"),
    (3, 1, 37, 20, True, True, 32, "token"), (4, 4, 256, 128, True, False, 128, "own"), (0, 2, 64, 0, False, None, 16, "own")])
def test_append(L, dt, nh, nkvh, dh, rot, halves, norm, page, layout):
    """Prompts and decoded tokens of several sequences, padding and every index that names nothing between them; everything else of
    the pool and of the queries' output stays as it was."""
    lib = L.load_library()
    r = np.random.default_rng(dh + page)
    seqs, per = 5, 6
    pages = seqs * per + 4
    table = r.permutation(pages)[:seqs * per].reshape(seqs, per).astype(np.int32)
    table[2, 1], table[3, 0], table[4, 5] = -1, pages, 2 ** 31 - 1
    todo = [(s, p) for s in range(seqs) for p in r.permutation(per * page)[:25]]
    todo += [(-1, 3), (seqs, 0), (2 ** 31 - 1, 1), (0, per * page), (1, 2 ** 32 - 1)]
    r.shuffle(todo)
    n = len(todo)
    n_pos = 50
    pos = r.integers(0, n_pos + 3, n).astype(np.uint32)  # not the slots: a shared prefix lies before them
    tok_seq, slot = (R.i32(np.array([x[i] for x in todo]).astype(np.uint32).astype(np.int64).astype(np.uint32).view(np.int32)) for i in (0, 1))
    q, k, v = R.rng_normal(1, (n, nh, dh), dt), R.rng_normal(2, (n, nkvh, dh), dt), R.rng_normal(3, (n, nkvh, dh), dt)
    q_w, k_w = (R.rng_normal(s, (dh,), dt) if norm else None for s in (4, 5))
    sin, cos = R.tables(n_pos, rot) if rot else (None, None)
    pool, args = pool_of(pages, page, nkvh, dh, dt, layout)
    qo = torch.full((n, nh, dh), 7.0, dtype=DT[dt], device=DEV)
    p = None if norm is None else prep(L, q_w, k_w, dt, sin, cos, rot, halves)
    post, tt = R.i32(pos.view(np.int32)), R.i32(table)
    L.check(lib.lcu_op_kv_append(L.KvPages(*args), tt.data_ptr(), per, seqs, tok_seq.data_ptr(), slot.data_ptr(), k.data_ptr(), nkvh * dh, dh, v.data_ptr(), nkvh * dh, dh,
                                 qo.data_ptr() if nh else None, nh * dh, dh, q.data_ptr() if nh else None, nh * dh, dh, post.data_ptr() if rot else None, p, n, nh, nkvh, dh,
                                 dt, R.stream()))
    fine = [0 <= s < seqs and sl < per * page and 0 <= table[s, sl // page] < pages and (not rot or pos[i] < n_pos) for i, (s, sl) in enumerate(todo)]
    assert 60 < sum(fine) < n - 5
    args = (1e-6, post.clamp(max=n_pos - 1), sin, cos, rot, halves)
    (qw, qm), (kw, km) = R.turn(q, q_w, *args), R.turn(k, k_w, *args)
    left = torch.ones(pool.shape, dtype=torch.bool, device=DEV)
    for i, (s, sl) in enumerate(todo):
        if not fine[i]:
            assert nh == 0 or (qo[i] == 7).all()
            continue
        at = int(table[s, sl // page]), sl % page
        close(place(pool, layout, *at, 0), kw[i], km[i], dt)
        assert torch.equal(place(pool, layout, *at, 1), v[i])
        if nh:
            close(qo[i], qw[i], qm[i], dt)
        for kv in (0, 1):
            place(left, layout, *at, kv)[:] = False
    assert (pool[left] == 7).all()


def test_append_behind_32_bits(L):
    """A page that begins behind 2^32 elements of the pool."""
    lib, dt, nkvh, dh, page = L.load_library(), 1, 8, 128, 128
    one = 2 * nkvh * page * dh
    pages = 2 ** 32 // one + 3
    pool, args = pool_of(pages, page, nkvh, dh, dt, "own", 0.0)
    table = R.i32([[pages - 1, 0]])
    slot = R.i32([5, 130])
    k, v = R.rng_normal(1, (2, nkvh, dh), dt), R.rng_normal(2, (2, nkvh, dh), dt)
    zero = R.i32([0, 0])
    L.check(lib.lcu_op_kv_append(L.KvPages(*args), table.data_ptr(), 2, 1, zero.data_ptr(), slot.data_ptr(), k.data_ptr(), nkvh * dh, dh, v.data_ptr(), nkvh * dh, dh, None, 0,
                                 0, None, 0, 0, None, None, 2, 0, nkvh, dh, dt, R.stream()))
    assert torch.equal(pool[pages - 1, 0, :, 5], k[0]) and torch.equal(pool[0, 1, :, 2], v[1])
    assert torch.equal(pool[pages - 1, 1, :, 5], v[0]) and torch.equal(pool[0, 0, :, 2], k[1])
    assert not pool[1:pages - 1].any()


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("dh,rot", [(128, 64), (128, 16), (128, 112), (64, 48), (32, 16), (96, 32), (256, 240), (192, 96), (16, 16), (16, 0),
                                    (8, 0), (24, 16), (40, 32), (72, 48), (72, 64), (104, 16), (248, 240)])
@pytest.mark.parametrize("n", [3, 1200])
def test_rotations_of_a_part_of_the_head(L, dt, dh, rot, n):
    test_norm_and_rotation(L, dt, n, 5, 2, dh, rot, True, "own", "whole")
    test_norm_and_rotation(L, dt, n, 5, 2, dh, rot - 8 if rot > 8 else rot, False, "f32", "cut")
