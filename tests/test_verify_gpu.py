"""Probabilities of rows of logits, and verification of drafted tokens (needs a B200)."""
import numpy as np
import pytest
import torch

import serve_ref as R
from serve_ref import DEV, DT

pytestmark = pytest.mark.gpu


def softmax(L, x, t, out=None):
    out = torch.full((x.shape[0], x.shape[1]), 7.0, device=DEV) if out is None else out
    L.check(L.load_library().lcu_op_softmax_rows(out.data_ptr(), out.stride(0), x.data_ptr(), x.stride(0), R.addr(t), x.shape[0], x.shape[1], {v: k for k, v in DT.items()}[x.dtype],
                                                 R.stream()))
    return out


def close(got, x, t):
    """32-bit arithmetic: the exponent's argument z is off by 3 roundings, so its value by 3 |z| 2^-24 relatively; two exponentials of 2 ulp, sums of up to
    64 values in a thread, 9 exchanges and 8 CTAs below 96 roundings in all; results below 2^-126 keep 2^-149."""
    want = R.softmax_rows(x, t)
    assert torch.equal(got.isnan(), want.isnan())
    z = (x.double() - x.double().amax(-1, keepdim=True)) / torch.where(t == 0, 1.0, t.double())[:, None]
    z = torch.nan_to_num(z, nan=0.0, posinf=0.0, neginf=0.0).abs()
    fine = ~want.isnan()
    off = (got.double() - want).abs()
    assert (off <= want * 2.0 ** -24 * (3 * z + 96) + 2.0 ** -148)[fine].all(), float(off[fine].max())


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("rows,n,shift", [(1, 1, 0), (3, 7, 0), (2, 512, 0), (5, 4097, 1), (1, 32000, 0), (3, 128256, 0), (2, 131073, 0), (1, 300001, 3), (70, 100, 0)])
def test_softmax(L, dt, rows, n, shift):
    wide = R.rng_normal(n + dt, (rows, n + 2 * shift), dt, 3.0)
    x = wide[:, shift:shift + n]
    t = torch.tensor([0.8, 1.0, 0.0, 1e-3, 50.0], device=DEV).repeat(rows // 5 + 1)[:rows].contiguous()
    got = softmax(L, x, t)
    close(got, x, t)
    greedy = t == 0
    assert torch.equal(got[greedy].double(), R.softmax_rows(x[greedy], t[greedy]))
    if rows > 1:
        one = torch.ones(rows, device=DEV)
        close(softmax(L, x, None), x, one)


def test_softmax_of_more_rows_than_a_grid_has(L):
    x = R.rng_normal(1, (66000, 9), 2)
    t = torch.ones(66000, device=DEV)
    got = softmax(L, x, t)
    assert (got.double() - torch.softmax(x.double(), -1)).abs().max() < 2.0 ** -24 * 200


def test_softmax_writes_rows_into_wider_ones(L):
    x = R.rng_normal(2, (4, 1000), 1)
    wide = torch.full((4, 1003), 7.0, device=DEV)
    t = torch.ones(4, device=DEV)
    close(softmax(L, x, t, wide)[:, :1000], x, t)
    assert (wide[:, 1000:] == 7).all()


@pytest.mark.parametrize("n", [5, 9000, 200000])
@pytest.mark.parametrize("temperature", [0.0, 1.0, 1e-38, 1e-45])
def test_softmax_of_rows_with_masks(L, n, temperature):
    inf, nan = torch.inf, torch.nan
    x = R.rng_normal(3, (9, n), 2)
    x[0] = -inf                            # nothing left
    x[1, 1:] = -inf                        # one token left
    x[2, :n // 2 + 1] = torch.finfo(torch.float32).min  # masked with the type's lowest value
    x[3] = torch.finfo(torch.float32).min  # ... everywhere
    x[4, n - 1] = nan
    x[5, 2] = x[5, n - 1] = inf
    x[6, 0], x[6, 1] = -inf, nan
    x[7] = 0.0                             # ties: -0 and 0 are equal
    x[7, 1] = -0.0
    x[8, n // 3] = x[8, n - 2] = 99.0      # a tie
    t = torch.full((9,), temperature, device=DEV)
    got = softmax(L, x, t)
    if temperature in (0.0, 1.0):
        close(got, x, t)
    else:  # as good as greedy, ties shared
        assert (got[0] == 0).all() and got[1, 0] == 1 and got[4].isnan().all() and got[5].isnan().all()
        assert (got[3] - 1 / n).abs().max() < 1e-6 and got[8, n // 3] == 0.5 and got[8, n - 2] == 0.5
    if temperature == 0:
        assert got[7, 0] == 1 and got[8, n // 3] == 1 and got[0].sum() == 0 and got[3, 0] == 1


def cases(seed, seqs, k, n, dt, kind):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    lg = torch.randn(seqs, k + 1, n, generator=g, device=DEV) * 2.5
    near = lg[:, :k] + torch.randn(seqs, k, n, generator=g, device=DEV) * 0.7
    target, draft = torch.softmax(lg, -1).to(DT[dt]), torch.softmax(near, -1).to(DT[dt])
    drafted = torch.multinomial(draft.float().view(-1, n) + 1e-30, 1, generator=g).view(seqs, k).int() if k else torch.zeros(seqs, 0, dtype=torch.int32, device=DEV)
    return target, draft if kind == "sampled" else None, drafted, torch.rand(seqs, k + 1, generator=g, device=DEV)


def run(L, target, draft, drafted, n_drafted, u):
    seqs, k1, n = target.shape
    accepted, tokens = torch.full((seqs,), 77, dtype=torch.int32, device=DEV), torch.full((seqs, k1), 77, dtype=torch.int32, device=DEV)
    L.check(L.load_library().lcu_op_verify_drafts(accepted.data_ptr(), tokens.data_ptr(), target.data_ptr(), target.stride(1), R.addr(draft), draft.stride(1) if draft is not None else 0,
                                                  drafted.data_ptr(), R.addr(n_drafted), u.data_ptr(), seqs, k1 - 1, n, {v: c for c, v in DT.items()}[target.dtype], R.stream()))
    return accepted, tokens


def host(t):
    return None if t is None else t.cpu().numpy() if t.dtype in (torch.int32, torch.float32) else t.float().cpu().numpy()


def same(L, target, draft, drafted, n_drafted, u):
    got = run(L, target, draft, drafted, n_drafted, u)
    want = R.verify(*(host(t) for t in (target, draft, drafted, n_drafted, u)))
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy(), b)
    return want


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("kind", ["sampled", "certain"])
@pytest.mark.parametrize("seqs,k,n", [(1, 4, 32000), (9, 3, 2047), (5, 0, 513), (3, 1, 1), (4, 40, 300), (33, 7, 4097), (2, 2, 128256)])
def test_verify(L, dt, kind, seqs, k, n):
    target, draft, drafted, u = cases(seqs + n, seqs, k, n, dt, kind)
    same(L, target, draft, drafted, None, u)
    counts = R.i32(np.random.default_rng(n).integers(-2, k + 3, seqs))  # clamped to [0, k]
    same(L, target, draft, drafted, counts, u)


def test_verify_accepts_and_rejects(L):
    """Both happen, at every place, and the last token comes from a rejected row as well as from the last one."""
    target, draft, drafted, u = cases(3, 200, 3, 500, 2, "sampled")
    accepted, _ = same(L, target, draft, drafted, None, u)
    assert set(accepted.tolist()) == {0, 1, 2, 3}


def test_verify_rows_off_every_alignment(L):
    seqs, k, n = 4, 3, 5001
    target, draft, drafted, u = cases(5, seqs, k, n, 1, "sampled")
    tw, dw = (torch.full((seqs * r, n + 6), torch.nan, dtype=torch.bfloat16, device=DEV) for r in (k + 1, k))
    tw[:, 3:3 + n], dw[:, 5:5 + n] = target.reshape(-1, n), draft.reshape(-1, n)
    want = R.verify(*(host(t) for t in (target, draft, drafted, None, u)))
    t, d = tw.view(seqs, k + 1, n + 6)[..., 3:3 + n], dw.view(seqs, k, n + 6)[..., 5:5 + n]
    for a, b in zip(run(L, t, d, drafted, None, u), want):
        assert np.array_equal(a.cpu().numpy(), b)


def test_verify_of_a_very_long_row(L):
    """More pieces than a CTA keeps: their size doubles."""
    target, draft, drafted, u = cases(6, 2, 1, 5000003, 2, "sampled")
    same(L, target, draft, drafted, None, u)


@pytest.mark.parametrize("kind", ["sampled", "certain"])
@pytest.mark.parametrize("n", [6, 9000])
def test_verify_at_the_borders(L, kind, n):
    """Random numbers of 0 and just below 1, probabilities of 0, rows without mass, drafts outside the vocabulary, values that are no probabilities."""
    seqs, k = 14, 2
    target, draft, drafted, u = cases(7, seqs, k, n, 2, kind)
    drafted.clamp_(max=n - 1)
    below = 1 - 2.0 ** -24
    u[0], u[1] = 0.0, below
    x = drafted[2:8, 0].long()
    at = torch.arange(2, 8, device=DEV)
    target[at, 0, x] = 0.0          # never accepted
    u[2, 0] = u[3, 0] = 0.0
    drafted[8, 0], drafted[9, 0], drafted[10, 1] = -1, n, 2 ** 31 - 1
    target[11] = 0.0                # no mass at all
    u[11] = 0.25
    target[12] = 0.0
    target[12, :, n - 1], target[12, :, 1] = torch.nan, -1.0
    target[12, :, 2] = 0.125
    u[12, 0] = below
    target[13, 0, 0] = torch.inf
    if draft is not None:
        draft[4] = target[4, :k]    # nothing left when the draft is rejected: p itself
        draft[5, 0] = 0.0
    accepted, tokens = same(L, target, draft, drafted, None, u)
    assert (accepted[2:10] == 0).all() and tokens[11, 0] == -1
    u[:, -1] = below
    same(L, target, draft, drafted, None, u)


def test_greedy_round(L):
    """Temperature 0 all along: drafts are accepted as long as they are the target's largest, then comes the target's."""
    n, k = 3001, 3
    lg = R.rng_normal(9, (4, k + 1, n), 1, 3.0)
    best = lg.float().argmax(-1).int()
    drafted = best[:, :k].clone()
    drafted[1, 0] = (drafted[1, 0] + 1) % n
    drafted[2, 2] = (drafted[2, 2] + 1) % n
    p = softmax(L, lg.view(-1, n), torch.zeros(4 * (k + 1), device=DEV)).view(4, k + 1, n)
    accepted, tokens = run(L, p, None, drafted, None, torch.full((4, k + 1), 0.999, device=DEV))
    assert accepted.tolist() == [3, 0, 2, 3]
    for b, a in enumerate(accepted.tolist()):
        assert tokens[b].tolist() == best[b, :a + 1].tolist() + [-1] * (k - a)


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("rows,n,pad", [(700, 2049, 0), (600, 20001, 0), (300, 50257, 6), (120, 100003, 1), (80, 200001, 0), (60, 262145, 0), (400, 5000, 3)])
def test_softmax_of_many_rows_that_begin_inside_a_piece(L, dt, rows, n, pad):
    """More rows than run at once, and strides that are no multiple of 16 bytes: the copy of the next row begins ahead of it."""
    x = R.rng_normal(n + dt, (rows, n + pad), dt, 3.0)[:, :n]
    t = torch.tensor([0.8, 1.0, 0.0, 1e-3, 50.0, 2.5, 0.3], device=DEV).repeat(rows // 7 + 1)[:rows].contiguous()
    x[5, 3:] = -torch.inf
    x[6] = -torch.inf
    wide = torch.full((rows, n + pad), 7.0, device=DEV)
    got = softmax(L, x, t, wide)[:, :n]
    assert (wide[:, n:] == 7).all()
    for at in range(0, rows, 100):  # (64 bits of all rows at once would take gigabytes)
        close(got[at:at + 100], x[at:at + 100], t[at:at + 100])


@pytest.mark.parametrize("rows,n", [(3, 1000), (1, 128256), (200, 30001), (90, 262144), (5, 300001)])
def test_softmax_in_place(L, rows, n):
    x = R.rng_normal(n, (rows, n), 2, 3.0)
    t = torch.tensor([0.7, 0.0, 1.0], device=DEV).repeat(rows // 3 + 1)[:rows].contiguous()
    want = softmax(L, x, t)
    assert torch.equal(softmax(L, x, t, x), want)
