"""Drafted tokens verified on a context of the framework's own: lcu_step_logits, then probabilities and verification, on logits whose rows are padded too
(needs a B200)."""
import numpy as np
import pytest
import torch

import serve_ref as R
import zefedra_models as M
from serve_ref import DEV
from test_verify_gpu import close, run as verify, softmax

pytestmark = pytest.mark.gpu


def context(L, kind):
    if kind == "llama":
        cfg = L.CONFIGS["tiny"]
        return cfg.vocab, L.load_model(cfg, L.synth_weights_numpy(cfg, 0))
    cfg, ctx = M.load(L, M.MIXED, M.weights(M.MIXED, 5), L.F32 if kind == "layered f32" else L.BF16)
    return cfg.vocab, ctx


@pytest.mark.parametrize("kind", ["llama", "layered f32", "layered bf16"])
def test_drafts_of_a_round(L, kind):
    vocab, ctx = context(L, kind)
    r, k, lens = np.random.default_rng(3), 3, (9, 2, 17)
    prompts = [r.integers(0, vocab, n) for n in lens]
    drafted = r.integers(0, vocab, (3, k))

    def logits():  # of each sequence's last token and its drafts (sequences of their own each time: states of layered models are not taken back)
        seqs = [ctx.seq_create() for _ in lens]
        ends = np.cumsum([n + k for n in lens])
        lg = ctx.step_logits([(s, 0, n + k) for s, n in zip(seqs, lens)], np.concatenate([np.concatenate([p, d]) for p, d in zip(prompts, drafted)]),
                             [int(e) - k - 1 + i for e in ends for i in range(k + 1)])
        for s in seqs:
            ctx.seq_free(s)
        return lg

    for i in range(k):  # drafts that the model itself would have given
        drafted[:, i] = logits().unflatten(0, (3, k + 1))[:, i].argmax(-1).cpu().numpy()
    drafted[1, 1] = (drafted[1, 1] + 1) % vocab
    lg = logits()
    assert lg.stride(0) == L.load_library().lcu_logits_stride(ctx.h) >= vocab and (kind == "llama") == (lg.stride(0) == vocab)
    best, counts = lg.unflatten(0, (3, k + 1)).argmax(-1).cpu().numpy(), R.i32([3, 3, 2])
    d = R.i32(drafted)
    for temperature in (0.0, 0.8):
        t = torch.full((3 * (k + 1),), temperature, device=DEV)
        p = softmax(L, lg, t)
        close(p, lg, t)
        p = p.view(3, k + 1, vocab)
        u = torch.as_tensor(r.random((3, k + 1), dtype=np.float32)).to(DEV)
        got = [x.cpu().numpy() for x in verify(L, p, None, d, counts, u)]
        want = R.verify(p.cpu().numpy(), None, drafted, [3, 3, 2], u.cpu().numpy())
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        if temperature == 0:
            assert got[0].tolist() == [3, 1, 2]
            for b, n in enumerate(got[0]):
                assert got[1][b].tolist() == best[b, :n + 1].tolist() + [-1] * (k - n)
    ctx.close()
