"""What the operators on a caller's pages and of drafted tokens refuse, and their sizes: before any GPU is asked."""
import ctypes as C

import pytest

P = 4096  # an address that is aligned and never read


def pages(L, **change):
    args = dict(k=P, v=P, stride_page=16 * 128 * 4, stride_tok=128, stride_head=16 * 128, n_pages=9, page_tokens=16)
    args.update(change)
    return L.KvPages(**args)


def prep(L, **change):
    args = dict(q_norm=P, k_norm=P, sin_t=P, cos_t=P, norm_dt=L.F16, eps=1e-6, n_pos=10, rot_dims=128, rot_halves=1)
    args.update(change)
    return L.QkPrep(**args)


def refused(L, rc, word):
    assert rc == L.ERR_INVALID, rc
    assert word in L.last_error(), L.last_error()


def norm_rope(L, n=3, nh=4, nkvh=2, dh=128, dt=0, q=P, qo=P, k=P, ko=P, pos=P, p="default"):
    return L.load_library().lcu_op_qk_norm_rope(qo, nh * dh, dh, q, nh * dh, dh, ko, nkvh * dh, dh, k, nkvh * dh, dh, pos, prep(L) if p == "default" else p, n, nh, nkvh, dh, dt, None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=3), "dtype"), (dict(n=-1), "tokens"), (dict(nh=0, nkvh=0), "heads"), (dict(nh=-1), "heads"), (dict(dh=257), "values"), (dict(dh=0), "values"),
    (dict(q=None), "null"), (dict(qo=None), "null"), (dict(k=None), "null"), (dict(ko=None), "null"), (dict(p=None), "null"), (dict(pos=None), "positions")])
def test_norm_rope_refuses(L, change, word):
    refused(L, norm_rope(L, **change), word)


@pytest.mark.parametrize("change,word", [
    (dict(rot_dims=127), "rotated"), (dict(rot_dims=-2), "rotated"), (dict(rot_dims=130), "rotated"), (dict(sin_t=None), "tables"), (dict(cos_t=None), "tables"),
    (dict(n_pos=0), "tables"), (dict(norm_dt=1), "norm weights"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")])
def test_prep_refuses(L, change, word):
    refused(L, norm_rope(L, p=prep(L, **change)), word)
    refused(L, append(L, p=prep(L, **change)), word)


def append(L, n=3, nh=4, nkvh=2, dh=128, dt=0, table=P, stride=4, seqs=2, tok=P, slot=P, k=P, v=P, q=P, qo=P, p="default", pg=None):
    return L.load_library().lcu_op_kv_append(pg or pages(L), table, stride, seqs, tok, slot, k, nkvh * dh, dh, v, nkvh * dh, dh, qo, nh * dh, dh, q, nh * dh, dh, P,
                                             prep(L) if p == "default" else p, n, nh, nkvh, dh, dt, None)


@pytest.mark.parametrize("change,word", [
    (dict(table=None), "null"), (dict(tok=None), "null"), (dict(slot=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q=None), "null"),
    (dict(qo=None), "null"), (dict(stride=0), "pages"), (dict(seqs=0), "sequences"), (dict(nkvh=0), "KV heads"), (dict(p=None), "queries"), (dict(dt=4), "dtype"),
    (dict(n=-3), "tokens"), (dict(dh=300), "values")])
def test_append_refuses(L, change, word):
    refused(L, append(L, **change), word)


PAGES = [(dict(k=None), "no pages"), (dict(v=None), "no pages"), (dict(n_pages=0), "no pages"), (dict(page_tokens=4), "power of two"), (dict(page_tokens=48), "power of two"),
         (dict(page_tokens=256), "power of two"), (dict(stride_page=0), "strides"), (dict(stride_tok=-1), "strides")]


@pytest.mark.parametrize("change,word", PAGES)
def test_pages_refused(L, change, word):
    refused(L, append(L, pg=pages(L, **change)), word)
    refused(L, attention(L, pg=pages(L, **change)), word)


def attention(L, n=3, nh=8, nkvh=2, dh=128, dt=0, o=P, q=P, prefix=100, ptab=P, table=P, stride=4, seqs=2, tok=P, ctx=P, scale=0.1, ws=P, ws_len=None, pg=None, sq=None):
    lib = L.load_library()
    need = lib.lcu_attention_prefix_workspace_size(n, nh, nkvh, dh, prefix)
    return lib.lcu_op_attention_prefix(o, nh * dh, dh, q, nh * dh if sq is None else sq, dh, pg or pages(L), ptab, prefix, table, stride, seqs, tok, ctx, n, nh, nkvh, dh, scale, dt, ws,
                                       need if ws_len is None else ws_len, None)


@pytest.mark.parametrize("change,word", [
    (dict(dt=2), "dtype"), (dict(dh=96), "dh"), (dict(dh=256), "dh"), (dict(n=-1), "tokens"), (dict(n=65536), "tokens"), (dict(nh=9), "query heads"), (dict(nh=34), "query heads"),
    (dict(nkvh=0), "query heads"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(prefix=2 ** 31), "prefix"), (dict(stride=-1), "pages"), (dict(stride=2 ** 28), "pages"), (dict(seqs=0), "sequences"), (dict(o=None), "null"), (dict(q=None), "null"),
    (dict(tok=None), "null"), (dict(ctx=None), "null"), (dict(ptab=None), "null"), (dict(table=None), "null"), (dict(q=P + 8), "16 bytes"), (dict(o=P + 2), "16 bytes"),
    (dict(sq=1028), "16 bytes")])
def test_attention_refuses(L, change, word):
    refused(L, attention(L, **change), word)


def test_attention_refuses_pages_off_16_bytes_and_short_workspaces(L):
    refused(L, attention(L, pg=pages(L, k=P + 8)), "16 bytes")
    refused(L, attention(L, pg=pages(L, stride_tok=132)), "16 bytes")
    refused(L, attention(L, pg=pages(L, stride_page=16 * 128 * 4 + 4)), "16 bytes")
    need = L.load_library().lcu_attention_prefix_workspace_size(3, 8, 2, 128, 100)
    if need:
        refused(L, attention(L, ws_len=need - 1), "workspace")
        refused(L, attention(L, ws=None), "workspace")
        refused(L, attention(L, ws=P + 16), "workspace")


def test_workspace_sizes(L):
    """Nothing without a prefix; bad shapes ask for nothing (the call refuses them)."""
    size = L.load_library().lcu_attention_prefix_workspace_size
    assert size(5, 8, 2, 128, 0) == 0 and size(0, 8, 2, 128, 100) == 0 and size(5, 8, 0, 128, 100) == 0 and size(-1, 8, 2, 128, 100) == 0 and size(5, 8, 3, 128, 9) == 0
    assert size(5, 8, 2, 0, 100) == 0 and size(5, -8, 2, 128, 100) == 0


def softmax(L, rows=2, n=100, dt=2, probs=P, logits=P, sp=100, sl=100):
    return L.load_library().lcu_op_softmax_rows(probs, sp, logits, sl, None, rows, n, dt, None)


@pytest.mark.parametrize("change,word", [(dict(dt=3), "dtype"), (dict(rows=-1), "rows"), (dict(n=0), "rows"), (dict(n=2 ** 31), "rows"), (dict(sp=99), "strides"), (dict(sl=99), "strides"),
                                         (dict(probs=None), "null"), (dict(logits=None), "null")])
def test_softmax_refuses(L, change, word):
    refused(L, softmax(L, **change), word)


def verify(L, seqs=2, k=3, n=100, dt=2, acc=P, tok=P, target=P, draft=P, drafted=P, u=P, st=100, sd=100):
    return L.load_library().lcu_op_verify_drafts(acc, tok, target, st, draft, sd, drafted, None, u, seqs, k, n, dt, None)


@pytest.mark.parametrize("change,word", [(dict(dt=3), "dtype"), (dict(seqs=-1), "sequences"), (dict(k=-1), "drafts"), (dict(k=65536), "drafts"), (dict(n=0), "tokens"), (dict(n=2 ** 31), "tokens"),
                                         (dict(acc=None), "null"), (dict(tok=None), "null"), (dict(target=None), "null"), (dict(drafted=None), "null"), (dict(u=None), "null"),
                                         (dict(st=99), "strides"), (dict(sd=99), "strides")])
def test_verify_refuses(L, change, word):
    refused(L, verify(L, **change), word)


def test_nothing_to_do_asks_no_gpu(L):
    assert norm_rope(L, n=0) == append(L, n=0) == attention(L, n=0) == softmax(L, rows=0) == verify(L, seqs=0) == L.OK


def test_accessors_refuse(L):
    lib = L.load_library()
    out, n = L.KvPages(), C.c_int()
    refused(L, lib.lcu_kv_layer_pages(None, 0, C.byref(out)), "null")
    refused(L, lib.lcu_seq_pages(None, 0, None, 0, C.byref(n)), "bad sequence")


def test_counts_whose_indices_would_not_fit(L):
    refused(L, softmax(L, rows=2 ** 30 + 1), "rows")
    refused(L, verify(L, seqs=2 ** 30 + 1), "sequences")
    refused(L, norm_rope(L, n=2 ** 30 + 1), "tokens")
    refused(L, append(L, n=2 ** 30 + 1), "tokens")
    size = L.load_library().lcu_attention_prefix_workspace_size
    assert size(65536, 8, 2, 128, 100) == size(2 ** 31 - 1, 2 ** 31 - 1, 1, 128, 2 ** 32 - 1) == size(3, 34, 2, 128, 100) == 0  # (what the call refuses)


def test_more_units_than_a_call_takes(L):
    refused(L, attention(L, n=65535, nh=64, nkvh=8, prefix=2 ** 31 - 1, stride=0), "more than a call takes")
    assert L.load_library().lcu_attention_prefix_workspace_size(65535, 64, 8, 128, 2 ** 31 - 1) == 0
