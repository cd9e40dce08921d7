"""Pages of one KV head: their stride from head to head names nothing, whatever it is, for those who write them and for those who read them."""
import numpy as np
import pytest
import torch

import test_serve_ops_cpu as S

STRIDES = [0, -7, 1, 3, 2 ** 31 - 1]


@pytest.mark.parametrize("stride", [0, -7])
def test_several_heads_need_a_stride(L, stride):
    S.refused(L, S.append(L, pg=S.pages(L, stride_head=stride)), "strides")
    S.refused(L, S.attention(L, pg=S.pages(L, stride_head=stride)), "strides")


@pytest.mark.parametrize("stride", STRIDES)
def test_one_head_needs_none(L, stride):
    """What is refused behind the pages is refused for its own reason."""
    pg = S.pages(L, stride_head=stride)
    S.refused(L, S.append(L, nkvh=1, dh=300, pg=pg), "values")
    S.refused(L, S.attention(L, nkvh=1, nh=8, q=None, pg=pg), "null")
    S.refused(L, S.attention(L, nkvh=1, nh=8, ws_len=0, ws=None, pg=pg, prefix=100), "workspace") if L.load_library().lcu_attention_prefix_workspace_size(3, 8, 1, 128, 100) else None


@pytest.mark.gpu
@pytest.mark.parametrize("stride", STRIDES)
@pytest.mark.parametrize("prefix,own", [(40, 100), (3000, 5), (0, 200)])
def test_one_head_written_and_read(L, stride, prefix, own):
    """Filled token by token and read, with the stride of a pool of several heads and with another: the same bits in both."""
    import serve_ref as R
    from test_prefix_gpu import Batch
    lib = L.load_library()
    b = Batch(prefix + own, [(own, 1)] * 3, prefix, 8, 1, 64, 1, 16)
    k = R.rng_normal(1, (b.n_pages * 16, 2, 1, 64), 1)
    table, n = R.i32(np.arange(b.n_pages)), k.shape[0]
    seq, slot = R.i32(np.zeros(n)), R.i32(np.arange(n))
    got = []
    for s in (16 * 64, stride):
        b.pool.zero_()
        args = list(b.pages_args())
        args[4] = s
        L.check(lib.lcu_op_kv_append(L.KvPages(*args), table.data_ptr(), b.n_pages, 1, seq.data_ptr(), slot.data_ptr(), k.data_ptr(), 128, 64, k[:, 1].data_ptr(), 128, 64, None, 0, 0,
                                     None, 0, 0, None, None, n, 0, 1, 64, 1, R.stream()))
        assert torch.equal(b.pool.transpose(2, 3).flatten(3), k.view(b.n_pages, 16, 2, 64).transpose(1, 2))
        b.pages_args = lambda: args
        b.run(L)
        del b.pages_args
        b.check()
        got.append(b.o.clone())
    assert torch.equal(got[0], got[1])
