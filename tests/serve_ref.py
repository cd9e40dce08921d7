"""Plain 64-bit forms of the operators on a caller's pages and of drafted tokens (tests only), and the calls."""
import ctypes as C

import numpy as np
import torch

DEV = "cuda:0"
DT = {0: torch.float16, 1: torch.bfloat16, 2: torch.float32}
HALF = {dt: torch.finfo(t).eps / 2 for dt, t in DT.items()}  # half a step, relative to the value


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def addr(t):
    return None if t is None else t.data_ptr()


def i32(a, device=DEV):
    return torch.as_tensor(np.ascontiguousarray(a, dtype=np.int32)).to(device)


def rng_normal(seed, shape, dt, std=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(DT[dt])


def tables(n_pos, rot):
    f = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * f
    return a.sin().float().to(DEV), a.cos().float().to(DEV)


def turn(x, w, eps, pos, sin, cos, rot, halves):
    """(value, sum of magnitudes that entered it) of rows [n, heads, dh], in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    out, mag = y.clone(), y.abs()
    for i in range(rot // 2):
        p, q = (i, i + rot // 2) if halves else (2 * i, 2 * i + 1)
        s, c = sin[pos.long(), i].double()[:, None], cos[pos.long(), i].double()[:, None]
        out[..., p], out[..., q] = y[..., p] * c - y[..., q] * s, y[..., p] * s + y[..., q] * c
        mag[..., p] = mag[..., q] = y[..., p].abs() + y[..., q].abs()
    return out, mag


def attention(q, k_prefix, v_prefix, k_own, v_own, scale):
    """One token: q [nh, dh], keys and values [positions, nkvh, dh] that it sees -> (o, sum of weights times |v|), in 64 bits."""
    k, v = torch.cat([k_prefix, k_own]).double(), torch.cat([v_prefix, v_own]).double()
    nh, nkvh = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return z, z
    s = torch.einsum("hgd,phd->hgp", q.double().view(nkvh, nh // nkvh, -1), k) * scale
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    return torch.einsum("hgp,phd->hgd", w, v).reshape(q.shape), torch.einsum("hgp,phd->hgd", w, v.abs()).reshape(q.shape)


def softmax_rows(x, temperature):
    """x [rows, n] (any type), in 64 bits with the operator's rules for rows without a largest value."""
    x = x.double()
    out = torch.zeros_like(x)
    for r in range(x.shape[0]):
        t = float(temperature[r])
        row = x[r]
        if t == 0:
            row = torch.where(row.isnan(), -torch.inf, row)
            if row.max() > -torch.inf:
                out[r, int((row == row.max()).nonzero()[0])] = 1
        elif row.isnan().any() or (row == torch.inf).any():
            out[r] = torch.nan
        elif row.max() > -torch.inf:
            e = torch.exp((row - row.max()) / t)
            out[r] = e / e.sum()
    return out


def verify(target, draft, drafted, n_drafted, u):
    """target [b, k + 1, n], draft [b, k, n] or None: numpy, any float type.  Returns accepted [b], tokens [b, k + 1]."""
    seqs, k1, n = target.shape
    accepted, tokens = np.zeros(seqs, np.int32), np.full((seqs, k1), -1, np.int32)
    def clean(w):
        return np.where(np.isfinite(w) & (w > 0), w, 0.0)
    for b in range(seqs):
        nd = k1 - 1 if n_drafted is None else min(max(int(n_drafted[b]), 0), k1 - 1)
        i = 0
        while i < nd:
            x = int(drafted[b, i])
            if not (0 <= x < n and float(u[b, i]) * (1.0 if draft is None else float(draft[b, i, x])) < float(target[b, i, x])):
                break
            tokens[b, i] = x
            i += 1
        accepted[b] = i
        p = target[b, i].astype(np.float64)
        w = clean(p)
        if i < nd:
            if draft is not None:
                rest = clean(p - draft[b, i].astype(np.float64))
            else:
                one = np.zeros(n)
                if 0 <= drafted[b, i] < n:
                    one[drafted[b, i]] = 1.0
                rest = clean(p - one)
            if rest.sum() > 0:
                w = rest
        if w.sum() > 0:
            run = np.cumsum(w)
            above = np.nonzero(run > float(u[b, -1]) * run[-1])[0]
            tokens[b, i] = above[0] if len(above) else np.nonzero(w)[0][-1]
    return accepted, tokens
