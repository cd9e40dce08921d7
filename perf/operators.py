"""Measured cases of the stand-alone operators of a serving round: queries and keys normed and rotated, keys and values appended to a
paged cache, attention of a batch that shares a long prefix, probabilities of rows of logits, verification of drafted tokens.

Sizes are those of `llama_cu_b200.CONFIGS` (32 or 64 query heads over 8 key/value heads of 64 or 128, vocabularies of 32000 and 128256)
and generic ones.  A cache is [page][k|v][kv head][token][head size], one layer of the framework's own page.

`run` computes a case with elementary torch operations in 32 bits (64 for sums and comparisons that choose a token), or, where `own` is
true, with the framework's operators.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"f16": 0, "bf16": 1, "f32": 2}  # lcu_dtype
EPS = 1e-6


def listed():
    return [
        # one decoded token: the launch is all there is
        {"name": "norm-rope-8b-1", "op": "norm_rope", "tokens": 1, "nh": 32, "nkvh": 8, "dh": 128, "rot": 128, "halves": True, "dtype": "bf16", "norm": True},
        # a long document's queries and keys, part of each head rotated in neighbouring pairs
        {"name": "norm-rope-1b-8000", "op": "norm_rope", "tokens": 8000, "nh": 32, "nkvh": 8, "dh": 64, "rot": 32, "halves": False, "dtype": "f16", "norm": True},
        # a decode round of 33 sequences
        {"name": "append-8b-33", "op": "append", "tokens": 33, "seqs": 33, "nh": 32, "nkvh": 8, "dh": 128, "rot": 128, "halves": False, "dtype": "f16",
         "norm": False, "page": 64, "past": 777, "pad": 0},
        # prompts of four sequences, the batch padded behind them
        {"name": "append-8b-4x2001-norm", "op": "append", "tokens": 8004, "seqs": 4, "nh": 32, "nkvh": 8, "dh": 128, "rot": 128, "halves": True, "dtype": "bf16",
         "norm": True, "page": 32, "past": 100, "pad": 60},
        # three answers to a short prompt
        {"name": "prefix-1b-3x100", "op": "prefix", "seqs": 3, "new": 1, "prefix": 100, "short": 1, "long": 40, "nh": 32, "nkvh": 8, "dh": 64, "dtype": "bf16", "page": 16, "pad": 0},
        # a service whose conversations begin with the same instructions
        {"name": "prefix-8b-33x2000", "op": "prefix", "seqs": 33, "new": 1, "prefix": 2000, "short": 30, "long": 500, "nh": 32, "nkvh": 8, "dh": 128, "dtype": "f16", "page": 64, "pad": 0},
        # four drafted tokens and the last one of every sequence, behind a long document
        {"name": "prefix-8b-drafts-16x8001", "op": "prefix", "seqs": 16, "new": 5, "prefix": 8001, "short": 5, "long": 300, "nh": 32, "nkvh": 8, "dh": 128, "dtype": "bf16", "page": 32, "pad": 0},
        # many samples of one long prompt
        {"name": "prefix-70b-256x32000", "op": "prefix", "seqs": 256, "new": 1, "prefix": 32000, "short": 1, "long": 200, "nh": 64, "nkvh": 8, "dh": 128, "dtype": "f16", "page": 64, "pad": 0},
        # one row of the smaller vocabulary
        {"name": "softmax-1x32000", "op": "softmax", "rows": 1, "vocab": 32000, "dtype": "f16"},
        # the rows of a round that verifies four drafted tokens of each of 32 sequences
        {"name": "softmax-160x128256", "op": "softmax", "rows": 160, "vocab": 128256, "dtype": "f32"},
        # one user, four drafted tokens
        {"name": "verify-1x4-32000", "op": "verify", "seqs": 1, "k": 4, "vocab": 32000, "dtype": "f32", "drafts": "sampled"},
        # a service under load
        {"name": "verify-64x4-128256", "op": "verify", "seqs": 64, "k": 4, "vocab": 128256, "dtype": "f32", "drafts": "sampled"},
    ]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Any operator; heads, types, pages, tokens, contexts and vocabularies over the whole range, odd ones among them."""
    op = rng.choice(["norm_rope", "append", "prefix", "prefix", "softmax", "verify"])
    if op == "softmax":
        vocab = log_uniform(rng, 8, 262144)
        return {"op": op, "rows": log_uniform(rng, 1, max(1, min(1000, 20000000 // vocab))), "vocab": vocab, "dtype": rng.choice(["f16", "bf16", "f32"])}
    if op == "verify":
        vocab = log_uniform(rng, 1000, 262144)
        k = rng.randint(0, 8)
        return {"op": op, "seqs": log_uniform(rng, 1, max(1, min(500, 8000000 // vocab))), "k": k, "vocab": vocab, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]),
                "drafts": rng.choice(["sampled", "sampled", "given"])}
    nh, nkvh = rng.choice([(32, 8), (32, 8), (64, 8), (8, 1), (4, 4), (12, 4), (20, 4), (16, 1), (7, 7)])
    dh = rng.choice([64, 128])
    if op == "prefix":
        seqs = log_uniform(rng, 1, 256)
        new = rng.randint(1, 8) if seqs <= 64 else 1
        prefix = log_uniform(rng, 1, min(32000, 256 * 32000 * 64 * 128 // (seqs * new * nh * dh))) if rng.random() < 0.9 else 0
        short = new + rng.randint(0, 60)
        return {"op": op, "seqs": seqs, "new": new, "prefix": prefix, "short": short, "long": min(short + log_uniform(rng, 1, 1000), 32000 // seqs + short), "nh": nh,
                "nkvh": nkvh, "dh": dh, "dtype": rng.choice(["f16", "bf16"]), "page": rng.choice([8, 16, 32, 64, 128]), "pad": rng.choice([0, 0, rng.randint(1, 9)])}
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    dh = rng.choice([dh, dh, 32, 80, 96, 192, 256])
    case = {"op": op, "tokens": log_uniform(rng, 1, 4000), "nh": nh, "nkvh": nkvh, "dh": dh, "rot": rng.choice([dh, dh, dh // 2]), "halves": rng.random() < 0.5,
            "dtype": dtype, "norm": rng.random() < 0.6}
    if op == "append":
        case |= {"seqs": rng.randint(1, min(40, case["tokens"])), "page": rng.choice([8, 16, 32, 64, 128]), "past": rng.randint(0, 500), "pad": rng.choice([0, 0, rng.randint(1, 20)])}
    return case


# ---------------------------------------------------------------------------------------------------------------------- inputs

def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, shape, dtype, std=1.0):
    """Normal values, drawn in the type itself: the largest caches are gigabytes in 32 bits."""
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def tables(n, rot):
    """sin and cos of position times frequency, [n, rot / 2] in 32 bits, angles in 64."""
    f = 5e5 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * f
    return a.sin().float(), a.cos().float()


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def prepare(case, seed):
    g, r = generator(seed), np.random.default_rng(seed)
    s = {"case": case}
    op = case["op"]
    dt = TYPES[case["dtype"]]
    if op in ("norm_rope", "append"):
        n, nh, nkvh, dh = case["tokens"], case["nh"], case["nkvh"], case["dh"]
        all_n = n + case.get("pad", 0)
        qkv = normal(g, (all_n, (nh + 2 * nkvh) * dh), dt)  # as a fused projection leaves them
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, dh)) for x in qkv.split([nh * dh, nkvh * dh, nkvh * dh], dim=1))
        s["q_out"] = torch.zeros(all_n, nh, dh, dtype=dt, device=DEV)
        s["q_w"], s["k_w"] = ((1 + 0.1 * normal(g, (dh,), torch.float32)).to(dt) for _ in range(2)) if case["norm"] else (None, None)
        if op == "norm_rope":
            s["k_out"] = torch.zeros(n, nkvh, dh, dtype=dt, device=DEV)
            pos = r.integers(0, 10) + np.arange(n)
        else:
            seqs, page = case["seqs"], case["page"]
            seq = np.arange(n) * seqs // n
            first = np.searchsorted(seq, seq)  # a sequence's first token of the round
            pos = r.integers(0, case["past"] + 1, seqs)[seq] + np.arange(n) - first
            per = (case["past"] + n // seqs) // page + 1
            s["table"] = i32(r.permutation(seqs * per).reshape(seqs, per))
            s["pool"] = torch.zeros(seqs * per, 2, nkvh, page, dh, dtype=dt, device=DEV)
            s["tok_seq"] = i32(np.concatenate([seq, np.full(case["pad"], -1)]))
            pos = np.concatenate([pos, np.zeros(case["pad"], pos.dtype)])
        s["pos"] = i32(pos)
        s["sin"], s["cos"] = tables(int(pos.max()) + 1, case["rot"])
    elif op == "prefix":
        seqs, new, page, nkvh, dh = case["seqs"], case["new"], case["page"], case["nkvh"], case["dh"]
        lens = r.integers(case["short"], case["long"] + 1, seqs)
        lens = np.maximum(lens, new)
        shared, per = -(-case["prefix"] // page), -(-int(lens.max()) // page)
        ids = r.permutation(shared + seqs * per + 3)
        s["prefix_table"], s["table"] = i32(ids[:shared]), i32(ids[shared:shared + seqs * per].reshape(seqs, per))
        s["pool"] = normal(g, (len(ids), 2, nkvh, page, dh), dt)
        pad = case["pad"]
        n = seqs * new + pad
        s["tok_seq"] = i32(np.concatenate([np.repeat(np.arange(seqs), new), np.full(pad, -1)]))
        s["tok_ctx"] = i32(np.concatenate([(lens[:, None] - new + 1 + np.arange(new)).reshape(-1), np.zeros(pad)]))
        s["q"] = normal(g, (n, case["nh"], dh), dt, 1.5)  # scores with a spread of 1.5
        s["o"] = torch.zeros(n, case["nh"], dh, dtype=dt, device=DEV)
    elif op == "softmax":
        s["logits"] = normal(g, (case["rows"], case["vocab"]), dt, 2.5)
        s["temperature"] = torch.from_numpy(r.choice(np.float32([0.0, 0.7, 0.8, 1.0, 1.3]), case["rows"], p=[0.1, 0.2, 0.3, 0.3, 0.1])).to(DEV)
        s["probs"] = torch.zeros(case["rows"], case["vocab"], dtype=torch.float32, device=DEV)
    else:
        seqs, k, vocab = case["seqs"], case["k"], case["vocab"]
        lg = normal(g, (seqs, k + 1, vocab), torch.float32, 2.5)
        s["target"] = torch.softmax(lg, -1).to(dt)
        near = lg[:, :k] + normal(g, (seqs, k, vocab), torch.float32, 0.7)  # a smaller model that mostly agrees
        if k:
            gumbel = -torch.log(-torch.log(torch.rand(seqs, k, vocab, device=DEV, generator=g).clamp_(1e-12, 1 - 1e-7)))
            s["drafted"] = (near + gumbel).argmax(-1).int() if case["drafts"] == "sampled" else near.argmax(-1).int()
        else:
            s["drafted"] = torch.zeros(seqs, 0, dtype=torch.int32, device=DEV)
        s["draft"] = torch.softmax(near, -1).to(dt) if case["drafts"] == "sampled" else None
        s["n_drafted"] = i32(r.integers(max(0, k - 1), k + 1, seqs))
        s["randoms"] = torch.from_numpy(r.random((seqs, k + 1), dtype=np.float32)).to(DEV)
        s["accepted"] = torch.zeros(seqs, dtype=torch.int32, device=DEV)
        s["tokens"] = torch.zeros(seqs, k + 1, dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------------------------- the plain form

def rotated(x, w, pos, sin, cos, rot, halves):
    """Rows [n, heads, dh]: divided by their root mean square and weighed (where there are weights), the first `rot` values rotated."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
    sn, cs = sin[pos.long()][:, None], cos[pos.long()][:, None]
    t = y[..., :rot]
    a, b = (t[..., :rot // 2], t[..., rot // 2:]) if halves else (t[..., 0::2], t[..., 1::2])
    u, v = a * cs - b * sn, a * sn + b * cs
    t = torch.cat([u, v], -1) if halves else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([t, y[..., rot:]], -1).to(x.dtype)


def plain_norm_rope(s):
    c = s["case"]
    args = s["pos"], s["sin"], s["cos"], c["rot"], c["halves"]
    s["q_out"][:] = rotated(s["q"], s["q_w"], *args)
    s["k_out"][:] = rotated(s["k"], s["k_w"], *args)
    return s["q_out"], s["k_out"]


def plain_append(s):
    c = s["case"]
    n = c["tokens"]
    pos = s["pos"][:n]
    args = pos, s["sin"], s["cos"], c["rot"], c["halves"]
    s["q_out"][:n] = rotated(s["q"][:n], s["q_w"], *args)
    page = s["table"][s["tok_seq"][:n].long(), (pos // c["page"]).long()].long()
    place = (pos % c["page"]).long()
    s["pool"][page, 0, :, place] = rotated(s["k"][:n], s["k_w"], *args)
    s["pool"][page, 1, :, place] = s["v"][:n]
    return s["pool"], s["q_out"]


def plain_prefix(s):
    c = s["case"]
    n, nkvh, dh, g = c["seqs"] * c["new"], c["nkvh"], c["dh"], c["nh"] // c["nkvh"]
    shared = s["pool"][s["prefix_table"].long()].transpose(0, 1).transpose(1, 2).flatten(2, 3)[:, :, :c["prefix"]].float()  # [k|v][head][prefix][dh]
    mine = s["pool"][s["table"].long()].permute(2, 0, 3, 1, 4, 5).flatten(3, 4).float()  # [k|v][seq][head][position][dh]
    q = s["q"][:n].view(c["seqs"], c["new"], nkvh, g, dh).permute(0, 2, 1, 3, 4).flatten(2, 3).float()  # [seq][head][token, group][dh]
    far = torch.einsum("shrd,hpd->shrp", q, shared[0])
    near = torch.einsum("shrd,shpd->shrp", q, mine[0])
    seen = torch.arange(near.shape[-1], device=DEV) < s["tok_ctx"][:n].view(c["seqs"], 1, c["new"], 1, 1)
    near = near.masked_fill(~seen.expand(-1, 1, -1, g, -1).flatten(2, 3), -math.inf)
    x = torch.cat([far, near], -1) / math.sqrt(dh)
    del far, near
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.einsum("shrp,hpd->shrd", x[..., :c["prefix"]], shared[1]) + torch.einsum("shrp,shpd->shrd", x[..., c["prefix"]:], mine[1])
    s["o"][:n] = o.unflatten(2, (c["new"], g)).permute(0, 2, 1, 3, 4).reshape(n, c["nh"], dh).to(s["o"].dtype)
    return s["o"]


def plain_softmax(s):
    x = s["logits"].float()
    t = s["temperature"][:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / torch.where(t == 0, torch.ones_like(t), t))
    at = torch.arange(x.shape[1], device=DEV)
    lowest = torch.where(x == top, at, x.shape[1]).amin(-1, keepdim=True)
    s["probs"][:] = torch.where(t == 0, (at == lowest).float(), e / e.sum(-1, keepdim=True))
    return s["probs"]


def plain_verify(s):
    c = s["case"]
    seqs, k, vocab = c["seqs"], c["k"], c["vocab"]
    p, drafted, u = s["target"], s["drafted"].long(), s["randoms"].double()
    px = p[:, :k].gather(2, drafted[..., None])[..., 0].double()
    qx = s["draft"].gather(2, drafted[..., None])[..., 0].double() if s["draft"] is not None else torch.ones_like(px)
    fine = (u[:, :k] * qx < px) & (torch.arange(k, device=DEV) < s["n_drafted"][:, None])
    n = fine.long().cumprod(-1).sum(-1)
    row = torch.arange(seqs, device=DEV)
    last = p[row, n].double()
    held = n < s["n_drafted"]  # a draft was rejected: its probability comes off
    if k:
        at = n.clamp(max=k - 1)
        if s["draft"] is not None:
            off = s["draft"][row, at].double()
        else:
            off = torch.zeros_like(last).scatter_(1, drafted[row, at][:, None], 1.0)
        rest = (last - off).clamp_min(0)
        last = torch.where((held & (rest.sum(-1) > 0))[:, None], rest, last)
    run = last.cumsum(-1)
    x = torch.searchsorted(run, u[:, k:] * run[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
    at = torch.arange(k + 1, device=DEV)
    more = torch.cat([drafted, drafted.new_zeros(seqs, 1)], 1)
    s["accepted"][:] = n
    s["tokens"][:] = torch.where(at < n[:, None], more, torch.where(at == n[:, None], x[:, None], -1))
    return s["accepted"], s["tokens"]


# ------------------------------------------------------------------------------------------------------------- the framework's operators

def library(s):
    """The binding, its library and the current stream; a state keeps what a program keeps: descriptions of its cache and a workspace."""
    import llama_cu_b200 as L
    return L, L.load_library(), L.stream_ptr()


def described(L, s):
    if "prep" not in s:
        c = s["case"]
        if "sin" in s:
            s["prep"] = L.QkPrep(L.ptr(s["q_w"]), L.ptr(s["k_w"]), s["sin"].data_ptr(), s["cos"].data_ptr(), CODES[c["dtype"]], EPS, s["sin"].shape[0], c["rot"],
                                 int(c["halves"]))
        if "pool" in s:
            pool = s["pool"]
            st = pool.stride()
            s["pages"] = L.KvPages(pool.data_ptr(), pool[:, 1].data_ptr(), st[0], st[3], st[2], pool.shape[0], pool.shape[3])
        s.setdefault("prep", None)
    return s["prep"], s.get("pages")


def own_norm_rope(s):
    L, lib, stream = library(s)
    c, (prep, _) = s["case"], described(L, s)
    q, k, qo, ko, dh = s["q"], s["k"], s["q_out"], s["k_out"], c["dh"]
    L.check(lib.lcu_op_qk_norm_rope(qo.data_ptr(), c["nh"] * dh, dh, q.data_ptr(), q.stride(0), dh, ko.data_ptr(), c["nkvh"] * dh, dh, k.data_ptr(), k.stride(0), dh,
                                    s["pos"].data_ptr(), prep, c["tokens"], c["nh"], c["nkvh"], dh, CODES[c["dtype"]], stream))
    return qo, ko


def own_append(s):
    L, lib, stream = library(s)
    c, (prep, pages) = s["case"], described(L, s)
    q, k, v, qo, dh = s["q"], s["k"], s["v"], s["q_out"], c["dh"]
    L.check(lib.lcu_op_kv_append(pages, s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["tok_seq"].data_ptr(), s["pos"].data_ptr(), k.data_ptr(), k.stride(0), dh,
                                 v.data_ptr(), v.stride(0), dh, qo.data_ptr(), c["nh"] * dh, dh, q.data_ptr(), q.stride(0), dh, s["pos"].data_ptr(), prep, q.shape[0],
                                 c["nh"], c["nkvh"], dh, CODES[c["dtype"]], stream))
    return s["pool"], qo


def own_prefix(s):
    L, lib, stream = library(s)
    c, (_, pages) = s["case"], described(L, s)
    n, nh, nkvh, dh = s["q"].shape[0], c["nh"], c["nkvh"], c["dh"]
    if "workspace" not in s:
        s["workspace"] = torch.empty(lib.lcu_attention_prefix_workspace_size(n, nh, nkvh, dh, c["prefix"]), dtype=torch.uint8, device=DEV)
    ws = s["workspace"]
    L.check(lib.lcu_op_attention_prefix(s["o"].data_ptr(), nh * dh, dh, s["q"].data_ptr(), nh * dh, dh, pages, s["prefix_table"].data_ptr(), c["prefix"],
                                        s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["tok_seq"].data_ptr(), s["tok_ctx"].data_ptr(), n, nh, nkvh, dh,
                                        1.0 / math.sqrt(dh), CODES[c["dtype"]], ws.data_ptr(), ws.numel(), stream))
    return s["o"]


def own_softmax(s):
    L, lib, stream = library(s)
    x = s["logits"]
    L.check(lib.lcu_op_softmax_rows(s["probs"].data_ptr(), x.shape[1], x.data_ptr(), x.shape[1], s["temperature"].data_ptr(), x.shape[0], x.shape[1],
                                    CODES[s["case"]["dtype"]], stream))
    return s["probs"]


def own_verify(s):
    L, lib, stream = library(s)
    c = s["case"]
    L.check(lib.lcu_op_verify_drafts(s["accepted"].data_ptr(), s["tokens"].data_ptr(), s["target"].data_ptr(), c["vocab"], L.ptr(s["draft"]), c["vocab"],
                                     s["drafted"].data_ptr(), s["n_drafted"].data_ptr(), s["randoms"].data_ptr(), c["seqs"], c["k"], c["vocab"], CODES[c["dtype"]], stream))
    return s["accepted"], s["tokens"]


PLAIN = {"norm_rope": plain_norm_rope, "append": plain_append, "prefix": plain_prefix, "softmax": plain_softmax, "verify": plain_verify}
OWN = {"norm_rope": own_norm_rope, "append": own_append, "prefix": own_prefix, "softmax": own_softmax, "verify": own_verify}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------------- work and 64-bit values

def work(case):
    op, e = case["op"], 4 if case["dtype"] == "f32" else 2
    if op in ("norm_rope", "append"):
        rows = case["nh"] + (2 if op == "append" else 1) * case["nkvh"]
        n, turned = case["tokens"], case["nh"] + case["nkvh"]
        return {"bytes": n * (2 * rows * case["dh"] * e + 4 * case["rot"] + 4), "flops": n * turned * (4 * case["dh"] * case["norm"] + 3 * case["rot"])}
    if op == "prefix":
        tokens, row = case["seqs"] * case["new"], case["nkvh"] * case["dh"] * e
        own_len = max((case["short"] + case["long"]) / 2, case["new"])
        keys = case["prefix"] + case["seqs"] * own_len
        seen = tokens * (case["prefix"] + own_len - (case["new"] - 1) / 2)
        return {"bytes": 2 * keys * row + 2 * tokens * case["nh"] * case["dh"] * e, "flops": 4 * case["nh"] * case["dh"] * seen}
    if op == "softmax":
        return {"bytes": case["rows"] * case["vocab"] * (e + 4), "flops": 4 * case["rows"] * case["vocab"]}
    rows = 2 if case["drafts"] == "sampled" and case["k"] else 1  # of a sequence: the target's and the draft's, where a draft was rejected
    return {"bytes": case["seqs"] * (rows * case["vocab"] * e + 40 * case["k"]), "flops": 2 * case["seqs"] * rows * case["vocab"]}


def exact_rows(x, w, pos, sin, cos, rot, halves):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
    at = torch.arange(rot // 2, device=y.device)
    i, j = (at, at + rot // 2) if halves else (2 * at, 2 * at + 1)
    turn = torch.complex(cos.double(), sin.double())[pos.long()][:, None]
    z = torch.complex(y[..., i], y[..., j]) * turn
    out = y.clone()
    out[..., i], out[..., j] = z.real, z.imag
    return out


def exact_prefix(case, s):
    """One sequence and one key/value head at a time, keys in the order of their positions."""
    new, prefix, page, dh, group = case["new"], case["prefix"], case["page"], case["dh"], case["nh"] // case["nkvh"]
    out = torch.zeros(s["o"].shape, dtype=torch.float64, device=DEV)
    pool, shared, table, ctx = s["pool"], s["prefix_table"].tolist(), s["table"].tolist(), s["tok_ctx"].tolist()
    for h in range(case["nkvh"]):
        heads = slice(h * group, (h + 1) * group)
        common = pool[shared, :, h].double()  # [page][k|v][token][dh]
        key, value = (common[:, i].reshape(-1, dh)[:prefix] for i in (0, 1))
        for b in range(case["seqs"]):
            tokens = slice(b * new, (b + 1) * new)
            most = max(ctx[tokens])
            mine = pool[table[b][:-(-most // page)], :, h].double()
            k, v = (mine[:, i].reshape(-1, dh)[:most] for i in (0, 1))
            q = s["q"][tokens, heads].double() * dh ** -0.5
            hide = torch.arange(most, device=DEV)[None, :] >= torch.tensor(ctx[tokens], device=DEV)[:, None]
            score = torch.cat([q @ key.T, (q @ k.T).masked_fill(hide[:, None], -math.inf)], -1)
            weight = (score - score.max(-1, keepdim=True).values).exp()
            out[tokens, heads] = (weight[..., :prefix] @ value + weight[..., prefix:] @ v) / weight.sum(-1, keepdim=True)
    return out


def exact_verify(s):
    """A sequence at a time, on the host."""
    target, drafted, n_drafted, randoms = (s[x].cpu().numpy() for x in ("target64", "drafted", "n_drafted", "randoms"))
    draft = s["draft64"].cpu().numpy() if s["draft"] is not None else None
    accepted, tokens = np.zeros(len(target), np.int32), np.full(s["tokens"].shape, -1, np.int32)
    for b in range(len(target)):
        u = randoms[b].astype(np.float64)
        i = 0
        while i < n_drafted[b]:
            x = drafted[b, i]
            q = draft[b, i] if draft is not None else np.eye(1, target.shape[2], x)[0]
            if not u[i] * q[x] < target[b, i, x]:
                break
            tokens[b, i] = x
            i += 1
        w = target[b, i]
        if i < n_drafted[b] and np.maximum(w - q, 0).sum() > 0:
            w = np.maximum(w - q, 0)
        run = np.cumsum(w)
        accepted[b], tokens[b, i] = i, min(int(np.sum(run <= u[-1] * run[-1])), len(w) - 1)
    return accepted, tokens


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm_rope", "append"):
        n = case["tokens"]
        args = s["pos"][:n], s["sin"], s["cos"], case["rot"], case["halves"]
        q = torch.zeros(s["q_out"].shape, dtype=torch.float64, device=DEV)
        q[:n] = exact_rows(s["q"][:n], s["q_w"], *args)
        k = exact_rows(s["k"][:n], s["k_w"], *args)
        if op == "norm_rope":
            return q, k
        pool = torch.zeros(s["pool"].shape, dtype=torch.float64, device=DEV)
        where = np.asarray([s["table"].cpu().numpy()[b, p // case["page"]] for b, p in zip(s["tok_seq"][:n].tolist(), s["pos"][:n].tolist())])
        flat = pool.transpose(2, 3).flatten(0, 2)  # a copy: row (page, k|v, token)
        row = torch.from_numpy(where).to(DEV).long() * 2 * case["page"] + s["pos"][:n].long() % case["page"]
        flat[row], flat[row + case["page"]] = k, s["v"][:n].double()
        return flat.view(pool.shape[0], 2, case["page"], case["nkvh"], case["dh"]).transpose(2, 3), q
    if op == "prefix":
        return exact_prefix(case, s)
    if op == "softmax":
        x, t = s["logits"].double(), s["temperature"].double().tolist()
        out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for i, temperature in enumerate(t):
            if temperature:
                z = torch.exp(x[i] / temperature - x[i].max() / temperature)
                out[i] = z / z.sum()
            else:
                out[i] = 0
                out[i, int((x[i] == x[i].max()).nonzero()[0])] = 1
        return out
    s["target64"] = s["target"].double()
    s["draft64"] = s["draft"].double() if s["draft"] is not None else None
    return exact_verify(s)
