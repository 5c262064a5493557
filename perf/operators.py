"""The sliding-window and paged-cache operators, as they are measured.

Five kinds of call:

  swa     attention with a causal window and sinks (the first tokens, which
          stay visible to everybody): forward of a [B, n, H, d] batch
  train   the same with every gradient (dq, dk, dv)
  append  a ragged batch of new keys and values into the paged cache: QKNorm,
          rotation at each token's own position, page summaries
  paged   attention of new tokens over the paged cache: one token per
          sequence (decode) or several (chunked prefill), whole or windowed
  prefix  decode of a batch whose sequences share their first pages

Shapes: 14 query / 2 KV heads at head dim 64 and 28 / 4 at head dim 128, the
two donors of this framework, window 1024, 4 or 8 sinks, 64-token pages; drawn
cases also take other groups.  Inputs are N(0, 1); cached keys are N(0, 1)
times the QKNorm gain d ** 0.25, so that scores have a standard deviation of 1.
"""
import os
import sys

import numpy as np
import torch

own = False

PAGE, EPS = 64, 1e-6
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SMALL = dict(Hq=14, Hkv=2, d=64)
LARGE = dict(Hq=28, Hkv=4, d=128)


def _hba():
    path = os.path.abspath("hierarchical-block-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hba_amd

    return hba_amd


# -------------------------------------------------------------------- cases --
def listed():
    return [
        # a short chat turn through one window layer: latency
        dict(name="swa_1k", kind="swa", dtype="bf16", B=1, n=1001, W=1024, S=4, padded=False, **SMALL),
        # prefill of a window layer at the native context
        dict(name="swa_32k", kind="swa", dtype="bf16", B=1, n=32768, W=1024, S=4, padded=False, **SMALL),
        # evaluation of a padded batch in fp32, as the gates run
        dict(name="swa_2k_f32", kind="swa", dtype="f32", B=2, n=2047, W=512, S=4, padded=True, **SMALL),
        # a training step of the larger donor's window layer
        dict(name="train_8k_d128", kind="train", dtype="bf16", B=1, n=8192, W=1024, S=8, padded=False, **LARGE),
        # a training step of a small padded batch
        dict(name="train_2k", kind="train", dtype="bf16", B=3, n=1999, W=512, S=4, padded=True, **SMALL),
        # prompts arriving together, at odd places of their pages
        dict(name="append_prompts", kind="append", dtype="bf16", Bd=6, new_lo=700, new_hi=4000, old_lo=0, old_hi=9000,
             m=4, draws=1, **LARGE),
        # a few accepted tokens per sequence of a running batch
        dict(name="append_few", kind="append", dtype="bf16", Bd=48, new_lo=0, new_hi=6, old_lo=10, old_hi=6000, m=4,
             draws=2, **SMALL),
        # one token of one window layer for a running batch
        dict(name="decode_window", kind="paged", dtype="bf16", Bd=64, new_lo=1, new_hi=1, old_lo=100, old_hi=16000,
             W=1024, S=4, draws=3, **SMALL),
        # one token over the whole cache, long contexts
        dict(name="decode_all_d128", kind="paged", dtype="bf16", Bd=24, new_lo=1, new_hi=1, old_lo=4000, old_hi=32000,
             W=0, S=0, draws=4, **LARGE),
        # chunked prefill: the next part of four prompts over what the cache holds
        dict(name="chunk_512", kind="paged", dtype="bf16", Bd=4, new_lo=300, new_hi=512, old_lo=1000, old_hi=8000, W=0,
             S=0, draws=5, **SMALL),
        # a batch behind one system prompt
        dict(name="prefix_8k", kind="prefix", dtype="bf16", Bd=64, shared=8192, new_lo=1, new_hi=1, old_lo=1,
             old_hi=700, draws=6, **SMALL),
        # a few fp32 sequences behind a short prefix
        dict(name="prefix_1k_f32", kind="prefix", dtype="f32", Bd=9, shared=1024, new_lo=1, new_hi=1, old_lo=0,
             old_hi=200, draws=7, **LARGE),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["swa", "train", "append", "paged", "paged", "prefix"])
    Hq, Hkv, d = rng.choice([(14, 2, 64), (28, 4, 128), (8, 8, 64), (16, 2, 128), (6, 6, 128), (12, 4, 64)])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]), Hq=Hq, Hkv=Hkv, d=d)
    if kind in ("swa", "train"):
        B, W = rng.choice([1, 2, 3]), _log(rng, 40, 2000)
        room = 8192 * 1024 * 28 * 128 // 2 if kind == "train" else 32768 * 1024 * 14 * 64 // 2
        if c["dtype"] == "f32":
            room //= 8
        most = max(64, min(16384, room // (B * W * Hq * d)))
        c.update(B=B, n=_log(rng, 40, most), W=W, S=rng.choice([0, 1, 4, 8, 70]), padded=rng.random() < 0.3)
    elif kind == "append":
        hi = _log(rng, 2, 3000)
        c.update(Bd=max(1, min(64, rng.randint(1, 10000 // hi))), new_lo=hi // 3, new_hi=hi, old_lo=0,
                 old_hi=_log(rng, 50, 6000), m=rng.choice([1, 4, 8]), draws=rng.randrange(1000))
    elif kind == "paged":
        hi = rng.choice([1, 1, _log(rng, 2, 400)])
        W = rng.choice([0, _log(rng, 30, 3000)])
        old = _log(rng, 60, 16000)
        Bd = max(1, min(40, rng.randint(1, max(1, 24 * 18000 * 4 // (old * Hkv)))))
        if hi > 1:
            Bd = max(1, min(Bd, 4 * 512 * 8000 * 14 // (hi * old * Hq)))
        c.update(Bd=Bd, new_lo=1 if hi == 1 else 0, new_hi=hi, old_lo=old // 4, old_hi=old, W=W,
                 S=rng.choice([1, 4, 70]) if W else 0, draws=rng.randrange(1000))
    else:
        c.update(Bd=_log(rng, 2, 60), shared=64 * _log(rng, 2, 100), new_lo=1, new_hi=1, old_lo=0,
                 old_hi=_log(rng, 20, 600), draws=rng.randrange(1000))
    return c


def _spread(lo, hi, count, draws):
    """`count` lengths of lo .. hi, both ends among them where there are two or more."""
    r = np.random.RandomState(draws)
    x = r.randint(lo, hi + 1, size=count)
    if count > 1:
        x[0], x[-1] = hi, lo
    return [int(v) for v in x]


def _lens(c):
    """Padded batches: the rows of each sequence, the first one whole."""
    return [max(1, c["n"] * (b + 2) // (2 * b + 2)) for b in range(c["B"])] if c["padded"] else [c["n"]] * c["B"]


def _ragged(c):
    """(tokens already there, new tokens) of each sequence; a shared prefix counts as there."""
    old = _spread(c["old_lo"], c["old_hi"], c["Bd"], c["draws"])
    new = _spread(c["new_lo"], c["new_hi"], c["Bd"], c["draws"] + 1)
    if sum(new) == 0:
        new[0] = 1
    return [x + c.get("shared", 0) for x in old], new


# ------------------------------------------------------------------- inputs --
def _key_off(d, dev):
    """Place of element t of token j within a key page, [64, d]."""
    j, t = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    tile, row = 2 * (j // 32) + j // 4 % 2, 4 * (j % 32 // 8) + j % 4
    return ((tile * (d // 32) + t // 32) * 64 + row + 16 * (t % 32 // 8)) * 8 + t % 8


def _val_off(d, dev):
    """Place of element t of token j within a value page, [64, d]."""
    j, t = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    return ((t // 16 * 2 + j // 32) * 64 + t % 16 + 16 * (j % 32 // 8)) * 8 + j % 8


def _tables(n, d, dev):
    ang = torch.outer(torch.arange(n, device=dev).double(),
                      1.0 / (1e6 ** (torch.arange(0, d, 2, device=dev).double() / d)))
    ang = torch.cat((ang, ang), -1)
    return ang.cos().float(), ang.sin().float()


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, d, Hq, Hkv = DT[c["dtype"]], c["d"], c["Hq"], c["Hkv"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    if c["kind"] in ("swa", "train"):
        B, n = c["B"], c["n"]
        s = dict(c=c, q=randn(B, n, Hq, d), k=randn(B, n, Hkv, d), v=randn(B, n, Hkv, d),
                 lens=_i32(_lens(c), dev) if c["padded"] else None)
        if c["kind"] == "train":
            s["dout"] = randn(B, n, Hq, d)
            if c["padded"]:   # nothing flows into padding
                s["dout"] *= (torch.arange(n, device=dev)[None] < s["lens"][:, None])[:, :, None, None]
        return s

    old, new = _ragged(c)
    L = [a + b for a, b in zip(old, new)]
    Bd, shared = c["Bd"], c.get("shared", 0) // PAGE
    mp = max(1, max((x + PAGE - 1) // PAGE for x in L))
    P = shared + Bd * (mp - shared) + 3
    phys = torch.randperm(P, generator=g, device=dev).int()
    table = torch.cat([phys[:shared].expand(Bd, shared), phys[shared:shared + Bd * (mp - shared)].view(Bd, -1)], 1)
    cos, sin = _tables(mp * PAGE, d, dev)
    gain = torch.full((max(Hq, Hkv),), d ** 0.25, device=dev)
    gain *= 1 + 0.1 * torch.randn(gain.shape, generator=g, device=dev)
    s = dict(c=c, table=table.contiguous(), seq_lens=_i32(L, dev), cos=cos, sin=sin, max_len=max(L),
             cu=_i32(np.cumsum([0] + new).tolist(), dev))
    T = sum(new)
    if c["kind"] == "append":
        m = c["m"]
        kv = randn(T, 2, Hkv, d)   # one projection's output: k and v are views of it
        s.update(k=kv[:, 0], v=kv[:, 1], gain=gain[:Hkv].contiguous(), probes=randn(Hkv, m, d).float() * d ** -0.5,
                 proj=torch.eye(d, device=dev) + 0.02 * torch.randn(Hkv, d, d, generator=g, device=dev))
        for name in ("kc", "kr", "vp"):
            s[name] = randn(P, Hkv, PAGE * d)
        s["summ"] = randn(P, Hkv, m, d)
        # what the plain form's program plans on the host: each token's sequence and
        # position, and the pages that this batch fills
        s["seq"] = torch.tensor(np.repeat(np.arange(Bd), new), device=dev)
        s["pos"] = torch.tensor(np.concatenate([np.arange(a, a + b) for a, b in zip(old, new)]), device=dev)
        full = [(i, p) for i, (a, b) in enumerate(zip(old, L)) for p in range(a // PAGE, b // PAGE)]
        s["full"] = torch.tensor(full, dtype=torch.long, device=dev).view(-1, 2)
        return s
    s.update(q=randn(T, Hq, d), gain=gain[:Hq].contiguous(), kr=randn(P, Hkv, PAGE * d) * d ** 0.25,
             vp=randn(P, Hkv, PAGE * d), scales=1.0 / d + torch.rand(Bd, generator=g, device=dev) * 0.1 / d)
    s["kr"] = s["kr"].to(dt)
    # each token's sequence and position: the plain form's program plans them on the host
    s["seq"] = torch.tensor(np.repeat(np.arange(Bd), new), device=dev)
    s["pos"] = torch.tensor(np.concatenate([np.arange(a, a + b) for a, b in zip(old, new)]), device=dev)
    s["most"] = max(new)
    return s


# --------------------------------------------------------------- plain forms --
def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_swa(q, k, v, W, S, lens):
    """Blocks of W queries against their own block of keys and the one before, and the sinks."""
    B, n, Hq, d = q.shape
    Hkv = k.shape[2]
    G, dev = Hq // Hkv, q.device
    c = min(W, n)
    nb = -(-n // c)
    pad = nb * c - n

    def heads(x, width):   # [B, n, Hkv * width, d] -> [B, Hkv, nb, width * c, d]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, pad)).view(B, nb, c, Hkv, width, d)
        return x.permute(0, 3, 1, 4, 2, 5).reshape(B, Hkv, nb, width * c, d)

    def two(x):            # each block behind the one before it
        return torch.cat((torch.cat((torch.zeros_like(x[:, :, :1]), x[:, :, :-1]), 2), x), 3)

    qb, kb, vb = heads(q, G), heads(k, 1), heads(v, 1)
    kw, vw = two(kb), two(vb)
    i = (torch.arange(nb, device=dev)[:, None] * c + torch.arange(c, device=dev)[None])[:, :, None]
    j = (torch.arange(nb, device=dev)[:, None] * c + torch.arange(-c, c, device=dev)[None])[:, None, :]
    near = (j >= 0) & (j <= i) & (j > i - W)
    s = (qb @ kw.transpose(-1, -2) * d ** -0.5).view(B, Hkv, nb, G, c, 2 * c)
    s = s.masked_fill(~near[:, None], float("-inf"))
    ns = min(S, n)
    ks, vs = k[:, :ns].float().permute(0, 2, 1, 3)[:, :, None], v[:, :ns].float().permute(0, 2, 1, 3)[:, :, None]
    far = torch.arange(ns, device=dev) <= i - W
    t = (qb @ ks.transpose(-1, -2) * d ** -0.5).view(B, Hkv, nb, G, c, ns)
    t = t.masked_fill(~far[:, None], float("-inf"))
    p = _softmax(torch.cat((s, t), -1)).reshape(B, Hkv, nb, G * c, 2 * c + ns)
    o = p[..., : 2 * c] @ vw + p[..., 2 * c:] @ vs
    o = o.view(B, Hkv, nb, G, c, d).permute(0, 2, 4, 1, 3, 5).reshape(B, nb * c, Hq, d)[:, :n]
    if lens is not None:
        o = o.masked_fill((torch.arange(n, device=dev)[None] >= lens[:, None])[:, :, None, None], 0.0)
    return o.to(q.dtype)


def _norm(x, gain):
    x = x.float()
    return x / x.square().mean(-1, keepdim=True).clamp_min(EPS).sqrt() * gain[:, None]


def _rotate(x, cos, sin, pos):
    h = x.shape[-1] // 2
    return x * cos[pos][:, None] + torch.cat((-x[..., h:], x[..., :h]), -1) * sin[pos][:, None]


def _plain_append(s):
    c, dev = s["c"], s["k"].device
    d, Hkv = c["d"], c["Hkv"]
    kc = _norm(s["k"], s["gain"])
    kr = _rotate(kc, s["cos"], s["sin"], s["pos"])
    page, slot = s["table"].long()[s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    at = (page[:, None] * Hkv + torch.arange(Hkv, device=dev))[..., None] * (PAGE * d)
    for name, x, off in (("kc", kc, _key_off(d, dev)), ("kr", kr, _key_off(d, dev)), ("vp", s["v"], _val_off(d, dev))):
        s[name].view(-1)[at + off[slot][:, None]] = x.to(s[name].dtype)
    full = s["table"].long()[s["full"][:, 0], s["full"][:, 1]]
    rows = s["kc"][full][..., _key_off(d, dev)].float()                  # [pages, Hkv, 64, d]
    att = _softmax(s["probes"][None] @ rows.transpose(-1, -2) * d ** -0.5)
    s["summ"][full] = (att @ rows @ s["proj"]).to(s["summ"].dtype)
    return s["kc"], s["kr"], s["vp"], s["summ"]


def _rows(s, pages):
    """Keys and values of a list of pages [..., n] as fp32 rows [..., Hkv, 64 n, d]."""
    d, dev = s["c"]["d"], s["kr"].device
    got = []
    for x, off in ((s["kr"], _key_off(d, dev)), (s["vp"], _val_off(d, dev))):
        x = x[pages].index_select(-1, off.view(-1)).float().unflatten(-1, (PAGE, d)).transpose(-4, -3)
        got.append(x.flatten(-3, -2))
    return got


def _plain_paged(s):
    c, dev = s["c"], s["q"].device
    Hq, Hkv, d, W, S, most = c["Hq"], c["Hkv"], c["d"], c["W"], c["S"], s["most"]
    Bd, G, mp = c["Bd"], Hq // Hkv, s["table"].shape[1]
    q = _rotate(_norm(s["q"], s["gain"]), s["cos"], s["sin"], s["pos"]) * s["scales"][s["seq"]][:, None, None]
    L = s["seq_lens"].long()
    first = L - (s["cu"][1:] - s["cu"][:-1])                             # position of the first new token
    if W:
        ns = -(-S // PAGE)
        w0 = (first - W + 1).clamp_min(0) // PAGE
        nw = min(mp, (W + most) // PAGE + 2)
        logical = torch.cat((torch.arange(ns, device=dev).expand(Bd, ns),
                             torch.maximum(w0, torch.tensor(ns, device=dev))[:, None]
                             + torch.arange(nw, device=dev)), 1)
    else:
        logical = torch.arange(mp, device=dev).expand(Bd, mp)
    k, v = _rows(s, s["table"].long().gather(1, logical.clamp_max(mp - 1)))
    j = (logical[:, :, None] * PAGE + torch.arange(PAGE, device=dev)).flatten(1)
    slot = torch.arange(len(s["seq"]), device=dev) - s["cu"][:-1].long()[s["seq"]]
    qp = torch.zeros(Bd, most, Hkv, G, d, device=dev)
    qp[s["seq"], slot] = q.view(-1, Hkv, G, d)
    i = first[:, None] + torch.arange(most, device=dev)
    seen = (j[:, None] <= i[:, :, None]) & (j < L[:, None])[:, None]
    if W:
        seen &= (j[:, None] > i[:, :, None] - W) | (j < S)[:, None]
    qp = qp.permute(0, 2, 1, 3, 4).reshape(Bd, Hkv, most * G, d)
    sc = (qp @ k.transpose(-1, -2)).view(Bd, Hkv, most, G, -1).masked_fill(~seen[:, None, :, None], float("-inf"))
    v = v.masked_fill((j >= L[:, None])[:, None, :, None], 0.0)
    o = (_softmax(sc).view(Bd, Hkv, most * G, -1) @ v).view(Bd, Hkv, most, G, d).permute(0, 2, 1, 3, 4)
    return o[s["seq"], slot].reshape(-1, Hq, d).to(s["q"].dtype)


def _plain_prefix(s):
    c, dev = s["c"], s["q"].device
    Hq, Hkv, d, Bd, n = c["Hq"], c["Hkv"], c["d"], c["Bd"], c["shared"]
    G, table = Hq // Hkv, s["table"].long()
    q = _rotate(_norm(s["q"], s["gain"]), s["cos"], s["sin"], s["pos"]) * s["scales"][:, None, None]
    q = q.view(Bd, Hkv, G, d)
    kp, vp = _rows(s, table[0, : n // PAGE])                             # the prefix, once
    ks, vs = _rows(s, table[:, n // PAGE:])
    j = n + torch.arange(ks.shape[2], device=dev)
    seen = j < s["seq_lens"][:, None]
    a = (q.transpose(0, 1).reshape(Hkv, Bd * G, d) @ kp.transpose(-1, -2)).view(Hkv, Bd, G, n).transpose(0, 1)
    b = (q @ ks.transpose(-1, -2)).masked_fill(~seen[:, None, None], float("-inf"))
    p = _softmax(torch.cat((a, b), -1))
    o = (p[..., :n].transpose(0, 1).reshape(Hkv, Bd * G, n) @ vp).view(Hkv, Bd, G, d).transpose(0, 1)
    o = o + p[..., n:] @ vs.masked_fill(~seen[:, None, :, None], 0.0)
    return o.reshape(Bd, Hq, d).to(s["q"].dtype)


def run(state):
    s = state
    c = s["c"]
    kind = c["kind"]
    if kind in ("swa", "train"):
        if kind == "swa":
            if own:
                return _hba().sliding_attention(s["q"], s["k"], s["v"], c["W"], sinks=c["S"], lens=s["lens"])
            return _plain_swa(s["q"], s["k"], s["v"], c["W"], c["S"], s["lens"])
        q, k, v = (s[x].detach().requires_grad_() for x in "qkv")
        if own:
            o = _hba().sliding_attention(q, k, v, c["W"], sinks=c["S"], lens=s["lens"])
        else:
            o = _plain_swa(q, k, v, c["W"], c["S"], s["lens"])
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), s["dout"]))
    if kind == "append":
        if not own:
            return _plain_append(s)
        _hba().ops.kv_append_ragged(s["k"], s["v"], s["cu"], s["gain"], EPS, s["cos"], s["sin"], s["table"],
                                    s["seq_lens"], s["kc"], s["kr"], s["vp"], s["probes"], s["proj"], s["summ"])
        return s["kc"], s["kr"], s["vp"], s["summ"]
    if not own:
        return _plain_paged(s) if kind == "paged" else _plain_prefix(s)
    return _hba().ops.paged_attn(s["q"], s["gain"], EPS, s["kr"], s["vp"], s["table"], s["seq_lens"], s["cos"],
                                 s["sin"], s["scales"], s["max_len"], window=c.get("W", 0), sinks=c.get("S", 0),
                                 cu=s["cu"] if c["new_hi"] > 1 else None, shared=c.get("shared", 0))


# ---------------------------------------------------------------------- work --
def _pairs(lo, hi, W, S):
    """Visible (query, key) pairs of query positions lo .. hi - 1."""
    i = np.arange(lo, hi, dtype=np.int64)
    if not W:
        return int((i + 1).sum())
    return int((np.minimum(i + 1, W) + np.clip(i + 1 - W, 0, S)).sum())


def work(case):
    c = case
    e, d, Hq, Hkv = 2 if c["dtype"] == "bf16" else 4, c["d"], c["Hq"], c["Hkv"]
    if c["kind"] in ("swa", "train"):
        rows = sum(_lens(c))
        pairs = sum(_pairs(0, x, c["W"], c["S"]) for x in _lens(c)) * Hq
        fwd = e * d * rows * 2 * (Hq + Hkv)                              # q, k, v read, out written
        if c["kind"] == "swa":
            return {"bytes": fwd, "flops": 4 * d * pairs}
        return {"bytes": fwd + e * d * rows * 2 * (Hq + Hkv), "flops": 14 * d * pairs}   # dout; dq, dk, dv
    old, new = _ragged(c)
    T, L = sum(new), [a + b for a, b in zip(old, new)]
    if c["kind"] == "append":
        full = sum(b // PAGE - a // PAGE for a, b in zip(old, L)) * Hkv
        part = sum(a % PAGE for a, b in zip(old, L) if b // PAGE > a // PAGE) * Hkv   # read back for a summary
        m = c["m"]
        return {"bytes": e * d * (5 * T * Hkv + part + full * m) + T * d * 8 + Hkv * (m + d) * d * 4,
                "flops": 10 * T * Hkv * d + full * m * d * (4 * PAGE + 2 * d)}
    W, S, shared = c.get("W", 0), c.get("S", 0), c.get("shared", 0)
    pairs = sum(_pairs(a, b, W, S) for a, b in zip(old, L)) * Hq
    keys = 0
    for a, b in zip(old, L):
        if not b > a:
            continue
        w0 = max(0, a - W + 1) if W else 0
        keys += b - w0 + min(S, w0) - (shared if c["kind"] == "prefix" else 0)
    return {"bytes": e * d * (2 * Hkv * (keys + shared) + 2 * T * Hq), "flops": 4 * d * pairs}


# --------------------------------------------------------------------- exact --
def _exact_rows(q, k, v, i, j, S, W, scale, dout=None):
    """Attention of query rows at positions i to key rows at positions j (one KV
    head; q [rows, G, d]) in 64 bits; with dout also dq, dk, dv."""
    vis = j[None] <= i[:, None]
    if W:
        vis = vis & ((j[None] > i[:, None] - W) | (j[None] < S))
    x = torch.einsum("rgd,kd->grk", q, k) * scale
    x = torch.where(vis, x, torch.full_like(x, -np.inf))
    p = torch.softmax(x, -1)
    o = torch.einsum("grk,kd->rgd", p, v)
    if dout is None:
        return o
    dv = torch.einsum("grk,rgd->kd", p, dout)
    dp = torch.einsum("rgd,kd->grk", dout, v)
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
    return o, torch.einsum("grk,kd->rgd", ds, k), torch.einsum("grk,rgd->kd", ds, q), dv


def _exact_swa(s):
    c = s["c"]
    G, d = c["Hq"] // c["Hkv"], c["d"]
    q, k, v = (s[x].double() for x in "qkv")
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if c["kind"] == "train" else None
    for b, n in enumerate(_lens(c)):
        for h in range(c["Hkv"]):
            hs = slice(h * G, h * G + G)
            for r0 in range(0, n, 512):
                r1 = min(n, r0 + 512)
                w0 = max(0, r0 - c["W"] + 1)
                j = torch.cat((torch.arange(min(c["S"], w0)), torch.arange(w0, r1))).to(q.device)
                i = torch.arange(r0, r1, device=q.device)
                a = (q[b, r0:r1, hs], k[b, j, h], v[b, j, h], i, j, c["S"], c["W"], d ** -0.5)
                if grads is None:
                    out[b, r0:r1, hs] = _exact_rows(*a)
                else:
                    o, dq, dk, dv = _exact_rows(*a, dout=s["dout"][b, r0:r1, hs].double())
                    out[b, r0:r1, hs], grads[0][b, r0:r1, hs] = o, dq
                    grads[1][b, :, h].index_add_(0, j, dk)
                    grads[2][b, :, h].index_add_(0, j, dv)
    return out if grads is None else (out, *grads)


def _exact_qk(x, gain, cos, sin):
    """QKNorm and rotation of rows x [..., d] in 64 bits: (normalised, rotated)."""
    x = x.double()
    y = gain.double()[:, None] * x / torch.sqrt(torch.clamp((x * x).mean(-1, keepdim=True), min=EPS))
    h = x.shape[-1] // 2
    a, b = y[..., :h], y[..., h:]
    co, si = cos.double()[:, None], sin.double()[:, None]
    return y, torch.cat((a * co[..., :h] - b * si[..., :h], b * co[..., h:] + a * si[..., h:]), -1)


def _exact_append(s):
    c, d = s["c"], s["c"]["d"]
    dev = s["k"].device
    kn, kt = _exact_qk(s["k"], s["gain"], s["cos"][s["pos"]], s["sin"][s["pos"]])
    pages = {n: s[n].double() for n in ("kc", "kr", "vp", "summ")}
    ko, vo = _key_off(d, dev), _val_off(d, dev)
    table, (old, new) = s["table"].cpu().tolist(), _ragged(c)
    t = 0
    for b in range(c["Bd"]):
        p = old[b]
        while p < old[b] + new[b]:
            n = min(PAGE - p % PAGE, old[b] + new[b] - p)
            at, sl = table[b][p // PAGE], slice(p % PAGE, p % PAGE + n)
            for h in range(c["Hkv"]):
                pages["kc"][at, h, ko[sl]] = kn[t:t + n, h]
                pages["kr"][at, h, ko[sl]] = kt[t:t + n, h]
                pages["vp"][at, h, vo[sl]] = s["v"][t:t + n, h].double()
                if p % PAGE + n == PAGE:
                    rows = pages["kc"][at, h][ko]
                    w = torch.softmax(s["probes"][h].double() @ rows.T / d ** 0.5, -1)
                    pages["summ"][at, h] = w @ rows @ s["proj"][h].double()
            t, p = t + n, p + n
    return pages["kc"], pages["kr"], pages["vp"], pages["summ"]


def _exact_paged(s):
    c, d = s["c"], s["c"]["d"]
    G, dev = c["Hq"] // c["Hkv"], s["q"].device
    W, S = c.get("W", 0), c.get("S", 0)
    q = _exact_qk(s["q"], s["gain"], s["cos"][s["pos"]], s["sin"][s["pos"]])[1]
    out = torch.zeros_like(q)
    old, new = _ragged(c)
    ko, vo, t = _key_off(d, dev), _val_off(d, dev), 0
    for b in range(c["Bd"]):
        if new[b]:
            L = old[b] + new[b]
            pages = s["table"][b, : -(-L // PAGE)].long()
            j, i = torch.arange(L, device=dev), torch.arange(old[b], L, device=dev)
            for h in range(c["Hkv"]):
                k = s["kr"][pages, h].double()[:, ko].reshape(-1, d)[:L]
                v = s["vp"][pages, h].double()[:, vo].reshape(-1, d)[:L]
                x = q[t:t + new[b], h * G:h * G + G]
                out[t:t + new[b], h * G:h * G + G] = _exact_rows(x, k, v, i, j, S, W, float(s["scales"][b].double()))
        t += new[b]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("swa", "train"):
        return _exact_swa(s)
    return _exact_append(s) if case["kind"] == "append" else _exact_paged(s)
