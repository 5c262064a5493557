"""The cache in 4 and 8 bits, as it is measured.

Four kinds of call:

  append  new keys and values into the cache: QKNorm, rotation at each token's
          own position, quantised; and those tokens read back as the values they
          stand for
  read    the last tokens of every sequence, or all of them, as rows
  paged   attention of new tokens over the cache: one token per sequence (decode)
          or several (a part of a prompt), whole or windowed with sinks
  prefix  decode of a batch whose sequences share their first pages

A cached element has 4 bits (e2m1) or 8 (e4m3); 32 neighbours of a token's head
share a power of two 2^(b - 127), held as the byte b: the smallest for which their
largest magnitude is at most 1.75 * 2^emax (7 or 448) times it.  b = 0: all are 0;
b = 255: one was not finite, all read as NaN.

Shapes: 14 query / 2 KV heads at head dim 64 and 28 / 4 at head dim 128, window
1024, 4 sinks, 64-token pages; drawn cases also take other groups.  Inputs are
N(0, 1); cached keys are N(0, 1) times the QKNorm gain d ** 0.25, so that scores have
a standard deviation of 1.
"""
import os
import sys

import numpy as np
import torch

own = False

PAGE, GROUP, EPS = 64, 32, 1e-6
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SMALL = dict(Hq=14, Hkv=2, d=64)
LARGE = dict(Hq=28, Hkv=4, d=128)
# bits -> (largest exponent, smallest exponent, mantissa bits, largest value)
FORMAT = {4: (2, 0, 1, 6.0), 8: (8, -6, 3, 448.0)}


def _hba():
    path = os.path.abspath("hierarchical-block-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hba_amd

    return hba_amd


# -------------------------------------------------------------------- cases --
def listed():
    return [
        # one token for each sequence of a running batch, one layer: latency
        dict(name="append_step", kind="append", dtype="bf16", bits=4, Bd=64, new_lo=1, new_hi=1, old_lo=10, old_hi=6000,
             draws=1, **SMALL),
        # a few accepted tokens per sequence, some with none, in 8 bits
        dict(name="append_few_8", kind="append", dtype="bf16", bits=8, Bd=48, new_lo=0, new_hi=6, old_lo=10,
             old_hi=6000, draws=2, **LARGE),
        # prompts arriving together, at odd places of their pages
        dict(name="append_prompts", kind="append", dtype="bf16", bits=4, Bd=6, new_lo=700, new_hi=4000, old_lo=0,
             old_hi=9000, draws=3, **LARGE),
        # a few fp32 sequences taken out of the cache
        dict(name="read_f32", kind="read", dtype="f32", bits=4, Bd=9, old_lo=20, old_hi=900, draws=4, **LARGE),
        # long contexts taken out of the cache whole
        dict(name="read_long_8", kind="read", dtype="bf16", bits=8, Bd=4, old_lo=8000, old_hi=32000, draws=5, **SMALL),
        # one user, one token, a short context: latency
        dict(name="decode_one", kind="paged", dtype="bf16", bits=4, Bd=1, new_lo=1, new_hi=1, old_lo=1501, old_hi=1501,
             W=0, S=0, draws=6, **SMALL),
        # one token of one window layer for a running batch, in 8 bits
        dict(name="decode_window_8", kind="paged", dtype="bf16", bits=8, Bd=64, new_lo=1, new_hi=1, old_lo=100,
             old_hi=16000, W=1024, S=4, draws=7, **SMALL),
        # one token over the whole cache, long contexts
        dict(name="decode_all_d128", kind="paged", dtype="bf16", bits=4, Bd=24, new_lo=1, new_hi=1, old_lo=4000,
             old_hi=32000, W=0, S=0, draws=8, **LARGE),
        # the same for a few fp32 sequences in 8 bits, as a check of a served model runs
        dict(name="decode_all_8_f32", kind="paged", dtype="f32", bits=8, Bd=9, new_lo=1, new_hi=1, old_lo=1000,
             old_hi=9000, W=0, S=0, draws=9, **LARGE),
        # chunked prefill: the next part of four prompts over what the cache holds
        dict(name="chunk_512", kind="paged", dtype="bf16", bits=4, Bd=4, new_lo=300, new_hi=512, old_lo=1000,
             old_hi=8000, W=0, S=0, draws=10, **SMALL),
        # the next parts of a few prompts in a window layer of the larger donor
        dict(name="chunk_window_8", kind="paged", dtype="bf16", bits=8, Bd=3, new_lo=1, new_hi=400, old_lo=500,
             old_hi=5000, W=1024, S=4, draws=11, **LARGE),
        # a batch behind one system prompt
        dict(name="prefix_8k", kind="prefix", dtype="bf16", bits=4, Bd=64, shared=8192, new_lo=1, new_hi=1, old_lo=1,
             old_hi=700, draws=12, **SMALL),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "paged", "paged", "prefix"])
    Hq, Hkv, d = rng.choice([(14, 2, 64), (28, 4, 128), (8, 8, 64), (16, 2, 128), (6, 6, 128), (12, 4, 64)])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]), bits=rng.choice([4, 4, 8]), Hq=Hq, Hkv=Hkv, d=d)
    if kind == "append":
        hi = rng.choice([1, _log(rng, 2, 3000)])
        c.update(Bd=max(1, min(64, rng.randint(1, 10000 // hi))), new_lo=1 if hi == 1 else hi // 3, new_hi=hi, old_lo=0,
                 old_hi=_log(rng, 50, 6000), draws=rng.randrange(1000))
    elif kind == "read":
        hi = _log(rng, 10, 16000)
        c.update(Bd=max(1, min(64, rng.randint(1, max(1, 40000 // hi)))), old_lo=0, old_hi=hi, draws=rng.randrange(1000))
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


def _ragged(c):
    """(tokens already there, the call's tokens) of each sequence; a shared prefix counts as there.
    A read's tokens are all there are."""
    old = _spread(c["old_lo"], c["old_hi"], c["Bd"], c["draws"])
    if c["kind"] == "read":
        old[0] = max(old[0], 1)
        return [0] * c["Bd"], old
    new = _spread(c["new_lo"], c["new_hi"], c["Bd"], c["draws"] + 1)
    if sum(new) == 0:
        new[0] = 1
    return [x + c.get("shared", 0) for x in old], new


def _one_each(c):
    return c.get("new_hi", 0) == 1 and c.get("new_lo", 0) == 1


# ------------------------------------------------------------------- layout --
def _page_bytes(d, bits):
    return PAGE * d * bits // 8 + 2 * d


def _key_off(d, bits, dev):
    """Byte of element t of key j within a key page [64, d], and of its group's scale [64, d / 32]."""
    j, t = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    tile, row = 2 * (j // 32) + j // 4 % 2, 4 * (j % 32 // 8) + j % 4
    at = (tile * (d // 4) + t % (d // 4)) * bits // 8
    g = torch.arange(d // GROUP, device=dev)[None]
    return (at // 16 * 64 + row + 16 * (t // (d // 4))) * 16 + at % 16, PAGE * d * bits // 8 + (row + 16 * g) * 4 + tile


def _val_off(d, bits, dev):
    """The same within a value page."""
    j, t = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    at = (t // 16 * 8 + j % 8) * bits // 8
    piece = j // 32 * (d * bits // 256) + at // 16
    g = torch.arange(d // GROUP, device=dev)[None]
    return (piece * 64 + t % 16 + 16 * (j % 32 // 8)) * 16 + at % 16, \
        PAGE * d * bits // 8 + (j // 8 * (d // GROUP) + g) * 8 + j % 8


def _high(d, keys, dev):
    """Whether an element has the high four bits of its byte, [64, d]."""
    j, t = torch.arange(PAGE, device=dev)[:, None], torch.arange(d, device=dev)[None]
    return ((t if keys else j) % 2 == 1).expand(PAGE, d)


# ------------------------------------------------------------- quantisation --
def _pow2(k):
    """2^k of whole numbers, with nothing rounded (a power function's result may be)."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _quantise(x, bits):
    """Codes (uint8, one each) and scale bytes of fp32 rows x [..., d]."""
    emax, emin, mant, top = FORMAT[bits]
    x = x.unflatten(-1, (-1, GROUP))
    big = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(big)                                              # big = m 2^e, m in [1/2, 1)
    b = (e - 1 - emax + (m > 0.875).int() + 127).clamp(1, 254)
    b = torch.where(big == 0, 0, b)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    a = (torch.where(bad, 0.0, x).double() * _pow2(127 - b)).abs()
    step = _pow2((torch.frexp(a)[1] - 1).clamp_min(emin) - mant)
    a = (torch.round(a / step) * step).clamp_max(top)
    m, e = torch.frexp(a)
    e = torch.where(a < 2.0 ** emin, emin, e - 1)                        # value a: exponent e, the rest in steps of 2^(e - mant)
    rest = (a * _pow2(mant - e)).int()                        # 2^mant .. 2^(mant + 1) - 1, less where subnormal
    code = torch.where(rest < 2 ** mant, rest, (e - emin + 1) * 2 ** mant + rest - 2 ** mant)
    code = code + (torch.signbit(x) & ~bad).int() * 2 ** (bits - 1)
    return code.flatten(-2).to(torch.uint8), torch.where(bad, 255, b).squeeze(-1).to(torch.uint8)


def _values(bits, dev):
    """The value of each code."""
    emax, emin, mant, top = FORMAT[bits]
    c = torch.arange(2 ** (bits - 1), device=dev)
    e, rest = c >> mant, (c & (2 ** mant - 1)).float()
    v = torch.where(e == 0, rest * 2.0 ** (emin - mant), (1 + rest * 2.0 ** -mant) * _pow2(e + emin - 1).float())
    return torch.cat((v, -v))


def _powers(dev):
    """The value of each scale byte."""
    p = _pow2(torch.arange(256, device=dev) - 127).float()
    p[0], p[255] = 0.0, float("nan")
    return p


def _place(pages, page, slot, rows, off, high, bits):
    """Rows [T, Hkv, d] as codes and scale bytes into pages [P, Hkv, bytes] at (page, slot) of each token."""
    code, b = _quantise(rows, bits)
    hkv = torch.arange(pages.shape[1], device=pages.device)
    base = ((page[:, None] * pages.shape[1] + hkv) * pages.shape[2])[..., None]
    flat = pages.view(-1)
    flat[base + off[1][slot][:, None]] = b
    where = (base + off[0][slot][:, None]).flatten()
    if bits == 8:
        flat[where] = code.flatten()
        return
    hi = high[slot][:, None].expand(code.shape).flatten()
    code = code.flatten()
    low, up = torch.where(~hi)[0], torch.where(hi)[0]   # two elements of a byte, one after the other
    flat[where[low]] = (flat[where[low]] & 240) | code[low]
    flat[where[up]] = (flat[where[up]] & 15) | (code[up] << 4)


def _rows(pages, ids, off, high, bits, d):
    """Pages ids [..., n] of [P, Hkv, bytes] as fp32 rows [..., n, Hkv, 64, d]."""
    x = pages[ids]
    code = x.index_select(-1, off[0].flatten()).unflatten(-1, (PAGE, d))
    if bits == 4:
        code = torch.where(high, code >> 4, code & 15)
    v = _values(bits, x.device).index_select(0, code.flatten().int()).view(code.shape)
    b = x.index_select(-1, off[1].flatten()).unflatten(-1, (PAGE, d // GROUP))
    s = _powers(x.device).index_select(0, b.flatten().int()).view(b.shape)
    return (v.unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)


# ------------------------------------------------------------------- inputs --
def _tables(n, d, dev):
    ang = torch.outer(torch.arange(n, device=dev).double(),
                      1.0 / (1e6 ** (torch.arange(0, d, 2, device=dev).double() / d)))
    ang = torch.cat((ang, ang), -1)
    return ang.cos().float(), ang.sin().float()


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _filled(P, Hkv, d, bits, std, off, high, g, dev):
    """Pages that hold quantised N(0, std^2) rows, 1024 pages at a time."""
    out = torch.empty(P, Hkv, _page_bytes(d, bits), dtype=torch.uint8, device=dev)
    for p in range(0, P, 1024):
        n = min(1024, P - p)
        code, b = _quantise(std * torch.randn(n, Hkv, PAGE, d, generator=g, device=dev), bits)
        part = out[p:p + n]
        part[..., off[1].flatten()] = b.flatten(-2)
        if bits == 8:
            part[..., off[0].flatten()] = code.flatten(-2)
        else:
            lo, hi = ~high.flatten(), high.flatten()
            at, code = off[0].flatten(), code.flatten(-2)
            part[..., at[lo]] = code[..., lo]
            part[..., at[hi]] |= code[..., hi] << 4
    return out


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, d, Hq, Hkv, bits = DT[c["dtype"]], c["d"], c["Hq"], c["Hkv"], c["bits"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    old, new = _ragged(c)
    L = [a + b for a, b in zip(old, new)]
    Bd, shared, T = c["Bd"], c.get("shared", 0) // PAGE, sum(new)
    mp = max(1, max((x + PAGE - 1) // PAGE for x in L))
    P = shared + Bd * (mp - shared) + 3
    phys = torch.randperm(P, generator=g, device=dev).int()
    table = torch.cat([phys[:shared].expand(Bd, shared), phys[shared:shared + Bd * (mp - shared)].view(Bd, -1)], 1)
    s = dict(c=c, T=T, table=table.contiguous(), seq_lens=_i32(L, dev), max_len=max(L),
             cu=None if _one_each(c) else _i32(np.cumsum([0] + new).tolist(), dev),
             koff=_key_off(d, bits, dev), voff=_val_off(d, bits, dev), khigh=_high(d, True, dev), vhigh=_high(d, False, dev))
    # each token's sequence and position: the plain form's program plans them on the host
    s["seq"] = torch.tensor(np.repeat(np.arange(Bd), new), device=dev)
    s["pos"] = torch.tensor(np.concatenate([np.arange(a, a + b) for a, b in zip(old, new)]), device=dev)
    s["kp"] = _filled(P, Hkv, d, bits, d ** 0.25, s["koff"], s["khigh"], g, dev)
    s["vp"] = _filled(P, Hkv, d, bits, 1.0, s["voff"], s["vhigh"], g, dev)
    if c["kind"] == "read":
        return s
    s["cos"], s["sin"] = _tables(mp * PAGE, d, dev)
    gain = torch.full((max(Hq, Hkv),), d ** 0.25, device=dev)
    gain *= 1 + 0.1 * torch.randn(gain.shape, generator=g, device=dev)
    if c["kind"] == "append":
        kv = randn(T, 2, Hkv, d)   # one projection's output: k and v are views of it
        s.update(k=kv[:, 0], v=kv[:, 1], gain=gain[:Hkv].contiguous())
        return s
    s.update(q=randn(T, Hq, d), gain=gain[:Hq].contiguous(), most=max(new),
             cu_all=_i32(np.cumsum([0] + new).tolist(), dev),
             scales=1.0 / d + torch.rand(Bd, generator=g, device=dev) * 0.1 / d)
    return s


# --------------------------------------------------------------- plain forms --
def _softmax(s):
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _norm(x, gain):
    return x / x.square().mean(-1, keepdim=True).clamp_min(EPS).sqrt() * gain[:, None]


def _rotate(x, cos, sin, pos):
    h = x.shape[-1] // 2
    return x * cos[pos][:, None] + torch.cat((-x[..., h:], x[..., :h]), -1) * sin[pos][:, None]


def _plain_read(s):
    c = s["c"]
    d, bits = c["d"], c["bits"]
    page, slot = s["table"].long()[s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    used, at = torch.unique(page, return_inverse=True)
    k = _rows(s["kp"], used, s["koff"], s["khigh"], bits, d)[at, :, slot]
    v = _rows(s["vp"], used, s["voff"], s["vhigh"], bits, d)[at, :, slot]
    return k.to(DT[c["dtype"]]), v.to(DT[c["dtype"]])


def _plain_append(s):
    c = s["c"]
    # a key next to a border between two codes falls to one side: in 64 bits, and rounded to 32 once
    k = _rotate(_norm(s["k"].double(), s["gain"].double()), s["cos"].double(), s["sin"].double(), s["pos"]).float()
    page, slot = s["table"].long()[s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    _place(s["kp"], page, slot, k, s["koff"], s["khigh"], c["bits"])
    _place(s["vp"], page, slot, s["v"].float(), s["voff"], s["vhigh"], c["bits"])
    return _plain_read(s)


def _pages(s, ids):
    """Keys and values of pages ids [..., n] as fp32 rows [..., Hkv, 64 n, d]."""
    c = s["c"]
    k = _rows(s["kp"], ids, s["koff"], s["khigh"], c["bits"], c["d"]).transpose(-4, -3).flatten(-3, -2)
    v = _rows(s["vp"], ids, s["voff"], s["vhigh"], c["bits"], c["d"]).transpose(-4, -3).flatten(-3, -2)
    return k, v


def _plain_paged(s):
    c, dev = s["c"], s["q"].device
    Hq, Hkv, d, W, S, most = c["Hq"], c["Hkv"], c["d"], c["W"], c["S"], s["most"]
    Bd, G, mp = c["Bd"], Hq // Hkv, s["table"].shape[1]
    q = _rotate(_norm(s["q"].float(), s["gain"]), s["cos"], s["sin"], s["pos"]) * s["scales"][s["seq"]][:, None, None]
    L, cu = s["seq_lens"].long(), s["cu_all"].long()
    first = L - (cu[1:] - cu[:-1])                                       # position of the first new token
    if W:
        ns = -(-S // PAGE)
        w0 = (first - W + 1).clamp_min(0) // PAGE
        nw = min(mp, (W + most) // PAGE + 2)
        logical = torch.cat((torch.arange(ns, device=dev).expand(Bd, ns),
                             torch.maximum(w0, torch.tensor(ns, device=dev))[:, None]
                             + torch.arange(nw, device=dev)), 1)
    else:
        logical = torch.arange(mp, device=dev).expand(Bd, mp)
    k, v = _pages(s, s["table"].long().gather(1, logical.clamp_max(mp - 1)))
    j = (logical[:, :, None] * PAGE + torch.arange(PAGE, device=dev)).flatten(1)
    slot = torch.arange(len(s["seq"]), device=dev) - cu[:-1][s["seq"]]
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
    q = _rotate(_norm(s["q"].float(), s["gain"]), s["cos"], s["sin"], s["pos"]) * s["scales"][:, None, None]
    q = q.view(Bd, Hkv, G, d)
    kp, vp = _pages(s, table[0, : n // PAGE])                            # the prefix, once
    ks, vs = _pages(s, table[:, n // PAGE:])
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
    if kind in ("append", "read"):
        if not own:
            return _plain_append(s) if kind == "append" else _plain_read(s)
        ops = _hba().ops
        if kind == "append":
            ops.kv_append_mx(s["k"], s["v"], s["cu"], s["gain"], EPS, s["cos"], s["sin"], s["table"], s["seq_lens"],
                             s["kp"], s["vp"])
        return ops.kv_read_mx(s["kp"], s["vp"], s["table"], s["seq_lens"], s["cu"], s["T"], c["d"], DT[c["dtype"]])
    if not own:
        return _plain_paged(s) if kind == "paged" else _plain_prefix(s)
    return _hba().ops.paged_attn_mx(s["q"], s["gain"], EPS, s["kp"], s["vp"], s["table"], s["seq_lens"], s["cos"],
                                    s["sin"], s["scales"], s["max_len"], window=c.get("W", 0), sinks=c.get("S", 0),
                                    cu=s["cu"], shared=c.get("shared", 0))


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
    held = d * c["bits"] // 8 + d // GROUP                               # bytes of a cached key or value
    old, new = _ragged(c)
    T, L = sum(new), [a + b for a, b in zip(old, new)]
    rows = 2 * T * Hkv * d * e                                           # keys and values of the call's tokens
    if c["kind"] == "read":
        return {"bytes": 2 * T * Hkv * held + rows, "flops": 2 * T * Hkv * d}
    if c["kind"] == "append":                                            # rows in, codes, rows out; cos and sin
        return {"bytes": 2 * rows + 2 * T * Hkv * held + T * d * 8, "flops": 16 * T * Hkv * d}
    W, S, shared = c.get("W", 0), c.get("S", 0), c.get("shared", 0)
    pairs = sum(_pairs(a, b, W, S) for a, b in zip(old, L)) * Hq
    keys = 0
    for a, b in zip(old, L):
        if not b > a:
            continue
        w0 = max(0, a - W + 1) if W else 0
        keys += b - w0 + min(S, w0) - (shared if c["kind"] == "prefix" else 0)
    return {"bytes": 2 * Hkv * (keys + shared) * held + 2 * T * Hq * d * e, "flops": 4 * d * pairs}


# --------------------------------------------------------------------- exact --
def exact(case, seed):
    """In 64 bits, sequence by sequence: what a page holds by its definition, the nearest
    code to each element, and attention as it is written."""
    c, s = case, prepare(case, seed)
    d, Hkv, bits = c["d"], c["Hkv"], c["bits"]
    G, dev = c["Hq"] // Hkv, s["kp"].device
    half = {4: [0, 0.5, 1, 1.5, 2, 3, 4, 6],
            8: [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]}
    grid = torch.tensor(half[bits], dtype=torch.float64, device=dev)
    powers = torch.tensor([2.0 ** k for k in range(-300, 301)], dtype=torch.float64, device=dev)
    middle, top = (grid[1:] + grid[:-1]) / 2, {4: 7.0, 8: 448.0}[bits]

    def nearest(x):
        """What rows x [..., d] are held as."""
        x = x.double().unflatten(-1, (d // 32, 32))
        big = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(big / top))
        e = e.nan_to_num(neginf=-126.0).long().clamp_min(-126)
        e = e + (big > top * powers[e + 300]).long() - (big <= top * powers[e + 299]).long()
        scale = powers[e.clamp_min(-126) + 300]
        a = (x / scale).abs()
        at = torch.bucketize(a, middle)                                  # how many middles are below
        at = at + ((a == middle[at.clamp_max(len(middle) - 1)]) & (at % 2 == 1)).long()
        y = torch.where(big == 0, 0.0, torch.sign(x) * grid[at.clamp_max(len(grid) - 1)] * scale)
        return y.flatten(-2)

    def held(pages, off, high, ids):
        """Rows [Hkv, 64 n, d] of pages ids [n]."""
        raw = pages[ids].long()
        code = raw[..., off[0]]
        if bits == 4:
            code = torch.where(high, code // 16, code % 16)
        signs, code = code // 2 ** (bits - 1), code % 2 ** (bits - 1)
        grown = torch.cat((grid, torch.full((1,), torch.nan, dtype=grid.dtype, device=dev)))
        b = raw[..., off[1]]
        scale = torch.where(b == 255, torch.nan, torch.where(b == 0, 0.0, powers[b + 300 - 127]))
        x = grown[code] * (1 - 2 * signs) * scale.repeat_interleave(32, -1)
        return x.transpose(0, 1).flatten(1, 2)

    def turned(x, gain, pos):
        """QKNorm and rotation at positions pos."""
        x = x.double()
        y = gain.double()[:, None] * x / torch.sqrt(torch.clamp((x * x).mean(-1, keepdim=True), min=EPS))
        co, si = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat((a * co[..., :d // 2] - b * si[..., :d // 2], b * co[..., d // 2:] + a * si[..., d // 2:]), -1)

    if c["kind"] == "append":
        return nearest(turned(s["k"], s["gain"], s["pos"]).float()), nearest(s["v"])
    old, new = _ragged(c)
    W, S, t, found = c.get("W", 0), c.get("S", 0), 0, []
    if c["kind"] != "read":
        q = turned(s["q"], s["gain"], s["pos"])
    for b in range(c["Bd"]):
        n = old[b] + new[b]
        if not new[b]:
            continue
        ids = s["table"][b, : -(-n // PAGE)].long()
        k, v = held(s["kp"], s["koff"], s["khigh"], ids)[:, :n], held(s["vp"], s["voff"], s["vhigh"], ids)[:, :n]
        if c["kind"] == "read":
            found.append((k.transpose(0, 1), v.transpose(0, 1)))
            continue
        i, j = torch.arange(old[b], n, device=dev)[:, None], torch.arange(n, device=dev)[None]
        see = j <= i
        if W:
            see = see & ((j > i - W) | (j < S))
        out = torch.empty(new[b], c["Hq"], d, dtype=torch.float64, device=dev)
        for h in range(c["Hq"]):
            x = q[t:t + new[b], h] @ k[h // G].T * float(s["scales"][b].double())
            out[:, h] = torch.softmax(torch.where(see, x, -torch.inf), -1) @ v[h // G]
        found.append(out)
        t += new[b]
    if c["kind"] == "read":
        return torch.cat([k for k, _ in found]), torch.cat([v for _, v in found])
    return torch.cat(found)
