"""The cache in 4 and 8 bits on the GPU: what append writes against the definition in 64
bits (the same bytes), what read gives (the same values), attention over it against 64-bit
results, and runs of all of them together."""
import pytest
import torch

import hba_amd
import mx64
from attn64 import E, assert_within, attend, norm_rotate, unit, visible
from hba_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 2.0 ** -20   # a number that fp32 has
FORMS = [(dt, d, bits) for dt in ("f32", "bf16") for d in (64, 128) for bits in (4, 8)]


def dev(s):
    return {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}


# ------------------------------------------------------------------- append --
def new_tokens(dt, d, bits, Hkv, lens, new, seed=0, gain=True, turn=True, maxp=None):
    """A ragged batch and pages full of random bytes."""
    g = torch.Generator().manual_seed(seed)
    Bd, T = len(lens), sum(new)
    maxp = maxp or max(1, max((n + 63) // 64 for n in lens))
    P = Bd * maxp + 2
    cos, sin = hba_amd.rope_tables(maxp * 64, d, 1e4, "cpu") if turn else (None, None)
    pages = [torch.randint(0, 256, (P, Hkv, mx64.page_bytes(d, bits)), generator=g).to(torch.uint8) for _ in range(2)]
    return dict(k=torch.randn(T, Hkv, d, generator=g).to(dt), v=torch.randn(T, Hkv, d, generator=g).to(dt),
                gain=1.5 + torch.rand(Hkv, generator=g) if gain else None, cos=cos, sin=sin, kp=pages[0], vp=pages[1],
                table=torch.randperm(P, generator=g)[:Bd * maxp].view(Bd, maxp).int(), new=new, bits=bits,
                lens=torch.tensor(lens, dtype=torch.int32), cu=torch.tensor([0] + new).cumsum(0).int())


def append(s, **kw):
    """The pages after the call."""
    a = dev({**s, **kw})
    ops.kv_append_mx(a["k"], a["v"], a["cu"], a["gain"], EPS, a["cos"], a["sin"], a["table"], a["lens"], a["kp"], a["vp"])
    return a["kp"].cpu(), a["vp"].cpu()


def appended(s):
    """The same by the definition: (sequence, position, row) of each token that has a place."""
    d, bits = s["k"].shape[2], s["bits"]
    kp, vp = s["kp"].clone(), s["vp"].clone()
    most = 64 * s["table"].shape[1]
    if s["cos"] is not None:
        most = min(most, s["cos"].shape[0])
    t = 0
    for b, (n, c) in enumerate(zip(s["lens"].tolist(), s["new"])):
        pos = torch.arange(n - c, n)
        ok = (pos >= 0) & (pos < most)
        at = pos.clamp(0, most - 1)
        cs, sn = (None, None) if s["cos"] is None else (s["cos"][at], s["sin"][at])
        k = norm_rotate(s["k"][t:t + c], s["gain"], EPS, cs, sn, 0.0)[1].float()
        kc, kb = mx64.quantise(k, bits)
        vc, vb = mx64.quantise(s["v"][t:t + c], bits)
        for p in range((most + 63) // 64):
            on = ok & (pos // 64 == p)
            page = int(s["table"][b, p])
            if not on.any() or not 0 <= page < kp.shape[0]:
                continue
            for h in range(kp.shape[1]):
                mx64.write(kp[page, h], pos[on] % 64, kc[on, h], kb[on, h], bits, True)
                mx64.write(vp[page, h], pos[on] % 64, vc[on, h], vb[on, h], bits, False)
        t += c
    return kp, vp


def same(got, want):
    for g, w, what in zip(got, want, ("keys", "values")):
        assert torch.equal(g, w), f"{what}: {int((g != w).sum())} of {g.numel()} bytes differ"


BATCHES = [([1], [1]), ([64], [64]), ([5, 70, 0, 300], [5, 3, 0, 299]), ([64, 640], [64, 65]), ([129, 900, 66], [0, 130, 1]),
           ([33, 41, 40, 77], [1, 2, 7, 13]), ([700, 127, 65], [700, 64, 2])]


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("lens,new", BATCHES)
def test_append_writes_the_definitions_bytes(lens, new, dt, d, bits):
    """Every byte of the pages: those of the new tokens, and all others as they were."""
    s = new_tokens(DT[dt], d, bits, 2, lens, new, seed=sum(lens))
    same(append(s), appended(s))


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("gain,turn", [(False, False), (True, False), (False, True)])
def test_append_without_norm_or_rotation(gain, turn, dt, d, bits):
    s = new_tokens(DT[dt], d, bits, 3, [200, 9, 65], [199, 2, 1], seed=1, gain=gain, turn=turn)
    same(append(s), appended(s))


@pytest.mark.parametrize("dt,d,bits", FORMS)
def test_append_one_token_each(dt, d, bits):
    """cu None: the newest of each sequence; as many calls leave what one call does."""
    s = new_tokens(DT[dt], d, bits, 2, [70, 1, 128, 9], [12, 1, 12, 9], seed=2)
    want = append(s)
    a = dev(s)
    at = s["cu"].tolist()
    for i in range(12):
        on = [b for b in range(4) if i < s["new"][b]]
        rows = torch.tensor([at[b] + i for b in on])
        lens = torch.tensor([s["lens"][b] - s["new"][b] + i + 1 for b in on], dtype=torch.int32)
        ops.kv_append_mx(a["k"][rows], a["v"][rows], None, a["gain"], EPS, a["cos"], a["sin"], a["table"][on], lens.cuda(),
                         a["kp"], a["vp"])
    same((a["kp"].cpu(), a["vp"].cpu()), want)


@pytest.mark.parametrize("dt,d,bits", FORMS)
def test_values_at_the_edges(dt, d, bits):
    """Zeros of both signs, groups that are tiny, subnormal, huge or not finite, magnitudes
    next to the scale's limit, and ties between two codes."""
    s = new_tokens(DT[dt], d, bits, 1, [120], [120], seed=3, gain=False, turn=False)
    for x in (s["k"], s["v"]):
        x[0] = 0.0
        x[1] = -0.0
        x[2, :, ::2] = 0.0
        x[3] *= 2.0 ** -120
        x[4] *= 2.0 ** -126
        x[5] *= 2.0 ** -132
        x[6] *= 2.0 ** 124
        x[7, :, 5] = float("nan")
        x[8, :, 40] = float("inf")
        x[9, :, 63] = float("-inf")
        x[10] = torch.finfo(x.dtype).max
        x[11] = -torch.finfo(x.dtype).max
        x[12], x[13], x[14] = 7.0, 7.03125, 448.0
        x[15, :, 1:] = 0.0
        for i in range(16, 120):   # multiples of 1/16 up to 8, of 1/64 and less in 8 bits
            x[i] = torch.randint(-128, 129, x[i].shape, generator=torch.Generator().manual_seed(i)) / (16.0 if i % 2 else 512.0)
            x[i, :, ::32] = 8.0 - i % 3
    got, want = append(s), appended(s)
    same(got, want)
    a = dev(s)
    k, v = ops.kv_read_mx(got[0].cuda(), got[1].cuda(), a["table"], a["lens"], a["cu"], 120, d, torch.float32)
    for x, y in ((s["k"], k), (s["v"], v)):
        want = mx64.values(*mx64.quantise(x, bits), bits)
        assert torch.equal(y.double().cpu().nan_to_num(77.0), want.nan_to_num(77.0))


@pytest.mark.parametrize("dt,d,bits", FORMS)
def test_what_is_not_appended(dt, d, bits):
    """A padded batch, lengths below the token count, past the page table and the rotation
    tables, pages outside the cache."""
    s = new_tokens(DT[dt], d, bits, 2, [100, 3, 70], [40, 3, 2], seed=4, maxp=2)
    pad = {n: torch.cat([s[n], torch.full((77, 2, d), float("nan"), dtype=DT[dt])]) for n in ("k", "v")}
    same(append({**s, **pad}), appended(s))
    short = {**s, "lens": torch.tensor([30, 1, 70], dtype=torch.int32)}
    same(append(short), appended(short))
    over = {**s, "lens": torch.tensor([150, 2 ** 31 - 1, -5], dtype=torch.int32)}
    same(append(over), appended(over))
    few = {**s, "cos": s["cos"][:80], "sin": s["sin"][:80]}
    same(append(few), appended(few))
    table = s["table"].clone()
    table[0, 1], table[1, 0] = 10 ** 8, -1
    same(append({**s, "table": table}), appended({**s, "table": table}))
    none = {n: s[n][:0] for n in ("k", "v")}
    same(append({**s, **none, "cu": s["cu"] * 0}), (s["kp"], s["vp"]))


def test_append_strides_streams_and_graphs():
    s = new_tokens(torch.bfloat16, 64, 4, 2, [300, 65], [200, 1], seed=5)
    want = append(s)
    both = torch.randn(201, 2, 3, 64).to(torch.bfloat16)
    both[:, :, 0], both[:, :, 2] = s["k"], s["v"]
    both = both.cuda()
    same(append({**s, "k": both[:, :, 0], "v": both[:, :, 2]}), want)
    same(append({**s, "k": torch.nn.functional.pad(s["k"], (1, 2)).cuda()[..., 1:-2]}), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = append(s)
    same(got, want)
    a = dev(s)
    start = a["kp"].clone(), a["vp"].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_append_mx(a["k"], a["v"], a["cu"], a["gain"], EPS, a["cos"], a["sin"], a["table"], a["lens"], a["kp"], a["vp"])
        out = ops.kv_read_mx(a["kp"], a["vp"], a["table"], a["lens"], a["cu"], 201, 64, torch.bfloat16)
    for seed in range(3):
        t = new_tokens(torch.bfloat16, 64, 4, 2, [300, 65], [200, 1], seed=seed)
        a["k"].copy_(t["k"])
        a["v"].copy_(t["v"])
        a["lens"].copy_(torch.tensor([300 - 50 * seed, 65 - seed]))
        a["kp"].copy_(start[0])
        a["vp"].copy_(start[1])
        graph.replay()
        torch.cuda.synchronize()
        now = {**s, "k": t["k"], "v": t["v"], "lens": a["lens"].cpu()}
        same((a["kp"].cpu(), a["vp"].cpu()), append(now))
        for x, y in zip(out, ops.kv_read_mx(a["kp"], a["vp"], a["table"], a["lens"], a["cu"], 201, 64, torch.bfloat16)):
            assert torch.equal(x, y)


def test_append_refusals():
    s = new_tokens(torch.float32, 64, 4, 2, [100, 65], [4, 5])
    bad = [dict(k=s["k"][:, :1]), dict(v=s["v"].bfloat16()), dict(k=s["k"].double(), v=s["v"].double()), dict(k=s["k"][0]),
           dict(kp=s["kp"].int()), dict(kp=s["kp"][..., :-1], vp=s["vp"][..., :-1]), dict(vp=s["vp"][:-1]),
           dict(kp=s["kp"][:0], vp=s["vp"][:0]), dict(kp=s["kp"].transpose(0, 1)), dict(table=s["table"].long()),
           dict(table=s["table"][0]), dict(lens=s["lens"][:1]), dict(cu=s["cu"].long()), dict(cu=s["cu"][:2]), dict(cu=None),
           dict(cos=None), dict(gain=s["gain"][:1]), dict(cos=s["cos"][:, :32], sin=s["sin"][:, :32])]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            append(s, **kw)


# --------------------------------------------------------------------- read --
@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("lens,new", BATCHES + [([3, 10], [5, 12]), ([0, 500], [0, 500])])
def test_read_gives_what_the_pages_hold(lens, new, dt, d, bits):
    """Random bytes are codes and scales of everything, NaN among them; tokens in no page
    are 0."""
    s = new_tokens(DT[dt], d, bits, 2, lens, new, seed=6)
    for p in (s["kp"], s["vp"]):     # scales that a bf16 value keeps all bits with
        sc = p[..., 64 * d * bits // 8:]
        sc[(sc < 20) | ((sc > 240) & (sc < 255))] = 127
    a = dev(s)
    T = sum(new) + 70
    got = ops.kv_read_mx(a["kp"], a["vp"], a["table"], a["lens"], a["cu"], T, d, DT[dt])
    for x, p, keys in ((got[0], s["kp"], True), (got[1], s["vp"], False)):
        assert x.shape == (T, 2, d) and x.dtype == DT[dt]
        want, t = torch.zeros(T, 2, d, dtype=torch.float64), 0
        held = mx64.rows(p, bits, d, keys)                                 # [P, Hkv, 64, d]
        for b, (n, c) in enumerate(zip(lens, new)):
            pos = torch.arange(n - c, n)
            on = pos >= 0
            at = pos.clamp_min(0)
            rows = held[s["table"][b].long()[at // 64], :, at % 64]
            want[t:t + c] = torch.where(on[:, None, None], rows, 0.0)
            t += c
        assert torch.equal(x.double().cpu().nan_to_num(77.0), want.nan_to_num(77.0))
        assert torch.equal(x.cpu().isnan(), want.isnan())


@pytest.mark.parametrize("bits", [4, 8])
def test_read_one_token_each_and_pages_that_there_are_none_of(bits):
    s = new_tokens(torch.float32, 64, bits, 2, [70, 1, 0, 128], [70, 1, 0, 128], seed=7)
    a = dev(s)
    append_to = a["kp"], a["vp"]
    ops.kv_append_mx(a["k"], a["v"], a["cu"], a["gain"], EPS, a["cos"], a["sin"], a["table"], a["lens"], *append_to)
    full = ops.kv_read_mx(*append_to, a["table"], a["lens"], a["cu"], 199, 64, torch.float32)
    one = ops.kv_read_mx(*append_to, a["table"], a["lens"], None, 4, 64, torch.float32)
    for x, y in zip(one, full):
        assert torch.equal(x[[0, 1, 3]], y[[69, 70, 198]]) and not x[2].any()
    table = a["table"].clone()
    table[0, 1], table[3, 0] = 10 ** 8, -1
    bad = ops.kv_read_mx(*append_to, table, a["lens"], a["cu"], 199, 64, torch.float32)
    for x, y in zip(bad, full):
        assert torch.equal(x[:64], y[:64]) and not x[64:70].any() and torch.equal(x[70], y[70])
        assert not x[71:135].any() and torch.equal(x[135:], y[135:])
    late = ops.kv_read_mx(*append_to, a["table"], a["lens"], a["cu"].clamp_min(5), 199, 64, torch.float32)
    for x, y in zip(late, full):     # sequence 0 has its last 65 tokens in places 5 ..
        assert not x[:5].any() and torch.equal(x[5:], y[5:])
    for x in ops.kv_read_mx(*append_to, a["table"][:0], a["lens"][:0], a["cu"][:1], 3, 64, torch.float32):
        assert x.shape == (3, 2, 64) and not x.any()
    assert ops.kv_read_mx(*append_to, a["table"], a["lens"], a["cu"] * 0, 0, 64, torch.float32)[0].shape == (0, 2, 64)
    past = torch.tensor([2 ** 31 - 1, 1, -4, 128], dtype=torch.int32).cuda()
    x = ops.kv_read_mx(*append_to, a["table"], past, a["cu"], 199, 64, torch.float32)[0]
    assert not x[:70].any() and torch.equal(x[70:], full[0][70:])
    for kw in (dict(tokens=-1), dict(head_dim=128), dict(dtype=torch.float16), dict(cu=None), dict(cu=a["cu"].long())):
        args = dict(cu=a["cu"], tokens=199, head_dim=64, dtype=torch.float32)
        args.update(kw)
        with pytest.raises((ValueError, TypeError)):
            ops.kv_read_mx(*append_to, a["table"], a["lens"], args["cu"], args["tokens"], args["head_dim"], args["dtype"])


# ---------------------------------------------------------------- attention --
def setup(dt, d, bits, Hq, Hkv, lens, new=None, shared=0, maxp=None, seed=0, gain=True):
    """Random rows, quantised, in permuted pages; everything behind a sequence's length is
    codes and scales of NaN and random bytes."""
    g = torch.Generator().manual_seed(seed)
    Bd, T = len(lens), len(lens) if new is None else sum(new)
    maxp = maxp or max(1, max((n + 63) // 64 for n in lens), shared // 64)
    P = Bd * maxp + 2
    table = torch.randperm(P, generator=g)[:Bd * maxp].view(Bd, maxp).int()
    table[:, :shared // 64] = table[0, :shared // 64]
    pages, held = [], []
    for keys in (True, False):
        p = torch.randint(0, 256, (P, Hkv, mx64.page_bytes(d, bits)), generator=g).to(torch.uint8)
        p[torch.rand(p.shape, generator=g) < 0.5] = 255
        c, b = mx64.quantise(torch.randn(P, Hkv, 64, d, generator=g) * (d ** 0.25 if keys else 1.0), bits)
        for s, n in enumerate(lens):
            for i in range((min(n, 64 * maxp) + 63) // 64):
                at, m = int(table[s, i]), 64 if i < shared // 64 else min(64, n - 64 * i)
                for h in range(Hkv):
                    mx64.write(p[at, h], torch.arange(m), c[at, h, :m], b[at, h, :m], bits, keys)
        pages.append(p)
        held.append(mx64.values(c, b, bits))
    rows = [[x[table[s].long()].transpose(0, 1).reshape(Hkv, -1, d) for x in held] for s in range(Bd)]
    cos, sin = hba_amd.rope_tables(maxp * 64, d, 1e4, "cpu")
    return dict(q=torch.randn(T, Hq, d, generator=g).to(dt), gain=1.2 + 0.1 * torch.randn(Hq, generator=g) if gain else None,
                kp=pages[0], vp=pages[1], table=table, lens=torch.tensor(lens, dtype=torch.int32), cos=cos, sin=sin,
                scales=(0.5 + torch.rand(Bd, generator=g)) / d, rows=rows, new=new, shared=shared, bits=bits,
                cu=None if new is None else torch.tensor([0] + new).cumsum(0).int(), max_len=max(1, max(lens)))


def call(s, W=0, S=0, **kw):
    a = dev({**s, **kw})
    return ops.paged_attn_mx(a["q"], a["gain"], EPS, a["kp"], a["vp"], a["table"], a["lens"], a["cos"], a["sin"],
                             a["scales"], a["max_len"], W, S, a["cu"], a["shared"])


def expect(s, W=0, S=0):
    """Results and bounds (attn64).  Keys and values are exact.  A query enters in parts.
    bf16 queries: two of bf16, u^2 of it lost at most, or (4 bits) three of e2m3 at least;
    fp32: three of bf16, 2^-24, or six of e2m3.  N parts of e2m3 (steps of 1/8 up to 2, of
    1/4 up to 4, of 1/2 up to 7.5) of a group whose largest magnitude is taken to (3.75,
    7.5]: the first leaves 1/4 at most, which 2^4 takes to 4, and the second 1/8 of its unit,
    which 2^5 takes to 4, and so on: 2^-(7 + 5 (N - 2)) of the first unit, over 3.75 of
    them.  A product of parts is up to six fp32 sums where the bounds count one: 5 d E more
    of a logit's |q||k|, 2 N E of a result's sum."""
    dt, (T, Hq, d) = s["q"].dtype, s["q"].shape
    Hkv = s["kp"].shape[1]
    G, u = Hq // Hkv, unit(dt)
    out, bound = torch.zeros(T, Hq, d, dtype=torch.float64), torch.zeros(T, Hq, d, dtype=torch.float64)
    t = 0
    for b, n in enumerate(s["lens"].tolist()):
        n = min(n, s["max_len"], 64 * s["table"].shape[1])
        c = 1 if s["new"] is None else s["new"][b]
        pos = torch.arange(n - c, n)
        at = pos.clamp(0, s["cos"].shape[0] - 1) if s["cos"] is not None else None
        cs, sn = (None, None) if at is None else (s["cos"][at], s["sin"][at])
        _, q, qe = norm_rotate(s["q"][t:t + c], s["gain"], EPS, cs, sn, u * u if dt == torch.bfloat16 else E)
        qe = qe + 5 * d * E * q.abs()
        if s["bits"] == 4:
            n6 = 3 if dt == torch.bfloat16 else 6
            qe = qe + 2.0 ** -(7 + 5 * (n6 - 2)) / 3.75 * q.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
        see = visible(pos, torch.arange(max(n, 0)), W or None, S)
        for h in range(Hkv):
            if n > 0 and c > 0:
                k, v = (r[h, :n] for r in s["rows"][b])
                hs = slice(h * G, h * G + G)
                a = (see, float(s["scales"][b]), u)
                out[t:t + c, hs], bound[t:t + c, hs] = attend(q[:, hs], k, v, *a, qerr=qe[:, hs])
                bound[t:t + c, hs] += 2 * n * E * attend(q[:, hs], k, v.abs(), *a)[0]
        t += c
    return out, bound


def check(s, W=0, S=0, **kw):
    got = call(s, W, S, **kw)
    assert got.dtype == s["q"].dtype and got.shape == s["q"].shape
    assert_within(got, *expect({**s, **kw}, W, S), "out")


LENS = [[1], [0, 1, 63], [64, 65, 128, 200], [700, 3, 0, 129], [1500]]
WINDOWS = [(0, 0), (1, 0), (1, 3), (64, 0), (70, 4), (63, 65), (500, 130), (5000, 2)]


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("W,S", WINDOWS)
@pytest.mark.parametrize("lens", LENS)
def test_decode(lens, W, S, dt, d, bits):
    check(setup(DT[dt], d, bits, 4, 2, lens, seed=len(lens)), W, S)


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("W,S", [(0, 0), (2100, 0), (2200, 70)])
@pytest.mark.parametrize("lens,Hq,Hkv", [([2049], 2, 1), ([0, 4000, 1, 63, 2600], 6, 2), ([0, 0, 2200, 0], 17, 1)])
def test_long_sequences_in_even_shares(lens, Hq, Hkv, W, S, dt, d, bits):
    check(setup(DT[dt], d, bits, Hq, Hkv, lens, seed=len(lens)), W, S)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("bd", [300, 1100])
def test_many_sequences_under_a_long_bound(bd, bits):
    s = setup(torch.bfloat16, 64, bits, 2, 1, [(37 * i) % 130 for i in range(bd)], seed=3)
    s["cos"], s["sin"] = hba_amd.rope_tables(4000, 64, 1e4, "cpu")
    check({**s, "table": torch.cat([s["table"], torch.zeros(bd, 60, dtype=torch.int32)], 1), "max_len": 4000})


@pytest.mark.parametrize("dt,bits", [("f32", 4), ("bf16", 4), ("f32", 8), ("bf16", 8)])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (40, 2), (6, 6)])
def test_groups(Hq, Hkv, dt, bits):
    check(setup(DT[dt], 64, bits, Hq, Hkv, [300, 65, 1], seed=Hq))
    check(setup(DT[dt], 64, bits, Hq, Hkv, [300, 65, 1], [40, 65, 1], seed=Hq), 50, 2)
    check(setup(DT[dt], 64, bits, Hq, Hkv, [300, 165, 129], shared=128, seed=Hq))


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("W,S", WINDOWS)
@pytest.mark.parametrize("lens,new", [([1], [1]), ([5, 70, 0, 300], [5, 3, 0, 299]), ([64, 640], [64, 65]),
                                      ([129, 900, 66], [0, 130, 1]), ([3, 10], [5, 12])])
def test_parts_of_prompts(lens, new, W, S, dt, d, bits):
    """The last case: more tokens than the cache holds, the first ones see nothing."""
    check(setup(DT[dt], d, bits, 6, 2, lens, new, seed=sum(new)), W, S)


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("shared,lens", [(64, [65, 64, 100]), (128, [129, 700, 130, 300]), (640, [641] * 20),
                                         (1024, [1100, 1024, 1500]), (128, [0, 5, 128, 200])])
def test_shared_prefix(shared, lens, dt, d, bits):
    check(setup(DT[dt], d, bits, 4, 2, lens, shared=shared, seed=shared))


@pytest.mark.parametrize("dt,d,bits", FORMS)
def test_shared_prefix_with_parts(dt, d, bits):
    check(setup(DT[dt], d, bits, 4, 2, [200, 300, 128, 129], [10, 150, 0, 129], shared=128))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shared,lens,new", [(0, [40, 20], [30, 1]), (0, [900, 700], [60, 65]), (0, [5, 0], [0, 0]),
                                             (64, [200, 130], [9, 66])])
def test_padded_batch(shared, lens, new, dt):
    s = setup(DT[dt], 64, 4, 6, 2, lens, new, shared=shared, seed=3)
    T = sum(new)
    s["q"] = torch.cat([s["q"], torch.full((300, 6, 64), float("nan"), dtype=DT[dt])])
    torch.full((T + 300, 6, 64), float("nan"), dtype=DT[dt], device="cuda")   # the output's memory, perhaps
    got = call(s)
    assert not got[T:].any() and got.shape[0] == T + 300
    if T:
        want, bound = expect({**s, "q": s["q"][:T]})
        assert_within(got[:T], want, bound, "out")


@pytest.mark.parametrize("dt,bits", [("f32", 4), ("bf16", 4), ("f32", 8), ("bf16", 8)])
@pytest.mark.parametrize("new", [None, [3, 60]])
def test_no_norm_no_rotation_and_sharp_logits(new, dt, bits):
    s = setup(DT[dt], 64, bits, 4, 2, [200, 90], new, gain=False)
    check(s, cos=None, sin=None)
    check({**s, "scales": s["scales"] * 40}, cos=None, sin=None)
    check({**s, "scales": s["scales"] * 0})


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("n", [2, 40, 200])
@pytest.mark.parametrize("parts", [False, True])
def test_all_parts_of_a_query_count(parts, n, dt, d, bits):
    """Logits so large that a query without its last part is out of bounds, in the form for
    single tokens and in that for parts of prompts."""
    s = setup(DT[dt], d, bits, 7, 1, [n] * 16, [1] * 16 if parts else None, seed=n)
    check({**s, "scales": s["scales"] * 16})


@pytest.mark.parametrize("dt,bits", [("bf16", 4), ("f32", 8)])
@pytest.mark.parametrize("W", [0, 20])
@pytest.mark.parametrize("lens,new,Hq,Hkv", [
    ([70 + i % 60 for i in range(1100)], [i % 3 for i in range(1100)], 2, 1),    # more sequences than are shared out
    ([40, 700, 1], [40, 700, 1], 400, 1),                                        # more row tiles
    ([300, 9, 0, 1500, 64], [300, 0, 0, 700, 64], 3, 3),                         # a workgroup's share crosses heads
    ([2000], [1], 32, 2), ([65] * 200, [1] * 200, 2, 2)])                        # a row tile's keys in many shares; pieces of one tile
def test_parts_shared_out(lens, new, Hq, Hkv, W, dt, bits):
    check(setup(DT[dt], 64, bits, Hq, Hkv, lens, new, seed=len(lens)), W, 3 if W else 0)


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("W,S", [(0, 0), (2100, 3)])
def test_parts_of_long_prompts(W, S, dt, d, bits):
    """Keys enough for shares in 4 bits too: a tile's keys in several shares, several tiles in
    one, shares that cross heads, sequences without tokens; and logits that need every part."""
    s = setup(DT[dt], d, bits, 6, 3, [2200, 9, 0, 3000, 64, 2600], [300, 0, 0, 700, 64, 1], seed=d + bits)
    check(s, W, S)
    check({**s, "scales": s["scales"] * 16}, W, S)


def test_max_len_and_long_tables():
    s = setup(torch.bfloat16, 64, 4, 4, 2, [300, 64], maxp=9)
    check({**s, "max_len": 576})
    check({**s, "max_len": 200}, 70, 1)         # a longer length is read as max_len
    s["lens"] = torch.tensor([10 ** 6, -5], dtype=torch.int32)      # past the page table, below 0
    s["max_len"] = 10 ** 6
    kp, vp = s["kp"] * 0, s["vp"] * 0
    out = call({**s, "kp": kp, "vp": vp})
    assert bool(torch.isfinite(out.float()).all()) and bool((out[1] == 0).all())
    bad = s["table"].clone()
    bad[0, 1], bad[0, 2] = 10 ** 8, -7          # clamped into the cache
    assert bool(torch.isfinite(call({**s, "kp": kp, "vp": vp, "table": bad}).float()).all())


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("which", ["kp", "vp"])
def test_masked_groups_have_no_effect(which, dt, d, bits):
    """A group of NaN in a key or value that only some tokens of a part see."""
    W, S, n = 40, 2, 200
    s = setup(DT[dt], d, bits, 4, 2, [n], [100])
    want, bound = expect(s, W, S)
    sc = mx64.places(d, bits, which == "kp")[2]
    s[which][int(s["table"][0, 130 // 64])][:, sc[130 % 64, 1]] = 255
    if which == "vp":
        c, high, _ = mx64.places(d, bits, False)
        for t in range(32, 64):
            page = s[which][int(s["table"][0, 130 // 64])]
            page[:, c[2, t]] &= 0 if bits == 8 else 240 if not high[2, t] else 15
    got = call(s, W, S).cpu()
    pos = torch.arange(100, 200)
    sees = (pos >= 130) & (pos < 130 + W)
    assert_within(got[~sees], want[~sees], bound[~sees], "out")
    if which == "vp":
        assert got[sees][..., 32:64].isnan().all()
    else:
        assert got[sees].isnan().all()
    one = {**s, "q": s["q"][-1:], "cu": None, "new": None}       # the newest token alone does not see it either
    assert_within(call(one, W, S).cpu(), *expect(one, W, S), "out")


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("which", ["kp", "vp"])
def test_masked_groups_in_shared_out_keys(which, dt, d, bits):
    """The same where a tile's keys lie in several workgroups' shares: tokens before the group
    do not see it, those from it on do."""
    n, at = 2400, 2250
    s = setup(DT[dt], d, bits, 32, 2, [n], [300])
    want, bound = expect(s)
    sc = mx64.places(d, bits, which == "kp")[2]
    page = s[which][int(s["table"][0, at // 64])]
    page[:, sc[at % 64, 1]] = 255
    if which == "vp":
        c, high, _ = mx64.places(d, bits, False)
        for t in range(32, 64):
            page[:, c[at % 64, t]] &= 0 if bits == 8 else 240 if not high[at % 64, t] else 15
    got = call(s).cpu()
    sees = torch.arange(n - 300, n) >= at
    assert_within(got[~sees], want[~sees], bound[~sees], "out")
    assert (got[sees][..., 32:64] if which == "vp" else got[sees]).isnan().all()
    if which == "vp":
        assert_within(got[sees][..., :32], want[sees][..., :32], bound[sees][..., :32], "out")


@pytest.mark.parametrize("bits", [4, 8])
def test_shared_out_keys_in_graphs_and_streams(bits):
    """Two graphs, replayed with other queries, lengths and offsets, and both at once on two
    streams."""
    s = setup(torch.bfloat16, 64, bits, 32, 2, [2400, 2100, 64], [250, 40, 10])
    a = dev(s)
    call(a), call(a, 2100, 3)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = call(a)
    with torch.cuda.graph(g2):
        o2 = call(a, 2100, 3)
    for seed in range(3):
        a["q"].copy_(torch.randn(300, 32, 64, generator=torch.Generator().manual_seed(seed)))
        a["lens"].copy_(torch.tensor([2400 - 70 * seed, 2100, 64 - seed]))
        a["cu"].copy_(torch.tensor([0, 250 - seed, 290, 300 - 2 * seed]))
        want = call(a), call(a, 2100, 3)
        torch.cuda.synchronize()
        streams = torch.cuda.Stream(), torch.cuda.Stream()
        for g, stream in zip((g1, g2), streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want[0]) and torch.equal(o2, want[1])
        for stream in streams:
            with torch.cuda.stream(stream):
                got = call(a)
            stream.synchronize()
            assert torch.equal(got, want[0])


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("W,S", [(0, 0), (70, 4)])
@pytest.mark.parametrize("lens,new,shared", [([1, 40, 100, 350], None, 0), ([40, 70, 129, 350], [40, 3, 128, 1], 0),
                                             ([135, 200], [7, 20], 128), ([135, 200, 129], None, 128),
                                             ([2410, 70], [1400, 60], 0)])
def test_what_lies_behind_a_sequence_changes_no_bit(lens, new, shared, W, S, dt, d, bits):
    if shared and W:
        W, S = 0, 0
    s = setup(DT[dt], d, bits, 6, 2, lens, new, shared=shared, seed=len(lens))
    want = call(s, W, S)
    assert torch.isfinite(want.float()).all()
    for fill in (0, 255, 127):
        t = dict(s)
        for name, keys in (("kp", True), ("vp", False)):
            fresh = torch.full_like(s[name], fill)
            for b, n in enumerate(lens):
                for i in range((n + 63) // 64):
                    m = 64 if i < shared // 64 else min(64, n - 64 * i)
                    at = int(s["table"][b, i])
                    c, high, sc = mx64.places(d, bits, keys)
                    for h in range(2):
                        old = s[name][at, h]
                        code = old[c[:m]]
                        if bits == 4:
                            code = torch.where(high[:m], code >> 4, code & 15)
                        mx64.write(fresh[at, h], torch.arange(m), code, old[sc[:m]], bits, keys)
            t[name] = fresh
        assert torch.equal(call(t, W, S), want), fill


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new", [None, [70, 3]])
def test_pages_far_apart(new, bits):
    """The same pages at the end of a cache of over 4 GiB: attention, append and read."""
    s = setup(torch.bfloat16, 64, bits, 4, 2, [2300, 190], new)
    near = call(s)
    P, extra = s["kp"].shape[0], 2 ** 32 // s["kp"][0].numel() + 100
    far = {**s, "table": s["table"] + extra}
    for n in ("kp", "vp"):
        far[n] = torch.empty(P + extra, *s[n].shape[1:], dtype=torch.uint8, device="cuda")
        far[n][extra:] = s[n].cuda()
    assert far["kp"].numel() > 2 ** 32
    assert torch.equal(call(far), near)
    t = {**new_tokens(torch.bfloat16, 64, bits, 2, [2300, 190], [100, 190]), "table": s["table"], "kp": s["kp"], "vp": s["vp"]}
    want = append(t)
    a = dev({**t, "table": far["table"], "kp": far["kp"], "vp": far["vp"]})
    ops.kv_append_mx(a["k"], a["v"], a["cu"], a["gain"], EPS, a["cos"], a["sin"], a["table"], a["lens"], a["kp"], a["vp"])
    assert torch.equal(a["kp"][extra:].cpu(), want[0]) and torch.equal(a["vp"][extra:].cpu(), want[1])
    x = ops.kv_read_mx(a["kp"], a["vp"], a["table"], a["lens"], a["cu"], 290, 64, torch.bfloat16)
    y = ops.kv_read_mx(*(w.cuda() for w in want), s["table"].cuda(), a["lens"], a["cu"], 290, 64, torch.bfloat16)
    assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_attention_strides_streams_and_graphs():
    s = setup(torch.bfloat16, 64, 4, 4, 2, [300, 65, 700, 1])
    want = call(s)
    q = torch.randn(4, 3, 4, 64).to(torch.bfloat16)
    q[:, 1] = s["q"]
    assert torch.equal(call({**s, "q": q.cuda()[:, 1]}), want)
    assert torch.equal(call({**s, "q": torch.nn.functional.pad(s["q"], (1, 2)).cuda()[..., 1:-2]}), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(s)
    stream.synchronize()
    assert torch.equal(got, want)
    a = dev(s)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = call(a)
    with torch.cuda.graph(g2):
        o2 = call(a, 70, 4)
    for seed in range(3):
        a["q"].copy_(torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(seed)))
        a["lens"].copy_(torch.tensor([300 - seed, 65, 700 - 10 * seed, min(seed, 1)]))   # what the pages hold
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        x, y = o1.clone(), o2.clone()
        assert torch.equal(x, call(a)) and torch.equal(y, call(a, 70, 4))


def test_attention_refusals():
    s = setup(torch.float32, 64, 4, 4, 2, [100, 65])
    bad = [(0, 1, {}), (-1, 0, {}), (4, -1, {}), (5, 0, dict(shared=64)), (0, 0, dict(shared=63)),
           (0, 0, dict(shared=64 * 100)), (0, 0, dict(shared=-64)), (0, 0, dict(q=s["q"][:1])),
           (0, 0, dict(q=s["q"][:, :3])), (0, 0, dict(q=s["q"].double())), (0, 0, dict(kp=s["kp"][:-1])),
           (0, 0, dict(vp=s["vp"].int())), (0, 0, dict(kp=s["kp"][..., 1:], vp=s["vp"][..., 1:])),
           (0, 0, dict(table=s["table"].long())), (0, 0, dict(lens=s["lens"][:1])),
           (0, 0, dict(cu=torch.tensor([0, 1], dtype=torch.int32))), (0, 0, dict(scales=s["scales"][:1])),
           (0, 0, dict(gain=s["gain"][:1])), (0, 0, dict(max_len=0)), (0, 0, dict(cos=None)),
           (0, 0, dict(cos=s["cos"][:10], sin=s["sin"][:10])), (0, 0, dict(q=s["q"][0]))]
    for W, S, kw in bad:
        with pytest.raises((ValueError, TypeError)):
            call(s, W, S, **kw)
    assert call(s, q=s["q"][:0], table=s["table"][:0], lens=s["lens"][:0], scales=s["scales"][:0]).shape == (0, 4, 64)


# ----------------------------------------------------------------- together --
class TestTogether:
    """Prompts in parts, single tokens, a shared beginning, rows taken out and put back."""

    def knobs(self, dt, batch, bits, d=64):
        torch.manual_seed(0)
        cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=d)
        return cfg, hba_amd.QKNorm(cfg).cuda(), [hba_amd.MXKVCache(cfg, batch, 512, dt, "cuda", bits=bits) for _ in range(2)]

    @pytest.mark.parametrize("dt,d,bits", FORMS)
    @pytest.mark.parametrize("window,sinks", [(None, 0), (70, 4)])
    def test_prompt_then_decode(self, window, sinks, dt, d, bits):
        """In parts and single tokens, against the sliding-window operator on what the cache
        says it holds, at every token."""
        cfg, qkn, (cache, _) = self.knobs(DT[dt], 2, bits, d)
        n, dt = 333, DT[dt]
        cos, sin = hba_amd.rope_tables(512, d, 1e4, "cuda")
        q, k, v = (torch.randn(2, n, h, d, device="cuda").to(dt) for h in (4, 2, 2))
        got, at = torch.empty(2, n, 4, d, device="cuda"), [0, 0]
        for counts in ([100, 64], [1, 1], [120, 3], [50, 200], [1, 1], [61, 64]):
            part = lambda x: torch.cat([x[s, at[s]:at[s] + counts[s]] for s in range(2)])  # noqa: E731
            if counts == [1, 1]:
                cache.append(part(k), part(v), qkn, cos, sin)
                cu = None
            else:
                cu = cache.extend(part(k), part(v), counts, qkn, cos, sin)
            out = hba_amd.cache_attention(part(q), cache, cfg, qkn, cos, sin, window, sinks, cu,
                                          scales=torch.full((2,), 1 / d, device="cuda"))
            for s in range(2):
                got[s, at[s]:at[s] + counts[s]] = out[sum(counts[:s]):][:counts[s]].float()
                at[s] += counts[s]
        assert at == [n, n] == cache.lens == cache.seq_lens.tolist()
        kr, vr, _ = cache.read(dtype=torch.float32)
        # bits: what 64 bits would hold, from the keys that the formula gives
        pos = torch.arange(n)
        for s in range(2):
            want = norm_rotate(k[s].cpu(), qkn.k.gain.detach().cpu(), qkn.k.eps, cos.cpu()[pos], sin.cpu()[pos], 0.0)[1]
            c, b = mx64.quantise(want.float(), bits)
            assert torch.equal(mx64.values(c, b, bits), kr.view(2, n, 2, d)[s].double().cpu())
        qr = torch.stack([norm_rotate(q[s].cpu(), qkn.q.gain.detach().cpu(), qkn.q.eps, cos.cpu()[pos], sin.cpu()[pos], 0.0)[1]
                          for s in range(2)]).float().cuda()
        want = hba_amd.sliding_attention(qr, kr.view(2, n, 2, d), vr.view(2, n, 2, d), window or n, sinks, scale=1 / d)
        # fp32: sums' orders and roundings of q; bf16: the probabilities' rounding and the result's, of values up to 5
        assert float((got - want).abs().max()) <= (d * 2.0 ** -20 if dt == torch.float32 else 5 * 2.0 ** -7)

    @pytest.mark.parametrize("bits", [4, 8])
    def test_shared_beginning_and_rows_put_back(self, bits):
        dt = torch.bfloat16
        cfg, qkn, (a, b) = self.knobs(dt, 3, bits)
        cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cuda")
        k, v = (torch.randn(200, 2, 64, device="cuda").to(dt) for _ in range(2))
        a.extend(k, v, [200, 0, 0], qkn, cos, sin)
        a.share(0, 192, [1, 2])
        b.extend(torch.cat((k, k[:192], k[:192])), torch.cat((v, v[:192], v[:192])), [200, 192, 192], qkn, cos, sin)
        assert len(a._free) == len(b._free) + 6
        k, v = (torch.randn(150, 2, 64, device="cuda").to(dt) for _ in range(2))
        for c in (a, b):
            cu = c.extend(k, v, [20, 0, 130], qkn, cos, sin)
        q = torch.randn(150, 4, 64, device="cuda").to(dt)
        x = hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, cu=cu, shared=192)
        y = hba_amd.cache_attention(q, b, cfg, qkn, cos, sin, cu=cu)
        assert float((x.float() - y.float()).abs().max()) <= 2e-2
        k, v = (torch.randn(3, 2, 64, device="cuda").to(dt) for _ in range(2))
        for c in (a, b):
            c.append(k, v, qkn, cos, sin)
        q = torch.randn(3, 4, 64, device="cuda").to(dt)
        x = hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, shared=192)
        y = hba_amd.cache_attention(q, b, cfg, qkn, cos, sin)
        assert float((x.float() - y.float()).abs().max()) <= 2e-2
        with pytest.raises(ValueError):
            hba_amd.cache_attention(q, b, cfg, qkn, cos, sin, shared=192)
        for m, n, p in zip(a.read(), b.read(), a.read([221, 193, 323])):
            assert torch.equal(m, n) and torch.equal(m, p)
        # out of one cache into another: the same bytes, so the same attention
        kr, vr, cu = b.read()
        other = hba_amd.MXKVCache(cfg, 3, 512, dt, "cuda", bits=bits)
        at = cu.tolist()
        for s in (2, 0, 1):
            other.load(s, kr[at[s]:at[s + 1]], vr[at[s]:at[s + 1]])
        assert torch.equal(hba_amd.cache_attention(q, other, cfg, qkn, cos, sin), y)
        page = b._table[2][1]
        assert torch.equal(b.key_rows(page), kr[at[2] + 64:at[2] + 128].transpose(0, 1))
        assert torch.equal(b.value_rows(torch.tensor([[page]]))[0, 0], vr[at[2] + 64:at[2] + 128].transpose(0, 1))

    def test_8_bits_are_near_the_whole_cache_and_4_bits_nearer_than_nothing(self):
        """The caches of 16, 8 and 4 bits of the same tokens: an element is off by 2^-4 of its
        size at most in 8 bits (or by 2^-10 of its group's largest), in 4 by a seventh of
        the group's largest or a quarter of its own."""
        dt = torch.float32
        torch.manual_seed(3)
        cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
        qkn, summ = hba_amd.QKNorm(cfg).cuda(), hba_amd.SlotSummarizer(cfg).cuda()
        cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cuda")
        k, v = (torch.randn(300, 2, 64, device="cuda") for _ in range(2))
        whole = hba_amd.PagedKVCache(cfg, 1, 512, dt, "cuda")
        whole.extend(k, v, [300], qkn, summ, cos, sin)
        pages = torch.tensor(whole._table[0], device="cuda")
        kr = whole.key_rows(pages, rotated=True).transpose(1, 2).reshape(-1, 2, 64)[:300]
        for bits in (8, 4):
            c = hba_amd.MXKVCache(cfg, 1, 512, dt, "cuda", bits=bits)
            c.extend(k, v, [300], qkn, cos, sin)
            for x, y in zip((kr, v), c.read()[:2]):
                g, h = x.unflatten(-1, (-1, 32)), y.unflatten(-1, (-1, 32))
                big = g.abs().amax(-1, keepdim=True)
                near = torch.maximum(g.abs() / 16, big / 1024) if bits == 8 else torch.maximum(g.abs() / 4, big / 7)
                assert bool(((g - h).abs() <= near * (1 + 2.0 ** -16)).all())
