"""Sliding-window attention with sinks (hba_amd.sliding_attention) against 64-bit
results: forward and gradients, lengths of one token to several tiles, windows and
sinks at tile borders, padded batches, strides, and what masked places may hold."""
import pytest
import torch

import hba_amd
from attn64 import assert_within, attend, sliding, unit
from hba_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(dt, B, n, Hq, Hkv, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, n, h, d, generator=g).to(dt) for h in (Hq, Hkv, Hkv, Hq)]


def run(q, k, v, W, S, scale=None, lens=None, dout=None):
    q, k, v = (t.cuda() for t in (q, k, v))
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32).cuda()
    if dout is None:
        return hba_amd.sliding_attention(q, k, v, W, S, scale, lens)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = hba_amd.sliding_attention(q, k, v, W, S, scale, lens)
    return (out, *torch.autograd.grad(out, (q, k, v), dout.cuda()))


def compare(got, q, k, v, W, S, scale, lens, dout=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, bound = sliding(q, k, v, W, S, scale, lens, unit(q.dtype), dout)
    if dout is None:
        got, want, bound = [got], [want], [bound]
    for name, a, b, c in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert a.dtype == q.dtype
        assert_within(a, b, c, name)


# n, W, S: one token; below, at and past a tile; a window of one key, at, past and
# off tile borders, as long as the sequence; sinks of none, some, over a tile, all
SIZES = [(1, 1, 0), (1, 64, 4), (2, 1, 0), (5, 3, 2), (63, 64, 0), (64, 64, 4), (65, 32, 1), (127, 1, 64),
         (130, 65, 63), (200, 17, 65), (257, 128, 4), (300, 299, 0), (301, 1000, 7), (333, 40, 333),
         (449, 100, 130)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,W,S", SIZES)
def test_forward_and_gradients(n, W, S, dt, d):
    q, k, v, do = make(DT[dt], 1, n, 4, 2, d, seed=n + W)
    compare(run(q, k, v, W, S), q, k, v, W, S, None, None)
    compare(run(q, k, v, W, S, dout=do), q, k, v, W, S, None, None, do)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,W,S", [(128, 128, 0), (190, 129, 66), (255, 255, 0), (256, 256, 0), (320, 256, 70), (700, 600, 3),
                                   (961, 2000, 0)])
@pytest.mark.parametrize("lens", [None, [0, 128], [100, 64]])
def test_few_rows_and_many_keys(n, W, S, lens, dt, d):
    """Sets of waves share the keys: odd and even tile counts, and workgroups without any."""
    q, k, v, _ = make(DT[dt], 2, n, 3, 1, d, seed=n)
    x = [t.clone() for t in (q, k, v)]
    for b, m in enumerate(lens or []):
        for t in x:
            t[b, m:] = float("nan")
    compare(run(*x, W, S, lens=lens), q, k, v, W, S, None, lens)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_two_sets_of_waves(dt, d):
    """More rows than four sets would have workgroups for."""
    q, k, v, _ = make(DT[dt], 2, 900, 14, 2, d, seed=5)
    compare(run(q, k, v, 300, 2, lens=[900, 511]), q, k, v, 300, 2, None, [900, 511])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_few_rows_spoiled(bad, dt):
    """A non-finite key or value spoils the rows that see it, whichever set of waves has it."""
    for at in (5, 300, 590):
        q, k, v, _ = make(DT[dt], 1, 600, 2, 1, 64, seed=at)
        want, bound = sliding(q, k, v, 300, 2, 64 ** -0.5, None, unit(q.dtype))
        k2, v2 = k.clone(), v.clone()
        k2[0, at], v2[0, at] = bad, bad
        got = run(q, k2, v2, 300, 2).cpu()
        sees = torch.arange(600)
        sees = (sees >= at) & (sees < at + 300)
        assert not got[0, sees].isfinite().any()
        assert_within(got[:, ~sees], want[:, ~sees], bound[:, ~sees], "out")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (14, 2), (8, 1), (33, 1), (6, 2)])
def test_groups(Hq, Hkv, dt):
    q, k, v, do = make(DT[dt], 2, 150, Hq, Hkv, 64, seed=Hq)
    compare(run(q, k, v, 50, 3, dout=do), q, k, v, 50, 3, None, None, do)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[0, 1, 200], [200, 64, 63], [130, 0, 0], [-5, 999, 65]])
def test_padded_batch(lens, dt):
    """Rows behind a sequence give 0 and have no effect, whatever they hold."""
    q, k, v, do = make(DT[dt], 3, 200, 4, 2, 64, seed=3)
    clamped = [max(0, min(200, x)) for x in lens]
    dirty = [t.clone() for t in (q, k, v, do)]
    for t in dirty:
        for b, m in enumerate(clamped):
            t[b, m:] = float("nan")
    got = run(*dirty[:3], 70, 5, lens=lens, dout=dirty[3])
    compare(got, q, k, v, 70, 5, None, clamped, do)
    for t in got:
        for b, m in enumerate(clamped):
            assert bool((t[b, m:] == 0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_scale_and_long_parts(dt):
    """A scale other than the default, and sinks that later rows see in several parts."""
    q, k, v, do = make(DT[dt], 1, 1500, 2, 1, 64, seed=5)
    compare(run(q, k, v, 64, 10, scale=0.3, dout=do), q, k, v, 64, 10, 0.3, None, do)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_large_logits(dt):
    """Maxima that grow from tile to tile: every rescaling of the running sums."""
    q, k, v, do = make(DT[dt], 1, 300, 2, 2, 64, seed=6)
    k = (k.float() * torch.linspace(0.1, 30, 300)[None, :, None, None]).to(k.dtype)
    compare(run(q, k, v, 200, 2, dout=do), q, k, v, 200, 2, None, None, do)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_places_have_no_effect(bad, dt):
    """A non-finite key, value, query or cotangent spoils only what sees it."""
    W, S, n, at = 40, 3, 200, 100
    q, k, v, do = make(DT[dt], 1, n, 4, 2, 64, seed=7)
    i = torch.arange(n)
    clean = run(q, k, v, W, S, dout=do)
    sees = (i >= at) & (i < at + W)              # the rows that see key `at`
    seen = ((i <= at) & (i > at - W)) | (i < S)  # the keys that row `at` sees
    for which in range(4):
        dirty = [t.clone() for t in (q, k, v, do)]
        dirty[which][:, at] = bad
        out, dq, dk, dv = run(*dirty[:3], W, S, dout=dirty[3])
        if which in (1, 2):                      # the keys' rows: through the rows that see them
            rows = sees
            keys = torch.zeros(n, dtype=torch.bool)
            for t in i[sees].tolist():
                keys |= ((i <= t) & (i > t - W)) | (i < S)
        else:
            rows, keys = i == at, seen
        for name, a, b, hit in (("out", out, clean[0], rows), ("dq", dq, clean[1], rows),
                                ("dk", dk, clean[2], keys), ("dv", dv, clean[3], keys)):
            a, b = a[:, ~hit].float().cpu(), b[:, ~hit].float().cpu()
            # computed again key by key: the same up to the roundings of two orders
            assert torch.isfinite(a).all(), (which, name)
            assert float((a - b).abs().max().detach()) <= (2e-2 if dt == "bf16" else 1e-5) * max(1.0, float(b.abs().max()))
        if which == 2:                           # a visible infinity arrives as it is
            assert not bool(torch.isfinite(out[:, sees].float()).any())


def test_visible_infinity_in_one_element():
    q, k, v, _ = make(torch.float32, 1, 100, 2, 1, 64, seed=8)
    v[0, 50, 0, 7] = float("inf")
    out = run(q, k, v, 20, 0)[0].cpu()
    hit = torch.zeros(100, dtype=torch.bool)
    hit[50:70] = True
    assert bool((out[hit][:, :, 7] == float("inf")).all())
    out[:, :, 7] = 0
    assert bool(torch.isfinite(out).all())
    assert bool(torch.isfinite(run(q, k, v, 20, 0)[0].cpu()[~hit]).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strided_views(dt):
    """One projection's output as q, k and v; heads before tokens; rows off 16 bytes."""
    g = torch.Generator().manual_seed(9)
    B, n, Hq, Hkv, d = 2, 90, 4, 2, 64
    qkv = torch.randn(B, n, Hq + 2 * Hkv, d, generator=g).to(DT[dt]).cuda()
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    want = hba_amd.sliding_attention(q.clone(), k.clone(), v.clone(), 33, 4)
    assert torch.equal(hba_amd.sliding_attention(q, k, v, 33, 4), want)
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(hba_amd.sliding_attention(*hm, 33, 4), want)
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (q, k, v)]
    assert torch.equal(hba_amd.sliding_attention(*odd, 33, 4), want)
    flip = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]
    assert torch.equal(hba_amd.sliding_attention(*flip, 33, 4), want)
    x = [t.detach().requires_grad_() for t in odd]
    o = hba_amd.sliding_attention(*x, 33, 4)
    a = torch.autograd.grad(o, x, torch.ones((), dtype=DT[dt], device="cuda").expand_as(o))
    y = [t.clone().requires_grad_() for t in (q, k, v)]
    b = torch.autograd.grad(hba_amd.sliding_attention(*y, 33, 4), y, torch.ones_like(want))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_rows_far_apart():
    """Rows just under 16 MiB apart: offsets within a sequence pass 32 bits."""
    q, k, v, do = make(torch.bfloat16, 1, 290, 4, 2, 64)
    far = torch.empty(290, 2 ** 23 - 64, dtype=torch.bfloat16, device="cuda")
    views = []
    for i, t in enumerate((q, k, v, do)):
        x = far[:, 1024 * i:1024 * i + t.shape[2] * 64].unflatten(1, (t.shape[2], 64))[None]
        x.copy_(t)
        views.append(x)
    leaves = [x.detach().requires_grad_() for x in views[:3]]
    out = hba_amd.sliding_attention(*leaves, 100, 3)
    compare((out, *torch.autograd.grad(out, leaves, views[3])), q, k, v, 100, 3, None, None, do)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_thousands_of_sinks(dt):
    """As many sinks as keys: tiles of sinks have longer parts than the others would."""
    n = 9000
    q, k, v, do = make(DT[dt], 1, n, 1, 1, 64, seed=9)
    got = run(q, k, v, 1, n, dout=do)
    i = torch.arange(n, device="cuda")
    want, bound = attend(q[0].cuda(), k[0, :, 0].cuda(), v[0, :, 0].cuda(), i[None] <= i[:, None], 64 ** -0.5,
                         unit(DT[dt]), do[0].cuda())
    for name, x, y, z in zip(("out", "dq", "dk", "dv"), got, want, bound):
        x = x[0] if name in ("out", "dq") else x[0, :, 0]
        assert_within(x, y.cpu(), z.cpu(), name)


def test_gradients_match_differences():
    q, k, v, do = make(torch.float32, 1, 70, 2, 1, 64, seed=10)
    _, *grads = run(q, k, v, 30, 2, dout=do)
    g = torch.Generator().manual_seed(11)
    for which, grad in enumerate(grads):
        x = [t.double() for t in (q, k, v)]
        way = torch.randn(x[which].shape, generator=g, dtype=torch.float64)
        step = 1e-4
        f = []
        for sign in (1, -1):
            y = list(x)
            y[which] = y[which] + sign * step * way
            f.append(float((sliding(*y, 30, 2, 64 ** -0.5, None, 0.0)[0] * do.double()).sum()))
        got = float((grad.double().cpu() * way).sum())
        size = float((grad.double().cpu() * way).abs().sum())
        assert abs(got - (f[0] - f[1]) / (2 * step)) <= 1e-5 * size


def test_same_bits_every_time_and_only_needed_gradients():
    q, k, v, do = (t.cuda() for t in make(torch.bfloat16, 2, 700, 14, 2, 64, seed=12))
    x = [t.requires_grad_() for t in (q, k, v)]
    first = torch.autograd.grad(hba_amd.sliding_attention(*x, 100, 4), x, do)
    for _ in range(3):
        again = torch.autograd.grad(hba_amd.sliding_attention(*x, 100, 4), x, do)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    kk = k.detach().requires_grad_()
    one, = torch.autograd.grad(hba_amd.sliding_attention(q.detach(), kk, v.detach(), 100, 4), kk, do)
    assert torch.equal(one, first[1])


def test_empty_batch_and_other_stream():
    q = torch.randn(0, 10, 4, 64, device="cuda")
    k = torch.randn(0, 10, 2, 64, device="cuda")
    assert hba_amd.sliding_attention(q, k, k, 5).shape == q.shape
    q = torch.randn(2, 0, 4, 64, device="cuda").requires_grad_()
    k = torch.randn(2, 0, 2, 64, device="cuda")
    hba_amd.sliding_attention(q, k, k, 5).sum().backward()
    assert q.grad.shape == q.shape
    q, k, v, _ = (t.cuda() for t in make(torch.bfloat16, 1, 300, 4, 2, 64))
    want = hba_amd.sliding_attention(q, k, v, 50, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = hba_amd.sliding_attention(q, k, v, 50, 2)
    s.synchronize()
    assert torch.equal(got, want)


def test_graph_replays():
    """Forward and backward captured once and replayed, with eager work between."""
    q, k, v, do = (t.cuda() for t in make(torch.bfloat16, 1, 260, 4, 2, 64, seed=13))
    x = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = hba_amd.sliding_attention(*x, 70, 3)
        return (o.detach(), *torch.autograd.grad(o, x, do))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        for t, new in zip((q, k, v, do), make(torch.bfloat16, 1, 260, 4, 2, 64, seed=20 + seed)):
            t.data.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_custom_ops_agree():
    q, k, v, do = (t.cuda() for t in make(torch.bfloat16, 1, 100, 4, 2, 64))
    out, lse = torch.ops.hba.swa_fwd(q, k, v, None, 30, 2, 0.125)
    assert torch.equal(out, hba_amd.sliding_attention(q, k, v, 30, 2, 0.125))
    x = [t.requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(hba_amd.sliding_attention(*x, 30, 2, 0.125), x, do)
    got = torch.ops.hba.swa_bwd(q, k, v, out, lse, do, None, 30, 2, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_traced():
    """In a traced graph the registered operators stand for the calls."""
    q, k, v, do = (t.cuda() for t in make(torch.bfloat16, 2, 70, 4, 2, 64))
    lens = torch.tensor([70, 33], device="cuda")

    def f(q, k, v):
        return hba_amd.sliding_attention(q, k, v, 20, 3, lens=lens)

    torch.compiler.reset()
    traced = torch.compile(f, backend="aot_eager", fullgraph=True)
    assert torch.equal(traced(q, k, v), f(q, k, v))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(f(*leaves), leaves, do)
    got = torch.autograd.grad(traced(*leaves), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_lse():
    q, k, v, _ = make(torch.float32, 1, 150, 2, 1, 64)
    _, lse = ops.swa_fwd(q.cuda(), k.cuda(), v.cuda(), None, 40, 1, 0.125)
    from attn64 import visible
    i = torch.arange(150)
    x = torch.einsum("ihd,jd->hij", q[0].double(), k[0, :, 0].double()) * 0.125
    x = x.masked_fill(~visible(i, i, 40, 1), float("-inf"))
    want = torch.logsumexp(x, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
    assert float((lse[0].double().cpu() - want).abs().max()) < 1e-5


def test_refusals():
    q, k, v, _ = (t.cuda() for t in make(torch.float32, 1, 20, 4, 2, 64))
    f = hba_amd.sliding_attention
    for args in ((q, k, v, 0), (q, k, v, 4, -1), (q, k, v, 4, 0, 0.0), (q, k, v, 4, 0, -1.0),
                 (q, k, v, 4, 0, float("inf")), (q, k, v, 4, 0, float("nan")), (q, k[:, :10], v, 4),
                 (q, k, v[:, :10], 4), (q[:, :, :3], k, v, 4), (q[0], k[0], v[0], 4),
                 (q, k, v, 4, 0, None, torch.ones(2, dtype=torch.int32)), (q, k, v, 4, 0, None, torch.ones(1)),
                 (q, k.cpu(), v, 4)):
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(TypeError):
        f(q, k.bfloat16(), v, 4)
    with pytest.raises(TypeError):
        f(q.half(), k.half(), v.half(), 4)
    with pytest.raises(ops.check.__globals__["HBAError"]):
        f(q[..., :32], k[..., :32], v[..., :32], 4)
