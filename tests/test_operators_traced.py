"""The window and cache operators where something records or transforms what runs: a
recorded graph holds the operator, not the memory of one call's result."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import hba_amd
from hba_amd import ops

EPS = 1e-6


def window(q, k, v):
    return hba_amd.sliding_attention(q, k, v, 20, 3)


def cache(dev, dt=torch.bfloat16, seed=0):
    """Two sequences of 5 and 100 tokens, 2 and 66 of them new: the arguments of both operators."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dt).to(dev)  # noqa: E731
    i = lambda x: torch.tensor(x, dtype=torch.int32).to(dev)  # noqa: E731
    cos, sin = (t.to(dev) for t in hba_amd.rope_tables(128, 64, 1e4, "cpu"))
    return dict(k=r(68, 2, 64), v=r(68, 2, 64), cu=i([0, 2, 68]), cos=cos, sin=sin, table=i([[3, 0], [1, 2]]),
                lens=i([5, 100]), kc=r(4, 2, 4096), kr=r(4, 2, 4096), vp=r(4, 2, 4096),
                probes=r(2, 4, 64).float(), proj=r(2, 64, 64).float(), summ=r(4, 2, 4, 64), q=r(68, 4, 64),
                gain=torch.ones(4).to(dev), scales=torch.full((2,), 1 / 64).to(dev))


def append(a):
    ops.kv_append_ragged(a["k"], a["v"], a["cu"], a["gain"][:2], EPS, a["cos"], a["sin"], a["table"], a["lens"],
                         a["kc"], a["kr"], a["vp"], a["probes"], a["proj"], a["summ"])
    return a["kr"]


def attend(a):
    return ops.paged_attn(a["q"], a["gain"], EPS, a["kr"], a["vp"], a["table"], a["lens"], a["cos"], a["sin"],
                          a["scales"], 128, cu=a["cu"])


def targets(g):
    return [str(n.target) for n in g.graph.nodes if n.op == "call_function"]


def test_eager_calls_go_past_the_dispatcher_and_nothing_else_does():
    t = torch.zeros(2, 2)
    assert ops._plain(t, None, torch.nn.Parameter(t))
    for state in (torch.no_grad(), torch.inference_mode(), torch.autocast("cpu", dtype=torch.bfloat16)):
        with state:
            assert ops._plain(t)
    seen = []

    def f(x):
        seen.append(ops._plain(x))
        return x * 2

    make_fx(f)(t)
    make_fx(f, pre_dispatch=True)(t)
    make_fx(f, tracing_mode="fake")(t)
    torch.jit.trace(f, (t,), check_trace=False)
    torch.func.vmap(f)(t)
    torch.func.jvp(f, (t,), (t,))
    torch.func.functionalize(f)(t)
    with FakeTensorMode() as mode:
        f(torch.zeros(2))
    assert not any(seen) and len(seen) == 8
    assert not ops._plain(mode.from_tensor(t))


@pytest.mark.parametrize("pre", [False, True])
def test_recorded_calls_of_tensors_without_memory(pre):
    with FakeTensorMode():
        q, k = torch.empty(1, 30, 4, 64, device="cuda"), torch.empty(1, 30, 2, 64, device="cuda")
        assert window(q, k, k).shape == q.shape
        assert "hba.swa_fwd.default" in targets(make_fx(window, pre_dispatch=pre)(q, k, k))
        a = cache("cuda")
        assert attend(a).shape == a["q"].shape and append(a) is a["kr"]
        assert "hba.paged_attn.default" in targets(make_fx(attend, pre_dispatch=pre)(a))
        assert "hba.kv_append_ragged.default" in targets(make_fx(append, pre_dispatch=pre)(a))


def recorded(f, args, how):
    return torch.jit.trace(f, args, check_trace=False) if how == "jit" else make_fx(f, pre_dispatch=how == "pre")(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["fx", "pre", "jit"])
def test_recorded_window(how):
    x = [torch.randn(1, 70, h, 64, device="cuda") for h in (4, 2, 2)]
    f = recorded(window, tuple(x), how)
    for t in x:
        t.normal_()
    y = [torch.randn_like(t) for t in x]
    for z in (x, y):
        assert torch.equal(f(*z), window(*z))


@pytest.mark.gpu
def test_recorded_gradients():
    x = [torch.randn(1, 70, h, 64, device="cuda") for h in (4, 2, 2, 4)]

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = window(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    g = make_fx(step)(*x)
    assert "hba.swa_fwd.default" in targets(g) and "hba.swa_bwd.default" in targets(g)
    x = [torch.randn_like(t) for t in x]
    assert all(torch.equal(a, b) for a, b in zip(g(*x), step(*x)))


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["fx", "pre", "jit"])
def test_recorded_cache_calls(how):
    names = list(cache("cpu"))

    def both(*ts):
        a = dict(zip(names, ts))
        append(a)
        return attend(a)

    f = recorded(both, tuple(cache("cuda").values()), how)
    a, b = cache("cuda", seed=1), cache("cuda", seed=1)
    got, want = f(*a.values()), both(*b.values())
    assert torch.equal(got, want)
    assert all(torch.equal(a[n], b[n]) for n in ("kc", "kr", "vp", "summ"))
    assert not torch.equal(a["kr"], cache("cuda", seed=1)["kr"])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "gain", "kr", "vp", "scales"])
def test_cache_attention_says_that_it_has_no_gradient(name):
    a = cache("cuda")
    want = attend(a)
    a[name].requires_grad_()
    got = attend(a)
    assert torch.equal(got, want) and got.requires_grad
    with pytest.raises(NotImplementedError):
        got.sum().backward()
    with torch.no_grad():
        assert not attend(a).requires_grad


@pytest.mark.gpu
def test_tangents_are_not_dropped():
    a = cache("cuda")
    q, k = torch.randn(1, 30, 4, 64, device="cuda"), torch.randn(1, 30, 2, 64, device="cuda")
    want = window(q, k, k)
    with forward_ad.dual_level():
        assert torch.equal(window(q, k, k), want)
        with pytest.raises(NotImplementedError):
            window(forward_ad.make_dual(q, q), k, k)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            window(q, k, forward_ad.make_dual(k, k))
        with pytest.raises(NotImplementedError):
            attend({**a, "q": forward_ad.make_dual(a["q"], a["q"])})
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: window(x, k, k), (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: attend({**a, "q": x}), (a["q"],), (a["q"],))


@pytest.mark.gpu
def test_compiled_cache_calls():
    """As the registered operators; a graph with a gradient through paged_attn is refused."""
    def both(a):
        append(a)
        return attend(a)

    torch.compiler.reset()
    f = torch.compile(both, backend="aot_eager", fullgraph=True)
    a, b = cache("cuda", seed=1), cache("cuda", seed=1)
    for x in (a, b):
        x["gain"].requires_grad_()
    with torch.no_grad():
        assert torch.equal(f(a), both(b))
    assert all(torch.equal(a[n], b[n]) for n in ("kc", "kr", "vp", "summ"))
    with pytest.raises(Exception, match="backward through hba.paged_attn"):
        f(a)


@pytest.mark.gpu
def test_mapped_calls():
    """vmap runs the registered operator for each; what it cannot map it refuses."""
    x = [torch.randn(3, 1, 30, h, 64, device="cuda") for h in (4, 2, 2)]
    want = torch.stack([window(*(t[i] for t in x)) for i in range(3)])
    assert torch.equal(torch.func.vmap(window)(*x), want)
    assert torch.equal(torch.func.vmap(window, (0, None, None))(x[0], x[1][0], x[2][0]),
                       torch.stack([window(x[0][i], x[1][0], x[2][0]) for i in range(3)]))
    a = cache("cuda")
    q = torch.randn(3, *a["q"].shape, device="cuda").bfloat16()
    got = torch.func.vmap(lambda t: attend({**a, "q": t}))(q)
    assert torch.equal(got, torch.stack([attend({**a, "q": t}) for t in q]))
    before = {n: a[n].clone() for n in ("kc", "kr", "vp", "summ")}
    k = torch.randn(3, *a["k"].shape, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: append({**a, "k": t}))(k)
    assert all(torch.equal(a[n], before[n]) for n in before)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: window(t, x[1][0], x[2][0]).sum())(x[0][0])
