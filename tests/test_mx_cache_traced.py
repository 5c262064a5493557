"""The operators of the cache in 4 and 8 bits where something records or transforms what
runs, and where a derivative is asked for."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from hba_amd import ops
from test_operators_traced import EPS, recorded, targets
from test_operators_traced import cache as plain_cache


def cache(dev, seed=0):
    """Two sequences of 5 and 100 tokens, 2 and 66 of them new."""
    a = plain_cache(dev, seed=seed)
    g = torch.Generator().manual_seed(seed)
    for n in ("kr", "vp"):
        p = torch.randint(0, 256, (4, 2, ops.mx_page_bytes(64, 4)), generator=g).to(torch.uint8)
        p[..., 2048:] = 120
        a[n] = p.to(dev)
    return {n: a[n] for n in ("k", "v", "cu", "cos", "sin", "table", "lens", "kr", "vp", "q", "gain", "scales")}


def append(a):
    ops.kv_append_mx(a["k"], a["v"], a["cu"], a["gain"][:2], EPS, a["cos"], a["sin"], a["table"], a["lens"], a["kr"], a["vp"])
    return a["kr"]


def read(a):
    return ops.kv_read_mx(a["kr"], a["vp"], a["table"], a["lens"], a["cu"], 68, 64, torch.bfloat16)


def attend(a):
    return ops.paged_attn_mx(a["q"], a["gain"], EPS, a["kr"], a["vp"], a["table"], a["lens"], a["cos"], a["sin"],
                             a["scales"], 128, cu=a["cu"])


def all_three(a):
    append(a)
    return (*read(a), attend(a))


@pytest.mark.parametrize("pre", [False, True])
def test_recorded_calls_of_tensors_without_memory(pre):
    with FakeTensorMode():
        a = cache("cuda")
        assert append(a) is a["kr"] and attend(a).shape == a["q"].shape
        assert [(tuple(x.shape), x.dtype) for x in read(a)] == [((68, 2, 64), torch.bfloat16)] * 2
        found = targets(make_fx(all_three, pre_dispatch=pre)(a))
        assert all(f"hba.{n}.default" in found for n in ("kv_append_mx", "kv_read_mx", "paged_attn_mx"))


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["fx", "pre", "jit"])
def test_recorded_calls(how):
    names = list(cache("cpu"))
    f = recorded(lambda *ts: all_three(dict(zip(names, ts))), tuple(cache("cuda").values()), how)
    a, b = cache("cuda", seed=1), cache("cuda", seed=1)
    for x, y in zip(f(*a.values()), all_three(b)):
        assert torch.equal(x, y)
    assert all(torch.equal(a[n], b[n]) for n in ("kr", "vp"))
    assert not torch.equal(a["kr"], cache("cuda", seed=1)["kr"])


@pytest.mark.gpu
def test_compiled_calls():
    torch.compiler.reset()
    f = torch.compile(all_three, backend="aot_eager", fullgraph=True)
    a, b = cache("cuda", seed=1), cache("cuda", seed=1)
    for x in (a, b):
        x["q"].requires_grad_()
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(f(a), all_three(b)))
    assert all(torch.equal(a[n], b[n]) for n in ("kr", "vp"))
    with pytest.raises(Exception, match="backward through hba.paged_attn_mx"):
        f(a)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "gain", "scales"])
def test_attention_says_that_it_has_no_gradient(name):
    a = cache("cuda")
    want = attend(a)
    a[name].requires_grad_()
    got = attend(a)
    assert torch.equal(got, want) and got.requires_grad
    with pytest.raises(NotImplementedError, match="paged_attn_mx"):
        got.sum().backward()
    with torch.no_grad():
        assert not attend(a).requires_grad


@pytest.mark.gpu
def test_tangents_are_not_dropped():
    a = cache("cuda")
    with forward_ad.dual_level():
        assert torch.equal(attend(a), attend(a))
        with pytest.raises(NotImplementedError):
            attend({**a, "q": forward_ad.make_dual(a["q"], a["q"])})
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: attend({**a, "q": x}), (a["q"],), (a["q"],))


@pytest.mark.gpu
def test_autograd_sees_the_append():
    a = cache("cuda")
    for n in ("kr", "vp"):
        before = a[n]._version
        append(a)
        assert a[n]._version > before
    with torch.inference_mode():
        b = {n: t.clone() for n, t in a.items()}
    append(b)


@pytest.mark.gpu
def test_mapped_calls():
    a = cache("cuda")
    q = torch.randn(3, *a["q"].shape, device="cuda").bfloat16()
    got = torch.func.vmap(lambda t: attend({**a, "q": t}))(q)
    assert torch.equal(got, torch.stack([attend({**a, "q": t}) for t in q]))
    before = {n: a[n].clone() for n in ("kr", "vp")}
    k = torch.randn(3, *a["k"].shape, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: append({**a, "k": t}))(k)
    assert all(torch.equal(a[n], before[n]) for n in before)
