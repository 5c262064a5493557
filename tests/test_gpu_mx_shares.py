"""Attention over the cache in 4 and 8 bits where keys are shared out over the workgroups: the
batches of mx_plan, which reach that code (test_mx_plan_host.py), against 64-bit results."""
import pytest
import torch

import hba_amd
import mx_plan
import test_gpu_mx_cache as mxc
from mx_plan import DECODE, PARTS
from test_gpu_mx_cache import DT, FORMS, assert_within, call, check, expect, setup

pytestmark = pytest.mark.gpu


def wide(s, max_len):
    """The same sequences under a bound and a page table that are far above their lengths."""
    d, more = s["q"].shape[2], mx_plan.ceil(max_len, 64) - s["table"].shape[1]
    cos, sin = hba_amd.rope_tables(max_len, d, 1e4, "cpu")
    return {**s, "table": torch.nn.functional.pad(s["table"], (0, more)), "max_len": max_len, "cos": cos, "sin": sin}


@pytest.mark.parametrize("dt,d,bits", [("bf16", 64, 4), ("bf16", 128, 8), ("f32", 128, 4), ("f32", 64, 8)])
@pytest.mark.parametrize("name", PARTS)
def test_parts_of_prompts(name, dt, d, bits):
    lens, new, Hq, Hkv, max_len = PARTS[name]
    s = wide(setup(DT[dt], d, bits, Hq, Hkv, lens, new, seed=len(lens)), max_len)
    for W, S in ((0, 0), (2100, 3), (20, 3)):
        check(s, W, S)


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("name", ["a share crosses heads", "a tile in many shares", "tokens behind the cache"])
def test_every_form(name, dt, d, bits):
    """Sharp logits, so that each part of a query and each share's maximum counts."""
    lens, new, Hq, Hkv, max_len = PARTS[name]
    s = wide(setup(DT[dt], d, bits, Hq, Hkv, lens, new, seed=d + bits), max_len)
    check({**s, "scales": s["scales"] * 16})


@pytest.mark.parametrize("dt,d,bits", FORMS)
def test_padded_batch(dt, d, bits):
    """Tokens before the first sequence's and behind the last one's, of NaN, give 0."""
    lens, new = [300, 9, 0, 1500, 64], [300, 0, 0, 200, 64]
    s = wide(setup(DT[dt], d, bits, 6, 3, lens, new, seed=d), 20000)
    T = sum(new)
    assert mx_plan.workspace(bits, T + 110, 5, 6, 3, d, 0, 0, 0, 20000)[0] == "shares"
    want, bound = expect(s)
    for front, behind in ((0, 110), (37, 0), (70, 40)):
        nan = torch.full((front + behind, 6, d), float("nan"), dtype=DT[dt])
        pad = {**s, "q": torch.cat((nan[:front], s["q"], nan[front:])), "cu": s["cu"] + front}
        torch.full(pad["q"].shape, float("nan"), dtype=DT[dt], device="cuda")   # the output's memory, perhaps
        got = call(pad)
        assert not got[:front].any() and not got[front + T:].any() and got.shape[0] == front + T + behind
        assert_within(got[front:front + T], want, bound, "out")


@pytest.mark.parametrize("dt,d,bits", FORMS)
@pytest.mark.parametrize("name", DECODE)
def test_single_tokens(name, dt, d, bits):
    """Both ways of sharing out; lists in one share, two and many; groups of more heads than 16;
    windows with sinks."""
    lens, Hq, Hkv, W, S = DECODE[name]
    s = mx_plan.pooled(DT[dt], d, bits, Hq, Hkv, lens, seed=len(lens) + d)
    check(s, W, S)


@pytest.mark.parametrize("bits", [4, 8])
def test_graphs_and_streams(bits):
    """Single tokens whose lists lie across shares: captured, replayed with other queries and
    lengths, and twice at once."""
    lens, Hq, Hkv, W, S = DECODE["uneven"]
    s = mx_plan.pooled(torch.bfloat16, 64, bits, Hq, Hkv, lens)
    a = mxc.dev(s)
    call(a)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call(a))
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        a["q"].copy_(torch.randn(s["q"].shape, generator=g))
        a["lens"].copy_(torch.tensor(lens)[torch.randperm(len(lens), generator=g)])
        want = call(a)
        torch.cuda.synchronize()
        for graph in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        now = {**s, "q": a["q"].cpu(), "lens": a["lens"].cpu(), "max_len": max(lens)}
        assert_within(want, *expect(now), "out")
