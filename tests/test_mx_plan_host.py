"""Which form attention over the cache in 4 and 8 bits takes, and the workspace that the form
asks for, on both sides of each of the rule's borders.  Needs a machine without a GPU: the
calls go as far as their checks."""
import pytest
import torch

import mx_plan
from mx_plan import MOST, PARTS, TILES

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would go on to a GPU")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("W,S", [(0, 0), (2100, 3), (20, 3)])
@pytest.mark.parametrize("name", PARTS)
def test_parts_of_prompts(name, W, S, d, bits):
    lens, new, Hq, Hkv, max_len = PARTS[name]
    a = (bits, sum(new), len(lens), Hq, Hkv, d, W, S, 0, max_len)
    form, nbytes = mx_plan.workspace(*a)
    assert mx_plan.asked(*a) == nbytes
    if W == 0:
        assert (form == "shares") == (not name.startswith("over"))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", mx_plan.DECODE)
def test_single_tokens(name, d, bits):
    """The batches reach both ways of sharing out, and lists in one to many shares."""
    lens, Hq, Hkv, W, S = mx_plan.DECODE[name]
    a = (bits, len(lens), len(lens), Hq, Hkv, d, W, S, 1, max(lens))
    form, nbytes = mx_plan.workspace(*a)
    assert form == "shares" and mx_plan.asked(*a) == nbytes
    one, most = mx_plan.decode_shares(bits, d, Hq, Hkv, lens, W, S, max(lens))
    assert one == (name == "alike") and most >= (2 if name == "windows" else 3)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_both_sides_of_every_border(d, bits):
    forms = set()
    for T, Bd, Hq, Hkv, max_len in (
            [(20, 1, 32, 2, n) for n in (64 * 32, 64 * 32 + 1)] +                       # pages of a list
            [(5, 5, h, h, n) for h in (1, 2, 8) for n in (64 * 42, 64 * 43, 64 * 85, 64 * 86, 64 * 170, 64 * 171,
                                                          64 * 341, 64 * 342)] +        # pages of all lists: 6 h times as many
            [(2, n, 2, 1, 5000) for n in (MOST - 2, MOST - 1, MOST, MOST + 1)] +
            [(n, 1, 128, 1, 5000) for n in (TILES - 2, TILES - 1, TILES)] +
            [(9, 40, h, h, 2200) for h in (12700, 12785, 12790)] +                      # row tiles of all heads
            [(9, 40, h, h, 64 * n) for h in (3000, 4000) for n in (3200, 4300, 4400)]):
        for W, S in ((0, 0), (1900, 3), (1990, 3), (3000, 100)):
            a = (bits, T, Bd, Hq, Hkv, d, W, S, 0, max_len)
            form, nbytes = mx_plan.workspace(*a)
            assert mx_plan.asked(*a) == nbytes, a
            forms.add(form)
    assert forms == {"shares", "runs", "whole"}
    forms = set()
    for Bd, Hq, Hkv in ((1, 1, 1), (1, 17, 1), (511, 4, 2), (512, 4, 2), (1023, 1, 1), (1024, 1, 1), (30, 34, 17), (31, 34, 17)):
        for max_len in (64 * 32, 64 * 32 + 1, 64 * 40, 10 ** 6):
            for W, S in ((0, 0), (1984, 0), (1985, 1), (3000, 100)):
                a = (bits, Bd, Bd, Hq, Hkv, d, W, S, 1, max_len)
                form, nbytes = mx_plan.workspace(*a)
                assert mx_plan.asked(*a) == nbytes, a
                forms.add(form)
    assert forms == {"shares", "whole"}
