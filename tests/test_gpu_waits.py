"""The count of barrier waits that gave up: 0 for calls that work, one more for a wait that nothing ends."""
from __future__ import annotations

import pytest
import torch

import engraft_ngram_b200 as eb
from engraft_ngram_b200 import _lib as L

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_a_wait_that_gives_up_is_counted_and_others_are_not():
    g = torch.Generator(device=DEV).manual_seed(0)
    u = torch.randn(300, 200, device=DEV, generator=g)
    x = torch.randn(50001, 40, device=DEV, generator=g)
    a, b = torch.randn(2, 40, 40, device=DEV, generator=g), torch.randn(2, 1040, 40, device=DEV, generator=g)
    index = torch.randint(0, 2, (50001,), device=DEV, generator=g).to(torch.int32)
    before = eb.waits_given_up()
    want = eb.orthogonalize(u), eb.adapter_add(None, x, a, b, index)
    assert eb.waits_given_up(DEV) == before
    L.check(L.load().engram_selftest_wait(L.stream_of(DEV)), "engram_selftest_wait")
    assert eb.waits_given_up(0) == before + 1
    got = eb.orthogonalize(u), eb.adapter_add(None, x, a, b, index)
    assert all(torch.equal(v, w) for v, w in zip(got, want)) and eb.waits_given_up() == before + 1
