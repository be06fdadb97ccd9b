"""Arguments of the live modes without the mode that takes them, and padding
where it would be taken for tokens: refused, or said, before any model call."""
from types import SimpleNamespace

import pytest
import torch

from tide_b200 import runtime
from tide_b200.config import TIDEConfig
from tide_b200.runtime import TIDERuntime

IDS = torch.arange(8).view(2, 4)
MASK = torch.tensor([[0, 1, 1, 1], [1, 1, 1, 1]])


class Reached(Exception):
    pass


def engine(**config):
    """An engine whose first use of its model raises Reached."""
    def reached(*args, **kw):
        raise Reached

    return SimpleNamespace(config=TIDEConfig(**config), _layers=[], _live_family=reached, model=reached,
                           _hidden_states=reached)


def generate(**kw):
    return TIDERuntime.generate(engine(), IDS, max_new_tokens=2, **kw)


def forward(config=None, **kw):
    return TIDERuntime.forward(engine(**(config or {})), IDS, **kw)


@pytest.mark.parametrize("mask", [MASK, MASK.bool(), MASK.float()])
def test_generate_live_refuses_padding_without_the_paged_cache(mask):
    with pytest.raises(ValueError, match="paged=True"):
        generate(live=True, attention_mask=mask)


@pytest.mark.parametrize("kw", [dict(), dict(attention_mask=None), dict(attention_mask=torch.ones_like(IDS)),
                                dict(paged=True, attention_mask=MASK)])
def test_generate_live_goes_on_without_padding_or_with_the_paged_cache(kw):
    with pytest.raises(Reached):
        generate(live=True, **kw)


@pytest.mark.parametrize("per_row", [False, True])
def test_generate_says_that_padding_counts_as_tokens(monkeypatch, per_row):
    """The reference's loop takes any keyword and no mask
    (python/TIDE/runtime.py:223-313): it goes on, but not in silence."""
    said = []
    monkeypatch.setattr(runtime.logger, "warning", said.append)
    with pytest.raises(Reached):
        generate(attention_mask=torch.ones_like(IDS), per_row_exit=per_row)
    assert not said
    with pytest.raises(Reached):
        generate(attention_mask=MASK, per_row_exit=per_row)
    assert len(said) == 1 and "padding" in said[0]


def test_generate_refuses_the_paged_cache_without_live():
    with pytest.raises(ValueError, match="live=True"):
        generate(paged=True)
    with pytest.raises(Reached):
        generate(paged=False)


@pytest.mark.parametrize("config,kw", [({}, {}), ({}, dict(live=False)),
                                       (dict(live_compaction=True), dict(live=False))])
def test_forward_refuses_packed_without_live(config, kw):
    with pytest.raises(ValueError, match="live"):
        forward(config, packed=True, **kw)
    with pytest.raises(Reached):
        forward(config, packed=False, **kw)


@pytest.mark.parametrize("config,kw", [({}, dict(live=True)), (dict(live_compaction=True), {})])
def test_forward_takes_packed_with_live(config, kw):
    with pytest.raises(Reached):
        forward(config, packed=True, **kw)
