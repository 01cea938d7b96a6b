"""Calls of the paged operators that are refused whatever the sizes are, on the CPU."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from autosage_b200 import paged
from test_paged_host import pages, scales, table

INT8 = torch.int8


def operands(coded=False):
    kind = INT8 if coded else torch.float32
    own = dict(key_pages=pages(kind), value_pages=pages(kind))
    if coded:
        own.update(key_scales=scales(), value_scales=scales())
    crow, col, lengths = table()
    return {
        "attention": (paged.csr_paged_attention, dict(own, crow=crow, col=col, lengths=lengths, query=torch.zeros(2, 4, 8))),
        "write": (paged.paged_cache_write, dict(own, slots=torch.tensor([0, 5, -1]), key=torch.zeros(3, 2, 8), value=torch.zeros(3, 2, 8))),
        "read": (paged.paged_cache_read, dict(own, slots=torch.tensor([0, 5]))),
    }


DIFFERENTIABLE = [("attention", "query"), ("attention", "key_pages"), ("attention", "value_pages"), ("attention", "key_scales"),
                  ("attention", "value_scales"), ("write", "key"), ("write", "value"), ("write", "key_pages"),
                  ("write", "value_pages"), ("write", "key_scales"), ("write", "value_scales"), ("read", "key_pages"),
                  ("read", "value_pages"), ("read", "key_scales"), ("read", "value_scales")]


@pytest.mark.parametrize("quiet", [False, True], ids=["grad", "no_grad"])
@pytest.mark.parametrize("operator, name", DIFFERENTIABLE)
def test_a_tangent_is_refused(operator, name, quiet):
    """A dual tensor has requires_grad False; its tangent would be dropped without a word."""
    call, given = operands(coded=name.endswith("scales"))[operator]
    with forward_ad.dual_level(), torch.set_grad_enabled(not quiet):
        given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(**given)


@pytest.mark.parametrize("operator, name", DIFFERENTIABLE)
def test_a_wanted_gradient_is_refused(operator, name):
    call, given = operands(coded=name.endswith("scales"))[operator]
    given[name] = given[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        call(**given)


def test_a_jvp_through_a_call_is_refused():
    call, given = operands()["attention"]
    query = given.pop("query")
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda q: call(query=q, **given), (query,), (torch.ones_like(query),))


def test_a_level_without_tangents_is_no_reason():
    call, given = operands()["attention"]
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="needs CUDA"):
        call(**given)
