"""Which parameters Muon takes, and what it says of those that it cannot."""

from __future__ import annotations

import warnings

import pytest
import torch

from minidist.fsdp import FullyShardedDataParallel, MixedPrecisionPolicy
from minidist.models import GPT, Block, GPTConfig
from minidist.optim import FusedAdamW, Muon, muon_groups
from tests.harness import run_distributed

CFG = GPTConfig(vocab_size=64, block_size=16, n_layer=2, n_head=2, n_embd=32, positions="rotary")


def _flat_shards_are_refused(rank: int, world: int) -> None:
    model = FullyShardedDataParallel(GPT(CFG), unit_types=(Block,), mixed_precision=MixedPrecisionPolicy(),
                                     device=torch.device("cpu"))
    for bad in (lambda: muon_groups(model), lambda: muon_groups(model, weight_decay=0.1),
                lambda: Muon(model.parameters()), lambda: muon_groups(model.module),
                lambda: Muon(model.module.parameters()), lambda: Muon([dict(params=list(model.parameters()))]),
                lambda: Muon([dict(params=list(model.parameters()), orthogonal=True)])):
        with pytest.raises(ValueError, match="whole matrices|not a float32 matrix"):
            bad()
    matrix = torch.nn.Parameter(torch.randn(4, 6))
    opt = Muon([dict(params=[matrix]), dict(params=list(model.parameters()), orthogonal=False)])
    assert [g["orthogonal"] for g in opt.param_groups] == [True, False]
    FusedAdamW(model.parameters())


@pytest.mark.parametrize("world", [1, 2])
def test_flat_shards_are_refused(world):
    run_distributed(_flat_shards_are_refused, world)


def test_a_mixed_group_says_what_it_leaves_to_adamw():
    vec, mat = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, 4))
    with pytest.warns(UserWarning, match="takes AdamW"):
        assert not Muon([vec, mat]).param_groups[0]["orthogonal"]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        Muon([mat])
        Muon([vec])
        Muon([dict(params=[vec, mat], orthogonal=False)])
        Muon(muon_groups(GPT(CFG)))


def test_named_parameters():
    lin = torch.nn.Linear(3, 4)
    opt = Muon([dict(params=[("weight", lin.weight)]), dict(params=[("bias", lin.bias)])], lr=0.1)
    assert [g["orthogonal"] for g in opt.param_groups] == [True, False]
    assert opt.param_groups[0]["param_names"] == ["weight"]
    before = lin.weight.detach().clone()
    lin(torch.randn(2, 3)).sum().backward()
    opt.step()
    assert not torch.equal(before, lin.weight) and "momentum_buffer" in opt.state[lin.weight]
    with pytest.warns(UserWarning, match="takes AdamW"):
        Muon(lin.named_parameters())


def test_precise_is_kept_with_the_group():
    mats = [torch.nn.Parameter(torch.randn(4, 6)) for _ in range(2)]
    opt = Muon([dict(params=[mats[0]], precise=True), dict(params=[mats[1]])])
    assert [g["precise"] for g in opt.param_groups] == [True, False]
    saved = opt.state_dict()
    del saved["param_groups"][1]["precise"]  # a state from before the option
    opt.load_state_dict(saved)
    for p in mats:
        p.grad = torch.ones_like(p)
    opt.step()
