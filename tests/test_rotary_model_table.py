"""The rotary table that a model keeps: made by whatever call comes first, good for every later one."""

from __future__ import annotations

import copy
import gc
import weakref

import pytest
import torch

import minidist as md
from minidist.models import GPT, GPTConfig

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _config(block_size=32, **kw):
    return GPTConfig(vocab_size=64, block_size=block_size, n_layer=3, n_head=2, n_embd=32, positions="rotary", **kw)


def _data(device):
    g = torch.Generator().manual_seed(0)
    return tuple(torch.randint(0, 64, (2, 32), generator=g).to(device) for _ in range(2))


@pytest.mark.parametrize("device", DEVICES)
def test_evaluate_in_inference_mode_then_train(device):
    model, twin = (GPT(_config(), device=device) for _ in range(2))
    ids, tgt = _data(device)
    with torch.inference_mode():
        model(ids)
    for net in (model, twin):
        net(ids, tgt)[1].backward()
    for p, q in zip(model.parameters(), twin.parameters()):
        assert torch.equal(p.grad, q.grad)
    assert not model.blocks[0].attn.rotary(ids.device).is_inference()


@pytest.mark.parametrize("device", DEVICES)
def test_one_table_for_the_layers_and_for_models_alike(device):
    model = GPT(_config(), device=device)
    ids, _ = _data(device)
    with torch.no_grad():
        model(ids)
    table = model.blocks[0].attn.rotary(ids.device)
    assert torch.equal(table, md.rotary_table(16, 32, device=device))
    other = GPT(_config(), device=device)
    for block in (*model.blocks, *other.blocks):
        assert block.attn.rotary(ids.device) is table
    for cfg in (_config(block_size=64), _config(rotary_fraction=0.5), _config(rotary_base=500.0),
                _config(rotary_scaling=md.RotaryScaling("linear", 2.0))):
        assert not torch.equal(GPT(cfg, device=device).blocks[0].attn.rotary(ids.device), table[:, :4])
    clone = copy.deepcopy(model)
    with torch.no_grad():
        assert torch.equal(clone(ids), model(ids))
    half = GPT(_config(), device=device).bfloat16()
    assert half.blocks[0].attn.rotary(ids.device).dtype == torch.float32
    ref = weakref.ref(table)
    del model, other, clone, half, table, block
    gc.collect()
    assert ref() is None  # kept by the models that use it, not by the process


@pytest.mark.gpu
def test_moved_model_and_capture_first():
    attn = GPT(_config(block_size=48)).blocks[0].attn
    host = attn.rotary(torch.device("cpu"))
    attn.cuda()
    want = md.rotary_table(16, 48, device="cuda")
    dev = want.device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.rotary(dev) * 2
    assert torch.equal(attn.rotary(dev), want)  # not the captured one, which no replay has filled yet
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want * 2)
    assert torch.equal(attn.rotary(dev).cpu(), want.cpu()) and host.device.type == "cpu"
    graph.reset()
