"""What ``muon_update_`` writes is known to autograd and to the fused block's bf16 copies."""

from __future__ import annotations

import pytest
import torch

from minidist.models import GPT, GPTConfig
from minidist.models.fused_gpt import bf16_weight
from minidist.ops import _native as nat
from minidist.ops import muon as M
from minidist.optim import Muon, muon_groups

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
CFG = GPTConfig(vocab_size=1000, block_size=128, n_layer=2, n_head=4, n_embd=256, positions="rotary")


@pytest.mark.parametrize("device", DEVICES)
def test_versions_go_up(device):
    w, g, m = ([torch.randn(24, 40, device=device) for _ in range(2)] for _ in range(3))
    sh = [torch.empty(24, 40, dtype=torch.bfloat16, device=device), None]
    old = [t._version for t in (*w, *m, sh[0])]
    kept = [t._version for t in g]
    M.muon_update_(w, g, m, lr=0.1, shadows=sh)
    assert all(t._version > v for t, v in zip((*w, *m, sh[0]), old))
    assert [t._version for t in g] == kept
    with torch.inference_mode():  # (tensors without a version)
        w, g, m = ([torch.randn(24, 40, device=device)] for _ in range(3))
        M.muon_update_(w, g, m, lr=0.1)


@pytest.mark.parametrize("device", DEVICES)
def test_autograd_sees_that_a_saved_weight_changed(device):
    w = torch.randn(24, 40, device=device, requires_grad=True)
    x = torch.randn(3, 24, device=device, requires_grad=True)
    y = (x @ w).sum()
    M.muon_update_([w], [torch.randn_like(w)], [torch.zeros_like(w)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_fused_block_computes_with_the_weights_of_a_direct_step():
    torch.manual_seed(0)
    model = GPT(CFG, device="cuda")
    ids = torch.randint(0, 1000, (2, 128), device="cuda")

    def run(net):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            return net(ids)

    before = run(model)
    mats = [p for p in model.blocks.parameters() if p.dim() == 2]
    M.muon_update_(mats, [torch.randn_like(p) for p in mats], [torch.zeros_like(p) for p in mats], lr=0.05)
    after = run(model)
    fresh = GPT(CFG, device="cuda")
    fresh.load_state_dict(model.state_dict())
    assert torch.equal(after, run(fresh)) and not torch.equal(after, before)
    nat.check_status()


@pytest.mark.gpu
def test_optimizer_keeps_its_copies_valid():
    """The copies that Muon refreshes are not cast again, those that were stale before its step are."""
    torch.manual_seed(0)
    model = GPT(CFG, device="cuda")
    opt = Muon(muon_groups(model), lr=1e-2)
    ids, tgt = (torch.randint(0, 1000, (2, 128), device="cuda") for _ in range(2))

    def step():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            model(ids, tgt)[1].backward()
        opt.step()
        opt.zero_grad(set_to_none=True)

    step()
    mats = opt.param_groups[0]["params"]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model(ids, tgt)[1].backward()
    with torch.no_grad():
        mats[0].mul_(0.5)
    opt.step()
    assert mats[0]._md_bf16_ver != mats[0]._version
    for p in mats[1:]:
        assert p._md_bf16_ver == p._version and torch.equal(p._md_bf16, p.detach().bfloat16())
    step()
    for p in mats:
        assert p._md_bf16_ver == p._version and torch.equal(p._md_bf16, p.detach().bfloat16())
    nat.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_copies_made_in_inference_mode_are_refreshed_outside(device):
    p = torch.nn.Parameter(torch.randn(16, 8, device=device))
    with torch.inference_mode():
        bf16_weight(p)
    with torch.no_grad():
        p.mul_(2.0)
    assert torch.equal(bf16_weight(p), p.detach().bfloat16())


@pytest.mark.gpu
def test_evaluate_in_inference_mode_then_step_one_matrix():
    model = GPT(CFG, device="cuda")
    ids = torch.randint(0, 1000, (2, 128), device="cuda")
    with torch.inference_mode(), torch.autocast("cuda", dtype=torch.bfloat16):
        model(ids)
    w = model.blocks[0].attn.proj.weight
    M.muon_update_([w], [torch.randn_like(w)], [torch.zeros_like(w)], lr=0.05)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        model(ids, ids)[1].backward()
    assert torch.equal(w._md_bf16, w.detach().bfloat16())
    nat.check_status()
