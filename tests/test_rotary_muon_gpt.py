"""A GPT with rotary positions, trained with Muon and scored with token log probabilities."""

from __future__ import annotations

import copy
import json
import math
import os
import subprocess
import sys

import pytest
import torch

import minidist as md
from minidist.models import GPT, GPTConfig
from minidist.ops import _native as nat
from minidist.ops.muon import muon_update_
from minidist.optim import FusedAdamW, Muon, muon_groups

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = GPTConfig(vocab_size=1000, block_size=256, n_layer=2, n_head=4, n_embd=256, positions="rotary")
SMALL = GPTConfig(vocab_size=64, block_size=32, n_layer=2, n_head=2, n_embd=32, positions="rotary")


def _data(cfg, device, B=4, S=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    S = S or cfg.block_size
    return tuple(torch.randint(0, cfg.vocab_size, (B, S), generator=g).to(device) for _ in range(2))


def test_rotary_model_has_no_position_table():
    model = GPT(SMALL)
    assert model.embedding.wpe is None and not any("wpe" in n for n in model.state_dict())
    assert not any("rotary" in n for n in model.state_dict())
    assert model.num_parameters() == SMALL.param_count()
    learned = GPT(GPTConfig(vocab_size=64, block_size=32, n_layer=2, n_head=2, n_embd=32))
    ids, tgt = _data(SMALL, "cpu")
    with torch.no_grad():
        assert not torch.allclose(model(ids), learned(ids))
    _, loss = model(ids, tgt)
    loss.backward()
    assert all(p.grad is not None for p in model.parameters())
    with pytest.raises(ValueError):
        model(torch.zeros(1, 33, dtype=torch.long))  # past the table


def test_rotary_attention_sees_relative_positions():
    """Scores depend on the distance between query and key: moving a whole sequence by an offset (its
    positions, not its tokens) leaves attention's output as it was."""
    attn = GPT(SMALL).blocks[0].attn
    x = torch.randn(1, 10, 32)
    q, k, _ = attn.qkv(x).view(1, 10, 2, 3, 16).unbind(3)
    table = attn.rotary(x.device)
    a, b = md.apply_rotary(q, k, table)
    c, d = md.apply_rotary(q, k, table, torch.arange(13, 23))
    s, t = (torch.einsum("bqhd,bkhd->bhqk", u, v) for u, v in ((a, b), (c, d)))
    # 16 products of fp32 numbers of size 1
    assert float((s - t).abs().max()) < 16 * 8 * 2.0**-24 * float(q.abs().max() * k.abs().max()) * 4


def test_config_refusals():
    for bad in (dict(positions="sinusoidal"), dict(positions="rotary", rotary_fraction=0.0),
                dict(positions="rotary", rotary_fraction=1.5), dict(positions="rotary", rotary_fraction=0.01)):
        with pytest.raises(ValueError):
            GPTConfig(n_embd=32, n_head=2, **bad)


def test_muon_groups_and_step_match_the_functions():
    model = GPT(SMALL)
    ids, tgt = _data(SMALL, "cpu")
    groups = muon_groups(model, weight_decay=0.1)
    hidden = {id(p) for p in groups[0]["params"]}
    want = {id(p) for n, p in model.named_parameters() if n.startswith("blocks.") and p.dim() == 2}
    assert hidden == want and sum(len(g["params"]) for g in groups) == len(list(model.parameters()))
    twin = copy.deepcopy(model)
    opt = Muon(groups, lr=1e-2, weight_decay=0.0)
    ref_groups = muon_groups(twin, weight_decay=0.1)
    adam = FusedAdamW(ref_groups[1:], lr=1e-2, betas=(0.9, 0.95), weight_decay=0.0)
    momenta = [torch.zeros_like(p) for p in ref_groups[0]["params"]]
    for _ in range(3):
        for m in (model, twin):
            for p in m.parameters():
                p.grad = None
            m(ids, tgt)[1].backward()
        opt.step()
        adam.step()
        mats = ref_groups[0]["params"]
        muon_update_(mats, [p.grad for p in mats], momenta, lr=1e-2, weight_decay=0.1)
    for (n, p), q in zip(model.named_parameters(), twin.parameters()):
        assert torch.equal(p, q), n
    other = Muon(muon_groups(copy.deepcopy(model)), lr=1e-2)
    other.load_state_dict(opt.state_dict())
    a, b = (o.state[o.param_groups[0]["params"][0]]["momentum_buffer"] for o in (opt, other))
    assert torch.equal(a, b)


def test_muon_refusals():
    vec, mat = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, 4))
    assert not Muon([vec, mat]).param_groups[0]["orthogonal"]
    assert Muon([mat]).param_groups[0]["orthogonal"]
    for bad in (lambda: Muon([dict(params=[vec], orthogonal=True)]), lambda: Muon([mat], momentum=1.0),
                lambda: Muon([mat], rms=0.0), lambda: Muon([mat], ns_steps=0), lambda: Muon([mat], lr=-1.0),
                lambda: Muon([dict(params=[torch.nn.Parameter(torch.zeros(4, 4).half())], orthogonal=True)])):
        with pytest.raises(ValueError):
            bad()


def _training(device, cfg, steps, amp):
    torch.manual_seed(0)
    model = GPT(cfg, device=device)
    opt = Muon(muon_groups(model), lr=3e-3)
    ids, tgt = _data(cfg, device)
    losses, scores = [], []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        with torch.autocast(device, dtype=torch.bfloat16, enabled=amp):
            _, loss = model(ids, tgt)
        loss.backward()
        opt.step()
        losses.append(loss.item())
        with torch.no_grad(), torch.autocast(device, dtype=torch.bfloat16, enabled=amp):
            r = md.token_logprobs(model(ids), tgt, entropy=True, top=1)
        scores.append((r.logprobs.mean().item(), r.entropy.mean().item()))
        assert bool((r.top_logprobs[..., 0] >= r.logprobs - 1e-4).all())
    return losses, scores


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_training_lowers_the_loss_and_the_scores_follow(device):
    cuda = device == "cuda"
    losses, scores = _training(device, CFG if cuda else SMALL, 8, cuda)
    assert losses[-1] < losses[0] - (0.5 if cuda else 0.1), losses
    # The score after a step is the next step's loss (bf16 logits: within a rounding of the loss).
    for loss, (lp, h) in zip(losses[1:], scores):
        assert abs(loss + lp) < (2e-2 if cuda else 1e-4)
        assert 0 < h <= math.log((CFG if cuda else SMALL).vocab_size) + 1e-3
    if cuda:
        nat.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("fraction", [1.0, 0.5])
def test_fused_rotary_matches_fp32(fraction):
    import dataclasses

    cfg = dataclasses.replace(CFG, rotary_fraction=fraction)
    torch.manual_seed(0)
    ref = GPT(cfg, device="cuda")
    fused = copy.deepcopy(ref)
    ids, tgt = _data(cfg, "cuda")
    _, loss_ref = ref(ids, tgt)
    loss_ref.backward()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        _, loss = fused(ids, tgt)
    loss.backward()
    nat.check_status()
    # (the bounds of the same comparison with learned positions)
    assert abs(loss.item() - loss_ref.item()) < 2e-2 * abs(loss_ref.item())
    for (n, p), (_, q) in zip(fused.named_parameters(), ref.named_parameters()):
        err = ((p.grad - q.grad).abs().max() / q.grad.abs().max().clamp(min=1e-8)).item()
        assert err < 6e-2, f"{n}: rel err {err:.3e}"


@pytest.mark.gpu
def test_muon_refreshes_the_bf16_copies_and_obeys_the_scaler():
    torch.manual_seed(0)
    model = GPT(CFG, device="cuda")
    opt = Muon(muon_groups(model), lr=1e-3)
    ids, tgt = _data(CFG, "cuda")
    for _ in range(2):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            _, loss = model(ids, tgt)
        loss.backward()
        opt.step()
    for p in opt.param_groups[0]["params"]:
        assert p._md_bf16_ver == p._version and torch.equal(p._md_bf16, p.detach().bfloat16())
    before = [p.detach().clone() for p in model.parameters()]
    buffers = [opt.state[p]["momentum_buffer"].clone() for p in opt.param_groups[0]["params"]]
    scaler = md.DistributedGradScaler(init_scale=2.0**10)
    opt.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        _, loss = model(ids, tgt)
    scaler.scale_loss(loss).backward()
    opt.param_groups[0]["params"][0].grad[0, 0] = float("inf")
    scaler.step(opt)
    scaler.update()
    assert scaler.num_skipped == 1
    assert all(torch.equal(a, b) for a, b in zip(before, model.parameters()))
    assert all(torch.equal(a, opt.state[p]["momentum_buffer"]) for a, p in zip(buffers, opt.param_groups[0]["params"]))


def test_trainer_rotary_muon_cpu(tmp_path):
    path = tmp_path / "m.jsonl"
    common = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--master-addr=127.0.0.1"]
    script = os.path.join(ROOT, "examples", "train_gpt.py")
    env = dict(os.environ, OMP_NUM_THREADS="1", CUDA_VISIBLE_DEVICES="")
    args = ["--layers", "2", "--embd", "64", "--heads", "4", "--vocab", "256", "--seq-len", "32", "--batch-size", "4",
            "--steps", "2", "--backend", "gloo", "--positions", "rotary", "--rotary-fraction", "0.5", "--optimizer", "muon"]
    for extra in (["--score-every", "1", "--metrics-jsonl", str(path)], ["--tp", "2"], ["--pp", "2", "--strategy", "none"]):
        proc = subprocess.run([*common, "--nproc-per-node=2", "--master-port=29581", script, *args, *extra],
                              capture_output=True, text=True, timeout=600, env=env, cwd=ROOT)
        assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
        assert "tok/s" in proc.stdout
    scores = [r for r in map(json.loads, path.read_text().splitlines()) if r.get("event") == "score"]
    assert len(scores) == 2 and all(-7.0 < s["logprob"] < -4.0 and 0 < s["entropy"] < 5.6 for s in scores), scores
    proc = subprocess.run([*common, "--nproc-per-node=2", "--master-port=29582", script, *args, "--strategy", "fsdp"],
                          capture_output=True, text=True, timeout=600, env=env, cwd=ROOT)
    assert proc.returncode != 0 and "whole matrices" in proc.stderr + proc.stdout


@pytest.mark.gpu
def test_trainer_rotary_muon_cuda_graph(tmp_path):
    metrics = tmp_path / "m.jsonl"
    cmd = [sys.executable, os.path.join(ROOT, "examples", "train_gpt.py"), "--precision", "bf16", "--cuda-graph",
           "--layers", "2", "--embd", "256", "--heads", "4", "--vocab", "4096", "--seq-len", "256", "--batch-size", "8",
           "--steps", "6", "--positions", "rotary", "--optimizer", "muon", "--score-every", "3",
           "--metrics-jsonl", str(metrics)]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
    recs = [json.loads(line) for line in metrics.read_text().splitlines()]
    losses = [r["loss"] for r in recs if "loss" in r]
    assert losses and all(7.0 < v < 9.5 for v in losses), losses  # ~ln(4096) = 8.3 for random tokens
    scores = [r for r in recs if r.get("event") == "score"]
    assert len(scores) == 2 and all(-9.5 < s["logprob"] < -7.0 for s in scores), scores
