"""Muon inside the framework's ways to train: captured steps, deferred gradient buckets, tensor parallelism."""

from __future__ import annotations

import copy
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import minidist as md
from minidist import ddp as ddp_mod
from minidist.ddp import DistributedDataParallel
from minidist.models import GPT, GPTConfig
from minidist.models.fused_gpt import bf16_weight
from minidist.ops import _native as nat
from minidist.ops.muon import muon_update_
from minidist.optim import Muon, muon_groups
from tests.harness import assert_close, run_distributed, solo_group

CFG = GPTConfig(vocab_size=64, block_size=16, n_layer=2, n_head=4, n_embd=32, positions="rotary", rotary_fraction=0.5,
                rotary_scaling=md.RotaryScaling("yarn", 4.0, original_positions=8))


def _data(seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randint(0, CFG.vocab_size, (4, CFG.block_size), generator=g) for _ in range(2))


SHAPES = [(96, 200), (96, 200), (300, 70), (33, 35), (768, 256)]


def _run(graph, grads, lrs):
    g = torch.Generator().manual_seed(1)
    mats = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda()) for s in SHAPES]
    vec = torch.nn.Parameter(torch.randn(40, generator=g).cuda())
    opt = Muon([dict(params=mats), dict(params=[vec])], lr=lrs[0], weight_decay=0.1, capturable=True)
    for p in mats[1:]:
        bf16_weight(p)  # copies to keep up to date

    def step(*gs):
        for p, t in zip((*mats, vec), gs):
            p.grad = t
        opt.step()

    run = md.GraphedStep(step, grads[0], warmup=2, optimizers=[opt]) if graph else step
    if not graph:
        for _ in range(2):
            step(*grads[0])
    states = []
    for gs, lr in zip(grads[1:], lrs):
        for group in opt.param_groups:
            group["lr"] = lr
        run(*gs)
        states.append([t.detach().clone() for t in (*mats, vec, *(opt.state[p]["momentum_buffer"] for p in mats),
                                                    *(p._md_bf16 for p in mats[1:]))])
        for p in mats[1:]:
            assert torch.equal(p._md_bf16, p.detach().bfloat16())
    if graph:
        run.release()
    nat.check_status()
    return states


@pytest.mark.gpu
def test_replayed_steps_are_the_eager_ones():
    """Bit for bit, with the learning rate changing between replays."""
    g = torch.Generator().manual_seed(2)
    grads = [[(torch.randn(*s, generator=g) * 1e-2).cuda() for s in (*SHAPES, (40,))] for _ in range(6)]
    lrs = [1e-2, 1e-2, 3e-3, 3e-3, 2e-2]
    eager, replayed = _run(False, grads, lrs), _run(True, grads, lrs)
    for i, (a, b) in enumerate(zip(eager, replayed)):
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i
    for a, b in zip(eager, eager[1:]):
        assert not any(torch.equal(x, y) for x, y in zip(a, b))  # every step changes every tensor


def _deferred(rank, world):
    solo = solo_group(rank, world)
    ids, tgt = _data()
    runs = []
    for defer in (0, 2):
        model = DistributedDataParallel(GPT(CFG, tp_group=solo), bucket_cap_mb=0.01, defer_last_buckets=defer)
        opt = Muon(muon_groups(model), lr=1e-2)
        before = copy.deepcopy(dict(model.named_parameters()))
        for it in range(3):
            x, y = ids.roll(it, 0).chunk(world)[rank], tgt.roll(it, 0).chunk(world)[rank]
            opt.zero_grad()
            model(x, y)[1].backward()
            if defer:
                # The optimizer honours the handles itself; its matrices are among those in flight.
                assert any(getattr(p, "_md_grad_event", None) is not None for p in opt.param_groups[0]["params"])
            opt.step()
            assert all(getattr(p, "_md_grad_event", None) is None for p in model.parameters())
        ddp_mod.wait_all_deferred()
        assert all(not torch.equal(p, before[n]) for n, p in model.named_parameters())
        runs.append(model)
    for (name, p), q in zip(runs[1].named_parameters(), runs[0].parameters()):
        assert torch.equal(p, q), f"[rank {rank}] deferred buckets with Muon differ at {name}"


def test_deferred_buckets():
    run_distributed(_deferred, 2)


def _tensor_parallel(rank, world):
    solo = solo_group(rank, world)
    sharded, whole = GPT(CFG, tp_group=None), GPT(CFG, tp_group=solo)
    torch.manual_seed(0)
    ids, tgt = _data()
    (logits, loss), (ref_logits, ref_loss) = sharded(ids, tgt), whole(ids, tgt)
    assert_close(loss, ref_loss, f"[rank {rank}] tp={world} rotary loss", tol=1e-5)
    assert_close(logits, ref_logits.chunk(world, -1)[rank], f"[rank {rank}] rotary logits", tol=1e-4)
    loss.backward()
    ref_loss.backward()
    for i in range(CFG.n_layer):
        a, b = sharded.blocks[i], whole.blocks[i]
        for part, dim in (("attn.qkv.weight", 0), ("attn.qkv.bias", 0), ("attn.proj.weight", 1), ("mlp.fc.weight", 0),
                          ("mlp.proj.weight", 1), ("ln1.weight", None), ("ln2.bias", None)):
            got, want = a.get_parameter(part).grad, b.get_parameter(part).grad
            assert_close(got, want if dim is None else want.chunk(world, dim)[rank],
                         f"[rank {rank}] block {i} {part} gradient", tol=1e-4)
    assert_close(sharded.embedding.wte.weight.grad, whole.embedding.wte.weight.grad.chunk(world, 0)[rank],
                 f"[rank {rank}] embedding gradient", tol=1e-4)
    # A shard is orthogonalised as a matrix of its own.
    opt = Muon(muon_groups(sharded), lr=1e-2, weight_decay=0.0)
    mats = opt.param_groups[0]["params"]
    twins, grads = [p.detach().clone() for p in mats], [p.grad.clone() for p in mats]
    opt.step()
    muon_update_(twins, grads, [torch.zeros_like(t) for t in twins], lr=1e-2)
    assert all(torch.equal(p, t) for p, t in zip(mats, twins))


@pytest.mark.parametrize("world", [2, 4])
def test_rotary_under_tensor_parallelism(world):
    run_distributed(_tensor_parallel, world)


def test_trainer_says_that_updates_depend_on_tp():
    root = Path(__file__).resolve().parent.parent
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--master-addr=127.0.0.1"]
    args = ["--layers", "1", "--embd", "32", "--heads", "2", "--vocab", "64", "--seq-len", "16", "--batch-size", "2", "--steps",
            "1", "--backend", "gloo", "--optimizer", "muon"]
    for tp in (1, 2):
        proc = subprocess.run([*cmd, "--nproc-per-node=2", "--master-port=29583", str(root / "examples" / "train_gpt.py"), *args,
                               "--tp", str(tp)], capture_output=True, text=True, timeout=300, cwd=root,
                              env=dict(os.environ, OMP_NUM_THREADS="1", CUDA_VISIBLE_DEVICES=""))
        assert proc.returncode == 0, proc.stderr[-3000:]
        assert ("updates depend on --tp" in proc.stdout) == (tp > 1)
