"""The vocabulary-parallel embedding kernel as a group of one rank, with and without position rows."""

from __future__ import annotations

import ctypes

import pytest
import torch

from minidist.ops import _native as nat
from minidist.parallel import collectives as C


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("M,S,width", [(1, 1, 8), (96, 32, 264), (1000, 125, 768), (64, 64, 4096)])
def test_world1(M, S, width, positions):
    V = 517
    wte, wpe = (torch.randn(n, width, device="cuda").bfloat16() for n in (V, S))
    ids = torch.randint(0, V, (M,), device="cuda")
    out = torch.full((M, width), 7.0, dtype=torch.bfloat16, device="cuda")
    flags = torch.zeros(int(nat.lib().md_symm_flag_bytes()) // 4, dtype=torch.int32, device="cuda")
    prm = C.EmbTpParams()
    prm.wte[0], prm.flags[0] = wte.data_ptr(), flags.data_ptr()
    prm.world, prm.rank, prm.channel = 1, 0, C._EMB_CHANNEL
    prm.timeout_ns, prm.status = 10**9, nat.status_ptr()
    prm.ids, prm.out, prm.ldo = ids.data_ptr(), out.data_ptr(), width
    if positions:
        prm.wpe, prm.ldp = wpe.data_ptr(), width
    prm.ldw, prm.vocab_rows, prm.M, prm.S, prm.C = width, V, M, S, width
    for _ in range(2):
        nat.check(nat.lib().md_embed_tp(ctypes.byref(prm), min(148, -(-M // 32)), ctypes.c_void_p(nat.stream_ptr())),
                  "md_embed_tp")
    nat.check_status()
    want = wte[ids]
    if positions:
        want = (want.float() + wpe.float()[torch.arange(M, device="cuda") % S]).bfloat16()
    assert torch.equal(out, want)
