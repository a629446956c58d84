"""Scratch of the un-quantised experts: bounded, whatever the batch."""
import pytest
import torch

from bitsmoe_b200 import capi
from bitsmoe_b200.layer import dense_experts
from tests import dense_bounds as db
from tests.test_gpu_grouped import expert_case, experts_exact

DEV = "cuda:0"
gpu = pytest.mark.gpu
MB = 1 << 20


def need(*sizes):
    return capi.lib().bm_dense_experts_workspace_bytes(*sizes)


def test_scratch_is_bounded():
    """(tokens, k, experts held, hidden, intermediate): k rows a token of 4 hidden + 6 intermediate bytes up to 256 MB, as many as experts are
    held up to 1 GB or four times the weights, and 12 bytes and a little for every assignment."""
    few, row = (10, 3, 2048, 512), 4 * 2048 + 6 * 512
    assert need(2000, *few) >= 2000 * 10 * row
    assert 16384 * 3 * row <= need(16384, *few) < 16384 * (3 * row + 121) + MB
    for T in (32768, 1000000):
        assert 1020 * MB < need(T, *few) < 1032 * MB + 12.1 * T * 10
    all_held = (8, 128, 2048, 768)                                   # 1.2 GB of weights
    assert need(16384, *all_held) >= 16384 * 8 * (4 * 2048 + 6 * 768)
    assert 4600 * MB < need(100000, *all_held) < 4620 * MB + 13 * 100000 * 8
    assert need(1, 32, 32, 1 << 24, 1) >= 32 * 4 * (1 << 24)          # a token's rows stay together


def held(routed, E):
    g2l = torch.full((routed,), -1, dtype=torch.int32, device=DEV)
    g2l[torch.randperm(routed, generator=torch.Generator().manual_seed(1))[:E].to(DEV)] = torch.arange(E, dtype=torch.int32, device=DEV)
    return g2l


def run(x, idx, w, gu, dn, g2l, most):
    """Eager twice and captured, within ``most`` bytes."""
    res = torch.randn_like(x)
    call = lambda: dense_experts(x, idx, w, gu, dn, global_to_local=g2l, residual=res)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = call()
    assert torch.cuda.max_memory_allocated() - before < most + got.nbytes
    value, err = experts_exact(x, idx, w, gu, dn, g2l, res)
    db.check(got, value, err, what="long batch")
    assert torch.equal(call(), got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, got)
    return got, res


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,k,E,H,I,routed", [(5003, 10, 3, 2048, 512, 512), (2100, 32, 2, 4096, 64, 2), (9001, 9, 8, 1024, 33, 8)])
def test_slots_that_name_one_expert_share_a_row(T, k, E, H, I, routed, dtype):
    """Ids drawn with repetition, and a map that sends two ids to one expert."""
    row = 4 * H + 6 * I
    assert T * k * row > 256 * MB and T * E * row < need(T, k, E, H, I) < T * (E * row + 12.1 * k) + MB
    x, idx, w, gu, dn = expert_case(31, T, k, E, H, I, dtype, routed=routed, dup=True)
    g2l = held(routed, E)
    g2l[:2] = g2l[:2].max()
    run(x, idx, w, gu, dn, g2l, T * E * row + 8 * MB)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("load", ["every slot", "one slot in 20", "the first tokens only", "none"])
def test_long_batches_go_through_in_windows(load, dtype):
    T, k, E, H, I = 30001, 32, 32, 512, 64
    row = 4 * H + 6 * I
    assert T * k * row > 2 * 1024 * MB and need(T, k, E, H, I) < 1040 * MB
    routed = 640 if load == "one slot in 20" else E
    x, idx, w, gu, dn = expert_case(33, T, k, E, H, I, dtype, routed=routed, dup=load == "one slot in 20")
    if load == "the first tokens only":
        idx[1024 * MB // (row * k):] = -1            # a window of tokens without rows follows one that is full
    elif load == "none":
        idx[:] = -1
    got, res = run(x, idx, w, gu, dn, held(routed, E), 1040 * MB)
    none = (idx < 0).all(dim=1)
    assert torch.equal(got[none], res[none])
