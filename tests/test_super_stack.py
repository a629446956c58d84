"""How a block stacks the weights of its un-quantised experts: order of copies and exchange, threads, streams."""
import threading
import time
from types import SimpleNamespace as NS

import pytest
import torch
import torch.nn as nn

from bitsmoe_b200.models.qwen3moe.bitsmoe_block import BitsMoE_Qwen3MoeSparseMoeBlock
from tests import helpers
from tests.test_dense_in_blocks import _by_modules, _qwen_block
from tests.test_gpu_blocks import DenseMLP

DEV = "cuda:0"
gpu = pytest.mark.gpu
HIDDEN, INTER = 32, 48


def host_block(experts, hidden_act="silu", num_experts=8):
    """A block on the CPU that has nothing but the given un-quantised experts {id: module}."""
    conf = NS(hidden_size=HIDDEN, intermediate_size=INTER, moe_intermediate_size=INTER, num_experts=num_experts, num_experts_per_tok=2,
              norm_topk_prob=True, hidden_act=hidden_act)
    src = NS(gate=nn.Linear(HIDDEN, num_experts, bias=False).half(), experts=[None] * num_experts)
    blk = BitsMoE_Qwen3MoeSparseMoeBlock(conf, 0, src, super_experts=sorted(experts), copy_source_experts=False)
    for e, m in experts.items():
        blk.set_expert(e, m, packed=False)
    blk._ensure_runtime_cache(torch.device("cpu"))
    return blk


def mlp(seed=0):
    torch.manual_seed(seed)
    return DenseMLP(HIDDEN, INTER).half()


def weights(m):
    return [getattr(m, n).weight for n in ("gate_proj", "up_proj", "down_proj")]


def test_copies_are_done_before_anything_else_sees_the_stack(monkeypatch):
    blk = host_block({1: mlp(1), 4: mlp(2)})
    before = [w.data_ptr() for e in (1, 4) for w in weights(blk.experts[e])]
    values = [w.detach().clone() for e in (1, 4) for w in weights(blk.experts[e])]
    seen = []

    def finish(device):
        seen.append((device.type, [w.data_ptr() for e in (1, 4) for w in weights(blk.experts[e])], blk._super_weights))

    monkeypatch.setattr(blk, "_finish_copies", finish, raising=False)
    gu, dn = blk._stacked_super_weights()
    assert seen == [("cpu", before, None)]             # once, with the parameters where they were and nothing published
    after = [w for e in (1, 4) for w in weights(blk.experts[e])]
    assert all(torch.equal(a, v) for a, v in zip(after, values))
    assert after[0].data_ptr() == gu[0].data_ptr() and after[4].data_ptr() == gu[1, INTER:].data_ptr() and after[5].data_ptr() == dn[1].data_ptr()
    assert blk._stacked_super_weights()[0] is gu and len(seen) == 1


def test_threads_in_their_first_call_share_one_stack(monkeypatch):
    blk = host_block({1: mlp(1), 4: mlp(2), 6: mlp(3)})
    values = [w.detach().clone() for e in (1, 4, 6) for w in weights(blk.experts[e])]
    monkeypatch.setattr(blk, "_finish_copies", lambda device: time.sleep(0.05), raising=False)
    got, gate = [], threading.Barrier(4)

    def call():
        gate.wait()
        got.append(blk._stacked_super_weights())

    threads = [threading.Thread(target=call) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(g[0] is got[0][0] and g[1] is got[0][1] for g in got)
    assert all(torch.equal(a, v) for a, v in zip((w for e in (1, 4, 6) for w in weights(blk.experts[e])), values))


@gpu
def test_first_call_on_a_side_stream():
    """Weights are loaded on one stream, the first call runs on another that is behind with its work, a third uses the block right
    away, and the first takes new memory meanwhile."""
    cfg, blk = _qwen_block([2, 5])
    x = torch.randn(1, 40, cfg.hidden, generator=torch.Generator().manual_seed(1)).to(DEV).half()
    want, _ = _by_modules(blk, x)
    kept = [w.detach().clone() for e in (2, 5) for w in weights(blk.experts[e])]
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)
    with torch.no_grad():
        with torch.cuda.stream(first):
            torch.cuda._sleep(100_000_000)
            a, _ = blk(x)
        junk = [torch.full_like(k, 7.0) for k in kept for _ in range(4)]
        with torch.cuda.stream(second):
            b, _ = blk(x)
    torch.cuda.synchronize()
    assert len(junk) == 24
    assert all(torch.equal(w, k) for w, k in zip((w for e in (2, 5) for w in weights(blk.experts[e])), kept))
    helpers.assert_close(a, want, what="first stream")
    helpers.assert_close(b, want, what="second stream")
