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


def test_devices_do_not_wait_for_one_another(monkeypatch):
    """A thread that waits for its device while it stacks must not keep another device's thread from launching what it waits for."""
    from bitsmoe_b200.models import base_block
    blocks = {torch.device("cuda", 0): host_block({1: mlp(1)}), torch.device("cuda", 1): host_block({1: mlp(2)})}
    both = threading.Barrier(2, timeout=20)
    real, mine = getattr(base_block, "_stacking_lock", None), threading.local()
    if real is not None:
        monkeypatch.setattr(base_block, "_stacking_lock", lambda device: real(mine.device))
    errors = []

    def call(device):
        mine.device = device
        try:
            blocks[device]._stacked_super_weights()
        except threading.BrokenBarrierError as e:
            errors.append(e)

    for b in blocks.values():
        monkeypatch.setattr(b, "_finish_copies", lambda device: both.wait())
    threads = [threading.Thread(target=call, args=(d,)) for d in blocks]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_loading_weights_keeps_the_stack():
    """What is loaded goes into the slices: the stack that a captured graph reads stays the one in use."""
    blk = host_block({1: mlp(1), 4: mlp(2)})
    gu, dn = blk._stacked_super_weights()
    ids = blk._super_global_to_local
    doubled = {k: v * 2 if "experts" in k else v for k, v in blk.state_dict().items()}
    blk.load_state_dict(doubled)
    blk._ensure_runtime_cache(torch.device("cpu"))
    again = blk._stacked_super_weights()
    assert blk._super_global_to_local is ids and again[0] is gu and again[1] is dn and torch.equal(gu[1, :INTER], doubled["experts.4.gate_proj.weight"])
    blk.set_expert(4, mlp(3), packed=False)                  # another module: another stack
    blk._ensure_runtime_cache(torch.device("cpu"))
    assert blk._stacked_super_weights()[0] is not gu


def test_shared_parameters_stay_where_they_are():
    """Ids, or blocks, that share an expert: each would move the parameters to a stack of its own in every call."""
    m = mlp(1)
    blk = host_block({1: m, 4: m})
    before = [w.data_ptr() for w in weights(m)]
    for _ in range(2):
        assert blk._stacked_super_weights() is None and [w.data_ptr() for w in weights(m)] == before
    first, second = host_block({1: m}), host_block({2: m, 3: mlp(2)})
    gu, _ = first._stacked_super_weights()
    for _ in range(2):
        assert second._stacked_super_weights() is None and first._stacked_super_weights()[0] is gu
    fused = torch.randn(2 * INTER, HIDDEN).half()
    views = mlp(3)
    views.gate_proj.weight, views.up_proj.weight = (nn.Parameter(v) for v in fused.chunk(2))
    assert host_block({0: views})._stacked_super_weights() is None and views.up_proj.weight.data_ptr() == fused[INTER].data_ptr()


def test_one_parameter_that_moved_is_taken_back():
    a, b = mlp(1), mlp(2)
    blk = host_block({1: a, 4: b})
    blk._stacked_super_weights()
    want = [w.detach().clone() for m in (a, b) for w in weights(m)]
    want[5] *= 2
    b.down_proj.weight.data = b.down_proj.weight.data * 2
    gu, dn = blk._stacked_super_weights()
    assert all(torch.equal(w, v) for w, v in zip((w for m in (a, b) for w in weights(m)), want)) and torch.equal(dn[1], want[5])


@gpu
def test_a_captured_block_follows_loaded_weights():
    cfg, blk = _qwen_block([1, 2])
    x = torch.randn(1, 24, cfg.hidden, generator=torch.Generator().manual_seed(2)).to(DEV).half()
    with torch.no_grad():
        blk(x)
        stack = blk._super_weights
        idx = torch.tensor([[1, 2]], dtype=torch.int32, device=DEV).expand(24, 2).contiguous()
        w = torch.full((24, 2), 0.5, device=DEV)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = blk._library_super_experts(x[0], idx, w, None)
        state = {k: v * 0.5 if "experts.2.up_proj" in k else v for k, v in blk.state_dict().items()}
        blk.load_state_dict(state)
        blk(x)
        assert blk._super_weights is stack
        g.replay()
        torch.cuda.synchronize()
        helpers.assert_close(out, sum(0.5 * blk.experts[e](x[0]).float() for e in (1, 2)), what="replayed experts")


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


# ---- which modules the library stands in for
class Gelu(DenseMLP):
    def forward(self, x):
        return self.down_proj(nn.functional.gelu(self.gate_proj(x)) * self.up_proj(x))


class Clamped(DenseMLP):
    def forward(self, x):
        return self.down_proj(nn.functional.silu(self.gate_proj(x)).clamp(max=7.0) * self.up_proj(x))


class Swapped(DenseMLP):
    def forward(self, x):
        return self.down_proj(self.gate_proj(x) * nn.functional.silu(self.up_proj(x)))


class Scaled(DenseMLP):
    def forward(self, x):
        return self.down_proj(nn.functional.silu(self.gate_proj(x)) * self.up_proj(x)) * 0.5


class Counting(DenseMLP):
    calls = 0

    def forward(self, x):
        self.calls += 1
        return DenseMLP.forward(self, x)


class Noisy(DenseMLP):
    def forward(self, x):
        h = self.up_proj(x) * nn.functional.silu(self.gate_proj(x))
        return self.down_proj(h + torch.randn_like(h) if self.noise else h)


class Recording(DenseMLP):
    def __init__(self, hidden, inter):
        super().__init__(hidden, inter)
        self.seen = []

    def forward(self, x):
        self.seen.append(x)
        return DenseMLP.forward(self, x)


class CountingSiLU(nn.Module):
    def __init__(self):
        super().__init__()
        self.calls = 0

    def forward(self, x):
        self.calls += 1
        return nn.functional.silu(x)


class WithAct(DenseMLP):
    def __init__(self, hidden, inter, act):
        super().__init__(hidden, inter)
        self.act_fn = act

    def forward(self, x):
        return self.down_proj(torch.mul(self.act_fn(self.gate_proj(x)), self.up_proj(x)))


class LowRankLinear(nn.Linear):
    def forward(self, x):
        return super().forward(x) + x.sum(dim=-1, keepdim=True)


def low_rank():
    m = mlp()
    m.up_proj = LowRankLinear(HIDDEN, INTER, bias=False).half()
    return m


def hooked(name=None, pre=False):
    m = mlp()
    on = m if name is None else getattr(m, name)
    on.register_forward_pre_hook(lambda mod, a: None) if pre else on.register_forward_hook(lambda mod, a, out: out * 2)
    return m


def forward_of_its_own():
    m = mlp()
    m.forward = lambda x: x
    return m


OTHER_KINDS = {
    "another activation in its forward": lambda: Gelu(HIDDEN, INTER).half(), "a clamp": lambda: Clamped(HIDDEN, INTER).half(),
    "gate and up the other way round": lambda: Swapped(HIDDEN, INTER).half(), "a factor": lambda: Scaled(HIDDEN, INTER).half(),
    "writes to itself": lambda: Counting(HIDDEN, INTER).half(), "an activation module": lambda: WithAct(HIDDEN, INTER, nn.GELU()).half(),
    "an activation function": lambda: WithAct(HIDDEN, INTER, torch.tanh).half(), "a record of its calls": lambda: Recording(HIDDEN, INTER).half(),
    "an activation that counts": lambda: WithAct(HIDDEN, INTER, CountingSiLU()).half(), "a Linear of another class": low_rank, "a hook": hooked,
    "a hook on a Linear": lambda: hooked("down_proj"), "a hook before it": lambda: hooked(pre=True), "a forward of its own": forward_of_its_own,
}


@pytest.mark.parametrize("kind", OTHER_KINDS)
def test_modules_of_another_kind_are_not_stacked(kind):
    other = OTHER_KINDS[kind]()
    blk = host_block({1: mlp(1), 4: other})
    where = [w.data_ptr() for w in weights(other)]
    assert blk._stacked_super_weights() is None and [w.data_ptr() for w in weights(other)] == where
    assert not getattr(other, "seen", None) and not getattr(getattr(other, "act_fn", None), "calls", 0)


def test_modules_that_are_swiglu_are_stacked():
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeMLP
    conf = NS(hidden_size=HIDDEN, intermediate_size=INTER, hidden_act="silu")
    kinds = [mlp(), Qwen3MoeMLP(conf).half(), WithAct(HIDDEN, INTER, nn.SiLU()).half(), WithAct(HIDDEN, INTER, nn.functional.silu).half()]
    assert host_block(dict(enumerate(kinds)))._stacked_super_weights()[0].shape == (4, 2 * INTER, HIDDEN)


def test_changes_of_a_module_are_noticed():
    act, noisy = WithAct(HIDDEN, INTER, nn.SiLU()).half(), Noisy(HIDDEN, INTER).half()
    noisy.noise = False
    blk = host_block({1: act, 4: noisy})
    assert blk._stacked_super_weights() is not None
    for change, back in ((lambda: setattr(act, "act_fn", nn.GELU()), lambda: setattr(act, "act_fn", nn.SiLU())),
                         (lambda: setattr(noisy, "noise", True), lambda: setattr(noisy, "noise", False))):
        change()
        assert blk._stacked_super_weights() is None
        back()
        assert blk._stacked_super_weights() is not None
    for on in (act, act.gate_proj, act.act_fn):
        handle = on.register_forward_hook(lambda *a: None)
        assert blk._stacked_super_weights() is None
        handle.remove()
        assert blk._stacked_super_weights() is not None


def test_a_shared_expert_of_another_kind_keeps_its_forward_in_4_bits(monkeypatch):
    """What holds a Linear in 4 bits does not make a SwiGLU of its MLP."""
    from bitsmoe_b200.quant.linear4 import Linear4
    blk = host_block({1: mlp(1)})
    ran = []
    monkeypatch.setattr(blk, "_library_dense_mlp4", lambda *a: ran.append(1) or a[0])
    x = torch.zeros(3, HIDDEN, dtype=torch.float16)
    for kind, runs in ((DenseMLP, 1), (Gelu, 0)):
        m = kind(HIDDEN, INTER)
        for n in ("gate_proj", "up_proj", "down_proj"):
            setattr(m, n, Linear4.from_linear(getattr(m, n), 32))
        del ran[:]
        assert (blk._library_dense_mlp(x, m) is not None) == bool(runs) and len(ran) == runs
