"""The dense parts of a MoE block on the library's kernels: un-quantised experts, shared experts and projections in 4 bits."""
import copy
from types import SimpleNamespace as NS

import pytest
import torch
import torch.nn as nn

from bitsmoe_b200 import synth
from bitsmoe_b200.models.auto import quantize_dense_inplace
from bitsmoe_b200.quant import linear4 as q4
from tests import helpers
from tests.test_gpu_blocks import DenseMLP, StubMoEGate, _conf, _fill

DEV = "cuda:0"
gpu = pytest.mark.gpu


def _qwen_block(supers, dtype=torch.float16, seed=9):
    from bitsmoe_b200.models.qwen3moe.bitsmoe_block import BitsMoE_Qwen3MoeSparseMoeBlock
    from bitsmoe_b200.models.qwen3moe.bitsmoe_mlp import BitsMoE_Qwen3MoeMLP
    torch.manual_seed(seed)
    cfg = synth.tiny(hidden=256, num_experts=8, intermediate=256, top_k=3, rank=64)
    layer = synth.make_layer(cfg, seed=seed, keep_full=True)
    conf = _conf(cfg)
    src = NS(gate=nn.Linear(cfg.hidden, cfg.num_experts, bias=False), experts=[None] * cfg.num_experts)
    blk = BitsMoE_Qwen3MoeSparseMoeBlock(conf, 3, src, super_experts=supers, copy_source_experts=False).to(DEV, dtype)
    _fill(blk, BitsMoE_Qwen3MoeMLP, conf, layer, skip=supers)
    for e in supers:
        blk.set_expert(e, DenseMLP(cfg.hidden, 384).to(DEV, dtype), packed=False)
    return cfg, blk


def _by_modules(blk, x):
    """The same block with its dense experts as torch modules: autograd on."""
    with torch.enable_grad():
        y, logits = blk(x)
    return y.detach(), logits.detach()


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 13, 300])
def test_block_with_super_experts_runs_them_in_the_library(tokens, dtype):
    cfg, blk = _qwen_block([2, 5], dtype)
    x = (torch.randn(1, tokens, cfg.hidden, generator=torch.Generator().manual_seed(tokens)) * 1.0).to(DEV, dtype)
    want, _ = _by_modules(blk, x)
    called = []
    real = blk._library_super_experts
    blk._library_super_experts = lambda *a: called.append(1) or real(*a)
    with torch.no_grad():
        got, _ = blk(x)
    assert called and blk._super_weights is not None
    eps = torch.finfo(dtype).eps
    # torch rounds after every product, sum and scaling (six times), this path between the products and at the end
    helpers.assert_close(got, want, rtol=8 * eps, atol=8 * eps * float(want.abs().max()), rel_max=8 * eps, rel_l2=4 * eps, what="super experts")
    dense = blk(x)[0] - 0     # still callable with autograd on afterwards
    helpers.assert_close(dense, want, what="modules again")


@gpu
def test_super_experts_follow_their_parameters():
    cfg, blk = _qwen_block([2, 5])
    x = torch.randn(1, 40, cfg.hidden, generator=torch.Generator().manual_seed(1)).to(DEV).half()
    with torch.no_grad():
        first, _ = blk(x)
        held = blk._super_weights
        w = blk.experts[5].down_proj.weight
        assert w.data_ptr() == held[1][1].data_ptr()                   # a slice of the stack, not a copy
        w.mul_(2.0)                                                     # in place
        second, _ = blk(x)
        helpers.assert_close(second, _by_modules(blk, x)[0], what="after an update in place")
        assert float((second - first).abs().max()) > 0
        blk.experts[5].down_proj.weight.data = w.data.clone().mul_(0.25)    # storage of its own
        third, _ = blk(x)
        helpers.assert_close(third, _by_modules(blk, x)[0], what="after an exchange of the storage")
        assert blk._super_weights is not held
        blk.load_state_dict({k: v.clone() * (0.5 if "experts.2.up_proj" in k else 1) if v.dtype == torch.float16 else v for k, v in blk.state_dict().items()})
        fourth, _ = blk(x)
        helpers.assert_close(fourth, _by_modules(blk, x)[0], what="after load_state_dict")
        other = copy.deepcopy(blk.experts[2])
        blk.set_expert(2, other, packed=False)
        other.gate_proj.weight.zero_()
        fifth, _ = blk(x)
        helpers.assert_close(fifth, _by_modules(blk, x)[0], what="after set_expert")
        assert bool(blk.experts[2].gate_proj.weight.any()) is False


@gpu
def test_block_with_super_experts_can_be_captured():
    cfg, blk = _qwen_block([1, 2, 7])
    gen = torch.Generator().manual_seed(2)
    xs = [torch.randn(1, 24, cfg.hidden, generator=gen).to(DEV).half() for _ in range(2)]
    with torch.no_grad():
        want = [blk(x)[0] for x in xs]
        static = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            blk(static)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, _ = blk(static)
        for x, w in zip(xs, want):
            static.copy_(x)
            g.replay()
            torch.cuda.synchronize()
            helpers.assert_close(out, w, what="replayed block")


@gpu
def test_first_call_in_inference_mode_leaves_ordinary_parameters():
    cfg, blk = _qwen_block([2, 5])
    x = torch.randn(1, 7, cfg.hidden, generator=torch.Generator().manual_seed(4)).to(DEV).half()
    with torch.inference_mode():
        first, _ = blk(x)
    assert blk._super_weights is not None
    w = blk.experts[5].gate_proj.weight
    assert not w.is_inference() and not blk._super_weights[0].is_inference()
    blk.experts[5](x[0]).float().sum().backward()                       # the modules still train
    assert w.grad is not None and w.grad.shape == w.shape
    with torch.no_grad():
        w.mul_(0.5)
        helpers.assert_close(blk(x)[0], _by_modules(blk, x)[0], what="after inference mode")


@gpu
def test_modules_of_another_kind_keep_their_own_forward():
    cfg, blk = _qwen_block([2])
    x = torch.randn(1, 9, cfg.hidden, generator=torch.Generator().manual_seed(3)).to(DEV).half()
    mlp = DenseMLP(cfg.hidden, 64).to(DEV).half()
    mlp.up_proj = nn.Linear(cfg.hidden, 64, bias=True).to(DEV).half()
    blk.set_expert(2, mlp, packed=False)
    with torch.no_grad():
        got, _ = blk(x)
        assert blk._super_weights is None
    helpers.assert_close(got, _by_modules(blk, x)[0], what="experts with a bias")


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [2, 70])
def test_shared_expert_in_4_bits(tokens, dtype):
    """Blocks with a gated shared expert (and un-quantised experts beside it): the 4-bit block against the same block whose shared
    expert holds the dequantised weights."""
    from bitsmoe_b200.models.qwen3next.bitsmoe_block import BitsMoE_Qwen3NextSparseMoeBlock
    from bitsmoe_b200.models.qwen3next.bitsmoe_mlp import BitsMoE_Qwen3NextMLP
    torch.manual_seed(11)
    cfg = synth.tiny(hidden=256, num_experts=16, intermediate=128, top_k=4, rank=48, shared_intermediate=192, shared_gated=True)
    layer = synth.make_layer(cfg, seed=10, keep_full=True)
    conf = _conf(cfg)
    shared = DenseMLP(cfg.hidden, cfg.shared_intermediate)
    src = NS(gate=nn.Linear(cfg.hidden, cfg.num_experts, bias=False), experts=[None] * cfg.num_experts, shared_expert=shared,
             shared_expert_gate=nn.Linear(cfg.hidden, 1, bias=False))
    blk = BitsMoE_Qwen3NextSparseMoeBlock(conf, 0, src, super_experts=[3], copy_source_experts=False).to(DEV, dtype)
    _fill(blk, BitsMoE_Qwen3NextMLP, conf, layer, skip=(3,))
    blk.set_expert(3, DenseMLP(cfg.hidden, 128).to(DEV, dtype), packed=False)
    assert blk.quantize_shared_experts(64) == 3 and blk.quantize_shared_experts(64) == 0
    x = torch.randn(1, tokens, cfg.hidden, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    ref = copy.deepcopy(blk)
    for n in ("gate_proj", "up_proj", "down_proj"):
        m = getattr(ref.shared_expert, n)
        lin = nn.Linear(m.in_features, m.out_features, bias=False, device=DEV, dtype=torch.float32)
        lin.weight.data = q4.dequantize_linear4(m.payload, m.scale, m.in_features, m.group_size)
        setattr(ref.shared_expert, n, lin.to(torch.float16 if dtype == torch.float16 else dtype))
    with torch.no_grad():
        got, want = blk(x)[0], ref(x)[0]
        helpers.assert_close(blk.to(dtype)(x)[0], got, what="cast again")
    helpers.assert_close(got, want, what="shared expert in 4 bits")
    helpers.assert_detects_damage(got, want)
    helpers.assert_close(_by_modules(blk, x)[0], want, what="modules with autograd on")


@gpu
def test_deepseek_block_with_super_experts_and_4_bit_shared_experts():
    from bitsmoe_b200.models.deepseekv2.bitsmoe_block import BitsMoE_DeepSeekSparseMoeBlock
    from bitsmoe_b200.models.deepseekv2.bitsmoe_mlp import BitsMoE_DeepSeekMLP
    torch.manual_seed(5)
    cfg = synth.tiny(hidden=256, num_experts=8, intermediate=160, top_k=3, rank=40, bit_probs=((2, 1.0),), norm_topk_prob=False, shared_intermediate=320)
    layer = synth.make_layer(cfg, seed=12, keep_full=True)
    conf = _conf(cfg, n_shared_experts=2)
    src = NS(gate=StubMoEGate(cfg.hidden, cfg.num_experts, cfg.top_k), experts=[None] * cfg.num_experts,
             shared_experts=DenseMLP(cfg.hidden, cfg.shared_intermediate).half())
    blk = BitsMoE_DeepSeekSparseMoeBlock(conf, 1, src, super_experts=[0, 6], copy_source_experts=False).to(DEV).eval()
    _fill(blk, BitsMoE_DeepSeekMLP, conf, layer, skip=(0, 6))
    for e in (0, 6):
        blk.set_expert(e, DenseMLP(cfg.hidden, 96).to(DEV).half(), packed=False)
    x = synth.activations(cfg, 60, seed=3, dtype=torch.float16).reshape(2, 30, cfg.hidden).to(DEV)
    with torch.no_grad():
        before = blk(x)
        with torch.enable_grad():
            modules = blk(x).detach()
        helpers.assert_close(before, modules, what="DeepSeek block with super experts")
        assert blk._super_weights is not None
        assert blk.quantize_shared_experts() == 3
        after = blk(x)
    with torch.enable_grad():
        helpers.assert_close(after, blk(x).detach(), what="4-bit shared experts")
    assert 1e-3 < float((after.float() - before.float()).norm() / before.float().norm()) < 0.3      # the weights did change, a little


# ---- projections of a patched model
def _tiny_model():
    transformers = pytest.importorskip("transformers")
    from bitsmoe_b200.models.auto import build_patched_model
    from tests import test_patcher as tp
    cfg = tp._config()
    _, state, _ = tp._checkpoint(cfg)
    return tp, transformers, build_patched_model(cfg, "qwen3moe", state, super_experts_by_layer=tp.SUPER)


def test_quantize_dense_replaces_projections_and_nothing_else():
    tp, _, model = _tiny_model()
    names = {n for n, m in model.named_modules() if isinstance(m, nn.Linear)}
    assert quantize_dense_inplace(model, group_size=32) == 4 * tp.LAYERS
    left = {n for n, m in model.named_modules() if isinstance(m, nn.Linear)}
    gone = names - left
    assert len(gone) == 4 * tp.LAYERS and all(n.split(".")[-1] in ("q_proj", "k_proj", "v_proj", "o_proj") for n in gone)
    assert quantize_dense_inplace(model, group_size=32) == 0
    assert isinstance(model.model.layers[0].self_attn.q_proj, q4.Linear4)


@gpu
def test_patched_model_runs_with_4_bit_projections():
    _, _, model = _tiny_model()
    quantize_dense_inplace(model, group_size=32)
    model = model.to(DEV).eval()
    ref = copy.deepcopy(model)
    for layer in ref.model.layers:
        for n in ("q_proj", "k_proj", "v_proj", "o_proj"):
            m = getattr(layer.self_attn, n)
            lin = nn.Linear(m.in_features, m.out_features, bias=False, device=DEV, dtype=torch.float16)
            lin.weight.data = q4.dequantize_linear4(m.payload, m.scale, m.in_features, m.group_size).half()
            setattr(layer.self_attn, n, lin)
    ids = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(3)).to(DEV)
    with torch.no_grad():
        got, want = model(input_ids=ids).logits, ref(input_ids=ids).logits
    helpers.assert_close(got, want, atol=2e-2 * float(want.abs().max()), what="logits")
