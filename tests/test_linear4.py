"""The 4-bit format of dense weights: packing on the CPU; products and MLP on the GPU against their definition in 64 bits."""
import pytest
import torch
import torch.nn as nn

from bitsmoe_b200 import capi
from bitsmoe_b200.layer import dense_mlp4, linear4
from bitsmoe_b200.quant import linear4 as q4
from bitsmoe_b200.quant.quantizer import quantize_symmetric
from tests import dense_bounds as db

DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


# ---- format (CPU)
@pytest.mark.parametrize("k", [1, 7, 8, 31, 32, 33, 100, 256])
def test_codes_come_back(k):
    codes = torch.randint(-8, 8, (5, k), generator=torch.Generator().manual_seed(k)).to(torch.int8)
    payload = q4.pack_codes4(codes)
    assert payload.dtype == torch.uint32 and payload.shape == (5, 4 * (-(-k // 32)))
    assert torch.equal(q4.unpack_codes4(payload, k), codes)
    words = payload.view(torch.int32).to(torch.int64) & 0xFFFFFFFF
    for r, c in ((0, 0), (4, k - 1), (2, k // 2)):
        assert int(words[r, c // 8] >> (4 * (c % 8)) & 15) - 8 == int(codes[r, c])
    if k % 32:
        assert bool((q4.unpack_codes4(payload, payload.shape[1] * 8)[:, k:] == 0).all())


@pytest.mark.parametrize("group", q4.GROUP_SIZES)
def test_quantiser_goes_group_by_group(group):
    w = torch.randn(9, 3 * group + 17, generator=torch.Generator().manual_seed(1)) * 0.02
    w[3, :group] = 0
    payload, scale = q4.quantize_linear4(w, group)
    assert scale.shape == (9, 4) and scale.dtype == torch.float16
    back = q4.dequantize_linear4(payload, scale, w.shape[1], group)
    for j in range(4):
        part = w[:, j * group:(j + 1) * group]
        alone = q4.quantize_linear4(part, group)
        assert torch.equal(q4.dequantize_linear4(*alone, part.shape[1], group), back[:, j * group:(j + 1) * group]) and torch.equal(scale[:, j], alone[1][:, 0])
        codes, s = quantize_symmetric(part, bits=4, dim=1)
        plain = codes.float() * s.unsqueeze(1)
        assert float((back[:, j * group:(j + 1) * group] - part).norm()) < float((plain - part).norm())
    assert not bool(back[3, :group].any())
    assert float((back - w).norm() / w.norm()) < 0.13         # 4-bit symmetric codes of a normal law are off by about 0.1


def test_module_keeps_its_format_and_refuses_a_bias():
    m = q4.Linear4.from_linear(nn.Linear(70, 12, bias=False), 32)
    scale = m.scale.clone()
    for cast in (lambda v: v.half(), lambda v: v.bfloat16(), lambda v: v.float(), lambda v: v.to(torch.float64)):
        cast(nn.Sequential(m))
        assert m.scale.dtype == torch.float16 and torch.equal(m.scale, scale) and m.payload.dtype == torch.uint32
    fresh = q4.Linear4(70, 12, 32)
    fresh.load_state_dict(m.state_dict())
    assert torch.equal(fresh.payload.view(torch.int32), m.payload.view(torch.int32)) and torch.equal(fresh.scale, m.scale)
    with pytest.raises(ValueError):
        q4.Linear4.from_linear(nn.Linear(8, 8))
    with pytest.raises(ValueError):
        q4.Linear4(8, 8, 48)
    with pytest.raises(ValueError):
        q4.quantize_linear4(torch.zeros(4, 4), 16)
    with pytest.raises(RuntimeError):
        m(torch.zeros(2, 70, dtype=torch.float16))          # no CPU path


# ---- products (GPU)
def rnd(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * std).to(dtype).to(DEV)


def matrix4(gen, n, k, group, device=None):
    """Random codes over their whole range, scales of different sizes, and what they stand for in 64 bits."""
    codes = torch.randint(-8, 8, (n, k), generator=gen).to(torch.int8)
    scale = (torch.rand(n, -(-k // group), generator=gen) * 0.02 + 0.002).half()
    w = codes.double() * scale.double().repeat_interleave(group, dim=1)[:, :k]
    return (q4.pack_codes4(codes).to(device or DEV), scale.to(device or DEV)), w.to(device or DEV)


def exact(x, w, residual=None):
    value, err = db.linear(x, w)
    if residual is not None:
        value = value + residual.double()
        err = err + 2.0 ** -23 * (value.abs() + residual.double().abs())
    return value, db.rounded(value, err, x.dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", q4.GROUP_SIZES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 8, 9, 16, 17, 32, 33, 64, 65, 130, 300])
def test_tokens(tokens, group, dtype):
    gen = torch.Generator().manual_seed(tokens)
    m, w = matrix4(gen, 272, 512, group)
    x, res = rnd(gen, tokens, 512, dtype=dtype), rnd(gen, tokens, 272, dtype=dtype)
    db.check(linear4(x, *m, group), *exact(x, w), what="linear4")
    db.check(linear4(x, *m, group, residual=res), *exact(x, w, res), what="with a residual")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,group", [(1, 1, 128), (5, 7, 32), (16, 32, 32), (17, 100, 64), (999, 1000, 128), (64, 129, 128), (48, 127, 128), (2048, 4096, 64),
                                       (31, 8200, 32), (4096, 257, 64), (130, 33, 64), (40000, 64, 32), (24, 20000, 128), (7, 65000, 128), (40, 120000, 64)])
@pytest.mark.parametrize("tokens", [1, 5, 40, 200])
def test_shapes(tokens, n, k, group, dtype):
    gen = torch.Generator().manual_seed(n + k)
    m, w = matrix4(gen, n, k, group)
    x = rnd(gen, tokens, k, dtype=dtype)
    db.check(linear4(x, *m, group), *exact(x, w), what="linear4")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", q4.GROUP_SIZES)
@pytest.mark.parametrize("n,k", [(4100, 4096), (2057, 8192), (20001, 1100)])
@pytest.mark.parametrize("tokens", [17, 24, 33, 64, 131])
def test_matrices_too_large_for_passes(tokens, n, k, group, dtype):
    """Sizes at which more than 16 tokens go to the tensor core: columns shared by two and four CTAs and whole, ends in every direction."""
    gen = torch.Generator().manual_seed(n + tokens)
    m, w = matrix4(gen, n, k, group)
    x, res = rnd(gen, tokens, k, dtype=dtype), rnd(gen, tokens, n, dtype=dtype)
    db.check(linear4(x, *m, group, residual=res), *exact(x, w, res), what="linear4")


@gpu
@pytest.mark.parametrize("tokens", [3, 100])
def test_values_far_from_one(tokens):
    """bf16 activations beyond fp16's range, infinities in one row, rows of zeros, scales of zero and subnormal scales."""
    gen = torch.Generator().manual_seed(3)
    (payload, scale), _ = matrix4(gen, 64, 300, 64)
    scale[0], scale[1, 2] = 0.0, 2.0 ** -24
    w = q4.unpack_codes4(payload, 300).double() * scale.double().repeat_interleave(64, dim=1)[:, :300]
    x = rnd(gen, tokens, 300, dtype=torch.bfloat16) * 1e6
    x[1] = 0
    db.check(linear4(x, payload, scale, 64), *exact(x, w), what="large rows")
    want = linear4(x, payload, scale, 64)
    x[2, 299] = float("inf")
    got = linear4(x, payload, scale, 64)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[3:], want[3:]) and not bool(got[2].isfinite().any())
    small = rnd(gen, tokens, 300, dtype=torch.float16) * 2.0 ** -13        # many of them subnormal
    db.check(linear4(small, payload, scale, 64), *exact(small, w), what="small rows")


@gpu
def test_code_zero_is_exact_and_sums_do_not_drift():
    """A matrix of code 0 gives zeros, one of equal codes a long sum of equal signs."""
    x = torch.full((2, 4096), 3.0, dtype=torch.float16, device=DEV)
    scale = torch.full((16, 32), 0.01, dtype=torch.float16, device=DEV)
    zero = q4.pack_codes4(torch.zeros(16, 4096, dtype=torch.int8, device=DEV))
    assert not bool(linear4(x, zero, scale).any())
    seven = q4.pack_codes4(torch.full((16, 4096), 7, dtype=torch.int8, device=DEV))
    want = 4096 * 3.0 * 7 * float(scale[0, 0])
    assert float((linear4(x, seven, scale).double() - want).abs().max()) <= want * (db.half_step(torch.float16) + 2.0 ** -20)


def mlp_case(seed, tokens, hidden, inter, group, dtype):
    gen = torch.Generator().manual_seed(seed)
    packs, mats = zip(*(matrix4(gen, *s, group) for s in ((inter, hidden), (inter, hidden), (hidden, inter))))
    return rnd(gen, tokens, hidden, std=0.3, dtype=dtype), packs, mats, rnd(gen, hidden, std=0.05, dtype=torch.float16), rnd(gen, tokens, hidden, dtype=dtype)


def mlp_exact(x, mats, token_gate, residual):
    y, err = db.swiglu(x, *mats, x.dtype)
    if token_gate is not None:
        logit, le = db.linear(x, token_gate.reshape(1, -1))
        f = torch.sigmoid(logit)
        err = f * err + (y.abs() + err) * (0.25 * le + db.EXP_REL * f)          # |sigmoid'| <= 1/4
        y = f * y
    if residual is not None:
        err = err + 2.0 ** -23 * (y.abs() + residual.double().abs())
        y = y + residual.double()
    return y, db.rounded(y, err, x.dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", q4.GROUP_SIZES)
@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 128), (5, 512, 352), (24, 264, 512), (70, 128, 333), (300, 512, 256), (1, 64, 1), (9, 1000, 37)])
def test_mlp(tokens, hidden, inter, group, dtype):
    x, packs, mats, tg, res = mlp_case(inter, tokens, hidden, inter, group, dtype)
    db.check(dense_mlp4(x, *packs, group), *mlp_exact(x, mats, None, None), what="mlp4")
    db.check(dense_mlp4(x, *packs, group, token_gate_weight=tg, residual=res), *mlp_exact(x, mats, tg, res), what="mlp4, gated, residual")
    db.check(dense_mlp4(x, *packs, group, token_gate_weight=tg.reshape(1, -1)), *mlp_exact(x, mats, tg, None), what="mlp4, gated")


@gpu
def test_strided_and_unaligned_rows():
    gen = torch.Generator().manual_seed(4)
    m, w = matrix4(gen, 40, 96, 32)
    wide = rnd(gen, 6, 200, dtype=torch.float16)
    db.check(linear4(wide[:, 5:101], *m, 32), *exact(wide[:, 5:101], w), what="strided")
    flat = rnd(gen, 6 * 96 + 1, dtype=torch.float16)[1:].view(6, 96)
    db.check(linear4(flat, *m, 32), *exact(flat, w), what="unaligned")
    res = rnd(gen, 40, 6).t()
    db.check(linear4(flat, *m, 32, residual=res), *exact(flat, w, res.half()), what="strided fp32 residual")
    assert linear4(flat[:0], *m, 32).shape == (0, 40)


@gpu
@pytest.mark.parametrize("tokens,hidden,inter", [(33, 2056, 4100), (150, 4096, 2050)])
def test_mlp_on_the_tensor_core(tokens, hidden, inter):
    x, packs, mats, tg, res = mlp_case(inter, tokens, hidden, inter, 128, torch.bfloat16)
    db.check(dense_mlp4(x, *packs, 128, token_gate_weight=tg, residual=res), *mlp_exact(x, mats, tg, res), what="mlp4")


@gpu
@pytest.mark.parametrize("tokens", [2, 150])
def test_streams_graphs_and_repeats(tokens):
    x, packs, _, tg, res = mlp_case(6, tokens, 512, 384, 128, torch.bfloat16)
    want = dense_mlp4(x, *packs, 128, token_gate_weight=tg, residual=res)
    for _ in range(3):
        assert torch.equal(dense_mlp4(x, *packs, 128, token_gate_weight=tg, residual=res), want)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = dense_mlp4(x, *packs, 128, token_gate_weight=tg, residual=res)
    side.synchronize()
    assert torch.equal(other, want)
    static, outs, graphs = torch.zeros_like(x), [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(dense_mlp4(static, *packs, 128, token_gate_weight=tg, residual=res))
        graphs.append(g)
    static.copy_(x)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens", [1, 40])
def test_weights_written_by_the_launch_before(tokens, gated):
    """Scales of the down matrix that a product of this library has just computed: its launch lets the next ones start early, and the down
    product fetches weights before it waits.  Every round writes other scales to the same place."""
    hidden, inter, group = 2048, 1024, 32
    x, packs, _, tg, res = mlp_case(21, tokens, hidden, inter, group, torch.float16)
    gen = torch.Generator().manual_seed(22)
    maker, _ = matrix4(gen, inter // group, 8192, 128)
    sources = [rnd(gen, hidden, 8192, std=0.02, dtype=torch.float16) for _ in range(3)]
    tg = tg if gated else None
    want = []
    for src in sources:
        s = linear4(src, *maker)
        torch.cuda.synchronize()
        want.append(dense_mlp4(x, packs[0], packs[1], (packs[2][0], s), group, token_gate_weight=tg, residual=res).clone())
        torch.cuda.synchronize()
        del s
    assert not torch.equal(want[0], want[1])
    for i in range(30):
        s = linear4(sources[i % 3], *maker)
        got = dense_mlp4(x, packs[0], packs[1], (packs[2][0], s), group, token_gate_weight=tg, residual=res)
        assert torch.equal(got, want[i % 3]), i
        del s, got


@gpu
def test_module_runs_on_the_kernels():
    lin = nn.Linear(192, 80, bias=False, device=DEV).half()
    m = q4.Linear4.from_linear(lin, 64)
    x = torch.randn(2, 7, 192, device=DEV).half()
    w = q4.dequantize_linear4(m.payload, m.scale, 192, 64)
    with torch.no_grad():
        got = m(x)
    assert got.shape == (2, 7, 80)
    db.check(got.reshape(14, 80), *exact(x.reshape(14, 192), w), what="Linear4")


@gpu
def test_refusals():
    gen = torch.Generator().manual_seed(7)
    (p, s), _ = matrix4(gen, 24, 96, 32)
    x = torch.zeros(4, 96, dtype=torch.float16, device=DEV)
    wrong = [lambda: linear4(x.float(), p, s, 32), lambda: linear4(x[:, :64], p, s, 32), lambda: linear4(x, p, s, 64), lambda: linear4(x, p, s, 48),
             lambda: linear4(x.cpu(), p, s, 32), lambda: linear4(x, p.cpu(), s, 32), lambda: linear4(x, p, s.cpu(), 32), lambda: linear4(x, p.view(torch.int32), s, 32),
             lambda: linear4(x, p, s.bfloat16(), 32), lambda: linear4(x, p[:-1], s, 32), lambda: linear4(x, p, s[:, :-1], 32), lambda: linear4(x[0], p, s, 32),
             lambda: linear4(x, p, s, 32, residual=torch.zeros(4, 23, dtype=torch.float16, device=DEV)), lambda: linear4(x, p.repeat(1, 2)[:, ::2], s, 32),
             lambda: linear4(x.clone().requires_grad_(), p, s, 32), lambda: linear4(x, p, s, 32, residual=torch.zeros(4, 24, dtype=torch.float16))]
    (d, ds), _ = matrix4(gen, 96, 24, 32)
    good = [(p, s), (p, s), (d, ds)]
    assert dense_mlp4(x, *good, 32).shape == (4, 96)
    for i in range(3):
        bad = list(good)
        bad[i] = (d, ds) if i < 2 else (p, s)
        wrong.append(lambda bad=bad: dense_mlp4(x, *bad, 32))
    wrong += [lambda: dense_mlp4(x, *good, 32, token_gate_weight=torch.zeros(95, dtype=torch.float16, device=DEV)),
              lambda: dense_mlp4(x, *good, 32, token_gate_weight=torch.zeros(96, dtype=torch.float16)),
              lambda: dense_mlp4(x, *good, 32, residual=torch.zeros(3, 96, dtype=torch.float16, device=DEV)),
              lambda: dense_mlp4(x.clone().requires_grad_(), *good, 32), lambda: dense_mlp4(x.float(), *good, 32)]
    for i, call in enumerate(wrong):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    lib, q, st = capi.lib(), x.data_ptr(), capi.stream_ptr(torch.device(DEV))
    assert lib.bm_linear4(q, 0, p.data_ptr(), s.data_ptr(), 4, 96, 24, 16, None, q, st) == 2
    assert lib.bm_linear4(q, 2, p.data_ptr(), s.data_ptr(), 4, 96, 24, 32, None, q, st) == 1
    assert lib.bm_linear4(q, 0, p.data_ptr() + 4, s.data_ptr(), 4, 96, 24, 32, None, q, st) == 1
    assert lib.bm_linear4(q, 0, None, s.data_ptr(), 4, 96, 24, 32, None, q, st) == 1
    assert lib.bm_linear4(q, 0, p.data_ptr(), s.data_ptr(), 0, 96, 24, 32, None, q, st) == 0
    need = lib.bm_dense_mlp4_workspace_bytes(4, 24)
    ptrs = [v.data_ptr() for pair in good for v in pair]
    assert lib.bm_dense_mlp4_forward(q, 0, *ptrs, None, 4, 96, 24, 32, None, q, q, need - 1, st) == 4
