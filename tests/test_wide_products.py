"""GPU: MLPs in fp16 whose product between the two matrices passes fp16's range where their output does not."""
import pytest
import torch

from bitsmoe_b200.layer import dense_experts, dense_mlp4
from tests import dense_bounds as db
from tests.test_gpu_grouped import expert_case, experts_exact
from tests.test_linear4 import mlp_case, mlp_exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP16 = torch.float16


def largest(x, gate, up):
    g, u = x.double() @ gate.double().T, x.double() @ up.double().T
    return float((db.silu(g) * u).abs().max())


@pytest.mark.parametrize("T,k,E,H,I", [(1, 8, 16, 256, 96), (7, 2, 5, 128, 40), (64, 4, 8, 256, 128), (333, 6, 12, 192, 72), (900, 8, 9, 128, 64),
                                       (9, 2, 3, 65, 33), (40, 3, 4, 130, 47), (40, 3, 4, 130, 48), (40, 3, 4, 256, 47), (30001, 32, 32, 512, 64)])
def test_dense_experts(T, k, E, H, I):
    x, idx, w, gu, dn = expert_case(16, T, k, E, H, I, FP16)
    rows = torch.arange(0, T, 3, device=DEV)
    calm = x.clone()
    x[rows] *= 500
    dn *= 2.0 ** -8
    res = torch.randn_like(x)
    assert largest(x[rows], gu[:, :I].reshape(-1, H), gu[:, I:].reshape(-1, H)) > 4 * 65504
    value, err = experts_exact(x, idx, w, gu, dn, residual=res)
    assert float(value.abs().max()) < 65504
    got = dense_experts(x, idx, w, gu, dn, residual=res)
    db.check(got, value, err, what="rows beyond fp16 between the products")
    assert torch.equal(dense_experts(x, idx, w, gu, dn, residual=res), got)
    others = torch.ones(T, dtype=torch.bool, device=DEV)
    others[rows] = False
    assert torch.equal(dense_experts(calm, idx, w, gu, dn, residual=res)[others], got[others])


def test_dense_experts_behind_a_map():
    T, k, E, routed = 90, 6, 3, 40
    x, idx, w, gu, dn = expert_case(17, T, k, E, 128, 48, FP16, routed=routed, dup=True)
    g2l = torch.full((routed,), -1, dtype=torch.int32, device=DEV)
    g2l[5], g2l[17], g2l[30] = 0, 2, 1
    idx[1, :], idx[3, 1], idx[3, 4] = 17, 5, 5
    x *= 600
    dn *= 2.0 ** -9
    value, err = experts_exact(x, idx, w, gu, dn, g2l)
    assert float(value.abs().max()) < 65504
    db.check(dense_experts(x, idx, w, gu, dn, global_to_local=g2l), value, err, what="behind a map")


def test_outputs_beyond_the_range_and_infinite_inputs():
    """What is infinite stays so, in its row alone, with its sign."""
    x, idx, w, gu, dn = expert_case(18, 30, 2, 4, 128, 64, FP16)
    want = dense_experts(x, idx, w, gu, dn)
    bad = x.clone()
    bad[3] *= 3000
    bad[11, 5], bad[12, 7] = float("inf"), float("nan")
    got = dense_experts(bad, idx, w, gu, dn)
    keep = torch.ones(30, dtype=torch.bool, device=DEV)
    keep[[3, 11, 12]] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[12].isnan().all()) and not bool(got[11].isfinite().any())
    value, err = experts_exact(bad[3:4], idx[3:4], w[3:4], gu, dn)
    far = value.abs() - err > 65520
    assert bool(far.any()) and bool((got[3:4][far] == value[far].sign() * float("inf")).all())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 128), (5, 512, 352), (24, 264, 512), (70, 128, 333), (300, 512, 256), (9, 1000, 37), (33, 2056, 1100)])
def test_dense_mlp4(tokens, hidden, inter, group, gated):
    x, packs, mats, tg, res = mlp_case(inter + 1, tokens, hidden, inter, group, FP16)
    rows = torch.arange(0, tokens, 4, device=DEV)
    calm = x.clone()
    x[rows] *= 12000 / hidden ** 0.5
    tg, res = (tg * 2.0 ** -9, res) if gated else (None, None)
    down = (packs[2][0], packs[2][1] * 2.0 ** -4)
    mats = (mats[0], mats[1], mats[2] * 2.0 ** -4)
    assert torch.equal(down[1].float() * 2 ** 4, packs[2][1].float())          # no scale has become subnormal
    assert largest(x[rows], mats[0], mats[1]) > 1.5 * 65504
    value, err = mlp_exact(x, mats, tg, res)
    assert float(value.abs().max()) < 65504
    got = dense_mlp4(x, packs[0], packs[1], down, group, token_gate_weight=tg, residual=res)
    db.check(got, value, err, what="rows beyond fp16 between the products")
    others = torch.ones(tokens, dtype=torch.bool, device=DEV)
    others[rows] = False
    assert torch.equal(dense_mlp4(calm, packs[0], packs[1], down, group, token_gate_weight=tg, residual=res)[others], got[others])


@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_dense_mlp4_with_infinities(tokens):
    """Rows of x, and scales of the down matrix, that are infinite or not a number keep to their rows and columns."""
    x, packs, mats, tg, res = mlp_case(9, tokens, 512, 352, 64, FP16)
    want = dense_mlp4(x, *packs, 64, token_gate_weight=tg, residual=res)
    bad = x.clone()
    bad[0, 3] = float("nan")
    bad[tokens // 2, 5] = float("inf")
    rows = torch.ones(tokens, dtype=torch.bool, device=DEV)
    rows[[0, tokens // 2]] = False
    got = dense_mlp4(bad, *packs, 64, token_gate_weight=tg, residual=res)
    assert torch.equal(got[rows], want[rows]) and not bool(got[~rows].isfinite().any())
    scale = packs[2][1].clone()
    scale[7, 2], scale[300, 0] = float("inf"), float("nan")
    cols = torch.ones(512, dtype=torch.bool, device=DEV)
    cols[[7, 300]] = False
    got = dense_mlp4(x, packs[0], packs[1], (packs[2][0], scale), 64, token_gate_weight=tg, residual=res)
    assert torch.equal(got[:, cols], want[:, cols]) and not bool(got[:, ~cols].isfinite().any())
