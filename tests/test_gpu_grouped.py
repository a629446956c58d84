"""GPU: products grouped by expert and un-quantised experts against their definition in 64 bits."""
import pytest
import torch

from bitsmoe_b200 import capi
from bitsmoe_b200.layer import dense_experts, grouped_linear, route_build, route_topk
from tests import dense_bounds as db

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16]


def rnd(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * std).to(dtype).to(DEV)


def offsets(sizes):
    return torch.tensor([0] + list(torch.tensor(sizes).cumsum(0)), dtype=torch.int32, device=DEV)


def grouped_exact(x, w, sizes, index=None):
    value = torch.zeros(sum(sizes), w.shape[1], dtype=torch.float64, device=DEV)
    err, at = torch.zeros_like(value), 0
    rows = torch.arange(sum(sizes), device=DEV) if index is None else index.long()
    for e, n in enumerate(sizes):
        r = rows[at:at + n]
        live = (r >= 0) & (r < x.shape[0])
        xe = torch.where(live[:, None], x[torch.where(live, r, 0)], torch.zeros_like(x[:1]))
        value[at:at + n], err[at:at + n] = db.linear(xe, w[e])
        at += n
    return value, db.rounded(value, err, x.dtype)


SIZES = {
    "one row": [1],
    "one group": [300],
    "empty groups around": [0, 0, 5, 0, 17, 0],
    "every size at a tile's edge": [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 2],
    "one long among short": [3, 1, 700, 2, 0, 1],
    "many groups": [(7 * i) % 5 for i in range(200)],
    "more groups than the tensor-core kernel's table holds": [(7 * i) % 3 for i in range(1100)],
    "rows enough to be brought into order first": [150, 0, 90, 131],
}
SHAPES = [(64, 128), (2048, 256), (768, 2048), (200, 136), (8, 1), (1000, 999), (72, 257)]     # (K, N): rows of 16-byte multiples
ODD = [(67, 33), (1, 1), (129, 70), (1001, 48)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("sizes", SIZES)
def test_group_sizes(sizes, gather, dtype):
    gen = torch.Generator().manual_seed(1)
    sizes = SIZES[sizes]
    A, K, N = sum(sizes), 192, 272
    x = rnd(gen, 41 if gather else A, K, dtype=dtype)
    w = rnd(gen, len(sizes), N, K, std=0.05, dtype=dtype)
    index = torch.randint(0, 41, (A,), generator=gen).to(torch.int32).to(DEV) if gather else None      # rows come up several times
    got = grouped_linear(x, w, offsets(sizes), index)
    db.check(got, *grouped_exact(x, w, sizes, index), what="grouped_linear")
    assert got.dtype == dtype


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES + ODD)
def test_shapes(shape, dtype):
    gen = torch.Generator().manual_seed(2)
    (K, N), sizes = shape, [5, 0, 40, 1]
    x, w = rnd(gen, 20, K, dtype=dtype), rnd(gen, 4, N, K, std=0.05, dtype=dtype)
    index = torch.randint(0, 20, (46,), generator=gen).to(torch.int32).to(DEV)
    db.check(grouped_linear(x, w, offsets(sizes), index), *grouped_exact(x, w, sizes, index), what="grouped_linear")
    x = rnd(gen, 46, K, dtype=dtype)
    db.check(grouped_linear(x, w, offsets(sizes)), *grouped_exact(x, w, sizes), what="grouped_linear, rows in order")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [96, 67])
def test_rows_that_no_expert_owns_stay(K, dtype):
    gen = torch.Generator().manual_seed(3)
    x, w = rnd(gen, 40, K, dtype=dtype), rnd(gen, 3, 48, K, std=0.1, dtype=dtype)
    out = torch.full((40, 48), 7.0, dtype=dtype, device=DEV)
    off = torch.tensor([2, 9, 9, 30], dtype=torch.int32, device=DEV)
    got = grouped_linear(x, w, off, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[:2] == 7).all()) and bool((out[30:] == 7).all())
    value, err = grouped_exact(x[2:], w, [7, 0, 21])
    db.check(out[2:30], value, err, what="rows owned")
    before = out.clone()
    assert torch.equal(grouped_linear(x, w, torch.zeros(4, dtype=torch.int32, device=DEV), out=out), before)


@pytest.mark.parametrize("K", [96, 67])
def test_indices_and_offsets_outside_their_ranges_are_harmless(K):
    """Tables come from the device, where the host cannot check them: an index outside x stands for zeros, offsets are limited to
    the rows there are, and a group whose end lies before its start is empty."""
    gen = torch.Generator().manual_seed(4)
    x, w = rnd(gen, 10, K, dtype=torch.float16), rnd(gen, 3, 24, K, std=0.1, dtype=torch.float16)
    index = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, -2 ** 31, 3, 4], dtype=torch.int32, device=DEV)
    db.check(grouped_linear(x, w, offsets([3, 2, 3]), index), *grouped_exact(x, w, [3, 2, 3], index), what="indices outside")
    out = torch.full((8, 24), 7.0, dtype=torch.float16, device=DEV)
    grouped_linear(x, w, torch.tensor([-5, 3, 1, 2 ** 30], dtype=torch.int32, device=DEV), index, out=out)       # [0, 3), none, [1, 8)
    value, err = grouped_exact(x, w[2:], [8], index)
    db.check(out[3:], value[3:], err[3:], what="offsets outside")


def test_offsets_that_descend_own_the_rows_before():
    """[0, 500), then a group whose end lies before its start: long enough to be brought into order first, to scratch that holds NaN."""
    gen = torch.Generator().manual_seed(14)
    x, w = rnd(gen, 40, 64, dtype=torch.float16), rnd(gen, 2, 72, 64, std=0.1, dtype=torch.float16)
    index = torch.randint(0, 40, (500,), generator=gen).to(torch.int32).to(DEV)
    out = torch.zeros(500, 72, dtype=torch.float16, device=DEV)
    poison = torch.full((500 * 64,), float("nan"), dtype=torch.float16, device=DEV)
    del poison
    grouped_linear(x, w, torch.tensor([0, 500, 400], dtype=torch.int32, device=DEV), index, out=out)
    db.check(out, *grouped_exact(x, w, [500, 0], index), what="descending offsets")


def test_nothing_to_do():
    x, w = torch.zeros(0, 64, dtype=torch.float16, device=DEV), torch.zeros(2, 32, 64, dtype=torch.float16, device=DEV)
    assert grouped_linear(x, w, offsets([0, 0])).shape == (0, 32)
    assert grouped_linear(torch.zeros(4, 64, dtype=torch.float16, device=DEV), w[:0], offsets([])).shape == (4, 32)
    nowhere = torch.tensor([0, -1, 5], dtype=torch.int32, device=DEV)             # no rows to pick from: rows of zeros
    assert not bool(grouped_linear(x, w + 1, offsets([1, 2]), nowhere).any())
    idx, tw = torch.zeros(0, 2, dtype=torch.int32, device=DEV), torch.zeros(0, 2, device=DEV)
    assert dense_experts(x, idx, tw, torch.zeros(1, 64, 64, dtype=torch.float16, device=DEV), torch.zeros(1, 64, 32, dtype=torch.float16, device=DEV)).shape == (0, 64)


def test_infinities_stay_in_their_rows():
    """A row with inf and NaN is nobody else's business, in its tile, its group or the next group."""
    gen = torch.Generator().manual_seed(5)
    x, w = rnd(gen, 50, 128, dtype=torch.bfloat16), rnd(gen, 2, 64, 128, std=0.1, dtype=torch.bfloat16)
    want = grouped_linear(x, w, offsets([20, 30]))
    bad = x.clone()
    bad[19, 3], bad[20, 5] = float("nan"), float("inf")
    got = grouped_linear(bad, w, offsets([20, 30]))
    keep = torch.ones(50, dtype=torch.bool, device=DEV)
    keep[19:21] = False
    assert torch.equal(got[keep], want[keep])
    assert bool(got[19].isnan().all()) and not bool(got[20].isfinite().any())
    big = grouped_linear(torch.full((3, 64), 300.0, dtype=torch.bfloat16, device=DEV), torch.full((1, 8, 64), 30000.0, dtype=torch.bfloat16, device=DEV), offsets([3]))
    assert bool((big == big[0, 0]).all()) and abs(float(big[0, 0]) / (64 * 300.0 * 30000.0) - 1) < 0.02      # past fp16's range


# ---- un-quantised experts
def selection(gen, T, k, routed, dup=False):
    if dup:
        idx = torch.randint(0, routed, (T, k), generator=gen)
    else:
        idx = torch.argsort(torch.rand(T, routed, generator=gen), dim=1)[:, :k]
    return idx.to(torch.int32).to(DEV), torch.rand(T, k, generator=gen).to(DEV)


def experts_exact(x, idx, w, gate_up, down, g2l=None, residual=None):
    E, I = down.shape[0], down.shape[2]
    local = idx.long()
    ok = (local >= 0) & (local < (E if g2l is None else g2l.numel()))
    local = torch.where(ok, local if g2l is None else g2l.long()[torch.where(ok, local, 0)], -1)
    value = torch.zeros(x.shape, dtype=torch.float64, device=DEV) if residual is None else residual.double()
    err, size = torch.zeros_like(value), value.abs()
    for e in range(E):
        t, s = torch.nonzero(local == e, as_tuple=True)
        if t.numel():
            d, de = db.swiglu(x[t], gate_up[e, :I], gate_up[e, I:], down[e], x.dtype)
            ws = w.double()[t, s, None]
            value = value.index_add(0, t, ws * d)
            err = err.index_add(0, t, ws.abs() * de)
            size = size.index_add(0, t, (ws * d).abs())
    return value, db.rounded(value, err + (idx.shape[1] + 1) * 2.0 ** -23 * size, x.dtype)


def expert_case(seed, T, k, E, H, I, dtype, routed=None, dup=False):
    gen = torch.Generator().manual_seed(seed)
    idx, w = selection(gen, T, k, routed or E, dup)
    return rnd(gen, T, H, dtype=dtype), idx, w, rnd(gen, E, 2 * I, H, std=0.08, dtype=dtype), rnd(gen, E, H, I, std=0.08, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,H,I", [(1, 1, 1, 64, 64), (1, 8, 16, 256, 96), (7, 2, 5, 128, 40), (64, 4, 8, 256, 128), (333, 6, 12, 192, 72),
                                       (2100, 8, 9, 128, 64), (5, 32, 40, 64, 32), (9, 2, 3, 65, 33), (200, 1, 2, 264, 136)])
def test_dense_experts(T, k, E, H, I, dtype):
    x, idx, w, gu, dn = expert_case(6, T, k, E, H, I, dtype)
    got = dense_experts(x, idx, w, gu, dn)
    db.check(got, *experts_exact(x, idx, w, gu, dn), what="dense_experts")
    res = torch.randn_like(x)
    db.check(dense_experts(x, idx.long(), w, gu, dn, residual=res), *experts_exact(x, idx, w, gu, dn, residual=res), what="with a residual")
    assert torch.equal(dense_experts(x, idx, w, gu, dn), got)          # the same bits from run to run


@pytest.mark.parametrize("dtype", TYPES)
def test_dense_experts_behind_a_map(dtype):
    """Experts held elsewhere, ids outside the map and map entries outside the experts held here add nothing; an expert that a
    token names twice counts twice; tokens with no expert here keep their residual."""
    T, k, E, routed = 90, 6, 3, 40
    x, idx, w, gu, dn = expert_case(7, T, k, E, 128, 48, dtype, routed=routed, dup=True)
    g2l = torch.full((routed,), -1, dtype=torch.int32, device=DEV)
    g2l[5], g2l[17], g2l[30], g2l[31] = 0, 2, 1, 99
    idx[0, 0], idx[0, 1], idx[1, :], idx[2, :] = -7, 2 ** 31 - 1, 17, 6
    idx[3, 1], idx[3, 4] = 5, 5
    res = torch.randn_like(x)
    clean = torch.where(g2l == 99, -1, g2l)
    got = dense_experts(x, idx, w, gu, dn, global_to_local=g2l, residual=res)
    db.check(got, *experts_exact(x, idx, w, gu, dn, clean, res), what="behind a map")
    assert torch.equal(got[2], res[2])
    none = torch.full_like(g2l, -1)
    assert torch.equal(dense_experts(x, idx, w, gu, dn, global_to_local=none, residual=res), res)
    assert not bool(dense_experts(x, idx, w, gu, dn, global_to_local=none).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_few_held_experts_of_many(dtype):
    """A long batch of which three of 300 experts are held here: lists much longer than what is in them."""
    T, k, E, routed = 3000, 10, 3, 300
    x, idx, w, gu, dn = expert_case(12, T, k, E, 64, 40, dtype, routed=routed)
    g2l = torch.full((routed,), -1, dtype=torch.int32, device=DEV)
    g2l[7], g2l[100], g2l[299] = 2, 0, 1
    res = torch.randn_like(x)
    got = dense_experts(x, idx, w, gu, dn, global_to_local=g2l, residual=res)
    db.check(got, *experts_exact(x, idx, w, gu, dn, g2l, res), what="three of 300")
    none = (g2l.long()[idx.long()] < 0).all(dim=1)
    assert torch.equal(got[none], res[none])


@pytest.mark.parametrize("T", [24, 1, 300])
def test_one_held_expert_of_many_takes_four_launches(T):
    """Fewer rows expected than one: no pass over the rows of x before the products."""
    x, idx, w, gu, dn = expert_case(13, T, 10, 1, 256, 64, torch.float16, routed=512)
    g2l = torch.full((512,), -1, dtype=torch.int32, device=DEV)
    g2l[idx[0, 0]] = 0
    lib = capi.lib()
    before = lib.bm_launch_count()
    got = dense_experts(x, idx, w, gu, dn, global_to_local=g2l)
    launches = lib.bm_launch_count() - before
    db.check(got, *experts_exact(x, idx, w, gu, dn, g2l), what="one of 512")
    assert launches == 4


def test_chain_from_logits_as_a_block_runs_it():
    """Router tail, routing build, grouped products with the routed lists, and the whole as one call: the same numbers."""
    gen = torch.Generator().manual_seed(8)
    T, E, k, H, I = 130, 24, 4, 256, 96
    x, gu, dn = rnd(gen, T, H, dtype=torch.float16), rnd(gen, E, 2 * I, H, std=0.05, dtype=torch.float16), rnd(gen, E, H, I, std=0.05, dtype=torch.float16)
    idx, w = route_topk(rnd(gen, T, E), k, True, torch.float16)
    tok, off, rw, _, _ = route_build(idx, w, E)
    h = grouped_linear(x, gu, off, tok)
    z = (torch.nn.functional.silu(h[:, :I].float()) * h[:, I:].float()).half()
    d = grouped_linear(z, dn, off)
    y = torch.zeros(T, H, device=DEV).index_add_(0, tok.long(), d.float() * rw[:, None])
    value, err = experts_exact(x, idx, w, gu, dn)
    db.check(dense_experts(x, idx, w, gu, dn), value, err, what="one call")
    assert float((y.double() - value).norm() / value.norm()) < 4 * db.half_step(torch.float16) * 2      # four 16-bit roundings on the way


def test_long_lists_pass_32_bits():
    """rows * N passes 2^31 elements: the last rows are as right as the first."""
    rows, K, N = 33000, 64, 66000
    gen = torch.Generator().manual_seed(9)
    x = rnd(gen, rows, K, dtype=torch.float16)
    w = rnd(gen, 2, N, K, std=0.1, dtype=torch.float16)
    got = grouped_linear(x, w, offsets([rows - 100, 100]))
    for r, e in ((slice(0, 4), 0), (slice(rows - 104, rows - 100), 0), (slice(rows - 100, rows), 1)):
        value, err = db.linear(x[r], w[e])
        db.check(got[r], value, db.rounded(value, err, torch.float16), what="long lists")


def test_strided_and_unaligned_inputs():
    gen = torch.Generator().manual_seed(10)
    wide = rnd(gen, 30, 200, dtype=torch.float16)
    x, w = wide[:, 7:135], rnd(gen, 2, 128, 40, std=0.1, dtype=torch.float16).transpose(1, 2)
    db.check(grouped_linear(x, w, offsets([13, 17])), *grouped_exact(x, w, [13, 17]), what="strided")
    flat = rnd(gen, 30 * 128 + 3, dtype=torch.float16)
    x = flat[3:].view(30, 128)                 # contiguous, off a 16-byte boundary
    db.check(grouped_linear(x, w, offsets([13, 17])), *grouped_exact(x, w, [13, 17]), what="unaligned x")
    out = torch.zeros(30 * 40 + 1, dtype=torch.float16, device=DEV)[1:].view(30, 40)
    db.check(grouped_linear(x, w, offsets([13, 17]), out=out), *grouped_exact(x, w, [13, 17]), what="unaligned out")


def test_another_stream_and_graph_replay():
    gen = torch.Generator().manual_seed(11)
    x, idx, w, gu, dn = expert_case(11, 40, 4, 8, 256, 128, torch.bfloat16)
    want = dense_experts(x, idx, w, gu, dn, residual=x)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = dense_experts(x, idx, w, gu, dn, residual=x)
    side.synchronize()
    assert torch.equal(other, want)
    static_x, static_idx, static_w = torch.zeros_like(x), torch.zeros_like(idx), torch.zeros_like(w)
    static_idx.copy_(idx)
    graphs, outs = [], []
    for _ in range(2):                        # two captured calls of one shape: neither may use the other's scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(dense_experts(static_x, static_idx, static_w, gu, dn, residual=static_x))
        graphs.append(g)
    for scale in (1.0, 0.5):
        static_x.copy_(x * scale)
        static_idx.copy_(idx.flip(0) if scale == 0.5 else idx)
        static_w.copy_(w)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        again = dense_experts(static_x, static_idx, static_w, gu, dn, residual=static_x)
        assert all(torch.equal(o, again) for o in outs)
    assert torch.equal(dense_experts(x, idx, w, gu, dn, residual=x), want)


def test_refusals():
    h = lambda *s, dtype=torch.float16, device=DEV: torch.zeros(*s, dtype=dtype, device=device)
    i32 = lambda *s: h(*s, dtype=torch.int32)
    x, w, off = h(6, 64), h(3, 32, 64), i32(4)
    wrong = [lambda: grouped_linear(x.float(), w.float(), off), lambda: grouped_linear(x, w.bfloat16(), off), lambda: grouped_linear(x.cpu(), w, off),
             lambda: grouped_linear(x, w.cpu(), off), lambda: grouped_linear(x, w[0], off), lambda: grouped_linear(x, h(3, 32, 72), off),
             lambda: grouped_linear(x, w, off[:-1]), lambda: grouped_linear(x, w, off.long()), lambda: grouped_linear(x, w, off.cpu()),
             lambda: grouped_linear(x, w, off, i32(6).long()), lambda: grouped_linear(x, w, off, i32(6).cpu()), lambda: grouped_linear(x, w, off, i32(12)[::2]),
             lambda: grouped_linear(x, w, off, out=h(5, 32)), lambda: grouped_linear(x, w, off, out=h(6, 32).bfloat16()),
             lambda: grouped_linear(x, w, off, out=h(32, 6).t()), lambda: grouped_linear(x.clone().requires_grad_(), w, off),
             lambda: grouped_linear(x, w.clone().requires_grad_(), off), lambda: grouped_linear(x.reshape(2, 3, 64), w, off)]
    buf = h(6 * 64 + 8)
    wrong.append(lambda: grouped_linear(buf[:384].view(6, 64), h(1, 64, 64), i32(2), out=buf[8:392].view(6, 64)))       # in place
    idx, tw, gu, dn = i32(6, 2), h(6, 2, dtype=torch.float32), h(3, 64, 64), h(3, 64, 32)
    good = dict(x=x, topk_idx=idx, topk_w=tw, w_gate_up=gu, w_down=dn)
    bad = [dict(x=x.float()), dict(x=h(5, 64)), dict(topk_idx=idx.float()), dict(topk_idx=idx.cpu()), dict(topk_w=h(6, 3)), dict(topk_w=idx),
           dict(w_gate_up=h(3, 63, 64)), dict(w_gate_up=h(2, 64, 64)), dict(w_down=h(3, 64, 31)), dict(w_down=h(3, 72, 32)), dict(w_down=dn.bfloat16()),
           dict(w_gate_up=gu.cpu()), dict(global_to_local=i32(6).long()), dict(global_to_local=i32(6).cpu()), dict(residual=h(5, 64)),
           dict(residual=h(6, 64, device="cpu")), dict(topk_idx=i32(6, 33), topk_w=h(6, 33, dtype=torch.float32)), dict(x=x.clone().requires_grad_())]
    wrong += [lambda b=b: dense_experts(**{**good, **b}) for b in bad]
    for i, call in enumerate(wrong):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert dense_experts(**good).shape == (6, 64)
    with torch.no_grad():
        assert grouped_linear(x, w.clone().requires_grad_(), off).shape == (6, 32)


def test_c_entry_refusals():
    lib = capi.lib()
    x = torch.zeros(8, 64, dtype=torch.float16, device=DEV)
    p = x.data_ptr()
    st = capi.stream_ptr(torch.device(DEV))
    off = torch.zeros(4, dtype=torch.int32, device=DEV).data_ptr()
    assert lib.bm_grouped_linear(p, 0, p, 8, 0, 4, 1, off, None, 8, p, None, 0, st) == 1
    assert lib.bm_grouped_linear(p, 2, p, 8, 64, 4, 1, off, None, 8, p, None, 0, st) == 1
    assert lib.bm_grouped_linear(p, 0, None, 8, 64, 4, 1, off, None, 8, p, None, 0, st) == 1
    assert lib.bm_grouped_linear(p, 0, p, 4, 64, 4, 1, off, None, 8, p, None, 0, st) == 1
    assert lib.bm_grouped_linear_workspace_bytes(64, 1, 0) == 0 and lib.bm_grouped_linear_workspace_bytes(64, 2, 5000) >= 5000 * 128
    assert lib.bm_grouped_linear(p, 0, p, 8, 64, 4, 2, off, off, 5000, p, p, 4999 * 128, st) == 4
    need = lib.bm_dense_experts_workspace_bytes(8, 2, 1, 64, 32)
    assert need > 0 and lib.bm_dense_experts_workspace_bytes(0, 2, 1, 64, 32) == 0
    assert lib.bm_dense_experts_forward(p, 0, off, off, None, 1, 8, 2, 1, p, p, 64, 32, None, p, p, need - 1, st) == 4
    assert lib.bm_dense_experts_forward(p, 0, off, off, None, 2, 8, 2, 1, p, p, 64, 32, None, p, p, need, st) != 0      # two routed, one held, no map
