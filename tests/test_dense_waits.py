"""GPU: the dense products' kernels leave cleanly when a wait gives up, and say so."""
import contextlib

import pytest
import torch

from bitsmoe_b200 import capi
from bitsmoe_b200.layer import check_dense_status, dense_experts, dense_mlp4, grouped_linear, linear4
from tests.test_gpu_grouped import expert_case, offsets, rnd
from tests.test_linear4 import matrix4, mlp_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def grouped(K, N, sizes, gather):
    gen = torch.Generator().manual_seed(1)
    rows = sum(sizes)
    x, w, off = rnd(gen, 50 if gather else rows, K, dtype=torch.bfloat16), rnd(gen, len(sizes), N, K, std=0.05, dtype=torch.bfloat16), offsets(sizes)
    index = torch.randint(0, 50, (rows,), generator=gen).to(torch.int32).to(DEV) if gather else None
    return lambda: grouped_linear(x, w, off, index)


def experts(T, k, E, H, I):
    case = expert_case(2, T, k, E, H, I, torch.float16)
    return lambda: dense_experts(*case)


def product4(tokens, n, k, group):
    gen = torch.Generator().manual_seed(3)
    m, _ = matrix4(gen, n, k, group)
    x = rnd(gen, tokens, k, dtype=torch.bfloat16)
    return lambda: linear4(x, *m, group)


def mlp4(tokens, hidden, inter, gated):
    x, packs, _, tg, res = mlp_case(4, tokens, hidden, inter, 128, torch.float16)
    return lambda: dense_mlp4(x, *packs, 128, token_gate_weight=tg if gated else None, residual=res)


CALLS = {
    "short groups in order": lambda: grouped(2048, 512, [1, 0, 3, 9], False), "short groups by index": lambda: grouped(2048, 512, [1, 0, 3, 9], True),
    "long groups": lambda: grouped(768, 2048, [300, 900, 17, 256], False), "long groups by index": lambda: grouped(768, 2048, [300, 900, 17, 40], True),
    "few columns": lambda: grouped(64, 24, [5, 6], False), "experts, one token": lambda: experts(1, 4, 8, 512, 128),
    "experts, long": lambda: experts(900, 4, 8, 512, 128), "4 bits, columns shared by four": lambda: product4(64, 4100, 4096, 128),
    "4 bits, columns shared by two": lambda: product4(131, 8200, 2048, 32), "4 bits, many tiles": lambda: product4(600, 20001, 1104, 64),
    "MLP in 4 bits": lambda: mlp4(300, 2048, 512, True), "MLP in 4 bits, wide": lambda: mlp4(150, 4096, 2050, False),
}


@contextlib.contextmanager
def wait_limit(us):
    capi.check(capi.lib().bm_dense_set_wait_limit(us))
    try:
        yield
    finally:
        capi.check(capi.lib().bm_dense_set_wait_limit(2000000))


@pytest.mark.parametrize("name", CALLS)
def test_kernels_leave_cleanly_when_a_wait_gives_up(name):
    """With the limit at 0 the roles of every CTA leave at their first wait that is not over, with copies and products under way: the launch
    ends, the time-out is reported once, and the next launches compute what they should."""
    call = CALLS[name]()
    want = call()
    check_dense_status()
    for _ in range(5):
        with wait_limit(0):
            call()
        with pytest.raises(capi.BitsMoEError, match="bounded wait"):
            check_dense_status(DEV)
        check_dense_status()                      # the report has cleared it
        assert torch.equal(call(), want)
        check_dense_status()


@pytest.mark.parametrize("tokens", [5, 600])
def test_products_without_waits_report_nothing(tokens):
    """Rows of 1100 16-bit elements do not start on 16-byte boundaries: the streaming kernel takes them, which waits for nobody."""
    call = product4(tokens, 20001, 1100, 64)
    want = call()
    with wait_limit(0):
        assert torch.equal(call(), want)
    check_dense_status()


def test_limits_that_are_refused():
    lib = capi.lib()
    for us in (-1, 2000001):
        assert lib.bm_dense_set_wait_limit(us) == 1
    assert lib.bm_dense_set_wait_limit(2000000) == 0
