"""The 8-bit path in the debug build, whose kernels check their indexes, over the forms that each kernel has; results as in the
product build's tests."""
import numpy as np
import pytest

from backpack_b200 import Q4KContext
from test_gpu_i8 import TYPES, check_product, check_rows, dtype_of, make_product, place, rows_reference
from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def debug():
    c = Q4KContext(0, debug=True)
    yield c
    c.close()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,V,k", [(1, 128256, 0), (1, 128256, 20), (1, 128256, 32), (3, 128256, 5), (40, 32003, 8), (160, 32 * 1024, 32), (160, 32 * 1024 - 1, 32),
                                   (300, 40001, 20), (300, 5000, 32), (700, 1031, 1), (1, 8 * 255 * 1024, 32), (1, 8 * 255 * 1024 + 3, 32), (2, 8 * 256 * 1024 + 9, 5)])
def test_log_probabilities(debug, kind, M, V, k):
    """One CTA a row and clusters; blocks of a step, of lines, of several steps; lines kept beside the blocks' largest values."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(M + V + k)
    x = (torch.randn(M, V, device="cuda", generator=g) * 3).to(dtype_of(kind))
    check(debug, x, torch.randint(0, V, (M, 2), device="cuda", generator=g, dtype=torch.int32), k)   # (and the device status)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,K,pad,offset", [(3, 700, 0, 0), (2, 9000, 0, 0), (2, 9001, 2, 1), (300, 1500, 0, 0), (2, 20001, 0, 0), (2, 20000, 0, 0), (2, 32768, 0, 0), (2, 32767, 0, 3)])
def test_rows(debug, kind, M, K, pad, offset):
    """8, 16 and 32 values a thread; single accesses and whole ones; with a norm, with a residual too, and without either."""
    import torch

    rng = np.random.default_rng(K)
    t = dtype_of(kind)
    x, r = (torch.from_numpy((rng.standard_normal((M, K)) * 3).astype(np.float32)).to(t) for _ in range(2))
    w = rng.uniform(-0.5, 2.0, K).astype(np.float32)
    xd, rd = place(x, kind, pad, offset)[1], place(r, kind, pad, offset)[1]
    eps = float(np.float32(1e-5))
    got, total = debug.add_rmsnorm_i8(xd, torch.from_numpy(w).cuda(), 1e-5, residual=rd)
    codes, scales, v = rows_reference(x.float().numpy(), r.float().numpy(), w, eps)
    check_rows(got, codes, scales, K)
    assert torch.equal(total.cpu(), torch.from_numpy(v).to(t))
    check_rows(debug.add_rmsnorm_i8(xd, torch.from_numpy(w).cuda(), 1e-5)[0], *rows_reference(x.float().numpy(), None, w, eps)[:2], K)
    check_rows(debug.quantize_i8(xd), *rows_reference(x.float().numpy(), None, None, 0.0)[:2], K)
    assert debug.device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,N,K", [(3, 1000, 4097), (20, 40000, 1024), (16, 300, 8192), (48, 520, 4096), (100, 500, 9000), (128, 1000, 16384), (180, 1030, 8200),
                                   (400, 20000, 512), (777, 555, 333)])
def test_products(debug, kind, M, N, K):
    """Few rows; a CTA with several tiles; shared tiles that exchange beside the ring and in it; pairs with one tile and with several."""
    host, (xr, wr, bias) = make_product(M, N, K, M + N + K, True)
    check_product(debug.matmul_i8(xr, wr, bias=bias, dtype=dtype_of(kind)), *host, kind)
    assert debug.device_status() == 0


def test_long_rows_in_one_cta(ctx, debug):
    """Where rows are many, or clusters are refused, a CTA takes a row of any length by itself: the same tokens as by several CTAs,
    and the same numbers to what both may be off by."""
    import torch

    M, V = 300, 600011
    x = torch.randn(M, V, device="cuda", dtype=torch.bfloat16) * 3
    given = torch.randint(0, V, (M,), device="cuda", dtype=torch.int32)
    for c in (ctx, debug):
        many = c.logprobs(x, given=given, top=32)
        for r in (0, 7, M - 1):
            one = c.logprobs(x[r:r + 1], given=given[r:r + 1], top=32)
            assert torch.equal(many.top_ids[r], one.top_ids[0])
            # S of either is off by (V / 512 + 80) half steps, the results' own roundings come on top
            bound = 2 * ((V / 512 + 80) * 2.0 ** -24 + 4 * 2.0 ** -24 * 30)
            assert float((many.top[r] - one.top[0]).abs().max()) <= bound and float((many.given[r] - one.given[0]).abs()) <= bound
            assert float((many.entropy[r] - one.entropy[0]).abs()) <= 3 * bound * 15
        assert c.device_status() == 0
