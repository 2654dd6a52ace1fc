"""Codes of products v * w that lie next to the middle between two codes, against whole numbers: v and w are whole mantissas of 24
bits, so a product has 48, and 254 |p| and (2k + 1) a, whose order decides, have up to 56, more than a double holds."""
import numpy as np
import pytest

# (v, w of the largest product, v, w beside it): 254 p and the nearest (2k + 1) a round to the same double and differ by 1 to 4
NEAR = [(14374551, 15341497, 8794469, 11353154), (15809411, 15930841, 12492902, 9921272), (11266187, 9016469, 4819963, 7384584),
        (11115507, 10714261, 6065789, 7807138), (13595645, 10876507, 13386201, 8741667), (16535716, 12242964, 9080669, 16764530),
        (12372689, 13931109, 8702256, 16765738), (12856587, 16222039, 9059099, 16768111), (13663921, 12763343, 5529028, 16764517),
        (14981597, 12695915, 6478636, 16759954), (9095098, 16491983, 6723015, 16777059), (13454083, 14778227, 9103842, 16766894),
        (14175818, 15815528, 5742033, 16755559), (12496675, 15070087, 11006493, 16773624), (14044451, 13371111, 9739883, 16775562),
        (10056281, 16472795, 9525616, 16774284), (12113213, 14303275, 10288869, 16773126), (16464876, 16772857, 12118880, 16776869)]


def whole_number_codes(v, w):
    """round_half_even(127 v w / max |v w|) of whole v, w."""
    p = [int(a) * int(b) for a, b in zip(v, w)]
    peak = max(abs(q) for q in p)
    codes = []
    for q in p:
        k, rest = divmod(127 * abs(q), peak)
        k += 2 * rest > peak or (2 * rest == peak and k % 2 == 1)
        codes.append(k if q >= 0 else -k)
    return np.array(codes)


def test_the_doubles_of_both_sides_are_equal():
    """What makes these products the hard ones."""
    for V, W, v, w in NEAR:
        a, p = V * W, v * w
        k = 127 * p // a
        assert 0 < abs(254 * p - (2 * k + 1) * a) <= 4 and float(254 * p) == float((2 * k + 1) * a)


@pytest.mark.gpu
@pytest.mark.parametrize("K,offset", [(2, 0), (4, 0), (64, 0), (1000, 1), (4096, 0), (9000, 0), (20000, 0), (20001, 3)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -90, 2.0 ** 30])
@pytest.mark.parametrize("residual", [False, True])
def test_codes_of_products_next_to_a_border(ctx, K, offset, scale, residual):
    """One row per pair, anywhere in it and of either sign, among products that are smaller."""
    import torch

    rng = np.random.default_rng(K)
    for i, (V, W, v, w) in enumerate(NEAR):
        vs, ws = rng.integers(1, 1 << 22, K), rng.integers(1, 1 << 22, K)
        at = rng.choice(K, 2, replace=False)
        vs[at], ws[at] = (V, v), (W, w)
        vs = vs * rng.choice([-1, 1], K)
        x = torch.from_numpy((vs * scale).astype(np.float32))
        buf = torch.zeros(K + offset, device="cuda")
        buf[offset:] = x
        r = torch.zeros(1, K, device="cuda") if residual else None
        got, _ = ctx.add_rmsnorm_i8(buf[offset:].view(1, K), torch.from_numpy((ws * scale).astype(np.float32)).cuda(), 0.0, residual=r)
        np.testing.assert_array_equal(got.codes[0].cpu().numpy(), whole_number_codes(vs, ws), err_msg=str(i))
    assert ctx.device_status() == 0
