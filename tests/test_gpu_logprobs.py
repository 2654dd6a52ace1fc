"""Log probabilities, entropy and most likely tokens (bpq4k_logprobs) against their definition in 64 bits.

Bounds: of n sums a thread adds at most n / 512 + 64 floats one after the other, so S is off by (n / 512 + 64) * 2^-24 and an
exponential by a few steps (two of its own, |x - m| 2^-24 from the argument, which its weight e^(x-m) makes less than one); ln S, x - m
and their difference round once each."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["f32", "f16", "bf16"]
LOWEST = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}


def dtype_of(kind):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def reference(x, given, k):
    """x: [M, V] in 64 bits."""
    M, V = x.shape
    lp = np.full((M, V), -np.inf)
    ent = np.zeros(M)
    for i in range(M):
        live = x[i] > -np.inf
        if live.any():
            m = x[i][live].max()
            e = np.exp(x[i][live] - m)
            s = e.sum()
            lp[i][live] = x[i][live] - m - np.log(s)
            ent[i] = np.log(s) - (e * np.maximum(x[i][live] - m, -1e300)).sum() / s
    ids = np.stack([np.lexsort((np.arange(V), -x[i]))[:k] for i in range(M)]) if k else np.zeros((M, 0), int)
    return (np.take_along_axis(lp, given, 1) if given is not None else None), ent, ids, np.take_along_axis(lp, ids, 1)


def close(got, want, V):
    got = got.cpu().numpy().astype(np.float64)
    want = np.where(want < -3.4028235677973366e38, -np.inf, want)   # (2^128 - 2^103: what a float rounds to -infinity)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine])
    bound = (V / 512 + 80) * U + 4 * U * np.abs(want[fine])
    assert (np.abs(got[fine] - want[fine]) <= bound).all(), float((np.abs(got[fine] - want[fine]) - bound).max())


def check(ctx, x, given, k):
    """x, given on the device."""
    import torch

    got = ctx.logprobs(x, given=given, top=k)
    V = x.shape[1]
    host = x.double().cpu().numpy()
    g2 = None if given is None else given.cpu().numpy().astype(np.int64).reshape(x.shape[0], -1)
    lp, ent, ids, top = reference(host, g2, k)
    if given is not None:
        assert got.given.shape == given.shape
        close(got.given.reshape(x.shape[0], -1), lp, V)
    else:
        assert got.given is None
    # entropy = ln S - T / S: both terms positive, T of 2 (n / 512 + 80) roundings
    np.testing.assert_allclose(got.entropy.cpu().numpy(), ent, rtol=3 * (V / 512 + 80) * U, atol=3 * (V / 512 + 80) * U)
    if k:
        assert np.array_equal(got.top_ids.cpu().numpy(), ids)
        close(got.top, top, V)
    else:
        assert got.top_ids is None and got.top is None
    assert ctx.device_status() == 0
    return got


SHAPES = [(1, 1), (1, 2), (2, 5), (3, 31), (2, 33), (1, 511), (4, 513), (2, 1000), (1, 4099), (5, 8192), (7, 20011), (1, 32003), (3, 32000), (1, 128256),
          (2, 131072), (40, 3001), (600, 32767), (160, 32768), (3, 262144 + 5), (2, 1100003), (300, 1031), (1000, 70)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,V", SHAPES)
@pytest.mark.parametrize("k", [0, 1, 5, 20, 32])
def test_logprobs_match_the_definition(ctx, kind, M, V, k):
    import torch

    g = torch.Generator(device="cuda").manual_seed(M * 131 + V + k)
    x = (torch.randn(M, V, device="cuda", generator=g) * 3).to(dtype_of(kind))   # (16-bit logits: many equal values)
    given = torch.randint(0, V, (M, 3), device="cuda", generator=g, dtype=torch.int32)
    check(ctx, x, given, min(k, V))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V,ld,offset", [(1000, 1001, 1), (1003, 1024, 3), (65, 67, 5), (7, 9, 2), (20001, 20007, 7)])
def test_rows_at_odd_addresses(ctx, kind, V, ld, offset):
    """Rows of a wider matrix, beginning anywhere, with NaNs between them."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(V)
    M = 9
    buf = torch.full((M * ld + offset,), float("nan"), dtype=dtype_of(kind), device="cuda")
    x = buf[offset:].view(M, ld)[:, :V]
    x.copy_(torch.randn(M, V, device="cuda", generator=g) * 2)
    check(ctx, x, torch.randint(0, V, (M,), device="cuda", generator=g, dtype=torch.int32), min(V, 16))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "two values", "steps"])
@pytest.mark.parametrize("V", [40, 4099, 50000])
def test_orders_and_ties(ctx, kind, order, V):
    import torch

    i = torch.arange(V, device="cuda")
    x = {"equal": i * 0.0 + 1.5, "ascending": i / 4096.0, "descending": -i / 4096.0, "two values": (i * 7 % 13 == 5) * 1.0,
         "steps": (i // 16) % 7 * 0.5}[order].float()[None].repeat(3, 1)
    x[1] = x[1].flip(0)
    x[2] = -x[2]                                    # zeros of both signs among them
    check(ctx, x.to(dtype_of(kind)).contiguous(), None, 32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [8 * 255 * 1024 - 5, 8 * 255 * 1024, 8 * 255 * 1024 + 3, 8 * 256 * 1024 + 9])
@pytest.mark.parametrize("equal", [False, True])
def test_long_rows_and_many_alternatives(ctx, kind, V, equal):
    """Eight CTAs share a row, around the most blocks of 1024 values that each has a thread for."""
    import torch

    x = torch.zeros(1, V, device="cuda") if equal else torch.randn(1, V, device="cuda")
    x[0, V // 3] = 7.5
    check(ctx, x.to(dtype_of(kind)), None, 32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("fill", ["-inf", "lowest"])
@pytest.mark.parametrize("V", [50, 4099, 32003])
def test_masked_rows(ctx, kind, fill, V):
    """Masks of -infinity and of the type's lowest value that leave all, few, one or no tokens."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(6, V, device="cuda", generator=g) * 3).to(dtype_of(kind))
    low = float("-inf") if fill == "-inf" else LOWEST[kind]
    for r, live in enumerate([V, V // 2, 7, 1, 0, 0]):
        keep = torch.randperm(V, device="cuda", generator=g)[:live]
        row = torch.full((V,), low, dtype=x.dtype, device="cuda")
        row[keep] = x[r][keep]
        x[r] = row
    x[5, V - 1] = LOWEST[kind]                       # the lowest value and nothing else
    given = torch.randint(0, V, (6, 8), device="cuda", generator=g, dtype=torch.int32)
    got = check(ctx, x, given, 20)
    if fill == "-inf":
        assert got.entropy[4] == 0 and bool((got.top[4] == -float("inf")).all()) and got.top_ids[4].tolist() == list(range(20))
        assert got.entropy[5] == 0 and got.top[5, 0] == 0 and got.top_ids[5, 0] == V - 1
    else:
        assert abs(float(got.entropy[4]) - np.log(V)) < 1e-4


@pytest.mark.parametrize("shift", [-3e38, -1e30, -1e4, 0.0, 1e4, 1e30, 3e38])
def test_logits_of_any_magnitude(ctx, shift):
    import torch

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 3000, device="cuda", generator=g) * 3 + shift
    x[1, 5] = -3.4e38
    x[2, 7] = 3.4e38
    check(ctx, x, torch.randint(0, 3000, (3, 2), device="cuda", generator=g, dtype=torch.int32), 8)


def test_rows_without_a_distribution(ctx):
    import torch

    for V in (9, 3000, 40001):
        x = torch.randn(5, V, device="cuda")
        x[1, V - 1] = float("nan")
        x[2, 0] = float("inf")
        x[3] = float("nan")
        given = torch.zeros(5, 2, dtype=torch.int32, device="cuda")
        got = ctx.logprobs(x, given=given, top=3)
        for r in (1, 2, 3):
            assert torch.isnan(got.given[r]).all() and torch.isnan(got.entropy[r]) and torch.isnan(got.top[r]).all() and (got.top_ids[r] == -1).all()
        # the other rows are as they are by themselves.  Which values a thread adds up follows from the row's place between
        # 16-byte boundaries (row 1 of two begins elsewhere than row 4 of five), so each result is within its own bound of the
        # exact value, and the two within twice that of each other
        rest = ctx.logprobs(x[::4].contiguous(), given=given[::4].contiguous(), top=3)
        assert torch.equal(got.top_ids[::4], rest.top_ids)
        for a, b, n in ((got.given, rest.given, 1), (got.entropy, rest.entropy, 3), (got.top, rest.top, 1)):
            bound = n * (V / 512 + 80) * U
            assert bool(((a[::4] - b).abs() <= 2 * (bound + (bound if n == 3 else 4 * U) * b.abs())).all())


def test_given_tokens_outside_the_row(ctx):
    import torch

    x = torch.randn(2, 100, device="cuda")
    got = ctx.logprobs(x, given=torch.tensor([[-1, 0, 99, 100], [2 ** 31 - 1, 5, 5, -2 ** 31]], dtype=torch.int32, device="cuda")).given
    assert torch.isnan(got).tolist() == [[True, False, False, True], [True, False, False, True]]
    assert got[1, 1] == got[1, 2]


def test_peaked_rows_keep_their_entropy(ctx):
    import torch

    x = torch.zeros(4, 5000, device="cuda")
    for r, top in enumerate((5.0, 15.0, 30.0, 200.0)):
        x[r, 1234] = top
    got = ctx.logprobs(x, given=torch.full((4,), 1234, dtype=torch.int32, device="cuda"), top=2)
    _, ent, _, _ = reference(x.double().cpu().numpy(), None, 0)
    # S = 1 + 4999 e^-top: the sums of a thread hold 4999 e^-top apart from the 1 only to half a step of it
    assert np.abs(got.entropy.cpu().numpy() - ent).max() <= 3 * (5000 / 512 + 80) * U
    assert got.top_ids[:, 0].tolist() == [1234] * 4 and got.top_ids[:, 1].tolist() == [0] * 4


def test_outputs_stay_inside_their_buffers(ctx):
    import torch

    M, V, G, k = 5, 999, 3, 7
    x = torch.randn(M, V, device="cuda")
    given = torch.randint(0, V, (M, G), dtype=torch.int32, device="cuda")
    lp, ent, top = (torch.full((n + 8,), -7777.0, device="cuda") for n in (M * G, M, M * k))
    ids = torch.full((M * k + 8,), -7777, dtype=torch.int32, device="cuda")
    st = ctx.lib.bpq4k_logprobs(ctx.h, 0, x.data_ptr(), M, V, V, given.data_ptr(), G, lp[4:].data_ptr(), ent[4:].data_ptr(), k, ids[4:].data_ptr(),
                                top[4:].data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert st == 0
    want = ctx.logprobs(x, given=given, top=k)
    for buf, w in ((lp, want.given), (ent, want.entropy), (ids, want.top_ids), (top, want.top)):
        assert torch.equal(buf[4:-4], w.reshape(-1)) and bool((buf[:4] == -7777).all()) and bool((buf[-4:] == -7777).all())
    # parts that are not asked for are not written
    ent.fill_(-7777.0)
    assert ctx.lib.bpq4k_logprobs(ctx.h, 0, x.data_ptr(), M, V, V, None, 0, None, ent[4:].data_ptr(), 0, None, None, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.allclose(ent[4:-4], want.entropy, rtol=1e-6)
    assert ctx.lib.bpq4k_logprobs(ctx.h, 0, x.data_ptr(), M, V, V, given.data_ptr(), G, lp[4:].data_ptr(), None, 0, None, None, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()


def test_many_given_tokens(ctx):
    import torch

    x = torch.randn(3, 5001, device="cuda")
    given = torch.randint(0, 5001, (3, 1000), dtype=torch.int32, device="cuda")
    check(ctx, x, given, 0)
    empty = ctx.logprobs(x, given=given[:, :0].contiguous(), top=1)
    assert tuple(empty.given.shape) == (3, 0)


def test_best_token_is_the_argmax(ctx):
    import torch

    x = torch.randn(4, 128256, device="cuda")
    ids = ctx.logprobs(x, top=1).top_ids
    for r in range(4):
        assert int(ids[r, 0]) == int(ctx.argmax(x[r].contiguous())[0])


def test_refusals(ctx):
    import torch

    x, given = torch.randn(2, 50, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    f, i = torch.empty(64, device="cuda"), torch.empty(64, dtype=torch.int32, device="cuda")

    def call(ft=0, x=x.data_ptr(), M=2, V=50, ld=50, g=given.data_ptr(), G=1, lp=f.data_ptr(), e=f[8:].data_ptr(), k=3, ids=i.data_ptr(), top=f[16:].data_ptr()):
        return ctx.lib.bpq4k_logprobs(ctx.h, ft, x, M, V, ld, g, G, lp, e, k, ids, top, 0)

    assert call() == 0 and call(M=0, x=None) == 0
    assert call(ft=3) == 2 and call(V=0) == 2 and call(V=1 << 31, ld=(1 << 32) - 1) == 2 and call(M=1 << 31) == 2
    assert call(k=33) == 2 and call(k=32) == 0 and call(V=2, k=3) == 2
    assert call(x=None) == 1 and call(ld=49) == 1 and call(g=None) == 1 and call(lp=None) == 1 and call(ids=None) == 1 and call(top=None) == 1
    assert call(g=None, lp=None, G=0, e=None, k=0, ids=None, top=None) == 1
    assert call(x=x.data_ptr() + 2) == 3 and call(ft=1, x=x.data_ptr() + 1) == 3 and call(ids=i.data_ptr() + 2) == 3 and call(e=f.data_ptr() + 1) == 3
    for bad in (lambda: ctx.logprobs(x, top=33), lambda: ctx.logprobs(x, top=-1), lambda: ctx.logprobs(x.double()), lambda: ctx.logprobs(x, given=given.long()),
                lambda: ctx.logprobs(x, given=given[:1]), lambda: ctx.logprobs(x.t()), lambda: ctx.logprobs(x.cpu())):
        with pytest.raises(ValueError):
            bad()
    torch.cuda.synchronize()
    assert ctx.device_status() == 0
