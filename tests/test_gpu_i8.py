"""The 8-bit path (bpq4k_add_rmsnorm_i8, bpq4k_quantize_i8, bpq4k_matmul_i8) against its definition in 64 bits.

Tolerances count roundings of half a step: 2^-24 of a float, 2^-11 of a half, 2^-8 of a bfloat16."""
import numpy as np
import pytest

from backpack_b200 import I8Rows, Q4KContext, Q4KError, pack_kq, synth
from oracle import q4k_oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TYPES = ["f32", "f16", "bf16"]
CANARY = -7777.0


def dtype_of(kind):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def place(host, kind, pad=0, offset=0, fill=float("nan")):
    """A device copy of a matrix whose rows are `pad` values further apart than they are long, `offset` values into a buffer
    that is otherwise full of `fill`; returns (buffer, matrix)."""
    import torch

    m, k = host.shape
    t = torch.as_tensor(host).to(dtype_of(kind))
    buf = torch.full((m * (k + pad) + offset + 64,), fill, dtype=t.dtype, device="cuda")
    view = buf[offset:offset + m * (k + pad)].view(m, k + pad)[:, :k]
    view.copy_(t)
    return buf, view


def codes_on_device(codes, fill=77):
    """Codes in rows that begin at multiples of 16 bytes, with `fill` between them."""
    import torch

    m, k = codes.shape
    buf = torch.full((m, (k + 15) // 16 * 16 + 16), fill, dtype=torch.int8, device="cuda")
    buf[:, :k] = torch.from_numpy(codes)
    return buf[:, :k]


def rows_reference(x, r, w, eps):
    """(codes, scales, sum) of host matrices in the element type's values, from the definition; the quotient in 64 bits."""
    v = x.astype(np.float32)
    if r is not None:
        v = v + r.astype(np.float32)
    p = v.astype(np.float64) * (w.astype(np.float64) if w is not None else 1.0)
    a = np.abs(p).max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        codes = np.rint(127.0 * p / np.where(a == 0, 1.0, a))
        rstd = 1.0 / np.sqrt((v.astype(np.float64) ** 2).mean(axis=1, keepdims=True) + eps) if w is not None else 1.0
        scales = np.where(a == 0, 0.0, a * rstd / 127.0)[:, 0]
    return codes, scales, v


def check_rows(got, codes, scales, k):
    assert np.array_equal(got.codes.cpu().numpy().astype(np.float64), codes)
    # the sum of squares: at most 32 additions in a thread, 5 + 5 over the block, each half a step of a float; half of that in
    # the root; the scale's own rounding; eps as a float
    np.testing.assert_allclose(got.scales.cpu().numpy().astype(np.float64), scales, rtol=((32 + 10) / 2 + 2) * U, atol=0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K,pad,offset", [(1, 4096, 0, 0), (3, 1, 0, 0), (2, 7, 1, 0), (5, 64, 0, 0), (4, 1000, 0, 0), (3, 1001, 0, 0), (2, 2048, 8, 0),
                                            (7, 768, 0, 1), (2, 8192, 0, 0), (2, 8200, 0, 0), (1, 28672, 0, 0), (3, 32768, 0, 0), (2, 32767, 0, 3),
                                            (150, 520, 0, 0), (700, 96, 3, 0), (200, 5120, 0, 0), (160, 16384, 0, 0)])
def test_norm_matches_the_definition(ctx, kind, residual, M, K, pad, offset):
    import torch

    rng = np.random.default_rng(M * 100003 + K)
    t = dtype_of(kind)
    wide = np.where(rng.random(K) < 0.02, 30.0, 1.0)
    x = torch.from_numpy((rng.standard_normal((M, K)) * wide).astype(np.float32)).to(t)
    r = torch.from_numpy((rng.standard_normal((M, K)) * 2).astype(np.float32)).to(t) if residual else None
    w = rng.uniform(-0.5, 2.0, K).astype(np.float32)
    _, xd = place(x, kind, pad, offset)
    rd = place(r, kind, pad, offset)[1] if residual else None
    got, total = ctx.add_rmsnorm_i8(xd, torch.from_numpy(w).cuda(), 1e-5, residual=rd)
    codes, scales, v = rows_reference(x.float().numpy(), r.float().numpy() if residual else None, w, float(np.float32(1e-5)))
    check_rows(got, codes, scales, K)
    if residual:
        assert total.dtype == t and torch.equal(total.cpu(), torch.from_numpy(v).to(t))
    else:
        assert total.data_ptr() == xd.data_ptr()
    assert ctx.device_status() == 0


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,K,pad,offset", [(1, 1, 0, 0), (1, 4096, 0, 0), (9, 333, 0, 0), (4, 14336, 0, 0), (2, 32768, 0, 0), (33, 100, 4, 5), (300, 2048, 0, 0)])
def test_quantize_matches_the_definition(ctx, kind, M, K, pad, offset):
    import torch

    rng = np.random.default_rng(K)
    x = torch.from_numpy((rng.standard_normal((M, K)) * 3).astype(np.float32)).to(dtype_of(kind))
    got = ctx.quantize_i8(place(x, kind, pad, offset)[1])
    codes, scales, _ = rows_reference(x.float().numpy(), None, None, 0.0)
    check_rows(got, codes, scales, K)


def test_codes_halfway_between_two_go_to_the_even_one(ctx):
    """Largest value 254: odd values lie exactly between two codes; their neighbours a step of a float away do not."""
    import torch

    odd = np.arange(-253, 254, 2, dtype=np.float32)
    x = np.stack([np.concatenate([[254.0], odd, np.nextafter(odd, np.float32(0)), np.nextafter(odd, np.float32(1000) * np.sign(odd))])]).astype(np.float32)
    got = ctx.quantize_i8(torch.from_numpy(x).cuda())
    codes, scales, _ = rows_reference(x, None, None, 0.0)
    check_rows(got, codes, scales, x.shape[1])
    ties = got.codes.cpu().numpy()[0, 1:1 + odd.size]
    assert (ties % 2 == 0).all()
    # the same through products that a float cannot hold: v * w with 24 bits each
    rng = np.random.default_rng(5)
    v = rng.uniform(1, 2, (4, 4096)).astype(np.float32)
    w = rng.uniform(0.5, 1, 4096).astype(np.float32)
    got, _ = ctx.add_rmsnorm_i8(torch.from_numpy(v).cuda(), torch.from_numpy(w).cuda(), 0.0)
    check_rows(got, *rows_reference(v, None, w, 0.0)[:2], 4096)


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-22, 1e-12, 1e12, 1e19, 1e30])
def test_norm_of_very_small_and_very_large_rows(ctx, scale):
    import torch

    rng = np.random.default_rng(3)
    x = (rng.uniform(0.5, 2, (5, 1536)) * rng.choice([-1, 1], (5, 1536)) * scale).astype(np.float32)
    w = rng.uniform(0.5, 2, 1536).astype(np.float32)
    got, _ = ctx.add_rmsnorm_i8(torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda(), 0.0)
    codes, scales, _ = rows_reference(x, None, w, 0.0)
    check_rows(got, codes, scales, 1536)


def test_rows_of_zeros_and_rows_without_a_finite_norm(ctx):
    import torch

    x = np.ones((6, 512), np.float32)
    x[0] = 0
    x[1, 17] = np.nan
    x[2, 500] = np.inf
    x[3, 3] = -np.inf
    x[4, ::2] = -0.0
    w = torch.ones(512, device="cuda")
    for eps in (0.0, 1e-5):
        got, _ = ctx.add_rmsnorm_i8(torch.from_numpy(x).cuda(), w, eps)
        s, c = got.scales.cpu().numpy(), got.codes.cpu().numpy()
        assert s[0] == 0 and not c[0].any()
        assert np.isnan(s[1:4]).all() and not c[1:4].any()
        assert np.isfinite(s[4:]).all() and (c[5] == 127).all()
    got = ctx.quantize_i8(torch.from_numpy(x).cuda())
    assert got.scales[0] == 0 and np.isnan(got.scales[1:4].cpu().numpy()).all()
    w[9] = float("nan")
    assert np.isnan(ctx.add_rmsnorm_i8(torch.from_numpy(x).cuda(), w, 1e-5)[0].scales.cpu().numpy()).all()
    # everything made of such a row is a NaN, everything made of a row of zeros is the bias
    y = ctx.matmul_i8(got, ctx.quantize_i8(torch.ones(40, 512, device="cuda")), bias=torch.full((40,), 3.0, device="cuda"))
    assert torch.isnan(y[1:4]).all() and torch.equal(y[0], torch.full((40,), 3.0, device="cuda")) and torch.isfinite(y[4:]).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", [1024, 999, 20000])
def test_sum_may_be_written_over_an_input(ctx, kind, K):
    import torch

    t = dtype_of(kind)
    x, r = torch.randn(6, K, device="cuda").to(t), torch.randn(6, K, device="cuda").to(t)
    w = torch.rand(K, device="cuda")
    want, total = ctx.add_rmsnorm_i8(x, w, 1e-6, residual=r)
    for place_in in ("residual", "x"):
        x2, r2 = x.clone(), r.clone()
        got, s = ctx.add_rmsnorm_i8(x2, w, 1e-6, residual=r2, sum_out=r2 if place_in == "residual" else x2)
        assert torch.equal(s, total) and torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        assert torch.equal(r2 if place_in == "x" else x2, r if place_in == "x" else x)
    got, s = ctx.add_rmsnorm_i8(x, w, 1e-6, residual=x)           # the same tensor twice
    assert torch.equal(s, (x.float() * 2).to(t))


def test_rows_stay_inside_their_buffers(ctx):
    import torch

    for kind in TYPES:
        for M, K in [(1, 1), (3, 17), (5, 1000), (4, 4096)]:
            t = dtype_of(kind)
            x, r = torch.randn(M, K).to(t), torch.randn(M, K).to(t)
            pad = (K + 15) // 16 * 16 + 16
            cbuf = torch.full((M + 2, pad), 55, dtype=torch.int8, device="cuda")
            sbuf = torch.full((M + 2,), CANARY, device="cuda")
            obuf, total = place(torch.zeros(M, K), kind, 8, 16, fill=3.0)
            out = I8Rows(cbuf[1:M + 1, :K], sbuf[1:M + 1])
            w = torch.rand(K) + 0.1
            ctx.add_rmsnorm_i8(place(x, kind, 8, 8)[1], place(w[None], "f32", 0, 4)[1][0], 1e-5, residual=place(r, kind, 16, 8)[1], sum_out=total, out=out)
            codes, scales, v = rows_reference(x.float().numpy(), r.float().numpy(), w.numpy(), float(np.float32(1e-5)))
            check_rows(out, codes, scales, K)
            assert torch.equal(total.cpu(), torch.from_numpy(v).to(t))
            cbuf[1:M + 1, :K] = 55
            total.fill_(3.0)
            assert bool((cbuf == 55).all()) and bool((obuf == 3.0).all()) and sbuf[0] == CANARY and sbuf[-1] == CANARY


# ---- the product ----------------------------------------------------------------------------------------------------------

def random_codes(rng, m, k):
    return np.clip(np.rint(rng.standard_normal((m, k)) * 40), -128, 127).astype(np.int8)


def product_reference(x, xs, w, ws, bias):
    """(Y, bound of a float result's error) in 64 bits.  The sum is exact; its conversion to a float and two products round
    once each, the bias' addition once more."""
    s = x.astype(np.float64) @ w.astype(np.float64).T
    prod = s * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    y = prod + (bias.astype(np.float64) if bias is not None else 0.0)
    return y, 3.01 * U * np.abs(prod) + (1.01 * U * np.abs(y) if bias is not None else 0.0)


def check_product(got, x, xs, w, ws, bias, kind):
    y, bound = product_reference(x, xs, w, ws, bias)
    got = got.float().cpu().numpy().astype(np.float64)
    if kind != "f32":
        bound = bound + HALF_STEP[kind] * (np.abs(y) + bound) + (2.0 ** -25 if kind == "f16" else 0.0)
    worst = np.max(np.abs(got - y) - bound)
    assert worst <= 0, worst


def make_product(M, N, K, seed, with_bias):
    import torch

    rng = np.random.default_rng(seed)
    x, w = random_codes(rng, M, K), random_codes(rng, N, K)
    xs, ws = rng.uniform(0.001, 0.02, M).astype(np.float32), rng.uniform(0.0005, 0.002, N).astype(np.float32)
    bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    xr, wr = I8Rows(codes_on_device(x), dev(xs)), I8Rows(codes_on_device(w, -99), dev(ws))
    return (x, xs, w, ws, bias), (xr, wr, dev(bias) if with_bias else None)


SHAPES = [(1, 1, 1), (1, 7, 15), (1, 1024, 4096), (1, 300, 127), (1, 129, 12289), (2, 128, 128), (3, 1000, 16), (4, 515, 2049), (5, 257, 4096),
          (8, 640, 1024), (9, 130, 8190), (16, 2048, 512), (17, 385, 640), (31, 96, 300), (32, 4096, 4096), (33, 250, 4096), (48, 1024, 1000),
          (64, 128, 4095), (65, 999, 129), (100, 300, 20000), (127, 77, 256), (128, 512, 512), (129, 2000, 768), (200, 1537, 1024),
          (255, 129, 1000), (256, 256, 4096), (130, 300, 4096), (180, 1030, 8200), (250, 4096, 2080), (400, 700, 9000), (257, 640, 384), (300, 4097, 513), (512, 1024, 2048), (777, 555, 333), (1030, 2305, 640)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("kind,with_bias", [("f32", True), ("f16", False), ("bf16", True)])
def test_matmul_matches_the_definition(ctx, M, N, K, kind, with_bias):
    host, (xr, wr, bias) = make_product(M, N, K, M * 7 + N * 3 + K, with_bias)
    got = ctx.matmul_i8(xr, wr, bias=bias, dtype=dtype_of(kind))
    assert got.dtype == dtype_of(kind)
    check_product(got, *host, kind)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("shares", range(1, 10))
@pytest.mark.parametrize("M", [9, 16, 30, 48, 50, 77, 112, 128])
def test_matmul_of_shared_tiles(ctx, M, shares):
    """Few tiles, whose K range CTAs share where each has four steps of 128 codes and more; the last step is a short one."""
    for N, K in ((200, shares * 512 - 20), (129 * (9 - min(shares, 8)), shares * 512 + 77)):
        host, (xr, wr, bias) = make_product(M, N, K, M * 11 + shares, True)
        check_product(ctx.matmul_i8(xr, wr, bias=bias), *host, "f32")
    assert ctx.device_status() == 0


@pytest.mark.parametrize("M", [1, 3, 20, 150, 400])
@pytest.mark.parametrize("K", [131071, 131056])
def test_matmul_of_the_largest_sums(ctx, M, K):
    """128 * 128 * 131071 is 16384 below 2^31."""
    import torch

    N = 130
    x, w = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    w[1::2] = 127
    ones = lambda n: np.ones(n, np.float32)  # noqa: E731
    got = ctx.matmul_i8(I8Rows(codes_on_device(x), torch.ones(M, device="cuda")), I8Rows(codes_on_device(w), torch.ones(N, device="cuda")))
    check_product(got, x, ones(M), w, ones(N), None, "f32")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("M,N,K,ldy", [(1, 100, 256, 131), (5, 257, 500, 300), (70, 130, 1024, 137), (140, 385, 640, 400), (300, 1000, 272, 1001)])
def test_matmul_stays_inside_its_buffers(ctx, M, N, K, ldy, kind):
    import torch

    host, (xr, wr, _) = make_product(M, N, K, N + K, False)
    t = dtype_of(kind)
    buf = torch.full((M + 2, ldy), CANARY, dtype=t, device="cuda")
    out = buf[1:M + 1, 3:N + 3] if ldy >= N + 3 else buf[1:M + 1, :N]
    ctx.matmul_i8(xr, wr, out=out)
    check_product(out, *host, kind)
    out.fill_(CANARY)
    assert bool((buf == torch.tensor(CANARY, dtype=t, device="cuda")).all())


def test_matmul_rows_and_views(ctx):
    """Row ranges of a weight, columns of wider codes, one activation row of many: the same values as the whole."""
    import torch

    host, (xr, wr, _) = make_product(37, 700, 1040, 11, False)
    whole = ctx.matmul_i8(xr, wr)
    assert torch.equal(ctx.matmul_i8(xr, wr.rows(129, 430)), whole[:, 129:430])
    assert torch.equal(ctx.matmul_i8(xr.rows(5, 6), wr), whole[5:6])
    part = ctx.matmul_i8(I8Rows(xr.codes[:, 16:1000], xr.scales), I8Rows(wr.codes[:, 16:1000], wr.scales))
    check_product(part, host[0][:, 16:1000], host[1], host[2][:, 16:1000], host[3], None, "f32")


def test_matmul_result_does_not_depend_on_the_batch(ctx):
    """Whichever kernel serves a number of rows: the sums are exact, so the bits are those of the row by itself."""
    import torch

    _, (xr, wr, bias) = make_product(600, 1300, 2000, 4, True)
    whole = ctx.matmul_i8(xr, wr, bias=bias)
    for m in (1, 2, 4, 5, 8, 16, 17, 40, 64, 65, 100, 128, 129, 200, 256, 257, 500):
        assert torch.equal(ctx.matmul_i8(xr.rows(0, m), wr, bias=bias), whole[:m]), m


@pytest.mark.parametrize("name,bits", [("bfloat16", 8), ("float16", 11)])
def test_every_16_bit_quotient(ctx, name, bits):
    """Each row has another mantissa n as its largest value, n * 2^-10, and all mantissas m, m * 2^-10-t for t = 0 .. 8, below it:
    codes round_half_even(127 m / (n 2^t)) in whole numbers."""
    import torch

    dtype, low, high = getattr(torch, name), 1 << (bits - 1), 1 << bits
    m, t = (a.reshape(1, -1) for a in np.meshgrid(np.arange(low, high), np.arange(9), indexing="ij"))
    n = np.arange(low, high).reshape(-1, 1)
    m = np.where((t == 0) & (m > n), n, m)
    x = torch.from_numpy(m * 0.5 ** (10 + t)).to(dtype)
    assert torch.equal(x.double(), torch.from_numpy(m * 0.5 ** (10 + t)))
    x[:, ::3] *= -1
    got = ctx.quantize_i8(x.cuda()).codes.cpu().numpy()
    num, den = 127 * m, n << t
    k, rest = num // den, 2 * (num % den)
    want = np.where((rest > den) | ((rest == den) & (k % 2 == 1)), k + 1, k)
    want[:, ::3] *= -1
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("K,pad,offset", [(700, 0, 0), (701, 3, 1), (9000, 0, 0), (20000, 0, 0), (20001, 2, 3)])
def test_16_bit_rows_full_of_borders(ctx, kind, K, pad, offset):
    """A largest value whose mantissa 127 divides (254, and 1143 = 9 * 127 in half), and odd multiples of a 254th of it."""
    import torch

    rows = []
    for peak, step, most in [(254.0, 1.0, 253)] + ([(1143.0, 4.5, 227)] if kind == "f16" else []):
        row = np.resize(step * np.arange(1, most + 1, 2), K)
        row[1::2] *= -1
        row[K // 2] = peak
        rows += [row, row / 1024]
    x = torch.from_numpy(np.stack(rows)).to(dtype_of(kind))
    assert torch.equal(x.double(), torch.from_numpy(np.stack(rows)))
    codes, scales, _ = rows_reference(x.float().numpy(), None, None, 0.0)
    check_rows(ctx.quantize_i8(place(x, kind, pad, offset)[1]), codes, scales, K)


def test_rows_of_several_dimensions(ctx):
    """[batch, tokens, K] and a single row [K] are rows like any others."""
    import torch

    x, r = torch.randn(3, 5, 256, device="cuda"), torch.randn(3, 5, 256, device="cuda")
    w = torch.rand(256, device="cuda")
    got, total = ctx.add_rmsnorm_i8(x, w, 1e-5, residual=r)
    flat, flat_total = ctx.add_rmsnorm_i8(x.view(15, 256), w, 1e-5, residual=r.view(15, 256))
    assert total.shape == x.shape and torch.equal(total.view(15, 256), flat_total) and torch.equal(got.codes, flat.codes)
    one, one_total = ctx.add_rmsnorm_i8(x[1, 2], w, 1e-5, residual=r[1, 2])
    assert torch.equal(one.codes[0], flat.codes[7]) and torch.equal(one_total, flat_total[7])
    assert torch.equal(ctx.quantize_i8(x).codes, ctx.quantize_i8(x.view(15, 256)).codes)
    head = ctx.quantize_i8(torch.randn(40, 256, device="cuda"))
    out = torch.empty(3, 5, 40, device="cuda")
    assert ctx.matmul_i8(got, head, out=out) is out and torch.equal(out.view(15, 40), ctx.matmul_i8(flat, head))


def test_nothing_to_do(ctx):
    import torch

    w = ctx.quantize_i8(torch.randn(10, 64, device="cuda"))
    empty = ctx.quantize_i8(torch.empty(0, 64, device="cuda"))
    assert tuple(empty.codes.shape) == (0, 64)
    assert tuple(ctx.matmul_i8(empty, w).shape) == (0, 10)
    assert tuple(ctx.matmul_i8(w, empty).shape) == (10, 0)
    got, total = ctx.add_rmsnorm_i8(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"), 1e-5, residual=torch.empty(0, 64, device="cuda"))
    assert tuple(total.shape) == (0, 64) and tuple(got.scales.shape) == (0,)


@pytest.mark.parametrize("qtype", [orc.Q4_K, orc.Q5_K, orc.Q6_K])
def test_kquant_weight_in_8_bits(ctx, qtype):
    N, K = 300, 1024
    raw = synth.make_kq_weights(qtype, N, K, 9)
    got = ctx.i8_weight(ctx.upload(pack_kq(qtype, raw, N, K)))
    deq = orc.dequant(raw, N, K) if qtype == orc.Q4_K else orc.kq_dequant(qtype, raw, N, K)
    codes, scales, _ = rows_reference(deq.reshape(N, K), None, None, 0.0)
    check_rows(got, codes, scales, K)


def test_refusals(ctx):
    import torch

    lib, h = ctx.lib, ctx.h
    x = torch.randn(4, 64, device="cuda")
    w = torch.rand(64, device="cuda")
    c, s = torch.empty(4, 64, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    y = torch.empty(4, 4, device="cuda")

    def norm(ft=0, x=x.data_ptr(), r=None, w=w.data_ptr(), eps=1e-5, sm=None, c=c.data_ptr(), s=s.data_ptr(), M=4, K=64, ldx=64, ldr=64, lds=64, ldc=64):
        return lib.bpq4k_add_rmsnorm_i8(h, ft, x, r, w, eps, sm, c, s, M, K, ldx, ldr, lds, ldc, 0)

    assert norm() == 0 and norm(M=0, x=None, w=None) == 0
    assert norm(ft=12) == 2 and norm(K=0) == 2 and norm(K=32769, ldx=40000, ldc=40000) == 2 and norm(M=1 << 31) == 2
    assert norm(x=None) == 1 and norm(w=None) == 1 and norm(c=None) == 1 and norm(s=None) == 1 and norm(sm=y.data_ptr()) == 1
    assert norm(ldx=63) == 1 and norm(ldc=48) == 1 and norm(r=x.data_ptr(), ldr=1) == 1 and norm(r=x.data_ptr(), sm=x.data_ptr(), lds=0) == 1
    assert norm(r=x.data_ptr(), M=2, sm=x.data_ptr(), lds=128) == 1
    assert norm(eps=-1.0) == 1 and norm(eps=float("nan")) == 1
    assert norm(x=x.data_ptr() + 2) == 3 and norm(c=c.data_ptr() + 8) == 3 and norm(ldc=72) == 3 and norm(s=s.data_ptr() + 1) == 3
    assert "multiple of 16" in (norm(ldc=72), lib.bpq4k_last_error_string(h).decode())[1]

    def quant(ft=0, x=x.data_ptr(), c=c.data_ptr(), s=s.data_ptr(), M=4, K=64, ldx=64, ldc=64):
        return lib.bpq4k_quantize_i8(h, ft, x, c, s, M, K, ldx, ldc, 0)

    assert quant() == 0 and quant(M=0, x=None) == 0 and quant(ft=2) == 2 and quant(x=None) == 1 and quant(K=0) == 2 and quant(c=c.data_ptr() + 1) == 3

    def product(ft=0, x=c.data_ptr(), xs=s.data_ptr(), w=c.data_ptr(), ws=s.data_ptr(), b=None, y=y.data_ptr(), M=4, N=4, K=64, ldx=64, ldw=64, ldy=4):
        return lib.bpq4k_matmul_i8(h, ft, x, xs, w, ws, b, y, M, N, K, ldx, ldw, ldy, 0)

    assert product() == 0 and product(M=0, x=None) == 0 and product(N=0, w=None) == 0
    assert product(ft=24) == 2 and product(K=0) == 2 and product(K=131072, ldx=131072, ldw=131072) == 2
    assert product(M=(1 << 24) + 1) == 2 and product(N=(1 << 24) + 1) == 2
    assert product(x=None) == 1 and product(xs=None) == 1 and product(w=None) == 1 and product(ws=None) == 1 and product(y=None) == 1
    assert product(ldx=48) == 1 and product(ldw=48) == 1 and product(ldy=3) == 1
    assert product(x=c.data_ptr() + 4) == 3 and product(w=c.data_ptr() + 8) == 3 and product(ldx=72) == 3 and product(ldw=65) == 3
    assert product(y=y.data_ptr() + 2) == 3 and product(ft=1, y=y.data_ptr() + 1) == 3 and product(b=s.data_ptr() + 2) == 3 and product(xs=s.data_ptr() + 1) == 3
    for args in (lambda: ctx.quantize_i8(x.double()), lambda: ctx.quantize_i8(x.cpu()), lambda: ctx.quantize_i8(x.t()),
                 lambda: ctx.matmul_i8(I8Rows(c, s), I8Rows(c[:, :48], s)), lambda: ctx.matmul_i8(I8Rows(c, s[:3]), I8Rows(c, s)),
                 lambda: ctx.matmul_i8(I8Rows(c, s), I8Rows(c, s), bias=torch.zeros(3, device="cuda")),
                 lambda: ctx.matmul_i8(I8Rows(c, s), I8Rows(c, s), out=torch.empty(4, 5, device="cuda")),
                 lambda: ctx.matmul_i8(I8Rows(c, s), I8Rows(c, s), out=y, dtype=torch.float16),
                 lambda: ctx.add_rmsnorm_i8(x, w[:10], 1e-5), lambda: ctx.add_rmsnorm_i8(x, w, 1e-5, sum_out=x),
                 lambda: ctx.add_rmsnorm_i8(x, w, 1e-5, residual=x[:2]), lambda: ctx.add_rmsnorm_i8(x, w, 1e-5, residual=x.half()),
                 lambda: ctx.quantize_i8(x, out=I8Rows(c[:2], s[:2]))):
        with pytest.raises(ValueError):
            args()
    with pytest.raises(Q4KError, match="multiple of 16"):
        ctx.matmul_i8(I8Rows(torch.zeros(3, 20, dtype=torch.int8, device="cuda"), s[:3]), I8Rows(c[:, :20], s))
    torch.cuda.synchronize()
    assert ctx.device_status() == 0


# ---- together, as a program uses them ---------------------------------------------------------------------------------------

def last_layer(ctx, x, r, nw, head, given):
    rows, total = ctx.add_rmsnorm_i8(x, nw, 1e-5, residual=r)
    logits = ctx.matmul_i8(rows, head)
    return total, logits, ctx.logprobs(logits, given=given, top=4)


def make_last_layer(M, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    K, V = 1024, 5003
    x, r = (torch.randn(M, K, device="cuda", generator=g) for _ in range(2))
    nw = torch.rand(K, device="cuda", generator=g) + 0.5
    head = torch.randn(V, K, device="cuda", generator=g) * 0.05
    return x, r, nw, head, torch.randint(0, V, (M,), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("M", [1, 6, 90, 300])
def test_norm_head_and_answer_together(ctx, M):
    import torch

    x, r, nw, head, given = make_last_layer(M, M)
    total, logits, lp = last_layer(ctx, x, r, nw, ctx.quantize_i8(head), given)
    v = x.double() + r.double()
    y = v * nw.double() / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)
    want = y @ head.double().T
    # codes are off by at most half a step of their row's scale on either side: |error| <= sum |y| sw/2 + |head| sx/2 + sx sw/4
    sx, sw = y.abs().amax(1) / 127, head.double().abs().amax(1) / 127
    bound = 0.5 * (y.abs().sum(1)[:, None] * sw + sx[:, None] * head.double().abs().sum(1)) + 0.25 * 1024 * sx[:, None] * sw
    assert bool(((logits.double() - want).abs() <= bound * 1.001).all())
    ref = torch.log_softmax(logits.double(), 1)
    assert torch.allclose(lp.given.double(), ref.gather(1, given.long()[:, None])[:, 0], rtol=0, atol=1e-5)
    assert torch.equal(lp.top_ids.long(), torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :4])
    assert torch.equal(total, x + r)


def test_captured_replayed_and_side_by_side(ctx):
    """Two graphs of the whole run replayed at once on two streams, and eager calls beside them: nothing is shared."""
    import torch

    sets, graphs, outs, wants = [make_last_layer(m, 100 + m) for m in (3, 200)], [], [], []
    heads = [ctx.quantize_i8(s[3]) for s in sets]
    for s, hd in zip(sets, heads):
        wants.append(last_layer(ctx, *s[:3], hd, s[4]))
    torch.cuda.synchronize()
    for s, hd in zip(sets, heads):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(last_layer(ctx, *s[:3], hd, s[4]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        last_layer(ctx, *sets[0][:3], heads[0], sets[0][4])
    torch.cuda.synchronize()
    for (t, y, lp), (wt, wy, wlp) in zip(outs, wants):
        assert torch.equal(t, wt) and torch.equal(y, wy) and torch.equal(lp.given, wlp.given)
        assert torch.equal(lp.entropy, wlp.entropy) and torch.equal(lp.top_ids, wlp.top_ids) and torch.equal(lp.top, wlp.top)
    assert ctx.device_status() == 0


FIRST_CALL_IS_CAPTURED = """
import torch, backpack_b200 as bp
ctx = bp.Q4KContext(0)
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, device="cuda", generator=g)
sets = [(r(m, k), r(m, k), torch.rand(k, device="cuda", generator=g), bp.I8Rows(torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g),
         torch.rand(n, device="cuda", generator=g))) for m, n, k in [(1, 512, 1024), (20, 512, 8192), (100, 1000, 4096), (300, 2000, 512)]]
def run(s):
    rows, total = ctx.add_rmsnorm_i8(s[0], s[2], 1e-5, residual=s[1])
    y = ctx.matmul_i8(rows, s[3])
    lp = ctx.logprobs(y, top=3)
    return total, y, lp.entropy, lp.top_ids
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [run(s) for s in sets]
for _ in range(3):
    graph.replay()
torch.cuda.synchronize()
for o, s in zip(outs, sets):
    assert all(torch.equal(a, b) for a, b in zip(o, run(s)))
assert ctx.device_status() == 0
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IS_CAPTURED], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_calls_on_another_stream_and_from_threads(ctx):
    """Calls queued on a stream that is not the current one's default, a handle per thread."""
    import threading

    import torch

    sets = [make_last_layer(m, 200 + m) for m in (2, 130)]
    want = [last_layer(ctx, *s[:3], ctx.quantize_i8(s[3]), s[4]) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        c = Q4KContext(0)
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(10):
                    t, y, lp = last_layer(c, *sets[i][:3], c.quantize_i8(sets[i][3]), sets[i][4])
                    st.synchronize()
                    if not (torch.equal(y, want[i][1]) and torch.equal(lp.top, want[i][2].top)):
                        bad.append(i)
        finally:
            c.close()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_offsets_beyond_32_bits(ctx):
    """More than 2^32 codes, values or outputs: the last rows are as they are by themselves."""
    import torch

    K, N = 32768, 131072 + 300
    w = I8Rows(torch.empty((N, K), dtype=torch.int8, device="cuda"), torch.rand(N, device="cuda"))
    for n in range(0, N, 8192):
        w.codes[n:n + 8192].random_(-127, 128)
    x = ctx.quantize_i8(torch.randn(200, K, device="cuda"))
    for m in (1, 20, 200):
        y = ctx.matmul_i8(x.rows(0, m), w)
        assert torch.equal(y[:, -500:], ctx.matmul_i8(x.rows(0, m), I8Rows(w.codes[-500:].clone(), w.scales[-500:].clone())))
        assert torch.equal(y[:, :500], ctx.matmul_i8(x.rows(0, m), w.rows(0, 500)))
        del y
    big = I8Rows(w.codes[:, :64].contiguous(), w.scales)
    xs = I8Rows(torch.empty((33000, 64), dtype=torch.int8, device="cuda").random_(-127, 128), torch.rand(33000, device="cuda"))
    y = ctx.matmul_i8(xs, big, dtype=torch.bfloat16)                      # 33000 x 131372: 4.3e9 outputs
    assert torch.equal(y[-3:], ctx.matmul_i8(xs.rows(32997, 33000), big, dtype=torch.bfloat16))
    given = torch.full((33000,), 131371, dtype=torch.int32, device="cuda")
    lp = ctx.logprobs(y, given=given, top=2)
    part = ctx.logprobs(y[-3:].clone(), given=given[-3:], top=2)
    assert torch.equal(lp.top_ids[-3:], part.top_ids) and torch.allclose(lp.given[-3:], part.given, rtol=1e-5)
    del y, lp, part
    v = torch.zeros((N + 8, K), dtype=torch.float16, device="cuda")
    v[-5:].normal_()
    got = ctx.quantize_i8(v, out=I8Rows(torch.empty((N + 8, K), dtype=torch.int8, device="cuda"), torch.empty(N + 8, device="cuda")))
    tail = ctx.quantize_i8(v[-5:].clone())
    assert torch.equal(got.codes[-5:], tail.codes) and torch.equal(got.scales[-5:], tail.scales) and not bool(got.scales[:-5].any())


def test_same_calls_on_the_debug_build():
    import torch

    c = Q4KContext(0, debug=True)
    try:
        for M, N, K in [(1, 7, 15), (5, 257, 500), (64, 300, 1024), (150, 385, 640), (300, 1000, 272)]:
            host, (xr, wr, bias) = make_product(M, N, K, 3, True)
            check_product(c.matmul_i8(xr, wr, bias=bias), *host, "f32")
            x = torch.randn(M, K, device="cuda")
            got, _ = c.add_rmsnorm_i8(x, torch.ones(K, device="cuda"), 1e-5, residual=x)
            check_rows(got, *rows_reference(x.cpu().numpy(), x.cpu().numpy(), np.ones(K, np.float32), float(np.float32(1e-5)))[:2], K)
            c.logprobs(x, given=torch.zeros(M, dtype=torch.int32, device="cuda"), top=min(K, 5))
        assert c.device_status() == 0
        assert c.launch_count() >= 15
    finally:
        c.close()
