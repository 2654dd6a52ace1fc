"""Waits of the 8-bit matmul that run out: the status word says so, and the next call is as if nothing had happened.  The loads and
products do complete; only the patience with them is short."""
import pytest

from backpack_b200 import I8Rows, Q4KContext, Q4KError, q4k

pytestmark = pytest.mark.gpu

TIMEOUT = 6
# one CTA a tile (few tiles; several a CTA; all steps of a tile in the ring at once), shared tiles that exchange their sums beside the
# ring and in it, pairs (one tile; several; few steps)
SHAPES = [(20, 700, 640), (20, 40000, 4096), (20, 4096, 512), (20, 500, 32768), (9, 129, 131071), (100, 500, 65536), (128, 1000, 16384),
          (300, 2048, 8192), (400, 20000, 4096), (600, 9000, 384)]
# a CTA takes in 92 GB/s, so the first sums of these are there after some 20 us (1024 / 8 steps of 18 KB, 512 / 8 of 29, 64 of 32): in the
# product build a single poll, of 4 us, is over before
SLOW = [(9, 129, 131071), (100, 500, 65536), (300, 2048, 8192)]


def status(ctx):
    try:
        return ctx.device_status()
    except Q4KError as e:
        return e.status


@pytest.fixture(scope="module", params=["product", "debug"])
def own(request):
    c = Q4KContext(0, debug=request.param == "debug")
    c.fine = request.param == "debug"              # polls of some 20 ns: waits run out anywhere
    yield c
    c.close()


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_a_wait_that_runs_out_is_reported(own, M, N, K):
    import torch

    g = torch.Generator(device="cuda").manual_seed(M + N + K)

    def rows(n):
        codes = torch.empty((n, (K + 15) // 16 * 16), dtype=torch.int8, device="cuda").random_(-127, 128, generator=g)[:, :K]
        return I8Rows(codes, torch.rand(n, device="cuda", generator=g))

    x, w = rows(M), rows(N)
    want = own.matmul_i8(x, w)
    assert status(own) == 0
    buf = torch.full((M + 2, N + 8), -7777.0, device="cuda")
    out, seen = buf[1:M + 1, :N], []
    try:
        for polls in (1, 1, 2, 4, 12, 25, 50, 75, 100, 150, 200, 300, 400, 600, 1000, 2000, 1):
            own.set_option(q4k.OPT_I8_WAIT_POLLS, polls)
            own.matmul_i8(x, w, out=out)
            own.set_option(q4k.OPT_I8_WAIT_POLLS, 0)
            after = own.matmul_i8(x, w)                # right behind a call that may have given up, on the same SMs
            seen.append(status(own))
            assert seen[-1] in (0, TIMEOUT)
            assert torch.equal(after, want) and (seen[-1] or torch.equal(out, want))
            assert status(own) == 0
    finally:
        own.set_option(q4k.OPT_I8_WAIT_POLLS, 0)
    if own.fine or (M, N, K) in SLOW:                # (in the debug build one poll is over before the first copy has come)
        assert seen[0] == seen[-1] == TIMEOUT, seen
    out.fill_(-7777.0)
    assert bool((buf == -7777.0).all())


def test_the_option(own):
    assert own.get_option(q4k.OPT_I8_WAIT_POLLS) == 0
    with pytest.raises(Q4KError):
        own.set_option(q4k.OPT_I8_WAIT_POLLS, -1)
    own.set_option(q4k.OPT_I8_WAIT_POLLS, 7)
    assert own.get_option(q4k.OPT_I8_WAIT_POLLS) == 7
    own.set_option(q4k.OPT_I8_WAIT_POLLS, 0)
