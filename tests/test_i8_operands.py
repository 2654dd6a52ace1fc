"""What the 8-bit path's binding takes as rows, and what it refuses; no device needed."""
import pytest

from backpack_b200 import Q4KContext, q4k


@pytest.fixture(scope="module")
def binding():
    import torch

    c = Q4KContext.__new__(Q4KContext)          # (a handle needs a device; its checks of operands do not)
    c._torch, c._dev, c._ftype = torch, torch.device("cpu"), {torch.float32: q4k.F32, torch.float16: q4k.F16, torch.bfloat16: q4k.BF16}
    return c


def test_rows_at_one_distance(binding):
    import torch

    x = torch.zeros(6, 4, 32)
    for t, want in ((x, (24, 32, 32)), (x[1, 2], (1, 32, 32)), (x[:, 1], (6, 32, 128)), (x[2:4, 0, :5], (2, 5, 128)), (x[:, :, :8], (24, 8, 32)),
                    (x[:, :, :1], (24, 1, 32)), (torch.zeros(0, 3, 32), (0, 32, 32)), (torch.zeros(3, 0, 32), (0, 32, 32))):
        _, ft, *rows = binding._rows(t, "x")
        assert ft == q4k.F32 and tuple(rows) == want, tuple(t.shape)


def test_what_is_not_rows(binding):
    import torch

    x = torch.zeros(6, 4, 32)
    for t in (x.transpose(0, 1), x[:, :2], torch.tensor(1.0), torch.zeros(3, 2, 0), x[:, :, ::2], x[0].t(), x.double(), torch.zeros(4, 4, dtype=torch.int8)):
        with pytest.raises(ValueError):
            binding._rows(t, "x")
    with pytest.raises(ValueError, match="distance"):
        binding.quantize_i8(x.transpose(0, 1))
