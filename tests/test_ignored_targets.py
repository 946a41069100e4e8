"""Which targets `ignore_index` leaves out (CPU), whatever integer type they come in: those equal to it as numbers."""
import pytest
import torch

from noetic_tensor_b200 import loss


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("ignore_index", [-100, 5, 156, 70000, 2**32 + 5, -(2**32) + 5, 2**31, -(2**31)])
@pytest.mark.parametrize("check", [False, True])
def test_ignored(dtype, ignore_index, check):
    info = torch.iinfo(dtype)
    numbers = [n for n in (1, 5, 156, 100, 0) if info.min <= n <= info.max]
    if not check and info.min <= -100:
        numbers += [-100, -1]
    elif info.min <= ignore_index <= info.max:
        numbers += [ignore_index]
    ids, keep = loss._targets(torch.tensor(numbers, dtype=dtype), 1, len(numbers), 512, ignore_index, check=check)
    assert keep.tolist() == [0.0 if n == ignore_index else 1.0 for n in numbers]
    assert ids.dtype == torch.int32
    for got, n in zip(ids.tolist(), numbers):
        want = 0 if n == ignore_index else n
        assert got == want or (not 0 <= want < 512 and not 0 <= got < 512)
