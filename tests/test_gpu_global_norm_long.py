"""The global norm and the clip of lists past 256 MB, whose reads and writes go round the last-level cache, and of lists with
more tensors than any table: the bounds of tests/test_gpu_global_norm.py."""
import pytest
import torch

from tests.test_gpu_global_norm import check, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)])
def test_past_the_cache(dtypes):
    """Odd offsets in a shared buffer, ragged ends, single values and long tensors."""
    sizes = [1, 3, 70_000_001, 4097, 33_333_333, 16383, 60_000_007, 5, 40_000_003]
    ts = []
    for i, dt in enumerate(dtypes):
        mine = [n for k, n in enumerate(sizes) if k % len(dtypes) == i]
        flat = tensors([sum(mine) + 1], (dt,), seed=i, scale=0.01)[0][1:]
        ts += list(torch.split(flat, mine))
    assert sum(t.numel() * t.element_size() for t in ts) > 256 << 20
    check(ts)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("count", [128, 129, 5000, 20000])
def test_many_tensors(count):
    flat = tensors([count * 3], (torch.float32,))[0]
    check(list(torch.split(flat, 3)))
