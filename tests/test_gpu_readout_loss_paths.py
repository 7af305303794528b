"""The read-out's cross-entropy at sizes that take the tiled kernels through each way they have of dividing the work, against
64 bits with the bounds of tests/test_gpu_readout_loss.py: classes in several pieces in the loss (the running rows carried
from one to the next) and in the gradient, a piece's classes in one launch of large and one of small tiles, large tiles with
their contraction split."""
import pytest
import torch

from tests.test_gpu_readout_loss import check, make

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16


@pytest.mark.parametrize("size,dtype,kind", [
    ((17, 4096, 50000), F, "i64"), ((17, 4096, 50000), F, "rows"),  # loss and gradient in two pieces, gx in large split tiles
    ((17, 2047, 300000), B, "i64"),                                  # likewise, W packed, gx in small tiles
    ((20000, 520, 26000), B, "i64"),                                 # two pieces, each one's dl in two launches
    ((1021, 333, 50021), B, "i64"), ((1021, 333, 50021), B, "rows"),  # loss and dl in two launches, gx in large split tiles
    ((1000, 2048, 50000), B, "i32"),                                 # likewise, x and W as they lie
    ((1021, 333, 50021), F, "i64"),                                  # loss and dl of three parts in two launches
    ((4000, 64, 9000), B, "i64"), ((4000, 64, 9000), F, "rows"),     # one of them in two launches
    ((5000, 200, 6000), F, "i64"),                                   # gW in large split tiles
    # up to 64 rows: gW's contraction has one or two steps, and small tiles beside gx's
    ((24, 256, 2000), B, "i64"), ((50, 64, 9000), B, "rows"), ((64, 72, 700), B, "i64"), ((17, 130, 513), B, "rows"),
    ((2048, 256, 8191), B, "rows"), ((2903, 51, 1293), B, "i64"),
])
def test_ways_of_dividing_the_work(size, dtype, kind):
    check(make(*size, dtype, kind))
    torch.cuda.empty_cache()
