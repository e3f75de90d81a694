"""What products with low-rank adapters refuse for their sizes, as far as no GPU is involved."""
import pytest

from tests.test_host_mx4 import refused
from tests.test_host_mx4_attention import adapters, fc_args


@pytest.mark.parametrize("in_type, size", [(0, 4), (1, 2), (3, 0)])
@pytest.mark.parametrize("K", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 4096])
def test_columns_that_32_bits_do_not_count(K, in_type, size):
    """Steps of 64 columns that go past the last of them would pass 2^31."""
    row = -(-(-(-K // 128)) * 68 // 16) * 16
    at = 1 << 50                       # (the sizes are larger than the distances between the others' addresses)
    args = fc_args(adapters(count=1, down=2 * at, up=3 * at), M=1, K=K, N=1, in_type=in_type, in_row=K * size or row, w_row=row,
                   x=4 * at, w=5 * at, ws=6 * at, ws_bytes=1 << 40, out_row=16)
    refused("mi355x_mx4_fc_adapters", args, "columns", -4)
