"""What products with low-rank adapters refuse for their sizes, as far as no GPU is involved."""
import numpy as np
import pytest

from glow_amd import capi
from tests.mx4_ref import row_bytes
from tests.test_host_mx4 import refused
from tests.test_host_mx4_attention import adapters, fc_args


@pytest.mark.parametrize("in_type, size", [(0, 4), (1, 2), (3, 0)])
@pytest.mark.parametrize("K", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 4096])
def test_columns_that_32_bits_do_not_count(K, in_type, size):
    """Steps of 64 columns that go past the last of them would pass 2^31."""
    row = row_bytes(K)
    at = 1 << 50                       # (the sizes are larger than the distances between the others' addresses)
    args = fc_args(adapters(count=1, down=2 * at, up=3 * at), M=1, K=K, N=1, in_type=in_type, in_row=K * size or row, w_row=row,
                   x=4 * at, w=5 * at, ws=6 * at, ws_bytes=1 << 40, out_row=16)
    refused("mi355x_mx4_fc_adapters", args, "columns", -4)


@pytest.mark.parametrize("in_type", [0, 1, 2, 3])
@pytest.mark.parametrize("M, K, N, rank", [(1, 1, 1, 1), (1, 4096, 64, 16), (64, 4096, 4096, 16), (300, 96, 64, 8), (4096, 4096, 4096, 64)])
def test_workspaces_hold_both_launches(M, K, N, rank, in_type):
    """A workspace of its own, of at least down's results and what the shared product asks for; none without rows, results or rank."""
    n = capi.mx4_fc_adapters_workspace_bytes(M, K, N, in_type, rank)
    assert n >= 4 * M * rank + capi.mx4_fc_workspace_bytes(M, K, N, in_type) and n % 16 == 0
    if in_type == 3:
        assert capi.mx4_fc_workspace_bytes(M, K, N, in_type) == 0
        assert capi.mx4_fc_adapters_workspace_bytes(M, K, N, in_type, 0) == 0
    assert capi.mx4_fc_adapters_workspace_bytes(0, K, N, in_type, rank) == capi.mx4_fc_adapters_workspace_bytes(M, K, 0, in_type, rank) == 0
    shape = dict(M=M, K=K, N=N, in_type=in_type, in_row=max(4 * K, row_bytes(K)), w_row=row_bytes(K), out_row=2 * N)
    for change in (dict(ws=0), dict(ws_bytes=n - 1)):
        refused("mi355x_mx4_fc_adapters", fc_args(adapters(rank=rank), **shape, **change), "workspace")


@pytest.mark.parametrize("change", [dict(x=(100,)), dict(weights=(80,)), dict(down=(100,)), dict(down=(4, 100)), dict(up=(5,)), dict(up=(5, 4))])
def test_the_convenience_refuses_arrays_of_other_ranks(change):
    shapes = dict(x=(2, 100), weights=(5, 80), down=(1, 4, 100), up=(1, 5, 4))
    shapes.update(change)
    x, weights, down, up = (np.zeros(shapes[k], np.uint8 if k == "weights" else np.float32) for k in ("x", "weights", "down", "up"))
    with pytest.raises(capi.MI355XError, match="of shape"):
        capi.mx4_fc_adapters(x, 0, weights, None, 100, down, up, np.zeros(2, np.int32))
