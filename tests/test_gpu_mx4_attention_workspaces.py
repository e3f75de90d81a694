"""Attention over microscaled rows with workspaces of exactly the bytes that are asked for, which no window, number of first tokens
or type is told: calls are made and write nothing behind them."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref
from tests.test_gpu_mx4_attention import queries
from tests.test_gpu_mx4_serving import Call

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("dim, kv_heads, group, lengths, new", [
    (64, 2, 4, [3000, 40], [1, 1]), (128, 8, 2, [3000, 40], [2, 1]), (128, 3, 2, [3000, 40], [1, 3]), (256, 1, 8, [3000], [2]),
    (64, 1, 8, [3000, 40], [8, 8]), (64, 1, 8, [3000, 40], [8, 9]), (128, 2, 4, [3000], [70]), (256, 1, 4, [3000, 700], [70, 70]),
    (128, 1, 16, [5000], [130]), (64, 2, 2, [2000], [1000])])
def test_exactly_what_is_asked_for(dim, kv_heads, group, lengths, new, type_):
    """Both kernels, and batches on either side of the choice between them."""
    rng = np.random.default_rng(dim + kv_heads)
    b = aref.Batch(rng, lengths, new, kv_heads, dim, 32)
    heads = kv_heads * group
    q = queries(rng, b, heads, type_)
    for window, sinks in ((0, 0), (1, 0), (17, 4), (600, 0), (600, 2000), (2000, 3), (2990, 1), (5000, 9), (2 ** 40, 2 ** 40)):
        call = Call(b, q, heads, type_, window=window, sinks=sinks)
        call.q_host, size = q, call.n
        call.ws = capi.to_device(np.full(size + GUARD, 0xa5, np.uint8))
        call.launch()
        got = call.out.numpy()
        assert (call.ws.numpy()[size:] == 0xa5).all()
        if rng.random() < 0.3:
            call.check(got)
    assert size > 0 or dim == 64 and new == [1000]
