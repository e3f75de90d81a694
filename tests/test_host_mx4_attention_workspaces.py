"""Workspaces of attention over microscaled rows, as far as no GPU is involved."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref
from tests.test_host_mx4 import refused
from tests.test_host_mx4_attention import attention_args, cache

MOST = 66 << 20


def sized(kv, dim):
    return cache(kv_heads=kv, head_dim=dim, row_bytes=ref.row_bytes(kv * dim), keys=1 << 50, values=1 << 51, n_pages=10 ** 6,
                 pages_per_sequence=10 ** 5)


@pytest.mark.parametrize("kv, dim, group", [(1, 64, 1), (2, 64, 4), (8, 128, 4), (3, 128, 2), (1, 256, 8)])
def test_what_is_asked_for_is_enough_and_no_less(kv, dim, group):
    """Few rows, which are cut alike whatever their type. (Windows and many rows: on the device, where such calls may be made.)"""
    c, asked = sized(kv, dim), 0
    for sequences, rows in ((1, 1), (3, 3), (3, 7), (1, 4), (20, 40)):
        for most in (10, 300, 5000, 131072, 10 ** 6):
            n = capi.mx4_attention_workspace_bytes(c, kv * group, sequences, rows, most)
            for type_ in (ref.F32, ref.F16, ref.BF16) if n else ():
                row = kv * group * dim * (4 if type_ == ref.F32 else 2)
                args = dict(c=c, out_type=type_, out_row=row, type_=type_, q_row=row, heads=kv * group, sequences=sequences, rows=rows,
                            most=most)
                # (the size is looked at before whether the workspace overlaps a tensor)
                refused("mi355x_mx4_attention", attention_args(**args, ws=(1 << 50) + 16, ws_bytes=n), "the workspace overlaps")
                refused("mi355x_mx4_attention", attention_args(**args, ws_bytes=n - 1), "a workspace of")
                asked += 1
    assert asked > 5


def test_one_size_holds_for_every_batch():
    rng = np.random.default_rng(1)
    sizes = []
    for _ in range(4000):
        kv, dim, group = int(rng.choice([1, 2, 3, 4, 5, 8, 16, 24])), int(rng.choice([64, 128, 256])), int(rng.integers(1, 17))
        sequences = int(2 ** rng.uniform(0, 10))
        rows = int(sequences * 2 ** rng.uniform(-1, 7)) + 1
        sizes.append(capi.mx4_attention_workspace_bytes(sized(kv, dim), kv * group, sequences, rows, int(2 ** rng.uniform(0, 20))))
    assert MOST // 2 < max(sizes) <= MOST
    # and the largest batch is not the one that asks for most
    n = [capi.mx4_attention_workspace_bytes(sized(8, 128), 32, s, s, 131072) for s in (1, 8, 256, 300)]
    assert 0 < n[0] < n[1] and n[2] > 0 and n[3] == 0
