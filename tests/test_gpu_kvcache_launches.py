"""GPU: kvcache.decode at numbers of workgroups on both sides of a choice between instances, against the plain 64-bit
form."""
import numpy as np
import pytest
import torch

from tests import serving_ref as R
from tests.test_gpu_kvcache import _check, _decode, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [72, 80, 128])
@pytest.mark.parametrize("batch", [95, 96, 97])  # 760, 768 and 776 workgroups of one chunk
def test_decode_f32_waves(gpu, dim, batch):
    rng = np.random.default_rng(31)
    lens = [0, 1] + rng.integers(2, 70, batch - 2).tolist()
    q, k, v, table, lens, _, scores = _inputs(31, "f32", batch, 1, 8, 8, dim, 16, lens, None)
    assert table.shape[1] * 16 <= 256  # one chunk
    want = R.attention(q, k, v, table, lens, dim ** -0.5, None, scores)
    out, lse, new = _decode(gpu, q, k, v, table, lens, None, scores)
    _check(out, want[0], want[3][0], "out")
    _check(lse, want[1], want[3][1], "lse")
    _check(new, want[2], want[3][2], "scores")


def test_decode_f32_waves_split(gpu):
    """The same sequences in tables that make 640 and 880 workgroups: chunks of one size, so the same sums."""
    q, k, v, table, lens, _, scores = _inputs(32, "f32", 10, 1, 8, 8, 128, 16, [1790 - 130 * i for i in range(10)], None)
    wide = torch.cat([table, torch.full((10, 2800 // 16 - table.shape[1]), -1, dtype=torch.int32)], 1)
    want = R.attention(q, k, v, table, lens, 128 ** -0.5, None, None)
    for t in (table, wide):
        out, lse = _decode(gpu, q, k, v, t.contiguous(), lens)
        _check(out, want[0], want[3][0], "out")
        _check(lse, want[1], want[3][1], "lse")
