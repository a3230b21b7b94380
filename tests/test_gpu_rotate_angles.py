"""GPU: the cosines and sines of kvcache.append_rotated, to the bound that its series has."""
import numpy as np
import pytest
import torch

from tests import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at", [1.0, 0.95, 0.5])
def test_cosines_and_sines_are_rounded_from_40_bits(gpu, at):
    """Angles around `at` of an eighth of a turn, where the series leave the most: half a step of float32 and 2^-40."""
    from tallax_amd import kvcache
    rng = np.random.default_rng(0)
    tokens, pairs = 256, 128
    k, v, table = R.make_cache(rng, 1, 1, 256, 16, 16, [tokens], torch.float32)
    x = torch.zeros((1, tokens, 1, 256), device=gpu)
    x[..., :pairs] = 1.0  # y0 = cos a, y1 = sin a
    # odd multiples of an eighth of a turn; or of a part of it, a quarter apart: 2 pi p / 4 + at pi / 4 = p f
    p = 1 + 2 * np.arange(tokens) if at == 1.0 else np.ones(tokens, np.int64)
    places = torch.from_numpy(p.astype(np.int32))[None].to(gpu)
    lens = torch.zeros(1, dtype=torch.int32, device=gpu)
    steps = np.arange(16 * pairs).reshape(16, pairs) - 8 * pairs
    for i in range(16):
        if at == 1.0:
            f = (np.round(np.pi / 4 * 2 ** 24) + steps[i]) * 2.0 ** -24
        else:
            f = at * np.pi / 4 + np.pi / 2 * rng.integers(0, 4, pairs) + steps[i] * 2.0 ** -20
        f = f.astype(np.float32)
        _, q = kvcache.append_rotated(k.to(gpu), v.to(gpu), table.to(gpu), lens, x, x, x, torch.from_numpy(f).to(gpu),
                                      token_positions=places)
        got = q[0, :, 0].cpu().numpy().astype(np.float64)
        a = p[:, None] * f.astype(np.float64)  # exact: 9 and 24 bits
        want = np.concatenate([np.cos(a), np.sin(a)], 1)
        # half a step of float32 (of the larger neighbour, where the rounding crosses a power of two), the series, and
        # 2^-43 for the angle in turns (up to 64 of them to 2^-52, twice, by 2 pi) and the reference's own rounding
        half = np.spacing(np.maximum(np.abs(got), np.abs(want)).astype(np.float32)).astype(np.float64) / 2
        off = np.abs(got - want) - half
        assert off.max() <= 2.0 ** -40 + 2.0 ** -43, (i, off.max(), int((off > 2.0 ** -40).sum()))
