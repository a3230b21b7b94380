"""The workspaces of kvcache and speculative: one that does not begin on 16 bytes is refused on the host (the kernels
store whole vectors and 64-bit atomics into it), one that does is used wherever it lies."""
import pytest
import torch

from tests.test_serving_host import _cache, _decode

OFF = (1, 2, 4, 8, 12, 17)


def _evict(ws, n):
    import ctypes
    from tallax_amd import _lib
    return _lib.LIB.tallax_kv_evict(ctypes.byref(_cache()), 4, 4, 4, 4, 8, 0, 0, 8, 8, 8, ws, n, None)


def _verify(ws, n):
    from tallax_amd import _lib
    return _lib.LIB.tallax_verify(4, 16, 0, 2, 3, 100, None, 4, None, 0, 4, 4, 4, 4, ws, n, None)


def test_refuses_workspaces_off_16_bytes():
    from tallax_amd import _lib
    calls = (lambda ws, n: _decode(_cache(), scores=4, out_scores=4, ws=ws, nws=n), _evict, _verify)
    for call in calls:
        for off in OFF:
            assert call(4096 + off, 1 << 20) == _lib.INVALID_ARGUMENT, off
            assert b"16 bytes" in _lib.LIB.tallax_last_error()
        assert call(4096 + 16, 8) == _lib.WORKSPACE_TOO_SMALL
        assert call(None, 1 << 20) == _lib.WORKSPACE_TOO_SMALL


@pytest.mark.gpu
def test_workspaces_that_begin_inside_a_buffer(gpu):
    from tallax_amd import kvcache, speculative
    gen = torch.Generator(device=gpu)
    gen.manual_seed(30)
    k, v = (torch.randn((20, 2, 16, 64), generator=gen, device=gpu) for _ in range(2))
    table = torch.arange(20, dtype=torch.int32, device=gpu).reshape(2, 10)
    lens = torch.tensor([150, 100], dtype=torch.int32, device=gpu)
    q = torch.randn((2, 2, 4, 64), generator=gen, device=gpu)
    scores = torch.rand((2, 2, 160), generator=gen, device=gpu)
    positions = torch.arange(160, dtype=torch.int32, device=gpu).expand(2, 2, 160).contiguous()
    draft = torch.zeros((2, 3), dtype=torch.int32, device=gpu)
    logits = torch.randn((2, 4, 100), generator=gen, device=gpu)
    u, noise = torch.rand((2, 3), generator=gen, device=gpu), torch.rand((2, 100), generator=gen, device=gpu) + 0.1
    calls = (lambda **ws: kvcache.decode(q, k, v, table, lens, scores=scores, **ws),
             lambda **ws: speculative.verify(draft, logits, u, noise, **ws),
             lambda **ws: kvcache.evict(k, v, table, lens, scores, positions, lens, budget=32, **ws))
    buf = torch.empty(1 << 20, dtype=torch.uint8, device=gpu)
    for call in calls:
        want = call()
        for off in (16, 48):
            assert all(torch.equal(x, y) for x, y in zip(call(workspace=buf[off:]), want, strict=True))
        for off in OFF:
            with pytest.raises(ValueError, match="16 bytes"):
                call(workspace=buf[off:])
