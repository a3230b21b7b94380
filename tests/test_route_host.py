"""Host checks of experts.route: strides of rows."""
from tests.test_layer_host import _route


def test_strides_that_no_memory_holds_are_refused():
    from tallax_amd import _lib
    assert _route(stride=(1 << 37) + 1) == _lib.UNSUPPORTED and b"2^37" in _lib.LIB.tallax_last_error()
    assert _route(stride=1 << 37, tokens=0, logits=None) == _lib.OK
    assert _route(stride=1 << 37, logits=None) == _lib.INVALID_ARGUMENT
