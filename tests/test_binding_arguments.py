"""Arguments that the Python binding refuses itself, before the library is called
(no GPU needed)."""
import ctypes

import pytest


@pytest.mark.parametrize("stream", [0, ctypes.c_void_p(None), ctypes.c_void_p(0)])
def test_the_default_stream_is_refused(q, stream):
    """0 is the default stream's handle, and no stream of its own would be a
    surprise to who passes it."""
    with pytest.raises(ValueError, match="default stream"):
        q.Context(0, stream)
    with pytest.raises(ValueError, match="default stream"):
        q.Context(0, stream=stream)
