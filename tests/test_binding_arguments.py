"""Arguments that the Python binding refuses itself, before the library is called
(no GPU needed)."""
import ctypes

import numpy as np
import pytest


@pytest.mark.parametrize("stream", [0, ctypes.c_void_p(None), ctypes.c_void_p(0)])
def test_the_default_stream_is_refused(q, stream):
    """0 is the default stream's handle, and no stream of its own would be a
    surprise to who passes it."""
    with pytest.raises(ValueError, match="default stream"):
        q.Context(0, stream)
    with pytest.raises(ValueError, match="default stream"):
        q.Context(0, stream=stream)


@pytest.mark.parametrize("pages", [[1.5], [2.0 ** 32], np.array([2 ** 32 + 1]), np.array([-2 ** 32]), np.array([2 ** 63], np.uint64),
                                   [float("nan")]])
def test_page_numbers_that_are_no_int32(q, pages):
    """A number that would be cut to another page's is refused, wherever it stands."""
    for src, dst, tokens in [(pages, [1], None), ([1], pages, None), ([1], [2], pages)]:
        with pytest.raises(ValueError, match="whole numbers"):
            q.cache_copy_pages(None, None, None, 1, 0, 8, 4, 8, src, dst, tokens)
    with pytest.raises(ValueError, match="whole numbers"):
        q.Runtime.page_fork(None, pages, 4)


@pytest.mark.parametrize("pages", [[3], (3,), np.array([3]), np.array([3], np.uint8), np.array([3.0])])
def test_page_numbers_of_other_types(q, pages):
    got = q._page_list(pages)
    assert got.dtype == np.int32 and got.tolist() == [3] and q._page_list([]).size == 0
