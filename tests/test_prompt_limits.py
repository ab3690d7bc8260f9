"""Sizes at which the prompt operators refuse a call, without a GPU: refusals that
come before anything of the context or of a buffer is looked at.  A call whose sizes
are taken goes on to its buffers, which are missing here."""
import ctypes

import pytest

from mlx_amd import abi
from test_prompt_abi import table  # noqa: F401

PAGES = [("op_paged_fork", abi.PagedForkArgs), ("op_paged_release", abi.PagedReleaseArgs), ("op_paged_compact", abi.PagedCompactArgs)]
UNSEEN = ctypes.create_string_buffer(1 << 16)  # a context that no refusal reads


def call(table, op, args):  # noqa: F811
    return getattr(table, op)(ctypes.addressof(UNSEEN), args)


@pytest.mark.parametrize("op,record", PAGES)
@pytest.mark.parametrize("over,taken", [(dict(), True), (dict(max_pages=2 ** 31 - 1 - 256), True), (dict(max_pages=2 ** 31 - 256), False),
                                        (dict(max_pages=2 ** 31 - 2), False), (dict(max_pages=2 ** 31 - 1), False),
                                        (dict(requests=2, max_pages=2 ** 30 - 1), True), (dict(requests=2, max_pages=2 ** 30), False),
                                        (dict(max_pages=2 ** 27, page_size=16), False), (dict(num_pages=1 << 22), True),
                                        (dict(num_pages=(1 << 22) + 1), False)])
def test_pages_in_use(table, op, record, over, taken):  # noqa: F811
    """Tables whose last columns' places, looked at 256 at a time, pass 31 bits are refused."""
    args = record(**{**dict(requests=1, max_pages=4, page_size=1, num_pages=8, free_count=8), **over})
    assert call(table, op, args) == (abi.ERR_INVALID_ARGUMENT if taken else abi.ERR_NOT_SUPPORTED)
