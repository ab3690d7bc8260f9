"""Ids of no page that are any number, in forks of each launch form."""
import pytest
import torch

from prompt_util import ints
from test_gpu_paged_pages import fork, held

pytestmark = pytest.mark.gpu

LOWEST = -2 ** 31


@pytest.mark.parametrize("forks", [3, 100, 1100])
def test_the_lowest_number_as_no_page(ctx, forks):
    """Where src's last page is none, so is dst's, whatever a former request left in its row; a list may hold such a number, too."""
    page = 4
    lens, table, shares, free, head = held(forks, [9, 6, 12, 3], forks, page, cols=4, extra=forks)
    table[0, 2], table[1, 0], table[1, 1] = LOWEST, LOWEST, -1
    table[4:] = 1  # names of former requests
    free[head + 1] = LOWEST
    src = torch.arange(forks, dtype=torch.int32) % 4
    got = fork(ctx, src, 4 + torch.arange(forks, dtype=torch.int32), lens, table, shares, free, head, page, f"{forks} forks")
    assert int(got["block_table"][4, 2]) == LOWEST
    # the same requests as sources once more
    some = ints([5, 4, 7])
    lens2, table2 = got["lens"], got["block_table"]
    lens2[0] = 0
    table2[0] = 1
    fork(ctx, some, ints([0, 0, 1]), lens2, table2, got["shares"], free, int(got["counts"][0]), page, "again")
