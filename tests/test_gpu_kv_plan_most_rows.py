"""The plan of a step with as many rows as a call takes, 2^31 - 1: the row counters' last steps pass 32 signed bits."""
import pytest
import torch

import periodicdent42_b200 as bsk

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("first,second", [(3, 5), (MOST - 40, 33), (MOST - 1000, 1000)])
def test_most_rows(no_device_error, cuda_dev, first, second):
    """A short step and padding, and requests that reach into the last 512 rows and to the last one."""
    page = 1024
    if torch.cuda.mem_get_info()[0] < 60 * 2 ** 30:
        pytest.skip("60 GB needed")
    i32 = dict(dtype=torch.int32, device=cuda_dev)
    width = -(-MOST // page)
    table = torch.zeros(2, width, **i32)
    pages = [-(-n // page) for n in (first, second)]
    free = torch.arange(sum(pages), **i32)
    slots, places, cu, lens, left = bsk.kv_cache_plan(torch.zeros(2, **i32), torch.tensor([first, second], **i32), table, free,
                                                      torch.tensor([sum(pages)], **i32), page, MOST)
    assert cu.tolist() == [0, first, first + second] and lens.tolist() == [first, second] and left.item() == 0
    assert slots.shape == places.shape == (MOST,)
    used, a = first + second, 0
    assert table[0, :pages[0]].flip(0).equal(free[pages[1]:]) and table[1, :pages[1]].flip(0).equal(free[:pages[1]])
    for i, n in enumerate((first, second)):
        for b in range(0, n, 2 ** 28):
            e = min(b + 2 ** 28, n)
            at = torch.arange(b, e, device=cuda_dev)
            assert torch.equal(places[a + b:a + e].long(), at)
            at.copy_(table[i][at // page].long() * page + at % page)
            assert torch.equal(slots[a + b:a + e], at)
        a += n
    for b in range(used, MOST, 2 ** 28):
        e = min(b + 2 ** 28, MOST)
        assert (slots[b:e] == -1).all() and (places[b:e] == 0).all()
