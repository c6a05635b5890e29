"""Lists of copied pages around the length at which their check moves to a kernel of its own, and pages of whole blocks that
are no power of two."""
import pytest
import torch

from ako4x_b200 import kv_pages, paged_decode
from test_paged_decode_gpu import TYPES, make, run_check

pytestmark = pytest.mark.gpu
PAGES = 6000


def lists(n, seed):
    """n pairs of distinct pages, pages 0 to 9 in none of them."""
    order = 10 + torch.randperm(PAGES - 10, generator=torch.Generator().manual_seed(seed)).int()
    return order[:n].clone(), order[n:2 * n].clone()


def copy(cache, src, dst):
    return kv_pages.copy([cache], src.cuda(), dst.cuda()).tolist()


CONFLICTS = {  # entry, entry: what the second one is given
    "the same destination": lambda s, d, i, j: d.__setitem__(j, int(d[i])),
    "a destination that is a source": lambda s, d, i, j: d.__setitem__(j, int(s[i])),
    "a source that is a destination": lambda s, d, i, j: s.__setitem__(j, int(d[i])),
    "two pages swapped": lambda s, d, i, j: (s.__setitem__(j, int(d[i])), d.__setitem__(j, int(s[i]))),
    "the same pair": lambda s, d, i, j: (s.__setitem__(j, int(s[i])), d.__setitem__(j, int(d[i])))}


@pytest.mark.parametrize("what", list(CONFLICTS))
@pytest.mark.parametrize("n", [2, 255, 256, 257, 258, 1024, 1025, 2900])
def test_a_list_that_depends_on_the_order_is_refused(built_lib, n, what):
    cache = torch.randn(PAGES, 5, device="cuda")
    before = cache.clone()
    for i, j in {(0, n - 1), (n - 1, 0), (n // 2 - 1, n // 2), (min(1023, n - 1), n - 1 if n < 1025 else 1024)}:
        if i == j:
            continue
        src, dst = lists(n, n + i)
        CONFLICTS[what](src, dst, i, j)
        assert copy(cache, src, dst) == [False] and torch.equal(cache, before)
        # the next one has the same workspace, with the numbers of this one in it
        src, dst = lists(n, n + i)
        assert copy(cache, src, dst) == [True]
        want = before.clone()
        want[dst.long()] = before[src.long()]
        assert torch.equal(cache, want)
        cache.copy_(before)


@pytest.mark.parametrize("n", [10, 256, 300, 1500])
def test_pairs_that_do_not_count_make_no_conflict(built_lib, n):
    """Out of range or from a page to itself: such an entry is neither a destination nor a source."""
    cache = torch.randn(PAGES, 5, device="cuda")
    before = cache.clone()
    src, dst = lists(n, n)
    src[1], dst[1] = -1, dst[0]
    src[2], dst[2] = dst[0], PAGES
    src[3], dst[3] = dst[4], dst[4]
    src[5], dst[5] = src[6], src[6]
    src[n - 1], dst[n - 1] = 2 ** 31 - 1, src[0]
    assert copy(cache, src, dst) == [True]
    want = before.clone()
    real = [i for i in range(n) if i not in (1, 2, 3, 5, n - 1)]
    want[dst[real].long()] = before[src[real].long()]
    assert torch.equal(cache, want)
    src[0], dst[7] = 4, 4                                    # and one that counts does
    assert copy(cache, src, dst) == [False]
    assert torch.equal(cache, want)


def test_lists_in_turn(built_lib):
    """Long lists whose destinations are the last one's sources, over one workspace."""
    cache = torch.arange(PAGES, dtype=torch.float32, device="cuda").view(PAGES, 1).repeat(1, 3)
    want = cache.clone()
    for step in range(6):
        src, dst = lists(2000 + step, 77)
        if step % 2:
            src, dst = dst, src
        if step == 3:
            dst[5] = dst[6]
        ok = copy(cache, src, dst)
        assert ok == [step != 3]
        if ok[0]:
            want[dst.long()] = want[src.long()].clone()
        assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("ps", [48, 80, 112, 144])
@pytest.mark.parametrize("lens,hk,group,dim,window", [([1, 47, 48, 49, 500, 0, 143], 2, 4, 128, 0), ([3000, 95], 1, 7, 64, 0), ([700, 81], 2, 5, 256, 130)])
def test_pages_of_three_blocks_and_more(built_lib, lens, hk, group, dim, window, ps, dtype, kind):
    run_check(make(lens, hk, group, dim, dtype, kind, ps, seed=ps + dim), **({"window": window} if window else {}))


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_a_window_without_an_end(built_lib, dtype, kind):
    a = make([1500, 17], 2, 4, 64, dtype, kind, 16, seed=31)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in a.items()}
    o, lse = paged_decode.run(**d)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1):
        o2, lse2 = paged_decode.run(**d, window=window)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
