"""The life of requests that continue others, on the CPU: the cache's own
bookkeeping, nothing is launched."""

import pytest
import torch

import sunshape_mlx_amd as S
from sunshape_mlx_amd import _hip, paged


@pytest.fixture(autouse=True)
def nothing_runs(monkeypatch):
    """CPU tensors pass for GPU ones, and launches do nothing."""
    monkeypatch.setattr(_hip, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "_launch", lambda *a: None)
    monkeypatch.setattr(paged, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(paged, "_scored_workspace_bytes", lambda *a: 0)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def forked():
    """Requests 1 and 2 continue 0, 3 is by itself."""
    c = S.PagedKVCache(n_requests=4, n_kv_heads=2, max_tokens=64, device="cpu")
    c.step([20, 0, 0, 4])
    c.share([1, 2], 0)
    c.step([0, 5, 3, 1])
    return c


def known(c):
    """What the cache knows of its requests."""
    return c._host, c._bound, c._version, c.plan, c.shared, list(c._parent), c.parents.tolist(), c._prefixes


def parents(c, *want):
    assert c._parent == list(want) and c.parents.tolist() == list(want) and c._prefixes == set(want) - {-1}


def test_a_child_that_ends_in_a_step_continues_nothing():
    c = forked()
    c.step([0, -5, 0, 0])
    parents(c, -1, -1, 0, -1)
    c.step([0, 7, 1, 0])  # another request in its place
    parents(c, -1, -1, 0, -1)
    c.step([0, 0, -4, 0])
    parents(c, -1, -1, -1, -1)
    c.step([0, 1, 1, 1])
    assert c.shared is None


def test_a_child_that_keeps_tokens_stays():
    c = forked()
    c.step([0, -4, 1, 0])
    parents(c, -1, 0, 0, -1)


@pytest.mark.parametrize("adds", [[-20, 0, 0, 0], [-1, 0, 0, 0], [-20, -5, 0, 0], [-20, -5, -2, 0], [-1, -5, 7, 0]])
def test_a_prefix_keeps_its_tokens_while_it_is_continued(adds):
    c = forked()
    before = known(c)
    with pytest.raises(ValueError, match="others continue"):
        c.step(adds)
    assert known(c) == before


@pytest.mark.parametrize("adds", [[-20, -5, -3, 0], [-1, -5, -3, 2]])
def test_a_prefix_gives_tokens_back_with_all_that_continue_it(adds):
    c = forked()
    c.step(adds)
    parents(c, -1, -1, -1, -1)


def test_a_prefix_whose_children_hold_nothing_yet_is_kept_too():
    c = forked()
    c.share([3], None)  # (continues nothing: nothing to undo)
    c.step([0, -5, -3, -5])
    c.share([3], 0)
    with pytest.raises(ValueError, match="others continue"):
        c.step([-20, 0, 0, 0])
    c.release([0, 3])
    parents(c, -1, -1, -1, -1)
    assert c._host == [0, 0, 0, 0]


def test_a_prefix_may_grow():
    c = forked()
    c.step([6, 1, 1, 0])
    parents(c, -1, 0, 0, -1)


def test_what_holds_tokens_is_not_detached():
    c = forked()
    before = known(c)
    for requests in ([1], [1, 2], [3, 2]):
        with pytest.raises(ValueError, match="behind"):
            c.share(requests, None)
        assert known(c) == before
    c.trim(3)
    c.share([2], None)
    parents(c, -1, 0, -1, -1)


def test_a_child_trimmed_to_nothing_goes_on_behind_its_prefix():
    c = forked()
    c.trim(9)
    assert c._host == [20, 0, 0, 0]
    parents(c, -1, 0, 0, -1)
    c.step([0, 2, 0, 0])
    assert c.shared is not None
    c.release([1, 2])
    parents(c, -1, -1, -1, -1)


def test_lengths_that_only_the_gpu_knows():
    """A list takes nothing from a prefix, as its children may hold tokens; release ends both."""
    c = forked()
    c.step(ints(0, 1, 1, 0), 2)
    for adds in ([-1, 0, 0, 0], [-20, -6, -4, 0]):
        before = known(c)
        with pytest.raises(ValueError, match="release"):
            c.step(adds)
        assert known(c) == before
    c.release([1])
    parents(c, -1, -1, 0, -1)
    with pytest.raises(ValueError, match="others continue"):
        c.release([0])
    c.trim(1)
    parents(c, -1, -1, 0, -1)
    c.release([0, 2])
    parents(c, -1, -1, -1, -1)


def test_a_step_that_fails_ends_nobody(monkeypatch):
    c = forked()
    before = known(c)

    def fail(*a):
        raise RuntimeError("no launch")

    monkeypatch.setattr(paged, "_launch", fail)
    for call in (lambda: c.step([0, -5, 0, 0]), lambda: c.release([1])):
        with pytest.raises(RuntimeError, match="no launch"):
            call()
        assert known(c) == before


# ------------------------------------------------- what attend is told


class Once(list):
    """A list that is not gone through again."""

    def __iter__(self):
        raise AssertionError("every attend goes through all requests")


@pytest.mark.parametrize("adds,longest", [([0, 1, 1, 1], 7), ([512, 1, 0, 0], 532), ([9, 0, 0, 0], 29),
                                          ([0, 0, 0, 200], 205), ([0, 0, 0, 0], 1)])
def test_attend_is_sized_for_the_requests_that_add_tokens(monkeypatch, adds, longest):
    """A prefix that goes on among them; no attend goes through the requests, of which there
    may be thousands."""
    c = S.PagedKVCache(n_requests=4, n_kv_heads=2, max_tokens=1000, device="cpu")
    c.step([20, 0, 0, 4])
    c.share([1, 2], 0)
    c.step([0, 6, 3, 1])
    plan = c.step(adds)
    told = []
    monkeypatch.setattr(paged, "_scored_workspace_bytes", lambda *a: told.append(a[6]) or 0)
    c._host = Once(c._host)
    n = sum(adds)
    c.attend(torch.zeros((n, 4, 128), dtype=torch.float16), 0.1)
    assert c.shared is not None and plan.slots.shape[0] == n
    assert told == ([longest] if n else [])


def test_attend_without_sharing_is_sized_for_the_longest(monkeypatch):
    c = S.PagedKVCache(n_requests=3, n_kv_heads=2, max_tokens=1000, device="cpu")
    told = []
    monkeypatch.setattr(paged, "_workspace_bytes", lambda *a: told.append(a[6]) or 0)
    q = torch.zeros((1, 4, 128), dtype=torch.float16)
    for adds in ([300, 2, 0], [0, 1, 0], ints(1, 0, 0)):
        c.step(adds, 400)
        c.attend(q.expand(400, 4, 128), 0.1)
    assert told == [300, 300, 700]
