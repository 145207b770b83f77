"""CPU: PeerWatch where a rank leaves between its beat of a step and the others'
look at it: it has arrived at that step, and is missed at the next."""
import pytest

from flash_deepseek_b200 import ep


class Store(dict):
    """A key-value store as torch.distributed's: values come back as bytes."""

    def set(self, k, v):
        self[k] = v.encode()

    def get(self, k):
        return self[k]

    def check(self, keys):
        return all(k in self for k in keys)


def ranks(n=2, timeout=0.05):
    store = Store()
    return [ep.PeerWatch(store, r, n, timeout=timeout) for r in range(n)]


def test_a_rank_that_left_after_its_beat_has_arrived():
    a, b = ranks()
    for w in (a, b):
        w.beat(2)
    b.wait(2)
    b.leave()
    a.wait(2)
    a.beat(3)
    with pytest.raises(ep.PeerLost) as e:
        a.wait(3)
    assert e.value.ranks == [1] and e.value.left == [1]


def test_a_rank_that_left_before_its_first_beat_is_lost_at_once():
    a, b = ranks(timeout=60.0)
    b.leave()
    a.beat(0)
    with pytest.raises(ep.PeerLost) as e:
        a.wait(0)
    assert e.value.left == [1]


def test_left_and_late_ranks_are_told_apart():
    a, b, c = ranks(3)
    for w in (a, b):
        w.beat(0)
    b.leave()
    with pytest.raises(ep.PeerLost) as e:
        a.wait(0)
    assert e.value.ranks == [2] and e.value.left == []
    c.beat(0)
    a.wait(0)
    c.beat(1)
    with pytest.raises(ep.PeerLost) as e:
        a.wait(1)
    assert e.value.ranks == [1] and e.value.left == [1]
