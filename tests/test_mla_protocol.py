"""The hand-offs inside the MLA attention kernel (k_mla, moe_mla.cu) as a
protocol model: which accesses of tensor memory are ordered by what the kernel
waits for.  Order comes from a role's own program, from an mbarrier that is
waited for, from a commit (after every product issued before it), and on the
tensor pipe only between products of the same accumulator and shape.  What the
model takes from the kernel's text is which barriers the issuing warp waits
for in front of a tile's scores."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash_deepseek_b200", "csrc", "moe_mla.cu")


def body(name):
    """The text of a member function, from its head to the closing brace at the head's indentation."""
    text = open(SRC).read()
    m = re.search(r"^( *)__device__ [\w<>, ]*\b%s\(.*?^\1\}" % name, text, re.S | re.M)
    assert m, name
    return m.group(0)


def waits_before_scores():
    """Barriers that scores() waits for in front of the first product of a tile."""
    b = body("scores")
    loop = b.index("for (int p = 0; p < NV; p++)")
    return set(re.findall(r"(?:wait_phase|then_wait)\((?:[\w.]+, )?&c->(\w+)", b[:loop]))


def unordered(tiles, waits):
    """Pairs of conflicting accesses to score tiles and weights without an order, for one segment of `tiles` tiles.

    Issuing warp: scores(0), scores(1), output(0), scores(2), output(1), ...  Softmax: reads scores(i), writes the
    weights over half of them.  output(i) reads the weights."""
    edges = {}

    def edge(a, b):
        edges.setdefault(a, set()).add(b)

    issued, last = [], None

    def issue(mma):
        nonlocal last
        node = ("issue",) + mma
        if last:
            edge(last, node)
        edge(node, mma)
        for m in issued:   # the pipe's own order: the same accumulator and shape
            if m[0] == mma[0] and (m[0] == "output" or m[1] % 2 == mma[1] % 2):
                edge(m, mma)
        issued.append(mma)
        last = node

    def commit(bar):
        for m in issued:
            edge(m, bar)

    for i in range(tiles + 1):
        if i < tiles:
            if "pv_done" in waits and i >= 2:
                edge(("pv_done", i - 2), ("issue", "scores", i))
            issue(("scores", i))
            commit(("s_full", i))
            edge(("s_full", i), ("softmax", i))
            edge(("softmax", i), ("p_full", i))
            if i:
                edge(("softmax", i - 1), ("softmax", i))
        if i:
            edge(("p_full", i - 1), ("issue", "output", i - 1))
            issue(("output", i - 1))
            commit(("pv_done", i - 1))

    reach = {}

    def after(a):
        if a not in reach:
            reach[a] = set()
            for b in edges.get(a, ()):
                reach[a] |= {b} | after(b)
        return reach[a]

    touch = {p: [] for p in (0, 1)}   # per score tile: (node, writes)
    for i in range(tiles):
        touch[i % 2] += [(("scores", i), True), (("softmax", i), True), (("output", i), False)]
    bad = []
    for nodes in touch.values():
        for k, (a, wa) in enumerate(nodes):
            for b, wb in nodes[k + 1:]:
                if (wa or wb) and b not in after(a) and a not in after(b):
                    bad.append((a, b))
    return bad


@pytest.mark.parametrize("tiles", [1, 2, 3, 9])
def test_scores_wait_for_the_product_that_reads_their_place(tiles):
    """The weights of tile i lie over its scores; the scores of tile i + 2 go to the same columns."""
    assert unordered(tiles, waits_before_scores()) == []


def test_issue_order_alone_orders_no_products_of_different_accumulators():
    bad = unordered(5, {"full_b"})
    assert bad and all(a[0] == "output" and b == ("scores", a[1] + 2) for a, b in bad)


def test_numbers_between_warps_are_released_and_acquired():
    """`used` goes from the copying warp to the softmax warps outside any barrier: a plain store and load of it would
    order nothing else (the rows that are then overwritten)."""
    text = open(SRC).read()
    uses = [m.start() for m in re.finditer(r"c->used\b", text)]
    handed = [m.end() - len("c->used") for m in re.finditer(r"(?:store_release|load_acquire)\(&c->used", text)]
    first = text.index("c->used = 0")   # the start value, in front of the block's barrier
    assert len(handed) == 2 and sorted(handed + [first]) == uses
    assert "store_release" in body("forward") and "load_acquire" in body("copies_used")


def test_roles_meet_at_bounded_waits_only():
    """Every wait of a role gives up after a while and the role returns.  A block barrier among them would hold the
    other warps for good: only the kernel's entry and exit, which all threads reach, have one."""
    text = open(SRC).read()
    roles = text[text.index("struct MlaKernel"):text.index("k_mla(MoeKvDev kv")]
    assert not re.search(r"bar\.sync|barrier\.sync|__syncthreads|cluster_sync", roles)
    assert "clean" in body("meet") and body("clean").count("meet(u)") == 2


class Phases:
    """An mbarrier: completed phases, arrivals of the present one."""

    def __init__(self, count):
        self.count, self.done, self.here = count, 0, 0

    def arrive(self):
        self.here += 1
        if self.here == self.count:
            self.done, self.here = self.done + 1, 0

    def passed(self, parity):
        return self.done & 1 != parity


def softmax_warps(tiles, gives_up, rng, patience=200):
    """Four warps over tiles that need cleaning, in random order; gives_up: {warp: tile in whose wait it gives up}.
    Returns for each warp the tiles that it finished; raises if one never returns."""
    bar, met = Phases(4), [0] * 4
    done, asleep = [0] * 4, [0] * 4
    live = {0, 1, 2, 3}
    arrived = [False] * 4
    for _ in range(100000):
        if not live:
            return done
        w = rng.choice(sorted(live))
        if done[w] == tiles or (gives_up.get(w) == done[w] and met[w] == 2 * done[w] and not arrived[w]):
            live.discard(w)
        elif not arrived[w]:
            bar.arrive()
            arrived[w], asleep[w] = True, 0
        elif bar.passed(met[w] & 1):
            met[w], arrived[w] = met[w] + 1, False
            done[w] = met[w] // 2
        else:
            asleep[w] += 1
            if asleep[w] > patience:
                live.discard(w)
    raise AssertionError("a warp never returned")


def test_a_warp_that_gives_up_leaves_no_other_behind():
    import random
    for seed in range(40):
        rng = random.Random(seed)
        assert softmax_warps(6, {}, rng) == [6] * 4
        w, t = rng.randrange(4), rng.randrange(6)
        done = softmax_warps(6, {w: t}, rng)
        assert done[w] == t and all(t <= d <= t + 1 for d in done)
