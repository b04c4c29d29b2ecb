"""The ring of K and V stages of vbs_cu_attention_tree's tcgen05 kernel, as a
model on the host: its loader, the two issuers and the softmax streams under
random delays. A barrier's parity tells two neighbouring phases apart and no
more, and with an odd number of stages an issuer meets every other phase of
each; so every wait has to come when the phase before the awaited one is
known to be over. Stage counts and both ways of sharing rows are those that
tree_tc_launch can choose."""
import heapq
import random

import pytest


class Bar:
    """A barrier: phases completed, and who waits."""
    def __init__(self):
        self.done = 0

    def passes(self, phase):
        """try_wait.parity of `phase`: true when the phase that the barrier is in has the other parity."""
        return (self.done & 1) != (phase & 1)


def run(ns, two, tiles, seed, output_first):
    """Returns the items (2 i: keys of tile i, 2 i + 1: values) that were used
    before they had landed, in one random schedule."""
    rng = random.Random(seed)
    steps = 2 * tiles if two else tiles
    full, empty = [Bar() for _ in range(ns)], [Bar() for _ in range(ns)]
    s_bar, o_bar, p_bar = [Bar(), Bar()], [Bar(), Bar()], [Bar(), Bar()]
    landed, stale, events, now = set(), [], [], [0.0]
    slow = rng.choice([0.3, 3.0, 30.0])      # memory beside the products' 1

    def later(delay, act):
        heapq.heappush(events, (now[0] + delay * rng.uniform(0.2, 3), rng.random(), act))

    def land(item):
        landed.add(item)
        full[item % ns].done += 1

    def use(item):
        if item not in landed:
            stale.append(item)

    def loader():
        for item in range(2 * tiles):
            if item >= ns:
                yield empty[item % ns], item // ns - 1
            later(slow, lambda item=item: land(item))

    order = {"qk": 0.0, "pv": 0.0}           # products of one issuer complete in turn

    def product(kind, acts):
        order[kind] = max(order[kind], now[0]) + rng.uniform(0.2, 2)

        def finish():
            for b in acts:
                b.done += 1
        heapq.heappush(events, (order[kind], rng.random(), finish))

    def qk():
        for n in range(steps):
            w, i = n & 1, n >> 1 if two else n
            waits = [(full[2 * i % ns], 2 * i // ns)]
            if n >= 2:
                waits.insert(0 if output_first else 1, (o_bar[w], n // 2 - 1))
            for x in waits:
                yield x
            use(2 * i)
            product("qk", [s_bar[w]] + ([empty[2 * i % ns]] if not two or w else []))

    def pv():
        for n in range(steps):
            w, i = n & 1, n >> 1 if two else n
            yield full[(2 * i + 1) % ns], (2 * i + 1) // ns
            yield p_bar[w], n >> 1
            use(2 * i + 1)
            product("pv", [o_bar[w]] + ([empty[(2 * i + 1) % ns]] if not two or w else []))

    def softmax(w):
        for n in range(w, steps, 2):
            yield s_bar[w], n >> 1
            if rng.random() < 0.3:           # a masked tile: its values are looked at
                i = n >> 1 if two else n
                yield full[(2 * i + 1) % ns], (2 * i + 1) // ns
                use(2 * i + 1)
            later(1.0, lambda: setattr(p_bar[w], "done", p_bar[w].done + 1))
            yield None, 0                    # until its weights are out
            yield p_bar[w], n >> 1

    waiting = []                             # (role, barrier, phase)
    for role in (loader(), qk(), pv(), softmax(0), softmax(1)):
        waiting.append([role, None, 0])
    while True:
        moved = True
        while moved:
            moved = False
            rng.shuffle(waiting)
            for x in list(waiting):
                if x[1] is None or x[1].passes(x[2]):
                    moved = True
                    try:
                        x[1], x[2] = next(x[0])
                    except StopIteration:
                        waiting.remove(x)
        if stale or not events:
            assert stale or not waiting, "stuck"
            return stale
        now[0], _, act = heapq.heappop(events)
        act()


RINGS = [(ns, two) for ns in (3, 4, 5, 6, 8) for two in (False, True)]


@pytest.mark.parametrize("ns,two", RINGS)
def test_no_stage_is_used_before_it_has_landed(ns, two):
    for seed in range(1500):
        assert not run(ns, two, 12, seed, output_first=True)


def test_three_stages_want_the_last_product_first():
    """Waiting for the stage and then for the product that used it last lets
    three stages pass a whole phase early, and no others."""
    found = {(ns, two): sum(bool(run(ns, two, 12, seed, output_first=False)) for seed in range(400)) for ns, two in RINGS}
    assert found[(3, False)] > 0
    assert not any(n for ring, n in found.items() if ring != (3, False))
