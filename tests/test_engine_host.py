"""Host-side decisions of the batched engine, on a host without a GPU: the launches are stood in for."""

from __future__ import annotations

import random
import time

import pytest
import torch

from tests.conftest import submodule


def bare_engine(max_seqs=8):
    """An engine without a model or device buffers."""
    engine = submodule("engine")
    eng = object.__new__(engine.B200SpeculativeEngine)
    eng.max_seqs = max_seqs
    return eng


# ------------------------------------------------------------------------------ samples of one prompt
class _Status:
    def __init__(self, error):
        self.error = error

    def raise_on_device_error(self):
        if self.error:
            raise RuntimeError(self.error)


def samples_engine(error, steps):
    """``steps[i]``: the tokens that step i yields for each sample (the last one repeats)."""
    engine = submodule("engine")
    eng = bare_engine()
    eng.model = _Status(error)
    eng.calls, eng.released = 0, []

    def step(slots):
        eng.calls += 1
        assert eng.calls < 50, "the same step again and again"
        row = steps[min(eng.calls, len(steps)) - 1]
        return engine.StepResult(tokens={s: list(row[s]) for s in slots}, finish={s: None for s in slots})

    eng.add_request = lambda *a, **kw: 0
    eng.prefill = lambda slots, **kw: engine.StepResult(tokens={s: [7] for s in slots}, finish={s: None for s in slots})
    eng.fork = lambda slot, n, **kw: list(range(1, n + 1))
    eng.step = step
    eng.release = eng.released.extend
    return eng


@pytest.mark.parametrize("steps,calls", [
    ([[(), (), ()]], 1),                          # the first step's blocks do not fit
    ([[(1,), (2, 3), (4,)], [(), (), ()]], 2),    # a later step's
    ([[(1,), (), (2,)]], 1),                      # one sample cannot go on
])
def test_samples_whose_step_yields_no_token_end_with_the_device_error(steps, calls) -> None:
    eng = samples_engine("out of KV blocks", steps)
    with pytest.raises(RuntimeError, match="out of KV blocks"):
        eng.generate_samples([1, 2, 3], 3, 40)
    assert eng.calls == calls and sorted(eng.released) == [0, 1, 2]


def test_samples_whose_step_yields_no_token_end_without_a_device_error_too() -> None:
    eng = samples_engine(None, [[(), (), ()]])
    with pytest.raises(RuntimeError, match="no token"):
        eng.generate_samples([1, 2, 3], 3, 40)
    assert sorted(eng.released) == [0, 1, 2]


# ------------------------------------------------------------------------------ who shares which blocks
def groups_of(slots, prefix_of=(), fork_of=(), max_seqs=16):
    """(blocks, slots) of the groups that ``_fill_groups`` makes, largest first; ``prefix_of`` /
    ``fork_of``: {slot: (holder / source, shared blocks)}."""
    eng = bare_engine(max_seqs)
    prefix_of, fork_of = dict(prefix_of), dict(fork_of)
    eng._prefix_of = {s: h for s, (h, _) in prefix_of.items()}
    eng._shared_count = {s: n for s, (_, n) in prefix_of.items()}
    eng._fork_of = {s: h for s, (h, _) in fork_of.items()}
    eng._fork_blocks = {s: n for s, (_, n) in fork_of.items()}
    host = torch.zeros((2, max_seqs), dtype=torch.int32)
    eng._fill_groups(slots, host)
    entry_group, prefix_blocks = host.tolist()
    assert all(g == -1 for g in entry_group[len(slots):])
    groups = {}
    for s, g in zip(slots, entry_group):
        if g >= 0:
            groups.setdefault(g, []).append(s)
    assert all(prefix_blocks[g] > 0 and len(members) > 1 for g, members in groups.items())
    return sorted(((prefix_blocks[g], members) for g, members in groups.items()), reverse=True)


def test_users_of_one_prefix_are_a_group() -> None:
    users = {s: (9, 128) for s in range(8)}
    assert groups_of(list(range(8)), users) == [(128, list(range(8)))]
    assert groups_of([3], users) == [] and groups_of([10, 11], users) == []
    # the holder's own entry is one of them; two holders' users are two groups
    assert groups_of([9, 0, 1], users) == [(128, [9, 0, 1])]
    two = {0: (9, 8), 1: (9, 8), 2: (10, 5), 3: (10, 5), 4: (11, 7)}
    assert groups_of([0, 2, 1, 3, 4], two) == [(8, [0, 1]), (5, [2, 3])]


@pytest.mark.parametrize("short", [0, 1])
def test_a_short_fork_does_not_cut_the_others_prefix(short) -> None:
    users = {s: (9, 128) for s in range(7)}
    assert groups_of(list(range(8)), {**users, 7: (9, short)}, {7: (0, short)}) == [(128, list(range(7)))]


def test_a_member_that_shares_most_blocks_stays() -> None:
    """Reading 100 blocks once for eight saves more than 128 once for seven."""
    users = {s: (9, 128) for s in range(7)}
    assert groups_of(list(range(8)), {**users, 7: (9, 100)}) == [(128, list(range(7)))]  # 6 x 128 > 7 x 100
    assert groups_of(list(range(8)), {**users, 7: (9, 120)}) == [(120, list(range(8)))]  # 7 x 120 > 6 x 128


def test_short_members_share_among_themselves() -> None:
    users = {**{s: (9, 128) for s in range(6)}, 6: (9, 2), 7: (9, 2), 8: (9, 1)}
    assert groups_of(list(range(9)), users) == [(128, list(range(6))), (2, [6, 7])]


def test_forks_share_what_their_source_holds_beyond_its_prefix() -> None:
    users = {0: (9, 4), 1: (9, 4), 2: (9, 4), 3: (9, 4), 4: (9, 4), 5: (9, 4)}
    forks = {1: (0, 200), 2: (0, 200), 3: (0, 200)}
    assert groups_of([1, 2, 3], users, forks) == [(200, [1, 2, 3])]
    assert groups_of([0, 1, 2, 3, 4, 5], users, forks) == [(200, [0, 1, 2, 3]), (4, [4, 5])]


def test_nested_forks_share_with_their_own_source() -> None:
    # 1 from 0 at 3 blocks; 2 and 3 from 1, which had run on to 50; 4 from 2 at 60
    forks = {1: (0, 3), 2: (1, 50), 3: (1, 50), 4: (2, 60)}
    assert groups_of([0, 1, 2, 3, 4], (), forks) == [(50, [1, 2, 3, 4])]
    assert groups_of([0, 2], (), forks) == [(3, [0, 2])]      # what the path between them shares
    assert groups_of([3, 4], (), forks) == [(50, [3, 4])]
    assert groups_of([0, 5, 6], (), {5: (0, 0), 6: (0, 0)}) == []


def test_many_entries_are_grouped_in_little_time() -> None:
    n = 256
    pairs = {s: (1000 + s // 2, 1 + s % 7) for s in range(n)}
    start = time.perf_counter()
    groups = groups_of(list(range(n)), pairs, max_seqs=n)
    chain = groups_of(list(range(n)), (), {s: (s - 1, s) for s in range(1, n)}, max_seqs=n)
    assert time.perf_counter() - start < 5.0
    assert len(groups) == n // 2
    assert sum(len(m) for _, m in chain) > n // 2


@pytest.mark.parametrize("seed", range(30))
def test_groups_read_blocks_that_all_members_have(seed) -> None:
    """Random trees of prefixes and forks, their tables written out: a group's first blocks are the same ids."""
    rng = random.Random(seed)
    tables, prefix_of, fork_of, ids = {}, {}, {}, iter(range(1 << 20))
    fresh = lambda n: [next(ids) for _ in range(n)]  # noqa: E731
    for holder in (14, 15):
        tables[holder] = fresh(rng.randint(1, 9))
    for s in range(14):
        kind = rng.randrange(3)
        if kind == 0:
            tables[s] = fresh(rng.randint(1, 12))
        elif kind == 1:
            holder = rng.choice((14, 15))
            n = rng.randint(0, len(tables[holder]))
            prefix_of[s] = (holder, n)
            tables[s] = tables[holder][:n] + fresh(rng.randint(1, 6))
        else:
            source = rng.choice([x for x in range(s)] + [14, 15])
            n = rng.randint(0, len(tables[source]))
            fork_of[s] = (source, n)
            holder = source if source >= 14 else prefix_of.get(source, (None, 0))[0]
            if holder is not None:
                prefix_of[s] = (holder, min(n, len(tables[holder]) if source >= 14 else prefix_of[source][1]))
            tables[s] = tables[source][:n] + fresh(rng.randint(1, 6))
    slots = rng.sample(range(16), rng.randint(2, 16))
    groups = groups_of(slots, prefix_of, fork_of)
    seen = [s for _, members in groups for s in members]
    assert len(seen) == len(set(seen))
    for blocks, members in groups:
        assert all(tables[s][:blocks] == tables[members[0]][:blocks] and len(tables[s]) >= blocks for s in members)
