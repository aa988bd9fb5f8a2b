"""The operators for many samples of one prompt in the engine, together: shared prefixes and forks
whose steps read the shared blocks once (``shared_prefix_attention``), drawn with ``ops.sample_logits``
and moved by compaction."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.conftest import submodule

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def make(pkg, cuda_device):
    submodule("build").build()
    weights = pkg.make_weights(pkg.SMALL_TEST, seed=0)
    models = {}

    def engine(kv_int8=False, shared=True, max_seqs=8, **kw):
        if kv_int8 not in models:
            models[kv_int8] = submodule("model").B200Model(
                pkg.SMALL_TEST, weights, num_slots=192 * 16, device=cuda_device, max_positions=640, max_rows=512,
                max_seqs=16, kv_int8=kv_int8)
        return submodule("engine").B200SpeculativeEngine(models[kv_int8], k=4, max_ngram=3, max_seqs=max_seqs,
                                                         max_model_len=512, num_blocks=192, sampling=True,
                                                         shared_prefix_attention=shared, **kw)

    return engine


def prompts_with_prefix(pkg, length, n):
    v = pkg.SMALL_TEST.vocab_size
    prefix = pkg.make_prompt(v, length, 3, False)
    return [prefix + pkg.make_prompt(v, 5 + 3 * i, 50 + i, i % 2 == 0) for i in range(n)]


@pytest.mark.parametrize("kv_int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "eager"])
def test_shared_prefix_requests_take_the_same_tokens(pkg, make, kv_int8, graphs) -> None:
    """Greedy requests on one prefix (more than fit at once, so slots change hands under captured steps)."""
    prompts = prompts_with_prefix(pkg, 200, 11)
    want = make(kv_int8, shared=False).generate(prompts, 20, shared_prefix=200)
    eng = make(kv_int8, cuda_graphs=graphs)
    assert eng.generate(prompts, 20, shared_prefix=200) == want
    assert eng.state.num_free_blocks() == 192
    # and the same engine without any sharing
    assert eng.generate(prompts[:5], 12) == make(kv_int8, shared=False).generate(prompts[:5], 12)


def test_two_prefixes_forks_and_loners_in_one_batch(pkg, make) -> None:
    a, b = prompts_with_prefix(pkg, 150, 2), [p[70:] for p in prompts_with_prefix(pkg, 150, 4)[2:]]
    lone = pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 40, 9, False)
    outs = {}
    for shared in (False, True):
        eng = make(shared=shared)
        pa, pb = eng.add_prefix(a[0][:150]), eng.add_prefix(b[0][:80])
        slots = eng.add_requests(a, [24, 24], ignore_eos=True, prefix=pa)
        slots += eng.add_requests(b, [24, 24], ignore_eos=True, prefix=pb)
        slots.append(eng.add_request(lone, 24, ignore_eos=True))
        res = eng.prefill(slots)
        out = {s: list(res.tokens[s]) for s in slots}
        for _ in range(2):
            for s, t in eng.step(slots).tokens.items():
                out[s] += t
        fork, = eng.fork(slots[-1])
        slots.append(fork)
        out[fork] = list(out[slots[-2]])
        eng.compact()
        live = list(slots)
        while live:
            res = eng.step(live)
            for s in list(live):
                out[s] += res.tokens[s]
                if res.finish[s] is not None:
                    live.remove(s)
        outs[shared] = [out[s] for s in slots]
        eng.release(slots)
        eng.drop_prefix(pa)
        eng.drop_prefix(pb)
        assert eng.state.num_free_blocks() == 192
    assert outs[True] == outs[False]
    assert outs[True][-1] == outs[True][-2]


def test_a_fork_in_a_reused_slot_gets_its_own_group(pkg, make) -> None:
    """The step's slot list stays the same while the fork in it is another one: the groups follow."""
    eng = make(max_seqs=2)
    prompt = prompts_with_prefix(pkg, 100, 1)[0]
    want = make(shared=False).generate([prompt], 60)[0]
    s = eng.add_request(prompt, 60, ignore_eos=True)
    out = list(eng.prefill([s]).tokens[s])
    for _ in range(3):
        fork, = eng.fork(s)
        theirs = list(out)
        for _ in range(4):
            res = eng.step(sorted([s, fork]))
            out += res.tokens[s]
            theirs += res.tokens[fork]
        assert theirs == out
        eng.release([fork])
    while len(out) < 60:
        out += eng.step([s]).tokens[s]
    assert out == want


def test_requests_in_reused_slots_leave_the_old_group(pkg, make) -> None:
    """Two requests on a prefix, then two without one in the same slots: the slot list stays the same."""
    shared = prompts_with_prefix(pkg, 200, 2)
    v = pkg.SMALL_TEST.vocab_size
    lone = [pkg.make_prompt(v, 230, 70 + i, i == 0) for i in range(2)]
    outs = {}
    for on in (False, True):
        eng = make(shared=on, max_seqs=3)
        holder = eng.add_prefix(shared[0][:200])
        outs[on] = []
        for prompts, prefix in ((shared, holder), (lone, None), (shared, holder)):
            slots = eng.add_requests(prompts, [20, 20], ignore_eos=True, prefix=prefix)
            assert sorted(slots) == [1, 2]
            res = eng.prefill(slots)
            out = {s: list(res.tokens[s]) for s in slots}
            live = list(slots)
            while live:
                res = eng.step(live)
                for s in list(live):
                    out[s] += res.tokens[s]
                    if res.finish[s] is not None:
                        live.remove(s)
            outs[on].append([out[s] for s in slots])
            eng.release([1, 2])
    assert outs[True] == outs[False]


@pytest.mark.parametrize("at", [1, 33, 48, 49, 160, 170])
def test_a_fork_cut_inside_the_prefix(pkg, make, at) -> None:
    """The fork shares fewer blocks than its source does: the group reads those only."""
    prompt = prompts_with_prefix(pkg, 160, 1)[0] + pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 12, 8, False)
    outs = {}
    for on in (False, True):
        eng = make(shared=on)
        holder = eng.add_prefix(prompt[:160])
        s = eng.add_request(prompt, 16, ignore_eos=True, prefix=holder)
        eng.prefill([s])
        slots = [s] + eng.fork(s, 2, at=at)
        out = {i: [] for i in slots}
        for _ in range(4):
            for i, t in eng.step(slots).tokens.items():
                out[i] += t
        outs[on] = [out[i] for i in slots]
        eng.release(slots)
        eng.drop_prefix(holder)
        assert eng.state.num_free_blocks() == 192
    assert outs[True] == outs[False]
    want = make(shared=False).generate([prompt[:at]], 8)[0]
    n = min(len(want), len(outs[True][1]))
    assert n >= 4 and outs[True][1][:n] == want[:n] and outs[True][2] == outs[True][1]


@pytest.mark.parametrize("on", [False, True], ids=["plain", "shared"])
def test_forks_of_a_prefix_itself_keep_it(pkg, make, on) -> None:
    """Forks of the handle that ``add_prefix`` gives are users of the prefix."""
    prompt = prompts_with_prefix(pkg, 160, 1)[0]
    eng = make(shared=on)
    holder = eng.add_prefix(prompt[:150])
    slots = eng.fork(holder, 2, at=140) + [eng.add_request(prompt, 8, ignore_eos=True, prefix=holder)]
    with pytest.raises(RuntimeError):
        eng.drop_prefix(holder)
    eng.state.max_new_tokens[torch.tensor(slots[:2], device=eng.model.device)] = 8
    res = eng.prefill(slots)
    out = {s: list(res.tokens[s]) for s in slots}
    while len(out[slots[2]]) < 8:
        for s, t in eng.step(slots).tokens.items():
            out[s] += t
    plain = make(shared=False)
    want = [plain.generate([p], 8)[0] for p in (prompt[:140], prompt[:140], prompt)]
    assert [out[s][:8] for s in slots] == want
    eng.release(slots)
    eng.drop_prefix(holder)
    assert eng.state.num_free_blocks() == 192


def steps_of(eng, slots, n):
    """The tokens of ``n`` steps, and whether they wrote the shared attention's workspace."""
    eng._groups_ws.zero_()
    out = {s: [] for s in slots}
    for _ in range(n):
        for s, t in eng.step(slots).tokens.items():
            out[s] += t
    return [out[s] for s in slots], bool(eng._groups_ws.any())


@pytest.mark.parametrize("kv_int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "eager"])
def test_steps_read_a_groups_prefix_through_its_first_member(pkg, make, kv_int8, graphs) -> None:
    """Users of a prefix and forks of a loner are the groups on the device, and the steps use them: the blocks
    that the other members' own tables name at a shared prefix are not read."""
    prompts = prompts_with_prefix(pkg, 150, 3)
    lone = pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 70, 9, False)
    outs = []
    for moved in (False, True):
        eng = make(kv_int8, cuda_graphs=graphs)
        holder = eng.add_prefix(prompts[0][:150])
        slots = eng.add_requests(prompts, [40] * 3, ignore_eos=True, prefix=holder)
        slots.append(eng.add_request(lone, 40, ignore_eos=True))
        eng.prefill(slots)
        slots += eng.fork(slots[3], 2)
        eng.step(slots)
        entry_group, prefix_blocks = eng._groups_dev.tolist()
        assert entry_group[:6] == [0, 0, 0, 1, 1, 1] and entry_group[6:] == [-1, -1]
        assert prefix_blocks[:3] == [9, 4, 0]  # (150 and 70 cached tokens)
        saved = eng.state.block_tables.clone()
        if moved:
            other = int(saved[holder, 9])  # (the prefix's last block, partly filled and shared with none)
            eng.state.block_tables[slots[1], :9] = other
            eng.state.block_tables[slots[2], 2:5] = other
            eng.state.block_tables[slots[5], :4] = other
        tokens, ran = steps_of(eng, slots, 4)
        assert ran
        outs.append(tokens)
        rows = torch.tensor(slots, device=saved.device)
        eng.state.block_tables[rows, :9] = saved[rows, :9]
        eng.release(slots)
        eng.drop_prefix(holder)
        assert eng.state.num_free_blocks() == 192
    assert outs[0] == outs[1]


def test_a_lone_sequences_steps_leave_the_shared_attention_alone(pkg, make) -> None:
    eng = make()
    s = eng.add_request(prompts_with_prefix(pkg, 60, 1)[0], 30, ignore_eos=True)
    eng.prefill([s])
    assert not steps_of(eng, [s], 3)[1]
    eng.release([s])


def test_reused_slots_and_forks_show_their_groups(pkg, make) -> None:
    """Requests, loners and forks in the same two slots, one after the other: the groups on the device follow."""
    eng = make(max_seqs=3)
    prompts = prompts_with_prefix(pkg, 200, 2)
    holder = eng.add_prefix(prompts[0][:200])

    def groups(slots):
        assert sorted(slots) == [1, 2]
        eng.step(slots)
        entry_group, prefix_blocks = eng._groups_dev.tolist()
        return entry_group[:2], prefix_blocks[0]

    def served(prompts, prefix):
        slots = eng.add_requests(prompts, [20] * len(prompts), ignore_eos=True, prefix=prefix)
        eng.prefill(slots)
        return slots

    for _ in range(2):
        slots = served(prompts, holder)
        assert groups(slots) == ([0, 0], 12)
        eng.release(slots)
        slots = served([p[100:] for p in prompts], None)
        assert groups(slots) == ([-1, -1], 0)
        eng.release(slots)
        slots = served([prompts[0]], None)
        slots += eng.fork(slots[0], 1, at=50)
        assert groups(slots) == ([0, 0], 3)
        eng.release(slots)


def test_a_short_fork_leaves_the_others_their_prefix(pkg, make) -> None:
    """One user's fork cut inside the first block, and one in the third: the group on the device holds the others
    and their whole prefix, and every sequence takes the tokens that it takes without sharing."""
    prompts = prompts_with_prefix(pkg, 160, 4)
    outs = {}
    for on in (False, True):
        eng = make(shared=on)
        holder = eng.add_prefix(prompts[0][:160])
        slots = eng.add_requests(prompts, [30] * 4, ignore_eos=True, prefix=holder)
        eng.prefill(slots)
        slots += eng.fork(slots[0], 1, at=5) + eng.fork(slots[0], 1, at=40)
        out = {s: [] for s in slots}
        for _ in range(4):
            for s, t in eng.step(slots).tokens.items():
                out[s] += t
        outs[on] = [out[s] for s in slots]
        if on:
            entry_group, prefix_blocks = eng._groups_dev.tolist()
            assert entry_group == [0, 0, 0, 0, -1, -1, -1, -1] and prefix_blocks[:2] == [10, 0]
        eng.release(slots)
        eng.drop_prefix(holder)
        assert eng.state.num_free_blocks() == 192
    assert outs[True] == outs[False]


def test_fork_step_and_sample_by_hand(pkg, make, cuda_device) -> None:
    """A user's own loop: prefill, fork, one step, and next tokens drawn from the step's logits with
    top-k, top-p and min-p; the draw equals the definition on those logits."""
    from tests.test_gpu_sample_logits import check

    ops = submodule("ops")
    eng = make()
    prompt = prompts_with_prefix(pkg, 120, 1)[0]
    s = eng.add_request(prompt, 40, ignore_eos=True, temperature=0.9, top_p=0.95, seed=1)
    eng.prefill([s])
    slots = [s] + eng.fork(s, 5, at=len(prompt), seeds=[2, 3, 4, 5, 6])
    eng.step(slots)
    rows = 6
    logits = eng.sampled_logits(rows)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    check(ops, logits, [(0.8, 20, 0.9, 0.01)] * rows, u)
    eng.release(slots)


@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "eager"])
def test_the_model_keeps_no_groups_between_launches(pkg, make, graphs) -> None:
    """The groups' arrays are the engine's: other users of the model, and later ones, never read them."""
    class Recorder:
        def __init__(self, lib):
            self.lib, self.bound = lib, []

        def __getattr__(self, name):
            return getattr(self.lib, name)

        def ne_model_set_prefix_groups(self, handle, groups, ws, size):
            self.bound.append(groups is not None)
            return self.lib.ne_model_set_prefix_groups(handle, groups, ws, size)

    prompts = prompts_with_prefix(pkg, 200, 3)
    eng = make(cuda_graphs=graphs)
    eng.lib = recorder = Recorder(eng.lib)
    eng.generate(prompts, 6, shared_prefix=200)
    n = len(recorder.bound)
    assert n and recorder.bound == [True, False] * (n // 2)
    recorder.ne_prefill = lambda *args: 1
    slots = eng.add_requests(prompts, [4] * 3)
    with pytest.raises(Exception):
        eng.prefill(slots)
    assert recorder.bound[n:] == [True, False]
    eng.release(slots)


def test_groups_whose_bounds_cannot_be_served_leave_steps_as_they_are(pkg, make, cuda_device) -> None:
    """Bounds past the shared attention's limits (here its units of work) are a forward without groups,
    not a failed one."""
    _lib = submodule("_lib")
    prompts = prompts_with_prefix(pkg, 60, 3)
    want = make(shared=False).generate(prompts, 10)
    eng = make(shared=False)
    entry_group = torch.full((16,), -1, dtype=torch.int32, device=cuda_device)
    prefix_blocks = torch.ones(16, dtype=torch.int32, device=cuda_device)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device=cuda_device)
    groups = _lib.PrefixGroups(num_groups=16, max_prefix_blocks=1 << 30, entry_group=entry_group.data_ptr(),
                               prefix_blocks=prefix_blocks.data_ptr())
    assert eng.lib.ne_model_set_prefix_groups(eng.model.handle, ctypes.byref(groups), ws.data_ptr(), ws.numel()) == 0
    try:
        assert eng.generate(prompts, 10) == want
    finally:
        eng.lib.ne_model_set_prefix_groups(eng.model.handle, None, None, 0)
    assert torch.count_nonzero(ws) == 0


def test_model_entry_refuses_bad_arguments(pkg, make, cuda_device) -> None:
    _lib = submodule("_lib")
    eng = make()
    lib, handle = eng.lib, eng.model.handle
    some = torch.zeros(256, dtype=torch.int32, device=cuda_device)
    ok = dict(num_groups=1, max_prefix_blocks=4, entry_group=some.data_ptr(), prefix_blocks=some.data_ptr())
    call = lambda ws=some.data_ptr(), **kw: lib.ne_model_set_prefix_groups(  # noqa: E731
        handle, ctypes.byref(_lib.PrefixGroups(**{**ok, **kw})), ws, 1024)
    assert lib.ne_model_set_prefix_groups(None, None, None, 0) == 1
    for bad in (dict(num_groups=-1), dict(num_groups=1025), dict(max_prefix_blocks=0), dict(entry_group=None),
                dict(prefix_blocks=None), dict(ws=None), dict(ws=some.data_ptr() + 4)):
        assert call(**bad) == 1
    assert call() == 0  # (a workspace too small for a step: its attention stays the ordinary one)
    prompt = prompts_with_prefix(pkg, 60, 1)[0]
    assert eng.generate([prompt], 8) == make(shared=False).generate([prompt], 8)
    assert lib.ne_model_set_prefix_groups(handle, None, None, 0) == 0
    with pytest.raises(ValueError):
        make(draft_model=submodule("model").B200Model(
            pkg.SMALL_TEST, pkg.make_weights(pkg.SMALL_TEST, seed=1), num_slots=32 * 16, device=cuda_device,
            max_positions=640, max_rows=512, max_seqs=16))
