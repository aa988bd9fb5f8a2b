"""Pages of the cache: copies within a pool, forks, trims and compaction, each against a plain
restatement on the host, and forked requests run through the engine."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import submodule

pytestmark = pytest.mark.gpu

BLOCK = 16
BAD_SLOT, NO_BLOCKS, HISTORY = 2, 4, 16


@pytest.fixture(scope="module")
def ops(cuda_device):
    submodule("build").build()
    return submodule("ops")


def pool(layers, blocks, nkv, int8, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, 2, blocks * BLOCK + 1, nkv, 128)
    if int8:
        return (torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).to(device),
                torch.randn(shape[:-1], generator=g).to(torch.bfloat16).to(device))
    return torch.randn(shape, generator=g).to(torch.bfloat16).to(device), None


def copied(t, pairs):
    """The pool's tensor after the copies, every source read first."""
    out = t.clone()
    blocks = t.shape[2] // BLOCK
    for s, d in pairs:
        if 0 <= s < blocks and 0 <= d < blocks:
            out[:, :, d * BLOCK:(d + 1) * BLOCK] = t[:, :, s * BLOCK:(s + 1) * BLOCK]
    return out


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("layers,blocks,nkv", [(1, 2, 1), (3, 40, 8), (28, 20, 8), (2, 33, 3), (5, 16, 2)])
def test_copy_blocks(ops, cuda_device, layers, blocks, nkv, int8) -> None:
    kv, scales = pool(layers, blocks, nkv, int8, cuda_device)
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(blocks)).tolist()
    half = blocks // 2
    pairs = list(zip(ids[:half], ids[half: 2 * half]))
    if len(pairs) > 2:
        pairs[1] = (pairs[0][0], pairs[1][1])  # one source, two destinations
        pairs[2] = (-1, pairs[2][1])           # no copy asked for
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    want, want_scales = copied(kv, pairs), copied(scales, pairs) if int8 else None
    src, dst = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in zip(*pairs))
    ops.copy_kv_blocks(kv, src, dst, scales=scales, status=status)
    assert torch.equal(kv, want) and int(status.item()) == 0
    if int8:
        assert torch.equal(scales, want_scales)


def test_copy_counts_bad_ids_and_refusals(ops, cuda_device) -> None:
    kv, _ = pool(2, 12, 2, False, cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    for count in (0, 1, 2, -5, 99):
        want = copied(kv, [(0, 6), (1, 7), (2, 8)][: max(count, 0)])
        ops.copy_kv_blocks(kv, ints([0, 1, 2]), ints([6, 7, 8]), count=ints([count]), status=status)
        assert torch.equal(kv, want) and int(status.item()) == 0
    for pair in ((12, 3), (3, 12), (3, -1), (1 << 30, 3), (3, 1 << 30)):
        status.zero_()
        want = copied(kv, [(0, 5)])
        ops.copy_kv_blocks(kv, ints([pair[0], 0]), ints([pair[1], 5]), status=status)
        assert torch.equal(kv, want) and int(status.item()) == BAD_SLOT
    ops.copy_kv_blocks(kv, ints([]), ints([]))
    for bad in (dict(kv=kv.float()), dict(kv=kv[:, :, ::2]), dict(kv=kv[:, :1]), dict(src=ints([0]).long()),
                dict(dst=ints([1, 2])), dict(scales=kv[..., 0]), dict(count=ints([1, 2]))):
        a = {**dict(kv=kv, src=ints([0]), dst=ints([1]), scales=None, count=None), **bad}
        with pytest.raises(ValueError):
            ops.copy_kv_blocks(a["kv"], a["src"], a["dst"], scales=a["scales"], count=a["count"])


def test_copies_far_into_a_large_pool(ops, cuda_device) -> None:
    """A pool of more than 2^32 bytes per plane pair: offsets pass 32 bits."""
    blocks = 70000
    kv = torch.zeros((2, 2, blocks * BLOCK + 1, 8, 128), dtype=torch.bfloat16, device=cuda_device)
    last = blocks - 1
    kv[:, :, :BLOCK] = torch.randn(2, 2, BLOCK, 8, 128, device=cuda_device).to(torch.bfloat16)
    ops.copy_kv_blocks(kv, torch.tensor([0], dtype=torch.int32, device=cuda_device),
                       torch.tensor([last], dtype=torch.int32, device=cuda_device))
    assert torch.equal(kv[:, :, last * BLOCK: blocks * BLOCK], kv[:, :, :BLOCK])
    assert torch.count_nonzero(kv[:, :, BLOCK: last * BLOCK].view(torch.int16)[:, :, ::BLOCK]) == 0


def fresh_state(cuda_device, tokens, cached, max_seqs=8, num_blocks=40, stride=256):
    """A state whose slot 0 holds ``tokens`` tokens, ``cached`` of them in blocks taken from the FIFO."""
    st = submodule("state").DeviceBatchState(max_seqs, stride, 4, num_blocks, device=cuda_device)
    st.load(0, list(range(100, 100 + tokens)), 50, ignore_eos=True, temperature=0.7, top_p=0.9, seed=77, draws=5)
    used = -(-cached // BLOCK)
    st.block_tables[0, :used] = torch.arange(used, dtype=torch.int32, device=cuda_device)
    st.num_blocks_used[0] = used
    st.num_cached[0] = cached
    st.ring_head_tail[0] = used
    return st


@pytest.mark.parametrize("tokens,at", [(40, 0), (33, 0), (34, 0), (1, 0), (16, 0), (17, 0), (40, 17), (40, 1), (40, 40),
                                       (40, 33), (40, 34)])
def test_fork_shares_full_blocks_and_copies_the_last(ops, cuda_device, tokens, at) -> None:
    st = fresh_state(cuda_device, tokens, tokens - 1)
    before = st.num_free_blocks()
    src, dst = st.fork(0, [3, 5], at)
    length = at or tokens
    cached = min(tokens - 1, length - 1)
    full, tail = cached // BLOCK, int(cached % BLOCK > 0)
    assert st.num_free_blocks() == before - 2 * tail
    for i, s in enumerate((3, 5)):
        assert st.tokens(s) == list(range(100, 100 + length))
        table = st.block_table(s)
        assert len(table) == full + tail and table[:full] == list(range(full))
        if tail:
            assert (int(src[i]), int(dst[i])) == (full, table[full])
            assert table[full] == -(-(tokens - 1) // BLOCK) + i  # the FIFO's next, in order
        else:
            assert (int(src[i]), int(dst[i])) == (-1, -1)
        assert int(st.num_cached[s]) == cached and int(st.num_shared_blocks[s]) == full
        assert int(st.num_prompt[s]) == min(tokens, length)
        assert float(st.temperature[s]) == pytest.approx(0.7) and int(st.rng_seed[s]) == 77 and int(st.rng_draws[s]) == 5
    # freeing the forks returns only what they own
    st.release([3, 5])
    assert st.num_free_blocks() == before
    assert st.block_table(0) == list(range(-(-(tokens - 1) // BLOCK)))


def test_fork_seeds_and_flags(ops, cuda_device) -> None:
    lib = submodule("_lib")
    st = fresh_state(cuda_device, 20, 19)
    st.flags[0] = lib.NE_SEQ_FINISHED | lib.NE_SEQ_IGNORE_EOS
    st.fork(0, [1, 2], 0, seeds=[9, (1 << 64) - 1])
    assert [int(st.rng_seed[s]) for s in (1, 2)] == [9, -1] and int(st.rng_draws[1]) == 0
    assert int(st.flags[1]) == int(st.flags[0])
    st.fork(0, [3], 10)
    assert int(st.flags[3]) == lib.NE_SEQ_IGNORE_EOS


def test_fork_refusals(ops, cuda_device) -> None:
    native = submodule("_lib").NativeError
    st = fresh_state(cuda_device, 20, 19)
    ring = st.ring_head_tail.clone()
    tables = st.block_tables.clone()
    with pytest.raises(native):
        st.fork(0, [1], 21)                     # beyond the history
    st.num_blocks_used[2] = 1
    for bad in ([0], [2], [99], [-3]):
        with pytest.raises(native):
            st.fork(0, bad)                     # the source, a slot with blocks, none at all
    assert torch.equal(st.ring_head_tail, ring) and torch.equal(st.block_tables, tables)
    with pytest.raises(native):
        st.fork(0, [4, 4])                      # listed twice: the first is made
    assert st.tokens(4) == st.tokens(0)
    assert int(st.ring_head_tail[0]) == int(ring[0]) + 1
    st.ring_head_tail[0] = st.ring_head_tail[1] - 1
    with pytest.raises(native, match="out of KV blocks"):
        st.fork(0, [5, 6])                      # one block left for two
    assert int(st.num_blocks_used[5]) == 0 and st.num_free_blocks() == 1
    for bad in ((8, [1], 0), (-1, [1], 0), (0, [1], -1), (0, [1], 10 ** 6)):
        with pytest.raises(ValueError):
            st.fork(*bad)
    with pytest.raises(ValueError):
        st.fork(0, [1], 0, seeds=[1, 2])


def test_trim_returns_the_blocks_past_the_cache(ops, cuda_device) -> None:
    st = fresh_state(cuda_device, 60, 59, num_blocks=10)
    st.num_cached[0] = 20
    st.trim([0, 0])
    assert st.block_table(0) == [0, 1]
    assert st.num_free_blocks() == 8
    head, tail = st.ring_head_tail.tolist()
    assert [int(st.free_ring[i % 10]) for i in range(head, tail)] == [4, 5, 6, 7, 8, 9, 2, 3]
    # shared blocks are another slot's
    st.fork(0, [1], 17)
    st.num_cached[1] = 0
    st.trim([1])
    assert st.block_table(1) == [0] and int(st.num_shared_blocks[1]) == 1
    with pytest.raises(submodule("_lib").NativeError):
        st.trim([-1])


@pytest.mark.parametrize("num_blocks", [1, 7, 64, 1500, 5000])
def test_compaction_keeps_every_sequence(ops, cuda_device, num_blocks) -> None:
    g = torch.Generator().manual_seed(num_blocks)
    st = submodule("state").DeviceBatchState(70, 2000, 4, num_blocks, device=cuda_device)
    ids = torch.randperm(num_blocks, generator=g).tolist()
    tables = {}
    for s in range(0, 70, 2):
        n = min(len(ids), int(torch.randint(0, 90, (1,), generator=g)))
        tables[s] = [ids.pop() for _ in range(n) if len(ids) > num_blocks // 3]
    tables[1] = tables[0][: len(tables[0]) // 2]  # shared blocks
    for s, t in tables.items():
        st.block_tables[s, : len(t)] = torch.tensor(t, dtype=torch.int32)
        st.num_blocks_used[s] = len(t)
    used = {b for t in tables.values() for b in t}
    st.ring_head_tail[0] = len(used)
    payload = torch.randn(1, 2, num_blocks * BLOCK + 1, 1, 128, device=cuda_device).to(torch.bfloat16)
    kv = payload.clone()
    copies = torch.full((num_blocks,), -1, dtype=torch.int32, device=cuda_device)
    for i, b in enumerate(tables[0]):
        copies[b] = i
    src, dst, count = st.compact(copies)
    ops.copy_kv_blocks(kv, src, dst, count=count)
    moved = int(count.item())
    assert moved == len([b for b in used if b >= len(used)])
    for s, t in tables.items():
        new = st.block_table(s)
        assert all(b < len(used) for b in new)
        for old_id, new_id in zip(t, new):
            assert torch.equal(kv[:, :, new_id * BLOCK:(new_id + 1) * BLOCK],
                               payload[:, :, old_id * BLOCK:(old_id + 1) * BLOCK])
    assert st.block_table(1) == st.block_table(0)[: len(tables[1])]
    assert [int(copies[b]) for b in st.block_table(0)] == list(range(len(tables[0])))
    assert int((copies >= 0).sum()) == len(tables[0])
    assert st.num_free_blocks() == num_blocks - len(used)
    assert st.free_ring[: num_blocks - len(used)].tolist() == list(range(len(used), num_blocks))
    again = st.compact(copies)
    assert int(again[2].item()) == 0


def test_compaction_reports_an_id_outside_the_pool(ops, cuda_device) -> None:
    st = fresh_state(cuda_device, 40, 39)
    st.block_tables[0, 1] = 4000
    with pytest.raises(submodule("_lib").NativeError):
        st.compact()


# ------------------------------------------------------------------------------ the engine
@pytest.fixture(scope="module")
def make_engine(pkg, cuda_device):
    submodule("build").build()
    weights = pkg.make_weights(pkg.SMALL_TEST, seed=0)
    models = {}

    def make(kv_int8=False, num_blocks=96, **kw):
        if kv_int8 not in models:
            models[kv_int8] = submodule("model").B200Model(
                pkg.SMALL_TEST, weights, num_slots=128 * 16, device=cuda_device, max_positions=512, max_rows=512,
                max_seqs=16, kv_int8=kv_int8, kv_copy_blocks=16 if kv_int8 else 0)
        return submodule("engine").B200SpeculativeEngine(models[kv_int8], k=4, max_ngram=3, max_seqs=8,
                                                         max_model_len=256, num_blocks=num_blocks, sampling=True, **kw)

    return make


@pytest.mark.parametrize("kv_int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("length", [33, 48, 61])
def test_samples_of_one_prompt(pkg, make_engine, kv_int8, length) -> None:
    """Greedy samples equal the request's own completion. Sampled ones are the same on every run and
    differ between seeds; they are not compared with requests run in another batch, whose GEMMs split
    their sums by the number of rows: a last bit of a logit moves a draw from this nearly flat
    random-weight distribution to a neighbouring id."""
    prompt = pkg.make_prompt(pkg.SMALL_TEST.vocab_size, length, 4, False)
    eng = make_engine(kv_int8)
    free = eng.state.num_free_blocks()
    seeds = [11, 12, 13, 14, 15]
    got = eng.generate_samples(prompt, 5, 24, temperature=0.8, top_p=0.9, seeds=seeds)
    assert eng.state.num_free_blocks() == free and len(eng.state.free_slots) == 8
    assert all(len(t) == 24 for t in got) and len({t[0] for t in got}) > 1 and len({tuple(t) for t in got}) == 5
    assert got == make_engine(kv_int8).generate_samples(prompt, 5, 24, temperature=0.8, top_p=0.9, seeds=seeds)
    greedy = make_engine(kv_int8).generate_samples(prompt, 3, 16, temperature=0.0)
    assert greedy == make_engine(kv_int8).generate([prompt], 16) * 3


@pytest.mark.parametrize("num_blocks", [2, 8, 12, 20])
def test_samples_that_outgrow_the_pool_end_with_an_error(pkg, make_engine, num_blocks) -> None:
    """The pool runs out in the prompt's prefill, in the forks' or in a step: the call raises, every slot
    and block is back, and samples that fit are served as ever."""
    eng = make_engine(num_blocks=num_blocks)
    prompt = pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 33, 4, False)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="out of KV blocks"):
            eng.generate_samples(prompt, 8, 200, temperature=0.8)
        assert eng.state.num_free_blocks() == num_blocks and len(eng.state.free_slots) == 8
    if num_blocks >= 8:  # (33 + 10 tokens and 4 guesses: three blocks of which two are shared)
        assert [len(t) for t in eng.generate_samples(prompt, 2, 10, temperature=0.8)] == [10, 10]


@pytest.mark.parametrize("kv_int8", [False, True], ids=["bf16", "int8"])
def test_a_fork_on_the_same_stream_draws_what_its_source_draws(pkg, make_engine, kv_int8) -> None:
    """Forked with all its tokens and without seeds, a sequence holds its source's very state: in one
    batch both take the same tokens, bit for bit."""
    eng = make_engine(kv_int8)
    s = eng.add_request(pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 45, 4, False), 30, ignore_eos=True,
                        temperature=0.9, top_p=0.95, seed=5)
    eng.prefill([s])
    eng.step([s])
    same, = eng.fork(s)
    other, = eng.fork(s, seeds=[6])
    outs = {x: [] for x in (s, same, other)}
    for _ in range(8):
        res = eng.step([s, same, other])
        for x, t in res.tokens.items():
            outs[x] += t
    assert outs[same] == outs[s] and outs[other] != outs[s]
    assert eng.draws_used(same) == eng.draws_used(s)
    eng.release([s, same, other])


@pytest.mark.parametrize("kv_int8", [False, True], ids=["bf16", "int8"])
def test_fork_trim_and_compact_in_mid_request_change_no_token(pkg, make_engine, kv_int8) -> None:
    """Two requests run; one ends and leaves holes; the other is forked in mid-way, the pool trimmed
    and compacted: source and fork go on as the request would have alone."""
    v = pkg.SMALL_TEST.vocab_size
    first, second = pkg.make_prompt(v, 50, 1, True), pkg.make_prompt(v, 70, 2, False)
    want = make_engine(kv_int8).generate([second], 40)[0]
    eng = make_engine(kv_int8)
    prefix = eng.add_prefix(second[:40])
    a = eng.add_request(first, 8, ignore_eos=True)
    b = eng.add_request(second, 40, ignore_eos=True, prefix=prefix)
    res = eng.prefill([a, b])
    out = list(res.tokens[b])
    for _ in range(3):
        out += eng.step([a, b]).tokens[b]
    fork = eng.fork(b, 2)
    nested = eng.fork(fork[0], 1)
    with pytest.raises(RuntimeError):
        eng.release([b])
    eng.release([a])
    eng.trim([b, *fork, *nested])
    assert eng.compact() >= 0
    lows = [i for s in (b, *fork, *nested, prefix) for i in eng.state.block_table(s)]
    assert max(lows) < eng.state.num_blocks - eng.state.num_free_blocks()
    outs = {s: list(out) for s in (b, *fork, *nested)}
    live = list(outs)
    while live:
        res = eng.step(live)
        for s in list(live):
            outs[s] += res.tokens[s]
            if res.finish[s] is not None:
                live.remove(s)
    assert all(t == want for t in outs.values())
    eng.release([b, *fork, *nested])
    eng.drop_prefix(prefix)
    assert eng.state.num_free_blocks() == 96 and len(eng.state.free_slots) == 8


def test_engine_fork_refusals(pkg, make_engine) -> None:
    eng = make_engine(num_blocks=8)
    prompt = pkg.make_prompt(pkg.SMALL_TEST.vocab_size, 40, 3, False)
    s = eng.add_request(prompt, 8, ignore_eos=True)
    with pytest.raises(ValueError):
        eng.fork(s)  # not prefilled
    eng.prefill([s])
    with pytest.raises(ValueError):
        eng.fork(7)  # a free slot
    with pytest.raises(ValueError):
        eng.fork(s, 1, at=0)
    with pytest.raises(RuntimeError):
        eng.fork(s, 8)  # more than the free slots
    free = list(eng.state.free_slots)
    with pytest.raises(RuntimeError, match="out of KV blocks"):
        eng.fork(s, 7)  # five blocks left
    assert eng.state.free_slots == free
    assert eng.fork(s, 0) == []
    with pytest.raises(ValueError):
        eng.generate_samples(prompt, 9, 4)
    with pytest.raises(ValueError):
        eng.generate_samples(prompt, 2, 4, seeds=[1])
