"""Attention over shared prompt prefixes (``ops.prefix_attention``) against a plain implementation in
64 bits: group layouts, lengths from one token on, head ratios, bf16 and int8 pools, rows that see
nothing, values in masked places, ids outside the pool, streams and captured graphs."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import submodule

pytestmark = pytest.mark.gpu

BLOCK, D = 16, 128
BAD_SLOT = 2


@pytest.fixture(scope="module")
def ops(cuda_device):
    submodule("build").build()
    return submodule("ops")


def make_case(seed, heads, kv_heads, q_lens, prefix_tokens, groups, suffixes, int8=False, poison=True, device="cuda:0",
              spare=3):
    """Entries with ``suffixes`` tokens between their prefix and their rows. ``prefix_tokens[g]`` is a
    multiple of 16; ``groups[b]`` is the entry's group or -1. With ``poison`` every slot that no row
    sees holds NaN (bf16) or the largest scale (int8)."""
    g = torch.Generator().manual_seed(seed)
    n = len(q_lens)
    prefix_blocks = [t // BLOCK for t in prefix_tokens]
    contexts = [(prefix_tokens[groups[b]] if groups[b] >= 0 else 0) + suffixes[b] + q_lens[b] for b in range(n)]
    totals = [-(-c // BLOCK) for c in contexts]
    shared = [prefix_blocks[groups[b]] if groups[b] >= 0 else 0 for b in range(n)]
    used = sum(prefix_blocks) + sum(t - s for t, s in zip(totals, shared))
    num_blocks = used + spare
    ids = torch.randperm(num_blocks, generator=g).tolist()
    take = lambda k: [ids.pop() for _ in range(k)]  # noqa: E731
    group_ids = [take(p) for p in prefix_blocks]
    stride = max(totals) + 2
    table = torch.full((n, stride), -1, dtype=torch.int32)
    for b in range(n):
        row = (group_ids[groups[b]] if groups[b] >= 0 else []) + take(totals[b] - shared[b])
        table[b, : len(row)] = torch.tensor(row, dtype=torch.int32)
    slots = num_blocks * BLOCK + 1
    seen = torch.zeros(slots, dtype=torch.bool)
    for b in range(n):
        if q_lens[b]:
            p = torch.arange(contexts[b])
            seen[table[b][p // BLOCK].long() * BLOCK + p % BLOCK] = True
    rows = sum(q_lens)
    q = (torch.randn(rows, heads, D, generator=g) * 1.5).to(torch.bfloat16)
    case = dict(q=q, table=table, heads=heads, kv_heads=kv_heads, q_lens=q_lens, contexts=contexts, int8=int8)
    for name in ("k", "v"):
        if int8:
            case[name] = torch.randint(-127, 128, (slots, kv_heads, D), generator=g, dtype=torch.int8)
            scale = ((torch.rand(slots, kv_heads, generator=g) + 0.5) / 73).to(torch.bfloat16)
            if poison:
                scale[~seen] = float("nan")
            case[name + "s"] = scale
        else:
            x = torch.randn(slots, kv_heads, D, generator=g).to(torch.bfloat16)
            if poison:
                x[~seen] = float("nan")
            case[name] = x
    starts = [sum(q_lens[:b]) for b in range(n)]
    positions = [p for b in range(n) for p in range(contexts[b] - q_lens[b], contexts[b])]
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    case.update(q_start=ints(starts), q_len=ints(q_lens), positions=ints(positions), entry_group=ints(groups),
                prefix_blocks=ints(prefix_blocks), max_prefix=max(prefix_tokens, default=0))
    return {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in case.items()}


def reference(c):
    """(output, sum of p |v|) per element in 64 bits."""
    out = torch.zeros(c["q"].shape, dtype=torch.float64, device=c["q"].device)
    spread = torch.zeros_like(out)
    group = c["heads"] // c["kv_heads"]
    starts, lens, pos = c["q_start"].tolist(), c["q_len"].tolist(), c["positions"].cpu()
    for b in range(len(lens)):
        for j in range(lens[b]):
            row = starts[b] + j
            n = int(pos[row]) + 1
            if n <= 0:
                continue
            p = torch.arange(n, device=out.device)
            ids = c["table"][b][p // BLOCK].long()
            at = ids * BLOCK + p % BLOCK
            good = (ids >= 0) & ((ids + 1) * BLOCK <= c["k"].shape[0] - 1)
            at = at[good]
            k, v = c["k"][at].double(), c["v"][at].double()
            if c["int8"]:
                k, v = k * c["ks"][at].double()[..., None], v * c["vs"][at].double()[..., None]
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            s = torch.einsum("hd,thd->ht", c["q"][row].double(), k) / D ** 0.5
            w = torch.softmax(s, -1)
            out[row] = torch.einsum("ht,thd->hd", w, v)
            spread[row] = torch.einsum("ht,thd->hd", w, v.abs())
    return out, spread


def call(ops, c, **kw):
    status = kw.pop("status", None)
    if status is None:
        status = torch.zeros(1, dtype=torch.int32, device=c["q"].device)
    got = ops.prefix_attention(
        c["q"], c["k"], c["v"], c["table"], c["q_start"], c["q_len"], c["positions"], c["entry_group"],
        c["prefix_blocks"], max_q_len=kw.pop("max_q_len", max(c["q_lens"])), max_context=kw.pop("max_context", max(c["contexts"])),
        max_prefix=kw.pop("max_prefix", c["max_prefix"]), k_scale=c.get("ks"), v_scale=c.get("vs"), status=status, **kw)
    return got, status


def assert_close(got, c, rows=None):
    """Each weight and the output are rounded to bf16 once (2^-8 relative at most), and scores in fp32
    are off by at most 128 x 2^-24 of the sum of their products' magnitudes (below 8 here, over the
    root of 128): 1e-3 of the weights covers both softmax sums."""
    want, spread = reference(c)
    err = (got.double() - want).abs()
    tol = (2.0 ** -8 + 1e-3) * spread + 2.0 ** -8 * want.abs() + 1e-30
    if rows is not None:
        err, tol = err[rows], tol[rows]
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = {
    "one_token": (2, 1, [1], [16], [0], [0]),
    "one_row_no_group": (2, 1, [1], [], [-1], [0]),
    "two_share_a_block": (16, 8, [1, 1], [16], [0, 0], [0, 5]),
    "tail_of_a_tile": (16, 8, [5, 5, 5, 5], [16 * 11], [0] * 4, [0, 3, 16, 33]),
    "many_share": (16, 8, [5] * 30, [528], [0] * 30, [(i * 37) % 90 for i in range(30)]),
    "idle_entries": (16, 8, [0, 5, 0, 1, 3], [160], [0] * 5, [4, 9, 1, 0, 70]),
    "groups_and_loners": (16, 8, [5, 1, 3, 5, 2, 4, 5], [256, 48, 16], [0, 1, -1, 0, 1, 2, -1],
                          [10, 0, 300, 44, 17, 1, 0]),
    "group_of_one": (16, 8, [5], [1024], [0], [100]),
    "long_prefix_few_rows": (4, 2, [1, 1, 1], [8192 + 16], [0] * 3, [5, 0, 40]),
    "wide_heads": (32, 8, [5] * 17, [400], [0] * 17, [i for i in range(17)]),
    "odd_head_ratio": (14, 2, [3, 1, 9, 4], [208], [0] * 4, [50, 2, 0, 31]),
    "one_kv_head_of_32": (32, 1, [2, 5], [336], [0, 0], [7, 90]),
    "no_head_sharing": (4, 4, [5, 5], [128], [0, 0], [20, 130]),
    "prefill_rows": (8, 2, [70, 33, 5], [256], [0, 0, 0], [0, 19, 4]),
    "long_own_context": (16, 8, [5, 1], [64], [0, -1], [2000, 1500]),
    "empty_group": (16, 8, [2, 2], [64, 32], [1, 1], [3, 9]),
    "rows_fill_two_tiles": (16, 8, [1] * 128, [272], [0] * 128, [i % 20 for i in range(128)]),
    "rows_just_past_two_tiles": (16, 8, [1] * 129, [272], [0] * 129, [i % 20 for i in range(129)]),
}


def _mixed(groups, blocks):
    """Groups of one query tile and of two in turn, so that a CTA's share of the work holds both."""
    q_lens, group = [], []
    for g in range(groups):
        for _ in range(1 if g % 2 else 10):
            q_lens.append(2 if g % 2 else 5)
            group.append(g)
    return (32, 8, q_lens, [16 * (blocks - g % 7) for g in range(groups)], group, [i % 23 for i in range(len(q_lens))])


CASES["one_and_two_tiles_in_turn"] = _mixed(40, 70)
CASES["one_and_two_tiles_short"] = _mixed(60, 20)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("name", list(CASES))
def test_matches_64_bits(ops, name, int8) -> None:
    c = make_case(len(name) + int8, *CASES[name], int8=int8)
    out = torch.full_like(c["q"], float("nan"))
    got, status = call(ops, c, out=out)
    assert int(status.item()) == 0
    assert got is out
    assert_close(got, c)


def test_equal_calls_give_equal_bits(ops) -> None:
    c = make_case(5, *CASES["groups_and_loners"])
    first, _ = call(ops, c)
    for _ in range(3):
        again, _ = call(ops, c)
        assert torch.equal(first, again)


def test_bounds_above_the_lengths_change_nothing_but_rounding(ops) -> None:
    """The host bounds only size the launch: a captured call keeps bounds above later lengths."""
    c = make_case(6, *CASES["many_share"])
    got, status = call(ops, c, max_q_len=9, max_context=4000, max_prefix=3000)
    assert int(status.item()) == 0
    assert_close(got, c)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_rows_that_see_nothing_or_only_part_of_the_prefix(ops, int8) -> None:
    c = make_case(7, 16, 8, [3, 4, 5, 2], [96], [0, 0, 0, 0], [0, 10, 20, 1], int8=int8, poison=False)
    pos = c["positions"]
    pos[0:3] = -1                                                                  # padding: no key at all
    pos[3:7] = torch.tensor([40, 41, 42, 100], dtype=torch.int32, device=pos.device)  # inside the prefix
    pos[7] = -1                                                                    # a padded first row
    got, status = call(ops, c)
    assert int(status.item()) == 0
    assert torch.count_nonzero(got[0:3]) == 0 and torch.count_nonzero(got[7]) == 0
    assert_close(got, c)


def test_later_rows_values_do_not_reach_earlier_rows(ops) -> None:
    """Row j's own key is masked for the rows before it: an infinite value there stays there."""
    c = make_case(8, 16, 8, [5, 5], [64], [0, 0], [11, 30])
    last = int(c["positions"][4])
    slot = int(c["table"][0][last // BLOCK]) * BLOCK + last % BLOCK
    c["v"][slot] = float("inf")
    got, _ = call(ops, c)
    assert bool(torch.isinf(got[4]).all())
    clean = [r for r in range(10) if r != 4]
    c["v"][slot] = 0.0
    assert_close(got, c, rows=clean)


@pytest.mark.parametrize("where", ["query", "prefix key", "own key", "prefix value", "own value"])
def test_nan_that_a_row_sees_reaches_it(ops, where) -> None:
    """NaN in a query, or in a key or value its row sees, gives NaN there; every other row and head
    stays as near the definition as it is without (a warp that meets a NaN takes all its rows' powers
    of two on the special-function unit, so not bit for bit)."""
    c = make_case(19, 16, 8, [5] * 6, [272], [0] * 6, [9, 30, 1, 0, 70, 3])
    hit = torch.zeros(30, 16, dtype=torch.bool, device=c["q"].device)
    if where == "query":
        c["q"][7, 3, 60] = float("nan")
        hit[7, 3] = True
    else:
        entry, at = (2, 100) if where.startswith("prefix") else (4, 300)
        slot = int(c["table"][entry][at // BLOCK]) * BLOCK + at % BLOCK
        c["k" if "key" in where else "v"][slot, 5, 7] = float("nan")
        rows = torch.arange(30, device=hit.device)
        seen = torch.ones_like(rows, dtype=torch.bool) if entry == 2 else (rows >= 20) & (rows < 25) & (c["positions"] >= at)
        hit[seen, 10:12] = True
    got, status = call(ops, c)
    assert int(status.item()) == 0
    bad = torch.isnan(got).any(-1)
    assert torch.equal(bad, hit), (int(bad.sum()), int(hit.sum()))
    assert_close(got, c, rows=~hit)


def test_rows_of_no_entry_stay_as_they_were(ops) -> None:
    c = make_case(9, 16, 8, [2, 3], [32], [0, 0], [5, 6])
    extra = torch.zeros(4, 16, D, dtype=torch.bfloat16, device=c["q"].device)
    c["q"] = torch.cat([c["q"], extra + float("nan")])
    c["positions"] = torch.cat([c["positions"], torch.full((4,), 7, dtype=torch.int32, device=extra.device)])
    out = torch.full_like(c["q"], 3.0)
    got, status = call(ops, c, out=out)
    assert int(status.item()) == 0
    assert bool((got[5:] == 3.0).all())
    c["q"], c["positions"] = c["q"][:5].contiguous(), c["positions"][:5].contiguous()
    assert_close(got[:5], c)


def test_rows_out_of_order_and_table_rows_by_index(ops) -> None:
    c = make_case(10, 16, 8, [2, 3, 1], [48], [0, -1, 0], [5, 60, 6])
    want, _ = call(ops, c)
    # the same entries with their rows stored in another order and their tables behind an index
    order = [3, 4, 5, 0, 1, 2]  # entry 2 and 0's rows move
    perm = torch.tensor([5, 0, 1, 2, 3, 4], device=c["q"].device)
    d = dict(c, q=c["q"][perm].contiguous(), positions=c["positions"][perm].contiguous(),
             q_start=torch.tensor([1, 3, 0], dtype=torch.int32, device=perm.device))
    rows = torch.tensor([2, 0, 1], dtype=torch.int32, device=perm.device)
    d["table"] = c["table"][[1, 2, 0]].contiguous()
    got, _ = call(ops, d, table_index=rows)
    assert len(order) == 6
    assert_close(got[torch.argsort(perm)], c)
    torch.testing.assert_close(got.float(), want[perm].float(), rtol=2 ** -6, atol=2 ** -6)


@pytest.mark.parametrize("bad", [-1, 1 << 20, (1 << 31) - 1, -(1 << 31)])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_an_id_outside_the_pool_is_reported_and_left_out(ops, bad, int8) -> None:
    c = make_case(11, 16, 8, [3, 3], [160], [0, 0], [40, 50], int8=int8)
    c["table"][:, 4] = bad   # inside the prefix
    c["table"][1, 11] = bad  # inside entry 1's own blocks
    got, status = call(ops, c)
    assert int(status.item()) == BAD_SLOT
    assert_close(got, c)


def test_entries_that_share_rows_are_reported(ops) -> None:
    """More rows of groups than there are rows: the prefixes are left out, nothing past the buffers is written."""
    c = make_case(20, 16, 8, [4, 4, 4], [64], [0, 0, 0], [5, 6, 7])
    c["q_start"].zero_()
    for name in ("q", "positions"):
        c[name] = c[name][:4].contiguous()
    got, status = call(ops, c)
    assert int(status.item()) == BAD_SLOT
    assert bool(torch.isfinite(got).all())


def test_a_bound_of_many_rows_an_entry(ops) -> None:
    """A captured prefill's bound may be far above the rows of a replay."""
    c = make_case(21, 16, 8, [3, 40], [160], [0, 0], [7, 30])
    got, status = call(ops, c, max_q_len=1 << 16, max_context=1 << 17)
    assert int(status.item()) == 0
    assert_close(got, c)


@pytest.mark.parametrize("where", ["prefix", "own"])
def test_a_large_value_at_a_key_of_no_weight_stays_out(ops, where) -> None:
    """Weights below fp32's range are zero, not its least number: 3e38 times that would be seen."""
    c = make_case(22, 16, 8, [5] * 4, [272], [0] * 4, [40, 30, 20, 35])
    c["q"] = c["q"].abs()
    entry, at = (0, 75) if where == "prefix" else (1, 280)
    slot = int(c["table"][entry][at // BLOCK]) * BLOCK + at % BLOCK
    c["k"][slot] = -60.0
    c["v"][slot] = 3e38
    got, status = call(ops, c)
    assert int(status.item()) == 0
    assert_close(got, c)


def test_a_table_shorter_than_the_context_is_reported(ops) -> None:
    c = make_case(12, 16, 8, [2], [32], [0], [40])
    c["table"] = c["table"][:, :3].contiguous()
    got, status = call(ops, c)
    assert int(status.item()) == BAD_SLOT
    assert bool(torch.isfinite(got).all())


def test_streams_and_a_replayed_graph_with_new_inputs(ops) -> None:
    c = make_case(13, *CASES["groups_and_loners"])
    dev = c["q"].device
    ws = ops.prefix_attention_workspace(c["q"].shape[0], 7, 3, 16, 8, 5, max(c["contexts"]), dev)
    out = torch.empty_like(c["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(ops, c, out=out, workspace=ws, status=torch.zeros(1, dtype=torch.int32, device=dev))
    torch.cuda.current_stream().wait_stream(side)
    assert_close(out, c)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ops, c, out=out, workspace=ws, status=status)
    # other lengths, groups and queries in the same buffers
    d = make_case(14, 16, 8, [1, 5, 2, 0, 5, 3, 1], [128, 64, 32], [1, 1, 0, -1, 0, 2, 2], [9, 30, 1, 0, 70, 3, 12])
    for name in ("k", "v"):
        assert d[name].shape[0] <= c[name].shape[0]
    bound = max(c["contexts"])
    assert max(d["contexts"]) <= bound
    merged = dict(c)
    for name in ("q_start", "q_len", "entry_group", "prefix_blocks"):
        c[name].copy_(d[name])
    rows = d["q"].shape[0]
    c["q"][:rows].copy_(d["q"])
    c["positions"][:rows].copy_(d["positions"])
    c["table"].fill_(-1)
    width = min(c["table"].shape[1], d["table"].shape[1])
    c["table"][:, :width].copy_(d["table"][:, :width])
    for name in ("k", "v"):
        c[name][: d[name].shape[0]].copy_(d[name])
    graph.replay()
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    assert merged["q"] is c["q"]
    assert_close(out[:rows], d)


def test_two_calls_at_once_with_a_workspace_each(ops) -> None:
    a, b = make_case(15, *CASES["many_share"]), make_case(16, *CASES["wide_heads"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(a["q"]), torch.empty_like(b["q"])]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, c, o in zip(streams, (a, b), outs):
            with torch.cuda.stream(s):
                call(ops, c, out=o)
    torch.cuda.synchronize()
    assert_close(outs[0], a)
    assert_close(outs[1], b)


def test_offsets_past_32_bits(ops, cuda_device) -> None:
    """A pool of more than 2^32 elements: blocks at its far end."""
    nkv, blocks = 8, (1 << 32) // (BLOCK * 8 * D) + 64
    slots = blocks * BLOCK + 1
    if torch.cuda.mem_get_info()[0] < 5 * slots * nkv * D:
        pytest.skip("not enough device memory for the pool")
    c = make_case(17, 16, 8, [5, 5, 1], [160], [0, 0, 0], [20, 3, 9], poison=False)
    k = torch.empty((slots, nkv, D), dtype=torch.bfloat16, device=cuda_device)
    v = torch.empty_like(k)
    small = c["k"].shape[0] - 1
    far = blocks * BLOCK - small
    assert far % BLOCK == 0
    k[far: far + small], v[far: far + small] = c["k"][:small], c["v"][:small]
    table = torch.where(c["table"] >= 0, c["table"] + far // BLOCK, c["table"]).int()
    got, status = call(ops, dict(c, k=k, v=v, table=table))
    assert int(status.item()) == 0
    assert_close(got, c)


def test_python_front_refuses_wrong_tensors(ops) -> None:
    c = make_case(18, 16, 8, [2, 2], [32], [0, 0], [5, 6])
    for bad in (dict(q=c["q"].float()), dict(q=c["q"][:, :, ::2]), dict(k=c["k"][:, ::2]), dict(v=c["v"].float()),
                dict(q_len=c["q_len"].long()), dict(positions=c["positions"][:1]), dict(table=c["table"][:1]),
                dict(entry_group=c["entry_group"][:1]), dict(k=c["k"].to(torch.int8))):
        with pytest.raises(ValueError):
            call(ops, {**c, **bad})
    with pytest.raises(ValueError):
        call(ops, c, out=torch.empty_like(c["q"]).float())
    with pytest.raises(submodule("_lib").NativeError):
        call(ops, c, workspace=torch.empty(0, dtype=torch.uint8, device=c["q"].device))
