"""What the operators for many samples of one prompt refuse, on a host without a GPU: NULL and
out-of-range arguments at the C entries (no device work), host tensors and wrong shapes in Python."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.conftest import submodule

INVALID, WORKSPACE = 1, 5
SOME = ctypes.c_void_p(4096)  # an address no refused call reads


@pytest.fixture(scope="module")
def lib():
    submodule("build").build()
    return submodule("_lib").load()


def _attention(lib, *, rows=None, groups=None, heads=16, kv_heads=8, block=16, slots=33, int8=0, workspace=4096,
               nbytes=1 << 30, q=SOME):
    _lib = submodule("_lib")
    fields = dict(max_rows=4, num_seqs=2, positions=4096, q_start=4096, q_len=4096, block_tables=4096,
                  block_table_stride=2, max_context=32, max_q_len=2)
    r = _lib.Rows(**{**fields, **(rows or {})})
    g = _lib.PrefixGroups(**{**dict(num_groups=1, max_prefix_blocks=1, entry_group=4096, prefix_blocks=4096),
                             **(groups or {})})
    return lib.ne_prefix_attention(q, SOME, SOME, SOME, None, None, int8, ctypes.byref(r), ctypes.byref(g), heads,
                                   kv_heads, block, slots, workspace, nbytes, None, None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(int8=1), dict(heads=15), dict(heads=264), dict(kv_heads=0), dict(block=32), dict(slots=1),
    dict(workspace=None), dict(workspace=4097), dict(rows=dict(num_seqs=0)), dict(rows=dict(num_seqs=1025)),
    dict(rows=dict(max_rows=0)), dict(rows=dict(max_q_len=0)), dict(rows=dict(positions=None)),
    dict(rows=dict(q_len=None)), dict(rows=dict(block_tables=None)), dict(groups=dict(num_groups=-1)),
    dict(groups=dict(entry_group=None)), dict(groups=dict(max_prefix_blocks=-1)),
])
def test_prefix_attention_refuses_bad_arguments(lib, bad) -> None:
    assert _attention(lib, **bad) == INVALID


def test_prefix_attention_refuses_a_small_workspace(lib) -> None:
    need = lib.ne_prefix_attention_workspace_bytes(4, 2, 1, 16, 8, 2, 32)
    assert need > 0
    assert _attention(lib, nbytes=need - 1) == WORKSPACE
    assert lib.ne_prefix_attention_workspace_bytes(4, 2, 1, 15, 8, 2, 32) == 0
    assert lib.ne_prefix_attention_workspace_bytes(-1, 2, 1, 16, 8, 2, 32) == 0


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(uniform=None), dict(tokens=None), dict(rows=-1), dict(vocab=0), dict(vocab=262145, stride=262145),
    dict(stride=99), dict(logits=ctypes.c_void_p(4097)), dict(fp32=1, logits=ctypes.c_void_p(4098)),
])
def test_sample_logits_refuses_bad_arguments(lib, bad) -> None:
    a = {**dict(logits=SOME, fp32=0, rows=2, vocab=100, stride=100, uniform=SOME, tokens=SOME), **bad}
    rc = lib.ne_sample_logits(a["logits"], a["fp32"], a["rows"], a["vocab"], a["stride"], None, None, None, None,
                              a["uniform"], a["tokens"], None, None, None)
    assert rc == INVALID


@pytest.mark.parametrize("bad", [
    dict(kv=None), dict(kv=ctypes.c_void_p(4104)), dict(int8=1), dict(scales=SOME), dict(layers=0), dict(heads=0),
    dict(slots=1), dict(src=None), dict(dst=None), dict(pairs=-1),
])
def test_copy_blocks_refuses_bad_arguments(lib, bad) -> None:
    a = {**dict(kv=SOME, scales=None, int8=0, layers=2, heads=2, slots=33, src=SOME, dst=SOME, pairs=1), **bad}
    assert lib.ne_kv_copy_blocks(a["kv"], a["scales"], a["int8"], a["layers"], a["heads"], a["slots"], a["src"],
                                 a["dst"], None, a["pairs"], None, None) == INVALID


def test_empty_calls_launch_nothing(lib) -> None:
    """No rows, no pairs and no slots are no work, whatever the pointers are."""
    assert lib.ne_kv_copy_blocks(SOME, None, 0, 2, 2, 33, None, None, None, 0, None, None) == 0
    assert lib.ne_sample_logits(SOME, 0, 0, 100, 100, None, None, None, None, SOME, SOME, None, None, None) == 0


def test_state_entries_refuse_bad_arguments(lib) -> None:
    assert lib.ne_state_fork_slots(None, 0, SOME, 1, 0, None, SOME, SOME, None, None) == INVALID
    assert lib.ne_state_trim_slots(None, SOME, 1, None, None) == INVALID
    assert lib.ne_state_compact(None, SOME, SOME, SOME, SOME, None, None, None) == INVALID
    _lib = submodule("_lib")
    fields = {name: 4096 for name, kind in _lib.BatchState._fields_ if kind is ctypes.c_void_p}
    st = _lib.BatchState(max_seqs=4, history_stride=64, block_table_stride=4, num_blocks=8, num_stop_ids=0, **fields)
    ref = ctypes.byref(st)
    for src, dst, n, at in ((4, SOME, 1, 0), (-1, SOME, 1, 0), (0, None, 1, 0), (0, SOME, -1, 0), (0, SOME, 1025, 0),
                            (0, SOME, 1, -1), (0, SOME, 1, 65)):
        assert lib.ne_state_fork_slots(ref, src, dst, n, at, None, SOME, SOME, None, None) == INVALID
    assert lib.ne_state_fork_slots(ref, 0, SOME, 1, 0, None, None, SOME, None, None) == INVALID
    assert lib.ne_state_fork_slots(ref, 0, None, 0, 0, None, None, None, None, None) == 0
    assert lib.ne_state_trim_slots(ref, None, 1, None, None) == INVALID
    assert lib.ne_state_trim_slots(ref, None, 0, None, None) == 0
    assert lib.ne_state_compact(ref, None, SOME, SOME, SOME, None, None, None) == INVALID


def test_python_front_refuses_host_tensors() -> None:
    ops = submodule("ops")
    with pytest.raises(ValueError):
        ops.sample_logits(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError):
        ops.copy_kv_blocks(torch.zeros(1, 2, 17, 1, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32),
                           torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.prefix_attention_workspace(4, 2, 1, 15, 8, 2, 32, "cpu")
