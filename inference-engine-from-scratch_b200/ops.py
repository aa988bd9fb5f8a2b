"""Torch front of the operators for many samples of one prompt (``include/nespec.h``).

* ``prefix_attention``   attention that reads a prompt prefix shared by many sequences once for all
* ``sample_logits``      temperature, top-k, top-p and min-p draws from given random numbers
* ``copy_kv_blocks``     copies of cache blocks within a pool (what forks and compaction ask for)

Each checks its arguments on the host (``ValueError``), launches on the current stream of its
tensors' device without waiting, and reports what only the device can see (an id outside the pool, a
row without a token) into ``status``, an int32 tensor of one element the caller may pass and read
(``_lib.describe_device_status``). Nothing is kept between calls; a workspace may be reused by calls
that follow one another on one stream.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

BLOCK_SIZE = 16
HEAD_DIM = 128


def _device_of(first: torch.Tensor, **others: torch.Tensor | None) -> torch.device:
    """The CUDA device all tensors lie on."""
    device = first.device
    if device.type != "cuda":
        raise ValueError("the operators run on CUDA tensors (the B200 path has no CPU fallback)")
    for name, t in others.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")
    return device


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape}, "
                         f"got {t.dtype} {tuple(t.shape)}{'' if t.is_contiguous() else ' (strided)'}")


def _vector(t: torch.Tensor | None, name: str, dtype: torch.dtype, n: int) -> int | None:
    if t is None:
        return None
    _check(t, name, dtype, (n,))
    return t.data_ptr()


def _status(status: torch.Tensor | None) -> int | None:
    return _vector(status, "status", torch.int32, 1)


def _launch(device: torch.device, what: str, entry, *args) -> None:
    """Call ``entry`` with the device current and its current stream as the last argument."""
    if device.index == torch.cuda.current_device():
        rc = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc, what)


# -------------------------------------------------------------------------------- attention
def prefix_attention_workspace(max_rows: int, num_seqs: int, num_groups: int, num_heads: int, num_kv_heads: int,
                               max_q_len: int, max_context: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """A workspace for ``prefix_attention`` calls within these bounds. Calls that may overlap (on
    different streams, or two captured graphs replayed side by side) need one each."""
    n = int(_lib.load().ne_prefix_attention_workspace_bytes(max_rows, num_seqs, num_groups, num_heads, num_kv_heads,
                                                            max_q_len, max_context))
    if n == 0:
        raise ValueError("negative bounds, or heads that do not divide into KV heads")
    return torch.empty(n, dtype=torch.uint8, device=device)


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     q_start: torch.Tensor, q_len: torch.Tensor, positions: torch.Tensor, entry_group: torch.Tensor,
                     prefix_blocks: torch.Tensor, *, max_q_len: int, max_context: int, max_prefix: int,
                     k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                     table_index: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of ``q`` [rows, heads, 128] (bf16) over a paged cache, with the prefixes that
    groups of sequences share read once per group.

    ``k_cache`` / ``v_cache`` [slots, KV heads, 128] are one layer's pool (the last slot is scratch),
    bf16, or int8 with ``k_scale`` / ``v_scale`` [slots, KV heads] bf16. Entry b has the rows
    ``q_start[b] .. + q_len[b]`` at the ascending ``positions`` [rows] and the block-table row b
    (``table_index[b]`` if given) of ``block_tables`` [*, blocks]; its group is ``entry_group[b]``
    (-1: none), whose members share their first ``prefix_blocks[group]`` blocks. The bounds
    ``max_q_len``, ``max_context`` and ``max_prefix`` (tokens) are the host's: they size the launch,
    and a captured call keeps them. Rows of no entry are left as they are in ``out``."""
    rows = q.shape[0] if q.dim() == 3 else 0
    heads = q.shape[1] if q.dim() == 3 else 0
    n = q_len.shape[0] if q_len.dim() == 1 else -1
    device = _device_of(q, k_cache=k_cache, v_cache=v_cache, block_tables=block_tables, q_start=q_start, q_len=q_len,
                        positions=positions, entry_group=entry_group, prefix_blocks=prefix_blocks, k_scale=k_scale,
                        v_scale=v_scale, table_index=table_index, out=out, workspace=workspace, status=status)
    _check(q, "q", torch.bfloat16, (rows, heads, HEAD_DIM))
    int8 = k_cache.dtype == torch.int8
    if k_cache.dim() != 3:
        raise ValueError("k_cache must be [slots, KV heads, 128]")
    slots, nkv = k_cache.shape[0], k_cache.shape[1]
    cache_type = torch.int8 if int8 else torch.bfloat16
    _check(k_cache, "k_cache", cache_type, (slots, nkv, HEAD_DIM))
    _check(v_cache, "v_cache", cache_type, (slots, nkv, HEAD_DIM))
    if int8 != (k_scale is not None) or int8 != (v_scale is not None):
        raise ValueError("an int8 cache needs k_scale and v_scale, a bf16 one has none")
    if int8:
        _check(k_scale, "k_scale", torch.bfloat16, (slots, nkv))
        _check(v_scale, "v_scale", torch.bfloat16, (slots, nkv))
    if n < 0 or nkv < 1 or heads % nkv:
        raise ValueError(f"{heads} heads over {nkv} KV heads, q_len of shape {tuple(q_len.shape)}")
    if block_tables.dim() != 2 or (table_index is None and block_tables.shape[0] < n):
        raise ValueError("block_tables must be [entries, blocks]")
    _check(block_tables, "block_tables", torch.int32, tuple(block_tables.shape))
    groups = prefix_blocks.shape[0] if prefix_blocks.dim() == 1 else -1
    table = _lib.PrefixGroups(num_groups=groups, max_prefix_blocks=-(-max_prefix // BLOCK_SIZE),
                              entry_group=_vector(entry_group, "entry_group", torch.int32, n),
                              prefix_blocks=_vector(prefix_blocks, "prefix_blocks", torch.int32, groups))
    if out is None:
        out = torch.zeros_like(q)
    else:
        _check(out, "out", torch.bfloat16, tuple(q.shape))
    if rows == 0 or n == 0 or max_q_len <= 0:
        return out
    if workspace is None:
        workspace = prefix_attention_workspace(rows, n, groups, heads, nkv, max_q_len, max_context, device)
    elif workspace.dtype != torch.uint8 or workspace.dim() != 1 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 vector (prefix_attention_workspace)")
    desc = _lib.Rows(max_rows=rows, num_seqs=n, positions=_vector(positions, "positions", torch.int32, rows),
                     q_start=_vector(q_start, "q_start", torch.int32, n),
                     q_len=_vector(q_len, "q_len", torch.int32, n), block_tables=block_tables.data_ptr(),
                     table_index=_vector(table_index, "table_index", torch.int32, n),
                     block_table_stride=block_tables.shape[1], max_context=max_context, max_q_len=max_q_len)
    _launch(device, "ne_prefix_attention", _lib.load().ne_prefix_attention, q.data_ptr(), out.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale), int(int8),
            ctypes.byref(desc), ctypes.byref(table), heads, nkv, BLOCK_SIZE, slots, workspace.data_ptr(),
            workspace.numel(), _status(status))
    return out


# -------------------------------------------------------------------------------- sampling
def sample_logits(logits: torch.Tensor, uniform: torch.Tensor, temperature: torch.Tensor | None = None,
                  top_k: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                  min_p: torch.Tensor | None = None, *,
                  status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token per row of ``logits`` [rows, vocab] (bf16 or fp32; rows may be strided) drawn with
    ``uniform`` [rows] (fp32, in [0, 1)) from the row's distribution after temperature, top-k, top-p
    and min-p (vectors of one value per row, or None): tokens [rows] int32 and their probabilities
    [rows] fp32. Temperature 0 takes the argmax. The exact rules are ne_sample_logits's."""
    device = _device_of(logits, uniform=uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                        status=status)
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or logits.stride(1) != 1:
        raise ValueError("logits must be [rows, vocab] in bf16 or fp32, each row contiguous")
    rows, vocab = logits.shape
    if vocab < 1 or (rows > 1 and logits.stride(0) < vocab):
        raise ValueError("logits need at least one token, and rows that do not overlap")
    tokens = torch.empty(rows, dtype=torch.int32, device=device)
    probs = torch.empty(rows, dtype=torch.float32, device=device)
    pointers = [_vector(uniform, "uniform", torch.float32, rows), _vector(temperature, "temperature", torch.float32, rows),
                _vector(top_k, "top_k", torch.int32, rows), _vector(top_p, "top_p", torch.float32, rows),
                _vector(min_p, "min_p", torch.float32, rows)]
    if rows:
        _launch(device, "ne_sample_logits", _lib.load().ne_sample_logits, logits.data_ptr(),
                int(logits.dtype == torch.float32), rows, vocab, max(logits.stride(0), vocab), *pointers[1:],
                pointers[0], tokens.data_ptr(), probs.data_ptr(), _status(status))
    return tokens, probs


# -------------------------------------------------------------------------------- pages
def copy_kv_blocks(kv: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, *, scales: torch.Tensor | None = None,
                   count: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Copy block ``src[i]`` to block ``dst[i]`` in every layer, K and V, of the pool ``kv``
    [layers, 2, slots, KV heads, 128] (bf16, or int8 with ``scales`` [layers, 2, slots, KV heads]).
    ``src`` / ``dst`` are int32 vectors on the device, ``count`` (one int32 on the device) limits the
    pairs to its value. No block may be written by one pair and read or written by another."""
    device = _device_of(kv, src=src, dst=dst, scales=scales, count=count, status=status)
    if kv.dim() != 5 or kv.dtype not in (torch.bfloat16, torch.int8):
        raise ValueError("kv must be [layers, 2, slots, KV heads, 128] in bf16 or int8")
    layers, _, slots, nkv, _ = kv.shape
    _check(kv, "kv", kv.dtype, (layers, 2, slots, nkv, HEAD_DIM))
    int8 = kv.dtype == torch.int8
    if int8 != (scales is not None):
        raise ValueError("an int8 pool needs its scales, a bf16 one has none")
    if int8:
        _check(scales, "scales", torch.bfloat16, (layers, 2, slots, nkv))
    pairs = src.shape[0] if src.dim() == 1 else -1
    _launch(device, "ne_kv_copy_blocks", _lib.load().ne_kv_copy_blocks, kv.data_ptr(), _lib.ptr(scales), int(int8),
            layers, nkv, slots, _vector(src, "src", torch.int32, pairs), _vector(dst, "dst", torch.int32, pairs),
            _vector(count, "count", torch.int32, 1), pairs, _status(status))
