"""Draws with temperature, top-k, top-p and min-p from given random numbers (``ops.sample_logits``)
against the definition in 64 bits on the host: tokens equal, probabilities within a few roundings."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.conftest import submodule

pytestmark = pytest.mark.gpu

SETTINGS = [(0.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.7, 20, 0.8, 0.0), (1.0, 50, 1.0, 0.0), (0.8, 0, 0.9, 0.0),
            (1.0, 0, 1.0, 0.05), (1.2, 200, 0.95, 0.02), (1.0, 0, 1.0, 0.0), (1.5, 0, 0.999, 0.0), (1.0, 1, 1.0, 0.0),
            (3.0, 5000, 0.7, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (0.05, 0, 0.5, 0.3), (1.0, 1 << 30, 1.0, -1.0)]


@pytest.fixture(scope="module")
def ops(cuda_device):
    submodule("build").build()
    return submodule("ops")


def expected(x, temperature, top_k, top_p, min_p, u, short=0.0):
    """(token, probability) of one row by the definition, in 64 bits; ``short``: taken off the mass that
    top-p is a share of."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    vocab, top = len(x), x.max()
    if top == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / temperature)))
    ranked = np.lexsort((np.arange(vocab), -x))
    if 0 < top_k < vocab:
        ranked = ranked[:top_k]
    mass = np.cumsum(w[ranked])
    kept = len(ranked)
    if top_p < 1:
        kept = min(kept, max(1, int((mass - w[ranked] < top_p * (mass[-1] - short)).sum())))
    if min_p > 0:
        kept = min(kept, max(1, int((w[ranked] >= min_p).sum())))
    ids = np.sort(ranked[:kept])
    p = w[ids]
    below = np.cumsum(p)
    at = min(int(np.searchsorted(below, u * below[-1], side="right")), kept - 1)
    return int(ids[at]), float(p[at] / below[-1])


def check(ops, logits, settings, uniform, **kw):
    dev = logits.device
    rows = logits.shape[0]
    columns = [torch.tensor([s[i] for s in settings], dtype=torch.int32 if i == 1 else torch.float32, device=dev)
               for i in range(4)]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    tokens, probs = ops.sample_logits(logits, uniform, *columns, status=status, **kw)
    host, u = logits.float().cpu().numpy(), uniform.cpu().numpy().astype(np.float64)
    floats = [c.cpu().numpy().astype(np.float64) for c in columns]
    for r in range(rows):
        row = (host[r], floats[0][r], int(columns[1][r]), floats[2][r], floats[3][r], u[r])
        token, p = expected(*row)
        if int(tokens[r]) != token:
            # Sums are in steps of 2^-45, a weight rounded down to them: V weights are short by less than
            # V 2^-45. The border of top-p may lie that much lower, and then leave out a token that starts
            # within it (seen: weights 1, 1, 8e-15 with top_p 0.5, where the second starts at 1 of 1 + 4e-15).
            token, p = expected(*row, short=logits.shape[1] * 2.0 ** -45)
        assert int(tokens[r]) == token, (r, settings[r], float(u[r]))
        # weights in 64 bits, sums in 2^-45 steps, one rounding to fp32
        assert abs(float(probs[r]) - p) <= 2.0 ** -23 * p + 1e-9, (r, settings[r])
    return tokens, probs, int(status.item())


def language_logits(rows, vocab, seed, device, dtype):
    g = torch.Generator(device=device).manual_seed(seed)
    rank = torch.argsort(torch.rand((rows, vocab), generator=g, device=device), dim=-1).float() + 1
    slope = torch.rand((rows, 1), generator=g, device=device) * 1.5 + 1
    x = 15 - slope * torch.log(rank) + torch.randn((rows, vocab), generator=g, device=device)
    u = torch.randint(0, 1 << 24, (rows,), generator=g, device=device).float() * 2.0 ** -24
    return x.to(dtype), u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 100, 1000, 4096, 8192, 8193, 16387, 50021, 151936, 262144])
def test_matches_the_definition(ops, cuda_device, vocab, dtype) -> None:
    logits, u = language_logits(len(SETTINGS), vocab, vocab, cuda_device, dtype)
    _, _, status = check(ops, logits, SETTINGS, u)
    assert status == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_many_rows(ops, cuda_device, dtype) -> None:
    rows = 200
    logits, u = language_logits(rows, 12345, 3, cuda_device, dtype)
    check(ops, logits, [SETTINGS[r % len(SETTINGS)] for r in range(rows)], u)


@pytest.mark.parametrize("rows", [297, 511, 512, 513, 1025, 4097])
@pytest.mark.parametrize("kind", ["mixed", "all slow", "none slow", "no temperature or top-k"])
def test_more_rows_than_run_at_once(ops, cuda_device, rows, kind) -> None:
    """Rows are taken in another order than they lie in: each is drawn, and with its own settings."""
    logits, u = language_logits(rows, 300, rows, cuda_device, torch.bfloat16)
    if kind == "no temperature or top-k":
        top_p = torch.tensor([(0.9, 1.0, 0.5)[r % 3] for r in range(rows)], device=cuda_device)
        tokens, _ = ops.sample_logits(logits, u, None, None, top_p)
        host, v = logits.float().cpu().numpy(), u.cpu().numpy().astype(np.float64)
        want = [expected(host[r], 1.0, 0, float(top_p[r]), 0.0, v[r])[0] for r in range(rows)]
        assert tokens.tolist() == want
        return
    settings = {"mixed": SETTINGS, "all slow": [(0.8, 0, 0.9, 0.0)], "none slow": [(0.0, 0, 0.5, 0.0), (1.0, 20, 0.9, 0.0)]}[kind]
    g = torch.Generator().manual_seed(rows)
    pick = torch.randint(0, len(settings), (rows,), generator=g).tolist()
    check(ops, logits, [settings[i] for i in pick], u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
def test_ties_go_to_the_lowest_ids(ops, cuda_device, vocab, dtype) -> None:
    """A handful of distinct values: every cut falls inside a group of equal logits."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randint(0, 5, (len(SETTINGS), vocab), generator=g).to(dtype).to(cuda_device)
    logits[3] = 1.5   # all equal
    logits[7] = -2.0
    logits[4] = 0.0
    logits[4, ::2] = -0.0  # equal to 0
    u = torch.rand(len(SETTINGS), generator=g).to(cuda_device)
    check(ops, logits, SETTINGS, u)


def test_first_and_last_random_number(ops, cuda_device) -> None:
    for u in (0.0, 1.0 - 2.0 ** -24):
        logits, uniform = language_logits(len(SETTINGS), 20000, 9, cuda_device, torch.bfloat16)
        uniform.fill_(u)
        check(ops, logits, SETTINGS, uniform)
    # a number of 1 or more takes the last kept token, one below 0 or NaN the first
    logits = torch.zeros(3, 10, device=cuda_device)
    tokens, probs = ops.sample_logits(logits, torch.tensor([1.0, -1.0, float("nan")], device=cuda_device))
    assert tokens.tolist() == [9, 0, 0]
    torch.testing.assert_close(probs, torch.full_like(probs, 0.1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_masked_infinite_and_nan_logits(ops, cuda_device, dtype) -> None:
    n = len(SETTINGS)
    logits, u = language_logits(n, 9001, 21, cuda_device, dtype)
    logits[:, ::3] = float("-inf")
    logits[:, 1::7] = float("nan")
    logits[:, 5] = torch.finfo(dtype).min
    _, _, status = check(ops, logits, SETTINGS, u)
    assert status == 0
    logits[:, 100] = float("inf")
    logits[:, 7000] = float("inf")
    logits[2, 7000] = float("nan")
    _, _, status = check(ops, logits, SETTINGS, u)
    assert status == 0
    only = torch.full_like(logits, float("-inf"))
    only[:, 4444] = -3.0
    check(ops, only, SETTINGS, u)
    only[1] = float("-inf")
    only[4] = float("nan")
    tokens, probs, status = check(ops, only, SETTINGS, u)
    assert status == 8 and tokens[1] == -1 and probs[4] == 0


def test_extreme_temperatures(ops, cuda_device) -> None:
    logits, u = language_logits(6, 3000, 5, cuda_device, torch.float32)
    settings = [(1e-6, 0, 1.0, 0.0), (1e-6, 0, 0.9, 0.0), (1e4, 0, 0.5, 0.0), (1e4, 700, 0.5, 0.0), (1e30, 0, 1.0, 0.0),
                (1e30, 0, 0.3, 0.5)]
    check(ops, logits, settings, u)


@pytest.mark.parametrize("temperature", [1e-1, 1e-3, 1e-5, 1e-6, 1e-7, 3e-8, 1e-8, 1e-12, 1e-30, 1e-42])
@pytest.mark.parametrize("top", [20.0, -37.7, 0.0])
def test_low_temperatures_beside_near_ties(ops, cuda_device, temperature, top) -> None:
    """Logits a few units in the last place (or a few temperatures) below the largest one."""
    g = torch.Generator().manual_seed(int(-math.log10(temperature)))
    n, vocab = 8, 3000
    step = max(temperature, np.spacing(np.float32(top)) / 2) if top else temperature
    near = top - torch.randint(0, 60, (n, vocab), generator=g).double() * step * 0.7
    logits = torch.where(torch.rand((n, vocab), generator=g) < 0.9, torch.tensor(top - 1.0).double(), near).float()
    settings = [(temperature, 0, 1.0, 0.0), (temperature, 0, 0.9, 0.0), (temperature, 40, 0.95, 0.01), (temperature, 0, 1.0, 1.0),
                (temperature, 0, 0.9, 1.0), (temperature, 0, 0.5, 2.0), (temperature, 2000, 0.999, 0.0), (temperature, 0, 1.0, 1e-6)]
    check(ops, logits.to(cuda_device), settings, torch.rand(n, generator=g).to(cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_logits_far_from_zero(ops, cuda_device, dtype) -> None:
    """A shift of all logits changes nothing but what it rounds away."""
    for shift in (300.0, -4096.0, 1e5, -3e7):
        logits, u = language_logits(len(SETTINGS), 9000, 31, cuda_device, torch.float32)
        check(ops, (logits + shift).to(dtype), SETTINGS, u)


def test_temperatures_up_to_infinity(ops, cuda_device) -> None:
    logits, u = language_logits(8, 3000, 41, cuda_device, torch.float32)
    logits[:, 5::9] = float("-inf")
    logits[:, 7::50] = torch.finfo(torch.float32).min
    inf = float("inf")
    check(ops, logits, [(inf, 0, 1.0, 0.0), (inf, 0, 0.4, 0.0), (inf, 30, 0.5, 0.0), (inf, 0, 1.0, 0.5), (1e31, 0, 0.7, 0.0),
                        (1e36, 0, 1.0, 0.0), (1e36, 2500, 0.9, 0.0), (1e36, 0, 1.0, 1.0)], u)
    logits = logits.sign() * 3.3e38  # differences that overflow
    logits[:, 0] = 3.3e38
    check(ops, logits, [(1e36, 0, 1.0, 0.0)] * 4 + [(1e36, 0, 0.9, 0.0)] * 4, u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_min_p_above_one_keeps_one_token(ops, cuda_device, dtype) -> None:
    logits = torch.zeros((6, 500), dtype=dtype, device=cuda_device)
    u = torch.linspace(0, 0.99, 6, device=cuda_device)
    check(ops, logits, [(1.0, 0, 1.0, 1.5), (1.0, 0, 0.9, 1.5), (1.0, 40, 1.0, 1.5), (0.5, 40, 0.5, 7.0), (1.0, 400, 0.9, 1.1),
                        (1.0, 0, 1.0, float("inf"))], u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strided_and_misaligned_rows(ops, cuda_device, dtype) -> None:
    for vocab, width, shift in ((1001, 1003, 0), (1001, 1008, 3), (9000, 9001, 1), (17, 40, 5)):
        base, u = language_logits(len(SETTINGS), width, vocab, cuda_device, dtype)
        check(ops, base[:, shift: shift + vocab], SETTINGS, u)


def test_no_settings_is_a_plain_draw_and_none_equals_neutral(ops, cuda_device) -> None:
    logits, u = language_logits(32, 6000, 6, cuda_device, torch.bfloat16)
    plain, p0 = ops.sample_logits(logits, u)
    neutral, p1 = ops.sample_logits(logits, u, torch.ones(32, device=cuda_device),
                                    torch.zeros(32, dtype=torch.int32, device=cuda_device),
                                    torch.ones(32, device=cuda_device), torch.zeros(32, device=cuda_device))
    assert torch.equal(plain, neutral) and torch.equal(p0, p1)
    check(ops, logits, [(1.0, 0, 1.0, 0.0)] * 32, u)


def test_equals_the_sampled_steps_draw(ops, cuda_device) -> None:
    """A draw without guesses in the verify step (temperature and top-p on a Philox stream) takes the
    same token as this operator with the stream's uniform."""
    serial = submodule("serial")
    from oracle.philox import uniform as philox_uniform
    logits, _ = language_logits(24, 4096, 8, cuda_device, torch.bfloat16)

    class Params:
        temperature, top_p = 0.9, 0.85

    for r in range(24):
        gen = serial.PhiloxGenerator(1000 + r)
        want = serial._logits_verifier(cuda_device).verify([], logits[r: r + 1], Params, gen)
        u = torch.tensor([float(philox_uniform(1000 + r, 0))], device=cuda_device)
        got, _ = ops.sample_logits(logits[r: r + 1], u, torch.tensor([0.9], device=cuda_device), None,
                                   torch.tensor([0.85], device=cuda_device))
        assert got.tolist() == want


def test_capture_and_side_stream(ops, cuda_device) -> None:
    logits, u = language_logits(len(SETTINGS), 30000, 12, cuda_device, torch.bfloat16)
    columns = [torch.tensor([s[i] for s in SETTINGS], dtype=torch.int32 if i == 1 else torch.float32,
                            device=cuda_device) for i in range(4)]
    want, _ = ops.sample_logits(logits, u, *columns)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = ops.sample_logits(logits, u, *columns)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, _ = ops.sample_logits(logits, u, *columns)
    other, u2 = language_logits(len(SETTINGS), 30000, 13, cuda_device, torch.bfloat16)
    logits.copy_(other)
    u.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    want, _ = ops.sample_logits(other, u2, *columns)
    assert torch.equal(got, want)


def test_no_rows_and_refusals(ops, cuda_device) -> None:
    tokens, probs = ops.sample_logits(torch.zeros(0, 8, device=cuda_device), torch.zeros(0, device=cuda_device))
    assert tokens.shape == (0,) and probs.shape == (0,)
    logits, u = torch.zeros(2, 8, device=cuda_device), torch.zeros(2, device=cuda_device)
    for args in ((logits.half(), u), (logits.t(), u), (logits, u[:1]), (logits, u.double()), (logits[:, ::2], u),
                 (logits[0], u), (torch.zeros(1, 8, device=cuda_device).expand(2, 8), u), (logits, u, None, u)):
        with pytest.raises(ValueError):
            ops.sample_logits(*args)
    with pytest.raises(submodule("_lib").NativeError):
        ops.sample_logits(torch.zeros(1, 262145, device=cuda_device), u[:1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("edge", [38704, 77408, 163776])
def test_either_side_of_the_slices_that_two_ctas_hold(ops, cuda_device, edge, dtype) -> None:
    """Vocabularies at which a row's cluster grows, and rows that start at once on one side only."""
    vocab = edge if dtype == torch.bfloat16 else edge // 2
    for v in (vocab - 1, vocab, vocab + 1, vocab + 500):
        logits, u = language_logits(45, v, v, cuda_device, dtype)
        _, _, status = check(ops, logits, [SETTINGS[r % len(SETTINGS)] for r in range(45)], u)
        assert status == 0
