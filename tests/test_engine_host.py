"""Host-side decisions of the batched engine, on a host without a GPU: the launches are stood in for."""

from __future__ import annotations

import pytest

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
