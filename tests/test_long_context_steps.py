"""The decode example takes no step whose tokens neither the index nor the window would hold."""
from __future__ import annotations

import pytest


def test_more_steps_than_window(capsys):
    from flashgann_amd import long_context
    with pytest.raises(ValueError, match="steps"):
        long_context.LongContext(tokens=100, steps=9, window=8)
    with pytest.raises(SystemExit):
        long_context.main(["--tokens", "100", "--steps", "9", "--window", "8"])
    assert "--steps must be at most --window" in capsys.readouterr().err


@pytest.mark.gpu
def test_no_step_past_the_last(gpu_available):
    """The last token of the last step still sees the first one after the index; one more step is refused."""
    import torch
    from flashgann_amd.long_context import LongContext
    ctx = LongContext(tokens=600, steps=2, heads=2, heads_kv=1, dim=64, k=8, beam=64, window=2, sinks=1)
    try:
        steps = [ctx.step() for _ in range(2)]
        assert [s.kv_lens.tolist() for s in steps] == [[601], [602]] and all(bool(torch.isfinite(s.lse).all()) for s in steps)
        with pytest.raises(RuntimeError, match="step"):
            ctx.step()
    finally:
        ctx.close()
