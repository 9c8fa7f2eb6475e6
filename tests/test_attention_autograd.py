"""The cache and attention operators beside autograd: they have no gradient, and say so."""
from __future__ import annotations

import pytest
import torch

from flashgann_amd import attention


def tensors(device):
    """Arguments of each call that may carry a gradient, and the others."""
    z = lambda *s, d=torch.bfloat16: torch.zeros(s, dtype=d, device=device)  # noqa: E731
    cache = dict(k_cache=z(4, 16, 2, 64), v_cache=z(4, 16, 2, 64))
    table, starts, lens = z(2, 2, d=torch.int32), z(3, d=torch.int32), z(2, d=torch.int32)
    return ((attention.attend, dict(q=z(3, 4, 64), **cache), dict(block_table=table, q_starts=starts, kv_lens=lens, max_q=1)),
            (attention.attend_retrieved, dict(q=z(2, 4, 64), **cache),
             dict(block_table=table, kv_lens=lens, ids=z(2, 2, 5, d=torch.int32), window=2)),
            (attention.cache_append, dict(k=z(3, 2, 64), v=z(3, 2, 64), **cache), dict(slots=z(3, d=torch.int64))))


def test_gradients_are_refused():
    """With autograd on, before anything else is looked at."""
    for call, maybe, rest in tensors("cpu"):
        for name in maybe:
            with pytest.raises(ValueError, match="gradient"):
                call(**{**maybe, name: maybe[name].clone().requires_grad_()}, **rest)
        with pytest.raises(ValueError, match="CUDA device"):
            call(**maybe, **rest)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call(**{n: t.clone().requires_grad_() for n, t in maybe.items()}, **rest)


@pytest.mark.gpu
def test_without_autograd(gpu_available):
    """Under no_grad, under inference_mode and detached the same tensors are taken."""
    for call, maybe, rest in tensors("cuda"):
        asking = {n: t.clone().requires_grad_() for n, t in maybe.items()}
        with pytest.raises(ValueError, match="gradient"):
            call(**asking, **rest)
        with torch.no_grad():
            call(**asking, **rest)
        with torch.inference_mode():
            call(**asking, **rest)
        call(**{n: t.detach() for n, t in asking.items()}, **rest)
    attend, maybe, rest = tensors("cuda")[0]
    for name, like in (("out", maybe["q"]), ("lse", torch.zeros((3, 4), device="cuda"))):
        with pytest.raises(ValueError, match="gradient"):
            attend(**maybe, **rest, **{name: like.clone().requires_grad_()})


@pytest.mark.gpu
def test_writes_in_place_are_counted(gpu_available):
    """What autograd saved and a call then overwrote is found out, as with torch's own writes."""
    (attend, maybe, rest), _, (append, rows, slots) = tensors("cuda")
    out, lse = torch.zeros_like(maybe["q"]), torch.zeros((3, 4), device="cuda")
    saved = [rows["k_cache"], rows["v_cache"], out, lse, rest["block_table"]]
    before = [t._version for t in saved]
    append(**rows, **slots)
    assert [t._version for t in saved] == [before[0] + 1, before[1] + 1, *before[2:]]
    attend(**maybe, **rest, out=out, lse=lse)
    attention.cache_plan(rest["kv_lens"], rest["kv_lens"], rest["block_table"], rest["kv_lens"], page_size=16, max_tokens=0)
    assert [t._version for t in saved] == [v + 1 for v in before]
    weight = torch.ones((), device="cuda", requires_grad=True)
    loss = (weight * rows["k_cache"]).sum()
    append(**rows, **slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # such tensors have no counter
        held = torch.zeros_like(rows["k_cache"])
        append(rows["k"], rows["v"], held, held.clone(), **slots)
    append(rows["k"], rows["v"], held, held, **slots)
