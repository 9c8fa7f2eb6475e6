"""Search, cache and attention together: the decode steps of
flashgann_amd.long_context against the 64-bit oracle on what the searches found."""
from __future__ import annotations

import pytest
import torch

import attention_oracle as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,heads_kv,dtype", ((128, 8, 2, torch.bfloat16), (96, 6, 1, torch.float16)))
def test_decode_over_an_index(gpu_available, dim, heads, heads_kv, dtype):
    from flashgann_amd.long_context import LongContext
    torch.cuda.set_device(0)
    ctx = LongContext(tokens=3000, steps=3, heads=heads, heads_kv=heads_kv, dim=dim, k=40, beam=128, window=32, sinks=4, dtype=dtype)
    try:
        for i in range(3):
            s = ctx.step()
            kv = [3001 + i]
            assert s.kv_lens.tolist() == kv
            q, k, v, table, ids = (t.cpu() for t in (s.q, ctx.k_cache, ctx.v_cache, ctx.table, s.ids))
            assert int(ids.min()) >= 0 and int(ids.max()) < 3000
            A.retrieved(q, k, v, table, kv, ids, dim ** -0.5, 32, 4).check(s.out, s.lse)
            A.dense(q, k, v, table, [0, 1], kv, dim ** -0.5).check(s.all_out, s.all_lse)
            # what was found adds to the first and the last tokens' weight and stays below all tokens'
            few = A.retrieved(q, k, v, table, kv, ids[:, :, :0], dim ** -0.5, 32, 4).lse
            assert bool((s.lse <= s.all_lse + 1e-4).all()) and bool((s.lse.cpu().double() > torch.from_numpy(few)).all())
    finally:
        ctx.close()


def test_command_line(gpu_available, capsys):
    from flashgann_amd import long_context
    assert long_context.main(["--tokens", "2000", "--steps", "2", "--k", "64", "--beam", "128"]) == 0
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 2 and "2002 tokens" in lines[1]
