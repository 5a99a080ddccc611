"""Edges of the cache held in 8 bits: values that are no numbers next to what a query sees, rows beside each other, workspaces,
and requests that are set back."""

import math

import pytest
import torch
from plain import q8_plain as plain
from test_q8_cache_gpu import DEV, Cache, attend_on_device, i32, starts, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,hd,page", [(8, 2, 128, 64), (8, 1, 64, 16), (16, 1, 128, 16), (6, 3, 48, 12), (8, 1, 256, 64), (2, 2, 32, 5)])
@pytest.mark.parametrize("window,rows", [
    (20, [(40, 1), (52, 1), (83, 1), (84, 1), (115, 1), (19, 1)]), (300, [(330, 1), (900, 1), (1023, 1)]), (33, [(70, 3), (95, 2)])])
def test_no_numbers_in_front_of_a_window(dtype, H, G, hd, page, window, rows, monkeypatch):
    """What the first query of a row does not see any more may hold NaN, in its keys and in its values: the row's
    outputs are those of the keys that are seen."""
    from scratch_llm_b200.kernels import ops
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: False)
    gen = torch.Generator().manual_seed(hd + window)
    c = Cache(G, hd, page, 1, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    for r, (before, _) in enumerate(rows):
        for pos in range(max(0, before - window + 1)):
            c.pages[int(c.table[r, pos // page]), :, :, pos % page] = 0x7F
    q = torch.randn(sum(m for _, m in rows), H * hd, generator=gen).to(dtype)
    for context in (None, 4096):
        got = attend_on_device(c, q.to(DEV), rows, c.device(), H, hd ** -0.5, window, context=context).double().cpu()
        want, spread, reach = plain.attend(q, c.pages, c.scales, c.table, rows, page, H, G, hd, hd ** -0.5, window)
        assert not want.isnan().any() and not got.isnan().any()
        assert ((got - want).abs() <= tolerance(dtype, hd, want, spread, reach)).all()
