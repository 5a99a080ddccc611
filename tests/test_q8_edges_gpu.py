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


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("planes", [(1,), (0, 1)])
def test_portions_beside_a_row_with_no_numbers(window, planes, monkeypatch):
    """Portions by way of 16 bits: a NaN in one row leaves the other rows' bits as they are, and of its own row those of the
    queries far in front of it and of the other kv heads; what sees it, or stands beside it in a tile, is right."""
    from scratch_llm_b200.kernels import ops
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: True)
    H, G, hd, page = 8, 2, 64, 16
    rows = [(300, 200), (20, 300), (0, 33), (250, 150)]
    gen = torch.Generator().manual_seed(31)
    c = Cache(G, hd, page, 8, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    q = torch.randn(sum(m for _, m in rows), H * hd, generator=gen).bfloat16()
    clean = attend_on_device(c, q.to(DEV), rows, c.device(), H, hd ** -0.5, window)
    bad = [(1, 250, 5), (3, 3, 9), (3, 280, 63)]                  # row, position, entry
    for r, pos, d in bad:
        for plane in planes:
            c.pages[int(c.table[r, pos // page]), plane, 1, pos % page, d] = 0xFF
    dev = c.device()
    for row_list in (None, [3, 0, 1]):
        got = attend_on_device(c, q.to(DEV), rows, dev, H, hd ** -0.5, window, row_list=row_list)
        s = starts(rows)
        for r in (0, 2):
            if row_list is None or r in row_list:
                assert torch.equal(got[s[r]:s[r + 1]], clean[s[r]:s[r + 1]])
        same = lambda a, z: torch.equal(got[a:z].view(-1, H, hd)[:, :4], clean[a:z].view(-1, H, hd)[:, :4])  # noqa: E731
        assert same(s[1], s[2]) and same(s[3], s[4])
        assert torch.equal(got[s[1]:s[1] + 100], clean[s[1]:s[1] + 100])
        for r in (1, 3):
            part = slice(s[r], s[r + 1])
            only = [(0, 0) if i != r else row for i, row in enumerate(rows)]
            want, spread, reach = plain.attend(q[part], c.pages, c.scales, c.table, only, page, H, G, hd, hd ** -0.5, window)
            mine = got[part].double().cpu()
            assert torch.equal(mine.isnan(), want.isnan()) and want.isnan().any() and not want.isnan().all()
            tol = tolerance(torch.bfloat16, hd, want, spread, reach, True)
            assert ((mine - want).abs() <= tol)[~want.isnan()].all()


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("hd", [64, 128, 48])
def test_small_probabilities_beside_a_key_of_zeros_in_32_bits(new, hd):
    """One key with nearly all of the probability and values of zero, as an attention sink has: the output comes from keys
    with probabilities of 2^-17 to 2^-20 of it.  In units of sum_j p_j |v_j|: a probability as two halves, the second scaled
    by 2^11, is off by at most 2^-36 against 2^5 * 2^-20 or more, 2^-21; scores are products of one entry, exact but
    for three roundings (scale, its unit, their product) of at most 10 (base 2), for the key and for the sink 2 * 30 * 2^-24,
    2^-18; the exponentials 2^-22 each; sums over 64 to 68 keys at most 2^-18 (16 keys an instruction, cut off at
    2^-23 of the sum's largest part, and five additions, for each of a warp's tiles), the meeting of four warps, the
    denominator, the division and the result 2^-20: less than 2^-16.5 together."""
    H, G, page, n = 4, 2, 16, 63
    gen = torch.Generator().manual_seed(hd)
    c = Cache(G, hd, page, 16, [n + new], gen).fill([(n + new, 0)], gen, 0.0)
    e4m3 = lambda x: plain.round_e4m3(torch.tensor(x).double()).view(torch.uint8)  # noqa: E731
    for pos in range(n + new):
        at, cell = int(c.table[0, pos // page]), pos % page
        c.scales[at, 0] = 127
        c.pages[at, 0, :, cell] = 0
        c.pages[at, 0, :, cell, 0] = e4m3(10.0 if pos == 0 else -8.0 - pos % 3)
        if pos == 0:
            c.pages[at, 1, :, cell] = 0
    q = torch.zeros(new, H, hd)
    q[:, :, 0] = 8.0
    scale = 0.97 * math.log(2.0) / 8.0
    rows = [(n, new)]
    got = attend_on_device(c, q.view(new, -1).to(DEV), rows, c.device(), H, scale).double().cpu()
    want, spread, _ = plain.attend(q.view(new, -1), c.pages, c.scales, c.table, rows, page, H, G, hd, scale)
    far = ((got - want).abs() / spread).max()
    assert far <= 2.0 ** -16.5, f"{float(far):.3g} of sum p |v|"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("listed", [[1], [2, 1], [3]])
def test_workspace_of_the_listed_rows(listed, dtype):
    """What a launch sets aside for the parts of its sums goes by the rows that it is asked for, not by the step's tokens."""
    H, G, hd, page = 16, 4, 128, 64
    rows = [(0, 3000), (8191, 1), (5000, 1), (6000, 3)]
    gen = torch.Generator().manual_seed(3)
    c = Cache(G, hd, page, 64, [b + m for b, m in rows], gen).fill([(b + m, 0) if r else (0, 0) for r, (b, m) in enumerate(rows)], gen, 0.5)
    n, s = sum(m for _, m in rows), starts(rows)
    q = torch.randn(n, H * hd, generator=gen).to(dtype)
    dev, out, on = c.device(), torch.full((n, H * hd), 7.0, dtype=dtype, device=DEV), q.to(DEV)
    attend_on_device(c, on, rows, dev, H, hd ** -0.5, row_list=listed, out=out)      # (what is loaded once)
    out.fill_(7.0)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    attend_on_device(c, on, rows, dev, H, hd ** -0.5, row_list=listed, out=out)
    took = torch.cuda.max_memory_allocated() - before
    # 64 shares at most, each with a head's sums, maximum and denominator for every token that a listed row may bring
    assert took <= 4 * 64 * len(listed) * 3 * H * (hd + 2) + (1 << 16), took
    for r in range(len(rows)):
        part = out[s[r]:s[r + 1]]
        if r not in listed:
            assert (part == 7).all()
            continue
        only = [row if i == r else (0, 0) for i, row in enumerate(rows)]
        want, spread, reach = plain.attend(q[s[r]:s[r + 1]], c.pages, c.scales, c.table, only, page, H, G, hd, hd ** -0.5)
        assert ((part.double().cpu() - want).abs() <= tolerance(dtype, hd, want, spread, reach)).all()


def test_captured_steps_whose_longest_rows_differ(model_dirs, monkeypatch):
    """Steps of the same padded sizes whose longest rows differ share no captured graph that would be too small for one of them,
    and launches are asked for no more than twice the longest row."""
    from configs import PAGE_SIZE
    from plain import llama_plain as P
    from scratch_llm_b200.engine import ModelRunner, RowInput
    from scratch_llm_b200.engine.runner import load_model
    from scratch_llm_b200.kernels import ops
    from test_q8_engine_gpu import PlainModel
    cfg, w = P.read_model_dir(model_dirs["B"])
    runner = ModelRunner(load_model(model_dirs["B"], "float32", verbose=False), PAGE_SIZE["B"], 60, 4, poison_free_pages=True,
                         cache_dtype="float8_e4m3fn")
    runner.capture_padded_after = 2
    asked, call = [], ops.attention_q8

    def attention(*a, **k):
        asked.append(a[10])
        return call(*a, **k)

    monkeypatch.setattr(ops, "attention_q8", attention)
    gen = torch.Generator().manual_seed(4)
    models = {n: PlainModel(cfg, w, PAGE_SIZE["B"], runner.cache.scale_block) for n in "abc"}
    for n in models:
        assert runner.admit(n)
    for step in [dict(a=8, b=8), dict(a=7, b=6), dict(a=5, b=8), dict(a=2, b=14), dict(a=14, b=2), dict(a=3, b=13), dict(a=8, b=8),
                 dict(a=4, b=3, c=3), dict(a=4, b=3, c=3), dict(a=2, b=9, c=2)]:
        ids = {n: torch.randint(0, cfg["vocab_size"], (k,), generator=gen).tolist() for n, k in step.items()}
        asked.clear()
        got = runner.step([RowInput(n, t, [len(t) - 1]) for n, t in ids.items()]).cpu()
        want = torch.cat([models[n].step(t)[-1:] for n, t in ids.items()])
        assert (got - want).norm() / want.norm() < 4e-3
        assert all(max(step.values()) <= m < 2 * max(step.values()) for m in asked)
    assert runner.replayed_steps >= 4


def test_requests_that_are_set_back_read_what_they_wrote(model_dirs):
    """A pool so small that requests are set back and their pages used again (free ones hold NaN): every token's
    log-probability is what the model, with room for all, says of the same tokens.  A request that comes in again stores its
    tokens in other portions; that moves a value only where a block's scale grew in between and the value is a subnormal of it,
    or where a 32-bit rounding lies at the border between two e4m3 numbers (one of a row's thousands, by 2^-3 of itself): some
    thousandths of a nat for this model, where a stale scale or a wrong page moves it by units."""
    from scratch_llm_b200 import LLM, Request, SamplingParams
    from scratch_llm_b200.engine import ModelRunner
    gen = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, 256, (n,), generator=gen).tolist() for n in (30, 25, 28, 9, 33, 20)]
    params = SamplingParams(temperature=0.0, max_tokens=40)
    make = lambda n, **k: LLM(model_dirs["A"], dtype="float32", max_tokens=n, page_size=16, max_requests=4,  # noqa: E731
                              cache_dtype="float8_e4m3fn", **k)
    small, big = make(160), make(2048)
    small.runner = ModelRunner(small.model, 16, 10, 4, poison_free_pages=True, cache_dtype="float8_e4m3fn")
    got = small.serve([Request(i, p, params) for i, p in enumerate(prompts)], want_logprobs=True)
    assert got.stats.preemptions > 0
    worst = 0.0
    for c, prompt in zip(got.completed, prompts):
        tokens = list(c.token_ids)
        assert len(tokens) == 40 and len(c.logprobs) == 40
        worst = max(worst, *(abs(a - b) for a, b in zip(c.logprobs, big.score(prompt, tokens))))
    assert worst < 0.05, worst
    small.runner.cache.check()
    assert not small.runner.cache.requests


@pytest.mark.parametrize("portions", [False, True])
def test_largest_values_reach_only_what_sees_them(portions, monkeypatch):
    """The largest bfloat16 numbers are stored as 2^128, for which bfloat16 has an infinity: queries that do not see them get
    what they get without them."""
    from scratch_llm_b200.kernels import ops
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: portions)
    H, G, hd, page = 8, 2, 64, 16
    rows = [(100, 60)]
    gen = torch.Generator().manual_seed(12)
    c = Cache(G, hd, page, 1, [160], gen).fill([(160, 0)], gen, 0.5)
    q = torch.randn(60, H * hd, generator=gen).bfloat16()
    clean = attend_on_device(c, q.to(DEV), rows, c.device(), H, hd ** -0.5)
    at = int(c.table[0, 130 // page]), 130 % page
    for plane, byte in ((0, 0x78), (1, 0xF8)):                    # 256, -256
        c.pages[at[0], plane, 1, at[1], 7], c.scales[at[0], plane, 1, at[1]] = byte, 247
    got = attend_on_device(c, q.to(DEV), rows, c.device(), H, hd ** -0.5)
    assert torch.equal(got[:30], clean[:30])
    assert torch.equal(got.view(60, H, hd)[:, :4], clean.view(60, H, hd)[:, :4])


@pytest.mark.parametrize("block", [1, 16])
def test_refused_drafts_leave_no_trace_in_blocks_of_one_token(block):
    """Loud drafts are stored, refused and written over: in blocks of one token the cache then holds what it holds without them; in
    larger ones a block keeps its scale, and no value of its earlier tokens moves by more than half a step of it."""
    from test_q8_cache_gpu import write_on_device
    H, G, hd, page = 2, 1, 64, 16
    gen = torch.Generator().manual_seed(2)
    c = Cache(G, hd, page, block, [40], gen)
    tokens = torch.randn(26, (H + 2 * G) * hd, generator=gen).bfloat16()
    loud = 3000.0 * torch.randn(4, (H + 2 * G) * hd, generator=gen).bfloat16()
    plainly, drafted = c.device(), c.device()
    write_on_device(c, tokens[:21], [(0, 21)], None, None, H, True, plainly)
    write_on_device(c, tokens[:21], [(0, 21)], None, None, H, True, drafted)
    write_on_device(c, loud, [(21, 4)], None, None, H, True, drafted)
    for dev in (plainly, drafted):
        write_on_device(c, tokens[21:], [(21, 5)], None, None, H, True, dev)
    held = [(dev[0].view(torch.uint8).cpu(), dev[1].view(torch.uint8).cpu()) for dev in (plainly, drafted)]
    a, b = (plain.values(*x, c.table[0], 26, page) for x in held)
    if block == 1:
        assert torch.equal(a, b)
    else:
        assert torch.equal(a[:, :16], b[:, :16])
        unit = plain.power(held[1][1][c.table[0].long()]).permute(1, 0, 3, 2).reshape(2, -1, G).repeat_interleave(block, 1)[:, :26]
        # (a first rounding to 2^-4 of the value at most on either side, or half a step of subnormals)
        assert ((a - b).abs() <= 2.0 ** -10 * unit[..., None] + 2.0 ** -3 * a.abs()).all()
        assert not torch.equal(held[0][1], held[1][1])
