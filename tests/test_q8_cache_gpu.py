"""The cache held in 8 bits: what is written, what is read back and the attention over it, against plain forms
(tests/plain/q8_plain.py)."""

import math

import pytest
import torch
from plain import q8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts(rows):
    at = [0]
    for _, m in rows:
        at.append(at[-1] + m)
    return at


def tables(hd, rot, most):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(most, dtype=torch.float64)[:, None] * inv
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


class Cache:
    """A cache on the CPU (bytes) whose free places hold NaN and scales of 2^120, with its device copy."""

    def __init__(self, G, hd, page, block, lengths, gen, spare=2):
        need = [-(-n // page) for n in lengths]
        n_pages = sum(need) + spare
        self.page, self.block, self.G, self.hd = page, block, G, hd
        self.pages = torch.full((n_pages, 2, G, page, hd), 0x7F, dtype=torch.uint8)
        self.scales = torch.full((n_pages, 2, G, page // block), 247, dtype=torch.uint8)
        self.table = torch.full((max(1, len(need)), max([1, *need])), -1, dtype=torch.int32)
        ids = torch.randperm(n_pages, generator=gen).int().tolist()
        for r, m in enumerate(need):
            for p in range(m):
                self.table[r, p] = ids.pop()

    def fill(self, rows, gen, spread=2.0):
        """Earlier tokens of each row, as a write would have left them (any bytes but NaN, scales of a few sizes)."""
        for r, (before, _) in enumerate(rows):
            for b0 in range(0, before, self.block):
                page, cell = int(self.table[r, b0 // self.page]), b0 % self.page
                t = min(self.block, before - b0)
                x = torch.randn(2, self.G, t, self.hd, generator=gen) * torch.exp(
                    spread * torch.randn(2, self.G, 1, 1, generator=gen))
                byte = plain.scale_byte(x.abs().amax((2, 3)))
                self.scales[page, :, :, cell // self.block] = byte.to(torch.uint8)
                self.pages[page, :, :, cell:cell + t] = plain.round_e4m3(
                    x.double() / plain.power(byte)[..., None, None]).view(torch.uint8)
        return self

    def device(self):
        return (self.pages.to(DEV).view(torch.float8_e4m3fn), self.scales.to(DEV).view(torch.float8_e8m0fnu),
                self.table.to(DEV))


def write_on_device(c, qkv, rows, cos, sin, H, interleaved, dev, bias=None, write=True, behind=0):
    """rope_kv_write_q8 on the device copy ``dev``; returns q_out with ``behind`` rows that nobody writes (filled with 7)."""
    from scratch_llm_b200.kernels import ops
    q_out = torch.full((qkv.shape[0], H * c.hd), 7.0, dtype=qkv.dtype, device=DEV)
    ops.rope_kv_write_q8(qkv.to(DEV), i32(starts(rows)), i32([b for b, _ in rows]), len(rows), max(m for _, m in rows),
                         cos.to(DEV) if cos is not None else None, sin.to(DEV) if sin is not None else None, q_out, dev[0],
                         dev[1], dev[2], c.page, H, c.G, c.hd, interleaved, write=write,
                         bias=bias.to(DEV) if bias is not None else None)
    return q_out


ROWS = [
    [(0, 1)], [(37, 1), (0, 1), (15, 1), (16, 1), (63, 1)],
    [(0, 70)], [(5, 3), (0, 0), (64, 40), (31, 1), (0, 16), (95, 34), (16, 0)],
]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,hd,rot,interleaved,bias,page,block", [
    (4, 2, 128, 128, True, False, 64, 16), (6, 6, 64, 32, False, True, 16, 16), (3, 1, 80, 40, True, True, 32, 32),
    (8, 2, 16, 0, True, False, 16, 1), (2, 2, 256, 256, False, False, 64, 64), (5, 1, 48, 46, False, False, 12, 3),
    (2, 1, 112, 2, True, False, 128, 128), (4, 4, 96, 96, False, False, 1, 1),
    (2, 1, 256, 254, True, True, 64, 32), (3, 3, 240, 2, False, False, 256, 256)])
def test_write(rows, dtype, H, G, hd, rot, interleaved, bias, page, block):
    gen = torch.Generator().manual_seed(hd + len(rows))
    c = Cache(G, hd, page, block, [b + m for b, m in rows], gen).fill(rows, gen)
    n, behind = sum(m for _, m in rows), 3
    width = (H + 2 * G) * hd
    # heads of several magnitudes, so that some blocks grow and some keep their scale; tokens behind the last row
    qkv = (torch.randn(n + behind, H + 2 * G, hd, generator=gen) *
           torch.exp(2 * torch.randn(H + 2 * G, 1, generator=gen))).to(dtype).view(-1, width)
    cos, sin = tables(hd, rot, 256) if rot else (None, None)
    b = 0.5 * torch.randn(width, generator=gen) if bias else None
    dev = c.device()
    q_out = write_on_device(c, qkv, rows, cos, sin, H, interleaved, dev, b)
    want = plain.write(qkv, rows, cos, sin, c.pages, c.scales, c.table, page, H, G, hd, interleaved, bias=b)
    assert torch.equal(dev[1].view(torch.uint8).cpu(), c.scales)
    assert torch.equal(dev[0].view(torch.uint8).cpu(), c.pages)       # (untouched places too)
    assert torch.equal(q_out[:n].cpu(), want)
    assert (q_out[n:] == 7).all()


@pytest.mark.parametrize("block", [1, 4, 16])
def test_write_token_by_token_is_within_the_roundings(block):
    """A row written in portions, its values growing: every stored value is within the roundings that its block's scales
    allow, and NaN and infinities stay with their own places."""
    H, G, hd, page = 2, 1, 32, 16
    gen = torch.Generator().manual_seed(block)
    cuts = [0, 1, 2, 3, 7, 8, 20, 21, 33, 48]
    total = cuts[-1]
    x = torch.randn(total, 2, G, hd, generator=gen).double() * torch.exp(0.3 * torch.arange(total).double())[:, None, None, None]
    x = x.float()
    x[5, 0, 0, 3], x[9, 1, 0, 31], x[21, 0, 0, 0] = math.inf, -math.inf, math.nan
    c = Cache(G, hd, page, block, [total], gen)
    dev = c.device()
    for a, z in zip(cuts, cuts[1:]):
        qkv = torch.cat([torch.zeros(z - a, H * hd), x[a:z, 0].reshape(z - a, -1), x[a:z, 1].reshape(z - a, -1)], 1)
        write_on_device(c, qkv, [(a, z - a)], None, None, H, True, dev)
    pages, scales = dev[0].view(torch.uint8).cpu(), dev[1].view(torch.uint8).cpu()
    got = plain.values(pages, scales, c.table[0], total, page).permute(1, 0, 2, 3)
    fine = x.isfinite()
    assert torch.equal(got.isfinite(), fine) and got[~fine].isnan().all()
    ids = c.table[0].long()
    unit = plain.power(scales[ids]).permute(0, 3, 1, 2).reshape(-1, 2, G).repeat_interleave(block, 0)[:total]
    # nothing saturates; a normal number is off by at most 2^-4 of itself per rounding, which only its first one is (a
    # scale that grows shifts exponents), what becomes subnormal by half a step of 2^-9 units: each growth at most
    # half the step at the scale of then, all of them together less than one step at the last scale
    tol = 2.0 ** -4 * x.double().abs() + 2.0 ** -9 * unit[..., None]
    assert ((got - x.double()).abs() <= tol)[fine].all()
    # the block's scale is the smallest for its largest value
    amax = torch.where(fine, x.abs(), torch.zeros(())).unflatten(0, (total // block, block)).amax((1, 4)) \
        if total % block == 0 else None
    if amax is not None:
        assert torch.equal(scales[ids].permute(0, 3, 1, 2).reshape(-1, 2, G)[:total // block].long(), plain.scale_byte(amax))


def test_write_small_and_large_values():
    """Zeros, subnormals, the largest 32-bit numbers, and values at the border 448 * 2^e."""
    H, G, hd, page, block = 1, 1, 16, 16, 1
    gen = torch.Generator().manual_seed(0)
    top = torch.finfo(torch.float32).max
    v = [0.0, 1e-45, 1.1754944e-38, 448.0, 448.00003, 464.0, 1.75, 1.7500001, 3.4e38, top, 2.0 ** -126 * 448, -top]
    x = torch.zeros(len(v), hd)
    x[:, 3] = torch.tensor(v)
    c = Cache(G, hd, page, block, [len(v)], gen)
    dev = c.device()
    qkv = torch.cat([x, x, -x], 1)
    write_on_device(c, qkv, [(0, len(v))], None, None, H, True, dev)
    plain.write(qkv, [(0, len(v))], None, None, c.pages, c.scales, c.table, page, H, G, hd, True)
    assert torch.equal(dev[1].view(torch.uint8).cpu(), c.scales)
    assert torch.equal(dev[0].view(torch.uint8).cpu(), c.pages)


def test_write_queries_only():
    H, G, hd, page, block = 4, 2, 64, 16, 16
    gen = torch.Generator().manual_seed(1)
    rows = [(5, 9), (30, 1)]
    c = Cache(G, hd, page, block, [14, 31], gen).fill(rows, gen)
    qkv = torch.randn(10, (H + 2 * G) * hd, generator=gen).bfloat16()
    cos, sin = tables(hd, hd, 64)
    dev = c.device()
    q = write_on_device(c, qkv, rows, cos, sin, H, True, dev, write=False)
    assert torch.equal(q.cpu(), plain.write(qkv, rows, cos, sin, c.pages, c.scales, c.table, page, H, G, hd, True, False))
    assert torch.equal(dev[0].view(torch.uint8).cpu(), c.pages) and torch.equal(dev[1].view(torch.uint8).cpu(), c.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_write_tokens_of_no_row(dtype):
    """Tokens before the first row and behind the last: as if they were not there, and their places are left alone."""
    from scratch_llm_b200.kernels import ops
    H, G, hd, page = 4, 2, 64, 16
    rows, n, front = [(20, 2), (0, 19), (5, 0), (31, 1)], 22, 37
    gen = torch.Generator().manual_seed(9)
    c = Cache(G, hd, page, 8, [b + m for b, m in rows], gen).fill(rows, gen)
    cos, sin = (t.to(DEV) for t in tables(hd, hd, 64))
    qkv = torch.randn(front + n + 9, (H + 2 * G) * hd, generator=gen).to(dtype).to(DEV)
    start, pos0, got = i32(starts(rows)), i32([b for b, _ in rows]), []
    for x, at in ((qkv[front:front + n].contiguous(), start), (qkv, start + front)):
        dev = c.device()
        q_out = torch.full((x.shape[0], H * hd), 7.0, dtype=dtype, device=DEV)
        ops.rope_kv_write_q8(x, at, pos0, len(rows), 19, cos, sin, q_out, *dev, page, H, G, hd, True)
        got.append((q_out, dev[0].view(torch.uint8), dev[1].view(torch.uint8)))
    assert torch.equal(got[1][0][front:front + n], got[0][0]) and (got[0][0] != 7).any()
    assert (got[1][0][:front] == 7).all() and (got[1][0][front + n:] == 7).all()
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][2], got[1][2])


def test_write_many_rows():
    """More rows than a warp has lanes, of mixed lengths, empty ones among them; a table wider than the rows need."""
    H, G, hd, page, block = 2, 1, 32, 16, 8
    gen = torch.Generator().manual_seed(2)
    rows = [(int(b), int(m)) for b, m in zip(torch.randint(0, 90, (131,), generator=gen), torch.randint(0, 12, (131,), generator=gen))]
    c = Cache(G, hd, page, block, [b + m for b, m in rows], gen).fill(rows, gen)
    qkv = torch.randn(sum(m for _, m in rows), (H + 2 * G) * hd, generator=gen)
    dev = c.device()
    wide = torch.full((len(rows), 40), -1, dtype=torch.int32)
    wide[:, :c.table.shape[1]] = c.table
    dev = (dev[0], dev[1], wide.to(DEV)[:, :c.table.shape[1] + 1])
    write_on_device(c, qkv, rows, None, None, H, True, dev)
    plain.write(qkv, rows, None, None, c.pages, c.scales, c.table, page, H, G, hd, True)
    assert torch.equal(dev[0].view(torch.uint8).cpu(), c.pages) and torch.equal(dev[1].view(torch.uint8).cpu(), c.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,hd,page,block", [(2, 128, 64, 16), (1, 48, 12, 3), (5, 16, 16, 1), (1, 256, 128, 128), (3, 80, 1, 1)])
def test_read(dtype, G, hd, page, block):
    from scratch_llm_b200.kernels import ops
    gen = torch.Generator().manual_seed(hd)
    spans = [(0, 37), (5, 5), (13, 130), (64, 65), (0, 1), (127, 128)]     # [from, to) of rows of 130 tokens
    c = Cache(G, hd, page, block, [130] * len(spans), gen).fill([(130, 0)] * len(spans), gen)
    c.pages[int(c.table[0, 0]), 0, 0, 0, 0] = 0xFF                         # a NaN comes back as one
    pages, scales, table = c.device()
    order = torch.randperm(c.table.numel(), generator=gen).int()
    out_table = order.view_as(c.table)
    out = torch.full((c.table.numel() + 1, 2, G, page, hd), 7.0, dtype=dtype, device=DEV)
    got = ops.kv_read_q8(pages, scales, table, page, i32([a for a, _ in spans]), i32([z for _, z in spans]), out,
                         out_table.to(DEV), len(spans), 130)
    assert got is out
    want = torch.full(out.shape, 7.0, dtype=torch.float64)
    for r, (a, z) in enumerate(spans):
        value = plain.values(c.pages, c.scales, c.table[r], z, page)
        for pos in range(a, z):
            want[int(out_table[r, pos // page]), :, :, pos % page] = value[:, pos]
    assert torch.equal(torch.nan_to_num(out.cpu().double(), nan=1e9), torch.nan_to_num(want, nan=1e9))


def attend_on_device(c, q, rows, dev, H, scale, window=0, row_list=None, out=None, context=None):
    from scratch_llm_b200.kernels import ops
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    listed = rows if row_list is None else [rows[r] for r in row_list]
    return ops.attention_q8(q, dev[0], dev[1], dev[2], c.page, i32(starts(rows)), i32([b for b, _ in rows]), out,
                            None if row_list is None else i32(row_list), len(listed), max(m for _, m in listed),
                            context or max(b + m for b, m in listed), H, c.G, c.hd, scale, window or None)


def tolerance(dtype, hd, want, spread, reach, portion=False):
    """The result's rounding; the probabilities' before they multiply v (11 bits, or 21 in the 32-bit form; in portions
    that the tcgen05 kernel takes 8 bits, a bfloat16 of them: off by at most 2^-8 of each, sum_j 2^-8 p_j |v_j|, and as
    much again for the denominator where it sums the rounded ones); a score's error, at most hd roundings of 32-bit sums (of 2^-22 each on the tensor cores) of the sum of its products' sizes, which
    moves its probability by as much; and the 32-bit sums over the keys."""
    H = reach.shape[1]
    moved = (2.0 ** -22 * hd * reach).expand(-1, -1, hd).reshape(want.shape)
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * want.abs() + ((2.0 ** -7 if portion else 2.0 ** -10) + 2 * moved) * spread
    return 2.0 ** -23 * want.abs() + (2.0 ** -19 + 2 * moved) * spread


def is_portion(c, rows, dtype, H, window=0, context=None):
    from scratch_llm_b200.kernels import ops
    new = max(m for _, m in rows)
    return dtype == torch.bfloat16 and new > 1 and ops._attention_q8_in_16_bits(
        torch.cuda.current_device(), len(rows), new, context or max(b + m for b, m in rows), H, c.G, c.hd, c.page, window or 0)


def check(c, q, rows, dtype, H, window=0, n=None, **kw):
    dev = c.device()
    scale = c.hd ** -0.5
    got = attend_on_device(c, q.to(DEV), rows, dev, H, scale, window, **kw)
    want, spread, reach = plain.attend(q, c.pages, c.scales, c.table, rows, c.page, H, c.G, c.hd, scale, window)
    n = want.shape[0]
    far = (got[:n].double().cpu() - want).abs()
    tol = tolerance(dtype, c.hd, want, spread, reach, is_portion(c, rows, dtype, H, window, **kw))
    assert not got[:n].isnan().any()
    assert (far <= tol).all(), f"worst {(far / tol.clamp(min=1e-300)).max():.3g} of the tolerance"
    assert (got[n:] == 7).all()
    return got


ATTEND_ROWS = [
    [(0, 1)], [(200, 1), (0, 1), (63, 1), (64, 1), (15, 1), (16, 1)],
    [(0, 5), (77, 3), (5, 0), (130, 1), (31, 9), (64, 2)],
    [(0, 75)], [(33, 140), (100, 20)],
]


@pytest.mark.parametrize("rows", ATTEND_ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,hd,page,block,window", [
    (8, 2, 128, 64, 16, 0), (4, 4, 64, 16, 16, 0), (12, 1, 80, 32, 8, 50), (6, 2, 48, 12, 3, 0), (3, 1, 16, 16, 1, 0),
    (4, 2, 256, 64, 64, 33), (20, 1, 96, 128, 128, 0), (7, 1, 112, 5, 5, 1), (34, 1, 32, 16, 4, 0), (2, 2, 192, 1, 1, 0)])
@pytest.mark.parametrize("portions", [False, True])
def test_attention(rows, dtype, H, G, hd, page, block, window, portions, monkeypatch):
    from scratch_llm_b200.kernels import ops
    if portions and (dtype == torch.float32 or not ops.attention_tc_supports(H, G, hd, page, window or None, bool(window))
                     or max(m for _, m in rows) == 1):
        pytest.skip("only rows of several tokens and shapes of the tcgen05 kernel are read back")
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: portions)
    gen = torch.Generator().manual_seed(hd + len(rows))
    n = sum(m for _, m in rows)
    c = Cache(G, hd, page, block, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    q = (1.5 * torch.randn(n + 2, H * hd, generator=gen)).to(dtype)
    check(c, q, rows, dtype, H, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,hd,window", [(8, 2, 128, 0), (4, 2, 64, 700), (16, 2, 96, 0), (2, 1, 256, 0), (4, 4, 80, 0)])
@pytest.mark.parametrize("rows", [[(1999, 1), (700, 1), (3, 1)], [(1100, 6), (1500, 1), (300, 4)], [(700, 200)]])
def test_attention_long_rows(dtype, H, G, hd, window, rows):
    gen = torch.Generator().manual_seed(hd)
    c = Cache(G, hd, 64, 16, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    q = (1.5 * torch.randn(sum(m for _, m in rows), H * hd, generator=gen)).to(dtype)
    check(c, q, rows, dtype, H, window)
    check(c, q, rows, dtype, H, window, context=4096)       # (a bound above what the rows have)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("context", [None, 4096])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("plan", [(1, 3, 0), (1, 8, 1), (1, 13, 2), (1, 13, 0), (1, 64, 0), (2, 5, 0), (2, 5, 2), (2, 2, 1)])
def test_attention_shares_of_ragged_rows(plan, window, context, dtype, monkeypatch):
    """However the keys are shared out: rows of fewer keys than shares, of none before their token, and a workspace that
    holds NaN beforehand."""
    from scratch_llm_b200.kernels import ops
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: False)
    monkeypatch.setattr(ops, "_attention_q8_plan", lambda *a: plan)
    H, G, hd = 8, 2, 64
    rows = [(1100, 4), (0, 1), (30, 2), (257, 4), (0, 0), (127, 1), (640, 3)]
    gen = torch.Generator().manual_seed(17)
    c = Cache(G, hd, 16, 16, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    n = sum(m for _, m in rows)
    q = (1.5 * torch.randn(n, H * hd, generator=gen)).to(dtype)
    for _ in range(2):
        gone = torch.full((n * H * plan[1] * (hd + 2),), float("nan"), device=DEV)
        del gone
        check(c, q, rows, dtype, H, window, context=context)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_listed_rows_and_strides(dtype):
    """Only the listed rows, in any order, the same bits as all of them; queries and outputs as column slices."""
    H, G, hd = 4, 2, 64
    rows = [(90, 1), (10, 4), (0, 2), (200, 1), (64, 3)]
    gen = torch.Generator().manual_seed(5)
    c = Cache(G, hd, 16, 8, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    n = sum(m for _, m in rows)
    wide = torch.randn(n, (H + 2 * G) * hd, generator=gen).to(dtype).to(DEV)
    dev, s = c.device(), starts(rows)
    whole = attend_on_device(c, wide[:, :H * hd], rows, dev, H, 0.1, context=256)
    out = torch.full((n, H * hd + 6), 7.0, dtype=dtype, device=DEV)
    attend_on_device(c, wide[:, :H * hd], rows, dev, H, 0.1, row_list=[3, 1], out=out[:, 2:2 + H * hd], context=256)
    for r in range(5):
        part = out[s[r]:s[r + 1], 2:2 + H * hd]
        if r in (1, 3):     # (how the work is split goes by the listed rows: two correct results)
            torch.testing.assert_close(part, whole[s[r]:s[r + 1]], rtol=2.0 ** -7, atol=2.0 ** -9)
        else:
            assert (part == 7).all()
    assert (out[:, :2] == 7).all() and (out[:, 2 + H * hd:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,hd,rows", [(8, 2, 128, [(40, 6)]), (4, 1, 64, [(3, 70)]), (2, 2, 48, [(64, 3), (9, 2)]),
                                         (8, 2, 128, [(500, 130)])])
@pytest.mark.parametrize("portions", [False, True])
def test_attention_values_that_are_no_numbers(dtype, H, G, hd, rows, portions, monkeypatch):
    """A NaN among the keys or values of a token reaches the queries that see it and no other."""
    from scratch_llm_b200.kernels import ops
    if portions and (dtype == torch.float32 or not ops.attention_tc_supports(H, G, hd, 16, None)):
        pytest.skip("only shapes of the tcgen05 kernel are read back")
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: portions)
    gen = torch.Generator().manual_seed(hd)
    c = Cache(G, hd, 16, 4, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    before, m = rows[0]
    bad = before + 2                                              # a token of this step: two queries come before it
    at = int(c.table[0, bad // 16]), bad % 16
    c.pages[at[0], 1, 0, at[1], 5] = 0x7F
    if G > 1:
        c.pages[at[0], 0, 1, at[1], 0] = 0xFF
    q = torch.randn(sum(k for _, k in rows), H * hd, generator=gen).to(dtype)
    got = attend_on_device(c, q.to(DEV), rows, c.device(), H, hd ** -0.5).double().cpu()
    want, spread, reach = plain.attend(q, c.pages, c.scales, c.table, rows, c.page, H, G, hd, hd ** -0.5)
    assert torch.equal(got.isnan(), want.isnan())
    assert want.isnan().any() and not want[:2].isnan().any()
    fine = ~want.isnan()
    tol = tolerance(dtype, hd, want, spread, reach, portions)
    assert ((got - want).abs() <= tol)[fine].all()


@pytest.mark.parametrize("window", [0, 150])
def test_attention_portions_in_several_launches(window, monkeypatch):
    """Portions whose keys and values in 16 bits do not fit the workspace at once, all rows and listed ones; what lies
    behind a window may have been given back."""
    from scratch_llm_b200.kernels import ops
    H, G, hd, page = 8, 2, 64, 16
    rows = [(300, 40), (20, 70), (0, 33), (511, 128), (7, 0), (64, 35)]
    gen = torch.Generator().manual_seed(11)
    c = Cache(G, hd, page, 8, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    q = torch.randn(sum(m for _, m in rows), H * hd, generator=gen).bfloat16()
    if window:
        for r, (b, _) in enumerate(rows):
            c.table[r, :max(0, b - window + 1) // page] = -1
    monkeypatch.setattr(ops, "Q8_WORKSPACE_BYTES", 2 * 4 * G * 640 * hd)
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: True)
    dev, s = c.device(), starts(rows)
    want, spread, reach = plain.attend(q, c.pages, c.scales, c.table, rows, page, H, G, hd, hd ** -0.5, window)
    tol = tolerance(torch.bfloat16, hd, want, spread, reach, True)
    got = attend_on_device(c, q.to(DEV), rows, dev, H, hd ** -0.5, window).double().cpu()
    assert ((got - want).abs() <= tol).all()
    got = attend_on_device(c, q.to(DEV), rows, dev, H, hd ** -0.5, window, row_list=[3, 0, 5, 1]).double().cpu()
    for r in range(len(rows)):
        part = slice(s[r], s[r + 1])
        if r in (0, 1, 3, 5):
            assert ((got[part] - want[part]).abs() <= tol[part]).all()
        else:
            assert (got[part] == 7).all()


def test_attention_far_scales():
    """Blocks whose scales lie far apart: what a huge block with a small probability adds and what a tiny one does both
    count, and a block of zeros counts in the denominator only."""
    H, G, hd, page, block = 4, 1, 64, 16, 16
    rows = [(95, 1)]
    gen = torch.Generator().manual_seed(9)
    c = Cache(G, hd, page, block, [96], gen).fill([(96, 0)], gen, 0.0)
    for p, shift in enumerate([0, -40, 30, -100, 0, 12]):
        c.scales[int(c.table[0, p]), 1] += shift
    zero = int(c.table[0, 4])
    c.pages[zero, 1], c.scales[zero, 1] = 0, 1
    c.pages[int(c.table[0, 2]), 1, 0, :, 32:] = 0                 # half of the entries only see the other blocks
    q = torch.randn(1, H * hd, generator=gen)
    # (a key's probability has 11 or 22 bits, below 2^-38 of the largest p_j 2^e_j fewer: 2^-32 of the largest |v|)
    dev = c.device()
    for dtype in (torch.bfloat16, torch.float32):
        got = attend_on_device(c, q.to(dtype).to(DEV), rows, dev, H, hd ** -0.5).double().cpu()
        want, spread, reach = plain.attend(q.to(dtype), c.pages, c.scales, c.table, rows, page, H, G, hd, hd ** -0.5)
        big = spread.view(H, hd).amax(-1, keepdim=True).expand(H, hd).reshape(want.shape)
        assert ((got - want).abs() <= tolerance(dtype, hd, want, spread, reach) + 2.0 ** -30 * big).all()


def test_attention_values_of_extreme_scales():
    """All values tiny, all values huge, and a cache whose values are zeros."""
    H, G, hd, page = 2, 1, 32, 16
    rows = [(50, 1), (20, 3)]
    gen = torch.Generator().manual_seed(3)
    for shift in (-100, 100, None):
        c = Cache(G, hd, page, 8, [51, 23], gen).fill([(51, 0), (23, 0)], gen, 0.0)
        for r, need in enumerate((4, 2)):
            for p in range(need):
                at = int(c.table[r, p])
                if shift is None:
                    c.pages[at, 1], c.scales[at, 1] = 0, 1
                else:
                    c.scales[at, 1] = (c.scales[at, 1].int() + shift).clamp(1, 230).to(torch.uint8)
        c.pages[int(c.table[1, 1]), :, :, 7:] = 0x7F
        check(c, torch.randn(4, H * hd, generator=gen), rows, torch.float32, H)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_large_queries(dtype):
    """Queries of every magnitude that the type holds, as long as the scores are numbers."""
    H, G, hd = 2, 1, 64
    rows = [(40, 2)]
    gen = torch.Generator().manual_seed(4)
    c = Cache(G, hd, 16, 16, [42], gen).fill([(42, 0)], gen, 0.0)
    for size in (1e-30, 1e-3, 3e4, 1e20):
        q = (torch.randn(2, H * hd, generator=gen) * size).to(dtype)
        scale = 1.0 / (size * hd ** 0.5)
        got = attend_on_device(c, q.to(DEV), rows, c.device(), H, scale).double().cpu()
        want, spread, reach = plain.attend(q, c.pages, c.scales, c.table, rows, 16, H, G, hd, scale)
        assert ((got - want).abs() <= tolerance(dtype, hd, want, spread, reach)).all(), size


def test_attention_captured_steps_share_nothing():
    """Two captured steps, replayed side by side on two streams and after the eager calls' memory was used again."""
    H, G, hd = 8, 2, 128
    gen = torch.Generator().manual_seed(6)
    kept = []
    for rows in ([(1800, 1), (900, 1)], [(1200, 4)]):
        c = Cache(G, hd, 64, 16, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
        q = torch.randn(sum(m for _, m in rows), H * hd, generator=gen).bfloat16().to(DEV)
        kept.append([c, rows, q, c.device()])
    from scratch_llm_b200.kernels import ops
    graphs = []

    def made(c, rows, q, dev, args):
        return lambda: ops.attention_q8(q, *dev, c.page, *args, None, len(rows), max(m for _, m in rows),
                                        max(b + m for b, m in rows), H, G, hd, 0.1)

    for c, rows, q, dev in kept:
        args = (i32(starts(rows)), i32([b for b, _ in rows]), torch.empty_like(q))
        call = made(c, rows, q, dev, args)
        want = call().clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, args, want, torch.cuda.Stream(), call))
    for _ in range(20):
        for graph, args, _, stream, _ in graphs:
            with torch.cuda.stream(stream):
                args[2].zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, args, want, _, _ in graphs:
        assert torch.equal(args[2], want)
    for _ in range(20):                                       # eager calls on two streams at once
        for _, args, _, stream, call in graphs:
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    for _, args, want, _, _ in graphs:
        assert torch.equal(args[2], want)


def test_write_read_attend_over_a_sequence():
    """A row's life: a prompt in portions, single tokens, drafts of which some are taken back and written again; the
    attention of every step over what the plain write leaves."""
    H, G, hd, page, block = 4, 2, 64, 16, 8
    gen = torch.Generator().manual_seed(8)
    c = Cache(G, hd, page, block, [120], gen)
    dev = c.device()
    cos, sin = tables(hd, hd, 128)
    at = 0
    for n, keep in [(30, 30), (21, 21), (1, 1), (1, 1), (5, 2), (5, 5), (4, 0), (1, 1), (6, 3), (1, 1)]:
        qkv = torch.randn(n, (H + 2 * G) * hd, generator=gen).bfloat16()
        q = write_on_device(c, qkv, [(at, n)], cos, sin, H, True, dev)
        want_q = plain.write(qkv, [(at, n)], cos, sin, c.pages, c.scales, c.table, page, H, G, hd, True)
        assert torch.equal(q.cpu(), want_q)
        assert torch.equal(dev[0].view(torch.uint8).cpu(), c.pages) and torch.equal(dev[1].view(torch.uint8).cpu(), c.scales)
        got = attend_on_device(c, q, [(at, n)], dev, H, hd ** -0.5).double().cpu()
        want, spread, reach = plain.attend(want_q, c.pages, c.scales, c.table, [(at, n)], page, H, G, hd, hd ** -0.5)
        assert ((got - want).abs() <= tolerance(torch.bfloat16, hd, want, spread, reach)).all()
        at += keep


@pytest.mark.parametrize("hd,page", [(128, 64), (64, 64), (48, 12)])
def test_pages_past_32_bits(hd, page, monkeypatch):
    """Pages that lie more than 2^32 bytes into a cache: written, read and attended to as the first ones are."""
    from scratch_llm_b200.kernels import ops
    H, G, tokens = 8, 2, 150
    n = (1 << 32) // (2 * G * page * hd) + 40
    pages = torch.empty((n, 2, G, page, hd), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scales = torch.empty((n, 2, G, 2), dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    gen = torch.Generator().manual_seed(hd)
    qkv = torch.randn(tokens, (H + 2 * G) * hd, generator=gen).bfloat16().to(DEV)
    need = -(-tokens // page)
    start, pos0, upto = i32([0, tokens]), i32([0]), i32([tokens])
    back_table = i32([list(range(need))])
    results = []
    for first in (0, n - need):
        table = i32([list(range(first, first + need))])
        q_out = torch.empty((tokens, H * hd), dtype=torch.bfloat16, device=DEV)
        ops.rope_kv_write_q8(qkv, start, pos0, 1, tokens, None, None, q_out, pages, scales, table, page, H, G, hd, True)
        back = torch.zeros((need, 2, G, page, hd), dtype=torch.bfloat16, device=DEV)
        ops.kv_read_q8(pages, scales, table, page, pos0, upto, back, back_table, 1, tokens)
        got = [q_out, back]
        for portions in (False, True):
            if portions and not ops.attention_tc_supports(H, G, hd, page, None, False):
                continue
            monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: portions)
            out = torch.empty_like(q_out)
            got.append(ops.attention_q8(q_out, pages, scales, table, page, start, pos0, out, None, 1, tokens, tokens, H, G, hd, 0.1))
        results.append(got)
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_a_row_that_is_listed_twice(dtype):
    H, G, hd = 8, 2, 64
    rows = [(700, 1), (900, 3), (20, 2)]
    gen = torch.Generator().manual_seed(21)
    c = Cache(G, hd, 16, 16, [b + m for b, m in rows], gen).fill([(b + m, 0) for b, m in rows], gen, 0.5)
    q = torch.randn(sum(m for _, m in rows), H * hd, generator=gen).to(dtype).to(DEV)
    dev = c.device()
    once = attend_on_device(c, q, rows, dev, H, 0.1, row_list=[1, 0], context=1024)
    twice = attend_on_device(c, q, rows, dev, H, 0.1, row_list=[1, 0, 1, 1], context=1024)
    torch.testing.assert_close(twice[:4], once[:4], rtol=2.0 ** -7, atol=2.0 ** -9)
    assert (twice[4:] == 7).all()
