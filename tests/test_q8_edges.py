"""Edges of the cache held in 8 bits and of drafted tokens that need no GPU: what launches are planned with, and what is refused."""

import subprocess
import sys

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from scratch_llm_b200.cache import CacheManager
from scratch_llm_b200.engine.batch import RowInput, build_batch
from scratch_llm_b200.kernels import ops
from scratch_llm_b200.kernels.ops import KernelError
from scratch_llm_b200.parts import KVSpec


class Stager:
    def upload(self, arrays):
        return [torch.from_numpy(np.asarray(a, dtype=np.int32)) for a in arrays]


@pytest.mark.parametrize("n_rows,new,before", [(8, 6, 2111), (16, 6, 2111), (32, 6, 2111), (8, 16, 4096), (16, 16, 4096), (32, 16, 4096),
                                               (1, 300, 3000), (3, 5, 100), (2, 200, 1000), (1, 500, 20)])
@pytest.mark.parametrize("decoded", [0, 20])
def test_a_padded_step_is_planned_by_its_longest_row(n_rows, new, before, decoded, monkeypatch):
    """Whatever a step is padded to, its portions go the way that the same step goes without padding."""
    H, G, hd, page = 32, 8, 128, 64
    monkeypatch.setattr(ops, "_sm_count", lambda device: 148)
    cache = CacheManager([KVSpec(G, hd, None)], [None], page, 4000, 64)
    rows = []
    for i in range(n_rows + decoded):
        cache.admit(i)
        assert cache.reserve(i, before)
        cache.commit(i, before)
        rows.append(RowInput(i, [1] * (new if i < n_rows else 1)))
        assert cache.reserve(i, len(rows[-1].tokens))
    width = 8
    while width * page < before + new:
        width *= 2
    exact = build_batch(cache, Stager(), rows, 10, 1 << 20)
    padded = build_batch(cache, Stager(), rows, 10, 1 << 20, table_width=width, pad=True)
    assert exact.max_row_multi == new <= padded.max_row_multi < 2 * new
    ways = [ops._attention_q8_in_16_bits.__wrapped__(0, b.n_multi, b.max_row_multi, context, H, G, hd, page, 0)
            for b, context in ((exact, exact.max_context), (padded, width * page))]
    assert ways[0] == ways[1]


def entry_statuses(library: str, calls: list[str]) -> list[int]:
    """What an entry of a built library returns for each call, in a process of its own (refusals come before any GPU is
    touched)."""
    done = subprocess.run([sys.executable, "-c", f"""
from ctypes import c_float, c_int, c_int64, c_void_p
from scratch_llm_b200.kernels import ops
lib = {library}
P, I, L, F = c_void_p, c_int, c_int64, c_float
print(*[int(x) for x in [{", ".join("lib." + c for c in calls)}]])
"""], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, f"the process ended with {done.returncode}: {done.stderr[-500:]}"
    return [int(x) for x in done.stdout.splitlines()[-1].split()]


def test_write_entry_refuses_large_heads():
    """A head for which a CTA has too few threads is an error code, whoever calls."""
    at = ", ".join(["P(0)"] * 4)
    calls = [f"sllm_rope_kv_write_q8({at}, I(1), I(1), I(1), P(0), P(0), I({rot}), I(1), P(0), P(0), P(0), P(0), I(1), I(16), "
             f"I(16), I(1), I(1), I({hd}), I(1), I(1), P(0))" for hd, rot in [(272, 0), (528, 2), (2064, 0), (4096, 8), (1 << 30, 0)]]
    assert entry_statuses("ops._core('sllm_kv_q8')", calls) == [1] * 5            # cudaErrorInvalidValue


F32, I32, BF16 = torch.float32, torch.int32, torch.bfloat16


@pytest.fixture
def fake(monkeypatch):
    """Tensors on a pretended cuda:0 (test_q8_refusals.py); ``at`` places them, and a call that passes every check raises Reached."""
    monkeypatch.setattr(ops, "_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda device: 0)
    monkeypatch.setattr(ops, "_attention_q8_plan", lambda *a: (1, 1, 0))
    monkeypatch.setattr(ops, "_attention_q8_in_16_bits", lambda *a: False)

    def reach(*a):
        raise Reached

    monkeypatch.setattr(ops, "_q8_function", lambda *a: reach)
    placed = []
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: next((at for t, at in placed if t is self), 1 << 40))

    def make(*shape, dtype=F32, at=None, stride=None):
        t = torch.empty(shape if stride is None else (shape[0], stride), dtype=dtype, device="cuda")
        t = t if stride is None else t[:, :shape[1]]
        placed.append((t, at if at is not None else (len(placed) + 1) << 24))
        return t

    make.placed = placed
    with FakeTensorMode():
        yield make


class Reached(Exception):
    pass


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_stride,out_stride,off,apart", [
    (64, 64, 0, False), (64, 64, 8, False), (64, 64, 5 * 64, True), (64, 64, -5 * 64, True), (64, 64, 4 * 64, False), (64, 64, -64, False),
    (160, 160, 64, True), (160, 160, 96, True), (160, 160, 104, False), (160, 160, 56, False), (160, 160, -64, True), (160, 160, -56, False),
    (160, 160, 160 + 64, True), (160, 96, 64, False), (96, 160, 4 * 96 + 64, True), (160, 96, 4 * 160 + 56, False)])
def test_attention_refuses_outputs_in_its_queries(fake, dtype, q_stride, out_stride, off, apart):
    """Outputs that share memory with queries, wholly or in part; columns side by side are taken."""
    size = 4 if dtype == F32 else 2
    pages, scales = fake(8, 2, 2, 16, 16, dtype=torch.float8_e4m3fn), fake(8, 2, 2, 1, dtype=torch.float8_e8m0fnu)
    q = fake(5, 64, dtype=dtype, stride=q_stride, at=1 << 32)
    out = fake(5, 64, dtype=dtype, stride=out_stride, at=(1 << 32) + off * size)
    with pytest.raises(Reached) if apart else pytest.raises(KernelError, match="memory of its own"):
        ops.attention_q8(q, pages, scales, fake(2, 4, dtype=I32), 16, fake(3, dtype=I32), fake(2, dtype=I32), out, None, 2, 1, 40, 4, 2,
                         16, 0.1)


@pytest.mark.parametrize("rows,q_row,out_row,off,apart", [(1, 0, 0, 0, False), (1, 0, 64, 32, False), (1, 0, 0, 64, True), (5, 0, 64, 0, False),
                                                          (5, 0, 64, 64, True), (1, 1, 1, -63, False), (1, 1, 1, -64, True)])
def test_attention_refuses_outputs_in_queries_that_all_rows_share(fake, rows, q_row, out_row, off, apart):
    """Rows that are one (a stride of 0), and a single row, whose stride says nothing."""
    pages, scales = fake(8, 2, 2, 16, 16, dtype=torch.float8_e4m3fn), fake(8, 2, 2, 1, dtype=torch.float8_e8m0fnu)
    views = []
    for row, at in ((q_row, 1 << 32), (out_row, (1 << 32) + 4 * off)):
        views.append(torch.empty(64 * rows, dtype=F32, device="cuda").as_strided((rows, 64), (row, 1)))
        fake.placed.append((views[-1], at))
    with pytest.raises(Reached) if apart else pytest.raises(KernelError, match="memory of its own"):
        ops.attention_q8(views[0], pages, scales, fake(2, 4, dtype=I32), 16, fake(3, dtype=I32), fake(2, dtype=I32), views[1], None, 2, 1,
                         40, 4, 2, 16, 0.1)


@pytest.mark.parametrize("off,apart", [(0, False), (4, False), (-4, False), (12, True), (-20, True), (-16, False), (8, False)])
def test_verify_refuses_tokens_in_its_drafts(fake, off, apart):
    with pytest.raises(Reached) if apart else pytest.raises(KernelError, match="memory of its own"):
        ops.verify_drafts(fake(5, 99), fake(3, dtype=I32, at=1 << 32), fake(3, dtype=I32), fake(5),
                          fake(5, dtype=I32, at=(1 << 32) + off), fake(2, dtype=I32), 3)


def test_verify_refuses_more_drafts_than_it_is_told(fake):
    args = lambda k, n: (fake(k + n, 99), fake(k, dtype=I32), fake(n + 1, dtype=I32), fake(k + n), fake(k + n, dtype=I32),  # noqa: E731
                         fake(n, dtype=I32))
    for k, n, most in ((3, 2, 1), (1, 1, 0), (9, 2, 4), (1, 0, 5)):
        with pytest.raises(KernelError, match="more than max_drafts"):
            ops.verify_drafts(*args(k, n), most)
    for k, n, most in ((3, 2, 2), (0, 1, 0), (8, 2, 4)):
        with pytest.raises(Reached):
            ops.verify_drafts(*args(k, n), most)


@pytest.mark.parametrize("new", [1, 6])
def test_attention_of_no_tokens(fake, new):
    """A step in which every row is empty asks for nothing (and for no workspace, which would have no address)."""
    pages, scales = fake(8, 2, 2, 16, 16, dtype=torch.float8_e4m3fn), fake(8, 2, 2, 1, dtype=torch.float8_e8m0fnu)
    out = fake(0, 64)
    assert ops.attention_q8(fake(0, 64), pages, scales, fake(2, 4, dtype=I32), 16, fake(3, dtype=I32), fake(2, dtype=I32), out, None, 2,
                            new, 40, 4, 2, 16, 0.1) is out
