"""Drafted tokens verified against the target's probabilities: the same tokens as the plain form in 64 bits."""

import math

import pytest
import torch
from plain import q8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def call(probs, drafts, counts, uniforms, near=None, stream=None):
    from scratch_llm_b200.kernels import ops
    at = [0]
    for k in counts:
        at.append(at[-1] + k)
    n = len(counts)
    tokens = torch.full((at[-1] + n,), -7, dtype=torch.int32, device=DEV)
    accepted = torch.full((n,), -7, dtype=torch.int32, device=DEV)
    ops.verify_drafts(probs.to(DEV), drafts.int().to(DEV), torch.tensor(at, dtype=torch.int32, device=DEV), uniforms.to(DEV),
                      tokens, accepted, max(counts, default=0), near.to(DEV) if near is not None else None)
    return tokens.tolist(), accepted.tolist()


def make(counts, V, seed, sharp=2.0, apart=0.7):
    gen = torch.Generator().manual_seed(seed)
    k, n = sum(counts), len(counts)
    logits = sharp * torch.randn(k + n, V, generator=gen)
    row = torch.tensor([r for r, c in enumerate(counts) for _ in range(c)], dtype=torch.long)
    near = torch.softmax(logits[torch.arange(k) + row] + apart * torch.randn(k, V, generator=gen), -1)
    drafts = torch.multinomial(near, 1, generator=gen)[:, 0] if k else torch.zeros(0, dtype=torch.long)
    return torch.softmax(logits, -1), drafts, near, torch.rand(k + n, generator=gen)


@pytest.mark.parametrize("counts", [[0], [1], [4, 0, 8, 1, 3], [40, 2], [2] * 70])
@pytest.mark.parametrize("V", [1, 2, 37, 1000, 4097, 32003])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify(counts, V, lookup):
    probs, drafts, near, u = make(counts, V, V + len(counts))
    near = None if lookup else near
    assert call(probs, drafts, counts, u, near) == plain.verify(probs, drafts, counts, u, near)


def test_verify_a_large_vocabulary_with_strides():
    counts, V = [3, 0, 5, 2], 128256
    probs, drafts, near, u = make(counts, V, 1)
    want = plain.verify(probs, drafts, counts, u, near)
    assert call(probs, drafts, counts, u, near) == want
    wide = torch.zeros(probs.shape[0], V + 3)
    wide[:, 1:V + 1] = probs
    wide_near = torch.zeros(near.shape[0], V + 1)
    wide_near[:, :V] = near
    assert call(wide.to(DEV)[:, 1:V + 1], drafts, counts, u, wide_near.to(DEV)[:, :V]) == want


def test_verify_borders():
    """Numbers at 0 and just below 1, drafts that agree in full, weights that vanish, rows of no probability."""
    V = 300
    eye = torch.eye(V)
    below = 1.0 - 2.0 ** -24
    cases = []
    # the draft is the target: always accepted, then a draw from the last row
    probs = torch.cat([eye[5:6], eye[9:10]])
    cases.append((probs, [5], [1], [below, below], eye[5:6]))
    # the draft has no probability: the target's own token
    cases.append((probs, [6], [1], [0.0, below], eye[6:7]))
    # p nowhere above q where the draft is refused: drawn from p itself
    half = torch.zeros(1, V)
    half[0, 3] = half[0, 4] = 0.5
    cases.append((torch.cat([half, half]), [7], [1], [0.5, 0.75], half))
    # nothing at all
    cases.append((torch.zeros(1, V), [], [0], [0.5], None))
    cases.append((torch.full((1, V), math.nan), [], [0], [0.5], None))
    # a NaN is never accepted and never drawn
    odd = torch.full((2, V), 1.0 / V)
    odd[0, 2] = math.nan
    cases.append((odd, [2], [1], [0.0, 0.0], None))
    # no draft of the vocabulary
    cases.append((odd, [-1], [1], [0.0, 0.999], None))
    cases.append((odd, [V], [1], [0.0, 0.999], odd[1:2].clone()))
    # the first and the last token of the row
    flat = torch.full((1, V), 1.0 / V)
    cases.append((flat, [], [0], [0.0], None))
    cases.append((flat, [], [0], [below], None))
    for probs, x, counts, u, near in cases:
        drafts, u = torch.tensor(x, dtype=torch.long), torch.tensor(u)
        assert call(probs, drafts, counts, u, near) == plain.verify(probs, drafts, counts, u, near), (x, u)


def test_verify_distribution():
    """Over many rows with numbers of their own the tokens follow the target's distribution, whatever the draft's is:
    each share of 20,000 rows is within five standard deviations."""
    V, rows = 12, 20000
    gen = torch.Generator().manual_seed(3)
    p, q = torch.softmax(torch.randn(V, generator=gen), 0), torch.softmax(1.5 * torch.randn(V, generator=gen), 0)
    drafts = torch.multinomial(q, rows, replacement=True, generator=gen)
    probs = torch.stack([p, torch.full((V,), 1.0 / V)]).repeat(rows, 1)
    tokens, accepted = call(probs, drafts, [1] * rows, torch.rand(2 * rows, generator=gen), q.expand(rows, V).contiguous())
    first = torch.tensor(tokens).view(rows, 2)[:, 0]
    share = torch.bincount(first, minlength=V).double() / rows
    assert ((share - p.double()).abs() < 5 * (p * (1 - p) / rows).sqrt()).all()
    assert 0 < sum(accepted) < rows


def test_verify_captured_and_on_another_stream():
    from scratch_llm_b200.kernels import ops
    counts, V = [3, 0, 2], 5003
    probs, drafts, near, u = (t.to(DEV) for t in make(counts, V, 7))
    at = torch.tensor([0, 3, 3, 5], dtype=torch.int32, device=DEV)
    drafts = drafts.int()
    tokens, accepted = torch.empty(8, dtype=torch.int32, device=DEV), torch.empty(3, dtype=torch.int32, device=DEV)
    want = call(probs, drafts, counts, u, near)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.verify_drafts(probs, drafts, at, u, tokens, accepted, 3, near)
    stream.synchronize()
    assert (tokens.tolist(), accepted.tolist()) == want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_drafts(probs, drafts, at, u, tokens, accepted, 3, near)
    u.copy_(torch.rand(8, generator=torch.Generator().manual_seed(1)))
    graph.replay()
    torch.cuda.synchronize()
    assert (tokens.tolist(), accepted.tolist()) == plain.verify(probs.cpu(), drafts.cpu(), counts, u.cpu(), near.cpu())
