"""The operators of a cache held in 8 bits and of drafted tokens, measured one by one.

A cache page holds keys, then values, as e4m3 numbers ``[pages, 2, kv heads, page size, head size]``; each block of
``block`` tokens has one power of two per plane and kv head (e8m0, ``[pages, 2, kv heads, page size / block]``).

* ``store``: a step's rotated queries; its keys and values written to the cache in 8 bits, and the blocks that it touched
  read back (what is held in 8 bits is returned as the values it stands for);
* ``read``: rows of the cache read back;
* ``attend``: attention of a step's queries over the cache;
* ``verify``: drafted tokens verified against the target's probabilities.

With ``own`` false ``run`` computes them in plain torch, in 32 bits (sums of probabilities in 64), else through the
framework's entry points.  Sizes are those of ``bench.py --sizes`` (Llama-3-8B, Llama-3.2-1B, Llama-2-13B).
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
THETA = 500000.0
NO_DRAFT_PROBS = "lookup"


def _layer(heads, kv, dim, page=64, block=16, interleaved=True, rot=0, bias=False):
    return dict(heads=heads, kv=kv, dim=dim, page=page, block=block, interleaved=interleaved, rot=rot or dim, bias=bias)


def _rows(rows, new, before, ragged=False):
    """``rows`` sequences that bring up to ``new`` tokens after up to ``before`` cached ones."""
    return dict(rows=rows, new=new, before=before, ragged=ragged)


LLAMA_8B, LLAMA_1B, LLAMA_13B = (32, 8, 128), (32, 8, 64), (40, 40, 128)


def listed():
    return [
        # a decode step of a small server: eight rows, one token each, in the middle of their blocks; latency counts
        dict(op="store", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(8, 1, 1001, True), name="store_decode_8"),
        # a prompt's step: whole blocks, bound by bandwidth
        dict(op="store", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(1, 8192, 0), name="store_prompt_8192"),
        # portions of several prompts that start and end inside blocks, biases, split halves, a part of each head turned
        dict(op="store", dtype="float32", **_layer(*LLAMA_13B, block=64, interleaved=False, rot=64, bias=True),
             **_rows(7, 301, 130, True), name="store_portions_32bit"),
        # a long row back in 16 bits, for a kernel or a transfer that takes plain pages
        dict(op="read", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(1, 0, 131072), name="read_131072"),
        # rows of mixed lengths in 32 bits, small pages
        dict(op="read", dtype="float32", **_layer(*LLAMA_1B, page=16), **_rows(9, 0, 1777, True), name="read_ragged_32bit"),
        # one user: the smallest decode step
        dict(op="attend", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(1, 1, 999), window=0, name="decode_1"),
        # a busy server with long contexts: bound by what the cache holds
        dict(op="attend", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(64, 1, 4095), window=0, name="decode_64"),
        # the 32-bit mode, mixed lengths, a window, blocks of one page
        dict(op="attend", dtype="float32", **_layer(*LLAMA_1B, page=16), **_rows(24, 1, 6001, True), window=4096,
             name="decode_24_32bit"),
        # drafted tokens: up to six a row beside rows that bring one
        dict(op="attend", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(32, 6, 2111, True), window=0, name="drafts_32"),
        # a portion of a long prompt: bound by the products
        dict(op="attend", dtype="bfloat16", **_layer(*LLAMA_8B), **_rows(1, 2048, 6144), window=0, name="portion_2048"),
        # verification for a small server, drafts from a draft model
        dict(op="verify", rows=4, drafts=4, vocab=128256, ragged=False, source="model", name="verify_4"),
        # for a large one, mixed numbers of drafts
        dict(op="verify", rows=64, drafts=8, vocab=128256, ragged=True, source="model", name="verify_64"),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend", "verify"])
    if op == "verify":
        return dict(op=op, rows=_between(rng, 1, 64), drafts=rng.randint(0, 8),
                    vocab=_between(rng, 1000, 130000), ragged=rng.random() < 0.6,
                    source=rng.choice(["model", "model", NO_DRAFT_PROBS]))
    heads, kv, dim = rng.choice([LLAMA_8B, LLAMA_1B, LLAMA_13B, (12, 12, 64), (24, 8, 96), (10, 2, 80), (16, 1, 256),
                                 (28, 4, 128)])
    page = rng.choice([16, 32, 64, 64, 128])
    block = rng.choice([b for b in (1, 4, 16, 32, 64, 128) if b <= page])
    rot = rng.choice([dim, dim, dim // 2])
    layer = _layer(heads, kv, dim, page, block, rng.random() < 0.6, rot, rng.random() < 0.3)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    most = (1 << 28) // (kv * dim)                      # cached tokens of a case
    case = dict(op=op, dtype=dtype, **layer)
    if op == "store":
        new = _between(rng, 1, 4096)
        rows = max(1, min(_between(rng, 1, 64), 6144 // new))
        return dict(case, **_rows(rows, new, rng.choice([0, _between(rng, 1, 4000)]), rng.random() < 0.7))
    if op == "read":
        rows = _between(rng, 1, 32)
        return dict(case, **_rows(rows, 0, max(1, min(_between(rng, 1, 65536), most // (2 * rows))), rng.random() < 0.7))
    window = rng.choice([0, 0, 0, _between(rng, 16, 8192)])
    if rng.random() < 0.5:                              # single tokens
        rows, new = _between(rng, 1, 96), 1
    elif rng.random() < 0.5:                            # drafts
        rows, new = _between(rng, 1, 32), rng.randint(2, 9)
    else:                                               # portions
        new = _between(rng, 16, 1500)
        rows = max(1, min(rng.randint(1, 4), 2000 // new))
    before = max(0, min(_between(rng, 1, 32768), most // (2 * rows), (1 << 23) // (rows * new)) - 1)
    return dict(case, **_rows(rows, new, before, rng.random() < 0.7), window=window)


# ------------------------------------------------------------------------------------------ what a case has

def _lengths(case):
    """(cached tokens, new tokens) of each row, from the case alone; the first row has the most of both."""
    rng = random.Random("%d %d %d" % (case["rows"], case["new"], case["before"]))
    got = []
    for r in range(case["rows"]):
        b, n = case["before"], case["new"]
        if case["ragged"] and r:
            b, n = rng.randint(b // 4, b), rng.randint(min(1, n), n)
        got.append((b, n))
    return got


def _counts(case):
    rng = random.Random("%d %d" % (case["rows"], case["drafts"]))
    return [rng.randint(0, case["drafts"]) if case["ragged"] and r else case["drafts"] for r in range(case["rows"])]


def _seen(case):
    """The pairs of a query and a key that it sees, and the keys that a row's queries see at all."""
    w, pairs, keys = case["window"], 0, 0
    for b, n in _lengths(case):
        pairs += sum(min(w, b + i + 1) if w else b + i + 1 for i in range(n))
        keys += min(b + n, w + n - 1) if w else b + n
    return pairs, keys


def work(case):
    if case["op"] == "verify":
        k = sum(_counts(case))
        rows = 1 if case["source"] == NO_DRAFT_PROBS else 2
        return {"bytes": 4 * case["rows"] * rows * case["vocab"] + 20 * k + 12 * case["rows"],
                "flops": 3 * case["rows"] * case["vocab"]}
    H, G, hd, es = case["heads"], case["kv"], case["dim"], 2 if case["dtype"] == "bfloat16" else 4
    lengths = _lengths(case)
    n = sum(x for _, x in lengths)
    if case["op"] == "read":
        t = sum(b for b, _ in lengths)
        return {"bytes": t * 2 * G * hd * (1 + es), "flops": t * 2 * G * hd}
    if case["op"] == "store":
        return {"bytes": n * (H + 2 * G) * hd * es + n * H * hd * es + n * 2 * G * hd * (1 + es) + n * case["rot"] * 4,
                "flops": n * (H + 2 * G) * hd * 4}
    pairs, keys = _seen(case)
    return {"bytes": keys * 2 * G * hd + 2 * n * H * hd * es, "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------------------------------ inputs

def _byte_for(amax):
    """The smallest e8m0 byte b >= 1 with amax <= 448 * 2^(b - 127), from a 32-bit number's own bits."""
    bits = amax.float().contiguous().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=1)


def _power(byte):
    """2^(byte - 127), from its bits (bytes of 1 and more)."""
    return (byte.int() << 23).view(torch.float32)


def _pool(case, gen):
    """A cache as earlier steps left it: every page full of values of a few magnitudes, per head and channel."""
    need = [max(1, -(-(b + n) // case["page"])) for b, n in _lengths(case)]
    G, hd, page, block = case["kv"], case["dim"], case["page"], case["block"]
    n_pages = sum(need) + 3
    head = torch.exp(0.7 * torch.randn(2, G, 1, 1, hd, generator=gen, device=DEV))
    x = torch.randn(n_pages, 2, G, page // block, block, hd, generator=gen, device=DEV).mul_(head)
    byte = _byte_for(x.abs().amax((-1, -2)))
    pages = x.mul_(1.0 / _power(byte)[..., None, None]).to(torch.float8_e4m3fn).view(n_pages, 2, G, page, hd)
    order = torch.randperm(n_pages, generator=gen, device=DEV).int()
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    place = torch.tensor([(r, p) for r, m in enumerate(need) for p in range(m)])
    table[place[:, 0], place[:, 1]] = order.cpu()[:len(place)]
    return pages, byte.to(torch.uint8).view(torch.float8_e8m0fnu), table.to(DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    if case["op"] == "verify":
        counts, V = _counts(case), case["vocab"]
        k, n = sum(counts), case["rows"]
        logits = 2.5 * randn(k + n, V)
        start = _i32(_starts(counts))
        row = torch.repeat_interleave(torch.arange(n, device=DEV), _i32(counts).long())
        at = torch.arange(k, device=DEV) + row             # the target's row for each draft
        near = torch.softmax(logits[at] + 0.5 * randn(k, V), -1)       # a draft model that is near the target
        drafts = torch.multinomial(near, 1, generator=gen)[:, 0] if k else torch.zeros(0, device=DEV)
        return dict(case=case, probs=torch.softmax(logits, -1), start=start, drafts=drafts.int(),
                    near=None if case["source"] == NO_DRAFT_PROBS else near, max_drafts=max(counts),
                    uniforms=torch.rand(k + n, generator=gen, device=DEV),
                    tokens=torch.empty(k + n, dtype=torch.int32, device=DEV),
                    accepted=torch.empty(n, dtype=torch.int32, device=DEV))
    lengths, dtype = _lengths(case), DTYPES[case["dtype"]]
    pages, scales, table = _pool(case, gen)
    s = dict(case=case, pages=pages, scales=scales, table=table, pos0=_i32([b for b, _ in lengths]),
             start=_i32(_starts([n for _, n in lengths])), n=sum(n for _, n in lengths),
             max_new=max(n for _, n in lengths), context=max(b + n for b, n in lengths))
    H, G, hd = case["heads"], case["kv"], case["dim"]
    page, block = case["page"], case["block"]
    if case["op"] == "attend":
        # (the queries of one product that also holds keys and values, as a layer's projection leaves them)
        s["q"] = (1.5 * randn(s["n"], (H + 2 * G) * hd)).to(dtype)[:, :H * hd]
        s["out"] = torch.zeros(s["n"], H * hd, dtype=dtype, device=DEV)
        return s
    first = [b // block * block if case["op"] == "store" else 0 for b, _ in lengths]
    end = [b + n for b, n in lengths]
    # plain pages for what is read back, one after the other in the rows' order
    back = torch.full(table.shape, -1, dtype=torch.int32)
    held = [(r, p) for r, (a, z) in enumerate(zip(first, end)) for p in range(a // page, -(-z // page))]
    where = torch.tensor(held).view(-1, 2)
    back[where[:, 0], where[:, 1]] = torch.arange(len(held), dtype=torch.int32)
    s |= dict(first=_i32(first), end=_i32(end), back_table=back.to(DEV), most=max(z - a for a, z in zip(first, end)),
              back=torch.zeros(len(held), 2, G, page, hd, dtype=dtype, device=DEV))
    if case["op"] == "store":
        rot = case["rot"]
        inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
        angle = torch.arange(max(end), dtype=torch.float64, device=DEV)[:, None] * inv
        s |= dict(cos=angle.cos().float().contiguous(), sin=angle.sin().float().contiguous(),
                  qkv=(randn(s["n"], H + 2 * G, hd) * torch.exp(0.7 * randn(H + 2 * G, hd))).to(dtype).view(s["n"], -1),
                  q_out=torch.empty(s["n"], H * hd, dtype=dtype, device=DEV),
                  bias=0.3 * randn((H + 2 * G) * hd) if case["bias"] else None)
    return s


# ------------------------------------------------------------------------------------------ plain forms

def _rows_of(start, n):
    return torch.searchsorted(start.long(), torch.arange(n, device=start.device), right=True) - 1


def _turn(x, cos, sin, interleaved):
    """x [N, heads, hd]: its first 2 * columns entries turned by the tokens' angles."""
    half = cos.shape[-1]
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    c, s = cos[:, None], sin[:, None]
    pair = (a * c - b * s, a * s + b * c)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([turned, rest], -1)


def _plain_store(s):
    case, H, G, hd = s["case"], s["case"]["heads"], s["case"]["kv"], s["case"]["dim"]
    page, block = case["page"], case["block"]
    row = _rows_of(s["start"], s["n"])
    pos = s["pos0"].long()[row] + torch.arange(s["n"], device=row.device) - s["start"].long()[row]
    x = s["qkv"].float()
    x = (x if s["bias"] is None else x + s["bias"]).view(-1, H + 2 * G, hd)
    qk = _turn(x[:, :H + G], s["cos"][pos], s["sin"][pos], case["interleaved"])
    kv = torch.stack([qk[:, H:], x[:, H + G:]], 1)                            # [N, 2, G, hd]
    pages, scales = s["pages"].view(torch.uint8), s["scales"].view(torch.uint8)
    page_of, off = s["table"].long()[row, pos // page], pos % page
    # blocks that the step touches, and what each of them needs
    unit, at = torch.unique(page_of * (page // block) + off // block, return_inverse=True)
    u_page, u_block = unit // (page // block), unit % (page // block)
    finite = torch.where(kv.isfinite(), kv.abs(), 0.0).amax(-1)               # [N, 2, G]
    amax = torch.zeros(len(unit), 2, G, device=kv.device)
    amax.scatter_reduce_(0, at[:, None, None].expand_as(finite), finite, "amax")
    begun = (s["pos0"].long()[row] - pos // block * block).clamp(min=0)       # earlier tokens of a token's block
    old = torch.zeros(len(unit), dtype=torch.long, device=kv.device).scatter_reduce_(0, at, begun, "amax")
    had = scales[u_page, :, :, u_block].int() * (old > 0)[:, None, None]
    byte = torch.maximum(_byte_for(amax), had)
    # the earlier tokens' values at the blocks' scales of now
    cells = pages.view(-1, 2, G, page // block, block, hd)
    held = cells[u_page, :, :, u_block]
    again = held.view(torch.float8_e4m3fn).float() * (_power(had.clamp(min=1)) / _power(byte))[..., None, None]
    earlier = (torch.arange(block, device=kv.device) < old[:, None])[:, None, None, :, None]
    cells[u_page, :, :, u_block] = torch.where(earlier, again.to(torch.float8_e4m3fn).view(torch.uint8), held)
    scales[u_page, :, :, u_block] = byte.to(torch.uint8)
    new = kv * (1.0 / _power(byte))[at][..., None]
    pages[page_of, :, :, off] = new.to(torch.float8_e4m3fn).view(torch.uint8)
    s["q_out"].copy_(qk[:, :H].reshape(s["n"], -1))
    return {"q": s["q_out"], "back": _plain_read(s)}


def _plain_read(s):
    """Positions [first, end) of every row, from the cache to pages of the compute dtype."""
    case, page, block = s["case"], s["case"]["page"], s["case"]["block"]
    count = (s["end"] - s["first"]).long()
    total = torch.cumsum(count, 0)
    i = torch.arange(int(total[-1]), device=total.device)
    row = torch.searchsorted(total, i, right=True)
    pos = s["first"].long()[row] + i - (total - count)[row]
    source, off = s["table"].long()[row, pos // page], pos % page
    byte = s["scales"].view(torch.uint8)[source, :, :, off // block]
    held = s["pages"].view(torch.uint8)[source, :, :, off].view(torch.float8_e4m3fn)
    value = held.to(s["back"].dtype) if s["back"].dtype == torch.bfloat16 else held.float()
    s["back"][s["back_table"].long()[row, pos // page], :, :, off] = value * _power(byte)[..., None].to(value.dtype)
    return s["back"]


def _plain_attend(s):
    case, H, G, hd = s["case"], s["case"]["heads"], s["case"]["kv"], s["case"]["dim"]
    page, R, T, C = case["page"], case["rows"], s["max_new"], s["context"]
    dev = s["q"].device
    kpos = torch.arange(C, device=dev)
    last = (s["pos0"] + s["start"].diff()).long()[:, None]                    # keys of a row
    source = s["table"].long().clamp(min=0)[:, kpos // page]                  # [R, C]
    byte = s["scales"].view(torch.uint8)[source, :, :, kpos % page // case["block"]]
    kv = s["pages"].view(torch.uint8)[source, :, :, kpos % page].view(torch.float8_e4m3fn).float()
    kv = kv * _power(byte)[..., None]
    kv = torch.where((kpos < last)[..., None, None, None], kv, 0.0)           # [R, C, 2, G, hd]
    row = _rows_of(s["start"], s["n"])
    t = torch.arange(s["n"], device=dev) - s["start"].long()[row]
    q = torch.zeros(R, T, G, H // G, hd, device=dev)
    q[row, t] = s["q"].float().view(-1, G, H // G, hd)
    score = torch.einsum("rtgjd,rcgd->rgtjc", q, kv[:, :, 0]) * hd ** -0.5
    qpos = s["pos0"].long()[:, None, None] + torch.arange(T, device=dev)[None, :, None]
    sees = (kpos <= qpos) & (kpos < last[..., None])
    if case["window"]:
        sees &= kpos > qpos - case["window"]
    score = torch.where(sees[:, None, :, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    out = torch.einsum("rgtjc,rcgd->rtgjd", p, kv[:, :, 1])
    out = out / p.sum(-1).permute(0, 2, 1, 3)[..., None].clamp(min=1e-30)
    s["out"].copy_(out.reshape(R, T, H * hd)[row, t])
    return s["out"]


def _plain_verify(s):
    start, n = s["start"].long(), s["case"]["rows"]
    counts, k = start.diff(), len(s["drafts"])
    row = _rows_of(s["start"], k)
    i = torch.arange(k, device=start.device) - start[row]
    x = s["drafts"].long()
    p = s["probs"][torch.arange(k, device=start.device) + row, x].double()
    q = 1.0 if s["near"] is None else s["near"][torch.arange(k, device=start.device), x].double()
    u = s["uniforms"].double()
    kept = u[torch.arange(k, device=start.device) + row] * q < p
    taken = counts.clone().scatter_reduce_(0, row, torch.where(kept, counts[row], i), "amin")
    # the distribution that the last token comes from
    at = start[:-1] + torch.arange(n, device=start.device) + taken
    w = s["probs"][at].double()
    refused, d = taken < counts, (start[:-1] + taken).clamp(max=max(k - 1, 0))
    if k and s["near"] is not None:
        w = torch.where(refused[:, None], (w - s["near"][d].double()).clamp(min=0), w)
    elif k:
        w = torch.where(refused[:, None] & (torch.arange(w.shape[1], device=w.device) == x[d][:, None]), 0.0, w)
    total = torch.cumsum(w, -1)
    goal = u[start[1:] + torch.arange(n, device=start.device)] * total[:, -1]
    token = (total <= goal[:, None]).sum(-1).clamp(max=w.shape[1] - 1)
    # a row's accepted drafts, the last token, and -1 behind it
    s["tokens"].fill_(-1)
    accepted = torch.where(i < taken[row], s["drafts"], -1)
    s["tokens"][torch.arange(k, device=start.device) + row] = accepted.int()
    s["tokens"][at] = token.int()
    s["accepted"].copy_(taken)
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


# ------------------------------------------------------------------------------------------ one pass

def _own(s):
    from scratch_llm_b200.kernels import ops

    case = s["case"]
    if case["op"] == "verify":
        ops.verify_drafts(s["probs"], s["drafts"], s["start"], s["uniforms"], s["tokens"], s["accepted"],
                          s["max_drafts"], draft_probs=s["near"])
        return {"tokens": s["tokens"], "accepted": s["accepted"]}
    R, H, G, hd, page = case["rows"], case["heads"], case["kv"], case["dim"], case["page"]
    if case["op"] == "attend":
        return ops.attention_q8(s["q"], s["pages"], s["scales"], s["table"], page, s["start"], s["pos0"], s["out"], None,
                                R, s["max_new"], s["context"], H, G, hd, hd ** -0.5, case["window"] or None)
    if case["op"] == "store":
        ops.rope_kv_write_q8(s["qkv"], s["start"], s["pos0"], R, s["max_new"], s["cos"], s["sin"], s["q_out"], s["pages"],
                             s["scales"], s["table"], page, H, G, hd, case["interleaved"], bias=s["bias"])
    ops.kv_read_q8(s["pages"], s["scales"], s["table"], page, s["first"], s["end"], s["back"], s["back_table"], R, s["most"])
    return s["back"] if case["op"] == "read" else {"q": s["q_out"], "back": s["back"]}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[
        state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------ in 64 bits

def _power64(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _round_e4m3(x):
    """To the nearest number with three bits behind the point at exponents of -6 and more, ties to even."""
    step = _power64((torch.frexp(x)[1] - 1).clamp(min=-6) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan)


def _exact_cache(s, r, length):
    """Keys and values [2, length, G, hd] of row r's first tokens."""
    case, page, block = s["case"], s["case"]["page"], s["case"]["block"]
    ids = s["table"][r, :-(-length // page)].long()
    x = s["pages"][ids].double().unflatten(3, (page // block, block)) * s["scales"][ids].double()[..., None, None]
    return x.flatten(3, 4).permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :length]


def _exact_store(s):
    case, H, G, hd = s["case"], s["case"]["heads"], s["case"]["kv"], s["case"]["dim"]
    page, block, half = case["page"], case["block"], case["rot"] // 2
    q_out, back = torch.zeros(s["n"], H, hd, dtype=torch.float64, device=DEV), torch.zeros_like(s["back"], dtype=torch.float64)
    x = s["qkv"].double()
    x = (x if s["bias"] is None else x + s["bias"].double()).view(-1, H + 2 * G, hd)
    for r, (before, n) in enumerate(_lengths(case)):
        t0 = int(s["start"][r])
        z = x[t0:t0 + n].clone()
        angle = torch.complex(s["cos"].double(), s["sin"].double())[before:before + n, None]
        i0 = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
        i1 = i0 + 1 if case["interleaved"] else i0 + half
        w = torch.complex(z[:, :H + G, i0], z[:, :H + G, i1]) * angle
        z[:, :H + G, i0], z[:, :H + G, i1] = w.real, w.imag
        q_out[t0:t0 + n] = z[:, :H]
        first = before // block * block
        old = _exact_cache(s, r, before)[:, first:]
        for b0 in range(first, before + n, block):
            fresh = torch.stack([z[:, H:H + G], z[:, H + G:]])[:, max(0, b0 - before):max(0, b0 + block - before)]
            amax = torch.where(fresh.isfinite(), fresh.abs(), 0.0).amax((1, 3))
            mantissa, e = torch.frexp(amax)                # amax = mantissa * 2^e, 0.5 <= mantissa < 1
            byte = torch.where(amax > 0, e - 9 + (mantissa > 0.875).int() + 127, 1).clamp(min=1)
            kept = old[:, :max(0, before - b0)] if b0 == first else old[:, :0]
            if kept.shape[1]:
                j = s["table"][r, b0 // page].long()
                byte = torch.maximum(byte, s["scales"].view(torch.uint8)[j, :, :, b0 % page // block].int())
            unit = _power64(byte - 127)[:, None, :, None]
            value = torch.cat([_round_e4m3(kept / unit), _round_e4m3(fresh / unit)], 1) * unit
            to = int(s["back_table"][r, b0 // page])
            back[to, :, :, b0 % page:b0 % page + value.shape[1]] = value.transpose(1, 2)
    return {"q": q_out.view(s["n"], -1), "back": back}


def _exact_attend(s):
    case, H, G, hd = s["case"], s["case"]["heads"], s["case"]["kv"], s["case"]["dim"]
    out = torch.zeros(s["n"], H, hd, dtype=torch.float64, device=DEV)
    for r, (before, n) in enumerate(_lengths(case)):
        t0, keys = int(s["start"][r]), before + n
        k, v = _exact_cache(s, r, keys)
        far = torch.arange(before, keys, device=DEV)[:, None] - torch.arange(keys, device=DEV)
        hidden = (far < 0) | (far >= (case["window"] or keys + 1))
        for g in range(G):
            q = s["q"][t0:t0 + n].double().view(n, G, H // G, hd)[:, g]
            z = (torch.matmul(q.transpose(0, 1), k[:, g].T) * hd ** -0.5).masked_fill(hidden, -math.inf)
            out[t0:t0 + n, g * (H // G):(g + 1) * (H // G)] = torch.matmul(torch.softmax(z, -1), v[:, g]).transpose(0, 1)
    return out.view(s["n"], -1)


def _exact_verify(s):
    tokens, accepted, at = [], [], 0
    u = s["uniforms"].double().tolist()
    for r, k in enumerate(_counts(s["case"])):
        a = at - r                                          # the row's first draft
        x = s["drafts"][a:a + k].tolist()
        i = 0
        while i < k and u[at + i] * (1.0 if s["near"] is None else float(s["near"][a + i, x[i]])) < float(s["probs"][at + i, x[i]]):
            i += 1
        w = s["probs"][at + i].double().clone()
        if i < k and s["near"] is None:
            w[x[i]] = 0.0
        elif i < k:
            w = (w - s["near"][a + i].double()).clamp(min=0.0)
        run_ = torch.cumsum(w.cpu(), 0)
        token = int(torch.searchsorted(run_, u[at + k] * float(run_[-1]), right=True))
        tokens += x[:i] + [min(token, len(w) - 1)] + [-1] * (k - i)
        accepted.append(i)
        at += k + 1
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "accepted": torch.tensor(accepted, dtype=torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    out = torch.zeros_like(s["back"], dtype=torch.float64)
    for r, (length, _) in enumerate(_lengths(case)):
        page = case["page"]
        value = _exact_cache(s, r, length).transpose(1, 2)
        for p in range(-(-length // page)):
            part = value[:, :, p * page:(p + 1) * page]
            out[int(s["back_table"][r, p]), :, :, :part.shape[2]] = part
    return out
