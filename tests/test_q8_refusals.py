"""What the 8-bit cache's operators and the verification of drafts refuse, checked without a GPU: tensors that only pretend to lie
on one reach the checks but no kernel."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from scratch_llm_b200.cache import CacheManager
from scratch_llm_b200.kernels import ops
from scratch_llm_b200.kernels.ops import KernelError
from scratch_llm_b200.parts import KVSpec

E4M3, E8M0, F32, I32, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float32, torch.int32, torch.bfloat16


class Reached(Exception):
    pass


@pytest.fixture
def fake(monkeypatch):
    """Tensors on a pretended cuda:0; a call that passes every check raises Reached instead of launching."""
    monkeypatch.setattr(ops, "_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda device: 0)

    def reach(*a):
        raise Reached

    monkeypatch.setattr(ops, "_q8_function", lambda *a: reach)
    monkeypatch.setattr(ops, "_attention_q8_plan", lambda *a: (1, 1, False))
    seen = []       # (kept alive, so that no address comes twice)

    def data_ptr(self):
        at = next((i for i, t in enumerate(seen) if t is self), None)
        if at is None:
            at = len(seen)
            seen.append(self)
        return (1 + at) << 20

    monkeypatch.setattr(torch.Tensor, "data_ptr", data_ptr)
    with FakeTensorMode():
        yield lambda *shape, dtype=F32, device="cuda": torch.empty(shape, dtype=dtype, device=device)


def cache(t, n_pages=8, G=2, page=16, hd=64, blocks=1):
    return t(n_pages, 2, G, page, hd, dtype=E4M3), t(n_pages, 2, G, blocks, dtype=E8M0)


def write_args(t, **change):
    pages, scales = cache(t)
    a = dict(qkv=t(5, 8 * 64, dtype=BF16), row_start=t(3, dtype=I32), row_pos0=t(2, dtype=I32), n_rows=2, max_new=4,
             cos=t(32, 32), sin=t(32, 32), q_out=t(5, 4 * 64, dtype=BF16), pages=pages, scales=scales,
             block_table=t(2, 4, dtype=I32), page_size=16, n_heads=4, n_kv_heads=2, head_dim=64, interleaved=True)
    return {**a, **change}


def test_what_passes(fake):
    with pytest.raises(Reached):
        ops.rope_kv_write_q8(**write_args(fake))
    pages, scales = cache(fake)
    rows, table = fake(2, dtype=I32), fake(2, 4, dtype=I32)
    with pytest.raises(Reached):
        ops.kv_read_q8(pages, scales, table, 16, rows, rows, fake(3, 2, 2, 16, 64), table, 2, 10)
    q = fake(5, 4 * 64)
    with pytest.raises(Reached):
        ops.attention_q8(q, pages, scales, table, 16, fake(3, dtype=I32), rows, fake(5, 4 * 64), None, 2, 1, 40, 4, 2, 64, 0.1)
    with pytest.raises(Reached):
        ops.verify_drafts(fake(5, 99), fake(3, dtype=I32), fake(3, dtype=I32), fake(5), fake(5, dtype=I32), rows, 3)


@pytest.mark.parametrize("change,says", [
    (dict(qkv=("f", 5, 8 * 64 + 16, BF16)), "qkv must be"), (dict(qkv=("f", 5, 8 * 64, torch.float16)), "unsupported dtype"),
    (dict(q_out=("f", 5, 4 * 64, F32)), "q_out must be torch.bfloat16"), (dict(q_out=("f", 4, 4 * 64, BF16)), "q_out must be"),
    (dict(row_start=("f", 2, I32)), "row_start must be"), (dict(row_start=("f", 3, torch.int64)), "row_start must be torch.int32"),
    (dict(row_pos0=("f", 1, I32)), "row_pos0 must be"), (dict(block_table=("f", 1, 4, I32)), "block_table must be"),
    (dict(cos=("f", 32, 33)), "cos must be"), (dict(sin=("f", 31, 32)), "sin must be"), (dict(sin=None), "sin must be"),
    (dict(bias=("f", 8 * 64 - 1)), "bias must be"), (dict(pages=("f", 8, 2, 2, 16, 64, torch.uint8)), "pages must be"),
    (dict(pages=("f", 8, 1, 2, 16, 64, E4M3)), "pages must be"), (dict(pages=("f", 8, 2, 2, 8, 64, E4M3)), "pages must be"),
    (dict(scales=("f", 8, 2, 2, 3, E8M0)), "divide"), (dict(scales=("f", 7, 2, 2, 1, E8M0)), "scales must be"),
    (dict(scales=("f", 8, 2, 2, 1, F32)), "scales must be"), (dict(pages=("f", 0, 2, 2, 16, 64, E4M3), scales=("f", 0, 2, 2, 1, E8M0)), "pages"),
    (dict(qkv=("f", 5, 8 * 64, BF16, "cpu")), "must be a CUDA tensor"), (dict(cos=("f", 32, 32, F32, "cuda:1")), "current device"),
    (dict(row_pos0=("f", 2, I32, "cuda:1")), "current device"),
])
def test_write_refuses(fake, change, says):
    def make(spec):
        if not isinstance(spec, tuple):
            return spec
        shape = [x for x in spec[1:] if isinstance(x, int)]
        dtype = next((x for x in spec if isinstance(x, torch.dtype)), F32)
        return fake(*shape, dtype=dtype, device=next((x for x in spec[1:] if isinstance(x, str)), "cuda"))

    with pytest.raises(KernelError, match=says):
        ops.rope_kv_write_q8(**write_args(fake, **{k: make(v) for k, v in change.items()}))


def test_write_refuses_layouts(fake):
    with pytest.raises(KernelError, match="qkv must be contiguous"):
        ops.rope_kv_write_q8(**write_args(fake, qkv=fake(5, 1024, dtype=BF16)[:, :512]))
    with pytest.raises(KernelError, match="contiguous rows"):
        ops.rope_kv_write_q8(**write_args(fake, block_table=fake(4, 2, dtype=I32).t()))
    for hd in (8, 24, 272):
        pages, scales = cache(fake, hd=hd)
        with pytest.raises(KernelError, match="head size"):
            ops.rope_kv_write_q8(**write_args(fake, pages=pages, scales=scales, head_dim=hd, cos=None, sin=None,
                                              qkv=fake(5, 8 * hd, dtype=BF16), q_out=fake(5, 4 * hd, dtype=BF16)))


def test_write_refuses_shared_and_unaligned_memory(fake, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 4096)
    with pytest.raises(KernelError, match="memory of its own"):
        ops.rope_kv_write_q8(**write_args(fake))
    for far in (5 * 8 * 64 * 2 - 16, -(5 * 4 * 64 * 2 - 16)):          # (q_out starts inside qkv, or ends there)
        monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 1 << 20 if self.shape[-1] == 8 * 64 else (1 << 20) + far)
        with pytest.raises(KernelError, match="memory of its own"):
            ops.rope_kv_write_q8(**write_args(fake))
    pages = write_args(fake)["pages"]
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 4096 if self.dtype == E4M3 else 4100 + id(self) % 9 * 16)
    with pytest.raises(KernelError, match="16-byte boundaries"):
        ops.rope_kv_write_q8(**write_args(fake, pages=pages))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 4104)
    with pytest.raises(KernelError, match="pages must start"):
        ops.rope_kv_write_q8(**write_args(fake, pages=pages))


def test_read_refuses(fake, monkeypatch):
    pages, scales = cache(fake)
    rows, table = fake(2, dtype=I32), fake(2, 4, dtype=I32)
    call = lambda out, **k: ops.kv_read_q8(pages, scales, k.get("table", table), 16, k.get("a", rows), k.get("z", rows), out,  # noqa: E731
                                           k.get("out_table", table), 2, 10)
    good = fake(3, 2, 2, 16, 64)
    with pytest.raises(KernelError, match="unsupported dtype"):
        call(fake(3, 2, 2, 16, 64, dtype=torch.float16))
    with pytest.raises(KernelError, match="out must be"):
        call(fake(3, 2, 2, 16 * 64))
    with pytest.raises(KernelError, match="out must be"):
        call(fake(3, 1, 2, 16, 64))
    with pytest.raises(KernelError, match="pages must be"):
        call(fake(3, 2, 2, 16, 32))
    with pytest.raises(KernelError, match="row_from"):
        call(good, a=fake(1, dtype=I32))
    with pytest.raises(KernelError, match="row_to"):
        call(good, z=fake(2))
    with pytest.raises(KernelError, match="out_table"):
        call(good, out_table=fake(1, 4, dtype=I32))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 4096 if self.dtype == E4M3 else 4096 + 16)
    with pytest.raises(KernelError, match="32-byte"):
        call(good)


def test_attention_refuses(fake):
    pages, scales = cache(fake)
    base = dict(q=fake(5, 256), pages=pages, scales=scales, block_table=fake(2, 4, dtype=I32), page_size=16,
                row_start=fake(3, dtype=I32), row_pos0=fake(2, dtype=I32), out=fake(5, 256), row_list=None, n_list=2, max_new=3,
                max_context=64, n_heads=4, n_kv_heads=2, head_dim=64, scale=0.1)
    for change, says in [
            (dict(q=fake(5, 255)), "q must be"), (dict(q=fake(256, 5).t()), "contiguous rows"), (dict(out=fake(5, 256, dtype=BF16)), "out must be"),
            (dict(out=fake(4, 256)), "out must be"), (dict(n_heads=5, q=fake(5, 320), out=fake(5, 320)), "group evenly"),
            (dict(row_list=fake(1, dtype=I32)), "row_list"), (dict(row_start=fake(2, dtype=I32)), "row_start"),
            (dict(row_pos0=fake(1, dtype=I32)), "row_pos0"), (dict(block_table=fake(1, 4, dtype=I32)), "block_table"),
            (dict(window=-1), "window"), (dict(q=fake(5, 256, dtype=torch.float16)), "unsupported dtype"),
            (dict(out=fake(5, 256, device="cuda:1")), "current device")]:
        with pytest.raises(KernelError, match=says):
            ops.attention_q8(**{**base, **change})
    assert ops.attention_q8(**{**base, "n_list": 0}) is base["out"]
    with pytest.raises(KernelError, match="memory of its own"):
        ops.attention_q8(**{**base, "out": base["q"]})


def test_attention_says_what_a_launch_holds(monkeypatch):
    monkeypatch.setattr(ops, "_attention_q8_form", lambda *a: (592, 32))
    plan = ops._attention_q8_plan.__wrapped__
    for rows, new in ((65536, 1), (1, 300000)):
        with pytest.raises(KernelError, match="at most 65,535 rows"):
            plan(0, 64, 0, rows, new, 300000, 32, 8, 0)
    for args in ((0, 64, 0, 1, 1, 1, 8, 8, 0), (0, 128, 1, 65535, 1, 1, 8, 8, 0), (0, 64, 0, 1, 100000, 200000, 32, 8, 100),
                 (0, 128, 1, 3, 4, 1 << 20, 32, 8, 0)):
        nt, n, merge = plan(*args)
        packed = args[4] * (args[6] // args[7])
        assert nt in (1, 2) and 1 <= n <= 64 and merge in (0, 1, 2) and (merge != 1 or n <= 8) and -(-packed // (8 * nt)) * n <= 65535


def test_verify_refuses(fake):
    base = dict(probs=fake(5, 99), drafts=fake(3, dtype=I32), draft_start=fake(3, dtype=I32), uniforms=fake(5),
                tokens=fake(5, dtype=I32), accepted=fake(2, dtype=I32), max_drafts=3)
    for change, says in [
            (dict(probs=fake(4, 99)), "probs must be"), (dict(probs=fake(99, 5).t()), "contiguous rows"), (dict(probs=fake(5, 0)), "probs must be"),
            (dict(probs=fake(5, 99, dtype=BF16)), "probs must be"), (dict(drafts=fake(3, dtype=torch.int64)), "drafts must be"),
            (dict(draft_start=fake(2, dtype=I32)), "draft_start"), (dict(uniforms=fake(4)), "uniforms"), (dict(tokens=fake(4, dtype=I32)), "tokens"),
            (dict(draft_probs=fake(5, 99)), "draft_probs"), (dict(draft_probs=fake(3, 98)), "draft_probs"), (dict(max_drafts=-1), "max_drafts"),
            (dict(accepted=fake(2, dtype=I32, device="cpu")), "CUDA tensor")]:
        with pytest.raises(KernelError, match=says):
            ops.verify_drafts(**{**base, **change})
    assert ops.verify_drafts(fake(0, 99), fake(0, dtype=I32), fake(1, dtype=I32), fake(0), fake(0, dtype=I32),
                             fake(0, dtype=I32), 0) is None


def test_cache_manager_pages_in_8_bits():
    spec = KVSpec(2, 32, None)
    m = CacheManager([spec, KVSpec(1, 16, 20)], [None, None], 8, 4, 2, dtype=E4M3, device="cpu", poison_free_pages=True)
    assert m.scale_block == 8
    g = m.groups[0]
    assert g.pages.dtype == E4M3 and g.scales.dtype == E8M0 and tuple(g.scales.shape) == (1, 4, 2, 2, 1)
    assert g.pages.float().isnan().all() and g.scales.float().isnan().all()
    assert tuple(m.entry_scales(1).shape) == (4, 2, 1, 1)
    m.admit("a")
    assert m.reserve("a", 9)
    g.pages.view(torch.uint8).zero_()
    g.scales.view(torch.uint8).fill_(127)
    held = m.table_of("a", 0)
    m.release("a")
    for p in range(4):
        assert bool(g.pages[0, p].float().isnan().all()) == bool(g.scales[0, p].float().isnan().all()) == (p in [0, 1])
    assert m.free_pages() == [4, 4] and held is not None
    m = CacheManager([spec], [None], 64, 4, 2, dtype=E4M3, device="cpu", scale_block=64)
    assert tuple(m.groups[0].scales.shape) == (1, 4, 2, 2, 1)
    assert CacheManager([spec], [None], 24, 4, 2, dtype=E4M3).scale_block == 8
    with pytest.raises(ValueError, match="divide"):
        CacheManager([spec], [None], 16, 4, 2, dtype=E4M3, scale_block=5)
    with pytest.raises(ValueError, match="belongs"):
        CacheManager([spec], [None], 16, 4, 2, dtype=F32, scale_block=8)
    with pytest.raises(ValueError, match="keys and values"):
        CacheManager([KVSpec(1, 16, None, planes=1)], [None], 16, 4, 2, dtype=E4M3, device="cpu")
    assert CacheManager([spec], [None], 16, 4, 2, dtype=F32, device="cpu").entry_scales(0) is None


def test_runner_refuses_mixers_without_8_bit_pages():
    from types import SimpleNamespace

    from deganex_util import CONFIGS as DEGANEX     # (its latent attention caches one vector per token)
    from nilevik_util import CONFIGS as NILEVIK
    from scratch_llm_b200.config import config_from_dict
    from scratch_llm_b200.engine import build_model
    from scratch_llm_b200.engine.runner import ModelRunner

    for raw in (*NILEVIK.values(), *DEGANEX.values()):
        model = build_model(config_from_dict(raw))
        model = SimpleNamespace(blocks=model.blocks, ctx=SimpleNamespace(dtype=F32))
        if not any(b.cache_owner is not None and b.cache_owner.kv_spec() is not None for b in model.blocks):
            continue
        with pytest.raises(ValueError, match="does not take a cache held in 8 bits"):
            ModelRunner._cache_dtype(model, "float8_e4m3fn")
        assert ModelRunner._cache_dtype(model, None) == F32
        with pytest.raises(ValueError, match="compute dtype"):
            ModelRunner._cache_dtype(model, "int8")
