"""A model served from a cache held in 8 bits: the attention part against the plain forms of what it writes and reads, and
whole steps through the engine against the plain model with a plain 8-bit cache."""

import math

import pytest
import torch
from configs import PAGE_SIZE
from plain import llama_plain as P
from plain import q8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bytes_of(t):
    return t.view(torch.uint8).cpu()


def make_part(dtype, hidden, H, G, hd, window=None, bias=False, value_dim=None, seed=0):
    from scratch_llm_b200.parts import MIXERS, POSITION_ENCODINGS, BuildContext, make
    from scratch_llm_b200.config.spec import PartSpec
    gen = torch.Generator().manual_seed(seed)
    mixer = make(MIXERS, "mixer", PartSpec("gqa_attention", dict(
        hidden_size=hidden, n_heads=H, n_kv_heads=G, head_dim=hd, scale=hd ** -0.5, window=window, bias=bias,
        value_dim=value_dim)))
    ctx = BuildContext(dtype=dtype, device=torch.device(DEV, torch.cuda.current_device()))
    mixer.load({n: torch.randn(s.shape, generator=gen) * (0.3 if len(s.shape) == 1 else s.shape[-1] ** -0.5)
                for n, s in mixer.param_specs().items()}, ctx)
    position = make(POSITION_ENCODINGS, "position encoding", PartSpec("rotary", dict(
        head_dim=hd, theta=10000.0, max_position=512, interleaved=not bias)))
    position.load({}, ctx)
    return mixer, position


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,G,hd,window,bias,value_dim,page", [
    (8, 2, 128, None, False, None, 64), (4, 4, 64, 40, False, None, 16), (6, 3, 48, None, True, 30, 16), (4, 1, 20, None, True, 36, 8)])
def test_attention_part(dtype, H, G, hd, window, bias, value_dim, page):
    """Steps of single tokens, of portions, of both, padded ones and runs that only read another run's entry."""
    from scratch_llm_b200.cache import CacheManager
    from scratch_llm_b200.engine.batch import BatchStager, RowInput, build_batch
    from scratch_llm_b200.parts import CacheView
    hidden = 64
    mixer, position = make_part(dtype, hidden, H, G, hd, window, bias, value_dim)
    spec = mixer.kv_spec()
    D = spec.head_dim
    cache = CacheManager([spec], [None], page, 40, 4, dtype=torch.float8_e4m3fn, device=mixer.qkv.weight.device,
                         poison_free_pages=True)
    stager = BatchStager(mixer.qkv.weight.device)
    gen = torch.Generator().manual_seed(1)
    names = ["a", "b", "c"]
    for n in names:
        cache.admit(n)
    shadow = bytes_of(cache.groups[0].pages[0]), bytes_of(cache.groups[0].scales[0])
    cos, sin = position.cos.cpu(), position.sin.cpu()
    steps = [dict(a=37, b=1), dict(a=1, b=1, c=50), dict(a=1, b=1, c=1), dict(a=6, b=1, c=5), dict(b=64, c=1), dict(a=1)]
    for i, step in enumerate(steps):
        rows = [RowInput(n, [1] * k) for n, k in step.items()]
        lens = [(cache.requests[n].n_tokens, k) for n, k in step.items()]
        for n, k in step.items():
            assert cache.reserve(n, k)
        batch = build_batch(cache, stager, rows, 10, 512, pad=i % 2 == 1)
        view = CacheView(pages=cache.entry_pages(0)[0], block_table=batch.block_tables[0], page_size=page,
                         scales=cache.entry_scales(0))
        x = torch.randn(batch.n_tokens, hidden, generator=gen).to(dtype).to(DEV)
        heads = torch.zeros(batch.n_tokens, H * D, dtype=dtype, device=DEV)
        mixer.activations_into(x, batch, view, True, position, [heads])
        qkv = mixer.qkv(x).cpu()
        n = sum(k for _, k in lens)
        width = -(-max(b + k for b, k in lens) // page)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for r, name in enumerate(step):
            held = torch.tensor(cache.table_of(name, 0), dtype=torch.int32)
            table[r, :len(held)] = held
        # (the plain form's own view of what the pages held before: pages given back were poisoned since)
        q = plain.write(qkv[:n], lens, cos, sin, *shadow, table, page, H, G, D, position.interleaved,
                        bias=mixer.bias.cpu() if mixer.bias is not None else None)
        now = bytes_of(cache.groups[0].pages[0]), bytes_of(cache.groups[0].scales[0])
        for r, (before, k) in enumerate(lens):
            last = before + k
            ids = table[r, max(0, before - 64) // page:-(-last // page)].long()
            ids = ids[ids >= 0]
            assert torch.equal(now[1][ids], shadow[1][ids])
            assert torch.equal(now[0][ids], shadow[0][ids])
        want, spread, reach = plain.attend(q, *shadow, table, lens, page, H, G, D, hd ** -0.5, window or 0)
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -7 * spread if dtype == torch.bfloat16 else \
            2.0 ** -23 * want.abs() + (2.0 ** -19 + 2.0 ** -21 * D * reach.expand(-1, -1, D).reshape(want.shape)) * spread
        assert ((heads[:n].cpu().double() - want).abs() <= tol).all()
        assert (heads[n:] == 0).all()
        # a run that reads the entry: its own queries, nothing stored
        out = torch.zeros_like(heads)
        mixer.activations_into(x, batch, view, False, position, [out])
        assert torch.equal(out, heads)
        assert torch.equal(bytes_of(cache.groups[0].pages[0]), now[0])
        assert torch.equal(bytes_of(cache.groups[0].scales[0]), now[1])
        for name, k in step.items():
            cache.commit(name, k)
        shadow = bytes_of(cache.groups[0].pages[0]), bytes_of(cache.groups[0].scales[0])


class PlainModel:
    """The plain Llama-style model (32 bits, CPU) with an 8-bit cache of its own per layer, for one sequence."""

    def __init__(self, cfg, w, page, block):
        self.cfg, self.w, self.page = cfg, w, page
        self.H, self.G = cfg["num_attention_heads"], cfg["num_key_value_heads"]
        self.hd, self.at = cfg["head_dim"], 0
        n = -(-cfg["max_position_embeddings"] // page)
        self.cos, self.sin = P.rope_tables(self.hd, cfg["max_position_embeddings"], cfg["rope_theta"])
        self.table = torch.arange(n, dtype=torch.int32)[None]
        self.layers = [(torch.zeros(n, 2, self.G, page, self.hd, dtype=torch.uint8),
                        torch.zeros(n, 2, self.G, page // block, dtype=torch.uint8)) for _ in range(cfg["num_hidden_layers"])]

    def step(self, ids):
        cfg, w, rows = self.cfg, self.w, [(self.at, len(ids))]
        eps = cfg["rms_norm_eps"]
        x = P.embed(torch.tensor(ids), w["model.embed_tokens.weight"])
        for i, held in enumerate(self.layers):
            p = f"model.layers.{i}"
            h = P.rmsnorm(x, w[f"{p}.input_layernorm.weight"], eps)
            qkv = torch.cat([h @ w[f"{p}.self_attn.{n}_proj.weight"].T for n in "qkv"], 1)
            q = plain.write(qkv, rows, self.cos, self.sin, *held, self.table, self.page, self.H, self.G, self.hd, True)
            out = plain.attend(q, *held, self.table, rows, self.page, self.H, self.G, self.hd, 1 / math.sqrt(self.hd))[0]
            x = x + out.float() @ w[f"{p}.self_attn.o_proj.weight"].T
            h = P.rmsnorm(x, w[f"{p}.post_attention_layernorm.weight"], eps)
            x = x + P.swiglu(h, *(w[f"{p}.mlp.{n}_proj.weight"] for n in ("gate", "up", "down")))
        self.at += len(ids)
        x = P.rmsnorm(x, w["model.norm.weight"], eps)
        return x @ (w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings") else w["lm_head.weight"]).T


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_steps_match_the_plain_model(name, model_dirs):
    """Portions and single tokens of three requests in 32 bits, decode steps replayed from captured graphs among them.  The
    engine's keys and values differ from the plain model's by 32-bit roundings, which now and then lie on two sides
    of a border between e4m3 numbers: such an entry is off by 2^-3 of itself, one of a row's thousands, and what it
    moves in the logits is far below the tolerance, which a whole token's mistake passes at once."""
    from scratch_llm_b200.engine import ModelRunner, RowInput
    from scratch_llm_b200.engine.runner import load_model
    cfg, w = P.read_model_dir(model_dirs[name])
    page = PAGE_SIZE[name]
    runner = ModelRunner(load_model(model_dirs[name], "float32", verbose=False), page, 60, 4, poison_free_pages=True,
                         cache_dtype="float8_e4m3fn")
    runner.capture_padded_after = 2
    assert runner.cache.groups[0].pages.dtype == torch.float8_e4m3fn
    gen = torch.Generator().manual_seed(3)
    models = {n: PlainModel(cfg, w, page, runner.cache.scale_block) for n in "abc"}
    for n in models:
        assert runner.admit(n)
    steps = [dict(a=17, b=3), dict(c=30), dict(a=1, b=1, c=1), dict(a=1, b=1, c=1), dict(a=1, b=1, c=1), dict(a=9, b=1),
             dict(a=9, b=1), dict(a=9, b=1), dict(b=2, c=11), dict(a=1, b=1, c=1)]
    for step in steps:
        ids = {n: torch.randint(0, cfg["vocab_size"], (k,), generator=gen).tolist() for n, k in step.items()}
        got = runner.step([RowInput(n, t, list(range(len(t))) if len(t) > 1 else [0]) for n, t in ids.items()]).cpu()
        want = torch.cat([models[n].step(t) for n, t in ids.items()])
        far = (got - want).norm() / want.norm()
        assert far < 4e-3, far
    assert runner.replayed_steps > 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_from_a_cache_in_8_bits(dtype, model_dirs):
    """Through the entry point: the same tokens with steps launched ahead and without, in a batch whose pool is so small that
    requests are set back; close to the model with an unquantised cache."""
    from scratch_llm_b200 import LLM, SamplingParams
    cfg, w = P.read_model_dir(model_dirs["D"])
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist() for n in (5, 140, 33, 64)]
    params = SamplingParams(temperature=0.0, max_tokens=12)
    make = lambda **k: LLM(model_dirs["D"], dtype=dtype, page_size=16, max_batch_tokens=96, chunk_size=64,  # noqa: E731
                           **{"max_tokens": 2048, "cache_dtype": "float8_e4m3fn", **k})
    llm = make()
    assert llm.runner.cache.groups[0].pages.element_size() == 1
    got = llm.generate(prompts, params)
    assert [len(t) for t in got] == [12] * 4
    assert make(lookahead=False).generate(prompts, params) == got
    score = llm.score(prompts[1], got[1])
    plain_score = make(cache_dtype=None).score(prompts[1], got[1])
    # e4m3 entries are off by 2^-4 of themselves at most, 2^-5.8 of them on average, with signs that cancel over a head: a
    # log-probability of this model moves by some hundredths; a wrong page or scale moves it by units
    assert max(abs(a - b) for a, b in zip(score, plain_score)) < 0.5
    small = make(max_tokens=288)
    again = small.generate(prompts, params)
    assert [len(t) for t in again] == [12] * 4


def test_command_line_with_a_cache_in_8_bits(tmp_path, monkeypatch, capsys, model_dirs):
    from scratch_llm_b200 import chat_cli
    answers = iter(["3 14 15 92"])

    def line(prompt=""):
        try:
            return next(answers)
        except StopIteration:
            raise EOFError from None

    monkeypatch.setattr("builtins.input", line)
    assert chat_cli.main(["--model", str(model_dirs["A"]), "--dtype", "float32", "--max-tokens", "6", "--cache-dtype",
                          "float8_e4m3fn"]) == 0
    out = [x for x in capsys.readouterr().out.splitlines() if x.startswith("bot>")]
    assert len(out) == 1 and len(out[0].split()) == 7
