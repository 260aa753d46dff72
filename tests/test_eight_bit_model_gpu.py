"""A Llama served with 8-bit weights and 8-bit pages: the engine against the same model put together from the definitions in 64 bits."""

import plain_eight_bit as plain
import pytest
import torch
from test_eight_bit_gpu import BF16, DEV, E4M3, F64

pytestmark = pytest.mark.gpu

CONFIG = {
    "architectures": ["LlamaForCausalLM"], "hidden_act": "silu", "rope_theta": 10000.0, "rms_norm_eps": 1e-5, "tie_word_embeddings": False,
    "hidden_size": 256, "intermediate_size": 400, "num_hidden_layers": 3, "num_attention_heads": 4, "num_key_value_heads": 2, "vocab_size": 300,
    "max_position_embeddings": 512,
}


def build(weight_dtype, cache_dtype, use_graphs=None, seed=3):
    from llmserve_triton_kernels_b200.cache import CacheManager
    from llmserve_triton_kernels_b200.config.registry import architecture_of
    from llmserve_triton_kernels_b200.engine.step import StepFunction
    from llmserve_triton_kernels_b200.models.load import random_model, resolve_cache_dtype

    config = architecture_of(CONFIG).config_class.from_dict(CONFIG)
    model = random_model(config, seed, BF16, DEV, std=0.06, weight_dtype=weight_dtype)
    cache = CacheManager(model.cache_specs(), model.plan.schedule, page_size=16, num_pages=100, max_requests=4, dtype=resolve_cache_dtype(cache_dtype, BF16, model), device=DEV)
    return model, cache, StepFunction(model, cache, use_graphs=use_graphs)


class Recorder:
    """Calls of the 8-bit operators as the engine makes them: what went in and what came out, in order."""

    def __init__(self, monkeypatch, names):
        from llmserve_triton_kernels_b200 import ops

        self.calls = []
        for name in names:
            monkeypatch.setattr(ops, name, self.around(name, getattr(ops, name)))

    def around(self, name, real):
        def call(*args, **kwargs):
            before = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            result = real(*args, **kwargs)
            after = args[0].clone() if isinstance(args[0], torch.Tensor) else None
            self.calls.append((name, before, kwargs, None if result is None else result.clone(), after))
            return result

        return call


def near(got, want, steps):
    """Within ``steps`` half steps of bfloat16 of the value, or of the row's size where terms cancel."""
    got, want = got.to(F64), want.to(F64)
    size = want.abs().amax(1, keepdim=True)
    return bool(((got - want).abs() <= steps * 2.0**-9 * size + 2.0**-8 * want.abs()).all())


@pytest.mark.parametrize("pages", [None, "float8"])
@pytest.mark.parametrize("counts", [(150,), (40, 1, 3), (1, 1)], ids=str)
def test_a_step_operator_by_operator(pages, counts, monkeypatch):
    """Every operator gets what the one in front left (rounded once), and leaves what its definition says of it: an 8-bit rounding near a
    border may fall either way, so that a whole pass in 64 bits drifts away from any other, but not from step to step."""
    from llmserve_triton_kernels_b200 import ops
    from llmserve_triton_kernels_b200.engine.batch import StepEntry

    model, cache, step = build("float8", pages, use_graphs=False)
    assert (cache.groups[0].pool.dtype == E4M3) == bool(pages)
    g = torch.Generator().manual_seed(2)
    held = [0] + [50, 90][: len(counts) - 1]
    tokens = [torch.randint(0, 300, (h + c,), generator=g).tolist() for h, c in zip(held, counts)]
    for r, (h, t) in enumerate(zip(held, tokens)):
        if h:
            step([StepEntry(r, t[:h])])
    write, attend = ("rope_kv_write8", "paged_attention8") if pages else ("rope_kv_write", "paged_attention")
    recorder = Recorder(monkeypatch, ["linear8", write, attend])
    logits = step([StepEntry(r, t[h:], [c - 1]) for r, (h, c, t) in enumerate(zip(held, counts, tokens))])
    calls, ctx = iter(recorder.calls), step.last_context
    x = model.embedding[ctx.token_ids.long()].float()  # the stream, as the engine adds it up
    n, H, KV, D = x.shape[0], 4, 2, 64

    def normed(part):
        v = x.to(F64)
        return (v * torch.rsqrt((v * v).mean(1, keepdim=True) + part.eps) * part.weight.to(F64)).to(BF16)

    def product(expected, w, dtype):
        name, (given, weights, *_), _, got, _ = next(calls)
        assert name == "linear8" and weights is w and near(given, expected, 1) and got.dtype == dtype
        want, size = plain.linear(given, w.values, w.scales)
        assert ((got.to(F64) - want).abs() <= 150 * 2.0**-23 * size * 1.01 + torch.finfo(dtype).eps / 2 * want.abs()).all()
        return got

    for block in model.blocks:
        a, f = block.mixer, block.feed_forward
        qkv = product(normed(block.mixer_norm), a.w_in, BF16)
        name, args, _, _, after = next(calls)
        assert name == write and torch.equal(args[0], qkv)
        turned = plain.turn(qkv.view(n, H + 2 * KV, D)[:, : H + KV], a.position.rotary_table, ctx.positions)
        assert near(after[:, : H * D], turned[:, :H].reshape(n, H * D), 1)
        name, args, kwargs, out, _ = next(calls)
        assert name == attend and torch.equal(args[0], after) and kwargs["scale"] == D**-0.5
        x = x + product(out, a.w_out, torch.float32)
        gate_up = product(normed(block.ff_norm), f.w_gate_up, BF16).to(F64)
        gate, up = gate_up.chunk(2, 1)
        x = x + product((gate * torch.sigmoid(gate) * up).to(BF16), f.w_down, torch.float32)
    assert next(calls, None) is None
    want = normed(model.final_norm)[ctx.logit_rows.long()].to(F64) @ model.head.to(F64).t()
    assert near(logits, want, 2)


def test_captured_steps_are_the_eager_ones(monkeypatch):
    """Prompts, portions and single tokens, kernel by kernel and as graphs: the same bits where the keys are shared out alike (a captured step's
    attention is laid out for the model's longest context)."""
    from llmserve_triton_kernels_b200 import ops
    from llmserve_triton_kernels_b200.engine.batch import StepEntry

    monkeypatch.setattr(ops, "_ATTENTION8_SPLIT", (8, 37))
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (200, 37, 90)]
    results = []
    for use_graphs in (False, True):
        model, cache, step = build("float8", "float8", use_graphs)
        rows = []
        for _ in range(3):  # the second time a shape has been seen it is captured, then replayed
            steps = [[(0, 0, 140), (1, 0, 1)], [(0, 140, 1), (1, 1, 30), (2, 0, 70)], [(2, 70, 17)]]
            at = [141, 31, 87]
            while any(a < len(s) for a, s in zip(at, seqs)):
                steps.append([(r, at[r], 1) for r in range(3) if at[r] < len(seqs[r])])
                at = [a + 1 if a < len(s) else a for a, s in zip(at, seqs)]
            for entries in steps:
                rows.append(step([StepEntry(r, seqs[r][a : a + n], [n - 1]) for r, a, n in entries]).clone())
            for r in range(3):
                cache.free_request(r)
            cache.check()
        assert step.last_was_graph == use_graphs
        results.append(rows)
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_generation_and_its_sizes():
    """``LLM.generate``: greedy tokens are those of the definition where it is sure of them; the 8-bit model and cache take half the memory."""
    from llmserve_triton_kernels_b200 import LLM, SamplingParams

    prompts = [[5, 17, 200, 9], list(range(30, 110))]
    llm = LLM(CONFIG, seed=3, max_batch_size=2, num_blocks=40, weight_dtype="float8", cache_dtype="float8", freeze_gc=False)
    plain_llm = LLM(CONFIG, seed=3, max_batch_size=2, num_blocks=40, freeze_gc=False)
    assert llm.cache.nbytes() < 0.52 * plain_llm.cache.nbytes()
    layers = sum(w.numel() for b in plain_llm.model.blocks for w in (b.mixer.w_in, b.mixer.w_out, b.feed_forward.w_gate_up, b.feed_forward.w_down))
    assert plain_llm.model.weight_bytes() - llm.model.weight_bytes() > 0.99 * layers  # a byte of two
    outputs = llm.generate(prompts, SamplingParams(max_new_tokens=12))
    again = llm.generate(prompts, SamplingParams(max_new_tokens=12))
    assert [o.token_ids for o in outputs] == [o.token_ids for o in again]
    assert all(len(o.token_ids) == 12 and o.finish_reason == "length" for o in outputs)
    llm.cache.check()


def test_programs_take_the_options(tmp_path, capsys, monkeypatch):
    import io
    import json

    from llmserve_triton_kernels_b200 import cli, replay
    from llmserve_triton_kernels_b200.config.presets import PRESETS

    monkeypatch.setitem(PRESETS, "small-test", CONFIG)
    cli.main(["--model", "small-test", "--max-new-tokens", "3", "--weight-dtype", "float8", "--cache-dtype", "float8", "--num-blocks", "16"])
    assert "decode=" in capsys.readouterr().out
    monkeypatch.setattr("sys.stdin", io.StringIO(json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [1, 2, 3], "want": [2]}]}) + "\n"))
    assert replay.main(["--random", "small-test", "--out", str(tmp_path), "--max-tokens", "64", "--weight-dtype", "float8", "--cache-dtype", "float8", "--seed", "3"]) == 0
    assert (tmp_path / "0.f32").stat().st_size == 4 * 300


def test_models_that_cannot_refuse():
    from llmserve_triton_kernels_b200 import LLM

    for options in ({"weight_dtype": "float8", "dtype": "float32"}, {"cache_dtype": "float8", "dtype": "float32"}, {"weight_dtype": "int4"}, {"cache_dtype": "int8"}):
        with pytest.raises(ValueError):
            LLM(CONFIG, num_blocks=8, freeze_gc=False, **options)
    for options in ({"weight_dtype": "float8"}, {"cache_dtype": "float8"}):
        with pytest.raises(ValueError, match="8-bit"):
            LLM("nurolorn-small", num_blocks=8, freeze_gc=False, **options)
