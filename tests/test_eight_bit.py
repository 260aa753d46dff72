"""8-bit weights and pages on the host: what is refused, what the cache manager keeps, how options reach the parts."""

from types import SimpleNamespace

import plain_eight_bit as plain
import pytest
import torch

from llmserve_triton_kernels_b200 import ops
from llmserve_triton_kernels_b200.cache import CacheManager, num_pages_for_budget
from llmserve_triton_kernels_b200.config.presets import PRESETS
from llmserve_triton_kernels_b200.config.registry import architecture_of
from llmserve_triton_kernels_b200.models.load import quantized_weights, random_model, resolve_cache_dtype
from llmserve_triton_kernels_b200.parts.base import PagedKVSpec, PagedRowSpec
from llmserve_triton_kernels_b200.models.plan import LayerRun

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def e4m3(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(E4M3)


def test_the_definition_agrees_with_torch_on_every_number():
    """The tests' own rounding against torch's conversion, over every e4m3 number, the middles between neighbours and beside them."""
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    every = every[every.isfinite()].sort().values
    x = torch.cat((every, (every[1:] + every[:-1]) / 2, torch.linspace(-448, 448, 5001, dtype=torch.float64)))
    assert torch.equal(plain.grid(x), x.float().to(E4M3).double())
    assert plain.exponents(torch.tensor([0.0, 448.0, 448.1, 1.75, 1.7500001, 1e-45, 3.4e38], dtype=torch.float64)).tolist() == [0, 0, 1, -8, -7, -126, 120]


@pytest.mark.parametrize("make", [
    lambda: ops.Quantized(e4m3(4, 256), torch.ones(4, 2), 2),
    lambda: ops.Quantized(torch.zeros(4, 256), torch.ones(4, 2)),
    lambda: ops.Quantized(e4m3(256, 4).t(), torch.ones(4, 2)),
    lambda: ops.Quantized(e4m3(4, 256), torch.ones(4, 3)),
    lambda: ops.Quantized(e4m3(4, 256), torch.ones(1, 2)),
    lambda: ops.Quantized(e4m3(4, 256), torch.ones(4, 2, dtype=BF16)),
    lambda: ops.Quantized(e4m3(4, 256), torch.ones(2, 4).t()),
], ids=["rows", "type", "strides", "columns", "blocks", "scales' type", "scales' strides"])
def test_a_matrix_in_8_bits_is_whole(make):
    with pytest.raises(ops.KernelError):
        make()


def test_products_refuse():
    w = ops.Quantized(e4m3(128, 64), torch.ones(1, 1), 128)
    x = torch.zeros(3, 64, dtype=BF16)
    for call, why in (
        (lambda: ops.quantize_blocks(x, rows=64), "1 or 128"), (lambda: ops.quantize_blocks(x.half()), "not supported"),
        (lambda: ops.quantize_blocks(x.t()), "unit inner stride"), (lambda: ops.quantize_blocks(x[0]), "matrix"),
        (lambda: ops.quantize_weight(torch.zeros(4, 40)), "multiple of 16"), (lambda: ops.quantize_weight(torch.zeros(4, 0)), "multiple of 16"),
        (lambda: ops.linear8(x, torch.zeros(128, 64)), "Quantized"), (lambda: ops.linear8(x, ops.Quantized(e4m3(3, 64), torch.ones(3, 1))), "every 128 rows"),
        (lambda: ops.linear8(x[:, :32], w), "do not match"), (lambda: ops.linear8(w, w), "scale for every row"),
        (lambda: ops.linear8(x[:, :8], ops.Quantized(e4m3(128, 8), torch.ones(1, 1), 128)), "multiple of 16"),
        (lambda: ops.linear8(x, w, out_dtype=torch.float16), "not supported"), (lambda: ops.linear8(x.double(), w), "not supported"),
        (lambda: ops.linear(x[:, :32], w), "do not match"),
    ):
        with pytest.raises(ops.KernelError, match=why):
            call()


def test_attention_refuses():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    pool, exps = e4m3(5, 2, 2, 16, 64), torch.zeros(5, 2, 2, 16, dtype=torch.uint8)
    q, table = torch.zeros(2, 8 * 64, dtype=BF16), torch.zeros(2, 3, dtype=torch.int32)
    ctx = SimpleNamespace(cu_tokens=i32(0, 1, 2), context_lens=i32(5, 6), host_cu_tokens=[0, 1, 2], max_context_len=6, max_query_len=1)
    good = dict(q=q, pool=pool, exponents=exps, page_table=table, ctx=ctx, num_heads=4, num_kv_heads=2, head_dim=64, scale=1.0, window=None)
    for change, why in (
        (dict(q=q.float()), "bfloat16"), (dict(q=q[:, ::2]), "rows of q"), (dict(num_heads=9), "rows of q"), (dict(num_heads=3), "query heads over"),
        (dict(pool=pool.view(torch.uint8)), "float8"), (dict(pool=pool[:, :1]), "pool plane"), (dict(num_kv_heads=4), "pool plane"), (dict(head_dim=32), "pool plane"),
        (dict(exponents=exps[:4]), "exponents"), (dict(exponents=exps.int()), "exponents"), (dict(window=0), "window"),
        (dict(pool=e4m3(5, 2, 2, 16, 32), head_dim=32), "lanes"), (dict(q=torch.zeros(2, 513, dtype=BF16)), "8 bytes"),
    ):
        with pytest.raises(ops.KernelError, match=why):
            ops.paged_attention8(**{**good, **change})
    qkv, slots, pos = torch.zeros(2, 8 * 64, dtype=BF16), i32(0, 1), i32(0, 1)
    good = dict(qkv=qkv, positions=pos, table=torch.zeros(9, 64), slot_map=slots, pool=pool, exponents=exps, num_heads=4, num_kv_heads=2, head_dim=64)
    for change, why in (
        (dict(qkv=qkv.float()), "bfloat16"), (dict(num_heads=5), "512|576"), (dict(exponents=exps[:, :1].contiguous()), "exponents"),
        (dict(qkv=torch.zeros(2, 515, dtype=BF16)), "16 bytes"), (dict(pool=pool.transpose(2, 3)), "pool plane"),
    ):
        with pytest.raises(ops.KernelError, match=why):
            ops.rope_kv_write8(**{**good, **change})


def test_the_cache_keeps_a_byte_for_every_vector():
    specs = [PagedKVSpec(2, 64), PagedKVSpec(2, 64), PagedKVSpec(4, 128, window=32)]
    cache = CacheManager(specs, [LayerRun(i) for i in range(3)], page_size=8, num_pages=6, max_requests=2, dtype=E4M3, device="cpu")
    assert [g.pool.dtype for g in cache.groups] == [E4M3, E4M3]
    assert [tuple(g.exponents.shape) for g in cache.groups] == [(2, 6, 2, 2, 8), (1, 6, 2, 4, 8)]
    assert cache.nbytes() == sum(g.pool.numel() + g.exponents.numel() for g in cache.groups) == sum(6 * g.bytes_per_page() for g in cache.groups)
    cache.add_request("a")
    cache.reserve([("a", 9)])
    tables, slots = cache.step_tables([("a", 9)])
    views = cache.views([(torch.from_numpy(t), torch.from_numpy(s)) for t, s in tables], torch.from_numpy(slots), slots.tolist())
    assert all(v.exponents.shape == v.pool.shape[:4] for v in views)
    assert views[1].exponents.data_ptr() == cache.groups[0].exponents[1].data_ptr()
    assert num_pages_for_budget(specs, 8, 1, 10 * sum(g.bytes_per_page() for g in cache.groups) + 3) == 10
    with pytest.raises(ValueError, match="latent"):
        CacheManager([PagedRowSpec(64)], [LayerRun(0)], page_size=8, num_pages=6, max_requests=2, dtype=E4M3, device="cpu")
    plain_cache = CacheManager(specs, [LayerRun(i) for i in range(3)], page_size=8, num_pages=6, max_requests=2, dtype=BF16, device="cpu")
    assert all(g.exponents is None for g in plain_cache.groups)


def _small(**kw):
    return {**PRESETS["tinyllama-1.1b"], "hidden_size": 256, "intermediate_size": 272, "num_hidden_layers": 2, "num_attention_heads": 4,
            "num_key_value_heads": 2, "vocab_size": 300, "max_position_embeddings": 64, **kw}


def test_options_are_checked():
    assert not quantized_weights(None) and quantized_weights("float8") and quantized_weights(E4M3)
    with pytest.raises(ValueError, match="weight_dtype"):
        quantized_weights("int8")
    assert resolve_cache_dtype(None, BF16) == BF16 and resolve_cache_dtype("float8", BF16) == E4M3
    with pytest.raises(ValueError, match="cache_dtype"):
        resolve_cache_dtype("bfloat16", BF16)

    def model(cfg, dtype):
        config = architecture_of(cfg).config_class.from_dict(cfg)
        return random_model(config, 0, dtype, "cpu")

    assert resolve_cache_dtype("float8", BF16, model(_small(), BF16)) == E4M3
    for cfg, dtype in ((_small(), torch.float32), (_small(num_attention_heads=8), BF16), (PRESETS["nurolorn-small"], BF16)):
        with pytest.raises(ValueError, match="8-bit pages"):
            resolve_cache_dtype("float8", BF16, model(cfg, dtype))
    with pytest.raises(ValueError, match="bfloat16 activations"):
        model(_small(), torch.float32).quantize_weights()


def test_parts_put_their_matrices_into_8_bits(monkeypatch):
    """By the plain definition: which matrices, in which blocks; the rest stays as it was, and a part that cannot refuses."""

    def quantize(w, rows=1):
        values, scales = plain.quantize(w, rows)
        return ops.Quantized(values.float().to(E4M3), scales.float(), rows)

    monkeypatch.setattr(ops, "quantize_blocks", quantize)
    cfg = _small()
    m = random_model(architecture_of(cfg).config_class.from_dict(cfg), 0, BF16, "cpu")
    block, before = m.blocks[0], m.weight_bytes()
    was = block.mixer.w_in.clone()
    m.quantize_weights()
    for w, shape in ((block.mixer.w_in, (512, 256)), (block.mixer.w_out, (256, 256)), (block.feed_forward.w_gate_up, (544, 256)), (block.feed_forward.w_down, (256, 272))):
        assert isinstance(w, ops.Quantized) and tuple(w.shape) == shape and w.rows == 128
    assert m.head.dtype == BF16 and block.mixer_norm.weight.dtype == torch.float32
    assert m.weight_bytes() < 0.75 * before
    # e4m3 keeps 4 bits of every value down to 2^-15 of its block's largest
    off = (block.mixer.w_in.dequantize() - was.float()).abs()
    assert (off <= was.float().abs() * 2.0**-4 + block.mixer.w_in.scales.max() * 2.0**-10).all()
    latent = random_model(architecture_of(PRESETS["nurolorn-small"]).config_class.from_dict(PRESETS["nurolorn-small"]), 0, BF16, "cpu")
    with pytest.raises(ValueError, match="8-bit weights are not built"):
        latent.quantize_weights()
