"""Grouped-query attention over a paged cache of keys and values.

Parity: src/llmserve/model/llama.py:57-88 (projections without bias, rotary encoding of q and k
before the cache write, head-major concatenation into the output projection) and
src/llmserve/kvcache/paged.py:81-110 (key j is visible to the query at position p iff j <= p;
consecutive query heads share a key/value head; softmax scale 1/sqrt(head_dim), which arrives
here as the parameter ``scale``).  ``window`` (None in Llama) limits a query to the last
``window`` keys, itself included.  With ``own_kv=False`` the layer has no key and value
projections and reads the cache that an earlier layer of the order wrote.  Over 8-bit pages (``cache.exponents``) the projection,
the rotation with the write, and the attention are kernels of their own.  ``qkv_bias`` and
``out_bias`` (both off in Llama; the reference's projections take the first as a flag,
src/llmserve/model/llama.py:64-66) give the projections bias vectors ``*_proj.bias``: such a layer
runs its products and the bias sums as kernels of their own, not the fused decode kernels.

Three options lead off the fused kernels onto the general ones (``ops.unit_norm_kv_write`` and
``ops.biased_paged_attention``): ``value_dim`` (values of another size than queries and keys), ``qk_norm_eps`` (every
query and key head is divided by its root mean square ``sqrt(mean(x^2) + eps)``, a norm without a weight), and
``distance_bias`` b (the score of key j for the query at position i loses ``slope_h * (i - j)`` with
``slope_h = 2^(-b (h+1) / num_heads)``).  ``tensor_names`` renames the four matrices.

The position encoding is a part of its own.  One whose ``rotary_layout`` is ``"half"`` (pairs
``(j, j + head_dim/2)`` over the whole head, angles tabulated as ``rotary_table``) is applied by the
kernels that also store keys and values; any other is asked to ``apply`` itself to q and k.
"""

from __future__ import annotations

import torch

from .. import ops
from .base import Mixer, PagedKVSpec, PartSpec, TensorSpec, build_part, register_part


class PagedAttention(Mixer):
    def __init__(
        self,
        hidden_size: int,
        num_heads: int,
        num_kv_heads: int,
        head_dim: int,
        scale: float,
        window: int | None = None,
        position: PartSpec | None = None,
        own_kv: bool = True,
        qkv_bias: bool = False,
        out_bias: bool = False,
        value_dim: int | None = None,
        qk_norm_eps: float | None = None,
        distance_bias: float | None = None,
        tensor_names: dict[str, str] | None = None,
    ):
        if num_heads % num_kv_heads:
            raise ValueError(f"num_heads {num_heads} is not a multiple of num_kv_heads {num_kv_heads}")
        if window is not None and window < 1:
            raise ValueError(f"window must be positive or None, got {window}")
        if not 1 <= int(head_dim) <= 256:
            raise ValueError(f"head_dim {head_dim} is not supported: the attention kernels take head sizes up to 256")
        self.hidden_size = int(hidden_size)
        self.num_heads = int(num_heads)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.scale = float(scale)
        self.window = None if window is None else int(window)
        self.own_kv = bool(own_kv)
        self.qkv_bias = bool(qkv_bias)
        self.out_bias = bool(out_bias)
        self.value_dim = self.head_dim if value_dim is None else int(value_dim)
        if not 1 <= self.value_dim <= 256:
            raise ValueError(f"value_dim {value_dim} is not supported: the attention kernels take value sizes up to 256")
        self.qk_norm_eps = None if qk_norm_eps is None else float(qk_norm_eps)
        self.distance_bias = None if distance_bias is None else float(distance_bias)
        self.general = self.value_dim != self.head_dim or self.qk_norm_eps is not None or self.distance_bias is not None
        if self.general and (position is not None or not own_kv or qkv_bias or out_bias):
            raise ValueError("value_dim, qk_norm_eps and distance_bias are built for layers with keys and values of their own, no position part and no biases")
        self.names = {"q": "q_proj.weight", "k": "k_proj.weight", "v": "v_proj.weight", "o": "o_proj.weight", **(tensor_names or {})}
        self.slopes: torch.Tensor | None = None  # [H] float32 with distance_bias
        self.b_in: torch.Tensor | None = None  # [(H + 2 KV) D] with qkv_bias
        self.b_out: torch.Tensor | None = None  # [hidden] with out_bias
        self.position = build_part("position", position) if position is not None else None
        self.w_in: torch.Tensor | None = None  # [(H + 2 KV) D, hidden], or [H D, hidden] without own_kv
        self.w_out: torch.Tensor | None = None  # [hidden, H D]

    def tensors(self) -> dict[str, TensorSpec]:
        q = self.num_heads * self.head_dim
        kv = self.num_kv_heads * self.head_dim
        n = self.names
        specs = {n["q"]: TensorSpec((q, self.hidden_size))}
        if self.own_kv:
            specs[n["k"]] = TensorSpec((kv, self.hidden_size))
            specs[n["v"]] = TensorSpec((self.num_kv_heads * self.value_dim, self.hidden_size))
        specs[n["o"]] = TensorSpec((self.hidden_size, self.num_heads * self.value_dim))
        if self.qkv_bias:
            specs[n["q"].replace(".weight", ".bias")] = TensorSpec((q,))
            if self.own_kv:
                specs[n["k"].replace(".weight", ".bias")] = TensorSpec((kv,))
                specs[n["v"].replace(".weight", ".bias")] = TensorSpec((kv,))
        if self.out_bias:
            specs[n["o"].replace(".weight", ".bias")] = TensorSpec((self.hidden_size,))
        return specs

    def bind(self, tensors, dtype, device) -> None:
        names = [self.names["q"]] + ([self.names["k"], self.names["v"]] if self.own_kv else [])
        fused = torch.cat([tensors[n].to(dtype) for n in names], dim=0)
        self.w_in = fused.to(device).contiguous()
        self.w_out = tensors[self.names["o"]].to(device=device, dtype=dtype).contiguous()
        if self.distance_bias is not None:
            heads = torch.arange(1, self.num_heads + 1, dtype=torch.float64)
            self.slopes = torch.pow(2.0, -self.distance_bias * heads / self.num_heads).to(torch.float32).to(device)
        if self.qkv_bias:
            self.b_in = torch.cat([tensors[n.replace(".weight", ".bias")].to(dtype) for n in names]).to(device).contiguous()
        if self.out_bias:
            self.b_out = tensors[self.names["o"].replace(".weight", ".bias")].to(device=device, dtype=dtype).contiguous()
        if self.position is not None:
            self.position.bind({}, dtype, device)

    def refuse_eight_bit_weights(self) -> str | None:
        if self.general:
            return "8-bit weights are not built for attention with value_dim, qk_norm_eps or distance_bias"
        return ops.refuse_quantize(self.w_in) or ops.refuse_quantize(self.w_out)

    def quantize_weights(self) -> None:
        super().quantize_weights()
        self.w_in, self.w_out = ops.quantize_weight(self.w_in), ops.quantize_weight(self.w_out)

    @property
    def eight_bit_pages(self) -> bool:
        return not self.general and self.head_dim in ops.ATTENTION8_HEAD_DIMS

    def cache_spec(self) -> PagedKVSpec:
        return PagedKVSpec(self.num_kv_heads, max(self.head_dim, self.value_dim), self.window)

    accepts_sink = True

    @property
    def graph_safe(self) -> bool:
        """The same launches whatever a step holds, if the position encoding's are too."""
        return self.position is None or bool(getattr(self.position, "graph_safe", False))

    def _rotary_table(self):
        """The table of a position encoding that the fused kernels know how to apply, else None."""
        if getattr(self.position, "rotary_layout", None) != "half":
            return None
        table = getattr(self.position, "rotary_table", None)
        return table if table is not None and table.shape[1] == self.head_dim else None

    def forward(self, x, ctx, cache, sink=None):
        H, KV, D = self.num_heads, self.num_kv_heads, self.head_dim
        if self.general:
            return self._forward_general(x, ctx, cache, sink)
        table = self._rotary_table()
        qkv = None
        eight_bit = getattr(cache, "exponents", None) is not None
        if (self.position is None or table is not None) and self.b_in is None and not eight_bit:
            # few rows: projection, rotation and the cache write in one kernel
            qkv = ops.linear_qkv_rope(
                x, self.w_in, ctx.positions, table, cache.slot_map, cache.pool, H, KV, D, write_kv=self.own_kv
            )
        if qkv is None:
            qkv = self._project_rotate_store(x, ctx, cache, table)
        heads = {"num_heads": H, "num_kv_heads": KV, "head_dim": D, "scale": self.scale, "window": self.window}
        if eight_bit:
            out = ops.paged_attention8(qkv, cache.pool, cache.exponents, cache.page_table, ctx, **heads)
        else:
            out = ops.paged_attention(qkv, cache.pool, cache.page_table, ctx, **heads)
        # the contribution to the 32-bit residual stream leaves the product in 32-bit: it is the sum's largest addend
        if self.b_out is not None:
            return ops.add_bias(ops.linear(out, self.w_out, out_dtype=torch.float32), self.b_out.float())
        if sink is not None:
            handed_on = sink.linear(out, self.w_out)
            if handed_on is not None:
                return handed_on
        return ops.linear(out, self.w_out, out_dtype=torch.float32)

    def _forward_general(self, x, ctx, cache, sink):
        """Projection, the unit-RMS norms with the cache write, attention with its bias, output projection."""
        H, KV = self.num_heads, self.num_kv_heads
        qkv = ops.linear(x, self.w_in)
        ops.unit_norm_kv_write(qkv, cache.slot_map, cache.pool, self.qk_norm_eps, H, KV, self.head_dim, self.value_dim)
        out = ops.biased_paged_attention(
            qkv, cache.pool, cache.page_table, ctx, num_heads=H, num_kv_heads=KV, key_dim=self.head_dim,
            value_dim=self.value_dim, scale=self.scale, window=self.window, slopes=self.slopes,
        )
        if sink is not None:
            handed_on = sink.linear(out, self.w_out)
            if handed_on is not None:
                return handed_on
        return ops.linear(out, self.w_out, out_dtype=torch.float32)

    def _project_rotate_store(self, x, ctx, cache, table):
        H, KV, D = self.num_heads, self.num_kv_heads, self.head_dim
        qkv = ops.linear(x, self.w_in)
        if self.b_in is not None:
            ops.add_bias(qkv, self.b_in)
        if self.position is not None and table is None:
            # a position encoding without a table: let it rewrite q and k, then store unrotated
            n = qkv.shape[0]
            q = qkv[:, : H * D].unflatten(1, (H, D))
            k = qkv[:, H * D : (H + KV) * D].unflatten(1, (KV, D)) if self.own_kv else qkv.new_empty((n, 0, D))
            self.position.apply(q, k, ctx.positions)
        if self.own_kv and getattr(cache, "exponents", None) is not None:
            ops.rope_kv_write8(qkv, ctx.positions, table, cache.slot_map, cache.pool, cache.exponents, H, KV, D)
            return qkv
        ops.rope_kv_write(
            qkv, ctx.positions, table, cache.slot_map, cache.pool, H, KV, D, write_kv=self.own_kv
        )
        return qkv


register_part("mixer", "attention", PagedAttention)
