"""What the operators on 8-bit numbers are measured by: products with 8-bit weights, and attention over 8-bit pages.

A case is one call of one operator:

* ``quantize``: a matrix to e4m3 values with a power of two for every block of 128 columns (of one row: activations; of 128 rows:
  weights);
* ``linear``: activations (quantised within the call) times a matrix held in e4m3 with a 32-bit scale for every block of 128 x 128;
* ``write``: a step's query heads and keys rotated, its keys and values written into 8-bit pages, a scale for every head's vector;
* ``attention``: a step's tokens over their requests' 8-bit pages.

Heads, widths and vocabularies are those of the Llama presets.  Weights and activations are normal numbers, a few columns of the
activations far larger than the others, as behind a trained model's norms.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False
DEVICE = "cuda:0"
F64 = torch.float64
E4M3 = torch.float8_e4m3fn

HEADS = {"tinyllama": (32, 4, 64), "llama2-7b": (32, 32, 128), "llama3-8b": (32, 8, 128)}  # query heads, key heads, lanes


def listed():
    def quantize(name, m, k, rows=1, dtype="bfloat16"):
        return {"name": name, "op": "quantize", "m": m, "k": k, "rows": rows, "dtype": dtype}

    def linear(name, m, n, k, dtype="bfloat16", out="bfloat16"):
        return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "out": out}

    def write(name, heads, requests, tokens, page):
        return {"name": name, "op": "write", "heads": heads, "requests": requests, "tokens": tokens, "page": page}

    def attention(name, heads, requests, context, tokens=1, page=16, window=0):
        return {"name": name, "op": "attention", "heads": heads, "requests": requests, "context": context, "tokens": tokens, "page": page,
                "window": window}

    return [
        # the down projection's input of a batch that decodes
        quantize("rows_of_a_decode_step", 8, 5632),
        # a matrix of the largest model as it is loaded, in 32 bits
        quantize("a_weight_matrix_32_bit", 4096, 14336, rows=128, dtype="float32"),
        # one user decodes on the small model: the stacked query, key and value projection
        linear("one_token_qkv", 1, 2560, 2048),
        # a batch of eight decodes on the large model: the stacked gate and up projection
        linear("eight_tokens_gate_up", 8, 28672, 4096),
        # the logits of a crowded step, in 32 bits
        linear("logits_of_33_rows", 33, 32000, 2048, out="float32"),
        # a full step of prompts on the large model, gate and up
        linear("prompts_of_4096_gate_up", 4096, 28672, 4096),
        # a batch of eight decodes on the small model
        write("write_a_decode_step", "tinyllama", 8, 1, 16),
        # a full step of prompts on the large model
        write("write_prompts", "llama3-8b", 5, 1023, 16),
        # one user, short conversation, small model
        attention("one_user_short", "tinyllama", 1, 173),
        # a batch of eight in the middle of long conversations
        attention("batch_of_8", "llama3-8b", 8, 3981),
        # many users with long contexts: the cache is most of what a step reads
        attention("many_users_long", "llama3-8b", 32, 8191, page=32),
        # a portion of a prompt behind what is cached already
        attention("portions_of_prompts", "tinyllama", 3, 1501, tokens=301),
    ]


def draw(rng):
    """One more case: the same operators, every size anywhere in its range, odd ones included."""

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("quantize", "linear", "linear", "write", "attention", "attention"))
        if op == "quantize":
            case = {"op": op, "m": log(1, 4096), "k": log(1, 14336), "rows": rng.choice((1, 1, 128)), "dtype": rng.choice(("bfloat16", "bfloat16", "float32"))}
        elif op == "linear":
            case = {"op": op, "m": log(1, 4096), "n": log(40, 32000), "k": 16 * log(8, 896), "dtype": rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32")),
                    "out": rng.choice(("bfloat16", "bfloat16", "float32"))}
        elif op == "write":
            case = {"op": op, "heads": rng.choice(tuple(HEADS)), "requests": log(1, 32), "tokens": rng.choice((1, log(1, 2048))), "page": rng.choice((8, 16, 32, 64))}
            if case["requests"] * case["tokens"] > 5200:
                continue
        else:
            case = {"op": op, "heads": rng.choice(tuple(HEADS)), "requests": log(1, 64), "context": log(1, 16384), "tokens": rng.choice((1, 1, 1, log(2, 512))),
                    "page": rng.choice((8, 16, 32, 64)), "window": rng.choice((0, 0, 0, log(16, 4096)))}
            case["tokens"] = min(case["tokens"], case["context"])
            # the plain form holds all of a step's scores at once
            if case["requests"] * case["tokens"] > 3000 or case["requests"] * case["tokens"] * case["context"] > 2_000_000:
                continue
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _counts(case):
    """Tokens that every request brings, and what it holds behind them: ragged, from the sizes alone."""
    part = (1.0, 0.61, 0.87, 0.33, 0.72, 0.49, 0.94, 0.21)
    n = [max(1, int(round(case["tokens"] * part[r % 8]))) for r in range(case["requests"])]
    held = [max(c, int(round(case.get("context", case["tokens"]) * part[(r * 5) % 8]))) for r, c in enumerate(n)]
    return n, held


def work(case):
    if case["op"] == "quantize":
        m, k = case["m"], case["k"]
        blocks = -(-m // case["rows"]) * -(-k // 128)
        return {"bytes": m * k * (_size(case["dtype"]) + 1) + 4 * blocks, "flops": 2 * m * k}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * _size(case["dtype"]) + n * k + 4 * -(-n // 128) * -(-k // 128) + m * n * _size(case["out"]), "flops": 2 * m * n * k}
    h, kv, d = HEADS[case["heads"]]
    counts, held = _counts(case)
    tokens = sum(counts)
    if case["op"] == "write":
        return {"bytes": tokens * ((2 * h + 2 * kv) * d * 2 + 4 * d + 8 + 2 * kv * (d + 1)), "flops": tokens * (h + 2 * kv) * 3 * d}
    keys = pairs = 0
    for c, n in zip(counts, held):
        span = case["window"] or n
        keys += min(n, span + c - 1)
        pairs += sum(min(p + 1, span) for p in range(n - c, n))
    return {"bytes": keys * 2 * kv * (d + 1) + 2 * tokens * h * d * 2 + 4 * -(-keys // case["page"]), "flops": 4 * pairs * h * d}


def _size(dtype):
    return {"bfloat16": 2, "float32": 4}[dtype]


# ---------------------------------------------------------------------------------------------- inputs
def _rows(g, m, k, dtype):
    """Rows as behind a norm: normal numbers, every fiftieth column some ten times larger."""
    x = torch.randn((m, k), generator=g, device=DEVICE)
    far = torch.rand((k,), generator=g, device=DEVICE) < 0.02
    return torch.where(far, 10.0 * x, x).to(dtype)


def _weights(g, n, k):
    """A matrix in 8 bits as a checkpoint carries it: e4m3 values and a 32-bit scale for every block of 128 x 128."""
    values = (torch.randn((n, k), generator=g, device=DEVICE) * 100.0).clamp(-448.0, 448.0).to(E4M3)
    scales = 2e-4 * (0.5 + torch.rand((-(-n // 128), -(-k // 128)), generator=g, device=DEVICE))
    return values, scales


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = getattr(torch, case.get("dtype", "bfloat16"))
    if case["op"] == "quantize":
        return {"case": case, "x": _rows(g, case["m"], case["k"], dtype)}
    if case["op"] == "linear":
        values, scales = _weights(g, case["n"], case["k"])
        return {"case": case, "x": _rows(g, case["m"], case["k"], dtype), "w": values, "scales": scales}
    h, kv, d = HEADS[case["heads"]]
    counts, held = _counts(case)
    page, requests = case["page"], case["requests"]
    width = -(-max(held) // page)
    pages = requests * width + 3
    # every request's pages lie anywhere in the pool
    table = torch.randperm(pages, generator=g, device=DEVICE)[: requests * width].view(requests, width).to(torch.int32)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    ints = {"dtype": torch.int32, "device": DEVICE}
    start = torch.tensor([n - c for c, n in zip(counts, held)], **ints)
    owner = torch.repeat_interleave(torch.arange(requests, device=DEVICE), torch.tensor(counts, device=DEVICE))
    cu_tokens = torch.tensor(cu, **ints)
    positions = torch.arange(cu[-1], **ints) - cu_tokens[owner] + start[owner]
    slots = table[owner, (positions // page).long()] * page + positions % page
    step = SimpleNamespace(
        num_tokens=cu[-1], num_requests=requests, token_request=owner.to(torch.int32), cu_tokens=cu_tokens, context_lens=torch.tensor(held, **ints),
        positions=positions, host_cu_tokens=cu, host_context_lens=held, max_query_len=max(counts), max_context_len=max(held), static_decode=False,
        fresh_requests=False, shared={},
    )
    state = {"case": case, "step": step, "table": table, "slots": slots, "cu": cu_tokens, "owner": owner, "held": step.context_lens, "positions": positions}
    qkv = torch.randn((cu[-1], (h + 2 * kv) * d), generator=g, device=DEVICE).to(torch.bfloat16)
    if case["op"] == "write":
        most = max(held)
        inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float32, device=DEVICE) / d)
        angle = torch.arange(most, dtype=torch.float32, device=DEVICE)[:, None] * inv
        state |= {"qkv": qkv, "rotary": torch.cat((angle.cos(), angle.sin()), dim=1).contiguous()}
        state["pool"] = torch.zeros((pages, 2, kv, page, d), dtype=torch.uint8, device=DEVICE).view(E4M3)
        state["exponents"] = torch.full((pages, 2, kv, page), 127, dtype=torch.uint8, device=DEVICE)
        return state
    state["q"] = qkv[:, : h * d].contiguous()
    # keys and values as the write leaves them: a vector's largest value in (224, 448], scales around one
    raw = torch.randn((pages, 2, kv, page, d), generator=g, device=DEVICE)
    state["pool"] = (raw * (336.0 / raw.abs().amax(-1, keepdim=True))).to(E4M3)
    state["exponents"] = (127 - 8 + torch.randint(0, 3, (pages, 2, kv, page), generator=g, device=DEVICE)).to(torch.uint8)
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "quantize":
        if own:
            from llmserve_triton_kernels_b200 import ops

            q = ops.quantize_blocks(state["x"], rows=case["rows"])
            return q.values, q.scales
        return _plain_quantize(state["x"], case["rows"])
    if case["op"] == "linear":
        out = getattr(torch, case["out"])
        if own:
            from llmserve_triton_kernels_b200 import ops

            return ops.linear8(state["x"], ops.Quantized(state["w"], state["scales"], 128), out_dtype=out)
        return _plain_linear(state["x"], state["w"], state["scales"], out)
    h, kv, d = HEADS[case["heads"]]
    if case["op"] == "write":
        qkv = state["qkv"].clone()  # the queries are rotated in place: a step's projection is a new tensor every time
        if own:
            from llmserve_triton_kernels_b200 import ops

            ops.rope_kv_write8(qkv, state["positions"], state["rotary"], state["slots"], state["pool"], state["exponents"], h, kv, d)
        else:
            _plain_write(qkv, state, h, kv, d)
        return qkv[:, : h * d], state["pool"], state["exponents"]
    if own:
        from llmserve_triton_kernels_b200 import ops

        return ops.paged_attention8(state["q"], state["pool"], state["exponents"], state["table"], state["step"], num_heads=h, num_kv_heads=kv,
                                    head_dim=d, scale=d**-0.5, window=case["window"] or None)
    return _plain_attention(state, h, kv, d)


def _exponent(largest):
    """The smallest e with ``largest <= 448 * 2^e``: 448 is 1.75 * 2^8, and frexp gives a mantissa in [1/2, 1)."""
    mantissa, power = torch.frexp(largest)
    e = power - 9 + (mantissa > 0.875).to(torch.int32)
    return torch.where(largest > 0, e.clamp(min=-126), torch.zeros_like(e))


def _plain_quantize(x, rows):
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // 128)
    x = x.float()
    padded = torch.nn.functional.pad(x, (0, kb * 128 - k, 0, mb * rows - m))
    largest = padded.view(mb, rows, kb, 128).abs().amax(dim=(1, 3))
    scales = torch.exp2(_exponent(largest).float())
    each = scales.repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    return (x / each).to(E4M3), scales


def _plain_linear(x, w, scales, out):
    (m, k), n = x.shape, w.shape[0]
    values, row_scales = _plain_quantize(x, 1)
    left = values.float() * row_scales.repeat_interleave(128, 1)[:, :k]
    right = w.float() * scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return (left @ right.t()).to(out)


def _plain_write(qkv, state, h, kv, d):
    n = qkv.shape[0]
    rows = state["rotary"][state["positions"].long()]
    cos, sin = rows[:, None, : d // 2], rows[:, None, d // 2 :]
    heads = qkv[:, : (h + kv) * d].view(n, h + kv, d).float()
    low, high = heads[..., : d // 2], heads[..., d // 2 :]
    turned = torch.cat((low * cos - high * sin, high * cos + low * sin), dim=-1)
    qkv[:, : h * d] = turned[:, :h].reshape(n, h * d).to(qkv.dtype)
    both = torch.stack((turned[:, h:], qkv[:, (h + kv) * d :].view(n, kv, d).float()), dim=1)  # [n, 2, kv, d]
    e = _exponent(both.abs().amax(-1))
    page = state["pool"].shape[3]
    at, off = (state["slots"] // page).long(), (state["slots"] % page).long()
    state["pool"].view(torch.uint8)[at, :, :, off] = (both / torch.exp2(e.float())[..., None]).to(E4M3).view(torch.uint8)
    state["exponents"][at, :, :, off] = (e + 127).to(torch.uint8)


def _plain_attention(state, h, kv, d):
    case, step = state["case"], state["step"]
    r, t, page = case["requests"], step.max_query_len, case["page"]
    length = state["table"].shape[1] * page
    table = state["table"].long()
    scales = torch.exp2(state["exponents"][table].float() - 127.0)  # [r, width, 2, kv, page]
    both = state["pool"][table].float() * scales[..., None]
    both = both.permute(2, 0, 3, 1, 4, 5).reshape(2, r, kv, length, d)
    # the queries of every request side by side, padded to the longest portion
    place = state["owner"] * t + (torch.arange(step.num_tokens, device=DEVICE) - state["cu"][state["owner"]])
    q = torch.zeros((r * t, h * d), dtype=torch.float32, device=DEVICE)
    q[place] = state["q"].float()
    pos = torch.full((r * t,), -1, dtype=torch.int64, device=DEVICE)
    pos[place] = state["positions"].long()
    q = q.view(r, t, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(r, kv, (h // kv) * t, d)
    scores = (q @ both[0].transpose(-1, -2)).view(r, kv, h // kv, t, length) * d**-0.5
    key = torch.arange(length, device=DEVICE)
    pos = pos.view(r, 1, 1, t, 1)
    seen = key <= pos
    if case["window"]:
        seen = seen & (key > pos - case["window"])
    p = torch.exp(scores.masked_fill_(~seen, float("-inf")) - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = (p.view(r, kv, (h // kv) * t, length) @ both[1]).view(r, kv, h // kv, t, d) / total
    return out.permute(0, 3, 1, 2, 4).reshape(r * t, h * d)[place].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _to_grid(x):
    """64-bit numbers of size up to 448 to the nearest e4m3 value, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3.0)
    return torch.round(x / step) * step


def _power(largest):
    """2^e for the smallest e with ``largest <= 448 * 2^e``, by trying the neighbours of the logarithm."""
    e = torch.ceil(torch.log2(torch.where(largest > 0, largest, torch.full_like(largest, 448.0)) / 448.0))
    e = torch.where(largest <= 448.0 * torch.exp2(e - 1.0), e - 1.0, e)
    e = torch.where(largest > 448.0 * torch.exp2(e), e + 1.0, e)
    return torch.exp2(e.clamp(min=-126.0))


def _exact_blocks(x, rows):
    """Values and scales of every block, by walking the blocks' columns."""
    x = x.to(F64)
    values, scales = torch.empty_like(x), []
    for k0 in range(0, x.shape[1], 128):
        piece = x[:, k0 : k0 + 128]
        top = piece.abs().amax(1)
        if rows > 1:
            top = torch.stack([t.max() for t in top.split(rows)])
        s = _power(top)
        scales.append(s)
        values[:, k0 : k0 + 128] = _to_grid(piece / s.repeat_interleave(rows)[: x.shape[0], None])
    return values, torch.stack(scales, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_blocks(state["x"], case["rows"])
    if case["op"] == "linear":
        values, scales = _exact_blocks(state["x"], 1)
        out = torch.zeros((case["m"], case["n"]), dtype=F64, device=DEVICE)
        for b, k0 in enumerate(range(0, case["k"], 128)):
            right = state["w"][:, k0 : k0 + 128].to(F64) * state["scales"][:, b].to(F64).repeat_interleave(128)[: case["n"], None]
            out += (values[:, k0 : k0 + 128] * scales[:, b : b + 1]) @ right.t()
        return out
    h, kv, d = HEADS[case["heads"]]
    counts, held = _counts(case)
    page = case["page"]
    if case["op"] == "write":
        rows = state["rotary"].to(F64)[state["positions"].long()]
        z = state["qkv"][:, : (h + kv) * d].to(F64).view(-1, h + kv, 2, d // 2)
        turn = torch.complex(rows[:, : d // 2], rows[:, d // 2 :])[:, None]
        z = torch.complex(z[:, :, 0], z[:, :, 1]) * turn
        z = torch.cat((z.real, z.imag), dim=-1)
        pool = state["pool"].to(F64)
        slots = state["slots"].long()
        for which, vectors in ((0, z[:, h:]), (1, state["qkv"][:, (h + kv) * d :].to(F64).view(-1, kv, d))):
            for head in range(kv):
                v = vectors[:, head]
                pool[slots // page, which, head, slots % page] = _to_grid(v / _power(v.abs().amax(1))[:, None])
        return z[:, :h].reshape(-1, h * d), pool, None
    out = torch.empty((sum(counts), h * d), dtype=F64, device=DEVICE)
    first = 0
    for r, (c, n) in enumerate(zip(counts, held)):
        where = torch.arange(n, device=DEVICE)
        pages, off = state["table"][r].long()[where // page], where % page
        i, j = torch.arange(n - c, n, device=DEVICE)[:, None], where[None]
        hidden = (j > i) | ((j <= i - case["window"]) if case["window"] else torch.zeros_like(j > i))
        for head in range(kv):
            k, v = (state["pool"][pages, w, head, off].to(F64) * torch.exp2(state["exponents"][pages, w, head, off].to(F64) - 127.0)[:, None] for w in (0, 1))
            for member in range(h // kv):
                lanes = slice((head * (h // kv) + member) * d, (head * (h // kv) + member + 1) * d)
                s = (state["q"][first : first + c, lanes].to(F64) @ k.t()) / math.sqrt(d)
                out[first : first + c, lanes] = torch.softmax(s.masked_fill(hidden, float("-inf")), dim=1) @ v
        first += c
    return out
