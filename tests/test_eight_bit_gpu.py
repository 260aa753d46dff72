"""Products with 8-bit weights and attention over 8-bit pages, each kernel against its definition in 64 bits."""

from types import SimpleNamespace

import plain_eight_bit as plain
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3, BF16, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64


def ops():
    from llmserve_triton_kernels_b200 import ops

    return ops


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def same(a, b):
    """Equal numbers, NaN where the other has NaN."""
    a, b = a.to(F64), b.to(F64)
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------------------------------------ quantize_blocks
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 127), (5, 128), (2, 136), (127, 260), (129, 257), (130, 1000), (300, 384)])
def test_quantize_is_its_definition(m, k, rows, dtype):
    x = torch.randn(m, k, generator=gen(m * 1000 + k), device=DEV)
    x = (x * torch.exp2(torch.randint(-20, 20, (m, 1), generator=gen(1), device=DEV).float())).to(dtype)
    x[0, 0] = 0.0
    pitched = torch.full((m, k + 11), 7.0, dtype=dtype, device=DEV)  # rows that start anywhere
    pitched[:, 3 : k + 3] = x
    wide = torch.full((m, k + 24), 7.0, dtype=dtype, device=DEV)  # rows on 16 bytes
    wide[:, 8 : k + 8] = x
    values, scales = plain.quantize(x, rows)
    for form in (x, pitched[:, 3 : k + 3], wide[:, 8 : k + 8]):
        q = ops().quantize_blocks(form, rows=rows)
        assert q.values.dtype == E4M3 and tuple(q.values.shape) == (m, k) and same(q.values, values)
        assert same(q.scales, scales)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("k", [128, 125])  # the kernel that loads sixteen bytes, and the one for every layout
def test_quantize_at_the_edges_of_the_numbers(k, dtype):
    """Blocks of zeros, of the smallest and largest numbers, with a largest value on and beside 448 * 2^e, with NaN and infinities, of ties."""
    g = gen(5)
    x = torch.zeros(16, k, device=DEV)
    x[1], x[2] = 2.0**-133, -(2.0**-126)  # numbers below the normal ones (as bfloat16 has them), and the smallest normal one
    x[3] = 3.3e38 * (2 * torch.rand(k, generator=g, device=DEV) - 1)
    x[4], x[5], x[6] = 448.0 * 2.0**5, 450.0 * 2.0**5, -446.0 * 2.0**-60
    x[7, 3], x[7, 4], x[7, 5], x[7, 6] = torch.nan, torch.inf, -torch.inf, 5.0
    x[8, 0] = torch.inf  # nothing finite but zeros
    x[9] = torch.nan
    x[10] = (2 * torch.arange(k, device=DEV) % 448 + 1.0) / 16  # odd multiples of half a step between e4m3 numbers
    x[10, 0] = 448.0
    x[11] = torch.exp2(-(torch.arange(k, device=DEV) % 40).float())  # down to where e4m3 ends
    x[12] = -1e-30 * torch.rand(k, generator=g, device=DEV)
    x[13, k - 1] = 1e-20
    x = x.to(dtype)
    values, scales = plain.quantize(x)
    q = ops().quantize_blocks(x)
    assert same(q.scales, scales) and same(q.values, values)
    tile = ops().quantize_blocks(x, rows=128)
    values, scales = plain.quantize(x, 128)
    assert same(tile.scales, scales) and same(tile.values, values)


def test_quantize_nothing():
    for shape in ((0, 128), (3, 0), (0, 0)):
        q = ops().quantize_blocks(torch.empty(shape, dtype=BF16, device=DEV))
        assert tuple(q.shape) == shape and tuple(q.scales.shape) == (shape[0], -(-shape[1] // 128))


# ------------------------------------------------------------------------------------------------ linear8
def weights(n, k, seed):
    g = gen(seed)
    values = (torch.randn(n, k, generator=g, device=DEV) * 120).clamp(-448, 448).to(E4M3)
    scales = torch.rand(-(-n // 128), -(-k // 128), generator=g, device=DEV) * 0.01 + 1e-4
    return ops().Quantized(values, scales, 128)


def check_product(got, x, w, what=""):
    """A 128-term block sum and the sum over blocks, in any order and with truncation: at most (128 + blocks + 8 warps + 2 scales)
    roundings of 2^-23 of the terms' sizes; then half a step of the output's type."""
    want, size = plain.linear(x, w.values, w.scales)
    steps = 128 + w.scales.shape[1] + 10
    out = torch.finfo(got.dtype).eps / 2
    off = (got.to(F64) - want).abs()
    assert (off <= steps * 2.0**-23 * size * (1 + out) + out * want.abs()).all(), f"{what}: {(off / size.clamp(min=1e-30)).max():.3g} of the terms' sizes"


@pytest.mark.parametrize("k", [16, 112, 128, 144, 1040, 2064])
@pytest.mark.parametrize("n", [1, 15, 16, 127, 128, 130, 400])
def test_linear_is_its_definition(n, k):
    w = weights(n, k, n * 31 + k)
    x = torch.randn(300, k, generator=gen(k), device=DEV)
    x[:, k // 2] *= 30
    for m in (1, 2, 7, 8, 9, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 257, 300):
        rows = x[:m].to(BF16) if m % 2 else x[:m].contiguous()
        for out in (BF16, F32):
            got = ops().linear8(rows, w, out_dtype=out)
            assert got.dtype == out and tuple(got.shape) == (m, n)
            check_product(got, rows, w, f"{m} rows, {out}")
    assert ops().linear8(x[:3].to(BF16), w).dtype == BF16 and ops().linear8(x[:3], w).dtype == F32
    assert tuple(ops().linear8(x[:0], w).shape) == (0, n)


def test_linear_of_many_tiles():
    """More tiles than SMs, ragged at both ends, in every tile width: column tiles cross the weights' blocks of 128."""
    for m, n, k in ((1100, 2000, 272), (513, 9000, 400), (65, 20000, 144), (2049, 700, 528)):
        w = weights(n, k, m)
        x = torch.randn(m, k, generator=gen(n), device=DEV).to(BF16)
        check_product(ops().linear8(x, w), x, w, f"{m} x {n} x {k}")
        check_product(ops().linear8(x, w, out_dtype=F32), x, w, f"{m} x {n} x {k}, 32-bit")


def spread(m, k, rows, seed, most=8):
    """Normal numbers, every block of ``rows`` by 128 times a power of two of its own."""
    g = gen(seed)
    e = torch.randint(-most, most + 1, (-(-m // rows), -(-k // 128)), generator=g, device=DEV).float()
    return torch.randn(m, k, generator=g, device=DEV) * torch.exp2(e).repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def check_scaled(got, x, w, what=""):
    """Sums of 32 terms and over K / 32 of them, with truncation, and at most four partial sums: (32 + 4 blocks + 4) steps of 2^-23 of the
    terms' sizes; then half a step of the output's type."""
    want, size = plain.linear(x, w.values, w.scales)
    steps = 32 + 4 * w.scales.shape[1] + 4
    out = torch.finfo(got.dtype).eps / 2
    off = (got.to(F64) - want).abs()
    assert (off <= steps * 2.0**-23 * size * (1 + out) + out * want.abs()).all(), f"{what}: {(off / size.clamp(min=1e-30)).max():.3g} of the terms' sizes"


@pytest.mark.parametrize("k", [16, 128, 144, 528, 1040, 2064])
@pytest.mark.parametrize("n", [1, 16, 130, 400])
def test_linear_with_powers_of_two(n, k):
    w = ops().quantize_weight(spread(n, k, 128, n + k))
    assert w.powers_of_two
    x = spread(300, k, 1, k)
    for m in (9, 17, 32, 33, 64, 65, 127, 128, 129, 300):
        for out in (BF16, F32):
            got = ops().linear8(x[:m], w, out_dtype=out)
            assert got.dtype == out and tuple(got.shape) == (m, n)
            check_scaled(got, x[:m], w, f"{m} rows, {out}")


@pytest.mark.parametrize("m,n,k", [(1100, 2000, 272), (513, 9000, 400), (65, 20000, 144), (2049, 1500, 528), (300, 19000, 1040), (40, 24000, 656), (900, 1100, 4112), (513, 2304, 6000), (257, 4097, 4096)])
def test_linear_of_many_tiles_with_powers_of_two(m, n, k):
    w = ops().quantize_weight(spread(n, k, 128, m))
    x = spread(m, k, 1, n).to(BF16)
    check_scaled(ops().linear8(x, w), x, w)
    check_scaled(ops().linear8(x, w, out_dtype=F32), x, w, "32-bit")
    q = ops().quantize_blocks(x)  # a caller's: its scales lie the other way round
    assert q.powers_of_two and torch.equal(ops().linear8(q, w), ops().linear8(x, w))
    # the same numbers without the promise, by the kernels for scales of any value
    plainer = ops().Quantized(w.values, w.scales, 128)
    check_product(ops().linear8(x, plainer), x, plainer)
    check_product(ops().linear8(ops().Quantized(q.values, q.scales), w), x, w)


@pytest.mark.parametrize("m,n", [(40, 200), (200, 200), (400, 9000)])
def test_linear_where_powers_of_two_end(m, n):
    """Scales at both ends of 32 bits' exponents whose products lie inside; blocks of zeros; NaN that stays in its row."""
    k = 640
    x, w = torch.randn(m, k, generator=gen(1), device=DEV), torch.randn(n, k, generator=gen(2), device=DEV)
    x[:, :128] *= 2.0**-118
    w[:, :128] *= 2.0**115
    x[:, 128:256] *= 2.0**110
    w[:, 128:256] *= 2.0**-113
    x[:, 256:384] = 0
    w[:, 384:512] = 0
    wq = ops().quantize_weight(w)
    want = ops().linear8(x, wq)
    check_scaled(want, x, wq)
    bad = x.clone()
    bad[m // 2, 300] = torch.nan
    bad[m - 1, 5] = torch.inf
    got = ops().linear8(bad, wq)
    spoilt = torch.zeros(m, dtype=torch.bool, device=DEV)
    spoilt[[m // 2, m - 1]] = True
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("m", [5, 40, 100])
def test_linear_of_rows_in_other_forms(m):
    k, n = 400, 200
    w = weights(n, k, m)
    x = torch.randn(m, k, generator=gen(m), device=DEV).to(BF16)
    want = ops().linear8(x, w)
    loose = torch.zeros(m, k + 5, dtype=BF16, device=DEV)
    loose[:, 3 : k + 3] = x
    assert torch.equal(ops().linear8(loose[:, 3 : k + 3], w), want)
    assert torch.equal(ops().linear8(ops().quantize_blocks(x), w), want)
    assert torch.equal(ops().linear(x, w), want)
    # activations with scales that are no powers of two, as another program may have quantised them
    q = ops().Quantized(ops().quantize_blocks(x).values, torch.rand(m, -(-k // 128), device=DEV) + 0.1, 1)
    left = q.values.to(F64) * plain.spread(q.scales, 1, m, k)
    right = w.values.to(F64) * plain.spread(w.scales, 128, n, k)
    got, size = ops().linear8(q, w, out_dtype=F32).to(F64), left.abs() @ right.abs().t()
    assert ((got - left @ right.t()).abs() <= 142 * 2.0**-23 * size).all()
    # factored rows, as a bfloat16 part in front may hand them on
    ss = torch.rand(3, m, device=DEV) * k
    normed = ops().NormedInput(x, ss, 1e-5)
    assert torch.equal(ops().linear(normed, w), ops().linear8(normed.materialize(), w))


@pytest.mark.parametrize("m", [9, 70])
def test_linear_rows_do_not_meet(m):
    """A row with NaN or infinities is NaN, the others are what they were; a row's bits do not depend on the rows beside it."""
    w = weights(300, 272, 3)
    x = torch.randn(m, 272, generator=gen(m), device=DEV).to(BF16)
    want = ops().linear8(x, w)
    bad = x.clone()
    bad[2, 200], bad[5, 0], bad[m - 1, 271] = torch.nan, torch.inf, -torch.inf
    got = ops().linear8(bad, w)
    spoilt = torch.zeros(m, dtype=torch.bool, device=DEV)
    spoilt[[2, 5, m - 1]] = True
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])
    assert torch.equal(ops().linear8(x[: m - 3], w), want[: m - 3])


@pytest.mark.parametrize("m", [3, 64, 65])
def test_linear_of_weights_just_written(m):
    """Weights quantised by the launch directly in front, over what lay there before: no kernel reads them early."""
    a = torch.randn(512, 1024, generator=gen(1), device=DEV)
    x = torch.randn(m, 1024, generator=gen(2), device=DEV).to(BF16)
    xq = ops().quantize_blocks(x)
    want = [ops().linear8(x, ops().quantize_weight(a * f)).clone() for f in (1.0, -3.0)]
    torch.cuda.synchronize()
    for turn in range(20):
        f = (1.0, -3.0)[turn % 2]
        scaled = a * f
        w = ops().quantize_weight(scaled)  # takes up the memory of the one before
        assert torch.equal(ops().linear8(xq, w), want[turn % 2])
        w = ops().quantize_weight(scaled)
        assert torch.equal(ops().linear8(x, w), want[turn % 2])


# ------------------------------------------------------------------------------------------------ rope_kv_write8
def a_step(counts, held, page_size, seed, more_pages=3):
    """A step's arrays: request r brings ``counts[r]`` tokens and holds ``held[r]`` behind them; its pages lie anywhere."""
    g, requests = gen(seed), len(counts)
    width = max(1, -(-max(held) // page_size))
    pages = requests * width + more_pages
    table = torch.randperm(pages, generator=g, device=DEV)[: requests * width].view(requests, width).to(torch.int32)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    i32 = {"dtype": torch.int32, "device": DEV}
    owner = torch.repeat_interleave(torch.arange(requests, device=DEV), torch.tensor(counts, device=DEV))
    cu_t = torch.tensor(cu, **i32)
    start = torch.tensor([n - c for n, c in zip(held, counts)], **i32)
    positions = torch.arange(cu[-1], **i32) - cu_t[owner] + start[owner]
    at = positions.clamp(min=0)
    slots = (table[owner, (at // page_size).long()] * page_size + at % page_size).to(torch.int32)
    ctx = SimpleNamespace(num_tokens=cu[-1], num_requests=requests, cu_tokens=cu_t, context_lens=torch.tensor(held, **i32), host_cu_tokens=cu,
                          max_query_len=max(counts), max_context_len=max(held), positions=positions, token_request=owner.to(torch.int32))
    return ctx, table, slots, pages


def pages8(pages, kv, page_size, d, seed):
    """Pages as a cache holds them: every vector's exponent its own."""
    g = gen(seed)
    pool = (torch.randn(pages, 2, kv, page_size, d, generator=g, device=DEV) * 100).clamp(-448, 448).to(E4M3)
    return pool, torch.randint(115, 123, (pages, 2, kv, page_size), generator=g, device=DEV).to(torch.uint8)


def rotary(d, places):
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=F32, device=DEV) / d)
    a = torch.arange(places, dtype=F32, device=DEV)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).contiguous()


@pytest.mark.parametrize("page_size", [1, 8, 16, 24])
@pytest.mark.parametrize("H,KV,D", [(8, 2, 64), (4, 4, 128), (5, 1, 64)])
def test_write_is_its_definition(H, KV, D, page_size):
    ctx, table, slots, pages = a_step([1, 19, 3], [40, 19, 7], page_size, H * 10 + D)
    n, width = ctx.num_tokens, (H + 2 * KV) * D
    wide = torch.randn(n, width + 16, generator=gen(7), device=DEV).to(BF16)
    wide[3, H * D + 5], wide[4, (H + KV) * D + 1] = torch.nan, torch.inf  # a key and a value that are not finite
    wide[5, H * D :] = 0.0
    wide[6, H * D :] *= 1e30
    wide[7, H * D :] *= 1e-37
    slots[9], slots[10] = -1, pages * page_size  # no place of the pool: not stored
    for rope in (rotary(D, 41), None):
        qkv = wide.clone()
        rows = qkv[:, :width]
        pool, exps = pages8(pages, KV, page_size, D, 2)
        was, was_exps = pool.clone(), exps.clone()
        ops().rope_kv_write8(rows, ctx.positions, rope, slots, pool, exps, H, KV, D)
        heads = wide[:, :width].view(n, H + 2 * KV, D)
        turned = heads[:, : H + KV].float() if rope is None else plain.turn(heads[:, : H + KV], rope, ctx.positions)
        assert same(qkv[:, : H * D], turned[:, :H].reshape(n, H * D).to(BF16))
        assert same(qkv[:, H * D :], wide[:, H * D :])  # nothing but the queries changes
        vectors = torch.stack((turned[:, H:], heads[:, H + KV :].float()), 1).to(F64)  # [n, 2, KV, D]
        e = plain.exponents(plain.finite_top(vectors, -1))
        want, want_exps = was.to(F64), was_exps.long()
        for t in range(n):
            if 0 <= int(slots[t]) < pages * page_size:
                page, off = divmod(int(slots[t]), page_size)
                want[page, :, :, off] = plain.grid(vectors[t] / torch.exp2(e[t].to(F64))[..., None])
                want_exps[page, :, :, off] = e[t] + 127
        assert same(pool, want) and torch.equal(exps.long(), want_exps)


# ------------------------------------------------------------------------------------------------ paged_attention8
def request_rows(pool, exps, table_row, length):
    """A request's keys and values ``[len, KV, D]`` in 64 bits."""
    page_size = pool.shape[3]
    j = torch.arange(length, device=DEV)
    at, off = table_row.long()[j // page_size], j % page_size
    both = pool[at, :, :, off].to(F64) * torch.exp2(exps[at, :, :, off].to(F64) - 127)[..., None]
    return both[:, 0], both[:, 1]


def check_attention(got, q, pool, exps, table, ctx, H, D, scale, window, what=""):
    """Weights in half precision (2^-11 of each), a 32-bit sum, the output's half step (2^-8); exponents of scores up to some 2^7 in
    32 bits (2^-24 * 2^7 * log 2 of each weight, and as much from the approximate exponential): relative to the values' sizes."""
    cu, held = ctx.host_cu_tokens, ctx.context_lens.tolist()
    for r in range(len(held)):
        a, b = cu[r], cu[r + 1]
        if a == b:
            continue
        k, v = request_rows(pool, exps, table[r], max(held[r], 0))
        rows = q[a:b, : H * D].view(b - a, H, D)
        want = plain.attention(rows, k, v, held[r] - (b - a), scale, window)
        size = plain.attention(rows, k, v.abs(), held[r] - (b - a), scale, window)
        off = (got[a:b].view(b - a, H, D).to(F64) - want).abs()
        bound = (2.0**-11 + 2.0**-15) * size + 2.0**-8 * want.abs()
        assert ((off <= bound) | (got[a:b].view_as(off).isnan() & want.isnan())).all(), f"{what}, request {r}: {(off / bound.clamp(min=1e-30)).max():.3g} of the bound"


CASES = {
    "one token each": ([1] * 6, [1, 2, 15, 16, 17, 300]), "long and short": ([1, 1, 1], [5, 2500, 64]), "portions": ([1, 40, 17, 2], [90, 40, 200, 2]),
    "one token alone": ([1], [1]), "one long one": ([1], [4000]), "a request without tokens": ([1, 0, 3], [20, 9, 30]), "a request that holds nothing": ([1, 1], [0, 33]),
}


@pytest.mark.parametrize("window", [None, 1, 7, 130])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("H,KV,D,page_size", [(8, 2, 64, 16), (4, 4, 128, 8), (20, 1, 64, 1), (34, 2, 128, 32), (2, 1, 128, 48), (3, 3, 64, 24)])
def test_attention_is_its_definition(H, KV, D, page_size, case, window):
    counts, held = CASES[case]
    ctx, table, _, pages = a_step(counts, held, page_size, H + D + page_size)
    pool, exps = pages8(pages, KV, page_size, D, 11)
    # what nobody sees is NaN: places behind a request's end, pages that are nobody's
    needed = torch.zeros(pages, page_size, dtype=torch.bool, device=DEV)
    for r, n in enumerate(held):
        j = torch.arange(max(n, 0), device=DEV)
        needed[table[r].long()[j // page_size], j % page_size] = True
    pool.view(torch.uint8).permute(0, 3, 1, 2, 4)[~needed] = 0x7F
    exps.permute(0, 3, 1, 2)[~needed] = 255
    q = torch.randn(ctx.num_tokens, H * D + 8, generator=gen(3), device=DEV).to(BF16)
    got = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.05, window=window)
    check_attention(got, q, pool, exps, table, ctx, H, D, 0.05, window, case)
    if 0 in held:
        assert not got[0].any()


@pytest.mark.parametrize("window", [None, 70])
@pytest.mark.parametrize("counts,held", [([130], [130]), ([300, 1, 40, 200, 5], [301, 700, 40, 260, 5]), ([1, 128], [0, 900]), ([129, 0, 31], [400, 9, 31])], ids=str)
@pytest.mark.parametrize("H,KV,D,page_size", [(8, 2, 64, 16), (4, 1, 128, 8), (3, 3, 64, 64), (4, 2, 128, 24)])
def test_attention_of_prompt_portions(H, KV, D, page_size, counts, held, window):
    """Requests of many tokens, over unpacked pages, beside others that are not; weights are rounded to bfloat16 there, which has 7 bits behind
    the leading one: half a step is 2^-8 of a weight."""
    ctx, table, _, pages = a_step(counts, held, page_size, H + D + page_size)
    pool, exps = pages8(pages, KV, page_size, D, 11)
    needed = torch.zeros(pages, page_size, dtype=torch.bool, device=DEV)
    for r, n in enumerate(held):
        j = torch.arange(n, device=DEV)
        needed[table[r].long()[j // page_size], j % page_size] = True
    pool.view(torch.uint8).permute(0, 3, 1, 2, 4)[~needed] = 0x7F
    exps.permute(0, 3, 1, 2)[~needed] = 255
    q = torch.randn(ctx.num_tokens, H * D + 8, generator=gen(3), device=DEV).to(BF16)
    got = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.05, window=window)
    cu = ctx.host_cu_tokens
    for r, n in enumerate(held):
        rows = q[cu[r] : cu[r + 1], : H * D].view(-1, H, D)
        k, v = request_rows(pool, exps, table[r], n)
        want, size = (plain.attention(rows, k, x, n - rows.shape[0], 0.05, window) for x in (v, v.abs()))
        off = (got[cu[r] : cu[r + 1]].view_as(want).to(F64) - want).abs()
        assert (off <= (2.0**-8 + 2.0**-14) * size + 2.0**-8 * want.abs()).all(), r


@pytest.mark.parametrize("split", [(2, 0), (8, 0), (8, 1), (8, 5), (8, 148), (2, 9)], ids=str)
@pytest.mark.parametrize("H,KV,D,page_size", [(8, 2, 64, 16), (40, 4, 64, 8), (16, 2, 128, 24), (20, 1, 128, 16), (4, 4, 128, 5)])
@pytest.mark.parametrize("longest", [900, 512])  # 513 keys and more of some request: stretches cut; fewer: they hold whole units
def test_attention_however_it_is_shared_out(monkeypatch, H, KV, D, page_size, split, longest):
    counts, held = [1, 1, 7, 0, 1, 30], [1, longest, 130, 40, 0, min(600, longest)]
    monkeypatch.setattr(ops(), "_ATTENTION8_SPLIT", split)
    ctx, table, _, pages = a_step(counts, held, page_size, 5)
    pool, exps = pages8(pages, KV, page_size, D, 12)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(4), device=DEV).to(BF16)
    for window in (None, 50):
        got = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1, window=window)
        check_attention(got, q, pool, exps, table, ctx, H, D, 0.1, window, f"{split} {window}")


def test_attention_of_many_short_requests():
    """More tiles of rows than there is room for at once: CTAs of two warps."""
    H, KV, D, page_size = 16, 16, 64, 16
    g = torch.Generator().manual_seed(8)
    held = torch.randint(1, 60, (50,), generator=g).tolist()
    ctx, table, _, pages = a_step([1] * 50, held, page_size, 9)
    pool, exps = pages8(pages, KV, page_size, D, 13)
    q = torch.randn(50, H * D, generator=gen(5), device=DEV).to(BF16)
    assert ops()._attention8_split(50, KV, 1, max(held), D) == (2, 0)
    got = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.125)
    check_attention(got, q, pool, exps, table, ctx, H, D, 0.125, None)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_reaches_the_rows_that_see(D):
    """NaN in a value or a key spoils the rows that see it and no other, also inside a tile of 16 keys that others see in part."""
    H, KV, page_size = 4, 2, 16
    ctx, table, _, pages = a_step([30, 1], [50, 40], page_size, 5)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(3), device=DEV).to(BF16)
    call = dict(num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    for which in (0, 1):
        for window in (None, 5):
            pool, exps = pages8(pages, KV, page_size, D, 12)
            want = ops().paged_attention8(q, pool, exps, table, ctx, window=window, **call)
            page, off = int(table[0, 37 // 16]), 37 % 16
            pool[page, which, 1, off, 9] = torch.nan  # position 37 of request 0 (token 17 of its 30), key head 1, lane 9
            got = ops().paged_attention8(q, pool, exps, table, ctx, window=window, **call)
            last = 30 if window is None else min(30, 17 + window)
            spoilt = torch.zeros(31, H, D, dtype=torch.bool, device=DEV)
            if which:
                spoilt[17:last, 2:, 9] = True
            else:
                spoilt[17:last, 2:] = True
            got, want = got.view(31, H, D), want.view(31, H, D)
            assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("what", ["large queries", "small queries", "values far apart", "scores far apart", "values of zero"])
@pytest.mark.parametrize("held", [40, 1200])
def test_attention_over_the_numbers_range(held, what):
    H, KV, D, page_size = 8, 2, 64, 16
    ctx, table, _, pages = a_step([1, 2], [held, held // 2], page_size, 8)
    pool, exps = pages8(pages, KV, page_size, D, 13)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(4), device=DEV)
    scale = 0.02
    if what == "large queries":
        q, scale = q * 1e30, 2e-32
    elif what == "small queries":
        q, scale = q * 1e-30, 2e28
    elif what == "values far apart":
        exps[:, 1] = torch.randint(60, 180, exps[:, 1].shape, generator=gen(9), device=DEV).to(torch.uint8)
    elif what == "scores far apart":
        scale = 1.0  # of hundreds: most weights vanish
        exps[:, 0] = 118
    else:
        pool.view(torch.uint8)[:, 1] = 0
        exps[:, 1] = 127
    q = q.to(BF16)
    got = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=scale)
    if what == "scores far apart":
        # a score of size S has an error of some S * 2^-22 (32-bit sums of 64 terms): with S up to 2^10 it shows in the weights
        cu, lens = ctx.host_cu_tokens, ctx.context_lens.tolist()
        for r in range(2):
            k, v = request_rows(pool, exps, table[r], lens[r])
            rows = q[cu[r] : cu[r + 1]].view(-1, H, D)
            want = plain.attention(rows, k, v, lens[r] - rows.shape[0], scale, None)
            size = plain.attention(rows, k, v.abs(), lens[r] - rows.shape[0], scale, None)
            off = (got[cu[r] : cu[r + 1]].view_as(want).to(F64) - want).abs()
            assert (off <= (2.0**-11 + 2.0**-10) * size + 2.0**-8 * want.abs()).all()
        return
    check_attention(got, q, pool, exps, table, ctx, H, D, scale, None, what)


def test_attention_of_pages_far_back_in_a_large_pool():
    """Places of the pool whose offset does not fit 32 bits."""
    H, KV, D, page_size, pages = 8, 8, 128, 16, 140_000  # 4.6 GB
    pool = torch.zeros(pages, 2, KV, page_size, D, dtype=torch.uint8, device=DEV).view(E4M3)
    exps = torch.full((pages, 2, KV, page_size), 127, dtype=torch.uint8, device=DEV)
    ctx, table, slots, _ = a_step([3, 1], [3, 1], page_size, 1)
    table = torch.tensor([[pages - 1], [pages - 2]], dtype=torch.int32, device=DEV)
    slots = (table[ctx.token_request.long(), 0] * page_size + ctx.positions).to(torch.int32)
    qkv = torch.randn(4, 3 * H * D, generator=gen(1), device=DEV).to(BF16)
    ops().rope_kv_write8(qkv, ctx.positions, rotary(D, 4), slots, pool, exps, H, KV, D)
    got = ops().paged_attention8(qkv, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    check_attention(got, qkv, pool, exps, table, ctx, H, D, 0.1, None)
    assert pool[pages - 1, :, :, :3].float().abs().amax(-1).min() > 200 and not pool[: pages - 2].view(torch.uint8).any()


def test_bad_pages_and_slots_touch_nothing():
    """Entries of a page table that name no page are read as one that exists, behind a request's end or not; a slot that is none is skipped."""
    H, KV, D, page_size = 4, 2, 64, 16
    ctx, table, slots, pages = a_step([2, 1], [40, 17], page_size, 2)
    pool, exps = pages8(pages, KV, page_size, D, 3)
    table[0, 2], table[1, 1] = 2**31 - 1, -7
    slots[:] = torch.tensor([-(2**31), 2**31 - 1, pages * page_size], dtype=torch.int32, device=DEV)
    was, was_exps = pool.clone(), exps.clone()
    qkv = torch.randn(3, (H + 2 * KV) * D, generator=gen(1), device=DEV).to(BF16)
    ops().rope_kv_write8(qkv, ctx.positions - 100, rotary(D, 4), slots, pool, exps, H, KV, D)
    assert same(pool, was) and torch.equal(exps, was_exps)
    got = ops().paged_attention8(qkv, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    assert got.isfinite().all()


# ------------------------------------------------------------------------------------------------ together
def chain(x, w_in, w_out, rope, pool, exps, ctx, table, slots, H, KV, D):
    qkv = ops().linear8(x, w_in)
    ops().rope_kv_write8(qkv, ctx.positions, rope, slots, pool, exps, H, KV, D)
    out = ops().paged_attention8(qkv, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=D**-0.5)
    return ops().linear8(out, w_out, out_dtype=F32), qkv, out


@pytest.mark.parametrize("counts,held", [([1, 1, 1], [1, 40, 700]), ([40, 1, 30], [40, 33, 300])])
def test_a_layers_run(counts, held):
    """The four as a layer runs them, each step held to its definition on what the one before it left."""
    H, KV, D, page_size, hidden = 8, 2, 64, 16, 272
    ctx, table, slots, pages = a_step(counts, held, page_size, 4)
    pool, exps = pages8(pages, KV, page_size, D, 5)
    w_in, w_out = weights((H + 2 * KV) * D, hidden, 1), weights(hidden, H * D, 2)
    x = torch.randn(ctx.num_tokens, hidden, generator=gen(6), device=DEV).to(BF16)
    rope = rotary(D, 800)
    y, qkv, out = chain(x, w_in, w_out, rope, pool, exps, ctx, table, slots, H, KV, D)
    check_attention(out, qkv, pool, exps, table, ctx, H, D, D**-0.5, None)
    check_product(y, out, w_out)
    fresh = ops().linear8(x, w_in)
    check_product(fresh, x, w_in)
    n = ctx.num_tokens
    turned = plain.turn(fresh.view(n, -1, D)[:, : H + KV], rope, ctx.positions)
    assert same(qkv[:, : H * D], turned[:, :H].reshape(n, -1).to(BF16))


def test_captured_replayed_and_beside_one_another():
    """The run as a graph, replayed on other inputs while the same run goes on eagerly on another stream."""
    H, KV, D, page_size, hidden = 8, 2, 64, 16, 256
    ctx, table, slots, pages = a_step([1] * 4, [30, 100, 600, 1], page_size, 4)
    w_in, w_out = weights((H + 2 * KV) * D, hidden, 1), weights(hidden, H * D, 2)
    rope = rotary(D, 800)
    inputs = [torch.randn(4, hidden, generator=gen(s), device=DEV).to(BF16) for s in range(4)]
    caches = [pages8(pages, KV, page_size, D, s) for s in (5, 5)]

    def go(x, cache):
        return chain(x, w_in, w_out, rope, *cache, ctx, table, slots, H, KV, D)[0]

    want = [go(x, pages8(pages, KV, page_size, D, 5)).clone() for x in inputs]
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(x, caches[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = go(x, caches[0])
    torch.cuda.synchronize()
    for turn in range(12):
        x.copy_(inputs[turn % 4])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = [go(inputs[(turn + i) % 4], caches[1]) for i in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(y, want[turn % 4])
        for i, o in enumerate(other):
            assert torch.equal(o, want[(turn + i) % 4])


def test_large_calls_beside_one_another():
    """Every kernel of the products and of the attention on two streams at once, with the results that each has alone."""
    o = ops()
    calls = []
    for m, n, k, powers in ((3, 4000, 1024, True), (40, 3000, 1040, True), (40, 3000, 1040, False), (200, 1000, 2064, True), (200, 1000, 2064, False), (700, 9000, 528, True),
                            (700, 9000, 528, False), (600, 1100, 4112, True), (500, 4000, 528, False)):
        w = o.quantize_weight(spread(n, k, 128, m + k)) if powers else weights(n, k, m + k)
        x = spread(m, k, 1, n).to(BF16)
        calls.append(lambda x=x, w=w: o.linear8(x, w))
    for H, KV, D, counts, held in ((16, 2, 128, [1] * 5, [3000, 20, 700, 1500, 1]), (8, 8, 64, [1] * 60, list(range(1, 61))), (8, 2, 64, [200, 1, 140], [500, 900, 140])):
        ctx, table, _, pages = a_step(counts, held, 16, H)
        cache = pages8(pages, KV, 16, D, H)
        q = torch.randn(ctx.num_tokens, H * D, generator=gen(H), device=DEV).to(BF16)
        calls.append(lambda q=q, cache=cache, table=table, ctx=ctx, heads=(H, KV, D): o.paged_attention8(
            q, *cache, table, ctx, num_heads=heads[0], num_kv_heads=heads[1], head_dim=heads[2], scale=0.1))
    want = [call().clone() for call in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for turn in range(8):
        got = []
        for i in range(len(calls)):
            for j, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    at = (i * (1 + 4 * j) + turn * j) % len(calls)
                    got.append((at, calls[at]()))
        torch.cuda.synchronize()
        for at, y in got:
            assert torch.equal(y, want[at]), at
    o.check_device_errors()


def test_operands_on_the_host_are_refused():
    o = ops()
    x, w = torch.randn(4, 128, device=DEV).to(BF16), weights(64, 128, 1)
    with pytest.raises(o.KernelError, match="current device"):
        o.quantize_blocks(x.cpu())
    with pytest.raises(o.KernelError, match="current device"):
        o.linear8(x, o.Quantized(w.values.cpu(), w.scales.cpu(), 128))
    ctx, table, slots, pages = a_step([1], [5], 16, 1)
    pool, exps = pages8(pages, 2, 16, 64, 1)
    q = torch.randn(1, 4 * 64, device=DEV).to(BF16)
    with pytest.raises(o.KernelError, match="current device"):
        o.paged_attention8(q.cpu(), pool, exps, table, ctx, num_heads=4, num_kv_heads=2, head_dim=64, scale=1.0)
