"""Attention over 8-bit pages where its numbers and its pages end; products whose work does not go round evenly."""

import plain_eight_bit as plain
import pytest
import torch
from test_eight_bit_gpu import (
    BF16, DEV, E4M3, F64, a_step, check_attention, check_product, check_scaled, gen, ops, pages8, request_rows, spread, weights,
)

pytestmark = pytest.mark.gpu


def a_token_that_draws(D, held, new, above, shift, seed):
    """A step over one request whose values have the size 2^(1 - shift), with one key at a place that every row sees; its score lies some
    ``above`` (0, 6 or 12) powers of two over the others', which lie within one of zero.  Returns ``(q, pool, exps, table, ctx, page, offset)``."""
    KV, page_size = 2, 16
    ctx, table, _, pages = a_step([new], [held], page_size, seed)
    pool, exps = pages8(pages, KV, page_size, D, seed)
    exps[:, 0] = 117  # keys of some 0.1
    exps[:, 1] = 120 - shift
    u = torch.randn(D, generator=gen(seed + 1), device=DEV).to(BF16)
    q = u.repeat(new, 8).contiguous()  # eight query heads, all alike
    at = (held - new) // 2
    page, off = int(table[0, at // page_size]), at % page_size
    pool[page, 0, :, off] = (448 * u.float().sign()).to(E4M3) if above else torch.zeros(D, device=DEV).to(E4M3)
    # 448 * sum|u| * 2^e * 0.05 * log2 e, sum|u| some 0.8 D: a power of two more for twice the lanes
    exps[page, 0, :, off] = {0: 127, 6: 119, 12: 120}[above] - (D == 128)
    return q, pool, exps, table, ctx, page, off


def attend(q, pool, exps, table, ctx, D, **kw):
    return ops().paged_attention8(q, pool, exps, table, ctx, num_heads=8, num_kv_heads=2, head_dim=D, scale=0.05, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("above", [0, 6, 12])
@pytest.mark.parametrize("shift", [0, 10, 24, 100])
@pytest.mark.parametrize("held,new", [(64, 1), (1500, 1), (90, 5)])
def test_a_value_of_zeros_draws_no_precision(D, above, shift, held, new):
    """A vector of zeros is written with scale one, whatever the others' scales: it takes its share of the weights' sum and nothing else."""
    q, pool, exps, table, ctx, page, off = a_token_that_draws(D, held, new, above, shift, held)
    pool.view(torch.uint8)[page, 1, 0, off] = 0
    pool.view(torch.uint8)[page, 1, 1, off] = 0x80  # the other zero
    exps[page, 1, :, off] = 127
    check_attention(attend(q, pool, exps, table, ctx, D), q, pool, exps, table, ctx, 8, D, 0.05, None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("above,far", [(0, 18), (6, 12), (12, 8)])
@pytest.mark.parametrize("held,new", [(64, 1), (1500, 1), (90, 5)])
def test_a_lane_far_above_the_others(D, above, far, held, new):
    """One lane of one value lies 2^far above everything else: where that value is zero the output is the others', whose weights (with their
    values' scales) lie within 2^-25 of the largest and keep their bits."""
    q, pool, exps, table, ctx, page, off = a_token_that_draws(D, held, new, above, 10, held)
    pool.view(torch.uint8)[page, 1, :, off] = 0
    pool[page, 1, :, off, 5] = 448.0
    exps[page, 1, :, off] = 110 + far
    check_attention(attend(q, pool, exps, table, ctx, D), q, pool, exps, table, ctx, 8, D, 0.05, None)


def small_weights_loss(q, pool, exps, table_row, length, new, H, D, scale, window):
    """What weights far below a row's largest may lose, ``[new, H, 1]``: with their values' scales they are held in half precision relative to a
    reference 2^11 to 2^15 below the largest, where a number has an error of 2^-25 at most: 2^-36 of the largest for every key, times a value of
    448 at most."""
    keys, _ = request_rows(pool, exps, table_row, length)
    at = torch.arange(length, device=DEV)
    ev = exps[table_row.long()[at // pool.shape[3]], 1, :, at % pool.shape[3]].to(F64) - 127  # [length, KV]
    group, place = H // pool.shape[2], torch.arange(length - new, length, device=DEV)
    s = torch.einsum("nhd,jhd->nhj", q[:, : H * D].view(new, H, D).to(F64), keys.repeat_interleave(group, 1)) * scale
    hidden = at[None] > place[:, None]
    if window is not None:
        hidden |= at[None] <= place[:, None] - window
    p = torch.softmax(s.masked_fill(hidden[:, None], -torch.inf), -1)
    largest = (p * torch.exp2(ev).t().repeat_interleave(group, 0)).amax(-1, keepdim=True)
    return length * 2.0**-36 * 448 * largest


def check_far_apart(got, q, pool, exps, table, held, new, H, D, scale, window):
    """As ``check_attention`` for one request, and what small weights may lose."""
    keys, values = request_rows(pool, exps, table[0], held)
    rows = q[:new, : H * D].view(new, H, D)
    want, size = (plain.attention(rows, keys, v, held - new, scale, window) for v in (values, values.abs()))
    off = (got[:new].view(new, H, D).to(F64) - want).abs()
    assert (off <= (2.0**-11 + 2.0**-15) * size + 2.0**-8 * want.abs() + small_weights_loss(q[:new], pool, exps, table[0], held, new, H, D, scale, window)).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("above", [0, 6, 12])
@pytest.mark.parametrize("far", [14, 30, 60, 120])
@pytest.mark.parametrize("held,new", [(64, 1), (1500, 1), (90, 5), (700, 21)])
def test_a_lane_beyond_half_precision(D, above, far, held, new):
    """... and however far: what the others lose then is small beside that lane."""
    q, pool, exps, table, ctx, page, off = a_token_that_draws(D, held, new, above, 10, held)
    pool.view(torch.uint8)[page, 1, :, off] = 0
    pool[page, 1, :, off, 5] = 448.0
    exps[page, 1, :, off] = 110 + far
    check_far_apart(attend(q, pool, exps, table, ctx, D), q, pool, exps, table, held, new, 8, D, 0.05, None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("held,new", [(40, 1), (1500, 1), (90, 5), (700, 21)])
@pytest.mark.parametrize("window", [None, 60])
def test_values_of_one_lane_with_scales_of_their_own(D, held, new, window):
    """Every value has one lane, and a scale anywhere in 2^-60 to 2^40: each lane's output is made of a few of them, whatever the others are."""
    ctx, table, _, pages = a_step([new], [held], 16, 8)
    pool, exps = pages8(pages, 2, 16, D, 9)
    lanes = torch.randint(0, D, exps[:, 1].shape, generator=gen(10), device=DEV)
    one = torch.nn.functional.one_hot(lanes, D).to(torch.bool)
    pool[:, 1] = torch.where(one, pool[:, 1].float(), 0.0).to(E4M3)
    exps[:, 1] = torch.randint(67, 167, exps[:, 1].shape, generator=gen(11), device=DEV).to(torch.uint8)
    q = torch.randn(new, 8 * D, generator=gen(12), device=DEV).to(BF16)
    check_far_apart(attend(q, pool, exps, table, ctx, D, window=window), q, pool, exps, table, held, new, 8, D, 0.05, window)


@pytest.mark.parametrize("exponent", [2, 8, 230])
def test_values_at_both_ends_of_the_exponents(exponent):
    """Scores that rise along the keys, so that references are moved, over values near the ends of what 32 bits and bfloat16 hold."""
    D, held = 64, 700
    ctx, table, _, pages = a_step([1], [held], 16, 3)
    pool, exps = pages8(pages, 2, 16, D, 4)
    exps[:, 1] = exponent
    q = torch.randn(1, 8 * D, generator=gen(5), device=DEV).to(BF16)
    check_attention(attend(q, pool, exps, table, ctx, D), q, pool, exps, table, ctx, 8, D, 0.05, None)


def nan_lanes(v, first, n, window):
    """Which rows and lanes see a NaN: ``v [len, KV, D]`` -> ``[n, KV, D]``."""
    bad, out = v.isnan(), []
    for p in range(first, first + n):
        out.append(bad[(0 if window is None else max(0, p - window + 1)) : p + 1].any(0))
    return torch.stack(out)


@pytest.mark.parametrize("D,page_size", [(64, 16), (128, 64), (128, 8), (64, 24)])
@pytest.mark.parametrize("window", [None, 5, 90])
def test_nan_reaches_the_rows_that_see_in_long_portions(D, page_size, window):
    """Values: the lanes that are NaN, for the rows that see them; keys: all lanes of those rows.  All other bits stay as they were."""
    H, KV, counts, held = 4, 2, [130, 1, 300, 40], [200, 70, 300, 50]
    ctx, table, _, pages = a_step(counts, held, page_size, 5)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(3), device=DEV).to(BF16)
    call = dict(num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1, window=window)
    clean = pages8(pages, KV, page_size, D, 12)
    want = ops().paged_attention8(q, *clean, table, ctx, **call).view(-1, H, D)
    # (request, position, key head, lane): seen by all of its rows, by some, by the last; two of one lane; beside a tile's end
    for which, places in ((1, [(0, 100, 0, 9)]), (1, [(0, 37, 1, 0), (2, 63, 0, D - 1), (2, 64, 0, 3), (2, 299, 1, 17), (3, 30, 1, 2)]), (1, [(2, 20, 0, 5), (2, 250, 0, 5)]),
                          (0, [(0, 150, 0, 9), (2, 299, 1, 1)]), (1, None)):
        pool, exps = (t.clone() for t in clean)
        if places is None:
            pool.view(torch.uint8)[:, 1] = 0xFF  # nothing but NaN
        for r, j, head, lane in places or ():
            pool[int(table[r, j // page_size]), which, head, j % page_size, lane] = torch.nan
        got = ops().paged_attention8(q, pool, exps, table, ctx, **call).view(-1, H, D)
        spoilt = []
        for r, n in enumerate(held):
            bad = nan_lanes(request_rows(pool, exps, table[r], n)[which], n - counts[r], counts[r], window)
            spoilt.append((bad if which else bad.any(-1, keepdim=True).expand_as(bad)).repeat_interleave(H // KV, 1))
        spoilt = torch.cat(spoilt)
        assert torch.equal(got.isnan(), spoilt) and torch.equal(got[~spoilt], want[~spoilt])


def test_nan_in_long_portions_as_a_graph():
    """Whether there is NaN is the device's business: a captured call finds it, and finds it gone."""
    H, KV, D = 4, 2, 64
    ctx, table, _, pages = a_step([200], [260], 16, 5)
    q = torch.randn(200, H * D, generator=gen(3), device=DEV).to(BF16)
    pool, exps = pages8(pages, KV, 16, D, 12)

    def go():
        return ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)

    want = go().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = go()
    place = (int(table[0, 100 // 16]), 1, 1, 100 % 16, 7)
    kept = pool[place].clone()
    for bad in (False, True, False):
        pool[place] = torch.nan if bad else kept.float()
        graph.replay()
        torch.cuda.synchronize()
        spoilt = torch.zeros(200, H, D, dtype=torch.bool, device=DEV)
        spoilt[40:, 2:, 7] = bad
        assert torch.equal(y.view(200, H, D).isnan(), spoilt) and torch.equal(y.view(200, H, D)[~spoilt], want.view(200, H, D)[~spoilt])


@pytest.mark.parametrize("KV,page_size,more_pages", [(1, 1, 0), (4, 3, 1), (2, 2, 0), (1, 4, 1), (3, 8, 1), (1, 16, 1)])
@pytest.mark.parametrize("counts,held", [([1, 3], [60, 33]), ([1], [2500])], ids=str)
def test_planes_of_a_cache(KV, page_size, more_pages, counts, held):
    """A cache's layers lie one after another in one allocation: the second and third start wherever the one in front ends."""
    D, H = 64, 2 * KV
    ctx, table, slots, pages = a_step(counts, held, page_size, 6, more_pages)
    if pages % 2 == 0:
        pages += 1
    pool, exps = pages8(3 * pages, KV, page_size, D, 7)
    pool, exps = pool.view(3, pages, 2, KV, page_size, D), exps.view(3, pages, 2, KV, page_size)
    qkv = torch.randn(ctx.num_tokens, (H + 2 * KV) * D, generator=gen(8), device=DEV).to(BF16)
    for plane in range(3):
        ops().rope_kv_write8(qkv, ctx.positions, None, slots, pool[plane], exps[plane], H, KV, D)
        got = ops().paged_attention8(qkv, pool[plane], exps[plane], table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
        check_attention(got, qkv, pool[plane], exps[plane], table, ctx, H, D, 0.1, None, f"plane {plane}")


def test_exponents_that_start_anywhere():
    """... and a caller's own, at any byte, over pages that hold tiles whole."""
    H, KV, D, page_size = 4, 2, 128, 16
    ctx, table, _, pages = a_step([1, 2, 130], [900, 40, 200], page_size, 6)
    pool, exps = pages8(pages, KV, page_size, D, 7)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(8), device=DEV).to(BF16)
    want = ops().paged_attention8(q, pool, exps, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    for offset in (1, 4, 8):
        room = torch.zeros(exps.numel() + offset, dtype=torch.uint8, device=DEV)
        moved = room[offset:].view(exps.shape)
        moved.copy_(exps)
        got = ops().paged_attention8(q, pool, moved, table, ctx, num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
        assert torch.equal(got, want), offset


def test_small_pages_in_the_engine():
    """Single-token pages, an odd number of them, two key heads: the second layer's exponents start on four bytes."""
    from llmserve_triton_kernels_b200 import LLM, SamplingParams
    from test_eight_bit_model_gpu import CONFIG

    prompts = [[5, 17, 200, 9], list(range(30, 45))]
    tokens = []
    for block_size, num_blocks in ((1, 101), (16, 8)):
        llm = LLM(CONFIG, seed=3, max_batch_size=2, block_size=block_size, num_blocks=num_blocks, cache_dtype="float8", freeze_gc=False)
        tokens.append([o.token_ids for o in llm.generate(prompts, SamplingParams(max_new_tokens=4))])
        llm.cache.check()
    assert [[len(t) for t in each] for each in tokens] == [[4, 4], [4, 4]]
    assert [t[0] for t in tokens[0]] == [t[0] for t in tokens[1]]


@pytest.mark.parametrize("counts,held", [([1, 3], [700, 33]), ([130], [200])], ids=str)
def test_windows_beyond_32_bits(counts, held):
    """A window that no context fills is none, however large the number."""
    H, KV, D = 4, 2, 64
    ctx, table, _, pages = a_step(counts, held, 16, 6)
    pool, exps = pages8(pages, KV, 16, D, 7)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(8), device=DEV).to(BF16)
    call = dict(num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    want = ops().paged_attention8(q, pool, exps, table, ctx, window=10_000, **call)
    for window in (2**31 - 1, 2**31, 2**32 + 5, 2**40):
        assert torch.equal(ops().paged_attention8(q, pool, exps, table, ctx, window=window, **call), want), window


@pytest.mark.parametrize("k", [1040, 2064, 2640, 2944, 4112])
@pytest.mark.parametrize("m", [20, 70, 300])
def test_k_blocks_shared_out_unevenly(m, k):
    """K-blocks that do not go evenly into the two or four CTAs, or the two pairs, of a tile: 9, 17, 21, 23 and 33."""
    x = spread(m, k, 1, k).to(BF16)
    for n in (130, 700):
        w = weights(n, k, n)
        check_product(ops().linear8(x, w), x, w, f"{n} features")
        w = ops().quantize_weight(spread(n, k, 128, n))
        check_scaled(ops().linear8(x, w), x, w, f"{n} features, powers of two")


@pytest.mark.parametrize("counts,held", [([130, 1], [200, 64]), ([40, 2], [200, 64])], ids=str)
@pytest.mark.parametrize("lowest", [torch.finfo(BF16).min, torch.finfo(BF16).max, 3.32e38], ids=str)
def test_values_of_the_types_lowest_number(counts, held, lowest):
    """bfloat16's largest numbers come to 2^128 in 8 bits, which 32 bits do not hold: rows that do not see them stay as they were, rows that do
    get their share.  (In long portions the largest bfloat16 number stands for 2^128: 2^-8 of it, as much as half a step of the output.)"""
    H, KV, D, page_size, place = 4, 2, 64, 16, 180
    ctx, table, _, pages = a_step(counts, held, page_size, 5)
    q = torch.randn(ctx.num_tokens, H * D, generator=gen(3), device=DEV).to(BF16)
    pool, exps = pages8(pages, KV, page_size, D, 12)
    call = dict(num_heads=H, num_kv_heads=KV, head_dim=D, scale=0.1)
    want = ops().paged_attention8(q, pool, exps, table, ctx, **call).view(-1, H, D)
    one = torch.zeros(1, 3 * KV * D, dtype=BF16, device=DEV)  # a key of zeros, and a value of zeros but for one lane
    one[0, 2 * KV * D + 7] = lowest
    slot = table[0, place // page_size] * page_size + place % page_size
    ops().rope_kv_write8(one, ctx.positions[:1], None, slot.view(1), pool, exps, KV, KV, D)
    got = ops().paged_attention8(q, pool, exps, table, ctx, **call).view(-1, H, D)
    first, last = held[0] - counts[0], place - (held[0] - counts[0])  # rows in front of `last` do not see the place
    assert torch.equal(got[:last], want[:last]) and torch.equal(got[counts[0] :], want[counts[0] :]) and not got.isnan().any()
    keys, values = request_rows(pool, exps, table[0], held[0])
    rows = q[: counts[0]].view(-1, H, D)
    exact, size = (plain.attention(rows, keys, v, first, 0.1, None) for v in (values, values.abs()))
    assert exact.abs().max() > 1e36
    # (long portions: weights in bfloat16, 2^-8 with the largest number's 2^-8; short ones: what small weights lose)
    loss = 0.0 if counts[0] >= 128 else small_weights_loss(q[: counts[0]], pool, exps, table[0], held[0], counts[0], H, D, 0.1, None)
    assert ((got[: counts[0]].to(F64) - exact).abs() <= (2.0**-7 + 2.0**-14) * size + 2.0**-8 * exact.abs() + loss).all()
