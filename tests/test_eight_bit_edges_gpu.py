"""Attention over 8-bit pages where its numbers and its pages end."""

import pytest
import torch
from test_eight_bit_gpu import BF16, DEV, E4M3, a_step, check_attention, gen, ops, pages8

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


@pytest.mark.parametrize("exponent", [2, 8, 230])
def test_values_at_both_ends_of_the_exponents(exponent):
    """Scores that rise along the keys, so that references are moved, over values near the ends of what 32 bits and bfloat16 hold."""
    D, held = 64, 700
    ctx, table, _, pages = a_step([1], [held], 16, 3)
    pool, exps = pages8(pages, 2, 16, D, 4)
    exps[:, 1] = exponent
    q = torch.randn(1, 8 * D, generator=gen(5), device=DEV).to(BF16)
    check_attention(attend(q, pool, exps, table, ctx, D), q, pool, exps, table, ctx, 8, D, 0.05, None)
