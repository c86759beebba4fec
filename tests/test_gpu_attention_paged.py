"""Paged attention where it is easily wrong: scores that rise all the time, what 16-bit probabilities lose, sums over long
contexts, values and queries that are not finite, tiny scales, windows beyond an int, page tables of one row."""
import math

import pytest
import torch

import q4kb200 as q
import serving_reference as ref
from test_gpu_paged import TYPES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scores_that_rise_with_every_block(kind, d):
    """Scores 6 higher in every block of 128 keys (8.7 in powers of two, so that the sums so far are scaled down at
    nearly every block): each half of a row's outputs is scaled before any product adds to it, in every repetition.

    A score is a sum of 8 x 96 and the rest of d products, at most 2 d / 16 steps that each lose up to 2^-23 of 112, with
    4 more roundings: 20 x 2^-23 x 112 = 2.7e-4, twice that in a probability (its own and the sum's)."""
    c = Case([300, 41], [2048, 1500], kind=kind, heads=32, kv=8, d=d, page=64, seed=11)
    c.q[..., 0] = 8.0
    for i, length in enumerate(c.ctx):
        at = torch.arange(length, device="cuda")
        c.k[c.table[i, at // 64].long(), :, at % 64, 0] = (6.0 * (at // 128)).to(c.k.dtype)[:, None]
    first = c.attend(scale=0.125)
    u, tiny = {"f32": (0.0, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}[kind]
    start = 0
    for i, (n, length) in enumerate(zip(c.new, c.ctx)):
        rows = slice(start, start + n)
        start += n
        k, v = (ref.paged_rows(t, c.table[i], length) for t in (c.k, c.v))
        want, want_lse, size, flat = ref.attention(c.q[rows], k, v, length - n, 0.125)
        err = (first[0][rows].double() - want).abs()
        assert (err <= u * (size + want.abs()) + tiny * (flat + 1) + 6e-4 * size).all(), (i, float((err / size).max()))
        assert ((first[1][rows].double() - want_lse).abs() <= 3e-4).all()
    for _ in range(40):
        assert all(torch.equal(x, y) for x, y in zip(first, c.attend(scale=0.125)))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,ctx", [([200, 33], [200, 1700]), ([700], [3000])])
def test_attention_of_16_bit_chunks_only_rounds_its_outputs(kind, d, new, ctx):
    """Probabilities reach the products as high and low parts, 2^-16 of each together in bf16 (a half step of a half step)
    and 2^-22 in fp16 (or 2^-32 of the row's largest, where a low part would be smaller than fp16's last place): what is
    left is the outputs' own rounding (2^-25 where those are small for fp16), and fp32's as in Case.check."""
    c = Case(new, ctx, kind=kind, heads=8, kv=2, d=d, page=32, seed=21)
    out, _ = c.attend()
    unit, parts = {"f16": (2.0 ** -11, 2.0 ** -22), "bf16": (2.0 ** -8, 2.0 ** -16)}[kind]
    start = 0
    for i, (n, length) in enumerate(zip(new, ctx)):
        rows = slice(start, start + n)
        start += n
        k, v = (ref.paged_rows(t, c.table[i], length) for t in (c.k, c.v))
        want, _, size, flat = ref.attention(c.q[rows], k, v, length - n, d ** -0.5)
        err = (out[rows].double() - want).abs()
        bound = unit * want.abs() + (parts + 2e-5) * size + (2.0 ** -25 + 2.0 ** -32 * flat if kind == "f16" else 0.0)
        assert (err <= bound).all(), (i, float((err / bound).max()))


@pytest.mark.parametrize("new", [[1] * 5, [3, 40, 1, 0, 150]])
def test_sequences_that_share_one_row_of_a_page_table(new):
    """Samples of one prompt: a page table expanded from one row, as if that row were repeated."""
    c = Case([200], [200], kind="f16", seed=4)
    n = len(new)
    c.new, c.ctx = new, [170 + i for i in range(n)]
    c.q_start = torch.tensor([0] + new).cumsum(0).int().cuda()
    c.kv_len = torch.tensor(c.ctx).int().cuda()
    c.tokens, c.max_new = sum(new), max(new)
    c.q = torch.randn(c.tokens, c.heads, c.d, device="cuda").half()
    row = c.table
    # what would be taken for the other rows
    store = torch.full((n, row.shape[1]), c.spare[0], dtype=torch.int32, device="cuda")
    store[:1] = row
    c.table = store[:1].expand(n, -1)
    out, lse = c.attend()
    c.check(out, lse)
    key = torch.randn(n, c.kv, c.d, device="cuda").half()
    one_each = q.PagedBatch(torch.arange(n + 1).int().cuda(), c.kv_len, c.table, max_new=1)
    k0, v0 = c.k.clone(), c.v.clone()
    q.paged_append(c.cache(), one_each, key, key)
    for i, length in enumerate(c.ctx):
        page, slot = int(row[0, (length - 1) // 16]), (length - 1) % 16
        assert torch.equal(c.v[page, :, slot], key[i])
        c.k[page, :, slot], c.v[page, :, slot] = k0[page, :, slot], v0[page, :, slot]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
    # rows that overlap in any other way are refused
    c.table = store.flatten()[: n + row.shape[1]].as_strided((n, row.shape[1]), (1, 1))
    with pytest.raises(q.InvalidArgument):
        c.attend()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,ctx,heads,kv", [([300], [330], 2, 2), ([300, 70], [700, 70], 8, 2), ([64, 900], [64, 1000], 5, 1)])
@pytest.mark.parametrize("window", [0, 1, 16, 40, 200])
def test_attention_of_chunks_with_several_values_that_are_not_finite(kind, new, ctx, heads, kv, window):
    """Keys whose values are not finite, further apart than a window and next to each other, in the first sequence: tokens
    that attend to none of them keep their results to the bit, those between two of them too."""
    c = Case(new, ctx, kind=kind, heads=heads, kv=kv)
    clean, _ = c.attend(window=window)
    n, length = new[0], ctx[0]
    position = torch.arange(length - n, length, device="cuda")
    sees = torch.zeros(n, dtype=torch.bool, device="cuda")
    for at in (length - n + 1, length - n + n // 3, length - n + n // 3 + 1, length - n + 3 * n // 4, length - 2):
        c.v[int(c.table[0, at // 16]), :, at % 16] = math.inf if at % 2 else math.nan
        sees |= (position >= at) & ((position - window < at) if window else torch.ones_like(sees))
        out, _ = c.attend(window=window)
        assert torch.equal(out[:n][~sees], clean[:n][~sees]) and torch.equal(out[n:], clean[n:])
        assert not out[:n][sees].isfinite().any()


@pytest.mark.parametrize("kind,ctx,group,new", [("f32", 65536, 1, 1), ("f32", 65536, 4, 3), ("f32", 65536, 4, 12), ("f16", 131072, 4, 1), ("f16", 131072, 4, 12),
                                                ("f16", 131072, 1, 40)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_attention_sums_over_long_contexts(kind, ctx, group, new, d, mean):
    """Many sequences over a long context, each tile's in one CTA: the tensor cores' truncated sums do not add up.

    A sum leaves them after 8 (fp32) or 64 (16-bit) blocks, 64 or 128 and 512 or 1024 MMAs, each of which may take its
    last place, 2^-23, off it and as much off what it adds, and is half grown on the average; queries and probabilities
    have 2^-21 as fp16 pairs. fp16 outputs are rounded without bias."""
    n, kv, page = 40, 8, 128
    act, cached = TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(31)
    k = torch.randn(ctx // page, kv, page, d, generator=g, device="cuda").to(cached)
    v = (torch.randn(ctx // page, kv, page, d, generator=g, device="cuda") + mean).to(cached)
    table = torch.randperm(ctx // page, generator=g, device="cuda").int()[None]
    query = torch.randn(n * new, kv * group, d, generator=g, device="cuda").to(act)
    q_start, kv_len = (torch.arange(n + 1) * new).int().cuda(), torch.full((n,), ctx, dtype=torch.int32, device="cuda")
    out = q.paged_attention(q.PagedKV(k, v), q.PagedBatch(q_start, kv_len, table.expand(n, -1), max_new=new), query)
    position = ctx - new + torch.arange(n * new, device="cuda") % new
    hidden = torch.arange(ctx, device="cuda") > position[:, None]
    mmas = (64 if new * group <= 16 else 128) * (1 if kind == "f32" else 8)
    for h in (0, kv * group - 1):
        keys, values = (t[table[0].long(), h // group].flatten(0, 1).double() for t in (k, v))
        want = torch.softmax((query[:, h].double() @ keys.T * d ** -0.5).masked_fill(hidden, -math.inf), -1) @ values
        err = out[:, h].double() - want
        assert abs(float((err * want).sum() / (want * want).sum())) <= mmas * 2.0 ** -23 + 2.0 ** -21
        if kind == "f32":
            assert err.norm() <= (mmas * 2.0 ** -23 + 2.0 ** -21) * want.norm()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,ctx", [([1, 3], [90, 200]), ([70, 5], [200, 5])])
@pytest.mark.parametrize("scale", [1e-45, 1e-30, 1e-13])
def test_attention_with_scales_that_leave_no_differences(kind, new, ctx, scale):
    """Queries of zeros or small values under scales whose product with them is below fp32's range: every key that a token
    sees weighs the same (to check()'s bounds: the scores are below 1e-10 and their differences round away)."""
    c = Case(new, ctx, kind=kind, seed=8)
    c.q[::2] = 0.0
    c.q[1::2] *= 1e-3
    c.check(*c.attend(scale=scale), scale=scale)
    c.check(*c.attend(scale=scale, window=20), window=20, scale=scale)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,ctx", [([1, 3], [90, 200]), ([70, 5], [200, 5])])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_of_queries_that_are_not_finite(kind, new, ctx, bad):
    """They reach no output but their own token's and head's."""
    c = Case(new, ctx, kind=kind, seed=9)
    clean, clean_lse = c.attend()
    c.q[1, 2, 5] = bad
    out, lse = c.attend()
    assert not out[1, 2].isfinite().any() and not lse[1, 2].isfinite()
    out[1, 2], lse[1, 2] = clean[1, 2], clean_lse[1, 2]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


def test_attention_windows_beyond_an_int():
    c = Case([1, 40], [300, 60], kind="f16")
    for window in (1 << 31, (1 << 32) + 5, 1 << 63):
        assert all(torch.equal(x, y) for x, y in zip(c.attend(window=window), c.attend()))
