"""The paged append and attention against 64-bit references: head layouts, page sizes, ragged and empty sequences,
windows, strides, streams, graphs, and what stands in places that no row may see."""
import math
import random

import pytest
import torch

import q4kb200 as q
import serving_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": (torch.float32, torch.float16), "f16": (torch.float16, torch.float16), "bf16": (torch.bfloat16, torch.bfloat16)}
LEFT = 7.0  # what outputs hold before a call


class Case:
    """A batch with its cache; `new` and `ctx`: new and cached tokens of each sequence."""

    def __init__(self, new, ctx, kind="f32", heads=8, kv=2, d=128, page=16, seed=1, pad=0, order="hnd", spare=3, max_new=None):
        self.new, self.ctx, self.kind, self.heads, self.kv, self.d, self.page = new, ctx, kind, heads, kv, d, page
        self.act, cached = TYPES[kind]
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        need = [max(1, -(-c // page)) for c in ctx]
        pages = sum(need) + spare
        shape = (pages, kv, page, d) if order == "hnd" else (pages, page, kv, d)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(cached) for _ in range(2))
        if order == "nhd":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        ids = list(range(pages))
        rng.shuffle(ids)
        self.spare = ids[sum(need):]
        self.table = torch.full((len(ctx), max(need) + 1), self.spare[0] if spare else 0, dtype=torch.int32)
        for i, n in enumerate(need):
            self.table[i, :n] = torch.tensor(ids[:n], dtype=torch.int32)
            ids = ids[n:]
        self.table = self.table.cuda()
        self.q_start = torch.tensor([0] + new).cumsum(0).int().cuda()
        self.kv_len = torch.tensor(ctx).int().cuda()
        self.tokens = sum(new) + pad
        self.q = (2.0 * torch.randn(self.tokens, heads, d, generator=g, device="cuda")).to(self.act)
        self.max_new = max(new) if max_new is None else max_new
        self.g = g

    def cache(self):
        return q.PagedKV(self.k, self.v)

    def batch(self):
        return q.PagedBatch(self.q_start, self.kv_len, self.table, max_new=self.max_new)

    def attend(self, query=None, **kw):
        query = self.q if query is None else query
        out = torch.full((self.tokens, self.heads, self.d), LEFT, dtype=self.act, device="cuda")
        lse = torch.full((self.tokens, self.heads), LEFT, device="cuda")
        q.paged_attention(self.cache(), self.batch(), query, out=out, lse=lse, **kw)
        return out, lse

    def check(self, out, lse, window=0, scale=None):
        """Per element: 16-bit types round each probability (u of sum p|v|; fp16 also 2^-25 of the row's largest below
        2^-14) and the output (u |o|); fp32 carries both as fp16 pairs (2^-22, and fp16's last place 2^-25 of 2^7
        times a probability) and adds fp32 sums. Scores are sums of d products in fp32: 1e-5 is 2^-23 for each
        of 8 blocks of 16 products with |s| up to 10, and moves a probability by as much."""
        scale = self.d ** -0.5 if scale is None else scale
        u, tiny = {"f32": (0.0, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}[self.kind]
        start = 0
        for i, (n, c) in enumerate(zip(self.new, self.ctx)):
            rows = slice(start, start + n)
            k, v = (ref.paged_rows(t, self.table[i], c) for t in (self.k, self.v))
            want, want_lse, size, flat = ref.attention(self.q[rows], k, v, c - n, scale, window)
            err = (out[rows].double() - want).abs()
            bound = u * (size + want.abs()) + tiny * (flat + 1) + 2e-5 * size
            worst = float((err / bound.clamp(min=1e-30)).max()) if n else 0.0
            assert bool(torch.isfinite(out[rows]).all()) and worst <= 1.0, (i, n, c, worst)
            if self.kind == "f32" and n and c:
                assert err.norm() <= 1e-5 * want.norm(), (i, n, c, float(err.norm() / want.norm()))
            none = want_lse == -math.inf
            assert (lse[rows][none] == -math.inf).all() and (out[rows][none] == 0).all()
            assert ((lse[rows].double() - want_lse)[~none].abs() <= 2e-5).all()
            start += n
        assert (out[start:] == LEFT).all() and (lse[start:] == LEFT).all()


LENGTHS = {
    "single tokens": ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 1000]),
    "some empty": ([1, 0, 3, 0, 1], [70, 40, 3, 0, 129]),
    "few each": ([2, 5, 8, 3], [2, 300, 129, 64]),
    "chunks": ([127, 1, 128, 129, 33], [127, 500, 640, 300, 1001]),
    "one chunk": ([300], [300]),
    "before the start": ([5, 1, 40], [3, 0, 17]),
}


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention(lengths, kind, d):
    c = Case(*LENGTHS[lengths], kind=kind, d=d, pad=3)
    c.check(*c.attend())


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 2), (32, 2), (40, 1), (32, 8)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", ["single tokens", "chunks"])
def test_attention_head_groups(heads, kv, kind, lengths):
    c = Case(*LENGTHS[lengths], kind=kind, heads=heads, kv=kv)
    c.check(*c.attend())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("order", ["hnd", "nhd"])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [700, 255, 257]), ([200, 3], [700, 257])])
def test_attention_pages(page, order, new, ctx):
    c = Case(new, ctx, kind="f16", page=page, order=order)
    c.check(*c.attend())


@pytest.mark.parametrize("window", [1, 2, 63, 64, 128, 300, 100000])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1], [5, 300, 900]), ([4, 2], [900, 70]), ([260, 1, 70], [700, 900, 70])])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_window(window, new, ctx, kind):
    c = Case(new, ctx, kind=kind)
    c.check(*c.attend(window=window), window=window)


@pytest.mark.parametrize("new,ctx", [([1, 1], [1, 33000]), ([1], [40001]), ([3, 90], [20000, 9000])])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attention_long(new, ctx, kind):
    c = Case(new, ctx, kind=kind, heads=4, kv=1, page=64)
    c.check(*c.attend())


@pytest.mark.parametrize("sequences", [1, 31, 300, 700])
def test_attention_many_sequences(sequences):
    rng = random.Random(sequences)
    c = Case([rng.randint(0, 2) for _ in range(sequences)], [rng.randint(2, 90) for _ in range(sequences)], heads=4, kv=1, d=64)
    c.check(*c.attend())


@pytest.mark.parametrize("max_new", [0, 1, 2, 50, 4096])
def test_attention_host_bound_of_new_tokens(max_new):
    """The bound chooses how the work is cut, not the result."""
    c = Case([1, 50, 7], [300, 60, 7], max_new=max_new)
    c.check(*c.attend())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,ctx", [([1, 1, 2], [3, 100, 130]), ([70, 1], [200, 129])])
def test_attention_ignores_what_no_row_sees(kind, new, ctx):
    """Rows of pages behind a sequence's end, pages of nobody and table entries behind the end hold NaN, infinities or
    bad pages; windows keep what lies before them out."""
    c = Case(new, ctx, kind=kind)
    clean = c.attend()
    windowed = c.attend(window=20)
    for i, n in enumerate(ctx):
        last = int(c.table[i, (n - 1) // 16])
        c.k[last, :, (n - 1) % 16 + 1:] = math.nan
        c.v[last, :, (n - 1) % 16 + 1:] = math.inf
        c.table[i, -(-n // 16):] = -5 if i % 2 else 1 << 30
    for p in c.spare:
        c.k[p], c.v[p] = math.inf, math.nan
    again = c.attend()
    assert all(torch.equal(x, y) for x, y in zip(clean, again))
    for i, (n, new_) in enumerate(zip(ctx, new)):
        first = max(0, n - new_ - 20 + 1)
        for p in range(first // 16):
            c.table[i, p] = -1
        if first % 16:
            c.k[int(c.table[i, first // 16]), :, :first % 16] = math.inf
            c.v[int(c.table[i, first // 16]), :, :first % 16] = math.nan
    again = c.attend(window=20)
    assert all(torch.equal(x, y) for x, y in zip(windowed, again))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("new,ctx,heads,kv", [([5], [70], 4, 2), ([2, 3], [131, 64], 4, 1), ([150, 3], [400, 3], 8, 2), ([300], [300], 2, 2)])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_new_tokens_do_not_see_later_ones(kind, new, ctx, heads, kv, window, bad):
    """A new token whose key and value are not finite: those that do not attend to it keep their results to the bit,
    those that do are not finite."""
    c = Case(new, ctx, kind=kind, heads=heads, kv=kv)
    clean, _ = c.attend(window=window)
    n, length = new[0], ctx[0]
    at = length - n + n // 2
    page, slot = int(c.table[0, at // 16]), at % 16
    c.v[page, :, slot] = bad
    for poison_key in (False, True):
        if poison_key:
            c.k[page, :, slot] = bad
        out, _ = c.attend(window=window)
        position = torch.arange(length - n, length, device="cuda")
        sees = (position >= at) & ((position - window < at) if window else torch.ones_like(position, dtype=torch.bool))
        assert torch.equal(out[:n][~sees], clean[:n][~sees]) and torch.equal(out[n:], clean[n:])
        assert not out[:n][sees].isfinite().any()


@pytest.mark.parametrize("new,ctx,d", [([2100], [9000], 64), ([700, 1], [5000, 4000], 128)])
def test_attention_fp32_over_many_blocks(new, ctx, d):
    """Sums over hundreds of products keep fp32 accuracy: as accurate as fp32 sums of the same length (2^-24 times the
    square root of the keys, 95 here) with the queries' and probabilities' 2^-22."""
    c = Case(new, ctx, kind="f32", heads=32, kv=8, d=d, page=64)
    out, _ = c.attend()
    start = 0
    for i, (n, length) in enumerate(zip(new, ctx)):
        k, v = (ref.paged_rows(t, c.table[i], length) for t in (c.k, c.v))
        for a in range(0, n, 700):
            b = min(n, a + 700)
            for h in range(0, 32, 8):
                want, *_ = ref.attention(c.q[start + a:start + b, h:h + 8], k[h // 4:h // 4 + 2], v[h // 4:h // 4 + 2], length - n + a, d ** -0.5)
                assert (out[start + a:start + b, h:h + 8].double() - want).norm() <= (95 * 2.0 ** -24 + 2.0 ** -21) * want.norm()
        start += n


@pytest.mark.parametrize("size", [1e-4, 30.0, 3000.0])
@pytest.mark.parametrize("kind", TYPES)
def test_attention_score_sizes(size, kind):
    """Flat and one-hot rows, queries that are large or small for their type. With scores of thousands a row's weight
    may sit on two keys whose scores fp32 cannot tell apart as well, so only rows led by more than that are compared."""
    c = Case([1, 60], [400, 200], kind=kind, seed=5)
    c.q = (c.q.float() * size).to(c.act)
    out, lse = c.attend()
    start = 0
    for i, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        k, v = (ref.paged_rows(t, c.table[i], ctx) for t in (c.k, c.v))
        want, want_lse, sizes, _ = ref.attention(c.q[start:start + n], k, v, ctx - n, c.d ** -0.5)
        # a score's error: 2^-23 for each of 8 blocks of products, of |q| |k| scale
        slack = 2.0 ** -20 * size * 2 * 11.4 * 11.4 * 1.5 * c.d ** -0.5
        u = {"f32": 1e-5, "f16": 2.0 ** -10 + 1e-3, "bf16": 2.0 ** -7}[kind]
        err = (out[start:start + n].double() - want).abs()
        assert (err <= (u + math.expm1(2 * slack)) * (sizes + want.abs())).all()
        assert ((lse[start:start + n].double() - want_lse).abs() <= 1e-5 + 2.0 ** -22 * want_lse.abs() + slack).all()
        start += n


def test_attention_huge_queries_stay_finite():
    """fp32 queries beyond fp16's range."""
    c = Case([1, 40], [100, 60], kind="f32")
    c.q *= 1e6
    out, lse = c.attend(scale=1e-6 * c.d ** -0.5)
    c.check(out, lse, scale=1e-6 * c.d ** -0.5)


def test_attention_strided_rows_and_scale():
    c = Case([1, 30], [90, 77], kind="bf16", heads=8, kv=2)
    fused = torch.randn(c.tokens, 12, c.d, device="cuda").to(c.act)
    fused[:, :8] = c.q
    whole = torch.full((c.tokens, 16, c.d), LEFT, dtype=c.act, device="cuda")
    got = q.paged_attention(c.cache(), c.batch(), fused[:, :8], out=whole[:, 8:], scale=0.3)
    assert (whole[:, :8] == LEFT).all()
    c.check(got, q_lse := c.attend(scale=0.3)[1], scale=0.3)
    assert q_lse.shape == (c.tokens, 8)


def test_offsets_past_32_bits():
    """Pages more than 2^32 elements apart."""
    d, page, kv = 64, 16, 1
    stride = (1 << 31) + 4096
    store = torch.empty(2 * stride + 2 * page * d, dtype=torch.float16, device="cuda")
    c = Case([2], [45], kind="f16", heads=2, kv=kv, d=d, spare=0)
    k = store.as_strided((3, kv, page, d), (stride, page * d, d, 1))
    v = store.as_strided((3, kv, page, d), (stride, page * d, d, 1), page * d)
    k.copy_(c.k)
    v.copy_(c.v)
    c.k, c.v = k, v
    c.check(*c.attend())
    key = torch.randn(2, kv, d, device="cuda").half()
    q.paged_append(c.cache(), c.batch(), key, key)
    assert torch.equal(v[int(c.table[0, 2]), :, 11:13], key.transpose(0, 1))


def test_attention_side_stream_and_graph():
    """A captured call follows the arrays' contents; another stream's work is ordered by that stream."""
    c = Case([1, 1, 1], [400, 10, 65])
    want = c.attend()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = q.paged_attention(c.cache(), c.batch(), c.q, stream=s)
    s.synchronize()
    assert torch.equal(out, want[0])
    out, lse = torch.empty_like(c.q), torch.empty(3, c.heads, device="cuda")
    cache, batch = c.cache(), c.batch()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.paged_attention(cache, batch, c.q, out=out, lse=lse)
    for ctx in ([400, 10, 65], [1, 416, 80], [0, 3, 64]):
        c.ctx = ctx
        c.kv_len.copy_(torch.tensor(ctx))
        big = c.table.max(1).values
        for i, n in enumerate(ctx):  # any pages will do, as long as every position has one of its own
            need = -(-n // 16)
            c.table[i, :need] = torch.randperm(c.k.shape[0], device="cuda")[:need].int()
        del big
        graph.replay()
        torch.cuda.synchronize()
        c.check(out, lse)


def test_attention_is_repeatable():
    c = Case([1, 60, 1], [3000, 900, 17], kind="bf16")
    first = c.attend()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, c.attend()))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("order,page", [("hnd", 16), ("nhd", 64)])
def test_append(kind, d, norm, order, page):
    """Norm and angles in fp32: 1e-5 covers a sum of d squares (2^-24 each) and the angle's 2^-22; then one rounding."""
    c = Case([1, 0, 40, 3, 1], [1, 9, 100, 3, 4000], kind=kind, d=d, page=page, order=order, pad=2)
    key, value = (torch.randn(c.tokens, c.kv, d, device="cuda").to(c.act) for _ in range(2))
    gq, gk = ((1 + 0.1 * torch.randn(d, device="cuda")) if norm else None for _ in range(2))
    k0, v0 = c.k.clone(), c.v.clone()
    out = torch.full_like(c.q, LEFT)
    got = q.paged_append(c.cache(), c.batch(), key, value, q=c.q, q_out=out, q_gamma=gq, k_gamma=gk, epsilon=1e-6, rope_base=1e6)
    assert got is out
    u = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
    u_act, u_kv = u[kind], 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    start, seen = 0, torch.zeros(c.k.shape[0], page, dtype=torch.bool, device="cuda")
    for i, (n, ctx) in enumerate(zip(c.new, c.ctx)):
        rows = slice(start, start + n)
        at = torch.arange(ctx - n, ctx, device="cuda")
        pages, slot = c.table[i, at // page].long(), at % page
        seen[pages, slot] = True
        pair = lambda x: torch.cat([x.abs()[..., :d // 2] + x.abs()[..., d // 2:]] * 2, -1)  # noqa: E731
        for x, gamma, y, unit in ((c.q, gq, out[rows], u_act), (key, gk, c.k[pages, :, slot], u_kv)):
            want = ref.normed_rotated(x[rows], gamma, ctx - n, 1e-6, 1e6)
            assert ((y.double() - want).abs() <= unit * want.abs() + 1e-5 * pair(want) + 2.0 ** -25).all()
        assert torch.equal(c.v[pages, :, slot], value[rows].to(c.v.dtype))
        start += n
    assert (out[start:] == LEFT).all()
    keep = ~seen
    assert torch.equal(c.k.transpose(1, 2)[keep], k0.transpose(1, 2)[keep]) and torch.equal(c.v.transpose(1, 2)[keep], v0.transpose(1, 2)[keep])


@pytest.mark.parametrize("position", [0, 1, 4095, 131071, 1 << 20, (1 << 24) + 1, (1 << 30) + 7])
def test_append_far_positions(position):
    """The angle's error does not grow with the position; a position past the table is rotated and not written."""
    c = Case([1], [1], kind="f32")
    c.ctx = [position + 1]
    c.kv_len.fill_(position + 1)
    k0 = c.k.clone()
    key = torch.randn(1, c.kv, c.d, device="cuda")
    out = q.paged_append(c.cache(), c.batch(), key, key, q=c.q)
    want = ref.normed_rotated(c.q, None, position, 1e-6, 1e6)
    assert (out.double() - want).abs().max() <= 1e-6 * want.abs().max()
    if position >= 16 * c.table.shape[1]:
        assert torch.equal(c.k, k0)


def test_append_skips_bad_places():
    """Positions before the cache's start, pages below zero or past the cache."""
    c = Case([4, 2, 1], [2, 20, 8], kind="f16")
    c.table[1, 1] = -1
    c.table[2, 0] = c.k.shape[0]
    k0, v0 = c.k.clone(), c.v.clone()
    key = torch.randn(7, c.kv, c.d, device="cuda").half()
    assert q.paged_append(c.cache(), c.batch(), key, key) is None
    p = int(c.table[0, 0])
    assert torch.equal(c.v[p, :, :2], key[2:4].transpose(0, 1))
    c.k[p, :, :2], c.v[p, :, :2] = k0[p, :, :2], v0[p, :, :2]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


def test_append_in_place_and_fused_rows():
    c = Case([1, 5], [30, 5], kind="bf16", heads=8, kv=2)
    qkv = torch.randn(c.tokens, 12, c.d, device="cuda").to(c.act)
    query, key, value = qkv.split((8, 2, 2), dim=1)
    want = q.paged_append(c.cache(), c.batch(), key, value, q=query)
    rest = qkv[:, 8:].clone()
    got = q.paged_append(c.cache(), c.batch(), key, value, q=query, q_out=query)
    assert torch.equal(got, want) and torch.equal(qkv[:, 8:], rest)


def test_rows_before_the_first_sequence_and_odd_lengths():
    """q_start need not begin at 0; negative lengths are empty caches; windows may be as long as an int."""
    c = Case([2, 3, 1], [40, 3, 5], kind="f16", max_new=1)
    base = c.attend(window=(1 << 31) - 1)
    assert all(torch.equal(x, y) for x, y in zip(base, c.attend()))
    k0, v0 = c.k.clone(), c.v.clone()
    c.q_start[0] = 1  # the first row is nobody's: a new token less
    c.kv_len[1] = -(1 << 31)
    out, lse = c.attend()
    assert (out[0] == LEFT).all() and (lse[0] == LEFT).all() and torch.equal(out[1], base[0][1]) and torch.equal(out[5], base[0][5])
    assert (out[2:5] == 0).all() and (lse[2:5] == -math.inf).all()
    key = torch.randn(6, c.kv, c.d, device="cuda").half()
    turned = torch.full_like(c.q, LEFT)
    q.paged_append(c.cache(), c.batch(), key, key, q=c.q, q_out=turned)
    assert (turned[0] == LEFT).all() and (turned[1:] != LEFT).any(-1).all()
    p, r = int(c.table[0, 2]), int(c.table[2, 0])
    assert torch.equal(c.v[p, :, 7], key[1]) and torch.equal(c.v[r, :, 4], key[5])
    c.k[p, :, 7], c.v[p, :, 7], c.k[r, :, 4], c.v[r, :, 4] = k0[p, :, 7], v0[p, :, 7], k0[r, :, 4], v0[r, :, 4]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


def test_empty_calls():
    c = Case([1], [4], kind="f16")
    batch = q.PagedBatch(torch.zeros(1, dtype=torch.int32, device="cuda"), c.kv_len[:0], c.table[:0])
    out = torch.full_like(c.q, LEFT)
    q.paged_attention(c.cache(), batch, c.q, out=out)
    assert (out == LEFT).all()
    q.paged_attention(c.cache(), c.batch(), c.q[:0])
    q.paged_append(c.cache(), c.batch(), c.q[:0, :2], c.q[:0, :2])
