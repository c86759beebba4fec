"""Sampling against long doubles: filters alone and together, ties, masked and odd values, sizes, streams and graphs."""
import math

import numpy as np
import pytest
import torch

import q4kb200 as q
import serving_reference as ref

pytestmark = pytest.mark.gpu


def check(logits, u, **settings):
    """Each row's token is the reference's; its log-probability is off by one fp32 rounding (and the weights' 2^-40)."""
    full = {k: torch.as_tensor(v, device="cuda") for k, v in settings.items()}
    rows = logits.shape[0]
    tokens, logprob = q.sample(logits, u, **full)
    x, uu = logits.double().cpu().numpy(), u.cpu().numpy()
    for r in range(rows):
        one = {k: v.cpu().numpy()[r].item() for k, v in full.items()}
        want, lp, near = ref.sample(x[r], uu[r], **one)
        got = int(tokens[r])
        assert got == want or got in near, (r, got, want, near, one, uu[r])
        if got == want:
            assert logprob[r] == lp or abs(float(logprob[r]) - lp) <= 2.0 ** -23 * abs(lp) + 1e-7, (r, float(logprob[r]), lp)
    return tokens


def rows_of(rows, vocab, dtype=torch.float32, seed=3, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * spread
    return logits.to(dtype), torch.rand(rows, generator=g, device="cuda")


def each(rows, value, dtype=torch.float32):
    return torch.full((rows,), value, dtype=dtype)


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 1024, 1025, 32768, 50001, 151936, 151937, 400000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_plain_draws(vocab, dtype):
    logits, u = rows_of(5, vocab, dtype)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    check(logits, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top_k", [1, 2, 50, 999, 1000, 5000])
@pytest.mark.parametrize("top_p", [0.0, 0.01, 0.5, 0.95, 1.0])
def test_top_k_and_top_p(dtype, top_k, top_p):
    logits, u = rows_of(6, 1000, dtype)
    check(logits, u, top_k=each(6, top_k, torch.int32), top_p=each(6, top_p))


@pytest.mark.parametrize("min_p", [0.0, 1e-6, 0.05, 0.9, 1.0, 3.0])
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 30.0])
def test_min_p_and_temperature(min_p, temperature):
    logits, u = rows_of(6, 5000)
    check(logits, u, temperature=each(6, temperature), min_p=each(6, min_p))


@pytest.mark.parametrize("rows", [1, 2, 9, 19, 40, 80, 200, 400])
@pytest.mark.parametrize("vocab", [700, 151936])
def test_rows_with_settings_of_their_own(rows, vocab):
    if rows * vocab > 13e6:
        rows = 86
    logits, u = rows_of(rows, vocab, torch.float16, spread=3.0)
    g = torch.Generator().manual_seed(rows)
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (rows,), generator=g)]  # noqa: E731
    check(logits, u, temperature=pick(0.0, 0.5, 1.0, 1.7), top_k=pick(0, 1, 40, 1 << 30).int(), top_p=pick(1.0, 0.3, 0.9, 0.999), min_p=pick(0.0, 0.1))


def test_ties():
    """Equal logits: the lowest indexes are kept, whatever filter cuts among them."""
    logits = torch.zeros(9, 3001, device="cuda")
    logits[3:6, ::3] = 1.0
    logits[6:, 100:] = -2.0
    logits[1, ::2] = -0.0
    u = torch.tensor([0.0, 0.5, 0.9999] * 3, device="cuda")
    for top_k in (0, 1, 7, 1001, 3000):
        for top_p in (1.0, 0.5, 0.25):
            check(logits, u, top_k=each(9, top_k, torch.int32), top_p=each(9, top_p))


def test_masked_and_odd_values():
    inf, low = math.inf, torch.finfo(torch.float32).min
    logits, u = rows_of(10, 2000)
    logits[0] = -inf
    logits[1, 1:] = -inf
    logits[2, :1999] = low
    logits[3] = math.nan
    logits[4, ::2] = math.nan
    logits[5, 7::100] = inf
    logits[6] = low
    logits[7, 500:] = -inf
    logits[8, :] = torch.finfo(torch.float32).max
    logits[9, 3] = torch.finfo(torch.float32).max
    for kw in ({}, {"top_k": each(10, 5, torch.int32)}, {"top_p": each(10, 0.9)}, {"min_p": each(10, 0.2)}, {"temperature": each(10, 0.0)},
               {"top_k": each(10, 600, torch.int32), "top_p": each(10, 0.6), "temperature": each(10, 1e-30)}):
        tokens = check(logits, u, **kw)
        assert int(tokens[0]) == -1 and int(tokens[3]) == -1
    # numbers outside [0, 1) draw the first or last kept token
    logits, _ = rows_of(3, 100)
    tokens, _ = q.sample(logits, torch.tensor([-1.0, 1.0, 2.0], device="cuda"))
    assert tokens.tolist() == [0, 99, 99]
    q.sample(logits, torch.full((3,), math.nan, device="cuda"), temperature=torch.full((3,), math.nan, device="cuda"))


def test_strided_rows_stream_and_graph():
    whole, u = rows_of(8, 4000)
    view = whole[:, 37:3040]
    check(view, u, top_p=each(8, 0.9))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    tokens, _ = q.sample(view, u, stream=s)
    s.synchronize()
    assert torch.equal(tokens, q.sample(view, u)[0])
    out, lp = torch.empty(8, dtype=torch.int32, device="cuda"), torch.empty(8, device="cuda")
    top_k = torch.full((8,), 20, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.sample(view, u, top_k=top_k, tokens=out, logprob=lp)
    for k in (20, 1, 0):
        top_k.fill_(k)
        u.copy_(torch.rand(8, device="cuda"))
        graph.replay()
        assert torch.equal(out, q.sample(view, u, top_k=top_k)[0])


def test_frequencies_follow_the_distribution():
    """The draw's own sums: over an even grid of uniform numbers each token comes as often as its probability says, to
    one grid step."""
    n = 4096
    logits, _ = rows_of(1, 50)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, _ = q.sample(logits.expand(n, 50).contiguous(), u)
    p = torch.softmax(logits[0].double(), 0).cpu().numpy()
    got = np.bincount(tokens.cpu().numpy(), minlength=50) / n
    assert np.abs(got - p).max() <= 1.0 / n + 1e-9


def test_step_of_serving():
    """Append, attend, project and sample as one step of a small batch, against the same step in 64 bits."""
    torch.manual_seed(0)
    heads, kv, d, page, vocab = 8, 2, 64, 16, 3000
    ctx = [5, 40, 17]
    k = torch.zeros(12, kv, page, d, device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    table = torch.tensor([[0, 3, 6, 9], [1, 4, 7, 10], [2, 5, 8, 11]], dtype=torch.int32, device="cuda")
    cache = q.PagedKV(k, v)
    gamma = 1 + 0.1 * torch.randn(d, device="cuda")
    w = torch.randn(vocab, heads * d, device="cuda") / 8
    kept_k = [torch.zeros(0, kv, d, dtype=torch.float64, device="cuda") for _ in ctx]
    kept_v = list(kept_k)
    done = [0, 0, 0]
    for step in range(4):
        new = ctx if step == 0 else [1, 2, 0]
        q_start = torch.tensor([0] + new).cumsum(0).int().cuda()
        done = [a + b for a, b in zip(done, new)]
        batch = q.PagedBatch(q_start, torch.tensor(done).int().cuda(), table, max_new=max(new))
        qkv = torch.randn(sum(new), heads + 2 * kv, d, device="cuda")
        query, key, value = qkv.split((heads, kv, kv), dim=1)
        turned = q.paged_append(cache, batch, key, value, q=query, q_gamma=gamma, k_gamma=gamma)
        out = q.paged_attention(cache, batch, turned)
        last = [int(q_start[i + 1]) - 1 for i in range(3) if new[i]]
        logits = out[last].flatten(1) @ w.T
        u = torch.rand(len(last), device="cuda")
        tokens, _ = q.sample(logits, u, temperature=torch.full_like(u, 0.8), top_k=torch.full_like(u, 100).int(), top_p=torch.full_like(u, 0.9))
        start = 0
        for i, n in enumerate(new):
            rows = slice(start, start + n)
            start += n
            kept_k[i] = torch.cat((kept_k[i], ref.normed_rotated(key[rows], gamma, done[i] - n, 1e-6, 1e6)))
            kept_v[i] = torch.cat((kept_v[i], value[rows].double()))
            want, _, size, _ = ref.attention(ref.normed_rotated(query[rows], gamma, done[i] - n, 1e-6, 1e6), kept_k[i].transpose(0, 1),
                                             kept_v[i].transpose(0, 1), done[i] - n, d ** -0.5)
            # keys and values are rounded to fp16: 2^-11 of a value, and of |q| |k| scale (at most 8 here) for a score
            assert ((out[rows].double() - want).abs() <= 2.0 ** -11 * (1 + 2 * 8) * (size + 1e-3)).all()
        for r in range(len(last)):
            got = int(tokens[r])
            want, _, near = ref.sample(logits[r].double().cpu().numpy(), float(u[r]), 0.8, 100, 0.9)
            assert got == want or got in near
