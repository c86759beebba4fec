"""The paged operators where a rule on sizes chooses another kernel, and calls on streams of their own."""
import random

import pytest
import torch

import q4kb200 as q
import serving_reference as ref
from test_gpu_paged import TYPES, Case

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("per_sm,more", [(2, -1), (2, 3), (8, 1), (16, -1), (16, 5)])
def test_append_of_many_tokens(kind, d, per_sm, more):
    """One to eight tokens a CTA: sequences that begin and end inside a CTA's tokens, empty ones, pages of nobody. The
    tolerances are test_append's."""
    rng = random.Random(per_sm * 10 + more)
    left, new, ctx = per_sm * sms() + more, [], []
    while left:
        n = min(left, rng.choice([0, 1, 1, 2, 7, 33, 150]))
        new.append(n)
        ctx.append(n + rng.randint(0, 40))
        left -= n
    c = Case(new, ctx, kind=kind, d=d, heads=4, kv=1, pad=3)
    key, value = (torch.randn(c.tokens, 1, d, generator=c.g, device="cuda").to(c.act) for _ in range(2))
    gq, gk = (1 + 0.1 * torch.randn(d, generator=c.g, device="cuda") for _ in range(2))
    # the longest sequence's last page is missing
    worst = ctx.index(max(ctx))
    c.table[worst, (ctx[worst] - 1) // 16] = -1
    k0, v0 = c.k.clone(), c.v.clone()
    out = torch.full_like(c.q, 7.0)
    q.paged_append(c.cache(), c.batch(), key, value, q=c.q, q_out=out, q_gamma=gq, k_gamma=gk)
    u = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
    u_act, u_kv = u[kind], 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    start, seen = 0, torch.zeros(c.k.shape[0], 16, dtype=torch.bool, device="cuda")
    pair = lambda x: torch.cat([x.abs()[..., :d // 2] + x.abs()[..., d // 2:]] * 2, -1)  # noqa: E731
    for i, (n, length) in enumerate(zip(new, ctx)):
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        at = torch.arange(length - n, length, device="cuda")
        pages, slot = c.table[i, at // 16].long(), at % 16
        held = pages >= 0
        seen[pages[held], slot[held]] = True
        want_q = ref.normed_rotated(c.q[rows], gq, length - n, 1e-6, 1e6)
        assert ((out[rows].double() - want_q).abs() <= u_act * want_q.abs() + 1e-5 * pair(want_q) + 2.0 ** -25).all()
        want_k = ref.normed_rotated(key[rows], gk, length - n, 1e-6, 1e6)[held]
        got_k = c.k[pages[held], :, slot[held]]
        assert ((got_k.double() - want_k).abs() <= u_kv * want_k.abs() + 1e-5 * pair(want_k) + 2.0 ** -25).all()
        assert torch.equal(c.v[pages[held], :, slot[held]], value[rows][held].to(c.v.dtype))
    assert (out[start:] == 7.0).all()
    keep = ~seen
    assert torch.equal(c.k.transpose(1, 2)[keep], k0.transpose(1, 2)[keep]) and torch.equal(c.v.transpose(1, 2)[keep], v0.transpose(1, 2)[keep])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sequences,kv", [(1, 2), (6, 3), (45, 8)])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_a_few_more_rows(kind, d, sequences, kv, window):
    """17 to 32 query rows per sequence and KV head, on either side of the rule that chooses their kernel."""
    rng = random.Random(sequences)
    new = [rng.randint(1, 8) for _ in range(sequences)]
    new[0] = 8
    c = Case(new, [n + rng.randint(0, 200) for n in new], kind=kind, heads=4 * kv, kv=kv, d=d, pad=1)
    c.check(*c.attend(window=window), window=window)


@pytest.mark.parametrize("kind,longest", [("f32", 1), ("f32", 70), ("bf16", 12)])
def test_attention_of_the_most_sequences(kind, longest):
    """8192 sequences, most of them without a new token."""
    rng = random.Random(longest)
    new = [0] * 8192
    for i in rng.sample(range(8192), 150) + [0, 8191]:
        new[i] = rng.randint(1, longest)
    new[8191] = longest
    c = Case(new, [n + rng.randint(0, 70) for n in new], kind=kind, heads=4, kv=2, d=64)
    out, lse = c.attend()
    keep = [i for i in range(8192) if new[i]]
    c.new, c.ctx, c.table = [new[i] for i in keep], [c.ctx[i] for i in keep], c.table[keep]
    c.check(out, lse)


def stream_of(x):
    """The stream that torch's allocator holds a tensor's memory for."""
    for segment in torch.cuda.memory_snapshot():
        if segment["address"] <= x.data_ptr() < segment["address"] + segment["total_size"]:
            return segment["stream"]
    raise AssertionError("no segment holds the tensor")


def test_allocations_are_the_streams():
    """A call on a stream of its own takes no memory that the current stream's work may still write."""
    c = Case([1] * 64, [200] * 64, kind="f16")
    logits, u = torch.randn(64, 5000, device="cuda"), torch.rand(64, device="cuda")
    turned, drawn = q.paged_append(c.cache(), c.batch(), c.q[:, :2], c.q[:, :2], q=c.q), q.sample(logits, u)
    want = c.attend()[0]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got_turned = q.paged_append(c.cache(), c.batch(), c.q[:, :2], c.q[:, :2], q=c.q, stream=s)
    got = q.paged_attention(c.cache(), c.batch(), c.q, stream=s)
    got_drawn = q.sample(logits, u, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(got_turned, turned) and torch.equal(got, want)
    assert all(torch.equal(x, y) for x, y in zip(got_drawn, drawn))
    assert {stream_of(x) for x in (got_turned, got, *got_drawn)} == {s.cuda_stream}
    assert stream_of(q.paged_attention(c.cache(), c.batch(), c.q)) != s.cuda_stream


def test_calls_on_two_streams_at_once():
    """Calls that may overlap, each with memory of its own, give what they give alone."""
    cases = [Case([1] * 40, [1500] * 40, kind="bf16", seed=2), Case([130, 5], [900, 700], kind="f32", seed=3)]
    alone = [c.attend()[0] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [q.paged_attention(c.cache(), c.batch(), c.q, stream=s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, alone))
