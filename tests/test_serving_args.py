"""Refusals of the paged cache's and sampling's entry points, made before any CUDA work."""
import ctypes as C

import pytest

import q4kb200 as q

A = 1 << 20  # an aligned address that nothing reads


def cache(**kw):
    c = dict(k=A, v=A, type=q.F16, kv_heads=2, head_dim=128, page_size=16, pages=10, page_stride=4096, head_stride=2048, row_stride=128)
    c.update(kw)
    return q._PagedKV(*c.values())


def batch(**kw):
    b = dict(sequences=1, max_new=1, q_start=A, kv_len=A, page_table=A, table_stride=4, table_width=4)
    b.update(kw)
    return q._PagedBatch(*b.values())


def append(c=None, b=None, **kw):
    a = dict(tokens=1, type=q.F32, q=A, ld_q=1024, heads=8, k=A, ld_k=256, v=A, ld_v=256, qg=None, kg=None, eps=1e-6, base=1e6, q_out=A, ld_out=1024)
    a.update(kw)
    return q.lib().q4k_paged_append(C.byref(c or cache()), C.byref(b or batch()), *a.values(), None)


def attend(c=None, b=None, **kw):
    a = dict(tokens=1, type=q.F32, q=A, ld_q=1024, heads=8, scale=0.0, window=0, out=A, ld_out=1024, lse=None, ws=A, ws_bytes=1 << 40)
    a.update(kw)
    return q.lib().q4k_paged_attention(C.byref(c or cache()), C.byref(b or batch()), *a.values(), None)


BAD_CACHES = [dict(k=None), dict(v=A + 8), dict(type=q.F32), dict(type=q.Q4_K), dict(type=q.BF16), dict(head_dim=96), dict(head_dim=256),
              dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(kv_heads=0), dict(pages=0), dict(row_stride=64),
              dict(row_stride=130), dict(page_stride=0), dict(head_stride=-128)]
BAD_BATCHES = [dict(sequences=-1), dict(max_new=-1), dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(table_width=0), dict(table_stride=3)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches(bad):
    assert append(cache(**bad)) == q.EINVAL and attend(cache(**bad)) == q.EINVAL


@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_bad_batches(bad):
    assert append(b=batch(**bad)) == q.EINVAL and attend(b=batch(**bad)) == q.EINVAL


@pytest.mark.parametrize("bad", [dict(pages=1 << 32), dict(page_stride=1 << 40)])
def test_out_of_range_caches(bad):
    assert append(cache(**bad)) == q.ERANGE and attend(cache(**bad)) == q.ERANGE


@pytest.mark.parametrize("bad", [dict(q=None), dict(q_out=None), dict(q=A + 4), dict(ld_q=1000), dict(ld_q=1026), dict(heads=0), dict(k=None),
                                 dict(v=A + 8), dict(ld_k=255), dict(ld_v=128), dict(base=0.0), dict(base=float("nan")), dict(qg=A, eps=0.0),
                                 dict(type=q.F16 + 5), dict(type=q.BF16), dict(ld_out=8)])
def test_bad_append_arguments(bad):
    assert append(**bad) == q.EINVAL


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=A + 8), dict(ld_q=512), dict(heads=0), dict(heads=7), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(window=-1), dict(out=None), dict(ld_out=1022), dict(type=q.Q6_K)])
def test_bad_attention_arguments(bad):
    assert attend(**bad) == q.EINVAL


def test_sizes_out_of_range():
    assert append(tokens=1 << 30) == q.ERANGE and attend(tokens=1 << 30) == q.ERANGE
    assert attend(b=batch(table_width=1 << 28, table_stride=1 << 28)) == q.ERANGE


def test_nothing_to_do():
    assert append(tokens=0) == q.OK and attend(tokens=0) == q.OK
    assert append(b=batch(sequences=0)) == q.OK and attend(b=batch(sequences=0)) == q.OK


def draw(**kw):
    a = dict(logits=A, type=q.F32, ld=100, rows=1, vocab=100, t=None, k=None, p=None, m=None, u=A, tokens=A, lp=None)
    a.update(kw)
    return q.lib().q4k_sample(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(type=q.Q4_K), dict(ld=99), dict(vocab=0), dict(u=None), dict(tokens=None)])
def test_bad_sampling_arguments(bad):
    assert draw(**bad) == q.EINVAL


def test_sampling_sizes():
    assert draw(vocab=400001, ld=400001) == q.ERANGE and draw(rows=1 << 24) == q.ERANGE and draw(rows=0) == q.OK


def test_python_refusals():
    import torch

    cpu = torch.zeros(4, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(q.InvalidArgument):
        q.PagedKV(cpu, cpu)
    with pytest.raises(q.InvalidArgument):
        q.PagedKV(cpu, cpu[:2])
    with pytest.raises(q.InvalidArgument):
        q.sample(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(q.InvalidArgument):
        q.PagedBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))


def test_packed_structures_are_the_ctypes_ones():
    kv, b = tuple(range(1, 11)), tuple(range(1, 8))
    assert bytes(q._PagedKV(*kv)) == q._pack_kv(*kv)
    assert len(q._pack_batch(*b)) == C.sizeof(q._PagedBatch) and bytes(q._PagedBatch(*b))[:44] == q._pack_batch(*b)[:44]
