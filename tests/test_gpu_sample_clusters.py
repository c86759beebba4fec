"""Rows that a cluster of CTAs shares unevenly."""
import pytest
import torch

import q4kb200 as q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [16385, 16900, 17281, 33000])
@pytest.mark.parametrize("rows", [1, 4])
def test_clusters_with_ctas_that_have_few_or_no_logits(vocab, rows):
    """The last CTAs of a row's cluster have little or nothing to load, and tell the others of their bounds at once; the
    largest logit in the first or last place, drawn in every repetition."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(rows, vocab, generator=g, device="cuda")
    u = torch.rand(rows, generator=g, device="cuda")
    for at in (0, vocab - 1):
        x = logits.clone()
        x[:, at] = 60.0  # e^-55 and less is left to the others
        for kw in ({}, {"temperature": torch.zeros(rows, device="cuda")}, {"top_p": torch.full((rows,), 0.9, device="cuda")}):
            for _ in range(50):
                assert (q.sample(x, u, **kw)[0] == at).all()
