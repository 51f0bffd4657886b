"""The token-model operators along the paths that only some sizes take: every form of the sort behind the table's gradient, sorted
gradients in recorded graphs, on side streams and in tables beyond 2^31 elements, log probabilities by warps, blocks and
clusters over masks, ties and specials."""
import math

import pytest
import torch

import cuv_b200 as cb
from test_gpu_tokens import gen

pytestmark = pytest.mark.gpu


def text_tokens(g, vocab, ncols, pad=0.1):
    """Text-like frequencies, some positions padding."""
    tok = ((torch.rand(ncols, device="cuda", generator=g, dtype=torch.float64) * math.log(vocab + 1)).exp().long() - 1).clamp(0, vocab - 1)
    tok[torch.rand(ncols, device="cuda", generator=g) < pad] = -7
    return tok


def whole_sums(tok, dout, vocab, before=None, factor=1.0):
    """The gradient of whole numbers, exact in 64 bits."""
    want = torch.zeros((vocab + 1, dout.shape[0]), dtype=torch.float64, device="cuda")
    want.index_add_(0, torch.where(tok < 0, vocab, tok), dout.t().double())
    want = want[:vocab].t() * factor
    return want if before is None else want + before.double()


@pytest.mark.parametrize("ncols", [300, 1500, 3000, 5000, 8192, 12000, 30000, 50000, 100000])
@pytest.mark.parametrize("vocab", [300, 20011, 300007])
def test_every_cluster_of_the_sort_beside_other_work(ncols, vocab):
    """Clusters of one to eight blocks, one to sixteen pairs a lane, one to three passes, again and again while another stream
    keeps the SMs busy, so that a cluster's blocks do not keep step.  Sums of whole numbers below 2^24: equality."""
    g, units = gen(ncols + vocab), 8
    dout = torch.randint(-100, 101, (ncols, units), device="cuda", generator=g).float().t()
    tok = text_tokens(g, vocab, ncols)
    want = whole_sums(tok, dout, vocab)
    other, load = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda", generator=g)
    torch.cuda.synchronize()
    got = [cb.colmajor_empty(units, vocab) for _ in range(12)]
    with torch.cuda.stream(other):
        for _ in range(12):
            load = torch.sin(load)
    for dtable in got:
        cb.embedding_grad(dtable, tok, dout)
    torch.cuda.synchronize()
    for dtable in got:
        assert torch.equal(dtable.double(), want)
