"""The token-model operators along the paths that only some sizes take: every form of the sort behind the table's gradient, sorted
gradients in recorded graphs, on side streams and in tables beyond 2^31 elements, log probabilities by warps, blocks and
clusters over masks, ties and specials."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import cuv_b200 as cb
from oracle import host_oracle as ho
from test_gpu_tokens import E32, TYPES, gen, matrix, near, plain_logprob

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


@pytest.mark.parametrize("ncols", [700, 5000, 40000, 140000])
@pytest.mark.parametrize("fold", [0.0, 1.0])
def test_sorted_gradients_recorded_on_side_streams(ncols, fold):
    """Two graphs recorded on a side stream, replayed at the same time on streams of their own, on contents that are not those
    of the recording: the sort, its dependent sums and joins, a workspace each.  Whole numbers: equality."""
    units, vocab = 40, 5003

    def operands(seed):
        g = gen(seed)
        return text_tokens(g, vocab, ncols), torch.randint(-30, 31, (ncols, units), device="cuda", generator=g).float().t()

    side, made = torch.cuda.Stream(), []
    for seed in (1, 2):
        (tok, dout), dtable = operands(seed), torch.ones((vocab, units), device="cuda").t()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            cb.embedding_grad(dtable, tok, dout, 1.0, fold)
        made.append((graph, tok, dout, dtable))
    torch.cuda.synchronize()
    for k, (graph, tok, dout, dtable) in enumerate(made):
        t, d = operands(11 + k)
        tok.copy_(t)
        dout.copy_(d)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for s, m in zip(streams, made):
            with torch.cuda.stream(s):
                m[0].replay()
    torch.cuda.synchronize()
    for graph, tok, dout, dtable in made:
        once = whole_sums(tok, dout, vocab)
        assert torch.equal(dtable.double(), 3 * once + 1.0 if fold else once)
    # and without a graph, on a side stream of which the current one knows nothing
    tok, dout = operands(21)
    dtable = torch.ones((vocab, units), device="cuda").t()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cb.embedding_grad(dtable, tok, dout, 1.0, fold)
    side.synchronize()
    assert torch.equal(dtable.double(), whole_sums(tok, dout, vocab) + (1.0 if fold else 0.0))


@pytest.mark.parametrize("ncols", [2000, 30000, 135000])
def test_a_sorted_gradient_recorded_on_its_very_first_call(ncols):
    """A process whose first call is the recorded one: what the sort needs set for its shared memory is set there."""
    code = """
import torch, cuv_b200 as cb
ncols = %d
dout = (torch.arange(ncols * 24, device="cuda") %% 17 - 8).float().view(ncols, 24).t()
tok = torch.arange(ncols, device="cuda") * 7919 %% 1009
dtable = cb.colmajor_empty(24, 1500)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    cb.embedding_grad(dtable, tok, dout)
graph.replay()
torch.cuda.synchronize()
want = torch.zeros((1500, 24), dtype=torch.float64, device="cuda")
want.index_add_(0, tok, dout.t().double())
assert torch.equal(dtable.double(), want.t())
print("same")
""" % ncols
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stderr[-2000:]


def test_sorted_gradients_beyond_32_bits():
    """A table, and then a batch, of more than 2^31 elements: the far end of either, absent columns there included."""
    units, vocab, ncols = 65536, 33000, 400
    g = gen(8)
    dout = torch.randint(-9, 10, (ncols, units), device="cuda", generator=g, dtype=torch.int8).to(torch.bfloat16).t()
    tok = torch.full((ncols,), -1, device="cuda")
    tok[:300] = vocab - 1 - torch.randint(0, 6, (300,), device="cuda", generator=g) * 2
    tok[300:350] = vocab - 40                                   # whose sums reach over chunks
    dtable = torch.full((vocab, units), 7.0, dtype=torch.bfloat16, device="cuda").t()
    cb.embedding_grad(dtable, tok, dout)
    rows = torch.where(tok < 0, 0, tok - (vocab - 40))
    want = torch.zeros((40, units), dtype=torch.float64, device="cuda")
    want.index_add_(0, rows[tok >= 0], dout.t().double()[tok >= 0])
    assert torch.equal(dtable[:, -40:], want.t().to(torch.bfloat16))                             # below 2^24: one rounding
    assert (dtable[:, :-40] == 0).all()
    del dtable
    ncols, vocab = 33000, 50
    big = torch.zeros((ncols, units), dtype=torch.bfloat16, device="cuda").t()
    big[:, -400:] = dout
    tok = torch.arange(ncols, device="cuda") % vocab
    dtable = cb.embedding_grad(cb.colmajor_empty(units, vocab), tok, big)
    want = torch.zeros((vocab, units), dtype=torch.float64, device="cuda")
    want.index_add_(0, tok[-400:], dout.t().double())
    assert torch.equal(dtable.double(), want.t())


def test_a_token_model_of_many_positions():
    """Embedding, dropout, a DIA layer, log probabilities and the way back to the table for 2100 positions, more than the
    gradient sums unsorted.  Against the same model in 64 bits: 32-bit sums of up to some 2100 terms, each of a dozen operations -
    the summed roundings stay below 2200 * 2^-24 of the largest value."""
    units, vocab, ncols, p, seed = 96, 130, 2100, 0.2, 5
    rng = np.random.default_rng(4)
    O = cb.dev_dia_matrix_f(vocab, units, np.arange(-60, 60, dtype=np.int32))
    O.set_vec(rng.standard_normal(O.num_dia * O.stride) * 0.1)
    table = cb.to_device(rng.standard_normal((units, vocab)))
    tok, target = (torch.from_numpy(rng.integers(-1, vocab, ncols)).cuda() for _ in range(2))
    E = cb.colmajor_empty
    x, y, logits = E(units, ncols), E(units, ncols), E(vocab, ncols)
    dlogits, dy, dx, dtable = E(vocab, ncols), E(units, ncols), E(units, ncols), torch.ones((vocab, units), device="cuda").t()
    cb.embedding(x, table, tok, 1.5)
    cb.dropout(y, x, p, seed, step=1)
    cb.prod(logits, O, y)
    r = cb.token_logprob(logits, target, entropy=True)
    dlogp, dent = torch.full((ncols,), -1.0 / ncols, device="cuda"), torch.full((ncols,), -0.01 / ncols, device="cuda")
    cb.token_logprob_grad(dlogits, logits, r.lse, target, dlogp, r.entropy, dent)
    cb.prod(dy, O, dlogits, "t")
    cb.dropout_grad(dx, dy, p, seed, step=1)
    cb.embedding_grad(dtable, tok, dx, 1.5)
    first = dtable.clone()
    cb.embedding_grad(dtable, tok, dx, 1.5, 1.0)                # a second batch's, added

    keep = torch.from_numpy(ho.uniform(units, ncols, seed, 1) >= np.float32(p)).cuda()
    t64, O64 = table.double().requires_grad_(), torch.from_numpy(cb.pull(O)).cuda().double()
    x64 = torch.where(tok >= 0, t64[:, tok.clamp(min=0)] * 1.5, 0.0)
    logq = torch.log_softmax(O64 @ torch.where(keep, x64 / (1.0 - float(np.float32(p))), 0.0), 0)
    logp = torch.where(target >= 0, logq.gather(0, target.clamp(min=0)[None])[0], 0.0)
    (-logp.sum() / ncols + 0.01 / ncols * (logq.exp() * logq).sum()).backward()
    bound = 2200 * E32 * t64.grad.abs().max()
    assert (first.double() - t64.grad).abs().max() <= bound
    assert (dtable.double() - 2 * t64.grad).abs().max() <= 2 * bound


# ---- token log probabilities ----------------------------------------------------------------------------------------

FAR = 24 * math.log(2.0)        # how far, at most, the logit that a column's sums are relative to lies below its largest one


def check(logits, tokens, scale, top, r):
    """Against 64 bits.  With z - R the exponents, R at most FAR below the largest z:  a power is off by 2^-22 and by four roundings
    of its exponent (the difference, log2(e), its product with the scale, the product), once more for what it is rescaled by when
    the reference grows; sums are taken in at most vocab/128 + 150 additions and rescaled at most vocab/1024 + 40 times, each time
    by a power and a product.  The logarithm and its product with ln 2 are off by 2^-22 of themselves, which R adds FAR to."""
    lse, logp, ent, logq, spread = plain_logprob(logits, tokens, scale)
    vocab, size = logits.shape[0], math.log(logits.shape[0]) + FAR
    err = (vocab / 1024 + 40) * (2.0 ** -22 + E32) + (vocab / 128 + 150) * E32 + 4 * E32 * (spread + 3 * FAR)
    near(r.lse, lse, err + 2.0 ** -22 * (lse.abs().nan_to_num(posinf=0.0) + size))
    if tokens is not None:
        near(r.logp, logp, err + 2.0 ** -22 * (logp.abs().nan_to_num(posinf=0.0) + size))
    if r.entropy is not None:
        near(r.entropy, ent, err * (1 + 2 * (spread + FAR)) + 2.0 ** -22 * (spread + size))
    if top:
        ranked = torch.where(torch.isnan(logits.float()), -math.inf, logits.float())
        value, index = torch.sort(ranked.t(), dim=1, descending=True, stable=True)
        index = torch.where(value == -math.inf, -1, index)[:, :top]
        index = torch.nn.functional.pad(index, (0, top - index.shape[1]), value=-1)
        assert torch.equal(r.top_index, index.int().t())
        want = torch.where(index < 0, -math.inf, logq.t().gather(1, index.clamp(min=0))).t()
        near(r.top_logp, want, err + 2.0 ** -22 * (want.abs().nan_to_num(posinf=0.0) + size))


# rows and columns: eight lanes, a warp, 128 threads, 256 threads and clusters of 2, 4 and 8 blocks a column
SHAPES = [(700, 800), (1000, 601), (3000, 2000), (8000, 1300), (40000, 700), (40000, 300), (40000, 40), (131072, 4)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ncols", SHAPES)
@pytest.mark.parametrize("top", [0, 3])
def test_a_token_far_above_the_others(kind, vocab, ncols, top):
    """One token anywhere in a column, 40 to 80 above the others, around what a sum of powers can hold too: certain, whatever the
    sums are relative to.  The others' powers sum up to 2^-25 at most, so each sum that has the token's power of one in it stays one,
    and what is left is their own share: vocab e^-40 of the log probability, and 80 times that of the entropy."""
    g, dtype = gen(vocab + top), TYPES[kind]
    x = (torch.rand((ncols, vocab), device="cuda", generator=g) - 1.0).to(dtype).t()
    place = torch.randint(0, vocab, (ncols,), device="cuda", generator=g)
    height = torch.rand(ncols, device="cuda", generator=g) * 40 + 40
    x.scatter_(0, place[None], height.to(dtype)[None])
    share = vocab * math.exp(-40.0)
    assert share < 2.0 ** -25
    for entropy in (False, True):
        r = cb.token_logprob(x, place, entropy=entropy, top=top)
        assert r.logp.abs().max() <= share
        assert torch.equal(r.lse, x.float().gather(0, place[None])[0])
        if entropy:
            assert r.entropy.abs().max() <= 81 * share
        if top:
            assert torch.equal(r.top_index[0], place.int()) and torch.equal(r.top_logp[0], r.logp)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ncols", SHAPES)
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_masks_ties_and_specials_on_every_path(kind, vocab, ncols, top):
    g, dtype, off = gen(vocab * 3 + top), TYPES[kind], vocab % 7 + 1

    def ask(logits, entropy=True):
        return cb.token_logprob(logits, tok, scale=0.8, entropy=entropy, top=top)

    x, buf = matrix(g, vocab, ncols, dtype, vocab + off, off, spread=6.0)
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    check(x, tok, 0.8, top, ask(x))
    check(x, tok, 0.8, top, ask(x, False))
    # the first half far below the rest, not at all, and by more than a sum of powers can hold
    for low in (-9.0, -30.0, -65.0, -75.0, -200.0):
        y = x.t().clone().t()
        y[:vocab // 2] += low
        check(y, tok, 0.8, top, ask(y))
        check(y, tok, 0.8, top, ask(y, False))
    # ties: few different values, then a single one
    y = torch.randint(0, 3, (ncols, vocab), device="cuda", generator=g).to(dtype).t()
    check(y, tok, 0.8, top, ask(y))
    y.fill_(1.5)
    r = ask(y)
    check(y, tok, 0.8, top, r)
    assert r.top_index is None or r.top_index[:, -1].tolist() == list(range(top))
    # forbidden tokens, the type's lowest value, columns with nothing left
    x[torch.rand((ncols, vocab), device="cuda", generator=g).t() < 0.5] = -math.inf
    x[torch.rand(vocab, device="cuda", generator=g) < 0.1] = torch.finfo(dtype).min
    x[:vocab // 3, ::2] = -math.inf
    x[:vocab // 3, 1::3] = torch.finfo(dtype).min
    x[:, 1] = -math.inf
    x[:, -1] = -math.inf
    want = ask(x)
    check(x, tok, 0.8, top, want)
    check(x, tok, 0.8, top, ask(x, False))
    assert want.lse[1] == -math.inf and want.entropy[1] == 0
    # NaN and +inf in single columns, which leave the others as they were
    x[vocab - 2, 0] = math.nan
    x[vocab // 2, 2] = math.inf
    r = ask(x)
    there = (tok >= 0) & (tok < vocab)
    for name in ("lse", "logp", "entropy"):
        a, b = getattr(r, name).clone(), getattr(want, name)
        for col in (0, 2):
            assert torch.isnan(a[col]) or name == "logp" and not there[col]
            a[col] = b[col]
        assert torch.equal(a, b)
    if top:
        rest = [c for c in range(ncols) if c not in (0, 2)]
        assert r.top_index[0, 2] == vocab // 2 and torch.equal(r.top_index[:, rest], want.top_index[:, rest])
        assert not (r.top_index[:, 0] == vocab - 2).any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ncols", SHAPES)
def test_far_logits_without_alternatives(kind, vocab, ncols):
    """Logits around 10000 (1000 in half precision): the differences cancel the offset."""
    g, dtype = gen(vocab), TYPES[kind]
    x = (torch.randn((ncols, vocab), device="cuda", generator=g) * 3 + (1000.0 if kind == "f16" else 10000.0)).to(dtype).t()
    tok = torch.randint(0, vocab, (ncols,), device="cuda", generator=g)
    for entropy in (False, True):
        check(x, tok, 1.0, 0, cb.token_logprob(x, tok, entropy=entropy))
