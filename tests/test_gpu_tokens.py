"""The token-model operators against plain implementations in 64 bits: column lookup by token and its gradient, dropout with
drawn masks, token log probabilities with entropy and alternatives, and their gradient.

Tolerances count roundings: a result rounded to type t is off by at most eps(t)/2 relative (half the smallest subnormal near
zero), an operation in 32 bits by 2^-24 relative, the kernels' power of two by 2^-22."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import cuv_b200 as cb
from oracle import host_oracle as ho

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(g, rows, cols, dtype, ld=None, offset=0, spread=1.0, fill=None):
    """A column-major matrix whose columns lie ld apart and that starts `offset` elements behind an aligned address, with
    its whole buffer (the rest of it NaN)."""
    ld = ld or rows
    buf = torch.full((offset + ld * cols + 8,), math.nan, dtype=dtype, device="cuda")
    m = buf[offset:offset + ld * cols].view(cols, ld).t()[:rows]
    if fill is None:
        m.copy_((torch.randn((cols, rows), device="cuda", generator=g) * spread).to(dtype).t())
    else:
        m.fill_(fill)
    return m, buf


def outside_untouched(buf, m):
    """Nothing but the matrix itself was written."""
    inside = torch.zeros_like(buf, dtype=torch.bool)
    inside.as_strided(m.shape, m.stride(), m.storage_offset() - buf.storage_offset()).fill_(True)
    assert torch.isnan(buf[~inside]).all()


def near(got, want, bound):
    """|got - want| <= bound where want is finite, equality elsewhere."""
    got, want = got.double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(nan=7.0), want[~fine].nan_to_num(nan=7.0))
    over = (got - want).abs()[fine] - (bound.expand_as(want)[fine] if isinstance(bound, torch.Tensor) else bound)
    assert not torch.isnan(got[fine]).any()
    assert over.numel() == 0 or over.max().item() <= 0, "over the bound by %g" % over.max().item()


# sizes, leading dimensions and offsets: whole vectors, odd ones, columns on any alignment
LAYOUTS = [(8, None, 0), (1, None, 0), (7, 9, 1), (64, 64, 0), (65, 72, 0), (257, 257, 3), (1000, 1004, 4), (1023, 1023, 0),
           (2048, 2048, 0), (4096, 4104, 8), (9001, 9001, 5), (16384, 16384, 0)]


# ---- lookup ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("units, ld, offset", LAYOUTS)
@pytest.mark.parametrize("ncols", [1, 5, 300])
def test_embedding(kind, units, ld, offset, ncols):
    g, dtype = gen(units + ncols), TYPES[kind]
    vocab = 37
    table, _ = matrix(g, units, vocab, dtype, ld, offset)
    dst, buf = matrix(g, units, ncols, dtype, ld, offset, fill=5.0)
    tok = torch.randint(-2, vocab + 2, (ncols,), device="cuda", generator=g)
    for scale, t in ((1.0, tok), (0.37, tok.int())):
        cb.embedding(dst, table, t, scale)
        there = (tok >= 0) & (tok < vocab)
        want = torch.where(there, table.double()[:, tok.clamp(0, vocab - 1)] * float(np.float32(scale)), 0.0)
        near(dst, want, want.abs() * (HALF[dtype] + E32) * 1.01 + TINY[dtype])
        outside_untouched(buf, dst)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("units", [*range(1, 42), 63, 64, 65, 127, 255, 257, 333, 511, 767, 1023, 1025, 1534, 2047, 2049])
def test_embedding_of_short_columns_that_lie_differently(kind, units):
    """Whole columns come out bit for bit, whatever the alignment of either side."""
    g, dtype, vocab, ncols = gen(units), TYPES[kind], 19, 41
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    there = (tok >= 0) & (tok < vocab)
    for shift, ld_from, ld_to in ((0, units, units), (3, units + 1, units + 2), (5, units + 3, units), (7, units, units + 5)):
        table, _ = matrix(g, units, vocab, dtype, ld_from, shift)
        dst, buf = matrix(g, units, ncols, dtype, ld_to, 7 - shift, fill=5.0)
        cb.embedding(dst, table, tok)
        assert torch.equal(dst, torch.where(there, table[:, tok.clamp(0, vocab - 1)], 0.0))
        outside_untouched(buf, dst)


def test_embedding_copies_bits_and_reads_no_other_column():
    table = torch.full((5, 64), math.nan, device="cuda").t()
    table[:, 3] = torch.tensor([0.0, -0.0, math.inf, -math.inf] * 16, device="cuda")
    dst = cb.colmajor_empty(64, 4)
    cb.embedding(dst, table, torch.tensor([3, -1, 5, 3], device="cuda"))
    assert torch.equal(dst[:, 0].view(torch.int32), table[:, 3].contiguous().view(torch.int32))
    assert torch.equal(dst[:, 3], dst[:, 0]) and (dst[:, 1:3] == 0).all()


# ---- gradient of the table ----------------------------------------------------------------------------------------

def grad_check(dout, tok, dtable, before, fnew, fold):
    """Against sums in 64 bits.  A sum of n terms is n additions in 32 bits at most, whatever their order; then two
    products, an addition and the rounding of the result."""
    units, vocab = dtable.shape
    there = (tok >= 0) & (tok < vocab)
    n = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, tok[there].long(), torch.ones_like(tok[there], dtype=torch.float64))
    total = torch.zeros((vocab, units), dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(total)
    total.index_add_(0, tok[there].long(), dout.t().double()[there])
    mass.index_add_(0, tok[there].long(), dout.t().double()[there].abs())
    fn, fo = float(np.float32(fnew)), float(np.float32(fold))
    want = (fn * total.t() + (fo * before.double() if fold else 0.0))
    old = before.double().abs() * abs(fo) if fold else 0.0
    bound = (abs(fn) * mass.t() * (n + 3) + 3 * old) * E32 * 1.01 + want.abs() * HALF[dtable.dtype] + TINY[dtable.dtype]
    near(dtable, want, bound)
    if fold == 1.0:
        assert torch.equal(dtable[:, n == 0].nan_to_num(7.0), before[:, n == 0].nan_to_num(7.0))


@pytest.mark.parametrize("kind, grad", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("units, ld, offset", [(8, None, 0), (1, 3, 1), (65, 72, 0), (257, 257, 3), (1023, 1023, 0), (2048, 2056, 0),
                                               (9001, 9001, 1)])
@pytest.mark.parametrize("vocab, ncols", [(1, 40), (37, 1), (37, 1000), (3001, 700)])
def test_embedding_grad(kind, grad, units, ld, offset, vocab, ncols):
    g = gen(units * 7 + vocab + ncols)
    dout, _ = matrix(g, units, ncols, TYPES[kind], ld, offset)
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    for fnew, fold, t in ((1.0, 0.0, tok), (0.5, 1.0, tok.int()), (-2.0, 0.25, tok)):
        dtable, buf = matrix(g, units, vocab, TYPES[grad], ld, offset)
        if fold == 0.0:
            dtable.fill_(math.nan)                          # not read
        before = dtable.clone()
        cb.embedding_grad(dtable, t, dout, fnew, fold)
        grad_check(dout, tok, dtable, before, fnew, fold)
        outside_untouched(buf, dtable)


@pytest.mark.parametrize("ncols", [31, 256, 257, 1024, 1025, 4095, 4097, 8192, 8193, 16384, 20000, 32769, 70001, 131072, 131073, 300001])
@pytest.mark.parametrize("vocab", [2, 511, 512, 131071, 300007])
def test_embedding_grad_sums_whole_numbers_exactly(ncols, vocab):
    """Whole numbers whose sums stay below 2^24: equality, whatever the order; text-like frequencies, so that single
    tokens fill many chunks, and a vocabulary of one, two and three digits of the sort."""
    g = gen(ncols + vocab)
    units = 24
    dout = torch.randint(-100, 101, (ncols, units), device="cuda", generator=g).float().t()
    tok = ((torch.rand(ncols, device="cuda", generator=g, dtype=torch.float64) * math.log(vocab + 1)).exp().long() - 1).clamp(0, vocab - 1)
    tok[torch.rand(ncols, device="cuda", generator=g) < 0.1] = -7
    dtable = cb.colmajor_empty(units, vocab)
    cb.embedding_grad(dtable, tok, dout)
    want = torch.zeros((vocab + 1, units), dtype=torch.float64, device="cuda")
    want.index_add_(0, torch.where(tok < 0, vocab, tok), dout.t().double())
    assert torch.equal(dtable.double(), want[:vocab].t())


@pytest.mark.parametrize("case", ["one token", "all padding", "no columns", "ascending", "descending"])
@pytest.mark.parametrize("many", [200, 2500])
def test_embedding_grad_extremes(case, many):
    units, vocab, ncols = 40, 3000, 0 if case == "no columns" else many
    dout = torch.randint(-9, 10, (ncols, units), device="cuda", generator=gen(1)).float().t()
    tok = {"one token": torch.full((ncols,), 17), "all padding": torch.full((ncols,), -1), "no columns": torch.empty(0, dtype=torch.long),
           "ascending": torch.arange(ncols), "descending": vocab - 1 - torch.arange(ncols)}[case].cuda()
    for fold in (0.0, 1.0, 2.0):
        dtable = torch.ones((vocab, units), device="cuda").t()
        cb.embedding_grad(dtable, tok, dout, 1.0, fold)
        want = torch.full((vocab, units), fold, dtype=torch.float64, device="cuda")
        keep = tok >= 0
        want.index_add_(0, tok[keep], dout.t().double()[keep])
        assert torch.equal(dtable.double(), want.t())


def test_embedding_grad_gives_the_same_bits_every_time():
    g = gen(4)
    dout = matrix(g, 513, 9000, torch.bfloat16)[0]
    tok = torch.randint(0, 60, (9000,), device="cuda", generator=g)
    first = cb.embedding_grad(cb.colmajor_empty(513, 60), tok, dout)
    for _ in range(3):
        assert torch.equal(cb.embedding_grad(cb.colmajor_empty(513, 60), tok, dout), first)


# ---- dropout --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows, ld, offset", LAYOUTS)
@pytest.mark.parametrize("ncols, residual", [(1, False), (19, True), (40, False)])
def test_dropout(kind, rows, ld, offset, ncols, residual):
    g, dtype = gen(rows + ncols), TYPES[kind]
    seed, step, col0, which, p = 0xABCDEF0123456789 + rows, 3, 11, 2, [0.1, 0.5, 0.9][rows % 3]
    src, _ = matrix(g, rows, ncols, dtype, ld, offset)
    res = matrix(g, rows, ncols, dtype, ld, offset)[0] if residual else None
    dst, buf = matrix(g, rows, ncols, dtype, ld, offset, fill=5.0)
    cb.dropout(dst, src, p, seed, step, col0, which, residual=res)
    keep = torch.from_numpy(ho.uniform(rows, ncols, seed, step, col0, which) >= np.float32(p)).cuda()
    kept = torch.where(keep, src.double() / (1.0 - float(np.float32(p))), 0.0)
    want = kept + res.double() if residual else kept
    # the factor 1/(1-p), the product, the sum, and the result's rounding
    near(dst, want, kept.abs() * 2 * E32 * 1.01 + want.abs() * (E32 * 1.01 + HALF[dtype]) + TINY[dtype])
    assert (dst[~keep] == (res[~keep] if residual else 0)).all()
    outside_untouched(buf, dst)


def test_dropout_layouts_may_differ():
    """src, residual and dst on different alignments and leading dimensions."""
    g = gen(9)
    src, res = matrix(g, 1001, 33, torch.float16, 1001, 1)[0], matrix(g, 1001, 33, torch.float16, 1008, 0)[0]
    dst, buf = matrix(g, 1001, 33, torch.float16, 1003, 6, fill=0.0)
    cb.dropout(dst, src, 0.3, 5, residual=res)
    same = cb.dropout(cb.colmajor_empty(1001, 33, dtype=torch.float16), src.t().contiguous().t(), 0.3, 5, residual=res.t().contiguous().t())
    assert torch.equal(dst, same)
    outside_untouched(buf, dst)


def test_dropout_borders_of_p_and_dropped_specials():
    x = torch.tensor([math.nan, math.inf, -math.inf, 1.0] * 64, device="cuda").view(4, 64).t()
    r = torch.randn(4, 64, device="cuda").t()
    out = cb.colmajor_empty(64, 4)
    assert (cb.dropout(out, x, 1.0, 1) == 0).all()
    assert torch.equal(cb.dropout(out, x, 1.0, 1, residual=r), r)
    assert torch.equal(cb.dropout(out, r, 0.0, 1), r)
    keep = torch.from_numpy(ho.uniform(64, 4, 1) >= np.float32(0.5)).cuda()
    cb.dropout(out, x, 0.5, 1)
    assert (out[~keep] == 0).all() and torch.equal(out[keep].nan_to_num(7.0, 8.0, 9.0), (x * 2)[keep].nan_to_num(7.0, 8.0, 9.0))
    # the smallest p drops exactly the elements whose number is zero, the largest below 1 all but the largest number
    tiny = cb.dropout(out, r, 2.0 ** -25, 1)
    assert (tiny != 0).all()


def test_dropout_in_place_and_backward():
    """The gradient against the formula (the same elements, the same factor) and against differences of a loss."""
    g = gen(2)
    x, y = matrix(g, 515, 21, torch.float32)[0], cb.colmajor_empty(515, 21)
    cb.dropout(y, x, 0.25, 77, step=4, which=1)
    z = x.t().clone().t()
    assert torch.equal(cb.dropout(z, z, 0.25, 77, step=4, which=1), y)
    z = x.t().clone().t()
    assert torch.equal(cb.dropout(z, torch.zeros(21, 515, device="cuda").t(), 0.25, 77, step=4, which=1, residual=z), x)
    dy = matrix(g, 515, 21, torch.float32)[0]
    dx = cb.dropout_grad(cb.colmajor_empty(515, 21), dy, 0.25, 77, step=4, which=1)
    v = matrix(g, 515, 21, torch.float32)[0]
    fv = cb.dropout(cb.colmajor_empty(515, 21), v, 0.25, 77, step=4, which=1)
    a, b = (dx.double() * v.double()).sum().item(), (dy.double() * fv.double()).sum().item()      # linear: <f'(dy), v> = <dy, f(v)>
    mass = (dy.double().abs() * fv.double().abs()).sum().item()
    assert abs(a - b) <= 4 * E32 * mass
    # every shard of the columns draws what the whole draws
    part = cb.dropout(cb.colmajor_empty(515, 6), x[:, 15:], 0.25, 77, step=4, col0=15, which=1)
    assert torch.equal(part, y[:, 15:])


# ---- token log probabilities ----------------------------------------------------------------------------------------

def plain_logprob(logits, tokens, scale):
    """In 64 bits: lse, logp, entropy, log probabilities, and the mean of |log2 p / pmax| that bounds count with."""
    z = logits.double() * float(np.float32(scale))
    m = z.amax(0).nan_to_num(neginf=0.0)
    logs = torch.log(torch.exp(z - m).sum(0))
    lse = m + logs
    logq = torch.where(lse == -math.inf, -math.inf, (z - m) - logs)     # z - lse loses logs where m is f32's lowest value
    q = torch.exp(logq)
    ent = -(q * torch.where(q == 0, 0.0, logq)).sum(0)
    vocab = logits.shape[0]
    logp = None
    if tokens is not None:
        there = (tokens >= 0) & (tokens < vocab)
        logp = torch.where(there, logq.gather(0, tokens.long().clamp(0, vocab - 1)[None])[0], 0.0)
    spread = (q * torch.where(q == 0, 0.0, (z - m).abs())).sum(0)
    return lse, logp, ent, logq, spread


def sum_error(vocab, spread):
    """Relative error of the sum of powers: a term's exponent d is off by two roundings of it (spread: their mean over the
    distribution), its power by 2^-22; the sum is taken in at most vocab/128 + 64 additions in 32 bits, and rescaled at most
    vocab/1024 + 32 times, each time by a power of two and a product."""
    return (vocab / 1024 + 34) * (2.0 ** -22 + E32) + (vocab / 128 + 64) * E32 + 4 * E32 * spread


def check_logprob(logits, tokens, scale, top, r):
    lse, logp, ent, logq, spread = plain_logprob(logits, tokens, scale)
    vocab = logits.shape[0]
    err = sum_error(vocab, spread)
    near(r.lse, lse, err + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0))
    if logp is not None:
        near(r.logp, logp, err + 2.0 ** -22 * (logp.abs().nan_to_num(posinf=0.0) + math.log(vocab)))
    if r.entropy is not None:
        near(r.entropy, ent, err * (1 + 2 * spread) + 2.0 ** -22 * (spread + math.log(vocab)))
    if top:
        ranked = torch.where(torch.isnan(logits.float()), -math.inf, logits.float())
        value, index = torch.sort(ranked.t(), dim=1, descending=True, stable=True)
        value, index = value[:, :top], index[:, :top]
        index = torch.where(value == -math.inf, -1, index)
        if index.shape[1] < top:
            index = torch.nn.functional.pad(index, (0, top - index.shape[1]), value=-1)
        assert torch.equal(r.top_index, index.int().t())
        want = torch.where(index < 0, -math.inf, logq.t().gather(1, index.clamp(min=0))).t()
        near(r.top_logp, want, (err + 2.0 ** -22 * (want.abs().nan_to_num(posinf=0.0) + math.log(vocab))))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ld, offset", [(1, None, 0), (2, 5, 1), (31, 31, 3), (256, None, 0), (257, 257, 5), (1000, 1008, 0),
                                               (4093, 4093, 1), (8192, None, 0), (32771, 32771, 7), (65536, None, 0)])
@pytest.mark.parametrize("ncols, top", [(1, 5), (3, 0), (37, 32), (300, 1)])
def test_token_logprob(kind, vocab, ld, offset, ncols, top):
    g, dtype = gen(vocab + ncols), TYPES[kind]
    logits, buf = matrix(g, vocab, ncols, dtype, ld, offset, spread=4.0)
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    keep = buf.clone()
    r = cb.token_logprob(logits, tok, scale=1.0, entropy=True, top=top)
    check_logprob(logits, tok, 1.0, top, r)
    r = cb.token_logprob(logits, tok.int(), scale=0.3, top=top)
    assert r.entropy is None
    check_logprob(logits, tok, 0.3, top, r)
    r = cb.token_logprob(logits, top=top)
    assert r.logp is None
    check_logprob(logits, None, 1.0, top, r)
    assert torch.equal(buf.nan_to_num(7.0), keep.nan_to_num(7.0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ncols", [(300, 5), (5000, 3), (40000, 2), (40000, 200)])
def test_token_logprob_masks_ties_and_specials(kind, vocab, ncols):
    g, dtype = gen(vocab), TYPES[kind]
    x = matrix(g, vocab, ncols, dtype, spread=2.0)[0]
    tok = torch.randint(0, vocab, (ncols,), device="cuda", generator=g)
    # most tokens forbidden, the given one of the first column among them; the lowest finite value as a mask elsewhere
    x[torch.rand(vocab, device="cuda", generator=g) < 0.9] = -math.inf
    x[tok[0], 0] = -math.inf
    x[torch.rand(vocab, device="cuda", generator=g) < 0.05] = torch.finfo(dtype).min
    check_logprob(x, tok, 1.0, 20, cb.token_logprob(x, tok, entropy=True, top=20))
    # nothing left in the last column
    x[:, -1] = -math.inf
    r = cb.token_logprob(x, tok, entropy=True, top=20)
    check_logprob(x, tok, 1.0, 20, r)
    assert r.lse[-1] == -math.inf and r.logp[-1] == -math.inf and r.entropy[-1] == 0 and (r.top_index[:, -1] == -1).all()
    # one token left: certain
    x[:, 0] = -math.inf
    x[vocab // 2, 0] = -3.0
    r = cb.token_logprob(x, torch.full((ncols,), vocab // 2, device="cuda"), entropy=True, top=2)
    assert r.logp[0] == 0 and r.entropy[0] == 0 and r.lse[0] == -3.0 and r.top_index[:, 0].tolist() == [vocab // 2, -1]
    # ties: few different values, all equal ones last
    y = torch.randint(0, 3, (ncols, vocab), device="cuda", generator=g).to(dtype).t()
    check_logprob(y, tok, 1.0, 32, cb.token_logprob(y, tok, entropy=True, top=32))
    y.fill_(1.5)
    r = cb.token_logprob(y, tok, entropy=True, top=32)
    check_logprob(y, tok, 1.0, 32, r)
    assert r.top_index[:, 0].tolist() == list(range(32))
    # ascending and descending logits: the alternatives' list turns over all the time, or never
    ramp = (torch.arange(vocab, device="cuda").float() * (8.0 / vocab)).to(dtype)
    y.copy_(ramp[:, None].expand(vocab, ncols))
    check_logprob(y, tok, 1.0, 32, cb.token_logprob(y, tok, entropy=True, top=32))
    y.copy_(ramp.flip(0)[:, None].expand(vocab, ncols))
    check_logprob(y, tok, 1.0, 32, cb.token_logprob(y, tok, entropy=True, top=32))
    # NaN and +inf make a column's numbers NaN and leave its neighbours alone; NaN is never among the likeliest
    z = matrix(g, vocab, ncols, dtype)[0]
    want = cb.token_logprob(z, tok, entropy=True, top=3)
    w = z.t().clone().t()
    w[vocab // 3, 0] = math.nan
    w[vocab - 1, 1] = math.inf
    r = cb.token_logprob(w, tok, entropy=True, top=3)
    for name in ("lse", "logp", "entropy"):
        a, b = getattr(r, name), getattr(want, name)
        assert torch.isnan(a[:2]).all() and torch.equal(a[2:], b[2:])
    assert r.top_index[0, 1] == vocab - 1 and torch.equal(r.top_index[:, 2:], want.top_index[:, 2:])
    left = z[:, 0].float().clone()
    left[vocab // 3] = -math.inf
    assert r.top_index[0, 0] == left.argmax()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ld, offset", [(1, None, 0), (3, 5, 1), (50, 50, 3), (256, None, 0), (509, 509, 5), (512, 1000, 0),
                                               (515, 515, 1), (1023, 1023, 7), (1031, 1031, 2)])
@pytest.mark.parametrize("ncols", [591, 593, 2111])
def test_token_logprob_of_many_short_columns(kind, vocab, ld, offset, ncols):
    g, dtype = gen(vocab + ncols), TYPES[kind]
    x, buf = matrix(g, vocab, ncols, dtype, ld, offset, spread=4.0)
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    keep = buf.clone()
    check_logprob(x, tok, 1.0, 0, cb.token_logprob(x, tok, entropy=True))
    check_logprob(x, tok, 0.3, 0, cb.token_logprob(x, tok.int(), scale=0.3))
    assert torch.equal(buf.nan_to_num(7.0), keep.nan_to_num(7.0))
    # forbidden tokens, the type's lowest value, columns without a token left, NaN and +inf in single columns
    x[torch.rand(vocab, ncols, device="cuda", generator=g) < 0.4] = -math.inf
    x[torch.rand(vocab, ncols, device="cuda", generator=g) < 0.05] = torch.finfo(dtype).min
    x[:, 7] = -math.inf
    x[:, -1] = -math.inf
    want = cb.token_logprob(x, tok, entropy=True)
    check_logprob(x, tok, 1.0, 0, want)
    assert want.lse[-1] == -math.inf and want.entropy[7] == 0
    x[vocab // 2, 3] = math.nan
    x[vocab - 1, 12] = math.inf
    r = cb.token_logprob(x, tok, entropy=True)
    there = (tok >= 0) & (tok < vocab)
    for name in ("lse", "logp", "entropy"):
        a, b = getattr(r, name).clone(), getattr(want, name)
        for col in (3, 12):
            assert torch.isnan(a[col]) or name == "logp" and not there[col]
            a[col] = b[col]
        assert torch.equal(a, b)


def test_token_logprob_of_far_logits():
    """A large offset cancels in logp and entropy, as the differences to the largest logit are exact."""
    g = gen(6)
    x = (torch.randn(4, 5000, device="cuda", generator=g) + 10000.0).t()
    tok = torch.arange(4, device="cuda")
    r = cb.token_logprob(x, tok, entropy=True, top=4)
    check_logprob(x, tok, 1.0, 4, r)


@pytest.mark.parametrize("vocab, ncols", [(50, 9), (3000, 2000), (40000, 3), (40000, 700)])
def test_token_logprob_gives_what_is_asked_for(vocab, ncols):
    """The C entry point with every choice of results; what is not asked for is not written."""
    from cuv_b200 import _capi
    x = matrix(gen(3), vocab, ncols, torch.float16, spread=3.0)[0]
    tok = torch.randint(0, vocab, (ncols,), device="cuda", generator=gen(4), dtype=torch.int32)
    all_of_them = cb.token_logprob(x, tok, scale=0.5, entropy=True, top=7)
    for choice in range(1, 16):
        logp, lse, ent = (torch.full((ncols,), 9.0, device="cuda") for _ in range(3))
        top_logp, top_index = torch.full((ncols, 7), 9.0, device="cuda"), torch.full((ncols, 7), 9, dtype=torch.int32, device="cuda")
        want = [choice >> k & 1 for k in range(4)]
        rc = _capi.lib().cuvdia_token_logprob(
            x.data_ptr(), vocab, _capi.T_F16, vocab, ncols, tok.data_ptr() if want[0] else None, _capi.T_I32, 0.5,
            logp.data_ptr() if want[0] else None, lse.data_ptr() if want[1] else None, ent.data_ptr() if want[2] else None,
            7 if want[3] else 0, top_logp.data_ptr() if want[3] else None, top_index.data_ptr() if want[3] else None,
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        check_logprob(x, tok, 0.5, 7 if want[3] else 0, cb.TokenLogprob(
            logp if want[0] else all_of_them.logp, lse if want[1] else all_of_them.lse, ent if want[2] else None,
            top_logp.t(), top_index.t()))
        for t, w in ((logp, want[0]), (lse, want[1]), (ent, want[2]), (top_logp, want[3]), (top_index, want[3])):
            assert w or (t == 9).all()


# ---- gradient of the log probabilities ------------------------------------------------------------------------------

def check_grad(dlogits, logits, lse, tok, dlogp, entropy, dentropy, scale):
    """The formula in 64 bits on the same lse and entropy.  The exponent x c - lse log2(e) carries the roundings of c, of the
    product lse log2(e) and of itself: |x c| and |lse| log2(e) each off by 2^-24 or twice that."""
    dtype, vocab = logits.dtype, logits.shape[0]
    s = float(np.float32(scale))
    z, l = logits.double() * s, lse.double()
    empty = l == -math.inf
    logq = z - l
    q = torch.where(empty, 0.0, torch.exp(logq))
    logq = torch.where(q == 0, 0.0, logq)
    there = (tok >= 0) & (tok < vocab) if dlogp is not None else torch.zeros_like(l, dtype=torch.bool)
    gw = torch.where(there & ~empty, dlogp.double(), 0.0) if dlogp is not None else torch.zeros_like(l)
    hot = torch.zeros_like(q)
    if dlogp is not None:
        cols = torch.arange(len(l), device="cuda")[there]
        hot[tok.long()[there], cols] = 1.0
    h = dentropy.double() if dentropy is not None else torch.zeros_like(l)
    H = entropy.double() if entropy is not None else torch.zeros_like(l)
    H = torch.where(empty, 0.0, H)
    w = gw + h * (logq + H)
    want = s * (gw * hot - q * w)
    far = z.abs().nan_to_num(posinf=0.0) + l.abs().nan_to_num(posinf=0.0)                        # natural units
    derr = far * 4 * E32                                        # of the exponent, in natural units
    werr = (gw.abs() + h.abs() * (logq.abs() + H.abs())) * 4 * E32 + h.abs() * derr
    bound = s * (q * (derr + 2.0 ** -22) * w.abs() + q * werr) + (want.abs() + s * (gw * hot).abs()) * 3 * E32
    # below 2^-126 a power is zero
    bound = bound * 1.01 + s * w.abs() * 2.0 ** -125 + want.abs() * HALF[dtype] + TINY[dtype]
    near(dlogits, want, bound)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ld, offset", [(1, None, 0), (2, 5, 1), (31, 31, 3), (256, None, 0), (257, 257, 5), (4093, 4093, 1),
                                               (8192, None, 0), (32771, 32771, 7), (65536, None, 0)])
@pytest.mark.parametrize("ncols", [1, 37])
def test_token_logprob_grad(kind, vocab, ld, offset, ncols):
    g, dtype = gen(vocab + ncols), TYPES[kind]
    x = matrix(g, vocab, ncols, dtype, ld, offset, spread=3.0)[0]
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    dlogp, dent = torch.randn(ncols, device="cuda", generator=g), torch.randn(ncols, device="cuda", generator=g)
    dlogp[tok < 0] = math.nan                                   # not used
    for scale in (1.0, 0.7):
        r = cb.token_logprob(x, tok, scale=scale, entropy=True)
        for t, a, e, b in ((tok, dlogp, None, None), (None, None, r.entropy, dent), (tok.int(), dlogp, r.entropy, dent)):
            d, buf = matrix(g, vocab, ncols, dtype, ld, offset, fill=5.0)
            cb.token_logprob_grad(d, x, r.lse, t, a, e, b, scale)
            check_grad(d, x, r.lse, tok, a, e, b, scale)
            outside_untouched(buf, d)
        # another alignment of the result, and in place
        d, buf = matrix(g, vocab, ncols, dtype, vocab + 3, 2, fill=5.0)
        cb.token_logprob_grad(d, x, r.lse, tok, dlogp, r.entropy, dent, scale)
        check_grad(d, x, r.lse, tok, dlogp, r.entropy, dent, scale)
        outside_untouched(buf, d)
        y, buf = matrix(g, vocab, ncols, dtype, ld, offset, fill=0.0)
        y.copy_(x)
        cb.token_logprob_grad(y, y, r.lse, tok, dlogp, r.entropy, dent, scale)
        assert torch.equal(y, d)
        outside_untouched(buf, y)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, ld, offset", [(1, None, 0), (3, 5, 1), (50, 50, 3), (256, None, 0), (257, 257, 5), (512, 1000, 0),
                                               (509, 509, 7), (515, 515, 1)])
@pytest.mark.parametrize("ncols", [591, 593, 2111])
def test_token_logprob_grad_of_many_short_columns(kind, vocab, ld, offset, ncols):
    g, dtype = gen(vocab + ncols), TYPES[kind]
    x = matrix(g, vocab, ncols, dtype, ld, offset, spread=3.0)[0]
    tok = torch.randint(-1, vocab + 1, (ncols,), device="cuda", generator=g)
    dlogp, dent = torch.randn(ncols, device="cuda", generator=g), torch.randn(ncols, device="cuda", generator=g)
    dlogp[tok < 0] = math.nan                                   # not used
    for masked in (False, True):
        if masked:
            x[torch.rand(vocab, ncols, device="cuda", generator=g) < 0.4] = -math.inf
            x[:, 7] = -math.inf
            x[:, -1] = -math.inf
        r = cb.token_logprob(x, tok, scale=0.7, entropy=True)
        for a, e, b in ((dlogp, None, None), (None, r.entropy, dent), (dlogp, r.entropy, dent)):
            d, buf = matrix(g, vocab, ncols, dtype, ld, offset, fill=5.0)
            cb.token_logprob_grad(d, x, r.lse, tok if a is not None else None, a, e, b, 0.7)
            check_grad(d, x, r.lse, tok, a, e, b, 0.7)
            outside_untouched(buf, d)
        other, buf = matrix(g, vocab, ncols, dtype, vocab + 3, 2, fill=5.0)         # another alignment, and in place
        cb.token_logprob_grad(other, x, r.lse, tok, dlogp, r.entropy, dent, 0.7)
        outside_untouched(buf, other)
        y, buf = matrix(g, vocab, ncols, dtype, ld, offset, fill=0.0)
        y.copy_(x)
        cb.token_logprob_grad(y, y, r.lse, tok, dlogp, r.entropy, dent, 0.7)
        assert torch.equal(y, d) and torch.equal(other, d)
        outside_untouched(buf, y)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_token_logprob_grad_masks(kind):
    g, dtype, vocab = gen(5), TYPES[kind], 3003
    x = matrix(g, vocab, 4, dtype, spread=2.0)[0]
    x[torch.rand(vocab, device="cuda", generator=g) < 0.5] = -math.inf
    x[:, 3] = -math.inf                                         # nothing left
    tok = torch.tensor([5, -1, 7, 8], device="cuda")
    x[5, 0] = -math.inf                                         # the given token is forbidden: probability zero
    x[7, 2] = torch.finfo(dtype).min
    dlogp, dent = torch.tensor([1.0, math.nan, -2.0, 3.0], device="cuda"), torch.tensor([0.5, 0.1, -1.0, 2.0], device="cuda")
    r = cb.token_logprob(x, tok, entropy=True)
    d = cb.colmajor_empty(vocab, 4, dtype=dtype)
    cb.token_logprob_grad(d, x, r.lse, tok, dlogp, r.entropy, dent)
    check_grad(d, x, r.lse, tok, dlogp, r.entropy, dent, 1.0)
    assert (d[:, 3] == 0).all() and torch.isfinite(d.float()).all()
    d.fill_(9.0)
    cb.token_logprob_grad(d, x, r.lse, tok, dlogp)
    check_grad(d, x, r.lse, tok, dlogp, None, None, 1.0)
    assert (d[:, 1] == 0).all() and (d[:, 3] == 0).all()


def test_token_logprob_grad_against_differences():
    """Central differences of the loss in 64 bits: off by their third derivative times step^2 (below |w| step^2 here, every
    derivative of log p and of the entropy being bounded by a few times |log p|) and by the cancellation, 1e-16 / step."""
    g = gen(12)
    x = matrix(g, 50, 3, torch.float32, spread=1.5)[0]
    tok = torch.tensor([4, 0, 49], device="cuda")
    dlogp, dent = torch.tensor([1.0, -0.5, 2.0], device="cuda"), torch.tensor([0.3, 1.0, -0.7], device="cuda")

    def loss(v):
        _, logp, ent, _, _ = plain_logprob(v, tok, 0.8)
        return (dlogp.double() * logp + dent.double() * ent).sum().item()

    r = cb.token_logprob(x, tok, scale=0.8, entropy=True)
    d = cb.token_logprob_grad(cb.colmajor_empty(50, 3), x, r.lse, tok, dlogp, r.entropy, dent, 0.8)
    step = 1e-4
    for v, j in [(4, 0), (7, 0), (0, 1), (30, 1), (49, 2), (12, 2)]:
        up, down = x.double(), x.double()
        up[v, j] += step
        down[v, j] -= step
        slope = (loss(up) - loss(down)) / (2 * step)
        assert abs(d[v, j].item() - slope) <= 20 * step ** 2 + 1e-11 / step + 1e-5 * abs(slope) + 1e-6


# ---- sizes beyond 32-bit offsets, streams, graphs, refusals ---------------------------------------------------------

def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 elements: what lies at the far end is read and written there."""
    rows, cols = 65536, 33000
    big = torch.empty((cols, rows), dtype=torch.bfloat16, device="cuda").t()
    big[:, -3:] = torch.randn(3, rows, device="cuda").t().to(torch.bfloat16)
    far = big[:, -3:].t().clone().t()
    out = cb.colmajor_empty(rows, 2, dtype=torch.bfloat16)
    assert torch.equal(cb.embedding(out, big, torch.tensor([cols - 1, cols - 3], device="cuda")), far[:, [2, 0]])
    r = cb.token_logprob(big, None, top=3)
    want = cb.token_logprob(far, None, top=3)
    # a call's blocks share a column by how many columns there are, so its sums may be added in another order: each is held
    # against 64 bits, as everywhere else
    for got in (cb.TokenLogprob(None, r.lse[-3:], None, r.top_logp[:, -3:], r.top_index[:, -3:]), want):
        check_logprob(far, None, 1.0, 3, got)
    seen = cb.dropout(cb.colmajor_empty(rows, 3, dtype=torch.bfloat16), far, 0.5, 9, col0=cols - 3)
    cb.dropout(big, big, 0.5, 9)
    assert torch.equal(big[:, -3:], seen)
    big[:, -3:] = far
    lse = torch.zeros(cols, device="cuda")
    lse[-3:] = want.lse
    tok = torch.full((cols,), -1, device="cuda")
    tok[-3:] = torch.tensor([1, 2, 3], device="cuda")
    ones = torch.ones(cols, device="cuda")
    cb.token_logprob_grad(big, big, lse, tok, ones)
    assert torch.equal(big[:, -3:], cb.token_logprob_grad(far, far, want.lse, tok[-3:], ones[-3:]))
    assert (big[:, :-3] == 0).all()
    tok[:-3] = -1
    g = torch.empty((cols, rows), dtype=torch.bfloat16, device="cuda").t()
    cb.embedding_grad(g, torch.tensor([cols - 1, cols - 1, cols - 2], device="cuda"), far)
    assert torch.equal(g[:, -2], far[:, 2])
    assert torch.equal(g[:, -1], (far[:, 0].float() + far[:, 1].float()).to(torch.bfloat16)) and (g[:, :-2] == 0).all()


def model_operands(seed, units=96, vocab=300, ncols=50):
    g = gen(seed)
    return dict(table=matrix(g, units, vocab, torch.float32)[0], tok=torch.randint(-1, vocab, (ncols,), device="cuda", generator=g),
                target=torch.randint(-1, vocab, (ncols,), device="cuda", generator=g))


def test_on_another_stream_and_in_a_graph():
    """All operators queued on a side stream, recorded on their first call of that size, replayed on new contents; two
    recorded graphs replayed in turn do not share anything."""
    def chain(m, b):
        cb.embedding(b["x"], m["table"], m["tok"], 2.0)
        cb.dropout(b["y"], b["x"], 0.3, 5, residual=b["x"])
        r = cb.token_logprob(b["y"], m["target"] % 90, entropy=True, top=4)
        cb.token_logprob_grad(b["dy"], b["y"], r.lse, m["target"] % 90, b["ones"], r.entropy, b["ones"])
        cb.dropout_grad(b["dx"], b["dy"], 0.3, 5)
        cb.embedding_grad(b["dt"], m["tok"], b["dx"], 2.0)
        return r

    def buffers():
        b = {k: cb.colmajor_empty(96, 50) for k in ("x", "y", "dy", "dx")}
        return dict(b, dt=cb.colmajor_empty(96, 300), ones=torch.ones(50, device="cuda"))

    want = []
    for seed in (1, 2):
        m, b = model_operands(seed), buffers()
        r = chain(m, b)
        want.append((b["dt"].clone(), r.logp.clone(), r.top_index.clone()))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    made = []
    for seed in (3, 4):
        m, b = model_operands(seed), buffers()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            r = chain(m, b)
        made.append((graph, m, b, r))
    torch.cuda.synchronize()
    for k, (graph, m, b, r) in enumerate(made):
        for name, t in model_operands(1 + k).items():
            m[name].copy_(t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(3):
        for s, (graph, m, b, r) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, m, b, r), w in zip(made, want):
        assert torch.equal(b["dt"], w[0]) and torch.equal(r.logp, w[1]) and torch.equal(r.top_index, w[2])


def test_recorded_on_their_very_first_call():
    """A process whose first call of every operator is the recorded one."""
    code = """
import torch, cuv_b200 as cb
E = cb.colmajor_empty
table, x, y, dy, dt = E(96, 300), E(96, 50), E(96, 50), E(96, 50), E(96, 300)
table.normal_()
tok, ones = torch.arange(50, device="cuda") % 7, torch.ones(50, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    cb.embedding(x, table, tok)
    cb.dropout(y, x, 0.5, 1)
    r = cb.token_logprob(y, tok, entropy=True, top=3)
    cb.token_logprob_grad(dy, y, r.lse, tok, ones, r.entropy, ones)
    cb.embedding_grad(dt, tok, dy)
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (x, y, r.lse, r.top_index, dy, dt)]
cb.embedding(x, table, tok)
cb.dropout(y, x, 0.5, 1)
r = cb.token_logprob(y, tok, entropy=True, top=3)
cb.token_logprob_grad(dy, y, r.lse, tok, ones, r.entropy, ones)
cb.embedding_grad(dt, tok, dy)
assert all(torch.equal(a, b) for a, b in zip(got, (x, y, r.lse, r.top_index, dy, dt)))
assert dt[:, :7].abs().sum() > 0 and (dt[:, 7:] == 0).all()
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stderr[-2000:]


def test_shapes_types_and_devices_are_refused():
    E = cb.colmajor_empty
    i64 = torch.zeros(3, dtype=torch.int64, device="cuda")
    bad = [
        lambda: cb.embedding(E(5, 3), E(4, 9), i64), lambda: cb.embedding(E(4, 2), E(4, 9), i64),
        lambda: cb.embedding(E(4, 3, dtype=torch.float16), E(4, 9), i64), lambda: cb.embedding(E(4, 3), E(4, 9), i64.float()),
        lambda: cb.embedding(E(4, 3), E(4, 9), i64.cpu()), lambda: cb.embedding(E(4, 3), E(4, 9), i64[:, None]),
        lambda: cb.embedding(E(4, 3, "cpu"), E(4, 9), i64),
        lambda: cb.embedding(E(4, 3), E(4, 9), torch.zeros(6, dtype=torch.int64, device="cuda")[::2]),
        lambda: cb.embedding_grad(E(5, 9), i64, E(4, 3)), lambda: cb.embedding_grad(E(4, 9, dtype=torch.float16), i64, E(4, 3)),
        lambda: cb.embedding_grad(E(4, 9, dtype=torch.float16), i64, E(4, 3, dtype=torch.bfloat16)),
        lambda: cb.embedding_grad(E(4, 9), i64[:2], E(4, 3)),
        lambda: cb.dropout(E(4, 3), E(4, 2), 0.5, 1), lambda: cb.dropout(E(4, 3), E(4, 3, dtype=torch.float16), 0.5, 1),
        lambda: cb.dropout(E(4, 3), E(4, 3), 0.5, 1, residual=E(4, 2)), lambda: cb.dropout(E(4, 3), E(4, 3), 1.5, 1),
        lambda: cb.dropout(E(4, 3), E(4, 3), 0.5, 1, which=-1), lambda: cb.dropout(E(4, 3), E(4, 3), 0.5, 1, step=1 << 32),
        lambda: cb.token_logprob(E(4, 3), i64[:2]), lambda: cb.token_logprob(E(4, 3), top=33), lambda: cb.token_logprob(E(4, 3), scale=0.0),
        lambda: cb.token_logprob_grad(E(4, 3), E(4, 3), torch.zeros(2, device="cuda"), i64, torch.zeros(3, device="cuda")),
        lambda: cb.token_logprob_grad(E(4, 3), E(4, 3), torch.zeros(3, device="cuda"), i64),
        lambda: cb.token_logprob_grad(E(4, 3), E(4, 3), torch.zeros(3, device="cuda"), i64, torch.zeros(3)),
        lambda: cb.token_logprob_grad(E(4, 3), E(4, 3), torch.zeros(3, device="cuda")),
        lambda: cb.token_logprob_grad(E(4, 3, dtype=torch.float16), E(4, 3), torch.zeros(3, device="cuda"), i64, torch.zeros(3, device="cuda")),
    ]
    before = cb.launch_count()
    for k, call in enumerate(bad):
        with pytest.raises(cb.CuvDiaError):
            call()
    assert cb.launch_count() == before


def test_no_columns():
    E = cb.colmajor_empty
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    cb.embedding(E(4, 0), E(4, 9), none)
    cb.dropout(E(4, 0), E(4, 0), 0.5, 1)
    r = cb.token_logprob(E(4, 0), none, entropy=True, top=3)
    assert r.lse.numel() == 0 and tuple(r.top_index.shape) == (3, 0)
    cb.token_logprob_grad(E(4, 0), E(4, 0), r.lse, none, r.logp)
    torch.cuda.synchronize()


# ---- together: a token model around a DIA layer ---------------------------------------------------------------------

def test_a_token_model_trains_around_a_dia_layer():
    """Embedding, dropout, a banded DIA layer, an output DIA layer whose rows are the vocabulary, log probabilities, and all
    the way back to the table and both layers' diagonals; one update.  Against the same model in 64 bits: 32-bit sums of a few
    hundred terms at most, a dozen operators deep - the summed roundings stay below 600 * 2^-24 of the largest value."""
    units, vocab, ncols, p, seed = 192, 256, 70, 0.2, 99
    rng = np.random.default_rng(3)
    offs = np.arange(-16, 16, dtype=np.int32)
    outs = np.arange(-64, 60, dtype=np.int32)
    W, O = cb.dev_dia_matrix_f(units, units, offs), cb.dev_dia_matrix_f(vocab, units, outs)
    for A in (W, O):
        A.set_vec(rng.standard_normal(A.num_dia * A.stride) * 0.1)
    table = cb.to_device(rng.standard_normal((units, vocab)))
    tok = torch.from_numpy(rng.integers(-1, vocab, ncols)).cuda()
    target = torch.from_numpy(rng.integers(-1, vocab, ncols)).cuda()
    E = cb.colmajor_empty

    def dense(A):
        return torch.from_numpy(cb.pull(A)).cuda().double()

    # forward
    x, y, hid, logits = E(units, ncols), E(units, ncols), E(units, ncols), E(vocab, ncols)
    cb.embedding(x, table, tok, 1.5)
    cb.dropout(y, x, p, seed, step=1)
    cb.prod(hid, W, y)
    cb.axpby(hid.t(), hid.t(), y.t(), 1.0, 1.0)                 # a residual path
    cb.prod(logits, O, hid)
    r = cb.token_logprob(logits, target, entropy=True, top=3)
    loss = -r.logp.sum() / ncols - 0.01 * r.entropy.sum()
    # backward
    dlogits, dhid, dy, dx = E(vocab, ncols), E(units, ncols), E(units, ncols), E(units, ncols)
    dlogp, dent = torch.full((ncols,), -1.0 / ncols, device="cuda"), torch.full((ncols,), -0.01, device="cuda")
    cb.token_logprob_grad(dlogits, logits, r.lse, target, dlogp, r.entropy, dent)
    dO, dW, dtable = cb.dev_dia_matrix_f(vocab, units, outs), cb.dev_dia_matrix_f(units, units, offs), E(units, vocab)
    for A in (dO, dW):
        A.vec.zero_()
    cb.densedense_to_dia(dO, None, dlogits, hid)
    cb.prod(dhid, O, dlogits, "t")
    cb.densedense_to_dia(dW, None, dhid, y)
    cb.prod(dy, W, dhid, "t")
    cb.axpby(dy.t(), dy.t(), dhid.t(), 1.0, 1.0)
    cb.dropout_grad(dx, dy, p, seed, step=1)
    cb.embedding_grad(dtable, tok, dx, 1.5)

    # the same model in 64 bits, differentiated by torch
    keep = torch.from_numpy(ho.uniform(units, ncols, seed, 1) >= np.float32(p)).cuda()
    t64, W64, O64 = table.double().requires_grad_(), dense(W).requires_grad_(), dense(O).requires_grad_()
    x64 = torch.where(tok >= 0, t64[:, tok.clamp(min=0)] * 1.5, 0.0)
    y64 = torch.where(keep, x64 / (1.0 - float(np.float32(p))), 0.0)
    h64 = W64 @ y64 + y64
    logq = torch.log_softmax(O64 @ h64, 0)
    logp = torch.where(target >= 0, logq.gather(0, target.clamp(min=0)[None])[0], 0.0)
    ent = -(logq.exp() * logq).sum(0)
    (-logp.sum() / ncols - 0.01 * ent.sum()).backward()

    def close(got, want):
        assert (got.double() - want).abs().max() <= 600 * E32 * want.abs().max()

    close(loss, (-logp.sum() / ncols - 0.01 * ent.sum()).detach())
    close(r.logp, logp.detach())
    close(r.entropy, ent.detach())
    close(dtable, t64.grad)
    for A, full in ((dO, O64.grad), (dW, W64.grad)):
        mask = torch.zeros_like(full, dtype=torch.bool)
        rows, cols = torch.meshgrid(torch.arange(full.shape[0]), torch.arange(full.shape[1]), indexing="ij")
        mask = ((cols - rows) >= int(A.offsets[0])) & ((cols - rows) <= int(A.offsets[-1]))
        close(dense(A), torch.where(mask.cuda(), full, 0.0))
    before = table.clone()
    cb.learn_step_weight_decay(table.t(), dtable.t(), 0.5)
    close(table, before.double() - 0.5 * t64.grad)
    assert torch.isfinite(r.top_logp).all()
