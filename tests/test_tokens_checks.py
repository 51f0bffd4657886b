"""Refusals of the token-model operators (column lookup by token, dropout, token log probabilities, their gradients): what the
C entry points and the Python layer turn away before anything touches a device."""
import ctypes
import os

import pytest
import torch

import cuv_b200 as cb
from cuv_b200 import _capi

F32, F16, BF16, I32, I64 = _capi.T_F32, _capi.T_F16, _capi.T_BF16, _capi.T_I32, _capi.T_I64
P = ctypes.c_void_p(1 << 20)            # never dereferenced: the checks come before any CUDA call
ODD = ctypes.c_void_p((1 << 20) + 1)
DRAW = _capi.Draw(1, 0, 0)


@pytest.fixture(scope="module")
def L():
    from cuv_b200 import build
    build.build()
    return _capi.lib()


def changed(good, **other):
    args = dict(good)
    assert set(other) <= set(args)
    args.update(other)
    return list(args.values())


EMB = dict(dst=P, ldd=8, table=P, ldt=8, type=BF16, units=8, vocab=5, tokens=P, token_type=I64, ncols=0, scale=1.0, stream=None)
GRAD = dict(dtable=P, ldt=8, grad_type=F32, dout=P, ldo=8, type=BF16, units=8, vocab=5, tokens=P, token_type=I32, ncols=5000,
            fnew=1.0, fold=0.0, work=P, bytes=1 << 30, stream=None)
DROP = dict(dst=P, ldd=8, src=P, lds=8, residual=None, ldr=0, type=F16, rows=8, ncols=0, p=0.5, draw=ctypes.byref(DRAW), which=0,
            stream=None)
LOGP = dict(logits=P, ld=8, type=F32, vocab=8, ncols=0, tokens=P, token_type=I64, scale=1.0, logp=P, lse=P, entropy=P, top=2,
            top_logp=P, top_index=P, stream=None)
LGRAD = dict(dlogits=P, ldd=8, logits=P, ld=8, type=F32, vocab=8, ncols=0, tokens=P, token_type=I64, scale=1.0, lse=P, dlogp=P,
             entropy=P, dentropy=P, stream=None)


def test_accepted_without_columns(L):
    assert L.cuvdia_embedding(*EMB.values()) == 0
    assert L.cuvdia_dropout(*DROP.values()) == 0
    assert L.cuvdia_token_logprob(*LOGP.values()) == 0
    assert L.cuvdia_token_logprob_grad(*LGRAD.values()) == 0


@pytest.mark.parametrize("other", [dict(dst=None), dict(table=None), dict(tokens=None), dict(type=_capi.T_I32), dict(type=I64),
                                   dict(type=7), dict(token_type=F32), dict(token_type=_capi.T_U8), dict(units=0), dict(vocab=0), dict(units=(1 << 30) + 1, ldd=(1 << 30) + 1, ldt=(1 << 30) + 1),
                                   dict(ncols=-1), dict(ldd=7), dict(ldt=7), dict(dst=ODD), dict(table=ODD), dict(tokens=ODD)])
def test_embedding_refuses(L, other):
    assert L.cuvdia_embedding(*changed(EMB, **other)) == _capi.ERR_INVALID
    assert L.cuvdia_last_error_message()


@pytest.mark.parametrize("other", [dict(dtable=None), dict(dout=None), dict(tokens=None), dict(work=None), dict(bytes=1000),
                                   dict(work=ODD), dict(grad_type=F16), dict(type=F32, grad_type=BF16), dict(type=I32),
                                   dict(token_type=F32), dict(units=0), dict(vocab=0), dict(ncols=-1), dict(ncols=(1 << 30) + 1),
                                   dict(ldt=7), dict(ldo=7), dict(dout=ODD), dict(dtable=ODD), dict(tokens=ODD)])
def test_embedding_grad_refuses(L, other):
    assert L.cuvdia_embedding_grad(*changed(GRAD, **other)) == _capi.ERR_INVALID


def test_embedding_grad_workspace(L):
    n = ctypes.c_longlong(-1)
    for bad in ((0, 5, 3), (8, 0, 3), (8, 5, -1), (8, 5, (1 << 30) + 1)):
        assert L.cuvdia_embedding_grad_workspace(*bad, ctypes.byref(n)) == _capi.ERR_INVALID
    assert L.cuvdia_embedding_grad_workspace(8, 5, 3, None) == _capi.ERR_INVALID
    assert L.cuvdia_embedding_grad_workspace(8, 5, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert L.cuvdia_embedding_grad_workspace(4096, 131072, 8, ctypes.byref(n)) == 0 and n.value == 0       # few: none
    last = 0
    for ncols in (5000, 100000, 1 << 24, 1 << 30):
        assert L.cuvdia_embedding_grad_workspace(4096, 131072, ncols, ctypes.byref(n)) == 0
        assert n.value > last
        last = n.value
        assert L.cuvdia_embedding_grad(*changed(GRAD, units=4096, vocab=131072, ldt=4096, ldo=4096, ncols=ncols, bytes=n.value - 1)) \
            == _capi.ERR_INVALID


@pytest.mark.parametrize("other", [dict(dst=None), dict(src=None), dict(draw=None), dict(type=I32), dict(rows=0), dict(ncols=-1),
                                   dict(rows=(1 << 30) + 1, ldd=(1 << 30) + 1, lds=(1 << 30) + 1),
                                   dict(ldd=7), dict(lds=7), dict(residual=P, ldr=7), dict(p=-0.1), dict(p=1.1),
                                   dict(p=float("nan")), dict(which=-1), dict(which=65536), dict(src=ODD), dict(dst=ODD),
                                   dict(residual=ODD, ldr=8), dict(draw=ctypes.byref(_capi.Draw(1, 1 << 32, 0))),
                                   dict(draw=ctypes.byref(_capi.Draw(1, 0, -1)))])
def test_dropout_refuses(L, other):
    assert L.cuvdia_dropout(*changed(DROP, **other)) == _capi.ERR_INVALID


@pytest.mark.parametrize("other", [dict(logits=None), dict(type=_capi.T_U8), dict(vocab=0), dict(vocab=(1 << 30) + 1, ld=(1 << 30) + 1),
                                   dict(ncols=-1), dict(ld=7), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=2e30),
                                   dict(scale=float("nan")), dict(tokens=None), dict(logp=None), dict(token_type=F32), dict(top=-1),
                                   dict(top=33), dict(top_logp=None), dict(top_index=None), dict(logits=ODD), dict(tokens=ODD), dict(logp=ODD),
                                   dict(lse=ODD), dict(entropy=ODD), dict(top_logp=ODD), dict(top_index=ODD),
                                   dict(tokens=None, logp=None, lse=None, entropy=None, top=0)])
def test_token_logprob_refuses(L, other):
    assert L.cuvdia_token_logprob(*changed(LOGP, **other)) == _capi.ERR_INVALID


@pytest.mark.parametrize("other", [dict(dlogits=None), dict(logits=None), dict(lse=None), dict(type=I64), dict(vocab=0), dict(ncols=-1),
                                   dict(ld=7), dict(ldd=7), dict(scale=0.0), dict(scale=float("nan")), dict(tokens=None),
                                   dict(dlogp=None), dict(entropy=None), dict(dentropy=None), dict(token_type=F16), dict(dlogits=ODD),
                                   dict(logits=ODD), dict(lse=ODD), dict(dlogp=ODD), dict(entropy=ODD), dict(dentropy=ODD),
                                   dict(tokens=None, dlogp=None, entropy=None, dentropy=None)])
def test_token_logprob_grad_refuses(L, other):
    assert L.cuvdia_token_logprob_grad(*changed(LGRAD, **other)) == _capi.ERR_INVALID


def test_the_new_element_types_are_not_reduced(L):
    assert L.cuvdia_reduce(P, F32, P, BF16, 4, 4, 0, 0, 1.0, 0.0, None) == _capi.ERR_UNSUPPORTED
    assert L.cuvdia_reduce(P, I64, P, F32, 4, 4, 0, 0, 1.0, 0.0, None) == _capi.ERR_UNSUPPORTED


# ---- the Python layer: shapes, types and layouts are looked at before the device ------------------------------------

def M(rows, cols, dtype=torch.float32):
    return torch.zeros((cols, rows), dtype=dtype).t()


TOK = torch.zeros(3, dtype=torch.int64)
V3 = torch.zeros(3)


@pytest.mark.parametrize("call, says", [
    (lambda: cb.embedding(M(4, 3), torch.zeros(4, 5), TOK), "column-major"),
    (lambda: cb.embedding(M(4, 3), M(4, 5, torch.float64), TOK), "float32, float16 or bfloat16"),
    (lambda: cb.embedding(None, M(4, 5), TOK), "CUDA"),
    (lambda: cb.embedding_grad(M(4, 5), TOK, torch.zeros(4, 3)), "column-major"),
    (lambda: cb.embedding_grad(M(4, 5), TOK, torch.zeros(3)), "2-D"),
    (lambda: cb.dropout(M(4, 3), torch.zeros(4, 3).expand(4, 3), 0.5, 1), "column-major"),
    (lambda: cb.dropout(M(4, 3), torch.zeros(4, 1).t().t().expand(4, 3), 0.5, 1), "overlapping"),
    (lambda: cb.dropout(M(4, 3), M(4, 3), 0.5, 1), "CUDA"),
    (lambda: cb.dropout_grad(M(4, 3), M(4, 3), 0.5, 1), "CUDA"),
    (lambda: cb.token_logprob(torch.zeros(4, 3)), "column-major"),
    (lambda: cb.token_logprob(M(4, 3)), "CUDA"),
    (lambda: cb.token_logprob_grad(M(4, 3), torch.zeros(3), V3), "2-D"),
])
def test_python_refuses(call, says):
    with pytest.raises(cb.CuvDiaError) as e:
        call()
    assert e.value.code == _capi.ERR_INVALID and says in str(e.value)


def test_calls_run_on_their_tensors_device(monkeypatch):
    """With another device current, a call enters the tensors' device and takes that device's stream."""
    import contextlib
    seen = []

    @contextlib.contextmanager
    def device(index):
        seen.append(("enter", index))
        yield
        seen.append(("leave", index))

    class Lib:
        def entry(self, *args):
            seen.append(args)
            return 0

    monkeypatch.setattr(_capi, "lib", lambda: Lib())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(cb, "_raw_stream", lambda index: 1000 + index)
    cb._call(0, "entry", 7)
    cb._call(2, "entry", 8)
    assert seen == [(7, 1000), ("enter", 2), (8, 1002), ("leave", 2)]


def test_cluster_barriers_order_what_came_before_them():
    """A block that has arrived may be read from no longer once the others leave the wait: every arrival releases, every wait
    acquires (a relaxed arrival orders no earlier read of another block's shared memory)."""
    import re
    from cuv_b200 import build
    found = []
    for name in sorted(os.listdir(build.CSRC)):
        with open(os.path.join(build.CSRC, name)) as f:
            found += re.findall(r"barrier\.cluster\.[a-z.]+", f.read())
    assert set(found) == {"barrier.cluster.arrive.release.aligned", "barrier.cluster.wait.acquire.aligned"}
