"""BlockDropout refuses in evaluation, and where p is 0, what it refuses in training."""

import pytest
import torch

import miniworld_b200 as mw

X = torch.zeros(2, 3, 4)
# name, shared, x, u
REFUSED = [("broadcast", None, X, X[:1]), ("broadcast x", None, X[:, :1], X), ("fewer dimensions", None, X, X[0]), ("float64", None, X.double(), X.double()),
           ("float64 alone", None, None, X.double()), ("whole numbers", None, X, X.long()), ("whole x", None, X.int(), X), ("no such dimension", 3, X, X),
           ("no such dimension", -4, X, X), ("another device", None, X, X.to("meta")), ("complex", None, X, X.to(torch.complex64))]


@pytest.mark.parametrize("name,shared,x,u", REFUSED)
def test_refusals(name, shared, x, u):
    for m in (mw.BlockDropout(0.3, shared).eval(), mw.BlockDropout(0.0, shared)):
        with pytest.raises(RuntimeError):
            m(x, u)


@pytest.mark.gpu
@pytest.mark.parametrize("name,shared,x,u", [r for r in REFUSED if "device" not in r[0]])
def test_training_refuses_them_too(name, shared, x, u):
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    for m in (mw.BlockDropout(0.3, shared), mw.BlockDropout(0.3, shared).eval(), mw.BlockDropout(0.0, shared)):
        with pytest.raises(RuntimeError):
            m(on(x), on(u))


@pytest.mark.parametrize("shared", [None, 0, -1, 2])
def test_what_training_takes(shared):
    for x, u in ((X, X + 1), (X.bfloat16(), X + 1), (X.half(), X.double() + 1), (None, X.half() + 1), (X[:0], X[:0])):
        for m in (mw.BlockDropout(0.3, shared).eval(), mw.BlockDropout(0.0, shared)):
            y = m(x, u)
            assert y.dtype == (u if x is None else x).dtype and bool((y == (u if x is None else x + u.to(x.dtype))).all())
