"""Gradients of rows that lean on few of many keys, where ds = p (dp - D) is a difference of nearly equal numbers.

D comes from the rounded output, and what its rounding leaves in ds is p_ij times one number e_i per row, far more than the rounding
of ds where p is near one.  sum_j ds_ij is zero, so the sum of a row's ds is that number: dk is computed with it taken out, and
so is dq with keys in one tile; with more keys dq has only e_i times the mean key taken out, and keeps
e_i times what the row's own mean key is away from that.

Bounds on the norm of the error, roundings being independent (u = eps / 2 for each, 1.7 times what a uniform rounding has): in ds u of
itself, and through D (for dk) p_ij times the sum of its row's roundings; for dq p_ij times the error of D, from the
roundings of out and of the forward pass's p; one rounding of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
C = 1 / math.sqrt(128)


@pytest.fixture(scope="module")
def ops(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import ops as _ops
    return _ops


def draw(Sq, Sk, spread, dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    n = lambda S, s=1.0: (torch.randn(1, 1, S, 128, generator=g, device=DEV) * s).to(dtype)  # noqa: E731
    return n(Sq, spread), n(Sk), n(Sk), n(Sq)


def exact(q, k, v, do):
    """dq, dk in 64 bits and the squares of their bounds."""
    u = torch.finfo(q.dtype).eps / 2
    q, k, v, do = (t[0, 0].double() for t in (q, k, v, do))
    p = torch.softmax(C * (q @ k.T), 1)
    out = p @ v
    ds = p * (do @ v.T - (do * out).sum(1, keepdim=True))
    dq, dk = C * (ds @ k), C * (ds.T @ q)
    km, qn, sq, p2 = k - k[:128].mean(0), q.square().sum(1), ds.square(), p.square()
    d_err = u * u * ((do * out).square().sum(1) + ((p2 @ v.square()) * do.square()).sum(1))
    rows = u * u * sq.sum(1)
    # scores in fp32: eight sums of sixteen products, each off by 2^-23 of a partial sum of up to twice the largest score, and the
    # exponent's argument, as a part of every p (and so of ds)
    e = (16 * 2.0 ** -23 * C * (q @ k.T).abs().amax(1) + 2.0 ** -20).square()
    e_dq = C * C * (((u * u + e[:, None]) * sq) @ km.square().sum(1) + d_err * (p @ km).square().sum(1))
    e_dk = C * C * (((u * u + e[:, None]) * sq + p2 * rows[:, None]).T @ qn)
    return dq, dk, float(e_dq.sum() + u * u * dq.square().sum()) ** 0.5, float(e_dk.sum() + u * u * dk.square().sum()) ** 0.5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spread", [1, 3, 10, 30])
@pytest.mark.parametrize("Sq,Sk", [(1000, 128), (1000, 129), (700, 2000), (60, 3000), (3000, 200), (300, 30000)])
def test_peaked_rows(ops, Sq, Sk, spread, dtype):
    q, k, v, do = draw(Sq, Sk, spread, dtype)
    out, lse = ops.attention_lse(q, k, v)
    dq, dk, _ = ops.attention_backward(do, q, k, v, out, lse)
    w_dq, w_dk, b_dq, b_dk = exact(q, k, v, do)
    for name, got, want, bound in (("dq", dq, w_dq, b_dq), ("dk", dk, w_dk, b_dk)):
        off = float((got[0, 0].double() - want).norm())
        assert off <= bound, f"{name}: {off / float(want.norm()):.3g} of the norm, {off / bound:.3g} of the bound"


def test_padded_rows_keep_out(ops):
    """The sums of rows that do not exist, whatever they hold, and lengths that leave one tile of many."""
    q, k, v, do = (t.repeat(3, 2, 1, 1) for t in draw(300, 1000, 10, torch.bfloat16))
    ql, kl = [300, 0, 131], [1000, 700, 100]
    q_lens, k_lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ql, kl))
    for b in range(3):
        q[b, :, ql[b]:] = do[b, :, ql[b]:] = math.nan
        k[b, :, kl[b]:] = v[b, :, kl[b]:] = math.inf
    out, lse = ops.attention_lse(q, k, v, q_lens=q_lens, k_lens=k_lens)
    dq, dk, dv = ops.attention_backward(do, q, k, v, out, lse, q_lens=q_lens, k_lens=k_lens)
    assert not dk[1].any() and not dv[1].any() and not dq[1].any()
    for b in (0, 2):
        one = tuple(t[b:b + 1, :1, :n].contiguous() for t, n in ((q, ql[b]), (k, kl[b]), (v, kl[b]), (do, ql[b])))
        w_dq, w_dk, b_dq, b_dk = exact(*one)
        for h in range(2):
            assert (dq[b, h, :ql[b]].double() - w_dq).norm() <= b_dq and (dk[b, h, :kl[b]].double() - w_dk).norm() <= b_dk
        assert not dq[b, :, ql[b]:].any() and not dk[b, :, kl[b]:].any()
