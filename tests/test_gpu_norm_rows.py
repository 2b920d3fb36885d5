"""LayerNorm + modulation and RMSNorm + rotary embedding, what the tests of single launches leave open: rows that share a CTA with
others, many row groups per CTA, values that are not finite, frozen parameters.

Tolerances (64-bit formulas, on the GPU).  Rows: as in ``test_gpu_norm_grad.py``, u of the value plus ``SLACK`` of the largest term, and a
value that is not a number fails.  Column sums: a thread adds the rows of its CTA, at least 148 CTAs share the rows of all samples
(``ROWS``), the join adds at most 8 x 148 / 32 partial sums per thread, five in a tree, and the samples: (ROWS + 37 + 5 + B) roundings of
the sum of absolute values, 128 for the errors of the terms."""
import pytest
import torch

from test_gpu_norm_grad import SLACK, _ln_reference, _rotate, _unit

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 1536, 5120, 8192])
def test_a_row_does_not_feel_its_neighbours(ops, D, dtype):
    """Rows with a small mean next to rows with a large one (which need a second pass over their statistics), a constant, NaN or
    infinity: every row has the bits that it has alone."""
    g = torch.Generator().manual_seed(D)
    S = 24
    x = torch.randn(1, S, D, generator=g) + 0.1
    x[0, 1::4] += 50  # a large mean in every second pair, as the second row
    x[0, 6] = 50 + x[0, 6]  # and as the first
    x[0, 9] = 3.25
    x[0, 12, 5], x[0, 15, 7] = float("nan"), float("inf")
    x = x.to(TYPES[dtype]).to(DEV)
    y, mean, rstd = ops.layernorm_modulate(x)
    for s in range(S):
        for a, b in zip((y, mean, rstd), ops.layernorm_modulate(x[:, s:s + 1])):
            assert torch.equal(a[:, s].nan_to_num(), b[:, 0].nan_to_num()) and torch.equal(a[:, s].isnan(), b[:, 0].isnan()), s
    z, zr = ops.rmsnorm_rope(x)
    for s in range(S):
        for a, b in zip((z, zr), ops.rmsnorm_rope(x[:, s:s + 1])):
            assert torch.equal(a[:, s].nan_to_num(), b[:, 0].nan_to_num()) and torch.equal(a[:, s].isnan(), b[:, 0].isnan()), s
    dy = torch.randn(1, S, D, generator=g).to(TYPES[dtype]).to(DEV)
    dx = ops.layernorm_modulate_backward(dy, x, mean, rstd)[0]
    dz = ops.rmsnorm_rope_backward(dy, x, zr)[0]
    for s in range(S):
        r = slice(s, s + 1)
        for a, b in ((dx, ops.layernorm_modulate_backward(dy[:, r], x[:, r], mean[:, r].contiguous(), rstd[:, r].contiguous())[0]),
                     (dz, ops.rmsnorm_rope_backward(dy[:, r], x[:, r], zr[:, r].contiguous())[0])):
            assert torch.equal(a[:, s].nan_to_num(), b[:, 0].nan_to_num()) and torch.equal(a[:, s].isnan(), b[:, 0].isnan()), s


def close(got, want, largest, what=""):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    bound = _unit(got.dtype) * want.abs() * (1 + 2 * SLACK) + SLACK * largest + tiny
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} elements"


def sums_close(got, want, absolute, B, S, what=""):
    rows = -(-B * S // 148) + 1
    bad = ~((got.double() - want).abs() <= (rows + 37 + 5 + B + 128) * 2.0 ** -24 * absolute + 1e-30)
    assert not bad.any(), f"{what}: {int(bad.sum())} elements"


def draw(B, S, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    t = TYPES[dtype]
    x, dy = (n(B, S, D) * 1.5 + n(D)).to(t), n(B, S, D).to(t)
    return x, dy, 1 + 0.2 * n(D), 0.3 * n(D), 0.3 * n(B, D), 0.3 * n(B, D)


def rms_reference(x, dy, w, cos, sin):
    xd, dyd, wd, cd, sd = x.double(), dy.double(), w.double(), cos[:, None].double(), sin[:, None].double()
    rstd = 1 / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6)
    n = xd * rstd
    y, back = _rotate(n * wd, cd, sd), _rotate(dyd, cd, -sd)
    pairs = lambda t: t.abs().unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(*t.shape[:-1], -1, 2).flatten(-2)  # noqa: E731
    ly, lb = pairs(n * wd), pairs(dyd)
    gr, lg = back * wd, lb * wd.abs()
    dx = rstd * (gr - n * (gr * n).mean(-1, keepdim=True))
    ldx = rstd * (lg + n.abs() * (lg * n.abs()).mean(-1, keepdim=True))
    return y, dx, (back * n).sum((0, 1)), ly, ldx, (lb * n.abs()).sum((0, 1)), rstd[..., 0]


# eight, sixteen and thirty-two elements per thread; six or more groups of rows for each CTA, the last of them not full
MANY = [(1, 15001, 512), (2, 8191, 1536), (1, 6001, 5120), (1, 3001, 8192)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,D", MANY)
def test_layernorm_over_many_row_groups(ops, B, S, D, dtype):
    x, dy, w, c, shift, scale = draw(B, S, D, dtype, 1)
    y_ref, dx_ref, sums, ly, ldx, mean_ref, rstd_ref = _ln_reference(x, dy, w, c, shift, scale)
    y, mean, rstd = ops.layernorm_modulate(x, ln_weight=w, ln_bias=c, shift=shift, scale=scale)
    close(y, y_ref, ly, "y")
    # the mean of D values of size |x|, D / 32 warps' worth of roundings and then some: SLACK of the mean of |x|
    assert bool(((mean.double() - mean_ref).abs() <= SLACK * x.double().abs().mean(-1)).all())
    assert bool(((rstd.double() - rstd_ref).abs() <= SLACK * rstd_ref * (1 + (mean_ref * rstd_ref) ** 2)).all())
    got = ops.layernorm_modulate_backward(dy, x, mean, rstd, ln_weight=w, ln_bias=c, scale=scale)
    close(got[0], dx_ref, ldx, "dx")
    for name, v in zip(("dweight", "dbias", "dshift", "dscale"), got[1:]):
        sums_close(v, *sums[name], B, S, name)
    frozen = ops.layernorm_modulate_backward(dy, x, mean, rstd, ln_weight=w, ln_bias=c, scale=scale, need_params=False)
    close(frozen[0], dx_ref, ldx, "dx of frozen parameters")
    assert frozen[1:] == (None,) * 4


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,D", MANY)
def test_rmsnorm_over_many_row_groups(ops, B, S, D, dtype):
    x, dy, w = draw(B, S, D, dtype, 2)[:3]
    ang = torch.rand(S, 64, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 6.28
    cos, sin = ang.cos(), ang.sin()
    y_ref, dx_ref, dw_ref, ly, ldx, ldw, rstd_ref = rms_reference(x, dy, w, cos, sin)
    y, rstd = ops.rmsnorm_rope(x, w, rope_cos=cos, rope_sin=sin)
    close(y, y_ref, ly, "y")
    assert bool(((rstd.double() - rstd_ref).abs() <= SLACK * rstd_ref).all())
    dx, dw = ops.rmsnorm_rope_backward(dy, x, rstd, w, rope_cos=cos, rope_sin=sin)
    close(dx, dx_ref, ldx, "dx")
    sums_close(dw, dw_ref, ldw, B, S, "dweight")
    frozen, none = ops.rmsnorm_rope_backward(dy, x, rstd, w, rope_cos=cos, rope_sin=sin, need_params=False)
    close(frozen, dx_ref, ldx, "dx of frozen parameters")
    assert none is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [256, 2048, 6144])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["x", "dy"])
def test_values_that_are_not_finite(ops, D, dtype, bad, where):
    """One such value: outputs and sums are NaN or infinite exactly where the formula makes them so, everything else is right."""
    B, S = 2, 37
    x, dy, w, c, shift, scale = draw(B, S, D, dtype, 4)
    (x if where == "x" else dy)[1, 8, 130] = bad
    ang = torch.rand(S, 64, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) * 6.28 + 0.1
    cos, sin = ang.cos(), ang.sin()

    def same(got, want, bound_of):
        finite = want.isfinite()
        assert torch.equal(got.isfinite(), finite)
        bound_of(torch.where(finite, got.double(), 0).to(got.dtype), torch.where(finite, want, 0))

    y_ref, dx_ref, sums, ly, ldx, _, _ = _ln_reference(x, dy, w, c, shift, scale)
    y, mean, rstd = ops.layernorm_modulate(x, ln_weight=w, ln_bias=c, shift=shift, scale=scale)
    same(y, y_ref, lambda a, b: close(a, b, ly.nan_to_num(0, 0, 0)))
    got = ops.layernorm_modulate_backward(dy, x, mean, rstd, ln_weight=w, ln_bias=c, scale=scale)
    same(got[0], dx_ref, lambda a, b: close(a, b, ldx.nan_to_num(0, 0, 0)))
    for name, v in zip(("dweight", "dbias", "dshift", "dscale"), got[1:]):
        same(v, sums[name][0], lambda a, b: sums_close(a, b, sums[name][1].nan_to_num(0, 0, 0), B, S, name))
    y_ref, dx_ref, dw_ref, ly, ldx, ldw, _ = rms_reference(x, dy, w, cos, sin)
    y, rstd = ops.rmsnorm_rope(x, w, rope_cos=cos, rope_sin=sin)
    same(y, y_ref, lambda a, b: close(a, b, ly.nan_to_num(0, 0, 0)))
    dx, dw = ops.rmsnorm_rope_backward(dy, x, rstd, w, rope_cos=cos, rope_sin=sin)
    same(dx, dx_ref, lambda a, b: close(a, b, ldx.nan_to_num(0, 0, 0)))
    same(dw, dw_ref, lambda a, b: sums_close(a, b, ldw.nan_to_num(0, 0, 0), B, S))
