"""LayerNorm + modulation and RMSNorm + rotary embedding with their gradients, against the formulas in 64 bits.

Tolerances.  u = eps / 2 of the output's type is the largest relative error of one rounding.  16-bit outputs are computed in
fp32 (relative error of a few 2^-24 times the terms that are added) and rounded once, so every element is within u of its
own value plus ``SLACK`` of the largest term that enters it; fp32 outputs have the second part alone.  ``SLACK``: a statistic
over D <= 8192 elements is added as at most 32 per thread, 5 shuffle steps and 16 warps, each step one rounding: 53 roundings,
two such statistics and fewer than 20 further operations per element: 128 * 2^-24 bounds their sum.  Column sums of R rows:
a CTA adds R / ctas rows in sequence, then at most 16 * 148 / 16 + 16 partial sums: (R + 164) roundings at worst against the sum
of absolute values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SLACK = 128 * 2.0 ** -24


@pytest.fixture(scope="module")
def ops(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import ops as _ops
    return _ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _unit(dt):
    return torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0


def _close(got, want, largest, dt):
    """|got - want| <= u |want| (1 + SLACK) + SLACK * largest, elementwise; fp16 results below its normal range are off by up
    to half of its smallest step."""
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0
    off = (got.double().cpu() - want).abs()
    bound = (_unit(dt) * want.abs()) * (1 + 2 * SLACK) + SLACK * largest + tiny
    bad = off > bound
    assert not bad.any(), f"{int(bad.sum())} elements, worst {float((off / bound.clamp_min(1e-300)).max()):.3g} of the bound"


def _sums_close(got, want, absolute, rows):
    bound = (rows + 164 + 128) * 2.0 ** -24 * absolute + 1e-30
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


def _ln_reference(x, dy, w, c, shift, scale, eps=1e-6):
    x, dy = x.double(), dy.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).pow(2).mean(-1, keepdim=True) + eps)
    n = (x - mean) * rstd
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    c = torch.zeros(x.shape[-1], dtype=torch.float64) if c is None else c.double()
    m = 1 + scale.double()[:, None] if scale is not None else torch.ones(1, 1, 1, dtype=torch.float64)
    y = (n * w + c) * m + (shift.double()[:, None] if shift is not None else 0)
    g = dy * m * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    largest_y = ((n.abs() * w.abs() + c.abs()) * m.abs() + (shift.double().abs()[:, None] if shift is not None else 0) + (mean.abs() * rstd) * (w * m).abs())
    largest_dx = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + (1 + n.abs() + mean.abs() * rstd) * (g * n).abs().mean(-1, keepdim=True)
                         + n.abs() * (g.abs() * mean.abs() * rstd).mean(-1, keepdim=True))
    noise = n.abs() + mean.abs() * rstd  # an error in n is relative to the terms x rstd and mean rstd
    sums = {"dweight": ((dy * m * n).sum((0, 1)), ((dy * m).abs() * noise).sum((0, 1))), "dbias": ((dy * m).sum((0, 1)), (dy * m).abs().sum((0, 1))),
            "dshift": (dy.sum(1), dy.abs().sum(1)), "dscale": ((dy * (n * w + c)).sum(1), (dy.abs() * (noise * w.abs() + c.abs())).sum(1))}
    return y, dx, sums, largest_y, largest_dx, mean[..., 0], rstd[..., 0]


LN_CASES = [  # B, S, D, dtype, affine, modulate
    (1, 1, 8, "bf16", True, True), (2, 3, 24, "f32", True, True), (3, 5, 264, "f16", False, True), (1, 17, 512, "bf16", False, True),
    (2, 63, 1536, "f16", True, False), (1, 700, 1536, "bf16", True, True), (2, 9, 2056, "bf16", True, True), (1, 33, 5120, "bf16", False, True),
    (2, 21, 5120, "f32", True, True), (1, 5, 5128, "f16", True, True), (1, 7, 8192, "f32", True, True), (1, 6, 8192, "bf16", True, True),
    (1, 4, 1032, "f32", False, False), (3, 1, 4096, "f16", False, False), (1, 2400, 64, "bf16", True, True), (4, 650, 128, "f32", True, True),
]


@pytest.mark.parametrize("B,S,D,dtype,affine,modulate", LN_CASES)
def test_layernorm_modulate(ops, B, S, D, dtype, affine, modulate):
    g, t = _gen(D + S), TYPES[dtype]
    x = (torch.randn(B, S, D, generator=g) * 1.5 + torch.randn(D, generator=g)).to(t)
    dy = (torch.randn(B, S, D, generator=g)).to(t)
    w, c = (1 + 0.2 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)) if affine else (None, None)
    shift, scale = (0.3 * torch.randn(B, D, generator=g), 0.3 * torch.randn(B, D, generator=g)) if modulate else (None, None)
    y_ref, dx_ref, sums, ly, ldx, mean_ref, rstd_ref = _ln_reference(x, dy, w, c, shift, scale)
    d = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    y, mean, rstd = ops.layernorm_modulate(d(x), ln_weight=d(w), ln_bias=d(c), shift=d(shift), scale=d(scale))
    got = ops.layernorm_modulate_backward(d(dy), d(x), mean, rstd, ln_weight=d(w), ln_bias=d(c), scale=d(scale))
    _close(y, y_ref, ly, t)
    _close(got[0], dx_ref, ldx, t)
    assert ((rstd.double().cpu() - rstd_ref).abs() <= SLACK * rstd_ref * (1 + (mean_ref * rstd_ref) ** 2)).all()
    for name, v in zip(("dweight", "dbias", "dshift", "dscale"), got[1:]):
        if v is None:
            assert (name in ("dweight", "dbias") and not affine) or (name in ("dshift", "dscale") and not modulate)
        else:
            _sums_close(v, *sums[name], B * S)


def _rotate(y, cos, sin):
    a, b = y.unflatten(-1, (-1, 64, 2)).unbind(-1)
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-3)


RMS_CASES = [  # B, S, D, dtype, weight, rotate
    (1, 1, 128, "bf16", True, True), (2, 3, 256, "f32", True, True), (3, 11, 384, "f16", True, True), (1, 19, 512, "bf16", True, True),
    (2, 40, 1536, "bf16", True, True), (1, 25, 5120, "bf16", True, True), (2, 6, 5120, "f32", True, True), (1, 5, 8192, "f16", True, True),
    (1, 5, 8192, "f32", True, True), (2, 31, 200, "bf16", True, False), (1, 9, 1040, "f32", False, False), (2, 7, 640, "f16", False, True),
    (1, 1800, 128, "f32", True, True),
]


@pytest.mark.parametrize("B,S,D,dtype,weight,rotate", RMS_CASES)
def test_rmsnorm_rope(ops, B, S, D, dtype, weight, rotate):
    g, t = _gen(D + S), TYPES[dtype]
    x, dy = (torch.randn(B, S, D, generator=g) * 2).to(t), torch.randn(B, S, D, generator=g).to(t)
    w = 1 + 0.2 * torch.randn(D, generator=g) if weight else None
    cos = sin = None
    if rotate:
        ang = torch.rand(S + 3, 64, generator=g) * 6.28
        cos, sin = ang.cos(), ang.sin()
    xd, dyd, wd = x.double(), dy.double(), (w.double() if weight else torch.ones(D, dtype=torch.float64))
    rstd_ref = 1 / torch.sqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6)
    n = xd * rstd_ref
    y_ref, back = n * wd, dyd
    ly, lback = (n * wd).abs(), dyd.abs()
    if rotate:
        cd, sd = cos[:S, None].double(), sin[:S, None].double()
        y_ref, back = _rotate(n * wd, cd, sd), _rotate(dyd, cd, -sd)
        ly, lback = _rotate(ly, cd.abs(), -sd.abs()).abs() + _rotate(ly, cd.abs(), sd.abs()).abs(), dyd.abs().unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(B, S, D // 2, 2).flatten(-2)
    gr = back * wd
    dx_ref = rstd_ref * (gr - n * (gr * n).mean(-1, keepdim=True))
    lg = lback * wd.abs()
    ldx = rstd_ref * (lg + n.abs() * (lg * n.abs()).mean(-1, keepdim=True))
    d = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    y, rstd = ops.rmsnorm_rope(d(x), d(w), rope_cos=d(cos), rope_sin=d(sin))
    dx, dw = ops.rmsnorm_rope_backward(d(dy), d(x), rstd, d(w), rope_cos=d(cos), rope_sin=d(sin))
    _close(y, y_ref, ly, t)
    _close(dx, dx_ref, ldx, t)
    if weight:
        _sums_close(dw, (back * n).sum((0, 1)), (lback * n.abs()).sum((0, 1)), B * S)
    else:
        assert dw is None


def test_layernorm_constant_rows_and_large_means(ops):
    """A constant row normalises to nothing; a mean far above the spread costs only what its own rounding costs."""
    D = 1536
    x = torch.full((1, 3, D), 7.3)
    x[0, 1] = 1000 + torch.randn(D, generator=_gen(0))
    x[0, 2] = 0
    y, mean, rstd = ops.layernorm_modulate(x.to(DEV))
    assert y[0, 0].abs().max() == 0 and y[0, 2].abs().max() == 0
    xd = x[0, 1].double()
    n = (xd - xd.mean()) / torch.sqrt(xd.var(correction=0) + 1e-6)
    # x - mean is exact to half an ulp of the mean's own rounding: 1000 * 2^-24, over a spread of one
    assert (y[0, 1].double().cpu() - n).abs().max() <= 1000 * 2.0 ** -24 + SLACK * 4


def test_strided_rows_and_gradients_of_any_layout(ops):
    """Rows inside a wider buffer, a token-strided batch, a gradient that is a broadcast scalar, an unaligned slice."""
    g = _gen(3)
    B, S, D = 2, 9, 520
    wide = torch.randn(B, S, 2 * D, generator=g).bfloat16().to(DEV)
    x = wide[:, :, D:]
    y, mean, rstd = ops.layernorm_modulate(x)
    y0, mean0, rstd0 = ops.layernorm_modulate(x.contiguous())
    assert torch.equal(y, y0) and torch.equal(mean, mean0) and torch.equal(rstd, rstd0)
    xt = torch.randn(S, B, D, generator=g).bfloat16().to(DEV).transpose(0, 1)
    assert torch.equal(ops.rmsnorm_rope(xt)[0], ops.rmsnorm_rope(xt.contiguous())[0])
    one = torch.ones((), device=DEV, dtype=torch.bfloat16).expand(B, S, D)
    got = ops.layernorm_modulate_backward(one, x, mean, rstd)[0]
    assert torch.equal(got, ops.layernorm_modulate_backward(one.contiguous(), x.contiguous(), mean, rstd)[0])
    odd = torch.randn(S, D + 3, generator=g).bfloat16().to(DEV)[:, 3:]
    assert torch.equal(ops.layernorm_modulate(odd)[0], ops.layernorm_modulate(odd.contiguous())[0])


def test_equal_inputs_give_equal_bits_and_streams_do_not_mix(ops):
    g = _gen(5)
    B, S, D = 2, 900, 1536
    x, dy = torch.randn(B, S, D, generator=g).bfloat16().to(DEV), torch.randn(B, S, D, generator=g).bfloat16().to(DEV)
    scale = torch.randn(B, D, generator=g).to(DEV)
    _, mean, rstd = ops.layernorm_modulate(x, shift=scale, scale=scale)
    ref = ops.layernorm_modulate_backward(dy, x, mean, rstd, scale=scale)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    res = []
    for _ in range(3):
        for st in (s1, s2):
            with torch.cuda.stream(st):
                res.append(ops.layernorm_modulate_backward(dy, x, mean, rstd, scale=scale))
    torch.cuda.synchronize()
    for r in res:
        for a, b in zip(r, ref):
            assert (a is None and b is None) or torch.equal(a, b)


def test_empty_inputs(ops):
    x = torch.empty(2, 0, 256, device=DEV, dtype=torch.bfloat16)
    scale = torch.ones(2, 256, device=DEV)
    y, mean, rstd = ops.layernorm_modulate(x, shift=scale, scale=scale)
    assert y.shape == x.shape and mean.shape == (2, 0)
    dx, _, _, dshift, dscale = ops.layernorm_modulate_backward(x, x, mean, rstd, scale=scale)
    assert dx.shape == x.shape and not dshift.any() and not dscale.any()
    dw = ops.rmsnorm_rope_backward(x, x, rstd, torch.ones(256, device=DEV))[1]
    assert not dw.any()
