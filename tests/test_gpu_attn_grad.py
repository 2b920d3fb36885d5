"""Attention with its gradient against the formulas in 64 bits.

Tolerances, elementwise, from the operators' definition (c = softmax scale, u = eps / 2 of the type = one rounding, w = 2^-23: an
addition in the tensor cores' fp32 accumulators, which need not round to nearest):
  scores     128 products:  |ds_ij| <= 128 w c sum_d |q k|; the exponential is relative, and lse carries the same error: a
             probability is off by at most  e_i = 4 * 128 w c max_j sum_d |q_i k_j| + 2^-20  of itself (2^-20: ex2.approx and the
             rounding of its argument); fp16 probabilities below 2^-14 by 2^-25 absolutely
  out        (u + e_i + Sk w) sum_j p |v|, and its own rounding u |out|
  D          sum_d |do| |error of out| + 128 w sum |do out|;   dp: 128 w sum |do v|
  ds         (u + e_i) |ds| + p (error of dp + error of D)   [fp16: + 2^-25]
  dq, dk, dv sums of those times |k|, |q|, of (u + e_i) p |do|, plus (terms) w of the absolute sums, and their own rounding"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
W = 2.0 ** -23


@pytest.fixture(scope="module")
def ops(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import ops as _ops
    return _ops


@pytest.fixture(autouse=True)
def device_status_clean():
    yield
    from dax_b200 import _lib
    assert _lib.device_status() == 0, "a kernel reported a timed-out wait"


def make(B, H, Sq, Sk, dtype, seed=0, offset=2.0):
    g = torch.Generator().manual_seed(seed)
    t = TYPES[dtype]
    q = torch.randn(B, Sq, H, 128, generator=g).to(t).transpose(1, 2)
    k = (torch.randn(B, Sk, H, 128, generator=g) + offset * torch.randn(1, 1, H, 128, generator=g)).to(t).transpose(1, 2)
    v = torch.randn(B, Sk, H, 128, generator=g).to(t).transpose(1, 2)
    do = torch.randn(B, Sq, H, 128, generator=g).to(t).transpose(1, 2)
    return [x.to(DEV) for x in (q, k, v, do)]


def reference(q, k, v, do, q_lens, k_lens, c, one_tile=False):
    """Results and their error bounds; padded tokens are replaced by zeros first (they take no part).  ``one_tile``: with at
    most 128 keys D is not taken from the rounded ``out`` but as sum_j p dp."""
    B, H, Sq, _ = q.shape
    Sk = k.shape[2]
    t = q.dtype
    u, tiny = torch.finfo(t).eps / 2, (2.0 ** -25 if t == torch.float16 else 0.0)
    qm = torch.arange(Sq, device=DEV) < (q_lens if q_lens is not None else torch.full((B,), Sq, device=DEV)).clamp(0, Sq)[:, None]
    km = torch.arange(Sk, device=DEV) < (k_lens if k_lens is not None else torch.full((B,), Sk, device=DEV)).clamp(0, Sk)[:, None]
    zero = lambda x, m: torch.where(m[:, None, :, None], x.double(), 0.0)  # noqa: E731
    q, do, k, v = zero(q, qm), zero(do, qm), zero(k, km), zero(v, km)
    seen = qm[:, None, :, None] & km[:, None, None, :]
    s = torch.where(seen, c * (q @ k.transpose(2, 3)), -math.inf)
    lse = torch.logsumexp(s, 3)
    p = torch.where(seen, torch.exp(s - lse[..., None]), 0.0)
    out = p @ v
    dp = do @ v.transpose(2, 3)
    D = (do * out).sum(3, keepdim=True)
    one = km.sum(1).eq(1)[:, None, None, None]
    ds = torch.where(one, 0.0, p * (dp - D))
    dq, dk, dv = c * (ds @ k), c * (ds.transpose(2, 3) @ q), p.transpose(2, 3) @ do
    qa, ka, va, da = q.abs(), k.abs(), v.abs(), do.abs()
    e = 4 * 128 * W * c * (qa @ ka.transpose(2, 3)).amax(3, keepdim=True) + 2.0 ** -20
    r = lambda x: u * x.abs() * (1 + 2 * u) + tiny  # the rounding of a result
    b_out = r(out) + (1 + u) * ((u + e + Sk * W) * (p @ va) + tiny * va.sum(2, keepdim=True))
    b_D = (da * b_out).sum(3, keepdim=True) + 128 * W * (da * out.abs()).sum(3, keepdim=True)
    if one_tile:
        # D as D' + sum_j p (dp - D') for a D' that is at most u |do||out| away: the errors of p (e), of dp (128 w) and of the
        # fp32 arithmetic (2^-18 covers 128 additions)
        b_D = (p * ((e + 2.0 ** -18) * (dp.abs() + 2 * D.abs()) + 128 * W * (da @ va.transpose(2, 3)))).sum(3, keepdim=True)
        b_D = b_D + (e + 2.0 ** -18) * (D.abs() + (da * out.abs()).sum(3, keepdim=True) * 2 * u)
    b_ds = torch.where(seen, (u + e) * ds.abs() + p * (128 * W * (da @ va.transpose(2, 3)) + b_D) * (1 + u) + tiny, 0.0)
    b_ds = torch.where(one, 0.0, b_ds)
    # dq is summed as r k - (sum of r) m with the rounded ds r and m the mean of the first (up to 128) keys; the exact ds of a
    # row add up to zero, so an error of ds counts with its key's distance from m
    first = (km & (torch.arange(Sk, device=DEV) < 128))[:, None, :, None].double()
    m = (k * first).sum(2, keepdim=True) / first.sum(2, keepdim=True).clamp_min(1)
    b_dq = r(dq) + (1 + u) * c * (b_ds @ torch.where(km[:, None, :, None], (k - m).abs(), 0.0) + (Sk + 300) * W * (ds.abs() @ (ka + m.abs())))
    b_dk = r(dk) + (1 + u) * c * (b_ds.transpose(2, 3) @ qa + Sq * W * (ds.abs().transpose(2, 3) @ qa))
    b_dv = r(dv) + (1 + u) * (((u + e + Sq * W) * p + tiny * seen).transpose(2, 3) @ da)
    b_lse = e[..., 0] + 2.0 ** -21 * (lse.abs().nan_to_num(posinf=0) + 1)
    return (out, lse, dq, dk, dv), (b_out, b_lse, b_dq, b_dk, b_dv)


def check(got, want, bound):
    for name, a, w, b in zip(("out", "lse", "dq", "dk", "dv"), got, want, bound):
        a = a.double()
        assert torch.equal(torch.isneginf(a), torch.isneginf(w)), name
        off = torch.where(torch.isneginf(w), 0.0, a - w).abs()
        bad = ~(off <= b)
        assert not bad.any(), f"{name}: {int(bad.sum())} elements, worst {float((off / b.clamp_min(1e-300)).max()):.3g} of the bound"


def run(ops, q, k, v, do, **kw):
    out, lse = ops.attention_lse(q, k, v, **kw)
    return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, **kw))


CASES = [  # B, H, Sq, Sk, dtype
    (1, 1, 128, 128, "bf16"), (1, 1, 1, 1, "bf16"), (1, 2, 1, 2, "f16"), (2, 3, 5, 3, "bf16"), (1, 1, 127, 129, "bf16"), (1, 2, 129, 127, "f16"),
    (2, 2, 256, 256, "bf16"), (1, 3, 257, 300, "f16"), (1, 1, 640, 1, "bf16"), (1, 1, 1, 900, "f16"), (1, 2, 1000, 77, "bf16"), (3, 1, 384, 513, "bf16"),
    (1, 4, 700, 700, "f16"), (1, 1, 3000, 200, "bf16"), (1, 1, 200, 3000, "bf16"), (1, 40, 130, 140, "bf16"), (1, 1, 9, 5000, "bf16"), (1, 1, 5000, 9, "f16"),
    (1, 160, 140, 260, "bf16"),
]


@pytest.mark.parametrize("B,H,Sq,Sk,dtype", CASES)
def test_attention_and_gradients(ops, B, H, Sq, Sk, dtype):
    q, k, v, do = make(B, H, Sq, Sk, dtype, seed=Sq + Sk)
    check(run(ops, q, k, v, do), *reference(q, k, v, do, None, None, 1 / math.sqrt(128)))


LENS = [  # B, H, Sq, Sk, dtype, q_lens, k_lens
    (2, 2, 200, 300, "bf16", None, [300, 1]), (3, 1, 130, 260, "f16", None, [0, 128, 129]), (3, 2, 300, 300, "bf16", [300, 0, 131], [300, 0, 131]),
    (2, 1, 513, 140, "bf16", [1, 512], None), (4, 1, 1, 70, "f16", [1, 0, 1, 1], [70, 70, 0, 33]), (2, 1, 40, 2000, "bf16", [39, 40], [1999, 130]),
    (2, 1, 2000, 40, "f16", [1, 1999], [40, 17]), (2, 1, 260, 260, "bf16", [-5, 9999], [9999, -1]), (2, 3, 384, 384, "bf16", [256, 128], [128, 256]),
    (1, 1, 700, 300, "bf16", [0], [300]), (1, 1, 300, 1500, "bf16", [300], [0]),
]


@pytest.mark.parametrize("B,H,Sq,Sk,dtype,q_lens,k_lens", LENS)
@pytest.mark.parametrize("fill", [None, math.nan, math.inf])
def test_padded_batches(ops, B, H, Sq, Sk, dtype, q_lens, k_lens, fill):
    """Tokens behind the lengths take no part, whatever they hold."""
    q, k, v, do = make(B, H, Sq, Sk, dtype, seed=Sk)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q_lens, k_lens = i32(q_lens), i32(k_lens)
    if fill is not None:
        for t, lens in ((q, q_lens), (do, q_lens), (k, k_lens), (v, k_lens)):
            if lens is not None:
                for b, n in enumerate(lens.clamp(0, t.shape[2]).tolist()):
                    t[b, :, n:] = fill
    check(run(ops, q, k, v, do, q_lens=q_lens, k_lens=k_lens), *reference(q, k, v, do, q_lens, k_lens, 1 / math.sqrt(128)))


@pytest.mark.parametrize("scale", [1e-3, 0.5])
def test_softmax_scale_and_peaked_rows(ops, scale):
    q, k, v, do = make(1, 2, 300, 400, "bf16", seed=3, offset=0.0)
    check(run(ops, q, k, v, do, sm_scale=scale), *reference(q, k, v, do, None, None, scale))


def test_keys_far_from_zero(ops):
    """An offset that all keys share has no part in dq; neither have the roundings of ds times that offset."""
    q, k, v, do = make(1, 3, 300, 500, "bf16", seed=13, offset=20.0)
    check(run(ops, q, k, v, do), *reference(q, k, v, do, None, None, 1 / math.sqrt(128)))


def test_rising_maxima(ops):
    """Scores that grow along the keys: every tile moves the running maximum by more than the rescaling threshold."""
    q, k, v, do = make(1, 1, 256, 1024, "bf16", seed=4, offset=0.0)
    q, k = q.abs(), (k.abs() * torch.linspace(0.1, 3, 1024, device=DEV)[:, None]).bfloat16()
    check(run(ops, q, k, v, do), *reference(q, k, v, do, None, None, 1 / math.sqrt(128)))


def test_layouts_and_gradients_of_any_layout(ops):
    """Head-major memory, heads inside a wider projection, every second token, a broadcast gradient, an unaligned slice."""
    B, H, S = 2, 3, 200
    q, k, v, do = make(B, H, S, S, "bf16", seed=5)
    want = run(ops, q, k, v, do)
    layouts = [lambda t: t.contiguous(), lambda t: torch.cat([t, t], 1)[:, :H], lambda t: torch.stack([t, t], 3).flatten(2, 3)[:, :, ::2],
               lambda t: torch.cat([t[..., :3], t], 3)[..., 3:], lambda t: t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)]
    for f in layouts:
        got = run(ops, f(q), f(k), f(v), f(do))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    one = torch.ones((), device=DEV, dtype=torch.bfloat16).expand(B, H, S, 128)
    a, b = run(ops, q, k, v, one), run(ops, q, k, v, one.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # keys and values that the samples share
    ks, vs = k[:1].expand(B, H, S, 128), v[:1].expand(B, H, S, 128)
    a, b = run(ops, q, ks, vs, do), run(ops, q, ks.contiguous(), vs.contiguous(), do)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_offsets_beyond_32_bits(ops):
    """Tokens that lie more than 2^32 bytes apart in one buffer."""
    S, stride = 300, 1 << 23
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    q, k, v, do = make(1, 1, S, S, "bf16", seed=6)
    buf = torch.empty(S * stride, dtype=torch.bfloat16, device=DEV)
    far = [torch.as_strided(buf, (1, 1, S, 128), (S * stride, S * stride, stride, 1), 128 * i) for i in range(4)]
    for f, t in zip(far, (q, k, v, do)):
        f.copy_(t)
    got, want = run(ops, *far), run(ops, q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shape", [(2, 3, 300, 500), (1, 1, 100, 4000), (1, 1, 4000, 100)])
def test_equal_inputs_give_equal_bits_on_any_stream(ops, shape):
    q, k, v, do = make(*shape, "bf16", seed=7)
    want = run(ops, q, k, v, do)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run(ops, q, k, v, do))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))


def test_captured_and_replayed_on_new_inputs(ops):
    """Two captured graphs, replayed alternately: their workspaces are their own, lengths are read at replay."""
    sets = [make(2, 2, 200, 700, "bf16", seed=s) for s in (8, 9)]
    lens = torch.tensor([700, 300], dtype=torch.int32, device=DEV)
    static = [[t.clone() for t in x] for x in sets]
    graphs, outs = [], []
    for st in static:
        run(ops, *st, k_lens=lens)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(ops, *st, k_lens=lens))
        graphs.append(g)
    lens.copy_(torch.tensor([129, 650], dtype=torch.int32))
    fresh = [make(2, 2, 200, 700, "bf16", seed=s) for s in (10, 11)]
    for st, new in zip(static, fresh):
        for a, b in zip(st, new):
            a.copy_(b)
    for g in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    for o, new in zip(outs, fresh):
        assert all(torch.equal(a, b) for a, b in zip(o, run(ops, *new, k_lens=lens)))


def test_gradient_against_differences(ops):
    """Central differences of the 64-bit loss along random directions, within the bounds of the gradients."""
    q, k, v, do = make(1, 1, 40, 60, "bf16", seed=12)
    got = run(ops, q, k, v, do)[2:]
    _, bound = reference(q, k, v, do, None, None, 1 / math.sqrt(128))
    x = [t.double() for t in (q, k, v)]

    def loss(q, k, v):
        return ((torch.softmax(q @ k.transpose(2, 3) / math.sqrt(128), 3) @ v) * do.double()).sum()

    g = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64).to(DEV)
        h = 1e-4
        up, down = [list(x) for _ in range(2)]
        up[i], down[i] = x[i] + h * d, x[i] - h * d
        diff = (loss(*up) - loss(*down)) / (2 * h)
        along = (got[i].double() * d).sum()
        # the difference quotient of a smooth loss is off by h^2 of its third derivative: 1e-5 of its size is ample
        assert (along - diff).abs() <= (bound[2 + i] * d.abs()).sum() + 1e-5 * (got[i].double() * d).abs().sum()


def test_empty_axes(ops):
    q, k, v, do = make(2, 2, 30, 40, "bf16")
    out, lse = ops.attention_lse(q, k[:, :, :0], v[:, :, :0])
    assert not out.any() and torch.isneginf(lse).all()
    dq, dk, dv = ops.attention_backward(do, q, k[:, :, :0], v[:, :, :0], out, lse)
    assert not dq.any() and dk.shape == dv.shape == (2, 2, 0, 128)
    out, lse = ops.attention_lse(q[:, :, :0], k, v)
    _, dk, dv = ops.attention_backward(do[:, :, :0], q[:, :, :0], k, v, out, lse)
    assert out.shape[2] == 0 and not dk.any() and not dv.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [None, [1, 1], [0, 1]])
def test_one_key_and_many_queries(ops, dtype, lens):
    """The queries are split over CTAs: the joined gradients through the scores are zero, that of the value is not."""
    q, k, v, do = make(2, 1, 6000, 1 if lens is None else 3, dtype, seed=14)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    check(run(ops, q, k, v, do, k_lens=lens), *reference(q, k, v, do, None, lens, 1 / math.sqrt(128)))


@pytest.mark.parametrize("rows", [128, 2000])
def test_fp16_probabilities_of_long_rows(ops, rows):
    """Equal probabilities of 1 / 225,000, 74.6 steps of the smallest fp16 numbers: they are rounded as normal numbers."""
    S = 225000
    g = torch.Generator(device=DEV).manual_seed(15)
    q = torch.zeros(1, 1, rows, 128, dtype=torch.float16, device=DEV)
    k, v = (torch.randn(1, 1, S, 128, generator=g, device=DEV).half() for _ in range(2))
    do = (64 * torch.rand(1, 1, rows, 128, generator=g, device=DEV)).half()
    dv = run(ops, q, k, v, do)[4].double()
    want = do.double().sum(2, keepdim=True) / S
    # the rounding of p, its exponential and that of lse (log 225,000 = 12.3: 2^-21), the additions, the rounding of the result
    bound = want * (2.0 ** -11 + 2.0 ** -20 + 2.0 ** -20 + rows * W) * (1 + 2.0 ** -10) + want * 2.0 ** -11 + 2.0 ** -25
    assert bool(((dv - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,Sq,Sk,k_lens", [(1, 2, 300, 2, None), (2, 1, 8, 8, None), (1, 1, 50, 128, None), (3, 2, 200, 300, [2, 128, 1]),
                                              (2, 1, 100, 3000, [5, 64]), (1, 1, 5000, 16, None)])
def test_few_keys_do_not_feel_the_rounding_of_out(ops, B, H, Sq, Sk, k_lens, dtype):
    q, k, v, do = make(B, H, Sq, Sk, dtype, seed=16)
    lens = None if k_lens is None else torch.tensor(k_lens, dtype=torch.int32, device=DEV)
    check(run(ops, q, k, v, do, k_lens=lens), *reference(q, k, v, do, None, lens, 1 / math.sqrt(128), one_tile=True))
