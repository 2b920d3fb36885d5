"""fp16 attention over the range of fp16 training: gradients far below one, long rows, dominant keys.

p and ds are much smaller than what they are made from (by the number of keys), and fp16 loses digits below 2^-14.  The
tolerances here are on the norm of an error and not elementwise: the bound on every element that all roundings fall the same way
is a hundred times what happens and would hide lost digits.  u = 2^-11 is the largest relative error of a rounding; roundings
are independent, so squares add; taking u for each (a uniform rounding has u / sqrt(3)) leaves a factor of 1.7 above
the expected norm, which the norm of ten thousand errors does not reach.  Results below 2^-14 are rounded to steps of 2^-24 by
their type: half a step absolutely, 2^-25."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U, HALF_STEP = 2.0 ** -11, 2.0 ** -25
W = 2.0 ** -23  # an addition in the tensor cores' fp32 sums


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


def run(ops, q, k, v, do, **kw):
    out, lse = ops.attention_lse(q, k, v, **kw)
    return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, **kw))


def exact_gradients(q, k, v, do, c):
    """One head ``[S, 128]`` in 64 bits: dq, dk, and for each the expected square of the error's norm (for dq by rows).

    dq_i = c sum_j ds_ij (k_j - m), m the mean of the first 128 keys (what the common part of the keys adds is zero): errors
    u ds_ij, and D_i off by the rounding of out and of the forward pass's p, which comes back as sum_j p_ij (k_j - m).
    dk_j = c sum_i ds_ij q_i: errors u ds_ij and p_ij times that of D_i.  The sums themselves are fp32: their errors, at most w
    of the running sum each, add up to less than sqrt(terms) w of sum |ds| |k|."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    km = k - k[:128].mean(0)
    kn, dk, dk_e = km.square().sum(1), torch.zeros_like(k), torch.zeros(k.shape[0], dtype=torch.float64, device=DEV)
    dq, dq_e = torch.zeros_like(q), torch.zeros(q.shape[0], dtype=torch.float64, device=DEV)
    for i in range(0, q.shape[0], 2048):
        r = slice(i, i + 2048)
        p = torch.softmax(c * (q[r] @ k.T), 1)
        out = p @ v
        dp = do[r] @ v.T
        ds = p * (dp - (do[r] * out).sum(1, keepdim=True))
        d_err = U * U * ((do[r] * out).square().sum(1) + p.square() @ v.square() @ torch.ones(128, dtype=torch.float64, device=DEV) * do[r].square().sum(1))
        dq[r] = c * (ds @ km)
        dk += c * (ds.T @ q[r])
        qn = q[r].square().sum(1)
        sq = ds.square()
        dq_e[r] = c * c * (U * U * (sq @ kn) + d_err * (p @ km).square().sum(1) + k.shape[0] * W * W * (ds.abs() @ km.abs()).square().sum(1))
        dk_e += c * c * (U * U * (sq.T @ qn) + p.square().T @ (d_err * qn) + q.shape[0] * W * W * (ds.abs().T @ q[r].abs()).square().sum(1))
    dq_e += U * U * dq.square().sum(1) + 128 * HALF_STEP ** 2
    return dq, dk, dq_e, dk_e.sum() + U * U * dk.square().sum() + dk.numel() * HALF_STEP ** 2


def close(got, want, square):
    off = float((got.double() - want).norm())
    assert off <= float(square) ** 0.5, f"error {off / float(want.norm()):.3g} of the norm, {off / float(square) ** 0.5:.3g} of the bound"


def draw(Sq, Sk, q_std, do_std, seed=0, v_std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = lambda S, std: (torch.randn(1, 1, S, 128, generator=g, device=DEV) * std).half()  # noqa: E731
    return t(Sq, q_std), t(Sk, 1 / q_std), t(Sk, v_std), t(Sq, do_std)


@pytest.mark.parametrize("Sq,Sk", [(700, 4095), (300, 32760), (2500, 32760), (5000, 700)])
@pytest.mark.parametrize("do_std", [1e-1, 1e-2, 1e-3])
@pytest.mark.parametrize("q_std", [0.25, 4.0])
def test_small_gradients_keep_their_digits(ops, Sq, Sk, do_std, q_std):
    """Scores of unit spread; q and k of different sizes bring dq (q_std 0.25) or dk (4) into the normal range."""
    q, k, v, do = draw(Sq, Sk, q_std, do_std)
    _, _, dq, dk, _ = run(ops, q, k, v, do)
    w_dq, w_dk, e_dq, e_dk = exact_gradients(q[0, 0], k[0, 0], v[0, 0], do[0, 0], 1 / math.sqrt(128))
    close(dq[0, 0], w_dq, e_dq.sum())
    close(dk[0, 0], w_dk, e_dk)


@pytest.mark.parametrize("Sq,Sk", [(300, 20000), (5000, 128), (600, 600)])
def test_rows_of_very_different_gradients(ops, Sq, Sk):
    """Output gradients from 1e-4 to 1e2 row by row: each row of dq is as exact as if it were alone."""
    q, k, v, do = draw(Sq, Sk, 0.25, 1.0, seed=1)
    do = (do.float() * torch.logspace(-4, 2, 7, device=DEV)[torch.arange(Sq, device=DEV) % 7, None]).half()
    _, _, dq, dk, _ = run(ops, q, k, v, do)
    w_dq, w_dk, e_dq, e_dk = exact_gradients(q[0, 0], k[0, 0], v[0, 0], do[0, 0], 1 / math.sqrt(128))
    for i in range(7):
        close(dq[0, 0, i::7], w_dq[i::7], e_dq[i::7].sum())
    close(dk[0, 0], w_dk, e_dk)


@pytest.mark.parametrize("Sq,Sk", [(300, 500), (200, 9), (2000, 64), (64, 4000)])
def test_large_gradients_of_the_scores(ops, Sq, Sk):
    """dp of a million: ds is far outside fp16, dq and dk are inside."""
    q, k, v, do = draw(Sq, Sk, 1.0, 300.0, seed=2, v_std=300.0)
    q, k = (q.float() / 32).half(), (k.float() / 32).half()
    _, _, dq, dk, _ = run(ops, q, k, v, do)
    w_dq, w_dk, e_dq, e_dk = exact_gradients(q[0, 0], k[0, 0], v[0, 0], do[0, 0], 1 / math.sqrt(128))
    assert w_dq.abs().max() < 65504 and w_dk.abs().max() < 65504
    close(dq[0, 0], w_dq, e_dq.sum())
    close(dk[0, 0], w_dk, e_dk)


@pytest.mark.parametrize("shape", [(2, 3, 300, 500), (1, 2, 5000, 70), (2, 1, 40, 9000)])
def test_factors_go_by_tokens_that_exist(ops, shape):
    """What lies behind the lengths has no say in the factors either, whatever it holds; empty samples and zero gradients."""
    B, H, Sq, Sk = shape
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, do = ((torch.randn(B, H, S, 128, generator=g, device=DEV) * s).half() for S, s in ((Sq, 0.25), (Sk, 4.0), (Sk, 1.0), (Sq, 1e-3)))
    ql, kl = ([Sq - 3] + [0] * (B - 1)), ([Sk - 5] + [Sk] * (B - 1))
    q_lens, k_lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ql, kl))
    want = run(ops, q[:1, :, :ql[0]], k[:1, :, :kl[0]], v[:1, :, :kl[0]], do[:1, :, :ql[0]])[2:]
    for fill in (0.0, 60000.0, math.inf, math.nan):
        for t, n in ((q, ql), (do, ql), (k, kl), (v, kl)):
            for b in range(B):
                t[b, :, n[b]:] = fill
        got = run(ops, q, k, v, do, q_lens=q_lens, k_lens=k_lens)[2:]
        for a, w, n in zip(got, want, (ql, kl, kl)):
            # other splits of the long axis may add in another order: fp32 sums, then one rounding
            assert ((a[:1, :, :n[0]].double() - w.double()).norm() <= U * w.double().norm() + w.numel() ** 0.5 * HALF_STEP)
            assert not a[:1, :, n[0]:].any() and not a[1:].any()
    zero = run(ops, q[:1, :, :ql[0]], k[:1, :, :kl[0]], v[:1, :, :kl[0]], torch.zeros_like(do[:1, :, :ql[0]]))[2:]
    assert not any(t.any() for t in zero)


def test_infinite_gradients_stay_in_their_rows_of_dq(ops):
    q, k, v, do = draw(200, 300, 1.0, 1e-2, seed=4)
    want = run(ops, q, k, v, do)[2]
    do[0, 0, 17, 5] = math.inf
    dq, dk = run(ops, q, k, v, do)[2:4]
    keep = torch.arange(200, device=DEV) != 17
    assert torch.equal(dq[0, 0, keep], want[0, 0, keep]) and not torch.isfinite(dq[0, 0, 17].float()).any()
    assert not torch.isfinite(dk.float()).all()


@pytest.mark.parametrize("gap", [10, 17, 21, 25])
@pytest.mark.parametrize("at", [0, 700, 1999])
@pytest.mark.parametrize("rows", [3, 5000])
def test_keys_far_below_the_largest_score(ops, gap, at, rows):
    """One key whose score is `gap` powers of two above all others and whose value is zero: the output is what the others add.
    Their p are 2^-gap of the largest, and rounded as normal numbers down to 2^-25 of it (u).  The offset
    of some keys and the rounding of k put them up to 2^0.03 lower (u times 1.03).  One product per score, so scores are exact
    but for the fp32 arithmetic of the exponent (2^-19); sums of S positive terms; the result's rounding."""
    S, c = 2000, 1 / math.sqrt(128)
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k = torch.zeros(1, 1, rows, 128, device=DEV), torch.zeros(1, 1, S, 128, device=DEV)
    q[..., 0], k[0, 0, at, 0] = 8.0, gap * math.log(2) / (8 * c)
    k[0, 0, :at, 0] = -0.01  # no two maxima in a row are the same
    v = 32 + 32 * torch.rand(1, 1, S, 128, generator=g, device=DEV)
    v[0, 0, at] = 0
    q, k, v = q.half(), k.half(), v.half()
    out, lse = ops.attention_lse(q, k, v)
    s = c * 8 * k[0, 0, :, 0].double()
    p = torch.softmax(s, 0)
    want = p @ v[0, 0].double()
    bound = (1.03 * U + 2.0 ** -19 + S * W) * want * (1 + U) + U * want + HALF_STEP
    assert bool(((out[0, 0].double() - want).abs() <= bound).all()), float(((out[0, 0].double() - want).abs() / want).max())
    assert bool(((lse.double() - torch.logsumexp(s, 0)).abs() <= 2.0 ** -18).all())


@pytest.mark.parametrize("step", [1.9, 3.9, 4.1, 7.9, 8.1, 30.0])
def test_maxima_that_rise_tile_by_tile(ops, step):
    """Every tile of 128 keys is `step` powers of two above the last: p stays inside fp16 whether the running maximum follows
    or not."""
    S, rows, c = 1024, 300, 1 / math.sqrt(128)
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k = torch.zeros(1, 1, rows, 128, device=DEV), torch.zeros(1, 1, S, 128, device=DEV)
    q[..., 0], k[0, 0, :, 0] = 8.0, (torch.arange(S, device=DEV) // 128) * (step * math.log(2) / (8 * c))
    v = 1 + torch.rand(1, 1, S, 128, generator=g, device=DEV)
    q, k, v = q.half(), k.half(), v.half()
    out, lse = ops.attention_lse(q, k, v)
    s = c * 8 * k[0, 0, :, 0].double()
    want = torch.softmax(s, 0) @ v[0, 0].double()
    # scores reach 7 * step * ln 2: the exponent's argument is off by 2^-24 of that, the rest as above
    err = U + 2.0 ** -19 + 2.0 ** -23 * 7 * step + S * W
    assert bool(((out[0, 0].double() - want).abs() <= (err * (1 + U) + U) * want).all())
    assert bool(((lse.double() - torch.logsumexp(s, 0)).abs() <= 2.0 ** -18 + 2.0 ** -22 * 7 * step).all())


def test_layouts_and_far_offsets(ops):
    """The largest norms are found through the tensors' own strides: heads inside a wider projection, every second token, tokens
    more than 2^32 bytes apart."""
    B, H, S, far = 2, 3, 300, 1 << 22
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v, do = ((torch.randn(B, S, H, 128, generator=g, device=DEV) * s).half().transpose(1, 2) for s in (1.0, 1.0, 1.0, 1e-3))
    v[1, 2, 250] *= 30
    want = run(ops, q, k, v, do)
    for f in (lambda t: t.contiguous(), lambda t: torch.cat([1000 * t, t], 1)[:, H:], lambda t: torch.stack([t, 1000 * t], 3).flatten(2, 3)[:, :, ::2]):
        assert all(torch.equal(a, b) for a, b in zip(run(ops, f(q), f(k), f(v), f(do)), want))
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    buf = torch.full((2 * S * far,), 1000.0, dtype=torch.float16, device=DEV)
    views = [torch.as_strided(buf, (B, H, S, 128), (S * far, 512, far, 1), 128 * i) for i in range(4)]
    for t, x in zip(views, (q, k, v, do)):
        t.copy_(x)
    assert all(torch.equal(a, b) for a, b in zip(run(ops, *views), want))


@pytest.mark.parametrize("shape", [(2, 2, 200, 700), (1, 1, 40, 4000), (1, 1, 4000, 40)])
def test_captured_factors_follow_the_inputs(ops, shape):
    """Two graphs replayed in turn on inputs a thousand times larger and smaller than those of the capture: the bits of eager calls."""
    B, H, Sq, Sk = shape
    g = torch.Generator(device=DEV).manual_seed(8)
    make = lambda s: [(torch.randn(B, H, S, 128, generator=g, device=DEV) * f).half() for S, f in ((Sq, 1.0), (Sk, 1.0), (Sk, s), (Sq, s))]  # noqa: E731
    static, graphs, outs = [make(0.1), make(3.0)], [], []
    for st in static:
        run(ops, *st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(ops, *st))
        graphs.append(graph)
    for s in (1e-3, 100.0):
        fresh = [make(s), make(s)]
        for st, new in zip(static, fresh):
            for a, b in zip(st, new):
                a.copy_(b)
        for graph in graphs + graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o, new in zip(outs, fresh):
            assert all(torch.equal(a, b) for a, b in zip(o, run(ops, *new)))


def test_equal_inputs_give_equal_bits_on_any_stream(ops):
    for shape in ((300, 500), (100, 4000), (4000, 100)):
        q, k, v, do = draw(*shape, 1.0, 1e-2, seed=9)
        want = run(ops, q, k, v, do)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for _ in range(3):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(run(ops, q, k, v, do))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
