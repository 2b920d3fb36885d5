"""The training operators together: as differentiable functions, chained through Wan blocks, captured into a graph."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ag(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import autograd as _ag
    return _ag


@pytest.fixture(autouse=True)
def device_status_clean():
    yield
    from dax_b200 import _lib
    assert _lib.device_status() == 0, "a kernel reported a timed-out wait"


class PlainProcessor:
    """The same block with elementary torch operations, in whatever type the model has."""

    def __call__(self, attn, x, encoder_hidden_states=None, attention_mask=None, rotary_emb=None):
        ctx = x if encoder_hidden_states is None else encoder_hidden_states
        heads = lambda t: t.unflatten(2, (attn.heads, 128)).transpose(1, 2)  # noqa: E731

        def norm(t, n):
            w = t if t.dtype == torch.float64 else t.float()
            y = w * torch.rsqrt(w.pow(2).mean(-1, keepdim=True) + n.eps) * n.weight.to(w.dtype)
            if rotary_emb is not None:
                r = rotary_emb.reshape(1, -1, 1, 64)
                c, s = r.real.to(w.dtype), r.imag.to(w.dtype)
                a, b = y.unflatten(2, (-1, 64, 2)).unbind(4)
                y = torch.stack((a * c - b * s, a * s + b * c), 4).flatten(2)
            return y.to(t.dtype)

        q, k, v = heads(norm(attn.to_q(x), attn.norm_q)), heads(norm(attn.to_k(ctx), attn.norm_k)), heads(attn.to_v(ctx))
        p = torch.softmax((q @ k.transpose(2, 3)) / math.sqrt(128), 3)
        return attn.to_out[1](attn.to_out[0]((p @ v).transpose(1, 2).flatten(2)))


def _plain_block(self, h, ctx, temb, rotary_emb):
    f = (lambda t: t) if h.dtype == torch.float64 else (lambda t: t.float())
    sm, cm, gm, cs, cc, cg = (f(self.scale_shift_table) + f(temb)).chunk(6, dim=1)
    ln = lambda t, n: F.layer_norm(f(t), n.normalized_shape, None if n.weight is None else f(n.weight), None if n.bias is None else f(n.bias), n.eps)  # noqa: E731
    h = (f(h) + f(self.attn1((ln(h, self.norm1) * (1 + cm) + sm).type_as(h), rotary_emb=rotary_emb)) * gm).type_as(h)
    h = h + self.attn2(ln(h, self.norm2).type_as(h), encoder_hidden_states=ctx)
    n = (ln(h, self.norm3) * (1 + cc) + cs).type_as(h)
    return (f(h) + f(self.ffn(n)) * cg).type_as(h)


def _blocks(dim=512, heads=4, layers=2):
    from dax_b200.adapters.wan.modules import WanTransformerBlock
    torch.manual_seed(0)
    net = torch.nn.ModuleList([WanTransformerBlock(dim, 2 * dim, heads) for _ in range(layers)])
    with torch.no_grad():
        for n, p in net.named_parameters():
            if "norm" in n and n.endswith("weight"):
                p.add_(0.1 * torch.randn(p.shape))
    return net


def _step(net, x, ctx, temb, rope, dy):
    params = dict(net.named_parameters())
    h = x.detach().requires_grad_()
    y = h
    for b in net:
        y = b(y, ctx, temb, rope)
    grads = torch.autograd.grad(y, [h, *params.values()], dy.to(y.dtype))
    return {"y": y.detach(), **dict(zip(["x", *params], grads))}


def test_training_block_is_as_exact_as_the_plain_composition(ag):
    """Two Wan blocks, batch of two: outputs and all gradients against 64 bits.  The kernels round where the plain bf16
    composition rounds, or less often, so each result has to be within 1.5 times that composition's error (roundings are
    independent; the norm of a few thousand of them does not move by a tenth), plus two units of rounding for results whose
    plain error is smaller than one."""
    import types
    from dax_b200.adapters.wan.modules import _Pipe, wan_rope_table
    from dax_b200.adapters.wan.training import enable_training
    net = _blocks()
    grid = (2, 8, 16)
    S, D = 256, 512
    g = torch.Generator().manual_seed(1)
    x, ctx, temb, dy = torch.randn(2, S, D, generator=g), torch.randn(2, 77, D, generator=g), torch.randn(2, 6, D, generator=g) * 0.3, torch.randn(2, S, D, generator=g)
    rope = wan_rope_table(grid, device=DEV)
    net = net.bfloat16()
    args = [t.bfloat16().to(DEV) for t in (x, ctx, temb)]
    results = []
    for kind in ("exact", "plain", "kernels"):
        m = copy.deepcopy(net).to(DEV)
        if kind == "exact":
            m = m.double()
        if kind == "kernels":
            assert enable_training(_Pipe(m)) == 2
        else:
            for b in m:
                b.attn1.processor = b.attn2.processor = PlainProcessor()
                b.forward = types.MethodType(_plain_block, b)
        a = [t.double() for t in args] if kind == "exact" else args
        results.append(_step(m, *a, rope, dy.bfloat16().to(DEV)))
    exact, plain, own = results
    for n in exact:
        norm = exact[n].norm()
        e_plain, e_own = ((r[n].double() - exact[n]).norm() / norm for r in (plain, own))
        assert e_own <= 1.5 * e_plain + 2 * 2.0 ** -9, (n, float(e_plain), float(e_own))


def test_context_lengths_and_refusals(ag):
    from dax_b200.adapters.wan.modules import Attention, _Pipe
    from dax_b200.adapters.wan.training import DAXWanTrainingAttnProcessor, enable_training
    from dax_b200.adapters.wan.transformer_adapter import quantize_transformer
    torch.manual_seed(2)
    attn = Attention(256, 2, processor=DAXWanTrainingAttnProcessor()).bfloat16().to(DEV)
    x, ctx = torch.randn(2, 130, 256, device=DEV).bfloat16(), torch.randn(2, 64, 256, device=DEV).bfloat16()
    lens = torch.tensor([64, 20], dtype=torch.int32, device=DEV)
    ctx_nan = ctx.clone()
    ctx_nan[1, 20:] = float("nan")
    proc = attn.processor
    a = proc(attn, x, encoder_hidden_states=ctx_nan, context_lens=lens)
    one = proc(attn, x[1:], encoder_hidden_states=ctx[1:, :20].contiguous())
    assert torch.equal(a[1:], one) and torch.isfinite(a.float()).all()
    with pytest.raises(NotImplementedError):
        proc(attn, x, encoder_hidden_states=ctx, attention_mask=lens)
    with pytest.raises(ValueError):
        proc(attn, x, context_lens=lens)
    net = _blocks(layers=1).bfloat16().to(DEV)
    quantize_transformer(net, "int8")
    with pytest.raises(NotImplementedError):
        enable_training(_Pipe(net))


def test_shapes_of_modulation_and_types_of_parameters(ag):
    """[D], [B, D], [B, 1, D] and a row for all samples; bf16 parameters get bf16 gradients, summed in fp32."""
    torch.manual_seed(3)
    x = torch.randn(3, 50, 384, device=DEV).bfloat16().requires_grad_()
    full = torch.randn(3, 384, device=DEV)
    dy = torch.randn(3, 50, 384, device=DEV).bfloat16()
    ref = None
    for shape in ((3, 384), (3, 1, 384)):
        s = full.clone().reshape(shape).requires_grad_()
        y = ag.layernorm_modulate(x, shift=s, scale=s * 2)
        gx, gs = torch.autograd.grad(y, (x, s), dy)
        assert gs.shape == shape
        if ref is not None:
            assert torch.equal(ref[0], gx) and torch.equal(ref[1], gs.reshape(3, 384))
        ref = (gx, gs.reshape(3, 384))
    row = full[0].clone().requires_grad_()
    per_sample = full[:1].expand(3, 384).clone().requires_grad_()
    g_row = torch.autograd.grad(ag.layernorm_modulate(x, shift=row, scale=row), row, dy)[0]
    g_each = torch.autograd.grad(ag.layernorm_modulate(x, shift=per_sample, scale=per_sample), per_sample, dy)[0]
    assert (g_row - g_each.sum(0)).abs().max() <= 8 * 2.0 ** -24 * g_each.abs().sum(0).max()
    w = torch.ones(384, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    g = torch.autograd.grad(ag.layernorm_modulate(x, ln_weight=w, ln_bias=w), w, dy)[0]
    assert g.dtype == torch.bfloat16 and g.shape == w.shape
    g = torch.autograd.grad(ag.rmsnorm_rope(x, w), w, dy)[0]
    assert g.dtype == torch.bfloat16
    x2 = x[0].detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ag.rmsnorm_rope(x2, w), x2, dy[0])[0], torch.autograd.grad(ag.rmsnorm_rope(x, w), x, dy)[0][0])


def test_shared_keys_get_the_sum_of_their_gradients(ag):
    """One context for a whole batch (expand): autograd adds the samples' gradients."""
    torch.manual_seed(4)
    q = torch.randn(3, 2, 140, 128, device=DEV).bfloat16().requires_grad_()
    k = torch.randn(1, 2, 50, 128, device=DEV).bfloat16().requires_grad_()
    v = torch.randn(1, 2, 50, 128, device=DEV).bfloat16().requires_grad_()
    do = torch.randn(3, 2, 140, 128, device=DEV).bfloat16()
    shared = torch.autograd.grad(ag.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)), (q, k, v), do)
    ke, ve = k.detach().repeat(3, 1, 1, 1).requires_grad_(), v.detach().repeat(3, 1, 1, 1).requires_grad_()
    each = torch.autograd.grad(ag.attention(q, ke, ve), (q, ke, ve), do)
    assert torch.equal(shared[0], each[0])
    for a, b in zip(shared[1:], each[1:]):
        assert torch.equal(a, b.sum(0, keepdim=True))


def test_frozen_parameters_and_second_derivatives(ag):
    x = torch.randn(2, 40, 256, device=DEV).bfloat16().requires_grad_()
    w = torch.ones(256, device=DEV)
    y = ag.layernorm_modulate(x, ln_weight=w)
    g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), x)


def test_training_step_captured_into_a_graph(ag):
    """Forward and backward of a block in one CUDA graph, replayed on new inputs."""
    from dax_b200.adapters.wan.modules import _Pipe, wan_rope_table
    from dax_b200.adapters.wan.training import enable_training
    net = _blocks(layers=1).bfloat16().to(DEV)
    enable_training(_Pipe(net))
    rope = wan_rope_table((2, 8, 16), device=DEV)
    gen = torch.Generator().manual_seed(5)
    make = lambda: [torch.randn(s, generator=gen).bfloat16().to(DEV) for s in ((2, 256, 512), (2, 77, 512), (2, 6, 512), (2, 256, 512))]  # noqa: E731
    static = make()

    def step(t):
        return _step(net, t[0], t[1], t[2], rope, t[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for _ in range(2):
        fresh = make()
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(fresh)
        for n in eager:
            assert torch.equal(captured[n], eager[n]), n


def test_whole_model_trains(ag):
    """Loss and gradients of a small DiT through the public calls; the criterion is that of the blocks' test, for gradients
    that have enough elements for it (4,096).  The others exist and are finite."""
    import types
    from dax_b200.adapters.wan.modules import WanDiT, _Pipe
    from dax_b200.adapters.wan.training import enable_training
    torch.manual_seed(3)
    net = WanDiT(layers=2, dim=256, ffn_dim=512, heads=2, text_dim=64, freq_dim=64).bfloat16()
    latents, target = (torch.randn(2, 16, 2, 8, 16).bfloat16().to(DEV) for _ in range(2))
    text, timestep = torch.randn(2, 20, 64).bfloat16().to(DEV), torch.tensor([900.0, 100.0], device=DEV)
    grads = []
    for kind in ("exact", "plain", "kernels"):
        m = copy.deepcopy(net).to(DEV)
        t = (lambda x: x.double()) if kind == "exact" else (lambda x: x)  # noqa: E731
        if kind == "exact":
            m = m.double()
        if kind == "kernels":
            assert enable_training(_Pipe(m)) == 2
        else:
            for b in m.blocks:
                b.attn1.processor = b.attn2.processor = PlainProcessor()
                b.forward = types.MethodType(_plain_block, b)
        out = m(t(latents), timestep, t(text))[0]
        (out - t(target)).square().mean().backward()
        grads.append({n: p.grad for n, p in m.named_parameters()})
    exact, plain, own = grads
    for n in exact:
        assert own[n] is not None and torch.isfinite(own[n]).all(), n
        if exact[n].numel() >= 4096:
            e_plain, e_own = ((r[n].double() - exact[n]).norm() / exact[n].norm() for r in (plain, own))
            assert e_own <= 1.5 * e_plain + 2 * 2.0 ** -9, (n, float(e_plain), float(e_own))


def test_captured_step_follows_its_rotary_table(ag):
    """The table is an input like the others: a graph captured after a warm-up step reads what it holds at the replay, and
    nothing that other tables' steps put in its place."""
    from dax_b200.adapters.wan import attn_adapter
    from dax_b200.adapters.wan.modules import _Pipe, wan_rope_table
    from dax_b200.adapters.wan.training import enable_training
    net = _blocks(layers=1).bfloat16().to(DEV)
    enable_training(_Pipe(net))
    torch.manual_seed(6)
    args = [torch.randn(s).bfloat16().to(DEV) for s in ((2, 256, 512), (2, 77, 512), (2, 6, 512))]
    dy = torch.randn(2, 256, 512).bfloat16().to(DEV)
    tables = [wan_rope_table((2, 8, 16), device=DEV).roll(i, 2) for i in range(6)]
    rope = tables[0].clone()
    cached = len(attn_adapter._ROPE_CACHE)

    def step(r):
        return _step(net, *args, r, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(rope)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(rope)
    for t in tables[1:]:
        want = step(t)
        rope.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(captured[n], want[n]), n
    assert len(attn_adapter._ROPE_CACHE) == cached


@pytest.mark.parametrize("shape", [(2, 3, 300, 500), (1, 1, 5000, 60), (1, 1, 40, 4000)])
def test_frozen_keys_and_values_cost_nothing(ag, monkeypatch, shape):
    """LoRA on self-attention alone leaves the keys and values of cross-attention without a gradient: theirs is not computed,
    that of the queries has the same bits."""
    from dax_b200 import ops
    B, H, Sq, Sk = shape
    torch.manual_seed(7)
    q, do = (torch.randn(B, H, Sq, 128, device=DEV).bfloat16() for _ in range(2))
    k, v = (torch.randn(B, H, Sk, 128, device=DEV).bfloat16() for _ in range(2))
    got = []
    backward = ops.attention_backward
    monkeypatch.setattr(ops, "attention_backward", lambda *a, **kw: got.append(backward(*a, **kw)) or got[-1])
    for t in (q, k, v):
        t.requires_grad_()
    dq, dk, dv = torch.autograd.grad(ag.attention(q, k, v), (q, k, v), do)
    only_q, = torch.autograd.grad(ag.attention(q, k.detach(), v.detach()), q, do)
    only_v, = torch.autograd.grad(ag.attention(q.detach(), k.detach(), v), v, do)
    assert torch.equal(only_q, dq) and torch.equal(only_v, dv)
    assert [r[1] is None and r[2] is None for r in got] == [False, True, False]
    assert ops.attention_backward(do[:, :, :0], q[:, :, :0], k, v, do[:, :, :0], torch.empty(B, H, 0, device=DEV), need_keys=False)[1:] == (None, None)
