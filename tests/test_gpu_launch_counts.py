"""The launch accounting against the kernel nodes of a captured graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops(built_library):
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    from dax_b200 import ops as _ops
    return _ops


def kernels_of(fn):
    """Kernel nodes of a capture of ``fn`` (copies of inputs would be among them: the tensors here need none)."""
    from cuda.bindings import runtime
    fn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        fn()
    raw = graph.raw_cuda_graph()
    err, _, n = runtime.cudaGraphGetNodes(raw)
    assert int(err) == 0
    err, nodes, n = runtime.cudaGraphGetNodes(raw, n)
    assert int(err) == 0
    kinds = [runtime.cudaGraphNodeGetType(node)[1] for node in nodes[:n]]
    return sum(k == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds)


def counted(ops, fn):
    before = ops.TRACE.launches
    fn()
    return ops.TRACE.launches - before


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("B,H,Sq,Sk", [(1, 40, 256, 256), (1, 1, 8, 30000), (1, 1, 30000, 8), (1, 2, 2000, 2000), (1, 1, 1, 1)])
def test_attention(ops, B, H, Sq, Sk, keys, dtype):
    q, do = (torch.randn(B, H, Sq, 128, device=DEV).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, H, Sk, 128, device=DEV).to(dtype) for _ in range(2))
    out, lse = ops.attention_lse(q, k, v)
    for fn in (lambda: ops.attention_lse(q, k, v), lambda: ops.attention_backward(do, q, k, v, out, lse, need_keys=keys)):
        assert counted(ops, fn) == kernels_of(fn)


@pytest.mark.parametrize("S", [40, 0])
def test_norms(ops, S):
    x = torch.randn(2, S, 256, device=DEV)
    w, scale = torch.ones(256, device=DEV), torch.ones(2, 256, device=DEV)
    _, mean, rstd = ops.layernorm_modulate(x)
    for fn in (lambda: ops.layernorm_modulate(x, shift=scale, scale=scale), lambda: ops.rmsnorm_rope(x, w),
               lambda: ops.layernorm_modulate_backward(x, x, mean, rstd, ln_weight=w, scale=scale),
               lambda: ops.layernorm_modulate_backward(x, x, mean, rstd, ln_weight=w, scale=scale, need_params=False),
               lambda: ops.layernorm_modulate_backward(x, x, mean, rstd),
               lambda: ops.rmsnorm_rope_backward(x, x, rstd, w), lambda: ops.rmsnorm_rope_backward(x, x, rstd, w, need_params=False)):
        assert counted(ops, fn) == kernels_of(fn)
