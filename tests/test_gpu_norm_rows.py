"""LayerNorm + modulation and RMSNorm + rotary embedding, what the tests of single launches leave open: rows that share a CTA with
others, many row groups per CTA, values that are not finite, frozen parameters."""
import pytest
import torch

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
