"""Refusals of the training operators, before anything is launched: CPU only."""
import ctypes

import pytest
import torch

from dax_b200 import _lib

I64x3 = ctypes.c_int64 * 3


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


ONE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def _fwd(lib, dtype=_lib.DAX_BF16, B=1, H=2, Sq=300, Sk=300, q=ONE, strides=(76800, 128, 256), scale=0.1, lse=ONE, ws=None, n=0):
    s = I64x3(*strides)
    return lib.dax_attn_forward_lse(q, ONE, ONE, dtype, B, H, Sq, Sk, s, s, s, scale, None, None, ONE, s, lse, ws, n, None)


def test_attention_forward_refusals(lib):
    assert _fwd(lib, B=0) == _lib.DAX_ERR_INVALID and b"bad shape" in lib.dax_last_error()
    assert _fwd(lib, dtype=_lib.DAX_F32) == _lib.DAX_ERR_UNSUPPORTED
    assert _fwd(lib, B=300, H=300) == _lib.DAX_ERR_UNSUPPORTED
    assert _fwd(lib, q=None) == _lib.DAX_ERR_INVALID
    assert _fwd(lib, q=ctypes.c_void_p(4104)) == _lib.DAX_ERR_ALIGN
    assert _fwd(lib, strides=(76800, 128, 252)) == _lib.DAX_ERR_ALIGN
    assert _fwd(lib, strides=(76800, 128, -256)) == _lib.DAX_ERR_INVALID
    assert _fwd(lib, lse=None) == _lib.DAX_ERR_INVALID
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _fwd(lib, scale=scale) == _lib.DAX_ERR_INVALID and b"softmax scale" in lib.dax_last_error()
    # few rows against many keys run split and need a workspace
    need = lib.dax_attn_lse_workspace_bytes(1, 1, 8, 30000)
    assert need > 0 and lib.dax_attn_lse_workspace_bytes(1, 40, 32760, 32760) == 0
    assert _fwd(lib, H=1, Sq=8, Sk=30000, ws=ONE, n=need - 1) == _lib.DAX_ERR_INVALID and b"workspace" in lib.dax_last_error()
    assert _fwd(lib, H=1, Sq=8, Sk=30000, ws=ctypes.c_void_p(4100), n=need) == _lib.DAX_ERR_ALIGN


def test_attention_backward_refusals(lib):
    s = I64x3(76800, 128, 256)
    need = lib.dax_attn_backward_workspace_bytes(1, 2, 300, 300)
    assert need >= 2 * 384 * 8

    def call(ws=ONE, n=need, dq=ONE, lse=ONE, dtype=_lib.DAX_F16, scale=0.1):
        return lib.dax_attn_backward(ONE, ONE, ONE, ONE, ONE, lse, dtype, 1, 2, 300, 300, s, s, s, s, s, scale, None, None, dq, ONE, ONE, s,
                                     s, s, ws, n, None)

    assert call(n=need - 1) == _lib.DAX_ERR_INVALID and b"workspace" in lib.dax_last_error()
    assert call(ws=None) == _lib.DAX_ERR_INVALID
    assert call(dq=ctypes.c_void_p(4100)) == _lib.DAX_ERR_ALIGN
    assert call(lse=None) == _lib.DAX_ERR_INVALID
    assert call(dtype=_lib.DAX_I8) == _lib.DAX_ERR_UNSUPPORTED
    assert call(scale=-1.0) == _lib.DAX_ERR_INVALID


def test_norm_refusals(lib):
    f32 = ctypes.c_float(1e-6)

    def ln(D=512, x=ONE, ss=512, w=None, c=None, shift=None, scale=None, B=1, S=4, dtype=_lib.DAX_BF16, mean=ONE):
        return lib.dax_layernorm_modulate(x, dtype, B, S, D, 4 * 512, ss, w, c, shift, scale, f32, ONE, 2048, 512, mean, ONE, None)

    assert ln(D=510) == _lib.DAX_ERR_UNSUPPORTED and ln(D=8200) == _lib.DAX_ERR_UNSUPPORTED and ln(D=0) == _lib.DAX_ERR_INVALID
    assert ln(dtype=_lib.DAX_E4M3) == _lib.DAX_ERR_UNSUPPORTED and ln(B=70000) == _lib.DAX_ERR_UNSUPPORTED
    assert ln(x=None) == _lib.DAX_ERR_INVALID and ln(mean=None) == _lib.DAX_ERR_INVALID
    assert ln(x=ctypes.c_void_p(4100)) == _lib.DAX_ERR_ALIGN and ln(ss=513) == _lib.DAX_ERR_ALIGN and ln(w=ctypes.c_void_p(4100)) == _lib.DAX_ERR_ALIGN
    assert ln(c=ONE) == _lib.DAX_ERR_INVALID and ln(shift=ONE) == _lib.DAX_ERR_INVALID and ln(scale=ONE) == _lib.DAX_ERR_INVALID
    assert ln(S=0) == _lib.DAX_OK

    def ln_b(dscale=None, ws=None, n=0):
        return lib.dax_layernorm_modulate_backward(ONE, ONE, _lib.DAX_BF16, 1, 64, 512, 0, 512, 0, 512, ONE, ONE, None, None, ONE, ONE, 0, 512, None,
                                                   None, None, dscale, ws, n, None)

    need = lib.dax_norm_backward_workspace_bytes(1, 64, 512)
    assert need > 0 and ln_b(dscale=ONE, ws=ONE, n=need // 4) == _lib.DAX_ERR_INVALID and b"workspace" in lib.dax_last_error()
    assert ln_b(dscale=ONE, ws=ctypes.c_void_p(4100), n=need) == _lib.DAX_ERR_ALIGN

    def rms(D=256, cos=None, sin=None):
        return lib.dax_rmsnorm_rope(ONE, _lib.DAX_BF16, 1, 4, D, 0, 256, None, cos, sin, f32, ONE, 0, 256, ONE, None)

    assert rms(cos=ONE) == _lib.DAX_ERR_INVALID and rms(D=200, cos=ONE, sin=ONE) == _lib.DAX_ERR_INVALID


def test_wrappers_refuse_wrong_tensors():
    """Shapes and types are looked at before the device: CPU tensors reach these refusals; right ones are told there is no
    CPU path."""
    from dax_b200 import ops
    q, k = torch.zeros(1, 2, 8, 128).bfloat16(), torch.zeros(1, 2, 9, 128).bfloat16()
    for bad in ((q[..., :64], k, k), (q, k[:, :1], k[:, :1]), (q, k, k[:, :, :4]), (q[0], k, k)):
        with pytest.raises(ValueError):
            ops.attention_lse(*bad)
    for bad in ((q.float(), k.float(), k.float()), (q, k.half(), k)):
        with pytest.raises(NotImplementedError):
            ops.attention_lse(*bad)
    for lens in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            ops.attention_lse(q, k, k, k_lens=lens)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            ops.attention_lse(q, k, k, sm_scale=scale)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attention_lse(q, k, k)
    lse = torch.zeros(1, 2, 8)
    for bad in (dict(dout=q[:, :, :4]), dict(dout=q.half()), dict(lse=lse[:, :1]), dict(lse=lse.double())):
        with pytest.raises(ValueError):
            ops.attention_backward(**{**dict(dout=q, q=q, k=k, v=k, out=q, lse=lse), **bad})
    x = torch.zeros(2, 3, 256).bfloat16()
    with pytest.raises(NotImplementedError):
        ops.layernorm_modulate(x.double())
    for kw in (dict(ln_weight=torch.zeros(255)), dict(ln_weight=torch.zeros(256).double()), dict(shift=torch.zeros(256), scale=torch.zeros(256))):
        with pytest.raises(ValueError):
            ops.layernorm_modulate(x, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layernorm_modulate(x)
    st = torch.zeros(2, 3)
    for bad in (dict(dy=x[:1]), dict(dy=x.half()), dict(mean=st[:1]), dict(rstd=st.double())):
        with pytest.raises(ValueError):
            ops.layernorm_modulate_backward(**{**dict(dy=x, x=x, mean=st, rstd=st), **bad})
    t = torch.zeros(3, 64)
    for kw in (dict(rope_cos=t), dict(rope_cos=t[:2], rope_sin=t[:2]), dict(rope_cos=t.double(), rope_sin=t), dict(rope_cos=t[:, :32], rope_sin=t)):
        with pytest.raises(ValueError):
            ops.rmsnorm_rope(x, **kw)
    with pytest.raises(ValueError):
        ops.rmsnorm_rope(x[..., :200], rope_cos=t, rope_sin=t)
    with pytest.raises(ValueError):
        ops.rmsnorm_rope(x[0, 0])


def test_an_optimised_pipe_is_not_trained():
    """Its forward ends in a quantising operator: gradients would stop there without a word."""
    from dax_b200.adapters.wan.modules import WanDiT, _Pipe
    from dax_b200.adapters.wan.training import enable_training
    from dax_b200.adapters.wan.transformer_adapter import replace_transformer
    net = WanDiT(layers=1, dim=128, ffn_dim=128, heads=1, text_dim=32, freq_dim=32)
    assert enable_training(_Pipe(net)) == 1
    replace_transformer(net)
    with pytest.raises(NotImplementedError, match="inference forward"):
        enable_training(_Pipe(net))


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_training_keeps_no_rotary_tables(dtype):
    """Tables are made for each call, on the stream of the call: a cache knows neither streams nor captured graphs."""
    from dax_b200.adapters.wan import attn_adapter, training
    before = dict(attn_adapter._ROPE_CACHE)
    ang = torch.rand(1, 1, 20, 64, dtype=torch.float64)
    table = torch.polar(torch.ones_like(ang), ang).to(dtype)
    for _ in range(2):
        cos, sin = training._rotary_tables(table)
        assert cos.dtype == sin.dtype == torch.float32 and cos.shape == sin.shape == (20, 64) and cos.is_contiguous() and sin.is_contiguous()
        assert torch.equal(cos, table[0, 0].real.float()) and torch.equal(sin, table[0, 0].imag.float())
        again = training._rotary_tables(table)
        assert again[0].data_ptr() != cos.data_ptr() and again[1].data_ptr() != sin.data_ptr()
        table.conj_physical_()
    assert attn_adapter._ROPE_CACHE.keys() == before.keys()


def test_attention_gradients_of_keys_and_values_come_together(lib):
    s = I64x3(76800, 128, 256)
    n = lib.dax_attn_backward_workspace_bytes(1, 2, 300, 300)

    def call(dk, dv, ws):
        return lib.dax_attn_backward(ONE, ONE, ONE, ONE, ONE, ONE, _lib.DAX_BF16, 1, 2, 300, 300, s, s, s, s, s, 0.1, None, None, ONE, dk, dv, s,
                                     s, s, ws, n, None)

    assert call(ONE, None, ONE) == _lib.DAX_ERR_INVALID and b"dv is null" in lib.dax_last_error()
    assert call(None, ONE, ONE) == _lib.DAX_ERR_INVALID and b"dk is null" in lib.dax_last_error()
    # neither is wanted: the next check is the workspace's
    assert call(None, None, None) == _lib.DAX_ERR_INVALID and b"workspace" in lib.dax_last_error()


@pytest.mark.parametrize("kw", [{}, {"int8_linear": True}, {"fuse_blocks": False}])
def test_a_pipe_in_training_is_not_optimised(kw):
    """The inference processors and forwards would replace the differentiable ones without a word; nothing is changed."""
    from dax_b200.adapters.wan import enable_training, optimize_pipe, quantize_transformer
    from dax_b200.adapters.wan.modules import WanDiT, _Pipe
    net = WanDiT(layers=1, dim=128, ffn_dim=128, heads=1, text_dim=32, freq_dim=32)
    pipe = _Pipe(net)
    assert enable_training(pipe) == 1
    before = (net.forward.__func__, net.blocks[0].forward.__func__, type(net.blocks[0].attn1.processor), type(net.blocks[0].ffn.net[2]))
    with pytest.raises(NotImplementedError, match="training"):
        optimize_pipe(pipe, sequence_parallel=False, overlap_comm=False, compile=False, **kw)
    with pytest.raises(NotImplementedError, match="training"):
        quantize_transformer(net, "int8")
    assert before == (net.forward.__func__, net.blocks[0].forward.__func__, type(net.blocks[0].attn1.processor), type(net.blocks[0].ffn.net[2]))
    assert enable_training(pipe) == 1  # again is fine
