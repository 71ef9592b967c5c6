"""What the C entry points of linear attention, of the query / key norms and of sampling refuse, by status and
message (no GPU needed: a refused call launches nothing), and the wrappers on CPU tensors."""
import ctypes as ct

import pytest
import torch

from hybrid_model_mamba_xlstm_b200 import _lib, kernels

ENTRIES = [(_lib.LinearAttnArgs, "hxm_linear_attn_fwd"), (_lib.LinearAttnBwdArgs, "hxm_linear_attn_bwd"),
           (_lib.LinearAttnStepArgs, "hxm_linear_attn_step"), (_lib.QkNormRopeArgs, "hxm_qk_norm_rope_fwd"),
           (_lib.QkNormRopeBwdArgs, "hxm_qk_norm_rope_bwd"), (_lib.SampleArgs, "hxm_sample_tokens")]


def call(fn, a):
    a.struct_size = ct.sizeof(a)
    if hasattr(a, "fwd"):
        a.fwd.struct_size = ct.sizeof(a.fwd)
    status = getattr(_lib.lib(), fn)(ct.byref(a), None)
    return status, _lib.lib().hxm_last_error_string().decode()


@pytest.mark.parametrize("cls,fn", ENTRIES)
def test_struct_sizes_and_null(cls, fn):
    assert getattr(_lib.lib(), fn)(None, None) == _lib.HXM_EBADARG
    a = cls()
    a.struct_size = ct.sizeof(a) + 8
    assert getattr(_lib.lib(), fn)(ct.byref(a), None) == _lib.HXM_EBADARG
    assert b"struct_size" in _lib.lib().hxm_last_error_string()


def attn(**kw):
    a = _lib.LinearAttnArgs()
    a.batch, a.seqlen, a.heads, a.dk, a.dv, a.io_dtype, a.scale = 1, 4, 2, 8, 8, _lib.HXM_F32, 1.0
    for n, x in kw.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("bad,status,text", [
    (dict(batch=-1), "HXM_EBADARG", "bad dims"), (dict(dk=0), "HXM_EBADARG", "bad dims"), (dict(dv=0), "HXM_EBADARG", "bad dims"),
    (dict(io_dtype=_lib.HXM_F16), "HXM_EBADARG", "io_dtype"), (dict(dk=520), "HXM_EUNSUPPORTED", "at most 512"),
    (dict(heads=70000), "HXM_EUNSUPPORTED", "at most"), (dict(batch=30000), "HXM_EUNSUPPORTED", "at most"),
    (dict(seqlen=2 ** 30 + 1), "HXM_EUNSUPPORTED", "2^30"), (dict(scale=0.0), "HXM_EBADARG", "scale"),
    (dict(scale=float("inf")), "HXM_EBADARG", "scale"), (dict(scale=float("nan")), "HXM_EBADARG", "scale"),
    (dict(), "HXM_EBADARG", "NULL tensor")])
def test_linear_attn(bad, status, text):
    got, said = call("hxm_linear_attn_fwd", attn(**bad))
    assert got == getattr(_lib, status) and text in said
    b = _lib.LinearAttnBwdArgs()
    b.fwd = attn(**bad)
    got, said = call("hxm_linear_attn_bwd", b)
    assert got == getattr(_lib, status) and text in said


def test_linear_attn_gradients_of_wide_values_and_without_workspace():
    b = _lib.LinearAttnBwdArgs()
    b.fwd = attn(dv=513)
    got, said = call("hxm_linear_attn_bwd", b)
    assert got == _lib.HXM_EUNSUPPORTED and "at most 512" in said
    # one head over a long time is cut into segments, whose states the caller has to lend
    f = attn(seqlen=100000, heads=1)
    for n in ("q", "k", "v", "out", "log_decay"):
        setattr(f, n, 1 << 20)
    f.struct_size = ct.sizeof(f)
    assert _lib.lib().hxm_linear_attn_workspace_size(f) > 0
    got, said = call("hxm_linear_attn_fwd", f)  # refused before the addresses are used
    assert got == _lib.HXM_EBADARG and "workspace" in said


@pytest.mark.parametrize("bad,status,text", [
    (dict(batch=-1), "HXM_EBADARG", "bad dims"), (dict(dk=0), "HXM_EBADARG", "bad dims"), (dict(io_dtype=9), "HXM_EBADARG", "io_dtype"),
    (dict(batch=70000), "HXM_EUNSUPPORTED", "65535"), (dict(), "HXM_EBADARG", "NULL tensor")])
def test_linear_attn_step(bad, status, text):
    a = _lib.LinearAttnStepArgs()
    a.batch, a.heads, a.dk, a.dv, a.io_dtype, a.scale = 1, 2, 8, 8, _lib.HXM_F32, 1.0
    for n, x in bad.items():
        setattr(a, n, x)
    got, said = call("hxm_linear_attn_step", a)
    assert got == getattr(_lib, status) and text in said


@pytest.mark.parametrize("bad,status,text", [
    (dict(seqlen=-1), "HXM_EBADARG", "bad dims"), (dict(dim=0), "HXM_EBADARG", "bad dims"), (dict(io_dtype=9), "HXM_EBADARG", "io_dtype"),
    (dict(dim=1025), "HXM_EUNSUPPORTED", "at most 1024"), (dict(rotary=3), "HXM_EBADARG", "rotary"),
    (dict(rotary=66), "HXM_EBADARG", "rotary"), (dict(rotary=-2), "HXM_EBADARG", "rotary"),
    (dict(rotary=4, rope_base=0.0), "HXM_EBADARG", "rope_base"), (dict(rotary=4, rope_base=float("inf")), "HXM_EBADARG", "rope_base"),
    (dict(heads_q=2 ** 20, heads_k=1), "HXM_EUNSUPPORTED", "heads"), (dict(), "HXM_EBADARG", "NULL")])
def test_qk_norm_rope(bad, status, text):
    def args():
        a = _lib.QkNormRopeArgs()
        a.batch, a.seqlen, a.heads_q, a.heads_k, a.dim, a.io_dtype, a.rope_base, a.eps = 1, 2, 2, 1, 64, _lib.HXM_F32, 1e4, 1e-6
        for n, x in bad.items():
            setattr(a, n, x)
        return a
    got, said = call("hxm_qk_norm_rope_fwd", args())
    assert got == getattr(_lib, status) and text in said
    b = _lib.QkNormRopeBwdArgs()
    b.fwd = args()
    got, said = call("hxm_qk_norm_rope_bwd", b)
    assert got == getattr(_lib, status) and text in said


@pytest.mark.parametrize("bad,status,text", [
    (dict(rows=-1), "HXM_EBADARG", "bad dims"), (dict(vocab=0), "HXM_EBADARG", "bad dims"), (dict(io_dtype=9), "HXM_EBADARG", "io_dtype"),
    (dict(vocab=2 ** 18 + 1), "HXM_EUNSUPPORTED", "at most"), (dict(rows=2 ** 27 + 1), "HXM_EUNSUPPORTED", "rows"),
    (dict(), "HXM_EBADARG", "NULL tensor")])
def test_sample(bad, status, text):
    a = _lib.SampleArgs()
    a.rows, a.vocab, a.io_dtype = 2, 10, _lib.HXM_F32
    for n, x in bad.items():
        setattr(a, n, x)
    got, said = call("hxm_sample_tokens", a)
    assert got == getattr(_lib, status) and text in said


def test_empty_calls_launch_nothing():
    assert call("hxm_linear_attn_fwd", attn(batch=0))[0] == _lib.HXM_OK
    a = _lib.LinearAttnStepArgs()
    a.batch, a.heads, a.dk, a.dv, a.io_dtype, a.scale = 0, 2, 8, 8, _lib.HXM_F32, 1.0
    assert call("hxm_linear_attn_step", a)[0] == _lib.HXM_OK
    s = _lib.SampleArgs()
    s.rows, s.vocab, s.io_dtype = 0, 10, _lib.HXM_F32
    assert call("hxm_sample_tokens", s)[0] == _lib.HXM_OK


def test_wrappers_on_cpu_tensors():
    x, ld = torch.zeros(1, 4, 2, 8), torch.zeros(2)
    for go in (lambda: kernels.linear_attention(x, x, x, ld),
               lambda: kernels.linear_attention(x.clone().requires_grad_(), x, x, ld),
               lambda: kernels.linear_attention_bwd(x, x, x, ld, x),
               lambda: kernels.linear_attention_step(x[0], x[0], x[0], ld, torch.zeros(4, 2, 8, 8)),
               lambda: kernels.qk_norm_rope(x, x),
               lambda: kernels.qk_norm_rope_bwd(x, x, None, None, x, x),
               lambda: kernels.sample_tokens(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA device"):
            go()


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_norms_eps(eps):
    a = _lib.QkNormRopeArgs()
    a.batch, a.seqlen, a.heads_q, a.heads_k, a.dim, a.io_dtype, a.rope_base, a.eps = 1, 2, 2, 1, 64, _lib.HXM_F32, 1e4, eps
    got, said = call("hxm_qk_norm_rope_fwd", a)
    assert got == _lib.HXM_EBADARG and "eps" in said
    b = _lib.QkNormRopeBwdArgs()
    b.fwd = a
    got, said = call("hxm_qk_norm_rope_bwd", b)
    assert got == _lib.HXM_EBADARG and "eps" in said


def test_forward_mode_is_refused():
    """A tangent would be lost silently: none of the operators has forward-mode derivatives."""
    x, ld = torch.zeros(1, 4, 2, 8), torch.zeros(2)
    calls = [lambda t: kernels.linear_attention(t, x, x, ld), lambda t: kernels.linear_attention(x, x, t, ld),
             lambda t: kernels.linear_attention(x, x, x, ld, initial_state=t.new_zeros(1, 2, 8, 8) + t[0, 0, 0, 0]),
             lambda t: kernels.linear_attention(x, x, x, t[0, 0, :, 0]),
             lambda t: kernels.linear_attention_step(x[0], t[0], x[0], ld, torch.zeros(4, 2, 8, 8)),
             lambda t: kernels.qk_norm_rope(t, x), lambda t: kernels.qk_norm_rope(x, x, None, t[0, 0, 0]),
             lambda t: kernels.linear_attention_bwd(x, x, x, ld, t), lambda t: kernels.qk_norm_rope_bwd(x, x, None, None, x, t)]
    for go in calls:
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                go(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
            with pytest.raises(RuntimeError, match="CUDA device"):  # no tangent: as ever
                go(x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: go(t), (x,), (torch.ones_like(x),))


def test_linear_attn_workspace_off_its_alignment():
    """The segments' sums are read in 16-byte pieces: such a workspace would be a misaligned access."""
    f = attn(seqlen=100000, heads=1)
    for n in ("q", "k", "v", "out", "log_decay"):
        setattr(f, n, 1 << 20)
    f.struct_size = ct.sizeof(f)
    f.workspace_bytes = _lib.lib().hxm_linear_attn_workspace_size(f)
    f.workspace = (1 << 20) + 4
    got, said = call("hxm_linear_attn_fwd", f)  # refused before the addresses are used
    assert got == _lib.HXM_EBADARG and "16-byte aligned" in said


@pytest.mark.parametrize("scale", [1e-39, -1e-39, 2e38])
def test_linear_attn_scales_without_a_reciprocal(scale):
    got, said = call("hxm_linear_attn_fwd", attn(scale=scale))
    assert got == _lib.HXM_EBADARG and "scale" in said
    with pytest.raises(ValueError, match="scale"):
        kernels.linear_attention(torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(2), scale=scale)
