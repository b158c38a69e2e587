"""The typed operators' refusals that need no GPU: the C entry points check every
argument before they touch the device, and the Python ones refuse CPU tensors."""
import ctypes

import pytest
import torch

from sgnn_amd import _hip, functional, muon

INVALID = _hip.SGNN_ERR_INVALID
P = 256   # a non-null pointer that no refused call reads


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


def _linear(lib, dtype=0, M=4, N=4, K=4, x=P, ldx=4, w=P, ldw=4, act=0, res=None, ldr=4, y=P, ldy=4, nws=1 << 30):
    return lib.sgnn_linear(dtype, M, N, K, x, ldx, w, ldw, None, act, res, ldr, None, y, ldy, P, nws, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(act=5), dict(act=-1), dict(M=-1), dict(N=-1), dict(K=-1), dict(x=None),
    dict(w=None), dict(y=None), dict(ldx=3), dict(ldw=3), dict(ldy=3), dict(res=P, ldr=3)])
def test_linear_refuses(lib, bad):
    assert _linear(lib, **bad) == INVALID
    assert "linear" in lib.sgnn_last_error().decode()


@pytest.mark.parametrize("big", [dict(M=(1 << 30) + 1), dict(N=(1 << 25) + 1), dict(K=(1 << 25) + 1)])
def test_linear_refuses_more_than_a_launch_holds(lib, big):
    far = dict(ldx=1 << 40, ldw=1 << 40)
    assert _linear(lib, **far, ldy=1 << 40, nws=1 << 62, **big) == _hip.SGNN_ERR_UNSUPPORTED
    assert _linear_bwd(lib, **far, ldd=1 << 40, nws=1 << 62, **big) == _hip.SGNN_ERR_UNSUPPORTED


def test_empty_calls_need_no_device(lib):
    assert _linear(lib, M=0) == _hip.SGNN_OK and _linear(lib, N=0) == _hip.SGNN_OK
    assert lib.sgnn_norm(0, 0, None, 4, 0, 4, None, None, None, 4, 1e-5, None, None, None, None) == _hip.SGNN_OK
    assert lib.sgnn_newton_schulz(0, None, 0, 5, 1.0, 0.0, 0.0, 0.0, None, 0, None) == _hip.SGNN_OK
    empty = (_hip.SgnnMatrix * 1)(_hip.SgnnMatrix(None, None, 0, 0, 0, 7))
    assert lib.sgnn_newton_schulz_workspace_bytes(empty, 1) == 0
    assert lib.sgnn_newton_schulz(0, empty, 1, 5, 1.0, 0.0, 0.0, 0.0, None, 0, None) == _hip.SGNN_OK


def _linear_bwd(lib, dtype=0, M=4, N=4, K=4, dy=P, ldd=4, slope=P, x=P, ldx=4, w=P, ldw=4, dx=P, dw=P, db=P,
                nws=1 << 30, ws=P):
    return lib.sgnn_linear_bwd(dtype, M, N, K, dy, ldd, slope, x, ldx, w, ldw, dx, dw, db, ws, nws, None)


@pytest.mark.parametrize("bad", [
    dict(dtype=7), dict(M=-1), dict(dy=None), dict(ldd=3), dict(x=None), dict(ldx=3),
    dict(w=None), dict(ldw=3), dict(nws=0), dict(ws=None)])
def test_linear_bwd_refuses(lib, bad):
    assert _linear_bwd(lib, **bad) == INVALID
    assert "linear_bwd" in lib.sgnn_last_error().decode()


def test_linear_bwd_workspace_of_slopes_of_0_and_1(lib):
    """SGNN_SLOPES_01: one plane of dz instead of two for the 16-bit types, nothing else; no other bit passes."""
    size = lambda dtype: lib.sgnn_linear_bwd_workspace_bytes(dtype, 1000, 512, 64, 1)
    for dtype in (1, 2):
        assert size(dtype) - size(dtype | 0x100) == 1000 * 512 * 2
    assert size(0) == size(0x100) > 0 and size(1 | 0x200) == 0
    assert _linear_bwd(lib, dtype=1 | 0x200) == INVALID and _linear_bwd(lib, dtype=3 | 0x100) == INVALID


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("M", [0, 4])
@pytest.mark.parametrize("slope", [None, P])
def test_linear_bwd_without_outputs(lib, dtype, M, slope):
    """N = 0: dw and db have no elements, and without dx there is nothing to launch."""
    assert lib.sgnn_linear_bwd_workspace_bytes(dtype, M, 0, 4, int(slope is not None)) == 0
    assert _linear_bwd(lib, dtype=dtype, M=M, N=0, dy=None, slope=slope, dx=None, ws=None, nws=0) == _hip.SGNN_OK


@pytest.mark.parametrize("bad", [
    dict(dtype=5), dict(dtype=1, wdtype=2), dict(n=-1), dict(width=0), dict(x=None), dict(y=None), dict(ldx=3),
    dict(res=P, ldr=3), dict(eps=-1.0), dict(eps=float("nan"))])
def test_norm_refuses(lib, bad):
    a = dict(dtype=0, wdtype=0, n=4, width=4, x=P, ldx=4, y=P, res=None, ldr=4, eps=1e-5)
    a.update(bad)
    if "wdtype" not in bad:
        a["wdtype"] = a["dtype"]
    assert lib.sgnn_norm(a["dtype"], a["wdtype"], a["x"], a["ldx"], a["n"], a["width"], None, None, a["res"],
                         a["ldr"], a["eps"], a["y"], None, None, None) == INVALID
    assert "norm" in lib.sgnn_last_error().decode()


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(n=-1), dict(width=0), dict(dy=None), dict(x=None), dict(mean=None),
                                 dict(rstd=None), dict(ldd=3), dict(ldx=3), dict(nws=0)])
def test_norm_bwd_refuses(lib, bad):
    a = dict(dtype=0, n=4, width=4, dy=P, ldd=4, x=P, ldx=4, mean=P, rstd=P, nws=1 << 20)
    a.update(bad)
    assert lib.sgnn_norm_bwd(a["dtype"], a["dtype"], a["dy"], a["ldd"], a["x"], a["ldx"], a["mean"], a["rstd"], None,
                             a["n"], a["width"], P, P, P, P, a["nws"], None) == INVALID
    assert "norm_bwd" in lib.sgnn_last_error().decode()


@pytest.mark.parametrize("bad", [dict(dtype=4), dict(count=-1), dict(steps=-1), dict(eps=-1.0), dict(null=True),
                                 dict(rows=-1), dict(ld=3), dict(in_=None), dict(nws=0), dict(ws=None)])
def test_newton_schulz_refuses(lib, bad):
    a = dict(dtype=0, count=1, steps=5, eps=0.0, null=False, rows=4, ld=4, in_=P, nws=1 << 30, ws=P)
    a.update(bad)
    cols = 4 if a["nws"] == 1 << 30 and a["ws"] else 400   # 4 x 4 needs no workspace
    a["rows"] = 400 if cols == 400 else a["rows"]
    mats = (_hip.SgnnMatrix * 1)(_hip.SgnnMatrix(a["in_"], P, max(a["ld"], cols) if cols == 400 else a["ld"], cols, a["rows"], cols))
    assert lib.sgnn_newton_schulz(a["dtype"], None if a["null"] else mats, a["count"], a["steps"], 1.0, 0.0, 0.0,
                                  a["eps"], a["ws"], a["nws"], None) == INVALID
    assert "newton_schulz" in lib.sgnn_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the matrices' addresses are none of a device")
@pytest.mark.parametrize("empty", [(0, 7), (7, 0), (0, 0)])
def test_newton_schulz_goes_on_behind_an_empty_matrix(lib, empty):
    """Without a device every call that has work ends in a launch error; one that skips its matrices reports success."""
    def status(shapes):
        mats = (_hip.SgnnMatrix * len(shapes))(*[_hip.SgnnMatrix(P, P, max(c, 1), max(c, 1), r, c) for r, c in shapes])
        return lib.sgnn_newton_schulz(0, mats, len(shapes), 5, 1.0, 0.0, 0.0, 0.0, P, 1 << 30, None)
    assert status([empty]) == _hip.SGNN_OK
    assert status([(4, 4)]) != _hip.SGNN_OK
    assert status([empty, (4, 4)]) != _hip.SGNN_OK
    assert status([empty, empty, (300, 200)]) != _hip.SGNN_OK


def test_matrix_struct_matches_header():
    assert ctypes.sizeof(_hip.SgnnMatrix) == 40


def test_python_entry_points_refuse_cpu_tensors():
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="GPU"):
        functional.linear(x, w)
    with pytest.raises(ValueError, match="GPU"):
        functional.layer_norm(x)
    with pytest.raises(ValueError, match="GPU"):
        muon.newton_schulz(x)


@pytest.mark.parametrize("bad", [dict(nseg=-1), dict(segs=None), dict(param=None), dict(update=None), dict(step=0)])
def test_muon_kernels_refuse(lib, bad):
    a = dict(segs=P, nseg=2, param=P, update=P, step=1)
    a.update(bad)
    assert lib.sgnn_muon_moments(a["segs"], a["nseg"], a["param"], P, P, P, a["update"], 0.95, 1, 0.1, 0.9, 0.999, 1e-8,
                                 a["step"], None) == INVALID
    if "step" not in bad:
        assert lib.sgnn_muon_apply(a["segs"], a["nseg"], a["param"], a["update"], 0.1, 0.0, None) == INVALID


@pytest.mark.parametrize("weight", [torch.zeros(3, 9, dtype=torch.bfloat16), torch.zeros(9, 3).t()], ids=["bf16", "strided"])
def test_fused_encoders_refuse_an_embedding_of_another_layout(weight):
    """The encoder kernels read fp32 rows: a 16-bit embedding beside an fp32 network would be read past its end."""
    from types import SimpleNamespace
    from sgnn_amd import engine, training
    t = torch.zeros(4)
    inp = SimpleNamespace(types=torch.zeros(4, dtype=torch.int64), ex_ptr=t, n_ex=1, vel_mean=t, vel_std=t, acc_mean=t, acc_std=t)
    with pytest.raises(ValueError, match="embedding"):
        training.emb_args(inp, weight)
    with pytest.raises(ValueError, match="embedding"):
        engine.step_in(inp, SimpleNamespace(n=4, T=6, dim=2, K=20), 1.0, weight, True)
    assert training.emb_args(inp, weight.float().contiguous())[3] == 1


def test_optimizers_refuse_each_other_s_state():
    """A checkpoint resumed with the other optimiser: refused before anything is changed."""
    from sgnn_amd import training
    module = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 3))
    flat = training.FlatParams(module)
    made = {"adam": training.Adam(flat, 0.5), "muon": muon.Muon(flat, module, 0.5)}
    for opt in made.values():
        opt.step_count = 3
        opt.exp_avg.fill_(2.0)
    for name, other in (("adam", "muon"), ("muon", "adam")):
        with pytest.raises(ValueError, match="optimiser"):
            made[name].load_state_dict(dict(made[other].state_dict(), lr=9.0))
        assert made[name].lr == 0.5 and made[name].step_count == 3 and (made[name].exp_avg == 2.0).all()
        made[name].load_state_dict(made[name].state_dict())


def test_optimizer_names():
    with pytest.raises(ValueError, match="adam"):
        muon.make_optimizer("sgd", None, None, 0.1)
