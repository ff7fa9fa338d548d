"""The linear layers' and the clipping's entry points refuse bad arguments on the host: no pointer is followed, nothing is
launched, so these run without a GPU."""
import ctypes

import pytest

from transformer_amd import _lib

BASE = {
    "mla_linear_act": (_lib.LinearActArgs, dict(x=4096, w=8192, bias=None, residual=None, y=12288, saved=None, M=64, N=16, K=24,
                                                x_stride=24, w_stride=24, residual_stride=0, y_stride=16, activation=0)),
    "mla_gated_linear": (_lib.GatedLinearArgs, dict(x=4096, w_gate=8192, w_up=8192, h=12288, saved=None, M=64, N=16, K=24,
                                                    x_stride=24, w_gate_stride=24, w_up_stride=24, h_stride=16, activation=2)),
    "mla_gated_linear_bwd": (_lib.GatedLinearBwdArgs, dict(dy=4096, w_down=8192, saved=16384, dgu=12288, M=64, N=16, K=24,
                                                           dy_stride=24, w_stride=16, dgu_stride=32, activation=2)),
    "mla_linear_dx": (_lib.LinearDxArgs, dict(dy=4096, w0=8192, w1=8192, dx=12288, M=64, N=16, K=24, dy_stride=32, w0_stride=24,
                                              w1_stride=24, dx_stride=24)),
    "mla_act_grad": (_lib.ActGradArgs, dict(dy=4096, saved=8192, dz=12288, db=16384, M=64, N=16, dy_stride=16, dz_stride=16,
                                            activation=2, db_dtype=0)),
}
SIZES = (dict(M=-1), dict(M=1 << 30), dict(N=0), dict(N=12), dict(N=1 << 20), dict(M=(1 << 30) - 1, N=(1 << 20) - 8))
BAD = {
    "mla_linear_act": (dict(K=0), dict(K=20), dict(K=1 << 20), dict(x=None), dict(w=None), dict(y=None), dict(x=4104),
                       dict(w=8200), dict(y=12290), dict(bias=4100), dict(residual=4104, residual_stride=16),
                       dict(residual=4096, residual_stride=8), dict(residual=4096, residual_stride=-16), dict(saved=8),
                       dict(x_stride=16), dict(x_stride=28), dict(w_stride=1 << 22), dict(y_stride=8), dict(activation=4),
                       dict(activation=-1)),
    "mla_gated_linear": (dict(K=0), dict(K=20), dict(x=None), dict(w_gate=None), dict(w_up=8200), dict(h=None), dict(saved=8),
                         dict(w_up_stride=16), dict(h_stride=20), dict(activation=0), dict(activation=9)),
    "mla_gated_linear_bwd": (dict(K=0), dict(dy=None), dict(w_down=8196), dict(saved=None), dict(saved=8), dict(dgu=None),
                             dict(dgu_stride=16), dict(w_stride=8), dict(K=1 << 19, dy_stride=1 << 19, w_stride=1 << 12),
                             dict(activation=0)),
    "mla_linear_dx": (dict(K=0), dict(dy=None), dict(w0=None), dict(w1=8200), dict(dx=8), dict(dy_stride=16),
                      dict(w1_stride=16), dict(w1_stride=32), dict(dx_stride=16), dict(N=1 << 19, dy_stride=1 << 20, w0_stride=1 << 12)),
    "mla_act_grad": (dict(M=0), dict(dy=None), dict(dz=None), dict(saved=None), dict(saved=8), dict(dy_stride=8), dict(dz_stride=8),
                     dict(db_dtype=3), dict(db=16386), dict(M=200, workspace_bytes=0), dict(activation=7)),
}


@pytest.mark.parametrize("entry", sorted(BASE))
def test_bad_arguments_are_refused(entry):
    lib = _lib.load()
    struct, good = BASE[entry]
    for change in (*SIZES, *BAD[entry]):
        a = struct(**{**good, **change})
        rc = getattr(lib, entry)(ctypes.byref(a), None)
        assert rc < 0 and entry.encode() in lib.mla_last_error(), (entry, change, rc)
    assert getattr(lib, entry)(None, None) == _lib.MLA_ERR_INVALID_ARG


def test_no_rows_is_no_work():
    lib = _lib.load()
    for entry in ("mla_linear_act", "mla_gated_linear", "mla_gated_linear_bwd", "mla_linear_dx"):
        struct, good = BASE[entry]
        a = struct(**{**good, "M": 0})
        assert getattr(lib, entry)(ctypes.byref(a), None) == _lib.MLA_OK


def _norm_args(at, counts, types, **change):
    n = len(at)
    keep = ((ctypes.c_void_p * n)(*at), (ctypes.c_int64 * n)(*counts), (ctypes.c_int32 * n)(*types))
    fields = dict(ptrs=ctypes.addressof(keep[0]), numels=ctypes.addressof(keep[1]), dtypes=ctypes.addressof(keep[2]), n_tensors=n,
                  norm=4096, workspace=8192, workspace_bytes=1 << 20, max_norm=1.0, norm_is_max=0)
    return _lib.GradNormArgs(**{**fields, **change}), keep


def test_grad_clip_refuses_bad_tables():
    lib = _lib.load()
    good = ([65536, 131072], [100, 200], [1, 0])
    for args, change in (((good[0], good[1], [1, 2]), {}), ((good[0], [100, -1], good[2]), {}),
                         (([65536, None], good[1], good[2]), {}), (([65538, 131072], good[1], good[2]), {}),
                         (([65536, 131073], good[1], good[2]), {}), (([65536, 65536], good[1], good[2]), {}),
                         (([65536, 65536 + 399], good[1], [1, 0]), {}), (([65536, 65536 + 398], good[1], [1, 0]), {}),
                         (good, dict(ptrs=None)), (good, dict(norm=None)), (good, dict(workspace=None)),
                         (good, dict(workspace_bytes=8)), (good, dict(max_norm=-1.0)), (good, dict(max_norm=float("nan"))),
                         (good, dict(n_tensors=-1)), (good, dict(n_tensors=1 << 20))):
        a, keep = _norm_args(*args, **change)
        assert lib.mla_grad_clip(ctypes.byref(a), None) < 0, (args, change)
        assert b"mla_grad_clip" in lib.mla_last_error()
    assert lib.mla_grad_clip(None, None) == lib.mla_grad_norm(None, None) == _lib.MLA_ERR_INVALID_ARG


def test_workspaces_and_saved_sizes():
    lib = _lib.load()
    a, _ = _norm_args([65536] * 3, [1] * 3, [1] * 3)
    assert 0 < lib.mla_grad_norm_workspace_bytes(ctypes.byref(a)) <= 1 << 14
    assert lib.mla_linear_saved_size(1, 8) == 3 << 10 and lib.mla_linear_saved_size(33, 40) == 12 << 10
    assert lib.mla_linear_saved_size(0, 8) == lib.mla_linear_saved_size(-5, 8) == lib.mla_linear_saved_size(1 << 62, 8) == 0


NEED = {  # sizes whose products are cut along k, or whose column sums come in several segments
    "mla_linear_act": dict(M=4090, N=328, K=4072, x_stride=4072, w_stride=4072, y_stride=328),
    "mla_gated_linear": dict(M=1000, N=264, K=1800, x_stride=1800, w_gate_stride=1800, w_up_stride=1800, h_stride=264),
    "mla_linear_dx": dict(M=300, N=1000, K=64, dy_stride=2000, w0_stride=64, w1_stride=64, dx_stride=64),
    "mla_act_grad": dict(M=200),
}


@pytest.mark.parametrize("entry", sorted(NEED))
def test_missing_short_and_unaligned_workspaces_are_refused(entry):
    lib = _lib.load()
    struct, good = BASE[entry]
    a = struct(**{**good, **NEED[entry]})
    need = getattr(lib, entry + "_workspace_bytes")(ctypes.byref(a))
    assert 0 < need <= 64 << 20
    for at, size in ((None, need), (1 << 20, need - 1), (1 << 20, 0), ((1 << 20) + 8, need)):
        a.workspace, a.workspace_bytes = at, size
        assert getattr(lib, entry)(ctypes.byref(a), None) == _lib.MLA_ERR_WORKSPACE, (at, size)
    small = struct(**{**good, "M": 64})
    assert getattr(lib, entry + "_workspace_bytes")(ctypes.byref(small)) == 0 or entry == "mla_linear_dx"
