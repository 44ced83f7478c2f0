"""What the layer norm, class log probability and grouped product entry points refuse, on the host (no GPU)."""
import ctypes as C

import pytest
import torch

import mgg_osdi23_b200 as mgg
from mgg_osdi23_b200 import _lib
from mgg_osdi23_b200._lib import ERR_INVALID_ARG, ERR_UNSUPPORTED, OK, lib

P = 4096     # stands for a device address: refused calls never look at it


def why():
    return lib.mggb_last_error().decode()


def test_layer_norm_forward():
    call = lambda out=P, x=2 * P, eps=1e-5, n=4, dim=8, ld_out=8, ld_x=8, dt=0: lib.mggb_layer_norm_forward(
        out, x, None, None, eps, None, None, n, dim, ld_out, ld_x, dt, None)
    for bad in (dict(out=None), dict(x=None), dict(n=-1), dict(dim=0), dict(ld_out=7), dict(ld_x=7), dict(dt=3), dict(dt=-1), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert call(**bad) == ERR_INVALID_ARG and "layer_norm_forward" in why(), bad
    assert call(n=0, out=None, x=None) == OK
    assert call(out=2 * P, ld_x=9) == ERR_INVALID_ARG and "in place" in why()


def test_layer_norm_backward():
    need = C.c_size_t()
    assert lib.mggb_layer_norm_backward_scratch_bytes(100, 8, C.byref(need)) == OK and need.value > 0
    assert lib.mggb_layer_norm_backward_scratch_bytes(100, 0, C.byref(need)) == ERR_INVALID_ARG
    assert lib.mggb_layer_norm_backward_scratch_bytes(-1, 8, C.byref(need)) == ERR_INVALID_ARG
    assert lib.mggb_layer_norm_backward_scratch_bytes(100, 8, None) == ERR_INVALID_ARG
    assert lib.mggb_layer_norm_backward_scratch_bytes(100, 8, C.byref(need)) == OK

    def call(dx=P, dw=2 * P, dy=3 * P, x=4 * P, mean=5 * P, rstd=6 * P, n=100, dim=8, ld=(8, 8, 8), dt=0, scratch=7 * P, nbytes=None):
        return lib.mggb_layer_norm_backward(dx, dw, None, dy, x, mean, rstd, None, n, dim, *ld, dt, scratch, need.value if nbytes is None else nbytes, None)
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(n=-1), dict(dim=0), dict(ld=(7, 8, 8)), dict(ld=(8, 7, 8)),
                dict(ld=(8, 8, 7)), dict(dt=5), dict(scratch=None), dict(nbytes=need.value - 1), dict(scratch=7 * P + 4), dict(dx=None, dw=None)):
        assert call(**bad) == ERR_INVALID_ARG and "layer_norm_backward" in why(), bad
    assert call(dx=3 * P, ld=(9, 8, 8)) == ERR_INVALID_ARG and "in place" in why()
    assert call(dx=4 * P, ld=(8, 8, 9)) == ERR_INVALID_ARG and "in place" in why()


def test_layer_norm_rows_beyond_the_limit():
    d, need = 2 ** 28 + 1, C.c_size_t()
    assert lib.mggb_layer_norm_forward(P, 2 * P, None, None, 1e-5, None, None, 1, d, d, d, 0, None) == ERR_INVALID_ARG and "2^28" in why()
    assert lib.mggb_layer_norm_backward_scratch_bytes(1, d, C.byref(need)) == ERR_INVALID_ARG and "2^28" in why()
    assert lib.mggb_layer_norm_backward(P, 2 * P, None, 3 * P, 4 * P, 5 * P, 6 * P, None, 1, d, d, d, d, 0, 16 * P, 2 ** 40, None) == ERR_INVALID_ARG
    assert "2^28" in why()


def test_class_logprob_forward():
    def call(lp=P, stats=None, ent=None, ids=None, tlp=None, top=0, z=2 * P, ld=10, labels=3 * P, n=4, c=10, dt=1):
        return lib.mggb_class_logprob_forward(lp, stats, ent, ids, tlp, top, z, ld, labels, n, c, dt, None)
    for bad in (dict(z=None), dict(n=-1), dict(c=0), dict(ld=9), dict(dt=9), dict(labels=None), dict(lp=None), dict(top=3), dict(top=-1),
                dict(top=11, ids=P), dict(top=33, ids=P, c=100, ld=100), dict(lp=None, labels=None)):
        assert call(**bad) == ERR_INVALID_ARG and "class_logprob_forward" in why(), bad
    assert call(n=0, z=None) == OK


def test_class_logprob_backward():
    def call(dz=P, z=2 * P, ld_dz=10, ld_z=10, labels=3 * P, stats=4 * P, dlp=5 * P, ent=None, dh=None, n=4, c=10, dt=2):
        return lib.mggb_class_logprob_backward(dz, z, ld_dz, ld_z, labels, stats, dlp, ent, dh, n, c, dt, None)
    for bad in (dict(dz=None), dict(z=None), dict(stats=None), dict(n=-1), dict(c=0), dict(ld_z=9), dict(ld_dz=9), dict(dt=3), dict(labels=None),
                dict(dlp=None), dict(dh=P), dict(dlp=None, labels=None), dict(dz=2 * P, ld_dz=11)):
        assert call(**bad) == ERR_INVALID_ARG and "class_logprob_backward" in why(), bad
    assert call(n=0, dz=None, z=None, stats=None) == OK


def test_grouped_dense():
    fwd = lambda out=P, x=2 * P, w=3 * P, ptr=4 * P, g=2, n=10, k=8, m=8, dt=0: lib.mggb_grouped_dense_forward(out, x, w, ptr, g, n, k, m, dt, None)
    for bad in (dict(out=None), dict(x=None), dict(w=None), dict(ptr=None), dict(g=0), dict(n=-1), dict(k=0), dict(m=0), dict(dt=4), dict(n=2 ** 31),
                dict(out=2 * P), dict(out=3 * P)):
        assert fwd(**bad) == ERR_INVALID_ARG and "grouped_dense_forward" in why(), bad
    assert fwd(n=0, out=None, x=None) == OK
    for bad in (dict(g=_lib.MAX_GROUPS + 1), dict(k=_lib.MAX_GROUPED_DIM + 1), dict(m=_lib.MAX_GROUPED_DIM + 1)):
        assert fwd(**bad) == ERR_UNSUPPORTED and "grouped_dense_forward" in why(), bad
    need = C.c_size_t()
    # one narrow type with many rows: the rows are split, so there are partial sums to keep
    size = lambda n=100_000, g=1, k=8, m=8, dt=0, out=C.byref(need): lib.mggb_grouped_dense_backward_scratch_bytes(n, g, k, m, dt, out)
    assert size() == OK
    for bad in (dict(n=-1), dict(g=0), dict(k=0), dict(m=0), dict(dt=3), dict(out=None)):
        assert size(**bad) == ERR_INVALID_ARG and "grouped_dense_backward_scratch_bytes" in why(), bad

    def bwd(dx=P, dw=2 * P, dy=3 * P, x=4 * P, w=5 * P, ptr=6 * P, g=1, n=100_000, k=8, m=8, dt=0, scratch=16 * P, nbytes=None):
        return lib.mggb_grouped_dense_backward(dx, dw, dy, x, w, ptr, g, n, k, m, dt, scratch, need.value if nbytes is None else nbytes, None)
    for bad in (dict(dy=None), dict(x=None), dict(w=None), dict(ptr=None), dict(dx=None, dw=None), dict(dx=3 * P), dict(dx=4 * P), dict(dx=5 * P),
                dict(g=0), dict(n=-1), dict(k=0), dict(m=0), dict(dt=4)):
        assert bwd(**bad) == ERR_INVALID_ARG and "grouped_dense_backward" in why(), bad
    for bad in (dict(dw=P), dict(dw=3 * P), dict(dw=4 * P)):
        assert bwd(**bad) == ERR_INVALID_ARG and "dw must not alias" in why(), bad
    if need.value:
        for bad in (dict(scratch=None), dict(nbytes=need.value - 1), dict(scratch=16 * P + 8)):
            assert bwd(**bad) == ERR_INVALID_ARG and "scratch" in why(), bad


def test_constants_match_the_header():
    import os
    import re
    text = open(os.path.join(os.path.dirname(_lib.PKG_DIR), "include", "mggb200.h")).read()
    for name in ("F32", "BF16", "F16"):
        assert re.search(rf"\bMGGB_{name} = {getattr(_lib, name)}\b", text), name
    for name in ("MAX_TOP", "MAX_GROUPS", "MAX_GROUPED_DIM"):
        assert re.search(rf"#define MGGB_{name} {getattr(_lib, name)}\b", text), name


def test_python_wrappers_refuse_host_tensors_and_wrong_types():
    x, v, i = torch.zeros(4, 8), torch.zeros(4), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mgg.layer_norm_forward(torch.zeros(4, 8), x)
    with pytest.raises(ValueError, match="CUDA"):
        mgg.layer_norm_backward(torch.zeros(4, 8), x, x, v, v)
    with pytest.raises(ValueError, match="CUDA"):
        mgg.class_logprob_forward(v, x, i)
    with pytest.raises(ValueError, match="CUDA"):
        mgg.class_logprob_backward(x, x, i, torch.zeros(4, 2), v)
    with pytest.raises(ValueError, match="CUDA"):
        mgg.grouped_dense_forward(torch.zeros(4, 3), x, torch.zeros(2, 8, 3), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="float32"):
        mgg.layer_norm_forward(x.double(), x.double())
    with pytest.raises(ValueError, match="matrix"):
        mgg.layer_norm_forward(x, [[1.0]])
    with pytest.raises(ValueError, match="matrix"):
        mgg.layer_norm_forward(v, v)
    with pytest.raises(ValueError, match="shape mismatch"):
        mgg.grouped_dense_forward(x, x, torch.zeros(2, 7, 8), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        mgg.grouped_dense_forward(x, x.double(), torch.zeros(2, 8, 8), torch.zeros(3, dtype=torch.int32))


class _CudaLike(torch.Tensor):
    """A host tensor that says it is on the current GPU, for the checks behind that one."""
    def get_device(self):
        return 0


def _cuda_like(t):
    return t.as_subclass(_CudaLike)


@pytest.fixture
def device0(monkeypatch):
    monkeypatch.setattr(mgg.api, "_current_device", lambda: 0)


def test_python_wrappers_refuse_strides_shapes_and_other_devices(device0, monkeypatch):
    c = _cuda_like
    x = c(torch.zeros(4, 8))
    with pytest.raises(ValueError, match="contiguous rows"):
        mgg.layer_norm_forward(x, c(torch.zeros(8, 4).t()))
    with pytest.raises(ValueError, match="contiguous rows"):
        mgg.layer_norm_forward(x, c(torch.zeros(1, 8).expand(4, 8)))
    with pytest.raises(ValueError, match="shape"):
        mgg.layer_norm_forward(c(torch.zeros(4, 7)), x)
    with pytest.raises(ValueError, match="dtype"):
        mgg.layer_norm_forward(c(torch.zeros(4, 8).half()), x)
    with pytest.raises(ValueError, match="weight"):
        mgg.layer_norm_forward(x, x, c(torch.zeros(7)))
    with pytest.raises(ValueError, match="weight"):
        mgg.layer_norm_forward(x, x, c(torch.zeros(8).half()))
    with pytest.raises(ValueError, match="mean"):
        mgg.layer_norm_forward(x, x, mean=c(torch.zeros(8)[::2]))
    with pytest.raises(ValueError, match="labels"):
        mgg.class_logprob_forward(c(torch.zeros(4)), x, c(torch.zeros(4, dtype=torch.int64)))
    with pytest.raises(ValueError, match="top_ids"):
        mgg.class_logprob_forward(None, x, None, top_ids=c(torch.zeros(4, dtype=torch.int32)))
    with pytest.raises(ValueError, match="top_logprobs needs top_ids"):
        mgg.class_logprob_forward(None, x, None, top_logprobs=c(torch.zeros(4, 2)))
    with pytest.raises(ValueError, match="stats"):
        mgg.class_logprob_backward(x, x, None, c(torch.zeros(4)), None)
    with pytest.raises(ValueError, match="x must be contiguous"):
        mgg.grouped_dense_forward(c(torch.zeros(4, 3)), c(torch.zeros(4, 9))[:, :8], c(torch.zeros(2, 8, 3)), c(torch.zeros(3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="group_ptr"):
        mgg.grouped_dense_forward(c(torch.zeros(4, 3)), x, c(torch.zeros(2, 8, 3)), c(torch.zeros(4, dtype=torch.int32)))
    with pytest.raises(ValueError, match="dw"):
        mgg.grouped_dense_backward(None, c(torch.zeros(2, 8, 3).half()), c(torch.zeros(4, 3)), x, c(torch.zeros(2, 8, 3)), c(torch.zeros(3, dtype=torch.int32)))
    monkeypatch.setattr(mgg.api, "_current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        mgg.layer_norm_forward(x, x)
