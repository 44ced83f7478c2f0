"""Outputs that lie partly over an input are refused, on the host (no GPU)."""
import ctypes as C

from mgg_osdi23_b200._lib import ERR_INVALID_ARG, lib

P = 1 << 20      # stands for a device address: refused calls never look at it


def why():
    return lib.mggb_last_error().decode()


def test_layer_norm_forward():
    call = lambda out, x, ld_out=8, ld_x=8, n=100, dim=8, dt=0: lib.mggb_layer_norm_forward(out, x, None, None, 1e-5, None, None, n, dim, ld_out, ld_x, dt, None)
    for shift in (4, -4, 8 * 4, -8 * 4, 99 * 32, 99 * 32 + 28):
        assert call(P + shift, P) == ERR_INVALID_ARG and "partly over" in why(), shift
    assert call(P + 8, P, ld_out=16, ld_x=16) == ERR_INVALID_ARG and "partly over" in why()            # columns 2..9 and 0..7 of one matrix
    assert call(P + 64 - 4, P, ld_out=16, ld_x=16) == ERR_INVALID_ARG and "partly over" in why()       # around the end of its rows
    assert call(P + 40, P, ld_out=16) == ERR_INVALID_ARG and "partly over" in why()                    # gaps in one of them
    assert call(P + 2, P, dt=1, n=1) == ERR_INVALID_ARG and "partly over" in why()


def test_layer_norm_backward():
    call = lambda dx, dy, x, ld=(8, 8, 8): lib.mggb_layer_norm_backward(dx, None, None, dy, x, 8 * P, 9 * P, None, 100, 8, *ld, 0, None, 0, None)
    for dx in (P + 4, P - 32, 2 * P + 16, 2 * P - 4):
        assert call(dx, P, 2 * P) == ERR_INVALID_ARG and "partly over" in why(), dx
    # in place over one of them and partly over the other
    assert call(P, P, P + 32) == ERR_INVALID_ARG and "partly over" in why()
    assert call(P + 32, P, P + 32) == ERR_INVALID_ARG and "partly over" in why()


def test_class_logprob_backward():
    call = lambda dz, z, ld=10: lib.mggb_class_logprob_backward(dz, z, ld, ld, 8 * P, 9 * P, 10 * P, None, None, 50, 10, 2, None)
    for shift in (2, -2, 20, -20, 49 * 20 + 18):
        assert call(P + shift, P) == ERR_INVALID_ARG and "partly over" in why(), shift
    assert call(P + 18, P, ld=20) == ERR_INVALID_ARG and "partly over" in why()


def test_grouped_products():
    n, k, m, g = 100, 16, 24, 3
    x, w, dy = n * k * 4, g * k * m * 4, n * m * 4
    fwd = lambda out: lib.mggb_grouped_dense_forward(out, P, 2 * P, 3 * P, g, n, k, m, 0, None)
    for out in (P + 4, P + x - 4, P - dy + 4, 2 * P + w - 4, 2 * P - 4):
        assert fwd(out) == ERR_INVALID_ARG and "partly over" in why(), out
    need = C.c_size_t()
    assert lib.mggb_grouped_dense_backward_scratch_bytes(n, g, k, m, 0, C.byref(need)) == 0
    bwd = lambda dx=10 * P, dw=11 * P: lib.mggb_grouped_dense_backward(dx, dw, P, 2 * P, 3 * P, 4 * P, g, n, k, m, 0, 16 * P, need.value, None)
    for dx in (P + 4, P - x + 4, 2 * P + 4, 2 * P - 4, 3 * P + 4):
        assert bwd(dx=dx) == ERR_INVALID_ARG and "dx lies partly over" in why(), dx
    for dw in (P + 4, P - w + 4, 2 * P + x - 4, 10 * P + 4):
        assert bwd(dw=dw) == ERR_INVALID_ARG and "dw lies partly over" in why(), dw
