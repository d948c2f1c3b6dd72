"""The host side of fused_sandwich_rmsnorm: what is refused, and which rows a gate's rows serve. Runs on the CPU."""

import ctypes

import pytest
import torch

import fma
from fma import KernelBackend
from fma.ops.fused_sandwich_rmsnorm import gate_rows


def test_library_refuses(lib):
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) & ~15  # never read: every call is refused on the host
    message = lambda: lib.fma_last_error_string().decode()  # noqa: E731

    def forward(x=p, w=None, gate=None, rows=0, width=0, out=p, B=4, H=64, dtype=2):
        return lib.fma_sandwich_rmsnorm_fwd(x, p, None, w, gate, rows, width, out, p, None, B, H, 1e-5, 1.0, dtype, None)

    assert forward(dtype=3) == -2
    assert forward(B=-1) == -3 and forward(B=1 << 31) == -3 and forward(H=0) == -3 and forward(H=65537) == -3
    assert forward(x=None) == -1 and forward(out=None) == -1
    assert forward(x=p + 1) == -6 and forward(w=p + 1) == -6 and forward(gate=p + 1, rows=1, width=64) == -6
    assert forward(gate=p, rows=3, width=64) == -3 and "divide" in message()
    assert forward(gate=p, rows=8, width=64) == -3 and forward(gate=p, rows=0, width=64) == -3
    assert forward(gate=p, rows=2, width=32) == -3 and "columns" in message()
    assert forward(B=0, x=None) == 0  # no rows: nothing to do

    def backward(x=p, weight=None, dw=None, gate=None, dg=None, dout=p, stats=p, B=4, H=64, nbytes=1 << 30, workspace=p, dtype=2):
        return lib.fma_sandwich_rmsnorm_bwd(
            x, p, None, weight, gate, 1, H, dout, None, stats, p, p, dg, None, dw, B, H, 1.0, workspace, nbytes, dtype, None
        )

    assert backward(dtype=3) == -2 and backward(B=-1) == -3 and backward(H=0) == -3 and backward(B=0) == -3
    assert backward(x=None) == -1 and backward(stats=None) == -1 and backward(workspace=None) == -1
    assert backward(dw=p) == -1 and "without its input" in message() and backward(dg=p) == -1
    assert backward(dout=p + 1) == -6 and backward(workspace=p + 4) == -6
    assert backward(nbytes=lib.fma_sandwich_rmsnorm_bwd_workspace_bytes(4, 64, 0, 0) - 1) == -7 and "workspace" in message()
    assert lib.fma_sandwich_rmsnorm_bwd_workspace_bytes(0, 64, 0, 0) == 0
    plain, group, scalar = (lib.fma_sandwich_rmsnorm_bwd_workspace_bytes(60000, 64, *g) for g in ((0, 0), (60, 64), (60, 1)))
    assert plain < group and scalar == plain + 4 * 60000


def test_rows_of_a_gate():
    x = torch.empty(6, 5, 8)
    for shape, rows in (
        ((), 1), ((1,), 1), ((8,), 1), ((1, 8), 1), ((1, 1, 8), 1), ((1, 1, 1), 1),
        ((6, 1, 1), 6), ((6, 1, 8), 6), ((6, 5, 1), 30), ((6, 5, 8), 30),
    ):  # fmt: skip
        assert gate_rows(torch.empty(shape), x) == rows
    # positions shared by the sequences, other sizes, more dimensions than x
    for shape in ((5, 8), (5, 1), (1, 5, 8), (6, 5, 4), (3, 1, 8), (6, 5, 8, 1), (1, 6, 5, 8), (2,)):
        with pytest.raises(AssertionError, match="does not fit"):
            gate_rows(torch.empty(shape), x)
    assert gate_rows(torch.empty(5, 8), torch.empty(1, 5, 8)) == 5 and gate_rows(torch.empty(4), torch.empty(4)) == 1
    assert gate_rows(torch.empty(0, 1), torch.empty(0, 8)) == 0


def test_arguments():
    x, w = torch.zeros(6, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU only"):
        fma.fused_sandwich_rmsnorm(x, x, w, w, None)
    with pytest.raises(ValueError, match="kernel_backend"):
        fma.fused_sandwich_rmsnorm(x, x, w, w, 1e-5, kernel_backend=KernelBackend.torch)
    for args, message in (
        ((x.double(), x.double(), None, None, None), "float32"),
        ((x[0, 0], x[0, 0], None, None, None), "rows"),
        ((x[:, :0], x[:, :0], None, None, None), "rows"),
        ((x, x[:5], None, None, None), "one shape"),
        ((x, x.half(), None, None, None), "one shape"),
        ((x, x, w[:4], None, None), "post_weight"),
        ((x, x, None, w.half(), None), "weight"),
        ((x, x, None, w[None], None), "weight"),
        ((x, x, w, w, None, w.half()), "gate"),
        ((x, x, w, w, None, torch.ones(3, 8)), "gate"),
    ):
        with pytest.raises(AssertionError, match=message):
            fma.fused_sandwich_rmsnorm(*args)
