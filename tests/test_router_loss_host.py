"""The host side of router_loss: what is refused. Runs on the CPU."""

import ctypes

import pytest
import torch

import fma
from fma import KernelBackend, MoE, swiglu_packed


def test_library_refuses(lib):
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) & ~15  # never read: every call is refused on the host
    message = lambda: lib.fma_last_error_string().decode()  # noqa: E731

    def forward(logits=p, mask=None, T=4, E=8, k=2, out=p, nbytes=1 << 20, dtype=2, workspace=p):
        return lib.fma_router_loss(logits, mask, T, E, k, out, p, p, p, workspace, nbytes, dtype, None)

    assert forward(dtype=3) == -2
    assert forward(T=-1) == -3 and forward(T=1 << 31) == -3
    assert forward(E=0) == -3 and forward(E=1025, k=1) == -4 and "1024" in message()
    assert forward(k=0) == -3 and forward(k=9) == -3 and "top_k" in message()
    assert forward(logits=None) == -1 and forward(out=None) == -1 and forward(workspace=None) == -1
    assert forward(logits=p + 1) == -6 and forward(workspace=p + 4) == -6 and "aligned" in message()
    assert forward(nbytes=lib.fma_router_loss_workspace_bytes(4, 8) - 1) == -7 and "workspace" in message()

    def backward(logits=p, T=4, E=8, table=p, grad=p, dtype=2):
        return lib.fma_router_loss_bwd(logits, None, T, E, table, p, None, grad, dtype, None)

    assert backward(dtype=5) == -2 and backward(E=1025) == -4 and backward(T=-1) == -3
    assert backward(logits=None) == -1 and backward(table=None) == -1 and backward(grad=None) == -1
    assert backward(grad=p + 1) == -6
    assert backward(T=0, logits=None, grad=None) == 0  # no tokens: nothing to do
    assert lib.fma_router_loss_workspace_bytes(0, 8) > 0 and lib.fma_router_loss_workspace_bytes(4, 1025) == 0
    sizes = [lib.fma_router_loss_workspace_bytes(T, 64) for T in (1, 128, 129, 10**5, 10**9)]
    assert sizes == sorted(sizes) and sizes[0] == sizes[1] < sizes[2] and sizes[3] == sizes[4]


def test_arguments():
    logits = torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        fma.router_loss(logits, 2)
    with pytest.raises(ValueError, match="kernel_backend"):
        fma.router_loss(logits, 2, kernel_backend=KernelBackend.torch)
    for bad, message in (
        (lambda: fma.router_loss(logits.double(), 2), "float32"),
        (lambda: fma.router_loss(logits.long(), 2), "float32"),
        (lambda: fma.router_loss(torch.zeros(()), 1), "dimension"),
        (lambda: fma.router_loss(torch.zeros(2, 1025), 2), "experts"),
        (lambda: fma.router_loss(torch.zeros(2, 0), 1), "experts"),
        (lambda: fma.router_loss(logits, 0), "num_experts_per_tok"),
        (lambda: fma.router_loss(logits, 9), "num_experts_per_tok"),
        (lambda: fma.router_loss(logits, 2, torch.ones(6)), "bool"),
        (lambda: fma.router_loss(logits, 2, torch.ones(7, dtype=torch.bool)), "does not fit"),
        # logits that know their batch take masks of its shape alone: a transposed one would name other tokens
        (lambda: fma.router_loss(torch.zeros(2, 3, 8), 2, torch.ones(3, 2, dtype=torch.bool)), "does not fit"),
        (lambda: fma.router_loss(torch.zeros(2, 3, 8), 2, torch.ones(6, dtype=torch.bool)), "does not fit"),
    ):
        with pytest.raises(AssertionError, match=message):
            bad()


def test_the_layer_passes_its_number_of_choices():
    moe = MoE(8, 3, 16, 16, swiglu_packed, True, False, 0.02)
    with pytest.raises(RuntimeError, match="GPU only"):
        moe.router_loss(torch.zeros(6, 8), torch.ones(2, 3, dtype=torch.bool))
    with pytest.raises(AssertionError, match="num_experts_per_tok should be in .1, 2., not 3"):
        moe.router_loss(torch.zeros(6, 2))
