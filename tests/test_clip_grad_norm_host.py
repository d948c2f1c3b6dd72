"""The host side of the gradient norm and of clipping: what is refused, and what needs no GPU. Runs on the CPU."""

import ctypes
import inspect
import math

import pytest
import torch

import fma
from fma import _lib
from fma.ops.clip_grad_norm.cuda_implementation import _is_dense


def _arrays(pointers, sizes, dtypes):
    n = len(pointers)
    return (ctypes.c_void_p * n)(*pointers), (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*dtypes), n


def _clip(lib, pointers, sizes, dtypes, max_norm=1.0, norm=True, workspace=True, nbytes=None):
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    nbytes = lib.fma_grad_norm_workspace_bytes(len(pointers)) if nbytes is None else nbytes
    return lib.fma_clip_grad_norm(*_arrays(pointers, sizes, dtypes), 0, max_norm, p if norm else None, p if workspace else None, nbytes, None)


def test_library_refuses(lib):
    p = 1 << 20  # an address that is never read: every call is refused on the host
    message = lambda: lib.fma_last_error_string().decode()  # noqa: E731
    assert _clip(lib, [p], [8], [7]) == -2 and "dtype" in message()
    assert _clip(lib, [p], [-1], [0]) == -3
    assert _clip(lib, [p], [(1 << 37) + 1], [0]) == -3
    assert _clip(lib, [None], [8], [0]) == -1
    assert _clip(lib, [p + 2], [8], [_lib.FMA_F32]) == -6 and "aligned" in message()
    assert _clip(lib, [p], [8], [0], max_norm=-1.0) == -3 and "max_norm" in message()
    assert _clip(lib, [p], [8], [0], max_norm=math.nan) == -3
    assert _clip(lib, [p], [8], [0], norm=False) == -1
    assert _clip(lib, [p], [8], [0], workspace=False) == -1
    assert _clip(lib, [p], [8], [0], nbytes=16) == -7 and "workspace" in message()
    # the same tensor twice, and two whose ends overlap
    for pointers, sizes in (([p, p], [8, 8]), ([p + 28, p], [8, 8]), ([p, p + 4096, p + 16], [64, 8, 4])):
        assert _clip(lib, pointers, sizes, [0] * len(sizes)) == -8 and "share memory" in message()
        assert lib.fma_scale_grads(*_arrays(pointers, sizes, [0] * len(sizes)), p, 1.0, None) == -8
    assert lib.fma_grad_norm(None, None, None, 3, 0, p, p, 1 << 20, None) == -1
    assert lib.fma_grad_norm(None, None, None, (1 << 20) + 1, 0, p, p, 1 << 20, None) == -3
    assert lib.fma_scale_grads(*_arrays([p], [8], [0]), None, 1.0, None) == -1
    assert lib.fma_scale_grads(None, None, None, 0, p, 1.0, None) == 0  # no tensors: nothing to do


def test_workspace_grows_with_the_launches(lib):
    sizes = [lib.fma_grad_norm_workspace_bytes(n) for n in (0, 1, 160, 161, 320, 1 << 20)]
    assert sizes == sorted(sizes) and sizes[1] == sizes[2] < sizes[3] == sizes[4] and sizes[0] >= 8
    assert lib.fma_grad_norm_workspace_bytes(-1) == 0


def test_arguments():
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    for call in (
        lambda **k: fma.clip_grad_norm_([p], **{"max_norm": 1.0, **k}),
        lambda **k: fma.get_total_norm([p.grad], **{n: v for n, v in k.items() if n != "max_norm"}),
    ):
        with pytest.raises(ValueError, match="norm_type"):
            call(norm_type=1.0)
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        fma.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        fma.clip_grads_with_norm_([p], math.nan, torch.ones(()))
    assert torch.equal(p.grad, torch.ones(3)) and p.grad._version == 0
    p.grad = torch.eye(3)[0].to_sparse()
    with pytest.raises(TypeError, match="layout"):
        fma.clip_grad_norm_([p], 1.0)
    p.grad = None
    assert fma.clip_grad_norm_([p], 1.0) == 0.0 and fma.get_total_norm([]) == 0.0 and fma.clip_grads_with_norm_(p, 1.0, torch.ones(())) is None


def test_tensors_of_other_kinds_are_refused():
    class Wrapped(torch.Tensor):
        pass

    with pytest.raises(TypeError, match="Wrapped"):
        fma.get_total_norm([torch.ones(3).as_subclass(Wrapped)])


def test_dense_layouts():
    t = torch.empty(4, 6, 5)
    for dense in (t, t.permute(2, 0, 1), t.transpose(0, 1), t[1:3], torch.empty(3, 1, 4).permute(1, 2, 0), torch.empty(0, 3), torch.empty(())):
        assert _is_dense(dense)
    for gaps in (t[:, ::2], t[..., 1:], t[0, 0, 0].expand(3), t.transpose(0, 2)[:, 1:]):
        assert not _is_dense(gaps)


def test_scaling_by_a_norm_in_64_bits_refuses_the_same(lib):
    p = 1 << 20  # never read, as above
    scale = lambda *a, norm=p, max_norm=1.0: lib.fma_scale_grads_norm64(*_arrays(*a), norm, max_norm, None)  # noqa: E731
    assert scale([p], [8], [7]) == -2 and scale([p], [-1], [0]) == -3 and scale([None], [8], [0]) == -1
    assert scale([p], [8], [0], max_norm=-1.0) == -3 and scale([p], [8], [0], max_norm=math.nan) == -3
    assert scale([p, p + 28], [8, 8], [0, 0]) == -8
    assert scale([p], [8], [0], norm=None) == -1
    assert scale([p], [8], [0], norm=p + 4) == -6 and "aligned" in lib.fma_last_error_string().decode()
    assert lib.fma_scale_grads(*_arrays([p], [8], [0]), p + 2, 1.0, None) == -6


def test_names_and_arguments_are_those_of_the_host_library():
    """a call of torch.nn.utils works here as it stands"""
    for name in ("clip_grad_norm_", "get_total_norm", "clip_grads_with_norm_"):
        ours, theirs = (inspect.signature(getattr(module, name)).parameters for module in (fma, torch.nn.utils))
        assert [(p.name, p.default) for p in ours.values()] == [(p.name, p.default) for p in theirs.values()], name
    p = torch.nn.Parameter(torch.ones(3))
    for foreach in (None, False, True):
        assert fma.clip_grad_norm_([p], 1.0, 2.0, False, foreach) == 0.0 and fma.get_total_norm([], foreach=foreach) == 0.0
        assert fma.clip_grads_with_norm_([p], 1.0, torch.ones(()), foreach) is None


def test_a_norm_inside_a_tensor_is_refused(lib):
    """every workgroup reads it while others write"""
    p = 1 << 20  # never read, as above
    for scale, aligned in ((lib.fma_scale_grads, 4), (lib.fma_scale_grads_norm64, 8)):
        for at in (p, p + 16, p + 64 - aligned):
            assert scale(*_arrays([p], [16], [0]), at, 1.0, None) == -8 and "norm" in lib.fma_last_error_string().decode()
            assert scale(*_arrays([p + 4096, p, p - 4096], [16, 16, 16], [0, 0, 0]), at, 1.0, None) == -8
        assert scale(*_arrays([p + 4], [16], [0]), p + 4 - 4 * (aligned == 8), 1.0, None) == -8
    assert lib.fma_clip_grad_norm(*_arrays([p], [16], [0]), 0, 1.0, p + 8, p + 4096, 1 << 20, None) == -8
