"""CPU: what the entry points for relative positions and the root-mean-square norm refuse, before anything is launched."""
import ctypes as C

import pytest
import torch

from bytetransformer_b200 import _abi

P = 1 << 20  # an address that is never followed: every call here is refused


@pytest.fixture(scope="module")
def lib():
    from bytetransformer_b200 import build
    build.build_core()
    return _abi.load()


def bias(lib, table=P, fp32=0, buckets=32, dist=128, both=1, heads=12, q=64, k=64, start=0, out=P, out_fp32=0):
    return lib.bt_relative_position_bias(table, fp32, buckets, dist, both, heads, q, k, start, out, out_fp32, None)


@pytest.mark.parametrize("change", [
    dict(table=None), dict(out=None), dict(out=P + 8), dict(table=P + 1), dict(table=P + 2, fp32=1), dict(buckets=33),
    dict(buckets=2), dict(buckets=1, both=0), dict(buckets=258), dict(dist=8), dict(dist=(1 << 20) + 1), dict(heads=0),
    dict(heads=65536), dict(q=0), dict(k=0), dict(q=-1), dict(k=(1 << 29) + 1), dict(start=-(1 << 29) - 1),
    dict(q=64 * 65535 + 1)])
def test_bias(lib, change):
    assert bias(lib, **change) == _abi.BT_ERR_INVALID_ARG


def grad(lib, grad=P, fp32=0, buckets=32, dist=128, both=1, batch=2, heads=12, q=64, k=64, start=0, out=P, ws=P, room=1 << 30):
    return lib.bt_relative_position_bias_grad(grad, fp32, buckets, dist, both, batch, heads, q, k, start, out, ws, room, None)


@pytest.mark.parametrize("change", [
    dict(grad=None), dict(out=None), dict(ws=None), dict(grad=P + 2), dict(ws=P + 4), dict(out=P + 2), dict(buckets=3),
    dict(dist=8), dict(batch=0), dict(batch=65536), dict(q=0), dict(k=0)])
def test_grad(lib, change):
    assert grad(lib, **change) == _abi.BT_ERR_INVALID_ARG


def test_grad_workspace(lib):
    n = C.c_size_t()
    assert lib.bt_relative_position_bias_grad_workspace(0, 32, 2, 12, 300, 300, C.byref(n)) == _abi.BT_OK
    assert n.value % (4 * 32 * 12 * 2) == 0
    assert grad(lib, q=300, k=300, room=n.value - 1) == _abi.BT_ERR_WORKSPACE
    assert lib.bt_relative_position_bias_grad_workspace(0, 32, 2, 12, 300, 300, None) == _abi.BT_ERR_INVALID_ARG
    assert lib.bt_relative_position_bias_grad_workspace(0, 32, 65535, 12, 1 << 29, 64, C.byref(n)) == _abi.BT_ERR_INVALID_ARG


def norm(lib, x=P, residual=P, gamma=P, total=P, out=P, scales=P, group=None, rows=4, hidden=768, eps=1e-6):
    if group is None:
        return lib.bt_add_residual_rmsnorm(x, 0, residual, gamma, 0, total, out, None, rows, hidden, eps, None)
    return lib.bt_add_residual_rmsnorm_e4m3(x, 0, residual, gamma, 0, total, out, scales, group, None, rows, hidden, eps, None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(gamma=None), dict(out=None), dict(x=P + 2), dict(residual=P + 8), dict(gamma=P + 4),
    dict(total=P + 2), dict(out=P + 8), dict(rows=0), dict(hidden=0), dict(hidden=12), dict(hidden=16392),
    dict(eps=-1.0), dict(eps=float("nan")), dict(group=64), dict(group=128, scales=None), dict(group=0, scales=P + 2)])
def test_norm(lib, change):
    assert norm(lib, **change) == _abi.BT_ERR_INVALID_ARG


def test_python_refuses_host_tensors(lib):
    from bytetransformer_b200 import encoder as E
    t = torch.zeros(32, 12, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        E.relative_position_bias(t, 8, 8)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        E.relative_position_bias_grad(torch.zeros(2, 8, 8), 32)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        E.add_residual_rmsnorm(t, None, t[0])
