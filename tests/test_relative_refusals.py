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


def window(lib, **change):
    f = dict(q=P, k=P, v=P, out=P, q_row_stride=768, k_row_stride=768, v_row_stride=768, out_row_stride=768, q_offsets=P,
             k_offsets=P, k_lens=None, batch=2, head_num=12, kv_head_num=12, q_rows=100, k_rows=100, max_q_len=60, max_k_len=60,
             left=-1, right=-1, sinks=0, scale=0.125, distance_bias=None, bias_len=0, bias_left=0, workspace=None, workspace_bytes=0)
    f.update(change)
    return lib.bt_window_attention(C.byref(_abi.bt_window_attention_args(**f)), None)


@pytest.mark.parametrize("change", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q_offsets=None), dict(k_offsets=None), dict(q=P + 8),
    dict(k=P + 2), dict(v=P + 4), dict(out=P + 8), dict(q_offsets=P + 2), dict(k_lens=P + 1), dict(distance_bias=P + 2, bias_len=9),
    dict(q_row_stride=760), dict(k_row_stride=767), dict(v_row_stride=772), dict(out_row_stride=0), dict(q_row_stride=(1 << 32) + 8),
    dict(head_num=0), dict(head_num=1025), dict(kv_head_num=0), dict(kv_head_num=5), dict(batch=0), dict(q_rows=0), dict(k_rows=-1),
    dict(max_q_len=0), dict(max_q_len=1 << 30), dict(max_k_len=-1), dict(max_k_len=1 << 30), dict(sinks=-1), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(distance_bias=P, bias_len=0),
    dict(distance_bias=P, bias_len=5, bias_left=5), dict(distance_bias=P, bias_len=5, bias_left=-1)])
def test_window(lib, change):
    assert window(lib, **change) == _abi.BT_ERR_INVALID_ARG
    assert lib.bt_window_attention(None, None) == _abi.BT_ERR_INVALID_ARG


def test_window_workspace(lib):
    n = C.c_size_t(7)
    ask = lib.bt_window_attention_workspace
    assert ask(2, 12, 12, 17, 100, -1, 0, C.byref(n)) == _abi.BT_OK and n.value == 0  # not few queries
    assert ask(2, 12, 12, 1, 100, -1, 0, C.byref(n)) == _abi.BT_OK and n.value == 0  # 100 keys are one range
    assert ask(1, 8, 2, 1, 1 << 20, -1, 0, C.byref(n)) == _abi.BT_OK and n.value == 2 * 148 * 16 * (64 * 4 + 8)
    assert ask(1, 8, 2, 1, 1 << 20, 500, 4, C.byref(n)) == _abi.BT_OK and n.value == 0  # four ranges, a cluster
    assert ask(40, 8, 8, 1, 3000, -1, 0, C.byref(n)) == _abi.BT_OK and n.value == 4 * 320 * 16 * (64 * 4 + 8)
    for bad in [(0, 8, 2, 1, 9, -1, 0), (1, 8, 3, 1, 9, -1, 0), (1, 8, 2, 0, 9, -1, 0), (1, 8, 2, 1, -1, -1, 0), (1, 8, 2, 1, 9, -1, -1)]:
        assert ask(*bad, C.byref(n)) == _abi.BT_ERR_INVALID_ARG
    assert ask(1, 8, 2, 1, 9, -1, 0, None) == _abi.BT_ERR_INVALID_ARG


X, RES, SUM, OUT = P, 2 * P, 3 * P, 4 * P


@pytest.mark.parametrize("x_fp32,group,total,out", [
    (0, None, SUM, SUM), (1, None, SUM, SUM), (0, None, X, X), (0, None, RES, RES),      # two results in one place
    (1, None, SUM, X), (1, None, X, OUT), (1, None, None, X), (1, 0, X, OUT),           # halves over single precision
    (0, 0, SUM, X), (0, 128, SUM, X), (1, 128, None, X), (0, 0, SUM, RES), (0, 128, None, RES)])  # 8 bits over something else
def test_norm_over_its_own_inputs(lib, x_fp32, group, total, out):
    """Elements of another size lie on other rows' inputs, which may not have been read yet.  (What is allowed reaches a launch: it
    is tested on the device.)"""
    args = [X, x_fp32, RES, 5 * P, 0, total, out]
    if group is None:
        rc = lib.bt_add_residual_rmsnorm(*args, None, 4, 768, 1e-6, None)
    else:
        rc = lib.bt_add_residual_rmsnorm_e4m3(*args, 6 * P, group, None, 4, 768, 1e-6, None)
    assert rc == _abi.BT_ERR_INVALID_ARG


class OnCuda(torch.Tensor):
    """A tensor without memory that says it is on the device: nothing here gets as far as reading it."""
    is_cuda = True


def big(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="meta").as_subclass(OnCuda)


CUT = (1 << 32) + 8  # 8 in 32 bits


def test_sizes_past_32_bits_are_refused_not_cut(lib):
    from bytetransformer_b200 import encoder as E
    off, two = big(3, dtype=torch.int32), big(2, dtype=torch.int32)
    q = big(64, 128)
    for call in [
            lambda: E.add_residual_rmsnorm(big(CUT, 8), None, big(8)),
            lambda: E.add_residual_rmsnorm(big(8, CUT), None, big(CUT)),
            lambda: E.add_residual_rmsnorm_e4m3(big(CUT, 8), None, big(8), group=128),
            lambda: E.add_residual_rmsnorm(big(CUT, 8), None, big(8), m_dev=big(1, dtype=torch.int32)),
            lambda: E.relative_position_bias(big(CUT, 4), 4, 4),
            lambda: E.relative_position_bias(big(32, CUT), 4, 4),
            lambda: E.relative_position_bias_grad(big(CUT, 4, 4), 32),
            lambda: E.relative_position_bias_grad(big(CUT, 1, 4, 4), 32),
            lambda: E.relative_position_bias_grad(big(2, 4, 4), CUT),
            lambda: E.relative_position_bias_grad(big(2, 4, 4), -32),
            lambda: E.window_attention(q, q, q, big(CUT, dtype=torch.int32), big(CUT, dtype=torch.int32), 8, 8),
            lambda: E.window_attention(big(CUT, 64), q[:, :64], q[:, :64], off, off, 8, 8),
            lambda: E.window_attention(q, big(CUT, 64), big(CUT, 64), off, off, 8, 8),
            lambda: E.window_attention(big(1, CUT * 64), q, q, two, two, 1, 8),
            lambda: E.window_attention(q, q, q, off, off, 8, 8, distance_bias=big(2, CUT, dtype=torch.float32), bias_left=4),
            lambda: E.window_attention(q, q, q, off, off, 8 - (1 << 32), 8),
            lambda: E.window_attention(q, q, q, off, off, 8, 8 - (1 << 32))]:
        with pytest.raises(RuntimeError, match="2\\^3"):
            call()
