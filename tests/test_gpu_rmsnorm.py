"""Root-mean-square norm with the residual's addition, fp16 and e4m3 results, against its definition in 64 bits.

Tolerances: the sum of squares is a chain of at most 8 * 4 + 5 + 16 single-precision additions, i.e. half of 53 * 2^-24 in
the square root, and s, the mean, the root, the quotient and the two products are one rounding each: 34 * 2^-24 < 2^-18
relative.  A result in fp16 adds half a step: 2^-11 relative, 2^-25 below the normal numbers; in e4m3 2^-4 and 2^-10."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SINGLE = 2.0 ** -18


def definition(x, residual, gamma, eps):
    s = x.double() + (residual.double() if residual is not None else 0.0)
    return s, s / torch.sqrt((s * s).mean(1, keepdim=True) + eps) * gamma.double()


def check_half(got, want):
    assert got.dtype == torch.float16
    assert ((got.double() - want).abs() <= want.abs() * (2.0 ** -11 + SINGLE) + 2.0 ** -25).all()


def check_e4m3(out, scales, y, group):
    rows, hidden = y.shape
    group = group or hidden
    top = torch.stack([p.abs().amax(1) for p in y.split(group, dim=1)], dim=1)
    want = top.clamp(min=2.0 ** -100) / 448.0
    assert scales.shape == want.shape
    assert ((scales.double() - want).abs() <= want * SINGLE).all()
    exact = y / scales.double().repeat_interleave(group, dim=1)[:, :hidden]
    assert ((out.double() - exact).abs() <= exact.abs() * (2.0 ** -4 + SINGLE) + 2.0 ** -10).all()
    # the largest value of a group takes the largest number there is
    assert (out.double().abs().amax(1) == 448.0).logical_or(top.amax(1) == 0).all()


def inputs(rows, hidden, x_fp32, gamma_fp32, residual, device, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 131 + hidden)
    x = torch.randn(rows, hidden, generator=g).to(torch.float32 if x_fp32 else torch.float16)
    r = (torch.randn(rows, hidden, generator=g) * 2).half() if residual else None
    gamma = (1 + 0.1 * torch.randn(hidden, generator=g)).to(torch.float32 if gamma_fp32 else torch.float16)
    return tuple(t.to(device) if t is not None else None for t in (x, r, gamma))


WIDTHS = [8, 16, 64, 120, 128, 136, 256, 264, 512, 520, 768, 776, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200, 12288, 12296, 16384]


@pytest.mark.parametrize("hidden", WIDTHS)
@pytest.mark.parametrize("x_fp32,gamma_fp32", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("residual", [True, False])
def test_against_the_definition(cuda_device, hidden, x_fp32, gamma_fp32, residual):
    from bytetransformer_b200 import encoder as E
    for rows in (1, 2, 7, 33):
        x, r, gamma = inputs(rows, hidden, x_fp32, gamma_fp32, residual, cuda_device)
        s, y = definition(x, r, gamma, 1e-6)
        out, total = E.add_residual_rmsnorm(x, r, gamma)
        check_half(out, y)
        if residual:
            assert ((total.double() - s).abs() <= s.abs() * 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -25).all()
        else:
            assert total is None
        for group in (0, 128):
            q, scales, total8 = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=group)
            check_e4m3(q, scales, y, group)
            assert (total8 is None) if not residual else torch.equal(total8, total)


def test_many_rows(cuda_device):
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(70001, 72, False, False, True, cuda_device)
    s, y = definition(x, r, gamma, 1e-6)
    check_half(E.add_residual_rmsnorm(x, r, gamma)[0], y)


def test_past_32_bits(cuda_device):
    from bytetransformer_b200 import encoder as E
    rows, hidden = 270_000, 8192  # 2.2e9 elements
    x = torch.ones(rows, hidden, dtype=torch.float16, device=cuda_device)
    x[-5:] = torch.randn(5, hidden, device=cuda_device).half()
    gamma = torch.ones(hidden, dtype=torch.float16, device=cuda_device)
    s, y = definition(x[-5:], x[-5:], gamma, 1e-6)
    out, total = E.add_residual_rmsnorm(x, x, gamma)
    check_half(out[-5:], y)
    assert (out[:-5] == 1).all() and (total[:-5] == 2).all() and torch.equal(total[-5:], x[-5:] * 2)
    del out, total
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, None, gamma, group=128)
    check_e4m3(q[-5:], scales[-5:], y, 128)


def test_rows_of_zeros_and_tiny_rows(cuda_device):
    from bytetransformer_b200 import encoder as E
    x = torch.zeros(3, 256, dtype=torch.float16, device=cuda_device)
    x[1] = 2.0 ** -24
    gamma = torch.ones(256, dtype=torch.float16, device=cuda_device)
    for eps in (1e-6, 0.0):
        s, y = definition(x[1:2], None, gamma, eps)
        for group in (0, 128):
            q, scales, _ = E.add_residual_rmsnorm_e4m3(x, None, gamma, eps, group=group)
            check_e4m3(q[1:2], scales[1:2], y, group)
            if eps > 0:
                assert (q[0].float() == 0).all() and (scales[0] > 0).all() and torch.isfinite(scales).all()
        check_half(E.add_residual_rmsnorm(x, None, gamma, eps)[0][1:2], y)


def test_infinities_and_nan_stay_in_their_row(cuda_device):
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(6, 768, False, False, True, cuda_device)
    s, y = definition(x, r, gamma, 1e-6)
    x[1, 5] = float("nan")
    x[3, 700] = float("inf")
    out, total = E.add_residual_rmsnorm(x, r, gamma)
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=128)
    keep = [0, 2, 4, 5]
    check_half(out[keep], y[keep])
    check_e4m3(q[keep], scales[keep], y[keep], 128)
    assert torch.isnan(out[1]).all() and torch.isnan(out[3, 700]) and torch.isnan(q[1].float()).all()
    assert torch.isnan(total[1, 5]) and torch.isinf(total[3, 700]) and torch.isfinite(total[1, 6:]).all()


@pytest.mark.parametrize("hidden", [256, 2048])
def test_rows_behind_the_device_count_are_left_as_they_were(cuda_device, hidden):
    from bytetransformer_b200 import _abi
    lib = _abi.load()
    x, r, gamma = inputs(37, hidden, False, False, True, cuda_device)
    s, y = definition(x, r, gamma, 1e-6)
    stream = torch.cuda.current_stream().cuda_stream
    for valid in (0, 1, 20, 37, 50, -3):
        m = torch.tensor([valid], dtype=torch.int32, device=cuda_device)
        out = torch.full((37, hidden), 7.0, dtype=torch.float16, device=cuda_device)
        total, scales = out.clone(), torch.full((37,), 7.0, device=cuda_device)
        assert lib.bt_add_residual_rmsnorm(x.data_ptr(), 0, r.data_ptr(), gamma.data_ptr(), 0, total.data_ptr(), out.data_ptr(),
                                           m.data_ptr(), 37, hidden, 1e-6, stream) == 0
        n = max(0, min(37, valid))
        check_half(out[:n], y[:n])
        assert (out[n:] == 7).all() and (total[n:] == 7).all()
        q = torch.full((37, hidden), 1.0, device=cuda_device).to(torch.float8_e4m3fn)
        assert lib.bt_add_residual_rmsnorm_e4m3(x.data_ptr(), 0, r.data_ptr(), gamma.data_ptr(), 0, None, q.data_ptr(),
                                                scales.data_ptr(), 0, m.data_ptr(), 37, hidden, 1e-6, stream) == 0
        assert (q[n:].float() == 1).all() and (scales[n:] == 7).all()


@pytest.mark.parametrize("hidden", [768, 4096])
def test_in_place(cuda_device, hidden):
    """The sum over the residual, the result over x: what a chain of layers does with two buffers."""
    from bytetransformer_b200 import _abi
    from bytetransformer_b200 import encoder as E
    lib = _abi.load()
    x, r, gamma = inputs(50, hidden, False, False, True, cuda_device)
    out, total = E.add_residual_rmsnorm(x, r, gamma)
    assert lib.bt_add_residual_rmsnorm(x.data_ptr(), 0, r.data_ptr(), gamma.data_ptr(), 0, r.data_ptr(), x.data_ptr(), None, 50,
                                       hidden, 1e-6, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x, out) and torch.equal(r, total)


def test_another_stream_and_a_captured_graph(cuda_device):
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(40, 768, False, False, True, cuda_device)
    want, _ = E.add_residual_rmsnorm(x, r, gamma)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = E.add_residual_rmsnorm(x, r, gamma)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, total = E.add_residual_rmsnorm(x, r, gamma)
        b, _ = E.add_residual_rmsnorm(a, total, gamma)  # a chain: each kernel starts ahead of the end of the one before
        q, scales, _ = E.add_residual_rmsnorm_e4m3(b, total, gamma)
    x2 = torch.randn_like(x)
    x.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    a2, total2 = E.add_residual_rmsnorm(x2, r, gamma)
    b2, _ = E.add_residual_rmsnorm(a2, total2, gamma)
    q2, scales2, _ = E.add_residual_rmsnorm_e4m3(b2, total2, gamma)
    assert torch.equal(b, b2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scales, scales2)


def test_python_refusals(cuda_device):
    from bytetransformer_b200 import BtError
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(4, 64, False, False, True, cuda_device)
    with pytest.raises(RuntimeError, match="residual must be"):
        E.add_residual_rmsnorm(x, r[:3], gamma)
    with pytest.raises(RuntimeError, match="gamma"):
        E.add_residual_rmsnorm(x, r, gamma[:32])
    with pytest.raises(RuntimeError, match="fp16 or fp32"):
        E.add_residual_rmsnorm(x.bfloat16(), r, gamma)
    with pytest.raises(RuntimeError, match="contiguous"):
        E.add_residual_rmsnorm(x.t(), None, gamma)
    with pytest.raises(RuntimeError, match="group"):
        E.add_residual_rmsnorm_e4m3(x, r, gamma, group=64)
    with pytest.raises(BtError):
        E.add_residual_rmsnorm(torch.zeros(4, 12, dtype=torch.float16, device=cuda_device), None,
                               torch.ones(12, dtype=torch.float16, device=cuda_device))
    assert E.add_residual_rmsnorm(x[:0], r[:0], gamma)[0].shape == (0, 64)


@pytest.mark.parametrize("hidden", [64, 520, 768, 2056, 4096, 12296])
@pytest.mark.parametrize("group", [0, 128])
def test_a_scale_says_where_its_group_holds_nan(cuda_device, hidden, group):
    """scale = max |y| over the group, which is NaN where a y is: by NaN in the row, by an infinity (it makes NaN of itself, the rest is
    finite), by NaN in gamma for its columns alone."""
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(7, hidden, False, False, True, cuda_device)
    clean = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=group)
    at = hidden - 3
    x[1, 2], x[4, at] = float("nan"), float("inf")
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=group)
    sick = torch.zeros_like(scales, dtype=torch.bool)
    sick[1] = True
    sick[4, at // 128 if group else 0] = True
    assert torch.equal(torch.isnan(scales), sick)
    wide = sick.repeat_interleave(group or hidden, dim=1)[:, :hidden]
    assert torch.equal(torch.isnan(q.float()), wide)
    keep = [0, 2, 3, 5, 6]
    assert torch.equal(q[keep].view(torch.uint8), clean[0][keep].view(torch.uint8)) and torch.equal(scales[keep], clean[1][keep])
    gamma[at] = float("nan")
    x, r, _ = inputs(7, hidden, False, False, True, cuda_device)
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=group)
    columns = torch.zeros(scales.shape[1], dtype=torch.bool, device=cuda_device)
    columns[at // 128 if group else 0] = True
    assert torch.equal(torch.isnan(scales), columns[None].expand_as(scales))
    assert torch.equal(scales[:, ~columns], clean[1][:, ~columns])


@pytest.mark.parametrize("hidden", [136, 768, 4096])
def test_every_group_uses_the_largest_number(cuda_device, hidden):
    """The largest value of each 128 columns, not of the row alone, is +-448."""
    from bytetransformer_b200 import encoder as E
    x, r, gamma = inputs(40, hidden, True, False, True, cuda_device)
    x[3, :128] = 0.0
    r[3, :128] = 0.0
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, r, gamma, group=128)
    top = torch.stack([p.double().abs().amax(1) for p in q.float().split(128, dim=1)], dim=1)
    want = torch.full_like(top, 448.0)
    want[3, 0] = 0.0
    assert torch.equal(top, want) and top.shape == scales.shape


@pytest.mark.parametrize("hidden", [768, 4096])
def test_in_place_the_other_ways(cuda_device, hidden):
    """The result over the residual and the sum over x; with 8 bits the sum over the residual."""
    from bytetransformer_b200 import _abi
    from bytetransformer_b200 import encoder as E
    lib, stream = _abi.load(), torch.cuda.current_stream().cuda_stream
    x, r, gamma = inputs(50, hidden, False, False, True, cuda_device)
    out, total = E.add_residual_rmsnorm(x, r, gamma)
    q, scales, _ = E.add_residual_rmsnorm_e4m3(x, r, gamma)
    x1, r1 = x.clone(), r.clone()
    assert lib.bt_add_residual_rmsnorm(x1.data_ptr(), 0, r1.data_ptr(), gamma.data_ptr(), 0, x1.data_ptr(), r1.data_ptr(), None, 50,
                                       hidden, 1e-6, stream) == 0
    assert torch.equal(r1, out) and torch.equal(x1, total)
    q1, scales1, r1 = torch.empty_like(q), torch.empty_like(scales), r.clone()
    assert lib.bt_add_residual_rmsnorm_e4m3(x.data_ptr(), 0, r1.data_ptr(), gamma.data_ptr(), 0, r1.data_ptr(), q1.data_ptr(),
                                            scales1.data_ptr(), 0, None, 50, hidden, 1e-6, stream) == 0
    assert torch.equal(q1.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scales1, scales) and torch.equal(r1, total)


def test_as_many_rows_as_32_bits_count(cuda_device):
    """2^31 - 1 rows of 8: the last block has room for a row that 32 bits do not count."""
    from bytetransformer_b200 import encoder as E
    rows = (1 << 31) - 1
    x = torch.empty(rows, 8, dtype=torch.float16, device=cuda_device)
    x[:5], x[-5:] = torch.randn(5, 8, device=cuda_device).half(), torch.randn(5, 8, device=cuda_device).half()
    x[5:-5].fill_(2.0)
    gamma = torch.linspace(0.5, 2.0, 8, device=cuda_device).half()
    out, _ = E.add_residual_rmsnorm(x, None, gamma)
    for part in (slice(0, 9), slice(rows // 2, rows // 2 + 9), slice(rows - 9, rows)):
        check_half(out[part], definition(x[part], None, gamma, 1e-6)[1])
