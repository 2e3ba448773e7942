"""Relative position bias by buckets and its gradient against their definition in whole numbers and 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# Single-precision additions that a value goes through at most: 127 down a diagonal's 128 rows, 3 with the neighbouring thread's
# share and the rows' ends (up to 7 of their own, instead of the 127), 8 within a block of 8 diagonals, 36 over a lane's
# share of a run of 257 blocks and its ends, 3 over the lanes; and the rounding of the result.
ROUNDINGS = 178


def bucket(d, buckets, dist, both):
    """Whole numbers: step j is reached when n^m * e^j >= D^j * e^m."""
    count, base, n = buckets, 0, max(-d, 0)
    if both:
        count = buckets // 2
        base, n = (count if d > 0 else 0), abs(d)
    e = count // 2
    if n < e:
        return base + n
    m, j = count - e, 0
    while j + 1 < m and n ** m * e ** (j + 1) >= dist ** (j + 1) * e ** m:
        j += 1
    return base + e + j


def by_distance(q, k, start, buckets, dist, both):
    """(bucket of every diagonal, index of the diagonal of every (query, key))"""
    ids = torch.tensor([bucket(d, buckets, dist, both) for d in range(-(q - 1) - start, k - start)])
    return ids, torch.arange(k)[None, :] + (q - 1 - torch.arange(q))[:, None]


BUCKETS = [(32, 128, True), (32, 128, False), (4, 3, True), (2, 2, False), (256, 129, False), (256, 1 << 20, False),
           (48, 400, False), (64, 1000, True), (18, 20, True)]
SHAPES = [(1, 1, 0), (1, 700, 699), (7, 5, 0), (64, 64, 0), (65, 1025, 3), (70, 263, 0), (70, 264, 0), (66, 265, 1), (3, 511, 0), (3, 513, 0), (5, 520, 0), (5, 521, 0), (130, 197, 1000), (257, 1032, -300), (128, 8, 0),
          (3, 4100, 2000), (200, 1027, 1 << 28), (5, 9, -(1 << 28))]


@pytest.mark.parametrize("q,k,start", SHAPES)
@pytest.mark.parametrize("buckets,dist,both", BUCKETS)
def test_bias(cuda_device, q, k, start, buckets, dist, both):
    from bytetransformer_b200 import encoder as E
    heads = 3
    g = torch.Generator().manual_seed(q * 7 + k)
    ids, at = by_distance(q, k, start, buckets, dist, both)
    for table_type in (torch.float16, torch.float32):
        table = torch.randn(buckets, heads, generator=g).to(table_type)
        want = table[ids].t()[:, at]
        for out_type in (torch.float16, torch.float32):
            got = E.relative_position_bias(table.to(cuda_device), q, k, max_distance=dist, bidirectional=both,
                                           q_start=start, out_dtype=out_type)
            assert got.dtype == out_type and torch.equal(got.cpu(), want.to(out_type))


def test_bias_of_the_longest_distances_told_apart(cuda_device):
    """One row over every border of the largest range."""
    from bytetransformer_b200 import encoder as E
    table = torch.arange(256.0)[:, None]
    k = (1 << 20) + 10
    got = E.relative_position_bias(table.to(cuda_device), 1, k, max_distance=1 << 20, bidirectional=False, q_start=k - 1,
                                   out_dtype=torch.float32).cpu().view(-1).flip(0).int().tolist()
    at = [n for n in range(1, k) if got[n] != got[n - 1]]
    for n in at:
        for m in (n - 1, n):
            assert got[m] == bucket(-m, 256, 1 << 20, False)
    assert got[0] == 0 and got[-1] == 255 and got == sorted(got)


GRAD_SHAPES = [(1, 1, 0, 1), (1, 700, 699, 2), (7, 5, 0, 3), (64, 64, 0, 2), (65, 1025, 3, 1), (130, 197, 0, 2),
               (257, 1032, -300, 1), (128, 8, 0, 2), (129, 2063, 7, 1), (3, 4100, 2000, 1), (300, 12, 0, 1), (200, 1027, 1 << 28, 1)]


@pytest.mark.parametrize("q,k,start,batch", GRAD_SHAPES + [(40, 96 + m, 0, 2) for m in range(8)])
@pytest.mark.parametrize("fp32", [False, True])
def test_grad(cuda_device, q, k, start, batch, fp32):
    from bytetransformer_b200 import encoder as E
    heads = 3
    g = torch.Generator().manual_seed(q * 11 + k)
    grad = torch.randn(batch, heads, q, k, generator=g).to(torch.float32 if fp32 else torch.float16)
    for buckets, dist, both in [(32, 128, True), (32, 128, False), (4, 3, True), (256, 1 << 20, False)]:
        ids, at = by_distance(q, k, start, buckets, dist, both)
        member = ids[at].reshape(-1)
        flat = grad.double().sum(0).reshape(heads, -1)
        want = torch.zeros(heads, buckets, dtype=torch.float64).index_add_(1, member, flat).t()
        size = torch.zeros(heads, buckets, dtype=torch.float64).index_add_(1, member, grad.double().abs().sum(0).reshape(heads, -1)).t()
        got = E.relative_position_bias_grad(grad.to(cuda_device), buckets, max_distance=dist, bidirectional=both,
                                            q_start=start).cpu().double()
        assert ((got - want).abs() <= ROUNDINGS * 2.0 ** -24 * size).all()


def test_grad_is_the_bias_gradient_by_differences(cuda_device):
    """The bias is linear in the table: moving one entry by t moves sum(w * bias) by t times its gradient."""
    from bytetransformer_b200 import encoder as E
    q, k, heads, buckets = 45, 67, 2, 16
    g = torch.Generator().manual_seed(5)
    w = torch.randn(heads, q, k, generator=g).double()
    grad = E.relative_position_bias_grad(w.float().to(cuda_device), buckets, max_distance=20).cpu().double()
    for b in range(buckets):
        for h in range(heads):
            table = torch.zeros(buckets, heads)
            table[b, h] = 1.0
            moved = E.relative_position_bias(table.to(cuda_device), q, k, max_distance=20, out_dtype=torch.float32).cpu().double()
            assert abs(float((w.float().double() * moved).sum()) - float(grad[b, h])) <= ROUNDINGS * 2.0 ** -24 * float((w * moved).abs().sum())


def test_grad_is_the_same_every_time(cuda_device):
    from bytetransformer_b200 import encoder as E
    grad = torch.randn(4, 6, 333, 517, device=cuda_device, dtype=torch.float16)
    first = E.relative_position_bias_grad(grad, 32)
    for _ in range(5):
        assert torch.equal(first, E.relative_position_bias_grad(grad, 32))


def test_grad_reads_nothing_beside_the_matrix(cuda_device):
    """Odd rows: the vectors at a row's ends and at the buffer's hold other rows' values, or none."""
    from bytetransformer_b200 import encoder as E
    for k in (61, 62, 63, 65, 66, 67):
        whole = torch.full((2 * 37 * k + 64,), float("nan"), dtype=torch.float16, device=cuda_device)
        grad = whole[:2 * 37 * k].view(2, 37, k)
        grad.fill_(0.25)
        got = E.relative_position_bias_grad(grad, 32)
        assert torch.equal(got.sum(0).cpu(), torch.full((2,), 0.25 * 37 * k))


def test_infinite_gradients_stay_in_their_bucket(cuda_device):
    from bytetransformer_b200 import encoder as E
    grad = torch.zeros(1, 40, 40, device=cuda_device)
    grad[0, 20, 18] = float("inf")
    grad[0, 5, 6] = float("nan")
    got = E.relative_position_bias_grad(grad, 32)[:, 0].cpu()
    assert got[2] == float("inf") and torch.isnan(got[17])
    keep = [b for b in range(32) if b not in (2, 17)]
    assert (got[keep] == 0).all()


def test_past_32_bits(cuda_device):
    """More than 2^31 elements, rows that start at every alignment, the last ones looked at."""
    from bytetransformer_b200 import encoder as E
    heads, q, k = 3, 27_001, 27_003
    table = torch.randn(32, heads, device=cuda_device, dtype=torch.float16)
    bias = E.relative_position_bias(table, q, k)
    for rows in (slice(0, 3), slice(q - 70, q)):
        n = rows.stop - rows.start
        part = E.relative_position_bias(table, n, k, q_start=rows.start)
        assert torch.equal(bias[:, rows], part)
    ids, at = by_distance(70, k, q - 70, 32, 128, True)
    assert torch.equal(bias[2, q - 70:].cpu(), table[:, 2].cpu()[ids][at])
    bias.fill_(1.0)  # as a gradient: the buckets' sizes
    got = E.relative_position_bias_grad(bias, 32).cpu().double()
    d = torch.arange(-(q - 1), k)
    many = torch.minimum(torch.minimum(d + q, k - d), torch.tensor(min(q, k))).double()
    member = torch.tensor([bucket(max(-200, min(200, int(x))), 32, 128, True) for x in d.tolist()])
    want = torch.zeros(32, dtype=torch.float64).index_add_(0, member, many)[:, None].expand(32, heads)
    assert ((got - want).abs() <= ROUNDINGS * 2.0 ** -24 * want).all()


def test_another_stream_a_captured_graph_and_empty_calls(cuda_device):
    from bytetransformer_b200 import encoder as E
    table = torch.randn(32, 12, device=cuda_device, dtype=torch.float16)
    grad = torch.randn(2, 12, 77, 91, device=cuda_device, dtype=torch.float16)
    want, want_grad = E.relative_position_bias(table, 77, 91), E.relative_position_bias_grad(grad, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_grad = E.relative_position_bias(table, 77, 91), E.relative_position_bias_grad(grad, 32)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_grad, want_grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_grad = E.relative_position_bias(table, 77, 91), E.relative_position_bias_grad(grad, 32)
    table.mul_(2)
    grad.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want * 2) and torch.equal(got_grad, want_grad * 2)
    assert E.relative_position_bias(table, 0, 5).shape == (12, 0, 5)
    assert torch.equal(E.relative_position_bias_grad(grad[:0], 32), torch.zeros(32, 12, device=cuda_device))


def test_python_refusals(cuda_device):
    from bytetransformer_b200 import BtError
    from bytetransformer_b200 import encoder as E
    table = torch.zeros(32, 12, device=cuda_device, dtype=torch.float16)
    with pytest.raises(BtError):
        E.relative_position_bias(table[:31], 4, 4)
    with pytest.raises(RuntimeError, match="fp16 or fp32"):
        E.relative_position_bias(table.bfloat16(), 4, 4)
    with pytest.raises(RuntimeError, match="contiguous"):
        E.relative_position_bias(table[:, :6], 4, 4)
    with pytest.raises(RuntimeError, match="out_dtype"):
        E.relative_position_bias(table, 4, 4, out_dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="grad must be"):
        E.relative_position_bias_grad(table, 32)


def test_the_general_path_takes_it_as_attention_bias(cuda_device):
    """Made on the device, used by the encoder: the same as the bias indexed by hand."""
    from bytetransformer_b200 import encoder as E
    from helpers import make_layer_weights, to_device_weights
    heads, B, S = 4, 2, 75
    g = torch.Generator().manual_seed(3)
    enc = E.Encoder(heads, 64, [to_device_weights(make_layer_weights(heads * 64, g), cuda_device)])
    x = torch.randn(B, S, heads * 64, generator=g).half().to(cuda_device)
    mask = torch.ones(B, S, S, dtype=torch.float16, device=cuda_device)
    table = torch.randn(32, heads, generator=g).half()
    ids, at = by_distance(S, S, 0, 32, 128, True)
    by_hand = table[ids].t()[:, at].contiguous().to(cuda_device)
    assert torch.equal(enc.forward_general(x, mask, E.relative_position_bias(table.to(cuda_device), S, S)),
                       enc.forward_general(x, mask, by_hand))


@pytest.mark.parametrize("table_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("out_type", [torch.float16, torch.float32])
def test_a_table_gets_its_gradient(cuda_device, table_type, out_type):
    """Through the bias into the table, from gradients of every layout, against the sum by buckets in 64 bits."""
    from bytetransformer_b200 import encoder as E
    heads, q, k, buckets, dist, start = 3, 45, 67, 16, 20, 5
    g = torch.Generator().manual_seed(61)
    ids, at = by_distance(q, k, start, buckets, dist, True)
    member = ids[at].reshape(-1)
    data = torch.randn(buckets, heads, generator=g).to(table_type).to(cuda_device)
    w = torch.randn(heads, q, k, generator=g).to(out_type).to(cuda_device)
    ones = torch.ones((), dtype=out_type, device=cuda_device)
    odd = torch.empty(w.numel() + 1, dtype=out_type, device=cuda_device)[1:].view(heads, q, k).copy_(w)
    for grad in (w, ones.expand(heads, q, k), w.transpose(1, 2).contiguous().transpose(1, 2), odd):
        table = data.clone().requires_grad_()
        bias = E.relative_position_bias(table, q, k, max_distance=dist, q_start=start, out_dtype=out_type)
        assert bias.requires_grad and torch.equal(bias.detach(), E.relative_position_bias(data, q, k, max_distance=dist, q_start=start,
                                                                                         out_dtype=out_type))
        bias.backward(grad)
        assert table.grad.dtype == table_type
        flat = grad.cpu().double().reshape(heads, -1)
        want = torch.zeros(heads, buckets, dtype=torch.float64).index_add_(1, member, flat).t()
        size = torch.zeros(heads, buckets, dtype=torch.float64).index_add_(1, member, flat.abs()).t()
        step = want.abs() * 2.0 ** -11 + 2.0 ** -25 if table_type == torch.float16 else 0.0
        assert ((table.grad.cpu().double() - want).abs() <= ROUNDINGS * 2.0 ** -24 * size * 1.001 + step).all()
    with torch.no_grad():
        assert not E.relative_position_bias(table, q, k).requires_grad
    assert not E.relative_position_bias(table.detach(), q, k).requires_grad
    with pytest.raises(RuntimeError):  # no second derivative
        table = data.clone().requires_grad_()
        first, = torch.autograd.grad(E.relative_position_bias(table, q, k).float().sum(), table, create_graph=True)
        first.float().sum().backward()


def test_the_gradient_of_a_shared_table_adds_up_and_by_differences(cuda_device):
    """A table used twice, as two layers use it, within a larger expression: linear in the table, so a difference is its gradient."""
    from bytetransformer_b200 import encoder as E
    table = torch.randn(16, 2, device=cuda_device, requires_grad=True)
    w = torch.randn(2, 9, 14, device=cuda_device)

    def total(t):
        a = E.relative_position_bias(t, 9, 14, max_distance=20, out_dtype=torch.float32)
        b = E.relative_position_bias(t, 1, 14, max_distance=20, q_start=13, bidirectional=False, out_dtype=torch.float32)
        return (a * w).double().sum() + (b * 3.0).double().sum()
    total(table).backward()
    step = torch.zeros_like(table)
    for at in range(table.numel()):
        step.view(-1)[at] = 1.0
        with torch.no_grad():
            moved = total(step)
        assert abs(float(moved) - float(table.grad.view(-1)[at])) <= (ROUNDINGS + 2) * 2.0 ** -24 * float(w.abs().sum() + 3 * 28)
        step.view(-1)[at] = 0.0
    assert E.relative_position_bias(table, 0, 5).sum().requires_grad
    E.relative_position_bias(table, 0, 5).sum().backward()


def test_a_captured_backward_pass_is_refused(cuda_device):
    """With a graph of the same table alive outside the capture, autograd would end the process; the forward pass and
    relative_position_bias_grad are captured as ever."""
    from bytetransformer_b200 import encoder as E
    table = torch.randn(32, 4, device=cuda_device, requires_grad=True)
    alive = E.relative_position_bias(table, 20, 20)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            E.relative_position_bias(table, 20, 20).sum().backward()
    torch.cuda.synchronize()
    del graph
    alive.sum().backward()
    want = E.relative_position_bias_grad(torch.ones(4, 20, 20, dtype=torch.float16, device=cuda_device), 32)
    assert torch.equal(table.grad, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bias = E.relative_position_bias(table, 20, 20)
        got = E.relative_position_bias_grad(bias.detach(), 32)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(bias, alive) and torch.equal(got, E.relative_position_bias_grad(alive.detach(), 32))
