"""Packed attention with a sliding window and first tokens that stay visible, against its definition in 64 bits.

Tolerance of an output element, A = sum of p|v| over the keys (p: the softmax weights): the weights are rounded to fp16, half a
step is 2^-11 of each; weights that the row's reference puts below fp16's normal numbers lose at most 2^-25 of the largest
weight each; scores are sums of 64 products in fp32 and pass a scale and an exponential (relative error of a weight: their
absolute error, at most `slack` below, twice because the sum of weights has it too); the result is rounded to fp16, 2^-11
of it or 2^-25."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 64


def definition(q, k, v, q_off, k_off, k_lens, left, right, sinks, bias, bias_left, scale=0.125):
    """(out, tolerance) in 64 bits; rows of no sequence: NaN."""
    heads, group = q.shape[1] // D, q.shape[1] // k.shape[1]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, float("nan"))
    q_off, k_off = q_off.tolist(), k_off.tolist()
    lens = k_lens.tolist() if k_lens is not None else [b - a for a, b in zip(k_off, k_off[1:])]
    for b, n in enumerate(lens):
        rows = slice(q_off[b], q_off[b + 1])
        m = rows.stop - rows.start
        if m == 0:
            continue
        p = torch.arange(m, device=q.device)[:, None] + n - m
        j = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= (j >= p - left) | (j < sinks)
        for h in range(heads):
            c, d = slice(h * D, h * D + D), slice(h // group * D, h // group * D + D)
            if n == 0:
                out[rows, c] = tol[rows, c] = 0.0
                continue
            qq, kk, vv = q[rows, c].double(), k[k_off[b]:k_off[b] + n, d].double(), v[k_off[b]:k_off[b] + n, d].double()
            s = qq @ kk.T * scale
            if bias is not None:
                s = s + bias[h].double()[(j - p + bias_left).clamp(0, bias.shape[1] - 1)]
            w = torch.softmax(s.masked_fill(~seen, -math.inf), dim=1).nan_to_num(0.0)
            o = w @ vv
            # a bias of the type's lowest value or beyond swallows the score, here and there, to the last bit
            small = bias[bias.abs() < 1e30] if bias is not None else torch.zeros(1)
            big = float((qq.norm(dim=1).max() * kk.norm(dim=1).max() * scale)) + (float(small.abs().max()) if small.numel() else 0.0)
            slack = big * 70 * 2.0 ** -24 + 2.0 ** -21
            out[rows, c] = o
            tol[rows, c] = (w @ vv.abs()) * (2.0 ** -11 + 2 * slack) * 1.01 + \
                seen.sum(1, keepdim=True) * 2.0 ** -25 * float(vv.abs().max()) + o.abs() * 2.0 ** -11 + 2.0 ** -25
    return out, tol


def packed(lens, heads, kv, device, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    off = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(device)
    qkv = torch.randn(sum(lens) + extra, (heads + 2 * kv) * D, generator=g).half().to(device)
    q, k, v = qkv.split([heads * D, kv * D, kv * D], dim=1)
    return q, k, v, off


def check(q, k, v, q_off, k_off, max_q, max_k, k_lens=None, left=-1, right=-1, sinks=0, bias=None, bias_left=0):
    from bytetransformer_b200 import encoder as E
    got = torch.full(q.shape, 7.0, dtype=torch.float16, device=q.device)
    E.window_attention(q, k, v, q_off, k_off, max_q, max_k, left=left, right=right, sinks=sinks, k_lens=k_lens, distance_bias=bias,
                       bias_left=bias_left, out=got)
    want, tol = definition(q, k, v, q_off, k_off, k_lens, left, right, sinks, bias, bias_left)
    none = torch.isnan(want)
    assert (got[none] == 7).all()
    bad = ((got.double() - want).abs() <= tol) | none
    assert bad.all(), "%d of %d outside, first at %s, largest excess %.3g" % (
        (~bad).sum(), bad.numel(), (~bad).nonzero()[0].tolist(), ((got.double() - want).abs() / tol).nan_to_num(0).max())
    return got


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (0, 0, 1), (5, 3, 0), (31, 32, 1), (64, 64, 4), (127, 0, 16), (128, 128, 17),
           (200, 0, 4), (300, 77, 130), (-1, 60, 3), (1000, -1, 2), (1, 100000, 5)]


@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("with_bias", [False, True])
def test_packed_sequences(cuda_device, left, right, sinks, with_bias):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 200, 255, 256, 257, 300, 513, 700]
    q, k, v, off = packed(lens, 3, 3, cuda_device, seed=left + 7 * right)
    bias = torch.randn(3, 101, device=cuda_device) if with_bias else None
    check(q, k, v, off, off, 700, 700, None, left, right, sinks, bias, 40)


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 2), (8, 4), (12, 12), (16, 2)])
def test_shared_heads(cuda_device, heads, kv):
    q, k, v, off = packed([40, 333, 1], heads, kv, cuda_device, seed=heads)
    check(q, k, v, off, off, 333, 333, None, 70, 9, 3)
    check(q, k, v, off, off, 400, 500, None, -1, 0, 0, torch.randn(heads, 7, device=cuda_device), 0)


def test_long_sequences_take_over_blocks(cuda_device):
    lens = [3000, 1, 2222, 4097, 0, 128, 1500]
    q, k, v, off = packed(lens, 6, 3, cuda_device, seed=3)
    for left, right, sinks in [(-1, -1, 0), (511, 0, 4), (256, 256, 1), (1500, 0, 200)]:
        check(q, k, v, off, off, 4097, 4097, None, left, right, sinks)
    check(q, k, v, off, off, 4097, 4097, None, 700, 100, 33, torch.randn(6, 513, device=cuda_device), 256)


def test_many_short_sequences(cuda_device):
    lens = [(i * 37) % 41 for i in range(700)]
    q, k, v, off = packed(lens, 2, 1, cuda_device, seed=4)
    check(q, k, v, off, off, 40, 40, None, 8, 0, 2)
    check(q, k, v, off, off, 128, 64, None, -1, -1, 0)


@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (20, 0, 4), (600, 0, 1), (20, 5, 40), (0, 0, 0)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_queries_at_the_end_of_longer_keys(cuda_device, left, right, sinks, with_bias):
    """Parts of prompts, single tokens, sequences without keys or with fewer keys than queries, over caches with room."""
    q_lens = [1, 1, 3, 130, 17, 5, 1, 260, 9, 0, 33]
    k_lens = [1, 900, 77, 500, 0, 2, 128, 261, 3, 50, 1000]
    heads, kv, room = 4, 2, 1003
    g = torch.Generator().manual_seed(11)
    q = torch.randn(sum(q_lens), heads * D, generator=g).half().to(cuda_device)
    kv_rows = torch.full((len(k_lens) * room, 2 * kv * D), float("nan")).half()
    for b, n in enumerate(k_lens):  # what lies behind a sequence's keys is nobody's
        kv_rows[b * room:b * room + n] = torch.randn(n, 2 * kv * D, generator=g).half()
    kv_rows = kv_rows.to(cuda_device)
    k, v = kv_rows[:, :kv * D], kv_rows[:, kv * D:]
    q_off = torch.tensor([0] + q_lens).cumsum(0).int().to(cuda_device)
    k_off = (torch.arange(len(k_lens) + 1) * room).int().to(cuda_device)
    lens = torch.tensor(k_lens).int().to(cuda_device)
    bias = torch.randn(heads, 65, device=cuda_device) if with_bias else None
    check(q, k, v, q_off, k_off, 260, room, lens, left, right, sinks, bias, 32)


@pytest.mark.parametrize("left", [-1, 0, 6, 300, 5000])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (16, 4), (24, 3), (40, 2)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_single_tokens(cuda_device, left, heads, kv, with_bias):
    lens = [0, 1, 2, 15, 16, 17, 31, 64, 65, 127, 300, 1025, 4100, 6001]
    room = 6005
    g = torch.Generator().manual_seed(heads)
    q = torch.randn(len(lens), heads * D, generator=g).half().to(cuda_device)
    cache = torch.full((len(lens), room, 2 * kv * D), float("nan")).half()
    for b, n in enumerate(lens):
        cache[b, :n] = torch.randn(n, 2 * kv * D, generator=g).half()
    cache = cache.view(-1, 2 * kv * D).to(cuda_device)
    q_off = torch.arange(len(lens) + 1, dtype=torch.int32, device=cuda_device)
    bias = torch.randn(heads, 65, device=cuda_device) if with_bias else None
    check(q, cache[:, :kv * D], cache[:, kv * D:], q_off, q_off * room, 1, room, torch.tensor(lens).int().to(cuda_device), left, 0, 4,
          bias, 64)


@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (-1, 0, 0), (40, 0, 20), (3, 2, 1), (700, 9, 100), (0, 0, 0)])
@pytest.mark.parametrize("q_len,heads,kv", [(16, 3, 3), (4, 8, 2), (5, 9, 3), (2, 8, 1)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_few_queries(cuda_device, left, right, sinks, q_len, heads, kv, with_bias):
    """Drafted tokens and the like: up to q_len queries for each sequence, one range of keys or several."""
    q_lens, k_lens, room = [q_len, 1, 0, q_len, min(3, q_len), q_len], [900, 70, 5, 2, 0, 2500], 2500
    g = torch.Generator().manual_seed(q_len + heads)
    q = torch.randn(sum(q_lens), heads * D, generator=g).half().to(cuda_device)
    cache = torch.full((len(k_lens), room, 2 * kv * D), float("nan")).half()
    for b, n in enumerate(k_lens):
        cache[b, :n] = torch.randn(n, 2 * kv * D, generator=g).half()
    cache = cache.view(-1, 2 * kv * D).to(cuda_device)
    q_off = torch.tensor([0] + q_lens).cumsum(0).int().to(cuda_device)
    k_off = (torch.arange(len(k_lens) + 1) * room).int().to(cuda_device)
    bias = torch.randn(heads, 65, device=cuda_device) if with_bias else None
    check(q, cache[:, :kv * D], cache[:, kv * D:], q_off, k_off, q_len, room, torch.tensor(k_lens).int().to(cuda_device), left, right,
          sinks, bias, 32)


def test_single_tokens_of_many_sequences(cuda_device):
    """More sequences than there are ranges to cut: the result is written without the second kernel."""
    lens = [(i * 97) % 300 for i in range(700)]
    g = torch.Generator().manual_seed(2)
    q = torch.randn(700, 2 * D, generator=g).half().to(cuda_device)
    kv = torch.randn(sum(lens), 2 * D, generator=g).half().to(cuda_device)
    q_off = torch.arange(701, dtype=torch.int32, device=cuda_device)
    k_off = torch.tensor([0] + lens).cumsum(0).int().to(cuda_device)
    check(q, kv[:, :D], kv[:, D:], q_off, k_off, 1, 300, None, 200, 0, 4)


@pytest.mark.parametrize("q_len", [1, 200])
def test_a_cache_past_32_bits(cuda_device, q_len):
    """Rows whose place is more than 2^32 halves from the first."""
    rows, heads, kv = 9_000_000, 4, 4
    cache = torch.empty(rows, 2 * kv * D, dtype=torch.float16, device=cuda_device)
    lens, starts = [300, 257, 900], [0, 4_500_000, 8_999_000]
    for n, at in zip(lens, starts):
        cache[at:at + n] = torch.randn(n, 2 * kv * D, device=cuda_device).half()
    q = torch.randn(3 * q_len, heads * D, device=cuda_device).half()
    q_off = torch.arange(4, dtype=torch.int32, device=cuda_device) * q_len
    k_off = torch.tensor(starts + [rows], dtype=torch.int32, device=cuda_device)
    check(q, cache[:, :kv * D], cache[:, kv * D:], q_off, k_off, q_len, rows, torch.tensor(lens).int().to(cuda_device), 150, 0, 4)


def test_large_scores(cuda_device):
    """References that move in every tile, weights that all but one vanish."""
    q, k, v, off = packed([900, 130], 2, 2, cuda_device, seed=5)
    ramp = torch.linspace(0, 12, q.shape[0], device=cuda_device).half()[:, None]
    q, k = (q.sign() * 2).half(), (k * 0 + ramp * q[:, :2 * D].sign()[:1]).half()
    check(q, k, v, off, off, 900, 900, None, 400, 50, 2)
    check(q, k, v, off, off, 900, 900, None, -1, -1, 0, torch.linspace(-60, 60, 600, device=cuda_device).repeat(2, 1), 300)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, -60000.0])
@pytest.mark.parametrize("one", [False, True])
def test_biases_that_mask(cuda_device, low, one):
    """The type's lowest value, minus infinity: as masks by distance, and where a row sees nothing else."""
    heads = 2
    bias = torch.randn(heads, 201, device=cuda_device)
    bias[0, :60] = low       # far to the left, for a head
    bias[0, 101:103] = low
    bias[1] = low            # every distance of the other
    if one:
        q, k, v, off = packed([300, 40, 1], heads, heads, cuda_device, seed=13)
        q = q[:3]
        q_off = torch.arange(4, dtype=torch.int32, device=cuda_device)
        got = check(q, k, v, q_off, off, 1, 300, None, -1, 0, 0, bias, 100)
    else:
        q, k, v, off = packed([300, 40, 1], heads, heads, cuda_device, seed=13)
        got = check(q, k, v, off, off, 300, 300, None, 250, 250, 2, bias, 100)
    assert torch.isfinite(got).all()
    if low == -math.inf:
        assert (got[:, D:] == 0).all() and (got[:, :D] != 0).any()


def test_infinite_and_nan_queries_stay_in_their_row(cuda_device):
    q, k, v, off = packed([200, 70], 2, 2, cuda_device, seed=14)
    clean = check(q, k, v, off, off, 200, 200, None, 60, 10, 2)
    q[50, 3] = float("nan")
    q[220, D + 5] = float("inf")
    from bytetransformer_b200 import encoder as E
    got = E.window_attention(q, k, v, off, off, 200, 200, left=60, right=10, sinks=2)
    assert torch.isnan(got[50, :D]).all() and not torch.isfinite(got[220, D:]).any()
    got[50, :D] = clean[50, :D]
    got[220, D:] = clean[220, D:]
    assert torch.isfinite(got).all() and ((got - clean).abs() <= 2.0 ** -9 * clean.abs() + 2.0 ** -14).all()


def test_bounds_beyond_every_distance_are_none(cuda_device):
    from bytetransformer_b200 import encoder as E
    q, k, v, off = packed([200, 70], 2, 2, cuda_device, seed=15)
    want = E.window_attention(q, k, v, off, off, 200, 200)
    for big in (200, 1 << 30, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 3, 1 << 70):
        assert torch.equal(want, E.window_attention(q, k, v, off, off, 200, 200, left=big, right=big, sinks=big))


def test_rows_around_the_sequences_do_not_matter(cuda_device):
    """NaN and infinities in the rows of the buffers that belong to no sequence, and in queries behind the last one."""
    lens = [100, 37, 140]
    for where in (float("nan"), float("inf")):
        q, k, v, off = packed(lens, 2, 2, cuda_device, seed=6, extra=50)
        clean = check(q, k, v, off, off, 140, 140, None, 30, 30, 2)[:277].clone()
        q[277:] = where
        k[277:] = where
        v[277:] = where
        from bytetransformer_b200 import encoder as E
        for left, right, sinks in [(30, 30, 2), (-1, -1, 0)]:
            got = E.window_attention(q, k, v, off, off, 140, 140, left=left, right=right, sinks=sinks)
            assert torch.isfinite(got[:277]).all()
            if left == 30:
                assert torch.equal(got[:277], clean)


def test_without_keys(cuda_device):
    from bytetransformer_b200 import encoder as E
    q = torch.randn(10, 2 * D, device=cuda_device).half()
    k = torch.empty(0, 2 * D, device=cuda_device, dtype=torch.float16)
    q_off = torch.tensor([0, 3, 10], dtype=torch.int32, device=cuda_device)
    k_off = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    assert (E.window_attention(q, k, k, q_off, k_off, 7, 0) == 0).all()
    assert E.window_attention(q[:0], k, k, q_off, k_off, 7, 0).shape == (0, 2 * D)


def test_the_same_every_time_and_with_other_neighbours(cuda_device):
    from bytetransformer_b200 import encoder as E
    q, k, v, off = packed([500, 1100, 90], 4, 4, cuda_device, seed=7)
    first = E.window_attention(q, k, v, off, off, 1100, 1100, left=200, right=0, sinks=4)
    for _ in range(5):
        assert torch.equal(first, E.window_attention(q, k, v, off, off, 1100, 1100, left=200, right=0, sinks=4))
    alone = torch.tensor([0, 1100], dtype=torch.int32, device=cuda_device)
    got = E.window_attention(q[500:1600], k[500:1600], v[500:1600], alone, alone, 1100, 1100, left=200, right=0, sinks=4)
    assert torch.equal(got, first[500:1600])


def test_offsets_that_fit_no_rows_are_reported(cuda_device):
    from bytetransformer_b200 import encoder as E
    from helpers import make_layer_weights, to_device_weights
    enc = E.Encoder(2, D, [to_device_weights(make_layer_weights(2 * D, torch.Generator().manual_seed(0)), cuda_device)])
    q, k, v, off = packed([100, 50, 60], 2, 2, cuda_device, seed=8)
    good = E.window_attention(q, k, v, off, off, 100, 100, left=10, right=10)
    assert enc.device_status() == 0
    cases = [([0, 100, 150, 500], [0, 100, 150, 210], None), ([0, 100, 90, 210], [0, 100, 150, 210], None),
             ([-5, 100, 150, 210], [0, 100, 150, 210], None), ([0, 100, 150, 210], [0, 100, 150, 211], None),
             ([0, 100, 150, 210], [0, 100, 40, 210], None), ([0, 100, 150, 210], [0, 100, 150, 210], [100, 51, 60]),
             ([0, 100, 150, 210], [0, 100, 150, 210], [100, -1, 60])]
    for q_off, k_off, k_lens in cases:
        out = torch.full_like(good, 7.0)
        as_ints = [torch.tensor(t, dtype=torch.int32, device=cuda_device) if t is not None else None for t in (q_off, k_off, k_lens)]
        E.window_attention(q, k, v, as_ints[0], as_ints[1], 100, 100, left=10, right=10, k_lens=as_ints[2], out=out)
        assert enc.device_status() == 0x301 and enc.device_status() == 0
        if q_off[1:2] == [100] and q_off[0] == 0 and k_off[1] == 100:
            assert torch.equal(out[:100], good[:100])
    for max_q, max_k in [(99, 100), (100, 99)]:
        E.window_attention(q, k, v, off, off, max_q, max_k, left=10, right=10)
        assert enc.device_status() == 0x301
    assert torch.equal(good, E.window_attention(q, k, v, off, off, 100, 100, left=10, right=10)) and enc.device_status() == 0


def test_another_stream_a_captured_graph_and_two_at_once(cuda_device):
    from bytetransformer_b200 import encoder as E
    q, k, v, off = packed([300, 20, 410], 4, 2, cuda_device, seed=9)
    bias = torch.randn(4, 33, device=cuda_device)

    def call(q):
        return (E.window_attention(q, k, v, off, off, 410, 410, left=100, right=20, sinks=2),
                E.window_attention(q, k, v, off, off, 410, 410, left=50, distance_bias=bias, bias_left=16))
    want = call(q)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call(q))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = call(q)
    lens2 = torch.tensor([0, 310, 330, 730], dtype=torch.int32, device=cuda_device)
    off.copy_(lens2)  # other lengths below the same bounds
    graph.replay()
    torch.cuda.synchronize()
    want2 = call(q)
    assert torch.equal(res[0], want2[0]) and torch.equal(res[1], want2[1]) and not torch.equal(res[0], want[0])


def test_agrees_with_the_packed_attention(cuda_device):
    """No window, no bias: what bt_attention computes; the two round alike but walk their keys differently."""
    from bytetransformer_b200 import encoder as E
    from helpers import make_layer_weights, to_device_weights
    heads = 4
    enc = E.Encoder(heads, D, [to_device_weights(make_layer_weights(heads * D, torch.Generator().manual_seed(0)), cuda_device)])
    q, k, v, off = packed([129, 64, 500], heads, heads, cuda_device, seed=10)
    qkv = torch.cat([q, k, v], dim=1).contiguous()
    want, tol = definition(q, k, v, off, off, None, -1, -1, 0, None, 0)
    got = E.window_attention(q, k, v, off, off, 500, 500)
    assert ((enc.attention(qkv, off, 500).double() - got.double()).abs() <= 2 * tol).all()


def test_a_layer_of_local_attention(cuda_device):
    """The operators together, as an encoder layer with relative positions runs them: norm, QKV product, windowed attention with
    the learned bias by distance, output product, norm with the residual."""
    from bytetransformer_b200 import _abi
    from bytetransformer_b200 import encoder as E
    from helpers import make_layer_weights, to_device_weights
    heads, lens = 4, [70, 200, 33]
    H, T = heads * D, sum(lens)
    g = torch.Generator().manual_seed(12)
    w = to_device_weights(make_layer_weights(H, g), cuda_device)
    enc = E.Encoder(heads, D, [w])
    off = torch.tensor([0] + lens).cumsum(0).int().to(cuda_device)
    x, r = (torch.randn(T, H, generator=g).half().to(cuda_device) for _ in range(2))
    gamma = (1 + 0.1 * torch.randn(H, generator=g)).half().to(cuda_device)
    table = torch.randn(32, heads, generator=g).to(cuda_device)
    bias = E.relative_position_bias(table, 1, 257, q_start=128, out_dtype=torch.float32).view(heads, 257)
    y, total = E.add_residual_rmsnorm(x, r, gamma)
    qkv = enc.gemm(y, w[0], w[1], epilogue=_abi.BT_EPI_BIAS)
    q, k, v = qkv.split([H, H, H], dim=1)
    ctx = E.window_attention(q, k, v, off, off, 200, 200, left=40, right=40, sinks=1, distance_bias=bias, bias_left=128)
    z = enc.gemm(ctx, w[2], w[3], epilogue=_abi.BT_EPI_BIAS)
    out, _ = E.add_residual_rmsnorm(z, total, gamma)
    # step by step in 64 bits, each from the rounded result of the one before
    s = x.double() + r.double()
    want = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * gamma.double()
    assert ((y.double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25).all()
    want, tol = definition(q, k, v, off, off, None, 40, 40, 1, bias, 128)
    assert ((ctx.double() - want).abs() <= tol).all()
    # the dense bias of the same table gives the same scores through the general path's layout
    dense = E.relative_position_bias(table, 200, 200, out_dtype=torch.float32)
    at = torch.arange(200)
    assert torch.equal(dense, bias[:, (at[None, :] - at[:, None] + 128).clamp(0, 256).to(cuda_device)])
    s = z.double() + total.double()
    want = s * torch.rsqrt((s * s).mean(1, keepdim=True) + 1e-6) * gamma.double()
    assert ((out.double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25).all()


def test_python_refusals(cuda_device):
    from bytetransformer_b200 import BtError
    from bytetransformer_b200 import encoder as E
    q, k, v, off = packed([20], 4, 2, cuda_device)
    call = E.window_attention
    with pytest.raises(RuntimeError, match="Tensor type: q"):
        call(q.float(), k, v, off, off, 20, 20)
    with pytest.raises(RuntimeError, match="k must be"):
        call(q, k[:, :60], v, off, off, 20, 20)
    with pytest.raises(RuntimeError, match="same shape"):
        call(q, k, v[:10], off, off, 20, 20)
    with pytest.raises(RuntimeError, match="q_offsets"):
        call(q, k, v, off.long(), off, 20, 20)
    with pytest.raises(RuntimeError, match="batch"):
        call(q, k, v, off, off[:1], 20, 20)
    with pytest.raises(RuntimeError, match="Tensor type: v"):
        call(q, k, v.float(), off, off, 20, 20)
    with pytest.raises(RuntimeError, match="v must be"):
        call(q, k, torch.empty(2 * D, 20, device=cuda_device, dtype=torch.float16).t(), off, off, 20, 20)
    with pytest.raises(RuntimeError, match="k_lens"):
        call(q, k, v, off, off, 20, 20, k_lens=off)
    with pytest.raises(RuntimeError, match="distance_bias"):
        call(q, k, v, off, off, 20, 20, distance_bias=torch.zeros(3, 5, device=cuda_device))
    with pytest.raises(RuntimeError, match="out must"):
        call(q, k, v, off, off, 20, 20, out=torch.empty(19, 4 * D, device=cuda_device, dtype=torch.float16))
    with pytest.raises(BtError):  # three heads cannot share two
        call(q[:, :3 * D], k, v, off, off, 20, 20)
    with pytest.raises(BtError):
        call(q, k, v, off, off, 20, 20, scale=0.0)
    with pytest.raises(BtError):  # rows that start anywhere
        call(torch.zeros(20, 4 * D + 4, device=cuda_device, dtype=torch.float16)[:, :4 * D], k, v, off, off, 20, 20)


def poisoned(q, k, v, off, k_off, max_q, max_k, rows, where, k_lens=None, **how):
    """Puts `where` into rows of k and v.  Rows of q that see none of them come out as without it (against the definition in
    64 bits); those that see one do not stay finite in the dimensions of v that hold it."""
    from bytetransformer_b200 import encoder as E
    args = {"left": -1, "right": -1, "sinks": 0, "bias": None, "bias_left": 0, **how}
    k, v = k.clone(), v.clone()
    k[rows], v[rows] = 0.0, 0.0
    group = q.shape[1] // k.shape[1]
    want, tol = definition(q, k, v, off, k_off, k_lens, *(args[n] for n in ("left", "right", "sinks", "bias", "bias_left")))
    mark = torch.zeros_like(v)
    mark[rows] = 1.0  # 1 of v: the weight of what is poisoned
    ask = {"left": args["left"], "right": args["right"], "sinks": args["sinks"], "k_lens": k_lens, "distance_bias": args["bias"],
           "bias_left": args["bias_left"]}
    weight = definition(q, k, mark, off, k_off, k_lens, *(args[n] for n in ("left", "right", "sinks", "bias", "bias_left")))[0]
    sees = (weight != 0).view(len(q), -1, D).any(2)  # [row, head]
    v[rows, 1::3] = where
    for poison_keys in (False, True):
        if poison_keys:
            k[rows, 5::7] = where
        got = E.window_attention(q, k, v, off, k_off, max_q, max_k, **ask).double()
        ok = ((got - want).abs() <= tol) | torch.isnan(want)
        ok = ok.view(len(q), -1, D)
        assert ok[~sees].all(), ((~ok).any(2) & ~sees).nonzero()[:8].tolist()
        hit = torch.zeros(v.shape[1], dtype=torch.bool, device=q.device)
        hit[1::3] = True
        hit = hit.view(-1, D).repeat_interleave(group, 0)  # [head, dimension]
        if not poison_keys:  # (a score that infinities in k make -inf leaves its key without weight)
            assert not torch.isfinite(got.view(len(q), -1, D)[sees[:, :, None] & hit[None]]).any()
    return sees


@pytest.mark.parametrize("where", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (70, 0, 0), (70, 0, 4), (3, 5, 40), (0, 0, 1)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_what_a_row_does_not_see_does_not_matter(cuda_device, where, left, right, sinks, with_bias):
    lens = [300, 1, 700, 130]
    q, k, v, off = packed(lens, 4, 2, cuda_device, seed=21)
    bias = torch.randn(4, 33, device=cuda_device) if with_bias else None
    how = {"left": left, "right": right, "sinks": sinks, "bias": bias, "bias_left": 16}
    for rows in ([299], [100, 301, 650], [4, 39, 305, 340, 1130], [64, 365, 1001 + 64]):
        sees = poisoned(q, k, v, off, off, 700, 700, rows, where, **how)
        assert sees.any() and not sees.all()


@pytest.mark.parametrize("where", [math.inf, math.nan])
@pytest.mark.parametrize("batch,room", [(3, 500), (12, 4000), (300, 200)])
@pytest.mark.parametrize("q_len,left,right,sinks", [(1, 60, 0, 4), (3, -1, 0, 0), (4, 20, 0, 33), (2, 60, 1, 5)])
def test_what_a_token_does_not_see_does_not_matter(cuda_device, batch, room, q_len, left, right, sinks, where):
    """Caches with what has left the window, tokens that follow one another; one range of keys, clusters, the second kernel."""
    heads, kv = 8, 2
    g = torch.Generator().manual_seed(22)
    q = torch.randn(batch * q_len, heads * D, generator=g).half().to(cuda_device)
    kv_rows = torch.randn(batch * room, 2 * kv * D, generator=g).half().to(cuda_device)
    lens = torch.randint(room // 2, room + 1, (batch,), generator=g)
    off = torch.arange(batch + 1, dtype=torch.int32, device=cuda_device) * q_len
    k_off = torch.arange(batch + 1, dtype=torch.int32, device=cuda_device) * room
    firsts = torch.arange(batch) * room
    lens_dev = lens.int().to(cuda_device)
    for spots in ([lens - 1], [firsts * 0 + 6, lens - 75], [firsts * 0 + 31, lens - 62, lens - 2]):
        rows = torch.cat([firsts + s for s in spots])[::2].tolist()
        poisoned(q, kv_rows[:, :kv * D], kv_rows[:, kv * D:], off, k_off, q_len, room, rows, where, k_lens=lens_dev, left=left, right=right,
                 sinks=sinks)


def test_what_a_bias_hides_does_not_matter(cuda_device):
    q, k, v, off = packed([300, 90], 2, 1, cuda_device, seed=23)
    bias = torch.randn(2, 201, device=cuda_device)
    bias[0, :70] = bias[1, 120:150] = -math.inf
    for where in (math.inf, math.nan):
        poisoned(q, k, v, off, off, 300, 300, [40, 200, 350], where, bias=bias, bias_left=100)
        ones = torch.arange(3, dtype=torch.int32, device=cuda_device)
        poisoned(q[:2], k, v, ones, off, 1, 300, [180, 350], where, bias=bias, bias_left=100)


def test_many_rows_that_do_not_see_something(cuda_device):
    """Every item of blocks that take over one another holds what some of its rows must not see."""
    lens = [(i * 53) % 400 + 1 for i in range(70)]
    q, k, v, off = packed(lens, 8, 4, cuda_device, seed=24)
    firsts = torch.tensor([0] + lens).cumsum(0)[:-1]
    rows = torch.cat([firsts + torch.tensor(lens) - 1, (firsts + 127)[torch.tensor(lens) > 128]]).tolist()
    poisoned(q, k, v, off, off, 400, 400, rows, math.nan, left=-1, right=0, sinks=0)
    poisoned(q, k, v, off, off, 400, 400, rows, math.inf, left=90, right=0, sinks=3)


def swallowed(q, k, v, off, rows_of, left, right, bias, bias_left):
    """`definition` where a bias of 1e9 and more leaves nothing of a score in single precision (a step is 128 there in the kernels' log2
    units, so a score of less than 44 changes nothing): such keys weigh by their bias alone.  A smaller bias costs a score half a
    step of the sum, twice because the sum of weights has it too."""
    heads, group = q.shape[1] // D, q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    ends = off.tolist()
    for b, (first, last) in enumerate(rows_of):
        n, m = ends[b + 1] - ends[b], last - first
        p = torch.arange(m, device=q.device)[:, None] + n - m
        j = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones(m, n, dtype=torch.bool, device=q.device)
        if right >= 0:
            seen &= j <= p + right
        if left >= 0:
            seen &= j >= p - left
        for h in range(heads):
            c, d = slice(h * D, h * D + D), slice(h // group * D, h // group * D + D)
            qq, kk, vv = (t.double() for t in (q[first:last, c], k[ends[b]:ends[b + 1], d], v[ends[b]:ends[b + 1], d]))
            s = qq @ kk.t() * 0.125
            assert float(s.abs().max()) < 44
            add = bias[h].double()[(j - p + bias_left).clamp(0, bias.shape[1] - 1)]
            low = add.abs() >= 1e9
            w = torch.softmax((torch.where(low, 0.0, s) + add).masked_fill(~seen, -math.inf), dim=1)
            finite = torch.where(low, 0.0, add)
            slack = float(qq.norm(dim=1).max() * kk.norm(dim=1).max() * 0.125) * 70 * 2.0 ** -24 + 2.0 ** -21
            slack = slack + float(finite.abs().max()) * 2.0 ** -23
            out[first:last, c] = w @ vv
            tol[first:last, c] = (w @ vv.abs()) * (2.0 ** -11 + 2 * slack) * 1.01 + \
                seen.sum(1, keepdim=True) * 2.0 ** -25 * float(vv.abs().max()) + (w @ vv).abs() * 2.0 ** -11 + 2.0 ** -25
    return out, tol


@pytest.mark.parametrize("low", [-1e4, -1e5, -1e9, -1e12, -1e29, 1e9, 1e12])
@pytest.mark.parametrize("side", ["left", "right", "both"])
@pytest.mark.parametrize("left,right", [(-1, -1), (-1, 0), (400, 300)])
@pytest.mark.parametrize("last", [0, 1])
def test_biases_that_swallow_the_scores(cuda_device, low, side, left, right, last):
    """Masks by distance like -1e9: whole tiles of nothing else ahead of, behind and between tiles with other biases, and rows that
    see nothing else, with scores far beyond fp16's range of exponents.  last: one query for each sequence."""
    from bytetransformer_b200 import encoder as E
    lens = [700, 260, 64]
    q, k, v, off = packed(lens, 2, 1, cuda_device, seed=31)
    q, k = (q * 2.2).half(), (k * 2.2).half()
    bias = torch.randn(2, 201, device=cuda_device)
    if side in ("left", "both"):
        bias[:, :70] = low
    if side in ("right", "both"):
        bias[:, 140:] = low
    bias[1] = low
    ends = off.tolist()
    if last:
        rows = [(i, i + 1) for i in range(3)]
        q = torch.stack([q[e - 1] for e in ends[1:]])
        q_off = torch.arange(4, dtype=torch.int32, device=cuda_device)
    else:
        rows, q_off = list(zip(ends, ends[1:])), off
    want, tol = swallowed(q, k, v, off, rows, left, right, bias, 100)
    got = E.window_attention(q, k, v, q_off, off, 1 if last else 700, 700, left=left, right=right, distance_bias=bias, bias_left=100)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist(), int((~torch.isfinite(got)).sum()))


@pytest.mark.parametrize("batch,room", [(3, 100), (2, 1500), (40, 3000), (300, 200)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_nan_in_a_token_or_in_a_key_that_it_sees_reaches_the_result(cuda_device, batch, room, with_bias):
    """One range of keys, clusters, the second kernel: a range, or a warp's share of one, all of whose scores are NaN is not one in which
    nothing is seen.  Other rows keep every bit."""
    from bytetransformer_b200 import encoder as E
    heads, kv = 8, 8
    g = torch.Generator().manual_seed(41)
    q = torch.randn(batch, heads * D, generator=g).half().to(cuda_device)
    cache = torch.randn(batch * room, 2 * kv * D, generator=g).half().to(cuda_device)
    off = torch.arange(batch + 1, dtype=torch.int32, device=cuda_device)
    bias = torch.randn(heads, 65, generator=g).to(cuda_device) if with_bias else None

    def call(q, cache, left):
        return E.window_attention(q, cache[:, :kv * D], cache[:, kv * D:], off, off * room, 1, room, left=left, right=0, distance_bias=bias,
                                  bias_left=64).view(batch, heads, D)
    for left in (-1, room // 2, 0):
        clean = call(q, cache, left)
        assert torch.isfinite(clean).all()
        sick = q.clone().view(batch, heads, D)
        sick[1, 2, 7] = sick[batch - 1, 0, 63] = float("nan")
        got = call(sick.view(batch, -1), cache, left)
        rows = torch.zeros(batch, heads, dtype=torch.bool, device=cuda_device)
        rows[1, 2] = rows[batch - 1, 0] = True
        assert torch.isnan(got[rows]).all() and torch.equal(got[~rows], clean[~rows])
        sick = cache.clone()
        sick[2 * room - 1, 2 * D + 9] = float("nan")  # the key of the token itself, for a head
        got = call(q, sick, left)
        rows[batch - 1, 0] = False
        assert torch.isnan(got[rows]).all() and torch.equal(got[~rows], clean[~rows])


def test_a_single_row_of_any_stride(cuda_device):
    """torch leaves the stride of a dimension of one element to chance: one token, one key, a result of one row."""
    from bytetransformer_b200 import encoder as E

    def row(t, stride):
        return t.reshape(1, -1).as_strided((1, t.numel()), (stride, 1))
    g = torch.Generator().manual_seed(51)
    q = torch.randn(1, 4 * D, generator=g).half().to(cuda_device)
    k, v = (torch.randn(30, 2 * D, generator=g).half().to(cuda_device) for _ in range(2))
    one = torch.tensor([0, 1], dtype=torch.int32, device=cuda_device)
    ends = torch.tensor([0, 30], dtype=torch.int32, device=cuda_device)
    want = E.window_attention(q, k, v, one, ends, 1, 30)
    want_one = E.window_attention(q, k[:1], v[:1], one, one, 1, 1)
    for stride in (0, 1, 7, 10 ** 6, 1 << 40):
        out = torch.empty_like(q)
        E.window_attention(row(q, stride), k, v, one, ends, 1, 30, out=row(out, stride))
        assert torch.equal(out, want)
        assert torch.equal(E.window_attention(q, row(k[0], stride), row(v[0], stride), one, one, 1, 1), want_one)
    many = torch.randn(200, 4 * D, generator=g).half().to(cuda_device)  # the block kernel over one key
    offs = torch.tensor([0, 200], dtype=torch.int32, device=cuda_device)
    assert torch.equal(E.window_attention(many, row(k[0], 1), row(v[0], 1), offs, one, 200, 1),
                       E.window_attention(many, k[:1], v[:1], offs, one, 200, 1))


def test_a_batch_without_queries(cuda_device):
    """The longest of no queries at all is 0: nothing is written."""
    from bytetransformer_b200 import encoder as E
    q, k, v, off = packed([30, 20], 4, 2, cuda_device, seed=52)
    none = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    out = torch.full_like(q, 7.0)
    assert E.window_attention(q, k, v, none, off, 0, 30, out=out) is out and (out == 7).all()
    assert (E.window_attention(q, k, v, none, off, 1, 30, out=out) == 7).all()
    assert E.window_attention(q, k, v, none, off, 0, 30).shape == q.shape


@pytest.mark.parametrize("size", [1.0, 30.0, 1000.0, 60000.0])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("q_len", [0, 1])
def test_scores_up_to_the_largest_that_halves_can_make(cuda_device, size, sign, with_bias, q_len):
    """Scores of up to 3e10, where a step of single precision is 2,048, all of one sign and either equal or so far apart that a row
    takes the values of the keys with the largest, weighed by their biases.  q_len 1: one query for each sequence.  The weights of those
    keys and their sum are rounded to fp16 in the one place: half a step of each, and of the result.  A bias loses half a step of its sum
    with the score, twice as the sum of weights has it too; where that leaves nothing of it, the result lies between those values."""
    from bytetransformer_b200 import encoder as E
    lens, heads = [700, 129, 64], 2
    g = torch.Generator().manual_seed(71)
    q, k, v, off = packed(lens, heads, heads, cuda_device, seed=71)
    T = sum(lens)
    signs = torch.randint(0, 2, (heads * D,), generator=g).mul(2).sub(1).half().to(cuda_device)
    ramp = (64 + 84 * torch.randperm(T, generator=g)[:T].float()).clamp(max=60000).half().to(cuda_device)
    q = (signs * sign * size).expand(T, -1).contiguous()
    k = ramp[:, None] * signs
    bias = torch.randn(heads, 65, device=cuda_device) if with_bias else None
    lost = 64 * size * 60000 * 0.125 * 2.0 ** -23 if with_bias else 0.0
    ends, ones = off.tolist(), torch.arange(4, dtype=torch.int32, device=cuda_device)
    last = [e - 1 for e in ends[1:]]
    for left, right in [(-1, -1), (-1, 0), (100, 30)]:
        if q_len:
            got = E.window_attention(q[last], k, v, ones, off, 1, 700, left=left, right=right, distance_bias=bias, bias_left=32)
        else:
            got = E.window_attention(q, k, v, off, off, 700, 700, left=left, right=right, distance_bias=bias, bias_left=32)
        for b, (first, end) in enumerate(zip(ends, ends[1:])):
            p = torch.arange(end - first, device=cuda_device)[:, None]
            d = p.t() - p
            seen = ((d <= right) | (right < 0)) & ((d >= -left) | (left < 0))
            for h in range(heads):
                c = slice(h * D, h * D + D)
                score = (64 * 0.125 * size * sign * ramp[first:end].double()).expand(end - first, -1)
                if with_bias:
                    score = score + bias[h].double()[(d + 32).clamp(0, 64)]
                w = torch.softmax(score.masked_fill(~seen, -math.inf), 1)
                vv = v[first:end, c].double()
                want, whole = w @ vv, w @ vv.abs()
                if lost < 0.25:
                    off_by = whole * (2.0 ** -11 + 2 * lost * ((w > 0).sum(1, keepdim=True) > 1))
                else:
                    high = torch.where((w > 0)[:, :, None], vv[None], -math.inf).amax(1)
                    low = torch.where((w > 0)[:, :, None], vv[None], math.inf).amin(1)
                    want, off_by = (high + low) / 2, (high - low) / 2 + torch.maximum(high.abs(), low.abs()) * 2.0 ** -11
                off_by = off_by * 1.01 + want.abs() * 2.0 ** -11 + 2.0 ** -25
                mine = got[b:b + 1, c] if q_len else got[first:end, c]
                ok = (mine.double() - want[-len(mine):]).abs() <= off_by[-len(mine):]
                assert ok.all(), (left, right, b, h, int((~ok).sum()), int((~torch.isfinite(mine)).sum()))
