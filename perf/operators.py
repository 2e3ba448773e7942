"""What is measured of the operators around an encoder layer with relative positions: the learned relative position
bias by buckets and its gradient, the root-mean-square norm with the residual's addition, and the packed attention
with a sliding window and first tokens that stay visible.

`own` false: the plain form, elementary torch operations.  `own` true: the package's entry points.
"""
import math
import random

import torch

own = False

HEAD = 64


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one short sequence: the bias of a call where latency is everything
        {"name": "bias_12h_64", "op": "bias", "heads": 12, "q": 64, "k": 64, "start": 0, "buckets": 32, "dist": 128,
         "both": True, "f32": False},
        # the longest dense bias that the general-mask path takes, 16 heads
        {"name": "bias_16h_1024", "op": "bias", "heads": 16, "q": 1024, "k": 1024, "start": 0, "buckets": 32,
         "dist": 128, "both": True, "f32": False},
        # the second part of a one-sided sequence, odd lengths: rows start at every alignment
        {"name": "bias_odd_777_1543", "op": "bias", "heads": 12, "q": 777, "k": 1543, "start": 766, "buckets": 48,
         "dist": 400, "both": False, "f32": False},
        # fine-tuning on short odd sequences: every score's gradient of eight sequences
        {"name": "grad_8x12h_197", "op": "grad", "batch": 8, "heads": 12, "q": 197, "k": 197, "start": 0,
         "buckets": 32, "dist": 128, "both": True, "f32": False},
        # the same at full length and a large batch
        {"name": "grad_16x16h_1024", "op": "grad", "batch": 16, "heads": 16, "q": 1024, "k": 1024, "start": 0,
         "buckets": 32, "dist": 128, "both": True, "f32": False},
        # a short request: 48 tokens of a 768-wide model
        {"name": "norm_48x768", "op": "norm", "rows": 48, "hidden": 768, "f32": False, "res": True, "group": -1},
        # the fp32 sums of a GEMM, normalised into 8-bit values with a scale for each 128 columns; odd row count
        {"name": "norm_18645x1024_e4m3", "op": "norm", "rows": 18645, "hidden": 1024, "f32": True, "res": True,
         "group": 128},
        # a whole micro-batch of the benchmark's size
        {"name": "norm_75776x768", "op": "norm", "rows": 75776, "hidden": 768, "f32": False, "res": True, "group": -1},
        # a small batch of short sequences, local attention on both sides
        {"name": "window_16x128", "op": "window", "batch": 16, "heads": 12, "kv": 12, "len": 128, "least": 16,
         "left": 32, "right": 32, "sinks": 1, "bias": False, "one": False, "lens": 1},
        # long documents of ragged lengths, local attention with the relative position bias
        {"name": "window_8x4096_bias", "op": "window", "batch": 8, "heads": 12, "kv": 12, "len": 4096, "least": 500,
         "left": 256, "right": 256, "sinks": 1, "bias": True, "one": False, "lens": 2},
        # one long sequence seen from the left only, heads that share keys and values
        {"name": "window_1x8192_shared", "op": "window", "batch": 1, "heads": 16, "kv": 4, "len": 8192, "least": 8192,
         "left": 2047, "right": 0, "sinks": 4, "bias": False, "one": False, "lens": 3},
        # one new token for each of 64 sequences over their caches
        {"name": "window_token_64x32768", "op": "window", "batch": 64, "heads": 16, "kv": 4, "len": 32768,
         "least": 100, "left": 4095, "right": 0, "sinks": 4, "bias": False, "one": True, "lens": 4},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["bias", "grad", "norm", "window", "window", "token"])
    if op in ("bias", "grad"):
        both = rng.random() < 0.6
        case = {"op": op, "heads": rng.choice([1, 4, 8, 12, 16]), "q": _log(rng, 1, 1100), "k": _log(rng, 1, 1600),
                "start": rng.choice([0, rng.randrange(0, 2000)]), "buckets": 2 * rng.randrange(4, 33),
                "dist": _log(rng, 70, 1000), "both": both, "f32": rng.random() < 0.3}
        if op == "grad":
            case["batch"] = rng.choice([1, 1, 2, 5, 8])
        return case
    if op == "norm":
        hidden = 8 * _log(rng, 4, 1024)
        return {"op": "norm", "rows": _log(rng, 1, min(40000, 50000000 // hidden)), "hidden": hidden,
                "f32": rng.random() < 0.4, "res": rng.random() < 0.8, "group": rng.choice([-1, -1, 0, 128])}
    kv = rng.choice([1, 2, 4, 6])
    case = {"op": "window", "heads": kv * rng.choice([1, 1, 2, 4]), "kv": kv, "sinks": rng.choice([0, 1, 4, 16, 40]),
            "bias": rng.random() < 0.4, "lens": rng.randrange(10 ** 6)}
    if op == "token":
        length = _log(rng, 1, 30000)
        return dict(case, batch=_log(rng, 1, 48), len=length, least=rng.choice([0, length]), right=0, one=True,
                    left=rng.choice([-1, _log(rng, 1, 8000)]))
    length = _log(rng, 1, 4000)
    batch = max(1, min(_log(rng, 1, 64), 800000000 // (case["heads"] * length * length)))
    return dict(case, batch=batch, len=length, least=rng.choice([1, length]), one=False,
                left=rng.choice([-1, _log(rng, 1, 2000)]), right=rng.choice([0, -1, _log(rng, 1, 2000)]))


def _lens(case):
    """Keys of each sequence: part of the case, so that the work is the case's alone."""
    r = random.Random(case["lens"])
    return [r.randint(case["least"], case["len"]) for _ in range(case["batch"])]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float16, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = {"case": case}
    dtype = torch.float32 if case.get("f32") else torch.float16
    if case["op"] == "bias":
        s["table"] = normal(case["buckets"], case["heads"], dtype=dtype)
    elif case["op"] == "grad":
        s["grad"] = normal(case["batch"], case["heads"], case["q"], case["k"], dtype=dtype, scale=0.02)
    elif case["op"] == "norm":
        s["x"] = normal(case["rows"], case["hidden"], dtype=dtype, scale=0.5)
        s["residual"] = normal(case["rows"], case["hidden"], scale=2.0) if case["res"] else None
        s["gamma"] = normal(case["hidden"], scale=0.1) + 1.0
    else:
        lens, heads, kv = _lens(case), case["heads"], case["kv"]
        if case["one"]:  # caches with room for `len` keys each; one query for each sequence
            rows = case["batch"] * case["len"]
            s["q"] = normal(case["batch"], heads * HEAD)
            keys = normal(rows, 2 * kv * HEAD)
            s["k"], s["v"] = keys[:, :kv * HEAD], keys[:, kv * HEAD:]
            s["q_offsets"] = torch.arange(case["batch"] + 1, dtype=torch.int32, device="cuda")
            s["k_offsets"] = s["q_offsets"] * case["len"]
            s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            s["max_q"] = 1
        else:  # the packed output of one product: queries, keys and values side by side
            offsets = [0]
            for n in lens:
                offsets.append(offsets[-1] + n)
            qkv = normal(offsets[-1], (heads + 2 * kv) * HEAD)
            s["q"], s["k"], s["v"] = qkv.split([heads * HEAD, kv * HEAD, kv * HEAD], dim=1)
            s["q_offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
            s["k_offsets"], s["k_lens"], s["max_q"] = s["q_offsets"], None, case["len"]
        # distances -128 .. 128, the nearest ones telling most apart
        s["bias"] = normal(heads, 257, dtype=torch.float32) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"bias": _plain_bias, "grad": _plain_grad, "norm": _plain_norm, "window": _plain_window}[case["op"]](s, case)


def _own(s, case):
    from bytetransformer_b200 import encoder as bt
    if case["op"] == "bias":
        return bt.relative_position_bias(s["table"], case["q"], case["k"], max_distance=case["dist"],
                                         bidirectional=case["both"], q_start=case["start"])
    if case["op"] == "grad":
        return bt.relative_position_bias_grad(s["grad"], case["buckets"], max_distance=case["dist"],
                                              bidirectional=case["both"], q_start=case["start"])
    if case["op"] == "norm":
        if case["group"] < 0:
            out, total = bt.add_residual_rmsnorm(s["x"], s["residual"], s["gamma"])
            return (out, total) if total is not None else (out,)
        out, scales, total = bt.add_residual_rmsnorm_e4m3(s["x"], s["residual"], s["gamma"], group=case["group"])
        out = out.to(torch.float16)  # the values that the 8 bits stand for
        return (out, scales, total) if total is not None else (out, scales)
    return bt.window_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["max_q"], case["len"],
                               left=case["left"], right=case["right"], sinks=case["sinks"], k_lens=s["k_lens"],
                               distance_bias=s["bias"], bias_left=128)


def _buckets(case, device):
    """The bucket of every (query, key), by the formula in 64 bits.  A distance on a border has a whole number there."""
    d = torch.arange(case["k"], device=device)[None, :] - torch.arange(case["q"], device=device)[:, None] - case["start"]
    count = case["buckets"] // 2 if case["both"] else case["buckets"]
    n = d.abs() if case["both"] else (-d).clamp(min=0)
    exact = count // 2
    step = torch.log(n.clamp(min=1).double() / exact) / math.log(case["dist"] / exact) * (count - exact)
    far = (exact + torch.floor(step + 1e-9).long()).clamp(max=count - 1)
    return torch.where(n < exact, n, far) + ((d > 0).long() * count if case["both"] else 0)


def _plain_bias(s, case):
    table = s["table"].float()[_buckets(case, s["table"].device)]
    return table.permute(2, 0, 1).contiguous().to(torch.float16)


def _plain_grad(s, case):
    total = s["grad"].double().sum(0).reshape(case["heads"], -1)
    member = _buckets(case, total.device).reshape(-1, 1) == torch.arange(case["buckets"], device=total.device)
    return (total @ member.double()).t().contiguous().float()


def _plain_norm(s, case):
    total = s["x"].float()
    if s["residual"] is not None:
        total = total + s["residual"].float()
    y = total * torch.rsqrt((total * total).mean(1, keepdim=True) + 1e-6) * s["gamma"].float()
    extra = (total.to(torch.float16),) if s["residual"] is not None else ()
    if case["group"] < 0:
        return (y.to(torch.float16),) + extra
    rows, hidden = y.shape
    group = case["group"] or hidden
    parts = -(-hidden // group)
    padded = torch.nn.functional.pad(y, (0, parts * group - hidden)).view(rows, parts, group)
    scale = padded.abs().amax(2).clamp(min=2.0 ** -100) / 448.0
    value = (padded / scale[:, :, None]).clamp(-448.0, 448.0).view(rows, -1)[:, :hidden]
    return (value.to(torch.float8_e4m3fn).to(torch.float16), scale) + extra


def _plain_window(s, case):
    heads, kv, device = case["heads"], case["kv"], s["q"].device
    q_off, k_off = s["q_offsets"].long(), s["k_offsets"].long()
    q_len = q_off[1:] - q_off[:-1]
    k_len = s["k_lens"].long() if s["k_lens"] is not None else k_off[1:] - k_off[:-1]
    qi = torch.arange(s["max_q"], device=device)
    kj = torch.arange(case["len"], device=device)
    # a padded batch: rows past a sequence's end repeat some row and are not seen
    q_at = (q_off[:-1, None] + qi).clamp(max=s["q"].shape[0] - 1)
    k_at = (k_off[:-1, None] + kj).clamp(max=s["k"].shape[0] - 1)
    q = s["q"].view(-1, heads, HEAD)[q_at].float().permute(0, 2, 1, 3).reshape(case["batch"], kv, -1, HEAD)
    k = s["k"].view(-1, kv, HEAD)[k_at].float().permute(0, 2, 3, 1)
    v = s["v"].view(-1, kv, HEAD)[k_at].float().permute(0, 2, 1, 3)
    score = (q @ k).mul_(HEAD ** -0.5).view(case["batch"], heads, s["max_q"], case["len"])
    dist = kj[None, None, :] - (qi[None, :, None] + (k_len - q_len)[:, None, None])
    if s["bias"] is not None:
        score += s["bias"][:, (dist + 128).clamp(0, s["bias"].shape[1] - 1)].transpose(0, 1)
    seen = (kj < k_len[:, None])[:, None, :].expand_as(dist)
    if case["right"] >= 0:
        seen = seen & (dist <= case["right"])
    if case["left"] >= 0:
        seen = seen & ((dist >= -case["left"]) | (kj < case["sinks"]))
    seen = seen[:, None]
    score.masked_fill_(~seen, -math.inf)
    top = score.amax(3, keepdim=True)
    score.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = score.sum(3, keepdim=True)
    out = (score.view(case["batch"], kv, -1, case["len"]) @ v).view(case["batch"], heads, s["max_q"], HEAD)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3).reshape(case["batch"], s["max_q"], -1)
    rows = torch.arange(s["q"].shape[0], device=device)
    b = torch.searchsorted(q_off, rows, right=True) - 1
    return out[b, rows - q_off[b]].to(torch.float16)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case.get("f32") else 2
    if case["op"] == "bias":
        return {"bytes": 2 * case["heads"] * case["q"] * case["k"] + size * case["heads"] * case["buckets"], "flops": 0}
    if case["op"] == "grad":
        n = case["batch"] * case["heads"] * case["q"] * case["k"]
        return {"bytes": size * n + 4 * case["heads"] * case["buckets"], "flops": n}
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        wide = size + (4 if case["res"] else 0) + (2 if case["group"] < 0 else 1)
        group = case["group"] or case["hidden"]
        scales = 0 if case["group"] < 0 else 4 * case["rows"] * -(-case["hidden"] // group)
        return {"bytes": wide * n + 2 * case["hidden"] + scales, "flops": 5 * n}
    pairs = keys = queries = 0
    for n in _lens(case):
        q = (1 if case["one"] else n)
        p = torch.arange(n - q, n, dtype=torch.int64)
        high = (p + case["right"] + 1).clamp(max=n) if case["right"] >= 0 else torch.full_like(p, n)
        low = (p - case["left"]).clamp(min=0) if case["left"] >= 0 else torch.zeros_like(p)
        first = torch.minimum(torch.minimum(low, high.clamp(min=0)), torch.tensor(case["sinks"]))
        seen = (high - low).clamp(min=0) + first.clamp(min=0)
        pairs += int(seen.sum()) if n else 0
        queries += q
        if n:
            keys += int(seen[0]) if case["one"] else n
    return {"bytes": 2 * HEAD * (2 * case["heads"] * queries + 2 * case["kv"] * keys),
            "flops": 4 * HEAD * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ 64 bits
def _bucket_of(d, case):
    """Bucket of one distance, in whole numbers: step j is reached when n^m * e^j >= D^j * e^m."""
    count, base = (case["buckets"] // 2, 0) if case["both"] else (case["buckets"], 0)
    if case["both"]:
        base, n = (count if d > 0 else 0), abs(d)
    else:
        n = max(-d, 0)
    e = count // 2
    if n < e:
        return base + n
    m, j = count - e, 0
    while j < m - 1 and n ** m * e ** (j + 1) >= case["dist"] ** (j + 1) * e ** m:
        j += 1
    return base + e + j


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("bias", "grad"):
        low = -(case["q"] - 1) - case["start"]
        by_distance = torch.tensor([_bucket_of(d, case) for d in range(low, case["k"] - case["start"])], device="cuda")
        at = (torch.arange(case["k"]) + (case["q"] - 1 - torch.arange(case["q"]))[:, None]).cuda()
        if case["op"] == "bias":
            return torch.stack([s["table"][:, h].double()[by_distance][at] for h in range(case["heads"])])
        out = torch.zeros(case["buckets"], case["heads"], dtype=torch.float64, device="cuda")
        diagonals = torch.zeros(by_distance.numel(), case["heads"], dtype=torch.float64, device="cuda")
        for i in range(case["q"]):  # row i lies on the diagonals from q-1-i on
            first = case["q"] - 1 - i
            diagonals[first:first + case["k"]] += s["grad"][:, :, i].double().sum(0).t()
        for b in range(case["buckets"]):
            out[b] = diagonals[by_distance == b].sum(0)
        return out
    if case["op"] == "norm":
        x = s["x"].double() + (s["residual"].double() if s["residual"] is not None else 0.0)
        y = x / torch.sqrt(torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / case["hidden"] + 1e-6)
        y = y * s["gamma"].double()
        extra = (x,) if s["residual"] is not None else ()
        if case["group"] < 0:
            return (y,) + extra
        group = case["group"] or case["hidden"]
        scales = torch.stack([part.abs().max(1).values for part in y.split(group, dim=1)], dim=1) / 448.0
        scales = torch.clamp(scales, min=2.0 ** -100 / 448.0)
        value = y / scales.repeat_interleave(group, dim=1)[:, :case["hidden"]]
        return (value.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double(), scales) + extra
    lens, group = _lens(case), case["heads"] // case["kv"]
    out = torch.zeros(s["q"].shape[0], case["heads"] * HEAD, dtype=torch.float64, device="cuda")
    q_off, k_off = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    for b, n in enumerate(lens):
        rows = q_off[b + 1] - q_off[b]
        p = torch.arange(rows, device="cuda")[:, None] + n - rows
        j = torch.arange(n, device="cuda")[None, :]
        seen = torch.ones(rows, n, dtype=torch.bool, device="cuda")
        if case["left"] >= 0:
            seen &= (p - j <= case["left"]) | (j < case["sinks"])
        if case["right"] >= 0:
            seen &= j - p <= case["right"]
        for h in range(case["heads"] if n else 0):
            c, d = slice(h * HEAD, (h + 1) * HEAD), slice(h // group * HEAD, (h // group + 1) * HEAD)
            key = s["k"][k_off[b]:k_off[b] + n, d].double()
            score = s["q"][q_off[b]:q_off[b + 1], c].double() @ key.T / math.sqrt(HEAD)
            if s["bias"] is not None:
                score = score + s["bias"][h].double()[torch.clamp(j - p, -128, 128) + 128]
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), dim=1).nan_to_num(0.0)
            out[q_off[b]:q_off[b + 1], c] = weight @ s["v"][k_off[b]:k_off[b] + n, d].double()
    return out
