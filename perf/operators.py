"""The transformer-layer operators, as they are measured: layer norm, linear with its epilogue, attention with a bucketed relative position bias.

`run` makes one pass: the forward alone (`train` false, as a served model calls it) or the forward and every gradient (`train` true, as a
training step calls it).  The plain forms are elementary torch operations in 32 bits, rounded once at the end; `exact` is the definition in
64 bits through autograd."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = {"none": 0, "silu": 1, "relu": 2, "sigmoid": 3}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------------------------ cases
def norm_case(name, rows, width, dtype, train, residual, weights="f32"):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "train": train, "residual": residual, "weights": weights}


def linear_case(name, rows, k, n, dtype, train, act, bias, residual):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train, "act": act, "bias": bias, "residual": residual}


def attention_case(name, batch, lq, lk, heads, kv_heads, dim, dtype, train, causal=False, ragged=False, groups=0, buckets=32, distance=128, both=True):
    return {"name": name, "op": "attention", "batch": batch, "lq": lq, "lk": lk, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "train": train, "causal": causal, "ragged": ragged, "groups": groups, "buckets": buckets, "distance": distance, "both": both}


def listed():
    return [
        # the post-norm of a decoder layer on one frame's 300 queries: latency
        norm_case("norm one frame", 300, 256, "bf16", False, True),
        # the token rows of eight 1088 x 608 frames (13566 each), a training step of the norm behind the input projection
        norm_case("norm tokens train", 108528, 256, "bf16", True, False),
        # an odd width, half precision, weights in the activations' type
        norm_case("norm odd train", 4099, 1283, "f16", True, True, "f16"),
        # a wide model in full precision
        norm_case("norm wide train", 16384, 4096, "f32", True, False),
        # one token through the first product of a feed-forward block: the weight is read once
        linear_case("linear one token", 1, 1024, 4096, "bf16", False, "silu", True, False),
        # the decoder's feed-forward block (256 -> 1024, ReLU) on 16 frames of 300 queries
        linear_case("linear decoder ffn train", 4800, 256, 1024, "bf16", True, "relu", True, False),
        # a large block: the matrix cores' rate
        linear_case("linear large train", 8192, 4096, 4096, "bf16", True, "silu", True, True),
        # full precision, nothing a multiple of a tile
        linear_case("linear ragged train", 1803, 514, 770, "f32", True, "sigmoid", True, True),
        # one new token for each of 32 sequences over their caches of up to 16384 keys, four query heads to a key head
        attention_case("attention one token", 32, 1, 16384, 16, 4, 64, "bf16", False, ragged=True, both=False),
        # the decoder's self-attention over 300 queries with the group mask that denoising training uses
        attention_case("attention queries train", 16, 300, 300, 8, 8, 32, "f16", True, groups=3),
        # a long causal sequence
        attention_case("attention long train", 2, 4096, 4096, 16, 16, 64, "bf16", True, causal=True, both=False),
        # full precision, odd lengths, shared heads, padded keys (one sequence without any)
        attention_case("attention ragged train", 3, 77, 401, 6, 2, 40, "f32", True, ragged=True, buckets=16, distance=50),
    ]


def spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    if op == "norm":
        width = spread(rng, 8, 8192)
        if rng.random() < 0.6:
            width = max(8, width // 8 * 8)
        rows = spread(rng, 1, min(200000, (1 << 26) // width))
        c = norm_case("", rows, width, dtype, train, rng.random() < 0.5, rng.choice(["f32", dtype]))
    elif op == "linear":
        k, n = spread(rng, 8, 4096), spread(rng, 8, 4096)
        if rng.random() < 0.7:
            k, n = max(8, k // 8 * 8), max(8, n // 8 * 8)
        rows = spread(rng, 1, 8192)
        c = linear_case("", rows, k, n, dtype, train, rng.choice(list(ACTS)), rng.random() < 0.8, rng.random() < 0.5)
    else:
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads, dim = kv_heads * rng.choice([1, 1, 2, 4]), 8 * rng.randint(1, 16)
        buckets, both = rng.choice([8, 16, 32, 48]), rng.random() < 0.5
        c = dict(buckets=buckets, distance=rng.randint(buckets, 256), both=both)
        kind = rng.choice(["token", "self", "cross"])
        if kind == "token":  # a few new tokens over a cache
            lq, lk, train = rng.randint(1, 8), spread(rng, 8, 32768), False
            batch = max(1, min(rng.randint(1, 32), (1 << 27) // (lk * kv_heads * dim)))
            c = attention_case("", batch, lq, lk, heads, kv_heads, dim, dtype, train, causal=True, ragged=True, **c)
        elif kind == "self":
            lq = spread(rng, 1, 2048)
            batch = max(1, min(rng.randint(1, 16), (1 << 27) // (lq * lq * heads)))
            c = attention_case("", batch, lq, lq, heads, kv_heads, dim, dtype, train, causal=rng.random() < 0.5, groups=rng.choice([0, 0, 3]), **c)
        else:
            lq, lk = spread(rng, 1, 1024), spread(rng, 1, 4096)
            batch = max(1, min(rng.randint(1, 16), (1 << 27) // (lq * lk * heads)))
            c = attention_case("", batch, lq, lk, heads, kv_heads, dim, dtype, train, ragged=rng.random() < 0.6, **c)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------------------------- inputs
def key_lengths(case):
    """Valid keys of each sequence: all of them, or (ragged) between a half and all, the second sequence of a training batch of three or more empty."""
    lk, batch = case["lk"], case["batch"]
    if not case["ragged"]:
        return [lk] * batch
    lens = [max(1, lk - (b * 7919) % (lk // 2 + 1)) for b in range(batch)]
    if case["train"] and batch >= 3:
        lens[1] = 0
    return lens


def first_position(case):
    """Position of the first query, one for each sequence: the queries are the last ones of a causal cache, else both count from zero."""
    return [n - case["lq"] if case["causal"] or case["lq"] == 1 else 0 for n in key_lengths(case)]


def group_mask(case):
    """True where a query must not see a key: the first two thirds are `groups` denoising groups, which see themselves and the rest; the rest
    does not see them."""
    if not case["groups"]:
        return None
    n = case["lq"]
    rest = n * 2 // 3
    group = np.where(np.arange(n) < rest, np.arange(n) * case["groups"] // max(1, rest), case["groups"])
    return (group[:, None] != group[None, :]) & (group[None, :] != case["groups"])


def bucket_of(relative, buckets, distance, both):
    """Bucket of a key at `relative` = its position - the query's: exact up to half the buckets, then logarithmic up to `distance`; in whole numbers."""
    n, base, m = abs(relative), 0, buckets
    if both:
        m = buckets // 2
        base = m if relative > 0 else 0
    elif relative > 0:
        n = 0
    near = m // 2
    if n < near:
        return base + n
    step = m - near
    t = max(0, min(step - 1, int(math.log(n / near) / math.log(distance / near) * step) - 1))
    while t < step - 1 and n ** step * near ** (t + 1) >= distance ** (t + 1) * near ** step:
        t += 1
    return base + near + t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = TYPES[case["dtype"]], case["train"]

    def rand(*shape, scale=1.0, shift=0.0, dtype=dt, grad=True):
        t = (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)
        return t.requires_grad_(True) if grad and train else t

    s = {"case": case}
    if case["op"] == "norm":
        m, c, wt = case["rows"], case["width"], TYPES[case["weights"]]
        s.update(x=rand(m, c, scale=2.0, shift=0.3), w=rand(c, scale=0.2, shift=1.0, dtype=wt), b=rand(c, scale=0.2, dtype=wt),
                 r=rand(m, c) if case["residual"] else None, dy=rand(m, c, grad=False) if train else None)
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        s.update(x=rand(m, k), w=rand(n, k, scale=k ** -0.5), b=rand(n, scale=0.5) if case["bias"] else None,
                 r=rand(m, n) if case["residual"] else None, dy=rand(m, n, grad=False) if train else None)
    else:
        b, lq, lk, h, hk, d = (case[x] for x in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
        s.update(q=rand(b, lq, h, d), k=rand(b, lk, hk, d), v=rand(b, lk, hk, d), table=rand(case["buckets"], h),
                 dy=rand(b, lq, h, d, grad=False) if train else None)
        far = case["distance"]
        s["lut"] = torch.tensor([bucket_of(x, case["buckets"], far, case["both"]) for x in range(-far, far + 1)], dtype=torch.uint8, device="cuda")
        s["k_len"] = torch.tensor(key_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        mask = group_mask(case)
        s["mask"] = None if mask is None else torch.from_numpy(mask).cuda()
        s["q_start"] = None if case["causal"] or lq == 1 else 0
    return s


# ------------------------------------------------------------------------------------------------------------------- plain
def plain_norm(s):
    x, r, dt = s["x"], s["r"], s["x"].dtype
    w, b = s["w"].float(), s["b"].float()
    t = x.float() if r is None else x.float() + r.float()
    t = t - t.mean(-1, keepdim=True)
    rstd = (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = t * rstd
    y = (xh * w + b).to(dt)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = ((g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rstd).to(dt)
    out = {"y": y, "dx": dx, "dw": (dy * xh).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}
    if r is not None:
        out["dr"] = dx
    return out


def plain_linear(s):
    x, w, r, dt, act = s["x"].float(), s["w"].float(), s["r"], s["x"].dtype, s["case"]["act"]
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    sg = 1 / (1 + torch.exp(-z)) if act in ("silu", "sigmoid") else None
    y = {"none": lambda: z, "silu": lambda: z * sg, "relu": lambda: z.clamp(min=0), "sigmoid": lambda: sg}[act]()
    if r is not None:
        y = y + r.float()
    y = y.to(dt)
    if s["dy"] is None:
        return {"y": y}
    dy = s["dy"].float()
    dz = {"none": lambda: dy, "silu": lambda: dy * (sg * (1 + z * (1 - sg))), "relu": lambda: dy * (z > 0), "sigmoid": lambda: dy * (sg * (1 - sg))}[act]()
    out = {"y": y, "dx": (dz @ w).to(dt), "dw": (dz.t() @ x).to(s["w"].dtype)}
    if s["b"] is not None:
        out["db"] = dz.sum(0).to(s["b"].dtype)
    if r is not None:
        out["dr"] = s["dy"]
    return out


def relative_positions(case, device):
    """[batch or 1, lq, lk] position of each key less the query's."""
    start = first_position(case) if len(set(first_position(case))) > 1 else first_position(case)[:1]
    at = torch.tensor(start, device=device)[:, None, None] + torch.arange(case["lq"], device=device)[None, :, None]
    return torch.arange(case["lk"], device=device)[None, None, :] - at


def hidden(case, mask, k_len, rel):
    """True where the score does not count: [batch or 1, 1, lq, lk] or None."""
    parts = []
    if case["causal"]:
        parts.append(rel > 0)
    if k_len is not None:
        parts.append((torch.arange(case["lk"], device=rel.device)[None, :] >= k_len[:, None])[:, None, :])
    if mask is not None:
        parts.append(mask[None])
    if not parts:
        return None
    out = parts[0]
    if len(parts) > 1:
        out = out | parts[1]
    if len(parts) > 2:
        out = out | parts[2]
    return out[:, None]


def plain_attention(s):
    case, q, k, v, dt = s["case"], s["q"], s["k"], s["v"], s["q"].dtype
    b, lq, lk, h, hk, d = (case[x] for x in ("batch", "lq", "lk", "heads", "kv_heads", "dim"))
    share, far, scale = h // hk, case["distance"], d ** -0.5
    rows = lambda t: t.float().transpose(1, 2).contiguous()  # noqa: E731
    qf, kf, vf = rows(q), rows(k), rows(v)
    if share > 1:
        kf, vf = kf.repeat_interleave(share, 1), vf.repeat_interleave(share, 1)
    rel = relative_positions(case, q.device)
    bias = s["table"].float()[s["lut"].long()[rel.clamp(-far, far) + far]].permute(0, 3, 1, 2)
    off = hidden(case, s["mask"], s["k_len"], rel)
    p = qf @ kf.transpose(2, 3).contiguous() * scale + bias
    del bias
    if off is not None:
        p = p.masked_fill(off, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    y = (p @ vf).transpose(1, 2).to(dt)
    if s["dy"] is None:
        return {"y": y}
    do = rows(s["dy"])
    dv = p.transpose(2, 3).contiguous() @ do
    ds = do @ vf.transpose(2, 3).contiguous()
    ds = p * (ds - (ds * p).sum(-1, keepdim=True))
    dq = (ds @ kf) * scale
    dk = (ds.transpose(2, 3).contiguous() @ qf) * scale
    if share > 1:
        dk, dv = dk.view(b, hk, share, lk, d).sum(2), dv.view(b, hk, share, lk, d).sum(2)
    # the table: sums along the diagonals (rows flipped and skewed so that a diagonal is a column), then over the diagonals of a bucket
    if rel.shape[0] == 1:
        ds, base = ds.double().sum(0, keepdim=True), first_position(case)[:1]
    else:
        ds, base = ds.double(), first_position(case)
    n = ds.shape[0]
    skew = torch.nn.functional.pad(ds.flip(2), (0, lq)).reshape(n, h, -1)[:, :, : lq * (lk + lq - 1)].view(n, h, lq, lk + lq - 1)
    by = skew.sum(2)  # column c holds the diagonal j - i = c - (lq - 1)
    at = torch.arange(lk + lq - 1, device=q.device)[None] - (lq - 1) - torch.tensor(base, device=q.device)[:, None]
    which = s["lut"].long()[at.clamp(-far, far) + far]
    dtable = torch.zeros(case["buckets"], h, dtype=torch.float64, device=q.device).index_add_(0, which.reshape(-1), by.permute(0, 2, 1).reshape(-1, h))
    back = lambda t: t.transpose(1, 2).to(dt)  # noqa: E731
    return {"y": y, "dq": back(dq), "dk": back(dk), "dv": back(dv), "dtable": dtable.to(s["table"].dtype)}


# -------------------------------------------------------------------------------------------------------------------- run
def gradients(s, y, names):
    names = {n: s[x] for n, x in names.items() if s[x] is not None}
    return dict(zip(names, torch.autograd.grad(y, list(names.values()), s["dy"])), y=y.detach())


def run_own(s):
    from mo_yolo_amd import modules
    case = s["case"]
    if case["op"] == "norm":
        y, names = modules.layer_norm(s["x"], s["w"], s["b"], EPS, residual=s["r"]), {"dx": "x", "dw": "w", "db": "b", "dr": "r"}
    elif case["op"] == "linear":
        y, names = modules.linear(s["x"], s["w"], s["b"], act=ACTS[case["act"]], residual=s["r"]), {"dx": "x", "dw": "w", "db": "b", "dr": "r"}
    else:
        y = modules.biased_attention(s["q"], s["k"], s["v"], s["table"], s["lut"], causal=case["causal"], q_start=s["q_start"], k_len=s["k_len"],
                                     attn_mask=s["mask"])
        names = {"dq": "q", "dk": "k", "dv": "v", "dtable": "table"}
    return gradients(s, y, names) if case["train"] else {"y": y}


def run(state):
    if own:
        return run_own(state)
    with torch.no_grad():
        return {"norm": plain_norm, "linear": plain_linear, "attention": plain_attention}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, c = case["rows"] * case["width"], case["width"]
        tensors = 2 + case["residual"] + (2 if case["train"] else 0)
        return {"bytes": n * size * tensors + 4 * c * TYPES[case["weights"]].itemsize, "flops": n * (18 if case["train"] else 8)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        there = m * k + n * k + n * case["bias"] + m * n * (1 + case["residual"])
        back = m * n + m * k + n * k + n * case["bias"]
        return {"bytes": (there + (back if case["train"] else 0)) * size, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    h, d, lq = case["heads"], case["dim"], case["lq"]
    lens, start, mask = key_lengths(case), first_position(case), group_mask(case)
    pairs = 0
    for n, at in zip(lens, start):
        seen = np.clip(np.arange(lq) + at + 1, 0, n) if case["causal"] else np.full(lq, n)
        if mask is None:
            pairs += int(seen.sum())
        else:
            pairs += int(((np.arange(case["lk"])[None, :] < seen[:, None]) & ~mask).sum())
    queries, keys = case["batch"] * lq * h * d, 2 * sum(lens) * case["kv_heads"] * d
    return {"bytes": size * ((2 * queries + keys) if not case["train"] else (4 * queries + 2 * keys)) + case["buckets"] * h * size,
            "flops": pairs * h * d * (14 if case["train"] else 4)}


# ------------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    wide = {n: t.detach().double().requires_grad_(t.requires_grad) if torch.is_tensor(t) and t.is_floating_point() else t for n, t in s.items()}
    with torch.enable_grad():
        if case["op"] == "norm":
            t = wide["x"] if wide["r"] is None else wide["x"] + wide["r"]
            spread_ = t.var(-1, unbiased=False, keepdim=True)
            y = (t - t.mean(-1, keepdim=True)) / torch.sqrt(spread_ + EPS) * wide["w"] + wide["b"]
            names = {"dx": "x", "dw": "w", "db": "b", "dr": "r"}
        elif case["op"] == "linear":
            z = torch.matmul(wide["x"], wide["w"].transpose(0, 1))
            z = z if wide["b"] is None else z + wide["b"]
            y = {"none": lambda t: t, "silu": lambda t: t * torch.sigmoid(t), "relu": torch.relu, "sigmoid": torch.sigmoid}[case["act"]](z)
            y = y if wide["r"] is None else y + wide["r"]
            names = {"dx": "x", "dw": "w", "db": "b", "dr": "r"}
        else:
            names = {"dq": "q", "dk": "k", "dv": "v", "dtable": "table"}
            share, far = case["heads"] // case["kv_heads"], case["distance"]
            ys = []
            for b, (n, at) in enumerate(zip(key_lengths(case), first_position(case))):  # one sequence at a time, its valid keys only
                if n == 0:
                    ys.append(wide["q"][b] * 0)
                    continue
                k, v = (wide[x][b, :n].repeat_interleave(share, 1).permute(1, 0, 2) for x in ("k", "v"))
                i, j = torch.arange(case["lq"], device="cuda")[:, None] + at, torch.arange(n, device="cuda")[None]
                bias = wide["table"].index_select(0, s["lut"].int()[(j - i).clamp(-far, far) + far].reshape(-1)).view(case["lq"], n, -1)
                score = torch.matmul(wide["q"][b].permute(1, 0, 2), k.transpose(1, 2)) / math.sqrt(case["dim"]) + bias.permute(2, 0, 1)
                off = (j > i) if case["causal"] else torch.zeros_like(j > i)
                if s["mask"] is not None:
                    off = off | s["mask"][:, :n]
                none = off.all(-1, keepdim=True)
                prob = torch.softmax(score.masked_fill(off & ~none, float("-inf")), -1).masked_fill(none, 0.0)
                ys.append(torch.matmul(prob, v).permute(1, 0, 2))
            y = torch.stack(ys)
        if not case["train"]:
            return {"y": y.detach()}
        wide["dy"] = s["dy"].double()
        return gradients(wide, y, names)
