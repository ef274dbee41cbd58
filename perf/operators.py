"""Cases of the image-transformer operators: group norm with an activation on channels-last maps, the gated
projection of a feed-forward block, and attention over a token grid with a learned relative position bias.

`run` computes a case in its plain form -- elementary torch operations in 32 bits, rounded once at the end -- or,
with `own` set, through pixelsplat_amd.  `exact` gives the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def _norm(name, n, h, w, c, groups, act, dtype, train):
    return dict(name=name, op="norm", n=n, h=h, w=w, c=c, groups=groups, act=act, dtype=dtype, train=train)


def _gated(name, rows, dim, hidden, act, dtype, train, bias=True):
    return dict(name=name, op="gated", rows=rows, dim=dim, hidden=hidden, act=act, dtype=dtype, train=train, bias=bias)


def _attention(name, batch, heads, gh, gw, dim, dtype, train, queries=0, masked=False, per_axis=32):
    return dict(name=name, op="attention", batch=batch, heads=heads, gh=gh, gw=gw, dim=dim, dtype=dtype, train=train,
                queries=queries, masked=masked, per_axis=per_axis)


def listed():
    return [
        # one scene's two context views as 4x4 patches of a 64x64 map: what a viewer pays per frame (latency)
        _norm("norm latency", 2, 16, 16, 128, 8, "relu", "bf16", False),
        # the 64x64 feature maps of seven scenes with two context views each: a training step of the encoder
        _norm("norm maps train", 14, 64, 64, 128, 32, "gelu", "fp32", True),
        # full-resolution maps of the refinement convolutions (twice the width) at 256x256, a training step in bf16
        _norm("norm full res train", 14, 256, 256, 256, 32, "gelu", "bf16", True),
        # an odd crop with a group width that is no power of two
        _norm("norm odd", 5, 61, 83, 120, 8, "silu", "fp16", False),
        # one token through the feed-forward of a 1024-wide transformer: weights are all that is read
        _gated("gated one token", 1, 1024, 4096, "silu", "bf16", False),
        # the self-attention blocks' feed-forward at the paper configuration: 14 images of 256 tokens, fp32 training
        _gated("gated tokens train", 14 * 256, 128, 256, "gelu", "fp32", True),
        # a long ragged prompt of a 768-wide backbone, forward only
        _gated("gated ragged", 1601, 768, 2050, "gelu", "fp16", False),
        # a training step of a wide transformer: the matrix products decide
        _gated("gated wide train", 16384, 1024, 4096, "silu", "bf16", True, bias=False),
        # self-attention over the 16x16 patch grid of 14 images, four heads of 128: the paper configuration's training
        _attention("attention patches train", 14, 4, 16, 16, 128, "fp32", True),
        # one token against every token of a 128x128 grid: a single query over a long key list
        _attention("attention one query", 4, 8, 128, 128, 64, "bf16", False, queries=1),
        # a ragged batch of odd grids with padded keys, one element of it padding alone
        _attention("attention ragged", 6, 6, 37, 23, 40, "fp16", False, masked=True),
        # 64x64 tokens, a feature map without patching: a training step in bf16
        _attention("attention maps train", 2, 8, 64, 64, 64, "bf16", True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "gated", "attention"])
    dtype, train = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5
    if op == "norm":
        while True:
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            c = _norm("", _spread(rng, 1, 28), _spread(rng, 8, 256), _spread(rng, 8, 256),
                      groups * _spread(rng, 1, max(1, 512 // groups)), groups, rng.choice(["none", "relu", "silu", "gelu"]), dtype, train)
            if c["n"] * c["h"] * c["w"] * c["c"] <= 14 * 256 * 256 * 128:
                break
    elif op == "gated":
        while True:
            c = _gated("", _spread(rng, 1, 16384), _spread(rng, 32, 2048), _spread(rng, 64, 8192),
                       rng.choice(["silu", "gelu", "sigmoid", "relu"]), dtype, train, rng.random() < 0.5)
            if rng.random() < 0.7:
                c["dim"] = max(32, c["dim"] // 8 * 8)
            if c["rows"] * c["dim"] * c["hidden"] <= 16384 * 1024 * 4096 // (8 if dtype == "fp32" else 1):
                break
    else:
        while True:
            gh = 1 if rng.random() < 0.25 else _spread(rng, 2, 96)
            gw = _spread(rng, 16, 4096) if gh == 1 else _spread(rng, 2, 96)
            c = _attention("", _spread(rng, 1, 16), _spread(rng, 1, 16), gh, gw, 8 * _spread(rng, 2, 16), dtype, train,
                           1 if rng.random() < 0.2 else 0, rng.random() < 0.4, rng.choice([8, 16, 32]))
            length = gh * gw
            most = 2 * 8 * 4096 * 4096 * 64 // (8 if dtype == "fp32" else 1)
            if length <= 8192 and c["batch"] * c["heads"] * length * length * c["dim"] <= most:
                break
    c.pop("name")
    return c


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _buckets(gh, gw, per_axis, device):
    """[2 gh - 1, 2 gw - 1] int32: the bucket of every (row, column) offset key - query; each axis has exact buckets
    near zero and logarithmic ones out to 128, a sign apart, and an axis of one token has one bucket."""
    def axis(n):
        if n == 1:
            return torch.zeros(1, dtype=torch.int64), 1
        d = torch.arange(-(n - 1), n, dtype=torch.float64)
        half, exact = per_axis // 2, per_axis // 4
        far = exact + (torch.log(d.abs().clamp(min=1) / exact) / math.log(128 / exact) * (half - exact)).floor()
        near = torch.where(d.abs() < exact, d.abs(), far.clamp(max=half - 1))
        return (near + half * (d > 0)).long(), per_axis
    (rows, _), (cols, n) = axis(gh), axis(gw)
    return (rows[:, None] * n + cols[None]).int().to(device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, scale=1.0, leaf=True):
        t = (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)
        return t.requires_grad_(train and leaf)

    s = dict(case=case)
    if case["op"] == "norm":
        shape = (case["n"], case["h"], case["w"], case["c"])
        s["x"] = (normal(*shape, leaf=False) * 1.5 + normal(1, 1, 1, case["c"], leaf=False)).requires_grad_(train)
        s["weight"] = (1 + normal(case["c"], scale=0.2, leaf=False)).requires_grad_(train)
        s["bias"] = normal(case["c"], scale=0.2)
        s["dy"] = normal(*shape, leaf=False) if train else None
    elif case["op"] == "gated":
        m, d, f = case["rows"], case["dim"], case["hidden"]
        s["x"] = normal(m, d)
        s["w_gate"], s["w_up"] = normal(f, d, scale=d ** -0.5), normal(f, d, scale=d ** -0.5)
        s["b_gate"], s["b_up"] = (normal(f, scale=0.1), normal(f, scale=0.1)) if case["bias"] else (None, None)
        s["dy"] = normal(m, f, leaf=False) if train else None
    else:
        b, h, d = case["batch"], case["heads"], case["dim"]
        length = case["gh"] * case["gw"]
        nq = case["queries"] or length
        # queries, keys and values as a packed projection leaves them: [batch, token, 3, head, dim], read as views
        packed = normal(b, length, 3, h, d, leaf=False)
        q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
        s["start"] = 0 if nq == length else int(torch.randint(0, length - nq + 1, (1,), generator=g, device=dev))
        s["q"] = q[:, :, s["start"]:s["start"] + nq].detach().requires_grad_(train)
        s["k"], s["v"] = k.detach().requires_grad_(train), v.detach().requires_grad_(train)
        s["buckets"] = _buckets(case["gh"], case["gw"], case["per_axis"], dev)
        rows = 1 if case["gh"] == 1 else case["per_axis"]
        cols = 1 if case["gw"] == 1 else case["per_axis"]
        s["table"] = normal(rows * cols, h, scale=0.5)
        s["mask"] = None
        if case["masked"]:   # True: a key that is there.  Ragged lengths; the second of a batch has no key at all
            lengths = torch.randint(1, length + 1, (b,), generator=g, device=dev)
            if b > 1:
                lengths[1] = 0
            s["mask"] = torch.arange(length, device=dev)[None] < lengths[:, None]
        s["dy"] = normal(b, h, nq, d, leaf=False) if train else None
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _act(name, z):
    """(act(z), act'(z))"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z * (z > 0), (z > 0).to(z.dtype)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-z))
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    return z * sig, sig * (1 + z * (1 - sig))


EPS = 1e-5


def _plain_norm(s):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    n, ch, groups = c["n"], c["c"], c["groups"]
    x = s["x"].float().reshape(n, -1, groups, ch // groups)
    w, b = s["weight"].float().view(groups, -1), s["bias"].float().view(groups, -1)
    mean = x.mean((1, 3), keepdim=True)
    x = x - mean
    rstd = torch.rsqrt((x * x).mean((1, 3), keepdim=True) + EPS)
    x = x * rstd
    y, slope = _act(c["act"], x * w + b)
    shape = s["x"].shape
    if not c["train"]:
        return y.reshape(shape).to(dtype)
    dz = s["dy"].float().reshape(x.shape) * slope
    db, dw = dz.sum((0, 1)), (dz * x).sum((0, 1))
    dz = dz * w
    dx = rstd * (dz - dz.mean((1, 3), keepdim=True) - x * (dz * x).mean((1, 3), keepdim=True))
    return y.reshape(shape).to(dtype), dx.reshape(shape).to(dtype), dw.reshape(-1).to(dtype), db.reshape(-1).to(dtype)


def _plain_gated(s):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    gate, up = x @ wg.T, x @ wu.T
    if c["bias"]:
        gate, up = gate + s["b_gate"].float(), up + s["b_up"].float()
    a, slope = _act(c["act"], gate)
    if not c["train"]:
        return (a * up).to(dtype)
    dy = s["dy"].float()
    dgate, dup = dy * up * slope, dy * a
    out = [a * up, dgate @ wg + dup @ wu, dgate.T @ x, dup.T @ x]
    if c["bias"]:
        out += [dgate.sum(0), dup.sum(0)]
    return tuple(t.to(dtype) for t in out)


def _offsets(s):
    """[queries, keys] index of the flattened bucket map."""
    c = s["case"]
    gh, gw = c["gh"], c["gw"]
    q = torch.arange(s["q"].shape[2], device=s["q"].device) + s["start"]
    k = torch.arange(gh * gw, device=s["q"].device)
    rows = k[None] // gw - q[:, None] // gw + gh - 1
    cols = k[None] % gw - q[:, None] % gw + gw - 1
    return rows * (2 * gw - 1) + cols


def _plain_attention(s):
    c, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    q, k, v, table = (s[n].float() for n in ("q", "k", "v", "table"))
    scale = c["dim"] ** -0.5
    bucket = s["buckets"].view(-1).long()[_offsets(s)]
    p = (q * scale) @ k.transpose(-1, -2) + table[bucket].permute(2, 0, 1)
    if s["mask"] is not None:
        p = p.masked_fill(~s["mask"][:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = p @ v
    if not c["train"]:
        return out.to(dtype)
    dy = s["dy"].float()
    dv = p.transpose(-1, -2) @ dy
    ds = p * (dy @ v.transpose(-1, -2) - (dy * out).sum(-1, keepdim=True))
    dq, dk = ds @ k * scale, ds.transpose(-1, -2) @ q * scale
    # up to 256 tables, summed at the end: the additions of one bucket would otherwise wait for one another
    n, copies = table.shape[0], min(256, q.shape[2])
    dtable = torch.zeros((copies * n, table.shape[1]), dtype=torch.float64, device=table.device)
    bucket = bucket + torch.arange(q.shape[2], device=table.device)[:, None] % copies * n
    dtable.index_add_(0, bucket.view(-1), ds.sum(0, dtype=torch.float64).flatten(1).T)
    dtable = dtable.view(copies, n, -1).sum(0)
    return out.to(dtype), dq.to(dtype), dk.to(dtype), dv.to(dtype), dtable.to(dtype)


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _own(s):
    c = s["case"]
    if c["op"] == "norm":
        from pixelsplat_amd.ops import group_norm
        leaves = [s["x"], s["weight"], s["bias"]]
        y = group_norm(s["x"], c["groups"], s["weight"], s["bias"], eps=EPS, activation=c["act"])
    elif c["op"] == "gated":
        from pixelsplat_amd.ops import gated_linear
        leaves = [s["x"], s["w_gate"], s["w_up"]] + ([s["b_gate"], s["b_up"]] if c["bias"] else [])
        y = gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=c["act"])
    else:
        from pixelsplat_amd.ops import relative_attention
        leaves = [s["q"], s["k"], s["v"], s["table"]]
        y = relative_attention(s["q"], s["k"], s["v"], s["table"], s["buckets"], key_mask=s["mask"],
                               query_start=s["start"])
    if not c["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "gated": _plain_gated, "attention": _plain_attention}[state["case"]["op"]](state)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "norm":
        n = case["n"] * case["h"] * case["w"] * case["c"]
        return {"bytes": n * e * (4 if train else 2) + case["c"] * e * (4 if train else 2), "flops": n * (35 if train else 12)}
    if case["op"] == "gated":
        m, d, f = case["rows"], case["dim"], case["hidden"]
        once = m * d + 2 * f * d + m * f + (2 * f if case["bias"] else 0)
        return {"bytes": once * e * (2 if train else 1), "flops": 4 * m * d * f * (3 if train else 1)}
    length = case["gh"] * case["gw"]
    nq = case["queries"] or length
    bh = case["batch"] * case["heads"]
    once = bh * case["dim"] * (2 * nq + 2 * length)
    return {"bytes": once * e * (2 if train else 1), "flops": bh * nq * length * case["dim"] * (14 if train else 4)}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_activation(name, t):
    if name == "none":
        return t
    if name == "relu":
        return t.clamp(min=0)
    if name == "sigmoid":
        return torch.sigmoid(t)
    if name == "silu":
        return t * torch.sigmoid(t)
    return t * 0.5 * torch.erfc(-t / math.sqrt(2))


def exact(case, seed):
    """Forward from the definition, one sample or head at a time; gradients by differentiating it in 64 bits."""
    s = prepare(case, seed)
    train = case["train"]
    up = lambda t: None if t is None else t.detach().double()  # noqa: E731
    if case["op"] == "norm":
        w, b = up(s["weight"]).requires_grad_(train), up(s["bias"]).requires_grad_(train)
        ys, dxs = [], []
        for i in range(case["n"]):
            x = up(s["x"][i]).requires_grad_(train)
            t = x.reshape(-1, case["groups"], case["c"] // case["groups"]).transpose(0, 1)
            var, mean = torch.var_mean(t, dim=(1, 2), unbiased=False, keepdim=True)
            t = ((t - mean) / torch.sqrt(var + EPS)).transpose(0, 1).reshape(-1, case["c"])
            y = _exact_activation(case["act"], t * w + b).reshape(x.shape)
            if train:
                y.backward(up(s["dy"][i]))
                dxs.append(x.grad)
            ys.append(y.detach())
        if not train:
            return torch.stack(ys)
        return torch.stack(ys), torch.stack(dxs), w.grad, b.grad
    if case["op"] == "gated":
        names = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if case["bias"] else [])
        t = {n: up(s[n]).requires_grad_(train) for n in names}
        f = torch.nn.functional.linear
        y = _exact_activation(case["act"], f(t["x"], t["w_gate"], t.get("b_gate"))) * f(t["x"], t["w_up"], t.get("b_up"))
        if not train:
            return y
        y.backward(up(s["dy"]))
        return (y.detach(), *(t[n].grad for n in names))
    gh, gw, length = case["gh"], case["gw"], case["gh"] * case["gw"]
    nq = s["q"].shape[2]
    where = torch.stack(torch.meshgrid(torch.arange(gh), torch.arange(gw), indexing="ij"), -1).reshape(length, 2).cuda()
    step = where[None] - where[s["start"]:s["start"] + nq][:, None]          # [nq, length, 2]
    bucket = s["buckets"].long()[step[..., 0] + gh - 1, step[..., 1] + gw - 1]
    one_hot_sum = torch.zeros(s["table"].shape, dtype=torch.float64, device=s["table"].device)
    outs = [torch.zeros(s[n].shape, dtype=torch.float64, device=s[n].device) for n in ("q", "q", "k", "v")]
    for b in range(case["batch"]):
        seen = torch.arange(length, device=s["q"].device) if s["mask"] is None else s["mask"][b].nonzero()[:, 0]
        if not len(seen):
            continue
        for h in range(case["heads"]):
            q, k, v = up(s["q"][b, h]), up(s["k"][b, h])[seen], up(s["v"][b, h])[seen]
            logits = q @ k.T / math.sqrt(case["dim"]) + up(s["table"])[:, h][bucket[:, seen]]
            p = torch.softmax(logits, -1)
            outs[0][b, h] = p @ v
            if train:
                dy = up(s["dy"][b, h])
                dp = dy @ v.T
                dl = p * (dp - (p * dp).sum(-1, keepdim=True))
                outs[1][b, h] = dl @ k / math.sqrt(case["dim"])
                outs[2][b, h, seen] = dl.T @ q / math.sqrt(case["dim"])
                outs[3][b, h, seen] = p.T @ dy
                one_hot_sum[:, h] += torch.bincount(bucket[:, seen].reshape(-1), dl.reshape(-1), s["table"].shape[0])
    return (*outs, one_hot_sum) if train else outs[0]
