"""Timed cases of the operators around a block's experts: pairs sorted by expert and back, products of
the sorted rows, norms at both ends of the block. Forward alone (serving) or with every gradient (tuning).

A case is one pass of one operator:

  sort     `dispatch.plan` of a routing, `dispatch.dispatch` of the tokens and `dispatch.combine` of the
           experts' rows; with gradients: those of the tokens, of the experts' rows and of the weights
  product  `grouped.product`: sorted rows times their experts' matrices; with gradients: those of the
           rows, of the matrices and of the biases
  norm     `norm.enter` (a norm before a block), or `norm.leave` (the norm behind it, its gate and scale, the
           residual sum and the next block's norm, in one pass); with gradients: those of all inputs

Inputs are N(0, 1) with a few channels much larger than the rest, as a trained model's residual stream
has them, weights N(0, 0.02), norm weights and gates near one; the routing follows a Zipf law where
`zipf` is set, and `drop` is the share of pairs that belong to no expert here (another device's, or
padding). Everything is made on the GPU from the seed alone.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6

# (hidden, projection outputs, experts, top-k) of the package's layer shapes; the outputs are those of the
# gate and up projections as one matrix.
_QWEN3 = dict(hidden=2048, inter=1536, experts=128, top_k=8, zipf=1.1)
_OLMOE = dict(hidden=2048, inter=2048, experts=64, top_k=8, zipf=0.0)
_E256 = dict(hidden=2048, inter=1024, experts=256, top_k=8, zipf=1.1)
_GPTOSS = dict(hidden=2880, inter=2880, experts=128, top_k=4, zipf=0.0)


def _sort(name, shape, tokens, dtype="bfloat16", train=False, drop=0.0, **other):
    c = dict(shape, **other)
    return dict(name=name, kind="sort", tokens=tokens, hidden=c["hidden"], experts=c["experts"], top_k=c["top_k"],
                zipf=c["zipf"], drop=drop, dtype=dtype, train=train)


def _product(name, shape, tokens, dtype="bfloat16", train=False, bias=False, drop=0.0, **other):
    return dict(shape, **other, name=name, kind="product", tokens=tokens, bias=bias, drop=drop, dtype=dtype, train=train)


def _norm(name, tokens, hidden, dtype="bfloat16", residual="bfloat16", form="leave", post=True, gate="none", next=True,
          train=False):
    return dict(name=name, kind="norm", tokens=tokens, hidden=hidden, dtype=dtype, residual=residual, form=form,
                post=post, gate=gate, next=next, train=train)


def listed():
    return [
        # 8 users of a many-expert layer: a decode step, all latency
        _sort("sort8", _E256, 8),
        # an ordinary prompt chunk
        _sort("sort2048", _QWEN3, 2048),
        # a tuning step's chunk: every gradient
        _sort("sort8192-train", _QWEN3, 8192, train=True),
        # one device's share of the experts, an odd width and count of tokens, fp32 rows
        _sort("sort1999-f32-drop", _OLMOE, 1999, "float32", train=True, drop=0.5, hidden=1001, experts=60),
        # one token through the gate and up matrices of its 8 experts
        _product("product1", _QWEN3, 1),
        # a short prompt through large experts with biases, fp16: every expert hit by few rows
        _product("product301-f16", _GPTOSS, 301, "float16", bias=True),
        # a tuning step of smaller, odd experts with biases, some pairs dropped
        _product("product701-train", _GPTOSS, 701, train=True, bias=True, drop=0.1, hidden=1000, inter=712, experts=60),
        # a tuning step's chunk
        _product("product4096-train", _QWEN3, 4096, train=True),
        # between two blocks of single-user generation
        _norm("norm1", 1, 2880),
        # between two blocks of a prompt chunk, a gate for each channel
        _norm("norm2048", 2048, 2048, gate="channel"),
        # a tuning step: residual stream in fp32, a gate for each token
        _norm("norm16384-train", 16384, 2048, residual="float32", gate="token", train=True),
        # the norm before a block alone, fp16, odd sizes, with gradients
        _norm("enter4999-f16-train", 4999, 1001, "float16", "float16", form="enter", train=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges: 1 to 16384 tokens, widths of 64 to 4096 values (odd ones too,
    products: multiples of 8), 4 to 256 experts, every type, with and without gradients."""
    kind = rng.choice(["sort", "product", "norm"])
    train = rng.random() < 0.5
    if kind == "norm":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        form = rng.choice(["enter", "leave", "leave"])
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), hidden=rng.choice([_log_int(rng, 64, 2048), 64 * rng.randint(8, 32)]),
                    dtype=dtype, residual=dtype if form == "enter" else rng.choice([dtype, "float32"]), form=form,
                    post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "token", "full"]),
                    next=rng.random() < 0.7, train=train)
    shape = dict(rng.choice([_QWEN3, _OLMOE, _E256, _GPTOSS]))
    if rng.random() < 0.6:
        shape.update(hidden=8 * _log_int(rng, 8, 360), inter=8 * _log_int(rng, 8, 360),
                     experts=rng.choice([4, 8, 16, 32, 60, 64, 96, 128, 160, 256]))
        shape["top_k"] = min(rng.choice([1, 2, 4, 6, 8]), shape["experts"])
    c = dict(shape, kind=kind, tokens=_log_int(rng, 1, 8192), drop=rng.choice([0.0, 0.0, 0.1, 0.5]), train=train)
    if kind == "sort":
        del c["inter"]
        c["dtype"] = rng.choice(["bfloat16", "float16", "float32"])
        if rng.random() < 0.4:
            c["hidden"] = _log_int(rng, 64, 2880)
    else:
        c.update(dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), bias=rng.random() < 0.5)
    top = [v for v in listed() if v["kind"] == kind and v["name"].endswith(("8192-train", "4096-train"))][0]
    most = work(top)
    while any(work(c)[k] > most[k] for k in most):
        c["tokens"] = c["tokens"] * 3 // 4
        if c["tokens"] < 64 and kind == "product":
            c["experts"] = max(c["top_k"], c["experts"] // 2)
    c["tokens"] = max(1, c["tokens"])
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed, *tags):
    g = torch.Generator(device=DEV)
    v = seed & 0xFFFFFFFF
    for t in tags:
        v = (v * 1000003 + t + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(v)
    return g


def _normal(shape, seed, *tags, dtype="float32", scale=1.0):
    return torch.randn(shape, generator=_gen(seed, *tags), device=DEV).mul_(scale).to(getattr(torch, dtype))


def _activations(rows, cols, dtype, seed, *tags):
    """N(0, 1), one channel in 64 twenty times larger."""
    g = _gen(seed, 7, *tags)
    x = torch.randn((rows, cols), generator=g, device=DEV)
    big = torch.rand(cols, generator=g, device=DEV) < 1 / 64
    return (x * torch.where(big, 20.0, 1.0)).to(getattr(torch, dtype))


def _routing(c, seed):
    """(experts [T, k] int32, -1 where dropped, weights [T, k] fp32 that sum to one over the k)."""
    E, T, k = c["experts"], c["tokens"], c["top_k"]
    g = _gen(seed, 8)
    z = -c["zipf"] * torch.log(torch.randperm(E, generator=g, device=DEV).double() + 1.0)
    u = torch.rand((T, E), generator=g, device=DEV, dtype=torch.float64).clamp(1e-12, 1 - 1e-12)
    v, idx = (z - torch.log(-torch.log(u))).topk(k, -1)
    idx = idx.int()
    if c["drop"]:
        idx = torch.where(torch.rand((T, k), generator=g, device=DEV) < c["drop"], -1, idx)
    return idx.contiguous(), torch.softmax(v, -1).float().contiguous()


class _State:
    """What a program holds between calls."""


def prepare(case, seed):
    c = case
    st = _State()
    st.case = c
    if own:
        from bigrig_amd import dispatch, grouped, lib, norm
        lib.init(0)
        st.dispatch, st.grouped, st.norm = dispatch, grouped, norm
    T, H, dt = c["tokens"], c["hidden"], c["dtype"]
    leaves = []
    if c["kind"] == "sort":
        st.idx, st.w = _routing(c, seed)
        n = st.idx.numel()
        st.x = _activations(T, H, dt, seed)
        st.y = _normal((n, H), seed, 1, dtype=dt)           # what the experts made of the rows
        leaves = [st.x, st.y, st.w]
        if c["train"]:
            st.drows = _normal((n, H), seed, 2, dtype=dt)
            st.dout = _normal((T, H), seed, 3, dtype=dt)
    elif c["kind"] == "product":
        idx, _ = _routing(c, seed)
        e = idx.reshape(-1)
        count = torch.bincount(e[e >= 0].long(), minlength=c["experts"])
        st.offsets = torch.cat((count.new_zeros(1), count.cumsum(0))).int()
        n = e.numel()
        st.rows = _activations(n, H, dt, seed)
        st.weight = _normal((c["experts"], c["inter"], H), seed, 4, dtype=dt, scale=0.02)
        st.bias = _normal((c["experts"], c["inter"]), seed, 5, dtype=dt, scale=0.02) if c["bias"] else None
        leaves = [st.rows, st.weight] + ([st.bias] if c["bias"] else [])
        if c["train"]:
            st.dout = _normal((n, c["inter"]), seed, 6, dtype=dt)
    else:
        near_one = lambda shape, tag: (_normal(shape, seed, tag) * 0.1 + 1.0).to(getattr(torch, dt))
        if c["form"] == "enter":
            st.x = _activations(T, H, dt, seed)
            st.weight = near_one((H,), 9)
            leaves = [st.x, st.weight]
        else:
            st.y = _normal((T, H), seed, 1, dtype=dt)
            st.r = _activations(T, H, c["residual"], seed)
            st.post = near_one((H,), 10) if c["post"] else None
            shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[c["gate"]]
            st.gate = None if shape is None else near_one(shape, 11)
            st.next = near_one((H,), 12) if c["next"] else None
            st.scale = 0.5
            leaves = [t for t in (st.y, st.r, st.post, st.gate, st.next) if t is not None]
            if c["train"]:
                st.dr = _normal((T, H), seed, 13, dtype=c["residual"])
        if c["train"] and (c["form"] == "enter" or c["next"]):
            st.dh = _normal((T, H), seed, 14, dtype=dt)
    st.leaves = leaves
    if own and c["train"]:
        for t in leaves:
            t.requires_grad_(True)
    return st


# ------------------------------------------------------------------ plain forms
def _sorted(idx, E):
    """(order [n] -1 behind the last, position [n] -1 where dropped, offsets [E + 1]), int32."""
    e = idx.reshape(-1)
    n = e.numel()
    kept = (e >= 0) & (e < E)
    order = torch.argsort(torch.where(kept, e, E), stable=True)
    count = torch.bincount(torch.where(kept, e, E).long(), minlength=E + 1)[:E]
    offsets = torch.cat((count.new_zeros(1), count.cumsum(0)))
    place = torch.arange(n, device=e.device)
    position = torch.empty_like(place)
    position[order] = place
    order = torch.where(place < offsets[-1], order, -1)
    return order.int(), torch.where(kept, position, -1).int(), offsets.int()


def _plain_sort(st):
    c = st.case
    T, k, H = c["tokens"], c["top_k"], c["hidden"]
    order, position, offsets = _sorted(st.idx, c["experts"])
    used = (order >= 0)[:, None]
    token = (order.clamp(min=0) // k).long()
    rows = torch.where(used, st.x[token], 0)
    at = position.clamp(min=0).long()
    on = (position >= 0).view(T, k, 1)
    mine = torch.where(on, st.y[at].float().view(T, k, H), 0.0)
    out = (mine * st.w[..., None]).sum(1).to(st.y.dtype)
    res = [order, offsets, rows, out]
    if c["train"]:
        res.append(torch.where(on, st.drows[at].float().view(T, k, H), 0.0).sum(1).to(st.x.dtype))
        w = st.w.reshape(-1)[order.clamp(min=0).long()]
        res.append(torch.where(used, w[:, None] * st.dout[token].float(), 0.0).to(st.y.dtype))
        res.append((mine * st.dout.float()[:, None]).sum(-1))
    return res


def _plain_product(st):
    c = st.case
    at = st.offsets.tolist()
    dt = st.rows.dtype
    out = torch.zeros((st.rows.shape[0], c["inter"]), dtype=dt, device=DEV)
    if c["train"]:
        drows = torch.zeros_like(st.rows)
        dweight = torch.zeros_like(st.weight)
        dbias = None if st.bias is None else torch.zeros_like(st.bias)
    for e in range(c["experts"]):
        lo, hi = at[e], at[e + 1]
        if lo == hi:
            continue
        x, w = st.rows[lo:hi].float(), st.weight[e].float()
        y = x @ w.T
        out[lo:hi] = (y if st.bias is None else y + st.bias[e].float()).to(dt)
        if c["train"]:
            d = st.dout[lo:hi].float()
            drows[lo:hi] = (d @ w).to(dt)
            dweight[e] = (d.T @ x).to(dt)
            if dbias is not None:
                dbias[e] = d.sum(0).to(dt)
    if not c["train"]:
        return out
    return [out, drows, dweight] + ([] if dbias is None else [dbias])


def _rms(x):
    """1 / root mean square of each row, fp32 [T, 1]."""
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _rms_back(x, rstd, g):
    """The gradient of x * rstd(x) given that of the result."""
    n = x * rstd
    return rstd * (g - n * (g * n).mean(-1, keepdim=True))


def _plain_norm(st):
    c = st.case
    dt = getattr(torch, c["dtype"])
    if c["form"] == "enter":
        x, w = st.x.float(), st.weight.float()
        s = _rms(x)
        h = (x * s * w).to(dt)
        if not c["train"]:
            return h
        d = st.dh.float()
        return [h, _rms_back(x, s, d * w).to(dt), (d * x * s).sum(0).to(dt)]
    y, r = st.y.float(), st.r.float()
    sy = _rms(y) if c["post"] else None
    u = y * sy * st.post.float() if c["post"] else y
    gate = 1.0 if st.gate is None else st.gate.float()
    new = (r + st.scale * gate * u).to(st.r.dtype)
    res = [new]
    if c["next"]:
        n = new.float()
        sn = _rms(n)
        res.append((n * sn * st.next.float()).to(dt))
    if not c["train"]:
        return res
    d = st.dr.float()
    if c["next"]:
        dh = st.dh.float()
        d = d + _rms_back(n, sn, dh * st.next.float())
    du = st.scale * gate * d
    res.append((_rms_back(y, sy, du * st.post.float()) if c["post"] else du).to(dt))
    res.append(d.to(st.r.dtype))
    if c["post"]:
        res.append((du * y * sy).sum(0).to(dt))
    if st.gate is not None:
        dg = st.scale * u * d
        dg = dg.sum(0) if c["gate"] == "channel" else dg.sum(-1, keepdim=True) if c["gate"] == "token" else dg
        res.append(dg.to(dt))
    if c["next"]:
        res.append((dh * n * sn).sum(0).to(dt))
    return res


def run(state):
    st, c = state, state.case
    if not own:
        return {"sort": _plain_sort, "product": _plain_product, "norm": _plain_norm}[c["kind"]](st)
    if c["kind"] == "sort":
        plan = st.dispatch.plan(st.idx, c["experts"])
        rows = st.dispatch.dispatch(st.x, plan)
        out = st.dispatch.combine(st.y, plan, st.w)
        res, grads = [plan.order, plan.offsets, rows, out], None
        if c["train"]:
            grads = torch.autograd.grad([rows, out], st.leaves, [st.drows, st.dout])
    elif c["kind"] == "product":
        out = st.grouped.product(st.rows, st.weight, st.offsets, st.bias)
        if not c["train"]:
            return out
        res, grads = [out], torch.autograd.grad(out, st.leaves, st.dout)
    elif c["form"] == "enter":
        h = st.norm.enter(st.x, st.weight, eps=EPS)
        if not c["train"]:
            return h
        res, grads = [h], torch.autograd.grad(h, st.leaves, st.dh)
    else:
        got = st.norm.leave(st.y, st.r, weight=st.post, gate=st.gate, scale=st.scale, next_weight=st.next, eps=EPS)
        res, grads = list(got) if c["next"] else [got], None
        if c["train"]:
            grads = torch.autograd.grad(res, st.leaves, [st.dr, st.dh] if c["next"] else [st.dr])
    return [t.detach() for t in res] + list(grads or [])


# ------------------------------------------------------------------ what a pass has to do
def _size(dtype):
    return 4 if dtype == "float32" else 2


def _distinct(c):
    """Experts the routing hits on average."""
    p = [1.0 / (i + 1.0) ** c["zipf"] for i in range(c["experts"])]
    total = sum(p)
    n = c["tokens"] * (1.0 - c["drop"])
    return sum(1.0 - (1.0 - min(1.0, c["top_k"] * v / total)) ** n for v in p)


def work(case):
    c = case
    T, H, s = c["tokens"], c["hidden"], _size(c["dtype"])
    if c["kind"] == "sort":
        n = T * c["top_k"]
        kept = int(n * (1.0 - c["drop"]))
        by = 4 * n + 4 * n + 4 * (c["experts"] + 1) + 4 * kept                    # idx, order, offsets, w
        by += s * H * (T + n + kept + T)                                          # x, rows, y, out
        fl = 2 * kept * H
        if c["train"]:
            by += s * H * (kept + T + T + n) + 4 * n                              # drows, dx, dout, dy, dw
            fl += 4 * kept * H
        return {"bytes": by, "flops": fl}
    if c["kind"] == "product":
        n, N, E = T * c["top_k"], c["inter"], c["experts"]
        kept = n * (1.0 - c["drop"])
        by = int(s * (kept * H + n * N + _distinct(c) * N * (H + bool(c["bias"])))) + 4 * (E + 1)
        fl = int(2 * kept * N * H)
        if c["train"]:
            by += int(s * (kept * N + n * H + E * N * (H + bool(c["bias"]))))
            fl *= 3
        return {"bytes": by, "flops": fl}
    if c["form"] == "enter":
        by, fl = s * (2 * T * H + H), 4 * T * H
        return {"bytes": by + (s * (2 * T * H + H) if c["train"] else 0), "flops": fl * (3 if c["train"] else 1)}
    rs = _size(c["residual"])
    gate = {"none": 0, "channel": H, "token": T, "full": T * H}[c["gate"]]
    once = T * H * (s + 2 * rs + (s if c["next"] else 0)) + s * (gate + H * (c["post"] + c["next"]))
    back = T * H * (2 * rs + s + (s if c["next"] else 0)) + s * (gate + H * (c["post"] + c["next"]))
    return {"bytes": once + (back if c["train"] else 0), "flops": T * H * (10 + (24 if c["train"] else 0))}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_sort(st):
    c = st.case
    T, k, E = c["tokens"], c["top_k"], c["experts"]
    ids = st.idx.cpu().reshape(-1).tolist()
    runs = [[] for _ in range(E)]
    for p, e in enumerate(ids):
        if 0 <= e < E:
            runs[e].append(p)
    order = [p for run in runs for p in run]
    n = len(order)
    offsets = [0]
    for run in runs:
        offsets.append(offsets[-1] + len(run))
    pair = torch.tensor(order, dtype=torch.long, device=DEV)
    x, y, w = st.x.double(), st.y.double(), st.w.double().reshape(-1)
    rows = torch.zeros((T * k, c["hidden"]), dtype=torch.float64, device=DEV)
    rows[:n] = x[pair // k]
    out = torch.zeros((T, c["hidden"]), dtype=torch.float64, device=DEV)
    out.index_add_(0, pair // k, w[pair, None] * y[:n])
    full = torch.full((T * k,), -1, dtype=torch.int32, device=DEV)
    full[:n] = pair.int()
    res = [full, torch.tensor(offsets, dtype=torch.int32, device=DEV), rows, out]
    if c["train"]:
        dout = st.dout.double()
        dx = torch.zeros_like(x).index_add_(0, pair // k, st.drows[:n].double())
        dy = torch.zeros_like(y)
        dy[:n] = w[pair, None] * dout[pair // k]
        dw = torch.zeros(T * k, dtype=torch.float64, device=DEV)
        dw[pair] = torch.linalg.vecdot(dout[pair // k], y[:n])
        res += [dx, dy, dw.view(T, k)]
    return res


def _exact_product(st):
    c = st.case
    P, E, N, H = st.rows.shape[0], c["experts"], c["inter"], c["hidden"]
    edge = st.offsets.cpu().numpy()
    out = torch.zeros((P, N), dtype=torch.float64, device=DEV)
    dx = torch.zeros((P, H), dtype=torch.float64, device=DEV)
    dw = torch.zeros((E, N, H), dtype=torch.float64, device=DEV) if c["train"] else None
    db = torch.zeros((E, N), dtype=torch.float64, device=DEV)
    for e in range(E):
        span = slice(int(edge[e]), int(edge[e + 1]))
        x, w = st.rows[span].double(), st.weight[e].double()
        out[span] = torch.mm(x, w.t().contiguous())
        if c["bias"]:
            out[span] += st.bias[e].double()
        if c["train"]:
            d = st.dout[span].double()
            dx[span] = torch.mm(d, w)
            dw[e] = torch.mm(d.t().contiguous(), x)
            db[e] = d.sum(0)
    if not c["train"]:
        return out
    return [out, dx, dw] + ([db] if c["bias"] else [])


def _exact_norm(st):
    c = st.case

    def normal(v):
        size = torch.sqrt(torch.linalg.vecdot(v, v) / v.shape[-1] + EPS)[:, None]
        return v / size, size

    def back(unit, size, g):
        return (g - unit * torch.linalg.vecdot(unit, g)[:, None] / unit.shape[-1]) / size

    if c["form"] == "enter":
        unit, size = normal(st.x.double())
        w = st.weight.double()
        if not c["train"]:
            return unit * w
        d = st.dh.double()
        return [unit * w, back(unit, size, w * d), (unit * d).sum(0)]
    y, r = st.y.double(), st.r.double()
    T, H = y.shape
    gate = st.scale * (st.gate.double() if st.gate is not None else torch.ones((), dtype=torch.float64, device=DEV))
    w = st.post.double() if c["post"] else None
    u = y
    if c["post"]:
        yu, ysize = normal(y)
        u = yu * w
    new = r + gate * u
    res = [new]
    if c["next"]:
        # the next block's norm is of the residual as it is held
        unit, size = normal(new.to(st.r.dtype).double())
        res.append(unit * st.next.double())
    if c["train"]:
        d = st.dr.double()
        if c["next"]:
            d = d + back(unit, size, st.next.double() * st.dh.double())
        du = d * gate
        res += [back(yu, ysize, w * du) if c["post"] else du, d]
        if c["post"]:
            res.append((yu * du).sum(0))
        if st.gate is not None:
            dg = st.scale * d * u
            res.append({"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True), "full": lambda: dg}[c["gate"]]())
        if c["next"]:
            res.append((unit * st.dh.double()).sum(0))
    return res


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"sort": _exact_sort, "product": _exact_product, "norm": _exact_norm}[case["kind"]](st)
