"""Performance cases of the operators of a small transformer's training step and
of its answers: attention with its gradients and over a cache of keys and values,
the root-mean-square norm with the residual's addition and its gradients, and
the AdamW step over all parameters.

``listed()`` names the cases that are reported, ``draw()`` gives more of the same
ranges.  ``run`` computes a case with the framework's operators where ``own`` is
true and in plain torch operations where it is not; ``exact`` gives the
definition's values in 64 bits.

Definitions
    attention   q [B, Tq, H, D], k and v [B, Tk, Hk, D]; head h reads key head
                h // (H / Hk).  Query i of sequence b sees the keys j with
                j < lengths[b] and, if causal, j <= starts[b] + i.
                p = softmax of scale (q . k) over them, y = sum p v;
                dv = sum p g, ds = p (g . v - sum p (g . v)),
                dq = scale sum ds k, dk = scale sum ds q, with sums over the
                queries of all heads that share a key head.  A query that sees
                nothing has y = 0 and no gradient.
    norm        s = x + residual (or x), r = (mean s^2 + eps)^-1/2, y = s r w;
                ds = gs + r (g w) - s r^3 mean(g w s), for x and the residual
                alike; dw = sum over rows of g s r
    adamw       m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
                p = p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
ALIGN = 64  # elements between the parameters in the one buffer that `run` returns


def listed() -> list[dict]:
    return [
        # The newest token of one short conversation: latency alone.
        _attn("attn_answer_one", "answer", 1, 1, 500, 8, 8, 64),
        # The newest tokens of 8 requests over a cache of up to 8192 tokens each,
        # four query heads to a key head: serving, every key read once.
        _attn("attn_answer", "answer", 8, 1, 8192, 32, 8, 128, ragged=True),
        # The next 333 tokens of three prompts of other lengths behind a cache;
        # odd sizes throughout.
        _attn("attn_prompt", "prompt", 3, 333, 1777, 6, 2, 80, ragged=True),
        # A first transformer's training step: 4 texts of 128 tokens.
        _attn("attn_train_small", "train", 4, 128, 128, 4, 4, 64),
        # A training step of ordinary size, 8192 tokens (the large MLP's batch)
        # at its width of 1024.
        _attn("attn_train", "train", 4, 2048, 2048, 16, 16, 64),
        # One long text, four query heads to a key head.
        _attn("attn_long", "train", 1, 8192, 8192, 16, 4, 128),
        # The norm before the small MLP, forward and backward.
        _norm("norm_small", 64, 256),
        # The norm of a training step at the large MLP's widths.
        _norm("norm_train", 8192, 4096),
        # A first norm, without a residual, in float64 and odd sizes.
        _norm("norm_odd", 1537, 1023, residual=False, dtype="float64"),
        # The parameters of the small MLP's size: latency.
        _adamw("adamw_small", 2, 64, 256, 1000),
        # Twelve blocks of width 1024 with a table of 32000: 184 million.
        _adamw("adamw_model", 12, 1024, 4096, 32000),
        # A table of 128000 x 2048 with little behind it: 1 GB of parameters.
        _adamw("adamw_table", 1, 2048, 2048, 128000),
    ]


def _attn(name, kind, B, Tq, Tk, H, Hk, D, causal=True, ragged=False, dtype="float32"):
    return {"name": name, "op": "attn", "kind": kind, "B": B, "Tq": Tq, "Tk": Tk, "H": H,
            "Hk": Hk, "D": D, "causal": causal, "ragged": ragged, "dtype": dtype}


def _norm(name, rows, D, residual=True, dtype="float32"):
    return {"name": name, "op": "norm", "rows": rows, "D": D, "residual": residual,
            "dtype": dtype}


def _adamw(name, blocks, width, hidden, vocabulary, dtype="float32"):
    return {"name": name, "op": "adamw", "blocks": blocks, "width": width, "hidden": hidden,
            "vocabulary": vocabulary, "step": 10, "dtype": dtype}


def _log(rng, lo: int, hi: int) -> int:
    """A size spread evenly over its logarithm; odd and even alike."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["attn", "attn", "norm", "adamw"])
    dtype = "float64" if rng.random() < 0.2 else "float32"
    wide = 2 if dtype == "float64" else 1
    if op == "norm":
        D = _log(rng, 8, 16384)
        rows = _log(rng, 1, min(16384, 8192 * 4096 // (wide * D)))
        case = _norm("", rows, D, rng.random() < 0.7, dtype)
    elif op == "adamw":
        width = _log(rng, 16, 1024)
        case = _adamw("", rng.randint(1, 6 // wide), width, _log(rng, 16, 4096),
                      _log(rng, 100, 32000), dtype)
        case["step"] = _log(rng, 1, 10000)
    else:
        kind = rng.choice(["answer", "prompt", "train"])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 3, 4, 8])
        D = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128, 160, 256, rng.randint(8, 128)])
        B = _log(rng, 1, 16)
        if kind == "answer":
            Tq = rng.choice([1, 1, 1, 2, 4])
            Tk = _log(rng, 16, max(16, min(32768, 2**26 // (B * Hk * D * wide))))
            Tk = max(Tk, Tq)
        else:
            # pairs of positions x width over all heads, a sixteenth of the longest
            # listed case's at most (64 bits: a quarter of that)
            most = 2**33 // (wide * wide)
            T = _log(rng, 5, max(6, min(4096, int(math.sqrt(most / (B * H * D))))))
            Tq, Tk = T, T
            if kind == "prompt":
                Tq = rng.randint(1, T)
        case = _attn("", kind, B, Tq, Tk, H, Hk, D, kind != "train" or rng.random() < 0.6,
                     rng.random() < 0.5, dtype)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs


def _shapes(case: dict) -> list[tuple[int, ...]]:
    """The parameters of a transformer: table, blocks, last norm."""
    w, h = case["width"], case["hidden"]
    block = [(w,), (w, w), (w, w), (w, w), (w, w), (w,), (w, h), (h,), (h, w), (w,)]
    return [(case["vocabulary"], w)] + block * case["blocks"] + [(w,)]


def _places(case: dict) -> tuple[list[int], int]:
    """Where each parameter begins in one buffer, and the buffer's size."""
    at, places = 0, []
    for shape in _shapes(case):
        places.append(at)
        at += -(-math.prod(shape) // ALIGN) * ALIGN
    return places, at


def _inputs(case: dict, seed: int, new) -> dict:
    """The case's inputs from the seed alone, {name: new(values)}."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = torch.float64 if case["dtype"] == "float64" else torch.float32
    out = {}

    def normal(name, *shape, scale=1.0):
        t = torch.randn(*shape, generator=gen, device="cuda", dtype=dt)
        out[name] = new(t if scale == 1.0 else t.mul_(scale))

    if case["op"] == "attn":
        B, Tq, Tk, H, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))
        normal("q", B, Tq, H, D, scale=1.5)
        normal("k", B, Tk, Hk, D)
        normal("v", B, Tk, Hk, D)
        if case["kind"] == "train":
            normal("g", B, Tq, H, D, scale=0.01)
        if case["ragged"]:
            u = torch.rand(B, generator=gen, device="cuda", dtype=torch.float64)
            n = Tk // 2 + (u * (Tk - Tk // 2 + 1)).long().clamp_(max=Tk - Tk // 2)
            out["lengths"] = new(n.to(torch.int32))
    elif case["op"] == "norm":
        rows, D = case["rows"], case["D"]
        normal("x", rows, D)
        normal("w", D)
        if case["residual"]:
            normal("residual", rows, D, scale=3.0)
        normal("g", 1 + case["residual"], rows, D)
    else:
        _, n = _places(case)
        live = torch.zeros(n, dtype=torch.bool, device="cuda")
        for at, shape in zip(_places(case)[0], _shapes(case)):
            live[at:at + math.prod(shape)] = True
        for name, scale in (("p", 0.02), ("g", 1e-3), ("m", 3e-4), ("v", 1e-3)):
            t = torch.randn(n, generator=gen, device="cuda", dtype=dt).mul_(scale)
            t = t.square_() if name == "v" else t
            out[name] = new(t.masked_fill_(~live, 0.0))  # what lies between them is zero
    return out


def _starts(case):
    """Training sequences begin at the first key; the queries of a prompt or an
    answer are the last tokens of theirs, which is the operator's default."""
    return 0 if case["kind"] == "train" else None


def prepare(case: dict, seed: int) -> dict:
    """The inputs, in the tensors of the side that computes: the framework works
    on its own ones."""
    s = _inputs(case, seed, _own_new if own else (lambda t: t))
    s["case"] = case
    if own:
        _own_prepare(s, case)
    torch.cuda.synchronize()
    return s


# -------------------------------------------------- the framework's operators


_NT_DTYPES = {torch.float32: "float32", torch.float64: "float64", torch.int32: "int32"}
_TYPESTR = {1: ("<i4", 4), 3: ("<f4", 4), 4: ("<f8", 8)}  # by dtype code


class _Memory:
    """A contiguous framework tensor's device memory under the array
    interface, so that torch reads it in place; keeps the tensor alive."""

    def __init__(self, t) -> None:
        storage = t.storage
        typestr, item = _TYPESTR[storage.dtype]
        self._tensor = t
        self.__cuda_array_interface__ = {
            "shape": t.shape, "typestr": typestr, "version": 2,
            "data": (storage.data_ptr() + t.strides[1] * item, False)}


def _torch(t) -> torch.Tensor:
    return torch.as_tensor(_Memory(t), device="cuda")


def _own_new(values: torch.Tensor):
    import nanotorch_amd as nt

    t = nt.zeros(*values.shape, dtype=getattr(nt, _NT_DTYPES[values.dtype]), device="cuda")
    nt.sync()
    _torch(t).copy_(values)
    torch.cuda.synchronize()
    return t


def _own_prepare(s, case):
    from nanotorch_amd import nn

    if case["op"] == "adamw":
        parameters = []
        for at, shape in zip(_places(case)[0], _shapes(case)):
            n = math.prod(shape)
            p = s["p"][at:at + n].reshape(*shape)
            p.enable_grad()
            (p * s["g"][at:at + n].reshape(*shape)).sum().backward()  # p.grad = g
            parameters.append(p)
        s["optimizer"] = nn.AdamW(parameters, LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                                  weight_decay=DECAY)
        s["optimizer"].load_moments(s.pop("m"), s.pop("v"), case["step"])
        return
    for name in ("q", "k", "v", "x", "w", "residual"):
        if name in s and case.get("kind", "train") == "train":
            s[name].enable_grad()


def run(s: dict):
    return (_RUN_OWN if own else _RUN_PLAIN)[s["case"]["op"]](s, s["case"])


def _own_attn(s, case):
    import nanotorch_amd as nt

    y = nt.attention(s["q"], s["k"], s["v"], causal=case["causal"], lengths=s.get("lengths"),
                     starts=_starts(case))
    out = {"y": _torch(y)}
    if case["kind"] == "train":
        dq, dk, dv = y.grad_fn.backward(s["g"])[:3]
        out |= {"dq": _torch(dq), "dk": _torch(dk), "dv": _torch(dv)}
    return out


def _own_norm(s, case):
    import nanotorch_amd as nt

    if not case["residual"]:
        y = nt.rms_norm(s["x"], s["w"], eps=EPS)
        dx, dw = y.grad_fn.backward(s["g"][0])[:2]
        return {"y": _torch(y), "ds": _torch(dx), "dw": _torch(dw)}
    y, total = nt.rms_norm(s["x"], s["w"], residual=s["residual"], eps=EPS)
    both = y.grad_fn.inputs[0]  # y and the sum, whose gradients arrive together
    dx, dw = both.grad_fn.backward(s["g"])[:2]
    return {"y": _torch(y), "s": _torch(total), "ds": _torch(dx), "dw": _torch(dw)}


def _own_adamw(s, case):
    s["optimizer"].step()
    m, v = s["optimizer"].moments()
    return {"p": _torch(s["p"]), "m": _torch(m), "v": _torch(v)}


_RUN_OWN = {"attn": _own_attn, "norm": _own_norm, "adamw": _own_adamw}


# ------------------------------------------------------------- plain forms


def _visible(s, case):
    """[B, 1, 1, Tq, Tk]: which keys each query sees."""
    Tq, Tk = case["Tq"], case["Tk"]
    j = torch.arange(Tk, device="cuda")
    n = s["lengths"].long() if "lengths" in s else torch.full((case["B"],), Tk, device="cuda")
    seen = j < n[:, None, None]
    if case["causal"]:
        start = _starts(case)
        first = n - Tq if start is None else torch.full_like(n, start)
        i = torch.arange(Tq, device="cuda")
        seen = seen & (j <= (first[:, None] + i)[:, :, None])
    return seen.expand(case["B"], Tq, Tk)[:, None, None]


def _plain_attn(s, case):
    B, Tq, Tk, H, Hk, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hk", "D"))
    G, scale = H // Hk, D ** -0.5

    def heads(x):  # [B, Tq, H, D] -> [B, Hk, G Tq, D]
        return x.reshape(B, Tq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Tq, D)

    def back(x):
        return x.reshape(B, Hk, G, Tq, D).permute(0, 3, 1, 2, 4).reshape(B, Tq, H, D)

    q = heads(s["q"])
    k, v = (s[n].permute(0, 2, 1, 3).contiguous() for n in "kv")
    seen = _visible(s, case)
    z = torch.matmul(q, k.transpose(2, 3)).mul_(scale).reshape(B, Hk, G, Tq, Tk)
    z = z.masked_fill_(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp_(z.sub_(torch.where(top > -math.inf, top, 0.0)))
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0)).reshape(B, Hk, G * Tq, Tk)
    out = {"y": back(torch.matmul(p, v))}
    if case["kind"] == "train":
        g = heads(s["g"])
        dp = torch.matmul(g, v.transpose(2, 3))
        dv = torch.matmul(p.transpose(2, 3), g)
        mean = (p * dp).sum(-1, keepdim=True)
        ds = dp.sub_(mean).mul_(p).mul_(scale)
        out["dq"] = back(torch.matmul(ds, k))
        out["dk"] = torch.matmul(ds.transpose(2, 3), q).permute(0, 2, 1, 3).contiguous()
        out["dv"] = dv.permute(0, 2, 1, 3).contiguous()
    return out


def _plain_norm(s, case):
    x = s["x"] + s["residual"] if case["residual"] else s["x"]
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    g, w = s["g"][0], s["w"]
    out = {"y": x * r * w}
    gw = g * w
    ds = r * gw - x * (r * r * r * (gw * x).mean(1, keepdim=True))
    out["ds"] = ds + s["g"][1] if case["residual"] else ds
    out["dw"] = (g * (x * r)).sum(0)
    if case["residual"]:
        out["s"] = x
    return out


def _plain_adamw(s, case):
    # all parameters as one buffer, as a program keeps them that has no step
    # over many tensors
    p, g, m, v = s["p"], s["g"], s["m"], s["v"]
    t = s["t"] = s.get("t", case["step"]) + 1
    m.mul_(BETA1).add_(g * (1 - BETA1))
    v.mul_(BETA2).add_(g * g * (1 - BETA2))
    p.mul_(1 - LR * DECAY)
    p.sub_(m * (LR / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS))
    return {"p": p, "m": m, "v": v}


_RUN_PLAIN = {"attn": _plain_attn, "norm": _plain_norm, "adamw": _plain_adamw}


# -------------------------------------------------------------------- work


def _pairs(case: dict) -> tuple[float, float]:
    """Per head: pairs of a query and a key that it sees, and keys that any
    query sees, over all sequences; ragged lengths by their mean."""
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    n = (Tk // 2 + Tk) / 2 if case["ragged"] else Tk
    if not case["causal"]:
        return B * Tq * n, B * n
    if case["kind"] == "train":
        m = min(n, Tq)
        return B * (m * (m + 1) / 2 + (Tq - m) * m), B * m
    m = min(Tq, n)  # queries that see anything
    return B * m * (n - (m - 1) / 2), B * n


def work(case: dict) -> dict:
    item = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "attn":
        H, Hk, D = case["H"], case["Hk"], case["D"]
        pairs, keys = _pairs(case)
        queries = case["B"] * case["Tq"]
        train = case["kind"] == "train"
        # q, y, (g, dq) and the keys and values that are seen, (all of dk and dv)
        moved = queries * H * D * (4 if train else 2) + 2 * keys * Hk * D
        if train:
            moved += 2 * case["B"] * case["Tk"] * Hk * D
        # two products forward, five backward
        return {"bytes": item * moved, "flops": 2 * pairs * H * D * (7 if train else 2)}
    if case["op"] == "norm":
        n = case["rows"] * case["D"]
        # x, g and y, ds; with a residual that, its sum and the sum's gradient
        return {"bytes": item * (n * (7 if case["residual"] else 4) + 2 * case["D"]),
                "flops": n * 14}
    n = sum(math.prod(shape) for shape in _shapes(case))
    return {"bytes": 7 * item * n, "flops": 15 * n}


# ------------------------------------------------------------------- exact


def exact(case: dict, seed: int):
    v = {k: (t.double() if t.is_floating_point() else t)
         for k, t in _inputs(case, seed, lambda t: t).items()}
    return {"attn": _exact_attn, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](v, case)


def _exact_attn(v, case):
    B, Tq, Tk, G = case["B"], case["Tq"], case["Tk"], case["H"] // case["Hk"]
    train = case["kind"] == "train"
    names = ("y", "dq", "dk", "dv") if train else ("y",)
    out = {n: torch.zeros_like(v[{"y": "q"}.get(n, n[1:])]) for n in names}
    for b in range(B):
        n = int(v["lengths"][b]) if case["ragged"] else Tk
        first = 0 if train else n - Tq
        hidden = torch.ones(Tq, Tk, dtype=torch.bool, device="cuda")
        hidden[:, :n] = False
        if case["causal"]:
            hidden |= torch.ones_like(hidden).triu(first + 1)
        live = ~hidden.all(1)
        for h in range(case["H"]):
            q, k, u = v["q"][b, :, h], v["k"][b, :, h // G], v["v"][b, :, h // G]
            z = torch.mm(q, k.T.contiguous()) / math.sqrt(case["D"])
            z.masked_fill_(hidden, -1e300)
            # (torch.softmax in float64 keeps only 24 bits of rows over 1024)
            p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) * live[:, None]
            y = torch.mm(p, u)
            out["y"][b, :, h] = y
            if not train:
                continue
            g = v["g"][b, :, h]
            d = p * (torch.mm(g, u.T.contiguous()) - (g * y).sum(1, keepdim=True))
            d /= math.sqrt(case["D"])
            out["dq"][b, :, h] = torch.mm(d, k)
            out["dk"][b, :, h // G] += torch.mm(d.T.contiguous(), q)
            out["dv"][b, :, h // G] += torch.mm(p.T.contiguous(), g)
    return out


def _exact_norm(v, case):
    x = v["x"] + v["residual"] if case["residual"] else v["x"]
    inverse = torch.rsqrt(x.square().mean(1) + EPS)
    n = x * inverse[:, None]  # rows of length about sqrt(D)
    out = {"y": n * v["w"], "dw": torch.linalg.vecdot(n, v["g"][0], dim=0)}
    dn = v["g"][0] * v["w"]
    out["ds"] = (dn - n * torch.linalg.vecdot(dn, n, dim=1)[:, None] / case["D"])
    out["ds"] *= inverse[:, None]
    if case["residual"]:
        out["ds"] += v["g"][1]
        out["s"] = x
    return out


def _exact_adamw(v, case):
    t = case["step"] + 1
    m = torch.lerp(v["g"], v["m"], BETA1)
    u = torch.lerp(v["g"] ** 2, v["v"], BETA2)
    rate = m / -math.expm1(t * math.log(BETA1))
    rate /= (u / -math.expm1(t * math.log(BETA2))).sqrt_().add_(ADAM_EPS)
    return {"p": v["p"] - LR * (rate + DECAY * v["p"]), "m": m, "v": u}
