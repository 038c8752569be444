"""Performance cases of the operators of a token model: the embedding lookup and
its gradient, dropout from a counter-based generator, and the log probabilities
of given tokens with entropy, top alternatives and the gradient.

``listed()`` names the cases that are reported, ``draw()`` gives more of the
same ranges.  ``run`` computes a case with the framework's operators where
``own`` is true and in plain torch operations where it is not; ``exact`` gives
the definition's values in 64 bits.

Definitions
    embedding   y[i] = scale * W[t_i];  dW[v] = scale * sum of g[i] over t_i = v
    dropout     y_i = x_i / (1 - p) where r_i >= round(p * 2^32), else 0, with
                r_i word i mod 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
                "Parallel random numbers: as easy as 1, 2, 3", SC 2011) under
                the key seed at the counter (i div 4, offset); i is the
                row-major index
    logprobs    lp = z_t - lse(z), H = -sum p log p, p = exp(z - lse(z)); the
                top alternatives by falling z, ties to the lowest token; rows
                whose token is -100 are left out: lp = H = 0, no alternatives
                (-inf, token -1), no gradient
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

IGNORED = -100


def listed() -> list[dict]:
    return [
        # The lookup of a first token model's training step (64 tokens, the
        # small MLP's width): bound by latency.
        {"name": "embed_small", "op": "embed", "V": 1000, "D": 64, "N": 64, "train": True,
         "dtype": "float32", "int32": False, "zipf": True, "scale": 1.0},
        # The newest token of 8 requests looked up: serving, latency again.
        {"name": "embed_answer", "op": "embed", "V": 50000, "D": 1024, "N": 8, "train": False,
         "dtype": "float32", "int32": False, "zipf": True, "scale": 32.0},
        # A training step of ordinary size: 8192 tokens (the large MLP's
        # batch) at its width of 1024; tokens numbered by how common they are.
        {"name": "embed_train", "op": "embed", "V": 32000, "D": 1024, "N": 8192, "train": True,
         "dtype": "float32", "int32": False, "zipf": True, "scale": 32.0},
        # A long batch over a large vocabulary: 1 GB of table, every row of
        # its gradient written.
        {"name": "embed_long", "op": "embed", "V": 128000, "D": 2048, "N": 65536, "train": True,
         "dtype": "float32", "int32": True, "zipf": True, "scale": 1.0},
        # Dropout behind the small MLP's hidden layer, forward and backward.
        {"name": "dropout_small", "op": "dropout", "rows": 64, "cols": 256, "p": 0.5,
         "dtype": "float32", "x_t": False},
        # Dropout behind the large MLP's hidden layer, forward and backward.
        {"name": "dropout_large", "op": "dropout", "rows": 8192, "cols": 4096, "p": 0.1,
         "dtype": "float32", "x_t": False},
        # Odd sizes, float64, the input a transposed view: data as it comes.
        {"name": "dropout_odd", "op": "dropout", "rows": 1537, "cols": 1023, "p": 0.3,
         "dtype": "float64", "x_t": True},
        # The loss of a small classifier's step: 64 rows over 1000 classes.
        {"name": "logp_small", "op": "logp", "rows": 64, "V": 1000, "train": True,
         "entropy": False, "top": 0, "masked": 0.0, "ignored": 0.0, "dtype": "float32",
         "int32": False},
        # The next token of 8 requests over a large vocabulary, with the
        # alternatives that a server returns: few rows, long ones.
        {"name": "logp_answer", "op": "logp", "rows": 8, "V": 128000, "train": False,
         "entropy": True, "top": 8, "masked": 0.0, "ignored": 0.0, "dtype": "float32",
         "int32": False},
        # Scoring given texts: odd rows, a tenth of the tokens forbidden
        # (-inf), five alternatives each.
        {"name": "logp_score", "op": "logp", "rows": 2000, "V": 50001, "train": False,
         "entropy": True, "top": 5, "masked": 0.1, "ignored": 0.0, "dtype": "float32",
         "int32": True},
        # Cross-entropy of the large MLP's batch over its 1000 classes,
        # forward and backward.
        {"name": "logp_classes", "op": "logp", "rows": 8192, "V": 1000, "train": True,
         "entropy": False, "top": 0, "masked": 0.0, "ignored": 0.0, "dtype": "float32",
         "int32": False},
        # A policy's training step over 1 GB of logits: weighted log
        # probabilities and an entropy bonus, a tenth of the rows padding.
        {"name": "logp_train", "op": "logp", "rows": 8192, "V": 32000, "train": True,
         "entropy": True, "top": 0, "masked": 0.0, "ignored": 0.1, "dtype": "float32",
         "int32": False},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A size spread evenly over its logarithm; odd and even alike."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["embed", "dropout", "logp"])
    dtype = "float64" if rng.random() < 0.2 else "float32"
    wide = 2 if dtype == "float64" else 1
    if op == "embed":
        return {"op": "embed", "V": _log(rng, 100, 128000), "D": _log(rng, 16, 2048 // wide),
                "N": _log(rng, 1, 65536), "train": rng.random() < 0.7, "dtype": dtype,
                "int32": rng.random() < 0.5, "zipf": rng.random() < 0.7,
                "scale": rng.choice([1.0, 8.0, 32.0])}
    if op == "dropout":
        return {"op": "dropout", "rows": _log(rng, 1, 8192 // wide), "cols": _log(rng, 8, 4096),
                "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "dtype": dtype,
                "x_t": rng.random() < 0.25}
    V = _log(rng, 10, 131072)
    rows = min(_log(rng, 1, 8192), 8192 * 32000 // (wide * V))
    train = rng.random() < 0.5
    return {"op": "logp", "rows": rows, "V": V, "train": train, "entropy": rng.random() < 0.5,
            "top": 0 if train else min(rng.choice([0, 1, 5, 20]), V),
            "masked": rng.choice([0.0, 0.0, 0.1]), "ignored": rng.choice([0.0, 0.25]),
            "dtype": dtype, "int32": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs


def _plain_new(shape, dtype):
    return torch.empty(*shape, dtype=dtype, device="cuda"), None


def _inputs(case: dict, seed: int, new=_plain_new) -> dict:
    """The case's inputs from the seed alone: {name: (torch tensor, the
    framework's tensor over the same memory or None)}."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = torch.float64 if case["dtype"] == "float64" else torch.float32
    it = torch.int32 if case.get("int32") else torch.int64
    out = {}

    def normal(name, *shape, scale=1.0):
        out[name] = new(shape, dt)
        t = out[name][0].normal_(generator=gen)
        return t if scale == 1.0 else t.mul_(scale)

    def tokens(n, V, zipf):
        out["t"] = new((n,), it)
        u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
        # numbered by how common they are: the k-th has a share of about 1 / k
        v = torch.exp(u * math.log(V + 1)).floor() - 1 if zipf else (u * V).floor()
        return out["t"][0].copy_(v.clamp_(0, V - 1))

    if case["op"] == "embed":
        normal("W", case["V"], case["D"], scale=0.02)
        tokens(case["N"], case["V"], case["zipf"])
        if case["train"]:
            normal("g", case["N"], case["D"])
    elif case["op"] == "dropout":
        r, c = case["rows"], case["cols"]
        normal("x", *((c, r) if case["x_t"] else (r, c)))
        normal("g", r, c)
    else:
        r, V = case["rows"], case["V"]
        z = normal("z", r, V, scale=2.5)
        t = tokens(r, V, True).long()
        if case["masked"]:  # tokens that a constraint forbids; never the given one
            hit = torch.rand(r, V, generator=gen, device="cuda") < case["masked"]
            hit.scatter_(1, t[:, None], False)
            z.masked_fill_(hit, -math.inf)
        if case["ignored"]:
            gone = torch.rand(r, generator=gen, device="cuda") < case["ignored"]
            out["t"][0].masked_fill_(gone, IGNORED)
        if case["train"]:
            normal("a", r)
            if case["entropy"]:
                normal("b", r, scale=0.1)
    return out


def prepare(case: dict, seed: int) -> dict:
    """The inputs, in the tensors of the side that computes: the framework
    works on its own ones, here made in place with the same values."""
    v = _inputs(case, seed, _own_new if own else _plain_new)
    s = {k: (b if own else a) for k, (a, b) in v.items()}
    if case["op"] == "dropout":
        s["seed"], s["offset"] = seed * 0x9E3779B97F4A7C15 % 2**64, seed % 1000
        if case["x_t"]:
            s["x"] = s["x"].T
    if own:
        for k in ("W", "x", "z"):
            if k in s and (case["op"] == "dropout" or case["train"]):
                s[k].enable_grad()
    s["case"] = case
    torch.cuda.synchronize()
    return s


# -------------------------------------------------- the framework's operators


_NT_DTYPES = {torch.float32: "float32", torch.float64: "float64", torch.int32: "int32",
              torch.int64: "int64"}
_TYPESTR = {1: ("<i4", 4), 2: ("<i8", 8), 3: ("<f4", 4), 4: ("<f8", 8)}  # by dtype code


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


def _own_new(shape, dtype):
    import nanotorch_amd as nt

    t = nt.zeros(*shape, dtype=getattr(nt, _NT_DTYPES[dtype]), device="cuda")
    nt.sync()
    return _torch(t), t


def run(s: dict):
    return (_RUN_OWN if own else _RUN_PLAIN)[s["case"]["op"]](s, s["case"])


def _own_embed(s, case):
    import nanotorch_amd as nt

    y = nt.embedding(s["W"], s["t"], case["scale"])
    if not case["train"]:
        return {"y": _torch(y)}
    return {"y": _torch(y), "dW": _torch(y.grad_fn.backward(s["g"])[0])}


def _own_dropout(s, case):
    import nanotorch_amd as nt

    y = nt.dropout(s["x"], case["p"], seed=s["seed"], offset=s["offset"])
    return {"y": _torch(y), "dx": _torch(y.grad_fn.backward(s["g"])[0])}


def _own_logp(s, case):
    import nanotorch_amd as nt

    z = s["z"]
    r = nt.token_logprobs(z, s["t"], entropy=case["entropy"], top=case["top"])
    out = {"logprob": _torch(r.logprob)}
    if case["entropy"]:
        out["entropy"] = _torch(r.entropy)
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = _torch(r.top_logprobs), _torch(r.top_tokens)
    if case["train"]:
        if case["entropy"]:
            z.zero_grad()
            (r.logprob * s["a"] + r.entropy * s["b"]).sum().backward()
            out["dz"] = _torch(z.grad)
        else:
            out["dz"] = _torch(r.logprob.grad_fn.backward(s["a"])[0])
    return out


_RUN_OWN = {"embed": _own_embed, "dropout": _own_dropout, "logp": _own_logp}


# ------------------------------------------------------------- plain forms


def _plain_embed(s, case):
    W, t = s["W"], s["t"].long()
    out = {"y": W[t] * case["scale"]}
    if case["train"]:
        dW = torch.zeros_like(W)
        dW.index_add_(0, t, s["g"])
        out["dW"] = dW * case["scale"]
    return out


def _mulhilo(m: int, b: torch.Tensor):
    """High and low words of m * b; 32-bit values held in int64."""
    low, high = b & 0xFFFF, b >> 16
    hi = (m * high + (m * low >> 16)) >> 16
    lo = (m * low + ((m * high & 0xFFFF) << 16)) & 0xFFFFFFFF
    return hi, lo


def _philox(i: torch.Tensor, offset: int, seed: int):
    """Philox4x32-10's four words for each counter (i, offset)."""
    c = [i & 0xFFFFFFFF, i >> 32, torch.full_like(i, offset & 0xFFFFFFFF),
         torch.full_like(i, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mulhilo(0xD2511F53, c[0])
        h1, l1 = _mulhilo(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack(c, 1).reshape(-1)


def _plain_dropout(s, case):
    x, g, p = s["x"], s["g"], case["p"]
    i = torch.arange((x.numel() + 3) // 4, device="cuda")
    r = _philox(i, s["offset"], s["seed"])[: x.numel()].reshape(x.shape)
    keep = r >= round(p * 2**32)
    return {"y": torch.where(keep, x * (1 / (1 - p)), 0.0),
            "dx": torch.where(keep, g * (1 / (1 - p)), 0.0)}


def _plain_logp(s, case):
    z, t, k = s["z"], s["t"].long(), case["top"]
    kept = t != IGNORED
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1)
    lse = torch.log(total)
    at = torch.where(kept, t, 0)[:, None]
    out = {"logprob": torch.where(kept, d.gather(1, at)[:, 0] - lse, 0.0)}
    if case["entropy"]:
        H = lse - (torch.where(e > 0, d, 0.0) * e).sum(1) / total
        out["entropy"] = torch.where(kept, H, 0.0)
    if k:
        value, token = torch.sort(d, dim=1, descending=True, stable=True)
        out["top_logprobs"] = torch.where(kept[:, None], value[:, :k] - lse[:, None], -math.inf)
        out["top_tokens"] = torch.where(kept[:, None], token[:, :k], -1)
    if case["train"]:
        a = torch.where(kept, s["a"], 0.0)
        p = e / total[:, None]
        dz = (p * -a[:, None]).scatter_add_(1, at, a[:, None])
        if case["entropy"]:
            b = torch.where(kept, s["b"], 0.0)
            log_p = torch.where(e > 0, d - lse[:, None], 0.0)
            dz -= p * (log_p + out["entropy"][:, None]) * b[:, None]
        out["dz"] = dz
    return out


_RUN_PLAIN = {"embed": _plain_embed, "dropout": _plain_dropout, "logp": _plain_logp}


# -------------------------------------------------------------------- work


def _distinct(case: dict) -> float:
    """How many different tokens the case has, on average."""
    N, V = case["N"], case["V"]
    if case["zipf"]:
        edge = np.log(np.arange(1, V + 2)) / math.log(V + 1)
        share = np.diff(edge)
    else:
        share = np.full(V, 1.0 / V)
    return float(np.sum(-np.expm1(N * np.log1p(-share))))


def work(case: dict) -> dict:
    item = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        token = 4 if case["int32"] else 8
        rows = _distinct(case)
        # rows that are looked up, tokens, y; then g and every row of dW
        n = token * N + item * D * (rows + N)
        if case["train"]:
            n += item * D * (N + V)
        return {"bytes": n, "flops": N * D * (2 if case["train"] else 1)}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * item * n, "flops": 2 * n}
    r, n = case["rows"], case["rows"] * case["V"] * (1 - case["ignored"])
    moved = item * n + r * (item + (4 if case["int32"] else 8))
    moved += r * (item * bool(case["entropy"]) + (item + 8) * case["top"])
    if case["train"]:
        # the logits again, every row of their gradient, the row weights
        moved += item * (n + case["rows"] * case["V"]) + r * item * (2 if case["entropy"] else 1)
    return {"bytes": moved, "flops": (10 if case["train"] else 5) * n}


# ------------------------------------------------------------------- exact


def _words(n: int, offset: int, seed: int) -> np.ndarray:
    """The first n words, in 64-bit unsigned arithmetic on the host."""
    low, u32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    x0 = np.arange(-(-n // 4), dtype=np.uint64)
    x1 = x0 >> u32
    x0 = x0 & low
    x2 = np.full_like(x0, offset & 0xFFFFFFFF)
    x3 = np.full_like(x0, offset >> 32)
    for r in range(10):
        k0 = np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        x0, x1, x2, x3 = (b >> u32) ^ x1 ^ k0, b & low, (a >> u32) ^ x3 ^ k1, a & low
    return np.stack([x0, x1, x2, x3], axis=1).reshape(-1)[:n]


def exact(case: dict, seed: int):
    v = {k: (t.double() if t.is_floating_point() else t.long())
         for k, (t, _) in _inputs(case, seed).items()}
    if case["op"] == "embed":
        out = {"y": torch.index_select(v["W"], 0, v["t"]).mul_(case["scale"])}
        if case["train"]:
            dW = torch.zeros(case["V"], case["D"], dtype=torch.float64, device="cuda")
            order = torch.argsort(v["t"], stable=True)
            out["dW"] = dW.index_add_(0, v["t"][order], v["g"][order]).mul_(case["scale"])
        return out
    if case["op"] == "dropout":
        shape = (case["rows"], case["cols"])
        key, offset = seed * 0x9E3779B97F4A7C15 % 2**64, seed % 1000
        kept = torch.from_numpy(
            _words(shape[0] * shape[1], offset, key) >= np.uint64(round(case["p"] * 2**32)))
        kept = kept.to("cuda").reshape(shape).double() / (1 - case["p"])
        x = v["x"].T if case["x_t"] else v["x"]
        return {"y": x * kept, "dx": v["g"] * kept}
    z, t = v["z"], v["t"]
    live = (t != IGNORED).double()
    at = t.clamp(min=0)[:, None]
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    plogp = (p * log_p.clamp(min=-1e300)).sum(1)
    out = {"logprob": log_p.gather(1, at)[:, 0].masked_fill(live == 0, 0.0)}
    if case["entropy"]:
        out["entropy"] = -plogp * live
    if case["top"]:
        value = torch.topk(log_p, case["top"], dim=1).values
        out["top_logprobs"] = value.masked_fill(live[:, None] == 0, -math.inf)
        out["top_tokens"] = None
    if case["train"]:
        a = v["a"] * live
        dz = -a[:, None] * p
        if case["entropy"]:
            part = log_p.clamp(min=-1e300).sub_(plogp[:, None])
            dz -= (v["b"] * live)[:, None] * p * part
        dz[torch.arange(case["rows"], device="cuda"), at[:, 0]] += a
        out["dz"] = dz
    return out
