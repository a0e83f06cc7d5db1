"""The training operators of ``hawk.stages`` as they are timed and checked:
what one pass reads and returns, in a plain torch form and through
``hawk.run``.

A case is a dict of plain values whose ``"kind"`` names the operator:

* ``recurrence``  a gated linear recurrence along the time axis, or its
  gradient (``"pass": "vjp"``): dense ``(S, T, C)`` planes, channel- or
  time-contiguous, or packed sequences ``(N, C)`` cut by offsets;
* ``logp``        the log-probability of each row's target, or its gradient;
* ``policy``      the clipped policy loss with a KL term: the loss
  (``"forward"``), loss and gradient in one pass (``"fused"``), the gradient
  from a saved forward (``"vjp"``);
* ``preference``  the loss of pairs of answers, alone or with its gradient
  (``"train"``);
* ``dropout``     dropout from a counter-based generator, with a residual, or
  its gradient.

The plain form computes in float32 and rounds once, to the output's type.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# -- the cases -------------------------------------------------------------------------

def listed():
    return [
        # one token of 64 running sequences: the serving form, all latency
        dict(name="recurrence_step", kind="recurrence", op="forward", S=64, T=1, C=2048, dtype="bf16", gate="sigmoid",
             reverse=False, time_major=False, packed=False, state=True),
        # sequences of ragged lengths packed into one axis, an odd channel count
        dict(name="recurrence_packed", kind="recurrence", op="forward", S=37, T=65793, C=1001, dtype="bf16",
             gate="value", reverse=False, time_major=False, packed=True, state=True),
        # the training step's gradient at a model's width
        dict(name="recurrence_vjp", kind="recurrence", op="vjp", S=16, T=4096, C=2048, dtype="bf16", gate="sigmoid",
             reverse=False, time_major=False, packed=False, state=False),
        # advantages of rollouts: discounted residuals summed backwards in time, done flags in the gate
        dict(name="recurrence_advantages", kind="recurrence", op="forward", S=16384, T=257, C=1, dtype="f32",
             gate="value", reverse=True, time_major=True, packed=False, state=False),
        # the old policy's and the reference's log-probabilities, an odd vocabulary
        dict(name="logp_odd", kind="logp", op="forward", N=4096, V=50001, dtype="bf16", scale=1.0),
        # the gradient of a model trained in float32
        dict(name="logp_vjp", kind="logp", op="vjp", N=1024, V=32768, dtype="f32", scale=0.5),
        # a policy's update: loss and gradient of every token of a batch, a large vocabulary
        dict(name="policy_large", kind="policy", op="fused", N=8192, V=131072, dtype="bf16", scale=1.0, kl=0.05),
        # a small agent's update: few rows, some tens of actions
        dict(name="policy_small", kind="policy", op="fused", N=200, V=48, dtype="f32", scale=1.0, kl=0.0),
        # pairs of answers after a prompt: loss and gradient
        dict(name="preference_train", kind="preference", op="train", P=8, L=384, V=32768, dtype="bf16", scale=1.0),
        # the same loss held out, of few short answers: few rows, a long vocabulary axis
        dict(name="preference_eval", kind="preference", op="forward", P=2, L=13, V=100003, dtype="f16", scale=1.0),
        # the residual branch of a layer
        dict(name="dropout_residual", kind="dropout", op="forward", rows=16384, cols=4096, dtype="bf16", p=0.1,
             residual=True),
        # its gradient, an odd width in float32
        dict(name="dropout_vjp", kind="dropout", op="vjp", rows=3001, cols=777, dtype="f32", p=0.25, residual=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "logp", "policy", "preference", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "recurrence":
        packed = rng.random() < 0.3
        T = _log(rng, 1, 65536 if packed else 16384)
        S, C = _log(rng, 1, 512), _log(rng, 1, 8192)
        most = 1 << 26
        if packed:
            S = min(S, max(1, T // 2))
            C = max(1, min(C, most // T))
        else:
            C = max(1, min(C, most // T))
            S = max(1, min(S, most // (T * C)))
        return dict(kind=kind, op=rng.choice(["forward", "vjp"]), S=S, T=T, C=C, dtype=dtype,
                    gate=rng.choice(["value", "sigmoid"]), reverse=rng.random() < 0.5,
                    time_major=not packed and rng.random() < 0.3, packed=packed, state=rng.random() < 0.5)
    if kind == "dropout":
        cols = _log(rng, 1, 16384)
        return dict(kind=kind, op=rng.choice(["forward", "vjp"]), rows=_log(rng, 1, (1 << 26) // cols), cols=cols,
                    dtype=dtype, p=rng.choice([0.05, 0.1, 0.25, 0.5]), residual=rng.random() < 0.5)
    V = _log(rng, 16, 131072)
    rows = (1 << 28) // V
    scale = rng.choice([1.0, 0.5, 1.25])
    if kind == "preference":
        L = _log(rng, 4, 1024)
        return dict(kind=kind, op=rng.choice(["forward", "train"]), P=max(1, min(_log(rng, 1, 32), rows // (2 * L))),
                    L=L, V=V, dtype=dtype, scale=scale)
    N = _log(rng, 1, min(16384, rows))
    if kind == "logp":
        return dict(kind=kind, op=rng.choice(["forward", "vjp"]), N=N, V=V, dtype=dtype, scale=scale)
    return dict(kind=kind, op=rng.choice(["forward", "fused", "vjp"]), N=N, V=V, dtype=dtype, scale=scale,
                kl=rng.choice([0.0, 0.05]))


def work(case):
    e = SIZE[case["dtype"]]
    kind = case["kind"]
    if kind == "recurrence":
        S, T, C = case["S"], case["T"], case["C"]
        n = T * C if case["packed"] else S * T * C
        sig = case["gate"] == "sigmoid"
        state = 4 * S * C * ((2 if case["op"] == "forward" else 3) if case["state"] else 0)
        if case["op"] == "forward":
            return {"bytes": 3 * e * n + state, "flops": (8 if sig else 2) * n}
        return {"bytes": (6 if sig else 5) * e * n + state, "flops": (12 if sig else 4) * n}
    if kind == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": e * n * (3 if case["residual"] and case["op"] == "forward" else 2), "flops": 2 * n}
    rows = case["N"] if "N" in case else 2 * case["P"] * case["L"]
    n = rows * case["V"]
    if case["op"] == "forward":
        return {"bytes": e * n, "flops": 4 * n}
    if case["op"] == "train":                # the gradient needs both answers' sums first
        return {"bytes": 3 * e * n, "flops": 8 * n}
    return {"bytes": 2 * e * n, "flops": (8 if case["op"] == "fused" else 4) * n}


# -- the inputs ------------------------------------------------------------------------

def _cuts(g, pieces, total):
    """``pieces`` ragged lengths that fill ``total``, one of them empty where there are three or more."""
    if pieces == 1:
        cut = torch.empty(0, dtype=torch.int64)
    else:
        cut = torch.sort(torch.randint(0, total + 1, (pieces - 1,), generator=g))[0]
        if pieces >= 3:
            cut[1] = cut[0]
    return torch.cat([torch.zeros(1, dtype=torch.int64), cut, torch.full((1,), total, dtype=torch.int64)])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    s = dict(case=case)
    if kind == "recurrence":
        S, T, C = case["S"], case["T"], case["C"]
        shape = (T, C) if case["packed"] else (S, T, C)

        def plane(x):
            return x.to(dtype).transpose(1, 2).contiguous().transpose(1, 2) if case["time_major"] else x.to(dtype)
        if case["gate"] == "sigmoid":
            gate = normal(*shape) + 2.0
        elif case["reverse"]:
            gate = 0.99 * 0.95 * (torch.rand(shape, generator=g, device=DEVICE) > 0.005)
        else:
            gate = torch.sigmoid(normal(*shape) + 2.0)
        s["gate"], s["x"] = plane(gate), plane(normal(*shape))
        if case["packed"]:
            s["offsets"] = _cuts(host, S, T).to(DEVICE)
        if case["state"]:
            s["h0"] = normal(S, C)
        if case["op"] == "forward":
            s["h"] = torch.empty_like(s["x"])
            if case["state"]:
                s["last"] = torch.empty_like(s["h0"])
        else:
            s["h"] = torch.empty_like(s["x"])
            s["h"].copy_(_recurrence(s)["h"])            # the forward's saved output
            s["bar_h"] = plane(normal(*shape))
            s["bar_gate"], s["bar_x"] = torch.empty_like(s["gate"]), torch.empty_like(s["x"])
            if case["state"]:
                s["bar_last"], s["bar_h0"] = normal(S, C), torch.empty_like(s["h0"])
        return s
    if kind == "dropout":
        shape = (case["rows"], case["cols"])
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ seed, seed % 1000
        s["x"] = normal(*shape).to(dtype)                # the vjp's bar_y
        s["y"] = torch.empty_like(s["x"])
        if case["residual"] and case["op"] == "forward":
            s["residual"] = normal(*shape).to(dtype)
        return s

    V = case["V"]
    if kind == "preference":
        # 2P answers of ragged lengths about L, a quarter of each a prompt that is left out
        P, L = case["P"], case["L"]
        lengths = torch.randint(L // 2, L + 1, (2 * P,), generator=host)
        lengths += (2 * P * L - int(lengths.sum())) // (2 * P)
        lengths[-1] += 2 * P * L - int(lengths.sum())
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(lengths, 0)])
        N = 2 * P * L
    else:
        N = case["N"]
    logits = normal(N, V).mul_(2.0)
    target = torch.randint(0, V, (N,), generator=g, device=DEVICE)
    logits[torch.arange(N, device=DEVICE), target] += 5.0
    s["logits"] = logits.to(dtype)
    del logits
    if kind == "preference":
        at = torch.arange(N)
        seq = torch.bucketize(at, offsets[1:], right=True)
        prompt = at - offsets[seq] < lengths[seq] // 4
        target[prompt.to(DEVICE)] = -1
        s["offsets"] = offsets.to(DEVICE)
    elif N >= 8:
        target[:: max(2, N // 8)] = -1                   # padding: rows left out
    s["target"] = target
    saved = _logp(s)
    if kind == "logp":
        if case["op"] == "forward":
            s["logp"], s["lse"] = torch.empty(N, device=DEVICE), torch.empty(N, device=DEVICE)
        else:
            s["lse"], s["bar_logp"] = saved["lse"], normal(N)
            s["bar_logits"] = torch.empty_like(s["logits"])
        return s
    s["ref_logp"] = saved["logp"] + 0.1 * normal(N)
    if kind == "policy":
        s["old_logp"] = saved["logp"] + 0.15 * normal(N)
        s["advantage"] = normal(N) + 0.25
        s["weight"] = (target >= 0).float() / (target >= 0).sum().clamp(min=1)
        if not case["kl"]:
            del s["ref_logp"]
    s["loss"] = torch.empty(1, device=DEVICE)
    s["logp"], s["lse"] = torch.empty(N, device=DEVICE), torch.empty(N, device=DEVICE)
    if case["op"] != "forward":
        s["bar_logits"] = torch.empty_like(s["logits"])
    if case["op"] == "vjp":
        s["logp"], s["lse"] = saved["logp"], saved["lse"]
    if kind == "preference":
        s["margin"] = torch.empty(case["P"], device=DEVICE)
    return s


# -- the plain forms -------------------------------------------------------------------

CLIP = (0.2, 0.28)
BETA, SMOOTHING = 0.1, 0.05


def _scan(a, b, dim):
    """``h_t = a_t h_{t-1} + b_t`` along ``dim``: each doubling step joins every element with the run before it."""
    n, T = 1, a.shape[dim]
    while n < T:
        b = torch.cat([b.narrow(dim, 0, n), b.narrow(dim, n, T - n) + a.narrow(dim, n, T - n) * b.narrow(dim, 0, T - n)],
                      dim)
        a = torch.cat([a.narrow(dim, 0, n), a.narrow(dim, n, T - n) * a.narrow(dim, 0, T - n)], dim)
        n *= 2
    return b


def _ends(s, reverse):
    """Packed sequences that are not empty, and each one's first row in the scan's direction."""
    offsets = s["offsets"]
    full = torch.nonzero(offsets[1:] > offsets[:-1])[:, 0]
    return full, (offsets[1:][full] - 1 if reverse else offsets[:-1][full])


def _gates(s):
    gate, x = s["gate"].float(), s["x"].float()
    if s["case"]["gate"] == "value":
        return gate, x
    a = 1.0 / (1.0 + torch.exp(-gate))
    return a, (1.0 - a) * x


def _run_scan(s, a, b, init, reverse):
    """The recurrence from ``init`` (or zero), in float32, along the case's time axis."""
    if s["case"]["packed"]:
        full, first = _ends(s, reverse)
        a, b = a.clone(), b.clone()
        if init is not None:
            b[first] += a[first] * init[full]
        a[first] = 0.0
        dim = 0
    else:
        dim = 1
        if init is not None:
            b = b.clone()
            b[:, -1 if reverse else 0] += a[:, -1 if reverse else 0] * init
    if reverse:
        return _scan(a.flip(dim), b.flip(dim), dim).flip(dim)
    return _scan(a, b, dim)


def _recurrence(s):
    case = s["case"]
    a, b = _gates(s)
    h = _run_scan(s, a, b, s.get("h0"), case["reverse"])
    out = {"h": h.to(s["x"].dtype)}
    if case["state"]:
        if case["packed"]:
            full, end = _ends(s, not case["reverse"])
            out["last"] = s["h0"].clone()
            out["last"][full] = h[end]
        else:
            out["last"] = h[:, 0 if case["reverse"] else -1].clone()
    return out


def _recurrence_vjp(s):
    case = s["case"]
    a, _ = _gates(s)
    x, h, bar_h = s["x"].float(), s["h"].float(), s["bar_h"].float()
    back = not case["reverse"]
    C = _run_scan(s, a, a * bar_h, s.get("bar_last"), back)      # C_t = a_t (bar_h_t + C_{t+1})
    dim = 0 if case["packed"] else 1
    T = case["T"]
    prior, after = torch.zeros_like(h), torch.zeros_like(h)      # h_{t-1} and C_{t+1} in the primal's direction
    if case["reverse"]:
        prior.narrow(dim, 0, T - 1).copy_(h.narrow(dim, 1, T - 1))
        after.narrow(dim, 1, T - 1).copy_(C.narrow(dim, 0, T - 1))
    else:
        prior.narrow(dim, 1, T - 1).copy_(h.narrow(dim, 0, T - 1))
        after.narrow(dim, 0, T - 1).copy_(C.narrow(dim, 1, T - 1))
    zero = torch.zeros((case["S"], case["C"]), device=h.device)
    h0, bar_last = s.get("h0", zero), s.get("bar_last", zero)
    out = {}
    if case["packed"]:
        full, first = _ends(s, case["reverse"])
        prior[first] = h0[full]
        _, end = _ends(s, back)
        after[end] = bar_last[full]
        if case["state"]:
            out["bar_h0"] = bar_last.clone()
            out["bar_h0"][full] = C[first]
    else:
        prior[:, -1 if case["reverse"] else 0] = h0
        after[:, 0 if case["reverse"] else -1] = bar_last
        if case["state"]:
            out["bar_h0"] = C[:, -1 if case["reverse"] else 0].clone()
    G = bar_h + after
    if case["gate"] == "value":
        bar_gate, bar_x = G * prior, G
    else:
        bar_gate, bar_x = G * (prior - x) * a * (1.0 - a), (1.0 - a) * G
    out["bar_gate"], out["bar_x"] = bar_gate.to(s["x"].dtype), bar_x.to(s["x"].dtype)
    return out


def _logp(s):
    x = s["logits"].float() * s["case"]["scale"]
    top = x.amax(1)
    lse = top + torch.log(torch.exp(x - top[:, None]).sum(1))
    target = s["target"]
    logp = x.gather(1, target.clamp(min=0)[:, None])[:, 0] - lse
    kept = target >= 0
    return {"logp": torch.where(kept, logp, 0.0), "lse": torch.where(kept, lse, 0.0)}


def _logits_gradient(s, lse, bar_logp):
    """``scale * bar_logp * (1[v = target] - p)``, zero in rows left out."""
    kept = s["target"] >= 0
    c = torch.where(kept, bar_logp, 0.0) * s["case"]["scale"]
    p = torch.exp(s["logits"].float() * s["case"]["scale"] - lse[:, None])
    grad = torch.where(kept[:, None], -c[:, None] * p, 0.0)
    grad.scatter_add_(1, s["target"].clamp(min=0)[:, None], c[:, None])
    return grad.to(s["logits"].dtype)


def _policy_terms(s, logp):
    """Each row's loss and its derivative by the row's log-probability."""
    kl, A = s["case"]["kl"], s["advantage"]
    r = torch.exp(logp - s["old_logp"])
    plain, clipped = r * A, torch.clamp(r, 1.0 - CLIP[0], 1.0 + CLIP[1]) * A
    loss = -torch.minimum(plain, clipped)
    slope = torch.where(plain <= clipped, -plain, 0.0)
    if kl:
        d = s["ref_logp"] - logp
        loss = loss + kl * (torch.exp(d) - d - 1.0)
        slope = slope + kl * (1.0 - torch.exp(d))
    kept = s["target"] >= 0
    return torch.where(kept, loss, 0.0), torch.where(kept, slope, 0.0)


def _policy(s):
    op = s["case"]["op"]
    saved = {"logp": s["logp"], "lse": s["lse"]} if op == "vjp" else _logp(s)
    loss, slope = _policy_terms(s, saved["logp"])
    out = {} if op == "vjp" else {"loss": (loss * s["weight"]).sum().reshape(1), **saved}
    if op != "forward":
        out["bar_logits"] = _logits_gradient(s, saved["lse"], slope * s["weight"])
    return out


def _preference(s):
    saved = _logp(s)
    N, P = s["target"].numel(), s["case"]["P"]
    seq = torch.bucketize(torch.arange(N, device=DEVICE), s["offsets"][1:], right=True)
    ratio = torch.where(s["target"] >= 0, saved["logp"] - s["ref_logp"], 0.0)
    sums = torch.zeros(2 * P, device=DEVICE).index_add_(0, seq, ratio).view(P, 2)
    margin = sums[:, 0] - sums[:, 1]
    z = BETA * margin
    soft = torch.log1p(torch.exp(-z.abs())) + torch.clamp(-z, min=0.0)       # -log sigma(z)
    loss = ((1.0 - SMOOTHING) * soft + SMOOTHING * (soft + z)).mean().reshape(1)
    out = {"loss": loss, "margin": margin, **saved}
    if s["case"]["op"] == "train":
        slope = SMOOTHING - 1.0 / (1.0 + torch.exp(z))                       # dL/dz
        bar = (BETA / P) * torch.stack([slope, -slope], 1).reshape(-1)[seq]
        out["bar_logits"] = _logits_gradient(s, saved["lse"], bar)
    return out


def _philox(counter, key):
    """Philox4x32-10 of int64 words below 2^32 (Salmon, Moraes, Dror and Shaw, 2011)."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(10):
        l0, h0 = _product(c0, 0xD2511F53)
        l1, h1 = _product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _product(x, m):
    """The low and the high word of a 32 x 32-bit product, in int64 arithmetic."""
    low, high = (x & 0xFFFF) * m, (x >> 16) * m
    return (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF, (high + (low >> 16)) >> 16


def _threshold(p):
    return int(round(p * 65536))


def _dropout(s):
    case, x = s["case"], s["x"]
    n = x.numel()
    group = torch.arange((n + 7) // 8, device=DEVICE)
    zero = torch.zeros_like(group)
    words = _philox((group & 0xFFFFFFFF, group >> 32, zero + (s["offset"] & 0xFFFFFFFF), zero + (s["offset"] >> 32)),
                    (s["seed"] & 0xFFFFFFFF, s["seed"] >> 32))
    words = torch.stack(words, 1)
    u = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n].view(x.shape)
    cut = _threshold(case["p"])
    y = torch.where(u >= cut, x.float() * (65536.0 / (65536 - cut)), 0.0)
    if "residual" in s:
        y = y + s["residual"].float()
    return {"bar_x" if case["op"] == "vjp" else "y": y.to(x.dtype)}


# -- one pass --------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _stage(kind, *options):
    """The stage a program makes once."""
    import hawk_amd as hawk
    return getattr(hawk.stages, kind)(**dict(options))


def _given(s, *names):
    return {n: s[n] for n in names if n in s}


def run(s):
    case = s["case"]
    kind, op = case["kind"], case["op"]
    if not own:
        if kind == "recurrence":
            return _recurrence_vjp(s) if op == "vjp" else _recurrence(s)
        if kind == "logp":
            return {"bar_logits": _logits_gradient(s, s["lse"], s["bar_logp"])} if op == "vjp" else _logp(s)
        return {"policy": _policy, "preference": _preference, "dropout": _dropout}[kind](s)

    import hawk_amd as hawk
    if kind == "recurrence":
        stage = _stage("recurrence", ("gate", case["gate"]), ("reverse", case["reverse"]))
        if op == "forward":
            hawk.run(stage, **_given(s, "gate", "x", "h", "h0", "last", "offsets"))
            return _given(s, "h", "last")
        hawk.run(stage.vjp, **_given(s, "gate", "x", "h", "h0", "offsets", "bar_h", "bar_last", "bar_gate", "bar_x",
                                     "bar_h0"))
        return _given(s, "bar_gate", "bar_x", "bar_h0")
    if kind == "logp":
        stage = _stage("token_logp", ("scale", case["scale"]))
        if op == "forward":
            hawk.run(stage, **_given(s, "logits", "target", "logp", "lse"))
            return _given(s, "logp", "lse")
        hawk.run(stage.vjp, **_given(s, "logits", "target", "lse", "bar_logp", "bar_logits"))
        return _given(s, "bar_logits")
    if kind == "policy":
        stage = _stage("policy_loss", ("clip", CLIP), ("kl", case["kl"]), ("scale", case["scale"]))
        planes = _given(s, "logits", "target", "old_logp", "advantage", "ref_logp", "weight", "logp", "lse")
        if op == "vjp":
            hawk.run(stage.vjp, bar_logits=s["bar_logits"], **planes)
            return _given(s, "bar_logits")
        hawk.run(stage, loss=s["loss"], **planes, **_given(s, "bar_logits"))
        return _given(s, "loss", "logp", "lse", "bar_logits")
    if kind == "preference":
        stage = _stage("preference_loss", ("beta", BETA), ("smoothing", SMOOTHING), ("scale", case["scale"]))
        hawk.run(stage, **_given(s, "logits", "target", "offsets", "ref_logp", "loss", "margin", "logp", "lse"))
        if op == "train":
            hawk.run(stage.vjp, **_given(s, "logits", "target", "offsets", "margin", "lse", "bar_logits"))
        return _given(s, "loss", "margin", "logp", "lse", "bar_logits")
    stage = _stage("dropout", ("p", case["p"]))
    if op == "vjp":
        hawk.run(stage.vjp, bar_y=s["x"], bar_x=s["y"], seed=s["seed"], offset=s["offset"])
        return {"bar_x": s["y"]}
    hawk.run(stage, **_given(s, "x", "residual", "y", "seed", "offset"))
    return _given(s, "y")


# -- from the definitions, in 64 bits --------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "recurrence":
        return _exact_recurrence(s)
    if kind == "dropout":
        return _exact_dropout(s)
    return _exact_rows(s)


def _exact_recurrence(s):
    """Step by step along the time axis, every sequence of a packed axis in turn."""
    case = s["case"]
    if case["packed"] and case["T"] > 1 << 18:
        return None
    wide = {n: v.double() for n, v in s.items() if n in ("gate", "x", "h", "bar_h", "h0", "bar_last")}
    if case["packed"]:
        cuts = s["offsets"].tolist()
        spans = [(k, range(cuts[k], cuts[k + 1])) for k in range(case["S"])]
        at = {n: list(v.unbind(0)) for n, v in wide.items() if n not in ("h0", "bar_last")}
    else:
        spans = [(slice(None), range(case["T"]))]
        at = {n: list(v.unbind(1)) for n, v in wide.items() if n not in ("h0", "bar_last")}
    nothing = torch.zeros((case["S"], case["C"]), dtype=torch.float64, device=DEVICE)
    a = [torch.special.expit(z) for z in at["gate"]] if case["gate"] == "sigmoid" else at["gate"]
    one, two = [None] * case["T"], [None] * case["T"]
    state = nothing.clone()
    for k, rows in spans:
        order = list(reversed(rows)) if case["reverse"] else list(rows)
        h0 = wide["h0"][k] if case["state"] else nothing[k]
        if case["op"] == "forward":
            h = h0
            for t in order:
                h = a[t] * h + (at["x"][t] * (1.0 - a[t]) if case["gate"] == "sigmoid" else at["x"][t])
                one[t] = h
            state[k] = h
            continue
        carry = wide["bar_last"][k] if case["state"] else nothing[k]
        for i in range(len(order) - 1, -1, -1):
            t = order[i]
            prior = at["h"][order[i - 1]] if i else h0
            G = at["bar_h"][t] + carry
            if case["gate"] == "sigmoid":
                one[t], two[t] = G * (prior - at["x"][t]) * a[t] * (1.0 - a[t]), (1.0 - a[t]) * G
            else:
                one[t], two[t] = G * prior, G
            carry = a[t] * G
        state[k] = carry
    dim = 0 if case["packed"] else 1
    if case["op"] == "forward":
        out = {"h": torch.stack(one, dim)}
        if case["state"]:
            out["last"] = state
        return out
    out = {"bar_gate": torch.stack(one, dim), "bar_x": torch.stack(two, dim)}
    if case["state"]:
        out["bar_h0"] = state
    return out


def _exact_rows(s):
    """The rows' losses and gradients, a block of rows at a time."""
    case, target = s["case"], s["target"]
    kind, op = case["kind"], case["op"]
    N, V = s["logits"].shape
    kept = target >= 0
    at = target.clamp(min=0)
    block = max(1, (1 << 27) // V)
    logp = torch.zeros(N, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros_like(logp)
    for r in range(0, N, block):
        w = slice(r, r + block)
        x = s["logits"][w].double() * case["scale"]
        lse[w] = torch.logsumexp(x, 1)
        logp[w] = x[torch.arange(x.shape[0], device=DEVICE), at[w]] - lse[w]
    lse, logp = lse * kept, logp * kept
    if op == "vjp":
        lse = s["lse"].double()                           # the saved forward is an input
        if kind == "policy":
            logp = s["logp"].double()
    out = {"logp": logp, "lse": lse}
    bar = None
    if kind == "logp":
        if op == "vjp":
            out, bar = {}, s["bar_logp"].double()
    elif kind == "policy":
        A, low, high = s["advantage"].double(), 1.0 - CLIP[0], 1.0 + CLIP[1]
        r = torch.exp(logp - s["old_logp"].double())
        one, two = r * A, r.clamp(low, high) * A
        loss, bar = -torch.where(one <= two, one, two), -one * (one <= two)
        if case["kl"]:
            d = s["ref_logp"].double() - logp
            loss, bar = loss + case["kl"] * (torch.expm1(d) - d), bar - case["kl"] * torch.expm1(d)
        weight = s["weight"].double() * kept
        out["loss"], bar = (loss * weight).sum().reshape(1), bar * weight
        if op == "vjp":
            out = {}
    else:
        P, cuts = case["P"], s["offsets"].tolist()
        ratio = (logp - s["ref_logp"].double()) * kept
        sums = torch.stack([ratio[cuts[k]:cuts[k + 1]].sum() for k in range(2 * P)])
        margin = sums[0::2] - sums[1::2]
        z = BETA * margin
        logsigmoid = torch.nn.functional.logsigmoid
        out["margin"] = margin
        out["loss"] = -((1.0 - SMOOTHING) * logsigmoid(z) + SMOOTHING * logsigmoid(-z)).mean().reshape(1)
        slope = BETA / P * (SMOOTHING * torch.sigmoid(z) - (1.0 - SMOOTHING) * torch.sigmoid(-z))
        bar = torch.cat([(slope if k % 2 == 0 else -slope)[k // 2].expand(cuts[k + 1] - cuts[k])
                         for k in range(2 * P)])
    if op != "forward":
        bar = bar * kept * case["scale"]
        grad = torch.empty((N, V), dtype=torch.float64, device=DEVICE)
        for r in range(0, N, block):
            w = slice(r, r + block)
            here = -bar[w, None] * torch.exp(s["logits"][w].double() * case["scale"] - lse[w, None])
            here[torch.arange(here.shape[0], device=DEVICE), at[w]] += bar[w]
            grad[w] = torch.where(kept[w, None], here, 0.0)
        out["bar_logits"] = grad
    return out


def _exact_dropout(s):
    """The generator in numpy's unsigned words."""
    case, n = s["case"], s["x"].numel()
    if n > 1 << 26:
        return None
    word, low = np.uint64, np.uint64(0xFFFFFFFF)
    shift = word(32)
    i = np.arange((n + 7) // 8, dtype=word)
    c = [i & low, i >> shift, np.full_like(i, s["offset"] & 0xFFFFFFFF), np.full_like(i, s["offset"] >> 32)]
    k = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for _ in range(10):
        p, q = c[0] * word(0xD2511F53), c[2] * word(0xCD9E8D57)
        c = [(q >> shift) ^ c[1] ^ word(k[0]), q & low, (p >> shift) ^ c[3] ^ word(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    u = np.empty((i.size, 8), dtype=np.uint16)
    for j in range(4):
        u[:, 2 * j] = c[j] & word(0xFFFF)
        u[:, 2 * j + 1] = c[j] >> word(16)
    cut = _threshold(case["p"])
    keep = torch.from_numpy(u.reshape(-1)[:n] >= cut).to(DEVICE).view(s["x"].shape)
    y = torch.where(keep, s["x"].double() * (65536.0 / (65536 - cut)), 0.0)
    if "residual" in s:
        y = y + s["residual"].double()
    return {"bar_x" if case["op"] == "vjp" else "y": y}
