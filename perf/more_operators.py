"""The stages of a policy with a matrix state (linear attention, layer norm, and
sampling its actions) as they are timed and checked: what one pass reads and
returns, in a plain torch form and through ``hawk.run``.

A case is a dict of plain values whose ``"kind"`` names the operator:

* ``linear``  linear attention with a decay for each head, or its gradient
  (``"op": "vjp"``): dense ``(S, T, H, D)`` planes, tokens or heads outermost, or
  packed sequences ``(N, H, D)`` cut by offsets;
* ``norm``    layer norm, or its gradient with those of the weight and the bias;
* ``sample``  a token drawn from each row of logits by a given random number, with
  temperature, top-k, top-p and min-p, for the call or for each row.

The plain form computes in float32, sampling in float64 (which token a number
falls to is decided at borders between sums), and rounds once, to the output's
type.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5


# -- the cases -------------------------------------------------------------------------

def listed():
    return [
        # one token of 64 running sequences: the serving form, the states' traffic
        dict(name="linear_step", kind="linear", op="forward", S=64, T=1, H=16, K=128, V=128, dtype="bf16", heads=False,
             packed=False, state=True),
        # one long prompt: few heads for the card, so the time axis has to be cut
        dict(name="linear_prompt", kind="linear", op="forward", S=1, T=32768, H=16, K=128, V=128, dtype="bf16",
             heads=False, packed=False, state=True),
        # prompts of ragged lengths packed into one axis, odd head sizes
        dict(name="linear_packed", kind="linear", op="forward", S=23, T=20011, H=5, K=72, V=100, dtype="f16", heads=False,
             packed=True, state=True),
        # the training step's gradient at a model's width
        dict(name="linear_vjp", kind="linear", op="vjp", S=8, T=4096, H=16, K=128, V=128, dtype="bf16", heads=False,
             packed=False, state=False),
        # a small policy trained in float32 over segments of episodes, heads outermost
        dict(name="linear_float", kind="linear", op="vjp", S=4, T=513, H=4, K=64, V=48, dtype="f32", heads=True,
             packed=False, state=True),
        # the norm before a layer
        dict(name="norm_forward", kind="norm", op="forward", rows=16384, cols=4096, dtype="bf16", weight="bf16"),
        # its gradient, weights held in float32
        dict(name="norm_vjp", kind="norm", op="vjp", rows=16384, cols=2048, dtype="bf16", weight="f32"),
        # a small model's gradient, an odd width in float32
        dict(name="norm_odd", kind="norm", op="vjp", rows=3001, cols=777, dtype="f32", weight="f32"),
        # a serving step: nucleus sampling of some tens of sequences over a large vocabulary
        dict(name="sample_serve", kind="sample", N=64, V=131072, dtype="bf16", temperature=0.8, top_k=0, top_p=0.95,
             min_p=0.0, masked=False, by_row=False),
        # actions of a rollout: the whole distribution, as the policy loss takes it
        dict(name="sample_rollout", kind="sample", N=4096, V=50001, dtype="f16", temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, masked=False, by_row=False),
        # a small agent's actions: some tens to choose from
        dict(name="sample_small", kind="sample", N=200, V=48, dtype="f32", temperature=1.0, top_k=8, top_p=1.0,
             min_p=0.05, masked=False, by_row=False),
        # requests with settings of their own, half of the vocabulary barred
        dict(name="sample_mixed", kind="sample", N=512, V=32768, dtype="f32", temperature=0.7, top_k=50, top_p=0.9,
             min_p=0.02, masked=True, by_row=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = (1 << 27) // SIZE[dtype]                          # the bytes of the largest listed plane
    if kind == "linear":
        packed = rng.random() < 0.3
        K, V = _log(rng, 8, 256), _log(rng, 8, 256)
        wide = max(K, V)
        T = _log(rng, 1, 32768)
        H = max(1, min(_log(rng, 1, 32), most // (wide * T)))
        if packed:
            S = max(1, min(_log(rng, 1, 64), T // 2))
        else:
            S = max(1, min(_log(rng, 1, 256), most // (wide * T * H), (1 << 25) // (H * K * V)))
        return dict(kind=kind, op=rng.choice(["forward", "forward", "vjp"]), S=S, T=T, H=H, K=K, V=V, dtype=dtype,
                    heads=not packed and rng.random() < 0.3, packed=packed, state=rng.random() < 0.5)
    if kind == "norm":
        cols = _log(rng, 8, 32768)
        return dict(kind=kind, op=rng.choice(["forward", "vjp"]), rows=_log(rng, 1, most // cols), cols=cols, dtype=dtype,
                    weight=rng.choice([dtype, "f32"]))
    V = _log(rng, 16, 200000)
    N = _log(rng, 1, min(8192, most // V))
    return dict(kind=kind, N=N, V=V, dtype=dtype, temperature=rng.choice([0.6, 0.8, 1.0, 1.3]),
                top_k=rng.choice([0, 0, _log(rng, 1, 2000)]), top_p=rng.choice([1.0, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.05]), masked=rng.random() < 0.3, by_row=rng.random() < 0.3)


def work(case):
    e = SIZE[case["dtype"]]
    kind = case["kind"]
    if kind == "linear":
        S, T, H, K, V = (case[n] for n in "STHKV")
        n = (T if case["packed"] else S * T) * H
        states = 4 * S * H * K * V if case["state"] else 0
        if case["op"] == "forward":                          # token by token: the update and the read of the state
            return {"bytes": e * n * 2 * (K + V) + 2 * states, "flops": 4 * n * K * V}
        return {"bytes": e * n * (4 * K + 3 * V) + 3 * states, "flops": 10 * n * K * V}
    if kind == "norm":
        n = case["rows"] * case["cols"]
        weights = SIZE[case["weight"]] * case["cols"]
        if case["op"] == "forward":
            return {"bytes": 2 * e * n + 8 * case["rows"] + 2 * weights, "flops": 8 * n}
        return {"bytes": 3 * e * n + 8 * case["rows"] + 3 * weights, "flops": 13 * n}
    n = case["N"] * case["V"]
    return {"bytes": e * n + 16 * case["N"], "flops": 6 * n}


# -- the inputs ------------------------------------------------------------------------

def _cuts(g, pieces, total):
    """``pieces`` ragged lengths that fill ``total``, one of them empty where there are three or more."""
    cut = torch.sort(torch.randint(0, total + 1, (pieces - 1,), generator=g))[0] if pieces > 1 else \
        torch.empty(0, dtype=torch.int64)
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
    if kind == "linear":
        S, T, H, K, V = (case[n] for n in "STHKV")

        def plane(width):
            if case["packed"]:
                return normal(T, H, width).to(dtype)
            if case["heads"]:
                return normal(S, H, T, width).to(dtype).transpose(1, 2)
            return normal(S, T, H, width).to(dtype)
        s["q"], s["k"], s["v"] = plane(K), plane(K), plane(V)
        s["scale"] = K ** -0.5
        # a head forgets within 8 tokens, another within thousands
        s["decay"] = 1.0 - torch.exp2(-3.0 - 8.0 * torch.arange(H, device=DEVICE) / H).float()
        if case["packed"]:
            cuts = _cuts(host, S, T)
            s["offsets"], s["longest"] = cuts.to(DEVICE), int((cuts[1:] - cuts[:-1]).max())
        if case["state"]:
            s["h0"] = normal(S, H, K, V)
        if case["op"] == "forward":
            s["o"] = torch.empty_like(s["v"])
            if case["state"]:
                s["last"] = torch.empty_like(s["h0"])
        else:
            s["bar_o"] = plane(V)
            for n in "qkv":
                s["bar_" + n] = torch.empty_like(s[n])
            if case["state"]:
                s["bar_last"], s["bar_h0"] = normal(S, H, K, V), torch.empty_like(s["h0"])
        return s
    if kind == "norm":
        rows, cols, wide = case["rows"], case["cols"], TYPES[case["weight"]]
        s["x"] = (1.5 * normal(rows, cols) + normal(rows, 1)).to(dtype)
        s["weight"], s["bias"] = (1.0 + 0.2 * normal(cols)).to(wide), (0.2 * normal(cols)).to(wide)
        s["mean"], s["rstd"] = torch.empty(rows, device=DEVICE), torch.empty(rows, device=DEVICE)
        if case["op"] == "forward":
            s["y"] = torch.empty_like(s["x"])
            return s
        saved = _norm(s)                                     # the forward's
        s["mean"], s["rstd"] = saved["mean"], saved["rstd"]
        s["bar_y"] = normal(rows, cols).to(dtype)
        s["bar_x"] = torch.empty_like(s["x"])
        s["bar_weight"], s["bar_bias"] = torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
        return s

    N, V = case["N"], case["V"]
    logits = normal(N, V).mul_(2.0)
    # a few tokens stand out, as a trained model's do
    likely = torch.randint(0, V, (N, 8), generator=g, device=DEVICE)
    logits.scatter_add_(1, likely, 3.0 + 3.0 * torch.rand(N, 8, generator=g, device=DEVICE))
    if case["masked"]:
        logits.masked_fill_(torch.rand(N, V, generator=g, device=DEVICE) < 0.5, -math.inf)
        logits[:, 0] = 0.0                                   # one is always allowed
    s["logits"] = logits.to(dtype)
    s["u"] = torch.rand(N, generator=g, device=DEVICE)
    s["token"], s["logp"] = torch.empty(N, dtype=torch.int64, device=DEVICE), torch.empty(N, device=DEVICE)
    if case["by_row"]:
        def spread(low, high):
            return low + (high - low) * torch.rand(N, generator=g, device=DEVICE)
        s["temperature"] = spread(0.5, 1.5) * (torch.rand(N, generator=g, device=DEVICE) > 0.1)     # some are greedy
        s["top_k"] = torch.randint(0, 2 * case["top_k"] + 2, (N,), generator=g, device=DEVICE, dtype=torch.int32)
        s["top_p"], s["min_p"] = spread(case["top_p"] - 0.1, 1.01), spread(-0.01, case["min_p"])
    return s


# -- the plain forms: linear attention ---------------------------------------------------

CHUNK = 128


def _rows_of(s, back):
    """Where each sequence's i-th token lies on the packed axis (from its end: ``back``), and whether there is one."""
    first, end = s["offsets"][:-1, None], s["offsets"][1:, None]
    at = torch.arange(s["longest"], device=DEVICE)
    rows = end - 1 - at if back else first + at
    return rows.clamp(0, s["case"]["T"] - 1), at < end - first


def _sequences(s, x, back):
    """A plane as ``(S, H, T, D)`` in float32, reversed in time if ``back``, zeros behind a sequence's last token."""
    if s["case"]["packed"]:
        rows, there = _rows_of(s, back)
        x = torch.where(there[:, :, None, None], x[rows].float(), 0.0)
    elif back:
        x = x.float().flip(1)
    return x.float().transpose(1, 2)


def _plane(s, x, back, dtype):
    """``(S, H, T, D)`` as the plane it belongs to."""
    x = x.transpose(1, 2)
    if s["case"]["packed"]:
        at = torch.arange(s["case"]["T"], device=DEVICE)
        seq = torch.bucketize(at, s["offsets"][1:], right=True)
        i = at - s["offsets"][seq]
        if back:
            i = s["offsets"][seq + 1] - 1 - at
        return x[seq, i].to(dtype)
    return (x.flip(1) if back else x).to(dtype)


def _power(s, n):
    """``decay^n`` of each head for whole numbers ``n``: ``(H, *n.shape)``, the exponent in float64."""
    log = torch.log(s["decay"].double()).reshape(-1, *[1] * n.dim())
    return torch.where(n > 0, torch.exp(n * log), torch.where(n == 0, 1.0, 0.0)).float()


def _lengths(s):
    return s["offsets"][1:] - s["offsets"][:-1] if s["case"]["packed"] else \
        torch.full((s["case"]["S"],), s["case"]["T"], device=DEVICE)


def _attend(s, a, b, c, start):
    """``out_i = sum_{j <= i} decay^(i - j) (a_i . b_j) c_j + decay^i a_i start`` of ``(S, H, T, D)`` planes, in chunks:
    products within one, a state between them that a doubling scan carries."""
    S, H, T, _ = a.shape
    n = -(-T // CHUNK)
    pad = (0, 0, 0, n * CHUNK - T)
    a, b, c = (torch.nn.functional.pad(x, pad).reshape(S, H, n, CHUNK, -1) for x in (a, b, c))
    at = torch.arange(CHUNK, device=DEVICE)
    inside = (a @ b.transpose(-1, -2)) * _power(s, at[:, None] - at[None, :])[None, :, None]
    out = inside @ c
    state = (b * _power(s, CHUNK - at)[None, :, None, :, None]).transpose(-1, -2) @ c      # what each chunk leaves
    state = torch.cat([start[:, :, None], state[:, :, :-1]], 2)
    step = 1
    while step < n:
        gain = _power(s, torch.full((1, 1, 1), step * CHUNK, device=DEVICE))[None]
        state = torch.cat([state[:, :, :step], state[:, :, step:] + gain * state[:, :, :-step]], 2)
        step *= 2
    out = out + (a * _power(s, at)[None, :, None, :, None]) @ state
    return out.reshape(S, H, n * CHUNK, -1)[:, :, :T]


def _leaves(s, b, c, start):
    """``sum_j decay^(T - 1 - j) b_j c_j^T + decay^T start``, T each sequence's length."""
    T = _lengths(s)
    left = T[:, None] - 1 - torch.arange(b.shape[2], device=DEVICE)
    return (b * _power(s, left).transpose(0, 1)[..., None]).transpose(-1, -2) @ c + \
        _power(s, T).transpose(0, 1)[..., None, None] * start


def _linear(s):
    q, k, v = (_sequences(s, s[n], False) for n in "qkv")
    decay = s["decay"][:, None, None]
    h0 = s.get("h0", torch.zeros((), device=DEVICE).expand(q.shape[0], q.shape[1], q.shape[3], v.shape[3]))
    out = {"o": _plane(s, s["scale"] * _attend(s, q, k, v, decay * h0), False, s["v"].dtype)}
    if s["case"]["state"]:
        out["last"] = _leaves(s, k, v, h0)
    return out


def _linear_vjp(s):
    """Each gradient is linear attention with the planes in other places: by q forward in time, by k and v backward."""
    dtype, scale = s["q"].dtype, s["scale"]
    decay = s["decay"][:, None, None]
    k, v, bar = (_sequences(s, s[n], False) for n in ("k", "v", "bar_o"))
    zero = torch.zeros((), device=DEVICE).expand(k.shape[0], k.shape[1], k.shape[3], v.shape[3])
    h0, bar_last = s.get("h0", zero), s.get("bar_last", zero)
    out = {"bar_q": _plane(s, scale * _attend(s, bar, v, k, (decay * h0).transpose(-1, -2)), False, dtype)}
    q, k, v, bar = (_sequences(s, s[n], True) for n in ("q", "k", "v", "bar_o"))
    out["bar_k"] = _plane(s, _attend(s, v, scale * bar, q, bar_last.transpose(-1, -2)), True, dtype)
    out["bar_v"] = _plane(s, _attend(s, k, scale * q, bar, bar_last), True, dtype)
    if s["case"]["state"]:
        some = (_lengths(s) > 0)[:, None, None, None]
        left = _leaves(s, scale * q, bar, bar_last / decay)
        out["bar_h0"] = torch.where(some, decay * left, bar_last)
    return out


# -- the plain forms: layer norm and sampling --------------------------------------------

def _norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
    y = (x - mean) * rstd * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _norm_vjp(s):
    rstd = s["rstd"][:, None]
    xh, bar_y = (s["x"].float() - s["mean"][:, None]) * rstd, s["bar_y"].float()
    g = bar_y * s["weight"].float()
    bar_x = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"bar_x": bar_x.to(s["x"].dtype), "bar_weight": (bar_y * xh).sum(0).to(s["weight"].dtype),
            "bar_bias": bar_y.sum(0).to(s["bias"].dtype)}


def _settings(s):
    """Each row's temperature, top_k, top_p and min_p, as columns."""
    def column(name):
        x = s[name].double() if name in s else torch.full((s["case"]["N"],), float(s["case"][name]), device=DEVICE,
                                                         dtype=torch.float64)
        return x[:, None]
    return column("temperature"), column("top_k"), column("top_p"), column("min_p")


def _filters(case):
    return case["by_row"] or case["top_k"] > 0 or case["top_p"] < 1.0 or case["min_p"] > 0.0


def _sample(s):
    x = s["logits"].double()
    V = x.shape[1]
    temperature, top_k, top_p, min_p = _settings(s)
    top, greedy = x.amax(1, keepdim=True), x.argmax(1)
    scaled = torch.where(x == top, 0.0, (x - top) / torch.where(temperature > 0.0, temperature, 1.0))
    w = torch.exp(scaled)
    if _filters(s["case"]):
        order = torch.sort(x, dim=1, descending=True, stable=True)[1]        # equal logits by index
        rank = torch.arange(V, device=DEVICE)
        some = torch.where(top_k > 0, top_k, V)
        ordered = w.gather(1, order)
        kept = torch.where(rank < some, ordered, 0.0)
        sums = kept.cumsum(1)
        keep = (rank < some) & ((sums - kept < top_p * sums[:, -1:]) | (top_p >= 1.0)) & (ordered >= min_p) | (rank == 0)
        w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    sums = w.cumsum(1)
    token = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(1)
    logp = scaled.gather(1, token[:, None])[:, 0] - torch.log(sums[:, -1])
    cold = temperature[:, 0] == 0.0
    return {"token": torch.where(cold, greedy, token), "logp": torch.where(cold, 0.0, logp).float()}


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
    kind = case["kind"]
    if not own:
        if kind == "linear":
            return _linear_vjp(s) if case["op"] == "vjp" else _linear(s)
        if kind == "norm":
            return _norm_vjp(s) if case["op"] == "vjp" else _norm(s)
        return _sample(s)

    import hawk_amd as hawk
    if kind == "linear":
        stage = _stage("linear_attention", ("scale", s["scale"]))
        planes = _given(s, "q", "k", "v", "decay", "h0", "offsets")
        if case["op"] == "forward":
            hawk.run(stage, **planes, **_given(s, "o", "last"))
            return _given(s, "o", "last")
        hawk.run(stage.vjp, **planes, **_given(s, "bar_o", "bar_last", "bar_q", "bar_k", "bar_v", "bar_h0"))
        return _given(s, "bar_q", "bar_k", "bar_v", "bar_h0")
    if kind == "norm":
        stage = _stage("layer_norm", ("eps", EPS))
        if case["op"] == "forward":
            hawk.run(stage, **_given(s, "x", "weight", "bias", "y", "mean", "rstd"))
            return _given(s, "y", "mean", "rstd")
        hawk.run(stage.vjp, **_given(s, "x", "weight", "mean", "rstd", "bar_y", "bar_x", "bar_weight", "bar_bias"))
        return _given(s, "bar_x", "bar_weight", "bar_bias")
    stage = _stage("sample", *((n, case[n]) for n in ("temperature", "top_k", "top_p", "min_p")))
    hawk.run(stage, **_given(s, "logits", "u", "temperature", "top_k", "top_p", "min_p", "token", "logp"))
    return _given(s, "token", "logp")


# -- from the definitions, in 64 bits --------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        return _exact_linear(s)
    if case["kind"] == "norm":
        return _exact_norm(s)
    return _exact_sample(s)


def _exact_linear(s):
    """Token by token: ``S_t = decay S_(t-1) + k_t v_t^T``, ``o_t = scale q_t S_t``, and its derivative backward."""
    case = s["case"]
    S, H, K, V = (case[n] for n in "SHKV")
    T = s["longest"] if case["packed"] else case["T"]
    cuts = s["offsets"] if case["packed"] else torch.arange(S + 1, device=DEVICE) * T
    decay = s["decay"].double()[:, None, None]

    def at(name, t):
        """The t-th token of every sequence (some token where there is none)."""
        x = s[name]
        rows = x[(cuts[:-1] + t).clamp(max=case["T"] - 1)] if case["packed"] else x[:, t]
        return rows.double()
    lengths = cuts[1:] - cuts[:-1]
    there = [(lengths > t)[:, None, None, None] for t in range(T)] if case["packed"] else [None] * T

    def kept(t, new, old):
        return new if there[t] is None else torch.where(there[t], new, old)

    def planes(rows, width):
        """Every token's row, where the plane has it."""
        if not case["packed"]:
            return torch.stack(rows, 1)
        out = torch.zeros(case["T"], H, width, dtype=torch.float64, device=DEVICE)
        bounds = cuts.tolist()
        every = torch.stack(rows, 1)
        for n in range(S):
            out[bounds[n]:bounds[n + 1]] = every[n, :bounds[n + 1] - bounds[n]]
        return out
    state = s["h0"].double() if case["state"] else torch.zeros(S, H, K, V, dtype=torch.float64, device=DEVICE)
    forward = case["op"] == "forward"
    rows = []
    for t in range(T):
        state = kept(t, decay * state + at("k", t)[..., :, None] * at("v", t)[..., None, :], state)
        if forward:
            rows.append(s["scale"] * (at("q", t)[..., :, None] * state).sum(-2))
        else:
            rows.append(s["scale"] * (at("bar_o", t)[..., None, :] * state).sum(-1))
    if forward:
        return {"o": planes(rows, V), **({"last": state} if case["state"] else {})}
    out = {"bar_q": planes(rows, K)}
    bar = s["bar_last"].double() if case["state"] else torch.zeros_like(state)
    bar_k, bar_v = [None] * T, [None] * T
    for t in reversed(range(T)):
        bar = kept(t, bar + s["scale"] * at("q", t)[..., :, None] * at("bar_o", t)[..., None, :], bar)
        bar_k[t] = (bar * at("v", t)[..., None, :]).sum(-1)
        bar_v[t] = (bar * at("k", t)[..., :, None]).sum(-2)
        bar = kept(t, decay * bar, bar)
    out["bar_k"], out["bar_v"] = planes(bar_k, K), planes(bar_v, V)
    if case["state"]:
        out["bar_h0"] = bar
    return out


def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    n = x.shape[1]
    if s["case"]["op"] == "forward":
        mean = x.sum(1) / n
        rstd = torch.rsqrt(torch.var(x, 1, correction=0) + EPS)
        y = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], w)
        return {"y": y, "mean": mean, "rstd": rstd}
    # the saved forward's numbers are inputs
    r = s["rstd"].double()[:, None]
    xh, bar = (x - s["mean"].double()[:, None]) * r, s["bar_y"].double()
    one, two = (bar @ w)[:, None] / n, ((bar * xh) @ w)[:, None] / n
    return {"bar_x": (bar * w - one - xh * two) * r, "bar_weight": torch.einsum("nc,nc->c", bar, xh),
            "bar_bias": bar.sum(0)}


def _exact_sample(s):
    """Row by row in blocks: probabilities, each token's place among them, the kept ones' inverse distribution."""
    case = s["case"]
    N, V = case["N"], case["V"]
    settings = [c[:, 0] for c in _settings(s)]
    token, logp = torch.empty(N, dtype=torch.int64, device=DEVICE), torch.zeros(N, dtype=torch.float64, device=DEVICE)
    block = max(1, (1 << 25) // V)
    for r in range(0, N, block):
        w = slice(r, r + block)
        temperature, top_k, top_p, min_p = (c[w, None] for c in settings)
        x = s["logits"][w].double()
        cold = temperature == 0.0
        p = torch.softmax(x / torch.where(cold, 1.0, temperature), 1)
        keep = torch.ones_like(p, dtype=torch.bool)
        if _filters(case):
            order = torch.argsort(-x, dim=1, stable=True)
            place = torch.empty_like(order).scatter_(1, order, torch.arange(V, device=DEVICE).expand_as(order))
            keep = (place < top_k) | (top_k <= 0)
            p = torch.where(keep, p, 0.0)
            p = p / p.sum(1, keepdim=True)
            along = p.gather(1, order)
            before = (along.cumsum(1) - along).gather(1, place)
            keep &= ((before < top_p) | (top_p >= 1.0)) & (p >= min_p * p.amax(1, keepdim=True))
            keep |= place == 0
        p = torch.where(keep, p, 0.0)
        p = p / p.sum(1, keepdim=True)
        upto = p.cumsum(1)
        found = torch.searchsorted(upto, s["u"][w].double()[:, None] * upto[:, -1:], right=True)
        first = (x == x.amax(1, keepdim=True)).double().argmax(1)
        token[w] = torch.where(cold[:, 0], first, found[:, 0].clamp(max=V - 1))
        logp[w] = torch.where(cold[:, 0], 0.0, torch.log(p.gather(1, token[w][:, None])[:, 0]))
    return {"token": token, "logp": logp}
