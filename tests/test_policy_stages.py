"""Layer norm, linear attention and sampling (``hawk.stages``) against plain
loops in 64 bits.

Tolerances.  ``u`` = 2^-24 is half an ulp of 1 in the arithmetic's type, ``r`` half an
ulp of 1 in the output's (2^-24, bfloat16 2^-8, float16 2^-11).  A sum of n numbers
added in lanes of at most n / 64 + 64 after each other errs by (n / 64 + 64) u times the
sum of their magnitudes; what is computed from it adds a few u.  Linear attention takes
its products to p = 2^-16 of each (16-bit planes) or 2^-23 (float32 and states), so with
the same sum of magnitudes M as the result's an output errs by (p + n u) M, n the terms
that are added after each other, at most (channels + 64) / 4 + tokens / 16 + 64, and
rounds by r.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

import hawk_amd as hawk
from hawk_amd import HawkError, _core, diff

TYPES = ("float32", "bfloat16", "float16")
U = 2.0 ** -24
R = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
P = {"float32": 2.0 ** -23, "bfloat16": 2.0 ** -16, "float16": 2.0 ** -16}
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -25}


def torch_type(name):
    import torch
    return getattr(torch, name)


def plane(x, dtype, device):
    """``x`` in ``dtype`` on the device, and the values it holds, in 64 bits."""
    import torch
    held = torch.from_numpy(np.asarray(x, dtype=np.float64)).to(torch_type(dtype)).to(device)
    return held, held.double().cpu().numpy()


def back(x):
    return x.double().cpu().numpy()


def within(got, want, bound):
    assert np.isfinite(got).all()
    worst = np.abs(got - want) - bound
    assert (worst <= 0).all(), f"off by {np.abs(got - want).max()} where {bound[np.unravel_index(worst.argmax(), worst.shape)]} is allowed"


def apart(t, extra, start=1):
    """The same values with rows further apart, at an odd address."""
    import torch
    wide = torch.full((*t.shape[:-1], t.shape[-1] + extra), 7.0, dtype=t.dtype, device=t.device)
    view = wide[..., start:start + t.shape[-1]]
    view.copy_(t)
    return view


# -- layer norm ------------------------------------------------------------------------------

EPS = 1e-5
NORMS = [(1, 1), (3, 5), (257, 8), (17, 127), (130, 128), (33, 129), (5, 512), (9, 777), (1500, 1024), (7, 2048), (4, 3001),
         (3, 4096), (2, 8192), (3, 9999), (2, 16384), (2, 16385), (3, 40001), (70, 33000), (0, 12), (4100, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_layer_norm_and_its_derivative(gpu, shape, dtype):
    import torch
    N, C = shape
    g = np.random.default_rng([N, C])
    n = C / 64 + 64
    for wide, affine, spread in ((False, True, False), (True, True, True), (False, False, True)):
        print(shape, dtype, wide, affine, spread, flush=True)
        kind = "float32" if wide else dtype
        x, xv = plane(g.normal(size=(N, C)) * 1.5 + 3 * g.normal(size=(N, 1)), dtype, gpu)
        w, wv = plane(1 + 0.3 * g.normal(size=C), kind, gpu)
        b, bv = plane(g.normal(size=C), kind, gpu)
        by, byv = plane(g.normal(size=(N, C)), dtype, gpu)
        given = dict(weight=w, bias=b) if affine else {}
        if not affine:
            wv, bv = np.ones(C), np.zeros(C)
        if spread:
            x, by = apart(x, 5), apart(by, 2)
        y = apart(torch.zeros(N, C, dtype=x.dtype, device=gpu), 3) if spread else torch.empty_like(x)
        mean, rstd = torch.empty(N, device=gpu), torch.empty(N, device=gpu)
        stage = hawk.stages.layer_norm(eps=EPS)
        hawk.run(stage, x=x, y=y, mean=mean, rstd=rstd, **given)
        m = xv.mean(1, keepdims=True)
        r = 1 / np.sqrt(((xv - m) ** 2).mean(1, keepdims=True) + EPS)
        size = np.abs(xv).mean(1, keepdims=True)
        xh = (xv - m) * r
        within(back(mean), m[:, 0], (n + 4) * U * size[:, 0] + 1e-37)
        # the variance about a mean that is off by d is more by d^2
        loose = (n + 8) * U + ((n + 4) * U * size * r) ** 2
        within(back(rstd), r[:, 0], (loose * r)[:, 0])
        want = xh * wv + bv
        off = (n + 8) * U * (np.abs(wv) * r * (size + np.abs(xv)) + np.abs(bv)) + loose * np.abs(xh * wv)
        within(back(y), want, off * (1 + R[dtype]) + R[dtype] * np.abs(want) + TINY[dtype])
        if spread and N > 1:                                    # what lies between the rows stays
            assert (torch.as_strided(y, (N - 1, 3), (y.stride(0), 1), y.storage_offset() + C) == 7).all()
        # the derivative at the mean and rstd that were saved
        mv, rv = back(mean)[:, None], back(rstd)[:, None]
        xh = (xv - mv) * rv
        bars = dict(bar_x=torch.empty(N, C, dtype=x.dtype, device=gpu))
        if affine:
            bars.update(bar_weight=torch.empty_like(w), bar_bias=torch.empty_like(b))
        hawk.run(stage.vjp, x=x, mean=mean, rstd=rstd, bar_y=by, **bars, **({"weight": w} if affine else {}))
        gy = byv * wv
        one, two = gy.mean(1, keepdims=True), (gy * xh).mean(1, keepdims=True)
        want = rv * (gy - one - xh * two)
        off = (n + 12) * U * rv * (np.abs(gy) + np.abs(gy).mean(1, keepdims=True) + np.abs(xh) * np.abs(gy * xh).mean(1, keepdims=True))
        within(back(bars["bar_x"]), want, off * (1 + R[dtype]) + R[dtype] * np.abs(want) + TINY[dtype])
        if affine:
            rows = N / 64 + 72
            for name, terms in (("bar_weight", byv * xh), ("bar_bias", byv)):
                want = terms.sum(0)
                within(back(bars[name]), want, rows * U * np.abs(terms).sum(0) * (1 + R[kind]) + R[kind] * np.abs(want) + TINY[kind])


@pytest.mark.gpu
def test_layer_norms_derivative_is_its_difference_quotient(gpu):
    """Central differences of sum(bar_y y), a sum of 24 numbers of order 1 in float32 rounded to 2^-24 each:
    24 * 2^-24 / e from rounding and e^2 from the third derivative, below 3e-4 at e = 2^-6."""
    import torch
    g = np.random.default_rng(3)
    base = {"x": g.normal(size=(2, 12)), "weight": 1 + 0.2 * g.normal(size=12), "bias": g.normal(size=12)}
    bar = torch.from_numpy(g.normal(size=(2, 12))).float().to(gpu)
    stage = hawk.stages.layer_norm()

    def put(values):
        return {n: torch.from_numpy(v).float().to(gpu) for n, v in values.items()}

    def forward(values):
        t = put(values)
        y = torch.empty_like(t["x"])
        hawk.run(stage, y=y, **t)
        return float((back(y) * back(bar)).sum())
    t = put(base)
    mean, rstd, y = torch.empty(2, device=gpu), torch.empty(2, device=gpu), torch.empty_like(t["x"])
    hawk.run(stage, y=y, mean=mean, rstd=rstd, **t)
    bars = {"bar_" + n: torch.empty_like(v) for n, v in t.items()}
    hawk.run(diff.vjp(stage), x=t["x"], weight=t["weight"], mean=mean, rstd=rstd, bar_y=bar, **bars)
    e = 2.0 ** -6
    for n in base:
        for index in [tuple(g.integers(0, d) for d in base[n].shape) for _ in range(8)]:
            ends = []
            for sign in (1, -1):
                moved = {m: v.copy() for m, v in base.items()}
                moved[n][index] += sign * e
                ends.append(forward(moved))
            slope = (ends[0] - ends[1]) / (2 * e)
            assert abs(slope - back(bars["bar_" + n])[index]) < 2e-3 * (1 + abs(slope)), (n, index)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [40, 3000, 50000])
def test_layer_norm_in_place_and_a_row_that_is_no_number(gpu, C):
    import torch
    N = 5
    g = torch.Generator(device=gpu).manual_seed(C)
    x = torch.randn(N, C, generator=g, device=gpu)
    x[1, C // 2], x[3, 0] = math.nan, math.inf
    x[4] = 3.0                                                  # a row without variance
    stage = hawk.stages.layer_norm(eps=1e-3)
    y, mean, rstd = torch.empty_like(x), torch.empty(N, device=gpu), torch.empty(N, device=gpu)
    hawk.run(stage, x=x, y=y, mean=mean, rstd=rstd)
    assert torch.isfinite(y[[0, 2, 4]]).all() and not torch.isfinite(y[[1, 3]]).all(1).any()
    assert (y[4] == 0).all() and mean[4] == 3.0 and abs(float(rstd[4]) - 1e-3 ** -0.5) < 1e-5
    bar = torch.randn(N, C, generator=g, device=gpu)
    out = torch.empty_like(x)
    hawk.run(stage.vjp, x=x, mean=mean, rstd=rstd, bar_y=bar, bar_x=out)
    for held in ("x", "bar_y"):                                 # over an input
        planes = dict(x=x.clone(), bar_y=bar.clone())
        hawk.run(stage.vjp, mean=mean, rstd=rstd, bar_x=planes[held], **planes)
        assert torch.equal(planes[held][[0, 2, 4]], out[[0, 2, 4]])
    hawk.run(stage, x=x, y=x)
    assert torch.equal(x[[0, 2, 4]], y[[0, 2, 4]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,C", [("float32", 50), ("bfloat16", 2049), ("float16", 16383), ("bfloat16", 16400), ("float32", 8200)])
def test_layer_norms_derivative_written_over_its_inputs(gpu, dtype, C):
    """``bar_x`` over ``x`` or ``bar_y``: the bits of the call that writes another plane."""
    import torch
    g, N = torch.Generator().manual_seed(C), 700
    x, by = (torch.randn(N, C, generator=g).to(gpu, getattr(torch, dtype)) for _ in range(2))
    w, y, mean, rstd = torch.randn(C, generator=g).to(gpu), torch.empty_like(x), torch.empty(N, device=gpu), torch.empty(N, device=gpu)
    stage = hawk.stages.layer_norm()
    hawk.run(stage, x=x, weight=w, y=y, mean=mean, rstd=rstd)

    def derivative(x, by, bx):
        bw, bb = torch.full((2, C), 7.0, device=gpu)
        hawk.run(stage.vjp, x=x, weight=w, mean=mean, rstd=rstd, bar_y=by, bar_x=bx, bar_weight=bw, bar_bias=bb)
        return bx, bw, bb

    want = derivative(x, by, torch.empty_like(x))
    a, b = x.clone(), by.clone()
    for got in (derivative(a, by, a), derivative(x, b, b)):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


# -- linear attention --------------------------------------------------------------------------

def spans(S, T, offsets):
    if offsets is None:
        return [(s, slice(0, T)) for s in range(S)]
    return [(s, slice(int(offsets[s]), int(offsets[s + 1]))) for s in range(S)]


def attention(q, k, v, decay, scale, h0, offsets):
    """The outputs, the states that leave, and the sums of their terms' magnitudes."""
    S = len(offsets) - 1 if offsets is not None else q.shape[0]
    H, K, V = q.shape[-2], q.shape[-1], v.shape[-1]
    o, size = np.zeros((*q.shape[:-1], V)), np.zeros((*q.shape[:-1], V))
    last, most = np.zeros((S, H, K, V)), np.zeros((S, H, K, V))
    for s, rows in spans(S, q.shape[-3], offsets):
        at = (lambda x: x[rows]) if offsets is not None else (lambda x: x[s])
        state = np.zeros((H, K, V)) if h0 is None else h0[s].copy()
        mass = np.abs(state)
        g = decay[:, None, None]
        for t in range(at(q).shape[0]):
            state = g * state + at(k)[t][:, :, None] * at(v)[t][:, None, :]
            mass = g * mass + np.abs(at(k)[t])[:, :, None] * np.abs(at(v)[t])[:, None, :]
            at(o)[t] = scale * np.einsum("hk,hkv->hv", at(q)[t], state)
            at(size)[t] = abs(scale) * np.einsum("hk,hkv->hv", np.abs(at(q)[t]), mass)
        last[s], most[s] = state, mass
    return o, last, size, most


def attention_vjp(q, k, v, decay, scale, h0, bar_o, bar_last, offsets):
    S = len(offsets) - 1 if offsets is not None else q.shape[0]
    H, K, V = q.shape[-2], q.shape[-1], v.shape[-1]
    bars = [np.zeros_like(x) for x in (q, k, v)]
    sizes = [np.zeros_like(x) for x in (q, k, v)]
    bar_h0, most = np.zeros((S, H, K, V)), np.zeros((S, H, K, V))
    g = decay[:, None, None]
    for s, rows in spans(S, q.shape[-3], offsets):
        at = (lambda x: x[rows]) if offsets is not None else (lambda x: x[s])
        state = np.zeros((H, K, V)) if h0 is None else h0[s].copy()
        mass = np.abs(state)
        for t in range(at(q).shape[0]):
            state = g * state + at(k)[t][:, :, None] * at(v)[t][:, None, :]
            mass = g * mass + np.abs(at(k)[t])[:, :, None] * np.abs(at(v)[t])[:, None, :]
            at(bars[0])[t] = scale * np.einsum("hv,hkv->hk", at(bar_o)[t], state)
            at(sizes[0])[t] = abs(scale) * np.einsum("hv,hkv->hk", np.abs(at(bar_o)[t]), mass)
        W = np.zeros((H, K, V)) if bar_last is None else bar_last[s].copy()
        mass = np.abs(W)
        for t in reversed(range(at(q).shape[0])):
            W = W + scale * at(q)[t][:, :, None] * at(bar_o)[t][:, None, :]
            mass = mass + abs(scale) * np.abs(at(q)[t])[:, :, None] * np.abs(at(bar_o)[t])[:, None, :]
            at(bars[1])[t] = np.einsum("hkv,hv->hk", W, at(v)[t])
            at(sizes[1])[t] = np.einsum("hkv,hv->hk", mass, np.abs(at(v)[t]))
            at(bars[2])[t] = np.einsum("hk,hkv->hv", at(k)[t], W)
            at(sizes[2])[t] = np.einsum("hk,hkv->hv", np.abs(at(k)[t]), mass)
            W, mass = g * W, g * mass
        bar_h0[s], most[s] = W, mass
    return bars, bar_h0, sizes, most


def close(got, want, size, terms, p, r, tiny):
    within(got, want, (p + terms * U) * size * (1 + r) + r * np.abs(want) + tiny)


def attention_case(S, T, H, K, V, dtype, layout, state, packed, device, seed):
    import torch
    g = np.random.default_rng([seed, S, T, H, K, V])
    lead = (T, H) if packed else (S, T, H)
    offsets = None
    if packed:
        cut = np.sort(g.integers(0, T + 1, S - 1)) if S > 1 else np.array([], int)
        if S >= 4:
            cut[1] = cut[0]
            cut[-1] = T
        offsets = np.concatenate([[0], cut, [T]])
    got, held = {}, {}
    for n, width in (("q", K), ("k", K), ("v", V), ("bar_o", V)):
        t, held[n] = plane(g.normal(size=(*lead, width)), dtype, device)
        if layout == "heads":                                   # heads outside the steps
            t = t.transpose(-2, -3).contiguous().transpose(-2, -3)
        elif layout == "sliced":
            t = apart(t, 3)
        got[n] = t
    if state:
        for n in ("h0", "bar_last"):
            got[n], held[n] = plane(g.normal(size=(S, H, K, V)), "float32", device)
    decay = np.float32(1 - 2.0 ** -np.linspace(1, 8, H)).astype(np.float64)
    if H > 2:
        decay[0], decay[1] = 0.0, 1.0
    got["decay"], held["decay"] = torch.from_numpy(decay).float().to(device), decay
    if packed:
        got["offsets"] = torch.from_numpy(offsets).to(device, torch.int32 if seed % 2 else torch.int64)
    return got, held, offsets


def check_attention(gpu, S, T, H, K, V, dtype, layout, state, packed, seed):
    import torch
    got, held, offsets = attention_case(S, T, H, K, V, dtype, layout, state, packed, gpu, seed)
    scale = 0.37
    stage = hawk.stages.linear_attention(scale=scale)
    planes = {n: got[n] for n in ("q", "k", "v", "decay", "h0", "offsets") if n in got}
    o = torch.zeros_like(got["v"])
    last = torch.empty(S, H, K, V, device=gpu)
    hawk.run(stage, o=o, last=last, **planes)
    want, want_last, size, most = attention(held["q"], held["k"], held["v"], held["decay"], scale, held.get("h0"), offsets)
    terms = (max(K, V) + 64) / 4 + T / 16 + 64
    close(back(o), want, size, terms, P[dtype], R[dtype], TINY[dtype])
    close(back(last), want_last, most, terms, P["float32"], U, 1e-37)
    if T * H * S > 64:                                          # what errors of either sign leave of those bounds
        assert np.linalg.norm(back(o) - want) <= max(R[dtype], 2.0 ** -20) * np.linalg.norm(want)
        assert np.linalg.norm(back(last) - want_last) <= 2.0 ** -20 * np.linalg.norm(want_last)
    bars = {n: torch.zeros_like(got[n[4:]]) for n in ("bar_q", "bar_k", "bar_v")}
    bars["bar_h0"] = torch.empty_like(last)
    if state:
        planes["bar_last"] = got["bar_last"]
    hawk.run(stage.vjp, bar_o=got["bar_o"], **planes, **bars)
    wants, want_h0, sizes, most = attention_vjp(held["q"], held["k"], held["v"], held["decay"], scale, held.get("h0"),
                                                held["bar_o"], held.get("bar_last"), offsets)
    for n, w, z in zip(("bar_q", "bar_k", "bar_v"), wants, sizes):
        close(back(bars[n]), w, z, terms, P[dtype], R[dtype], TINY[dtype])
    close(back(bars["bar_h0"]), want_h0, most, terms, P["float32"], U, 1e-37)


ATTENTIONS = [(1, 1, 1, 1, 1), (3, 1, 3, 16, 16), (2, 2, 2, 33, 5), (1, 31, 3, 32, 64), (2, 64, 1, 64, 65), (1, 65, 4, 40, 130),
              (2, 130, 3, 128, 128), (1, 200, 2, 129, 17), (5, 33, 2, 7, 256), (1, 97, 1, 256, 256), (4, 300, 3, 20, 48)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ATTENTIONS, ids=str)
def test_linear_attention_and_its_derivative_are_the_loop(gpu, shape, dtype):
    for k, (layout, state, packed) in enumerate([("steps", True, False), ("heads", False, False), ("sliced", True, False),
                                                 ("steps", True, True), ("sliced", False, True)]):
        print(shape, dtype, layout, state, packed, flush=True)
        check_attention(gpu, *shape, dtype, layout, state, packed, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,packed", [((1, 1500, 2, 48, 80), False), ((3, 700, 1, 130, 24), False), ((1, 2049, 1, 16, 16), True),
                                          ((7, 3000, 1, 64, 32), True), ((700, 1500, 8, 9, 12), True), ((300, 2600, 2, 20, 33), True)],
                         ids=str)
def test_a_long_sequence_is_cut_and_joined(gpu, shape, packed, dtype):
    check_attention(gpu, *shape, dtype, "steps", True, packed, 1)


@pytest.mark.gpu
def test_linear_attentions_derivative_is_its_difference_quotient(gpu):
    """The form is linear in each plane, so central differences of sum(w o) + sum(x last) err by rounding alone:
    sums of some hundred float32 numbers, 2^-24 * 100 / e, below 1e-3 at e = 2^-4."""
    import torch
    g = np.random.default_rng(11)
    S, T, H, K, V = 1, 7, 2, 3, 4
    base = {"q": g.normal(size=(S, T, H, K)), "k": g.normal(size=(S, T, H, K)), "v": g.normal(size=(S, T, H, V)),
            "h0": g.normal(size=(S, H, K, V))}
    decay = torch.tensor([0.5, 0.9], device=gpu)
    w, x = g.normal(size=(S, T, H, V)), g.normal(size=(S, H, K, V))
    stage = hawk.stages.linear_attention(scale=0.5)

    def put(v):
        return torch.from_numpy(v).float().to(gpu)

    def forward(values):
        o, last = torch.empty(S, T, H, V, device=gpu), torch.empty(S, H, K, V, device=gpu)
        hawk.run(stage, decay=decay, o=o, last=last, **{n: put(v) for n, v in values.items()})
        return (back(o) * w).sum() + (back(last) * x).sum()
    t = {n: put(v) for n, v in base.items()}
    bars = {"bar_" + n: torch.empty_like(v) for n, v in t.items()}
    hawk.run(diff.vjp(stage), decay=decay, bar_o=put(w), bar_last=put(x), **t, **bars)
    e = 2.0 ** -4
    for n in base:
        for index in [tuple(g.integers(0, d) for d in base[n].shape) for _ in range(8)]:
            ends = []
            for sign in (1, -1):
                moved = {m: v.copy() for m, v in base.items()}
                moved[n][index] += sign * e
                ends.append(forward(moved))
            slope = (ends[0] - ends[1]) / (2 * e)
            assert abs(slope - back(bars["bar_" + n])[index]) < 1e-3 * (1 + abs(slope)), (n, index)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [5, 200, 1500])
def test_a_token_that_is_no_number_leaves_earlier_ones(gpu, T, dtype):
    import torch
    H, K, V = 2, 24, 40
    at = T // 2 + 1
    for name, bad in (("v", math.nan), ("v", math.inf), ("k", math.nan), ("k", -math.inf), ("q", math.nan)):
        g = torch.Generator(device=gpu).manual_seed(T)
        t = {n: torch.randn(1, T, H, w, generator=g, device=gpu).to(torch_type(dtype)) for n, w in (("q", K), ("k", K), ("v", V))}
        decay = torch.tensor([0.9, 1.0], device=gpu)
        stage = hawk.stages.linear_attention()
        clean, o = torch.empty_like(t["v"]), torch.empty_like(t["v"])
        hawk.run(stage, decay=decay, o=clean, **t)
        t[name][0, at, 1, 3] = bad
        hawk.run(stage, decay=decay, o=o, **t)
        assert torch.equal(o[:, :, 0], clean[:, :, 0])                       # the other head
        # a chunk with such a token is summed in another order: the same within its rounding
        near = 2 * R[dtype] * clean.double().abs() + 1e-3 * clean.double().abs().max() * (1 if dtype != "float32" else 1e-2)
        assert ((o.double() - clean.double()).abs() <= near)[:, :at].all()
        if name == "q":
            assert not torch.isfinite(o[:, at, 1]).any() and torch.isfinite(o[:, at + 1:]).all()
        elif name == "v":
            assert not torch.isfinite(o[:, at:, 1, 3]).any() and torch.isfinite(o[:, :, 1, :3]).all()
        else:
            assert not torch.isfinite(o[:, at:, 1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_token_at_a_time_is_the_whole_prompt(gpu, dtype):
    """The states are float32 on both ways, so outputs differ by their rounding and 1e-5 of their terms."""
    import torch
    S, T, H, K, V = 3, 70, 2, 32, 24
    g = torch.Generator(device=gpu).manual_seed(1)
    q, k, v = (torch.randn(S, T, H, w, generator=g, device=gpu).to(torch_type(dtype)) for w in (K, K, V))
    decay = torch.tensor([0.8, 0.99], device=gpu)
    stage = hawk.stages.linear_attention(scale=K ** -0.5)
    o, last = torch.empty_like(v), torch.empty(S, H, K, V, device=gpu)
    hawk.run(stage, q=q, k=k, v=v, decay=decay, o=o, last=last)
    state, step = torch.zeros(S, H, K, V, device=gpu), torch.empty(S, 1, H, V, dtype=v.dtype, device=gpu)
    for t in range(T):
        hawk.run(stage, q=q[:, t:t + 1], k=k[:, t:t + 1], v=v[:, t:t + 1], decay=decay, o=step, h0=state, last=state)
        off = (step[:, 0].double() - o[:, t].double()).abs()
        assert (off <= 2 * R[dtype] * o[:, t].double().abs() + 1e-4).all(), t
    assert (state - last).abs().max() < 1e-4
    # the prompt in two parts
    one, two, mid = torch.empty_like(v[:, :33]), torch.empty_like(v[:, 33:]), torch.empty_like(last)
    hawk.run(stage, q=q[:, :33], k=k[:, :33], v=v[:, :33], decay=decay, o=one, last=mid)
    hawk.run(stage, q=q[:, 33:], k=k[:, 33:], v=v[:, 33:], decay=decay, o=two, h0=mid, last=mid)
    assert ((torch.cat([one, two], 1).double() - o.double()).abs() <= 2 * R[dtype] * o.double().abs() + 1e-4).all()
    assert (mid - last).abs().max() < 1e-4


@pytest.mark.gpu
def test_heads_that_share_keys_and_values(gpu):
    """Expanded planes: the outputs are those of copies, a gradient is the sum over the heads."""
    import torch
    S, T, H, K, V = 2, 90, 6, 16, 32
    g = torch.Generator(device=gpu).manual_seed(2)
    q, bar = torch.randn(S, T, H, K, generator=g, device=gpu), torch.randn(S, T, H, V, generator=g, device=gpu)
    k, v = (torch.randn(S, T, 1, w, generator=g, device=gpu).expand(S, T, H, w) for w in (K, V))
    decay = torch.linspace(0.5, 1, H, device=gpu)
    stage = hawk.stages.linear_attention()
    outs = []
    for a, b in ((k, v), (k.contiguous(), v.contiguous())):
        o = torch.empty(S, T, H, V, device=gpu)
        hawk.run(stage, q=q, k=a, v=b, decay=decay, o=o)
        bars = [torch.empty(S, T, H, w, device=gpu) for w in (K, K, V)]
        hawk.run(stage.vjp, q=q, k=a, v=b, decay=decay, bar_o=bar, bar_q=bars[0], bar_k=bars[1], bar_v=bars[2])
        outs.append([o, *bars])
    assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.gpu
def test_linear_attention_without_steps_sequences_or_heads(gpu):
    import torch
    stage = hawk.stages.linear_attention()
    h0 = torch.randn(2, 3, 4, 5, device=gpu)
    z = lambda *s: torch.zeros(s, device=gpu)  # noqa: E731
    last = torch.empty_like(h0)
    hawk.run(stage, q=z(2, 0, 3, 4), k=z(2, 0, 3, 4), v=z(2, 0, 3, 5), decay=z(3), o=z(2, 0, 3, 5), h0=h0, last=last)
    assert torch.equal(last, h0)
    hawk.run(stage, q=z(0, 3, 4), k=z(0, 3, 4), v=z(0, 3, 5), decay=z(3), o=z(0, 3, 5), last=last,
             offsets=torch.zeros(3, dtype=torch.int32, device=gpu))
    assert (last == 0).all()
    out = torch.empty_like(h0)
    hawk.run(stage.vjp, q=z(2, 0, 3, 4), k=z(2, 0, 3, 4), v=z(2, 0, 3, 5), decay=z(3), bar_o=z(2, 0, 3, 5), bar_last=h0,
             bar_h0=out)
    assert torch.equal(out, h0)
    hawk.run(stage, q=z(0, 4, 3, 4), k=z(0, 4, 3, 4), v=z(0, 4, 3, 5), decay=z(3), o=z(0, 4, 3, 5))
    hawk.run(stage, q=z(1, 4, 0, 4), k=z(1, 4, 0, 4), v=z(1, 4, 0, 5), decay=z(0), o=z(1, 4, 0, 5))
    # a decay that is none gives NaN, in its own head
    q = torch.ones(1, 3, 3, 4, device=gpu)
    o = torch.empty_like(q)
    hawk.run(stage, q=q, k=q, v=q, decay=torch.tensor([0.5, 1.5, math.nan], device=gpu), o=o)
    assert torch.isfinite(o[:, :, 0]).all() and torch.isnan(o[:, :, 1:]).all()


# -- sampling ----------------------------------------------------------------------------------

def draw(x, u, T, top_k, top_p, min_p):
    """One row: the token and its log-probability."""
    V = len(x)
    if np.isnan(x).any() or np.isnan(u) or not T >= 0:
        return -1, math.nan
    if V == 0 or x.max() == -np.inf:
        return -1, -math.inf
    if T == 0:
        return int(x.argmax()), 0.0
    with np.errstate(invalid="ignore"):
        l = np.where(x == x.max(), 0.0, (x - x.max()) / T)
    w = np.exp(l)
    order = np.argsort(-x, kind="stable")
    keep = np.ones(V, bool)
    if 0 < top_k < V:
        keep[order[top_k:]] = False
    if top_p < 1:
        ws = np.where(keep[order], w[order], 0.0)
        keep[order[np.cumsum(ws) - ws >= max(top_p, 0.0) * ws.sum()]] = False
    if min_p > 0:
        keep &= w >= min_p
    keep[order[0]] = True
    w = np.where(keep, w, 0.0)
    c = np.cumsum(w)
    at = min(int(np.searchsorted(c, u * c[-1], side="right")), int(np.nonzero(w)[0][-1])) if u > 0 else int(np.nonzero(w)[0][0])
    return at, l[at] - math.log(c[-1])


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 40, 0.8, 0.02), (0.0, 0, 1.0, 0.0), (2.0, 0, 0.0, 0.0),
            (1.0, 1, 1.0, 0.0), (0.9, 0, 1.0, 2.0), (1.5, 1500, 0.999, 1e-6), (100.0, 3000, 0.5, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 1), (40, 7), (9, 48), (5, 1000), (4, 4097), (7, 9001), (3, 50001), (2, 131072), (1, 1000003),
                                   (130, 17001), (515, 20011)], ids=str)
def test_the_drawn_token_is_the_one_of_64_bits(gpu, shape, dtype):
    """A border between two tokens is within 2^-36 of the plain form's, so of these few hundred draws none falls
    between the two; the log-probability is rounded once, and errs by the sum's 2^-40 before."""
    import torch
    N, V = shape
    g = np.random.default_rng([N, V])
    for k, setting in enumerate(SETTINGS):
        if N > 100 and k not in (0, 3, 8) or V > 200000 and k not in (2, 3, 4):
            continue
        print(shape, dtype, setting, flush=True)
        x = g.normal(size=shape) * (2 if k % 2 else 0.3)
        x[:, g.integers(0, V)] += 4
        if k % 3 == 1:
            x[g.random(shape) < 0.4] = -np.inf                  # barred tokens, a whole row among them
            x[0] = -np.inf
        if k % 4 == 2:
            x = np.round(2 * x) / 2                             # many equal logits
        t, xv = plane(x, dtype, gpu)
        if k % 2:
            t = apart(t, 3)
        u = g.random(N) if k % 2 else np.float32(g.random(N)).astype(np.float64)
        token = torch.empty(N, dtype=torch.int32 if k % 2 else torch.int64, device=gpu)
        logp = torch.empty(N, device=gpu)
        stage = hawk.stages.sample(**dict(zip(("temperature", "top_k", "top_p", "min_p"), setting)))
        hawk.run(stage, logits=t, u=torch.from_numpy(u).to(gpu, torch.float64 if k % 2 else torch.float32), token=token,
                 logp=logp)
        want = [draw(xv[n], u[n], *setting) for n in range(N)]
        assert token.cpu().tolist() == [a for a, _ in want], setting
        b = np.array([b for _, b in want])
        fine = np.isfinite(b)
        assert (back(logp)[~fine] == b[~fine]).all()
        assert np.abs(back(logp)[fine] - b[fine]).max(initial=0) <= U * np.abs(b[fine]).max(initial=0) + 2.0 ** -36


@pytest.mark.gpu
@pytest.mark.parametrize("V", [60, 5000, 30000])
def test_rows_sample_with_settings_of_their_own(gpu, V):
    import torch
    N = 64
    g = np.random.default_rng(V)
    x, xv = plane(g.normal(size=(N, V)) * 2, "float32", gpu)
    u = np.float32(g.random(N))
    cells = {"temperature": np.float32(np.where(g.random(N) < 0.2, 0, g.uniform(0.3, 2, N))), "top_k": g.integers(-1, V + 9, N),
             "top_p": np.float32(g.uniform(0.3, 1.2, N)), "min_p": np.float32(g.uniform(-0.1, 0.1, N))}
    cells["temperature"][3], cells["temperature"][4] = -1, math.nan
    planes = {n: torch.from_numpy(c).to(gpu, torch.int32 if n == "top_k" else torch.float32) for n, c in cells.items()}
    token = torch.empty(N, dtype=torch.int64, device=gpu)
    logp = torch.empty(N, device=gpu)
    u[7] = math.nan
    hawk.run(hawk.stages.sample(temperature=9.0, top_k=1, top_p=0.1, min_p=0.9), logits=x, u=torch.from_numpy(u).to(gpu),
             token=token, logp=logp, **planes)
    want = [draw(xv[n], float(u[n]), *(float(cells[c][n]) if c != "top_k" else int(cells[c][n])
                                       for c in ("temperature", "top_k", "top_p", "min_p"))) for n in range(N)]
    assert token.cpu().tolist() == [a for a, _ in want]
    b = np.array([b for _, b in want])
    assert (np.isnan(back(logp)) == np.isnan(b)).all() and np.isnan(b).sum() == 3
    assert np.nanmax(np.abs(back(logp) - b)) < 1e-6 * 20


@pytest.mark.gpu
@pytest.mark.parametrize("V", [600, 3000, 60000])
def test_sampling_at_the_borders_and_past_the_range(gpu, V):
    import torch
    z = torch.zeros(6, V, device=gpu)
    token, logp = torch.empty(6, dtype=torch.int64, device=gpu), torch.empty(6, device=gpu)
    # equal weights: token floor(u V) exactly, and u outside [0, 1) the first and the last
    u = torch.tensor([0.0, 0.25, 0.5, 1.0, -3.0, math.inf], device=gpu)
    hawk.run(hawk.stages.sample(), logits=z, u=u, token=token, logp=logp)
    assert token.tolist() == [0, V // 4, V // 2, V - 1, 0, V - 1] and (logp + math.log(V)).abs().max() < 1e-6
    # ties at the filters' borders go to the lowest index
    hawk.run(hawk.stages.sample(top_k=10), logits=z, u=u, token=token)
    assert token.tolist() == [0, 2, 5, 9, 0, 9]
    hawk.run(hawk.stages.sample(top_p=0.5), logits=z, u=u, token=token)
    assert token.tolist() == [0, V // 8, V // 4, V // 2 - 1, 0, V // 2 - 1]
    # infinities share the whole, a NaN anywhere is one, the type's lowest values are numbers
    z[0, [5, 9]], z[1, V - 1], z[2] = math.inf, math.nan, -math.inf
    z[3] = torch.finfo(torch.float32).min
    z[4], z[4, 17] = -math.inf, -1e30
    z[5, :] = torch.finfo(torch.float32).min
    z[5, 8] = torch.finfo(torch.float32).max
    u = torch.tensor([0.5, 0.5, 0.5, 0.5, 0.5, 0.5], device=gpu)
    for planes in ({}, dict(top_k=torch.full((6,), 500, dtype=torch.int32, device=gpu), top_p=torch.full((6,), 0.999, device=gpu))):
        hawk.run(hawk.stages.sample(), logits=z, u=u, token=token, logp=logp, **planes)
        at = token.tolist()
        assert at[0] == 9 and at[1:3] == [-1, -1] and at[4:] == [17, 8], at
        assert at[3] == (V // 2 if not planes else 250), at
        assert abs(float(logp[0]) + math.log(2)) < 1e-6 and math.isnan(logp[1]) and float(logp[2]) == -math.inf
        assert logp[4] == 0 and logp[5] == 0
    hawk.run(hawk.stages.sample(), logits=z[:, :0], u=u, token=token, logp=logp)
    assert (token == -1).all() and (logp == -math.inf).all()


@pytest.mark.gpu
def test_many_equal_logits_past_the_candidates(gpu):
    """A border inside more equal logits than are ranked at once, and one among logits that differ in the last bit."""
    import torch
    V = 70001
    x = torch.full((4, V), -2.0, device=gpu)
    x[1] = torch.from_numpy(np.float32(-2.0 + np.arange(V) * 2.0 ** -22)).to(gpu)      # one bin, all different
    x[2, ::3] = -1.0
    x[3] = x[1].flip(0)
    u = np.array([0.3, 0.6, 0.9, 0.1])
    held = back(x)
    for setting in ((1.0, 20000, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (0.5, 30000, 0.7, 0.0), (1.0, 65537, 0.25, 0.0)):
        want = [draw(held[n], u[n], *setting)[0] for n in range(4)]
        for times in (1, 33):                                   # rows in parts, and of a workgroup each
            token = torch.empty(4 * times, dtype=torch.int64, device=gpu)
            hawk.run(hawk.stages.sample(**dict(zip(("temperature", "top_k", "top_p", "min_p"), setting))), logits=x.repeat(times, 1),
                     u=torch.from_numpy(np.tile(u, times)).to(gpu), token=token)
            assert token.tolist() == want * times, (setting, times)


# -- together, captured, refused ---------------------------------------------------------------

@pytest.mark.gpu
def test_a_layer_trained_and_served_with_the_stages(gpu):
    """Norm, linear attention, dropout, policy loss and back: the weights' gradients are those of the same
    layer in float64, within 1e-4 of their norm (sums of some thousand float32 numbers and products)."""
    import torch
    from hawk_amd import stages
    S, T, H, K, V, C, A = 3, 40, 2, 8, 12, 24, 17
    g = torch.Generator(device=gpu).manual_seed(5)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=gpu) * scale
    u, weight, bias = normal(S, T, C), 1 + normal(C, scale=0.1), normal(C, scale=0.1)
    wq, wk, wv, wo, wa = (normal(a, b, scale=a ** -0.5) for a, b in ((C, H * K), (C, H * K), (C, H * V), (H * V, C), (C, A)))
    decay = torch.tensor([0.7, 0.95], device=gpu)
    norm, mix, choose, loss_of = (stages.layer_norm(), stages.linear_attention(scale=0.5), stages.sample(temperature=1.0),
                                  stages.policy_loss(clip=0.2))
    logp_of = stages.token_logp()

    def layer():
        x, mean, rstd = torch.empty_like(u), torch.empty(S * T, device=gpu), torch.empty(S * T, device=gpu)
        hawk.run(norm, x=u, weight=weight, bias=bias, y=x, mean=mean, rstd=rstd)
        q, k, v = ((x @ w).view(S, T, H, -1) for w in (wq, wk, wv))
        o = torch.empty_like(v)
        hawk.run(mix, q=q, k=k, v=v, decay=decay, o=o)
        y = u + o.reshape(S, T, H * V) @ wo
        return x, mean, rstd, q, k, v, o, y, (y @ wa).reshape(S * T, A)
    logits = layer()[-1]
    token, old = torch.empty(S * T, dtype=torch.int64, device=gpu), torch.empty(S * T, device=gpu)
    hawk.run(choose, logits=logits, u=torch.rand(S * T, generator=g, device=gpu), token=token, logp=old)
    logp, lse = torch.empty_like(old), torch.empty_like(old)
    hawk.run(logp_of, logits=logits, target=token, logp=logp, lse=lse)
    assert (logp - old).abs().max() < 1e-5                      # what was drawn has the probability the loss reads
    gain, loss = normal(S * T), torch.empty(1, device=gpu)
    x, mean, rstd, q, k, v, o, y, logits = layer()
    bar_logits = torch.empty_like(logits)
    hawk.run(loss_of, logits=logits, target=token, old_logp=old, advantage=gain, loss=loss, bar_logits=bar_logits)
    bar_y = (bar_logits @ wa.t()).view(S, T, C)
    bar_o = (bar_y @ wo.t()).view(S, T, H, V)
    bars = [torch.empty_like(p) for p in (q, k, v)]
    hawk.run(mix.vjp, q=q, k=k, v=v, decay=decay, bar_o=bar_o, bar_q=bars[0], bar_k=bars[1], bar_v=bars[2])
    bar_x = sum(b.reshape(S, T, -1) @ w.t() for b, w in zip(bars, (wq, wk, wv)))
    bar_w, bar_b, bar_u = torch.empty_like(weight), torch.empty_like(bias), torch.empty_like(u)
    hawk.run(norm.vjp, x=u, weight=weight, mean=mean, rstd=rstd, bar_y=bar_x, bar_x=bar_u, bar_weight=bar_w, bar_bias=bar_b)
    got = {"u": bar_u + bar_y, "weight": bar_w, "bias": bar_b, "wq": x.reshape(-1, C).t() @ bars[0].reshape(S * T, -1),
           "wv": x.reshape(-1, C).t() @ bars[2].reshape(S * T, -1)}
    # the same in float64 on the CPU, by autograd over the plain sums
    p = {n: t.double().cpu().requires_grad_() for n, t in dict(u=u, weight=weight, bias=bias, wq=wq, wk=wk, wv=wv, wo=wo, wa=wa).items()}
    xh = torch.nn.functional.layer_norm(p["u"], (C,), p["weight"], p["bias"])
    qq, kk, vv = ((xh @ p[n]).view(S, T, H, -1) for n in ("wq", "wk", "wv"))
    far = torch.arange(T)[:, None] - torch.arange(T)[None]
    power = torch.where(far >= 0, decay.double().cpu()[:, None, None] ** far.clamp(min=0), 0.0)
    oo = 0.5 * torch.einsum("sthk,sjhk,htj,sjhv->sthv", qq, kk, power, vv)
    ll = torch.log_softmax(((p["u"] + oo.reshape(S, T, -1) @ p["wo"]) @ p["wa"]).reshape(S * T, A), 1)
    ratio = torch.exp(ll.gather(1, token.cpu()[:, None])[:, 0] - old.double().cpu())
    A_ = gain.double().cpu()
    want = -torch.minimum(ratio * A_, ratio.clamp(0.8, 1.2) * A_).mean()
    want.backward()
    assert abs(float(loss) - float(want.detach())) < 1e-5
    for n, t in got.items():
        ref = p[n].grad
        assert (t.double().cpu() - ref).norm() < 1e-4 * ref.norm(), n
    # served a token at a time, greedily: the same logits
    state = torch.zeros(S, H, K, V, device=gpu)
    cold = stages.sample(temperature=0.0)
    for t in range(T):
        now = u[:, t:t + 1].contiguous()
        xt = torch.empty_like(now)
        hawk.run(norm, x=now, weight=weight, bias=bias, y=xt)
        q1, k1, v1 = ((xt @ w).view(S, 1, H, -1) for w in (wq, wk, wv))
        o1 = torch.empty_like(v1)
        hawk.run(mix, q=q1, k=k1, v=v1, decay=decay, o=o1, h0=state, last=state)
        one = ((now + o1.reshape(S, 1, -1) @ wo) @ wa).reshape(S, A)
        whole = logits.view(S, T, A)[:, t]
        assert (one - whole).abs().max() < 1e-4
        best = torch.empty(S, dtype=torch.int64, device=gpu)
        hawk.run(cold, logits=one, u=torch.zeros(S, device=gpu), token=best)
        assert (best == one.argmax(1)).all()


@pytest.mark.gpu
def test_the_stages_replayed_from_graphs_and_on_two_streams(gpu):
    """Each replay, with other work between, gives the eager call's bits; so do two streams at once."""
    import torch
    g = torch.Generator(device=gpu).manual_seed(9)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=gpu)
    q, k, v = normal(1, 1200, 2, 32), normal(1, 1200, 2, 32), normal(1, 1200, 2, 48)
    decay, x, w = torch.tensor([0.9, 0.99], device=gpu), normal(700, 300), normal(300)
    mean, rstd = x.mean(1), 1 / (x.var(1, correction=0) + 1e-5).sqrt()
    logits, u = normal(30, 20000), torch.rand(30, generator=g, device=gpu)
    mix, norm, pick = hawk.stages.linear_attention(), hawk.stages.layer_norm(), hawk.stages.sample(top_k=300, top_p=0.9)

    def calls(stream=None):
        out = dict(o=torch.empty_like(v), bar_q=torch.empty_like(q), bar_k=torch.empty_like(k), bar_v=torch.empty_like(v),
                   bar_weight=torch.empty_like(w), bar_bias=torch.empty_like(w), token=torch.empty(30, dtype=torch.int64, device=gpu),
                   logp=torch.empty(30, device=gpu))

        def go():
            hawk.run(mix, q=q, k=k, v=v, decay=decay, o=out["o"])
            hawk.run(mix.vjp, q=q, k=k, v=v, decay=decay, bar_o=v, bar_q=out["bar_q"], bar_k=out["bar_k"], bar_v=out["bar_v"])
            hawk.run(norm.vjp, x=x, weight=w, mean=mean, rstd=rstd, bar_y=x, bar_weight=out["bar_weight"], bar_bias=out["bar_bias"])
            hawk.run(pick, logits=logits, u=u, token=out["token"], logp=out["logp"])
        return out, go
    want, go = calls()
    go()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        out, go = calls()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            go()
        graphs.append((out, graph))
    for round_ in range(3):
        for out, _ in graphs:
            for t in out.values():
                t.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (out, graph), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager, go = calls()
        go()
        torch.cuda.synchronize()
        for out in (eager, *(o for o, _ in graphs)):
            for n in want:
                assert torch.equal(out[n], want[n]), (round_, n)
    # launchers, on streams of their own
    launchers = []
    for _ in range(2):
        s, o = torch.cuda.Stream(), torch.zeros_like(v)
        launchers.append((mix.prepare(q=q, k=k, v=v, decay=decay, o=o, stream=s), o))
    torch.cuda.synchronize()
    for launch, _ in launchers:
        launch()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want["o"]) for _, o in launchers)


@pytest.mark.gpu
def test_planes_whose_offsets_pass_32_bits(gpu):
    import torch
    # two tokens, 2^32 + 3 bytes and more apart
    far = (1 << 31) + 64
    room = torch.zeros(far + 4096, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(4)
    H, K = 1, 16
    vals = torch.randn(2, H, K, generator=g, device=gpu).to(torch.bfloat16)
    q = room.as_strided((1, 2, H, K), (1, far, K, 1))
    q.copy_(vals[None])
    decay = torch.tensor([0.5], device=gpu)
    o, want = torch.empty(1, 2, H, K, dtype=torch.bfloat16, device=gpu), torch.empty(1, 2, H, K, dtype=torch.bfloat16, device=gpu)
    stage = hawk.stages.linear_attention()
    hawk.run(stage, q=q, k=q, v=q, decay=decay, o=o)
    near = q.contiguous()
    hawk.run(stage, q=near, k=near, v=near, decay=decay, o=want)
    assert torch.equal(o, want)
    rows = room.as_strided((2, 2000), (far, 1))
    rows.copy_(torch.randn(2, 2000, generator=g, device=gpu))
    close_rows = rows.contiguous()
    y, wy = torch.empty_like(close_rows), torch.empty_like(close_rows)
    norm = hawk.stages.layer_norm()
    hawk.run(norm, x=rows, y=y)
    hawk.run(norm, x=close_rows, y=wy)
    assert torch.equal(y, wy)
    u, token, wt = torch.tensor([0.3, 0.8], device=gpu), *(torch.empty(2, dtype=torch.int64, device=gpu) for _ in range(2))
    hawk.run(hawk.stages.sample(top_p=0.9), logits=rows, u=u, token=token)
    hawk.run(hawk.stages.sample(top_p=0.9), logits=close_rows, u=u, token=wt)
    assert torch.equal(token, wt)


def test_options_out_of_range_are_refused():
    s = hawk.stages
    for bad in (-1.0, math.nan, math.inf, "1", True):
        with pytest.raises(HawkError, match="eps="):
            s.layer_norm(eps=bad)
    for bad in (math.nan, math.inf, None, True):
        with pytest.raises(HawkError, match="scale="):
            s.linear_attention(scale=bad)
    for name, values in (("temperature", (-0.1, math.nan, "a", True)), ("top_k", (-1, 1.5, True, 1 << 63)),
                         ("top_p", (-0.1, math.nan, None)), ("min_p", (math.nan, "x"))):
        for bad in values:
            with pytest.raises(HawkError, match=f"{name}="):
                s.sample(**{name: bad})
    with pytest.raises(HawkError, match="no derivative"):
        diff.vjp(s.sample())
    assert diff.vjp(s.layer_norm()).name == "layer_norm_vjp" and diff.vjp(s.linear_attention()).name == "linear_attention_vjp"


@pytest.mark.gpu
def test_planes_that_do_not_fit_are_refused(gpu):
    import torch
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=gpu)  # noqa: E731
    norm, mix, pick = hawk.stages.layer_norm(), hawk.stages.linear_attention(), hawk.stages.sample()
    x, d = z(4, 9), z(3)
    q, v = z(2, 5, 3, 4), z(2, 5, 3, 6)
    l, u = z(4, 9), z(4)
    t = torch.zeros(4, dtype=torch.int64, device=gpu)
    bad = [
        (norm, dict(x=x, y=z(4, 8)), "'y'"),
        (norm, dict(x=x.double(), y=x.double()), "float32"),
        (norm, dict(x=z(9, 4).t(), y=x.clone()), "contiguous"),
        (norm, dict(x=x, y=z(40).as_strided((4, 9), (5, 1))), "overlap"),
        (norm, dict(x=z(4, 3, 2, 9)[:, :2], y=z(4, 2, 2, 9)), "evenly apart"),
        (norm, dict(x=x, y=x.clone(), weight=z(8)), "'weight'"),
        (norm, dict(x=x, y=x.clone(), weight=z(9).half()), "'weight'"),
        (norm, dict(x=x.half(), y=x.half(), weight=z(9), bias=z(9).half()), "'bias'"),
        (norm, dict(x=x, y=x.clone(), mean=z(3)), "'mean'"),
        (norm, dict(x=x), "no output"),
        (norm.vjp, dict(x=x, bar_y=x, bar_x=x.clone(), mean=z(4)), "'rstd' is not given"),
        (norm.vjp, dict(x=x, bar_y=x, mean=z(4), rstd=z(4), bar_weight=z(9), weight=z(9).half()), "'weight'"),
        (mix, dict(q=q[0], k=q[0], v=v[0], decay=d, o=v[0].clone()), "offsets"),
        (mix, dict(q=q, k=z(2, 5, 3, 5), v=v, decay=d, o=v.clone()), "'k'"),
        (mix, dict(q=q, k=q, v=v, decay=z(2), o=v.clone()), "'decay'"),
        (mix, dict(q=q, k=q, v=v, decay=d.double(), o=v.clone()), "'decay'"),
        (mix, dict(q=q, k=q, v=v.half(), decay=d, o=v.clone()), "float16"),
        (mix, dict(q=z(2, 5, 3, 257), k=z(2, 5, 3, 257), v=v, decay=d, o=v.clone()), "256 channels"),
        (mix, dict(q=q, k=q, v=v[..., :0], decay=d, o=v[..., :0].clone()), "256 channels"),
        (mix, dict(q=q.transpose(1, 3).contiguous().transpose(1, 3), k=q, v=v, decay=d, o=v.clone()), "contiguous"),
        (mix, dict(q=q, k=q, v=v, decay=d, o=v), "one tensor"),
        (mix, dict(q=q, k=q, v=v, decay=d, o=v.clone(), h0=z(2, 3, 4, 5)), "state"),
        (mix, dict(q=q, k=q, v=v, decay=d, o=v.clone(), offsets=t), "packed planes"),
        (mix.vjp, dict(q=q, k=q, v=v, decay=d, bar_o=v, bar_q=q), "one tensor"),
        (mix.vjp, dict(q=q, k=q, v=v, decay=d, bar_o=v), "no output"),
        (mix, dict(q=q, k=q, v=v, decay=d, o=z(2, 5, 1, 6).expand(2, 5, 3, 6)), "repeats memory"),
        (pick, dict(logits=l.double(), u=u, token=t), "float32"),
        (pick, dict(logits=z(9, 4).t(), u=u, token=t), "contiguous"),
        (pick, dict(logits=l, u=z(3), token=t), "'u'"),
        (pick, dict(logits=l, u=u.half(), token=t), "'u'"),
        (pick, dict(logits=l, u=u, token=t.float()), "int32 or int64"),
        (pick, dict(logits=l, u=u, token=t[:3]), "'token'"),
        (pick, dict(logits=l, u=u, token=t, top_k=t), "'top_k'"),
        (pick, dict(logits=l, u=u, token=t, temperature=z(4).double()), "'temperature'"),
        (pick, dict(logits=l, u=u), "no output"),
        (pick, dict(logits=l, u=u, logp=u), "one tensor"),
        (pick, dict(logits=z(1).expand(2, (1 << 22) + 1), u=z(2), token=t[:2]), "2\\^22"),
    ]
    for stage, planes, text in bad:
        with pytest.raises(HawkError, match=text):
            hawk.run(stage, **planes)
        with pytest.raises(HawkError, match=text):
            stage.prepare(**planes)


def test_the_entries_refuse_bad_jobs():
    """The C entries check their jobs before any launch."""
    L = _core.lib()
    n = _core.LayerNormJob()
    n.rows, n.cols = 2, 5
    ref = ctypes.byref(n)
    assert L.hk_layer_norm(None, None, None) == 1 and L.hk_layer_norm_vjp(None, None, None) == 1
    assert L.hk_layer_norm(ref, None, None) == 1 and b"required" in L.hk_last_error()
    assert L.hk_layer_norm_vjp(ref, None, None) == 1 and b"required" in L.hk_last_error()
    n.x = n.bar_y = n.mean = n.rstd = n.bar_weight = 16
    assert L.hk_layer_norm_scratch_bytes(ref, 1) == 2 * 5 * 4 and L.hk_layer_norm_scratch_bytes(ref, 0) == 0
    assert L.hk_layer_norm_vjp(ref, None, None) == 1 and b"scratch" in L.hk_last_error()
    n.eps = -1.0
    assert L.hk_layer_norm(ref, None, None) == 1 and b"eps" in L.hk_last_error()
    n.eps, n.dtype = 0.0, 1
    assert L.hk_layer_norm(ref, None, None) == 1 and b"16-bit" in L.hk_last_error()
    n.dtype, n.weight_dtype = 2, 3
    assert L.hk_layer_norm(ref, None, None) == 1 and b"weights" in L.hk_last_error()
    n.weight_dtype, n.rows = 0, -1
    assert L.hk_layer_norm(ref, None, None) == 1 and b">= 0" in L.hk_last_error()
    n.rows = 0
    assert L.hk_layer_norm(ref, None, None) == 0
    a = _core.LinearAttentionJob()
    a.seqs, a.steps, a.heads, a.keys, a.values = 1, 4, 2, 8, 8
    ref = ctypes.byref(a)
    assert L.hk_linear_attention(None, None, None) == 1
    assert L.hk_linear_attention(ref, None, None) == 1 and b"missing" in L.hk_last_error()
    a.keys = 257
    assert L.hk_linear_attention(ref, None, None) == 1 and b"256" in L.hk_last_error()
    assert L.hk_linear_attention_scratch_bytes(ref, 0) == 0
    a.keys, a.dtype = 8, 1
    assert L.hk_linear_attention_vjp(ref, None, None) == 1 and b"16-bit" in L.hk_last_error()
    a.dtype, a.steps = 0, -1
    assert L.hk_linear_attention(ref, None, None) == 1 and b">= 0" in L.hk_last_error()
    a.steps, a.seqs = 4, 0
    assert L.hk_linear_attention(ref, None, None) == 0
    a.seqs, a.steps = 1, 100000
    for name in ("q", "k", "v", "o"):
        getattr(a, name).data = 16
    a.decay = 16
    assert L.hk_linear_attention_scratch_bytes(ref, 0) > 0
    assert L.hk_linear_attention(ref, None, None) == 1 and b"scratch" in L.hk_last_error()
    s = _core.SampleJob()
    s.rows, s.vocab = 2, 5
    ref = ctypes.byref(s)
    assert L.hk_sample(None, None, None) == 1
    assert L.hk_sample(ref, None, None) == 1 and b"required" in L.hk_last_error()
    s.vocab = (1 << 22) + 1
    assert L.hk_sample(ref, None, None) == 1 and b"2^22" in L.hk_last_error()
    s.vocab, s.dtype = 5, 1
    assert L.hk_sample(ref, None, None) == 1 and b"16-bit" in L.hk_last_error()
    s.dtype, s.rows = 0, 0
    assert L.hk_sample(ref, None, None) == 0


def test_the_jobs_are_laid_out_as_the_header_has_them():
    assert ctypes.sizeof(_core.LayerNormJob) == 10 * 8 + 6 * 8 + 4 * 4
    assert ctypes.sizeof(_core.SampleJob) == 8 * 8 + 4 * 8 + 3 * 8 + 4 * 4
    assert ctypes.sizeof(_core.HeadPlane) == 32
    assert ctypes.sizeof(_core.LinearAttentionJob) == 8 * 32 + 6 * 8 + 3 * 8 + 6 * 4
