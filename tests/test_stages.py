"""The training stages (``hawk.stages``) against plain loops in 64 bits.

Tolerances.  ``u`` is half an ulp of 1 in the arithmetic's type (2^-24, 2^-53
for float64), ``r`` half an ulp of 1 in the output's type (2^-8 for bfloat16, 2^-11
for float16).  A recurrence of T steps joins each step's term through at most T
products and sums, each with a relative error of at most u (a sigmoid gate's
own error is below 24 u for |z| <= 8), so its error is at most ``(c T + 16) u``
times the same recurrence of absolute values, c = 4 or 28; the output rounds
once, by r.  A row's log-sum-exp errs by 8 u (1 + |lse|) (its terms are joined in
a tree), and a gradient element by the exponent's absolute error, 16 u (1 + |l|),
times itself.
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import numpy as np
import pytest

import hawk_amd as hawk
from hawk_amd import HawkError, _core, diff

TYPES = ("float32", "bfloat16", "float16", "float64")
U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -24, "float16": 2.0 ** -24, "float64": 2.0 ** -53}
R = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float64": 2.0 ** -53}
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -25, "float64": 1e-300}


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


# -- the plain forms, in 64 bits -------------------------------------------------------------

def gates(gate, x, form):
    if form == "value":
        return gate, x
    a = np.where(gate >= 0, 1 / (1 + np.exp(-np.abs(gate))), np.exp(-np.abs(gate)) / (1 + np.exp(-np.abs(gate))))
    return a, (1 - a) * x


def loop(a, b, state):
    """``h_t = a_t h_{t-1} + b_t``, a gate of 0 cutting, over axis 0."""
    out = np.empty_like(b)
    for t in range(len(b)):
        state = np.where(a[t] == 0, b[t], a[t] * state + b[t])
        out[t] = state
    return out, state


def spans(S, T, offsets):
    if offsets is None:
        return [(s, slice(0, T)) for s in range(S)]
    return [(s, slice(int(offsets[s]), int(offsets[s + 1]))) for s in range(len(offsets) - 1)]


def take(x, s, rows, packed):
    return x[rows] if packed else x[s][rows]


def oracle_forward(gate, x, h0, offsets, form, reverse):
    packed = offsets is not None
    S = len(offsets) - 1 if packed else gate.shape[0]
    C = gate.shape[-1]
    h, scale = np.zeros_like(x), np.zeros_like(x)
    last = np.zeros((S, C))
    for s, rows in spans(S, gate.shape[-2], offsets):
        a, b = gates(take(gate, s, rows, packed), take(x, s, rows, packed), form)
        if reverse:
            a, b = a[::-1], b[::-1]
        start = np.zeros(C) if h0 is None else h0[s]
        out, last[s] = loop(a, b, start)
        size, _ = loop(np.abs(a), np.abs(b), np.abs(start))
        if reverse:
            out, size = out[::-1], size[::-1]
        take(h, s, rows, packed)[:] = out
        take(scale, s, rows, packed)[:] = size
    return h, last, scale


def oracle_vjp(gate, x, h, h0, bar_h, bar_last, offsets, form, reverse):
    packed = offsets is not None
    S = len(offsets) - 1 if packed else gate.shape[0]
    C = gate.shape[-1]
    bar_gate, bar_x = np.zeros_like(gate), np.zeros_like(gate)
    size_gate, size_x = np.zeros_like(gate), np.zeros_like(gate)
    bar_h0, size_0 = np.zeros((S, C)), np.zeros((S, C))
    for s, rows in spans(S, gate.shape[-2], offsets):
        g, xs = take(gate, s, rows, packed), take(x, s, rows, packed) if x is not None else None
        hs, bs = take(h, s, rows, packed), take(bar_h, s, rows, packed)
        a, _ = gates(g, xs if xs is not None else g, form)
        order = range(len(g))
        order = list(order) if reverse else list(reversed(order))
        carry = np.zeros(C) if bar_last is None else bar_last[s]
        mass = np.abs(carry)
        for i, t in enumerate(order):
            before = order[i + 1] if i + 1 < len(order) else None
            prior = hs[before] if before is not None else (np.zeros(C) if h0 is None else h0[s])
            G, m = bs[t] + carry, np.abs(bs[t]) + mass
            if form == "sigmoid":
                bg, bx = G * (prior - xs[t]) * a[t] * (1 - a[t]), (1 - a[t]) * G
                mg, mx = m * (np.abs(prior) + np.abs(xs[t])) * a[t] * (1 - a[t]), (1 - a[t]) * m
            else:
                bg, bx, mg, mx = G * prior, G, m * np.abs(prior), m
            take(bar_gate, s, rows, packed)[t], take(bar_x, s, rows, packed)[t] = bg, bx
            take(size_gate, s, rows, packed)[t], take(size_x, s, rows, packed)[t] = mg, mx
            carry, mass = np.where(a[t] == 0, 0, a[t] * G), np.abs(a[t]) * m
        bar_h0[s], size_0[s] = carry, mass
    return (bar_gate, bar_x, bar_h0), (size_gate, size_x, size_0)


def close(got, want, size, T, form, dtype, state=False):
    c = 28 if form == "sigmoid" else 4
    r = U[dtype] if state else R[dtype]
    bound = ((c * T + 16) * U[dtype] + r) * size * (1 + 2 * r) + TINY["float64" if state else dtype]
    assert np.isfinite(got).all()
    worst = np.abs(got - want) - bound
    assert (worst <= 0).all(), f"off by {np.abs(got - want).max()} where {bound[np.unravel_index(worst.argmax(), worst.shape)]} is allowed"


def recurrence_case(S, T, C, dtype, form, reverse, layout, state, packed, device, seed=0):
    g = np.random.default_rng([seed, S, T, C])
    shape = (T, C) if packed else (S, T, C)
    gate = g.normal(size=shape) + 1.0 if form == "sigmoid" else 1 / (1 + np.exp(-g.normal(size=shape) - 2))
    if form == "value":
        gate *= g.random(shape) > 0.03
        gate = np.where(g.random(shape) < 0.1, -gate, gate)
    offsets = None
    if packed:
        cut = np.sort(g.integers(0, T + 1, S - 1)) if S > 1 else np.array([], int)
        if S >= 4:
            cut[1] = cut[0]
            cut[-1] = T
        offsets = np.concatenate([[0], cut, [T]])
    got, held = {}, {}

    def put(name, x):
        t, held[name] = plane(x, dtype, device)
        if layout == "steps":
            t = t.transpose(-1, -2).contiguous().transpose(-1, -2)
        elif layout == "sliced":                                # odd strides, odd alignment
            import torch
            wide = torch.zeros((*t.shape[:-1], t.shape[-1] + 3), dtype=t.dtype, device=device)
            wide[..., 1:1 + t.shape[-1]] = t
            t = wide[..., 1:1 + t.shape[-1]]
        elif layout == "scattered":                             # neither axis contiguous
            import torch
            wide = torch.zeros((*t.shape[:-2], 2 * t.shape[-2], 2 * t.shape[-1]), dtype=t.dtype, device=device)
            wide[..., ::2, ::2] = t
            t = wide[..., ::2, ::2]
        got[name] = t
    for n in ("gate", "x", "bar_h"):
        put(n, gate if n == "gate" else g.normal(size=shape))
    sd = "float64" if dtype == "float64" else "float32"
    if state:
        for n in ("h0", "bar_last"):
            got[n], held[n] = plane(g.normal(size=(S, C)), sd, device)
    return got, held, offsets


SHAPES = [(1, 1, 1), (3, 1, 5), (2, 2, 8), (1, 7, 64), (5, 33, 9), (2, 129, 24), (3, 300, 1), (1, 1025, 40),
          (1, 2500, 3), (70, 5, 2), (2, 640, 513)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["value", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_recurrence_and_its_derivative_are_the_loop(gpu, shape, dtype, form):
    import torch
    S, T, C = shape
    for k, (layout, reverse, state, packed) in enumerate([
            ("channels", False, True, False), ("steps", True, True, False), ("sliced", True, False, False),
            ("steps", False, False, False), ("channels", False, True, True), ("sliced", True, True, True),
            ("scattered", False, True, False)]):
        print(shape, dtype, form, layout, reverse, state, packed, flush=True)
        got, held, offsets = recurrence_case(S, T, C, dtype, form, reverse, layout, state, packed, gpu, seed=k)
        stage = hawk.stages.recurrence(gate=form, reverse=reverse)
        planes = {n: got[n] for n in ("gate", "x", "h0") if n in got}
        if packed:
            planes["offsets"] = torch.from_numpy(offsets).to(gpu, torch.int64 if k % 2 else torch.int32)
        h = torch.empty_like(got["x"])
        last = torch.empty_like(got["h0"]) if state else None
        hawk.run(stage, h=h, last=last, **planes)
        want, want_last, size = oracle_forward(held["gate"], held["x"], held.get("h0"), offsets, form, reverse)
        close(back(h), want, size, T, form, dtype)
        if state:
            mass = np.abs(want_last) + (np.abs(size).max() if size.size else 0) + np.abs(held["h0"])
            close(back(last), want_last, mass, T, form, dtype, state=True)
        # the derivative, of the h the forward wrote
        bars = {n: torch.empty_like(got["x"]) for n in ("bar_gate", "bar_x")}
        if state:
            bars["bar_h0"] = torch.empty_like(got["h0"])
            planes["bar_last"] = got["bar_last"]
        hawk.run(stage.vjp, h=h, bar_h=got["bar_h"], **planes, **bars)
        wants, sizes = oracle_vjp(held["gate"], held["x"], back(h), held.get("h0"), held["bar_h"],
                                  held.get("bar_last"), offsets, form, reverse)
        for n, w, z in zip(("bar_gate", "bar_x", "bar_h0"), wants, sizes):
            if n in bars:
                close(back(bars[n]), w, z, T, form, dtype, state=n == "bar_h0")


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["value", "sigmoid"])
def test_the_recurrences_derivative_is_its_difference_quotient(gpu, form):
    """Central differences of sum(w h) + sum(v last) in float64: an error of e^2 / 6 times the third
    derivative and of 1e-16 / e from rounding, so 1e-8 at e = 1e-5 for sums of order 1."""
    import torch
    g = np.random.default_rng(7)
    S, T, C = 2, 19, 3
    base = {"gate": g.uniform(0.2, 0.9, (S, T, C)) if form == "value" else g.normal(size=(S, T, C)),
            "x": g.normal(size=(S, T, C)), "h0": g.normal(size=(S, C))}
    w, v = g.normal(size=(S, T, C)), g.normal(size=(S, C))
    stage = hawk.stages.recurrence(gate=form)

    def forward(values):
        t = {n: torch.from_numpy(x).to(gpu) for n, x in values.items()}
        h, last = torch.empty_like(t["x"]), torch.empty_like(t["h0"])
        hawk.run(stage, h=h, last=last, **t)
        return h, last
    h, _ = forward(base)
    bars = {"bar_" + n: torch.empty_like(torch.from_numpy(x)).to(gpu) for n, x in base.items()}
    hawk.run(diff.vjp(stage), **{n: torch.from_numpy(x).to(gpu) for n, x in base.items()}, h=h,
             bar_h=torch.from_numpy(w).to(gpu), bar_last=torch.from_numpy(v).to(gpu), **bars)
    e = 1e-5
    for n in base:
        for index in [tuple(g.integers(0, d) for d in base[n].shape) for _ in range(8)]:
            ends = []
            for sign in (1, -1):
                moved = {m: x.copy() for m, x in base.items()}
                moved[n][index] += sign * e
                hh, ll = forward(moved)
                ends.append((back(hh) * w).sum() + (back(ll) * v).sum())
            slope = (ends[0] - ends[1]) / (2 * e)
            assert abs(slope - back(bars["bar_" + n])[index]) < 1e-7 * (1 + abs(slope)), (n, index)


@pytest.mark.gpu
def test_a_gate_of_zero_and_a_sequences_start_cut_infinities_and_nan(gpu):
    import torch
    T = 700
    for C, layout in ((1, "steps"), (16, "channels")):
        x = torch.randn(1, T, C, device=gpu)
        gate = torch.full_like(x, 0.5)
        x[0, 100] = math.nan
        x[0, 300] = math.inf
        gate[0, 200] = 0.0
        gate[0, 301] = 0.0
        h = torch.empty_like(x)
        hawk.run(hawk.stages.recurrence(), gate=gate, x=x, h=h)
        assert torch.isnan(h[0, 100:200]).all() and torch.isfinite(h[0, :100]).all()
        assert torch.isfinite(h[0, 200:300]).all() and torch.isinf(h[0, 300]).all() and torch.isfinite(h[0, 301:]).all()
        want, _, _ = oracle_forward(back(gate[:, 200:300]), back(x[:, 200:300]), None, None, "value", False)
        assert np.abs(back(h[:, 200:300]) - want).max() < 1e-5
        # the same through packed sequences: nothing crosses a bound
        gate.fill_(0.5)
        offsets = torch.tensor([0, 200, 200, 301, T], device=gpu)
        for reverse in (False, True):
            hp = torch.empty(T, C, device=gpu)
            hawk.run(hawk.stages.recurrence(reverse=reverse), gate=gate[0].contiguous(), x=x[0].contiguous(), h=hp,
                     offsets=offsets)
            assert torch.isfinite(hp[301:]).all() and torch.isfinite(hp[200:300] if not reverse else hp[101:200]).all()
            assert torch.isnan(hp[100]).all()
        # a NaN gate is not lost where the state is 0
        z = torch.zeros_like(x)
        gate[0, 5] = math.nan
        hawk.run(hawk.stages.recurrence(), gate=gate, x=z, h=h)
        assert torch.isnan(h[0, 5:]).all() and (h[0, :5] == 0).all()


def far_gates(T, dtype, sign, seed):
    """Gates that grow for a while and shrink for as long, (T, 1): a run's product passes the type's largest number,
    or its least, while a state that starts low stays an ordinary number.  With the number it starts from."""
    octaves, every = (1600, 1) if dtype == "float64" else (200, 1 if T < 3000 else 8)
    t = np.arange(T)
    gate = np.where(t % every == 0, np.where(t // (octaves * every) % 2 == 0, 2.0, 0.5), 1.0)
    if sign:
        gate = gate * np.where(np.random.default_rng(seed).random(T) < 0.5, -1, 1)
    return gate[:, None], 2.0 ** (-octaves / 2)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["channels", "steps", "sliced", "packed"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float64"])
@pytest.mark.parametrize("T,C", [(190, 16), (700, 40), (3500, 3), (9001, 8), (12001, 1)], ids=str)
def test_gates_whose_product_leaves_the_types_range(gpu, T, C, dtype, layout):
    """The states are ordinary numbers throughout, so the bounds are those of any recurrence."""
    import torch
    packed = layout == "packed"
    for k, (sign, reverse) in enumerate([(False, False), (True, True), (True, False)]):
        print(T, C, dtype, layout, sign, reverse, flush=True)
        got, held, offsets = recurrence_case(1 if not packed else 2, T, C, dtype, "value", reverse,
                                             "channels" if packed else layout, True, packed, gpu, seed=60 + k)
        low = far_gates(T, dtype, sign, k)[1]
        gate = np.tile(far_gates(T, dtype, sign, k)[0], (1, C))
        if packed:                                             # both sequences start where the gates grow
            offsets = np.array([0, T - 150, T])
            gate = np.concatenate([gate[:T - 150], gate[:150]])
            more = gate[T - 150:]
            gate = np.concatenate([gate[:T - 150][::-1], more[::-1]]) if reverse else gate
        elif reverse:
            gate = gate[::-1]
        g, held["gate"] = plane(np.ascontiguousarray(gate if packed else gate[None]), dtype, gpu)
        got["gate"].copy_(g)
        for n in ("x", "h0"):
            t, held[n] = plane(held[n] * low, dtype if n == "x" else "float64" if dtype == "float64" else "float32", gpu)
            got[n].copy_(t)
        planes = {n: got[n] for n in ("gate", "x", "h0")}
        if packed:
            planes["offsets"] = torch.from_numpy(offsets).to(gpu)
        stage = hawk.stages.recurrence(reverse=reverse)
        h, last = torch.empty_like(got["x"]), torch.empty_like(got["h0"])
        hawk.run(stage, h=h, last=last, **planes)
        want, want_last, size = oracle_forward(held["gate"], held["x"], held["h0"], offsets, "value", reverse)
        close(back(h), want, size, T, "value", dtype)
        ends = np.array([np.abs(size[rows if packed else (0, rows)]).max(0) for _, rows in spans(1, T, offsets)])
        close(back(last), want_last, ends, T, "value", dtype, state=True)
        # the derivative: adjoints that start low where the gates grow in its direction
        stage = hawk.stages.recurrence(reverse=not reverse)
        bars = {n: torch.empty_like(got["x"]) for n in ("bar_gate", "bar_x")}
        bars["bar_h0"] = torch.empty_like(got["h0"])
        saved, held_h = plane(np.random.default_rng(k).normal(size=held["x"].shape), dtype, gpu)
        hawk.run(stage.vjp, gate=got["gate"], h=saved, bar_h=got["x"], bar_last=got["h0"], h0=torch.ones_like(last),
                 **{n: planes[n] for n in ("offsets",) if packed}, **bars)
        wants, sizes = oracle_vjp(held["gate"], None, held_h, np.ones_like(held["h0"]), held["x"], held["h0"], offsets,
                                  "value", not reverse)
        for n, w, z in zip(("bar_gate", "bar_x", "bar_h0"), wants, sizes):
            close(back(bars[n]), w, z, T, "value", dtype, state=n == "bar_h0")


@pytest.mark.gpu
@pytest.mark.parametrize("T,C,layout", [(200, 16, "channels"), (300, 1, "steps"), (9000, 8, "channels"), (9000, 2, "steps")],
                         ids=str)
def test_large_and_infinite_states_through_many_small_gates(gpu, T, C, layout):
    import torch

    def put(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "steps" else x
    zero, h = put(torch.zeros(1, T, C, device=gpu)), put(torch.empty(1, T, C, device=gpu))
    sign = torch.where(torch.arange(T, device=gpu) % 2 == 0, -1.0, 1.0)[None, :, None].expand(1, T, C)
    steps = torch.arange(1, T + 1, device=gpu, dtype=torch.float64)[None, :, None]
    for stage, gate in ((hawk.stages.recurrence(), torch.full_like(zero, -0.5)),
                        (hawk.stages.recurrence("sigmoid"), torch.zeros_like(zero))):
        alternating = stage.gate == "value"
        # halved exactly while it is a normal number, gone below the least: no floor that a product is held at
        hawk.run(stage, gate=put(gate), x=zero, h=h, h0=torch.full((1, C), 1e35, device=gpu))
        want = float(torch.tensor(1e35)) * 0.5 ** steps * (sign if alternating else 1.0)
        u = 2.0 ** -24 * (4 if alternating else 28 * T)
        assert ((h.double() - want).abs() <= u * want.abs() + 2.0 ** -149).all()
        # an infinity stays one, of the sign that the gates give it
        hawk.run(stage, gate=put(gate), x=zero, h=h, h0=torch.full((1, C), math.inf, device=gpu))
        assert torch.equal(h, put(torch.full_like(zero, math.inf) * (sign if alternating else 1.0)))
        bar = put(torch.empty_like(zero))
        hawk.run(stage.vjp, gate=put(gate), x=zero, h=put(torch.ones_like(zero)), bar_h=zero, bar_x=bar,
                 bar_last=torch.full((1, C), math.inf, device=gpu))
        assert torch.isinf(bar).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["channels", "steps"])
@pytest.mark.parametrize("T,C", [(7, 16), (100, 16), (5000, 3)], ids=str)
def test_gates_below_the_least_normal_number(gpu, T, C, layout):
    """A gate of few bits is the number it holds, in a thread's own steps and in the products that are joined."""
    import torch

    def put(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "steps" else x
    gate = torch.ones(1, T, C, device=gpu)
    gate[0, T // 2], gate[0, T // 2 + 1] = 1e-40, -3e35
    x, h, h0 = put(torch.zeros_like(gate)), put(torch.empty_like(gate)), torch.full((1, C), 1e35, device=gpu)
    hawk.run(hawk.stages.recurrence(), gate=put(gate), x=x, h=h, h0=h0)
    want = h0.double() * torch.cumprod(gate.double(), 1)
    assert ((h.double() - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()
    bar = put(torch.empty_like(gate))
    hawk.run(hawk.stages.recurrence(reverse=True).vjp, gate=put(gate), h=x, bar_h=x, bar_last=h0, bar_x=bar)
    want = torch.cat([h0.double()[:, None], want[:, :-1]], 1)            # the adjoint before each step's gate
    assert ((bar.double() - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,C", [(1, 16), (8, 5), (40, 16), (9000, 8)], ids=str)
def test_a_sigmoid_gate_below_the_least_number_cuts_in_every_form(gpu, T, C):
    """sigma(-100) is no float32 of full precision and sigma(-inf) is 0: neither lets the state pass, dense or packed."""
    import torch
    x = torch.randn(1, T, C, device=gpu)
    gate = torch.randn(1, T, C, device=gpu)
    h0 = torch.full((1, C), math.inf, device=gpu)
    stage, offsets = hawk.stages.recurrence("sigmoid"), torch.tensor([0, T], device=gpu)
    for low in (-100.0, -math.inf):
        for at in sorted({0, T // 2, T - 1}):
            z = gate.clone()
            z[0, at] = low
            h, p = torch.empty_like(x), torch.empty(T, C, device=gpu)
            hawk.run(stage, gate=z, x=x, h=h, h0=h0)
            hawk.run(stage, gate=z[0], x=x[0], h=p, h0=h0, offsets=offsets)
            for got in (h, p[None]):
                assert torch.isinf(got[0, :at]).all()
                want, _, size = oracle_forward(back(z[:, at:]), back(x[:, at:]), None, None, "sigmoid", False)
                close(back(got[:, at:]), want, size, T - at, "sigmoid", "float32")
            # the adjoint that would pass the cut, in both forms
            bars = [torch.empty_like(x), torch.empty(T, C, device=gpu)]
            hawk.run(stage.vjp, gate=z, x=x, h=h.nan_to_num(posinf=0, neginf=0), bar_h=torch.zeros_like(x), bar_last=h0, bar_x=bars[0])
            hawk.run(stage.vjp, gate=z[0], x=x[0], h=p.nan_to_num(posinf=0, neginf=0), bar_h=torch.zeros(T, C, device=gpu), bar_last=h0,
                     bar_x=bars[1], offsets=offsets)
            for got in (bars[0][0], bars[1]):
                assert torch.isinf(got[at:]).all() and (got[:at] == 0).all()


@pytest.mark.gpu
def test_one_token_at_a_time_is_the_whole_sequence(gpu):
    import torch
    S, T, C = 5, 37, 130
    g = torch.Generator(device=gpu).manual_seed(3)
    z, x = (torch.randn(S, T, C, generator=g, device=gpu) for _ in range(2))
    stage = hawk.stages.recurrence(gate="sigmoid")
    whole = torch.empty_like(x)
    hawk.run(stage, gate=z, x=x, h=whole)
    state = torch.zeros(S, C, device=gpu)
    one = torch.empty(S, 1, C, device=gpu)
    for t in range(T):
        hawk.run(stage, gate=z[:, t:t + 1], x=x[:, t:t + 1], h=one, h0=state, last=state)      # in place
        assert (one[:, 0] - whole[:, t]).abs().max() <= 64 * 2.0 ** -24 * (1 + whole[:, t].abs().max())
        assert torch.equal(one[:, 0], state)


@pytest.mark.gpu
def test_recurrences_in_place_replayed_and_on_two_streams(gpu):
    import torch
    S, T, C = 3, 1500, 72
    g = torch.Generator(device=gpu).manual_seed(4)
    gate = torch.rand(S, T, C, generator=g, device=gpu).bfloat16()
    x = torch.randn(S, T, C, generator=g, device=gpu).bfloat16()
    stage = hawk.stages.recurrence()
    want = torch.empty_like(x)
    hawk.run(stage, gate=gate, x=x, h=want)
    held = x.clone()
    hawk.run(stage, gate=gate, x=held, h=held)
    assert torch.equal(held, want)
    # the same bits whatever stream, and however many run at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(x) for _ in range(8)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for k, out in enumerate(outs):
        hawk.run(stage, gate=gate, x=x, h=out, stream=streams[k % 2])
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
    # a captured call
    h = torch.empty_like(x)
    launch = stage.prepare(gate=gate, x=x, h=h)
    launch()
    torch.cuda.synchronize()
    assert torch.equal(h, want)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        captured = stage.prepare(gate=gate, x=x, h=h, stream=side)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured()
    other = torch.randn_like(x)
    for k in range(4):
        x.copy_(other * (k + 1))
        h.zero_()
        graph.replay()
        eager = torch.empty_like(x)
        hawk.run(stage, gate=gate, x=x, h=eager)
        torch.cuda.synchronize()
        assert torch.equal(h, eager)


def test_states_written_over_those_that_enter_have_room_for_a_copy():
    L = _core.lib()
    for steps, offsets, copied in ((4, None, False), (4, 8, True), (5000, None, True), (5000, 8, True)):
        for vjp, names in ((0, ("h0", "last")), (1, ("bar_last", "bar_h0"))):
            job = _core.RecurrenceJob()
            job.seqs, job.steps, job.chans, job.offsets = 3, steps, 72, offsets
            for n in ("gate", "x", "h", "bar_h", "bar_gate", "bar_x"):
                plane = getattr(job, n)
                plane.data, plane.seq, plane.step, plane.chan = 8, 72 * steps, 72, 1
            without = L.hk_recurrence_scratch_bytes(ctypes.byref(job), vjp)
            setattr(job, names[0], 8)
            assert L.hk_recurrence_scratch_bytes(ctypes.byref(job), vjp) == without
            setattr(job, names[1], 8)
            assert L.hk_recurrence_scratch_bytes(ctypes.byref(job), vjp) == without + copied * 4 * 3 * 72


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("T", [40, 2500, 9000])
def test_states_may_be_written_over_those_that_enter(gpu, T, dtype, packed):
    """The bits of a call whose states that leave have a tensor of their own."""
    import torch
    S, C, d = 3, 72, getattr(torch, dtype)
    g = torch.Generator(device=gpu).manual_seed(T)
    shape = (T, C) if packed else (S, T, C)
    gate = 0.9 + 0.1 * torch.rand(shape, generator=g, device=gpu, dtype=d)
    x, bar = (torch.randn(shape, generator=g, device=gpu, dtype=d) for _ in range(2))
    h0 = torch.randn(S, C, generator=g, device=gpu, dtype=d)
    more = dict(offsets=torch.tensor([0, 13, T - 5, T], device=gpu)) if packed else {}
    stage = hawk.stages.recurrence()
    want, last, to_gate, to_x, to_h0 = (torch.empty_like(y) for y in (x, h0, x, x, h0))
    hawk.run(stage, gate=gate, x=x, h=want, h0=h0, last=last, **more)
    hawk.run(stage.vjp, gate=gate, h=want, bar_h=bar, h0=last, bar_last=h0, bar_gate=to_gate, bar_x=to_x, bar_h0=to_h0, **more)
    for _ in range(4):
        h, a, b = (torch.full_like(x, float("nan")) for _ in range(3))
        state = h0.clone()
        hawk.run(stage, gate=gate, x=x, h=h, h0=state, last=state, **more)
        assert torch.equal(h, want) and torch.equal(state, last)
        state = h0.clone()
        hawk.run(stage.vjp, gate=gate, h=want, bar_h=bar, h0=last, bar_last=state, bar_gate=a, bar_x=b, bar_h0=state, **more)
        assert torch.equal(a, to_gate) and torch.equal(b, to_x) and torch.equal(state, to_h0)
    state = h0.clone()
    launch = stage.prepare(gate=gate, x=x, h=h, h0=state, last=state, **more)
    launch()
    assert torch.equal(h, want) and torch.equal(state, last)


@pytest.mark.gpu
def test_recurrence_without_steps_sequences_or_channels(gpu):
    import torch
    stage = hawk.stages.recurrence()
    h0 = torch.randn(3, 5, device=gpu)
    last = torch.empty_like(h0)
    e = torch.empty(3, 0, 5, device=gpu)
    hawk.run(stage, gate=e, x=e.clone(), h=e.clone(), h0=h0, last=last)
    assert torch.equal(last, h0)
    bar = torch.empty_like(h0)
    hawk.run(stage.vjp, gate=e, h=e.clone(), bar_h=e.clone(), bar_last=h0, bar_h0=bar)
    assert torch.equal(bar, h0)
    p = torch.empty(0, 5, device=gpu)
    last.zero_()
    hawk.run(stage, gate=p, x=p.clone(), h=p.clone(), h0=h0, last=last,
             offsets=torch.zeros(4, dtype=torch.int32, device=gpu))
    assert torch.equal(last, h0)
    for shape in ((0, 4, 5), (3, 4, 0)):
        e = torch.empty(shape, device=gpu)
        hawk.run(stage, gate=e, x=e.clone(), h=e.clone())


# -- rows of logits --------------------------------------------------------------------------

ROW_TYPES = ("float32", "bfloat16", "float16")
ROWS = [(1, 1), (3, 2), (7, 33), (64, 48), (5, 257), (2, 1000), (9, 1024), (3, 4097), (2, 32768), (3, 50001), (1, 140001)]


def rows_case(N, V, dtype, device, seed=0, masked=True, strided=False):
    import torch
    g = np.random.default_rng([seed, N, V])
    logits, held = plane(g.normal(size=(N, V)) * 3, dtype, device)
    if strided:
        wide = torch.zeros((N, V + 5), dtype=logits.dtype, device=device)
        wide[:, 3:3 + V] = logits
        logits = wide[:, 3:3 + V]
    target = g.integers(0, V, N)
    if masked and N >= 3:
        target[1] = -1
        target[N - 1] = -100
    return logits, held, target


def oracle_rows(held, target, scale):
    l = held * scale
    top = l.max(1)
    lse = top + np.log(np.exp(l - top[:, None]).sum(1))
    kept = target >= 0
    logp = l[np.arange(len(l)), np.maximum(target, 0)] - lse
    return np.where(kept, logp, 0), np.where(kept, lse, 0), l


def oracle_gradient(l, target, lse, c, scale):
    kept = target >= 0
    p = np.exp(l - lse[:, None])
    grad = -c[:, None] * p
    grad[np.arange(len(l)), np.maximum(target, 0)] += c
    size = np.abs(c)[:, None] * p
    size[np.arange(len(l)), np.maximum(target, 0)] += np.abs(c)
    return np.where(kept[:, None], grad * scale, 0), size * scale


def close_row(got, want, lse):
    assert (np.abs(got - want) <= 8 * 2.0 ** -24 * (2 + np.abs(lse) + np.abs(want))).all(), np.abs(got - want).max()


def close_gradient(got, want, size, l, lse, dtype, slack=0.0):
    reach = 16 * 2.0 ** -24 * (1 + np.abs(l) + np.abs(lse[:, None])) + slack
    bound = size * (reach + R[dtype] * (1 + reach)) + TINY[dtype]
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) - bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ROW_TYPES)
@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_token_logp_and_its_derivative(gpu, shape, dtype):
    import torch
    N, V = shape
    for k, (scale, strided, wide) in enumerate([(1.0, False, True), (0.7, True, False)]):
        print(shape, dtype, scale, strided, flush=True)
        logits, held, target = rows_case(N, V, dtype, gpu, k, strided=strided)
        y = torch.from_numpy(target).to(gpu, torch.int64 if wide else torch.int32)
        logp, lse = torch.empty(N, device=gpu), torch.empty(N, device=gpu)
        stage = hawk.stages.token_logp(scale=scale)
        hawk.run(stage, logits=logits, target=y, logp=logp, lse=lse)
        want, want_lse, l = oracle_rows(held, target, scale)
        close_row(back(logp), want, want_lse)
        close_row(back(lse), want_lse, want_lse)
        c = np.random.default_rng(k).normal(size=N).astype(np.float32)
        bar = torch.empty_like(logits)
        hawk.run(stage.vjp, logits=logits, target=y, lse=lse, bar_logp=torch.from_numpy(c).to(gpu), bar_logits=bar)
        grad, size = oracle_gradient(l, target, back(lse), c.astype(np.float64), scale)
        close_gradient(back(bar), grad, size, l, back(lse), dtype)
        # in place, and only logp
        again = torch.empty(N, device=gpu)
        hawk.run(stage, logits=logits, target=y, logp=again)
        assert torch.equal(again, logp)
        hawk.run(stage.vjp, logits=logits, target=y, lse=lse, bar_logp=torch.from_numpy(c).to(gpu), bar_logits=logits)
        assert torch.equal(logits, bar)


def oracle_policy(logp, target, old, A, ref, weight, clip, kl, bar):
    kept = target >= 0
    r = np.exp(logp - old)
    plain, clipped = r * A, np.clip(r, 1 - clip[0], 1 + clip[1]) * A
    loss, slope = -np.minimum(plain, clipped), np.where(plain <= clipped, -plain, 0.0)
    if kl:
        d = ref - logp
        loss, slope = loss + kl * (np.expm1(d) - d), slope - kl * np.expm1(d)
    return np.where(kept, loss * weight, 0), np.where(kept, slope * weight * bar, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kl", [0.0, 0.1])
@pytest.mark.parametrize("dtype", ROW_TYPES)
@pytest.mark.parametrize("shape", ROWS, ids=str)
def test_policy_loss_and_its_gradient_in_one_pass_and_two(gpu, shape, dtype, kl):
    import torch
    N, V = shape
    print(shape, dtype, kl, flush=True)
    clip, scale = (0.2, 0.3), 0.9
    logits, held, target = rows_case(N, V, dtype, gpu, 5, strided=True)
    logp64, lse64, l = oracle_rows(held, target, scale)
    g = np.random.default_rng([11, N, V])
    f32 = lambda x: np.asarray(x, dtype=np.float32)  # noqa: E731
    old, ref = f32(logp64 + 0.3 * g.normal(size=N)), f32(logp64 + 0.3 * g.normal(size=N))
    A, weight = f32(g.normal(size=N)), f32(g.uniform(0.5, 1.5, N) / N)
    y = torch.from_numpy(target).to(gpu)
    dev = {n: torch.from_numpy(v).to(gpu) for n, v in (("old_logp", old), ("ref_logp", ref), ("advantage", A),
                                                       ("weight", weight))}
    out = {n: torch.empty(k, device=gpu) for n, k in (("loss", 1), ("logp", N), ("lse", N))}
    stage = hawk.stages.policy_loss(clip=clip, kl=kl, scale=scale)
    bar, cell = torch.empty_like(logits), torch.tensor([1.5], device=gpu)
    hawk.run(stage, logits=logits, target=y, bar_logits=bar, bar_loss=cell, **dev, **out)
    close_row(back(out["logp"]), logp64, lse64)
    close_row(back(out["lse"]), lse64, lse64)
    # the loss and slope of the log-probability that was written: a row near a bound of the ratio
    # may fall on either side of it by an ulp of logp, so the slopes are the written logp's
    logp = back(out["logp"])
    loss, slope = oracle_policy(logp, target, *(v.astype(np.float64) for v in (old, A, ref, weight)), clip, kl, 1.5)
    mass = np.abs(loss).sum() + np.abs(weight).sum() * (1 + np.abs(A).max())
    assert abs(back(out["loss"])[0] - loss.sum()) <= 32 * 2.0 ** -24 * mass
    edge = np.isclose(np.exp(logp - old), 1 - clip[0], atol=1e-6) | np.isclose(np.exp(logp - old), 1 + clip[1], atol=1e-6)
    assert not edge.any()
    grad, size = oracle_gradient(l, target, back(out["lse"]), slope, scale)
    big = oracle_gradient(l, target, back(out["lse"]), 1.5 * weight * (np.abs(A) * 2 + 4 * kl), scale)[1]
    close_gradient(back(bar), grad, np.maximum(size, big), l, back(out["lse"]), dtype)
    two = torch.empty_like(logits)
    saved = {n: out[n] for n in ("logp", "lse")}
    hawk.run(stage.vjp, logits=logits, target=y, bar_logits=two, bar_loss=cell, **dev, **saved)
    close_gradient(back(two), grad, np.maximum(size, big), l, back(out["lse"]), dtype)
    # the loss alone, and the mean where no weight is given
    alone = torch.empty(1, device=gpu)
    hawk.run(stage, logits=logits, target=y, loss=alone, **dev)
    assert torch.equal(alone, out["loss"])
    del dev["weight"]
    hawk.run(stage, logits=logits, target=y, loss=alone, **dev)
    loss, _ = oracle_policy(logp, target, old.astype(np.float64), A.astype(np.float64), ref.astype(np.float64),
                            np.full(N, 1.0 / N), clip, kl, 1.0)
    assert abs(back(alone)[0] - loss.sum()) <= 32 * 2.0 ** -24 * (np.abs(loss).sum() + 1 + np.abs(A).max())
    # in place
    held_bar = bar.clone()
    dev["weight"] = torch.from_numpy(weight).to(gpu)
    hawk.run(stage, logits=logits, target=y, bar_logits=logits, bar_loss=cell, **dev, **out)
    assert torch.equal(logits, held_bar)


@pytest.mark.gpu
def test_rows_that_are_masked_hold_anything(gpu):
    """A left-out row, and one of weight 0, reach neither loss nor gradient whatever they hold; a target
    past the vocabulary and a row with no finite logit are loud."""
    import torch
    for V in (40, 3000, 70000):
        for dtype in (torch.float32, torch.bfloat16):
            N = 6
            logits = torch.randn(N, V, device=gpu).to(dtype)
            logits[1] = math.nan
            logits[2] = -math.inf
            logits[4, 3:] = torch.finfo(dtype).min           # masked vocabulary
            logits[4, 1] = -math.inf
            target = torch.tensor([1, -1, 2, 3, 0, 1], device=gpu)
            old = torch.zeros(N, device=gpu)
            old[1], old[2] = math.nan, math.inf
            A = torch.ones(N, device=gpu)
            A[1] = A[2] = math.nan
            weight = torch.full((N,), 0.25, device=gpu)
            weight[1] = math.nan
            weight[2] = 0.0
            loss, logp, lse = (torch.empty(k, device=gpu) for k in (1, N, N))
            bar = torch.empty_like(logits)
            stage = hawk.stages.policy_loss(kl=0.1)
            planes = dict(logits=logits, target=target, old_logp=old, advantage=A, ref_logp=old, weight=weight)
            hawk.run(stage, loss=loss, logp=logp, lse=lse, bar_logits=bar, **planes)
            assert torch.isfinite(loss).all() and torch.isfinite(bar).all()
            assert (bar[1] == 0).all() and (bar[2] == 0).all() and logp[1] == 0 and lse[1] == 0
            assert (bar[4, 3:] == 0).all() and bar[4, 0] != 0
            want = torch.log_softmax(logits[4].double()[:3], 0)[0]
            assert abs(logp[4].double() - want) < 1e-5
            two = torch.empty_like(bar)
            hawk.run(stage.vjp, logp=logp, lse=lse, bar_logits=two, **planes)
            assert torch.isfinite(two).all() and (two[2] == 0).all()
            target[3] = V
            hawk.run(stage, loss=loss, logp=logp, bar_logits=bar, **planes)
            assert torch.isnan(loss).all() and torch.isnan(logp[3]) and torch.isnan(bar[3]).all()
            assert torch.isfinite(bar[0]).all()
            # a row with no finite logit has no distribution
            hawk.run(hawk.stages.token_logp(), logits=logits, target=target.clamp(max=V - 1), logp=logp, lse=lse)
            assert torch.isnan(logp[2]) and lse[2] == -math.inf and torch.isfinite(logp[0])
            # a row of the lowest value throughout is a row of equal logits
            logits[0] = torch.finfo(dtype).min
            hawk.run(hawk.stages.token_logp(), logits=logits, target=target.clamp(max=V - 1), logp=logp)
            assert abs(float(logp[0]) + math.log(V)) < 1e-5


@pytest.mark.gpu
def test_the_policy_gradient_is_the_losss_difference_quotient(gpu):
    """float32: a step of 2^-6 gives a truncation of about e^2 and a rounding of 2^-24 / e relative to
    the loss, both below 1e-3."""
    import torch
    N, V = 5, 12
    g = torch.Generator(device=gpu).manual_seed(9)
    logits = torch.randn(N, V, generator=g, device=gpu)
    target = torch.tensor([3, 0, 11, -1, 5], device=gpu)
    base = torch.log_softmax(logits, 1)[torch.arange(N), target.clamp(min=0)]
    planes = dict(target=target, old_logp=base + torch.tensor([0.05, -0.4, 0.4, 0.0, 0.1], device=gpu),
                  ref_logp=base + 0.2, advantage=torch.tensor([1.0, 0.7, -0.8, 1.0, -0.5], device=gpu))
    stage = hawk.stages.policy_loss(kl=0.2)
    bar, loss = torch.empty_like(logits), torch.empty(1, device=gpu)
    hawk.run(stage, logits=logits, loss=loss, bar_logits=bar, **planes)
    e = 2.0 ** -6
    for n, v in [(0, 3), (0, 1), (1, 0), (1, 7), (2, 11), (2, 2), (3, 4), (4, 5)]:
        ends = []
        for sign in (1, -1):
            moved = logits.clone()
            moved[n, v] += sign * e
            hawk.run(stage, logits=moved, loss=loss, **planes)
            ends.append(float(loss))
        assert abs((ends[0] - ends[1]) / (2 * e) - float(bar[n, v])) < 1e-3, (n, v)


def oracle_pairs(logp, target, ref, offsets, weight, beta, eps, margin=None):
    ratio = np.where(target >= 0, logp - ref, 0)
    sums = np.array([ratio[offsets[k]:offsets[k + 1]].sum() for k in range(len(offsets) - 1)])
    margin = sums[0::2] - sums[1::2] if margin is None else margin
    z = beta * margin
    soft = np.log1p(np.exp(-np.abs(z)))
    loss = (1 - eps) * (soft + np.maximum(-z, 0)) + eps * (soft + np.maximum(z, 0))
    up = 1 / (1 + np.exp(-z))
    return margin, (weight * loss).sum(), beta * weight * (eps * up - (1 - eps) * (1 - up))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ROW_TYPES)
@pytest.mark.parametrize("lengths,V", [((1, 1), 5), ((3, 0, 0, 2), 17), ((30, 41, 7, 64, 129, 2), 300),
                                       ((5, 4, 3, 9, 0, 0, 8, 1, 2, 6), 5003)], ids=str)
def test_preference_loss_and_its_gradient(gpu, lengths, V, dtype):
    import torch
    N, P = sum(lengths), len(lengths) // 2
    print(lengths, V, dtype, flush=True)
    beta, eps, scale = 0.3, 0.1, 1.2
    logits, held, target = rows_case(N, V, dtype, gpu, 3)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    g = np.random.default_rng([13, N, V])
    logp64, lse64, l = oracle_rows(held, target, scale)
    ref = (logp64 + 0.2 * g.normal(size=N)).astype(np.float32)
    weight = g.uniform(0.5, 1.5, P).astype(np.float32)
    stage = hawk.stages.preference_loss(beta=beta, smoothing=eps, scale=scale)
    planes = dict(logits=logits, target=torch.from_numpy(target).to(gpu),
                  offsets=torch.from_numpy(offsets).to(gpu, torch.int32 if P % 2 else torch.int64))
    out = {n: torch.empty(k, device=gpu) for n, k in (("loss", 1), ("margin", P), ("logp", N), ("lse", N))}
    w = torch.from_numpy(weight).to(gpu)
    hawk.run(stage, ref_logp=torch.from_numpy(ref).to(gpu), weight=w, **planes, **out)
    margin, loss, slope = oracle_pairs(logp64, target, ref.astype(np.float64), offsets, weight.astype(np.float64), beta,
                                       eps)
    close_row(back(out["logp"]), logp64, lse64)
    # the sums are in 64 bits over log-probabilities that are not rounded: each token's has the
    # error of its row's sum of exponentials, whose terms err by their exponents' rounding,
    # u log2(e) |x - m| each (|x - m| of the terms that weigh is below 16): 24 u; the cell rounds
    tokens = np.add.reduceat(np.ones(N), np.minimum(offsets[:-1], N - 1)) * (np.diff(offsets) > 0)
    allowed = 24 * 2.0 ** -24 * (tokens[0::2] + tokens[1::2]) + 2.0 ** -24 * np.abs(margin)
    assert (np.abs(back(out["margin"]) - margin) <= allowed).all()
    assert abs(back(out["loss"])[0] - loss) <= 16 * 2.0 ** -24 * (abs(loss) + weight.sum()) + beta * (weight * allowed).sum()
    # the slope is the written margin's
    _, _, slope = oracle_pairs(logp64, target, ref.astype(np.float64), offsets, weight.astype(np.float64), beta, eps,
                               margin=back(out["margin"]))
    seq = np.searchsorted(offsets, np.arange(N), side="right") - 1
    c = 1.5 * np.where(seq % 2 == 0, slope[seq // 2], -slope[seq // 2])
    grad, size = oracle_gradient(l, target, back(out["lse"]), c, scale)
    bar = torch.empty_like(logits)
    hawk.run(stage.vjp, margin=out["margin"], lse=out["lse"], weight=w, bar_loss=torch.tensor(1.5, device=gpu),
             bar_logits=bar, **planes)
    # sigma's own error: 32 u relative
    close_gradient(back(bar), grad, size, l, back(out["lse"]), dtype, slack=64 * 2.0 ** -24)
    # the loss alone, no reference: 1 / pairs each
    hawk.run(stage, loss=out["loss"], **planes)
    _, mean, _ = oracle_pairs(logp64, target, np.zeros(N), offsets, np.full(P, 1.0 / P), beta, eps)
    assert abs(back(out["loss"])[0] - mean) <= 1e-5 * (1 + abs(mean) + np.abs(logp64).sum())


@pytest.mark.gpu
def test_a_pair_of_weight_zero_and_an_extreme_margin(gpu):
    import torch
    logits = torch.randn(4, 50, device=gpu)
    target = torch.tensor([0, 1, 2, 3], device=gpu)
    planes = dict(logits=logits, target=target, offsets=torch.tensor([0, 1, 2, 3, 4], device=gpu))
    ref = torch.tensor([0.0, 0.0, -2000.0, 3000.0], device=gpu)
    out = {n: torch.empty(k, device=gpu) for n, k in (("loss", 1), ("margin", 2), ("lse", 4))}
    stage = hawk.stages.preference_loss(beta=1.0)
    hawk.run(stage, ref_logp=ref, **planes, **out)
    assert torch.isfinite(out["loss"]).all()
    hawk.run(stage, ref_logp=-ref, **planes, **out)
    assert abs(float(out["loss"]) - 2500) < 10            # half of about 5000: the losing pair's -log sigma(z) = -z
    ref[2] = math.nan
    weight = torch.tensor([1.0, 0.0], device=gpu)
    hawk.run(stage, ref_logp=ref, weight=weight, **planes, **out)
    assert torch.isfinite(out["loss"]).all() and torch.isnan(out["margin"][1])
    bar = torch.empty_like(logits)
    hawk.run(stage.vjp, weight=weight, margin=out["margin"], lse=out["lse"], bar_logits=bar, **planes)
    assert torch.isfinite(bar).all() and (bar[2:] == 0).all() and (bar[:2] != 0).any()


@pytest.mark.gpu
def test_row_losses_replayed_from_a_graph_and_repeated(gpu):
    import torch
    N, V = 40, 9001
    logits = torch.randn(N, V, device=gpu).bfloat16()
    target = torch.randint(0, V, (N,), device=gpu)
    old, A = -9.0 + torch.randn(N, device=gpu), torch.randn(N, device=gpu)
    stage = hawk.stages.policy_loss()
    planes = dict(logits=logits, target=target, old_logp=old, advantage=A)
    loss, bar = torch.empty(1, device=gpu), torch.empty_like(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    launch = stage.prepare(loss=loss, bar_logits=bar, stream=side, **planes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        launch()
    for k in range(4):
        logits.copy_(torch.randn(N, V, device=gpu))
        want, wbar = torch.empty(1, device=gpu), torch.empty_like(logits)
        hawk.run(stage, loss=want, bar_logits=wbar, **planes)
        loss.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.equal(bar, wbar)


@pytest.mark.gpu
def test_plain_calls_captured_on_a_stream_of_their_own(gpu):
    """Two graphs captured on a stream that no call ran on before, replayed in
    either order and between plain calls: none leans on what another cleared."""
    import torch
    N, V, T, C = 40, 48, 3000, 40
    target = torch.randint(0, V, (N,), device=gpu)
    old, A = -4.0 + torch.randn(N, device=gpu), torch.randn(N, device=gpu)
    logits = torch.randn(N, V, device=gpu)
    few = torch.randn(3, 200003, device=gpu)
    gate, x = torch.rand(1, T, C, device=gpu), torch.randn(1, T, C, device=gpu)
    loss_stage, logp_stage, scan = hawk.stages.policy_loss(), hawk.stages.token_logp(), hawk.stages.recurrence()

    def calls():
        loss, bar, logp, h = torch.empty(1, device=gpu), torch.empty_like(logits), torch.empty(3, device=gpu), torch.empty_like(x)

        def run():
            hawk.run(loss_stage, logits=logits, target=target, old_logp=old, advantage=A, loss=loss, bar_logits=bar)
            hawk.run(logp_stage, logits=few, target=target[:3].contiguous(), logp=logp)
            hawk.run(scan, gate=gate, x=x, h=h)
        return run, (loss, bar, logp, h)

    eager, want = calls()
    eager()
    torch.cuda.synchronize()
    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        run, outs = calls()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        graphs.append((graph, outs))
    for k in (1, 0, 1, 1, 0):
        logits.copy_(torch.randn(N, V, device=gpu))
        x.copy_(torch.randn(1, T, C, device=gpu))
        eager()
        graph, outs = graphs[k]
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    with torch.cuda.stream(side):
        for o in want:
            o.fill_(float("nan"))
        eager()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(graphs[0][1], want))


@pytest.mark.gpu
def test_plain_calls_captured_on_a_stream_that_ran_before(gpu):
    """Graphs captured on a warmed stream, replayed on two others beside each other and beside plain calls on
    that stream: each works in memory of its own."""
    import torch
    N, V, T, C = 40, 48, 6000, 40
    target = torch.randint(0, V, (N,), device=gpu)
    old, A = -4.0 + torch.randn(N, device=gpu), torch.randn(N, device=gpu)
    logits, few = torch.randn(N, V, device=gpu), torch.randn(3, 200003, device=gpu)
    gate, x = torch.rand(1, T, C, device=gpu), torch.randn(1, T, C, device=gpu)
    offsets = torch.arange(0, N + 1, N // 8, device=gpu)[:9]
    loss_stage, logp_stage, scan = hawk.stages.policy_loss(), hawk.stages.token_logp(), hawk.stages.recurrence()
    pairs = hawk.stages.preference_loss()

    def calls():
        loss, bar, logp = torch.empty(1, device=gpu), torch.empty_like(logits), torch.empty(3, device=gpu)
        h, to_gate, to_x = (torch.empty_like(x) for _ in range(3))
        both = torch.empty(1, device=gpu)

        def run():
            hawk.run(loss_stage, logits=logits, target=target, old_logp=old, advantage=A, loss=loss, bar_logits=bar)
            hawk.run(logp_stage, logits=few, target=target[:3].contiguous(), logp=logp)
            hawk.run(scan, gate=gate, x=x, h=h)
            hawk.run(scan.vjp, gate=gate, h=h, bar_h=x, bar_gate=to_gate, bar_x=to_x)
            hawk.run(pairs, logits=logits, target=target, offsets=offsets, loss=both)
        return run, (loss, bar, logp, h, to_gate, to_x, both)

    eager, want = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            eager()
    torch.cuda.synchronize()
    want = tuple(o.clone() for o in want)
    graphs = []
    for _ in range(2):
        run, outs = calls()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        graphs.append((graph, outs, torch.cuda.Stream()))
    plain, plain_outs = calls()
    for k in range(6):
        for _, outs, _ in graphs:
            for o in outs:
                o.fill_(float("nan"))
        for o in plain_outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(side):
            plain()
        torch.cuda.synchronize()
        for outs in (graphs[0][1], graphs[1][1], plain_outs):
            assert all(torch.equal(o, w) for o, w in zip(outs, want)), k


@pytest.mark.gpu
def test_a_launcher_made_under_capture_runs_before_and_after_a_replay(gpu):
    import torch
    logits, few = torch.randn(40, 48, device=gpu), torch.randn(3, 200003, device=gpu)
    target = torch.randint(0, 48, (40,), device=gpu)
    planes = dict(logits=logits, target=target, old_logp=torch.full((40,), -4.0, device=gpu),
                  advantage=torch.randn(40, device=gpu))
    policy, rows = hawk.stages.policy_loss(), hawk.stages.token_logp()
    loss, logp, want, want_logp = (torch.empty(k, device=gpu) for k in (1, 3, 1, 3))
    hawk.run(policy, loss=want, **planes)
    hawk.run(rows, logits=few, target=target[:3].contiguous(), logp=want_logp)
    side, graph, y = torch.cuda.Stream(), torch.cuda.CUDAGraph(), target[:3].contiguous()
    with torch.cuda.graph(graph, stream=side):
        launches = policy.prepare(loss=loss, **planes), rows.prepare(logits=few, target=y, logp=logp)
        for launch in launches:
            launch()
    for k in range(4):
        loss.fill_(float("nan"))
        logp.fill_(float("nan"))
        torch.cuda.synchronize()
        if k % 2:
            graph.replay()
        else:
            for launch in launches:
                launch()
        torch.cuda.synchronize()
        # a row in one piece or in parts: the terms are joined in another tree
        assert abs(float(loss) - float(want)) <= 2.0 ** -20 * 10
        assert (logp - want_logp).abs().max() <= 16 * 2.0 ** -24 * (2 + want_logp.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ROW_TYPES)
@pytest.mark.parametrize("shape", [(2, 131072), (5, 262147), (64, 131081), (65, 131081)], ids=str)
def test_few_long_rows_over_several_workgroups(gpu, shape, dtype):
    """Rows whose first parts hold nothing, rows of the type's lowest value, and calls one
    after another that find the workgroups' words as the call before left them."""
    import torch
    N, V = shape
    g = np.random.default_rng([3, N, V])
    x = g.normal(size=(N, V)) * 3
    x[0, :V - 5] = -np.inf
    target = g.integers(0, V, N)
    target[0] = V - 2
    if N > 2:
        x[1] = float(torch.finfo(torch_type(dtype)).min) / 2
        x[2, ::2] = -np.inf
        target[2] |= 1
        target[3] = -1
    logits, held = plane(x, dtype, gpu)
    del x
    y = torch.from_numpy(target).to(gpu)
    want, want_lse, l = oracle_rows(held, target, 1.0)
    c = g.normal(size=N).astype(np.float32)
    bar_logp = torch.from_numpy(c).to(gpu)
    stage = hawk.stages.token_logp()
    out = [torch.empty(N, device=gpu) for _ in range(2)]
    held_launch = stage.prepare(logits=logits, target=y, logp=out[0], lse=out[1])
    first = None
    for k in range(3):
        logp, lse = torch.empty(N, device=gpu), torch.empty(N, device=gpu)
        hawk.run(stage, logits=logits, target=y, logp=logp, lse=lse)
        held_launch()
        close_row(back(logp), want, want_lse)
        close_row(back(lse), want_lse, want_lse)
        first = logp if first is None else first
        assert torch.equal(logp, first) and torch.equal(logp, out[0]) and torch.equal(lse, out[1])
    bar = torch.empty_like(logits)
    hawk.run(stage.vjp, logits=logits, target=y, lse=lse, bar_logp=bar_logp, bar_logits=bar)
    grad, size = oracle_gradient(l, target, back(lse), c.astype(np.float64), 1.0)
    # a masked logit's gradient is 0, whatever its distance
    reach = np.where(np.isinf(l), 0, l)
    close_gradient(back(bar), grad, size, reach, back(lse), dtype)
    del bar
    # the policy loss of the same rows: its slope is -r A at r = 1, then in place
    loss, both = torch.empty(1, device=gpu), torch.empty_like(logits)
    planes = dict(target=y, old_logp=logp, advantage=-bar_logp, weight=torch.ones(N, device=gpu))
    policy = hawk.stages.policy_loss()
    hawk.run(policy, logits=logits, loss=loss, bar_logits=both, **planes)
    close_gradient(back(both), grad, size, reach, back(lse), dtype, slack=8 * 2.0 ** -24 * (2 + 2 * np.abs(back(lse)).max()))
    total = np.where(target >= 0, c, 0).astype(np.float64).sum()
    assert abs(back(loss)[0] - total) <= 8 * 2.0 ** -24 * (2 + np.abs(want_lse)) @ np.abs(c) * 2
    hawk.run(policy, logits=logits, bar_logits=logits, **planes)
    assert torch.equal(logits, both)


@pytest.mark.gpu
def test_a_ratio_past_the_largest_number_is_the_minimums(gpu):
    """r = inf: -min(r A, clamp(r) A) is bounded for A > 0, an infinity for A < 0 and, like inf * 0, a NaN for A = 0."""
    import torch
    logits, target = torch.zeros(4, 9, device=gpu), torch.arange(4, device=gpu)
    A = torch.tensor([1.0, -1.0, 0.0, 0.5], device=gpu)
    old = torch.tensor([-200.0, -200.0, -200.0, -2.0], device=gpu)
    stage, loss, bar = hawk.stages.policy_loss(clip=0.2), torch.empty(1, device=gpu), torch.empty_like(logits)
    for n, want in enumerate((-1.2, math.inf, math.nan, None)):
        weight = torch.zeros(4, device=gpu)
        weight[n] = 1.0
        hawk.run(stage, logits=logits, target=target, old_logp=old, advantage=A, weight=weight, loss=loss, bar_logits=bar)
        if want is None:
            assert math.isfinite(float(loss)) and torch.isfinite(bar).all()
        else:
            assert float(loss) == pytest.approx(want, rel=1e-6, nan_ok=True)
            assert torch.isnan(bar[n]).all() if math.isnan(want) else not math.isfinite(want) or (bar[n] == 0).all()
        assert (bar[torch.arange(4) != n] == 0).all()


@pytest.mark.gpu
def test_the_kl_term_of_a_target_without_probability_is_infinite(gpu):
    import torch
    logits, target = torch.randn(3, 50, device=gpu), torch.tensor([1, 2, 3], device=gpu)
    logits[1, 2] = -math.inf
    planes = dict(logits=logits, target=target, old_logp=torch.full((3,), -4.0, device=gpu),
                  ref_logp=torch.full((3,), -4.0, device=gpu), advantage=torch.ones(3, device=gpu))
    loss = torch.empty(1, device=gpu)
    hawk.run(hawk.stages.policy_loss(kl=0.1), loss=loss, **planes)
    assert float(loss) == math.inf
    hawk.run(hawk.stages.policy_loss(), loss=loss, **{n: x for n, x in planes.items() if n != "ref_logp"})
    assert math.isfinite(float(loss))
    # a step of the policy that e^d overflows for
    planes["ref_logp"][1] = 0.0
    logits[1, 2] = -200.0
    hawk.run(hawk.stages.policy_loss(kl=0.1), loss=loss, **planes)
    assert float(loss) == math.inf


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ROW_TYPES)
@pytest.mark.parametrize("V", [5, 300, 3000, 9000, 70000, 200003])
def test_an_infinite_logit_is_the_rows_sum(gpu, V, dtype):
    """lse = +inf: every other logit has probability 0 and log-probability -inf, its own is inf - inf."""
    import torch
    for N in (6, 600) if V <= 9000 else (6,):
        logits = torch.randn(N, V, device=gpu).to(torch_type(dtype))
        target = torch.full((N,), 2, device=gpu)
        logits[0, V - 1] = math.inf                        # another element's
        logits[1, 2] = math.inf                            # the target's own
        logits[2, 1], logits[2, 0] = math.inf, math.nan    # a NaN beside it
        logits[3] = math.inf
        logits[4, V - 1] = math.inf
        logits[4, 2] = -math.inf
        stage = hawk.stages.token_logp()
        logp, lse, bar = torch.empty(N, device=gpu), torch.empty(N, device=gpu), torch.empty_like(logits)
        hawk.run(stage, logits=logits, target=target, logp=logp, lse=lse)
        assert (lse[[0, 1, 3, 4]] == math.inf).all() and torch.isnan(lse[2])
        assert (logp[[0, 4]] == -math.inf).all() and torch.isnan(logp[[1, 2, 3]]).all()
        assert torch.isfinite(lse[5:]).all() and torch.isfinite(logp[5:]).all()
        hawk.run(stage.vjp, logits=logits, target=target, lse=lse, bar_logp=torch.ones(N, device=gpu), bar_logits=bar)
        assert bar[0, 2] == 1 and (bar[0, 3:V - 1] == 0).all() and (bar[0, :2] == 0).all() and torch.isnan(bar[0, V - 1])
        assert torch.isnan(bar[2]).all() and torch.isnan(bar[3]).all()
        # the same sum in the other rows' kernels
        both, again = torch.empty_like(logits), torch.empty(N, device=gpu)
        hawk.run(hawk.stages.policy_loss(), logits=logits, target=target, old_logp=logp.nan_to_num(0.0, 0.0, 0.0),
                 advantage=torch.ones(N, device=gpu), lse=again, bar_logits=both)
        assert torch.equal(again.nan_to_num(-1.0), lse.nan_to_num(-1.0)) or (again - lse)[5:].abs().max() < 1e-4
        assert (again[[0, 1, 3, 4]] == math.inf).all() and torch.isnan(again[2])
        assert torch.isfinite(both[5:]).all() and (both[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [1, 128, 129, 400])
def test_an_infinite_margin_costs_what_its_side_of_the_loss_says(gpu, pairs):
    """A sequence with a masked target has log-probability -inf.  Against it the preferred one's loss is 0, whatever the
    weight 0 of the smoothing's other side; with smoothing it is infinite."""
    import torch
    logits = torch.zeros(2 * pairs, 8, device=gpu)
    target = torch.zeros(2 * pairs, dtype=torch.int64, device=gpu)
    planes = dict(logits=logits, target=target, offsets=torch.arange(2 * pairs + 1, device=gpu))
    loss, margin, lse = torch.empty(1, device=gpu), torch.empty(pairs, device=gpu), torch.empty(2 * pairs, device=gpu)
    rest = math.log(2) * (pairs - 1) / pairs               # every other margin is 0
    for row, side, want in ((1, math.inf, {0.0: rest, 0.25: math.inf, 1.0: math.inf}),
                            (0, -math.inf, {0.0: math.inf, 0.25: math.inf, 1.0: rest})):
        logits.zero_()
        logits[row, 0] = -math.inf
        for smoothing, value in want.items():
            stage, bar = hawk.stages.preference_loss(beta=0.5, smoothing=smoothing), torch.empty_like(logits)
            hawk.run(stage, loss=loss, margin=margin, lse=lse, **planes)
            assert float(margin[0]) == side and (margin[1:] == 0).all()
            assert float(loss) == pytest.approx(value, rel=1e-6, abs=1e-7)
            hawk.run(stage.vjp, margin=margin, lse=lse, bar_logits=bar, **planes)
            assert torch.isfinite(bar).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 3000, 20000])
def test_a_weight_of_zero_leaves_a_row_out_whatever_its_target(gpu, V):
    """A target past the vocabulary is a NaN, in a row or pair of weight 0 nothing: in every form of the gradient."""
    import torch
    logits = torch.randn(6, V, device=gpu)
    target = torch.tensor([1, V, 2, V + 5, 0, 3], device=gpu)
    old = torch.full((6,), -5.0, device=gpu)
    for weight, loud in (([1.0, 0.0, 1.0, 0.0, 1.0, 1.0], ()), ([1.0, 0.5, 1.0, 0.0, 1.0, 1.0], (1,))):
        stage = hawk.stages.policy_loss()
        planes = dict(logits=logits, target=target, old_logp=old, advantage=torch.ones(6, device=gpu),
                      weight=torch.tensor(weight, device=gpu))
        loss, logp, lse = (torch.empty(k, device=gpu) for k in (1, 6, 6))
        one, two = torch.empty_like(logits), torch.empty_like(logits)
        hawk.run(stage, loss=loss, logp=logp, lse=lse, bar_logits=one, **planes)
        hawk.run(stage.vjp, logp=logp, lse=lse, bar_logits=two, **planes)
        for bar in (one, two):
            for n in range(6):
                if n in loud:
                    assert torch.isnan(bar[n]).all()
                else:
                    assert torch.isfinite(bar[n]).all() and (n not in (1, 3) or (bar[n] == 0).all())
        assert math.isnan(float(loss)) == bool(loud)
    pair, bar = hawk.stages.preference_loss(), torch.empty_like(logits)
    planes = dict(logits=logits, target=target, offsets=torch.arange(7, device=gpu))
    margin, lse = torch.empty(3, device=gpu), torch.empty(6, device=gpu)
    for weight, loud in (([0.0, 0.0, 1.0], ()), ([0.0, 1.0, 1.0], (2, 3))):
        planes["weight"] = torch.tensor(weight, device=gpu)
        hawk.run(pair, margin=margin, lse=lse, loss=loss, **planes)
        assert math.isnan(float(loss)) == bool(loud)
        hawk.run(pair.vjp, margin=margin, lse=lse, bar_logits=bar, **planes)
        for n in range(6):
            assert torch.isnan(bar[n]).all() if n in loud else torch.isfinite(bar[n]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [((1 << 28) + 3, 2), ((1 << 26) + 5, 280)], ids=str)
def test_more_rows_than_one_launch_has_threads_for(gpu, N, V):
    """A launch has fewer than 2^32 threads along its grid: 2^28 rows of 16 lanes each, 2^26 of 64, are past that."""
    import torch
    block = torch.randn(1 << 16, V, device=gpu).bfloat16()
    logits = torch.empty(N, V, dtype=torch.bfloat16, device=gpu)
    for first in range(0, N, len(block)):
        part = logits[first:first + len(block)]
        part.copy_(block[:len(part)])
    target = torch.zeros(N, dtype=torch.int32, device=gpu)
    target[1::2] = 1
    logp, lse = torch.empty(N, device=gpu), torch.empty(N, device=gpu)
    stage = hawk.stages.token_logp()
    hawk.run(stage, logits=logits, target=target, logp=logp, lse=lse)
    want = torch.log_softmax(block.double(), 1)
    at = torch.arange(len(block), device=gpu) % 2
    for first in (0, N - N % len(block) - len(block), N // 2 // len(block) * len(block)):
        rows = slice(first, first + len(block))
        assert (logp[rows].double() - want[torch.arange(len(block), device=gpu), at]).abs().max() < 1e-5
    tail = N % len(block)
    assert (logp[N - tail:].double() - want[torch.arange(tail, device=gpu), at[:tail]]).abs().max() < 1e-5
    hawk.run(stage.vjp, logits=logits, target=target, lse=lse, bar_logp=torch.ones(N, device=gpu), bar_logits=logits)
    grad = -want.exp()
    grad[torch.arange(len(block), device=gpu), at] += 1
    for first in list(range(0, N - len(block), len(block) * 331)) + [N - tail - len(block)]:
        assert (logits[first:first + len(block)].double() - grad).abs().max() < 2.0 ** -8
    assert (logits[N - tail:].double() - grad[:tail]).abs().max() < 2.0 ** -8


# -- dropout ---------------------------------------------------------------------------------

def philox(group, offset, seed):
    """Philox4x32-10 in Python integers."""
    low = 0xFFFFFFFF
    c = [group & low, group >> 32, offset & low, offset >> 32]
    k = [seed & low, seed >> 32]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def kept(n, cut, offset, seed):
    out = np.empty(n, bool)
    for g in range((n + 7) // 8):
        w = philox(g, offset, seed)
        for j in range(min(8, n - 8 * g)):
            out[8 * g + j] = (w[j // 2] >> (16 * (j % 2)) & 0xFFFF) >= cut
    return out


def test_the_generator_is_philox_4x32_10():
    """The generator's published known answers."""
    assert philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert philox(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox(0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (65, 129), (2, 3, 40), (1000, 17), (31, 512)], ids=str)
def test_dropout_and_its_derivative_are_the_generators_mask(gpu, shape, dtype):
    import torch
    print(shape, dtype, flush=True)
    g = np.random.default_rng(21)
    n = int(np.prod(shape))
    for p, seed, offset in ((0.25, 5, 0), (0.1, (1 << 64) - 3, (1 << 40) + 7), (0.0, 1, 2), (1.0, 1, 2)):
        x, xv = plane(g.normal(size=shape), dtype, gpu)
        res, rv = plane(g.normal(size=shape), dtype, gpu)
        cut = round(p * 65536)
        mask = kept(n, cut, offset, seed).reshape(shape)
        stage = hawk.stages.dropout(p)
        y = torch.empty_like(x)
        hawk.run(stage, x=x, y=y, seed=seed, offset=offset)
        # two roundings: the factor and the product in the arithmetic's type, then the output's
        want = np.where(mask, xv * (65536.0 / (65536 - cut) if cut < 65536 else 0), 0)
        assert (np.abs(back(y) - want) <= (4 * U[dtype] + R[dtype]) * 1.01 * np.abs(want) + TINY[dtype]).all()
        assert ((back(y) == 0) == ~mask).all() or p == 0
        hawk.run(stage, x=x, residual=res, y=y, seed=seed, offset=offset)
        size = np.abs(want) + np.abs(rv)
        assert (np.abs(back(y) - want - rv) <= (8 * U[dtype] + R[dtype]) * 1.01 * size + TINY[dtype]).all()
        bar = torch.empty_like(x)
        hawk.run(diff.vjp(stage), bar_y=x, bar_x=bar, seed=seed, offset=offset)
        assert (np.abs(back(bar) - want) <= (4 * U[dtype] + R[dtype]) * 1.01 * np.abs(want) + TINY[dtype]).all()
        # the offset from a cell, in place, and through rows apart: the same mask
        hawk.run(stage, x=x.clone(), y=bar, seed=seed, offset=torch.tensor([offset], device=gpu))
        hawk.run(stage, x=x, y=y, seed=seed, offset=offset)
        assert torch.equal(bar, y)
        if len(shape) > 1:
            wide = torch.zeros((*shape[:-1], shape[-1] + 3), dtype=x.dtype, device=gpu)
            apart = wide[..., 1:1 + shape[-1]]
            apart.copy_(x)
            hawk.run(stage, x=apart, y=apart, seed=seed, offset=offset)
            assert torch.equal(apart, y) and (wide[..., 0] == 0).all() and (wide[..., -2:] == 0).all()
        hawk.run(stage, x=x, y=x, seed=seed, offset=offset)
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_dropout_drops_infinities_and_keeps_its_rate(gpu):
    import torch
    n = 1 << 20
    x = torch.full((n,), math.inf, device=gpu)
    y = torch.empty_like(x)
    hawk.run(hawk.stages.dropout(0.5), x=x, y=y, seed=3)
    assert ((y == 0) | torch.isinf(y)).all()
    hawk.run(hawk.stages.dropout(0.1), x=torch.ones_like(x), y=y, seed=4, offset=9)
    rate = float((y == 0).double().mean())
    cut = 6554 / 65536                                    # round(0.1 * 2^16) / 2^16
    assert abs(rate - cut) < 6 * math.sqrt(cut * (1 - cut) / n)
    other = torch.empty_like(y)
    hawk.run(hawk.stages.dropout(0.1), x=torch.ones_like(x), y=other, seed=4, offset=10)
    assert abs(float(((y == 0) & (other == 0)).double().mean()) - cut ** 2) < 6 * cut / math.sqrt(n)


@pytest.mark.gpu
def test_dropout_draws_a_new_mask_a_replay(gpu):
    import torch
    x = torch.ones(5000, device=gpu)
    y, cell = torch.empty_like(x), torch.zeros(1, dtype=torch.int64, device=gpu)
    stage = hawk.stages.dropout(0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    launch = stage.prepare(x=x, y=y, seed=8, offset=cell, stream=side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        launch()
        cell.add_(1)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(x)
        hawk.run(stage, x=x, y=want, seed=8, offset=k)
        assert torch.equal(y, want)


def test_dropout_refuses_a_single_row_that_is_not_contiguous():
    """Planes are addressed by rows: one row with gaps, or of one element repeated, is refused as several are."""
    import torch
    base, m, one = torch.zeros(1000), torch.zeros(300, 7), torch.zeros(())
    gaps = torch.zeros(1, 1000)[:, ::2]
    for x in (base[::2], m[:, 3], gaps, one.expand(500), torch.zeros(1, 1, 1).expand(1, 1, 9)):
        like = torch.zeros(x.shape)
        drop = hawk.stages.dropout(0.5)
        for stage, planes in ((drop, dict(x=x, y=like)), (drop, dict(x=like, y=x)), (drop, dict(x=like, residual=x, y=like)),
                              (drop.vjp, dict(bar_y=x, bar_x=like)), (drop.vjp, dict(bar_y=like, bar_x=x))):
            with pytest.raises(HawkError, match="is contiguous, got strides"):
                stage._make(planes)
    # one row that is contiguous, and rows of one element, are planes like any other
    wide = torch.zeros(3, 64)
    for x in (wide[1], wide[1:2, :7], wide[:, 3:4], torch.zeros(1, 1, 5)[:, :, 1:4], torch.zeros(4, 1).expand(4, 1), one):
        assert hawk.stages.dropout(0.5)._make(dict(x=x, y=torch.zeros(x.shape))).job.cols > 0


def test_dropout_takes_whole_numbers_as_they_are_and_refuses_others():
    """An offset that is no cell is never taken for 0: a mask would repeat from step to step."""
    import torch
    stage = hawk.stages.dropout(0.5)
    for name in ("seed", "offset"):
        for x, want in ((5, 5), (np.int64(5), 5), (np.uint64((1 << 64) - 1), (1 << 64) - 1), (np.int32(0), 0)):
            assert stage._value(name, x) == want
        for x in (7.0, np.float64(7), "7", True, np.bool_(True), -1, np.int64(-1), 1 << 64, [5], np.array([5, 6])):
            with pytest.raises(HawkError, match=f"{name}= is an int"):
                stage._value(name, x)
    assert stage._value("offset", None) == 0 and stage._value("offset", torch.zeros(1, dtype=torch.int64)) == 0
    for x in (None, torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(HawkError, match="seed= is an int"):
            stage._value("seed", x)


# -- refusals --------------------------------------------------------------------------------

def test_options_out_of_range_are_refused():
    s = hawk.stages
    for call, text in ((lambda: s.recurrence(gate="tanh"), "gate="), (lambda: s.dropout(1.5), "p="),
                       (lambda: s.dropout(1e-7), "resolution"), (lambda: s.dropout(True), "p="),
                       (lambda: s.policy_loss(clip=-0.1), "clip="), (lambda: s.policy_loss(kl=math.nan), "kl="),
                       (lambda: s.token_logp(scale=0.0), "scale="), (lambda: s.token_logp(scale=math.inf), "scale="),
                       (lambda: s.preference_loss(smoothing=1.5), "smoothing="),
                       (lambda: s.preference_loss(beta=math.inf), "beta=")):
        with pytest.raises(HawkError, match=text):
            call()


def test_names_missing_planes_and_launch_options_are_refused():
    import torch
    x = torch.zeros(1, 2, 3)
    scan = hawk.stages.recurrence()
    with pytest.raises(HawkError, match="no plane is named 'y'"):
        hawk.run(scan, gate=x, x=x, y=x)
    with pytest.raises(HawkError, match="'x' is not given"):
        hawk.run(scan, gate=x, h=x)
    with pytest.raises(HawkError, match="no output"):
        hawk.run(scan.vjp, gate=x, h=x, bar_h=x)
    with pytest.raises(HawkError, match="not on a ROCm device"):
        hawk.run(scan, gate=x, x=x, h=x)
    with pytest.raises(HawkError, match="torch tensor"):
        hawk.run(scan, gate=x.numpy(), x=x, h=x)
    with pytest.raises(HawkError, match="no base="):
        hawk.run(scan, base=1, gate=x, x=x, h=x)
    with pytest.raises(HawkError, match="seed"):
        hawk.run(hawk.stages.dropout(0.5), x=x, y=x)
    with pytest.raises(HawkError, match="wrt="):
        diff.vjp(scan, wrt=("x",))
    with pytest.raises(HawkError, match="no derivative"):
        diff.vjp(scan.vjp)


def test_a_stage_is_no_traced_kernel():
    for stage in (hawk.stages.recurrence(), hawk.stages.policy_loss().vjp, hawk.stages.dropout(0.5)):
        with pytest.raises(HawkError, match=f"{stage.name}: a stage has no forward-mode derivative"):
            diff.jvp(stage)
        with pytest.raises(HawkError, match="not a traced kernel"):
            hawk.chain(stage, name="both")
        with pytest.raises(HawkError, match="takes a traced kernel"):
            hawk.steps(stage, 2)


@pytest.mark.gpu
def test_planes_that_do_not_fit_are_refused(gpu):
    import torch
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=gpu)  # noqa: E731
    scan, x = hawk.stages.recurrence(), z(2, 5, 3)
    bad = [
        (scan, dict(gate=x, x=z(2, 5, 4), h=x.clone()), "x.*is"),
        (scan, dict(gate=x, x=x.half(), h=x.clone()), "float16"),
        (scan, dict(gate=x.int(), x=x.int(), h=x.int()), "planes are"),
        (scan, dict(gate=x[0], x=x[0], h=x[0].clone()), "offsets"),
        (scan, dict(gate=x, x=x, h=z(2, 1, 3).expand(2, 5, 3)), "repeats memory"),
        (scan, dict(gate=x, x=x, h=x.clone(), h0=z(2, 4)), "state"),
        (scan, dict(gate=x, x=x, h=x.clone(), h0=z(2, 3, dtype=torch.float64)), "state"),
        (scan, dict(gate=x[0], x=x[0], h=x[0].clone(), offsets=z(3)), "int32 or int64"),
        (scan, dict(gate=x, x=x, h=x.clone(), offsets=z(3, dtype=torch.int32)), "packed planes"),
        (scan.vjp, dict(gate=x, h=x, bar_h=x, bar_x=x), "one tensor"),
        (hawk.stages.recurrence("sigmoid").vjp, dict(gate=x, h=x, bar_h=x, bar_gate=x.clone()), "'x' is not given"),
    ]
    t = torch.zeros(4, dtype=torch.int64, device=gpu)
    logp, pol, pref = hawk.stages.token_logp(), hawk.stages.policy_loss(kl=0.1), hawk.stages.preference_loss()
    l = z(4, 9)
    bad += [
        (logp, dict(logits=l.double(), target=t, logp=z(4)), "float32"),
        (logp, dict(logits=z(9, 4).t(), target=t, logp=z(4)), "contiguous"),
        (logp, dict(logits=l, target=t[:3], logp=z(4)), "rows"),
        (logp, dict(logits=l, target=t.float(), logp=z(4)), "int32 or int64"),
        (logp, dict(logits=l, target=t, logp=z(5)), "'logp'"),
        (logp, dict(logits=l, target=t), "no output"),
        (logp.vjp, dict(logits=l, target=t, lse=z(4), bar_logp=z(4), bar_logits=l.half()), "bar_logits"),
        (logp.vjp, dict(logits=l, target=t, lse=z(4), bar_logp=z(4), bar_logits=z(40).as_strided((4, 9), (5, 1))),
         "overlap"),
        (pol, dict(logits=l, target=t, old_logp=z(4), advantage=z(4), loss=z(1)), "ref_logp"),
        (pol, dict(logits=l, target=t, old_logp=z(4), advantage=z(4), ref_logp=z(4), loss=z(2)), "'loss'"),
        (pref, dict(logits=l, target=t, offsets=t, loss=z(1)), "2 \\* pairs"),
        (pref, dict(logits=l, target=t, offsets=t[:3], loss=z(1), margin=z(2)), "'margin'"),
    ]
    d = hawk.stages.dropout(0.5)
    bad += [
        (d, dict(x=l, y=z(4, 8), seed=0), "'y'"),
        (d, dict(x=l, y=l.half(), seed=0), "float16"),
        (d, dict(x=l, y=l.clone(), seed=-1), "seed="),
        (d, dict(x=l, y=l.clone(), seed=0, offset=1 << 64), "offset="),
        (d, dict(x=l, y=l.clone(), seed=0, offset=z(1)), "int64 cell"),
        (d, dict(x=z(9, 4).t(), y=l.clone(), seed=0), "contiguous"),
        (d, dict(x=z(4, 3, 2, 9)[:, :2], y=z(4, 2, 2, 9), seed=0), "evenly apart"),
    ]
    for stage, planes, text in bad:
        with pytest.raises(HawkError, match=text):
            hawk.run(stage, **planes)
        with pytest.raises(HawkError, match=text):
            stage.prepare(**planes)


def test_the_entries_refuse_bad_jobs():
    """The C entries check their jobs before any launch."""
    L = _core.lib()
    r = _core.RecurrenceJob()
    r.seqs, r.steps, r.chans = 1, 4, 4
    ref = ctypes.byref(r)
    assert L.hk_recurrence(None, None, None) == 1
    assert L.hk_recurrence(ref, None, None) == 1 and b"plane is missing" in L.hk_last_error()
    r.steps = -1
    assert L.hk_recurrence_vjp(ref, None, None) == 1 and b">= 0" in L.hk_last_error()
    r.steps, r.dtype = 4, 9
    assert L.hk_recurrence(ref, None, None) == 1 and b"element type" in L.hk_last_error()
    assert L.hk_recurrence_scratch_bytes(None, 0) == 0
    w = _core.RowLossJob()
    w.rows, w.vocab, w.scale = 2, 5, 1.0
    ref = ctypes.byref(w)
    for fn in (L.hk_token_logp, L.hk_token_logp_vjp, L.hk_policy_loss, L.hk_policy_loss_vjp, L.hk_preference_loss,
               L.hk_preference_loss_vjp):
        assert fn(None, None, None) == 1
        assert fn(ref, None, None) == 1 and b"required" in L.hk_last_error()
    w.scale = 0.0
    assert L.hk_token_logp(ref, None, None) == 1 and b"scale" in L.hk_last_error()
    w.scale, w.dtype = 1.0, 1
    assert L.hk_token_logp(ref, None, None) == 1 and b"16-bit" in L.hk_last_error()
    d = _core.DropoutJob()
    d.rows, d.cols, d.cut = 1, 4, 70000
    assert L.hk_dropout(ctypes.byref(d), None) == 1 and b"cut" in L.hk_last_error()
    d.cut = 5
    assert L.hk_dropout(ctypes.byref(d), None) == 1 and b"required" in L.hk_last_error()
    # nothing to do is not an error
    r.dtype, r.seqs = 0, 0
    assert L.hk_recurrence(ctypes.byref(r), None, None) == 0
    w.dtype, w.rows = 0, 0
    assert L.hk_token_logp(ctypes.byref(w), None, None) == 0


def test_planes_past_the_grids_threads_are_refused_before_the_launch():
    """Dropout and the recurrence cut their launches no finer: what does not fit one is told by the entry."""
    L = _core.lib()
    d = _core.DropoutJob()
    d.rows, d.cols, d.cut, d.dtype = 1, 1 << 37, 5, 2
    d.x = d.y = 16
    assert L.hk_dropout(ctypes.byref(d), None) == 1 and b"grid limit" in L.hk_last_error()
    d.rows, d.cols = 1 << 34, 9
    assert L.hk_dropout(ctypes.byref(d), None) == 1 and b"grid limit" in L.hk_last_error()
    r = _core.RecurrenceJob()
    r.seqs, r.steps, r.chans, r.dtype = 1 << 29, 1 << 10, 1, 2
    for n in ("gate", "x", "h"):
        plane = getattr(r, n)
        plane.data, plane.seq, plane.step, plane.chan = 16, 2 << 10, 2, 3
    assert L.hk_recurrence(ctypes.byref(r), 16, None) == 1 and b"grid limit" in L.hk_last_error()


def test_a_stage_takes_the_scratch_its_entry_works_in():
    """Rows without a sum over them work in the stream's state alone, their gradients in neither."""
    import torch
    N = 4096
    l, t, f = torch.zeros(N, 8), torch.zeros(N, dtype=torch.int64), torch.zeros(N)
    logp, policy = hawk.stages.token_logp(), hawk.stages.policy_loss()
    plan = logp._make(dict(logits=l, target=t, logp=f))
    assert plan.scratch == 1 and plan.state is not None
    plan = logp.vjp._make(dict(logits=l, target=t, lse=f, bar_logp=f, bar_logits=l))
    assert plan.scratch == 0 and plan.state is None
    plan = policy._make(dict(logits=l, target=t, old_logp=f, advantage=f, logp=f))
    assert plan.scratch >= 12 * N and plan.state is not None
    assert logp._make(dict(logits=l[:0], target=t[:0], logp=f[:0])).scratch == 0


def test_the_jobs_are_laid_out_as_the_header_has_them():
    assert ctypes.sizeof(_core.SeqPlane) == 32
    assert ctypes.sizeof(_core.RecurrenceJob) == 6 * 32 + 5 * 8 + 3 * 8 + 4 * 4
    assert ctypes.sizeof(_core.RowLossJob) == 15 * 8 + 5 * 8 + 6 * 4 + 3 * 4 + 4
    assert ctypes.sizeof(_core.DropoutJob) == 4 * 8 + 5 * 8 + 2 * 8 + 2 * 4


def test_the_binding_puts_words_where_they_belong_and_refuses_others():
    import torch
    seen = []
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(ctypes.c_uint64), ctypes.c_void_p, ctypes.c_void_p)(
        lambda job, scratch, stream: seen.append((job[0], job[1], job[2], scratch, stream)) or 5)
    address = ctypes.cast(entry, ctypes.c_void_p).value
    Call, x = _core.bind().Call, torch.zeros(3)
    job = (1).to_bytes(8, "little") + (2).to_bytes(8, "little") + (3).to_bytes(8, "little")
    call = Call(address, False, True, 0, job, 2, (("x", x, 0), ("seed", None, 1)), ())
    assert call.launch([(1, 7), (2, 1 << 63)], 16, 32) == 5 and seen == [(1, 7, 1 << 63, 16, 32)]
    with pytest.raises(ValueError):
        call.launch([(3, 0)], 0, 0)
    # no tensor of the plan's device, another count, another name: nothing runs
    for arrays in ({"x": x, "seed": 4}, {"x": x}, {"seed": 4, "x": x}, {"x": 1, "seed": 4}, {}):
        assert call.run(arrays, 0, 0) == -1
    # by-value words alone: bound once the stream has its space, refused out of range
    call = Call(address, False, True, 0, job, 2, (("seed", None, 1),), ())
    assert call.run({"seed": 4}, 0, 32) == -1
    call.space(32, 48, 64)
    assert call.run({"seed": 4}, 0, 32) == 5 and seen[1:] == [(1, 4, 64, 48, 32)]
    for bad in (True, -1, 1 << 64, 1.0, None):
        assert call.run({"seed": bad}, 0, 32) == -1
    assert call.run({"seed": 4}, 1, 32) == -1 and call.run({"seed": 4}, 0, 33) == -1
    for planes, apart, size, error in (((("x", x, 3),), (), 24, ValueError), ((("x", 1, 0),), (), 24, TypeError),
                                       ((("x", x, 0),), ((0, 1),), 24, ValueError), ((), (), 23, ValueError)):
        with pytest.raises(error):
            Call(address, False, True, 0, job[:size], 2, planes, apart)


def bare_stage(entry):
    """A stage of planes ``x`` and ``y`` on the CPU, whose entry is the given function's address."""
    from hawk_amd import stages

    class Bare(stages._Stage):
        name, reads, writes = "bare", ("x",), ("y",)

        def _placed(self, arrays):
            return {n: t for n, t in arrays.items() if t is not None}

        def _make(self, t):
            job = (ctypes.c_uint64 * 2)()
            return stages._Plan(job, {"x": 0, "y": 1}, ctypes.cast(entry, ctypes.c_void_p), 0)
    return Bare()


def test_a_plan_is_found_once_it_can_be_called(monkeypatch):
    """Threads that meet a new set of shapes at once each call a whole plan; a plan that could not be bound is
    not kept."""
    import threading

    import torch
    from hawk_amd import stages
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)(lambda *_: 0)
    stage, x = bare_stage(entry), torch.zeros(3)
    bind, inside, leave, seen = stages._Plan.bind, threading.Event(), threading.Event(), []

    def slow(plan, *args):
        inside.set()
        leave.wait(10)
        bind(plan, *args)
    monkeypatch.setattr(stages._Plan, "bind", slow)
    first = threading.Thread(target=lambda: seen.append(stage._found({"x": x, "y": x})[0]))
    first.start()
    assert inside.wait(10)
    assert not stage._plans and stage._last is None
    monkeypatch.setattr(stages._Plan, "bind", bind)
    second = stage._found({"x": x, "y": x})[0]                 # meets the same shapes meanwhile
    leave.set()
    first.join()
    assert second.call is not None and seen[0].call is not None
    assert stage._found({"x": x, "y": x})[0].call is not None and len(stage._plans) == 1

    def broken(plan, *args):
        raise HawkError("the binding is not built")
    monkeypatch.setattr(stages._Plan, "bind", broken)
    stage = bare_stage(entry)
    for _ in range(2):
        with pytest.raises(HawkError, match="not built"):
            stage._found({"x": x, "y": x})
    assert not stage._plans and stage._last is None


def test_a_captured_call_works_apart_from_the_streams_others(monkeypatch):
    """A stream's space is not bound into a graph, which may be replayed on another stream: while the stream is
    captured every call asks for space of its own, and none of it is kept."""
    from types import SimpleNamespace

    from hawk_amd import stages
    seen, made, capturing = [], [], [False]
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(ctypes.c_uint64), ctypes.c_void_p, ctypes.c_void_p)(
        lambda job, scratch, stream: seen.append((scratch, job[2])) or 0)
    asked = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)(lambda stream: int(capturing[0]))
    monkeypatch.setattr(_core, "stream_capturing", lambda stream: capturing[0])
    monkeypatch.setattr(_core, "stream_capturing_entry", lambda: ctypes.cast(asked, ctypes.c_void_p).value)

    def space(device, stream, nbytes, state):
        made.append(SimpleNamespace(scratch=1000 + len(made), state=2000 + len(made)))
        return made[-1], not capturing[0]
    monkeypatch.setattr(stages, "_space", space)

    class Fixed(stages._Stage):
        """By-value words alone, which the binding's quick check takes on the CPU too."""
        name, values = "fixed", ("seed",)

        def _names(self, arrays):
            pass

        def _placed(self, arrays):
            return {}

        def _make(self, t):
            return stages._Plan((ctypes.c_uint64 * 3)(), {}, ctypes.cast(entry, ctypes.c_void_p), 64, state=2,
                                cells=(("seed", 1),))

        def _value(self, name, x):
            return x
    stage, arrays = Fixed(), {"seed": 7}
    for now in (False, False, True, True, False, True, False):
        capturing[0] = now
        stage.run(arrays, stream=96)
    kept = (1000, 2000)
    assert seen == [kept, kept, (1001, 2001), (1002, 2002), kept, (1003, 2003), kept] and len(made) == 4
    assert _core.lib().hk_stream_capturing(None) == 0


def test_a_launcher_made_under_capture_takes_no_state(monkeypatch):
    """Its clearing would be the graph's: a call of the launcher before a replay would find what the memory held."""
    import torch
    from hawk_amd import stages
    seen, capturing, made = [], [False], []
    words = ctypes.POINTER(ctypes.c_uint64)
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)(
        lambda job, scratch, stream: seen.append((scratch, ctypes.cast(job, words)[2])) or 0)
    monkeypatch.setattr(_core, "stream_capturing", lambda stream: capturing[0])
    monkeypatch.setattr(stages, "_on", lambda stream: contextlib.nullcontext())

    def on_host(make):
        def called(*args, device=None, **more):
            made.append(make(*args, **more))
            return made[-1]
        return called
    stage, x = bare_stage(entry), torch.zeros(3)
    plan = stages._Plan((ctypes.c_uint64 * 3)(), {"x": 0, "y": 1}, entry, 64, state=2)
    monkeypatch.setattr(stage, "_found", lambda arrays: (plan, [], -1))
    monkeypatch.setattr(torch, "empty", on_host(torch.empty))
    monkeypatch.setattr(torch, "zeros", on_host(torch.zeros))
    for capturing[0], tensors in ((False, 2), (True, 1)):
        made.clear()
        stage.prepare(stream=96, x=x, y=x)()
        assert len(made) == tensors
        assert seen[-1] == (made[0].data_ptr(), made[1].data_ptr() if tensors == 2 else 0)


@pytest.mark.parametrize("one,two,apart", [((0, 32), (0, 64), True), ((0, 32), (1, 32), True), ((0, 32), (0, 32), False)], ids=str)
def test_calls_wait_for_those_of_their_own_stream_alone(one, two, apart):
    """A launch that blocks holds the calls of its stream, whose scratch it works in, and no others."""
    import threading
    inside, met, order = threading.Event(), threading.Event(), []

    def first(job, scratch, stream):
        inside.set()
        order.append(("first", met.wait(20 if apart else 0.3)))
        return 0

    def second(job, scratch, stream):
        order.append(("second", None))
        met.set()
        return 0
    kind = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p)
    calls = []
    for entry, (device, stream) in ((kind(first), one), (kind(second), two)):
        call = _core.bind().Call(ctypes.cast(entry, ctypes.c_void_p).value, False, True, device, bytes(8), -1, (("seed", None, 0),), ())
        call.space(stream, 48, 0)
        calls.append((call, entry, device, stream))
    running = threading.Thread(target=lambda: calls[0][0].run({"seed": 1}, *calls[0][2:]))
    running.start()
    assert inside.wait(20)
    assert calls[1][0].run({"seed": 1}, *calls[1][2:]) == 0
    running.join()
    assert order == ([("second", None), ("first", True)] if apart else [("first", False), ("second", None)])


@pytest.mark.gpu
def test_the_recurrent_policy_example_learns(gpu):
    """All stages together: recall by chance is 1 in 16."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "recurrent_policy.py"
    spec = importlib.util.spec_from_file_location("recurrent_policy", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.train(gpu, rounds=60)
    assert got["rewards"][0] < 0.2 and got["rewards"][-1] > 0.5
    assert got["right"] > 0.8 and got["preference"][-1] < got["preference"][0]


@pytest.mark.gpu
@pytest.mark.parametrize("T,C,layout,packed,dtype", [
    (70001, 8, "channels", False, "float32"), (150001, 1, "steps", False, "float32"),
    (40003, 10, "channels", True, "bfloat16"), (30001, 3, "channels", True, "float64")], ids=str)
def test_a_long_recurrence_is_many_tiles_in_order(gpu, T, C, layout, packed, dtype):
    """More tiles than one look back sees, and the same bits every time."""
    import torch
    print(T, C, layout, packed, dtype, flush=True)
    for reverse in (False, True):
        got, held, offsets = recurrence_case(5 if packed else 1, T, C, dtype, "value", reverse, layout, True, packed, gpu,
                                             seed=40)
        # slow gates: a state reaches back over many tiles
        gate = 1 - 0.001 * np.random.default_rng(3).random(held["gate"].shape)
        if packed:
            gate[T // 2] = 0.0
        t, held["gate"] = plane(gate, dtype, gpu)
        got["gate"] = t.transpose(-1, -2).contiguous().transpose(-1, -2) if layout == "steps" else t
        stage = hawk.stages.recurrence(reverse=reverse)
        planes = {n: got[n] for n in ("gate", "x", "h0")}
        if packed:
            planes["offsets"] = torch.from_numpy(offsets).to(gpu)
        outs = []
        for _ in range(3):
            h, last = torch.empty_like(got["x"]), torch.empty_like(got["h0"])
            hawk.run(stage, h=h, last=last, **planes)
            bars = {n: torch.empty_like(got["x"]) for n in ("bar_gate", "bar_x")}
            bars["bar_h0"] = torch.empty_like(got["h0"])
            hawk.run(stage.vjp, h=h, bar_h=got["bar_h"], bar_last=got["bar_last"], **planes, **bars)
            outs.append((h, last, *bars.values()))
        assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))
        want, want_last, size = oracle_forward(held["gate"], held["x"], held["h0"], offsets, "value", reverse)
        close(back(h), want, size, T, "value", dtype)
        close(back(last), want_last, np.abs(size).max() + np.abs(want_last), T, "value", dtype, state=True)
        wants, sizes = oracle_vjp(held["gate"], None, back(h), held["h0"], held["bar_h"], held["bar_last"], offsets,
                                  "value", reverse)
        for n, w, z in zip(("bar_gate", "bar_x", "bar_h0"), wants, sizes):
            close(back(bars[n]), w, z, T, "value", dtype, state=n == "bar_h0")


@pytest.mark.gpu
def test_planes_whose_offsets_pass_32_bits(gpu):
    """Two sequences, rows or steps more than 2^31 elements apart."""
    import torch
    far = (1 << 31) + 40
    buffer = torch.empty(far + 4096, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(6)

    def apart(shape, strides):
        t = buffer.as_strided(shape, strides)
        t.copy_(torch.randn(shape, generator=g, device=gpu))
        return t
    # sequences apart, then steps apart
    for strides in ((far, 24, 1), (24, far, 1)):
        x = apart((2, 2, 24), strides)
        gate = torch.rand(2, 2, 24, generator=g, device=gpu).bfloat16()
        near, want = x.contiguous(), torch.empty(2, 2, 24, dtype=torch.bfloat16, device=gpu)
        hawk.run(hawk.stages.recurrence(), gate=gate, x=near, h=want)
        hawk.run(hawk.stages.recurrence(), gate=gate, x=x, h=x)
        assert torch.equal(x, want)
        hawk.run(hawk.stages.recurrence().vjp, gate=gate, h=x, bar_h=near, bar_x=near)
        bar, again = torch.empty_like(want), x.clone()
        hawk.run(hawk.stages.recurrence().vjp, gate=gate, h=want, bar_h=again, bar_x=bar)
        hawk.run(hawk.stages.recurrence().vjp, gate=gate, h=want, bar_h=x, bar_x=x)
        assert torch.equal(x, bar)
    logits = apart((2, 300), (far, 1))
    near = logits.contiguous()
    target = torch.tensor([3, 299], device=gpu)
    out, want, lse = (torch.empty(2, device=gpu) for _ in range(3))
    hawk.run(hawk.stages.token_logp(), logits=near, target=target, logp=want, lse=lse)
    hawk.run(hawk.stages.token_logp(), logits=logits, target=target, logp=out)
    assert torch.equal(out, want)
    c, bar = torch.ones(2, device=gpu), torch.empty_like(near)
    hawk.run(hawk.stages.token_logp().vjp, logits=near, target=target, lse=lse, bar_logp=c, bar_logits=bar)
    hawk.run(hawk.stages.token_logp().vjp, logits=logits, target=target, lse=lse, bar_logp=c, bar_logits=logits)
    assert torch.equal(logits, bar)
    for width in (300, 301):
        x = apart((2, width), (far, 1))
        near = x.contiguous()
        hawk.run(hawk.stages.dropout(0.3), x=near, y=near, seed=5)
        hawk.run(hawk.stages.dropout(0.3), x=x, y=x, seed=5)
        assert torch.equal(x, near)


@pytest.mark.gpu
def test_a_stage_of_many_shapes_keeps_a_bounded_number_of_plans(gpu):
    import torch
    from hawk_amd import stages
    scan = hawk.stages.recurrence()
    for n in range(1, stages.PLANS + 60):
        x = torch.ones(1, n, 2, device=gpu)
        h = torch.empty_like(x)
        hawk.run(scan, gate=x, x=x, h=h)
        if n % 37 == 0:
            assert torch.equal(h[0, :, 0], torch.arange(1, n + 1, device=gpu, dtype=torch.float32))
    assert len(scan._plans) <= stages.PLANS
    # planes in another order, of another type, and with a plane left out
    h64 = torch.empty(1, 4, 2, dtype=torch.float64, device=gpu)
    ones = torch.ones_like(h64)
    hawk.run(scan, h=h64, x=ones, gate=ones, h0=None)
    assert torch.equal(h64[0, :, 1], torch.arange(1, 5, device=gpu, dtype=torch.float64))
    with pytest.raises(HawkError, match="'x' is not given"):
        hawk.run(scan, h=h64, x=None, gate=ones)


@pytest.mark.gpu
def test_stages_from_several_threads(gpu):
    """One stage, one stream, four threads: a call's launches and scratch stay together."""
    import threading

    import torch
    scan, loss_of = hawk.stages.recurrence(), hawk.stages.policy_loss()
    g = torch.Generator(device=gpu).manual_seed(12)
    work = []
    for k in range(4):
        T = 700 + 300 * k
        gate = torch.rand(2, T, 40, generator=g, device=gpu)
        x = torch.randn(2, T, 40, generator=g, device=gpu)
        logits = torch.randn(50 + k, 3000, generator=g, device=gpu)
        n = len(logits)
        planes = dict(logits=logits, target=torch.randint(0, 3000, (n,), generator=g, device=gpu),
                      old_logp=torch.full((n,), -9.0, device=gpu), advantage=torch.randn(n, generator=g, device=gpu))
        h, loss = torch.empty_like(x), torch.empty(1, device=gpu)
        hawk.run(scan, gate=gate, x=x, h=h)
        hawk.run(loss_of, loss=loss, **planes)
        work.append((gate, x, h, planes, loss))
    torch.cuda.synchronize()
    wrong = []

    def run(k):
        gate, x, want, planes, want_loss = work[k]
        for _ in range(40):
            h, loss = torch.empty_like(x), torch.empty(1, device=gpu)
            hawk.run(scan, gate=gate, x=x, h=h)
            hawk.run(loss_of, loss=loss, **planes)
            if not torch.equal(h, want) or not torch.equal(loss, want_loss):
                wrong.append(k)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_more_rows_than_one_run_of_the_loss_sum(gpu):
    import torch
    N, V = 70001, 5
    g = np.random.default_rng(8)
    logits = torch.from_numpy(g.normal(size=(N, V)).astype(np.float32)).to(gpu)
    target = torch.from_numpy(g.integers(0, V, N)).to(gpu)
    A = torch.from_numpy(g.normal(size=N).astype(np.float32)).to(gpu)
    logp, loss, old = torch.empty(N, device=gpu), torch.empty(1, device=gpu), torch.full((N,), -1.6, device=gpu)
    hawk.run(hawk.stages.policy_loss(), logits=logits, target=target, old_logp=old, advantage=A, logp=logp, loss=loss)
    want, _ = oracle_policy(back(logp), target.cpu().numpy(), back(old), back(A), None, np.full(N, 1.0 / N), (0.2, 0.2),
                            0.0, 1.0)
    # each row's loss errs by 8 u of itself, their sum in 64 bits by nothing, the cell by u
    assert abs(back(loss)[0] - want.sum()) <= 10 * 2.0 ** -24 * np.abs(want).sum()
    # pairs past one workgroup's
    P = 300
    offsets = torch.arange(0, 2 * P + 1, device=gpu) * 3
    n = 6 * P
    out = {k: torch.empty(m, device=gpu) for k, m in (("loss", 1), ("margin", P), ("logp", n))}
    hawk.run(hawk.stages.preference_loss(beta=0.5), logits=logits[:n], target=target[:n], offsets=offsets, **out)
    margin, total, _ = oracle_pairs(back(out["logp"]), target[:n].cpu().numpy(), np.zeros(n), offsets.cpu().numpy(),
                                    np.full(P, 1.0 / P), 0.5, 0.0)
    # six written log-probabilities a pair, each rounded by u of itself
    assert np.abs(back(out["margin"]) - margin).max() <= 2.0 ** -24 * (24 * 6 + 6 * np.abs(back(out["logp"])).max())
    assert abs(back(out["loss"])[0] - total) <= 2.0 ** -24 * (16 * (1 + total) + 0.5 * (24 * 6 + 6 * 10))
