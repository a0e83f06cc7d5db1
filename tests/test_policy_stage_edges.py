"""Linear attention, layer norm and sampling (``hawk.stages``) where their digits, their
planes' layouts and their launches end, against plain sums in 64 bits.

``u`` = 2^-24 is the most that one rounding to 24 bits is off, relative to the value.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import hawk_amd as hawk
from hawk_amd import HawkError, _core

U = 2.0 ** -24


def back(x):
    return x.double().cpu().numpy()


# -- linear attention --------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("S", [1, 13], ids=["cut", "whole"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_the_state_is_made_and_read_to_24_bits(gpu, dtype, S):
    """Two channels of the state that cancel: one made of the first token, one that entered.  From the
    second chunk on a result is their difference alone, whose error is that of the states' digits.

    Each channel has at most half of the magnitudes' sum M.  Its roundings: the token's factor, its product
    and that one's parts and sum (4), two a chunk for each of five chunks, two where segments are joined, the
    parts as it is read (1), six products added: 23.  A float16 result is a multiple of 2^-24."""
    import torch
    T, H, V = 130, 32, 16
    g = np.random.default_rng([S, len(dtype)])
    kind = getattr(torch, dtype)
    decay = np.float32(1 - 2.0 ** -8 * g.random(H))
    v = torch.zeros(S, T, H, V, dtype=kind)
    v[:, 0] = torch.from_numpy(g.uniform(0.5, 2, (S, H, V))).to(kind)
    first = back(v[:, 0])
    h0 = np.zeros((S, H, 2, V), np.float32)
    h0[:, :, 1] = first / decay.astype(np.float64)[:, None]
    q, k = torch.empty(S, T, H, 2, dtype=kind), torch.zeros(S, T, H, 2, dtype=kind)
    q[..., 0], q[..., 1], k[:, 0, :, 0] = 1, -1, 1
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    o = torch.empty_like(v)
    hawk.run(hawk.stages.linear_attention(), q=q, k=k, v=v, decay=torch.from_numpy(decay).to(gpu),
             h0=torch.from_numpy(h0).to(gpu), o=o)
    power = decay.astype(np.float64)[None, :] ** np.arange(T + 1)[:, None]           # (T + 1, H)
    made = power[None, :T, :, None] * first[:, None]
    entered = power[None, 1:, :, None] * h0[:, None, :, 1].astype(np.float64)
    off = np.abs(back(o) - (made - entered)) - (24 * U * (made + np.abs(entered)) + 2.0 ** -25)
    assert (off[:, 64:] <= 0).all(), off[:, 64:].max()


@pytest.mark.gpu
@pytest.mark.parametrize("S,T,K", [(100, 8192, 16), (1, 65536, 64)], ids=["whole", "cut"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_state_that_fades_slowly_is_off_by_roundings_of_either_sign(gpu, dtype, S, T, K):
    """Tokens of zeros: the state only decays, a factor a chunk (of 32 tokens at least) or a segment.  Each
    rounds every number, by u / sqrt(3) in the mean square, so the mean over a head's numbers errs by
    sqrt(n / (3 numbers)) u; six times that, and u for the factor of the last tokens, which are no whole chunk.
    A factor that is itself rounded moves all numbers the same way, by up to u for each of the n."""
    import torch
    decay = np.float32([1 - 2.0 ** -10, 1 - 2.0 ** -11, 1 - 2.0 ** -13, 1 - 2.0 ** -16])
    H = len(decay)
    plane = torch.zeros(K, dtype=getattr(torch, dtype), device=gpu).expand(S, T, H, K)
    g = np.random.default_rng(S)
    h0 = torch.from_numpy(g.uniform(1, 2, (S, H, K, K)).astype(np.float32)).to(gpu)
    for stage, planes in ((hawk.stages.linear_attention(), dict(h0=h0, last=torch.empty_like(h0))),
                          (hawk.stages.linear_attention().vjp, dict(bar_o=plane, bar_last=h0, bar_h0=torch.empty_like(h0)))):
        hawk.run(stage, q=plane, k=plane, v=plane, decay=torch.from_numpy(decay).to(gpu), **planes)
        left = back(planes.get("last", planes.get("bar_h0")))
        want = back(h0) * (decay.astype(np.float64) ** T)[None, :, None, None]
        off = (left / want - 1).mean((0, 2, 3))
        allowed = U * (1 + 6 * np.sqrt(T / 32 / (3 * S * K * K)))
        assert (np.abs(off) <= allowed).all(), (off / U, allowed / U)


@pytest.mark.gpu
@pytest.mark.parametrize("bounds", [(0, 5, 5, 40), (0, 300, 1700, 2000)], ids=str)
def test_packed_planes_have_no_sequence_stride(gpu, bounds):
    """The C entries' ``seq`` of a packed plane is not looked at: the bits of a job that has 0 there, and
    nothing is written where the strides would lead."""
    import torch
    S, T, H, K, V = len(bounds) - 1, bounds[-1], 2, 8, 12
    g = torch.Generator(device=gpu).manual_seed(T)
    stray = T * H * V                                           # S times this is allocated behind each plane
    width = {"q": K, "k": K, "v": V, "o": V, "bar_o": V, "bar_q": K, "bar_k": K, "bar_v": V}
    L, got = _core.lib(), []
    values = {n: torch.randn(T * H * width[n], generator=g, device=gpu) for n in ("q", "k", "v", "bar_o")}
    states = {n: torch.randn(S, H, K, V, generator=g, device=gpu) for n in ("h0", "bar_last")}
    for seq in (0, stray):
        job = _core.LinearAttentionJob()
        planes = {n: torch.full((T * H * w + S * stray,), 7.0, device=gpu) for n, w in width.items()}
        held = {**states, **{n: torch.zeros(S, H, K, V, device=gpu) for n in ("last", "bar_h0")},
                "decay": torch.tensor([0.9, 0.999], device=gpu), "offsets": torch.tensor(bounds, device=gpu)}
        for n, x in values.items():
            planes[n][:len(x)] = x
        for n, x in planes.items():
            at = getattr(job, n)
            at.data, at.seq, at.step, at.head = x.data_ptr(), seq, H * width[n], width[n]
        for n, x in held.items():
            setattr(job, n, x.data_ptr())
        job.seqs, job.steps, job.heads, job.keys, job.values = S, T, H, K, V
        job.scale, job.dtype, job.offsets64 = 0.5, 0, 1
        ref = ctypes.byref(job)
        for vjp, entry in ((0, L.hk_linear_attention), (1, L.hk_linear_attention_vjp)):
            room = torch.empty(max(1, L.hk_linear_attention_scratch_bytes(ref, vjp)), dtype=torch.uint8, device=gpu)
            assert entry(ref, room.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
            torch.cuda.synchronize()
        got.append({**planes, **held})
    for n, w in width.items():
        assert torch.equal(got[0][n], got[1][n]) and (got[1][n][T * H * w:] == 7).all(), n
    assert all(torch.equal(got[0][n], got[1][n]) for n in ("last", "bar_h0"))
    assert torch.isfinite(got[1]["o"]).all() and (got[1]["o"][:T * H * V] != 7).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_numbers_up_to_the_types_largest_are_numbers(gpu, dtype):
    """A state, a token's share of one and a product q . k above the largest bfloat16, read with small factors:
    results of some 1e35, in three of four cases of one term, within 8 roundings to 24 bits or 2^-16."""
    import torch
    T, V, kind = 70, 16, getattr(torch, dtype)
    most = (2 - 2.0 ** -8) * 2.0 ** 127                         # halfway from there to 2^128
    small = 2.0 ** -10
    z = lambda w: torch.zeros(1, T, 1, w, dtype=torch.float64)  # noqa: E731
    stage, one = hawk.stages.linear_attention(), torch.ones(1, device=gpu)

    def results(q, k, v, **planes):
        o = torch.empty(1, T, 1, V, dtype=kind, device=gpu)
        hawk.run(stage, q=q.to(gpu, kind), k=k.to(gpu, kind), v=v.to(gpu, kind), decay=one, o=o, **planes)
        return back(o)[0, :, 0]

    r = {"float32": 8 * U, "bfloat16": 2.0 ** -8 + 2.0 ** -16}[dtype]
    q, k, v = z(2), z(2), z(V)
    q[..., 0] = small
    for x in (most, -(2 - 2.0 ** -23) * 2.0 ** 127):
        h0 = torch.zeros(1, 1, 2, V, device=gpu)
        h0[..., 0, :] = x
        got = results(q, k, v, h0=h0)
        assert (np.abs(got - x * small) <= r * abs(x) * small).all()
    # q . k, of two numbers that bfloat16 has, of which the product is above its largest
    q, k, v = z(2), z(2), z(V)
    big = 1.453125 * 2.0 ** 127
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 1.375, big, small
    got, want = results(q, k, v), 1.375 * big * small
    assert most < 1.375 * big < 2.0 ** 128 and (np.abs(got - want) <= r * want).all()
    # a token's v, and its sum with what entered
    if dtype == "float32":
        q, k, v = z(2), z(2), z(V)
        q[..., 0], k[:, 0, :, 0], v[:, 0] = 1, small, most
        assert (np.abs(results(q, k, v) - most * small) <= r * most * small).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(3, 1, 2, 128, 128), (2, 3, 2, 72, 100), (1, 8, 1, 256, 256), (2, 2, 3, 129, 65), (5, 1, 4, 65, 256),
                                   (1, 8, 2, 64, 64), (1, 9, 1, 256, 256), (2, 9, 3, 129, 65)], ids=str)
def test_a_few_tokens_of_wide_heads(gpu, shape, dtype):
    """Up to 8 tokens as they stand: a state takes two roundings a token, a result K / 16 + 16 sums and three
    roundings more.  Nine go by way of chunks, whose products are taken to 2^-16 (16-bit planes) or 2^-23."""
    import torch
    S, T, H, K, V = shape
    g, kind = np.random.default_rng(shape), getattr(torch, dtype)
    q, k, v = (torch.from_numpy(g.normal(size=(S, T, H, w))).to(kind) for w in (K, K, V))
    h0 = torch.from_numpy(g.normal(size=(S, H, K, V))).float()
    decay = np.float32([0.9, 1.0, 0.0, 0.97])[:H]
    gain, scale = decay.astype(np.float64)[None, :, None, None], 0.37
    state = back(h0)
    mass, want, size = np.abs(state), [], []
    for t in range(T):
        kv = back(k[:, t])[..., :, None] * back(v[:, t])[..., None, :]
        state, mass = gain * state + kv, gain * mass + np.abs(kv)
        want.append(scale * np.einsum("shk,shkv->shv", back(q[:, t]), state))
        size.append(scale * np.einsum("shk,shkv->shv", np.abs(back(q[:, t])), mass))
    want, size = np.stack(want, 1), np.stack(size, 1)
    r = {"float32": U, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    if T <= 8:
        p_state = (2 * T + 2) * U
        p = p_state + (K / 16 + 19) * U
    else:
        p_state = 2.0 ** -23 + ((max(K, V) + 64) / 4 + 65) * U
        p = p_state + (0 if dtype == "float32" else 2.0 ** -16)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    stage, decay = hawk.stages.linear_attention(scale=scale), torch.from_numpy(decay).to(gpu)
    for held in (False, True):                                  # the state beside what entered, or over it
        o, h = torch.empty_like(v), h0.to(gpu)
        last = h if held else torch.full_like(h, 7.0)
        hawk.run(stage, q=q, k=k, v=v, decay=decay, o=o, h0=h, last=last)
        assert (np.abs(back(o) - want) <= p * size * (1 + r) + r * np.abs(want) + 2.0 ** -25).all()
        assert (np.abs(back(last) - state) <= p_state * mass).all()
        h = h0.to(gpu)
        hawk.run(stage, q=q, k=k, v=v, decay=decay, h0=h, last=h)
        assert torch.equal(h, last)                             # without results


# -- layer norm ------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(12,), (2, 3), (300000,), ()], ids=str)
def test_rows_without_columns_have_no_mean(gpu, lead):
    import torch
    stage, N = hawk.stages.layer_norm(), int(np.prod(lead))
    x = torch.empty(*lead, 0, device=gpu)
    mean, rstd = torch.full((2, N), 7.0, device=gpu)
    hawk.run(stage, x=x, y=torch.empty_like(x), mean=mean, rstd=rstd)
    assert torch.isnan(mean).all() and torch.isnan(rstd).all()
    mean.fill_(7)
    hawk.run(stage, x=x, mean=mean)
    assert torch.isnan(mean).all()
    hawk.run(stage, x=x, y=torch.empty_like(x))
    none = torch.empty(0, device=gpu)
    hawk.run(stage.vjp, x=x, mean=mean, rstd=rstd, bar_y=x, bar_x=torch.empty_like(x), bar_weight=none, bar_bias=torch.empty(0, device=gpu))


@pytest.mark.gpu
def test_the_sums_over_rows_of_more_columns_than_a_launch_has_threads_for(gpu):
    """One row at mean 0 and rstd 1: bar_bias is bar_y, bar_weight its product with x, which float32 holds whole."""
    import torch
    C = (1 << 26) + 53
    g = torch.Generator(device=gpu).manual_seed(3)
    x, bar = (torch.randn(1, C, generator=g, device=gpu, dtype=torch.bfloat16) for _ in range(2))
    mean, rstd = torch.zeros(1, device=gpu), torch.ones(1, device=gpu)
    bw, bb = torch.full((2, C), 7.0, device=gpu)
    hawk.run(hawk.stages.layer_norm().vjp, x=x, mean=mean, rstd=rstd, bar_y=bar, bar_weight=bw, bar_bias=bb)
    assert torch.equal(bb, bar[0].float()) and torch.equal(bw, bar[0].float() * x[0].float())


def test_the_layer_norm_entries_refuse_rows_that_lie_in_two_ways():
    L, n = _core.lib(), _core.LayerNormJob()
    ref = ctypes.byref(n)
    n.x = n.y = n.bar_y = n.bar_x = n.mean = n.rstd = 1 << 20
    n.rows, n.cols, n.x_stride, n.y_stride, n.bar_y_stride, n.bar_x_stride = 3, 8, 8, 9, 8, 8
    for entry in (L.hk_layer_norm, L.hk_layer_norm_vjp):
        assert entry(ref, None, None) == 1 and b"row distance" in L.hk_last_error()
    n.y = None
    for x, bar_y in ((8, 9), (9, 8)):
        n.x_stride, n.bar_y_stride = x, bar_y
        assert L.hk_layer_norm_vjp(ref, None, None) == 1 and b"row distance" in L.hk_last_error()


@pytest.mark.gpu
def test_an_output_over_an_input_lies_as_it_does(gpu):
    """At one address with other strides a call would write over what it has not read yet."""
    import torch
    room = torch.zeros(400, device=gpu)
    near, far = room.as_strided((5, 8), (8, 1)), room.as_strided((5, 8), (9, 1))
    block = torch.zeros(2, 4, 8, device=gpu)
    turned = block, block.as_strided((2, 4, 8), (32, 1, 4))
    other, m = torch.zeros(5, 8, device=gpu), torch.ones(5, device=gpu)
    target, s = torch.zeros(5, dtype=torch.int64, device=gpu), hawk.stages
    gate = torch.zeros(2, 4, 8, device=gpu)
    norm, logp, drop, scan = s.layer_norm(), s.token_logp(), s.dropout(0.5), s.recurrence()
    calls = [(norm, lambda a, b: dict(x=a, y=b)),
             (norm.vjp, lambda a, b: dict(x=a, bar_y=other, bar_x=b, mean=m, rstd=m)),
             (norm.vjp, lambda a, b: dict(x=other, bar_y=a, bar_x=b, mean=m, rstd=m)),
             (logp.vjp, lambda a, b: dict(logits=a, target=target, lse=m, bar_logp=m, bar_logits=b)),
             (drop, lambda a, b: dict(x=a, y=b, seed=1)),
             (drop, lambda a, b: dict(x=other, residual=a, y=b, seed=1)),
             (scan, lambda a, b: dict(gate=gate, x=a, h=b)),
             (scan, lambda a, b: dict(gate=a, x=gate, h=b)),
             (scan.vjp, lambda a, b: dict(gate=gate, h=gate, bar_h=a, bar_gate=b))]
    for stage, planes in calls:
        a, b = turned if "gate" in stage.planes else (near, far)
        for one, two in ((a, b), (b, a)):
            with pytest.raises(HawkError, match="lies in two ways"):
                hawk.run(stage, **planes(one, two))
            with pytest.raises(HawkError, match="lies in two ways"):
                stage.prepare(**planes(one, two))
            hawk.run(stage, **planes(one, one))                 # over the input itself, as before
    hawk.run(norm, x=near[:1], y=far[:1])                       # one row has no distance


@pytest.mark.gpu
def test_layer_norms_outputs_are_tensors_of_their_own(gpu):
    import torch
    stage = hawk.stages.layer_norm()
    x, y, m, r, w = torch.ones(5, 1, device=gpu), *(torch.ones(5, 1, device=gpu), *torch.ones(2, 5, device=gpu)), torch.ones(1, device=gpu)
    for planes in (dict(x=x, mean=m, rstd=m), dict(x=x, y=y, mean=y[:, 0]), dict(x=x, y=y, rstd=y[:, 0]), dict(x=x, mean=x[:, 0]),
                   dict(x=x, rstd=x[:, 0])):
        with pytest.raises(HawkError, match="one tensor"):
            hawk.run(stage, **planes)
    for bars in (dict(bar_x=m[:, None]), dict(bar_x=r[:, None]), dict(bar_x=y, bar_weight=y[0]), dict(bar_x=y, bar_bias=y[0])):
        with pytest.raises(HawkError, match="one tensor"):
            hawk.run(stage.vjp, x=x, mean=m, rstd=r, bar_y=x, **bars)
    hawk.run(stage, x=x, y=x, mean=m, rstd=r)
    hawk.run(stage.vjp, x=x, mean=m, rstd=r, bar_y=y, bar_x=x, bar_weight=w)


# -- sampling ----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("V", [131072, 1000003, 1 << 20, 1 << 22])
@pytest.mark.parametrize("low", [25.0, 28.5, 30.5])
def test_a_flat_tail_far_below_the_highest_logit(gpu, V, low):
    """One token above V - 1 equal ones.  A weight is a whole number of units of 2^-shift, so many that V of them
    stay below 2^63, and half a unit off: sums by E = V 2^-(shift + 1) of the highest weight, shares of the whole
    by 2 E, its logarithm by E.  The weights' polynomial adds 2^-48."""
    import torch
    shift = min(51, 63 - V.bit_length())
    E = V * 2.0 ** -(shift + 1) + 2.0 ** -48
    at, w = V // 3, float(np.exp(-np.float64(np.float32(low))))
    x = torch.full((1, V), -low, device=gpu)
    x[0, at] = 0
    whole = 1 + w * (V - 1)
    tail = w * (V - 1) / whole
    u = torch.from_numpy(np.array([0.0, tail / 5, tail / 3 + 2.5 * E, 0.5, 1 - 2 * tail / 3 - 2.5 * E, 1 - tail / 3, 1 - 2.0 ** -50])).to(gpu)
    N = len(u)
    for filters in ({}, dict(min_p=1e-30), dict(top_k=V - 1)):
        token, logp = torch.empty(N, dtype=torch.int64, device=gpu), torch.empty(N, device=gpu)
        hawk.run(hawk.stages.sample(**filters), logits=x.expand(N, V), u=u, token=token, logp=logp)
        got = token.cpu().numpy()
        upto = (w * (got + 1) + (got >= at) * (1 - w)) / whole  # the whole's share up to the token, and before it
        before = upto - np.where(got == at, 1, w) / whole
        assert (before <= back(u) + 2 * E).all() and (upto >= back(u) - 2 * E).all(), (got, back(u))
        want = np.where(got == at, 0, -np.float64(np.float32(low))) - np.log(whole)
        assert (np.abs(back(logp) - want) <= E + U * np.abs(want)).all()
        assert got[3] == at


# -- options -----------------------------------------------------------------------------------

@pytest.mark.parametrize("big", [3.5e38, 1e300, 1 << 200, 1 << 2000])
def test_numbers_past_float32_are_refused(big):
    with pytest.raises(HawkError, match="scale="):
        hawk.stages.linear_attention(scale=-big)
    with pytest.raises(HawkError, match="eps="):
        hawk.stages.layer_norm(eps=big)
    hawk.stages.linear_attention(scale=-3.4e38), hawk.stages.layer_norm(eps=3.4e38), hawk.stages.layer_norm(eps=0)
