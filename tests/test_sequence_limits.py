"""The selective scan where its forms could part from the recurrence: rows cut into segments, numbers of states that are padded,
infinities, growing states.  Against the recurrence in 64 bits, with an error bound that decays with the states.

The bound.  `recurrence` carries along with every value its magnitude (the same formulas with every term's absolute value) and a bound
on its error in float32.  U = 2^-24 is half a step; exp2, log2 and reciprocals of the hardware are off by 2 U.  raw = dt + dt_bias is off
by |raw| U, e^raw by another (2 |raw| + 2) U, the logarithm and its correction by 14 U at most: d by (3 |raw| + 16) U.  The exponent d A
has a constant and a product more (4 U), its exp2 3 U; where a row is cut, d is first summed over a segment and a stretch of segments (at
most SUMMED additions, U each).  A state is what is kept of the one before, with that one's error, and its own terms; a cut row adds it up
twice.  So an error lives as long as the state it is in, and the bound does not grow with the row.
"""
import struct

import numpy as np
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from metaworld_amd import sequence

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U, SUMMED = 2.0 ** -24, 300
NAMES = ("y", "last", "du", "ddt", "dA", "dB", "dC", "dD", "dz", "dbias", "dstate")


def recurrence(u, dt, A, B, C, D, z, bias, state, reset, lengths, dy, dlast, keep_state=lambda t, h: h):
    """{name: (value, bound on its error in float32)}, token by token, all rows at once"""
    batch, time, width = u.shape
    states = A.shape[1]
    ends = lengths.long() if lengths is not None else torch.full((batch,), time)
    reset = reset if reset is not None else torch.zeros(batch, time, dtype=torch.bool)
    raw = dt + bias
    d = torch.logaddexp(raw, torch.zeros_like(raw))
    rel_d = (3 * raw.abs() + 16) * U
    sig = torch.sigmoid(z)
    gate = z * sig
    gate_rel = (2 * z.abs() + 9) * U
    slope, slope_err = sig * (1 + z * (1 - sig)), sig * (1 + z.abs()) * (4 * z.abs() + 16) * U
    zero = torch.zeros((), dtype=torch.float64)
    h, hm, he = state.clone(), state.abs(), torch.zeros_like(state)
    out = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in zip(NAMES, (u, state, u, dt, A, B, C, D, z, bias, state))}
    tape = []
    for t in range(time):
        on = (t < ends)[:, None]
        a = torch.exp(d[:, t, :, None] * A)
        rel_a = d[:, t, :, None] * A.abs() * (rel_d[:, t, :, None] + (SUMMED + 4) * U) + 3 * U
        fresh = reset[:, t, None, None]
        keep, km, ke = (torch.where(fresh, zero, v) for v in (a * h, a * hm, a * he + a * hm * rel_a))
        x = (d[:, t] * u[:, t])[..., None] * B[:, t, None]
        new, nm = keep + x, km + x.abs()
        ne = ke + x.abs() * (rel_d[:, t, :, None] + 3 * U) + 3 * U * nm
        o, om = (new * C[:, t, None]).sum(-1) + D * u[:, t], (nm * C[:, t, None].abs()).sum(-1) + (D * u[:, t]).abs()
        oe = (ne * C[:, t, None].abs()).sum(-1) + (states + 4) * U * om
        out["y"][0][:, t] = torch.where(on, o * gate[:, t], zero)
        out["y"][1][:, t] = torch.where(on, (oe + om * gate_rel[:, t]) * gate[:, t].abs(), zero)
        h, hm, he = (torch.where(on[..., None], n, v) for n, v in ((keep_state(t, new), h), (nm, hm), (ne, he)))
        tape.append((on, a, rel_a, fresh, keep, km, ke, new, nm, ne, o, om, oe))
    out["last"] = h, he
    if dy is None:
        return out
    g, gm, ge = dlast.clone(), dlast.abs(), torch.zeros_like(dlast)
    adds = {n: torch.zeros_like(out[n][0]) for n in ("dA", "dD", "dbias")}           # magnitudes: a sum over all tokens adds as many roundings
    for t in range(time - 1, -1, -1):
        on, a, rel_a, fresh, keep, km, ke, new, nm, ne, o, om, oe = tape[t]
        on3, dt_, rd, Bt, Ct, ut = on[..., None], d[:, t], rel_d[:, t], B[:, t, None], C[:, t, None], u[:, t]
        dyt = torch.where(on, dy[:, t], zero)
        do = dyt * gate[:, t]
        dom, doe = do.abs(), do.abs() * gate_rel[:, t]
        G, Gm = g + do[..., None] * Ct, gm + dom[..., None] * Ct.abs()
        Ge = ge + doe[..., None] * Ct.abs() + 3 * U * Gm
        live = [torch.where(on3, v, zero) for v in (G, Gm, Ge)]
        both = lambda v, m, e, over: ((v).sum(over), (e + 40 * U * m).sum(over))         # a sum over channels or states, by lanes, waves and blocks
        du_ = dt_ * ut

        def put(name, value, error):
            out[name][0][:, t], out[name][1][:, t] = torch.where(on.view(batch, *[1] * (value.dim() - 1)), value, zero), torch.where(on.view(batch, *[1] * (value.dim() - 1)), error, zero)
        put("dz", dyt * o * slope[:, t], dyt.abs() * (oe * slope[:, t].abs() + om * (slope_err[:, t] + 4 * U)))
        put("dC", *both(do[..., None] * new, dom[..., None] * nm, dom[..., None] * ne + doe[..., None] * nm, 1))
        put("dB", *both(live[0] * du_[..., None], live[1] * du_.abs()[..., None], live[2] * du_.abs()[..., None] + live[1] * (du_.abs() * (rd + U))[..., None], 1))
        gB, gBm, gBe = ((x * y).sum(-1) for x, y in zip(live, (Bt, Bt.abs(), Bt.abs())))
        put("du", D * do + dt_ * gB, D.abs() * doe + dt_ * (gBe + gBm * (rd + (states + 4) * U)) + 4 * U * (D.abs() * dom + dt_ * gBm))
        gk, gkm, gke = live[0] * keep, live[1] * km, live[2] * km + live[1] * ke
        dd, ddm = ut * gB + (gk * A).sum(-1), ut.abs() * gBm + (gkm * A.abs()).sum(-1)
        dde = ut.abs() * gBe + (gke * A.abs()).sum(-1) + (states + 10) * U * ddm
        s = torch.sigmoid(raw[:, t])
        draw, drawm, drawe = dd * s, ddm * s, dde * s + ddm * s * (3 * raw[:, t].abs() + 8) * U
        draw, drawm, drawe = (torch.where(on, v, zero) for v in (draw, drawm, drawe))
        put("ddt", draw, drawe)
        for name, v, m, e in (("dbias", draw, drawm, drawe), ("dD", do * ut, dom * ut.abs(), doe * ut.abs()),
                              ("dA", gk * dt_[..., None], gkm * dt_[..., None], gke * dt_[..., None] + gkm * (dt_ * (rd + 4 * U))[..., None])):
            v, m, e = (torch.where(on.view(batch, *[1] * (v.dim() - 1)), x, zero).sum(0) for x in (v, m, e))
            out[name] = out[name][0] + v, out[name][1] + e
            adds[name] = adds[name] + m
        cg, cm, ce = (torch.where(fresh, zero, v) for v in (a * G, a * Gm, a * Ge + a * Gm * rel_a))
        g, gm, ge = (torch.where(on3, n, v) for n, v in ((cg, g), (cm, gm), (ce, ge)))
    out["dstate"] = g, ge
    for name, m in adds.items():
        out[name] = out[name][0], out[name][1] + (batch * time + 40) * U * m
    return out


def beyond(got, want, error):
    """how far off, in tolerances: the bound, with a twentieth for terms of second order, and the rounding of the output's type.  What passes through
    numbers below float32's smallest normal one, 2^-126, is off by 2^-150 an operation there: together, with the factors that follow, under 2^-126 as
    long as operations times factors stay under 2^24 (at most 500 tokens x 32 states, factors under 100, that decay from there)"""
    kind, g = got.dtype, got.detach().double().cpu()
    error = 1.05 * error + 2.0 ** -126
    tol = error + torch.finfo(kind).eps / 2 * (want.abs() + error) + torch.finfo(kind).tiny * torch.finfo(kind).eps
    return (g - want).abs() / tol


def rand(gen, *shape, scale=1.0, kind=torch.float64):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(kind).double()


def inputs(seed, batch, time, width, states, kind, slow=2e-3):
    """rates from `slow` to 4 and steps around 0.1: memories of a few to some thousand tokens"""
    gen = torch.Generator().manual_seed(seed)
    u, dt, z, B, C = (rand(gen, batch, time, n, kind=kind) for n in (width, width, width, states, states))
    A = -torch.exp(torch.rand((width, states), generator=gen, dtype=torch.float64) * (np.log(4) - np.log(slow)) + np.log(slow)).float().double()
    D, bias, state = rand(gen, width, kind=torch.float32), (rand(gen, width, scale=0.5) - 2.2).float().double(), rand(gen, batch, width, states, kind=torch.float32)
    dy, dlast = rand(gen, batch, time, width, kind=kind), rand(gen, batch, width, states, kind=torch.float32)
    return (u, dt * 0.5, A, B, C, D, z, bias, state), dy, dlast, gen


def on_gpu(ins, kind, grad=False):
    return [t.to("cuda", kind if k in (0, 1, 3, 4, 6) else torch.float32).requires_grad_(grad) for k, t in enumerate(ins)]


def gpu_or_none(*all_):
    return [t.cuda() if t is not None else None for t in all_]


# ---- values and gradients within the bound ----
@gpu
@pytest.mark.parametrize("batch,time,width,states", [(1, 700, 70, 16), (2, 1500, 33, 4), (1, 500, 130, 32), (2, 90, 256, 16), (3, 50, 192, 7), (2, 60, 128, 32), (2, 70, 250, 20)])
def test_scan_within_the_decaying_bound(batch, time, width, states):
    """rows cut into segments, blocks of one to four waves, more than 16 states in two pairs of waves"""
    ins, dy, dlast, gen = inputs(time + width, batch, time, width, states, torch.float32)
    few = torch.rand((batch, time), generator=gen) < 2.0 / time
    ends = torch.randint(time // 2, time, (batch,), generator=gen, dtype=torch.int32)
    for reset, lengths in ((None, None), (few, ends)):
        want = recurrence(*ins, reset, lengths, dy, dlast)
        leaves = on_gpu(ins, torch.float32, True)
        r, n = gpu_or_none(reset, lengths)
        y, last = sequence.selective_scan(*leaves[:8], state=leaves[8], reset=r, lengths=n)
        grads = torch.autograd.grad((y, last), leaves, (dy.float().cuda(), dlast.float().cuda()))
        for name, got in zip(NAMES, (y, last, *grads)):
            off = beyond(got, *want[name])
            assert off.max() <= 1, f"{name}: {int((off > 1).sum())} of {off.numel()} values off, by up to {float(off.max()):.3g} of the tolerance"


@pytest.mark.parametrize("batch,time,width,states", [(1, 700, 70, 16), (2, 1500, 33, 4)])
def test_the_bound_tells_a_state_of_fewer_bits(batch, time, width, states):
    """the mistakes are planted in the recurrence itself: its states, or every 48th of them (what a segment begins with), or what a segment begins with
    left out by a thousandth; float32 states pass"""
    ins, *_ = inputs(time + width, batch, time, width, states, torch.float32)
    want = recurrence(*ins, None, None, None, None)

    def off(keep):
        got = recurrence(*ins, None, None, None, None, keep_state=keep)
        return [float(beyond(got[n][0].float(), *want[n]).max()) for n in ("y", "last")]
    at_borders = lambda f: lambda t, h: f(h) if t % 48 == 47 else h
    assert max(off(lambda t, h: h.float().double())) <= 1
    assert off(lambda t, h: h.bfloat16().double())[0] > 1
    assert off(at_borders(lambda h: h.bfloat16().double()))[0] > 1
    assert off(at_borders(lambda h: h * 0.999))[0] > 1


# ---- recorded or not ----
@gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.float16])
@pytest.mark.parametrize("batch,time,width,states", [(4, 1000, 600, 12), (6, 1000, 768, 12), (2, 1000, 600, 20), (3, 700, 340, 9)])
def test_recording_changes_no_bit_of_cut_rows(kind, batch, time, width, states):
    """numbers of states whose padding differs with recording, at sizes where the number of chains over the segments, so padded, would lie on both sides of a limit"""
    gen = torch.Generator(device="cuda").manual_seed(time + width + states)
    r = lambda *s, k=kind: torch.randn(s, generator=gen, device="cuda").to(k)
    args = [r(batch, time, width), r(batch, time, width) - 2, -torch.rand(width, states, generator=gen, device="cuda"), r(batch, time, states), r(batch, time, states)]
    state = r(batch, width, states, k=torch.float32)
    with torch.no_grad():
        y, last = sequence.selective_scan(*args, state=state)
    again, last2 = sequence.selective_scan(*[t.requires_grad_() for t in args], state=state)
    assert torch.equal(y, again) and torch.equal(last, last2)


# ---- growing states ----
@gpu
@pytest.mark.parametrize("at,count,step,start", [(40, 8, 12.0, 1e-20), (40, 8, 17.0, 1e-38), (200, 8, 12.0, 1e-20), (33, 60, 1.5, 1e-20), (40, 8, 17.0, 1e-20)])
@pytest.mark.parametrize("width,states", [(20, 4), (70, 9)])
def test_states_that_grow_in_a_cut_row(width, states, at, count, step, start):
    """rates above zero, no steps but `count` large ones: a segment's factor of up to 2^138 or 2^196 on a state of 1e-20 or 1e-38 is a number, and what
    passes the range (the last case) is an infinity, as token by token"""
    time = 400
    dt = torch.full((1, time, width), -20.0, dtype=torch.float64)
    dt[:, at:at + count] = step
    u, C = torch.zeros(1, time, width, dtype=torch.float64), torch.ones(1, time, states, dtype=torch.float64)
    A = torch.linspace(-1, 1, width * states, dtype=torch.float64).view(width, states).float().double()
    small = torch.full((1, width, states), start, dtype=torch.float64).float().double()
    ins = (u, dt, A, C, C, torch.zeros(width, dtype=torch.float64), torch.full_like(u, 1.0), torch.zeros(width, dtype=torch.float64), small)
    dy, dlast = torch.zeros_like(u), small * 0.5
    want = recurrence(*ins, None, None, dy, dlast)
    leaves = on_gpu(ins, torch.float32, True)
    y, last = sequence.selective_scan(*leaves[:8], state=leaves[8])
    outputs = [y, last]
    most = torch.finfo(torch.float32).max
    passes = want["last"][0].max() > 2 * most
    if not passes:                   # (where a state passes the range, so do factors of gradients that do not)
        outputs += torch.autograd.grad((y, last), leaves, (dy.float().cuda(), dlast.float().cuda()))
    for name, got in zip(NAMES, outputs):
        value, error = want[name]
        inside = (value.abs() + 2 * error) < most / 2
        assert inside.any() and torch.isfinite(got.cpu()[inside]).all(), name
        assert (beyond(got, value, error)[inside] <= 1).all(), name
        assert torch.isposinf(got.cpu()[value - 2 * error > 2 * most]).all(), name
    assert passes == (step == 17.0 and start == 1e-20) and want["last"][0].max() > 1e18


# ---- infinities ----
def classes(t):
    t = t.detach().double().cpu()
    return torch.where(t.isnan(), 3.0, torch.where(t.isinf(), t.sign(), 0.0))


@gpu
@pytest.mark.parametrize("states,kind", [(1, TYPES[0]), (3, TYPES[1]), (5, TYPES[2]), (6, TYPES[0]), (9, TYPES[1]), (12, TYPES[0]), (12, TYPES[2]), (13, TYPES[1]), (18, TYPES[0]), (20, TYPES[2]), (24, TYPES[1]),
                                         (29, TYPES[2]), (31, TYPES[0]), (32, TYPES[1])])
@pytest.mark.parametrize("where", ["u", "dt"])
def test_infinite_inputs_give_infinities(where, states, kind):
    """an infinite input or step makes states infinite, until an episode begins: not the padding of a number of states, which counts for nothing, NaN"""
    batch, time, width = 2, 60, 40
    ins, dy, dlast, gen = inputs(states, batch, time, width, states, kind)
    u, dt, A, B, C, D, z, bias, state = ins
    B, C, z, u, D = B.abs() + 0.25, C.abs() + 0.25, z.abs() + 0.25, u.abs() + 0.25, D.abs()
    (u if where == "u" else dt)[0, 17, ::3] = float("inf")
    (u if where == "u" else dt)[1, 59, 1] = float("inf")
    reset = torch.zeros(batch, time, dtype=torch.bool)
    reset[0, 33] = True
    u, B, C, z, D = (t.to(kind).double() for t in (u, B, C, z, D))          # the numbers that the kernels get
    ins = (u, dt, A, B, C, D, z, bias, state)
    want = recurrence(*ins, reset, None, None, None)
    leaves = on_gpu(ins, kind)
    y, last = sequence.selective_scan(*leaves[:8], state=leaves[8], reset=reset.cuda())
    for name, got in (("y", y), ("last", last)):
        value, error = want[name]
        assert torch.equal(classes(got), classes(value)) and (classes(value) == 1).any(), name
        assert (beyond(got, value, error)[classes(value) == 0] <= 1).all(), name
    for t in leaves:
        t.requires_grad_()
    again = sequence.selective_scan(*leaves[:8], state=leaves[8], reset=reset.cuda())
    assert torch.equal(torch.nan_to_num(again[0]), torch.nan_to_num(y)) and torch.equal(torch.nan_to_num(again[1]), torch.nan_to_num(last))
    # where the formula has a number, padding makes it no NaN: gradients of the tokens before an infinite step, which wipes the states, and of those of the other episode
    grads = torch.autograd.grad(again, leaves, (dy.to("cuda", kind), dlast.float().cuda()))
    want = recurrence(*ins, reset, None, dy, dlast)
    for name, got in zip(NAMES[2:], grads):
        value, error = want[name]
        inside = torch.isfinite(value) & torch.isfinite(error)
        assert torch.isfinite(got.cpu()[inside]).all() and (beyond(got, value, error)[inside] <= 1).all(), name


@gpu
def test_an_infinite_state_stays_one_over_segments():
    """a state that is infinite decays to an infinity, also where a segment's factor as a whole is too small for a number"""
    batch, time, width, states = 1, 500, 30, 8
    ins, *_ = inputs(3, batch, time, width, states, torch.float32, slow=1.0)
    u, dt, A, B, C, D, z, bias, state = ins
    dt = torch.full_like(dt, 3.0)
    state[0, ::2] = float("inf")
    ins = (u, dt, A, B, C, D, z, bias, state)
    want = recurrence(*ins, None, None, None, None)
    leaves = on_gpu(ins, torch.float32)
    y, last = sequence.selective_scan(*leaves[:8], state=leaves[8])
    assert torch.equal(classes(last), classes(want["last"][0])) and (classes(last) == 1).any() and torch.equal(classes(y), classes(want["y"][0]))


@gpu
@pytest.mark.parametrize("time,end", [(13, 13), (24, 19)])
def test_an_infinity_in_a_rows_last_token_reaches_no_rate(time, end):
    """what comes behind a row's last token counts for nothing: dA has no term of the last state"""
    ins, dy, dlast, _ = inputs(5, 1, time, 9, 8, torch.float32)
    ins[0][0, end - 1, 4] = float("inf")
    dy[0, end - 1] = 0
    lengths = torch.tensor([end], dtype=torch.int32)
    want = recurrence(*ins, None, lengths, dy, dlast)["dA"]
    leaves = on_gpu(ins, torch.float32, True)
    out = sequence.selective_scan(*leaves[:8], state=leaves[8], lengths=lengths.cuda())
    dA, = torch.autograd.grad(out, leaves[2:3], (dy.float().cuda(), dlast.float().cuda()))
    assert torch.isfinite(want[0]).all() and (beyond(dA, *want) <= 1).all()


# ---- what the calls refuse ----
def test_tracing_is_refused():
    """a traced function would hold the outputs' memory and not the kernels that fill it"""
    w, A = torch.zeros(6, 4), -torch.ones(6, 3)
    x, s = torch.zeros(2, 5, 6), torch.zeros(2, 5, 3)
    held, h = torch.zeros(2, 3, 6), torch.zeros(2, 6, 3)
    for call in (lambda x: sequence.layer_norm(x), lambda x: sequence.causal_conv(x, w), lambda x: sequence.causal_conv_step(x[:, 0], w, state=held),
                 lambda x: sequence.selective_scan(x, x, A, s, s), lambda x: sequence.selective_scan_step(x[:, 0], x[:, 0], A, s[:, 0], s[:, 0], state=h)):
        for trace in (lambda: torch.jit.trace(call, (x,)), lambda: make_fx(call)(x)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                trace()


def test_a_recorded_scan_is_refused_where_its_backward_pass_would_be():
    """more of dB and dC than is counted: said by the forward pass that keeps states, before it launches anything"""
    lib = sequence.library()
    args = struct.pack("@26Q17q4i", *[64] * 11, 0, 0, *[64] * 13, 1 << 17, 1 << 10, *[0] * 14, 1 << 60, 8, 16, 1, 0)
    for f in (lib.mws_scan_backward, lib.mws_scan_forward):
        assert f(args, None) == -1 and "count" in lib.mws_last_error().decode()
