"""AdamW over many tensors (xdfm_adamw_*, models/adamw.py) against the formula in 64 bits.

m and v are two products and their sum in fp32, each rounded once: the reference forms them the same way on the CPU,
so they are equal in every bit, and so are the codes and scales of the 8-bit states (integer arithmetic from there).
p: u = 2^-24 per rounding.  step * m / (sqrt(v) * inv_root + eps) passes through seven operations, three of which
(root, division, and the reciprocal root of 1 - beta2^t) are good to 2 u at worst, and step and inv_root are each off
by a few u where they come from the device's step count (expm1 of a rounded logarithm): 24 u of the quotient in all;
(p - lr wd p) - that: 3 u of what is added up.
"""
import math

import numpy as np
import pytest
import torch

from recommenders_amd import _lib
from recommenders_amd.models.deeprec.models.adamw import AdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
RAGGED = [1, 0, 3, 63, 64, 65, 20, 4095, 4096, 4097, 130, 10007, 2, 257, 1 << 15]


# ------------------------------------------------------------------ reference
def random_bits(n, tensor, step, seed, start=0):
    """32 bits for each element: two rounds of xor-shift and multiplication, modulo 2^32."""
    M = 0xFFFFFFFF

    def mix(a, b):
        return ((a ^ (a >> 15)) * 0x9E3779B1 + b) & M

    key = mix(mix(mix(seed & M, seed >> 32), step & M), tensor)
    i = np.arange(start, start + n, dtype=np.uint64)
    a = ((i & M) + mix(key, 1)) * 0x9E3779B1 & M
    high = np.array([mix(key, 2 + int(h)) for h in np.unique(i >> 32)], dtype=np.uint64)[np.searchsorted(
        np.unique(i >> 32), i >> 32)]
    a = (a ^ (a >> 15) ^ high) * 0x6A09E667 & M
    return a ^ (a >> 16)


def encode(x, span, r20):
    """fp32 values -> (codes, scales): the definition in include/xdfm.h, in integers and 64-bit floats."""
    x = x.astype(np.float32)
    n = x.size
    codes, scales = np.zeros(n, dtype=np.uint8), np.zeros((n + 63) // 64, dtype=np.uint8)
    for b in range(len(scales)):
        part = slice(b * 64, min(n, b * 64 + 64))
        v = x[part].astype(np.float64)
        if not np.isfinite(v).all():
            scales[b] = 255
            continue
        top = np.abs(v).max()
        s = max(48, math.frexp(top)[1] - 1 + 127 if top else 0)
        scales[b] = s
        q = np.abs(v) * 2.0 ** (127 + span - s)
        low = np.maximum(np.frexp(q)[1] - 4, 0)
        k = (np.rint(q * 2.0 ** (20 - low)).astype(np.int64) + r20[part].astype(np.int64)) >> 20
        if span == 32:
            k = np.where((v > 0) & (k == 0), 1, k)
        c = k + 8 * low
        if span == 16:
            c = c + 128 * np.signbit(v)
        codes[part] = c
    return codes, scales


def decode(codes, scales, span):
    c = codes.astype(np.int64)
    size = c & 127 if span == 16 else c
    e, f = size >> 3, size & 7
    v = np.where(e > 0, (8.0 + f) * 2.0 ** np.maximum(e - 1, 0), f)
    s = np.repeat(scales.astype(np.int64), 64)[:c.size]
    v = np.where(s == 255, np.nan, v * 2.0 ** (np.minimum(s, 254) - 127.0 - span))
    return np.where(c >= 128, -v, v) if span == 16 else v


def moments(m, v, g, b1=0.9, b2=0.999):
    f = np.float32
    m, v, g = m.astype(f), v.astype(f), g.astype(f)
    return m * f(b1) + g * f(1 - b1), v * f(b2) + (g * g) * f(1 - b2)


def check_p(got, p, m, v, lr, wd, t, eps=1e-8, b1=0.9, b2=0.999):
    p, m, v = p.astype(np.float64), m.astype(np.float64), v.astype(np.float64)
    move = lr / (1 - b1 ** t) * m / (np.sqrt(v) / math.sqrt(1 - b2 ** t) + eps)
    wd = float(np.float32(wd))
    exp = p - lr * wd * p - move
    tol = 24 * U * np.abs(move) + 3 * U * (np.abs(p) + np.abs(exp)) + 1e-45
    assert (np.abs(got.astype(np.float64) - exp) <= tol).all(), float((np.abs(got - exp) / tol).max())


class Setup(object):
    """Tensors of the given sizes, each in an allocation of its own, at addresses off by `shift` elements."""

    def __init__(self, sizes, bits, gdtype=torch.float32, seed=0, shift=0, decay=None):
        rng = np.random.default_rng(seed)
        self.sizes, self.bits = sizes, bits
        scale = [10.0 ** rng.uniform(-5, 1) for _ in sizes]

        def put(a, dtype):
            t = torch.zeros((a.size + shift,), dtype=dtype, device="cuda")[shift:]
            t.copy_(torch.from_numpy(np.ascontiguousarray(a)))
            return t

        def normal(n):
            return rng.standard_normal(n).astype(np.float32)

        self.p = [put(0.05 * normal(n), torch.float32) for n in sizes]
        self.g = [put((s * normal(n) * (rng.random(n) > 0.1)).astype(np.float32), gdtype) for n, s in zip(sizes, scale)]
        m = [(0.3 * s * normal(n)).astype(np.float32) for n, s in zip(sizes, scale)]
        v = [(s * s * normal(n) ** 2 * 10.0 ** rng.uniform(-6, 0, n)).astype(np.float32) for n, s in zip(sizes, scale)]
        self.decay = decay if decay is not None else [0.01 * (k % 3) for k in range(len(sizes))]
        if bits == 32:
            self.m, self.v = [put(a, torch.float32) for a in m], [put(a, torch.float32) for a in v]
            more = {}
        else:
            half = [np.full(n, 1 << 19) for n in sizes]
            em, ev = [encode(a, 16, r) for a, r in zip(m, half)], [encode(a, 32, r) for a, r in zip(v, half)]
            self.m, self.v = [put(c, torch.uint8) for c, _ in em], [put(c, torch.uint8) for c, _ in ev]
            self.sm, self.sv = [put(s, torch.uint8) for _, s in em], [put(s, torch.uint8) for _, s in ev]
            more = dict(scale_m=self.sm, scale_v=self.sv)
        self.opt = AdamW(self.p, self.g, weight_decay=self.decay, state_bits=bits, slot_m=self.m, slot_v=self.v, **more)

    def host(self):
        """(p, g, m, v) per tensor as they stand: fp32 numpy, decoded."""
        out = []
        for k in range(len(self.sizes)):
            p, g = self.p[k].cpu().numpy(), self.g[k].float().cpu().numpy()
            m, v = self.m[k].cpu().numpy(), self.v[k].cpu().numpy()
            if self.bits == 8:
                m = decode(m, self.sm[k].cpu().numpy(), 16).astype(np.float32)
                v = decode(v, self.sv[k].cpu().numpy(), 32).astype(np.float32)
            out.append((p, g, m, v))
        return out

    def check_step(self, before, lr, t, seed=0, eps=1e-8):
        for k, (p, g, m, v) in enumerate(before):
            if not p.size:
                continue
            m, v = moments(m, v, g)
            check_p(self.p[k].cpu().numpy(), p, m, v, lr, self.decay[k], t, eps)
            gm, gv = self.m[k].cpu().numpy(), self.v[k].cpu().numpy()
            if self.bits == 32:
                assert np.array_equal(gm, m) and np.array_equal(gv, v), k
                continue
            r = random_bits(p.size, k, t, seed)
            for got, scale, exact, span, r16 in ((gm, self.sm[k], m, 16, r & 0xFFFF), (gv, self.sv[k], v, 32, r >> 16)):
                codes, scales = encode(exact, span, (r16 << 4) + 8)
                assert np.array_equal(scale.cpu().numpy(), scales), (k, span)
                same = got == codes
                # (-0 and 0 stand for one value)
                assert (same | ((got & 127) + (codes & 127) == 0)).all(), (k, span, int((~same).sum()))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_steps_match_the_formula(bits, gdtype, shift):
    s = Setup(RAGGED, bits, gdtype, seed=shift, shift=shift)
    for t in (1, 2, 3, 1000):
        before = s.host()
        print("adamw", bits, gdtype, shift, t, flush=True)
        s.opt.step(lr=0.01, step=t, seed=77)
        torch.cuda.synchronize()
        s.check_step(before, 0.01, t, seed=77)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [[1], [5000001], [7] * 700, [1 << 22, 1, 1 << 20]])
def test_few_and_many_tensors(bits, sizes):
    s = Setup(sizes, bits, seed=1)
    before = s.host()
    print("adamw", bits, len(sizes), flush=True)
    s.opt.step(lr=1e-3, step=9, seed=(5 << 32) + 1)
    torch.cuda.synchronize()
    if sum(sizes) > 1 << 20:  # the reference codes block by block: the ends and the middle of long tensors
        for k, (p, g, m, v) in enumerate(before):
            n = p.size
            for at in {0, n // 2 // 64 * 64, max(0, n - 1000) // 64 * 64}:
                part = slice(at, min(n, at + 2000))
                pm, pv = moments(m[part], v[part], g[part])
                check_p(s.p[k].cpu().numpy()[part], p[part], pm, pv, 1e-3, s.decay[k], 9)
                got = s.m[k].cpu().numpy()[part], s.v[k].cpu().numpy()[part]
                if bits == 32:
                    assert np.array_equal(got[0], pm) and np.array_equal(got[1], pv)
                else:
                    r = random_bits(pm.size, k, 9, (5 << 32) + 1, at)
                    whole = pm.size // 64 * 64 if part.stop < n else pm.size
                    cm, _ = encode(pm, 16, ((r & 0xFFFF) << 4) + 8)
                    cv, _ = encode(pv, 32, ((r >> 16) << 4) + 8)
                    assert (((got[0] == cm) | ((got[0] & 127) + (cm & 127) == 0))[:whole]).all()
                    assert (got[1] == cv)[:whole].all()
    else:
        s.check_step(before, 1e-3, 9, seed=(5 << 32) + 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_lies_beside_the_tensors_is_left_alone(bits):
    """Tensors carved out of one buffer with gaps of one element: the gaps keep their bytes."""
    sizes = [5, 64, 1, 200, 4099]
    dt = torch.float32 if bits == 32 else torch.uint8

    def carve(counts, dtype, fill):
        buf = torch.full((sum(counts) + len(counts) + 1,), fill, dtype=dtype, device="cuda")
        mask, views, at = torch.ones_like(buf, dtype=torch.bool), [], 1
        for n in counts:
            views.append(buf[at:at + n])
            mask[at:at + n] = False
            at += n + 1
        return buf, mask, views

    blocks = [(n + 63) // 64 for n in sizes]
    bufs = [carve(sizes, torch.float32, 7.0), carve(sizes, dt, 7), carve(sizes, dt, 7)]
    grads = [torch.randn(n, device="cuda") for n in sizes]
    more = {}
    if bits == 8:
        bufs += [carve(blocks, dt, 7), carve(blocks, dt, 7)]
        more = dict(scale_m=bufs[3][2], scale_v=bufs[4][2])
    opt = AdamW(bufs[0][2], grads, state_bits=bits, slot_m=bufs[1][2], slot_v=bufs[2][2], **more)
    for t in (1, 2):
        opt.step(lr=0.1, step=t)
    torch.cuda.synchronize()
    for buf, mask, views in bufs:
        assert (buf[mask] == 7).all()
        assert not any((v == 7).all() for v in views)


def test_states_from_the_beginning():
    """New states: zeros.  The first step moves each parameter by lr (bias corrections cancel), zeros stay zeros."""
    p = [torch.zeros(100, device="cuda") for _ in range(2)]
    g = [torch.full((100,), 3e-4, device="cuda"), torch.zeros(100, device="cuda")]
    for bits in (32, 8):
        q = [t.clone() for t in p]
        opt = AdamW(q, g, weight_decay=0.0, state_bits=bits)
        opt.step(lr=0.5, step=1, eps=1e-30)
        # m / sqrt(v) of one gradient: sqrt(1 - b2) (1 - b1) over their roundings; 24 u as in check_p, b's roundings 4 u
        assert (q[0] + 0.5).abs().max() <= 0.5 * 28 * U and (q[1] == 0).all()
        assert all((s == 0).all() for s in (opt.slot_m[1], opt.slot_v[1]))


def test_rounding_is_unbiased_and_differs_by_step_and_element():
    """One v of 1 and gradients of 0: v (1 - 0.001) lies 0.001 below a code; it is rounded down with the probability
    that the distance is of the step under 1 (a sixteenth): 1.6 %.  4096 x 64 draws: standard deviation of the mean
    0.0156 sqrt(p (1 - p) / n), 5 of them allowed.  To the nearest it would never move."""
    n, seeds = 4096, 64
    v0 = np.ones(n, dtype=np.float32)
    codes, scales = encode(v0, 32, np.full(n, 1 << 19))
    zero = torch.zeros(n, device="cuda")
    total, moved = 0.0, []
    for seed in range(seeds):
        v, sv = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()
        m, sm = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(64, dtype=torch.uint8, device="cuda")
        opt = AdamW([zero.clone()], [zero], state_bits=8, slot_m=[m], slot_v=[v], scale_m=[sm], scale_v=[sv])
        opt.step(lr=0.0, step=1, seed=seed)
        values = opt.read_state()[1].double()
        moved.append((values < 1).cpu().numpy())
        total += float(values.mean())
    step = 1 / 16  # the codes under 1 are 15/16 apart from it by a sixteenth
    prob = 0.001 / step
    sigma = step * math.sqrt(prob * (1 - prob) / (n * seeds))
    assert abs(total / seeds - 0.999) <= 5 * sigma + 2.0 ** -20
    moved = np.array(moved)
    per_element, per_seed = moved.sum(0), moved.sum(1)
    # binomial(64, 1.6 %) and binomial(4096, 1.6 %): no element or seed stands out by more than 8 deviations
    assert per_element.max() <= 64 * prob + 8 * math.sqrt(64 * prob)
    assert abs(per_seed - n * prob).max() <= 8 * math.sqrt(n * prob)


def test_second_moments_converge_and_never_vanish():
    """400 steps of beta2 = 0.9 on a constant gradient: v approaches g^2 as 1 - 0.9^400.  Each rounding is within a
    step (an eighth of the value at most); the mean over 64 x 64 elements is unbiased, its deviation an eighth / 64 /
    sqrt(1 - 0.9^2) at most, five of which are allowed; a value never reads as zero."""
    n = 4096
    g = torch.full((n,), 0.3, device="cuda")
    g[::2] = 1e-5  # far below the block's largest
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], [g], state_bits=8, weight_decay=0.0)
    for t in range(1, 401):
        opt.step(lr=0.0, step=t, beta1=0.9, beta2=0.9, seed=3)
    m, v = (x.double() for x in opt.read_state())
    assert (v > 0).all()
    big = slice(1, None, 2)
    allowed = 5 * 0.125 / math.sqrt(n / 2) / math.sqrt(1 - 0.81)
    assert abs(float(v[big].mean()) / 0.09 - 1) <= allowed
    assert abs(float(m[big].mean()) / 0.3 - 1) <= allowed


def test_values_and_codes_convert_both_ways():
    sizes = [1, 64, 65, 4097, 0, 9000]
    s = Setup(sizes, 8, seed=4)
    m, v = s.opt.read_state()
    at = 0
    for k, n in enumerate(sizes):
        assert np.array_equal(m[at:at + n].double().cpu().numpy(), decode(s.m[k].cpu().numpy(), s.sm[k].cpu().numpy(), 16))
        assert np.array_equal(v[at:at + n].double().cpu().numpy(), decode(s.v[k].cpu().numpy(), s.sv[k].cpu().numpy(), 32))
        at += n
    rng = np.random.default_rng(8)
    xm = (rng.standard_normal(at) * 10.0 ** rng.uniform(-9, 3, at)).astype(np.float32)
    xv = (10.0 ** rng.uniform(-30, 3, at)).astype(np.float32)
    xv[::7] = 0
    s.opt.write_state(torch.from_numpy(xm).cuda(), torch.from_numpy(xv).cuda())
    torch.cuda.synchronize()
    at = 0
    for k, n in enumerate(sizes):
        half = np.full(n, 1 << 19)
        for x, codes, scale, span in ((xm, s.m[k], s.sm[k], 16), (xv, s.v[k], s.sv[k], 32)):
            ec, es = encode(x[at:at + n], span, half)
            assert np.array_equal(scale.cpu().numpy(), es)
            got = codes.cpu().numpy()
            assert ((got == ec) | ((got & 127) + (ec & 127) == 0)).all() if span == 16 else np.array_equal(got, ec)
        at += n


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
def test_what_is_not_finite_stays_in_its_block(bad):
    """3e38: the square overflows, so v does."""
    n = 1000
    for bits in (32, 8):
        a, b = Setup([n], bits, seed=6), Setup([n], bits, seed=6)
        b.g[0][130] = bad
        for s in (a, b):
            s.opt.step(lr=0.01, step=5, seed=1)
            s.opt.step(lr=0.01, step=6, seed=1)
        torch.cuda.synchronize()
        block = np.arange(128, 192) if bits == 8 else np.array([130])
        keep = np.setdiff1d(np.arange(n), block)
        for x, y in ((a.p, b.p), (a.m, b.m), (a.v, b.v)):
            assert np.array_equal(x[0].cpu().numpy()[keep], y[0].cpu().numpy()[keep])
        if bits == 8:
            assert int(b.sv[0][2]) == 255 and (b.sv[0].cpu().numpy() == 255).sum() == 1
            m, v = b.opt.read_state()
            assert torch.isnan(v[128:192]).all() and torch.isfinite(v[192:]).all()
            assert torch.isnan(b.p[0][128:192]).all()


def test_step_count_from_the_device_equals_the_hosts():
    for bits in (32, 8):
        a, b = Setup([500, 70], bits, seed=2), Setup([500, 70], bits, seed=2)
        state = torch.tensor([1.0, 1.0, 0.0, 0.0], device="cuda")
        for t in range(1, 4):
            before = b.host()
            _lib.check(_lib.lib.xdfm_opt_advance(state.data_ptr(), 0.01, 0.9, 0.999, 1e-8, None,
                                                 torch.cuda.current_stream().cuda_stream))
            a.opt.step(lr=0.01, step=t, seed=9)
            b.opt.step(lr=0.01, opt_state=state, seed=9)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(a.m + a.v, b.m + b.v))
            b.check_step(before, 0.01, t, seed=9)


def test_a_step_count_that_was_not_advanced_counts_as_the_first():
    a, b = Setup([500, 70], 8, seed=2), Setup([500, 70], 8, seed=2)
    a.opt.step(lr=0.01, opt_state=torch.tensor([1.0, 1.0, 0.0, 0.0], device="cuda"), seed=9)
    b.opt.step(lr=0.01, opt_state=torch.tensor([0.9, 0.999, 0.0, 1.0], device="cuda"), seed=9)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a.p + a.m + a.v, b.p + b.m + b.v))
    for bad in (torch.zeros(3, device="cuda"), torch.zeros(4), torch.zeros(4, device="cuda", dtype=torch.float64),
                torch.zeros(8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="opt_state"):
            a.opt.step(lr=0.01, opt_state=bad)
    with pytest.raises(ValueError, match="either"):
        a.opt.step(lr=0.01)
    with pytest.raises(ValueError, match="elements of"):
        a.opt.read_state(torch.zeros(5, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("bits", [32, 8])
def test_the_class_refuses_tensors_that_do_not_fit(bits):
    n = 100
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for kw in (dict(params=[p.double()]), dict(grads=[g.double()]), dict(grads=[g[:50]]), dict(params=[p.repeat(2)[::2]]),
               dict(grads=[g.cpu()]), dict(slot_m=[p.half()]), dict(slot_v=[]), dict(weight_decay=[0.1, 0.1])):
        a = dict(params=[p], grads=[g], state_bits=bits)
        a.update(kw)
        with pytest.raises(ValueError):
            AdamW(**a)
    # the library's own refusals come through
    with pytest.raises(_lib.XdfmError, match="overlap"):
        AdamW([p, p], [g, g], state_bits=bits)
    with pytest.raises(_lib.XdfmError, match="gradient"):
        AdamW([p], [p], state_bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_replayed_with_two_optimizers(bits):
    """Two graphs of two optimizers, replayed in turn with eager steps of twins and waits between: equal in every bit."""
    pairs = [(Setup(RAGGED, bits, seed=k), Setup(RAGGED, bits, seed=k)) for k in (10, 11)]
    states = [[torch.tensor([1.0, 1.0, 0.0, 0.0], device="cuda") for _ in range(2)] for _ in pairs]

    def one(s, state):
        _lib.check(_lib.lib.xdfm_opt_advance(state.data_ptr(), 0.01, 0.9, 0.999, 1e-8, None,
                                             torch.cuda.current_stream().cuda_stream))
        s.opt.step(lr=0.01, opt_state=state, seed=4)

    graphs = []
    for (s, twin), (st, st2) in zip(pairs, states):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one(s, st)
        side.synchronize()
        one(twin, st2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one(s, st)
        graphs.append(graph)
    for k in range(4):
        for graph, (s, twin), (st, st2) in zip(graphs, pairs, states):
            graph.replay()
            one(twin, st2)
            if k % 2:
                torch.cuda.synchronize()
    torch.cuda.synchronize()
    for s, twin in pairs:
        assert all(torch.equal(x, y) for x, y in zip(s.p + s.m + s.v, twin.p + twin.m + twin.v))


def test_more_than_2_31_elements():
    """One tensor whose element offsets pass 32 bits of bytes in 32-bit states and 2^31 elements in 8-bit ones."""
    n = (1 << 31) + 200
    p = torch.zeros(n, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-150:] = 0.25
    g[:10] = 0.25
    opt = AdamW([p], [g], state_bits=8, weight_decay=0.0)
    opt.step(lr=0.5, step=1, seed=12)
    torch.cuda.synchronize()
    assert (p[:10] + 0.5).abs().max() <= 1e-5 and (p[-150:] + 0.5).abs().max() <= 1e-5
    assert float(p[10:-150].abs().max()) == 0
    start = n - 200
    m, v = moments(np.zeros(200), np.zeros(200), g[start:].float().cpu().numpy())
    assert start % 64 == 0
    r = random_bits(200, 0, 1, 12, start)
    codes, scales = encode(v, 32, ((r >> 16) << 4) + 8)
    assert np.array_equal(opt.slot_v[0][start:].cpu().numpy(), codes)
    assert np.array_equal(opt.scale_v[0][start // 64:].cpu().numpy(), scales)
