"""xdfm_layer_norm_fwd / _bwd through the C ABI against the formula in 64 bits.

Tolerances are counted, per element, from the roundings on the way to it (u = 2^-24, half a step of fp32 relative
to the value; the half step of the element type at the end):

* a sum of n terms in the kernels passes through at most `chain(n)` additions one behind the other, so it is off by
  chain(n) u sum|terms|;
* xhat = (x - mean) rstd: two roundings, and what mean and rstd are off by;
* u = gamma xhat + beta: two more;  activations: 8 u of the value (expf / tanhf / expm1f are good to 2 ulp, and up to
  three operations follow), their slopes are at most 1, so an error of u goes through undiminished at most.
"""
import ctypes

import numpy as np
import pytest
import torch

from recommenders_amd import _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACT = {"identity": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "elu": 4}
TYPES = {"fp32": (torch.float32, 0), "bf16": (torch.bfloat16, 1), "fp16": (torch.float16, 2)}
SIZES = [(1, 1), (4, 1), (1, 7), (3, 20), (130, 20), (5, 64), (2, 65), (17, 257), (64, 1000), (33, 1024), (9, 2048), (7, 2496),
         (5, 4097), (3, 8192), (2, 16387), (2, 40001), (4099, 33), (2500, 512), (70, 200), (45, 700), (300, 129),
         (1029, 100), (3000, 8), (2, 16384), (600, 2600), (1100, 1600), (20, 6001), (300, 9000)]


def half_step(dtype, value):
    """Half a step of dtype at |value| (a bound: relative, and the smallest step below the normal numbers)."""
    tiny = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]
    return torch.finfo(dtype).eps / 2 * value.abs() + tiny


def chain(n):
    # a thread's own terms (at least 8 threads share a row; 512 at most lie one behind the other), then a tree
    return min(n, max(n / 8, 16) + 16, 600.0)


def act_of(u, act):
    return {"identity": lambda: u, "relu": lambda: u.clamp(min=0), "sigmoid": lambda: torch.sigmoid(u),
            "tanh": lambda: torch.tanh(u), "elu": lambda: torch.nn.functional.elu(u)}[act]()


def slope_of(u, act):
    return {"identity": lambda: torch.ones_like(u), "relu": lambda: (u > 0).double(),
            "sigmoid": lambda: torch.sigmoid(u) * (1 - torch.sigmoid(u)), "tanh": lambda: 1 - torch.tanh(u) ** 2,
            "elu": lambda: torch.where(u > 0, torch.ones_like(u), torch.exp(u))}[act]()


def make(rows, cols, dtype, seed, pad=0, offset=0):
    """x, dy as views of wider buffers whose other elements are 77; gamma, beta."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def view(values):
        buf = torch.full((rows * (cols + pad) + offset,), 77.0, dtype=dtype, device="cuda")
        v = buf[offset:].view(rows, cols + pad)[:, :cols]
        v.copy_(values)
        return v

    x = view(rand(rows, cols) * (0.5 + torch.rand((rows, 1), generator=gen, device="cuda")) + rand(rows, 1))
    dy = view(rand(rows, cols) * 0.1)
    return x, dy, 1 + 0.2 * rand(cols), 0.2 * rand(cols), view


def stream():
    return torch.cuda.current_stream().cuda_stream


def fwd(x, code, gamma, beta, act, y, stats, eps=1e-5):
    print("layer_norm_fwd", tuple(x.shape), x.dtype, act, flush=True)
    _lib.check(_lib.lib.xdfm_layer_norm_fwd(x.data_ptr(), x.stride(0), code, x.shape[0], x.shape[1], gamma.data_ptr(),
                                            beta.data_ptr(), eps, ACT[act], y.data_ptr(), y.stride(0),
                                            stats.data_ptr() if stats is not None else None, stream()))


def workspace(rows, cols):
    need = ctypes.c_size_t()
    _lib.check(_lib.lib.xdfm_layer_norm_bwd_workspace_floats(rows, cols, ctypes.byref(need)))
    return torch.full((need.value + 4,), float("nan"), device="cuda")


def bwd(x, dy, code, gamma, beta, stats, act, dx, ws=None):
    rows, cols = x.shape
    print("layer_norm_bwd", (rows, cols), x.dtype, act, flush=True)
    ws = workspace(rows, cols) if ws is None else ws
    dg, db = torch.full((cols,), 5.0, device="cuda"), torch.full((cols,), 5.0, device="cuda")
    _lib.check(_lib.lib.xdfm_layer_norm_bwd(x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), code, rows, cols,
                                            gamma.data_ptr(), beta.data_ptr(), stats.data_ptr(), ACT[act],
                                            dx.data_ptr(), dx.stride(0), dg.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                            stream()))
    return dg, db


def stats_exact(x, eps=1e-5):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    return mean, 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)


def within(got, exp, tol, what):
    err = (got.double() - exp).abs()
    bad = ~(err <= tol)
    assert not bad.any(), "%s: %d of %d off, by up to %.3g of the allowed" % (
        what, int(bad.sum()), bad.numel(), float((err / tol)[bad].max()))


def check_fwd(x, gamma, beta, act, y, stats, eps=1e-5):
    n = x.shape[1]
    xd = x.double()
    mean, rstd = stats_exact(x, eps)
    d = xd - mean
    e_mean = (chain(n) + 1) * U * xd.abs().mean(1, keepdim=True) + U * mean.abs()
    # sum of squares: each off by 2 |d| e_mean + 3 u d^2; then chain, the division, eps, root and reciprocal
    e_var = (2 * d.abs() * (e_mean + U * d.abs())).mean(1, keepdim=True) + e_mean ** 2 + (chain(n) + 4) * U * (d ** 2).mean(
        1, keepdim=True) + U * (1 / rstd ** 2)
    e_rstd = rstd * (0.5 * e_var * rstd ** 2 * (1 + e_var * rstd ** 2) + 4 * U)
    xhat = d * rstd
    e_xhat = rstd * (e_mean + 2 * U * d.abs()) + d.abs() * e_rstd + e_mean * e_rstd
    u = gamma.double() * xhat + beta.double()
    e_u = gamma.double().abs() * (e_xhat + 2 * U * xhat.abs()) + U * u.abs()
    exp = act_of(u, act)
    within(y, exp, e_u + 8 * U * exp.abs() + half_step(y.dtype, exp.abs() + e_u), "y")
    if stats is not None:
        within(stats[0], mean[:, 0], (e_mean + U * mean.abs())[:, 0] + 1e-40, "mean")
        within(stats[1], rstd[:, 0], e_rstd[:, 0], "rstd")


def exact_bwd(x, dy, gamma, beta, stats, act):
    """(dx, dgamma, dbeta) in 64 bits from the 32-bit statistics, and how far 32 bits may be off."""
    rows, n = x.shape
    g, b = gamma.double(), beta.double()
    mean, rstd = stats[0].double()[:, None], stats[1].double()[:, None]
    d = x.double() - mean
    xhat = d * rstd
    e_xhat = 2 * U * xhat.abs()
    u = g * xhat + b
    e_u = g.abs() * (e_xhat + U * xhat.abs()) + U * u.abs() + U * b.abs()
    s = slope_of(u, act)
    # (relu: exact; identity: exact; the others' slopes change by at most their second derivative, 1 at most, times e_u)
    e_s = torch.zeros_like(u) if act in ("identity", "relu") else e_u + 8 * U
    du = dy.double() * s
    e_du = dy.double().abs() * e_s + U * du.abs()
    t = du * g
    e_t = e_du * g.abs() + U * t.abs()
    q = t * xhat
    e_q = e_t * xhat.abs() + t.abs() * e_xhat + U * q.abs()
    a, c = t.mean(1, keepdim=True), q.mean(1, keepdim=True)
    e_a = e_t.mean(1, keepdim=True) + (chain(n) + 2) * U * t.abs().mean(1, keepdim=True)
    e_c = e_q.mean(1, keepdim=True) + (chain(n) + 2) * U * q.abs().mean(1, keepdim=True)
    dx = rstd * (t - a - xhat * c)
    e_dx = rstd * (e_t + e_a + xhat.abs() * e_c + e_xhat * c.abs() + 4 * U * (t.abs() + a.abs() + (xhat * c).abs()))
    w = du * xhat
    e_w = e_du * xhat.abs() + du.abs() * e_xhat + U * w.abs()
    many = min(rows, 600) + 2
    dg, e_dg = w.sum(0), e_w.sum(0) + many * U * w.abs().sum(0)
    db, e_db = du.sum(0), e_du.sum(0) + many * U * du.abs().sum(0)
    return (dx, e_dx), (dg, e_dg), (db, e_db)


def check_bwd(x, dy, gamma, beta, stats, act, dx, dg, db):
    (edx, tdx), (edg, tdg), (edb, tdb) = exact_bwd(x, dy, gamma, beta, stats, act)
    within(dx, edx, tdx + half_step(dx.dtype, edx.abs() + tdx), "dx")
    within(dg, edg, tdg + 1e-40, "dgamma")
    within(db, edb, tdb + 1e-40, "dbeta")


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("kind", list(TYPES))
def test_forward_and_backward_match_the_formula(rows, cols, kind):
    dtype, code = TYPES[kind]
    act = list(ACT)[(rows + cols) % 5]
    x, dy, gamma, beta, view = make(rows, cols, dtype, seed=rows * 7 + cols)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    stats = torch.empty((2, rows), device="cuda")
    fwd(x, code, gamma, beta, act, y, stats)
    check_fwd(x, gamma, beta, act, y, stats)
    dg, db = bwd(x, dy, code, gamma, beta, stats, act, dx)
    check_bwd(x, dy, gamma, beta, stats, act, dx, dg, db)


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols,pad,offset", [(1017, 513, 0, 0), (1031, 1000, 3, 1), (4099, 1024, 0, 0),
                                                  (1100, 1025, 5, 0), (1024, 1536, 8, 0), (2051, 1537, 0, 3),
                                                  (1500, 2041, 7, 1), (1019, 2048, 0, 0), (4101, 2049, 0, 1),
                                                  (4096, 2496, 6, 0), (4200, 2560, 0, 0), (1500, 700, 1, 2),
                                                  (511, 2561, 1, 0), (1027, 4096, 0, 1), (700, 5113, 7, 2),
                                                  (257, 5121, 0, 0), (263, 8192, 0, 0), (259, 10233, 3, 1),
                                                  (7, 8200, 0, 0), (261, 12289, 1, 1), (300, 16384, 0, 0),
                                                  (4097, 2700, 1, 1), (4099, 5119, 0, 0), (5, 18432, 0, 0),
                                                  (9, 20479, 1, 1), (3, 20481, 0, 0)])
def test_many_rows_of_a_few_waves_each(act, kind, rows, cols, pad, offset):
    """2 to 6 pieces a lane, 1 to 16 waves a row: out of place, and in place with the same bits."""
    dtype, code = TYPES[kind]
    x, dy, gamma, beta, view = make(rows, cols, dtype, seed=rows + cols, pad=pad, offset=offset)
    y, dx = view(torch.zeros_like(x)), view(torch.zeros_like(x))
    stats = torch.empty((2, rows), device="cuda")
    fwd(x, code, gamma, beta, act, y, stats)
    check_fwd(x, gamma, beta, act, y, stats)
    dg, db = bwd(x, dy, code, gamma, beta, stats, act, dx)
    check_bwd(x, dy, gamma, beta, stats, act, dx, dg, db)
    for target in ("dy", "x"):
        x2, dy2 = view(x), view(dy)
        on = dy2 if target == "dy" else x2
        dg2, db2 = bwd(x2, dy2, code, gamma, beta, stats, act, on)
        assert torch.equal(on, dx) and torch.equal(dg, dg2) and torch.equal(db, db2)
    over = view(x)
    fwd(over, code, gamma, beta, act, over, None)
    assert torch.equal(over, y)
    for t in (y, dx, over, on):
        whole = t._base.reshape(-1) if t._base is not None else t.reshape(-1)
        gaps = torch.ones_like(whole, dtype=torch.bool)
        gaps[offset:].view(rows, cols + pad)[:, :cols] = False
        assert (whole[gaps] == 77).all()


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cols,pad,offset", [(20, 3, 1), (1001, 6, 3), (512, 0, 1), (2496, 5, 0)])
def test_strides_and_odd_addresses_leave_the_gaps_alone(act, kind, cols, pad, offset):
    dtype, code = TYPES[kind]
    rows = 37
    x, dy, gamma, beta, view = make(rows, cols, dtype, seed=cols + pad, pad=pad, offset=offset)
    y, dx = view(torch.zeros_like(x)), view(torch.zeros_like(x))
    # weights at odd addresses too
    gamma, beta = torch.cat([gamma[:1], gamma])[1:], torch.cat([beta[:1], beta])[1:]
    stats = torch.empty((2, rows), device="cuda")
    fwd(x, code, gamma, beta, act, y, stats)
    check_fwd(x, gamma, beta, act, y, stats)
    dg, db = bwd(x, dy, code, gamma, beta, stats, act, dx)
    check_bwd(x, dy, gamma, beta, stats, act, dx, dg, db)
    for t in (x, dy, y, dx):
        base = t._base if t._base is not None else t
        whole = base.reshape(-1)
        gaps = torch.ones_like(whole, dtype=torch.bool)
        gaps[offset:].view(rows, cols + pad)[:, :cols] = False
        assert (whole[gaps] == 77).all()


@pytest.mark.parametrize("cols", [20, 700, 2496, 9000, 40001])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_in_place_equals_out_of_place(cols, kind):
    dtype, code = TYPES[kind]
    x, dy, gamma, beta, _ = make(21, cols, dtype, seed=3)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    stats, stats2 = torch.empty((2, 21), device="cuda"), torch.empty((2, 21), device="cuda")
    fwd(x, code, gamma, beta, "relu", y, stats)
    dg, db = bwd(x, dy, code, gamma, beta, stats, "relu", dx)
    over = x.clone()
    fwd(over, code, gamma, beta, "relu", over, stats2)
    assert torch.equal(over, y) and torch.equal(stats, stats2)
    fwd(x, code, gamma, beta, "relu", over, None)  # without statistics
    assert torch.equal(over, y)
    for target in ("dy", "x"):
        x2, dy2 = x.clone(), dy.clone()
        dg2, db2 = bwd(x2, dy2, code, gamma, beta, stats, "relu", dy2 if target == "dy" else x2)
        assert torch.equal(dy2 if target == "dy" else x2, dx) and torch.equal(dg, dg2) and torch.equal(db, db2)


@pytest.mark.parametrize("rows,cols", [(257, 20), (4099, 100), (2049, 512), (1003, 2496)])
def test_infinite_dx_on_x_stays_out_of_the_weights_gradients(rows, cols):
    """dx beyond the type's range, written where x was: other rows' threads that look past the last row see it there."""
    x, dy, gamma, beta, view = make(rows, cols, torch.float16, 31)
    dy *= 3e4
    gamma = gamma.abs() * 100  # dx ~ 3e3 * 100 * rstd
    mean, rstd = stats_exact(x)
    stats = torch.cat([mean, rstd], 1).t().float().contiguous()
    out = torch.empty_like(x)
    dg, db = bwd(x, dy, 2, gamma, beta, stats, "identity", out)
    assert torch.isinf(out).any() and torch.isfinite(dg).all() and torch.isfinite(db).all()
    for _ in range(3):
        on = x.clone()
        dg2, db2 = bwd(on, dy, 2, gamma, beta, stats, "identity", on)
        torch.cuda.synchronize()
        assert torch.equal(on, out) and torch.equal(dg2, dg) and torch.equal(db2, db)


def test_no_rows_and_rows_without_spread():
    gamma, beta = torch.randn(50, device="cuda"), torch.randn(50, device="cuda")
    x = torch.empty((0, 50), device="cuda")
    stats = torch.empty((2, 0), device="cuda")
    fwd(x, 0, gamma, beta, "identity", x, stats)
    dg, db = bwd(x, x, 0, gamma, beta, stats, "identity", x)
    assert (dg == 0).all() and (db == 0).all()
    # equal elements: xhat = 0 exactly where their mean is the element itself (a power of two)
    x = torch.tensor([0.0, 4.0, -0.5], device="cuda")[:, None].expand(3, 50).contiguous()
    stats, y = torch.empty((2, 3), device="cuda"), torch.empty_like(x)
    fwd(x, 0, gamma, beta, "identity", y, stats)
    check_fwd(x, gamma, beta, "identity", y, stats)
    one = torch.randn((5, 1), device="cuda")
    y = torch.empty_like(one)
    fwd(one, 0, gamma[:1], beta[:1], "identity", y, None)
    assert torch.equal(y, beta[:1].expand(5, 1))


def test_rows_far_from_zero():
    """mean 1000, spread 1: the variance is formed around the mean, not from the sum of squares."""
    x = 1000 + torch.randn((65, 1024), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    gamma, beta = torch.ones(1024, device="cuda"), torch.zeros(1024, device="cuda")
    y, stats = torch.empty_like(x), torch.empty((2, 65), device="cuda")
    fwd(x, 0, gamma, beta, "identity", y, stats)
    check_fwd(x, gamma, beta, "identity", y, stats)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_row(bad):
    for cols in (20, 1024, 9000):
        x, dy, gamma, beta, _ = make(40, cols, torch.float32, seed=9)
        y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty((2, 40), device="cuda")
        fwd(x, 0, gamma, beta, "tanh", y, stats)
        bwd(x, dy, 0, gamma, beta, stats, "tanh", dx)
        x2, dy2 = x.clone(), dy.clone()
        x2[7, 3] = bad
        y2, dx2, stats2 = torch.empty_like(x), torch.empty_like(x), torch.empty((2, 40), device="cuda")
        fwd(x2, 0, gamma, beta, "tanh", y2, stats2)
        assert torch.isnan(y2[7]).all()
        dy2[11, cols - 1] = bad
        dg, db = bwd(x2, dy2, 0, gamma, beta, stats2, "tanh", dx2)
        keep = [r for r in range(40) if r not in (7, 11)]
        assert torch.equal(y2[keep], y[keep]) and torch.equal(y2[11], y[11]) and torch.equal(dx2[keep], dx[keep])
        assert torch.isnan(dx2[7]).all() and not torch.isfinite(dx2[11]).any()
        assert torch.isnan(dg).all() and torch.isfinite(db[:3]).sum() == 0


def test_relu_is_on_by_the_exact_sign():
    """gamma xhat and beta that cancel to the last bits of 32: the sign comes from 64."""
    rows, cols = 64, 2048
    x, dy, gamma, _, _ = make(rows, cols, torch.float32, seed=21)
    stats = torch.empty((2, rows), device="cuda")
    y = torch.empty_like(x)
    fwd(x, 0, gamma, torch.zeros(cols, device="cuda"), "relu", y, stats)
    # beta = -(gamma xhat) of one row per column, rounded to 32 bits
    pick = torch.arange(cols, device="cuda") % rows
    mean, rstd = stats.double()
    beta = -(gamma.double() * (x.double()[pick, torch.arange(cols, device="cuda")] - mean[pick]) * rstd[pick])
    beta = beta.float().contiguous()
    dx = torch.empty_like(x)
    dg, db = bwd(x, dy, 0, gamma, beta, stats, "relu", dx)
    check_bwd(x, dy, gamma, beta, stats, "relu", dx, dg, db)


def test_two_runs_agree_in_every_bit_and_other_streams_too():
    x, dy, gamma, beta, _ = make(5000, 300, torch.bfloat16, seed=2)
    stats, y, dx = torch.empty((2, 5000), device="cuda"), torch.empty_like(x), torch.empty_like(x)
    fwd(x, 1, gamma, beta, "elu", y, stats)
    ref = bwd(x, dy, 1, gamma, beta, stats, "elu", dx)
    torch.cuda.synchronize()
    for _ in range(3):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            y2, dx2 = torch.empty_like(x), torch.empty_like(x)
            fwd(x, 1, gamma, beta, "elu", y2, stats)
            again = bwd(x, dy, 1, gamma, beta, stats, "elu", dx2)
        side.synchronize()
        assert torch.equal(y, y2) and torch.equal(dx, dx2) and all(torch.equal(a, b) for a, b in zip(ref, again))


def test_two_calls_at_once():
    """Two streams, each with its own workspace, under way together: the same bits as alone."""
    sets = [make(20000, c, torch.float32, seed=c) for c in (500, 512)]
    alone = []
    for x, dy, gamma, beta, _ in sets:
        y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty((2, 20000), device="cuda")
        fwd(x, 0, gamma, beta, "sigmoid", y, stats)
        alone.append((y, stats, dx) + bwd(x, dy, 0, gamma, beta, stats, "sigmoid", dx))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, (x, dy, gamma, beta, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty((2, 20000), device="cuda")
                fwd(x, 0, gamma, beta, "sigmoid", y, stats)
                got.append((y, stats, dx) + bwd(x, dy, 0, gamma, beta, stats, "sigmoid", dx))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed on changing inputs with eager work and waits between the replays."""
    rows, cols = 777, 513
    x, dy, gamma, beta, _ = make(rows, cols, torch.float32, seed=5)
    stats, y, dx = torch.empty((2, rows), device="cuda"), torch.empty_like(x), torch.empty_like(x)
    ws = workspace(rows, cols)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fwd(x, 0, gamma, beta, "relu", y, stats)
        bwd(x, dy, 0, gamma, beta, stats, "relu", dx, ws)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fwd(x, 0, gamma, beta, "relu", y, stats)
        dg, db = bwd(x, dy, 0, gamma, beta, stats, "relu", dx, ws)
    for k in range(4):
        nx, ndy, _, _, _ = make(rows, cols, torch.float32, seed=50 + k)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        if k % 2:
            torch.cuda.synchronize()
        y2, dx2, stats2 = torch.empty_like(x), torch.empty_like(x), torch.empty((2, rows), device="cuda")
        fwd(x, 0, gamma, beta, "relu", y2, stats2)
        dg2, db2 = bwd(x, dy, 0, gamma, beta, stats2, "relu", dx2)
        torch.cuda.synchronize()
        assert torch.equal(y, y2) and torch.equal(dx, dx2) and torch.equal(dg, dg2) and torch.equal(db, db2)


def test_offsets_beyond_32_bits():
    """Rows so far apart that an element's offset passes 2^31 (bf16: 2^32 bytes are passed too)."""
    cols, rows = 24, 2300
    gap = 1 << 20
    buf = torch.empty((rows - 1) * gap + cols, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((rows, cols), (gap, 1))
    x.copy_(torch.randn((rows, cols), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    gamma, beta = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
    packed = x.contiguous()
    y, y2 = torch.empty_like(packed), torch.empty_like(packed)
    stats, stats2 = torch.empty((2, rows), device="cuda"), torch.empty((2, rows), device="cuda")
    fwd(x, 1, gamma, beta, "identity", y, stats)
    fwd(packed, 1, gamma, beta, "identity", y2, stats2)
    assert torch.equal(y, y2) and torch.equal(stats, stats2)
    dx = torch.empty_like(packed)
    dg, db = bwd(packed, y, 1, gamma, beta, stats, "identity", dx)
    dg2, db2 = bwd(x, y, 1, gamma, beta, stats, "identity", x)
    assert torch.equal(x.contiguous(), dx) and torch.equal(dg, dg2) and torch.equal(db, db2)


@pytest.mark.parametrize("act", ["identity", "tanh", "sigmoid", "elu"])
def test_gradients_against_differences(act):
    """Central differences of the kernel's own forward pass in fp32 along random directions.  With steps of h the
    quotient is off by h^2/6 times the third derivative (at most ~10 over 24 unit-size elements here) and by twice the
    output's rounding over 2 h: |sum| 1e-6 / h."""
    rows, cols, h = 6, 24, 2e-3
    x, _, gamma, beta, _ = make(rows, cols, torch.float32, seed=31)
    w = torch.randn((rows, cols), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    stats, y, dx = torch.empty((2, rows), device="cuda"), torch.empty_like(x), torch.empty_like(x)
    fwd(x, 0, gamma, beta, act, y, stats)
    dg, db = bwd(x, w, 0, gamma, beta, stats, act, dx)

    def loss(xv, g, b):
        out = torch.empty_like(xv)
        fwd(xv, 0, g, b, act, out, None)
        return float((out.double() * w.double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(8)
    for arg, grad in (("x", dx), ("gamma", dg), ("beta", db)):
        v = torch.randn(grad.shape, generator=gen, device="cuda")
        v /= v.norm()

        def moved(s):
            return (x + s * v if arg == "x" else x, gamma + s * v if arg == "gamma" else gamma,
                    beta + s * v if arg == "beta" else beta)

        diff = (loss(*moved(h)) - loss(*moved(-h))) / (2 * h)
        tol = h * h / 6 * 10 * float(w.abs().sum()) / cols + 1e-6 / h * float((y.abs() * w.abs()).sum()) ** 0.5 + 1e-4
        assert abs(diff - float((grad.double() * v.double()).sum())) <= tol, arg
