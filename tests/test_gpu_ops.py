"""The operators on device tensors (popvae_amd.ops) against plain 64-bit formulas.

Tolerances count roundings (u = 2^-24, float32; h = finfo.eps / 2 of the tensors' type, plus half the smallest subnormal):
a float32 sum of K products is off by at most (K + 2) u times the sum of their absolute values -- 6 K + 8 terms where an
operand is cut into three bf16 parts and six partial products are added -- an activation has a slope of at most 1.13 and is
evaluated to 8 u (1 + |z|), its derivative to 16 u (1 + |z|), and each stored value is rounded once (h).  In the gradients g = dy f'(z)
is rounded to the tensors' type first: h |g| in every product."""
import math

import pytest
import torch

from popvae_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def f64(t):
    return None if t is None else t.double().contiguous()


def act64(z, name):
    return {"linear": lambda: z, "relu": lambda: z.clamp(min=0), "elu": lambda: torch.where(z > 0, z, torch.expm1(z)),
            "sigmoid": lambda: torch.sigmoid(z), "tanh": lambda: torch.tanh(z), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.erfc(-z / math.sqrt(2)) / 2}[name]()


def dact64(z, name):
    z = z.clone().requires_grad_(True)
    act64(z, name).sum().backward()
    return z.grad


def check(got, want, bound, what):
    got = got.double()
    bad = ((got - want).abs() > bound) | (got.isnan() != want.isnan())
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()), float(bound.max()))


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def check_forward(x, w, b, act, r, y, z=None):
    X, W = f64(x), f64(w)
    k = X.shape[1]
    z64 = X @ W + (0 if b is None else f64(b))
    S = X.abs() @ W.abs() + (0 if b is None else f64(b).abs())
    e = (6 * k + 8) * U * S
    if z is not None:
        check(z, z64, e + U * z64.abs(), "pre")
    want = act64(z64, act) + (0 if r is None else f64(r))
    h, tiny = half(y.dtype)
    bound = 1.13 * e + 8 * U * (1 + z64.abs()) + 4 * U * want.abs()
    check(y, want, bound + h * (want.abs() + bound) + tiny, "y")


def check_backward(dy, x, w, z, act, add, dx, dw, db):
    X, W, DY = f64(x), f64(w), f64(dy)
    m, n = DY.shape
    zz = torch.zeros_like(DY) if z is None else f64(z)
    G = DY * (dact64(zz, act) if m * n else zz)
    h, tiny = half(dy.dtype)
    eg = 16 * U * (1 + zz.abs()) * DY.abs() + 2 * U * G.abs()  # g in float32
    hr, tr = (h, tiny) if dy.dtype != F32 else (0.0, 0.0)
    er = eg + hr * (G.abs() + eg) + tr                         # g as it enters the products
    if dx is not None:
        want = G @ W.t().contiguous() + (0 if add is None else f64(add))
        e = er @ W.t().abs().contiguous() + (6 * n + 8) * U * ((G.abs() + er) @ W.t().abs().contiguous()) + 4 * U * want.abs()
        check(dx, want, e + h * (want.abs() + e) + tiny, "dx")
    if dw is not None:
        want = X.t().contiguous() @ G
        e = X.t().abs().contiguous() @ er + (6 * m + 8) * U * (X.t().abs().contiguous() @ (G.abs() + er)) + 4 * U * want.abs()
        check(dw, want, e + h * (want.abs() + e) + tiny, "dw")
    if db is not None:
        want = G.sum(0)
        e = eg.sum(0) + (m + 8) * U * (G.abs() + eg).sum(0)
        check(db, want, e + h * (want.abs() + e) + tiny, "db")


SIZES = [(1, 1, 1), (1, 128, 128), (3, 5, 7), (32, 128, 128), (33, 65, 129), (64, 64, 64), (100, 1, 300), (65, 300, 1), (1, 1000, 3),
         (2, 4097, 9), (7, 200, 1001), (8, 128, 4096), (9, 128, 513), (128, 512, 512), (257, 130, 515), (300, 1000, 40),
         (1000, 24, 1100), (513, 1025, 770)]
ACTS = list(ops.ACTIVATIONS)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_dense_and_gradients(m, k, n, dtype):
    for i, act in enumerate(ACTS[(m + k + n) % 3::3]):
        for w_t in (False, True):
            s = 10 * i + w_t
            x, r, dy = (rnd(m, j, dtype=dtype, seed=s + q) for q, j in ((1, k), (2, n), (3, n)))
            w = rnd(n, k, dtype=dtype, seed=s + 4, scale=k ** -0.5).t() if w_t else rnd(k, n, dtype=dtype, seed=s + 4, scale=k ** -0.5)
            b = rnd(n, dtype=dtype, seed=s + 5)
            z = torch.full((m, n), float("nan"), device="cuda")
            y = ops.dense(x, w, b, act, residual=r, pre=z)
            check_forward(x, w, b, act, r, y, z)
            plain = ops.dense(x, w, activation=act)
            check_forward(x, w, None, act, None, plain)
            got = ops.dense_backward(dy, x, w, z, act)
            check_backward(dy, x, w, z, act, None, *got)
            again = ops.dense_backward(dy, x, w, z, act)
            assert all(torch.equal(p, q) for p, q in zip(got, again))  # no order of sums that changes from run to run


# the large product kernel's forms: whole and ragged tiles, few and many of them, contractions in pieces, operands as they lie
# (aligned) and laid out (not), either orientation
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(2048, 1344, 2048), (2100, 1408, 2208), (192, 8192, 256), (640, 1024, 1152), (1543, 1021, 2027),
                                   (130, 70_001, 129), (5, 2048, 4099), (1024, 64, 3000), (4000, 64, 64), (600, 2500, 17), (4001, 30, 100)])
def test_large_products(m, k, n, dtype):
    act = ACTS[(m + n) % 7]
    for w_t in (False, True):
        x, r, dy = rnd(m, k, dtype=dtype, seed=1), rnd(m, n, dtype=dtype, seed=2), rnd(m, n, dtype=dtype, seed=3)
        w = rnd(n, k, dtype=dtype, seed=4, scale=k ** -0.5).t() if w_t else rnd(k, n, dtype=dtype, seed=4, scale=k ** -0.5)
        b, z = rnd(n, dtype=dtype, seed=5), torch.empty(m, n, device="cuda")
        check_forward(x, w, b, act, r, ops.dense(x, w, b, act, residual=r, pre=z), z)
        add = rnd(m, k, dtype=dtype, seed=6)
        check_backward(dy, x, w, z, act, add, *ops.dense_backward(dy, x, w, z, act, dx_add=add))
        dx, dw, db = ops.dense_backward(dy, x, w, z, act, need_dx=False, need_dw=False)
        assert dx is None and dw is None
        check_backward(dy, x, w, z, act, None, None, None, db)


@pytest.mark.parametrize("m,k,n", [(0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0), (3, 0, 9), (600, 5, 0), (600, 0, 5), (0, 300, 400)])
def test_empty_sizes(m, k, n):
    x, w, b, r, dy = rnd(m, k), rnd(k, n, seed=1), rnd(n, seed=2), rnd(m, n, seed=3), rnd(m, n, seed=4)
    z = torch.full((m, n), 7.0, device="cuda")
    y = ops.dense(x, w, b, "elu", residual=r, pre=z)
    assert y.shape == (m, n)
    check_forward(x, w, b, "elu", r, y, z)
    dx, dw, db = ops.dense_backward(dy, x, w, z, "elu")
    check_backward(dy, x, w, z, "elu", None, dx, dw, db)
    assert dx.shape == (m, k) and dw.shape == (k, n) and db.shape == (n,)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(5, 37, 70), (40, 128, 256), (200, 300, 130), (600, 256, 512)])
def test_strides_offsets_and_destinations(m, k, n, dtype):
    """Rows cut out of wider tensors (odd offsets and row strides), an expanded residual, the output over the residual."""
    wide = rnd(m, k + 13, dtype=dtype, seed=1)
    x = wide[:, 3:3 + k]
    w = rnd(k + 2, n + 9, dtype=dtype, seed=2, scale=k ** -0.5)[1:1 + k, 5:5 + n]
    b = rnd(n + 1, dtype=dtype, seed=3)[1:]
    row = rnd(1, n, dtype=dtype, seed=4)
    buf = torch.full((m + 2, n + 11), 3.0, dtype=dtype, device="cuda")
    out = buf[1:1 + m, 7:7 + n]
    zbuf = torch.full((m, n + 3), -1.0, device="cuda")
    got = ops.dense(x, w, b, "silu", residual=row.expand(m, n), pre=zbuf[:, 2:2 + n], out=out)
    assert got.data_ptr() == out.data_ptr()
    check_forward(x, w, b, "silu", row.expand(m, n), out, zbuf[:, 2:2 + n])
    keep = buf.clone()
    keep[1:1 + m, 7:7 + n] = 3.0
    assert bool((keep == 3.0).all()) and bool((zbuf[:, :2] == -1).all()) and bool((zbuf[:, 2 + n:] == -1).all())
    r = rnd(m, n, dtype=dtype, seed=5)
    r0 = r.clone()
    ops.dense(x, w, b, "tanh", residual=r, out=r)
    check_forward(x, w, b, "tanh", r0, r)
    dy = rnd(m, n + 4, dtype=dtype, seed=6)[:, 1:1 + n]
    z = zbuf[:, 2:2 + n]
    add = rnd(m, k, dtype=dtype, seed=7)
    for a in (None, add, add[:1].expand(m, k)):
        got = ops.dense_backward(dy, x, w, z, "silu", dx_add=a)
        check_backward(dy, x, w, z, "silu", a, *got)
    dx, dw, db = ops.dense_backward(dy, x, w, z, "silu", need_dx=False)
    assert dx is None
    check_backward(dy, x, w, z, "silu", None, dx, dw, db)
    dx, dw, db = ops.dense_backward(dy, x, w, activation="linear", need_dw=False, need_bias=False)
    assert dw is None and db is None
    check_backward(dy, x, w, None, "linear", None, dx, dw, db)


def test_gradients_against_differences():
    """The gradient of sum(dy * dense(...)) against central differences of the operator itself: off by the third derivative
    (|f'''| <= 2 for all of them, times what multiplies the parameter, cubed) times step^2 / 6, and by the roundings of y
    (16 u (1 + |z|) each) over the step."""
    m, k, n = 5, 6, 4
    for act in ("elu", "gelu", "silu", "tanh", "sigmoid"):
        x, w, b, dy = rnd(m, k, seed=1), rnd(k, n, seed=2, scale=0.3), rnd(n, seed=3), rnd(m, n, seed=4)
        z = torch.empty(m, n, device="cuda")
        ops.dense(x, w, b, act, pre=z)
        if act == "elu":  # its derivative bends at 0: move every z away from it by more than a step reaches
            assert float(z.abs().min()) > 1e-3
        dx, dw, db = ops.dense_backward(dy, x, w, z, act)
        step = 2.0 ** -8 if act == "elu" else 2.0 ** -6

        by = max(1.0, float(x.abs().max()), float(w.abs().max())) ** 3 * float(max(dy.abs().sum(0).max(), dy.abs().sum(1).max()))
        tol = by * step * step / 3 + float(dy.abs().sum()) * 16 * U * (1 + float(z.abs().max())) / step

        def loss():
            return float((dy.double() * ops.dense(x, w, b, act).double()).sum())

        for t, g in ((x, dx), (w, dw), (b, db)):
            flat, gf = t.view(-1), g.reshape(-1)
            for i in range(0, flat.numel(), 3):
                v = float(flat[i])
                flat[i] = v + step
                up, hi = loss(), float(flat[i])
                flat[i] = v - step
                down, lo = loss(), float(flat[i])
                flat[i] = v
                assert abs((up - down) / (hi - lo) - float(gf[i])) <= tol, (act, i)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(4, 70, 300), (40, 128, 200), (300, 256, 520)])
def test_infinities_and_nan_stay_where_they_belong(m, k, n, dtype):
    x, w = rnd(m, k, dtype=dtype, seed=1), rnd(k, n, dtype=dtype, seed=2)
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    w[7, 9] = float("-inf")
    y = ops.dense(x, w)
    want = f64(x) @ f64(w)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y[y.isinf()].double(), want[want.isinf()])
    lo = torch.finfo(dtype).min
    x = torch.zeros(m, k, dtype=dtype, device="cuda")
    x[:, 0] = lo
    w = torch.zeros(k, n, dtype=dtype, device="cuda")
    w[0] = 1.0
    assert bool((ops.dense(x, w) == lo).all())


def test_offsets_beyond_32_bits():
    m, k, n = 70_001, 3, 40_000  # 2.8e9 elements of y
    x, w = rnd(m, k, dtype=BF16, seed=1), rnd(k, n, dtype=BF16, seed=2)
    y = ops.dense(x, w, activation="relu")
    for rows in (slice(0, 3), slice(53_600, 53_900), slice(m - 3, m)):
        check_forward(x[rows], w, None, "relu", None, y[rows])
    del y
    dy = torch.zeros(m, n, dtype=BF16, device="cuda")
    dy[-2:] = rnd(2, n, dtype=BF16, seed=3)
    dx, dw, db = ops.dense_backward(dy, x, w)
    check_backward(dy[-2:], x[-2:], w, None, "linear", None, dx[-2:], dw, db)
    assert bool((dx[:-2] == 0).all())


def on_stream(f):
    """f on a stream of its own, ordered behind and before the current one."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r = f()
    torch.cuda.current_stream().wait_stream(s)
    return r


@pytest.mark.parametrize("m,k,n,dtype", [(4, 300, 200, F32), (32, 128, 128, F32), (300, 256, 300, F32), (300, 256, 300, BF16),
                                         (700, 520, 900, F32), (700, 512, 901, F16)])
def test_streams_and_graphs(m, k, n, dtype):
    x, w, b, dy = (rnd(*s, dtype=dtype, seed=i) for i, s in enumerate([(m, k), (k, n), (n,), (m, n)]))
    z, z2 = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
    p, mo, v = rnd(k, n, seed=8), torch.zeros(k, n, device="cuda"), torch.zeros(k, n, device="cuda")
    step = torch.ones((), dtype=torch.int32, device="cuda")

    def work(z, p, mo, v):
        y = ops.dense(x, w, b, "elu", pre=z)
        g = ops.dense_backward(dy, x, w, z, "elu")
        norm = ops.adam_step([p], [g[1]], [mo], [v], step, clip_norm=0.1)
        return [y, *g, norm]

    q, qm, qv = p.clone(), mo.clone(), v.clone()
    eager = [t.clone() for t in work(z, q, qm, qv)]
    q2, qm2, qv2 = p.clone(), mo.clone(), v.clone()
    other = on_stream(lambda: work(z2, q2, qm2, qv2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(eager + [q, qm, qv], other + [q2, qm2, qv2]))
    q2, qm2, qv2 = p.clone(), mo.clone(), v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(z2, q2, qm2, qv2)
    for i in range(4):  # replays, with other work and new inputs between them
        x.copy_(rnd(m, k, dtype=dtype, seed=50 + i))
        step.fill_(i + 1)
        junk = [rnd(100, 100) @ rnd(100, 100) for _ in range(3)]
        q.copy_(q2), qm.copy_(qm2), qv.copy_(qv2)
        graph.replay()
        got = [t.clone() for t in outs + [q2, qm2, qv2]]
        want = work(z, q, qm, qv)
        assert all(torch.equal(a, c) for a, c in zip(got, want + [q, qm, qv])), i
        del junk


# ---- many tensors --------------------------------------------------------------------------------
def tensors(sizes, dtypes, seed=0, scale=1.0):
    return [rnd(n, dtype=dtypes[i % len(dtypes)], seed=seed + i, scale=scale) for i, n in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


MANY = [[1], [4, 3, 2, 1], [8192, 8193, 8191, 0, 5], [7] * 100, [100_003, 1, 33, 4096], [3_000_001, 128, 16_384]]


@pytest.mark.parametrize("dtypes", [[F32], [BF16], [F16, F32, BF16]])
@pytest.mark.parametrize("sizes", MANY)
def test_norm_and_clipping(sizes, dtypes):
    ts = tensors(sizes, dtypes)
    want = norm64(ts)
    assert abs(float(ops.global_norm(ts)) - want) <= 2 * U * want
    for c in (want * 0.37, want * 1.01, 1e30):
        out = [torch.full_like(t, 9.0) for t in ts]
        n = ops.clip_by_global_norm(ts, c, out=out)
        assert abs(float(n) - want) <= 2 * U * want
        s = min(1.0, c / want)
        for t, o in zip(ts, out):
            h, tiny = half(t.dtype)
            w64 = t.double() * s
            check(o, w64, (h + 3 * U) * w64.abs() + tiny, "clipped") if s < 1 else None
            assert s < 1 or torch.equal(t, o)
        held = ops.TensorSet([t.clone() for t in ts])
        ops.clip_by_global_norm(held, c)
        assert all(torch.equal(a, b) for a, b in zip(held.tensors, out))


def test_norm_over_and_underflow_of_squares():
    for scale in (1e30, 1e-30):
        t = [rnd(5000, seed=3, scale=scale), rnd(17, seed=4, scale=scale)]
        want = norm64(t)
        assert abs(float(ops.global_norm(t)) - want) <= 2 * U * want
        ops.clip_by_global_norm(t, want / 2)
        assert abs(float(ops.global_norm(t)) - want / 2) <= 8 * U * want
    assert float(ops.global_norm([torch.zeros(5, device="cuda"), torch.zeros(0, device="cuda")])) == 0.0
    assert float(ops.global_norm([torch.zeros(0, device="cuda")])) == 0.0


def test_norm_of_unaligned_views_and_many_tensors():
    base = rnd(100_000, seed=1)
    ts, at = [], 1
    for i in range(300):
        ts.append(base[at:at + 1 + i % 37])
        at += 40 + i % 3
    want = norm64(ts)
    assert abs(float(ops.global_norm(ts)) - want) <= 2 * U * want
    before = base.clone()
    ops.clip_by_global_norm(ts, want / 4)
    touched = torch.zeros_like(base, dtype=torch.bool)
    for t in ts:
        touched[t.storage_offset():t.storage_offset() + t.numel()] = True
    assert torch.equal(base[~touched], before[~touched])
    check(base[touched], before[touched].double() / 4, 4 * U * before[touched].double().abs(), "clipped views")
    # the same gradient twice (a shared parameter) counts twice
    assert abs(float(ops.global_norm([ts[0], ts[0]])) - norm64([ts[0], ts[0]])) <= 2 * U * want


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_norm_that_is_not_finite_makes_all_nan(bad):
    ts = tensors([10, 20_000], [F32, BF16])
    ts[1][19_999] = bad
    out = [torch.empty_like(t) for t in ts]
    n = ops.clip_by_global_norm(ts, 1.0, out=out)
    assert not math.isfinite(float(n)) and all(bool(o.isnan().all()) for o in out)


def adam64(p, g, m, v, t, lr, b1, b2, eps, clip):
    n = norm64(g)
    s = 1.0 if clip is None else min(1.0, clip / n)
    out = []
    for a, b, c, d in zip(p, g, m, v):
        b = b.double() * s
        c = c.double() + (b - c.double()) * (1 - b1)
        d = d.double() + (b * b - d.double()) * (1 - b2)
        out.append((a.double() - lr * math.sqrt(1 - b2 ** t) / (1 - b1 ** t) * c / (d.sqrt() + eps), c, d))
    return n, out


@pytest.mark.parametrize("gdtypes", [[F32], [BF16, F16, F32]])
@pytest.mark.parametrize("sizes", MANY)
@pytest.mark.parametrize("clip", [None, 0.4])
def test_adam_step(sizes, gdtypes, clip):
    p, m = tensors(sizes, [F32], 1), tensors(sizes, [F32], 200, 0.1)
    v = [x.square() for x in tensors(sizes, [F32], 400, 0.1)]
    lr, b1, b2, eps = 3e-3, 0.8, 0.99, 1e-5
    for t in (1, 2, 1000):
        g = tensors(sizes, gdtypes, 600 + t)
        n, want = adam64(p, g, m, v, t, lr, b1, b2, eps, clip)
        old = [x.clone() for x in p]
        om, ov = [x.double().abs() for x in m], [x.double().abs() for x in v]
        got = ops.adam_step(p, g, m, v, t, lr, b1, b2, eps, clip_norm=clip)
        assert (got is None) == (clip is None)
        if got is not None:
            assert abs(float(got) - n) <= 2 * U * n
        for a, b, c, (wa, wb, wc), q, gg, xm, xv in zip(p, m, v, want, old, g, om, ov):
            s = 1.0 if clip is None else min(1.0, clip / n)
            ga = gg.double().abs() * s
            em, ev = 6 * U * (xm + ga), 8 * U * (xv + ga * ga)
            check(b, wb, em, "m")
            check(c, wc, ev, "v")
            # the update is off by its own roundings, the moment's error, and sqrt(v)'s: sqrt(ev) where v is tiny
            upd = (wa - q.double()).abs()
            rel = torch.sqrt(ev) / (torch.sqrt(wc.clamp(min=0)) + eps)
            alpha = lr * math.sqrt(1 - b2 ** t) / (1 - b1 ** t)
            den = (torch.sqrt((wc - ev).clamp(min=0)) + eps)
            check(a, wa, 2 * U * q.double().abs() + upd * (12 * U + torch.minimum(rel, ev / den / den)) + alpha * em / den, "p")


def test_adam_step_number_on_the_gpu():
    a, b = [rnd(1000, seed=1)], [rnd(1000, seed=1)]
    g = [rnd(1000, seed=2)]
    z = [[torch.zeros(1000, device="cuda")] for _ in range(4)]
    t = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    ops.adam_step(a, g, z[0], z[1], 7)
    ops.adam_step(b, g, z[2], z[3], t)
    assert torch.equal(a[0], b[0])


def test_refusals_on_the_gpu():
    x, w, b = rnd(4, 8), rnd(8, 6), rnd(6)
    for args, kw in [((x, w.bfloat16()), {}), ((x, rnd(7, 6)), {}), ((x, w, rnd(5)), {}), ((x, w, b, "softmax"), {}),
                     ((x.double(), w.double()), {}), ((x.t(), rnd(4, 6)), {}), ((x.cpu(), w.cpu()), {}), ((x[0], w), {}),
                     ((x, w[:, ::2][:, :3]), {}), ((x, w, b), {"residual": rnd(4, 5)}), ((x, w, b), {"pre": rnd(4, 6).half()}),
                     ((x, w, b), {"out": rnd(3, 6)}), ((x, rnd(8, 8)), {"out": x[:, :8]}), ((x, w[:1].expand(8, 6)), {}),
                     ((rnd(1, 8).expand(4, 8), w), {})]:
        with pytest.raises(ValueError):
            ops.dense(*args, **kw)
    with pytest.raises(ValueError, match="overlaps"):
        buf = rnd(8, 6)
        ops.dense(x, w, b, residual=buf[1:5], out=buf[:4])
    with pytest.raises(ValueError, match="overlaps"):
        buf = rnd(4, 6)
        ops.dense(x, w, b, out=buf, pre=buf)
    with pytest.raises(ValueError, match="pre"):
        ops.dense_backward(rnd(4, 6), x, w, activation="elu")
    with pytest.raises(ValueError):
        ops.dense_backward(rnd(4, 5), x, w)
    t = rnd(100)
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_by_global_norm([t, t], 1.0)
    with pytest.raises(ValueError, match="overlap"):
        ops.clip_by_global_norm([t[:50], t[50:]], 1.0, out=[t[10:60], rnd(50)])
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([t], 0.0)
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([t], float("nan"))
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([t], 1.0, out=[rnd(99)])
    with pytest.raises(ValueError):
        ops.global_norm([rnd(4, 6).t()])
    with pytest.raises(ValueError):
        ops.global_norm([])
    with pytest.raises(ValueError):
        ops.global_norm([t.double()])
    m, v = torch.zeros_like(t), torch.zeros_like(t)
    for bad in [dict(step=0), dict(step=1, beta1=1.0), dict(step=1, eps=0.0), dict(step=1, lr=float("nan")), dict(step=1, clip_norm=-1.0)]:
        with pytest.raises(ValueError):
            ops.adam_step([t], [t.clone()], [m], [v], **bad)
    with pytest.raises(ValueError, match="overlap"):
        ops.adam_step([t], [t], [m], [v], 1)
    with pytest.raises(ValueError, match="overlap"):
        ops.adam_step([t], [t.clone()], [m], [m], 1)
    with pytest.raises(ValueError):
        ops.adam_step([t.half()], [t.clone()], [m], [v], 1)
    s = ops.TensorSet([t])
    t.data = torch.zeros(100, device="cuda")
    with pytest.raises(ValueError, match="storage"):
        ops.global_norm(s)


def test_a_training_step_of_residual_layers():
    """The operators together, as a training program uses them: forward through three residual layers, their gradients, one
    clipped update -- captured into a graph, replayed, and followed in 64 bits."""
    torch.manual_seed(0)
    B, W, L = 48, 96, 3
    xs = rnd(B, W, seed=1)
    target = rnd(B, W, seed=2)
    params = [p for i in range(L) for p in (rnd(W, W, seed=10 + i, scale=W ** -0.5), rnd(W, seed=20 + i, scale=0.1))]
    m, v = [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params]
    grads = [torch.empty_like(p) for p in params]
    sets = [ops.TensorSet(t) for t in (params, grads, m, v)]
    pre = [torch.empty(B, W, device="cuda") for _ in range(L)]
    step = torch.zeros((), dtype=torch.int32, device="cuda")
    norms = torch.zeros((), device="cuda")
    lr, clip = 1e-2, 0.5

    def train():
        step.add_(1)
        acts = [xs]
        for i in range(L):
            acts.append(ops.dense(acts[-1], params[2 * i], params[2 * i + 1], "elu", residual=acts[-1], pre=pre[i]))
        dy = (acts[-1] - target) / B
        for i in reversed(range(L)):
            dx, dw, db = ops.dense_backward(dy, acts[i], params[2 * i], pre[i], "elu", dx_add=dy)
            grads[2 * i].copy_(dw)
            grads[2 * i + 1].copy_(db)
            dy = dx
        norms.copy_(ops.adam_step(sets[0], sets[1], sets[2], sets[3], step, lr=lr, clip_norm=clip))

    ref = [p.double() for p in params]
    rm, rv = [torch.zeros_like(p) for p in ref], [torch.zeros_like(p) for p in ref]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        keep = [[t.clone() for t in q] for q in (params, m, v)]
        train()
        for q, k in zip((params, m, v), keep):
            for a, b in zip(q, k):
                a.copy_(b)
        step.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        train()
    for t in range(1, 6):
        graph.replay()
        leaves = [p.clone().requires_grad_(True) for p in ref]
        h = xs.double()
        for i in range(L):
            h = torch.nn.functional.elu(h @ leaves[2 * i] + leaves[2 * i + 1]) + h
        (0.5 * (h - target.double()).square().sum() / B).backward()
        n, new = adam64(ref, [q.grad for q in leaves], rm, rv, t, lr, 0.9, 0.999, 1e-7, clip)
        # gradients to ~1e-6 of their norm (sums of up to W + B float32 products through three layers); Adam's ratio m / sqrt(v) turns
        # a gradient's relative error into the same one of a step of lr, small gradients excepted: those are held by the norm
        assert abs(float(norms) - n) <= 1e-5 * n
        for a, b, (w, c, d) in zip(params, m, new):
            assert float((b.double() - c).norm()) <= 1e-5 * float(c.norm())
            assert float((a.double() - w).norm()) <= 1e-3 * lr * t * a.numel() ** 0.5 + 1e-6 * float(w.norm())
        ref, rm, rv = [w for w, _, _ in new], [c for _, c, _ in new], [d for _, _, d in new]


@pytest.mark.parametrize("m,k,n", [(4, 128, 200), (40, 128, 200), (600, 100, 600), (600, 1024, 1200)])
def test_subnormal_halves_are_kept(m, k, n):
    """float16 values below 2^-14 enter the products as they are (rows, slim, tile and large kernels)."""
    x, w = rnd(m, k, dtype=F16, seed=1, scale=2.0 ** -18), rnd(k, n, dtype=F16, seed=2)
    check_forward(x, w, None, "linear", None, ops.dense(x, w))
    dy = rnd(m, n, dtype=F16, seed=3, scale=2.0 ** -18)
    check_backward(dy, x, w, None, "linear", None, *ops.dense_backward(dy, x, w))


def test_products_of_one_hot_rows_are_exact():
    """A row of zeros and a one picks a row of w, to the bit, whatever the kernel."""
    for m, k, n, dtype in ((3, 50, 70, F32), (60, 50, 70, F32), (500, 40, 900, F32), (500, 512, 900, F32), (500, 1024, 900, BF16)):
        w = rnd(k, n, dtype=dtype, seed=1)
        pick = torch.arange(m, device="cuda") % k
        x = torch.zeros(m, k, dtype=dtype, device="cuda")
        x[torch.arange(m, device="cuda"), pick] = 1
        assert torch.equal(ops.dense(x, w), w[pick])
        assert torch.equal(ops.dense(x, w.t().contiguous().t()), w[pick])


def test_two_streams_at_once():
    """Calls on two streams that overlap in time share nothing."""
    m, k, n = 900, 700, 800
    ins = [[rnd(*s, seed=10 * i + j) for j, s in enumerate([(m, k), (k, n), (n,), (m, n)])] for i in range(2)]
    z = [torch.empty(m, n, device="cuda") for _ in range(2)]

    def work(i):
        x, w, b, dy = ins[i]
        y = ops.dense(x, w, b, "tanh", pre=z[i])
        out = [torch.empty_like(x), torch.empty_like(w)]
        norm = ops.clip_by_global_norm([x, w], 1.0 + i, out=out)
        return [y, *ops.dense_backward(dy, x, w, z[i], "tanh"), norm, *out]

    want = [[t.clone() for t in work(i)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = work(i)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


# sizes at which the choice of kernel changes: few rows of odd weights, long and short contractions
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(1, 700, 8000), (2, 120, 1559), (3, 20_000, 5), (4, 5000, 70), (2, 3, 20_000), (9, 1216, 1301), (31, 300, 5003),
                                   (48, 2401, 500), (130, 130, 515), (600, 130, 2500), (7, 2401, 7003), (5, 520, 100_003)])
def test_what_lies_beside_an_operand_never_enters(m, k, n, dtype):
    """Every operand is cut out of a buffer of NaN."""
    def inside(t):
        buf = torch.full((t.shape[0] + 2, t.shape[1] + 17), float("nan"), dtype=t.dtype, device="cuda")
        view = buf[1:-1, 9:9 + t.shape[1]]
        view.copy_(t)
        return view

    act = ACTS[(m + k + n) % 7]
    for w_t in (False, True):
        x, r, dy = (inside(rnd(m, j, dtype=dtype, seed=q)) for q, j in ((1, k), (2, n), (3, n)))
        w = rnd(k, n, dtype=dtype, seed=4, scale=k ** -0.5)
        w = inside(w.t()).t() if w_t else inside(w)
        b, z = inside(rnd(1, n, dtype=dtype, seed=5))[0], inside(torch.zeros(m, n, device="cuda"))
        check_forward(x, w, b, act, r, ops.dense(x, w, b, act, residual=r, pre=z), z)
        check_backward(dy, x, w, z, act, None, *ops.dense_backward(dy, x, w, z, act))
