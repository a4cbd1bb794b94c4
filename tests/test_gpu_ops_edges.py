"""The operators on device tensors (popvae_amd.ops) at the edges of what they take, against 64-bit formulas.

Where the inputs are small whole numbers and f' is 0 or 1 (linear, relu), every product and every sum is exact in float32
(below 2^24), so a result is the exact one rounded once to its type: such tests compare bit for bit, and one product lost,
added or taken from a neighbour shows.  Elsewhere the tolerances count roundings: u = 2^-24, h = finfo.eps / 2 of the type,
tiny = half its smallest subnormal."""
import ctypes as C
import math

import pytest
import torch

from popvae_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def whole(*shape, dtype=F32, seed=0, top=2):
    """Whole numbers -top .. top."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(dtype)


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def f64(t):
    return t.double().contiguous()


def half(t):
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def act64(z, name):
    return {"linear": lambda: z, "relu": lambda: torch.relu(z), "elu": lambda: torch.where(z > 0, z, torch.expm1(z)),
            "sigmoid": lambda: torch.sigmoid(z), "tanh": lambda: torch.tanh(z), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.erfc(-z / math.sqrt(2)) / 2}[name]()


def dact64(z, name):
    z = z.clone().requires_grad_(True)
    act64(z, name).sum().backward()
    return z.grad


def grads64(dy, x, w, z, act):
    """dx, dw and db in 64 bits."""
    g = f64(dy) if act == "linear" else f64(dy) * dact64(f64(z), act)
    return g @ f64(w).t().contiguous(), f64(x).t().contiguous() @ g, g.sum(0)


def check(got, want, bound, what):
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs().max()), float(bound.max()))


def check_exact(x, w, dy, z, dtype):
    """Forward and gradients of whole numbers, bit for bit."""
    pre = torch.empty(x.shape[0], w.shape[1], device="cuda")
    y = ops.dense(x, w, activation="relu", pre=pre)
    want = f64(x) @ f64(w)
    assert torch.equal(pre.double(), want) and torch.equal(y, want.clamp(min=0).to(dtype))
    for act in ("relu", "linear"):
        got = ops.dense_backward(dy, x, w, z, act)
        for name, a, b in zip(("dx", "dw", "db"), got, grads64(dy, x, w, z, act)):
            assert torch.equal(a, b.to(dtype)), (act, name, int((a.double() != b).sum()))


# one column, or one row, of weights cut out of a wider tensor: neither stride is 1
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [3, 40, 600, 2000])
def test_a_single_column_or_row_of_weights_with_any_strides(m, dtype):
    k, n = 70, 70
    x, dy, z = whole(m, k, dtype=dtype, seed=1), whole(m, 1, dtype=dtype, seed=2), rnd(m, 1, seed=3)
    w = whole(k, 10, dtype=dtype, seed=4)[:, ::5][:, :1]
    assert w.stride() == (10, 5)
    check_exact(x, w, dy, z, dtype)
    x, dy, z = whole(m, 1, dtype=dtype, seed=5), whole(m, n, dtype=dtype, seed=6), rnd(m, n, seed=7)
    w = whole(9, 3 * n, dtype=dtype, seed=8)[::7, ::3][:1]
    assert w.stride() == (21 * n, 3)
    check_exact(x, w, dy, z, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_single_row_of_weights_in_the_large_kernel(dtype):
    """k = 1 and a result of 2^30 elements, w's only row with neither stride 1: every product is exact."""
    m = n = 1 << 15
    x, w = whole(m, 1, dtype=dtype, seed=1), whole(9, 3 * n, dtype=dtype, seed=2)[::7, ::3][:1]
    assert torch.equal(ops.dense(x, w), x * w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [2, 9, 40, 300, 700])
@pytest.mark.parametrize("dy_ld,pre_ld", [(1, 4), (1, 7), (5, 1), (3, 2)])
def test_a_single_output_with_strided_pre_or_dy(m, dy_ld, pre_ld, dtype):
    """n = 1: dy's rows lie next to each other and pre's do not, or the other way round."""
    k = 33
    x, w = whole(m, k, dtype=dtype, seed=1), whole(k, 1, dtype=dtype, seed=2)
    dy = whole(m, dy_ld, dtype=dtype, seed=3)[:, dy_ld // 2:][:, :1]
    z = rnd(m, pre_ld, seed=4)[:, pre_ld // 2:][:, :1]
    check_exact(x, w, dy, z, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(5, 9, 4), (40, 70, 50), (260, 24, 20), (700, 256, 300)])
@pytest.mark.parametrize("act", ["silu", "relu", "elu"])
def test_infinities_in_the_gradients_operands(m, k, n, act, dtype):
    """An infinite x or w makes the gradients that it enters infinite, with the formula's sign, whatever kernel runs; NaN
    only where the formula has it (0 times infinity, infinities of both signs)."""
    x, w, dy, z = rnd(m, k, dtype=dtype, seed=1), rnd(k, n, dtype=dtype, seed=2), rnd(m, n, dtype=dtype, seed=3), rnd(m, n, seed=4)
    x[1, 3], x[m - 1, 0], w[2, 1], w[k - 1, n - 1] = float("inf"), float("-inf"), float("-inf"), float("inf")
    dy[0] = 1.0  # exact in every type
    for name, a, b in zip(("dx", "dw", "db"), ops.dense_backward(dy, x, w, z, act), grads64(dy, x, w, z, act)):
        assert torch.equal(a.isnan(), b.isnan()), (name, int(a.isnan().sum()), int(b.isnan().sum()))
        assert torch.equal(a.isinf(), b.isinf()) and torch.equal(a[a.isinf()].double(), b[b.isinf()]), name


def check_gradients_rounded_once(dy, x, w, z, act, dtype):
    """dx and dw are off by what f' (16 u (1 + |z|)), g's two terms (bf16: 2^-16 of g -- what cutting the first
    off leaves is below 2^-7 of g, and the second is off by 2^-9 of that; f16: 2^-21 and 2^-35; float32: u) and
    float32 sums (u a term) are off by, and one rounding of the result: a rounding of g to a 16-bit type is not in it."""
    dx, dw, _ = ops.dense_backward(dy, x, w, z, act)
    X, W, DY, Z = f64(x), f64(w), f64(dy), f64(z)
    G = DY * dact64(Z, act)
    rel, least = {F32: (2 * U, 0.0), BF16: (2.0 ** -16, 0.0), F16: (2.0 ** -21, 2.0 ** -35)}[dtype]
    eg = 16 * U * (1 + Z.abs()) * DY.abs() + rel * G.abs() + least
    h, tiny = half(dtype)
    for what, got, want, e, terms, size in (
            ("dx", dx, G @ W.t().contiguous(), eg @ W.t().abs().contiguous(), W.shape[1], (G.abs() + eg) @ W.t().abs().contiguous()),
            ("dw", dw, X.t().contiguous() @ G, X.t().abs().contiguous() @ eg, X.shape[0], X.t().abs().contiguous() @ (G.abs() + eg))):
        # a sum of `terms` values (twice as many with two terms of g) is off by u a term of the values' sizes
        e = e + (2 * terms + 8) * U * size
        check(got, want, e + h * (want.abs() + e) + tiny, (what, act))


# few terms to a sum, so that a second rounding could not hide among others; both kernels of the gradients
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 5, 3), (2, 300, 2), (3, 40, 1), (40, 30, 3), (200, 17, 40), (300, 260, 2), (700, 300, 3),
                                   (700, 512, 16), (260, 2000, 1), (2048, 24, 8), (513, 130, 70), (1024, 256, 512)])
def test_gradients_are_rounded_once(m, k, n, dtype):
    for act in ("gelu", "tanh"):
        x, w, dy, z = rnd(m, k, dtype=dtype, seed=1), rnd(k, n, dtype=dtype, seed=2), rnd(m, n, dtype=dtype, seed=3), rnd(m, n, seed=4)
        check_gradients_rounded_once(dy, x, w, z, act, dtype)
        check_gradients_rounded_once(dy, x, rnd(n, k, dtype=dtype, seed=5).t(), z, act, dtype)


@pytest.mark.parametrize("m,k,n", [(3, 20, 4), (40, 30, 50), (300, 30, 50), (700, 256, 300)])
def test_half_precision_gradients_beyond_the_types_range(m, k, n):
    """float16: dy f'(pre) below the least subnormal or above the largest value, while the gradients themselves fit."""
    z = rnd(m, n, seed=4)
    small = rnd(m, n, dtype=F16, seed=3, scale=2.0 ** -22)
    x, w = rnd(m, k, dtype=F16, seed=1, scale=2.0 ** 10), rnd(k, n, dtype=F16, seed=2, scale=2.0 ** 10)
    for act in ("silu", "sigmoid"):
        check_gradients_rounded_once(small, x, w, z, act, F16)
    large = torch.where(rnd(m, n, seed=5) > 0, 60000.0, -61000.0).to(F16)  # times gelu'(sqrt 2) = 1.128: above 65504
    z = torch.full((m, n), math.sqrt(2.0), device="cuda")
    x, w = rnd(m, k, dtype=F16, seed=1, scale=2.0 ** -9), rnd(k, n, dtype=F16, seed=2, scale=2.0 ** -9)
    check_gradients_rounded_once(large, x, w, z, "gelu", F16)


def test_activations_far_from_zero():
    """The tails of the activations and their derivatives in float32, relative to their own size: exp, the sum and the
    reciprocal are off by 5 u together, every product by u more."""
    z = torch.cat([torch.linspace(-80, 80, 40_001, device="cuda"), -torch.logspace(-6, 1.9, 999, device="cuda")])[:, None].contiguous()
    one = torch.ones(1, 1, device="cuda")
    Z = z.double()
    s, q = torch.sigmoid(Z), torch.sigmoid(-Z)
    check(ops.dense(z, one, activation="sigmoid"), s, 8 * U * s, "sigmoid")
    check(ops.dense(z, one, activation="silu"), Z * s, 10 * U * (Z * s).abs(), "silu")

    def slope(act):
        return ops.dense_backward(torch.ones_like(z), z, one, z, act, need_dw=False, need_bias=False)[0]

    check(slope("sigmoid"), s * q, 18 * U * s * q, "sigmoid'")
    check(slope("elu"), torch.exp(Z.clamp(max=0)), 4 * U * torch.exp(Z.clamp(max=0)), "elu'")
    check(slope("silu"), s * (1 + Z * q), 18 * U * s * (1 + Z.abs() * q), "silu'")
    phi = torch.exp(-Z * Z / 2) / math.sqrt(2 * math.pi)
    # z^2 / 2 is rounded before exp sees it (u z^2 / 2, relative); Phi comes from 1 + erf: 4 u absolute
    check(slope("gelu"), torch.special.ndtr(Z) + Z * phi, 4 * U + (10 + Z * Z) * U * (Z * phi).abs(), "gelu'")


def test_activations_of_infinities_and_nan():
    z = torch.tensor([[float("inf")], [float("-inf")], [float("nan")], [3e38], [-3e38]], device="cuda")
    one = torch.ones(1, 1, device="cuda")
    for act in ("sigmoid", "tanh", "relu", "elu"):
        y = ops.dense(z, one, activation=act)
        assert torch.equal(torch.nan_to_num(y.double(), 7.0, 8.0, 9.0), torch.nan_to_num(act64(z.double(), act), 7.0, 8.0, 9.0)), act
        g = ops.dense_backward(torch.ones_like(z), z, one, z, act, need_dw=False, need_bias=False)[0]
        want = {"sigmoid": [0.0, 0.0, 0.0, 0.0], "tanh": [0.0, 0.0, 0.0, 0.0], "relu": [1.0, 0.0, 1.0, 0.0], "elu": [1.0, 0.0, 1.0, 0.0]}[act]
        assert g[[0, 1, 3, 4], 0].tolist() == want, act


# contractions in pieces and their remainders, ragged ends, unaligned rows, long sums over rows: nothing may be lost, added
# or taken twice
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 8192, 96), (2, 70_001, 33), (4, 1000, 4099), (8, 3159, 2001), (16, 8192, 130), (33, 5000, 65),
                                   (64, 4001, 403), (130, 70_001, 129), (192, 8192, 256), (5, 2048, 4099), (5, 520, 100_003),
                                   (600, 2500, 17), (20_011, 24, 40), (4000, 64, 64), (1543, 1021, 515), (70_001, 130, 3)])
def test_whole_numbers_are_exact(m, k, n, dtype):
    x, dy, z = whole(m, k, dtype=dtype, seed=1), whole(m, n, dtype=dtype, seed=2), rnd(m, n, seed=3)
    check_exact(x, whole(k, n, dtype=dtype, seed=4), dy, z, dtype)
    check_exact(x, whole(n, k, dtype=dtype, seed=5).t(), dy, z, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 4, 1), (32, 128, 128), (33, 65, 129), (700, 40, 70), (600, 256, 513)])
def test_g_itself(m, k, n, dtype):
    """pvae_dense_bwd's dpre, unrounded, from both kernels, alone and beside the gradients."""
    x, w, dy, z = rnd(m, k, dtype=dtype, seed=1), rnd(k, n, dtype=dtype, seed=2), rnd(m, n, dtype=dtype, seed=3), rnd(m, n, seed=4)
    L = ops.lib()
    for act in ("linear", "relu", "gelu"):
        G = f64(dy) if act == "linear" else f64(dy) * dact64(f64(z), act)
        bound = 0 * G if act != "gelu" else 16 * U * (1 + f64(z).abs()) * f64(dy).abs() + U * G.abs()
        for alone in (False, True):
            g = torch.full((m + 1, n), float("nan"), device="cuda")
            dx, dw, db = torch.empty_like(x), torch.empty(k, n, dtype=dtype, device="cuda"), torch.empty(n, dtype=dtype, device="cuda")
            a = ops._DenseBwd(dtype=ops.DTYPES[dtype], act=ops.ACTIVATIONS[act], m=m, k=k, n=n, dy=dy.data_ptr(), lddy=n, x=x.data_ptr(),
                              ldx=k, w=w.data_ptr(), w_sk=n, w_sn=1, pre=z.data_ptr(), ldp=n, dpre=g.data_ptr())
            if not alone:
                a.dx, a.lddx, a.dw, a.dbias = dx.data_ptr(), k, dw.data_ptr(), db.data_ptr()
            need = L.pvae_dense_bwd_workspace(C.byref(a))
            work = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
            assert L.pvae_dense_bwd(C.byref(a), work.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
            check(g[:m], G, bound, act)
            assert bool(g[m].isnan().all())
            if not alone:
                want = ops.dense_backward(dy, x, w, z, act)
                assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 30, 20), (4, 70, 33), (40, 128, 64), (300, 130, 200), (700, 256, 512)])
def test_operands_that_are_columns_of_one_buffer(m, k, n, dtype):
    """x, the residual, y and dy side by side in one buffer; w and dw's source likewise: nothing beside an output is written."""
    buf = whole(m, k + 3 * n + 5, dtype=dtype, seed=1)
    x, r, y, dy = buf[:, 1:1 + k], buf[:, 1 + k:1 + k + n], buf[:, 1 + k + n:1 + k + 2 * n], buf[:, 3 + k + 2 * n:3 + k + 3 * n]
    both = whole(k, 2 * n, dtype=dtype, seed=2)
    w, z = both[:, :n], torch.empty(m, 2 * n, device="cuda")
    before, want = buf.clone(), (f64(x) @ f64(w)).clamp(min=0) + f64(r)
    assert ops.dense(x, w, activation="relu", residual=r, pre=z[:, n:], out=y).data_ptr() == y.data_ptr()
    assert torch.equal(y, want.to(dtype)) and torch.equal(z[:, n:].double(), f64(x) @ f64(w))
    before[:, 1 + k + n:1 + k + 2 * n] = y
    assert torch.equal(buf, before)
    for name, a, b in zip(("dx", "dw", "db"), ops.dense_backward(dy, x, w, z[:, n:], "relu"), grads64(dy, x, w, z[:, n:], "relu")):
        assert torch.equal(a, b.to(dtype)), name
    if m > 1:
        with pytest.raises(ValueError, match="overlaps"):
            ops.dense(x, w, out=buf[:, k:k + n])  # x's last column
        with pytest.raises(ValueError, match="overlaps"):
            ops.dense(x, w, out=buf.view(-1)[k + 1:k + 1 + m * n].view(m, n))  # rows of another length


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(2, 5, 1), (40, 30, 50), (300, 70, 1), (700, 256, 300)])
def test_an_expanded_row_as_dy(m, k, n, dtype):
    x, w, z = whole(m, k, dtype=dtype, seed=1), whole(k, n, dtype=dtype, seed=2), rnd(m, n, seed=3)
    dy = whole(1, n, dtype=dtype, seed=4).expand(m, n)
    check_exact(x, w, dy, z, dtype)
    for a, b in zip(ops.dense_backward(dy, x, w, z, "gelu"), ops.dense_backward(dy.contiguous(), x, w, z, "gelu")):
        assert torch.equal(a, b)


def test_autograd_is_not_left_in_the_dark():
    """A tensor that requires a gradient is refused where autograd would record; without recording the same call runs."""
    x, w, b, r, z, dy = rnd(5, 6, seed=1), rnd(6, 4, seed=2), rnd(4, seed=3), rnd(5, 4, seed=4), rnd(5, 4, seed=5), rnd(5, 4, seed=6)
    y = ops.dense(x, w, b, "elu", residual=r)
    for t in (x, w, b, r):
        t.requires_grad_(True)
        with pytest.raises(ValueError, match="no_grad"):
            ops.dense(x, w, b, "elu", residual=r)
        with torch.no_grad():
            assert torch.equal(ops.dense(x, w, b, "elu", residual=r), y)
        t.requires_grad_(False)
    for t in (x, w, dy, z):
        t.requires_grad_(True)
        with pytest.raises(ValueError, match="no_grad"):
            ops.dense_backward(dy, x, w, z, "elu")
        with torch.inference_mode():
            ops.dense_backward(dy, x, w, z, "elu")
        t.requires_grad_(False)
    # parameters that require a gradient are what an optimizer updates
    p = [w.clone().requires_grad_(True)]
    ops.adam_step(p, [rnd(6, 4, seed=7)], [torch.zeros_like(w)], [torch.zeros_like(w)], 1)
    assert p[0].requires_grad and not torch.equal(p[0].detach(), w)


def test_what_is_written_in_place_counts_as_changed():
    """A tensor that autograd has saved and an operator overwrites makes the backward fail, as torch's own in-place operations do."""
    x, w, g = rnd(5, 6, seed=1), rnd(6, 6, seed=2), rnd(5, 6, seed=3)
    m, v = torch.zeros_like(g), torch.zeros_like(g)

    def writes():
        yield "out", lambda t: ops.dense(x, w, out=t)
        yield "pre", lambda t: ops.dense(x, w, pre=t)
        yield "clip in place", lambda t: ops.clip_by_global_norm([t], 0.1)
        yield "clip into", lambda t: ops.clip_by_global_norm([g], 0.1, out=[t])
        yield "parameters", lambda t: ops.adam_step([t], [g], [m], [v], 1)
        yield "first moment", lambda t: ops.adam_step([m], [g], [t], [v], 1)
        yield "second moment", lambda t: ops.adam_step([m], [g], [v], [t], 1)

    for name, write in writes():
        a, saved = rnd(5, 6, seed=4).requires_grad_(True), rnd(5, 6, seed=5).abs()
        loss = (a * saved).sum()  # saves `saved`
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
            raise AssertionError(name)
        loss = (a * saved).sum()
        loss.backward()
        assert torch.equal(a.grad, saved), name


def test_a_set_keeps_the_storage_that_it_describes():
    """A tensor of the set that lets go of its storage and later gets another of fewer elements: the allocator may hand out the
    same address again, so the set holds on to the storage and refuses the tensor."""
    t = rnd(1000, seed=1)
    s, at = ops.TensorSet([t]), t.data_ptr()
    t.data = torch.empty(0, device="cuda")
    others = [torch.zeros(990, device="cuda") for _ in range(64)]
    assert at not in [o.data_ptr() for o in others]
    for o in others:
        t.data = o
        with pytest.raises(ValueError, match="storage"):
            ops.global_norm(s)
