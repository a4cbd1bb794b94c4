"""The operators' C ABI and refusals without a GPU: a refused call launches nothing, so these run on the CPU."""
import ctypes as C
import os
import re

import pytest
import torch

from popvae_amd import ops


def test_header_symbols():
    hdr = open(os.path.join(os.path.dirname(__file__), "..", "include", "pvae_ops.h")).read()
    declared = set(re.findall(r"\b(pvae_\w+)\s*\(", hdr))
    assert declared == set(ops.OPS_SYMBOLS)
    for s in declared:
        assert hasattr(ops.lib(), s)


def test_structures_match_the_header():
    hdr = open(os.path.join(os.path.dirname(__file__), "..", "include", "pvae_ops.h")).read()
    for name, struct in (("pvae_dense_args", ops._Dense), ("pvae_dense_bwd_args", ops._DenseBwd), ("pvae_tensor", ops._Tensor)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, hdr, re.S).group(1)
        fields = [f.strip(" *") for line in re.findall(r"[^;]+;", body) for f in
                  re.sub(r"^\s*(const\s+)?(int32_t|int64_t|void|float)\b", "", line.strip().rstrip(";")).split(",")]
        assert fields == [f for f, _ in struct._fields_]


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 3), torch.zeros(3, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.dense(x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.dense_backward(torch.zeros(2, 4), x, w)
    with pytest.raises(ValueError):
        ops.global_norm([x])
    with pytest.raises(ValueError):
        ops.TensorSet([x])


def dense_args(**kw):
    a = dict(dtype=0, act=0, m=2, k=4, n=8, x=4096, ldx=4, w=8192, w_sk=8, w_sn=1, bias=None, residual=None, ldr=0, y=16384, ldy=8,
             pre=None, ldp=0)
    a.update(kw)
    return ops._Dense(**a)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "type"), (dict(act=7), "activation"), (dict(m=-1), "sizes"), (dict(n=1 << 31), "sizes"), (dict(x=None), "x is NULL"),
    (dict(x=4097), "aligned"), (dict(ldx=3), "x: row stride"), (dict(ldx=1 << 60), "too large"), (dict(w_sk=7), "w: row stride"),
    (dict(w_sk=16, w_sn=2), "neither"), (dict(n=1, ldy=1, w_sk=0), "w: row stride"), (dict(n=1, ldy=1, w_sk=-4), "w: row stride"), (dict(w_sk=1, w_sn=3), "w\\^T"), (dict(y=None), "y is NULL"), (dict(ldy=7), "y: row stride"),
    (dict(residual=4096, ldr=5), "residual"), (dict(pre=4098, ldp=8), "pre is not aligned"), (dict(pre=65536, ldp=4), "pre: row"), (dict(y=4096), "y overlaps x"), (dict(y=8192 + 60), "y overlaps w"),
    (dict(pre=16384 + 32, ldp=8), "y overlaps pre"), (dict(residual=16384 + 4, ldr=8), "y overlaps residual"),
    (dict(residual=16384, ldr=12), "y overlaps residual"), (dict(pre=4096, ldp=8, residual=16384, ldr=8), "pre overlaps x"),
    (dict(bias=16384 + 8), "y overlaps bias")])
def test_dense_refusals(kw, text):
    a = dense_args(**kw)
    assert ops.lib().pvae_dense(C.byref(a), None, 0, None) < 0
    assert re.search(text, ops.lib().pvae_ops_last_error().decode())
    assert ops.lib().pvae_dense_workspace(C.byref(a)) == 0


def bwd_args(**kw):
    a = dict(dtype=0, act=2, m=2, k=4, n=8, dy=4096, lddy=8, x=8192, ldx=4, w=12288, w_sk=8, w_sn=1, pre=16384, ldp=8, dx=20480, lddx=4,
             dx_add=None, ldadd=0, dw=24576, dbias=28672, dpre=32768)
    a.update(kw)
    return ops._DenseBwd(**a)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=-1), "type"), (dict(act=9), "activation"), (dict(k=-1), "sizes"), (dict(dy=None), "dy is NULL"), (dict(lddy=7), "dy: row"),
    (dict(pre=None), "pre is NULL"), (dict(pre=16386), "pre is not aligned"), (dict(x=None), "x is NULL"), (dict(w=None), "w is NULL"),
    (dict(lddx=3), "dx: row"), (dict(dx_add=40960, ldadd=2), "dx_add: row"), (dict(dw=24577), "dw is not aligned"),
    (dict(dbias=28673), "dbias is not aligned"), (dict(dpre=32769), "dpre is not aligned"), (dict(dx=4096), "dx overlaps dy"),
    (dict(dw=8192), "dw overlaps x"), (dict(dbias=12288), "dbias overlaps w"), (dict(dpre=16384), "dpre overlaps pre"),
    (dict(dx=24576), "dx overlaps dw"), (dict(dx_add=20484, ldadd=4), "dx overlaps dx_add")])
def test_dense_bwd_refusals(kw, text):
    a = bwd_args(**kw)
    assert ops.lib().pvae_dense_bwd(C.byref(a), None, 0, None) < 0
    assert re.search(text, ops.lib().pvae_ops_last_error().decode())


def test_packed_arguments_are_the_structures():
    for struct, packed in ((ops._Dense, ops._pack_dense), (ops._DenseBwd, ops._pack_bwd)):
        values = list(range(1, len(struct._fields_) + 1))
        assert packed(*values) == bytes(struct(*values))


def test_empty_calls_do_nothing():
    assert ops.lib().pvae_dense(C.byref(dense_args(m=0, x=None, y=None)), None, 0, None) == 0
    assert ops.lib().pvae_dense(C.byref(dense_args(n=0, w=None, y=None)), None, 0, None) == 0
    assert ops.lib().pvae_dense(None, None, 0, None) == -1


def test_a_missing_workspace_is_refused():
    a = dense_args(m=64, k=100_000, n=64, x=1 << 32, ldx=100_000, w=1 << 33, w_sk=64, y=1 << 34, ldy=64)
    need = ops.lib().pvae_dense_workspace(C.byref(a))
    assert need > 0
    for ptr, have in ((None, need), (4096, need - 1), (4097, need)):
        assert ops.lib().pvae_dense(C.byref(a), ptr, have, None) < 0
        assert "workspace" in ops.lib().pvae_ops_last_error().decode()


def table(*rows):
    return (ops._Tensor * len(rows))(*rows)


def test_many_tensor_refusals():
    L = ops.lib()
    need = L.pvae_norm_workspace()
    ok = table((4096, 10, 0, 0))
    for t, n in ((ok, -1), (ok, 65537), (None, 1), (table((None, 5, 0, 0)), 1), (table((4097, 5, 0, 0)), 1), (table((4096, 5, 3, 0)), 1),
                 (table((4096, -5, 0, 0)), 1), (table((4096, 8, 0, 4)), 1)):
        assert L.pvae_global_norm(t, n, 64, 4096, need, None) < 0
    assert L.pvae_global_norm(ok, 1, None, 4096, need, None) < 0
    assert L.pvae_global_norm(ok, 1, 64, 4096, need - 1, None) < 0
    for out, c in ((table((4100, 10, 0, 0)), 1.0), (table((8192, 9, 0, 0)), 1.0), (table((8192, 10, 1, 0)), 1.0), (ok, 0.0),
                   (ok, float("nan")), (ok, -1.0)):
        assert L.pvae_clip_by_global_norm(ok, out, 1, c, None, 4096, need, None) < 0
    p, g, m, v = (table((i * 4096, 8, 0, 0)) for i in range(1, 5))
    good = [1e-3, 0.9, 0.999, 1e-7, 1, None, 0.0]

    def adam(p=p, g=g, m=m, v=v, **kw):
        a = dict(zip(("lr", "b1", "b2", "eps", "step", "step_dev", "clip"), good), **kw)
        return L.pvae_adam_step(p, g, m, v, 1, a["lr"], a["b1"], a["b2"], a["eps"], a["step"], a["step_dev"], a["clip"], None, None, 0, None)

    for kw in (dict(lr=float("inf")), dict(b1=1.0), dict(b2=-0.1), dict(eps=0.0), dict(eps=1e-60), dict(eps=1e60), dict(step=0), dict(clip=-1.0), dict(clip=1.0),
               dict(p=g), dict(m=v), dict(p=table((4096, 8, 1, 0))), dict(g=table((8192, 9, 0, 0))), dict(p=table((4096, 8, 0, 4))),
               dict(p=table((4096, 8, 0, 4)), m=table((4096 + 16, 8, 0, 4)), v=table((4096 + 16, 8, 0, 4)))):
        assert adam(**kw) < 0, kw
    assert L.pvae_adam_step(p, g, m, v, 0, *good, None, None, 0, None) == 0  # no tensors: nothing to do


K = 100_000  # a contraction that is split: an accepted call asks for a workspace, a refused one for none
X, W, Y = 1 << 30, 1 << 31, 1 << 32


@pytest.mark.parametrize("kw,ok", [
    (dict(), True), (dict(y=X + 4 * K, ldy=K + 8), True), (dict(y=X + 4 * K - 4, ldy=K + 8), False), (dict(y=X + 4 * K + 4, ldy=K + 8), False),
    (dict(y=X - 32, ldy=K + 8), True), (dict(y=X - 28, ldy=K + 8), False), (dict(y=X + 4 * K, ldy=K + 9), False),
    (dict(y=X + 4 * (2 * K + 8), ldy=K + 8), True), (dict(m=1, y=X + 4 * K, ldy=8), True), (dict(m=1, y=X + 4 * K - 4, ldy=8), False),
    (dict(w_sk=20, y=W + 32, ldy=20), True), (dict(w_sk=20, y=W + 28, ldy=20), False), (dict(w_sk=20, y=W + 52, ldy=20), False),
    (dict(w_sk=1, w_sn=K + 8, y=W + 4 * K, ldy=K + 8), True), (dict(w_sk=1, w_sn=K + 8, y=W + 4 * K - 4, ldy=K + 8), False),
    (dict(ldy=16, pre=Y + 32, ldp=16), True), (dict(ldy=16, pre=Y + 28, ldp=16), False), (dict(ldy=16, pre=Y + 32, ldp=15), False),
    (dict(ldy=16, bias=Y + 32), True), (dict(ldy=16, bias=Y + 28), False), (dict(ldy=16, bias=Y + 36), False),
    (dict(ldy=16, residual=Y + 32, ldr=0), True), (dict(ldy=16, residual=Y + 28, ldr=0), False), (dict(ldy=16, residual=Y, ldr=16), True),
    (dict(ldy=16, residual=Y, ldr=0), False)])
def test_columns_of_one_buffer_are_apart(kw, ok):
    """An output may lie between the rows of an operand, at the byte."""
    a = dense_args(**dict(dict(m=2, k=K, n=8, x=X, ldx=K + 8, w=W, w_sk=8, y=Y, ldy=8), **kw))
    assert (ops.lib().pvae_dense_workspace(C.byref(a)) > 0) == ok
    if not ok:
        assert "overlaps" in ops.lib().pvae_ops_last_error().decode()
