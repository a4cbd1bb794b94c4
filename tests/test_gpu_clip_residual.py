"""Clipping by the global gradient norm and residual hidden layers in the engine (pvae_set_clip_norm, pvae_set_residual)."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import popvae_oracle as O
from popvae_amd import engine, prep

pytestmark = pytest.mark.gpu


def make(L, W, D, K, B, N=150, seed=0, lr=1e-3):
    g = np.random.default_rng(seed)
    dc = g.binomial(2, np.clip(g.beta(0.5, 0.5, L), 0.02, 0.98), size=(N, L)) * 0.5
    w = [x + (0.05 * g.normal(size=x.shape).astype(np.float32) if x.ndim == 1 else 0) for x in O.init_weights(L, W, D, K, seed=seed, dtype=np.float32)]

    def new():
        e = engine.Engine(n_snps=L, width=W, depth=D, latent_dim=K, batch_size=B, seed=3, lr=lr)
        e.load_genotypes(prep.pack_dc(dc))
        e.set_weights(w)
        return e
    return new, dc, w


def vae64(w, x, eps, D, K, residual):
    """Loss and gradients of the model in 64 bits (torch, CPU): popvae.py:392-424, residual hidden layers if asked for."""
    p = [torch.from_numpy(np.asarray(t, np.float64)).requires_grad_(True) for t in w]
    it = iter(p)
    X = torch.from_numpy(np.asarray(x, np.float64))
    E = torch.from_numpy(np.asarray(eps, np.float64))
    elu = torch.nn.functional.elu
    h = elu(X @ next(it) + next(it))
    for _ in range(D - 1):
        y = elu(h @ next(it) + next(it))
        h = y + h if residual else y
    mu = h @ next(it) + next(it)
    s = h @ next(it) + next(it)
    z = mu + torch.exp(s) * E
    h = z @ next(it) + next(it)
    for _ in range(D - 1):
        y = elu(h @ next(it) + next(it))
        h = y + h if residual else y
    a = h @ next(it) + next(it)
    rec = torch.nn.functional.binary_cross_entropy_with_logits(a, X, reduction="none").sum(1)
    kl = -0.5 * (1 + s - mu * mu - torch.exp(s)).sum(1)
    loss = (rec + kl).mean()
    loss.backward()
    return float(loss.detach()), [t.grad.numpy() for t in p], (mu.detach().numpy(), s.detach().numpy())


CASES = [(1000, 128, 6, 2, 32), (700, 32, 3, 3, 32), (900, 512, 2, 2, 32), (600, 100, 1, 2, 32), (800, 256, 3, 2, 48),
         (1300, 128, 3, 2, 100), (1000, 128, 2, 2, 140)]


@pytest.mark.parametrize("L,W,D,K,B", CASES)
def test_residual_layers_against_64_bits(L, W, D, K, B):
    new, dc, w = make(L, W, D, K, B)
    e = new()
    e.set_residual()
    g = np.random.default_rng(5)
    n = min(B, 32) if B == 32 else B - 3  # a short tile at the end
    rows = g.choice(150, n, replace=False).astype(np.int32)
    eps = g.normal(size=(n, K)).astype(np.float32)
    loss, grads, (mu, s) = vae64(w, dc[rows], eps, D, K, True)
    got = e.grad_step(rows, eps)[0]
    assert abs(got - loss) <= 1e-4 * abs(loss)
    for i, (a, b) in enumerate(zip(e.get_grads(), grads)):
        assert np.abs(a - b).max() <= 1e-4 * max(np.abs(b).max(), 1e-30), i
    m, lv, _ = e.encode(rows, eps)
    assert np.abs(m - mu).max() <= 1e-4 * np.abs(mu).max() and np.abs(lv - s).max() <= 1e-4 * np.abs(s).max()
    z = g.normal(size=(40, K)).astype(np.float32)
    it = iter([np.asarray(t, np.float64) for t in w[2 * D + 4:]])
    h = z.astype(np.float64) @ next(it) + next(it)
    for _ in range(D - 1):
        a = h @ next(it) + next(it)
        h = np.where(a > 0, a, np.expm1(np.minimum(a, 0))) + h
    p = 1 / (1 + np.exp(-(h @ next(it) + next(it))))
    assert np.abs(e.decode(z) - p).max() <= 1e-5
    # back to plain layers: the plain engine's results, bit for bit
    e.set_residual(False)
    f = new()
    assert e.train_step(rows, eps) == f.train_step(rows, eps)
    assert all(np.array_equal(a, b) for a, b in zip(e.get_weights(), f.get_weights()))
    e.close(), f.close()


def keras_update(w, m, v, g, t, lr, scale):
    out = []
    for a, b, c, d in zip(w, m, v, g):
        d = d.astype(np.float64) * scale
        b = b + (d - b) * 0.1
        c = c + (d * d - c) * 0.001
        out.append((a - lr * np.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t) * b / (np.sqrt(c) + 1e-7), b, c))
    return [list(x) for x in zip(*out)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("L,W,D,K,B", CASES)
def test_clipped_steps_against_64_bits(L, W, D, K, B, residual):
    """Each clipped step against the formula on the engine's own dumped gradients (held to 64 bits elsewhere)."""
    lr = 1e-3
    new, dc, w = make(L, W, D, K, B, lr=lr)
    e, probe = new(), new()
    for x in (e, probe):
        x.set_residual(residual)
    g = np.random.default_rng(7)
    m = [np.zeros_like(x, dtype=np.float64) for x in w]
    v = [np.zeros_like(x, dtype=np.float64) for x in w]
    for t, share in ((1, 0.3), (2, 2.0), (3, 0.05)):  # clipped, not clipped, clipped hard
        n = B if t != 2 else max(1, B - 7)
        rows = g.choice(150, n, replace=False).astype(np.int32)
        eps = g.normal(size=(n, K)).astype(np.float32)
        old = [x.astype(np.float64) for x in e.get_weights()]
        probe.set_weights(e.get_weights())
        loss = probe.grad_step(rows, eps)
        grads = probe.get_grads()
        norm = np.sqrt(sum((x.astype(np.float64) ** 2).sum() for x in grads))
        e.set_clip_norm(norm * share)
        assert e.train_step(rows, eps) == pytest.approx(loss, rel=1e-5)
        assert abs(e.grad_norm - norm) <= 2e-5 * norm
        new_w, m, v = keras_update(old, m, v, grads, t, lr, min(1.0, share))
        for i, (a, b, c) in enumerate(zip(e.get_weights(), new_w, old)):
            # the step is at most a few lr; where a gradient is rounding noise its sign is too: 2 % of the steps' norm
            assert np.linalg.norm(a - b) <= 2e-2 * np.linalg.norm(b - c) + 1e-6 * np.linalg.norm(b), (t, i)
        for which, mine in ((0, m), (1, v)):
            for i, (a, b) in enumerate(zip(e.get_moments(which), mine)):
                assert np.abs(a - b).max() <= 1e-4 * max(np.abs(b).max(), 1e-30), (t, which, i)
        m = [x.astype(np.float64) for x in e.get_moments(0)]
        v = [x.astype(np.float64) for x in e.get_moments(1)]
    e.close(), probe.close()


@pytest.mark.parametrize("L,W,D,K,B", CASES)
def test_an_epoch_with_clipping_equals_its_steps(L, W, D, K, B):
    new, dc, w = make(L, W, D, K, B)
    a, b = new(), new()
    g = np.random.default_rng(9)
    perm, val = g.permutation(110).astype(np.int32), np.arange(110, 150, dtype=np.int32)
    for e in (a, b):
        e.set_clip_norm(5.0)
    la, va = a.train_epoch(perm, val)
    losses = [b.train_step(perm[i:i + B])[0] for i in range(0, 110, B)]
    assert la == pytest.approx(float(np.mean(losses)), rel=1e-5)
    assert np.isfinite(va)
    for x, y in zip(a.get_weights(), b.get_weights()):
        assert np.array_equal(x, y)
    assert a.grad_norm == b.grad_norm
    # off again: the plain step's launches
    a.set_clip_norm(None)
    c = new()
    c.set_weights(a.get_weights())
    with pytest.raises(RuntimeError, match="no train step"):
        a.grad_norm
    rows, eps = perm[:16], np.zeros((16, K), np.float32)
    assert a.eval_step(rows, eps) == c.eval_step(rows, eps)
    for e in (a, b, c):
        e.close()


def test_a_bound_never_reached_leaves_the_trajectory():
    new, dc, w = make(1000, 128, 3, 2, 32, lr=1e-4)
    a, b = new(), new()
    a.set_clip_norm(1e30)
    g = np.random.default_rng(1)
    for _ in range(5):
        rows, eps = g.choice(150, 32, replace=False).astype(np.int32), g.normal(size=(32, 2)).astype(np.float32)
        assert a.train_step(rows, eps)[0] == pytest.approx(b.train_step(rows, eps)[0], rel=1e-5)
    for x, y in zip(a.get_moments(0), b.get_moments(0)):
        assert np.abs(x - y).max() <= 1e-4 * np.abs(y).max()
    a.close(), b.close()


def test_residual_layers_in_the_staged_step():
    """The calls that sharding cuts a step into, on one rank: the same gradients as the whole step."""
    new, dc, w = make(900, 128, 4, 2, 32)
    e = new()
    e.set_residual()
    rows, eps = np.arange(20, dtype=np.int32), np.random.default_rng(2).normal(size=(20, 2)).astype(np.float32)
    loss = e.grad_step(rows, eps)
    grads = e.get_grads()
    e.stage_a(rows, eps, engine.MODE_GRAD)
    e.stage_b(engine.MODE_GRAD)
    assert e.stage_c(engine.MODE_GRAD) == loss
    assert all(np.array_equal(a, b) for a, b in zip(e.get_grads(), grads))
    e.stage_a(rows, eps, engine.MODE_ENCODE)
    assert all(np.array_equal(a, b) for a, b in zip(e.stage_encode(20), e.encode(rows, eps)))
    e.close()


def test_refusals():
    new, _, _ = make(300, 32, 2, 2, 32)
    e = new()
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="clip_norm"):
            e.set_clip_norm(bad)
    e.set_clip_norm(1.0)
    rows = np.arange(8, dtype=np.int32)
    with pytest.raises(RuntimeError, match="clipping"):
        e.train_step_noalloc(rows)
    e.stage_a(rows, None, engine.MODE_TRAIN)
    with pytest.raises(RuntimeError, match="clip"):
        e.stage_b(engine.MODE_TRAIN)
    e.close()
    s = engine.Engine(n_snps=320, width=32, depth=2, n_snps_global=640, rank=0, world=2)
    with pytest.raises(RuntimeError, match="shard"):
        s.set_clip_norm(1.0)
    s.close()


def test_command_line(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    vcf = os.path.join(root, "tests", "golden", "pabu_test_genotypes.vcf.gz")
    out = str(tmp_path / "run")
    p = subprocess.run([sys.executable, os.path.join(root, "popvae.py"), "--infile", vcf, "--out", out, "--seed", "1", "--max_epochs", "8",
                        "--depth", "4", "--clip_norm", "20", "--residual"], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0, p.stderr[-2000:]
    import pandas as pd
    h = pd.read_csv(out + "_history.txt", sep="\t")
    assert len(h) == 8 and np.isfinite(h["loss"]).all() and np.isfinite(h["val_loss"]).all()
    p = subprocess.run([sys.executable, os.path.join(root, "popvae.py"), "--infile", vcf, "--out", out, "--clip_norm", "-1"],
                       capture_output=True, text=True, timeout=100)
    assert p.returncode != 0 and "clip_norm" in p.stderr


def test_weights_of_a_residual_model_on_the_command_line(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    vcf = os.path.join(root, "tests", "golden", "pabu_test_genotypes.vcf.gz")
    out = str(tmp_path / "run")

    def run(*more):
        return subprocess.run([sys.executable, os.path.join(root, "popvae.py"), "--infile", vcf, "--out", out, "--seed", "1", "--max_epochs", "2",
                               "--depth", "3", *more], capture_output=True, text=True, timeout=100)

    p = run("--residual", "--save_weights")
    assert p.returncode == 0, p.stderr[-2000:]
    p = run("--init_weights", out + "_weights.hdf5")
    assert p.returncode != 0 and "residual" in p.stderr
    p = run("--init_weights", out + "_weights.hdf5", "--residual")
    assert p.returncode == 0, p.stderr[-2000:]


def test_a_bound_below_float32_is_refused_not_taken_for_off():
    new, _, _ = make(300, 32, 2, 2, 32)
    e = new()
    with pytest.raises(RuntimeError, match="clip_norm"):
        e.set_clip_norm(1e-50)
    e.set_clip_norm(1e-40)  # a subnormal bound is one
    e.train_step(np.arange(8, dtype=np.int32))
    assert e.grad_norm > 0
    e.close()


def test_residual_layers_in_the_step_that_allocates_nothing():
    new, dc, w = make(900, 128, 4, 2, 32)
    a, b = new(), new()
    for e in (a, b):
        e.set_residual()
    g = np.random.default_rng(3)
    for n in (32, 5):
        rows, eps = g.choice(150, n, replace=False).astype(np.int32), g.normal(size=(n, 2)).astype(np.float32)
        assert a.train_step(rows, eps) == b.train_step_noalloc(rows, eps)
    assert all(np.array_equal(x, y) for x, y in zip(a.get_weights(), b.get_weights()))
    a.close(), b.close()
