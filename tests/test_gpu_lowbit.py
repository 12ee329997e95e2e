"""GPU tests of the 4-bit dense layers and 8-bit checkpoints against the 64-bit NumPy oracle.

Tolerance of a product: every piece product is exact in float32, so only the accumulation of at most 3 L + 8 terms and the
last rounding to the output's type count: |err| <= (3 L + 8) 2^-23 sum|a b| + (eps / 2 + 2^-23) |y|, L the length of the sum,
2^-23 twice the rounding of an addition (a matrix instruction may round a partial sum once more)."""
import numpy as np
import pytest
import torch

from gp_vae_amd import GpvaeError, ops
from oracle import lowbit_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def normal(rng, shape, dt, scale=1.0):
    return torch.tensor(rng.standard_normal(shape) * scale, dtype=F32, device=DEV).to(dt)


def close(got, want, absum, L, dt):
    eps = torch.finfo(dt).eps
    tiny = torch.finfo(dt).smallest_normal * eps  # below the smallest normal the step is fixed
    tol = (3 * L + 8) * 2.0 ** -23 * absum + (eps / 2 + 2.0 ** -23) * np.abs(want) + tiny
    err = np.abs(np64(got) - want)
    bad = ~(err <= tol)
    assert not bad.any(), "worst %g of its tolerance at %s" % (np.nanmax(err / tol), np.argwhere(bad)[:3].tolist())


def w4_np(w4):
    return orc.load_w4(w4.codes.cpu().numpy(), w4.exps.cpu().numpy(), w4.K, w4.N)


def q8_np(q):
    return orc.load_q8(q.codes.cpu().numpy(), q.exps.cpu().numpy(), q.M, q.K, q.relu)


def strided(t, pad_rows=0, lead=3, shift=1):
    """The same matrix inside a larger buffer: other leading dimension, unaligned base."""
    M, K = t.shape
    buf = torch.full((M + 1, K + lead + shift), 7.0, dtype=t.dtype, device=t.device)
    v = buf[:M, shift:shift + K]
    v.copy_(t)
    return buf, v


# ---- formats ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (32, 32), (50, 300), (33, 65), (7, 129), (100, 31)])
def test_quant_w4_is_the_formats_definition(K, N, dt):
    rng = np.random.default_rng(K * 1000 + N)
    W = normal(rng, (K, N), dt) * torch.tensor(10.0 ** rng.integers(-3, 3, (K, 1)), dtype=dt, device=DEV)
    _, V = strided(W)
    for M in (W, V):
        w4 = ops.quant_w4(M)
        c, e = orc.quant_w4(np64(W))
        assert np.array_equal(w4.codes.cpu().numpy().view(np.uint32), c) and np.array_equal(w4.exps.cpu().numpy(), e)
    for out in (F32, BF16):
        assert np.array_equal(np64(ops.load_w4(w4, out)), orc.load_w4(c, e, K, N))


def test_quant_w4_special_values():
    W = torch.zeros((40, 48), device=DEV)
    W[0, 0], W[0, 9], W[0, 17], W[0, 25] = float("inf"), float("nan"), 3.4e38, 1e-45
    W[8, :7] = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0])   # ties, with the tile's 6 below
    W[9, 0] = 6.0
    W[16, :8] = torch.tensor([1e-38, -2e-38, 3e-39, -1e-45, 0.0, -0.0, 1.2e-38, 5e-39])
    w4 = ops.quant_w4(W)
    c, e = orc.quant_w4(np64(W))
    assert np.array_equal(w4.codes.cpu().numpy().view(np.uint32), c) and np.array_equal(w4.exps.cpu().numpy(), e)
    got = np64(ops.load_w4(w4))
    assert np.isnan(got[:8, :16]).all() and np.isfinite(got[:8, 16:]).all() and np.isfinite(got[8:]).all()
    assert np.array_equal(got, orc.load_w4(c, e, 40, 48), equal_nan=True)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (8, 8), (8, 32), (100, 35), (13, 129), (257, 64), (3, 1000)])
@pytest.mark.parametrize("relu", [False, True])
def test_store_q8_is_the_formats_definition(M, K, relu, dt):
    rng = np.random.default_rng(M * 1000 + K)
    X = normal(rng, (M, K), dt) * torch.tensor(10.0 ** rng.integers(-3, 3, (1, K)), dtype=dt, device=DEV)
    Yw, c, e = orc.store_q8(np64(X), relu)
    buf, V = strided(X)
    for src in (X, V):
        if relu:
            Y, q = ops.store_q8(src, relu=True)
            assert np.array_equal(np64(Y), Yw)
        else:
            q = ops.store_q8(src)
        assert np.array_equal(q.codes.cpu().numpy(), c) and np.array_equal(q.exps.cpu().numpy(), e)
    assert np.array_equal(np64(ops.load_q8(q)), orc.load_q8(c, e, M, K, relu))
    assert np.array_equal(np64(ops.load_q8(q, BF16)), orc.load_q8(c, e, M, K, relu))
    if relu:  # in place, inside a larger buffer whose rest stays as it was
        Y, q = ops.store_q8(V, relu=True, out=V)
        assert Y is V and np.array_equal(np64(V), Yw) and np.array_equal(q.codes.cpu().numpy(), c)
        rest = buf.clone()
        rest[:M, 1:1 + K] = 7.0
        assert (rest == 7.0).all()


@pytest.mark.parametrize("relu", [False, True])
def test_store_q8_special_values(relu):
    X = torch.zeros((16, 64), device=DEV)
    X[0, 0], X[1, 1], X[0, 2], X[2, 9], X[0, 17], X[0, 25] = float("inf"), -1.0, 2.0, float("nan"), 3.4e38, 1e-45
    X[3, 10], X[4, 33] = -float("inf"), -float("inf")
    X[8, :8] = torch.tensor([1.0, 1e-6, -1e-6, 254.5 / 255, .5 / 255, 1.5 / 255, 2.5 / 255, 1e-45])
    Yw, c, e = orc.store_q8(np64(X), relu)
    q = ops.store_q8(X, relu=relu)
    if relu:
        Y, q = q
        assert np.array_equal(np64(Y), Yw, equal_nan=True)
        mask = q.codes.cpu().numpy().transpose(0, 2, 1).reshape(16, 64) != 0
        assert np.array_equal(mask, ~(np64(X) <= 0))
    assert np.array_equal(q.codes.cpu().numpy(), c) and np.array_equal(q.exps.cpu().numpy(), e)
    assert np.array_equal(np64(ops.load_q8(q)), orc.load_q8(c, e, 16, 64, relu), equal_nan=True)


# ---- products ---------------------------------------------------------------------------------------------------------
SHAPES = [(1, 50, 4096), (1, 1, 1), (2, 35, 300), (3, 300, 17), (16, 64, 128), (17, 1024, 65), (33, 31, 1000), (64, 100, 96),
          (65, 700, 33), (100, 33, 625), (130, 257, 260), (256, 96, 129), (300, 513, 1030),
          (22, 65, 97), (43, 130, 31), (350, 70, 99), (400, 129, 260), (1030, 65, 33), (515, 400, 640)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_dense_w4(M, K, N, dt):
    rng = np.random.default_rng(M + 10 * K + 100 * N)
    w4 = ops.quant_w4(normal(rng, (K, N), F32, K ** -0.5))
    X, b = normal(rng, (M, K), dt), normal(rng, (N,), dt)
    Wd, Xd, bd = w4_np(w4), np64(X), np64(b)
    S = np.abs(Xd) @ np.abs(Wd) + np.abs(bd)
    close(ops.dense_w4(X, w4), Xd @ Wd, S, K, dt)
    Y = ops.dense_w4(X, w4, b, relu=True)
    close(Y, orc.dense(Xd, Wd, bd, True), S, K, dt)
    assert torch.equal(Y, ops.dense_w4(X, w4, b, relu=True))  # same inputs, same bits
    buf, Xs = strided(X)
    obuf = torch.full((M + 2, N + 5), 7.0, dtype=dt, device=DEV)
    out = obuf[1:1 + M, 3:3 + N]
    assert ops.dense_w4(Xs, w4, b, relu=True, out=out) is out and torch.equal(out, Y)
    obuf[1:1 + M, 3:3 + N] = 7.0
    assert (obuf == 7.0).all()                                # nothing beside the output was written


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_dense_vjp_w4(M, K, N, dt):
    rng = np.random.default_rng(1 + M + 10 * K + 100 * N)
    w4 = ops.quant_w4(normal(rng, (K, N), F32, K ** -0.5))
    dY, A = normal(rng, (M, N), dt), normal(rng, (M, K), dt)
    _, q = ops.store_q8(A, relu=True)
    Wd, dYd = w4_np(w4), np64(dY)
    S = np.abs(dYd) @ np.abs(Wd).T
    close(ops.dense_vjp_w4(dY, w4), dYd @ Wd.T, S, N, dt)
    dX = ops.dense_vjp_w4(dY, w4, q)
    close(dX, orc.dense_vjp(dYd, Wd, np64(A) > 0), S, N, dt)
    assert (dX[A <= 0] == 0).all() and torch.equal(dX, ops.dense_vjp_w4(dY, w4, q))
    _, dYs = strided(dY)
    obuf = torch.full((M + 2, K + 5), 7.0, dtype=dt, device=DEV)
    out = obuf[1:1 + M, 3:3 + K]
    assert ops.dense_vjp_w4(dYs, w4, q, out=out) is out and torch.equal(out, dX)
    obuf[1:1 + M, 3:3 + K] = 7.0
    assert (obuf == 7.0).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("M,K,N", SHAPES + [(0, 5, 7), (1000, 50, 64), (2049, 33, 40)])
def test_dense_grads_q8(M, K, N, relu, dt):
    rng = np.random.default_rng(2 + M + 10 * K + 100 * N)
    A, dY = normal(rng, (M, K), dt), normal(rng, (M, N), dt)
    q = ops.store_q8(A, relu=relu)
    q = q[1] if relu else q
    Xd, dYd = q8_np(q), np64(dY)
    dW, db = ops.dense_grads_q8(q, dY)
    assert dW.dtype == F32 and db.dtype == F32
    want = orc.dense_grads(Xd, dYd)
    close(dW, want[0], np.abs(Xd).T @ np.abs(dYd), M, F32)
    close(db, want[1], np.abs(dYd).sum(0), M, F32)
    again = ops.dense_grads_q8(q, dY)
    assert torch.equal(again[0], dW) and torch.equal(again[1], db)
    if M:
        _, dYs = strided(dY)
        obuf = torch.full((K + 2, N + 5), 7.0, device=DEV)
        out = obuf[1:1 + K, 3:3 + N]
        ops.dense_grads_q8(q, dYs, out=(out, None))
        assert torch.equal(out, dW)
        obuf[1:1 + K, 3:3 + N] = 7.0
        assert (obuf == 7.0).all()


def test_gradients_agree_with_differences():
    """d/dX and d/db of sum(C * dense) by central differences in 64 bits of the oracle's layer at the stored weights."""
    rng = np.random.default_rng(9)
    M, K, N = 5, 41, 37
    w4 = ops.quant_w4(normal(rng, (K, N), F32))
    X, Cc = normal(rng, (M, K), F32), normal(rng, (M, N), F32)
    Wd, Xd, Cd = w4_np(w4), np64(X), np64(Cc)
    f = lambda x: float((orc.dense(x, Wd, relu=True) * Cd).sum())
    Y = ops.dense_w4(X, w4, relu=True)
    dX = np64(ops.dense_vjp_w4(Cc * (Y > 0), w4))
    for m, k in [(0, 0), (2, 17), (4, 40)]:
        h = 1e-6
        P, Q = Xd.copy(), Xd.copy()
        P[m, k] += h
        Q[m, k] -= h
        assert abs((f(P) - f(Q)) / (2 * h) - dX[m, k]) < 1e-4 * np.abs(dX).max()


@pytest.mark.parametrize("M", [1, 20, 200])
def test_infinities_and_nan_reach_what_they_touch_and_nothing_else(M):
    rng = np.random.default_rng(4)
    K, N = 70, 90
    W = normal(rng, (K, N), F32)
    w4 = ops.quant_w4(W)
    Wd = w4_np(w4)
    X = normal(rng, (M, K), F32)
    X[0, 3] = float("inf")
    if M > 1:
        X[1, 69] = float("nan")
        X[M - 1, 0] = 3.4e38
    Y, want = np64(ops.dense_w4(X, w4)), np64(X) @ Wd
    with np.errstate(invalid="ignore", over="ignore"):
        want32 = want.astype(np.float32).astype(np.float64)
    rows = [r for r in range(M) if r not in (0, 1, M - 1)]
    assert np.isfinite(Y[rows]).all()
    nz = Wd[3] != 0
    assert np.isnan(Y[0, ~nz]).all() and np.array_equal(Y[0, nz], np.sign(Wd[3, nz]) * np.inf)  # inf * 0 = NaN
    if M > 1:
        assert np.isnan(Y[1]).all()
        big = np.abs(want32[M - 1]) < 3e38
        assert np.isfinite(Y[M - 1][big]).all()
    dY = normal(rng, (M, N), F32)
    dY[0, 89] = -float("inf")
    dX = np64(ops.dense_vjp_w4(dY, w4))
    nz = Wd[:, 89] != 0
    assert np.isfinite(dX[1:]).all() and np.array_equal(dX[0, nz], -np.sign(Wd[nz, 89]) * np.inf) and np.isnan(dX[0, ~nz]).all()
    # a weight tile that is not finite: its rows' and columns' outputs are NaN, the others are not
    W[9, 17] = float("nan")
    bad = ops.quant_w4(W)
    Y = ops.dense_w4(torch.ones((M, K), device=DEV), bad)
    assert torch.isnan(Y[:, 16:24]).all() and torch.isfinite(Y[:, :16]).all() and torch.isfinite(Y[:, 24:]).all()
    dX = ops.dense_vjp_w4(torch.ones((M, N), device=DEV), bad)
    assert torch.isnan(dX[:, 8:16]).all() and torch.isfinite(dX[:, :8]).all() and torch.isfinite(dX[:, 16:]).all()
    # the gradient of a checkpoint with a NaN in it
    A = normal(rng, (M, K), F32)
    A[0, 5] = float("nan")
    dW, db = ops.dense_grads_q8(ops.store_q8(A), torch.ones((M, N), device=DEV))
    assert torch.isnan(dW[:8]).all() and torch.isfinite(dW[8:]).all() and torch.isfinite(db).all()


def test_float16_and_float32_extremes_keep_their_accuracy():
    """Smallest and largest magnitudes of the types: every piece of the split carries its share."""
    rng = np.random.default_rng(8)
    w4 = ops.quant_w4(normal(rng, (64, 40), F32))
    Wd = w4_np(w4)
    for dt, lo, hi in ((F16, -24, 14), (F32, -100, 100), (BF16, -100, 100)):
        X = (normal(rng, (6, 64), F32) * torch.tensor(2.0 ** rng.integers(lo, hi, (6, 1)), dtype=F32, device=DEV)).to(dt)
        Xd = np64(X)
        want = Xd @ Wd
        top = torch.finfo(dt).max
        ok = np.abs(want) < 0.9 * top
        got, S = ops.dense_w4(X, w4), np.abs(Xd) @ np.abs(Wd)
        close(torch.where(torch.tensor(ok, device=DEV), got, torch.zeros_like(got)), np.where(ok, want, 0), S, 64, dt)


def test_other_layouts_and_empty_calls():
    rng = np.random.default_rng(6)
    K, N, M = 40, 50, 12
    w4 = ops.quant_w4(normal(rng, (K, N), F32))
    X = normal(rng, (M, K), F32)
    assert torch.equal(ops.dense_w4(X.t().contiguous().t(), w4), ops.dense_w4(X, w4))            # column-major rows
    one = normal(rng, (1, K), F32)
    assert torch.equal(ops.dense_w4(one.expand(M, K), w4), ops.dense_w4(one.repeat(M, 1), w4))  # a broadcast row
    g = torch.ones((), device=DEV).expand(M, N)
    assert torch.equal(ops.dense_vjp_w4(g, w4), ops.dense_vjp_w4(g.contiguous(), w4))
    q = ops.store_q8(X)
    assert torch.equal(ops.dense_grads_q8(q, g)[0], ops.dense_grads_q8(q, g.contiguous())[0])
    k1 = ops.quant_w4(normal(rng, (1, N), F32))
    col = normal(rng, (M, 3), F32)[:, 1:2]
    close(ops.dense_w4(col, k1), np64(col) @ w4_np(k1), np.abs(np64(col)) @ np.abs(w4_np(k1)), 1, F32)
    assert ops.dense_w4(X[:0], w4).shape == (0, N) and ops.dense_vjp_w4(torch.empty((0, N), device=DEV), w4).shape == (0, K)
    q0 = ops.store_q8(X[:0])
    dW, db = ops.dense_grads_q8(q0, torch.empty((0, N), device=DEV))
    assert ops.load_q8(q0).shape == (0, K) and (dW == 0).all() and (db == 0).all()


def test_refusals():
    w4 = ops.quant_w4(torch.ones((40, 50), device=DEV))
    X = torch.ones((3, 40), device=DEV)
    Y, q = ops.store_q8(X, relu=True)
    bad = [lambda: ops.dense_w4(X.double(), w4), lambda: ops.dense_w4(X[:, :39], w4), lambda: ops.dense_w4(X[0], w4),
           lambda: ops.dense_w4(X, w4, torch.ones(49, device=DEV)), lambda: ops.dense_w4(X, w4, torch.ones(50, device=DEV).half()),
           lambda: ops.dense_w4(X, w4, out=torch.empty((3, 49), device=DEV)), lambda: ops.dense_w4(X, w4, out=torch.empty((50, 3), device=DEV).t()),
           lambda: ops.dense_w4(X, w4, torch.ones(50)), lambda: ops.dense_vjp_w4(X, w4),
           lambda: ops.dense_vjp_w4(torch.ones((3, 50), device=DEV), w4, ops.store_q8(X)),
           lambda: ops.dense_vjp_w4(torch.ones((4, 50), device=DEV), w4, q), lambda: ops.quant_w4(torch.ones((0, 3), device=DEV)),
           lambda: ops.store_q8(X, out=X), lambda: ops.store_q8(X.long()), lambda: ops.dense_grads_q8(q, torch.ones((4, 5), device=DEV)),
           lambda: ops.dense_grads_q8(q, torch.ones((3, 0), device=DEV)),
           lambda: ops.dense_grads_q8(q, X, out=(torch.empty((40, 39), device=DEV), None))]
    sq = ops.quant_w4(torch.ones((40, 40), device=DEV))
    bad.append(lambda: ops.dense_w4(X, sq, out=X))
    for i, call in enumerate(bad):
        with pytest.raises(GpvaeError):
            call()
            pytest.fail("call %d was not refused" % i)


def test_offsets_past_32_bits():
    """More than 2^32 bytes of codes: rows and columns at both ends."""
    K, N = 65600, 131104
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    kb, np_ = K // 32, N
    codes = torch.randint(-2 ** 31, 2 ** 31 - 1, (kb, np_, 4), dtype=torch.int32, device=DEV, generator=g)
    exps = torch.randint(120, 125, (kb, np_ // 8, 4), dtype=torch.uint8, device=DEV, generator=g)
    assert codes.numel() * 4 > 2 ** 32
    w4 = ops.W4(codes, exps, K, N)
    X = torch.randn((2, K), device=DEV, generator=g)
    Y = ops.dense_w4(X, w4)
    cut = ops.W4(codes[:, -64:].contiguous(), exps[:, -8:].contiguous(), K, 64)  # the last 64 columns
    Wd = w4_np(cut)
    close(Y[:, -64:], np64(X) @ Wd, np.abs(np64(X)) @ np.abs(Wd), K, F32)
    dY = torch.randn((2, N), device=DEV, generator=g)
    dX = ops.dense_vjp_w4(dY, w4)
    cut = ops.W4(codes[-2:].contiguous(), exps[-2:].contiguous(), 64, N)         # the last 64 rows
    Wd = w4_np(cut)
    close(dX[:, -64:], np64(dY) @ Wd.T, np.abs(np64(dY)) @ np.abs(Wd).T, N, F32)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(5, 256, 70), (20, 384, 200), (130, 128, 66), (300, 256, 258)])
def test_alignment_changes_no_bit(M, K, N, dt):
    """Whatever loads an operand's strides and alignment allow, the same sums in the same order."""
    rng = np.random.default_rng(M + K + N)
    w4, b = ops.quant_w4(normal(rng, (K, N), F32)), normal(rng, (N,), dt)
    X, dY = normal(rng, (M, K), dt), normal(rng, (M, N), dt)
    Y, q = ops.store_q8(X, relu=True)
    Yd, dX, (dW, db) = ops.dense_w4(X, w4, b), ops.dense_vjp_w4(dY, w4, q), ops.dense_grads_q8(q, dY)
    for lead, shift in [(0, 0), (3, 1), (2, 1), (8, 0), (6, 2), (5, 8), (64, 64)]:
        vx, vy = strided(X, lead=lead, shift=shift)[1], strided(dY, lead=lead, shift=shift)[1]
        Y2, q2 = ops.store_q8(vx, relu=True)
        assert torch.equal(Y2, Y) and torch.equal(q2.codes, q.codes) and torch.equal(q2.exps, q.exps)
        buf, out = strided(torch.zeros_like(Yd), lead=lead, shift=shift)
        assert torch.equal(ops.dense_w4(vx, w4, b, out=out), Yd) and torch.equal(ops.dense_vjp_w4(vy, w4, q), dX)
        assert (buf[M] == 7).all() and (buf[:, :shift] == 7).all() and (buf[:M, shift + N:] == 7).all()
        wbuf, wout = strided(torch.zeros_like(dW), lead=lead, shift=shift)
        got = ops.dense_grads_q8(q, vy, out=(wout, torch.empty_like(db)))
        assert torch.equal(got[0], dW) and torch.equal(got[1], db)
        assert (wbuf[K] == 7).all() and (wbuf[:, :shift] == 7).all() and (wbuf[:K, shift + N:] == 7).all()


def test_gradients_are_not_written_over_their_input():
    q = ops.store_q8(torch.ones((6, 6), device=DEV))
    dY = torch.ones((6, 6), device=DEV)
    for out in [(dY, None), (torch.empty((6, 6), device=DEV), dY[0])]:
        with pytest.raises(GpvaeError):
            ops.dense_grads_q8(q, dY, out=out)


def test_operands_past_32_bits():
    """Operands, their pieces, codes and outputs of more than 2^32 bytes: rows and columns at both ends."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    M, K, N = 66000, 65600, 40
    X = torch.randn((M, K), device=DEV, generator=g, dtype=BF16)
    q = ops.store_q8(X)
    assert q.codes.numel() > 2 ** 32
    for rows in (slice(0, 16), slice(M - 16, M)):
        mb = slice(rows.start // 8, rows.stop // 8)
        cut = ops.store_q8(X[rows].contiguous())
        assert torch.equal(q.codes[mb], cut.codes) and torch.equal(q.exps[mb], cut.exps)
    dY = torch.randn((M, N), device=DEV, generator=g, dtype=BF16)
    dW, db = ops.dense_grads_q8(q, dY)
    for cols in (slice(0, 64), slice(K - 64, K)):
        t = ops.load_q8(ops.Q8(q.codes[:, cols].contiguous(), q.exps[:, cols.start // 8:cols.stop // 8].contiguous(), M, 64)).double()
        want, S = t.t() @ dY.double(), t.abs().t() @ dY.double().abs()
        close(dW[cols], want.cpu().numpy(), S.cpu().numpy(), M, F32)
    del q, dW
    w4 = ops.quant_w4(torch.randn((K, N), device=DEV, generator=g))
    Wd = ops.load_w4(w4).double()
    rows = torch.cat([torch.arange(8), torch.arange(M - 8, M)]).to(DEV)
    got = ops.dense_w4(X, w4)[rows]                                    # many rows, read in place
    want, S = X[rows].double() @ Wd, X[rows].double().abs() @ Wd.abs()
    close(got, want.cpu().numpy(), S.cpu().numpy(), K, BF16)
    X = X[:24000].float()
    rows = torch.cat([torch.arange(8), torch.arange(24000 - 8, 24000)]).to(DEV)
    got = ops.dense_w4(X, w4)[rows]                                    # many rows, pieces of 9.4 GB
    want, S = X[rows].double() @ Wd, X[rows].double().abs() @ Wd.abs()
    close(got, want.cpu().numpy(), S.cpu().numpy(), K, F32)
    wt = ops.quant_w4(Wd.t().contiguous().float())                     # [N, K]: its transposed product reduces over K
    got = ops.dense_vjp_w4(X, wt)[rows]
    Wt = ops.load_w4(wt).double()
    want, S = X[rows].double() @ Wt.t(), X[rows].double().abs() @ Wt.abs().t()
    close(got, want.cpu().numpy(), S.cpu().numpy(), K, F32)


@pytest.mark.parametrize("M", [3, 22])
def test_very_long_reductions(M):
    """Small integers: the sums are exact."""
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    K, N = 67200001, 8
    w4 = ops.quant_w4(torch.randint(0, 2, (K, N), device=DEV, generator=g).mul_(2).sub_(1).to(BF16))
    X = torch.randint(-1, 2, (M, K), device=DEV, generator=g, dtype=torch.int8).float()
    want = sum(X[:, k:k + 2 ** 22].double() @ ops.load_w4(ops.W4(w4.codes[k // 32:(k + 2 ** 22) // 32].contiguous(), w4.exps[k // 32:(k + 2 ** 22) // 32].contiguous(), min(2 ** 22, K - k), N)).double()
               for k in range(0, K, 2 ** 22))
    assert torch.equal(ops.dense_w4(X, w4).double(), want)


def test_gradients_of_rows_far_apart():
    buf = torch.zeros((2, 2 ** 26 + 64), dtype=BF16, device=DEV)
    buf[:, :5] = torch.arange(1, 11, device=DEV).reshape(2, 5)
    q = ops.store_q8(torch.ones((2, 3), device=DEV))
    with pytest.raises(GpvaeError):
        ops.dense_grads_q8(q, buf[:, :5])                      # more than 2^26 elements from row to row
    one = ops.store_q8(torch.ones((1, 3), device=DEV))
    dW, db = ops.dense_grads_q8(one, buf[:1, :5])              # a single row has no distance
    assert db.tolist() == [1, 2, 3, 4, 5] and dW.tolist() == [[1, 2, 3, 4, 5]] * 3
    dW, db = ops.dense_grads_q8(q, buf[:, :2 ** 26 - 1][:, -3:].contiguous())
    assert (dW == 0).all() and (db == 0).all()


# ---- streams and graphs -------------------------------------------------------------------------------------------------
def test_side_stream_and_replayed_graph():
    rng = np.random.default_rng(12)
    M, K, N = 24, 96, 200
    w4 = ops.quant_w4(normal(rng, (K, N), F32))
    Xs = [normal(rng, (M, K), F32) for _ in range(4)]
    dYs = [normal(rng, (M, N), F32) for _ in range(4)]
    b = normal(rng, (N,), F32)

    def step(X, dY):
        A, q = ops.store_q8(X, relu=True)
        Y = ops.dense_w4(A, w4, b, relu=True)
        return (Y, ops.dense_vjp_w4(dY, w4, q), *ops.dense_grads_q8(q, dY))

    want = [[t.clone() for t in step(X, dY)] for X, dY in zip(Xs, dYs)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(Xs[0], dYs[0])
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(got, want[0]))
    sx, sdy = Xs[0].clone(), dYs[0].clone()
    graphs = []
    for _ in range(2):  # two graphs of the same calls
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(sx, sdy)
        graphs.append((g, outs))
    for i in (1, 2, 3, 1, 0):
        sx.copy_(Xs[i])
        sdy.copy_(dYs[i])
        for g, outs in graphs:
            g.replay()
            step(Xs[(i + 1) % 4], dYs[(i + 1) % 4])  # the program's own eager work between replays
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs, want[i])), i


# ---- values at the edges of the types ---------------------------------------------------------------------------------
NAN_BITS = {F32: (torch.int32, [0x7f800001, 0x7f80ffff, 0x7fbfffff, -0x7fffff, -0x7f0001, 0x7fc00000]),
            BF16: (torch.int16, [0x7f81, 0x7fbf, -0x7f, 0x7fc0]), F16: (torch.int16, [0x7c01, 0x7dff, -0x3ff, 0x7e00])}


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M", [1, 20, 300])
def test_every_nan_stays_a_nan(M, dt):
    """Signalling ones too, whose set mantissa bits may all lie below the first bfloat16 piece."""
    rng = np.random.default_rng(M)
    K, N = 200, 150
    w4 = ops.quant_w4(normal(rng, (K, N), F32))
    X, dY = normal(rng, (M, K), dt), normal(rng, (M, N), dt)
    bits, patterns = NAN_BITS[dt]
    A, q = ops.store_q8(X, relu=True)
    for i, p in enumerate(patterns):
        for k in (0, 67, K - 1):
            V = X.clone()
            V.view(bits)[M - 1, k] = p
            for src in (V, strided(V)[1]):
                assert torch.isnan(ops.dense_w4(src, w4, relu=bool(i & 1))[M - 1]).all()
                assert torch.isfinite(ops.dense_w4(src, w4)[:M - 1]).all()
            assert torch.isnan(ops.load_q8(ops.store_q8(V))[M - 1, k]) and torch.isnan(ops.load_w4(ops.quant_w4(V))[M - 1, k])
        for n in (0, 33, N - 1):
            V = dY.clone()
            V.view(bits)[M - 1, n] = p
            for src in (V, strided(V)[1]):
                dX = ops.dense_vjp_w4(src, w4)
                assert torch.isnan(dX[M - 1]).all() and torch.isfinite(dX[:M - 1]).all()
                dX = ops.dense_vjp_w4(src, w4, q)                       # the mask selects: 0 where it is 0
                assert torch.isnan(dX[M - 1][A[M - 1] > 0]).all() and (dX[A <= 0] == 0).all()
                dW, db = ops.dense_grads_q8(q, src)
                rest = [j for j in range(N) if j != n]
                assert torch.isnan(dW[:, n]).all() and torch.isnan(db[n])
                assert torch.isfinite(dW[:, rest]).all() and torch.isfinite(db[rest]).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("relu", [False, True])
def test_gradients_of_the_largest_checkpoints(relu, dt):
    """Tiles whose power of two is the format's largest, next to zeros: powers of two times them are exact."""
    M, K, N = 70, 40, 9
    X = torch.zeros((M, K), device=DEV)
    X[0, 0], X[1, 1], X[2, 2], X[3, 9], X[20, 17], X[69, 39] = 2e38, -2e38, 3.4e38, 1.7e38, 1.0, -3e38
    q = ops.store_q8(X, relu=relu)
    q = q[1] if relu else q
    assert int(q.exps.max()) == 127 + (120 if relu else 121)
    dY = torch.zeros((M, N), device=DEV, dtype=dt)
    for m in (0, 1, 2, 3, 20, 69):
        dY[m, m % N] = -2.0 ** -(m % 14 + 10)
    want, S = q8_np(q).T @ np64(dY), np.abs(q8_np(q)).T @ np.abs(np64(dY))
    dW, db = ops.dense_grads_q8(q, dY)
    close(dW, want, S, M, F32)
    close(db, np64(dY).sum(0), np.abs(np64(dY)).sum(0), M, F32)


def ends(M, *cuts):
    """Rows at both ends and on both sides of the cuts."""
    near = [torch.arange(max(0, c - 9), min(M, c + 9)) for c in (0, *cuts, M)]
    return torch.cat(near).unique().to(DEV)


def test_more_rows_than_a_launch_has_room_for():
    """2^24 rows of more than 512 reduction indices, a workgroup for each row's pieces: 2^32 threads."""
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    M, K, N = 2 ** 24 + 70, 520, 33
    X = torch.randn((2 ** 18 + 1, K), device=DEV, generator=g).to(BF16).repeat(65, 1)[:M]
    w4 = ops.quant_w4(torch.randn((K, N), device=DEV, generator=g))
    Y, rows, Wd = ops.dense_w4(X, w4), ends(M, 2 ** 20, 2 ** 23, 2 ** 24), ops.load_w4(w4).double()
    close(Y[rows], (X[rows].double() @ Wd).cpu().numpy(), (X[rows].double().abs() @ Wd.abs()).cpu().numpy(), K, BF16)


@pytest.mark.parametrize("dt", TYPES)
def test_rows_in_several_launches(dt):
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    M, K, N = 2 ** 20 + 100, 140, 24
    rand = lambda *s: torch.randn(s, device=DEV, generator=g)
    w4, wt = ops.quant_w4(rand(K, N)), ops.quant_w4(rand(N, K))  # reductions over 140 both ways
    X, b, rows = rand(M, K).to(dt), rand(N).to(dt), ends(M, 2 ** 19, 2 ** 20)
    A, q = ops.store_q8(rand(M, N).to(dt), relu=True)
    Wd, Wt, Xd = ops.load_w4(w4).double(), ops.load_w4(wt).double().t(), X[rows].double()
    obuf = torch.full((M + 2, N + 3), 7.0, dtype=dt, device=DEV)
    out = obuf[1:1 + M, 2:2 + N]
    ops.dense_w4(X, w4, b, relu=True, out=out)
    close(out[rows], torch.relu(Xd @ Wd + b.double()).cpu().numpy(), (Xd.abs() @ Wd.abs() + b.double().abs()).cpu().numpy(), K, dt)
    S = (Xd.abs() @ Wt.abs()).cpu().numpy()
    ops.dense_vjp_w4(X, wt, q, out=out)
    close(out[rows], ((Xd @ Wt) * (A[rows] > 0)).cpu().numpy(), S, K, dt)
    assert (out[A <= 0] == 0).all() and (out[A > 0] != 0).float().mean() > 0.99
    obuf[1:1 + M, 2:2 + N] = 7.0
    assert (obuf == 7.0).all()


# Reductions split over workgroups, whose parts a second launch adds and finishes, by few and by many rows
SPLIT = [(1, 32768, 130), (1, 9000, 33), (3, 8192, 200), (21, 5000, 97), (40, 9001, 65), (130, 9000, 260), (300, 6000, 130),
         (700, 4100, 300), (1024, 4096, 1024)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,L,O", SPLIT)
def test_split_reductions_in_both_directions(M, L, O, dt):
    g = torch.Generator(device=DEV)
    g.manual_seed(M + L + O)
    rand = lambda *s: torch.randn(s, device=DEV, generator=g)
    w4, wt = ops.quant_w4(rand(L, O) * L ** -0.5), ops.quant_w4(rand(O, L) * L ** -0.5)
    X, b = rand(M, L).to(dt), rand(O).to(dt)
    A, q = ops.store_q8(rand(M, O).to(dt), relu=True)
    lib, code = ops._lib.load_lowbit(), ops._LB_DT[dt]
    work = lib.gpvae_dense_w4_workspace_bytes(code, M, L, O), lib.gpvae_dense_vjp_w4_workspace_bytes(code, M, O, L)
    assert min(work) >= 2 * M * O * 4
    obuf = torch.full((M + 1, O + 3), 7.0, dtype=dt, device=DEV)
    out = obuf[:M, 2:2 + O]
    Wd, Wt, Xd, bd = ops.load_w4(w4).double(), ops.load_w4(wt).double().t(), X.double(), b.double()
    for bias, relu in ((None, False), (b, False), (b, True)):
        want, S = Xd @ Wd + (0 if bias is None else bd), Xd.abs() @ Wd.abs() + (0 if bias is None else bd.abs())
        torch.full((max(work) // 4,), float("nan"), device=DEV)  # whatever the workspace held before
        ops.dense_w4(X, w4, bias, relu=relu, out=out)
        close(out, (torch.relu(want) if relu else want).cpu().numpy(), S.cpu().numpy(), L, dt)
        assert torch.equal(out, ops.dense_w4(strided(X)[1], w4, bias, relu=relu))
    want, S = Xd @ Wt, Xd.abs() @ Wt.abs()
    for act in (None, q):
        torch.full((max(work) // 4,), float("nan"), device=DEV)
        ops.dense_vjp_w4(X, wt, act, out=out)
        close(out, (want if act is None else want * (A > 0)).cpu().numpy(), S.cpu().numpy(), L, dt)
        assert torch.equal(out, ops.dense_vjp_w4(strided(X)[1], wt, act))
    assert (out[A <= 0] == 0).all()
    X[M - 1, L - 1] = float("inf")  # the mask selects: what it hides is 0 whatever it is
    ops.dense_vjp_w4(X, wt, q, out=out)
    hit = (A[M - 1] > 0) & (ops.load_w4(wt)[:, L - 1] != 0)
    assert (out[A <= 0] == 0).all() and torch.isinf(out[M - 1][hit]).all() and torch.isfinite(out[:M - 1]).all()
    obuf[:M, 2:2 + O] = 7.0
    assert (obuf == 7.0).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", [(2000, 300, 200), (1111, 130, 257), (4096, 40, 1000)])
def test_gradients_whose_rows_are_split(M, K, N, dt):
    g = torch.Generator(device=DEV)
    g.manual_seed(M + K + N)
    dY = torch.randn((M, N), device=DEV, generator=g).to(dt)
    work = ops._lib.load_lowbit().gpvae_dense_grads_q8_workspace_bytes(ops._LB_DT[dt], M, K, N)
    assert work >= 2 * (K + 1) * N * 4
    for relu in (False, True):
        q = ops.store_q8(torch.randn((M, K), device=DEV, generator=g), relu=relu)
        q = q[1] if relu else q
        V, D = ops.load_q8(q).double(), dY.double()
        obuf = torch.full((K + 1, N + 3), 7.0, device=DEV)
        out = obuf[:K, 2:2 + N], torch.empty(N, device=DEV)
        torch.full((work // 4,), float("nan"), device=DEV)
        dW, db = ops.dense_grads_q8(q, dY, out=out)
        close(dW, (V.t() @ D).cpu().numpy(), (V.abs().t() @ D.abs()).cpu().numpy(), M, F32)
        close(db, D.sum(0).cpu().numpy(), D.abs().sum(0).cpu().numpy(), M, F32)
        assert torch.equal(dW, ops.dense_grads_q8(q, strided(dY)[1])[0])
        obuf[:K, 2:2 + N] = 7.0
        assert (obuf == 7.0).all()


def test_bfloat16_operands_past_32_bits_read_in_place():
    """Rows of whole steps of 128: the tiles read the operand itself, more than 2^32 bytes of it."""
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    M, L, O = 33000, 65664, 40
    X = torch.randn((M, L), device=DEV, generator=g, dtype=BF16)
    assert X.numel() * 2 > 2 ** 32
    w4, wt, rows = ops.quant_w4(torch.randn((L, O), device=DEV, generator=g)), ops.quant_w4(torch.randn((O, L), device=DEV, generator=g)), ends(M, 2 ** 15)
    Xd = X[rows].double()
    for got, W in ((ops.dense_w4(X, w4), ops.load_w4(w4).double()), (ops.dense_vjp_w4(X, wt), ops.load_w4(wt).double().t())):
        close(got[rows], (Xd @ W).cpu().numpy(), (Xd.abs() @ W.abs()).cpu().numpy(), L, BF16)
