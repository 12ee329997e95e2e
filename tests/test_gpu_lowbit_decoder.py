"""GPU tests of the decoder in 4 bits: its layers run together, and behind VAEInference.

Error bounds are carried through the layers in 64 bits: a dense layer adds (3 L + 8) 2^-23 sum|a b| + 2^-22 |y| of its own
(see test_gpu_lowbit) to |W|^T times its input's error; a ReLU and a mask do not enlarge an error."""
import math

import numpy as np
import pytest
import torch

from gp_vae_amd import GpvaeError, ops
from gp_vae_amd.inference import VAEInference
from oracle import lowbit_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -23
NAMES = ("V1", "c1", "V2", "c2", "V3", "c3")


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def params(rng, n, h0, h1, z):
    w = {"V1": (z, h1), "c1": (h1,), "V2": (h1, h0), "c2": (h0,), "V3": (h0, n), "c3": (n,)}
    return {k: rng.standard_normal(s) * (s[0] ** -0.5 if len(s) == 2 else 0.1) for k, s in w.items()}


def flat(p):
    return torch.tensor(np.concatenate([p[k].reshape(-1) for k in NAMES]), dtype=torch.float32, device=DEV)


def layer(X, eX, W, b):
    """(y, bound of its error) of a dense layer with input X +- eX."""
    S = np.abs(X) @ np.abs(W) + np.abs(b)
    y = X @ W + b
    own = (3 * W.shape[0] + 8) * U * (S + eX @ np.abs(W)) + 2 * U * np.abs(y)
    return y, eX @ np.abs(W) + own


def within(got, want, bound):
    err = np.abs(np64(got) - want)
    assert (err <= bound + 1e-30).all(), "worst %g of its bound" % np.max(err / (bound + 1e-30))


@pytest.mark.parametrize("dims", [(1, 300, 35, 30, 10), (7, 625, 50, 30, 15), (100, 1024, 64, 32, 16), (256, 333, 130, 70, 33), (5, 19, 3, 2, 1)])
def test_decoder_forward_backward_and_parameter_gradients(dims):
    C, n, h0, h1, z = dims
    rng = np.random.default_rng(sum(dims))
    dec = ops.quant_decoder_w4(flat(params(rng, n, h0, h1, z)), n, h0, h1, z)
    Z = torch.tensor(rng.standard_normal((C, z)), dtype=torch.float32, device=DEV)
    dF = torch.tensor(rng.standard_normal((C, n)), dtype=torch.float32, device=DEV)
    W = [orc.load_w4(w.codes.cpu().numpy(), w.exps.cpu().numpy(), w.K, w.N) for w in dec.layers]
    b = [np64(t) for t in dec.biases]
    F, acts = ops.decoder_fwd_w4(dec, Z, keep=True)
    assert torch.equal(F, ops.decoder_fwd_w4(dec, Z))
    y1, e1 = layer(np64(Z), 0 * np64(Z), W[0], b[0])
    y2, e2 = layer(np.maximum(y1, 0), e1, W[1], b[1])
    f, ef = layer(np.maximum(y2, 0), e2, W[2], b[2])
    within(F, f, ef)
    # masks: those of the activations wherever their sign is certain
    X = [orc.load_q8(a.codes.cpu().numpy(), a.exps.cpu().numpy(), a.M, a.K, a.relu) for a in acts]
    for y, e, x in ((y1, e1, X[1]), (y2, e2, X[2])):
        sure = np.abs(y) > e
        assert ((x > 0) == (y > 0))[sure].all()
    # backward: the checkpoints' masks and values are what it is to use
    dZ, g = ops.decoder_vjp_w4(dec, acts, dF, grads=True)
    assert torch.equal(dZ, ops.decoder_vjp_w4(dec, acts, dF))
    d, ed = np64(dF), np.zeros((C, n))
    want, bound = [], []
    for i in (2, 1, 0):
        dW, db = orc.dense_grads(X[i], d)
        S, Sb = np.abs(X[i]).T @ (np.abs(d) + ed), (np.abs(d) + ed).sum(0)
        want = [dW, db] + want
        bound = [np.abs(X[i]).T @ ed + (3 * C + 8) * U * S + 2 * U * np.abs(dW), ed.sum(0) + (3 * C + 8) * U * Sb + 2 * U * np.abs(db)] + bound
        d, ed = layer(d, ed, W[i].T, np.zeros(W[i].shape[0]))
        if i:
            d, ed = np.where(X[i] > 0, d, 0), np.where(X[i] > 0, ed, 0)
    within(dZ, d, ed)
    within(g, np.concatenate([a.reshape(-1) for a in want]), np.concatenate([a.reshape(-1) for a in bound]))


def test_gradients_against_differences_of_the_4_bit_decoder():
    rng = np.random.default_rng(3)
    C, n, h0, h1, z = 3, 40, 24, 17, 6
    dec = ops.quant_decoder_w4(flat(params(rng, n, h0, h1, z)), n, h0, h1, z)
    W = [orc.load_w4(w.codes.cpu().numpy(), w.exps.cpu().numpy(), w.K, w.N) for w in dec.layers]
    b = [np64(t) for t in dec.biases]
    Z, dF = rng.standard_normal((C, z)), rng.standard_normal((C, n))

    def loss(Zv, W, b):
        h = np.maximum(np.maximum(Zv @ W[0] + b[0], 0) @ W[1] + b[1], 0)
        return float(((h @ W[2] + b[2]) * dF).sum())

    Zt = torch.tensor(Z, dtype=torch.float32, device=DEV)
    Z = np64(Zt)
    F, acts = ops.decoder_fwd_w4(dec, Zt, keep=True)
    dFt = torch.tensor(dF, dtype=torch.float32, device=DEV)
    dF = np64(dFt)
    dZ, g = ops.decoder_vjp_w4(dec, acts, dFt, grads=True)
    dZ = np64(dZ)
    for c, j in ((0, 0), (1, 3), (2, 5)):
        E = np.zeros_like(Z)
        E[c, j] = 1e-6
        assert abs((loss(Z + E, W, b) - loss(Z - E, W, b)) / 2e-6 - dZ[c, j]) < 1e-4 * np.abs(dZ).max()
    # parameters: the layers' inputs are kept to within 1/127 of their tile's largest value, so the gradient of a weight is that
    # of the difference to within sum over the chains of max|x| / 127 * |d|; the biases' gradients carry no such error
    o = 0
    parts = {}
    for k, w in ((z, h1), (h1, h0), (h0, n)):
        parts[len(parts)] = (np64(g[o:o + k * w]).reshape(k, w), np64(g[o + k * w:o + k * w + w]))
        o += k * w + w
    h = [Z, np.maximum(Z @ W[0] + b[0], 0)]
    h.append(np.maximum(h[1] @ W[1] + b[1], 0))
    d = [None, None, dF]
    d[1] = (d[2] @ W[2].T) * (h[2] > 0)
    d[0] = (d[1] @ W[1].T) * (h[1] > 0)
    for i in range(3):
        for j in (0, W[i].shape[1] - 1):
            bp, bm = [v.copy() for v in b], [v.copy() for v in b]
            bp[i][j] += 1e-6
            bm[i][j] -= 1e-6
            assert abs((loss(Z, W, bp) - loss(Z, W, bm)) / 2e-6 - parts[i][1][j]) < 1e-4 * max(1.0, np.abs(parts[i][1]).max())
            Wp, Wm = [v.copy() for v in W], [v.copy() for v in W]
            Wp[i][0, j] += 1e-6
            Wm[i][0, j] -= 1e-6
            fd = (loss(Z, Wp, b) - loss(Z, Wm, b)) / 2e-6
            assert abs(fd - parts[i][0][0, j]) <= np.abs(h[i]).max() / 127 * np.abs(d[i][:, j]).sum() + 1e-4 * max(1.0, abs(fd))


def test_inference_with_a_4_bit_decoder():
    rng = np.random.default_rng(11)
    n, h0, h1, z = 300, 35, 30, 10
    p = params(rng, n, h0, h1, z)
    as_list = lambda q: [(q["V1"], q["c1"]), (), (q["V2"], q["c2"]), (), (q["V3"], q["c3"])]
    x, obs = np.arange(n) / n, [20, 23, 100, 110, 117, 130, 133, 140, 170, 190]
    y = np.sin(6 * x)
    args = {"num_warmup": 5, "num_samples": 6, "num_chains": 4, "max_tree_depth": 4}
    inf = VAEInference(None, as_list(p), z, 1, x, y, obs, args, seed=2, weights="w4")
    # the same model in 64 bits at the weights the codes stand for
    W = [orc.load_w4(w.codes.cpu().numpy(), w.exps.cpu().numpy(), w.K, w.N) for w in inf.dec_w4.layers]
    q = dict(zip(NAMES, (W[0], np64(inf.dec_w4.biases[0]), W[1], np64(inf.dec_w4.biases[1]), W[2], np64(inf.dec_w4.biases[2]))))
    ref = VAEInference(None, as_list(q), z, 1, x, np64(inf.y), obs, args, dtype=torch.float64)
    Zc = torch.tensor(rng.standard_normal((6, z)), dtype=torch.float32, device=DEV)
    ls = torch.tensor(np.log(rng.uniform(0.05, 0.3, 6)), dtype=torch.float32, device=DEV)
    y1, e1 = layer(np64(Zc), 0 * np64(Zc), W[0], q["c1"])
    y2, e2 = layer(np.maximum(y1, 0), e1, W[1], q["c2"])
    f, ef = layer(np.maximum(y2, 0), e2, W[2], q["c3"])
    within(inf.predict(Zc), f, ef)
    U4, dz4, du4 = inf.potential_and_grad(Zc, ls)
    Ur, dzr, dur = ref.potential_and_grad(Zc.double(), ls.double())
    # a residual off by e moves r^2 / (2 s^2) by at most (|r| + e) e / s^2; sums of up to 32 float32 terms and exp(log s)
    # (relative 4 eps) add 64 eps of the terms' magnitudes
    s2 = np.exp(2 * np64(ls))[:, None]
    r = f[:, obs] - np64(inf.y)[obs]
    mag = ((r * r) / s2).sum(1) + (np64(Zc) ** 2).sum(1) + 200
    tol = ((np.abs(r) + ef[:, obs]) * ef[:, obs] / s2).sum(1) + 64 * U * mag
    assert (np.abs(np64(U4) - np64(Ur)) <= tol).all()
    assert (np.abs(np64(du4) - np64(dur)) <= 2 * tol).all()
    # gradients: relative to the largest, the residual's error and the sums' over s^2
    scale = np.abs(np64(dzr)).max()
    assert np.abs(np64(dz4) - np64(dzr)).max() <= 1e-4 * scale
    post = inf.run_mcmc(1)
    assert post["z"].shape == (24, z) and torch.isfinite(post["z"]).all() and torch.isfinite(post["f"]).all()
    assert torch.equal(post["f"], ops.decoder_fwd_w4(inf.dec_w4, post["z"]))
    prior, pred = inf.fit(rng_key=3, num_prior=50)
    assert prior.shape == (50, n) and pred.shape == (24, n) and torch.isfinite(prior).all() and torch.isfinite(pred).all()


def test_a_training_step_and_its_replayed_graph():
    """Weights quantised, forward, backward with parameter gradients, Adam: eager, and captured and replayed."""
    rng = np.random.default_rng(5)
    C, n, h0, h1, z = 64, 200, 48, 40, 8
    p0 = flat(params(rng, n, h0, h1, z))
    Z = torch.tensor(rng.standard_normal((C, z)), dtype=torch.float32, device=DEV)
    Y = torch.tensor(rng.standard_normal((C, n)), dtype=torch.float32, device=DEV)

    def step(p, m, v):
        dec = ops.quant_decoder_w4(p, n, h0, h1, z)
        F, acts = ops.decoder_fwd_w4(dec, Z, keep=True)
        dZ, g = ops.decoder_vjp_w4(dec, acts, (F - Y) / C, grads=True)
        ops.adam_(p, g, m, v, 1, 1e-3)
        return F, dZ, g

    def fresh():
        return p0.clone(), torch.zeros_like(p0), torch.zeros_like(p0)

    st = fresh()
    eager = []
    for _ in range(3):
        eager.append([t.clone() for t in (*step(*st), *st)])
    sg = fresh()
    step(*sg)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(*sg)
    for rounds in range(2):
        for t, v in zip(sg, fresh()):
            t.copy_(v)
        for i in range(3):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((*outs, *sg), eager[i])), (rounds, i)
        step(*fresh())  # eager work between the replays


def test_refusals():
    rng = np.random.default_rng(1)
    n, h0, h1, z = 30, 9, 7, 4
    p = params(rng, n, h0, h1, z)
    fl = flat(p)
    dec = ops.quant_decoder_w4(fl, n, h0, h1, z)
    Z = torch.zeros((3, z), device=DEV)
    F, acts = ops.decoder_fwd_w4(dec, Z, keep=True)
    lst = [(p["V1"], p["c1"]), (), (p["V2"], p["c2"]), (), (p["V3"], p["c3"])]
    for call in (lambda: ops.quant_decoder_w4(fl[:-1], n, h0, h1, z), lambda: ops.quant_decoder_w4(fl.double(), n, h0, h1, z),
                 lambda: ops.decoder_fwd_w4(dec, Z.half()), lambda: ops.decoder_fwd_w4(dec, Z[:, :3]),
                 lambda: ops.decoder_vjp_w4(dec, acts, F[:2]), lambda: ops.decoder_vjp_w4(dec, acts, F.half()),
                 lambda: ops.DecoderW4(dec.layers[::-1], dec.biases), lambda: ops.DecoderW4(dec.layers, dec.biases[::-1]),
                 lambda: VAEInference(None, lst, z, 1, np.arange(n) / n, np.zeros(n), [1, 2], {}, dtype=torch.float64, weights="w4")):
        with pytest.raises(GpvaeError):
            call()
    with pytest.raises(ValueError):
        VAEInference(None, lst, z, 1, np.arange(n) / n, np.zeros(n), [1, 2], {}, weights="w8")
    assert math.isfinite(float(F.sum()))


def test_inference_with_a_decoder_wider_than_the_float_one():
    """Hidden widths above 1024: predictions, and the potential's gradient against autograd in 64 bits."""
    rng = np.random.default_rng(21)
    n, h0, h1, z = 500, 1200, 1100, 12
    p = params(rng, n, h0, h1, z)
    x, obs = np.arange(n) / n, [3, 77, 78, 250, 499]
    y = np.cos(5 * x)
    inf = VAEInference(None, [(p["V1"], p["c1"]), (), (p["V2"], p["c2"]), (), (p["V3"], p["c3"])], z, 1, x, y, obs, {}, weights="w4")
    W = [ops.load_w4(w).double() for w in inf.dec_w4.layers]
    b = [t.double() for t in inf.dec_w4.biases]
    Z = torch.tensor(rng.standard_normal((7, z)), dtype=torch.float32, device=DEV)
    u = torch.tensor(np.log(rng.uniform(0.1, 0.3, 7)), dtype=torch.float32, device=DEV)
    y1, e1 = layer(np64(Z), 0 * np64(Z), np64(W[0]), np64(b[0]))
    y2, e2 = layer(np.maximum(y1, 0), e1, np64(W[1]), np64(b[1]))
    f, ef = layer(np.maximum(y2, 0), e2, np64(W[2]), np64(b[2]))
    within(inf.predict(Z), f, ef)
    zd, ud = Z.double().requires_grad_(), u.double().requires_grad_()
    F = torch.relu(torch.relu(zd @ W[0] + b[0]) @ W[1] + b[1]) @ W[2] + b[2]
    r = F[:, obs] - inf.y.double()[obs]
    s = torch.exp(ud)
    U = 0.5 * (r * r).sum(1) / s ** 2 + len(obs) * ud + 0.5 * (zd * zd).sum(1) + 0.5 * (s / 0.1) ** 2 - ud
    U.sum().backward()
    got = inf.potential_and_grad(Z, u)
    # the residual's error e counts (|r| + e) e / s^2 in U; float32 sums of fewer than 32 terms and exp add 64 eps of the terms
    s2, rr = np.exp(2 * np64(u))[:, None], np.abs(np64(r))
    const = (got[0].double() - U).detach()  # the potential's constant terms
    tol = ((rr + ef[:, obs]) * ef[:, obs] / s2).sum(1) + 64 * 2 * U.detach().abs().cpu().numpy() * 2.0 ** -23 + 64 * 2.0 ** -23 * ((rr ** 2 / s2).sum(1) + 100)
    assert (np.abs(np64(const - const.mean())) <= tol + tol.mean()).all()
    # gradients: relative to the largest, as above
    assert np.abs(np64(got[1]) - np64(zd.grad)).max() <= 1e-4 * np.abs(np64(zd.grad)).max()
    assert np.abs(np64(got[2]) - np64(ud.grad)).max() <= 1e-4 * max(1.0, np.abs(np64(ud.grad)).max())
