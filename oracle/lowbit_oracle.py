"""NumPy restatement, in 64 bits, of the low-bit formats and dense layers of include/gpvae_lowbit.h (test infrastructure).

Loops over tiles and searches for the exponent and the nearest value by comparison: written from the definitions, not from
the kernels."""
import numpy as np

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def up(a, b):
    return -(-a // b) * b


def tile_exponent(amax, top, lowest):
    """Exponent byte of a tile: smallest e >= lowest with amax <= top 2^e as long as top 2^e is a finite float (larger
    values saturate), 0 for zeros, 255 if not finite."""
    if not np.isfinite(amax):
        return 255
    if amax == 0:
        return 127
    e = lowest
    while amax > top * 2.0 ** e and top * 2.0 ** (e + 1) < 2.0 ** 128:
        e += 1
    return e + 127


def e2m1_nearest(v):
    """Code of the nearest E2M1 value of every |v| <= 6, ties to the even code; bit 3 the sign."""
    d = np.abs(np.abs(v)[..., None] - E2M1)
    best = d.min(-1, keepdims=True)
    tie = d == best
    even = tie & (np.arange(8) % 2 == 0)
    pick = np.where(even.any(-1), even.argmax(-1), tie.argmax(-1))
    return pick + 8 * (v < 0)


def quant_w4(W):
    """codes [kb, Np, 4] uint32, exps [kb, Np/8, 4] uint8 of W [K, N] (float64 values of the stored type)."""
    K, N = W.shape
    Kp, Np = up(K, 32), up(N, 32)
    P = np.zeros((Kp, Np))
    P[:K, :N] = W
    codes = np.zeros((Kp // 32, Np, 4), np.uint32)
    exps = np.zeros((Kp // 32, Np // 8, 4), np.uint8)
    for kt in range(Kp // 8):
        for t in range(Np // 8):
            T = P[8 * kt:8 * kt + 8, 8 * t:8 * t + 8]
            eb = tile_exponent(np.abs(T).max() if np.isfinite(T).all() else np.inf, 6, -125)
            exps[kt // 4, t, kt % 4] = eb
            if eb == 255:
                continue
            c = e2m1_nearest(np.clip(T / 2.0 ** (eb - 127), -6, 6)).astype(np.uint32)
            codes[kt // 4, 8 * t:8 * t + 8, kt % 4] = (c << (4 * np.arange(8, dtype=np.uint32))[:, None]).sum(0, dtype=np.uint32)
    return codes, exps


def load_w4(codes, exps, K, N):
    codes = codes.view(np.uint32)
    kb, Np, _ = codes.shape
    c = (codes[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    v = np.where(c >= 8, -1.0, 1.0) * E2M1[c & 7]  # [kb, n, j, i]
    s = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    v = v * np.repeat(s, 8, 1)[..., None]
    return v.transpose(0, 2, 3, 1).reshape(kb * 32, Np)[:K, :N]


def store_q8(X, relu):
    """(Y or None, codes [mb, Kp, 8] uint8, exps [mb, Kp/8] uint8)."""
    Y = np.where(X < 0, 0.0, X) if relu else X
    M, K = X.shape
    Mp, Kp = up(M, 8), up(K, 32)
    P = np.zeros((Mp, Kp))
    P[:M, :K] = Y
    codes = np.zeros((Mp // 8, Kp, 8), np.uint8)
    exps = np.zeros((Mp // 8, Kp // 8), np.uint8)
    for mb in range(Mp // 8):
        for t in range(Kp // 8):
            T = P[8 * mb:8 * mb + 8, 8 * t:8 * t + 8]
            eb = tile_exponent(np.abs(T).max() if np.isfinite(T).all() else np.inf, 255 if relu else 127, -126)
            exps[mb, t] = eb
            q = np.zeros((8, 8)) if eb == 255 else np.rint(np.clip(T / 2.0 ** (eb - 127), -255 if relu else -127, 255 if relu else 127))
            if relu:
                q = np.where((q == 0) & ~(T <= 0), 1, q)
            codes[mb, 8 * t:8 * t + 8] = q.astype(np.int64).astype(np.uint8).T
    return (Y if relu else None), codes, exps


def load_q8(codes, exps, M, K, relu):
    q = codes.astype(np.float64) if relu else codes.view(np.int8).astype(np.float64)
    s = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    v = q * np.repeat(s, 8, 1)[..., None]
    return v.transpose(0, 2, 1).reshape(-1, codes.shape[1])[:M, :K]


def dense(X, W, b=None, relu=False):
    Y = X @ W + (0 if b is None else b)
    return np.where(Y < 0, 0.0, Y) if relu else Y


def dense_vjp(dY, W, mask=None):
    dX = dY @ W.T
    return dX if mask is None else np.where(mask, dX, 0.0)


def dense_grads(X, dY):
    return X.T @ dY, dY.sum(0)
