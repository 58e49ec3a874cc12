"""What the operators on dictionaries in 4 bits and columns in 8 keep of float32's and double's precision, against the NumPy
oracle in 64 bits: every bound here is a rounding or two of the formula, with no factor for the kernels' order."""
import numpy as np
import pytest

from oracle import lowbit_oracle as lo

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch


@pytest.fixture(scope="module")
def eng(torch):
    from onmf_ontf_ndl_amd.engine import get_engine
    return get_engine()


def host(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def kept_values(eng, X):
    K = eng.keep8(eng.dev(X))
    return K, lo.values8(K.codes.cpu().numpy().astype(np.float64), host(K.scales), K.n)


# ------------------------------------------------------------------------------------------------- the gradient
@pytest.mark.parametrize("d,r,n", [(256, 64, 8000), (512, 128, 20000), (1200, 100, 8191), (300, 300, 4000), (60, 20, 3000)])
def test_gradient_at_the_least_squares_dictionary(eng, torch, d, r, n):
    """Where W (H H^T) and X H^T cancel down to the rounding of W itself.  Everything up to dW is in double, several runs of
    groups included: 2^-53 a rounding of the terms' magnitudes, in a chain of at most n / 128 groups, 16 for their runs and
    r + 8 for W A (the oracle's own: n + 2 r), and half a float32 step of the result."""
    rs = np.random.RandomState(d + r)
    H = np.maximum(rs.randn(r, n), 0).astype(np.float32)
    X = np.maximum(np.maximum(rs.randn(d, r), 0) @ H + rs.rand(d, n), 0).astype(np.float32)
    (KX, Xh), (KH, Hh) = kept_values(eng, X), kept_values(eng, H)
    assert eng.lib.onmf_keep8_workspace(d, r, n, 1) > 8 * r * (r + d) + 512          # several runs
    W = np.linalg.solve(Hh @ Hh.T, Hh @ Xh.T).T.astype(np.float32)
    g = host(eng.keep8_gradient(eng.dev(W), KX, KH))
    W64 = W.astype(np.float64)
    want = W64 @ (Hh @ Hh.T) - Xh @ Hh.T
    size = np.abs(W64) @ (np.abs(Hh) @ np.abs(Hh).T) + np.abs(Xh) @ np.abs(Hh).T
    assert np.abs(want).max() <= 1e-6 * size.max()
    assert (np.abs(g - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -53 * (n / 128 + 16 + r + 8 + n + 2 * r) * size).all()


@pytest.mark.parametrize("d,r,n", [(700, 256, 500), (4100, 300, 400), (4100, 330, 400), (6000, 640, 300), (1300, 1030, 700),
                                   (150, 2050, 300), (260, 2050, 300)])
@pytest.mark.parametrize("kind", ["even", "dead", "rescaled", "apart", "signed", "dominated"])
def test_gradient_holds_the_terms_that_are_summed(eng, torch, d, r, n, kind):
    """W (H H^T) in double or in whole digits, whichever a size takes: an entry is off by at most half a float32 step of itself
    and half a step of its own terms, |W| |H H^T| + |X| |H|^T - of an atom that no column uses, of scales moved from W to H, of
    small entries beside large ones that meet zeros."""
    rs = np.random.RandomState(d + r + n)
    W = np.maximum(rs.randn(d, r) + 0.4, 0).astype(np.float32)
    H = np.maximum(rs.randn(r, n), 0).astype(np.float32)
    if kind == "dead":
        H[3] = 0
        H[r - 1] = 0
        W[:, 3] *= 1e4
        W[:, r - 1] *= 1e30
    elif kind == "rescaled":
        for j, f in ((5, 1e-4), (6, 1e6), (7, 1e-15), (r - 2, 1e12)):
            W[:, j] *= f
            H[j] /= f
    elif kind == "apart":
        H *= np.arange(r)[:, None] % min(n, r) == np.arange(n)[None, :] % min(n, r)
        W *= 10.0 ** rs.randint(-6, 1, size=(d, r))
    elif kind == "signed":
        W = rs.randn(d, r).astype(np.float32)
    elif kind == "dominated":
        W[:, 1:] *= 1e-5
        W[::3, 0] = 0
    live = np.where(H.any(1), np.abs(W).max(0), 0) if kind != "dead" else np.where(H.any(1), 1, 0)
    X = np.maximum((W * (live > 0)).astype(np.float64) @ H + 0.1 * rs.rand(d, n), 0).astype(np.float32)
    (KX, Xh), (KH, Hh) = kept_values(eng, X), kept_values(eng, H)
    g = host(eng.keep8_gradient(eng.dev(W), KX, KH))
    W64 = W.astype(np.float64)
    A, B = Hh @ Hh.T, Xh @ Hh.T
    want = W64 @ A - B
    size = np.abs(W64) @ A + np.abs(Xh) @ np.abs(Hh).T
    bound = 2.0 ** -24 * np.abs(want) + 2.0 ** -25 * (1 + 2.0 ** -20) * size + 2.0 ** -53 * (2 * n + 4 * r + 64) * size
    assert np.isfinite(g).all() and (np.abs(g - want) <= bound).all()
    # ... and every entry depends on its own row of W alone, whichever way its neighbours are computed
    other = rs.randn(d, r).astype(np.float32) * np.float32(1e3)
    other[::7] = W[::7]
    assert np.array_equal(host(eng.keep8_gradient(eng.dev(other), KX, KH))[::7], g[::7])


# ------------------------------------------------------------------------------------------------- the aggregates
@pytest.mark.parametrize("d,r,n", [(40, 20, 1000), (100, 60, 300), (130, 129, 700), (300, 300, 260), (200, 30, 5000)])
def test_aggregates_keep_float32s_range(eng, torch, d, r, n):
    """Scales whose own product float32 does not hold: small columns and codes (two roundings a group and its addition, half a
    step each, as ever), and large ones that never meet, whose sums are zeros."""
    rs = np.random.RandomState(d + n)
    X, H = (rs.rand(d, n) * 1e-20).astype(np.float32), (rs.rand(r, n) * 1e-16).astype(np.float32)
    (KX, Xh), (KH, Hh) = kept_values(eng, X), kept_values(eng, H)
    _, B = eng.keep8_aggregate(KX, KH, 1.0)
    assert (np.abs(host(B) - Hh @ Xh.T) <= 2.0 ** -24 * (n / 128 + 4) * (Hh @ Xh.T)).all()
    early = np.arange(n) % 128 < 64
    X, H = (rs.rand(d, n) * early * 1e36).astype(np.float32), (rs.rand(r, n) * ~early * 1e8).astype(np.float32)
    (KX, Xh), (KH, Hh) = kept_values(eng, X), kept_values(eng, H)
    A, B = eng.keep8_aggregate(KX, KH, 1.0)
    assert np.array_equal(host(B), np.zeros((r, d)))
    assert (np.abs(host(A) - Hh @ Hh.T) <= 2.0 ** -24 * (n / 128 + 4) * (Hh @ Hh.T)).all()


# ------------------------------------------------------------------------------------------------- the two products
STEP = 2.0 ** -23          # a rounding, or what a matrix instruction cuts off
# every kernel of either product: one column, few in one launch, ranges and slabs, weights resident, weights laid out
PATHS = [(441, 25, 1, 64), (2500, 70, 1, 128), (1030, 20, 1, 32), (100, 16, 2, 64), (2100, 33, 2, 32), (1100, 8200, 2, 32),
         (441, 72, 3, 64), (250, 40, 20, 32), (441, 72, 50, 128), (2500, 8200, 8, 64), (8192, 72, 3, 32), (4096, 40, 100, 64),
         (2100, 3000, 31, 32), (300, 70, 1501, 64), (1200, 100, 8192, 64), (441, 100, 1101, 32), (33, 3, 1025, 32),
         (1300, 900, 1031, 32), (3000, 300, 1026, 128)]


def packed(eng, q, z, s, d, group):
    from onmf_ontf_ndl_amd import PackedDictionary
    codes, scales = lo.to_codes4(q, z, s)
    t = eng.torch
    return PackedDictionary(t.from_numpy(codes).to(eng.device), t.from_numpy(scales).to(eng.device), d, group)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1e-30, 1e35, 1.5e38])
@pytest.mark.parametrize("d,r,b,group", PATHS)
def test_products_keep_float32s_range(eng, torch, d, r, b, group, size, dtype):
    """Columns near either end of what float32 holds, entries of a dictionary far from zero beside their scale: the result is
    finite and as near as ever - 2^-23 a rounding, at most K / 4 + 64 of them one after another, of the magnitudes that are
    added up - where those have a sum that float32 holds."""
    rs = np.random.RandomState(d + r + b)
    groups = -(-d // group)
    q = rs.randint(0, 16, size=(r, groups * group))
    q[:, d:] = 0
    z = rs.randint(225, 241, size=(r, groups))
    for K, other, call in ((d, r, "dict4_correlate"), (r, d, "dict4_product")):
        # entries of up to 255 2^-e, K of them: their sum's magnitude stays below 1.5 times the largest |x|
        s = np.full((r, groups), 2.0 ** -np.ceil(np.log2(255 * K / 1.5)))
        P = packed(eng, q, z, s, d, group)
        W = lo.values4(q, z, s, d)
        W = W.T if call == "dict4_correlate" else W
        X = eng.dev((rs.rand(K, b) * size).astype(np.float32))
        X = X.bfloat16() if dtype == "bfloat16" else X
        got, want = host(getattr(eng, call)(P, X)), W @ host(X)
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= STEP * (K / 4 + 64) * want).all()


def one_each(rs, K, b, values):
    """K x b columns with one entry that is not zero, at a random place; (matrix, places)"""
    X, at = np.zeros((K, b), dtype=np.float32), rs.randint(K, size=b)
    X[at, np.arange(b)] = values
    return X, at


@pytest.mark.parametrize("d,r,b,group", PATHS)
def test_products_use_every_bit_of_a_column(eng, torch, d, r, b, group):
    """One entry a column, with all of float32's 24 bits, against weights that are powers of two (by q, or by z alone): the
    result is that entry shifted, whatever pieces it is taken in, so it has to be equal."""
    rs = np.random.RandomState(d + 2 * r + b)
    groups = -(-d // group)
    for by_z in (False, True):
        q = np.zeros((r, groups * group), dtype=int) if by_z else 2 ** rs.randint(0, 4, size=(r, groups * group))
        q[:, d:] = 0
        z = 2 ** rs.randint(3, 8, size=(r, groups)) * rs.choice([-1, 1], size=(r, groups)) if by_z else np.zeros((r, groups), dtype=int)
        s = 2.0 ** rs.randint(-12, 5, size=(r, groups))
        P = packed(eng, q, z, s, d, group)
        W = lo.values4(q, z, s, d)
        for K, M, call in ((d, W.T, "dict4_correlate"), (r, W, "dict4_product")):
            x = (rs.randint(2 ** 23, 2 ** 24, size=b) | 1) * rs.choice([-1.0, 1.0], size=b) * 2.0 ** rs.randint(-60, 20, size=b)
            X, at = one_each(rs, K, b, x)
            assert np.array_equal(host(getattr(eng, call)(P, eng.dev(X))), M[:, at] * x)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,r,b,group", PATHS)
def test_products_use_every_bit_of_a_weight(eng, torch, d, r, b, group, dtype):
    """Weights of 16 bits, s (q + z) = 129 * 255 2^e.  One entry a column: of 9 bits in float32, 257, which makes 24 bits and
    needs the weight's lower half times the entry's second piece, or 1 in bfloat16 - both exact.  And any entry, within three
    roundings or cuts of 2^-23 of the product and one of the scale, where what is left out (2^-25) has its place too."""
    rs = np.random.RandomState(d + 3 * r + b)
    groups = -(-d // group)
    q = np.full((r, groups * group), 15)
    q[:, d:] = 0
    z = np.full((r, groups), 240)
    s = 129 * 2.0 ** rs.randint(-20, 0, size=(r, groups))
    P = packed(eng, q, z, s, d, group)
    W = lo.values4(q, z, s, d)
    for K, M, call in ((d, W.T, "dict4_correlate"), (r, W, "dict4_product")):
        x = (257.0 if dtype == "float32" else 1.0) * rs.choice([-1.0, 1.0], size=b) * 2.0 ** rs.randint(-10, 10, size=b)
        X, at = one_each(rs, K, b, x)
        X = eng.dev(X).bfloat16() if dtype == "bfloat16" else eng.dev(X)
        assert np.array_equal(host(getattr(eng, call)(P, X)), M[:, at] * x)
        X, at = one_each(rs, K, b, rs.randn(b))
        X = eng.dev(X).bfloat16() if dtype == "bfloat16" else eng.dev(X)
        want = M[:, at] * host(X)[at, np.arange(b)]
        assert (np.abs(host(getattr(eng, call)(P, X)) - want) <= 4 * STEP * np.abs(want)).all()
