"""GPU tests of dictionaries held in 4 bits and columns held in 8, through the engine and the C-ABI, against the NumPy
oracle in 64 bits.

Tolerances.  What is whole (codes, offsets, scales) is equal.  Products of small whole numbers whose sums stay
below 2^24 are equal too, whatever the order: these tests find a wrong index anywhere.  For real values an element's
error is at most 2^-23 L M with M = sum of the magnitudes that are added up (s (q + |z|) |x| for a 4-bit dictionary)
and L the additions one after another: no kernel has a chain of more than K / 4 + 64 for a contraction of length K
(four waves or sixteen-wide matrix instructions share it at least), and 2^-23, twice half a float32 step, also covers
matrix instructions that cut instead of round and the pieces that three bfloat16 leave over (2^-24)."""
import ctypes as C

import numpy as np
import pytest

from oracle import lowbit_oracle as lo

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23


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


def as_type(torch, eng, a, dtype):
    """(tensor of that type, the float64 values it holds)"""
    t = eng.dev(np.asarray(a, dtype=np.float32))
    t = t.bfloat16() if dtype == "bfloat16" else t
    return t, host(t)


def whole_dictionary(eng, rs, d, r, group):
    """A 4-bit dictionary of small whole numbers: scales 1 and 2, offsets -20..20."""
    from onmf_ontf_ndl_amd import PackedDictionary
    groups = -(-d // group)
    q = rs.randint(0, 16, size=(r, groups * group))
    q.reshape(r, -1)[:, d:] = 0
    z = rs.randint(-20, 21, size=(r, groups))
    s = 2.0 ** rs.randint(0, 2, size=(r, groups))
    codes, scales = lo.to_codes4(q, z, s)
    t = eng.torch
    return PackedDictionary(t.from_numpy(codes).to(eng.device), t.from_numpy(scales).to(eng.device), d, group), (q, z, s)


# ------------------------------------------------------------------------------------------------- packing
@pytest.mark.parametrize("d,r,group", [(1, 1, 32), (32, 3, 32), (100, 16, 64), (441, 25, 64), (129, 300, 128), (1200, 7, 128)])
def test_pack_is_the_oracles(eng, torch, d, r, group):
    rs = np.random.RandomState(d + r)
    W = np.maximum(rs.randn(d, r) + 0.4, 0).astype(np.float32)
    W[:, 0] = rs.randn(d)                                      # signed
    if r > 3:
        W[:, 1] = 1 + 1e-3 * rs.rand(d)                        # far from zero
        W[:, 2] = 0
        W[:, 3] *= 1e-40                                       # below the smallest scale
    if r > 6:
        W[d // 2, 4] = np.nan
        W[d - 1, 5] = -np.inf
        W[:, 6] = np.round(W[:, 6] * 4) / 4 + 0.125            # quotients on and next to halves
    P = eng.dict4_pack(eng.dev(W), group)
    q, z, s = lo.pack4(W, group)
    codes, scales = lo.to_codes4(q, z, s)
    assert np.array_equal(P.codes.cpu().numpy(), codes)
    fine = np.isfinite(s)
    got = P.scales.cpu().numpy()
    assert np.array_equal(got[fine], scales[fine])
    assert np.isnan((got.view(np.uint32) & 0xFFFF0000).view(np.float32)[~fine]).all()
    # (the float32 product s (q + z): an eight-bit scale times at most eight bits is exact)
    assert np.array_equal(host(P.unpack()), lo.values4(q, z, s, d), equal_nan=True)


# ------------------------------------------------------------------------------------------------- products
SHAPES = [  # d, r, b, group: single columns, a few, many; ragged and whole; one split and several
    (1, 1, 1, 32), (441, 25, 1, 64), (1024, 256, 1, 64), (2500, 70, 1, 128), (4100, 9, 1, 32), (7, 1000, 1, 32),
    (100, 16, 2, 64), (2100, 33, 2, 32), (441, 25, 3, 64), (1030, 130, 4, 128), (513, 257, 5, 32), (1500, 40, 8, 64),
    (9000, 5, 8, 128), (1, 1, 9, 32), (33, 129, 9, 32), (441, 25, 17, 64), (100, 16, 130, 64), (128, 128, 128, 128),
    (257, 300, 33, 32), (1200, 100, 257, 64), (1024, 256, 300, 128), (130, 2000, 65, 64), (4096, 40, 100, 64),
    (8192, 20, 3, 64), (1100, 8200, 2, 32), (700, 9000, 31, 64), (2100, 4000, 64, 128), (3, 5000, 64, 32),
    (60, 40, 1100, 32), (300, 70, 1501, 64), (200, 6001, 200, 32), (2100, 600, 601, 128), (33, 3, 1025, 32), (90, 33, 1030, 64), (777, 1400, 1027, 64),
    (1300, 900, 1031, 32), (3000, 300, 1026, 128), (700, 4000, 1025, 64),
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,r,b,group", SHAPES)
def test_products_of_whole_numbers_are_exact(eng, torch, d, r, b, group, dtype):
    rs = np.random.RandomState(d + 3 * r + 7 * b)
    P, parts = whole_dictionary(eng, rs, d, r, group)
    W = lo.values4(*parts, d)
    X, Xh = as_type(torch, eng, rs.randint(-4, 5, size=(d, b)), dtype)
    H, Hh = as_type(torch, eng, rs.randint(-4, 5, size=(r, b)), dtype)
    assert max(np.abs(W).sum(0).max(), np.abs(W).sum(1).max()) * 4 < 2 ** 24
    C_, R = eng.dict4_correlate(P, X), eng.dict4_product(P, H)
    assert C_.dtype is torch.float32 and tuple(C_.shape) == (r, b) and tuple(R.shape) == (d, b)
    assert np.array_equal(host(C_), W.T @ Xh)
    assert np.array_equal(host(R), W @ Hh)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,r,b,group", SHAPES)
def test_products_of_real_values(eng, torch, d, r, b, group, dtype):
    rs = np.random.RandomState(d + 5 * r + 11 * b)
    W = np.maximum(rs.randn(d, r) + 0.4, 0).astype(np.float32)
    if r > 1:
        W[:, 1] = 0.5 + 1e-2 * rs.randn(d)
    P = eng.dict4_pack(eng.dev(W), group)
    q, z, s = lo.pack4(W, group)
    Wq, M = lo.values4(q, z, s, d), lo.reach4(q, z, s, d)
    X, Xh = as_type(torch, eng, rs.randn(d, b) * 10.0 ** rs.randint(-4, 4, size=(d, 1)), dtype)
    H, Hh = as_type(torch, eng, rs.randn(r, b) * 10.0 ** rs.randint(-4, 4, size=(r, 1)), dtype)
    C_, R = host(eng.dict4_correlate(P, X)), host(eng.dict4_product(P, H))
    assert (np.abs(C_ - Wq.T @ Xh) <= STEP * (d / 4 + 64) * (M.T @ np.abs(Xh))).all()
    assert (np.abs(R - Wq @ Hh) <= STEP * (r / 4 + 64) * (M @ np.abs(Hh))).all()


@pytest.mark.parametrize("b", [1, 3, 8, 40, 601, 1101])
def test_products_take_views(eng, torch, b):
    """Columns of a wider matrix, a transposed one, every second column, one value for all."""
    rs = np.random.RandomState(b)
    d, r = 300, 37
    P, parts = whole_dictionary(eng, rs, d, r, 64)
    W = lo.values4(*parts, d)
    wide = eng.dev(rs.randint(-3, 4, size=(d, 2 * b + 7)).astype(np.float32))
    tall = eng.dev(rs.randint(-3, 4, size=(b, d)).astype(np.float32))
    one = eng.dev(rs.randint(-3, 4, size=(d, 1)).astype(np.float32))
    for X in (wide[:, 1:b + 1], wide[:, 4:b + 4], tall.t(), wide[:, 0:2 * b:2], one.expand(d, b), wide.bfloat16()[:, 3:b + 3]):
        assert np.array_equal(host(eng.dict4_correlate(P, X)), W.T @ host(X))
    codes = eng.dev(rs.randint(-3, 4, size=(r, 2 * b + 7)).astype(np.float32))
    for H in (codes[:, 1:b + 1], codes.bfloat16()[:, 2:b + 2], codes[:, 0:2 * b:2], codes.bfloat16()[:, 5:b + 5], codes[:b, :r].t()[:, :1] if b <= r else codes[:, :1]):
        if H.shape[0] == r:
            assert np.array_equal(host(eng.dict4_product(P, H)), W @ host(H))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_that_lie_far_apart(eng, torch, dtype):
    """Offsets that pass 32 bits, in bytes and in elements: 40 rows of 2^26 + 1 values, of which the first few count."""
    rs = np.random.RandomState(4)
    d, ld = 40, 2 ** 26 + 1
    held = torch.empty(d * ld, dtype=getattr(torch, dtype), device=eng.device)
    wide = held.view(d, ld)
    P, parts = whole_dictionary(eng, rs, d, 37, 32)
    W = lo.values4(*parts, d)
    Q, qarts = whole_dictionary(eng, rs, 37, d, 32)
    V = lo.values4(*qarts, 37)
    for b in (1, 2, 5, 20, 41, 601, 1101):
        X, Xh = as_type(torch, eng, rs.randint(-4, 5, size=(d, b)), dtype)
        wide[:, 7:7 + b] = X
        view = wide[:, 7:7 + b]
        assert np.array_equal(host(eng.dict4_correlate(P, view)), W.T @ Xh)
        assert np.array_equal(host(eng.dict4_product(Q, view)), V @ Xh)
        K = eng.keep8(view)
        q, s = lo.keep8(Xh)
        assert np.array_equal(K.codes.cpu().numpy(), q) and np.array_equal(host(K.scales), s)
    # ... and by way of the workspace
    P, parts = whole_dictionary(eng, rs, d, 20000, 32)
    Q, qarts = whole_dictionary(eng, rs, 5000, d, 32)
    b = 1101
    X, Xh = as_type(torch, eng, rs.randint(-4, 5, size=(d, b)), dtype)
    wide[:, 7:7 + b] = X
    assert np.array_equal(host(eng.dict4_correlate(P, wide[:, 7:7 + b])), lo.values4(*parts, d).T @ Xh)
    assert np.array_equal(host(eng.dict4_product(Q, wide[:, 7:7 + b])), lo.values4(*qarts, 5000) @ Xh)


@pytest.mark.parametrize("b", [1, 2, 4, 7, 8, 9, 100, 601, 1101])
def test_a_column_that_is_not_finite_touches_no_other(eng, torch, b):
    rs = np.random.RandomState(b)
    d, r = 200, 150
    P, parts = whole_dictionary(eng, rs, d, r, 64)
    W = lo.values4(*parts, d)
    X, H = rs.randint(-3, 4, size=(d, b)).astype(np.float32), rs.randint(-3, 4, size=(r, b)).astype(np.float32)
    bad = b // 2
    X[5, bad], H[5, bad] = np.nan, np.inf
    others = np.arange(b) != bad
    C_, R = host(eng.dict4_correlate(P, eng.dev(X))), host(eng.dict4_product(P, eng.dev(H)))
    assert np.array_equal(C_[:, others], W.T @ X.astype(np.float64)[:, others])
    assert np.array_equal(R[:, others], W @ H.astype(np.float64)[:, others])
    assert np.isnan(C_[:, bad]).all() and not np.isfinite(R[W[:, 5] != 0, bad]).any()


@pytest.mark.parametrize("b", [1, 5, 40, 1101])
def test_product_leaves_what_lies_behind_its_rows(eng, torch, b):
    from onmf_ontf_ndl_amd.engine import _ptr
    rs = np.random.RandomState(b)
    d, r, ld = 130, 50, b + 5
    P, parts = whole_dictionary(eng, rs, d, r, 32)
    H = eng.dev(rs.randint(-3, 4, size=(r, b)).astype(np.float32))
    out = torch.full((d + 2, ld), 7.0, device=eng.device)
    n = eng.lib.onmf_dict4_workspace(1, d, r, b, 32)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=eng.device)
    rc = eng.lib.onmf_dict4_product(eng.ctx, d, r, b, 32, _ptr(P.codes), _ptr(P.scales), _ptr(H), 0, b, _ptr(out), ld,
                                    _ptr(ws), n, eng.stream())
    assert rc == 0
    got = host(out)
    assert np.array_equal(got[:d, :b], lo.values4(*parts, d) @ host(H))
    assert (got[:d, b:] == 7).all() and (got[d:] == 7).all()


def test_the_two_products_are_each_others_gradient(eng, torch):
    """L = sum(T * (W H)): its difference along a direction against <W^T T, direction>."""
    rs = np.random.RandomState(0)
    d, r, b = 257, 60, 20
    P = eng.dict4_pack(eng.dev(rs.rand(d, r)), 32)
    T, H, D = eng.dev(rs.randn(d, b)), eng.dev(rs.randn(r, b)), eng.dev(rs.randn(r, b))
    grad = host(eng.dict4_correlate(P, T))
    up, down = host(eng.dict4_product(P, H + D)), host(eng.dict4_product(P, H - D))
    got = (host(T) * (up - down)).sum() / 2
    # linear in H: only rounding is left - each of the d b products sums r terms of size <= about 3
    size = np.abs(host(T)).sum() * r * 3 * 2.0 ** -23
    assert abs(got - (grad * host(D)).sum()) <= size


def test_library_refuses_what_the_engine_would_not_send(eng, torch):
    from onmf_ontf_ndl_amd.engine import _ptr
    P, _ = whole_dictionary(eng, np.random.RandomState(0), 64, 300, 64)
    X, out = eng.zeros(64, 16), eng.zeros(300, 16)
    lib, ctx = eng.lib, eng.ctx

    def call(d=64, r=300, b=16, group=64, codes=P.codes, x=X, kind=0, ld=16, c=out, ws=None, n=0):
        return lib.onmf_dict4_correlate(ctx, d, r, b, group, _ptr(codes), _ptr(P.scales), _ptr(x), kind, ld, _ptr(c),
                                        _ptr(ws), n, eng.stream())
    for bad in (dict(d=0), dict(d=1 << 19), dict(r=0), dict(b=0), dict(b=-1), dict(group=63), dict(kind=2), dict(ld=15),
                dict(x=None), dict(c=None), dict(codes=None), dict(b=2 ** 31 - 5, ld=2 ** 31 - 1)):
        assert call(**bad) == -1, bad
        assert b"dict4_correlate" in lib.onmf_last_error(ctx)
    need = lib.onmf_dict4_workspace(0, 8192, 25, 16, 64)
    assert need > 0
    big, _ = whole_dictionary(eng, np.random.RandomState(0), 8192, 25, 64)
    xx, c = eng.zeros(8192, 16), eng.zeros(25, 16)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=eng.device)
    for where, n in ((_ptr(ws), need - 1), (None, need), (ws.data_ptr() + 4, need)):
        assert call(d=8192, r=25, codes=big.codes, x=xx, c=c, ws=None, n=0) == -1
        assert lib.onmf_dict4_correlate(ctx, 8192, 25, 16, 64, _ptr(big.codes), _ptr(big.scales), _ptr(xx), 0, 16, _ptr(c), where, n,
                                        eng.stream()) == -1
    need = lib.onmf_dict4_workspace(1, 64, 5000, 16, 64)
    assert need > 0
    big, _ = whole_dictionary(eng, np.random.RandomState(0), 64, 5000, 64)
    h, out, ws = eng.zeros(5000, 16), eng.zeros(64, 16), torch.empty(need, dtype=torch.uint8, device=eng.device)
    for bad in (dict(ldr=15), dict(ldh=15), dict(n=need - 1), dict(kind=7), dict(b=0)):
        a = dict(dict(b=16, kind=0, ldh=16, ldr=16, n=need), **bad)
        assert lib.onmf_dict4_product(ctx, 64, 5000, a["b"], 64, _ptr(big.codes), _ptr(big.scales), _ptr(h), a["kind"], a["ldh"], _ptr(out),
                                      a["ldr"], _ptr(ws), a["n"], eng.stream()) == -1, bad


# ------------------------------------------------------------------------------------------------- columns in 8 bits
def awkward_columns(rs, d, n):
    X = (rs.randn(d, n) * 10.0 ** rs.randint(-6, 6, size=(d, 1))).astype(np.float32)
    X[0] = 0
    if d > 3:
        X[1] = np.round(rs.rand(n) * 254) / 2 - 63.5            # with a largest of 63.5: quotients on halves
        X[1, 0] = 63.5
        X[2] *= np.float32(1e-41 / 1e-6)                        # at and below the smallest scale
    if d > 6:
        X[4, n // 2] = np.nan
        X[5, n - 1] = np.inf
        X[6, 0] = -3e38
    return X


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,n", [(1, 1), (3, 128), (7, 129), (25, 1000), (100, 127), (441, 260), (2, 4099)])
def test_keep_is_the_oracles(eng, torch, d, n, dtype):
    rs = np.random.RandomState(d + n)
    X, Xh = as_type(torch, eng, awkward_columns(rs, d, n), dtype)
    K = eng.keep8(X)
    q, s = lo.keep8(Xh)
    assert np.array_equal(host(K.scales), s, equal_nan=True)
    assert np.array_equal(K.codes.cpu().numpy(), q)
    want = lo.values8(q, s, n)
    back = host(K.expand())                                    # one float32 rounding of s q
    fine = np.isfinite(want)
    assert np.isnan(back[~fine]).all()
    assert (np.abs(back - want)[fine] <= 2.0 ** -24 * np.abs(want)[fine] + 2.0 ** -150).all()
    idx = np.concatenate([rs.randint(-n, n, size=37), [0, n - 1, -n, -1, 0]])
    assert np.array_equal(host(K.expand(idx)), back[:, idx], equal_nan=True)


@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_keep_takes_views(eng, torch, shift):
    rs = np.random.RandomState(shift)
    wide = eng.dev(rs.randn(9, 400))
    for X in (wide[:, shift:shift + 300], wide[:, shift::2], wide.t()[shift:], wide[:1].expand(5, 400),
              wide.bfloat16()[:, shift:shift + 131]):
        q, s = lo.keep8(host(X))
        K = eng.keep8(X)
        assert np.array_equal(K.codes.cpu().numpy(), q) and np.array_equal(host(K.scales), s)


def whole_columns(eng, rs, d, n, most=15):
    """Kept columns of small whole numbers: scales 1 and 2."""
    from onmf_ontf_ndl_amd import KeptColumns
    groups = -(-n // 128)
    q = rs.randint(-most, most + 1, size=(d, groups * 128))
    q[:, n:] = 0
    s = 2.0 ** rs.randint(0, 2, size=(d, groups))
    t = eng.torch
    return KeptColumns(t.from_numpy(q.astype(np.int8)).to(eng.device), eng.dev(s), n), lo.values8(q, s, n)


SUMS = [(1, 1, 1), (3, 2, 128), (441, 25, 1000), (100, 16, 127), (130, 129, 700), (1200, 100, 1500), (257, 300, 129),
        (64, 1, 5000), (1, 64, 5000), (1024, 256, 2048), (40, 600, 257),
        (300, 40, 9), (33, 333, 16), (200, 531, 17), (17, 15, 64), (1000, 70, 128), (8300, 20, 100), (8300, 129, 65), (1, 1000, 2),
        (4100, 330, 300), (5000, 1030, 140), (700, 1100, 2000)]        # the last three: W (H H^T) by whole digits


@pytest.mark.parametrize("d,r,n", SUMS)
def test_aggregates_of_whole_numbers_are_exact(eng, torch, d, r, n):
    rs = np.random.RandomState(d + r + n)
    X, Xh = whole_columns(eng, rs, d, n)
    H, Hh = whole_columns(eng, rs, r, n)
    assert n * 30 * 30 * 2 < 2 ** 24
    A, B = rs.randint(-50, 50, size=(r, r)) * 4.0, rs.randint(-50, 50, size=(r, d)) * 4.0
    for w, a, b in ((1.0, None, None), (0.5, A, B), (0.25, A, None), (0.25, None, B)):
        got = eng.keep8_aggregate(X, H, w, None if a is None else eng.dev(a), None if b is None else eng.dev(b))
        want = lo.aggregate(Xh, Hh, w, 0 if a is None else a, 0 if b is None else b)
        # rounded once: sums below 2^24, halves and quarters of them below 2^22 are exact; above, half a step
        for x, y in zip(got, want):
            assert (np.abs(host(x) - y) <= 2.0 ** -24 * np.abs(y)).all()
    W = rs.randint(-2, 3, size=(d, r)).astype(np.float64)
    g = host(eng.keep8_gradient(eng.dev(W), X, H))
    want = lo.gradient(W, Xh, Hh)
    assert (np.abs(g - want) <= 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("d,r,n", SUMS)
def test_aggregates_and_gradient_of_real_values(eng, torch, d, r, n):
    """Inside a group sums are exact; a workgroup adds at most n / 128 groups in float32, each with three roundings
    (the product of the scales, its product with the whole sum - that one fused - and the conversion of a whole sum
    of up to 2^21, exact): an element is within 2^-24 (n / 128 + 3) of the sum of magnitudes, and one more half step
    where float32 comes out."""
    rs = np.random.RandomState(d * r + n)
    W = np.maximum(rs.randn(d, r), 0).astype(np.float32)
    H = np.maximum(rs.randn(r, n), 0).astype(np.float32)
    X = np.maximum(W @ H + 0.1 * rs.rand(d, n), 0).astype(np.float32)
    KX, KH = eng.keep8(eng.dev(X)), eng.keep8(eng.dev(H))
    Xh, Hh = lo.values8(*lo.keep8(X), n), lo.values8(*lo.keep8(H), n)
    eps = 2.0 ** -24 * (n / 128 + 4)
    A, B = eng.keep8_aggregate(KX, KH, 1.0)
    assert (np.abs(host(A) - Hh @ Hh.T) <= eps * (np.abs(Hh) @ np.abs(Hh).T)).all()
    assert (np.abs(host(B) - Hh @ Xh.T) <= eps * (np.abs(Hh) @ np.abs(Xh).T)).all()
    A0, B0 = rs.rand(r, r).astype(np.float32), rs.rand(r, d).astype(np.float32)
    A1, B1 = eng.keep8_aggregate(KX, KH, 0.3, eng.dev(A0), eng.dev(B0))
    wa, wb = lo.aggregate(Xh, Hh, 0.3, A0.astype(np.float64), B0.astype(np.float64))
    assert (np.abs(host(A1) - wa) <= 2 * eps * np.abs(wa)).all() and (np.abs(host(B1) - wb) <= 2 * eps * np.abs(wb)).all()
    W1 = np.maximum(W + 0.2 * rs.randn(d, r), 0).astype(np.float32)
    g = host(eng.keep8_gradient(eng.dev(W1), KX, KH))
    W64 = W1.astype(np.float64)
    # the gradient's sums are doubles, rounded to float32 once a run; what is cut off its digits is bounded as below
    A64, want = np.abs(Hh) @ np.abs(Hh).T, lo.gradient(W64, Xh, Hh)
    size = np.abs(W64) @ A64 + np.abs(Xh) @ np.abs(Hh).T
    bound = 2.0 ** -24 * (1 + 2.0 ** -10) * size + 2.0 ** -24 * np.abs(want)
    if d * r * r > 4e8:
        most = np.abs(W64).max(1)[:, None]
        bound += 2.0 ** -26 * most * (A64.sum(0) + r * A64.max(0))[None, :]
    assert (np.abs(g - want) <= bound).all()


def test_gradient_by_digits_row_by_row(eng, torch):
    """Rows of W of very different size, a zero one and ones that are not finite: each keeps its own precision (2^-26 of its
    largest entry times the row sum of |A|, as for the sums' float32 runs) and touches no other."""
    rs = np.random.RandomState(8)
    d, r, n = 4100, 330, 400
    X, H = np.maximum(rs.randn(d, n), 0).astype(np.float32), np.maximum(rs.randn(r, n), 0).astype(np.float32)
    W = rs.randn(d, r).astype(np.float32)
    W[1] *= 1e-30
    W[2] *= 1e28
    W[3] = 0
    W[4, 7], W[5, 0] = np.nan, np.inf
    W[6, :-1] *= 1e-5
    KX, KH = eng.keep8(eng.dev(X)), eng.keep8(eng.dev(H))
    Xh, Hh = host(KX.expand()), host(KH.expand())
    g = host(eng.keep8_gradient(eng.dev(W), KX, KH))
    rest = np.setdiff1d(np.arange(d), [4, 5])
    assert np.isnan(g[4]).all() and not np.isfinite(g[5]).any()
    W64, A = W.astype(np.float64)[rest], Hh @ Hh.T
    want = W64 @ A - (Xh @ Hh.T)[rest]
    size = np.abs(W64) @ A + (Xh @ Hh.T)[rest]
    most = np.abs(W64).max(1)[:, None] * A.sum(0)[None, :] + r * np.abs(W64).max(1)[:, None] * A.max(0)[None, :]
    # a run's sum and the result rounded to float32, digits cut at 2^-27 on both sides and 2^-28 left out
    assert (np.abs(g[rest] - want) <= 2.0 ** -24 * 2 * size + 2.0 ** -26 * most).all()
    alone = np.zeros((d, r), dtype=np.float32)
    alone[6] = W[6]
    assert np.array_equal(host(eng.keep8_gradient(eng.dev(alone), KX, KH))[6], g[6])


def test_gradient_is_the_losses_difference(eng, torch):
    rs = np.random.RandomState(3)
    d, r, n = 60, 9, 300
    X, H, W = rs.rand(d, n), rs.rand(r, n), rs.rand(d, r).astype(np.float32)
    KX, KH = eng.keep8(eng.dev(X)), eng.keep8(eng.dev(H))
    Xh, Hh = host(KX.expand()), host(KH.expand())
    g = host(eng.keep8_gradient(eng.dev(W), KX, KH))
    for i, k in ((0, 0), (59, 8), (30, 4)):
        e = np.zeros((d, r))
        e[i, k] = 1e-3
        diff = (lo.loss(W + e, Xh, Hh) - lo.loss(W - e, Xh, Hh)) / 2e-3          # quadratic: the central difference is exact
        assert abs(diff - g[i, k]) <= 1e-5 * np.abs(W).sum(1).max() * n


@pytest.mark.parametrize("n", [500, 5000])          # one run of groups, and several that are added up
def test_aggregates_in_place(eng, torch, n):
    from onmf_ontf_ndl_amd.engine import _ptr
    rs = np.random.RandomState(4)
    d, r = 200, 30
    X, H = eng.keep8(eng.dev(rs.rand(d, n))), eng.keep8(eng.dev(rs.rand(r, n)))
    A, B = eng.dev(rs.rand(r, r)), eng.dev(rs.rand(r, d))
    want = eng.keep8_aggregate(X, H, 0.25, A, B)
    nbytes = eng.lib.onmf_keep8_workspace(d, r, n, 0)
    assert (nbytes > 0) == (n > 1024)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=eng.device)
    rc = eng.lib.onmf_keep8_aggregate(eng.ctx, d, r, n, _ptr(X.codes), _ptr(X.scales), _ptr(H.codes), _ptr(H.scales), 0.25,
                                      _ptr(A), _ptr(B), _ptr(A), _ptr(B), _ptr(ws), nbytes, eng.stream())
    assert rc == 0 and torch.equal(A, want[0]) and torch.equal(B, want[1])
    for short, where in ((nbytes - 1, ws), (nbytes, None)) if nbytes else ():
        assert eng.lib.onmf_keep8_aggregate(eng.ctx, d, r, n, _ptr(X.codes), _ptr(X.scales), _ptr(H.codes), _ptr(H.scales), 0.25,
                                            _ptr(A), _ptr(B), _ptr(A), _ptr(B), _ptr(where), short, eng.stream()) == -1
    assert eng.lib.onmf_keep8(eng.ctx, d, n, _ptr(A), 0, n - 1, _ptr(X.codes), _ptr(X.scales), eng.stream()) == -1
    assert eng.lib.onmf_keep8(eng.ctx, d, n, _ptr(A), 5, n, _ptr(X.codes), _ptr(X.scales), eng.stream()) == -1


def test_gradient_refuses_results_over_its_input_and_a_workspace_askew(eng, torch):
    from onmf_ontf_ndl_amd.engine import _ptr
    rs = np.random.RandomState(1)
    d, r = 64, 16
    both = eng.dev(rs.rand(2 * d, r))
    for n in (50, 3000):
        X, H = eng.keep8(eng.dev(rs.rand(d, n))), eng.keep8(eng.dev(rs.rand(r, n)))
        need = eng.lib.onmf_keep8_workspace(d, r, n, 1)
        ws = torch.empty(need + 32, dtype=torch.uint8, device=eng.device)

        def call(dW, shift=0, nbytes=need):
            return eng.lib.onmf_keep8_gradient(eng.ctx, d, r, n, both.data_ptr(), _ptr(X.codes), _ptr(X.scales), _ptr(H.codes),
                                               _ptr(H.scales), dW, ws.data_ptr() + shift, nbytes, eng.stream())
        for row in (0, 1, d - 1):
            assert call(both[row].data_ptr()) == -1
        assert call(both[d:].data_ptr(), 8) == -1
        assert call(both[d:].data_ptr()) == 0
        assert torch.equal(both[d:], eng.keep8_gradient(both[:d], X, H))
        if need:
            assert call(both[d:].data_ptr(), 0, need - 1) == -1


# ------------------------------------------------------------------------------------------------- streams and graphs
def every_operator(eng, P, X, H, KX, KH, W, A, B):
    kept = eng.keep8(X)
    return [eng.dict4_correlate(P, X), eng.dict4_correlate(P, X[:, :3]), eng.dict4_product(P, H), eng.dict4_product(P, H[:, :1]),
            kept.codes, kept.scales, eng.keep8_expand(KX), *eng.keep8_aggregate(KX, KH, 0.5, A, B), eng.keep8_gradient(W, KX, KH),
            eng.dict4_product(P, H[:, :9]), eng.keep8_gradient(W, eng.keep8(X[:, :100]), eng.keep8(H[:, :100]))]


def state(eng, seed):
    rs = np.random.RandomState(seed)
    d, r, b = 1030, 70, 200
    W = eng.dev(rs.rand(d, r))
    X, H = eng.dev(rs.rand(d, b)), eng.dev(rs.rand(r, b))
    return (eng.dict4_pack(W, 64), X, H, eng.keep8(X), eng.keep8(H), W, eng.dev(rs.rand(r, r)), eng.dev(rs.rand(r, d)))


def test_results_are_the_same_every_time_and_on_two_streams_at_once(eng, torch):
    states = [state(eng, 1), state(eng, 2)]
    want = [every_operator(eng, *s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = [None, None]
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = every_operator(eng, *states[i])
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


def test_calls_from_several_threads(eng, torch):
    """The operators take nothing from the engine's context but its device: threads with streams of their own may call at
    once."""
    import threading
    states = [state(eng, 10 + i) for i in range(4)]
    want = [every_operator(eng, *s) for s in states]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = every_operator(eng, *states[i])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:                                  # (a thread's exception would be lost)
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong, wrong


def test_captured_calls_replay(eng, torch):
    """Two graphs of the same calls, replayed in turn with new inputs, eager work and synchronizations in between."""
    s = state(eng, 5)
    every_operator(eng, *s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(every_operator(eng, *s))
        graphs.append(g)
    for turn in range(6):
        s[1].copy_(torch.rand_like(s[1]))
        s[2].copy_(torch.rand_like(s[2]))
        s[5].copy_(torch.rand_like(s[5]))
        want = every_operator(eng, *s)
        torch.cuda.synchronize()
        graphs[turn % 2].replay()
        again = every_operator(eng, *s)
        torch.cuda.synchronize()
        for a, b, c in zip(outs[turn % 2], want, again):
            assert torch.equal(a, b) and torch.equal(a, c)


# ------------------------------------------------------------------------------------------------- the framework's paths
def test_coding_with_a_packed_dictionary_is_coding_with_what_it_stands_for(eng, torch):
    from onmf_ontf_ndl_amd import Online_NMF, pack_dictionary, update_code_within_radius
    rs = np.random.RandomState(6)
    W = rs.rand(200, 20)
    W /= np.linalg.norm(W, axis=0)
    X = eng.dev(rs.rand(200, 333))
    P = pack_dictionary(W, 32)
    nmf = Online_NMF(X, n_components=20, rng="device", seed=1)
    H0 = eng.dev(rs.rand(20, 333))
    a = update_code_within_radius(X, P, H0=H0)
    b = update_code_within_radius(X, P.unpack(), H0=H0)
    assert torch.equal(a, b)
    assert tuple(nmf.sparse_code(X, P).shape) == (20, 333)
    # one solve per column: W^T X from the codes differs from the float32 product by rounding
    h = eng.sparse_code_each(X, P, H0=H0, alpha=1, stopping_diff=0)
    k = eng.sparse_code_each(X, P.unpack(), H0=H0, alpha=1, stopping_diff=0)
    assert np.linalg.norm(host(h) - host(k)) <= 2e-5 * np.linalg.norm(host(k))
    assert torch.equal(eng.patch_product(P, h), eng.dict4_product(P, h))


def test_training_from_kept_columns_is_training_from_what_they_stand_for(eng, torch):
    from onmf_ontf_ndl_amd import Online_NMF, keep_columns
    rs = np.random.RandomState(7)
    K = keep_columns(rs.rand(64, 500))
    dense = K.expand()
    W0 = eng.dev(rs.rand(64, 8))
    agg = [eng.zeros(8, 8), eng.zeros(8, 64)]
    for subsample in (False, True):
        out = []
        for X in (K, dense):
            np.random.seed(11)
            nmf = Online_NMF(X, n_components=8, iterations=6, batch_size=50, ini_dict=W0, ini_agg=agg, subsample=subsample)
            W, sums, code = nmf.train_dict()
            out.append((W, *sums, code))
        assert all(torch.equal(a, b) for a, b in zip(*out))
        # the same object trained again, the other way round
        nmf.subsample = not subsample
        nmf.train_dict()
    nmf = Online_NMF(K, n_components=8, iterations=3, batch_size=50, subsample=True, rng="device")
    nmf.train_dict()
    nmf.subsample = False
    nmf.train_dict()
    H, (A, B), W = nmf.step(K, agg, W0, 3)
    assert tuple(H.shape) == (8, 500)


def test_images_reconstruct_with_a_packed_dictionary(eng, torch):
    from onmf_ontf_ndl_amd import pack_dictionary
    from onmf_ontf_ndl_amd.image_reconstruction import Image_Reconstructor
    rs = np.random.RandomState(8)
    img = rs.rand(24, 20, 3)
    rec = Image_Reconstructor(img, n_components=12, patch_size=4, is_color=True)
    rec.W = rs.rand(48, 12)
    P = pack_dictionary(rec.W, 32)
    out = []
    for W in (P, P.unpack().cpu().numpy().astype(np.float64)):
        rec.W = W
        np.random.seed(3)
        out.append(np.array(rec.reconstruct_image_color(img)))
    assert np.linalg.norm(out[0] - out[1]) <= 1e-4 * np.linalg.norm(out[1])
    grey = Image_Reconstructor(rs.rand(20, 20), n_components=6, patch_size=4, is_color=False, downscale_factor=1)
    W = rs.rand(16, 6)
    Pg = pack_dictionary(W, 32)
    out = []
    for W in (Pg, Pg.unpack().cpu().numpy().astype(np.float64)):
        grey.W = W
        np.random.seed(3)
        grey.reconstruct_image(grey.data, patch_size=4)
        out.append(np.array(grey.img_recons))
    assert np.linalg.norm(out[0] - out[1]) <= 1e-5 * np.linalg.norm(out[1])


def test_a_training_loop_on_low_bits(eng, torch):
    """Together as they would be used: columns and codes kept in 8 bits, aggregates from them, the dictionary pass,
    the dictionary packed in 4 bits and coded with again."""
    from onmf_ontf_ndl_amd import dictionary_gradient, keep_columns
    rs = np.random.RandomState(9)
    d, r, n = 144, 12, 2000
    W = eng.dev(rs.rand(d, r) / 12)
    X = eng.dev(np.maximum(rs.randn(d, r) + 0.3, 0) @ np.maximum(rs.randn(r, n), 0) / 12)
    K = keep_columns(X)
    A = B = None
    for t in range(1, 4):
        P = eng.dict4_pack(W, 64)
        C_ = eng.dict4_correlate(P, K.expand())
        H, _, _ = eng.sparse_code(K.expand(), P.unpack(), seed=t)
        KH = keep_columns(H)
        A, B = eng.keep8_aggregate(K, KH, 1.0 / t, A, B)
        dW = dictionary_gradient(W, K, KH)
        W = eng.update_dict(W, A, B)
        assert tuple(C_.shape) == tuple(H.shape) and tuple(dW.shape) == (d, r)
        assert all(bool(torch.isfinite(v).all()) for v in (C_, H, A, B, dW, W))
    Hh, Xh = host(KH.expand()), host(K.expand())
    want = lo.gradient(host(W), Xh, Hh)
    assert np.linalg.norm(host(dictionary_gradient(W, K, KH)) - want) <= 1e-5 * np.linalg.norm(want)
