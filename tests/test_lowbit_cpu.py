"""Dictionaries in 4 bits and columns in 8, without a GPU: the oracle's own properties, what the containers and the
host side refuse, and the sizes the library asks for."""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as lo

from onmf_ontf_ndl_amd import KeptColumns, PackedDictionary, _lib
from onmf_ontf_ndl_amd.engine import Engine


# ------------------------------------------------------------------------------------------------- the format
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind", ["plain", "zeros", "signed", "far", "constant", "tiny", "huge"])
def test_an_entry_moves_by_at_most_half_its_scale(group, kind):
    rs = np.random.RandomState(group)
    W = rs.rand(2 * group + 5, 7).astype(np.float32)
    if kind == "zeros":
        W = np.maximum(W - 0.6, 0).astype(np.float32)
    elif kind == "signed":
        W = (W - 0.5).astype(np.float32)
    elif kind == "far":
        W = (W * 1e-3 + 1).astype(np.float32)
    elif kind == "constant":
        W[:] = np.float32(0.3)
    elif kind == "tiny":
        W = (W * 1e-30).astype(np.float32)
    elif kind == "huge":
        W = (W * 1e35).astype(np.float32)
    q, z, s = lo.pack4(W, group)
    assert q.min() >= 0 and q.max() <= 15 and np.abs(z).max() <= 255
    assert np.abs(q.reshape(7, -1, group) + z[:, :, None]).max() <= 255
    back = lo.values4(q, z, s, W.shape[0])
    half = np.repeat(s, group, axis=1)[:, :W.shape[0]].T / 2
    assert (np.abs(back - W) <= half * (1 + 1e-12)).all()
    if kind == "zeros":
        assert (back[W == 0] == 0).all()                     # zeros stay zeros
    codes, scales = lo.to_codes4(q, z, s)
    assert codes.shape == (7, 3 * group // 2) and scales.shape == (7, 3)
    assert ((scales.view(np.uint32) & 0xFFFF0000).view(np.float32) == s).all()       # a scale is a bfloat16


def test_bf16_up_is_the_next_bfloat16():
    for v in (1.0, 1.0 + 2.0 ** -20, 0.1, 3.3e38, 1e-38, 1e-45, 0.99999999, 2.0 ** -126, 2.0 ** -130):
        u = lo.bf16_up(v)
        assert u >= v
        bits = int(np.float32(u).view(np.uint32))
        assert float(np.float32(u)) == u and bits & 0xFFFF == 0
        below = float(np.uint32(bits - 0x10000).view(np.float32))
        assert below < v


def test_kept_columns_move_by_at_most_half_their_scale():
    rs = np.random.RandomState(1)
    X = (rs.rand(5, 300) - 0.3).astype(np.float32)
    X[2, :128] = 0
    q, s = lo.keep8(X)
    assert np.abs(q).max() == 127
    step = np.repeat(s, 128, axis=1)[:, :300]
    assert (np.abs(lo.values8(q, s, 300) - X) <= step / 2 * (1 + 1e-12)).all()
    assert s[2, 0] == 0


def test_gradient_is_the_losses_difference():
    rs = np.random.RandomState(2)
    W, H, X = rs.rand(6, 3), rs.rand(3, 9), rs.rand(6, 9)
    g = lo.gradient(W, X, H)
    for i, k in ((0, 0), (5, 2), (3, 1)):
        e = np.zeros_like(W)
        e[i, k] = 1e-4
        assert abs((lo.loss(W + e, X, H) - lo.loss(W - e, X, H)) / 2e-4 - g[i, k]) < 1e-8


# ------------------------------------------------------------------------------------------------- refusals
def packed(d=100, r=5, group=64):
    groups = -(-d // group)
    return PackedDictionary(torch.zeros(r, groups * group // 2, dtype=torch.uint8),
                            torch.zeros(r, groups, dtype=torch.int32), d, group)


def kept(d=4, n=200):
    groups = -(-n // 128)
    return KeptColumns(torch.zeros(d, groups * 128, dtype=torch.int8), torch.zeros(d, groups), n)


def test_containers_know_their_shapes():
    P, K = packed(), kept()
    assert P.shape == (100, 5) and P.nbytes() == 5 * 64 + 4 * 10 and P.device.type == "cpu"
    assert K.shape == (4, 200) and K.nbytes() == 4 * 256 + 4 * 8


@pytest.mark.parametrize("change", [dict(d=0), dict(d=200), dict(group=48), dict(codes=torch.zeros(5, 63, dtype=torch.uint8)),
                                    dict(codes=torch.zeros(5, 64, dtype=torch.int8)), dict(scales=torch.zeros(5, 2)),
                                    dict(scales=torch.zeros(4, 2, dtype=torch.int32)),
                                    dict(codes=torch.zeros(0, 64, dtype=torch.uint8), scales=torch.zeros(0, 2, dtype=torch.int32)),
                                    dict(codes=torch.zeros(64, 5, dtype=torch.uint8).t()),
                                    dict(codes=torch.zeros(5 * 64, dtype=torch.uint8))])
def test_packed_dictionary_refuses(change):
    P = packed()
    args = dict(codes=P.codes, scales=P.scales, d=100, group=64)
    PackedDictionary(**args)
    args.update(change)
    with pytest.raises(ValueError):
        PackedDictionary(**args)


@pytest.mark.parametrize("change", [dict(n=0), dict(n=257), dict(n=128), dict(codes=torch.zeros(4, 256)),
                                    dict(scales=torch.zeros(4, 2, dtype=torch.float64)), dict(scales=torch.zeros(4, 1)),
                                    dict(codes=torch.zeros(256, 4, dtype=torch.int8).t()), dict(scales=torch.zeros(2, 4).t())])
def test_kept_columns_refuse(change):
    K = kept()
    args = dict(codes=K.codes, scales=K.scales, n=200)
    KeptColumns(**args)
    args.update(change)
    with pytest.raises(ValueError):
        KeptColumns(**args)


class NoLibrary:
    """Nothing may reach the library in these tests."""
    def __getattr__(self, name):
        raise AssertionError("the library was called: " + name)


@pytest.fixture
def host_side():
    eng = Engine.__new__(Engine)
    eng.torch, eng.lib, eng.ctx, eng.device, eng.index = torch, NoLibrary(), None, torch.device("cpu"), 0
    return eng


def test_products_refuse_before_the_library_is_called(host_side):
    eng, P, K = host_side, packed(), kept()
    X = torch.zeros(100, 3)
    for bad in (torch.zeros(99, 3), torch.zeros(100), torch.zeros(100, 0), torch.zeros(100, 3, dtype=torch.float64),
                torch.zeros(100, 3, dtype=torch.float16), np.zeros((100, 3), dtype=np.float32),
                torch.zeros(100, 3, device="meta"), torch.zeros(1, 100, 3)):
        with pytest.raises(ValueError):
            eng.dict4_correlate(P, bad)
    for bad in (torch.zeros(100, 3), torch.zeros(5, 0), torch.zeros(5, 3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            eng.dict4_product(P, bad)
    for what in (eng.dict4_correlate, eng.dict4_product):
        with pytest.raises(ValueError):
            what(X, X)
        with pytest.raises(ValueError):
            what(K, X)
    with pytest.raises(ValueError):
        eng.dict4_unpack(K)
    for group in (0, 16, 48, 256):
        with pytest.raises(ValueError):
            eng.dict4_pack(X, group)
    for bad in (torch.zeros(0, 3), torch.zeros(3), torch.zeros(3, 4).t(), torch.zeros(3, 4, dtype=torch.bfloat16),
                np.zeros((3, 4), dtype=np.float32)):
        with pytest.raises(ValueError):
            eng.dict4_pack(bad)


def test_stores_refuse_before_the_library_is_called(host_side):
    eng, K = host_side, kept()
    for bad in (torch.zeros(4, 0), torch.zeros(0, 4), torch.zeros(4), torch.zeros(4, 4, dtype=torch.int8)):
        with pytest.raises(ValueError):
            eng.keep8(bad)
    with pytest.raises(ValueError):
        eng.keep8_expand(packed())
    for idx in ([], [[0, 1]]):
        with pytest.raises(ValueError):
            eng.keep8_expand(K, np.array(idx, dtype=np.int64))
    for idx in ([0, 200], [-201]):
        with pytest.raises(IndexError):
            eng.keep8_expand(K, np.array(idx))
    H = kept(3, 200)
    with pytest.raises(ValueError):
        eng.keep8_aggregate(K, kept(3, 201), 0.5)
    with pytest.raises(ValueError):
        eng.keep8_aggregate(K, torch.zeros(3, 200), 0.5)
    for A, B in ((torch.zeros(4, 4), None), (None, torch.zeros(4, 3)), (torch.zeros(3, 3, dtype=torch.float64), None)):
        with pytest.raises(ValueError):
            eng.keep8_aggregate(K, H, 0.5, A, B)
    for W in (torch.zeros(3, 4), torch.zeros(3, 4).t(), torch.zeros(4, 3, dtype=torch.bfloat16)):
        if tuple(W.shape) == (4, 3) and W.dtype is torch.float32 and W.is_contiguous():
            continue
        with pytest.raises(ValueError):
            eng.keep8_gradient(W, K, H)


def test_sizes_that_no_int_holds_are_refused(host_side):
    """The library counts in ints: a view of more columns, rows or atoms than one holds (it takes no memory) is refused here
    and not cut off on the way."""
    from onmf_ontf_ndl_amd import KeptColumns, PackedDictionary
    eng, one = host_side, torch.zeros(1, 1)
    far = 2 ** 32 + 5
    P = packed()
    for bad in (one.expand(1, far), one.expand(far, 1), one.bfloat16().expand(1, far)):
        with pytest.raises(ValueError):
            eng.keep8(bad)
    with pytest.raises(ValueError):
        eng.dict4_correlate(P, one.expand(P.shape[0], far))
    with pytest.raises(ValueError):
        eng.dict4_product(P, one.expand(P.shape[1], far))
    for bad in (one.expand(1, far), one.expand(far, 1)):
        with pytest.raises(ValueError):
            eng.dict4_pack(bad)
    with pytest.raises(ValueError):
        eng.keep8_expand(kept(), torch.zeros(1, dtype=torch.int64).expand(far))
    with pytest.raises(ValueError):
        KeptColumns(torch.zeros(1, 1, dtype=torch.int8).expand(1, 2 ** 28 + 128), torch.zeros(1, 1).expand(1, 2 ** 21 + 1), 2 ** 28 + 1)
    with pytest.raises(ValueError):
        KeptColumns(torch.zeros(1, 1, dtype=torch.int8).expand(far, 128), torch.zeros(1, 1).expand(far, 1), 3)
    with pytest.raises(ValueError):
        PackedDictionary(torch.zeros(1, 1, dtype=torch.uint8).expand(far, 16), torch.zeros(1, 1, dtype=torch.int32).expand(far, 1), 3, 32)


# ------------------------------------------------------------------------------------------------- the library's host side
def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    assert lib.onmf_dict4_pack(None, 8, 8, 64, None, None, None, None) == -1
    assert lib.onmf_dict4_correlate(None, 8, 8, 1, 64, None, None, None, 0, 1, None, None, 0, None) == -1
    assert lib.onmf_keep8(None, 8, 8, None, 0, 8, None, None, None) == -1
    assert lib.onmf_keep8_gradient(None, 8, 8, 8, None, None, None, None, None, None, None, 0, None) == -1


def test_workspaces_are_bounded():
    """A call never asks for more than a few times its output or a fixed amount: 768 slabs of one output tile."""
    lib = _lib.load()
    for which in (0, 1):
        for d in (1, 31, 441, 4096, 8192):
            for r in (1, 25, 256, 32768):
                for b in (1, 3, 8, 9, 64, 1000, 65536):
                    # the weights in bfloat16 (two pieces) with their scales, and 1024 pieces of a result's tile
                    # of 256 x 128 - or, a column or a few of them, of 512 features
                    n = lib.onmf_dict4_workspace(which, d, r, b, 64)
                    laid = (4 * r + r // 8 + 128) * (d + 128) if b > 8 else 0
                    assert n % 4 == 0 and n <= laid + 1024 * 256 * 128 * 4
        assert lib.onmf_dict4_workspace(which, 0, 4, 4, 64) == 0
        assert lib.onmf_dict4_workspace(which, 4, 4, 4, 48) == 0
    for d, r, n in ((441, 25, 128), (8192, 1024, 1), (4096, 300, 100)):     # by way of the residual: none
        assert lib.onmf_keep8_workspace(d, r, n, 1) == 0
    # a slab for each run of groups (512 workgroups of 256 x 128 results at most), and the sums as doubles
    for d, r, n in ((441, 25, 1000), (1024, 256, 65536), (8192, 1024, 129), (60000, 20, 100), (60, 1024, 100)):
        plain, with_gradient = lib.onmf_keep8_workspace(d, r, n, 0), lib.onmf_keep8_workspace(d, r, n, 1)
        sums, digits = 8 * r * (r + d), 4 * (d + r) * (r + 63) + 8 * (d + r)
        assert plain <= 512 * 256 * 128 * 4 and plain + sums <= with_gradient <= plain + sums + 512 + digits
    assert lib.onmf_keep8_workspace(0, 4, 4, 0) == 0


def test_workspaces_of_sizes_that_the_calls_refuse():
    """The largest ints go through no arithmetic that could overflow."""
    lib = _lib.load()
    large = 2 ** 31 - 1
    for which in (0, 1):
        assert lib.onmf_dict4_workspace(which, 2 ** 18 + 1, 64, 64, 64) == 0
        assert lib.onmf_dict4_workspace(which, 64, large, 64, 64) == 0
        assert lib.onmf_dict4_workspace(which, 64, 64, large, 64) == 0
        assert lib.onmf_keep8_workspace(large, 64, 4096, which) == 0
        assert lib.onmf_keep8_workspace(64, large, 4096, which) == 0
        assert lib.onmf_keep8_workspace(64, 64, 2 ** 28 + 1, which) == 0
        assert 0 < lib.onmf_dict4_workspace(which, 2 ** 18, 2 ** 18, 2 ** 18, 32) < 2 ** 62
        # (sums of one run go straight to A and B: no workspace)
        assert (which == 1) <= lib.onmf_keep8_workspace(2 ** 18, 2 ** 18, 2 ** 28, which) < 2 ** 62
    assert lib.onmf_keep8_workspace(2 ** 18 + 1, 64, 4096, 1) == 0 and lib.onmf_keep8_workspace(64, 2 ** 18 + 1, 4096, 1) == 0
