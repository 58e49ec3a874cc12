"""The framework's paths that take columns in 8 bits and dictionaries in 4, without a GPU: what they hand to the engine."""
import numpy as np
import pytest
import torch

from onmf_ontf_ndl_amd import KeptColumns, Online_NMF, Online_NTF, PackedDictionary
from onmf_ontf_ndl_amd import onmf as onmf_module
from onmf_ontf_ndl_amd import ontf as ontf_module


class HostEngine:
    """An engine on the CPU for what the paths call: it refuses what the real one refuses, and keeps the calls."""
    device = torch.device("cpu")

    def __init__(self):
        self.torch = torch
        self.calls = []

    def dev(self, a, dtype=None):
        if isinstance(a, (KeptColumns, PackedDictionary)):
            raise TypeError("dev: not an array: %s" % type(a).__name__)
        return torch.as_tensor(np.asarray(a)).to(dtype or torch.float32).contiguous()

    def zeros(self, *shape):
        return torch.zeros(*shape)

    def numpy_rand(self, *shape):
        return torch.from_numpy(np.random.rand(*shape)).float()

    def next_seed(self, base=0):
        return base

    def keep8_expand(self, K, idx=None):
        if not isinstance(K, KeptColumns):
            raise ValueError("keep8_expand needs a KeptColumns, not %s" % type(K).__name__)
        self.calls.append("expand all" if idx is None else "expand some")
        X = K.codes[:, :K.n].float() * K.scales.repeat_interleave(128, dim=1)[:, :K.n]
        return X if idx is None else X[:, torch.as_tensor(idx)]

    def dict4_unpack(self, P):
        self.calls.append("unpack")
        return torch.full(P.shape, 0.5)

    def surrogate_loss(self, W, A, B, C):
        assert isinstance(W, torch.Tensor)
        return float(W.sum())

    def sparse_code_lars(self, X, W, alpha=2.0, max_iter=1000):
        assert isinstance(W, torch.Tensor)
        return torch.ones(W.shape[1], X.shape[1])

    def sparse_code_each(self, X, W, H0=None, want_sweeps=False, **kw):
        assert isinstance(W, (torch.Tensor, PackedDictionary))
        self.calls.append("each from " + type(W).__name__)
        return torch.ones(W.shape[1], X.shape[1]), torch.ones(X.shape[1], dtype=torch.int32)

    def ntf_step(self, X, A, B, W, w, **kw):
        assert isinstance(W, torch.Tensor)
        return torch.ones(W.shape[1], X.shape[1]), A, B, W

    def gather_columns(self, X, idx):
        if not isinstance(X, torch.Tensor):
            raise ValueError("gather_columns needs a tensor, not %s" % type(X).__name__)
        self.calls.append("gather")
        return X[:, torch.as_tensor(idx)]

    def step(self, X, A, B, C, W, w, **kw):
        assert isinstance(X, torch.Tensor) and isinstance(W, torch.Tensor)
        self.calls.append("step")
        H = torch.ones(W.shape[1], X.shape[1]) * X.mean()
        return H, A + H @ H.t(), B + H @ X.t(), C, W + 1, 1, None

    def code_accumulate(self, code, idx, H):
        if idx is None:
            code += H
        else:
            code.index_add_(1, torch.as_tensor(idx), H)


@pytest.fixture
def engine(monkeypatch):
    eng = HostEngine()
    for module in (onmf_module, ontf_module):
        monkeypatch.setattr(module, "get_engine", lambda device=None: eng)
    return eng


def kept(d=4, n=200):
    g = torch.Generator().manual_seed(d + n)
    groups = -(-n // 128)
    codes = torch.randint(-127, 128, (d, groups * 128), generator=g, dtype=torch.int8)
    codes[:, n:] = 0
    return KeptColumns(codes, torch.rand(d, groups, generator=g), n)


@pytest.mark.parametrize("order", [(False, True), (True, False), (False, True, False), (True, False, True)])
def test_kept_columns_are_trained_on_again_with_and_without_subsampling(engine, order):
    """One object, trained several times with `subsample` turned on and off in between: each time as a fresh object that
    starts from the same dictionary."""
    K = kept()
    nmf = Online_NMF(K, n_components=3, iterations=4, batch_size=20)
    for subsample in order:
        nmf.subsample = subsample
        engine.calls.clear()
        np.random.seed(5)
        W, agg, _ = nmf.train_dict()
        calls = list(engine.calls)
        fresh = Online_NMF(K, n_components=3, iterations=4, batch_size=20, subsample=subsample)
        np.random.seed(5)
        W1, agg1, _ = fresh.train_dict()
        assert torch.equal(W, W1) and all(torch.equal(a, b) for a, b in zip(agg, agg1))
        assert ("expand some" in calls) == subsample and "gather" not in calls


def packed(d=4, r=3):
    return PackedDictionary(torch.zeros(r, 16, dtype=torch.uint8), torch.zeros(r, 1, dtype=torch.int32), d, 32)


def test_a_step_reads_a_packed_dictionary(engine):
    X, agg = np.random.RandomState(0).rand(4, 10), [np.zeros((3, 3)), np.zeros((3, 4))]
    H, (A, B), W = Online_NMF(X, n_components=3).step(X, agg, packed(), 1)
    assert H.shape == (3, 10) and A.shape == (3, 3) and B.shape == (3, 4)
    assert isinstance(W, np.ndarray) and W.shape == (4, 3)


def test_training_starts_from_a_packed_dictionary(engine):
    X, P = np.random.RandomState(0).rand(4, 10), packed()
    agg = [np.zeros((3, 3)), np.zeros((3, 4))]
    W, _, _ = Online_NMF(X, n_components=3, iterations=3, ini_dict=P, ini_agg=agg).train_dict()
    dense = Online_NMF(X, n_components=3, iterations=3, ini_dict=np.full((4, 3), 0.5), ini_agg=agg).train_dict()[0]
    assert np.array_equal(W, dense) and engine.calls.count("unpack") == 1


def test_the_loss_reads_a_packed_dictionary(engine):
    assert onmf_module.surrogate_loss(packed(), np.zeros((3, 3)), np.zeros((3, 4))) == 6.0


@pytest.mark.parametrize("coder", ["lars", "cd"])
def test_tensor_columns_are_coded_with_a_packed_dictionary(engine, coder):
    ntf = Online_NTF(np.zeros((2, 2, 5)), n_components=3, coder=coder)
    H = ntf.joint_sparse_code_tensor(np.zeros((4, 5)), packed())
    assert H.shape == (5, 3)
    assert engine.calls == (["unpack"] if coder == "lars" else ["each from PackedDictionary"])


def test_a_tensor_step_reads_a_packed_dictionary(engine):
    ntf = Online_NTF(np.zeros((2, 2, 5)), n_components=3)
    H, A, B, W = ntf.step(np.zeros((4, 5)), np.zeros((3, 3)), np.zeros((3, 4)), packed(), 1)
    assert H.shape == (5, 3) and isinstance(W, np.ndarray) and W.shape == (4, 3)
