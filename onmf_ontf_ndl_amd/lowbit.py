"""What a dictionary held in 4 bits and columns held in 8 bits are to the host (the arithmetic is in
libonmf_hip.so, the formats are described in include/onmf_hip.h).

    P = pack_dictionary(W, group=64)         # W (d x r): an eighth of its room and a little
    H = nmf.sparse_code(X, P)                # wherever a dictionary is read
    P.unpack()                               # the float32 matrix it stands for

    K = keep_columns(X)                      # X (d x n): a quarter of its room
    Online_NMF(K, ...).train_dict()          # learn from columns that are held in 8 bits
    dW = dictionary_gradient(W, K, keep_columns(H))

The reference has neither: its dictionaries and patches are float64 arrays.
"""
from __future__ import annotations

__all__ = ["PackedDictionary", "KeptColumns", "pack_dictionary", "keep_columns", "dictionary_gradient", "GROUPS4",
           "GROUP8"]

GROUPS4 = (32, 64, 128)      # features that may share a scale in a 4-bit dictionary
GROUP8 = 128                 # columns that share a scale in an 8-bit store
MOST = 2 ** 31 - 1           # what the library's sizes hold
MOST8 = 2 ** 28              # columns of an 8-bit store


class PackedDictionary:
    """A d x r dictionary in 4 bits: ``codes`` uint8 (r, bytes of a padded atom), ``scales`` int32 (r, groups)."""

    __slots__ = ("codes", "scales", "d", "group")

    def __init__(self, codes, scales, d, group):
        d, group = int(d), int(group)
        if group not in GROUPS4:
            raise ValueError("a group is 32, 64 or 128 features, not %d" % group)
        groups = -(-d // group)
        shape = codes.shape
        if d <= 0 or len(shape) != 2 or shape[0] == 0 or shape[1] * 2 != groups * group or \
                scales.shape != (shape[0], groups):
            raise ValueError("codes must be (r, %d) and scales (r, %d) for d=%d, group=%d"
                             % (groups * group // 2, groups, d, group))
        if shape[0] > MOST or d > MOST:
            raise ValueError("a dictionary has at most 2^31 - 1 atoms and features")
        if str(codes.dtype) != "torch.uint8" or str(scales.dtype) != "torch.int32" or codes.device != scales.device:
            raise ValueError("codes must be uint8 and scales int32, on one device")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous")
        self.codes, self.scales, self.d, self.group = codes, scales, d, group

    @property
    def shape(self):
        return (self.d, self.codes.shape[0])

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + 4 * self.scales.numel()

    def unpack(self):
        """The float32 matrix (d x r) that this dictionary stands for."""
        from .engine import get_engine
        return get_engine(self.device).dict4_unpack(self)


class KeptColumns:
    """A d x n matrix in 8 bits: ``codes`` int8 (d, padded n), ``scales`` float32 (d, groups)."""

    __slots__ = ("codes", "scales", "n")

    def __init__(self, codes, scales, n):
        n = int(n)
        groups = -(-n // GROUP8)
        shape = codes.shape
        if n <= 0 or len(shape) != 2 or shape[0] == 0 or shape[1] != groups * GROUP8 or \
                scales.shape != (shape[0], groups):
            raise ValueError("codes must be (d, %d) and scales (d, %d) for n=%d" % (groups * GROUP8, groups, n))
        if shape[0] > MOST or n > MOST8:
            raise ValueError("a store has at most 2^31 - 1 rows and 2^28 columns")
        if str(codes.dtype) != "torch.int8" or str(scales.dtype) != "torch.float32" or codes.device != scales.device:
            raise ValueError("codes must be int8 and scales float32, on one device")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous")
        self.codes, self.scales, self.n = codes, scales, n

    @classmethod
    def _made(cls, codes, scales, n):
        """What the engine has just made itself: nothing to check (1.5 us of a short call's 15)."""
        K = object.__new__(cls)
        K.codes, K.scales, K.n = codes, scales, n
        return K

    @property
    def shape(self):
        return (self.codes.shape[0], self.n)

    @property
    def device(self):
        return self.codes.device

    def nbytes(self):
        return self.codes.numel() + 4 * self.scales.numel()

    def expand(self, idx=None):
        """The float32 columns this store stands for: all of them, or those at ``idx``."""
        from .engine import get_engine
        return get_engine(self.device).keep8_expand(self, idx)


def pack_dictionary(W, group=64, *, device=None):
    """W (d x r, NumPy or torch) in 4 bits on the GPU; every entry moves by at most half its group's scale."""
    from .engine import get_engine
    eng = get_engine(device)
    return eng.dict4_pack(eng.dev(W), group)


def keep_columns(X, *, device=None):
    """X (d x n, NumPy or torch) in 8 bits on the GPU; every entry moves by at most 1/254 of the largest among the
    128 columns of its row that share a scale."""
    from .engine import get_engine
    eng = get_engine(device)
    return eng.keep8(X if eng.is_columns(X) else eng.dev(X))


def dictionary_gradient(W, X, H, *, device=None):
    """The gradient of 1/2 |X - W H|^2 to W, W (H H^T) - X H^T, from kept X (d x n) and H (r x n)."""
    from .engine import get_engine
    from .onmf import _is_torch, _out
    eng = get_engine(X.device if device is None else device)
    return _out(eng.keep8_gradient(eng.dev(W), X, H), _is_torch(W))
