"""The drivers with a dictionary in 4 bits: what they make of it is what they make of the matrix it stands for."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch


def dense(P):
    return P.unpack().cpu().numpy().astype(np.float64)


def close(a, b):
    """Codes come from the same float32 matrix, or from products that differ by rounding; ten sweeps or a path of
    a dozen atoms pass that on, and W H adds its own."""
    a, b = np.asarray(a), np.asarray(b)
    return np.linalg.norm(a - b) <= 1e-4 * np.linalg.norm(b)


def test_tensor_images_reconstruct_with_a_packed_dictionary(torch):
    from onmf_ontf_ndl_amd import pack_dictionary
    from onmf_ontf_ndl_amd.image_reconstruction_tensor import Image_Reconstructor
    rs = np.random.RandomState(3)
    img = rs.rand(18, 21, 3)
    rec = Image_Reconstructor(img, n_components=12, patch_size=4, is_color=True)
    P = pack_dictionary(rs.rand(48, 12) / 4, 32)
    out = []
    for W in (P, dense(P)):
        rec.W = W
        out.append(np.array(rec.reconstruct_image_color(img)))
    assert out[0].shape == img.shape and np.abs(out[1]).max() > 0 and close(*out)
    grey = Image_Reconstructor(rs.rand(16, 15), n_components=6, patch_size=4, is_color=False, downscale_factor=1)
    P = pack_dictionary(2 * rs.rand(16, 6), 32)
    out = []
    for W in (P, dense(P)):
        grey.W = W
        code = grey.reconstruct_image(grey.data, patch_size=4)
        out.append((np.array(code), np.array(grey.img_recons)))
    assert np.abs(out[1][0]).max() > 0 and close(out[0][0], out[1][0]) and close(out[0][1], out[1][1])


@pytest.mark.parametrize("coder", ["lars", "cd"])
def test_networks_reconstruct_with_a_packed_dictionary(torch, coder):
    from onmf_ontf_ndl_amd import pack_dictionary
    from onmf_ontf_ndl_amd.network_reconstruction import Network_Reconstructor
    rs = np.random.RandomState(4)
    n = 40
    edges = np.array([(i, (i + 1) % n) for i in range(n)] + [(a, b) for a, b in rs.randint(n, size=(70, 2)) if a != b])
    P = pack_dictionary(rs.rand(36, 8), 32)
    out = []
    for W in (P, dense(P)):
        rec = Network_Reconstructor(edges, n_components=8, k1=0, k2=5, is_glauber_recons=False, seed=17)
        rec.W = W
        _, mean, count = rec.reconstruct_network(recons_iter=100, return_weights=True, coder=coder)
        out.append((np.array(mean), np.array(count)))
    assert np.array_equal(out[0][1], out[1][1]) and np.abs(out[1][0]).max() > 0 and close(out[0][0], out[1][0])


def test_steps_and_training_take_a_packed_dictionary(torch):
    from onmf_ontf_ndl_amd import Online_NMF, pack_dictionary
    from onmf_ontf_ndl_amd.onmf import surrogate_loss
    rs = np.random.RandomState(5)
    X = rs.rand(60, 300)
    P = pack_dictionary(rs.rand(60, 8) / 8, 32)
    agg = [rs.rand(8, 8), rs.rand(8, 60)]
    out = []
    for W in (P, dense(P)):
        np.random.seed(1)
        nmf = Online_NMF(X, n_components=8, iterations=4, ini_dict=W, ini_agg=agg)
        H, (A, B), W1 = nmf.step(X, agg, W, 2)
        W2, (A2, B2), _ = nmf.train_dict()
        out.append((H, A, B, W1, W2, A2, B2, surrogate_loss(W, A, B)))
    assert all(np.array_equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("hug", [False, True])
def test_threads_that_find_a_step_not_waited_for(torch, hug):
    """Four threads, streams of their own, call at once while a deferred step's verdicts have not been looked at - with a
    tolerance that no sweep's bounds decide its solve is run again there: once, and to the same bits."""
    import threading
    from onmf_ontf_ndl_amd import _lib
    from onmf_ontf_ndl_amd.engine import get_engine
    eng = get_engine()
    d, r, b = 200, 64, 3000
    g = torch.Generator(device=eng.device).manual_seed(3)
    X, W = torch.rand(d, b, device=eng.device, generator=g), torch.rand(d, r, device=eng.device, generator=g)
    W = W / torch.linalg.norm(W, dim=0).clamp(min=1)
    Y = torch.rand(d, 300, device=eng.device, generator=g)
    P = eng.dict4_pack(W.contiguous(), 64)
    A, B = eng.zeros(r, r), eng.zeros(r, d)
    tol = 0.01
    if hug:
        eng.set_option(_lib.OPT_EXACT_STOP, 1)
        _, _, dist = eng.sparse_code(X, W, seed=5, stopping_diff=0.0)
        eng.set_option(_lib.OPT_EXACT_STOP, 0)
        tol = float(dist[5] * 0.995)
    def step(defer):
        return eng.step(X, A, B, None, W, 0.5, seed=5, stopping_diff=tol, defer=defer)
    want = step(False)
    corr, kept = eng.dict4_correlate(P, Y), eng.keep8(Y)
    torch.cuda.synchronize()
    wrong = []

    def work(start):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(3):
                    c, k = eng.dict4_correlate(P, Y), eng.keep8(Y)
                    stream.synchronize()
                    if not (torch.equal(c, corr) and torch.equal(k.codes, kept.codes)):
                        wrong.append("a result")
                try:
                    eng.dict4_correlate(P, Y[:5])
                    wrong.append("no refusal")
                except ValueError:
                    pass
                if eng.lib.onmf_keep8(eng.ctx, 1, 1, None, 0, 1, None, None, None) != -1 or not eng.lib.onmf_last_error(eng.ctx):
                    wrong.append("no error")
        except Exception as e:                                  # (a thread's exception would be lost)
            wrong.append(e)
    eng.set_option(_lib.OPT_DEFER_VERDICT, 1)
    try:
        for _ in range(4):
            before = eng.counters()
            got = step(True)
            start = threading.Barrier(4)
            threads = [threading.Thread(target=work, args=(start,)) for _ in range(4)]
            for th in threads:
                th.start()
            for th in threads:
                th.join()
            eng.settle()
            torch.cuda.synchronize()
            after = eng.counters()
            assert not wrong, wrong
            assert after["sweeps_total"] - before["sweeps_total"] == want[5]
            assert all(torch.equal(got[i], want[i]) for i in (0, 1, 2, 4))
    finally:
        eng.set_option(_lib.OPT_DEFER_VERDICT, 0)
