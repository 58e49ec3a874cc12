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
