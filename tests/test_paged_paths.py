"""Paths of the paged-serving kernels that the operators' own tests do not choose: sampling with every split
of a row and slices up to the largest, single tokens in the order of their lengths, and both sides of the
bounds between the attention kernels."""
from __future__ import annotations

import sys

import numpy as np
import pytest

from conftest import REPO
from oracle import paged_oracle as PO

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


def test_device_tables_are_the_generators():
    sys.path.insert(0, str(REPO / "llaccel_b200" / "csrc"))
    import gen_luts
    assert (REPO / "llaccel_b200" / "csrc" / "device_luts.h").read_text() == gen_luts.render_device()


@pytest.fixture(scope="module")
def calls():
    from llaccel_b200 import build
    build.build()
    import test_paged_ops
    return test_paged_ops


# rows and vocabulary; CTAs a row and vectors a CTA, as launch_sample chooses them
SPLITS = [(300, 51180, 1, 6399), (300, 102380, 2, 6400), (80, 204780, 4, 6400), (128, 151936, 4, 4749), (300, 262144, 8, 4097),
          (9, 262144, 16, 2049)]


@gpu
@pytest.mark.parametrize("R,V,C,slice_", SPLITS)
def test_sample_splits(calls, R, V, C, slice_):
    """Eight rows with settings of their own, again and again from row starts of every alignment."""
    vecs, got = (V + 14) // 8, 1
    while got < 16 and ((R * got < 296 and vecs > got * 512) or vecs > got * 6400):
        got *= 2
    assert (got, -(-vecs // got)) == (C, slice_)
    rng = np.random.default_rng(V + R)
    x = calls.logits(rng, 8, V, -10)
    x[3] = 7  # flat
    x[4] = rng.integers(-40, 40, V)  # many ties
    x[5, [0, V // 2, V - 1]] = 32767
    t = np.float32([1.0, 0.0, 0.7, 1.0, 1.0, 3.0, 2.0, 1.5])
    k = np.int32([0, 0, 50, 0, 300, 0, 5000, 0])
    p = np.float32([0.95, 1.0, 0.9, 0.5, 1.0, 0.999, 0.8, 1.0])
    m = np.float32([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.02])
    u = rng.random(8)
    u[3], u[6] = 1 - 2.0 ** -53, 0.0
    want = [PO.sample(x[i], float(u[i]), -10, t[i].item(), k[i].item(), p[i].item(), m[i].item()) for i in range(8)]
    pick = np.arange(R) % 8
    wide = torch.zeros((R, V + 3), dtype=torch.int16, device="cuda")
    wide[:, :V] = calls.dev(x)[calls.dev(pick)]
    col = lambda a: calls.dev(a[pick])  # noqa: E731
    token, prob = calls.sampling.sample(wide, col(u), exponent=-10, vocab=V, temperature=col(t), top_k=col(k), top_p=col(p), min_p=col(m))
    assert token.cpu().tolist() == [want[i][0] for i in pick]
    # one double division, rounded to float32: half a step, relative to the value
    ref = np.array([want[i][1] for i in pick])
    assert (np.abs(prob.cpu().numpy() - ref) <= ref * (np.finfo(np.float32).eps / 2 + 2.0 ** -52)).all()


@gpu
@pytest.mark.parametrize("n", [65, 200, 512, 513])
@pytest.mark.parametrize("D", [64, 128])
def test_single_tokens_in_the_order_of_their_lengths(calls, n, D):
    """More clusters than a wave holds: the longest sequences start first (up to 512 of them).  Equal lengths,
    sequences without rows, slots in any order."""
    rng = np.random.default_rng(n + D)
    lens = rng.choice([1, 5, 16, 17, 64, 90, 90, 90, 130, 300], n)
    rows = (rng.random(n) > 0.1).astype(int)
    rows[0] = 1
    assert calls.attention_case(rng, 8, 8, D, 16, rows.tolist(), lens.tolist(), slots=rng.permutation(n + 5)[:n].tolist(), pad=2) == 0


@gpu
@pytest.mark.parametrize("H,Hkv,rows", [(2, 2, [32, 1]), (2, 2, [33, 1]), (16, 2, [4, 1]), (16, 2, [5, 1]), (32, 1, [1, 1]), (33, 1, [1, 1])])
@pytest.mark.parametrize("D", [64, 128])
def test_pairs_on_both_sides_of_the_few_row_kernels_bound(calls, H, Hkv, rows, D):
    rng = np.random.default_rng(H + rows[0] + D)
    assert calls.attention_case(rng, H, Hkv, D, 32, rows, [333, 1000]) == 0


@gpu
@pytest.mark.parametrize("D,H,most", [(128, 8, 80000), (128, 8, 100000), (128, 4, 170000), (128, 4, 200000), (64, 8, 90000), (64, 8, 110000)])
def test_lengths_on_both_sides_of_the_few_row_kernels_bound(calls, D, H, most):
    """A launch's bound beyond what a cluster's shared memory holds, over short contexts and over long ones."""
    rng = np.random.default_rng(most)
    assert calls.attention_case(rng, H, 1, D, 64, [1, 0, 1], [1000, most, 64], max_len=most) == 0
    assert calls.attention_case(rng, H, 1, D, 64, [1], [most - 7], max_len=most) == 0
