"""The paged 4-bit decode step at the ends of its numbers' ranges, against
tests/ragged_ref.py."""
import numpy as np
import pytest
import torch

from tests import ragged_ref as ref
from tests.test_ragged_gpu import History, cu

pytestmark = pytest.mark.gpu

# heads and widths of every slab width, and heads that are not multiples of 32
SHAPES = [(1, 32), (2, 32), (1, 128), (2, 128), (4, 16), (8, 16), (4, 24), (16, 16)]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import ops as _ops

    assert _ops.read_status() >= 0
    return _ops


def store(h, kv):
    """Fill the stored positions of a History with the rows kv[b, i] [2D]."""
    n = h.n_pages * h.page
    rows, slots = [], []
    for b in range(h.B):
        i = np.arange(max(0, int(h.pos[b])))
        slots.append(h.table[b, i // h.page] * h.page + i % h.page)
        rows.append(kv[b, i])
    x = cu(np.concatenate(rows).astype(np.float32))
    assert len(x) <= n
    h.ops.kv4_write(x[:, : h.D], x[:, h.D:], cu(np.concatenate(slots).astype(np.int32)), h.pages)


def history(h, b, pages):
    """k and v [t+1, D] in 64 bits that sequence b's row sums over."""
    i = range(int(h.pos[b]) + 1)
    kv = np.stack([ref.unpack_row(pages[h.table[b, j // h.page], :, j % h.page]) for j in i])
    return kv[:, 0], kv[:, 1]


def check(h, spread):
    """The step's rows against the 64-bit ones.  A channel is off by at most
    2 (6 X + 8 + n) 2^-24 max |v| of the channel: X = `spread` bounds the
    exponents' size, each carries up to 6 roundings of X 2^-24, exp and sigmoid
    4 half steps, sums of n terms n half steps, in numerator and denominator."""
    pages, z, _ = h.expect()
    got = h.step().double().cpu().numpy()
    assert h.ops.read_status() == 0 and np.array_equal(h.pages.cpu().numpy(), pages)
    assert np.array_equal(np.isnan(got), np.isnan(z))
    for b in range(h.B):
        n = int(h.pos[b]) + 1
        top = np.abs(history(h, b, pages)[1]).max(0)
        tol = 2 * (6 * spread + 8 + n) * 2.0**-24 * top
        bad = ~(np.abs(got[b] - z[b]) <= tol) & ~np.isnan(z[b])
        assert not bad.any(), (b, np.argwhere(bad)[:4], got[b][bad][:4], z[b][bad][:4])
    return got


@pytest.mark.parametrize("H,hs", SHAPES)
@pytest.mark.parametrize("kind", ["sum", "weight", "shares"])
def test_aft_decode4_huge_values(ops, H, hs, kind):
    """Values of up to 9e36: neither the sum of many of them nor one of them
    times a weight above the reference may overflow, in a group beside
    ordinary ones."""
    rng = np.random.default_rng(H * hs)
    D, T = H * hs, 900 if kind == "shares" else 120
    w = np.zeros((H, T, T), np.float32)
    lens = [T - 1] if kind == "shares" else [T - 1, 70]
    kv = rng.standard_normal((len(lens), T, 2 * D))
    kv[..., :32] = 0
    if kind == "weight":  # 2^15.9 above the reference of a lane's first rows, which stays
        kv[..., :D] = 0
        w[:, :, 2::4] = w[:, :, 3::4] = 11.0
        kv[..., D: D + 32] = 9e33
    else:
        kv[..., D: D + 32] = 9e36 * np.where(rng.random((len(lens), T, 32)) < 0.2, -1.0, 1.0)
    h = History(ops, rng, len(lens), H, hs, T, 8, "f32", lens, w=w)
    store(h, kv)
    h.qkv[:, D: D + 32] = 0
    if kind == "weight":
        h.qkv[:, D: 2 * D] = 0
    got = check(h, 20)
    assert np.isfinite(got).all() and np.abs(got[0, :32]).max() > 1e33


LOWEST = float(np.finfo(np.float32).min)


@pytest.mark.parametrize("H,hs", SHAPES)
@pytest.mark.parametrize("kind", ["absorbed", "levels", "above", "cancel", "nan", "row", "below", "shares"])
def test_aft_decode4_huge_bias(ops, H, hs, kind):
    """Finite biases beside which fp32 holds nothing of a key, and keys that
    outweigh them all the same: exponents are the sums in 64 bits."""
    rng = np.random.default_rng(H * hs + 1)
    D, T = H * hs, 900 if kind == "shares" else 120
    lens = [T - 1] if kind == "shares" else [T - 1, 70]
    w = (0.5 * rng.standard_normal((H, T, T))).astype(np.float32)
    kv = rng.standard_normal((len(lens), T, 2 * D))
    key = kv[..., :32]  # one group, beside ordinary ones
    if kind == "absorbed":
        w[:] = 1e30
        kv[..., :32] = 2e36 * key
    elif kind in ("levels", "shares"):  # every position masked, some of them less
        w[:] = LOWEST
        w[:, :, 5::7] = -3e38
    elif kind == "above":
        w[:, :, ::3] = -1e30
        kv[..., :32] = 1e33 * key
    elif kind == "cancel":
        w[:, :, 5] = -2.0**119
        kv[:, 5, :32] = 2.0**119
    elif kind == "nan":
        w[:, :, 5] = LOWEST
        kv[0, 5, 3] = np.nan
    elif kind == "row":
        w[:] = -1e9
    elif kind == "below":
        w[:] = LOWEST
        kv[..., :32] = -9e36 * np.abs(key) / np.abs(key).max()
    h = History(ops, rng, len(lens), H, hs, T, 8, "f32", lens, w=w)
    store(h, kv)
    got = check(h, 20)
    if kind == "nan":
        assert np.isnan(got).sum() == 32
