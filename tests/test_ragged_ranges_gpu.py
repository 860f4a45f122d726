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


@pytest.mark.parametrize("H,hs,T,page,B,odd", [
    (1, 64, 5000, 32, 1, 0), (1, 64, 4097, 16, 2, 1), (2, 128, 2000, 16, 3, 0), (8, 16, 1500, 8, 2, 1),
    (1, 32, 3000, 64, 40, 0), (16, 16, 300, 8, 150, 1), (5, 64, 400, 128, 90, 0), (1, 128, 700, 256, 500, 0),
    (2, 48, 2500, 64, 1, 0)])
def test_aft_decode4_every_position_counts_once(ops, H, hs, T, page, B, odd):
    """Keys of zero, biases of 0 or -inf and values that are whole numbers
    0..15 make every weight 0 or 1 and both sums whole numbers below 2^24, so a
    row is their quotient, rounded once (and halved by the gate): a position
    that is lost or counted twice at a border of shares, blocks or pages is off
    by 1 / (t + 1), far above that."""
    rng = np.random.default_rng(T + B)
    D, width = H * hs, -(-T // page)
    v = rng.integers(0, 16, (B, T, D)).astype(np.float32)
    v[..., ::32], v[..., 1::32] = 0, 15  # a group's low is 0, its step 1
    keep = rng.random((H, T)) < 0.7
    n_pages = B * width + 2
    table = rng.permutation(n_pages)[: B * width].reshape(B, width).astype(np.int32)
    pages = ops.kv4_pages(n_pages, page, D)
    i = np.arange(T)
    slots = cu((table[:, i // page] * page + i % page).reshape(-1).astype(np.int32))
    flat = torch.from_numpy(v.reshape(B * T, D)).cuda()
    ops.kv4_write(torch.zeros_like(flat), flat, slots, pages)
    w = torch.zeros(H, T, T + odd, device="cuda")[:, :, odd:]
    w.masked_fill_(cu(~keep)[:, None], float("-inf"))
    on = np.repeat(keep, hs, 0).T  # [T, D]
    ws, qkv, t_table = ops.aft_decode4_workspace(B, D), torch.zeros(B, 3 * D, device="cuda"), cu(table)
    num = np.cumsum(np.where(on, v, 0), 1, dtype=np.float32)  # whole numbers: exact
    den = np.cumsum(on, 0, dtype=np.float32)
    assert num.max() < 2**24
    rows = np.arange(B)
    for k in range(25):
        pos = rng.integers(0, T, B) if k % 3 else np.minimum(T - 1, T - 1 - k + rng.integers(0, 2, B))
        if B > 2:
            pos[rng.random(B) < 0.1] = rng.integers(0, 20)
        qkv[:, 2 * D:] = cu(v[rows, pos])
        got = ops.aft_decode4(qkv, w, pages, t_table, cu(pos.astype(np.int32)), ws).cpu().numpy()
        n, d = num[rows, pos], den[pos]
        want = 0.5 * np.where(d > 0, n / np.maximum(d, 1), 0)
        assert np.all(np.abs(got - want) <= 2.0**-23 * want), (k, np.argwhere(np.abs(got - want) > 2.0**-23 * want)[:4])
    assert ops.read_status() == 0


@pytest.mark.parametrize("H,hs", SHAPES)
@pytest.mark.parametrize("T", [200, 1100])
def test_aft_decode4_keys_far_apart(ops, H, hs, T):
    """Channels of a group whose keys lie hundreds apart are summed again,
    whatever the slab's width, by a CTA alone or the last of several."""
    rng = np.random.default_rng(H * hs + T)
    D = H * hs
    h = History(ops, rng, 2, H, hs, T, 8, "f32", [T - 1, T // 2])
    kv = rng.standard_normal((2, T, 2 * D))
    kv[..., :D] = 40 * kv[..., :D] + 150 * rng.standard_normal(D)
    store(h, kv)
    check(h, 900)


@pytest.mark.parametrize("H,hs", SHAPES)
@pytest.mark.parametrize("T", [90, 700])
def test_aft_decode4_not_finite_under_masks(ops, H, hs, T):
    """A value that is not finite reaches its group's outputs from a position
    that -inf masks too (0 * NaN), wherever it lies, and no others; a sequence
    whose positions are all masked stays zero."""
    rng = np.random.default_rng(H * hs + T)
    D = H * hs
    for at in (0, 1, 17, T - 2):
        w = (0.5 * rng.standard_normal((H, T, T))).astype(np.float32)
        w[:, :, : T // 2] = -np.inf
        w[:, T - 1, at] = -np.inf
        kv = rng.standard_normal((2, T, 2 * D))
        kv[0, at, D + 5] = np.nan
        h = History(ops, rng, 2, H, hs, T, 8, "f32", [T - 1, T // 2 - 1], w=w)
        store(h, kv)
        got = check(h, 20)
        assert np.flatnonzero(np.isnan(got[0])).tolist() == list(range(32)) and not got[1].any()


@pytest.mark.parametrize("H,hs", SHAPES)
@pytest.mark.parametrize("size", [1e-10, 1e-20, 1e-28, 1e-33])
def test_aft_decode4_small_values(ops, H, hs, size):
    """Values whose products with small weights fall below fp32's range:
    channels up to 40 nats below their group's reference."""
    rng = np.random.default_rng(H * hs)
    D, T = H * hs, 150
    h = History(ops, rng, 2, H, hs, T, 8, "f32", [T - 1, 60])
    kv = rng.standard_normal((2, T, 2 * D))
    kv[..., :D] += rng.uniform(-20, 20, D)
    kv[..., D:] *= size
    store(h, kv)
    h.qkv[:, 2 * D:] *= size
    check(h, 40)
