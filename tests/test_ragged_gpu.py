"""Ragged-generation operators on the GPU (page tables, the paged 4-bit k/v
history and the AFT decode step over it, logit controls, the per-row pick)
against tests/ragged_ref.py."""
import numpy as np
import pytest
import torch

from tests import ragged_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import ops as _ops

    assert _ops.read_status() >= 0  # start from a cleared status word
    return _ops


def cu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


# ------------------------------------------------------------ page tables
def tables_case(rng, B, page, width, most, spare=0, start_most=None):
    cap = page * width
    start = rng.integers(0, (start_most if start_most is not None else cap // 2) + 1, B)
    count = np.minimum(rng.integers(0, most + 1, B), cap - start)
    need = -(-start // page)
    free = rng.permutation(B * width + 5).astype(np.int32)
    table = np.full((B, width), -7, np.int32)
    for b in range(B):
        table[b, : need[b]] = 100000 + b * width + np.arange(need[b])
    return start.astype(np.int32), count.astype(np.int32), free, table


def run_tables(ops, start, count, free, head, table, page, n_slots, ld, inplace=False):
    t_table, t_head = cu(table), cu(np.array([head], np.int32))
    slots = torch.full((n_slots,), -99, dtype=torch.int32, device="cuda")
    row = torch.full((len(start) + 1,), -99, dtype=torch.int32, device="cuda")
    out = t_head if inplace else torch.zeros_like(t_head)
    ops.page_tables(cu(start), cu(count), cu(free), t_head, t_table, page, slots=slots, ld_slots=ld, row_start=row,
                    head_out=None if inplace else out)
    return t_table.cpu().numpy(), slots.cpu().numpy(), row.cpu().numpy(), int(out), ops.read_status()


@pytest.mark.parametrize("B,page,width,most,ld", [
    (1, 8, 1, 1, 0), (1, 16, 40, 600, 0), (3, 8, 7, 20, 20), (64, 16, 32, 1, 0), (64, 16, 32, 1, 1),
    (33, 256, 3, 300, 0), (1024, 32, 4, 9, 0), (1025, 8, 5, 11, 11), (2500, 64, 3, 40, 0), (7, 128, 9, 1000, 1000)])
def test_page_tables(ops, B, page, width, most, ld):
    rng = np.random.default_rng(B * 7 + page)
    start, count, free, table = tables_case(rng, B, page, width, most)
    n_slots = B * most + 3
    want = ref.page_tables(start, count, free, 2, table, page, n_slots, ld)
    for inplace in (False, True):
        got = run_tables(ops, start, count, free, 2, table, page, n_slots, ld, inplace)
        for a, b in zip(got[:4], want[:4]):
            assert np.array_equal(a, b)
        assert got[4] == 0 and not want[4]


@pytest.mark.parametrize("case", ["pool", "row", "slots", "ld", "inactive", "head", "hole"])
def test_page_tables_runs_out(ops, case):
    """Free list, table row, slots array or padded row too short: the tokens
    that have no page get -1 and the status says so; everything else stands."""
    rng = np.random.default_rng(11)
    B, page, width = 9, 8, 6
    start, count, free, table = tables_case(rng, B, page, width, 20, start_most=20)
    head, n_slots, ld, bad = 0, 400, 0, True
    if case == "pool":
        free = free[:5]
    elif case == "row":
        count[4] = 2000
        start[4] = 3
        n_slots = 4000
    elif case == "slots":
        n_slots = 40
    elif case == "ld":
        ld = 7
        n_slots = B * ld
    elif case == "inactive":
        start[::2] = -1
        count[1] = -5
        bad = False
    elif case == "head":
        head = len(free) + 10
    else:  # the page that a request's tokens end in is missing
        start[2], count[2] = 11, 3
        table[2] = -1
    want = ref.page_tables(start, count, free, head, table, page, n_slots, ld)
    got = run_tables(ops, start, count, free, head, table, page, n_slots, ld)
    for a, b in zip(got[:4], want[:4]):
        assert np.array_equal(a, b)
    assert got[4] == (0x100 if bad else 0) and want[4] == bad


def test_page_tables_huge_counts(ops):
    """Counts whose sum passes 2^31: nothing is written outside slots."""
    start = np.zeros(8, np.int32)
    count = np.full(8, 2**31 - 1, np.int32)
    free = np.arange(40, dtype=np.int32)
    table = np.full((8, 2), -1, np.int32)
    t, slots, row, head, status = run_tables(ops, start, count, free, 0, table, 8, 64, 0)
    assert np.array_equal(t, np.arange(16).reshape(8, 2)) and head == 16 and status == 0x100
    assert np.array_equal(slots, np.where(np.arange(64) < 16, np.arange(64), -1))
    assert row[0] == 0 and row[-1] == 2**31 - 1


# ------------------------------------------------------------ 4-bit history
def special_rows(rng, n, D):
    """Normal rows with channel means, and groups where quantisation can go
    wrong: constants, zeros, a small range far from zero, exact ties, huge and
    tiny magnitudes, values that are not finite."""
    x = (rng.standard_normal((n, D)) + 2 * rng.standard_normal(D)).astype(np.float32)
    tie = (np.arange(32) % 31 * 0.5).astype(np.float32)  # low 0, step 1: every half is a border
    kinds = [np.full(32, 1.2345678), np.zeros(32), 100 + 0.1 * rng.standard_normal(32), tie, -tie, tie + 2.0**-20,
             9e36 * rng.uniform(-1, 1, 32), 1e-39 * rng.standard_normal(32), 1e-42 * rng.standard_normal(32),
             np.where(np.arange(32) == 7, np.nan, 1.0), np.where(np.arange(32) == 31, np.inf, 1.0),
             np.where(np.arange(32) == 0, -np.inf, 0.5), np.full(32, -0.0), np.where(np.arange(32) == 3, 1.5e37, 0.0),
             -3.0 + 1e-6 * rng.standard_normal(32), np.abs(rng.standard_normal(32)) * 1e-30]
    for i, g in enumerate(kinds):
        r, c = i % n, (i // n) % (D // 32)
        x[r, 32 * c: 32 * c + 32] = g.astype(np.float32)
    return x


@pytest.mark.parametrize("n,D,page,dtype,ld", [
    (1, 32, 8, "f32", 0), (16, 64, 8, "f32", 64), (16, 96, 16, "bf16", 0), (16, 128, 32, "f32", 128),
    (20, 160, 8, "bf16", 16), (17, 256, 64, "f32", 0), (16, 512, 256, "bf16", 0), (3, 544, 8, "f32", 0)])
def test_kv4_write(ops, n, D, page, dtype, ld):
    """Bytes equal to the exact definition; skipped rows, other slots and
    their values stay; the values are what the codes stand for."""
    rng = np.random.default_rng(n * D)
    n_pages = -(-n // page) + 2
    W = ref.slab(D)
    host = torch.from_numpy(np.concatenate([special_rows(rng, n, D), special_rows(rng, n, D)], 1)).to(DT[dtype])
    wide = torch.zeros(n, 2 * D + ld, dtype=DT[dtype])
    wide[:, : 2 * D] = host
    x = wide.cuda()
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    if n > 2:
        slots[1] = -1
    pages = ops.kv4_pages(n_pages, page, D)
    pages.fill_(0xAB)
    vals = torch.full((n, 2 * D + ld), 3.0, dtype=DT[dtype], device="cuda")
    ops.kv4_write(x[:, :D], x[:, D: 2 * D], cu(slots), pages, values=(vals[:, :D], vals[:, D: 2 * D]))
    want = np.full((n_pages, D // W, page, W * 5 // 4), 0xAB, np.uint8)
    wval = np.full((n, 2 * D), 3.0)
    f = host.float().numpy()
    for r in range(n):
        if slots[r] < 0:
            continue
        rec, val = ref.pack_row(f[r, :D], f[r, D:])
        want[slots[r] // page, :, slots[r] % page] = rec
        wval[r] = val.reshape(-1)
    assert np.array_equal(pages.cpu().numpy(), want)
    got = vals[:, : 2 * D].float().cpu().numpy().astype(np.float64)
    # one rounding of low + step * code to fp32 (exact in float64 here), a
    # second to bf16
    tol = np.abs(wval) * (2.0**-24 + (2.0**-8 if dtype == "bf16" else 0)) + 1e-45
    assert np.array_equal(np.isnan(got), np.isnan(wval))
    ok = ~np.isnan(wval)
    assert np.all(np.abs(got - wval)[ok] <= tol[ok])
    assert torch.all(vals[:, 2 * D:] == 3.0)
    assert ops.read_status() == 0
    # in place: the same values over k and v
    ops.kv4_write(x[:, :D], x[:, D: 2 * D], cu(slots), pages, values=(x[:, :D], x[:, D: 2 * D]))
    keep = cu(slots >= 0)
    assert torch.equal(torch.nan_to_num(x[keep][:, : 2 * D], 7.0), torch.nan_to_num(vals[keep][:, : 2 * D], 7.0))
    assert torch.equal(torch.nan_to_num(x[~keep].cpu(), 7.0), torch.nan_to_num(wide[(~keep).cpu()], 7.0))


def test_kv4_write_error_bound(ops):
    """A stored value is off by at most half a step, and the step exceeds
    1/15 of the group's range by the two bf16 roundings only."""
    rng = np.random.default_rng(5)
    n, D = 64, 256
    x = cu((rng.standard_normal((n, 2 * D)) * 3 + 10).astype(np.float32))
    pages = ops.kv4_pages(8, 8, D)
    v = torch.empty_like(x)
    ops.kv4_write(x[:, :D], x[:, D:], torch.arange(n, dtype=torch.int32, device="cuda"), pages, values=(v[:, :D], v[:, D:]))
    g = x.double().view(n, -1, 32)
    span = g.amax(-1) - g.amin(-1)
    # step <= (span + |low| 2^-7) / 15 * (1 + 2^-7); values rounded to fp32
    step = (span + g.amin(-1).abs() * 2.0**-7) / 15 * (1 + 2.0**-7)
    err = (v.double() - x.double()).view(n, -1, 32).abs().amax(-1)
    assert torch.all(err <= step / 2 * (1 + 1e-9) + 32 * 2.0**-24)


def test_kv4_write_bad_slots(ops):
    """Slots behind the pool write nothing and set status bit 0x200."""
    pages = ops.kv4_pages(2, 8, 64)
    x = torch.randn(4, 128, device="cuda")
    slots = torch.tensor([3, 16, 2**31 - 1, -5], dtype=torch.int32, device="cuda")
    ops.kv4_write(x[:, :64], x[:, 64:], slots, pages)
    assert ops.read_status() == 0x200
    used = pages.view(2, 1, 8, 80).sum((1, 3)).view(-1) > 0
    assert used.nonzero()[:, 0].tolist() == [3]


# ------------------------------------------------------------ decode step
class History:
    """A paged 4-bit history with its bytes known on the host."""

    def __init__(self, ops, rng, B, H, hs, T, page, dtype, lens, w=None):
        self.ops, self.B, self.H, self.hs, self.D, self.page, self.T = ops, B, H, hs, H * hs, page, T
        D = self.D
        width = -(-T // page)
        self.n_pages = B * width + 3
        self.pos = np.asarray(lens, np.int32)
        self.table = rng.permutation(self.n_pages)[: B * width].reshape(B, width).astype(np.int32)
        self.pages = ops.kv4_pages(self.n_pages, page, D)
        self.pages.copy_(torch.from_numpy(rng.integers(0, 256, tuple(self.pages.shape), dtype=np.uint8)))
        n = self.n_pages * page
        kv = torch.from_numpy((rng.standard_normal((n, 2 * D)) + rng.standard_normal(2 * D)).astype(np.float32)).cuda()
        # positions behind pos keep arbitrary bytes (NaN steps among them)
        slots = np.full(n, -1, np.int32)
        for b in range(B):
            i = np.arange(max(0, min(self.pos[b], T)))
            s = self.table[b, i // page] * page + i % page
            slots[s] = s
        ops.kv4_write(kv[:, :D], kv[:, D:], cu(slots), self.pages)
        self.qkv = torch.from_numpy(rng.standard_normal((B, 3 * D)).astype(np.float32)).to(DT[dtype]).cuda()
        self.w = (0.5 * rng.standard_normal((H, T, T))).astype(np.float32) if w is None else w
        self.ws = ops.aft_decode4_workspace(B, D)
        self.dtype = dtype

    def step(self, **kw):
        return self.ops.aft_decode4(self.qkv, cu(self.w), self.pages, cu(self.table), cu(self.pos), self.ws, **kw)

    def expect(self):
        """(pages, z, bound): the bytes after the append, the rows in 64 bits
        and how far fp32 arithmetic may be off."""
        pages = self.pages.cpu().numpy().copy()
        x = self.qkv.float().cpu().numpy()
        z, tol = np.zeros((self.B, self.D)), np.zeros((self.B, self.D))
        for b in range(self.B):
            t = int(self.pos[b])
            if t < 0 or t >= self.T:
                continue
            rec, _ = ref.pack_row(x[b, self.D: 2 * self.D], x[b, 2 * self.D:])
            pages[self.table[b, t // self.page], :, t % self.page] = rec
            kv = np.stack([ref.unpack_row(pages[self.table[b, i // self.page], :, i % self.page]) for i in range(t + 1)])
            w = self.w[:, t, : t + 1]
            z[b] = ref.aft_row(x[b, : self.D], kv[:, 0], kv[:, 1], w, self.hs)
            # weights: exponents of size X carry up to 6 roundings of X 2^-24
            # in either log base, exp and sigmoid 4 half steps; sums of t+1
            # terms t+1 half steps; all relative to the weighted mean of |v|,
            # at most max |v|, twice (numerator and denominator)
            fin = np.where(np.abs(w) < 1e30, w, 0)
            X = np.nanmax(np.abs(kv[:, 0])) + np.abs(fin).max()
            tol[b] = 2 * (6 * X + 8 + t + 1) * 2.0**-24 * np.nanmax(np.abs(kv[:, 1]))
        if self.dtype == "bf16":
            tol = tol + 2.0**-8 * np.abs(z)
        return pages, z, tol

    def check(self, status=0):
        pages, z, tol = self.expect()
        got = self.step()
        assert self.ops.read_status() == status
        assert np.array_equal(self.pages.cpu().numpy(), pages)
        g = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(z))
        bad = ~(np.abs(g - z) <= tol) & ~np.isnan(z)
        assert not bad.any(), (np.abs(g - z)[bad].max(), np.argwhere(bad)[:4])
        counters = -(-4 * self.B * (self.D // 32) // 256) * 256  # at the end, left at zero
        assert torch.count_nonzero(self.ws[-counters:]) == 0
        again = self.step()  # idempotent, the same bits
        assert self.ops.read_status() == status
        assert torch.equal(torch.nan_to_num(again, 7.0), torch.nan_to_num(got, 7.0))
        return got


@pytest.mark.parametrize("H,hs,T,page,dtype,lens", [
    (1, 32, 1, 8, "f32", [0]), (2, 16, 16, 8, "f32", [0, 15, 7]), (3, 32, 70, 16, "bf16", [69, 0, 1, 33, 8]),
    (4, 16, 100, 64, "f32", [99, 50, 15, 16, 17]), (1, 128, 300, 32, "f32", [299, 255, 256]),
    (4, 128, 130, 16, "f32", [129, 64, 0]), (5, 64, 90, 128, "bf16", [89, 2]), (16, 8, 40, 8, "f32", [39, 38, 31, 32]),
    (4, 8, 33, 256, "bf16", [32, 5]), (17, 32, 48, 8, "f32", [47, 11])])
def test_aft_decode4(ops, H, hs, T, page, dtype, lens):
    rng = np.random.default_rng(H * hs + T)
    History(ops, rng, len(lens), H, hs, T, page, dtype, lens).check()


@pytest.mark.parametrize("H,hs,T,page,dtype,lens", [
    (2, 128, 1500, 64, "f32", [1499, 3]), (1, 64, 2100, 16, "bf16", [2099]), (2, 16, 1030, 8, "f32", [1029, 1024, 511, 0])])
def test_aft_decode4_long(ops, H, hs, T, page, dtype, lens):
    rng = np.random.default_rng(T)
    History(ops, rng, len(lens), H, hs, T, page, dtype, lens).check()


@pytest.mark.parametrize("masked", [0, 4800])
def test_aft_decode4_many_shares(ops, masked):
    """One sequence over many CTAs, whose first shares a mask may leave empty."""
    T = 5000
    rng = np.random.default_rng(masked)
    w = (0.5 * rng.standard_normal((1, T, T))).astype(np.float32)
    w[:, :, :masked] = -np.inf
    History(ops, rng, 2, 1, 64, T, 32, "f32", [T - 1, T - 100], w=w).check()


def test_aft_decode4_many_sequences(ops):
    """More sequences than SMs, lengths from one to long, in one call."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 60, 400)
    lens[[5, 399]] = 199
    lens[[0, 17, 398]] = -1
    h = History(ops, rng, 400, 2, 16, 200, 8, "f32", lens)
    z = h.check()
    assert torch.count_nonzero(z[[0, 17, 398]]) == 0


@pytest.mark.parametrize("B,H,hs,T,page,dtype", [(40, 24, 64, 120, 16, "f32"), (50, 5, 128, 90, 8, "bf16"),
                                                 (80, 14, 32, 60, 64, "f32"), (36, 32, 24, 70, 8, "f32"),
                                                 (150, 2, 128, 130, 32, "f32")])
def test_aft_decode4_uneven_shares(ops, B, H, hs, T, page, dtype):
    """More (sequence, slab) items than parts of their own would fit: shares
    that begin and end inside items, of lengths from one position up."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, T, B)
    lens[rng.random(B) < 0.3] = rng.integers(0, 4)
    lens[[0, B - 1]] = T - 1, -1
    History(ops, rng, B, H, hs, T, page, dtype, lens).check()


def test_aft_decode4_inactive_and_full(ops):
    rng = np.random.default_rng(4)
    h = History(ops, rng, 4, 2, 32, 24, 8, "f32", [-1, 24, 23, -2**31])
    z = h.check(status=0x40)
    h2 = History(ops, rng, 2, 2, 32, 24, 8, "f32", [-1, -1])
    assert torch.count_nonzero(h2.check()) == 0
    assert torch.count_nonzero(z[[0, 1, 3]]) == 0 and torch.count_nonzero(z[2]) == 64


@pytest.mark.parametrize("fill", [-np.inf, np.finfo(np.float32).min])
def test_aft_decode4_masked_bias(ops, fill):
    """-inf and the type's lowest value in the bias: masked positions, whole
    rows masked for one head (zero, respectively the plain mean) or for all."""
    rng = np.random.default_rng(6)
    H, hs, T = 4, 32, 80
    w = (0.5 * rng.standard_normal((H, T, T))).astype(np.float32)
    w[0][rng.random((T, T)) < 0.7] = fill
    w[1] = fill
    w[2, :, 3:] = fill
    w[3, 60] = fill
    w[:, 41] = fill
    h = History(ops, rng, 5, H, hs, T, 16, "f32", [79, 60, 41, 0, 2], w=w)
    z = h.check()
    if fill == -np.inf:
        assert torch.count_nonzero(z[2]) == 0 and torch.count_nonzero(z[0, 32:64]) == 0


def test_aft_decode4_not_finite(ops):
    """NaN and inf in the appended row reach that group's outputs only."""
    rng = np.random.default_rng(7)
    h = History(ops, rng, 2, 2, 64, 40, 8, "f32", [20, 33])
    h.qkv[0, 128 + 5] = float("nan")
    h.qkv[1, 256 + 70] = float("inf")
    z = h.check()
    bad = torch.isnan(z)
    assert bad[0].nonzero()[:, 0].tolist() == list(range(32))
    assert bad[1].nonzero()[:, 0].tolist() == list(range(64, 96))


def test_aft_decode4_wide_spread(ops):
    """Channels of one group whose keys lie far apart, rising with the
    position: the running maximum is each channel's own."""
    rng = np.random.default_rng(8)
    h = History(ops, rng, 2, 1, 64, 200, 8, "f32", [199, 120])
    n = h.n_pages * h.page
    kv = torch.randn(n, 128, device="cuda")
    kv[:, :64] = kv[:, :64] * 40 + 150 * torch.randn(64, device="cuda")
    slots = np.full(n, -1, np.int32)
    for b in range(2):
        i = np.arange(h.pos[b])
        s = h.table[b, i // 8] * 8 + i % 8
        slots[s] = s
    h.ops.kv4_write(kv[:, :64], kv[:, 64:], cu(slots), h.pages)
    h.check()


def test_aft_decode4_far_above(ops):
    """The last key of one channel lies 2^126 above what came before: for the
    group's other channels, 2^90 below it, that is not yet lost."""
    T, rng = 1024, np.random.default_rng(9)
    w = np.zeros((1, T, T), np.float32)
    w[0, :, 2::4] = w[0, :, 3::4] = 11.05
    w[0, T - 1, T - 1] = 25.03
    h = History(ops, rng, 1, 1, 32, T, 16, "f32", [T - 1], w=w)
    slots = np.full(h.n_pages * 16, -1, np.int32)
    i = np.arange(T - 1)
    slots[:T - 1] = h.table[0, i // 16] * 16 + i % 16
    kv = torch.ones(len(slots), 64, device="cuda")
    kv[:, :32] = 0
    ops.kv4_write(kv[:, :32], kv[:, 32:], cu(slots), h.pages)
    h.qkv[:] = 0
    h.qkv[0, 32] = 62.34375
    h.qkv[0, 64:] = -1
    h.check()


def test_aft_decode4_huge_keys(ops):
    """Keys of up to 9e36: each channel takes the value of its largest."""
    rng = np.random.default_rng(13)
    h = History(ops, rng, 2, 2, 32, 60, 8, "f32", [59, 17])
    n = h.n_pages * h.page
    kv = torch.randn(n, 128, device="cuda")
    kv[:, :64] *= 2e36
    slots = np.full(n, -1, np.int32)
    for b in range(2):
        i = np.arange(h.pos[b])
        s = h.table[b, i // 8] * 8 + i % 8
        slots[s] = s
    ops.kv4_write(kv[:, :64], kv[:, 64:], cu(slots), h.pages)
    z = h.expect()[1]
    got = h.step().double().cpu().numpy()
    # a weight is 1 or 0: what is left is the value's and the gate's rounding
    assert np.all(np.abs(got - z) <= 2.0**-20 * np.abs(z) + 1e-30) and ops.read_status() == 0


def test_aft_decode4_one_workspace(ops):
    """A workspace of a large call serves smaller ones in between."""
    rng = np.random.default_rng(14)
    big = History(ops, rng, 40, 8, 64, 200, 16, "f32", rng.integers(100, 200, 40))
    small = History(ops, rng, 1, 1, 32, 900, 16, "f32", [899])
    mid = History(ops, rng, 3, 4, 32, 700, 16, "bf16", [699, 650, 3])
    small.ws = mid.ws = big.ws
    for h in (big, small, big, mid, small, mid, big):
        pages, z, tol = h.expect()
        assert np.all(np.abs(h.step().double().cpu().numpy() - z) <= tol)
    assert ops.read_status() == 0


def test_aft_decode4_bad_page(ops):
    """A page id outside the pool: its positions are left out, status 0x200."""
    rng = np.random.default_rng(9)
    h = History(ops, rng, 2, 2, 32, 64, 8, "f32", [60, 60])
    good = h.table.copy()
    h.table[0, 2], h.table[1, 3] = -1, h.n_pages
    got = h.step()
    assert ops.read_status() == 0x200
    h.table = good
    h.w[:, 60, 16:24], keep = -np.inf, h.w.copy()
    z0 = h.expect()[1][0]
    h.w = keep
    h.w[:, 60, 24:32] = -np.inf
    z1 = h.expect()[1][1]
    assert np.abs(got[0].cpu().numpy() - z0).max() < 1e-4 and np.abs(got[1].cpu().numpy() - z1).max() < 1e-4


def test_aft_decode4_shared_pages_and_strides(ops):
    """Two sequences that share the pages of a common beginning; qkv, out and
    w as columns and corners of wider tensors."""
    rng = np.random.default_rng(10)
    h = History(ops, rng, 2, 2, 32, 64, 8, "f32", [40, 35])
    h.table[1, :4] = h.table[0, :4]
    pages, z, tol = h.expect()
    wide = torch.zeros(2, 3 * 64 + 12, device="cuda")
    wide[:, : 192] = h.qkv
    w = torch.zeros(2, 70, 77, device="cuda")
    w[:, :64, :64] = cu(h.w)
    out = torch.full((2, 80), 5.0, device="cuda")
    got = ops.aft_decode4(wide[:, :192], w[:, :64, :64], h.pages, cu(h.table), cu(h.pos), h.ws, out=out[:, :64])
    assert np.all(np.abs(got.cpu().numpy() - z) <= tol) and torch.all(out[:, 64:] == 5.0)
    assert np.array_equal(h.pages.cpu().numpy(), pages) and ops.read_status() == 0


def test_aft_decode4_captured(ops):
    """A captured step replayed on another stream as the positions advance:
    page_tables takes each request's next page, the decode appends."""
    rng = np.random.default_rng(12)
    B, H, hs, T, page = 3, 2, 32, 48, 8
    D = H * hs
    w = cu((0.5 * rng.standard_normal((H, T, T))).astype(np.float32))
    pages = ops.kv4_pages(B * 6, page, D)
    free = cu(rng.permutation(B * 6).astype(np.int32))
    head = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.full((B, 6), -1, dtype=torch.int32, device="cuda")
    pos = cu(np.array([0, -1, 0], np.int32))
    one = torch.ones(B, dtype=torch.int32, device="cuda")
    rows = cu(rng.standard_normal((T, B, 3 * D)).astype(np.float32))
    qkv, z = torch.zeros(B, 3 * D, device="cuda"), torch.zeros(B, D, device="cuda")
    ws = ops.aft_decode4_workspace(B, D)

    def step():
        ops.page_tables(pos, one, free, head, table, page)
        ops.aft_decode4(qkv, w, pages, table, pos, ws, out=z)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        qkv.copy_(rows[0])
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        for i in range(1, 20):
            pos[::2] += 1
            qkv.copy_(rows[i])
            g.replay()
    s.synchronize()
    assert ops.read_status() == 0 and int(head) == 2 * 3
    del g
    x = rows.cpu().numpy()
    for b in (0, 2):
        kv = np.stack([ref.pack_row(x[i, b, D: 2 * D], x[i, b, 2 * D:])[1] for i in range(20)])
        want = ref.aft_row(x[19, b, :D], kv[:, 0], kv[:, 1], w[:, 19, :20].cpu().numpy(), hs)
        tol = 2 * (6 * 8 + 8 + 20) * 2.0**-24 * np.abs(kv).max()
        assert np.abs(z[b].cpu().numpy() - want).max() <= tol
    assert torch.count_nonzero(z[1]) == 0


# ------------------------------------------------------------ logit controls
@pytest.mark.parametrize("B,V,T,dtype,which", [
    (1, 1, 1, "f32", "rpfbm"), (1, 65, 30, "f32", "r"), (3, 97, 200, "bf16", "rpfBM"), (5, 8192, 64, "f32", "rpfbM"),
    (2, 50257, 700, "bf16", "rpfBm"), (4, 4097, 300, "f32", "fb"), (2, 33, 40, "f32", "p"), (3, 20000, 5, "bf16", "M"),
    (2, 131, 9, "f32", "B"), (2, 64, 9, "f32", ""), (600, 25001, 40, "bf16", "rpfbm"), (600, 17003, 40, "f32", "rf")])
@pytest.mark.parametrize("ld", [0, 3])
def test_logits_controls(ops, B, V, T, dtype, which, ld):
    rng = np.random.default_rng(B * V + T)
    host = torch.from_numpy((3 * rng.standard_normal((B, V + ld))).astype(np.float32)).to(DT[dtype])
    x = host.cuda()[:, :V]
    tokens = rng.integers(0, min(V, 50), (B, T)).astype(np.int32)
    tokens[:, ::3] = rng.integers(0, V, tokens[:, ::3].shape)
    tokens[:, 1::7] = -1  # ids outside [0, V) are ignored
    tokens[:, 4::7] = V
    pos = rng.integers(-1, T, B).astype(np.int32)
    pos[-1] = T - 1
    prompt = rng.integers(0, T + 1, B).astype(np.int32)
    rep = rng.uniform(0.8, 1.6, B).astype(np.float32) if "r" in which else None
    pres = rng.uniform(-1, 1, B).astype(np.float32) if "p" in which else None
    freq = rng.uniform(-0.3, 0.6, B).astype(np.float32) if "f" in which else None
    bias = rng.standard_normal((B, V) if "B" in which else V).astype(np.float32) if "b" in which.lower() else None
    words = (V + 31) // 32
    mask = None
    if "m" in which.lower():
        mask = rng.integers(-2**31, 2**31, (B, words) if "M" in which else words).astype(np.int32)
        mask.reshape(-1, words)[0] = 0  # a row (or all) that allows nothing
    opt = lambda a: None if a is None else cu(a)  # noqa: E731
    want = ref.logits_controls(host[:, :V].float().numpy(), tokens, pos, prompt, rep, pres, freq, bias, mask)
    out = torch.full((B, V + ld), 9.0, dtype=DT[dtype], device="cuda")
    got = ops.logits_controls(x, cu(tokens), cu(pos), prompt_len=cu(prompt), repetition=opt(rep), presence=opt(pres),
                              frequency=opt(freq), bias=opt(bias), mask=opt(mask), out=out[:, :V])
    assert torch.all(out[:, V:] == 9.0)
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isneginf(g), np.isneginf(want))
    ok = np.isfinite(want)
    # at most 5 fp32 operations on values of at most |x| + f T + |p| + |b|,
    # then one rounding to the type
    size = 1.6 * np.abs(host[:, :V].float().numpy()).max() + 0.6 * T + 1 + 5
    tol = 5 * 2.0**-24 * size + (2.0**-8 if dtype == "bf16" else 0) * np.abs(np.where(ok, want, 0))
    assert np.all(np.abs(np.where(ok, g, 0) - np.where(ok, want, 0)) <= tol)
    # in place
    y = host.cuda()
    ops.logits_controls(y[:, :V], cu(tokens), cu(pos), prompt_len=cu(prompt), repetition=opt(rep), presence=opt(pres),
                        frequency=opt(freq), bias=opt(bias), mask=opt(mask), out=y[:, :V])
    assert torch.equal(y[:, :V], got) and torch.equal(y[:, V:].cpu(), host[:, V:])
    assert ops.read_status() == 0


def test_logits_controls_not_finite(ops):
    """inf, -inf and NaN logits: penalties keep them, the mask hides NaN."""
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), 1.0, float("nan")]], device="cuda")
    tokens = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    mask = torch.tensor([0b01111], dtype=torch.int32, device="cuda")
    one = torch.ones(1, device="cuda")
    y = ops.logits_controls(x, tokens, pos, repetition=2 * one, presence=one, frequency=one, mask=mask)[0].tolist()
    assert y[0] == float("inf") and y[1] == float("-inf") and y[2] != y[2] and y[3] == 0.5 - 2 and y[4] == float("-inf")


def test_logits_controls_position_behind_the_row(ops):
    """Positions past the tokens' capacity, up to the largest int."""
    tokens = torch.tensor([[1, 2, 2], [1, 2, 2], [1, 2, 2]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([2, 3, 2**31 - 1], dtype=torch.int32, device="cuda")
    y = ops.logits_controls(torch.zeros(3, 5, device="cuda"), tokens, pos, frequency=torch.ones(3, device="cuda"))
    assert y.tolist() == [[0, -1, -2, 0, 0]] * 3


def test_single_rows_of_any_stride(ops):
    """A tensor of one row has no row stride."""
    rng = np.random.default_rng(21)
    h = History(ops, rng, 1, 1, 32, 20, 8, "f32", [19])
    want = h.step().clone()
    wide = torch.zeros(2, 97, device="cuda")
    wide[0, :96] = h.qkv[0]
    h.qkv = wide[:1, :96]
    assert torch.equal(h.step(), want) and ops.read_status() == 0


def test_logits_controls_shared_position(ops):
    rng = np.random.default_rng(2)
    B, V, T = 4, 300, 20
    x, tokens = rng.standard_normal((B, V)).astype(np.float32), rng.integers(0, V, (B, T)).astype(np.int32)
    rep = np.full(B, 1.3, np.float32)
    got = ops.logits_controls(cu(x), cu(tokens), cu(np.array([11], np.int32)), repetition=cu(rep))
    want = ref.logits_controls(x, tokens, np.full(B, 11), None, rep, None, None, None, None)
    assert np.abs(got.cpu().numpy() - want).max() <= 2.0**-23 * np.abs(x).max() * 1.3


def test_logits_controls_long_history(ops):
    """One token repeated over a history longer than the vocabulary chunk."""
    V, T = 100, 20001
    tokens = torch.full((1, T), 42, dtype=torch.int32, device="cuda")
    pos = torch.tensor([T - 1], dtype=torch.int32, device="cuda")
    prompt = torch.tensor([1], dtype=torch.int32, device="cuda")
    f = torch.full((1,), 0.5, device="cuda")
    y = ops.logits_controls(torch.zeros(1, V, device="cuda"), tokens, pos, prompt_len=prompt, frequency=f)
    assert float(y[0, 42]) == -0.5 * (T - 1) and int(torch.count_nonzero(y)) == 1


# ------------------------------------------------------------ pick
@pytest.mark.parametrize("B,V,D,dtype,ld", [(1, 1, 1, "f32", 0), (3, 65, 32, "f32", 0), (64, 8192, 512, "f32", 0),
                                            (5, 50257, 48, "bf16", 3), (2, 131073, 7, "f32", 1), (300, 130, 4, "bf16", 0),
                                            (40, 70001, 9, "bf16", 3), (400, 9000, 5, "f32", 1)])
def test_greedy_embed_rows(ops, B, V, D, dtype, ld):
    rng = np.random.default_rng(V)
    T = 12
    x = torch.from_numpy(rng.standard_normal((B, V + ld)).astype(np.float32)).to(DT[dtype])
    x[:, V:] = 100.0
    if V > 2:
        x[0, [V // 3, V - 1]] = 50.0  # a tie: the lowest index
    if B > 1:
        x[1, :V] = float("-inf")  # nothing allowed: token 0
        if V > 1:
            x[B - 1, :V // 2] = float("nan")
    tokens = rng.integers(0, V, (B, T)).astype(np.int32)
    pos = rng.integers(-1, T - 1, B).astype(np.int32)
    pos[0] = 0
    status = 0
    if B > 2:
        pos[2], status = T - 1, 0x40
    wte, wpe = rng.standard_normal((V, D)).astype(np.float32), rng.standard_normal((T, D)).astype(np.float32)
    t_tok, t_x = cu(tokens), torch.full((B, D), 3.0, device="cuda")
    out = torch.zeros(B, dtype=torch.int32, device="cuda")
    ops.greedy_embed_rows(x.cuda()[:, :V], t_tok, cu(pos), wte=cu(wte), wpe=cu(wpe), x=t_x, pos_out=out)
    want_tok, want_x, want_pos = tokens.copy(), np.full((B, D), 3.0, np.float32), pos.copy()
    f = x[:, :V].float().numpy()
    for b in range(B):
        if 0 <= pos[b] < T - 1:
            row = np.where(np.isnan(f[b]), -np.inf, f[b])
            finite = np.flatnonzero(~np.isnan(f[b]))
            tok = int(finite[np.argmax(row[finite])])
            want_tok[b, pos[b] + 1] = tok
            want_x[b] = wte[tok] + wpe[pos[b] + 1]
            want_pos[b] += 1
    assert ops.read_status() == status
    assert np.array_equal(t_tok.cpu().numpy(), want_tok) and np.array_equal(out.cpu().numpy(), want_pos)
    assert np.array_equal(t_x.cpu().numpy(), want_x)
    # in place, without an embedding
    p = cu(pos)
    t2 = cu(tokens)
    ops.greedy_embed_rows(x.cuda()[:, :V], t2, p)
    assert torch.equal(t2, t_tok) and torch.equal(p, out) and ops.read_status() == status
