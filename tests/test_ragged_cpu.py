"""Host-side checks of the ragged-generation entry points: what they refuse,
before any CUDA call, and the 64-bit definitions against each other."""
import ctypes

import numpy as np
import pytest
import torch

from tests import ragged_ref as ref

FAKE = 0x1000  # never dereferenced: validation returns first


@pytest.fixture(scope="module")
def L():
    from dart_cuda_b200 import lib

    return lib()


def tables(L, B=2, page=16, n_free=4, ldtab=3, slots=FAKE, n_slots=8, ld=0, start=FAKE, table=FAKE, head=FAKE):
    return L.dc_page_tables(start, FAKE, B, page, FAKE, n_free, head, FAKE, table, ldtab, slots, n_slots, ld, None, None)


@pytest.mark.parametrize("bad", [dict(B=-1), dict(page=7), dict(page=4), dict(page=512), dict(page=24), dict(n_free=-1),
                                 dict(ldtab=0), dict(n_slots=-1), dict(ld=-1), dict(ld=5), dict(start=None),
                                 dict(table=None), dict(head=None), dict(B=2**20, ldtab=2**12),
                                 dict(n_free=2**30), dict(B=1, ldtab=2**30)])
def test_page_tables_refuses(L, bad):
    assert tables(L, **bad) == 1 and L.dc_last_error()
    assert tables(L, B=0) == 0


def write(L, k=FAKE, v=FAKE, ld=64, dtype=0, slots=FAKE, n=3, D=64, pages=FAKE, n_pages=2, page=8, vk=None, vv=None, ldv=0):
    return L.dc_kv4_write(k, v, ld, dtype, slots, n, D, pages, n_pages, page, vk, vv, ldv, None)


@pytest.mark.parametrize("bad", [dict(D=48), dict(D=0), dict(page=6), dict(n_pages=0), dict(n_pages=2**30), dict(n=-1),
                                 dict(dtype=2), dict(ld=60), dict(ld=66), dict(ld=68, dtype=1), dict(k=None),
                                 dict(v=None), dict(slots=None), dict(pages=None), dict(k=FAKE + 4), dict(pages=FAKE + 8),
                                 dict(vk=FAKE), dict(vk=FAKE, vv=FAKE, ldv=32), dict(vk=FAKE, vv=FAKE + 4, ldv=64)])
def test_kv4_write_refuses(L, bad):
    assert write(L, **bad) == 1 and L.dc_last_error()
    assert write(L, n=0) == 0


def decode(L, qkv=FAKE, ldq=192, dtype=0, w=FAKE, ldw=32, pages=FAKE, n_pages=9, page=8, table=FAKE, ldtab=4, B=2, H=2,
           hs=32, pos=FAKE, Tmax=32, Z=FAKE, ldz=64, ws=FAKE, nb=1 << 30):
    return L.dc_aft_decode4(qkv, ldq, dtype, w, ldw, 1024, pages, n_pages, page, table, ldtab, B, H, hs, pos, Tmax, Z,
                            ldz, ws, nb, None)


@pytest.mark.parametrize("bad", [dict(B=-1), dict(H=0), dict(hs=0), dict(hs=12), dict(hs=4, H=16), dict(H=1, hs=24),
                                 dict(Tmax=2**20, ldw=2**20, ldtab=2**18), dict(B=2**20, Tmax=2**15, ldw=2**15, ldtab=2**12),
                                 dict(H=2**20, hs=2**12), dict(Tmax=0), dict(ldtab=0), dict(dtype=7), dict(ldq=188),
                                 dict(ldq=194), dict(ldz=63), dict(ldz=68, dtype=1), dict(ldw=31), dict(page=9),
                                 dict(n_pages=0), dict(qkv=None), dict(w=None), dict(pages=None), dict(table=None),
                                 dict(pos=None), dict(Z=None), dict(ws=None), dict(qkv=FAKE + 4), dict(Z=FAKE + 8),
                                 dict(ws=FAKE + 8)])
def test_aft_decode4_refuses(L, bad):
    assert decode(L, **bad) == 1 and L.dc_last_error()
    assert decode(L, nb=8) == 4  # DC_ERR_NOMEM
    assert decode(L, B=0) == 0


def controls(L, x=FAKE, ldl=100, out=FAKE, ldo=100, dtype=0, B=2, V=100, tokens=FAKE, ldt=8, pos=FAKE, stride=1, rep=FAKE,
             bias=None, ldb=0, mask=None, ldm=0):
    return L.dc_logits_controls(x, ldl, out, ldo, dtype, B, V, tokens, ldt, pos, stride, None, rep, None, None, bias, ldb,
                                mask, ldm, None)


@pytest.mark.parametrize("bad", [dict(B=-1), dict(V=0), dict(ldl=99), dict(ldo=99), dict(ldo=104), dict(dtype=3),
                                 dict(x=None), dict(out=None), dict(tokens=None), dict(pos=None), dict(ldt=0),
                                 dict(stride=2), dict(bias=FAKE, ldb=50), dict(mask=FAKE, ldm=3)])
def test_logits_controls_refuses(L, bad):
    assert controls(L, **bad) == 1 and L.dc_last_error()
    assert controls(L, B=0) == 0


def pick(L, x=FAKE, ldl=100, dtype=0, B=2, V=100, wte=FAKE, wpe=FAKE, pos=FAKE, out=FAKE, D=8, tokens=FAKE, ldt=8, e=FAKE):
    return L.dc_greedy_embed_rows(x, ldl, dtype, B, V, wte, wpe, pos, out, D, tokens, ldt, e, None)


@pytest.mark.parametrize("bad", [dict(B=-1), dict(V=0), dict(ldl=99), dict(ldt=0), dict(dtype=9), dict(x=None),
                                 dict(pos=None), dict(out=None), dict(tokens=None), dict(wte=None), dict(wpe=None),
                                 dict(D=0)])
def test_greedy_embed_rows_refuses(L, bad):
    assert pick(L, **bad) == 1 and L.dc_last_error()
    assert pick(L, B=0) == 0


def test_pool_size(L):
    n = ctypes.c_size_t(0)
    for pages, page, D in ((1, 8, 32), (7, 16, 96), (100000, 64, 2048)):
        assert L.dc_kv4_pages_size(pages, page, D, ctypes.byref(n)) == 0
        assert n.value == pages * page * D * 5 // 4
    assert L.dc_kv4_pages_size(1, 8, 33, ctypes.byref(n)) == 1
    assert L.dc_kv4_pages_size(1, 8, 32, None) == 1


def test_workspace_size_grows(L):
    """A workspace of B sequences of D channels holds those of smaller calls."""
    size = L.dc_aft_decode4_workspace_size
    assert size(0, 64) == 0 and size(3, 40) == 0
    last = 0
    for D in range(32, 2100, 32):
        assert size(64, D) >= last and size(63, D) <= size(64, D)
        last = size(64, D)


def test_python_calls_refuse_host_tensors():
    """The Python layer refuses tensors that are not on the current device
    before it reaches the library."""
    if torch.cuda.is_available():
        pytest.skip("the refusal of host tensors is checked without a GPU")
    from dart_cuda_b200 import DcError, ops

    with pytest.raises((DcError, RuntimeError, AssertionError)):
        ops.kv4_write(torch.zeros(2, 32), torch.zeros(2, 32), torch.zeros(2, dtype=torch.int32),
                      torch.zeros(1, 1, 8, 40, dtype=torch.uint8))


def test_reference_packs_and_unpacks():
    """pack_row and unpack_row agree, and a value is within half a step."""
    rng = np.random.default_rng(1)
    for D in (32, 96, 128, 256, 512):
        k, v = (rng.standard_normal((2, D)) * 4).astype(np.float32)
        rec, values = ref.pack_row(k, v)
        assert np.array_equal(ref.unpack_row(rec), values)
        for x, y in ((k, values[0]), (v, values[1])):
            for g in range(D // 32):
                s = slice(32 * g, 32 * g + 32)
                _, step, _ = ref.quantise_group(x[s])
                assert np.abs(x[s].astype(np.float64) - y[s]).max() <= float(step) / 2


@pytest.mark.parametrize("call,bad", [(controls, dict(V=2**30, ldl=2**30, ldo=2**30)),
                                      (controls, dict(V=2**31 - 1, ldl=2**31 - 1, ldo=2**31 - 1)),
                                      (controls, dict(ldt=2**30)), (controls, dict(ldt=2**31 - 1)),
                                      (pick, dict(V=2**30, ldl=2**30)), (pick, dict(V=2**31 - 1, ldl=2**31 - 1))])
def test_rows_past_the_kernels_indices_are_refused(L, call, bad):
    """The kernels step through logits and tokens in 32 bits."""
    assert call(L, **bad) == 1 and b"2^30" in L.dc_last_error()
