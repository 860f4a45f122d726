"""AftDecoder generation over the paged 4-bit history (prompts of different
lengths) and with logit controls."""
import numpy as np
import pytest
import torch

from tests import ragged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import decoder, ops
    ops.read_status()
    return decoder, ops


def model(decoder, seed=7, **kw):
    base = dict(vocab=37, d_model=64, n_layers=2, n_heads=2, block_size=48)
    base.update(kw)
    return decoder.AftDecoder(decoder.DecoderConfig(**base), seed=seed, std=0.3)


def prompts(vocab, B, T0, seed=8):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (B, T0), generator=g, dtype=torch.int32).cuda()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("page_size,lens", [(8, [5, 17, 1, 12, 16]), (16, [17, 16, 15, 2, 9]), (64, [3, 3, 3, 3, 3])])
def test_ragged_matches_single_sequences(mods, page_size, lens):
    """Each sequence of a ragged batch gets the logits and tokens that it gets
    alone.  GEMMs of other sizes add in another order (2^-24 relative), which
    moves a 4-bit code only where a value lies that near a border: logits
    agree to far less than one code's step (2e-2 of their norm)."""
    decoder, ops = mods
    m = model(decoder)
    B, T0, n_new = 5, 17, 20
    p = prompts(37, B, T0)
    m.prefill(p, lens=lens, cache_bits=4, n_new=n_new, page_size=page_size)
    logits = [m._dec["logits"].clone()]
    for _ in range(n_new - 1):
        m.decode_step()
        logits.append(m._dec["logits"].clone())
    toks, pos = m._dec["tokens"].clone(), m._dec["pos"].tolist()
    assert pos == [n + n_new - 1 for n in lens] and ops.read_status() == 0
    used = sum(-(-(n + n_new - 1) // page_size) for n in lens)
    assert int(m._dec["head"]) == used
    for b, n in enumerate(lens):
        assert torch.equal(toks[b, :n], p[b, :n])
        one = p[b: b + 1, :n].contiguous()
        m.prefill(one, lens=[n], cache_bits=4, n_new=n_new, page_size=page_size)
        for i in range(n_new):
            if i:
                m.decode_step()
            got, want = logits[i][b], m._dec["logits"][0]
            assert rel(got, want) < 2e-2, (b, i)
            top = torch.topk(want, 2).values
            if float(top[0] - top[1]) <= 4e-2 * float(want.norm()):
                break  # the two may pick differently from here on
            assert int(toks[b, n + i]) == int(m._dec["tokens"][0, n + i])
    assert ops.read_status() == 0


def test_history_holds_the_prefill(mods):
    """The pages hold the quantised k and v of the prefill's projections, and
    the forward attended to exactly these values."""
    decoder, ops = mods
    m = model(decoder)
    lens, T0, page = [9, 4, 11], 11, 8
    p = prompts(37, 3, T0)
    m.prefill(p, lens=lens, cache_bits=4, page_size=page)
    s, d = m._dec, 64
    table = s["table"].cpu().numpy()
    for l in range(2):
        pages = s["cache"][l].cpu().numpy()
        qkv = m._bufs["qkv"][l].view(3, T0, 3 * d).cpu().numpy()
        for b, n in enumerate(lens):
            for i in range(n):
                k, v = ref.unpack_row(pages[table[b, i // page], :, i % page])
                assert np.array_equal(k.astype(np.float32), qkv[b, i, d: 2 * d])
                assert np.array_equal(v.astype(np.float32), qkv[b, i, 2 * d:])


@pytest.mark.parametrize("cache_bits", [4, 32])
def test_generate_graph_matches_eager(mods, cache_bits):
    decoder, ops = mods
    m = model(decoder)
    p = prompts(37, 4, 10)
    c = decoder.LogitControls(repetition=1.2, presence=0.1, frequency=[0.1, 0.2, 0.0, 0.3])
    a = m.generate(p, 25, graph=False, cache_bits=cache_bits, controls=c).clone()
    b = m.generate(p, 25, graph=True, cache_bits=cache_bits, controls=c).clone()
    assert torch.equal(a, b) and torch.equal(a[:, :10], p) and ops.read_status() == 0


def test_four_bits_stay_near_32(mods):
    """Logits after the prompt: a 4-bit value is off by at most half a step,
    at most 1/30 of its group's range, so the logits stay near the 32-bit
    ones (within 0.2 of their norm), and are not the same."""
    decoder, _ = mods
    m = model(decoder)
    p = prompts(37, 6, 20)
    m.prefill(p)
    m.decode_step()
    a = m._dec["logits"].clone()
    tok = m._dec["tokens"].clone()
    m.prefill(p, cache_bits=4)
    same = (m._dec["tokens"][:, 20] == tok[:, 20]).nonzero()[:, 0]
    assert len(same) >= 3
    m.decode_step()
    err = rel(m._dec["logits"][same], a[same])
    assert 0 < err < 0.2


@pytest.mark.parametrize("cache_bits", [4, 32])
def test_controls(mods, cache_bits):
    """A mask keeps generation inside its tokens, a bias forces one, a large
    presence penalty forbids repeating a generated token, a large repetition
    penalty those of the prompt too."""
    decoder, ops = mods
    m = model(decoder)
    B, T0, n = 3, 6, 12
    p = prompts(37, B, T0)
    C = decoder.LogitControls
    allow = [2, 5, 31, 32, 36]
    words = np.zeros(2, np.int64)
    for v in allow:
        words[v // 32] |= 1 << (v % 32)
    mask = torch.from_numpy(words.astype(np.uint32).view(np.int32)).cuda()
    out = m.generate(p, n, cache_bits=cache_bits, controls=C(mask=mask))[:, T0:]
    assert set(out.unique().tolist()) <= set(allow)
    bias = torch.zeros(B, 37)
    bias[torch.arange(B), torch.tensor([7, 0, 36])] = 1e4
    out = m.generate(p, n, cache_bits=cache_bits, controls=C(bias=bias))[:, T0:]
    assert out.tolist() == [[7] * n, [0] * n, [36] * n]
    out = m.generate(p, n, cache_bits=cache_bits, controls=C(presence=1e4))[:, T0:]
    assert all(len(set(r)) == n for r in out.tolist())
    out = m.generate(p, n, cache_bits=cache_bits, controls=C(bias=torch.full((37,), 1e3), mask=mask, frequency=[1e4, 0.0, 1e4]))
    counts = [[r.count(v) for v in allow] for r in out[:, T0:].tolist()]
    assert max(counts[0]) - min(counts[0]) <= 1 and max(counts[2]) - min(counts[2]) <= 1
    assert ops.read_status() == 0


def test_decode_step_leaves_out_finished_sequences(mods):
    decoder, ops = mods
    m = model(decoder)
    p = prompts(37, 3, 8)
    m.prefill(p, lens=[8, 3, 5], cache_bits=4)
    m.decode_step()
    m._dec["pos"][1] = -1
    before, head = m._dec["tokens"].clone(), int(m._dec["head"])
    m.decode_step()
    assert m._dec["pos"].tolist() == [10, -1, 7]
    assert torch.equal(m._dec["tokens"][1], before[1]) and int(m._dec["head"]) == head
    assert ops.read_status() == 0


def test_pool_runs_out(mods):
    """Steps past the pages that n_new asked for set the status bits."""
    decoder, ops = mods
    m = model(decoder)
    m.prefill(prompts(37, 2, 8), cache_bits=4, n_new=4, page_size=8)
    assert m._dec["n_pages"] == 4
    for _ in range(8):
        m.decode_step()
    assert ops.read_status() == 0
    m.decode_step()
    assert ops.read_status() == 0x300


def test_refusals(mods):
    decoder, _ = mods
    m = model(decoder)
    p = prompts(37, 2, 8)
    for kw in (dict(cache_bits=8), dict(lens=[8, 4]), dict(lens=[8, 9], cache_bits=4), dict(lens=[8, 0], cache_bits=4),
               dict(lens=[8], cache_bits=4), dict(cache_bits=4, page_size=0)):
        with pytest.raises(ValueError):
            m.prefill(p, **kw)
    with pytest.raises(ValueError):
        m.generate(p, 41, cache_bits=4)
    m.generate(p, 43, lens=[5, 3], cache_bits=4)
    with pytest.raises(ValueError):
        model(decoder, d_model=48, n_heads=4).prefill(p, cache_bits=4)
    from dart_cuda_b200 import DcError
    with pytest.raises(DcError):
        m.prefill(p, cache_bits=4, page_size=12)
    with pytest.raises(DcError):
        m.generate(p, 3, controls=decoder.LogitControls(bias=torch.zeros(36)))
