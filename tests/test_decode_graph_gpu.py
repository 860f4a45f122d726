"""A captured decode step that is kept across prefills: it follows the new
prompt and controls, or refuses the replay."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decoder():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import decoder, ops
    ops.read_status()
    return decoder


def model(decoder):
    return decoder.AftDecoder(decoder.DecoderConfig(vocab=37, d_model=64, n_layers=2, n_heads=2, block_size=64), seed=7,
                              std=0.3)


def prompts(B, T0, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 37, (B, T0), generator=g, dtype=torch.int32).cuda()


def eager(m, p, n, **kw):
    return m.generate(p, n, graph=False, **kw).clone()


def replayed(m, g, p, n, **kw):
    m.prefill(p, **kw)
    for _ in range(n - 1):
        g.replay()
    return m._dec["tokens"][:, : p.shape[1] + n].clone()


def captured(m, p, **kw):
    m.prefill(p, **kw)
    m.decode_step()
    return m.capture_decode_step()


def mask_of(allow):
    words = [0, 0]
    for v in allow:
        words[v // 32] |= 1 << v % 32
    return torch.tensor([w - 2**32 if w >= 2**31 else w for w in words], dtype=torch.int32)


@pytest.mark.parametrize("cache_bits", [4, 32])
def test_new_prompt(decoder, cache_bits):
    m = model(decoder)
    g = captured(m, prompts(3, 9, 1), cache_bits=cache_bits)
    for seed, T0 in ((2, 9), (3, 5), (4, 12)):
        p = prompts(3, T0, seed)
        want = eager(m, p, 20, cache_bits=cache_bits)
        assert torch.equal(replayed(m, g, p, 20, cache_bits=cache_bits), want)


@pytest.mark.parametrize("cache_bits", [4, 32])
def test_new_controls_of_the_host(decoder, cache_bits):
    """Penalties, a bias and a mask given as numbers or host tensors are the
    last prefill's in every replay."""
    m = model(decoder)
    C, B, n = decoder.LogitControls, 3, 24
    p = prompts(B, 9, 1)

    def controls(k):
        bias = torch.zeros(37)
        bias[k % 37] = 2.0 * k
        return C(repetition=1.0 + 0.2 * k, presence=[0.3 * k] * B, frequency=torch.full((B,), 0.1 * k), bias=bias,
                 mask=mask_of(range(k, 37, 2)))

    g = captured(m, p, cache_bits=cache_bits, controls=controls(1))
    seen = []
    for k in (2, 5, 1):
        want = eager(m, p, n, cache_bits=cache_bits, controls=controls(k))
        assert torch.equal(replayed(m, g, p, n, cache_bits=cache_bits, controls=controls(k)), want)
        seen.append(want[:, 9:])
        assert set(want[:, 9:].unique().tolist()) <= set(range(k, 37, 2))
    assert not torch.equal(seen[0], seen[1])


def test_controls_on_the_device(decoder):
    """A device tensor is read at every step: rewritten it counts, another one
    needs another capture."""
    m = model(decoder)
    C = decoder.LogitControls
    p = prompts(2, 6, 3)
    mask = mask_of([1, 2, 3]).cuda()
    g = captured(m, p, cache_bits=4, controls=C(mask=mask))
    mask.copy_(mask_of([20, 36]))
    out = replayed(m, g, p, 10, cache_bits=4, controls=C(mask=mask))[:, 6:]
    assert set(out.unique().tolist()) <= {20, 36}
    m.prefill(p, cache_bits=4, controls=C(mask=mask.clone()))
    with pytest.raises(RuntimeError):
        g.replay()
    m.prefill(p, cache_bits=4, controls=C(mask=mask))
    g.replay()


def test_replay_refused(decoder):
    """Another history or another set of controls than the captured one."""
    m = model(decoder)
    C = decoder.LogitControls
    p = prompts(2, 8, 5)
    small = dict(cache_bits=4, n_new=4, page_size=8)
    g = captured(m, p, **small)
    before = m._dec["tokens"].clone()
    for kw in (dict(cache_bits=4, n_new=40, page_size=8), dict(cache_bits=4, page_size=16), dict(cache_bits=32)):
        m.prefill(p, **kw)
        with pytest.raises(RuntimeError):
            g.replay()
    g = captured(m, p, cache_bits=32)
    m.prefill(prompts(3, 8, 5))
    with pytest.raises(RuntimeError):
        g.replay()
    g = captured(m, p, controls=C(presence=1.0))
    for controls in (None, C(frequency=1.0), C(presence=1.0, bias=torch.zeros(37))):
        m.prefill(p, controls=controls)
        with pytest.raises(RuntimeError):
            g.replay()
    m.prefill(p, controls=C(presence=2.0))
    g.replay()
    assert before.shape == m._dec["tokens"].shape
