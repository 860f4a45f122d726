"""Prompts and lengths as a caller may hold them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import decoder, ops
    ops.read_status()
    return decoder.AftDecoder(decoder.DecoderConfig(vocab=37, d_model=64, n_layers=2, n_heads=2, block_size=48), seed=7,
                              std=0.3)


def prompts(B, T0):
    g = torch.Generator().manual_seed(8)
    return torch.randint(0, 37, (B, T0), generator=g, dtype=torch.int32).cuda()


def test_lengths_of_any_iterable(m):
    p, lens = prompts(3, 9), [4, 9, 2]
    want = m.generate(p, 6, lens=lens, cache_bits=4).clone()
    for given in (tuple(lens), torch.tensor(lens), torch.tensor(lens).cuda(), iter(lens)):
        assert torch.equal(m.generate(p, 6, lens=given, cache_bits=4), want)
    m.prefill(p, lens=iter(lens), cache_bits=4)
    assert m._dec["prompt_len"].tolist() == lens


@pytest.mark.parametrize("cache_bits", [4, 32])
def test_prompts_of_any_strides(m, cache_bits):
    """Columns of a wider tensor, a transposed one, one row of another."""
    wide = prompts(4, 30)
    for p in (wide[:, 3:12], wide[::2, :9], wide[:, :4].t(), wide[1:2, 5:20]):
        want = m.generate(p.contiguous(), 6, cache_bits=cache_bits).clone()
        got = m.generate(p, 6, cache_bits=cache_bits)
        assert torch.equal(got, want) and torch.equal(got[:, : p.shape[1]], p)


def test_prompts_refused(m):
    p = prompts(2, 9)
    for bad in (p.long(), p.cpu(), p[0], p.float(), prompts(2, 49)):
        with pytest.raises(ValueError):
            m.prefill(bad)
