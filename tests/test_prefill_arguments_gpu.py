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
