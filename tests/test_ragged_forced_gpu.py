"""Every step of a ragged batch against the sequences alone, on the same tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page_size,lens", [(8, [5, 17, 1, 12, 16]), (16, [17, 16, 15, 2, 9]), (32, [3, 14, 3, 8, 1])])
def test_ragged_steps_match_single_sequences(page_size, lens):
    """The single run is given the ragged run's tokens, so that all steps
    compare, and the same padded prompt: the prefill's AFT scales a sequence's
    operands by their maxima over its whole row before it rounds them to tf32,
    so another padding moves every operand.  What is left are sums in another
    order, about 2^-22, which move an operand of a tf32 product to its
    neighbour (2^-11 of one of 64 terms) now and then: below 1e-3 of the
    logits' norm.  A 4-bit code moves more rarely still, and then one channel of
    one position by a step, 1/15 of its group's range: below 2e-2.  One position
    left out of 20 is about 5e-2 of its row.  Picks compare where the best two
    logits lie further apart than that."""
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from dart_cuda_b200 import decoder, ops

    ops.read_status()
    m = decoder.AftDecoder(decoder.DecoderConfig(vocab=37, d_model=64, n_layers=2, n_heads=2, block_size=48), seed=7, std=0.3)
    g = torch.Generator().manual_seed(8)
    B, T0, n_new = 5, 17, 20
    p = torch.randint(0, 37, (B, T0), generator=g, dtype=torch.int32).cuda()
    m.prefill(p, lens=lens, cache_bits=4, n_new=n_new, page_size=page_size)
    logits = [m._dec["logits"].clone()]
    for _ in range(n_new - 1):
        m.decode_step()
        logits.append(m._dec["logits"].clone())
    toks = m._dec["tokens"].clone()
    errors, picks = [], 0
    for b, n in enumerate(lens):
        m.prefill(p[b: b + 1], lens=[n], cache_bits=4, n_new=n_new, page_size=page_size)
        s = m._dec
        for i in range(n_new):
            got, want = logits[i][b].double(), s["logits"][0].double()
            errors.append(float((got - want).norm() / want.norm()))
            top = torch.topk(want, 2).values
            if float(top[0] - top[1]) > 4e-2 * float(want.norm()):
                assert int(toks[b, n + i]) == int(s["tokens"][0, n + i])
                picks += 1
            tok = toks[b, n + i]
            s["tokens"][0, n + i] = tok
            s["x"][0] = m.P["wte"][tok.long()] + m.P["wpe"][n + i]
            if i + 1 < n_new:
                m.decode_step()
    errors.sort()
    assert errors[-1] < 2e-2 and errors[len(errors) * 9 // 10] < 1e-3, errors[-12:]
    assert picks >= 25 and ops.read_status() == 0
