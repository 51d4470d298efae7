"""Draws at low temperatures, where powers of probabilities are below fp32's numbers."""
import numpy as np
import pytest

from test_gpu_texts import Texts64, check_draws

pytestmark = pytest.mark.gpu


# Logits are off by some 1e-4 of these models (test_gpu_sampling: probabilities by up to 2.4e-5), so a cumulative probability by 1e-4 / (4 temperature) at most
# (the steepest slope of a share): 2.5e-3 at 0.01, of which four times are allowed; from 0.001 on the largest takes all, or the two largest share it in
# any way where they are within 1e-3 of one another, so that only draws apart from both would be seen as wrong.
@pytest.mark.parametrize("V", [65, 300])
@pytest.mark.parametrize("temperature,near", [(0.02, 5e-3), (0.01, 0.01), (0.001, 0.1)])
def test_cold_draws_are_of_the_likely_tokens(bmb, cuda, V, temperature, near):
    T = 48
    t = bmb.Trainer(seed=7, max_seq_len=T, vocab_size=V, padded_vocab=-(-V // 128) * 128, n_layer=3, n_head=3, n_embd=96, B=2, T=T, math=bmb.MATH_FP32)
    m = Texts64(cuda, t)
    starts = [3, 11, 40, V - 1]
    out = t.generate_batch([[s] for s in starts], T // 2, seed=21, temperature=temperature)
    close = sum(check_draws(m, [s], o, 21 + i, temperature, 1.0, 0.0, 0.0, near) for i, (s, o) in enumerate(zip(starts, out)))
    assert close <= 3
    for i, s in enumerate(starts):
        assert check_draws(m, [s], t.generate(s, T // 2, seed=21 + i, temperature=temperature), 21 + i, temperature, 1.0, 0.0, 0.0, near) <= 2
    t.close()


def test_as_cold_as_can_be(bmb, cuda):
    """The most likely token, to the last one, at temperatures whose inverse is infinity."""
    T, V = 48, 300
    t = bmb.Trainer(seed=7, max_seq_len=T, vocab_size=V, padded_vocab=384, n_layer=3, n_head=3, n_embd=96, B=2, T=T, math=bmb.MATH_FP32)
    m = Texts64(cuda, t)
    text = [5]
    for tok in t.generate_batch([[5]], T - 1, seed=1, temperature=1e-40)[0]:
        x = m.logits(text)
        assert x[tok] > x.max() - 2e-3
        text.append(tok)
    t.close()
