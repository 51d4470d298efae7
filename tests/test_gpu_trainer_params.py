"""Parameters that a trainer is given are in place, rounded copies too, when the call returns."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("math", ["MATH_TF32", "MATH_BF16"])
@pytest.mark.parametrize("fused", [0, 1])
@pytest.mark.parametrize("layers,heads,width", [(1, 2, 64), (3, 3, 192), (3, 4, 256)])
def test_rounded_weights_follow_the_parameters(bmb, cuda, layers, heads, width, fused, math, tmp_path):
    """The loss after parameters are set or loaded over others (zeros) is to the bit that after they are set where they are already: the
    forward pass has no atomics, so only weights rounded before the new parameters had arrived can tell them apart."""
    rng = np.random.default_rng(0)
    x = rng.integers(0, 65, (2, 65)).astype(np.int32)
    t = bmb.Trainer(seed=7, max_seq_len=64, vocab_size=65, padded_vocab=128, n_layer=layers, n_head=heads, n_embd=width, B=2, T=64, math=getattr(bmb, math), fused=fused)
    t.upload(np.ascontiguousarray(x[:, :-1]), np.ascontiguousarray(x[:, 1:]))
    w = np.empty(t.num_params, np.float32)
    t.get_params(w)
    w *= 3
    t.set_params(w)
    t.set_params(w)
    right = t.forward_loss()
    path = tmp_path / "w.bin"
    t.save(path)
    seen = []
    for _ in range(15):
        t.set_params(np.zeros_like(w))
        t.set_params(w)
        seen.append(t.forward_loss())
        t.set_params(np.zeros_like(w))
        t.load(path)
        seen.append(t.forward_loss())
    t.close()
    assert seen == [right] * 30
