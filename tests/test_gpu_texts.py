"""Several texts drawn at once from a model (a paged cache, attention over it, penalties), against the model in 64 bits (plain torch)."""
import numpy as np
import pytest

from test_gpu_sampling import Model64

pytestmark = pytest.mark.gpu


class Texts64(Model64):
    def logits(self, tokens):
        torch, F, c = self.torch, self.torch.nn.functional, self.c
        wte, wpe, l1w, l1b, qw, qb, aw, ab, l2w, l2b, fw, fb, pw, pb, lw, lb = self.p
        n, C, NH = len(tokens), c.n_embd, c.n_head
        x = wte[torch.as_tensor(tokens, device="cuda").long()] + wpe[:n]
        mask = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for i in range(c.n_layer):
            q, k, v = (F.layer_norm(x, (C,), l1w[i], l1b[i]) @ qw[i].T + qb[i]).reshape(n, 3, NH, C // NH).permute(1, 2, 0, 3)
            s = (q @ k.transpose(1, 2) / (C // NH) ** 0.5).masked_fill(mask, float("-inf"))
            x = x + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, C) @ aw[i].T + ab[i]
            x = x + F.gelu(F.layer_norm(x, (C,), l2w[i], l2b[i]) @ fw[i].T + fb[i], approximate="tanh") @ pw[i].T + pb[i]
        return (F.layer_norm(x[-1], (C,), lw, lb) @ wte.T)[:c.vocab_size].cpu().numpy()


def check_draws(m, prompt, drawn, seed, temperature, repetition, frequency, presence, near):
    """Walks along the drawn tokens: each is the one that the model in 64 bits draws there, or next to it with the coin within `near` of
    the border between them.  How many were."""
    bits = np.random.MT19937()
    bits._legacy_seeding(seed)
    text, close = list(prompt), 0
    for tok in drawn:
        # the generator's next number as a float below 1, the way the C++ library makes one
        coin = float(min(np.float32(bits.random_raw()) * np.float32(2.0 ** -32), np.nextafter(np.float32(1), np.float32(0))))
        x = m.logits(text)
        for v in set(text):
            times = text[len(prompt):].count(v)
            x[v] = x[v] / repetition if x[v] > 0 else x[v] * repetition
            x[v] -= frequency * times + presence * (times > 0)
        p = np.exp((x - x.max()) / temperature)
        cdf = np.cumsum(p / p.sum())
        want = int(np.searchsorted(cdf, coin, side="right"))
        if tok != want:
            assert 0 <= tok < len(cdf) and abs(coin - cdf[min(tok, want)]) < near and abs(coin - cdf[max(tok, want) - 1]) < near, (tok, want, coin)
            close += 1
        text.append(int(tok))
    return close


CONFIGS = [(3, 32, 4, 48, 65, 1), (2, 64, 1, 70, 300, 1), (2, 128, 3, 33, 65, 1), (3, 64, 2, 40, 65, 0)]   # heads, head size, B, T, vocabulary, flash


# How near a border a coin may fall: in fp32 test_gpu_sampling measured up to 2.4e-5 between these models' probabilities and theirs in 64
# bits, 1e-4 is four times that; a cumulative sum of them is off by no more than their sum of differences, which this bounds too as most
# tokens' are far smaller.  Keys and values of 8 bits (bf16) are off by 2^-9 each; through three layers of gains and weights at three times their
# usual size a probability may be off by some tens of that.
@pytest.mark.parametrize("heads,hs,B,T,V,flash", CONFIGS)
@pytest.mark.parametrize("penalties", [(1.0, 0.0, 0.0), (1.3, 0.4, 0.2)])
@pytest.mark.parametrize("cache,near", [("TYPE_FP32", 2e-4), ("TYPE_BF16", 0.1), ("TYPE_FP16", 0.02)])
def test_texts_drawn_together(bmb, cuda, heads, hs, B, T, V, flash, penalties, cache, near):
    t = bmb.Trainer(seed=7, max_seq_len=T, vocab_size=V, padded_vocab=-(-V // 128) * 128, n_layer=3, n_head=heads, n_embd=heads * hs, B=B, T=T,
                    use_flash=flash, math=bmb.MATH_FP32, fused=0)
    m = Texts64(cuda, t)
    rng = np.random.default_rng(3)
    steps = T // 2
    prompts = [list(map(int, rng.integers(0, V, k))) for k in (1, T // 3, 2, T - steps, 5)]
    how = dict(temperature=0.9, repetition=penalties[0], frequency=penalties[1], presence=penalties[2], cache=getattr(bmb, cache))
    out = t.generate_batch(prompts, steps, seed=11, **how)
    assert [len(o) for o in out] == [steps] * 5
    close = sum(check_draws(m, p, o, 11 + i, 0.9, *penalties, near) for i, (p, o) in enumerate(zip(prompts, out)))
    assert close <= (3 if cache == "TYPE_FP32" else 5 * steps // 4)
    t.close()


@pytest.mark.parametrize("math", ["MATH_TF32", "MATH_BF16"])
@pytest.mark.parametrize("fused", [0, 1])
def test_texts_in_the_other_arithmetics(bmb, cuda, math, fused):
    """Runs on trainers of the tensor-core modes too; draws follow the model to these modes' precision."""
    t = bmb.Trainer(seed=7, max_seq_len=64, vocab_size=65, padded_vocab=128, n_layer=3, n_head=3, n_embd=192, B=2, T=64, math=getattr(bmb, math), fused=fused)
    m = Texts64(cuda, t)
    prompts = [[1, 2, 3], [5], list(range(30))]
    out = t.generate_batch(prompts, 20, seed=5, temperature=0.9)
    close = sum(check_draws(m, p, o, 5 + i, 0.9, 1.0, 0.0, 0.0, 0.02 if math == "MATH_TF32" else 0.15) for i, (p, o) in enumerate(zip(prompts, out)))
    assert close <= 15
    t.close()


def test_a_text_ends_with_its_stop_token(bmb, cuda):
    """Texts that end give their pages back and rest; the others' draws are what they are without that."""
    t = bmb.Trainer(seed=3, max_seq_len=96, vocab_size=20, padded_vocab=128, n_layer=2, n_head=2, n_embd=64, B=1, T=96, math=bmb.MATH_FP32)
    prompts = [[i % 20] for i in range(40)]
    whole = t.generate_batch(prompts, 60, seed=100)
    ended = t.generate_batch(prompts, 60, seed=100, stop=7)
    assert sum(len(a) < 60 for a in ended) > 10
    for a, b in zip(whole, ended):
        assert b == (a[:a.index(7) + 1] if 7 in a else a)
    t.close()


def test_one_text_is_what_generate_draws(bmb, cuda):
    t = bmb.Trainer(seed=9, max_seq_len=64, vocab_size=65, padded_vocab=128, n_layer=4, n_head=4, n_embd=128, B=2, T=64, math=bmb.MATH_FP32)
    texts = [t.generate(3, 50, seed=s, temperature=0.8) for s in range(8)]
    same = [t.generate_batch([[3]], 50, seed=s, temperature=0.8)[0] == texts[s] for s in range(8)]
    together = t.generate_batch([[3]] * 8, 50, seed=0, temperature=0.8)
    # 400 draws from 65 tokens, probabilities within 1e-5: one that falls otherwise is a chance of a few per cent, and spoils one text
    assert sum(same) >= 7 and sum(a == b for a, b in zip(together, texts)) >= 7
    t.close()


def test_texts_leave_the_trainer_alone(bmb, cuda):
    """Between two steps: parameters, gradients, the resident batch and its loss are what they were, to the bit.  (The losses of two
    trainings cannot say so: the token embedding's gradient is added up by atomics, in another order each time.)"""
    t = bmb.Trainer(seed=9, max_seq_len=32, vocab_size=65, padded_vocab=128, n_layer=2, n_head=2, n_embd=64, B=2, T=32, math=bmb.MATH_FP32)
    rng = np.random.default_rng(0)
    for step in range(1, 4):
        x = rng.integers(0, 65, (2, 33)).astype(np.int32)
        t.upload(np.ascontiguousarray(x[:, :-1]), np.ascontiguousarray(x[:, 1:]))
        t.step(1e-3, step)
        seen = []
        for _ in range(2):
            params, grads = np.empty(t.num_params, np.float32), np.empty(t.num_params, np.float32)
            t.get_params(params)
            t.get_grads(grads)
            seen.append((params, grads, t.forward_loss()))
            t.generate_batch([[1], [2, 3]], 10, seed=1, frequency=0.5)
        for a, b in zip(*seen):
            assert np.array_equal(a, b)
    t.close()


def test_refusals(bmb, cuda):
    t = bmb.Trainer(seed=9, max_seq_len=32, vocab_size=65, padded_vocab=128, n_layer=1, n_head=2, n_embd=64, B=1, T=32, math=bmb.MATH_FP32)
    assert t.generate_batch([], 5, seed=1) == [] and t.generate_batch([[1]], 0, seed=1) == [[]]
    for prompts, steps, how in [([[1] * 20], 13, {}), ([[]], 3, {}), ([[65]], 3, {}), ([[-1]], 3, {}), ([[1]], 3, dict(temperature=0.0)), ([[1]], 3, dict(repetition=0.0)),
                                ([[1]], 3, dict(frequency=float("nan"))),
                                ([[1]], 3, dict(presence=float("inf"))), ([[1]], 3, dict(temperature=float("inf"))), ([[1]], 3, dict(cache=3)), ([[1]], -1, {})]:
        with pytest.raises(bmb.BmbError):
            t.generate_batch(prompts, steps, seed=1, **how)
    assert len(t.generate_batch([[1] * 20], 12, seed=1)[0]) == 12
    t.close()
    wide = bmb.Trainer(seed=9, max_seq_len=32, vocab_size=65, padded_vocab=128, n_layer=1, n_head=1, n_embd=256, B=1, T=32, use_flash=0, math=bmb.MATH_FP32)
    with pytest.raises(bmb.BmbError, match="head size 256"):
        wide.generate_batch([[1]], 3, seed=1)
    wide.close()


def test_the_command_draws_several_texts(bmb, cuda, tmp_path):
    import os
    import subprocess
    t = bmb.Trainer(seed=9, max_seq_len=32, vocab_size=5, padded_vocab=128, n_layer=1, n_head=2, n_embd=64, B=1, T=32, math=bmb.MATH_FP32)
    t.save(tmp_path / "m.bin", itos=b"\nabcd")
    exe = os.path.join(os.path.dirname(bmb.LIB_PATH), "bmb_train_gpt")
    got = subprocess.run([exe, "--load", str(tmp_path / "m.bin"), "--len", "400", "--texts", "3", "--frequency", "0.2", "--seed", "4"], capture_output=True, text=True,
                         timeout=120)
    assert got.returncode == 0 and "[text 2]" in got.stdout and "[text 3]" in got.stdout, got
    want = t.generate_batch([[0]] * 3, 31, seed=5, temperature=0.8, frequency=0.2)
    for text in want:
        assert "".join("\nabcd"[tok] for tok in text) in got.stdout
    t.close()
