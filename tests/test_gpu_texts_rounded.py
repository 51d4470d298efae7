"""Texts drawn over 16-bit caches, against the model in 64 bits with keys and values rounded where the cache rounds them."""
import numpy as np
import pytest

from test_gpu_texts import CONFIGS, Texts64, check_draws

pytestmark = pytest.mark.gpu


class RoundedTexts64(Texts64):
    """A prompt's rows see one another as they are; rows behind it see the cache's keys and values, their own included."""
    cache, prompt, alone = None, 0, False

    def logits(self, tokens):
        torch, F, c = self.torch, self.torch.nn.functional, self.c
        wte, wpe, l1w, l1b, qw, qb, aw, ab, l2w, l2b, fw, fb, pw, pb, lw, lb = self.p
        n, C, NH = len(tokens), c.n_embd, c.n_head
        x = wte[torch.as_tensor(tokens, device="cuda").long()] + wpe[:n]
        mask = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for i in range(c.n_layer):
            q, k, v = (F.layer_norm(x, (C,), l1w[i], l1b[i]) @ qw[i].T + qb[i]).reshape(n, 3, NH, C // NH).permute(1, 2, 0, 3)
            ways = []
            for k_, v_ in ((k, v), [a.float().to(self.cache).double() for a in (k, v)]):
                s = (q @ k_.transpose(1, 2) / (C // NH) ** 0.5).masked_fill(mask, float("-inf"))
                ways.append((torch.softmax(s, -1) @ v_).transpose(0, 1).reshape(n, C))
            of_prompt = (torch.arange(n, device="cuda") < (0 if self.alone else self.prompt))[:, None]
            x = x + torch.where(of_prompt, *ways) @ aw[i].T + ab[i]
            x = x + F.gelu(F.layer_norm(x, (C,), l2w[i], l2b[i]) @ fw[i].T + fb[i], approximate="tanh") @ pw[i].T + pb[i]
        return (F.layer_norm(x[-1], (C,), lw, lb) @ wte.T)[:c.vocab_size].cpu().numpy()


# How near a border a coin may fall where the drawn token is another: keys and values are rounded alike but where fp32 and 64 bits (2^-20 apart, after three
# layers) lie on two sides of a rounding border.  bf16: steps of 2^-8 at most, so one element in 2^11, 2 of a layer's 2 * 24 * 96; a value's
# moves its column by 2^-8 / 20 of itself, a key's a score by 2^-8 / sqrt(hs), either 2e-4 at most behind a softmax over 20 tokens, so a cumulative
# probability by some 5e-4 over three layers, of which four times are allowed.  fp16: steps of an eighth, 8 times as many of them, which add up like
# sqrt(8): 3 / 8 of that, and the fp32 error itself besides.  How many draws: as over an fp32 cache.  (Measured: none of 475; of a model that rounds
# keys and values to another type 5 to 16 of a configuration's, or one beyond the border.)
@pytest.mark.parametrize("heads,hs,B,T,V,flash", CONFIGS)
@pytest.mark.parametrize("penalties", [(1.0, 0.0, 0.0), (1.3, 0.4, 0.2)])
@pytest.mark.parametrize("cache,near", [("TYPE_BF16", 2e-3), ("TYPE_FP16", 1e-3)])
@pytest.mark.parametrize("alone", [False, True])
def test_texts_over_a_cache_of_16_bits(bmb, cuda, heads, hs, B, T, V, flash, penalties, cache, near, alone):
    """`alone`: prompts of one token each, whose first row goes over the cache too."""
    t = bmb.Trainer(seed=7, max_seq_len=T, vocab_size=V, padded_vocab=-(-V // 128) * 128, n_layer=3, n_head=heads, n_embd=heads * hs, B=B, T=T,
                    use_flash=flash, math=bmb.MATH_FP32, fused=0)
    m = RoundedTexts64(cuda, t)
    m.cache, m.alone = cuda.bfloat16 if cache == "TYPE_BF16" else cuda.float16, alone
    rng = np.random.default_rng(3)
    steps = T // 2
    prompts = [list(map(int, rng.integers(0, V, k))) for k in ([1] * 5 if alone else (1, T // 3, 2, T - steps, 5))]
    out = t.generate_batch(prompts, steps, seed=11, temperature=0.9, repetition=penalties[0], frequency=penalties[1], presence=penalties[2], cache=getattr(bmb, cache))
    assert [len(o) for o in out] == [steps] * 5
    close = 0
    for i, (p, o) in enumerate(zip(prompts, out)):
        m.prompt = len(p)
        close += check_draws(m, p, o, 11 + i, 0.9, *penalties, near)
    assert close <= 3
    t.close()
