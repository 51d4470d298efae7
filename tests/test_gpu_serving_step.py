"""A step of several requests as the documents have it: rows of new tokens one behind the other, queries gathered from them."""
import numpy as np
import pytest

import serving_oracle
from test_gpu_serving import Serving, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,heads,kv,hs,page", [("fp32", 4, 2, 64, 16), ("bf16", 6, 6, 32, 8)])
def test_a_step_of_requests_that_add_different_numbers_of_tokens(bmb, cuda, name, heads, kv, hs, page):
    """Prompts, single tokens, requests that rest and requests that have ended, in one step: row starts[i + 1] - 1 is request i's newest token,
    and its attention is over its own text.  (Row i is another request's, as soon as one before it adds none or several.)"""
    torch, n = cuda, 7
    s = Serving(bmb, torch, n, heads, kv, hs, page, 400 // page, 300 // page, 250, name)
    rng = np.random.default_rng(heads)
    C, st, texts, moved = heads * hs, torch.cuda.current_stream().cuda_stream, [[] for _ in range(n)], 0
    q = torch.empty(n, C, device="cuda")
    for step in range(25):
        new = np.array([int(rng.integers(2, 30)) if not t and rng.random() < 0.5 else int(len(t) > 0 and rng.random() < 0.7) for t in texts])
        if step % 5 == 4:
            new[0] = 0                                        # (nothing of the first one: starts[1] is 0)
        s.new.copy_(i32(torch, new))
        s.qkv.copy_(torch.randn(s.room, s.qkv.shape[1], device="cuda"))
        s.bmb.call("bmb_pages_assign", s.tables, s.lens, s.slots, s.positions, s.owners, s.starts, s.free, s.lens, s.new, s.stack, s.free, n, s.tables.shape[1],
                   page, s.pages, s.room, st)
        s.bmb.call("bmb_paged_kv_write", s.cache, s.qkv[:, C:], s.qkv[:, C + kv * hs:], s.qkv.shape[1], s.slots, s.room, st)
        torch.index_select(s.qkv[:, :C], 0, (s.starts[1:] - 1).clamp(min=0), out=q)
        s.bmb.call("bmb_paged_attention", s.out, None, q, s.cache, s.tables, s.lens, n, heads, C, C, s.tables.shape[1], hs ** -0.5, s.ws, s.ws.numel(), st)
        lens, begins = s.lens.tolist(), np.concatenate([[0], np.cumsum(new)])
        for i in range(n):
            if lens[i] == len(texts[i]) + new[i]:
                texts[i] += [s.qkv[begins[i] + j].clone() for j in range(new[i])]
            assert lens[i] == len(texts[i])
            if new[i] == 0 or not texts[i] or not torch.equal(texts[i][-1], s.qkv[begins[i + 1] - 1]):
                continue
            moved += begins[i + 1] - 1 != i
            rows = torch.stack(texts[i])[:, C:].to(s.k.dtype).reshape(1, len(texts[i]), 2, kv, hs)
            want, _, size, top, count = serving_oracle.attention(torch, s.qkv[begins[i + 1] - 1, :C].reshape(1, heads, hs), rows[:, :, 0], rows[:, :, 1], [[0]],
                                                                 [len(texts[i])], hs ** -0.5)
            assert ((s.out[i].view(1, heads, hs).double() - want).abs() <= serving_oracle.attention_bounds(hs, size, top, count)[0][..., None]).all()
        done = np.array([len(t) > 50 or rng.random() < 0.1 for t in texts])
        s.done.copy_(i32(torch, done))
        s.release(st)
        texts = [[] if d else t for t, d in zip(texts, done)]
    assert moved > 20
