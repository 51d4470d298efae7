"""Serving operators at the ends of what they accept: counters that reach the last int, the largest finite numbers, infinities and NaN."""
import numpy as np
import pytest

import serving_oracle
from test_gpu_serving import TYPES, dtype_of, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before", [0, 1100])
def test_assign_of_as_many_tokens_as_an_int_counts(bmb, cuda, before):
    """max_tokens of 2^31 - 1, all of them asked for: a thread's step behind its last token ends beyond an int.  `before`: requests of a later
    stretch, which begins where the tokens end."""
    torch = cuda
    T, new = 2 ** 31 - 1, [5, 2 ** 31 - 1] + [3] * before
    n = len(new)
    tables = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    slots, positions, owners = (torch.full((T + 1,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    lens, free = i32(torch, [0] * n), i32(torch, [4])
    starts = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    bmb.call("bmb_pages_assign", tables, lens, slots, positions, owners, starts, free, lens, i32(torch, new), i32(torch, [3, 2, 1, 0]), free, n, 2, 16, 4, T,
             torch.cuda.current_stream().cuda_stream)
    assert slots[:5].tolist() == [0, 1, 2, 3, 4] and (slots[5:T] == -1).all()
    assert owners[:5].tolist() == [0] * 5 and (owners[5:T] == 1).all() and positions[:5].tolist() == [0, 1, 2, 3, 4]
    for at in range(5, T, 1 << 28):
        to = min(at + (1 << 28), T)
        assert torch.equal(positions[at:to], torch.arange(at - 5, to - 5, dtype=torch.int32, device="cuda"))
    assert [int(x[T]) for x in (slots, positions, owners)] == [77] * 3
    assert starts.tolist() == [0, 5] + [T] * (n - 1) and lens.tolist() == [5] + [0] * (n - 1) and int(free) == 3


def test_attention_of_rows_that_are_longer_than_an_int_counts(bmb, cuda):
    """2^25 heads of 64: a row of outputs has 2^31 elements, and all of them are written, of a request without tokens too."""
    torch = cuda
    heads, hs = 1 << 25, 64
    k, v = (torch.randn(1, 16, 1, hs, device="cuda").bfloat16() for _ in range(2))
    q = torch.ones(heads * hs, device="cuda")
    out, lse = torch.full((2, heads * hs), 77.0, device="cuda"), torch.full((2, heads), 77.0, device="cuda")
    ws = torch.empty(bmb.paged_attention_workspace(heads, 1, hs), dtype=torch.uint8, device="cuda")
    bmb.call("bmb_paged_attention", out, lse, q, bmb.KvCache.of(k, v), i32(torch, [[0], [0]]), i32(torch, [0, 1]), 2, heads, 0, heads * hs, 1, 0.0, ws, ws.numel(),
             torch.cuda.current_stream().cuda_stream)
    for part in out[0].split(1 << 28):
        assert (part == 0).all()
    for part in out[1].view(heads, hs).split(1 << 22):
        assert (part == v[0, 0].float()).all()               # (one token: its weight is 1, and a bf16 value's product with that is exact)
    assert (lse[0] == -float("inf")).all() and (lse[1] == 0).all()
