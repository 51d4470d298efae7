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


# ---- infinities, NaN, the largest numbers -------------------------------------------------------------------------------

def formula(torch, q, k, v, lens, scale):
    """Softmax attention of q [n, heads, hs] over k and v [n, longest, kv, hs] in 64 bits, with what IEEE makes of infinities and NaN, a score
    of -infinity having weight 0; and how far fp32 may be from it where it is finite.  As serving_oracle.attention_bounds has it (errors of a score
    d; of a weight twice that), but for each column by itself and with two roundings for each token in the sums, which are one chain
    where a sum is not finite or an element is near the largest.  Of an fp16 cache the rest of an element of q behind its first piece is a half too, in
    units in which the row's largest is 2^14 at least: off by 2^-25 (half the smallest half) at most, 2^-39 of the row's largest, besides what is counted above."""
    n, heads, hs = q.shape
    group, u = heads // k.shape[2], 2.0 ** -24
    out, bound = torch.zeros(2, n, heads, hs, dtype=torch.float64, device=q.device)
    lse, lse_bound = torch.full((n, heads), -float("inf"), dtype=torch.float64, device=q.device), torch.zeros(n, heads, dtype=torch.float64, device=q.device)
    for i in range(n):
        for h in range(heads):
            x, y = k[i, :lens[i], h // group].double(), v[i, :lens[i], h // group].double()
            terms = x * q[i, h].double()
            s = terms.sum(1) * scale
            if torch.isnan(s).any() or (s == float("inf")).any():
                out[i, h] = lse[i, h] = float("nan")
                continue
            some = s > -float("inf")
            if not some.any():
                continue
            top = s.max()
            w = torch.exp(s - top)
            out[i, h] = (w[:, None] * y).sum(0) / w.sum()
            lse[i, h] = top + torch.log(w.sum())
            d = (hs / 4 + 8) * u * (terms[some].abs().sum(1) * abs(scale)).max()
            if k.dtype == torch.float16:
                d = d + 2.0 ** -39 * q[i, h].double().abs().max() * (x[some].abs().sum(1) * abs(scale)).max()
            rest = (2 * lens[i] + 64) * u
            bound[i, h] = (2 * d + rest) * torch.where(torch.isfinite(y), y, 0.0).abs().amax(0)
            lse_bound[i, h] = d + rest + 2 * u * lse[i, h].abs()
    return out, bound, lse, lse_bound


def check_limits(bmb, torch, q, k, v, lens, scale, width, loose=None, least=0.0):
    """Against the formula; `width`: pages of a row of the tables, by which attention is divided.  loose: (request, head, column) where NaN and
    an infinity are alike, a weight being 0 in fp32 that is not in 64 bits.
    least: what an output may be off besides."""
    n, heads, hs = q.shape
    longest, kv = k.shape[1:3]
    page = 16
    each = -(-longest // page)
    ids = torch.randperm(n * each)
    tables = torch.full((n, width), -1, dtype=torch.int32)
    tables[:, :each] = ids.view(n, each)
    pools = []
    for x in (k, v):
        pool = torch.full((n * each, page, kv, hs), float("nan"), dtype=x.dtype, device="cuda")
        rows = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, each * page - longest)).view(n * each, page, kv, hs)
        pool[ids.cuda()] = rows
        pools.append(pool)
    out, lse = torch.full((n, heads, hs), 77.0, device="cuda"), torch.full((n, heads), 77.0, device="cuda")
    ws = torch.empty(bmb.paged_attention_workspace(heads, kv, hs), dtype=torch.uint8, device="cuda")
    bmb.call("bmb_paged_attention", out, lse, q, bmb.KvCache.of(*pools), tables.cuda(), i32(torch, lens), n, heads, heads * hs, heads * hs, width, scale, ws,
             ws.numel(), torch.cuda.current_stream().cuda_stream)
    want, bound, want_lse, lse_bound = formula(torch, q, k, v, lens, scale)
    for got, want, bound in ((out.double(), want, bound + least), (lse.double(), want_lse, lse_bound)):
        finite = torch.isfinite(want)
        same = torch.where(finite, (got - want).abs() <= bound, (got == want) | (torch.isnan(got) & torch.isnan(want)))
        if loose is not None and got.dim() == 3:
            same[loose] = ~torch.isfinite(got[loose])
        assert same.all(), (torch.argwhere(~same)[:4].tolist(), got[~same][:4].tolist(), want[~same][:4].tolist(), bound[~same][:4].tolist())
    return out


def texts(torch, name, n, longest, heads, kv, hs, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    dt = dtype_of(torch, name)
    return r(n, heads, hs), r(n, longest, kv, hs).to(dt), r(n, longest, kv, hs).to(dt)


# heads, kv heads, head size, longest text, pages of a table's row: a cluster for each head; one block; the line, its heads in one
# warp, in several of a block, over blocks
FORMS = [(6, 2, 64, 40, 4), (2, 1, 32, 700, 44), (3, 3, 128, 300, 20), (18, 1, 64, 150, 10), (12, 12, 32, 33, 3000), (18, 1, 64, 300, 3000), (2, 1, 128, 6000, 3000),
         (1, 1, 128, 20000, 3000)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,hs,longest,width", FORMS)
def test_a_value_that_is_not_finite_is_seen_however_small_its_weight(bmb, cuda, name, heads, kv, hs, longest, width):
    """One token takes all and the other tokens' weights are 0 in fp32, those of whole parts of the text together; 0 times NaN is NaN."""
    torch = cuda
    for at in (0, longest // 3, longest - 2):
        q, k, v = texts(torch, name, 2, longest, heads, kv, hs)
        k[:, :, :, 0] = 0
        k[:, longest // 2, :, 0] = 30
        q[:, :, 0] = 30
        v[0, at, 0, 5], v[0, at + 1, kv - 1, 9], v[1, at, kv - 1, 3] = float("nan"), float("inf"), -float("inf")
        group = heads // kv
        loose = torch.zeros(2, heads, hs, dtype=torch.bool, device="cuda")
        loose[0, :group, 5] = loose[0, -group:, 9] = loose[1, -group:, 3] = True
        check_limits(bmb, torch, q, k, v, [longest, longest - 1], 1.0, width, loose)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,hs,longest,width", FORMS)
@pytest.mark.parametrize("what", ["key", "value", "query", "both"])
def test_infinities_do_what_they_do_in_the_formula(bmb, cuda, name, heads, kv, hs, longest, width, what):
    """Keys, values and queries of both infinities, beside queries and weights of both signs and zeros: scores of -infinity have no weight, those of
    infinity and NaN leave NaN, an infinite value stays what it is unless it meets the other infinity."""
    torch, inf = cuda, float("inf")
    for seed in range(3):
        q, k, v = texts(torch, name, 3, longest, heads, kv, hs, seed)
        a, b = longest // 5, longest - 3
        if what == "key":
            q[:, :, 3] = q[:, :, 3].abs()                     # (whole texts whose scores are -infinity, and others whose are infinity)
            q[1, 0, 4] = 0.0
            k[0, a, 0, 3], k[1, b, kv - 1, 4], k[2, a, 0, 5], k[2, b, 0, 6] = -inf, inf, inf, -inf
            k[0, b, 0, 3] = -inf
        elif what == "value":
            v[0, a, 0, 3], v[0, b, 0, 4], v[1, a, kv - 1, 5], v[1, b, kv - 1, 5], v[2, b, 0, 0] = inf, -inf, inf, -inf, inf
        elif what == "query":
            q[0, 0, 3], q[1, heads - 1, 4], q[2, 0, 0] = inf, -inf, float("nan")
        else:
            q[:, :, 3] = 1.0
            k[0, :, 0, 3] = -inf                              # nothing of a weight is left
            k[1, a:, :, 3] = -inf
            v[1, 0, 0, 7] = inf
        check_limits(bmb, torch, q, k, v, [longest, longest, longest - 1], hs ** -0.5, width)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,hs,longest,width", FORMS)
def test_the_largest_numbers_are_finite(bmb, cuda, name, heads, kv, hs, longest, width):
    """The largest and lowest value of the cache's type among values, and keys and queries of that size whose scores are ordinary."""
    torch = cuda
    for seed in range(2):
        q, k, v = texts(torch, name, 2, longest, heads, kv, hs, seed)
        most = torch.finfo(k.dtype).max
        v[0, longest // 2, 0, 3], v[0, 1, kv - 1, 4], v[1, longest - 2, 0, 5] = most, -most, most
        check_limits(bmb, torch, q, k, v, [longest, longest - 1], hs ** -0.5, width)
        k[0, longest // 3, :, 2], k[1, 0, :, 2] = most, -most
        q[:, :, 2] = 8.0 / most
        check_limits(bmb, torch, q, k, v, [longest, longest - 1], hs ** -0.5, width)
        q[:, :, 2], k[:, :, :, 2] = torch.finfo(torch.float32).max, 0.0
        check_limits(bmb, torch, q, k, v, [longest, longest - 1], hs ** -0.5, width)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv,hs,longest,width", FORMS)
def test_the_smallest_numbers(bmb, cuda, name, heads, kv, hs, longest, width):
    """Values down to the type's smallest ones: of an fp32 value the second piece ends at 2^-136 (its 10 bits behind 2^-126), so each of the two
    products that a weight's pieces make with it is off by that at most, and the weights' sum is 1."""
    torch = cuda
    q, k, v = texts(torch, name, 2, longest, heads, kv, hs)
    tiny = torch.finfo(v.dtype).tiny
    for scale in (64.0, 1.0, 2.0 ** -6):
        check_limits(bmb, torch, q, k, (v.double() * tiny * scale).to(v.dtype), [longest, longest - 1], hs ** -0.5, width, least=2.0 ** -135)
