"""Serving several requests: pages, cache writes, attention over pages and adjusted logits against plain forms in 64 bits (whole
numbers and single roundings exactly), at the sizes, layouts and lengths where they can go wrong, and as a step runs them together."""
import numpy as np
import pytest

import serving_oracle

pytestmark = pytest.mark.gpu
TYPES = ["fp32", "bf16", "fp16"]


def dtype_of(torch, name):
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[name]


def i32(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


# ---- pages ----------------------------------------------------------------------------------------------------------

def run_assign(bmb, torch, tables, lens, new, stack, free, page, pages, T, optional=True, in_place=False):
    n, width = tables.shape
    t, l, a, s, f = (i32(torch, x) for x in (tables, lens, new, stack, [free]))
    lo, fo = (l, f) if in_place else (torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"), torch.full((2,), 77, dtype=torch.int32, device="cuda"))
    slots, pos, own = (torch.full((T + 5,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    starts = torch.full((n + 2,), 77, dtype=torch.int32, device="cuda")
    bmb.call("bmb_pages_assign", t, lo, slots, pos if optional else None, own if optional else None, starts if optional else None, fo, l, a, s, f, n,
             width, page, pages, T, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = serving_oracle.assign(np.asarray(tables), lens, new, stack, free, page, pages, T)
    assert np.array_equal(t.cpu().numpy(), want[0])
    assert np.array_equal(lo[:n].cpu().numpy(), want[1])
    assert np.array_equal(slots[:T].cpu().numpy(), want[2])
    assert int(fo[0]) == want[6]
    assert (slots[T:] == 77).all() and (in_place or (lo[n:] == 77).all() and (fo[1:] == 77).all())
    if optional:
        assert np.array_equal(pos[:T].cpu().numpy(), want[3]) and np.array_equal(own[:T].cpu().numpy(), want[4])
        assert np.array_equal(starts[:n + 1].cpu().numpy(), want[5])
        assert (pos[T:] == 77).all() and (own[T:] == 77).all() and (starts[n + 1:] == 77).all()
    assert np.array_equal(s.cpu().numpy(), np.asarray(stack))


# n, page, table width, longest, longest new, share of pages that are free, tokens left out of max_tokens (negative: padding)
ASSIGN = [(1, 16, 4, 40, 20, 2.0, -3), (1, 1, 90, 40, 50, 1.0, 0), (7, 16, 8, 100, 30, 0.6, -9), (64, 16, 64, 1000, 1, 1.0, 0),
          (33, 24, 12, 200, 100, 1.5, 100), (300, 8, 40, 300, 30, 0.5, -1000), (1024, 16, 10, 150, 2, 0.9, -1), (1025, 100, 3, 250, 60, 0.8, -40),
          (2500, 7, 9, 50, 5, 0.7, 500), (5, 4096, 3, 9000, 3500, 1.0, -1), (16, 16, 600, 5, 9000, 0.8, 0), (3, 128, 300, 9, 38000, 0.9, -70000)]


@pytest.mark.parametrize("n,page,width,longest,new_longest,room,cut", ASSIGN)
@pytest.mark.parametrize("in_place", [False, True])
def test_assign(bmb, cuda, n, page, width, longest, new_longest, room, cut, in_place):
    rng = np.random.default_rng(n * 7 + page)
    lens, new = rng.integers(0, longest + 1, n), rng.integers(0, new_longest + 1, n)
    lens[rng.random(n) < 0.1] *= -1                                  # negative lengths count as none
    new[rng.random(n) < 0.1] = -1
    held = -(-np.maximum(lens, 0) // page)
    asked = int(np.maximum(-(-(np.maximum(lens, 0) + np.maximum(new, 0)) // page) - held, 0).sum())
    free = int(room * asked)
    pages = free + int(np.minimum(held, width).sum()) + 3
    ids = rng.permutation(pages)
    tables, at = np.full((n, width), -1, np.int64), 0
    for i in range(n):
        k = min(int(held[i]), width)
        tables[i, :k] = ids[at:at + k]
        at += k
    if n > 4:                                                        # pages that are none: a corrupt table gives no slot
        for i, bad in ((1, -5), (3, pages), (4, 2 ** 31 - 1)):
            tables[i, max(int(held[i]) - 1, 0) % width] = bad
    stack = np.zeros(pages, np.int64)
    stack[:free] = ids[at:at + free]
    T = max(int(np.maximum(new, 0).sum()) - cut, 0)
    run_assign(bmb, cuda, tables, lens, new, stack, free, page, pages, T, optional=not in_place, in_place=in_place)


def test_assign_corners(bmb, cuda):
    none = np.zeros((0, 4), np.int64)
    run_assign(bmb, cuda, none, [], [], [1, 2, 3], 2, 16, 3, 10)
    run_assign(bmb, cuda, np.full((2, 4), -1), [0, 0], [1, 1], np.arange(6), 99, 16, 6, 10)         # more free pages than there are
    run_assign(bmb, cuda, np.full((2, 4), -1), [0, 0], [1, 1], np.arange(6), -4, 16, 6, 10)         # fewer than none
    run_assign(bmb, cuda, np.full((2, 4), -1), [0, 0], [1, 1], np.arange(6), 6, 16, 6, 0)           # no room for tokens
    run_assign(bmb, cuda, np.full((3, 4), -1), [0, 0, 0], [60, 3, 70], [9, -1, 2 ** 31 - 1, 3], 4, 16, 4, 140)   # a corrupt stack
    big = 2 ** 31 - 1
    run_assign(bmb, cuda, np.full((3, 4), -1), [big, 5, big], [big, 2, 3], np.arange(6), 6, 16, 6, 10)   # lengths whose sums pass an int
    run_assign(bmb, cuda, np.full((3, 4), -1), [0, 2, 0], [40, 2, 2], [5, 4, 3, 2], 2, 16, 6, 50)   # the first waits, a later one needs no page


def run_release(bmb, torch, stack, free, lens, tables, done, page, pages, in_place=False):
    s, l, t, d, f = (i32(torch, x) for x in (stack, lens, tables, done, [free]))
    n = len(lens)
    lo, fo = (l, f) if in_place else (torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"), torch.full((2,), 77, dtype=torch.int32, device="cuda"))
    bmb.call("bmb_pages_release", s, fo, lo, f, l, t, d, n, np.asarray(tables).shape[1], page, pages, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = serving_oracle.release(np.asarray(stack), free, lens, np.asarray(tables), done, page, pages)
    assert np.array_equal(s.cpu().numpy(), want[0]) and int(fo[0]) == want[1] and np.array_equal(lo[:n].cpu().numpy(), want[2])
    assert in_place or (lo[n:] == 77).all() and (fo[1:] == 77).all()
    assert np.array_equal(t.cpu().numpy(), np.asarray(tables))


@pytest.mark.parametrize("n,page,longest,share,in_place", [(1, 16, 200, 1.0, False), (5, 1, 70, 0.5, True), (64, 16, 1024, 0.25, False),
                                                            (200, 24, 3001, 0.8, True), (1023, 8, 99, 0.5, False), (1030, 16, 300, 1.0, True),
                                                            (2100, 128, 400, 0.3, False), (40, 16, 50000, 0.6, False),
                                                            (300, 16, 30000, 0.9, True), (3, 1, 200000, 1.0, False)])
def test_release(bmb, cuda, n, page, longest, share, in_place):
    rng = np.random.default_rng(n + page)
    lens = rng.integers(-3, longest + 1, n)
    held = -(-np.maximum(lens, 0) // page)
    pages, width = int(held.sum()) + 6, max(int(held.max()), 1)
    ids, at = rng.permutation(pages), 0
    tables = np.full((n, width), -1, np.int64)
    for i in range(n):
        tables[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    tables[rng.random((n, width)) < 0.02] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31])   # entries that are no pages
    stack = np.full(pages, -7, np.int64)
    stack[:pages - at] = ids[at:]
    run_release(bmb, cuda, stack, pages - at, lens, tables, (rng.random(n) < share) * rng.integers(1, 9, n), page, pages, in_place)


def test_release_corners(bmb, cuda):
    ends = np.zeros(1500, np.int64)
    ends[[0, 1, 700, 1023, 1024, 1499]] = 1                                                         # few among many
    run_release(bmb, cuda, np.zeros(4600, np.int64), 11, np.arange(1500) % 49, np.arange(4500).reshape(1500, 3), ends, 16, 4600)
    t = np.array([[0, 1, 2], [3, 4, 5]])
    run_release(bmb, cuda, np.zeros(6, np.int64), 0, [], np.zeros((0, 3), np.int64), [], 16, 6)
    run_release(bmb, cuda, np.zeros(6, np.int64), 4, [48, 48], t, [1, 1], 16, 6)                    # no room for all of them
    run_release(bmb, cuda, np.zeros(6, np.int64), -3, [2 ** 31 - 1, 1], t, [1, 1], 16, 6)           # a length beyond its table
    run_release(bmb, cuda, np.zeros(6, np.int64), 99, [48, 48], t, [1, 0], 16, 6)
    run_release(bmb, cuda, np.zeros(6, np.int64), 2, [48, 48], t, [0, 0], 16, 6)


# ---- cache ----------------------------------------------------------------------------------------------------------

LAYOUTS = ["tokens", "heads", "interleaved"]


def pool(torch, layout, pages, page, heads, hs, dtype, fill=None):
    """k and v as (pages, page, heads, hs) views of memory in another order; `tokens`: as they are seen."""
    if layout == "interleaved":                                       # keys and values of a page side by side, padded rows
        both = torch.empty(pages, 2, page, heads, hs + 8, dtype=dtype, device="cuda")
        k, v = both[:, 0, :, :, :hs], both[:, 1, :, :, :hs]
    elif layout == "heads":
        k, v = (torch.empty(pages, heads, page, hs, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        k, v = (torch.empty(pages, page, heads, hs, dtype=dtype, device="cuda") for _ in range(2))
    if fill is not None:
        k.fill_(fill)
        v.fill_(fill)
    return k, v


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tokens,heads,hs,page,shift,pad", [(1, 1, 32, 1, 0, 0), (37, 3, 64, 24, 0, 0), (37, 3, 64, 24, 1, 0), (300, 12, 64, 16, 0, 3),
                                                            (70, 8, 128, 100, 2, 5), (5000, 2, 32, 64, 0, 4)])
def test_kv_write(bmb, cuda, name, layout, tokens, heads, hs, page, shift, pad):
    torch, dt = cuda, dtype_of(cuda, name)
    pages = -(-tokens // page) + 2
    k, v = pool(torch, layout, pages, page, heads, hs, dt, 5.0)
    torch.manual_seed(tokens + hs)
    width = 2 * heads * hs + 64 + pad
    rows = torch.randn(tokens * width + 8, device="cuda")[shift:shift + tokens * width].view(tokens, width) * 30
    rows[0, :6] = torch.tensor([0.0, -0.0, 7e4, -1e30, float("inf"), float("nan")], device="cuda")
    slots = torch.randperm(pages * page, device="cuda")[:tokens].int()
    slots[tokens // 3::7] = -1
    if tokens > 10:
        slots[2], slots[5] = pages * page, -2 ** 31
    before = k.clone(), v.clone()
    C = heads * hs
    bmb.call("bmb_paged_kv_write", bmb.KvCache.of(k, v), rows, rows[:, C:], width, slots, tokens, torch.cuda.current_stream().cuda_stream)
    ok = (slots >= 0) & (slots < pages * page)
    for c, was, begin in ((k, before[0], 0), (v, before[1], C)):
        flat = was.reshape(pages * page, heads, hs)
        flat[slots[ok].long()] = rows[ok, begin:begin + C].reshape(-1, heads, hs).to(dt)
        assert torch.equal(torch.nan_to_num(c.reshape(pages * page, heads, hs).float(), 123.0), torch.nan_to_num(flat.float(), 123.0))


def check_attention(bmb, torch, name, layout, lens, heads, kv, hs, page, scale=None, big=1.0, shift=1.0, bad_pages=False, spare=2, lse=True, seed=0):
    """Tokens that no request has are NaN throughout, so that reading one is seen."""
    dt = dtype_of(torch, name)
    torch.manual_seed(seed + sum(lens) + hs)
    counts = [-(-x // page) for x in lens]
    pages, width = sum(counts) + spare, max(max(counts + [0]), 1) + 1
    k, v = pool(torch, layout, pages, page, kv, hs, dt, float("nan"))
    ids = torch.randperm(pages).tolist()
    tables = np.full((len(lens), width), -1, np.int64)
    for i, c in enumerate(counts):
        for j in range(c):
            tables[i, j] = ids.pop()
            used = min(page, lens[i] - j * page)
            k[tables[i, j], :used] = (torch.randn(used, kv, hs, device="cuda") + shift * torch.randn(1, kv, hs, device="cuda")).to(dt)
            v[tables[i, j], :used] = torch.randn(used, kv, hs, device="cuda").to(dt)
        for j in range(c, width):
            tables[i, j] = [0, -1, pages + 5, 2 ** 31 - 1][(i + j) % 4]      # entries behind the last page mean nothing
        if bad_pages:
            for j in range(c):
                if (i * 3 + j * 5) % 4 == 0:
                    tables[i, j] = [-1, pages, -2 ** 31, 2 ** 31 - 1][(i + j) % 4]
    n = len(lens)
    qkv = torch.full((n, heads * hs + 64), float("nan"), device="cuda")
    qkv[:, :heads * hs] = torch.randn(n, heads * hs, device="cuda") * big
    out = torch.full((n + 1, heads * hs + 3), 77.0, device="cuda")
    got_lse = torch.full((n + 1, heads), 77.0, device="cuda") if lse else None
    size = bmb.paged_attention_workspace(heads, kv, hs)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    scale = hs ** -0.5 if scale is None else scale
    bmb.call("bmb_paged_attention", out, got_lse, qkv, bmb.KvCache.of(k, v), i32(torch, tables), i32(torch, lens), n, heads, qkv.stride(0), out.stride(0),
             width, scale, ws, size, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (ws[size:] == 255).all()
    assert (out[n:] == 77).all() and (out[:, heads * hs:] == 77).all()
    q = qkv[:, :heads * hs].reshape(n, heads, hs)
    want, want_lse, s, top, count = serving_oracle.attention(torch, q, k, v, tables, lens, scale)
    d_out, d_lse = serving_oracle.attention_bounds(hs, s, top, count)
    err = (out[:n, :heads * hs].reshape(n, heads, hs).double() - want).abs()
    assert (err <= d_out[..., None]).all(), (err.max().item(), (err / d_out[..., None].clamp(min=1e-30)).max().item())
    if lse:
        assert (got_lse[n:] == 77).all()
        none = count == 0
        assert (got_lse[:n][none] == -float("inf")).all()
        e = (got_lse[:n].double() - want_lse)[~none].abs()
        assert (e <= (d_lse + 2.0 ** -23 * want_lse.abs())[~none]).all(), e.max().item()
    return out[:n, :heads * hs]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_lengths(bmb, cuda, name, hs, layout):
    lens = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 511, 513, 1000, 0]
    check_attention(bmb, cuda, name, layout, lens, 4, 2, hs, 16)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("page", [1, 3, 8, 24, 100, 1024])
def test_attention_page_sizes(bmb, cuda, name, page):
    check_attention(bmb, cuda, name, "tokens", [1, 23, 24, 25, 99, 100, 101, 0, 700], 3, 3, 64, page)
    check_attention(bmb, cuda, name, "heads", [5, 130, 1025], 4, 2, 128, page, bad_pages=True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 2), (71, 1), (12, 12), (24, 3), (30, 2), (128, 8)])
def test_attention_shared_heads(bmb, cuda, name, heads, kv):
    for hs in (32, 128):
        check_attention(bmb, cuda, name, "heads", [3, 200, 0, 77, 513], heads, kv, hs, 32)


@pytest.mark.parametrize("name", TYPES)
def test_attention_long_and_uneven(bmb, cuda, name):
    check_attention(bmb, cuda, name, "tokens", [70001], 1, 1, 64, 64)
    check_attention(bmb, cuda, name, "tokens", [40000, 3, 0, 1, 9000, 1], 8, 1, 128, 100)
    check_attention(bmb, cuda, name, "heads", [1 + 37 * (i % 29) for i in range(700)], 2, 2, 32, 16)
    check_attention(bmb, cuda, name, "heads", [20000] + [i % 3 for i in range(1100)], 2, 1, 32, 16)
    check_attention(bmb, cuda, name, "heads", [0] * 700 + [60] + [0] * 1500 + [3, 3000, 0, 9] + [0] * 400, 4, 2, 64, 16)
    check_attention(bmb, cuda, name, "heads", [5] + [0] * 31 + [3] + [0] * 32 + [2000] + [0] * 33 + [4] + [0] * 200, 1, 1, 128, 16)


@pytest.mark.parametrize("name", TYPES)
def test_attention_large_scores_and_pages_that_are_none(bmb, cuda, name):
    check_attention(bmb, cuda, name, "tokens", [1, 50, 333, 2000], 6, 2, 64, 16, big=40.0, shift=3.0)       # one token takes all
    check_attention(bmb, cuda, name, "tokens", [1, 50, 333, 2000], 6, 2, 64, 16, big=1e-20)
    check_attention(bmb, cuda, name, "tokens", [9, 64, 500], 6, 2, 64, 16, scale=0.0)
    check_attention(bmb, cuda, name, "tokens", [9, 64, 500], 6, 2, 64, 16, scale=-0.2)
    check_attention(bmb, cuda, name, "tokens", [1, 16, 17, 2000, 3000], 6, 2, 128, 16, bad_pages=True, lse=False)


def test_attention_queries_of_very_different_sizes(bmb, cuda):
    """Rows of q from 2^-60 to 2^40 side by side, and within a row elements 2^30 apart: what a score is made of is what counts."""
    torch = cuda
    for name in TYPES:
        hs, heads, L = 64, 8, 100
        k, v = (torch.randn(1, L, 1, hs, device="cuda").to(dtype_of(torch, name)) for _ in range(2))
        q = torch.randn(1, heads * hs, device="cuda") * (2.0 ** torch.tensor([-60, -30, -12, 0, 4, 8, 20, 40], device="cuda")).repeat_interleave(hs)
        q[:, ::3] *= 2.0 ** -30
        out, ws = torch.empty(1, heads * hs, device="cuda"), torch.empty(bmb.paged_attention_workspace(heads, 1, hs), dtype=torch.uint8, device="cuda")
        bmb.call("bmb_paged_attention", out, None, q, bmb.KvCache.of(k, v), i32(torch, [[0]]), i32(torch, [L]), 1, heads, heads * hs, heads * hs, 1, 0.125, ws,
                 ws.numel(), torch.cuda.current_stream().cuda_stream)
        want, _, s, top, count = serving_oracle.attention(torch, q.view(1, heads, hs), k, v, [[0]], [L], 0.125)
        err = (out.view(1, heads, hs).double() - want).abs()
        assert (err <= serving_oracle.attention_bounds(hs, s, top, count)[0][..., None]).all()


def test_attention_lengths_beyond_the_table(bmb, cuda):
    """A length that its table cannot hold is clamped to it; a negative one is none."""
    torch = cuda
    k, v = (torch.randn(3, 16, 1, 32, device="cuda") for _ in range(2))
    q, ws = torch.randn(3, 32, device="cuda"), torch.empty(bmb.paged_attention_workspace(1, 1, 32), dtype=torch.uint8, device="cuda")
    outs = []
    for lens in ([48, 2 ** 31 - 1, -5], [48, 48, 0]):
        out = torch.full((3, 32), 9.0, device="cuda")
        bmb.call("bmb_paged_attention", out, None, q, bmb.KvCache.of(k, v), i32(torch, [[0, 1, 2], [2, 0, 1], [1, 1, 1]]), i32(torch, lens), 3, 1, 32, 32, 3, 0.2, ws,
                 ws.numel(), torch.cuda.current_stream().cuda_stream)
        outs.append(out)
    assert torch.equal(*outs) and (outs[0][2] == 0).all() and not (outs[0][1] == 0).any()


def test_attention_not_finite(bmb, cuda):
    """NaN in a key or value that counts reaches its head's outputs and no other's."""
    torch = cuda
    for name in TYPES:
        k, v = (torch.randn(4, 16, 2, 64, device="cuda").to(dtype_of(torch, name)) for _ in range(2))
        k[1, 3, 0, 5] = float("nan")
        v[2, 0, 1, 7] = float("inf")
        q, out = torch.randn(2, 4 * 64, device="cuda"), torch.empty(2, 4 * 64, device="cuda")
        ws = torch.empty(bmb.paged_attention_workspace(4, 2, 64), dtype=torch.uint8, device="cuda")
        bmb.call("bmb_paged_attention", out, None, q, bmb.KvCache.of(k, v), i32(torch, [[0, 1], [3, 2]]), i32(torch, [32, 20]), 2, 4, 256, 256, 2, 0.125, ws,
                 ws.numel(), torch.cuda.current_stream().cuda_stream)
        bad = ~torch.isfinite(out.view(2, 4, 64))
        assert bad[0, :2].all() and not bad[0, 2:].any() and not bad[1, :2].any()
        assert bad[1, 2:, 7].all() and bad[1, 2:].sum() == 2


def test_offsets_beyond_32_bits(bmb, cuda):
    """A cache whose last pages begin more than 2^32 bytes and 2^31 elements behind its first."""
    torch = cuda
    pages, page, heads, hs = 9000, 1024, 4, 64
    k, v = (torch.empty(pages, page, heads, hs, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    C, T = heads * hs, 2000
    rows = torch.randn(T, 3 * C, device="cuda")
    ids = [pages - 1, pages - 2]
    slots = torch.tensor([ids[t // page] * page + t % page for t in range(T)], dtype=torch.int32, device="cuda")
    c = bmb.KvCache.of(k, v)
    st = torch.cuda.current_stream().cuda_stream
    bmb.call("bmb_paged_kv_write", c, rows[:, C:], rows[:, 2 * C:], 3 * C, slots, T, st)
    out, ws = torch.empty(1, C, device="cuda"), torch.empty(bmb.paged_attention_workspace(heads, heads, hs), dtype=torch.uint8, device="cuda")
    bmb.call("bmb_paged_attention", out, None, rows[-1:], c, i32(torch, [ids]), i32(torch, [T]), 1, heads, 3 * C, C, 2, 0.125, ws, ws.numel(), st)
    near = [rows[:, (j + 1) * C:(j + 2) * C].to(torch.bfloat16).reshape(1, T, heads, hs) for j in range(2)]
    want, _, s, top, count = serving_oracle.attention(torch, rows[-1:, :C].reshape(1, heads, hs), near[0], near[1], [[0]], [T], 0.125)
    assert ((out.view(1, heads, hs).double() - want).abs() <= serving_oracle.attention_bounds(hs, s, top, count)[0][..., None]).all()


# ---- logits ---------------------------------------------------------------------------------------------------------

def run_adjust(bmb, torch, logits, V, in_place=False, **parts):
    n, stride = logits.shape
    x = torch.from_numpy(logits).cuda()
    out = x if in_place else torch.full_like(x, 77.0)
    rules = {{"lens": "history_lens", "prompts": "prompt_lens", "rep": "repetition", "freq": "frequency", "pres": "presence"}.get(key, key):
             torch.from_numpy(np.ascontiguousarray(a).view(np.int32) if np.asarray(a).dtype == np.uint32 else np.ascontiguousarray(a)).cuda()
             for key, a in parts.items()}
    bmb.call("bmb_logits_adjust", out, x, n, V, stride, bmb.LogitRules.of(**rules), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = serving_oracle.adjust(logits, V, **parts)
    got = out.cpu().numpy()
    same = (got[:, :V] == want[:, :V]) | (np.isnan(got[:, :V]) & np.isnan(want[:, :V]))
    assert same.all(), (np.argwhere(~same)[:5], got[:, :V][~same][:5], want[:, :V][~same][:5])
    assert np.array_equal(got[:, V:], logits[:, V:] if in_place else np.full_like(got[:, V:], 77.0))
    return got


def all_rules(rng, n, V, H, nb):
    history = (V * rng.random((n, H)) ** 3).astype(np.int32)
    history[rng.random((n, H)) < 0.05] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31])
    lens = rng.integers(0, H + 1, n).astype(np.int32)
    lens[0] = H
    f = lambda lo, hi: rng.uniform(lo, hi, n).astype(np.float32)
    d = dict(history=history, lens=lens, prompts=(lens * rng.random(n)).astype(np.int32), rep=f(0.7, 1.6), freq=f(-0.5, 1), pres=f(-0.5, 1))
    if nb:
        ids = (V * rng.random((n, nb)) ** 2).astype(np.int32)
        ids[rng.random((n, nb)) < 0.1] = rng.choice([-1, V, 2 ** 31 - 1])
        d.update(bias_ids=ids, bias=(rng.standard_normal((n, nb)) * 9).astype(np.float32), bias_lens=rng.integers(0, nb + 1, n).astype(np.int32))
    allowed = rng.integers(0, 2 ** 32, (n, (V + 31) // 32 + 1), dtype=np.uint32)
    allowed[n // 2] = 0
    allowed[0] = 2 ** 32 - 1
    d["allowed"] = allowed
    return d


@pytest.mark.parametrize("n,V,stride,H,nb", [(1, 1, 1, 1, 1), (3, 31, 40, 50, 4), (2, 32, 33, 7, 0), (5, 65, 128, 300, 9), (4, 257, 257, 1000, 600),
                                             (3, 4096, 4096, 64, 5), (3, 4097, 4099, 64, 5), (7, 50257, 50304, 2000, 300), (2, 131071, 131073, 9000, 40),
                                             (2, 300001, 300004, 500, 40), (300, 1000, 1024, 33, 3), (1, 50257, 50257, 40000, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust(bmb, cuda, n, V, stride, H, nb, in_place):
    rng = np.random.default_rng(V + H)
    logits = (rng.standard_normal((n, stride)) * 5).astype(np.float32)
    lowest = np.finfo(np.float32).min
    special = np.array([np.nan, np.inf, -np.inf, lowest, -lowest, 0.0, -0.0, 1e-42], np.float32)
    logits[0, :min(V, 8)] = special[:min(V, 8)]
    d = all_rules(rng, n, V, H, nb)
    d["history"][0, :min(H, 8)] = np.arange(min(H, 8)) % V
    run_adjust(bmb, cuda, logits, V, in_place, **d)


def test_adjust_single_rules(bmb, cuda):
    rng = np.random.default_rng(4)
    n, V = 6, 5003
    logits = (rng.standard_normal((n, V)) * 5).astype(np.float32)
    d = all_rules(rng, n, V, 400, 30)
    text = {k: d[k] for k in ("history", "lens")}
    run_adjust(bmb, cuda, logits, V)                                                       # no rules: a copy
    run_adjust(bmb, cuda, logits, V, **text)                                               # a text and nothing made of it
    for key in ("rep", "freq", "pres"):
        run_adjust(bmb, cuda, logits, V, **text, **{key: d[key]})
        run_adjust(bmb, cuda, logits, V, **text, prompts=d["prompts"], **{key: d[key]})
    run_adjust(bmb, cuda, logits, V, **{k: d[k] for k in ("bias_ids", "bias", "bias_lens")})
    got = run_adjust(bmb, cuda, logits, V, allowed=d["allowed"])
    assert np.isneginf(got[n // 2]).all()
    wild = dict(text, lens=np.array([-5, 0, 399, 400, 401, 2 ** 31 - 1], np.int32), prompts=np.array([-5, 2 ** 31 - 1, 0, 400, 200, -1], np.int32))
    run_adjust(bmb, cuda, logits, V, **wild, rep=d["rep"], freq=d["freq"], pres=d["pres"])  # lengths beyond the arrays


def test_adjust_many_times_one_token(bmb, cuda):
    """All of a long text one token: counted exactly."""
    V, H = 70, 100000
    logits = np.ones((2, V), np.float32)
    history = np.full((2, H), 5, np.int32)
    history[1] = np.arange(H) % V
    one = np.ones(2, np.float32)
    run_adjust(bmb, cuda, logits, V, history=history, lens=np.array([H, H], np.int32), rep=one * 3, freq=one * 0.5, pres=one)


# ---- streams, graphs, and a step of all of them ---------------------------------------------------------------------------

class Serving:
    """A cache, its pool, and the steps of several texts with one attention layer, the way a program holds them."""

    def __init__(self, bmb, torch, n, heads, kv, hs, page, pages, width, room, name="bf16"):
        self.bmb, self.torch, self.n, self.heads, self.kv, self.hs, self.page, self.pages, self.room = bmb, torch, n, heads, kv, hs, page, pages, room
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.k, self.v = pool(torch, "tokens", pages, page, kv, hs, dtype_of(torch, name), float("nan"))
        self.cache = bmb.KvCache.of(self.k, self.v)
        self.tables, self.lens, self.new, self.done, self.stack = z(n, width).fill_(-1), z(n), z(n), z(n), torch.randperm(pages, device="cuda").int()
        self.free, self.slots, self.positions, self.owners, self.starts = z(1).fill_(pages), z(room), z(room), z(room), z(n + 1)
        self.qkv = torch.zeros(room, (heads + 2 * kv) * hs, device="cuda")
        self.out = torch.zeros(n, heads * hs, device="cuda")
        self.ws = torch.empty(bmb.paged_attention_workspace(heads, kv, hs), dtype=torch.uint8, device="cuda")

    def step(self, stream):
        """Pages for the new tokens, their keys and values into the cache, and attention of the first n rows' queries."""
        call, n = self.bmb.call, self.n
        call("bmb_pages_assign", self.tables, self.lens, self.slots, self.positions, self.owners, self.starts, self.free, self.lens, self.new, self.stack,
             self.free, n, self.tables.shape[1], self.page, self.pages, self.room, stream)
        at = self.heads * self.hs
        call("bmb_paged_kv_write", self.cache, self.qkv[:, at:], self.qkv[:, at + self.kv * self.hs:], self.qkv.shape[1], self.slots, self.room, stream)
        call("bmb_paged_attention", self.out, None, self.qkv, self.cache, self.tables, self.lens, n, self.heads, self.qkv.shape[1], self.out.shape[1],
             self.tables.shape[1], self.hs ** -0.5, self.ws, self.ws.numel(), stream)

    def release(self, stream):
        self.bmb.call("bmb_pages_release", self.stack, self.free, self.lens, self.free, self.lens, self.tables, self.done, self.n, self.tables.shape[1],
                      self.page, self.pages, stream)


def simulate(bmb, torch, run_step, s, texts, steps, seed):
    """Several texts that begin, grow, end and begin again, against rows kept in a plain list."""
    rng = np.random.default_rng(seed)
    C, K, hs = s.heads * s.hs, s.kv * s.hs, s.hs
    for step in range(steps):
        new = np.array([int(rng.integers(2, 40)) if not t and rng.random() < 0.6 else int(bool(t)) for t in texts])
        s.new.copy_(i32(torch, new))
        s.qkv.copy_(torch.randn(s.room, s.qkv.shape[1], generator=torch.Generator().manual_seed(seed + step)))
        before = [len(t) for t in texts]
        free = int(s.free)
        run_step()
        torch.cuda.synchronize()
        lens, rows = s.lens.cpu().numpy(), s.qkv.clone()
        begin = 0
        for i in range(s.n):
            served = lens[i] == before[i] + new[i]
            assert served or lens[i] == before[i]
            if served:
                texts[i] += [rows[begin + j] for j in range(new[i])]
            begin += new[i]
        held = sum(-(-len(t) // s.page) for t in texts)
        assert int(s.free) == s.pages - held and int(s.free) <= free
        for i in range(s.n):
            if not texts[i]:
                assert (s.out[i] == 0).all()
                continue
            dt = s.k.dtype
            kv = torch.stack(texts[i])[:, C:].to(dt).reshape(1, len(texts[i]), 2, s.kv, hs)
            want, _, size, top, count = serving_oracle.attention(torch, rows[i:i + 1, :C].reshape(1, s.heads, hs), kv[:, :, 0], kv[:, :, 1], [[0]], [len(texts[i])], hs ** -0.5)
            err = (s.out[i].view(1, s.heads, hs).double() - want).abs()
            assert (err <= serving_oracle.attention_bounds(hs, size, top, count)[0][..., None]).all()
        done = np.array([len(t) > 60 or rng.random() < 0.1 for t in texts])
        s.done.copy_(i32(torch, done))
        s.release(torch.cuda.current_stream().cuda_stream)
        texts = [[] if d else t for t, d in zip(texts, done)]
    assert int(s.free) == s.pages - sum(-(-len(t) // s.page) for t in texts)


@pytest.mark.parametrize("name,heads,kv,hs,page,pages", [("bf16", 6, 2, 64, 8, 60), ("fp32", 4, 4, 32, 3, 300), ("fp16", 8, 1, 128, 16, 30)])
def test_steps_together(bmb, cuda, name, heads, kv, hs, page, pages):
    s = Serving(bmb, cuda, 9, heads, kv, hs, page, pages, 120 // page, 200, name)
    simulate(bmb, cuda, lambda: s.step(cuda.cuda.current_stream().cuda_stream), s, [[] for _ in range(9)], 30, 5)


@pytest.mark.parametrize("width", [15, 800])
def test_a_captured_step_follows_the_lengths(bmb, cuda, width):
    """One graph of a whole step, replayed while texts begin, grow and end: nothing of its shape came from the host.  (Tables for short
    texts, and for long ones, whose attention is divided over the GPU.)"""
    torch = cuda
    s = Serving(bmb, torch, 9, 6, 2, 64, 8, 70, width, 200)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            s.step(torch.cuda.current_stream().cuda_stream)
    simulate(bmb, torch, graph.replay, s, [[] for _ in range(9)], 20, 11)


def test_two_streams_at_once(bmb, cuda):
    """Calls on two streams, each with its own workspace, beside one another."""
    torch = cuda
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for j in range(2):
        torch.manual_seed(j)
        L, heads, hs = 5000 + 777 * j, 8, 64
        k, v = (torch.randn(1, L, 2, hs, device="cuda") for _ in range(2))
        q = torch.randn(3, heads * hs, device="cuda")
        out, ws = torch.empty(3, heads * hs, device="cuda"), torch.empty(bmb.paged_attention_workspace(heads, 2, hs), dtype=torch.uint8, device="cuda")
        work.append((k, v, q, out, ws, i32(torch, [[0]] * 3), i32(torch, [L, 11, L - 5]), [L, 11, L - 5]))
    torch.cuda.synchronize()
    for _ in range(20):
        for side, (k, v, q, out, ws, tables, lens, _) in zip(sides, work):
            bmb.call("bmb_paged_attention", out, None, q, bmb.KvCache.of(k, v), tables, lens, 3, 8, 512, 512, 1, 0.125, ws, ws.numel(), side.cuda_stream)
    torch.cuda.synchronize()
    for k, v, q, out, ws, tables, _, lens in work:
        want, _, s, top, count = serving_oracle.attention(torch, q.view(3, 8, 64), k, v, [[0]] * 3, lens, 0.125)
        assert ((out.view(3, 8, 64).double() - want).abs() <= serving_oracle.attention_bounds(64, s, top, count)[0][..., None]).all()


def test_the_same_call_twice_gives_the_same_bits(bmb, cuda):
    a = check_attention(bmb, cuda, "bf16", "tokens", [9000, 40, 1234, 0, 1], 16, 2, 128, 16, seed=3)
    b = check_attention(bmb, cuda, "bf16", "tokens", [9000, 40, 1234, 0, 1], 16, 2, 128, 16, seed=3)
    assert cuda.equal(a, b)


@pytest.mark.parametrize("name", TYPES)
def test_attention_with_blocks_for_each_head(bmb, cuda, name):
    """Few and short heads, which a cluster of 1 to 8 blocks each serves without a second launch, and their like beyond that form's borders."""
    for hs in (32, 64, 128):
        keys = 4096 // (hs * (4 if name == "fp32" else 2))
        for L in (1, keys, 4 * keys + 1, 9 * keys, 15 * keys - 3, 32 * keys - 16, 33 * keys, 64 * keys + 5, 100 * keys):
            check_attention(bmb, cuda, name, "tokens", [L], 6, 3, hs, 16)
            check_attention(bmb, cuda, name, "heads", [max(L - 7 * i, 0) for i in range(5)], 24, 12, hs, 16, bad_pages=True)
            check_attention(bmb, cuda, name, "heads", [max(L - 7 * i, 0) for i in range(24)], 12, 12, hs, 16, lse=False)
            check_attention(bmb, cuda, name, "interleaved", [L, 3, 0], 17, 1, hs, 24)
        check_attention(bmb, cuda, name, "tokens", [0, 5, 0], 9, 1, hs, 16)


def test_write_of_as_many_rows_as_an_int_counts(bmb, cuda):
    """2^31 - 1 rows, all but the first and the last left out: the threads behind the last row are beyond an int."""
    torch = cuda
    tokens = 2 ** 31 - 1
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    slots[0], slots[-1] = 3, 17
    k, v = (torch.zeros(2, 16, 1, 32, device="cuda") for _ in range(2))
    row = torch.arange(64, dtype=torch.float32, device="cuda")
    bmb.call("bmb_paged_kv_write", bmb.KvCache.of(k, v), row, row[32:], 0, slots, tokens, torch.cuda.current_stream().cuda_stream)
    for got, want in ((k, row[:32]), (v, row[32:])):
        rows = got.view(32, 32)
        assert torch.equal(rows[[3, 17]], want.expand(2, 32)) and not rows[[i for i in range(32) if i not in (3, 17)]].any()
