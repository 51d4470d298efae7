"""The serving entry points without a GPU: every call that they refuse is refused before anything is launched, and the plain
forms that the GPU tests compare with behave as the definitions say."""
import ctypes as C

import numpy as np
import pytest

import serving_oracle

P = 4096                                  # an address that is never followed: the calls below end before that


def cache(bmb, **change):
    d = dict(k=P, v=P, page_stride=16 * 2 * 64, token_stride=2 * 64, head_stride=64, type=bmb.TYPE_FP32, pages=8, page_size=16, heads=2, head_size=64)
    d.update(change)
    return bmb.KvCache(**d)


BAD_CACHES = [
    (dict(k=None), "E_ARG"), (dict(v=None), "E_ARG"), (dict(type=3), "E_ARG"), (dict(type=-1), "E_ARG"), (dict(pages=0), "E_ARG"),
    (dict(page_size=0), "E_ARG"), (dict(heads=0), "E_ARG"), (dict(head_size=96), "E_UNSUPPORTED"), (dict(head_size=0), "E_UNSUPPORTED"),
    (dict(pages=1 << 20, page_size=1 << 12), "E_LIMIT"), (dict(k=P + 8), "E_ARG"), (dict(v=P + 4), "E_ARG"), (dict(token_stride=130), "E_ARG"),
    (dict(head_stride=32), "E_ARG"), (dict(page_stride=-2048), "E_ARG"), (dict(type=1, head_stride=68), "E_ARG"),
]


@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches_are_refused(bmb, change, code):
    lib, want = bmb.lib(), getattr(bmb, code)
    assert lib.bmb_paged_kv_write(cache(bmb, **change), P, P, 384, P, 4, None) == want
    assert lib.bmb_paged_attention(P, P, P, cache(bmb, **change), P, P, 1, 2, 384, 128, 4, 0.125, P, 1 << 24, None) == want


@pytest.mark.parametrize("at,value,code", [
    (0, None, "E_ARG"), (2, None, "E_ARG"), (3, None, "E_ARG"), (4, None, "E_ARG"), (5, None, "E_ARG"), (6, -1, "E_ARG"), (7, 3, "E_ARG"), (7, 0, "E_ARG"),
    (8, -1, "E_ARG"), (9, 127, "E_ARG"), (10, 0, "E_ARG"), (10, 1 << 28, "E_LIMIT"), (12, None, "E_ARG"), (12, P + 8, "E_ARG"), (13, 0, "E_ARG"),
    (6, (1 << 31) - 1, "E_LIMIT"), (0, P + 2, "E_ARG"), (1, P + 2, "E_ARG"), (2, P + 1, "E_ARG"), (4, P + 2, "E_ARG"), (5, P + 3, "E_ARG"),
])
def test_attention_refuses(bmb, at, value, code):
    args = [P, P, P, cache(bmb), P, P, 1, 2, 384, 128, 4, 0.125, P, 1 << 24, None]
    args[at] = value
    assert bmb.lib().bmb_paged_attention(*args) == getattr(bmb, code)
    assert bmb.lib().bmb_last_error().startswith(b"paged_attention")


def test_attention_of_no_requests_is_nothing(bmb):
    assert bmb.lib().bmb_paged_attention(None, None, None, cache(bmb), None, None, 0, 2, 384, 128, 4, 0.125, None, 0, None) == 0
    assert bmb.lib().bmb_paged_kv_write(cache(bmb), None, None, 384, None, 0, None) == 0


@pytest.mark.parametrize("at,value", [(1, None), (2, None), (3, -1), (4, None), (5, -1), (1, P + 2), (4, P + 2)])
def test_write_refuses(bmb, at, value):
    args = [cache(bmb), P, P, 384, P, 4, None]
    args[at] = value
    assert bmb.lib().bmb_paged_kv_write(*args) == bmb.E_ARG


@pytest.mark.parametrize("at,value,code", [
    (0, None, "E_ARG"), (1, None, "E_ARG"), (2, None, "E_ARG"), (6, None, "E_ARG"), (7, None, "E_ARG"), (8, None, "E_ARG"), (9, None, "E_ARG"),
    (10, None, "E_ARG"), (11, -1, "E_ARG"), (12, 0, "E_ARG"), (13, 0, "E_ARG"), (14, -1, "E_ARG"), (15, -1, "E_ARG"), (14, 1 << 28, "E_LIMIT"),
    (12, 1 << 28, "E_LIMIT"),
] + [(i, P + 2, "E_ARG") for i in range(11)])
def test_assign_refuses(bmb, at, value, code):
    args = [P] * 11 + [4, 8, 16, 32, 64, None]
    args[at] = value
    assert bmb.lib().bmb_pages_assign(*args) == getattr(bmb, code)


@pytest.mark.parametrize("at,value,code", [
    (0, None, "E_ARG"), (1, None, "E_ARG"), (2, None, "E_ARG"), (3, None, "E_ARG"), (4, None, "E_ARG"), (5, None, "E_ARG"), (6, None, "E_ARG"),
    (7, -1, "E_ARG"), (8, 0, "E_ARG"), (9, 0, "E_ARG"), (10, -1, "E_ARG"), (10, 1 << 28, "E_LIMIT"),
] + [(i, P + 1, "E_ARG") for i in range(7)])
def test_release_refuses(bmb, at, value, code):
    args = [P] * 7 + [4, 8, 16, 32, None]
    args[at] = value
    assert bmb.lib().bmb_pages_release(*args) == getattr(bmb, code)


@pytest.mark.parametrize("rules,more", [
    (dict(repetition=P), {}), (dict(frequency=P), {}), (dict(presence=P), {}), (dict(history=P, history_stride=4), {}),
    (dict(history=P, history_lens=P, history_stride=-1), {}), (dict(bias_ids=P, bias_lens=P), {}), (dict(bias=P, bias_lens=P), {}),
    (dict(bias_ids=P, bias=P), {}), (dict(bias_ids=P, bias=P, bias_lens=P, bias_stride=-1), {}), (dict(allowed=P, allowed_stride=3), {}),
    (dict(history=P, history_lens=P + 2, history_stride=4), {}), (dict(allowed=P + 1, allowed_stride=4), {}), ({}, dict(out=P + 2)),
    ({}, dict(out=None)), ({}, dict(logits=None)), ({}, dict(n=-1)), ({}, dict(V=-1)), ({}, dict(stride=99)),
])
def test_adjust_refuses(bmb, rules, more):
    d = dict(out=P, logits=P, n=2, V=100, stride=100)
    d.update(more)
    assert bmb.lib().bmb_logits_adjust(d["out"], d["logits"], d["n"], d["V"], d["stride"], bmb.LogitRules(**rules), None) == bmb.E_ARG
    assert bmb.lib().bmb_logits_adjust(d["out"], d["logits"], 2, 100, 100, None, None) == bmb.E_ARG


def test_adjust_of_nothing_is_nothing(bmb):
    assert bmb.lib().bmb_logits_adjust(None, None, 0, 100, 100, bmb.LogitRules(), None) == 0
    assert bmb.lib().bmb_logits_adjust(None, None, 3, 0, 0, bmb.LogitRules(), None) == 0


def test_workspace_is_stated(bmb):
    assert bmb.paged_attention_workspace(12, 12, 64) % 16 == 0
    assert 16 <= bmb.paged_attention_workspace(71, 1, 128) < 1 << 25


def test_struct_layouts(bmb):
    """The ctypes mirrors have the C structs' sizes: pointers and 64-bit strides first, then ints."""
    assert C.sizeof(bmb.KvCache) == 5 * 8 + 5 * 4 + 4 and C.sizeof(bmb.LogitRules) == 10 * 8 + 3 * 4 + 4


def test_long_texts_are_refused(bmb):
    for rules in (dict(history=P, history_lens=P, history_stride=(1 << 30) + 1), dict(bias_ids=P, bias=P, bias_lens=P, bias_stride=(1 << 30) + 1)):
        assert bmb.lib().bmb_logits_adjust(P, P, 2, 100, 100, bmb.LogitRules(**rules), None) == bmb.E_LIMIT
    assert bmb.lib().bmb_logits_adjust(P, P, 1 << 30, 5000, 5000, bmb.LogitRules(), None) == bmb.E_LIMIT
    assert bmb.lib().bmb_paged_kv_write(cache(bmb, heads=1 << 26), P, P, 384, P, 4, None) == bmb.E_LIMIT


def test_structs_of_tensors(bmb):
    import torch
    k = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    c = bmb.KvCache.of(k, k.clone())
    assert (c.page_stride, c.token_stride, c.head_stride, c.type, c.pages, c.page_size, c.heads, c.head_size) == (2048, 128, 64, bmb.TYPE_BF16, 3, 16, 2, 64)
    t = k.transpose(1, 2)
    c = bmb.KvCache.of(t, t)
    assert (c.page_size, c.heads, c.token_stride, c.head_stride) == (2, 16, 64, 128)
    for a, b in ((k, k.float()), (k, k[:2]), (k.double(), k.double()), (k[0], k[0]), (k.transpose(2, 3), k.transpose(2, 3)), (k, t.contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            bmb.KvCache.of(a, b)
    r = bmb.LogitRules.of(history=torch.zeros(2, 7, dtype=torch.int32), history_lens=torch.zeros(2, dtype=torch.int32), allowed=torch.zeros(2, 4, dtype=torch.int32))
    assert (r.history_stride, r.bias_stride, r.allowed_stride) == (7, 0, 4) and r.bias is None


def test_oracle_assign_by_hand():
    tables = np.full((4, 3), -1, np.int32)
    tables[1, 0] = 6
    t, lens, slots, pos, own, starts, left = serving_oracle.assign(tables, [0, 3, 0, 4], [5, 1, 9, 0], np.array([7, 2, 5, 0]), 3, 4, 8, 16)
    # request 0 takes two pages from the end of the stack of three, 1 fills its page, 2 needs three pages (one is left), 3 rests
    assert t.tolist() == [[5, 2, -1], [6, -1, -1], [-1, -1, -1], [-1, -1, -1]]
    assert lens.tolist() == [5, 4, 0, 4] and left == 1 and starts.tolist() == [0, 5, 6, 15, 15]
    assert slots.tolist() == [20, 21, 22, 23, 8, 27] + [-1] * 10
    assert pos.tolist() == [0, 1, 2, 3, 4, 3, 0, 1, 2, 3, 4, 5, 6, 7, 8, 0] and own.tolist() == [0] * 5 + [1] + [2] * 9 + [-1]


def test_oracle_release_by_hand():
    stack, free, lens = serving_oracle.release(np.array([7, 2, 0, 0, 0, 0, 0, 0]), 2, [5, 4, 9], np.array([[5, -3, 1], [6, 9, 9], [3, 8, 4]]), [1, 0, 1], 4, 8)
    assert stack.tolist() == [7, 2, 5, 3, 4, 0, 0, 0] and free == 5 and lens.tolist() == [0, 4, 0]


@pytest.mark.parametrize("blocks", [1, 2, 7, 148])
@pytest.mark.parametrize("type_,hs", [(0, 128), (1, 32), (2, 64)])
def test_every_tile_is_worked_on_once(bmb, blocks, type_, hs):
    """The division of attention's work over warps and blocks, for lengths of all kinds."""
    rng = np.random.default_rng(blocks + hs)
    cases = [[0], [1], [5000], [0, 0, 0], [100000, 0, 1, 1], [1] * 500, [0] * 129 + [300], [300] + [0] * 700 + [2, 0], list(range(1, 260))]
    cases += [list((rng.integers(0, 10 ** int(rng.integers(1, 5)), int(rng.integers(1, 700))) * (rng.random() < 0.9)).astype(int)) for _ in range(20)]
    most = 0
    for i, lens in enumerate(cases):
        for heads, kv in ((1, 1), (6, 6), (32, 8), (71, 1), (24, 2)):
            tiles, joined = C.c_longlong(), C.c_int()
            a = np.array(lens, np.int32)
            cap = 20000 if i % 5 else 10 ** 6
            s = bmb.lib().bmb_paged_attention_schedule_check(a.ctypes.data, len(lens), heads, kv, hs, type_, cap, blocks, C.byref(tiles), C.byref(joined))
            assert s == 0, bmb.lib().bmb_last_error()
            keys = 4096 // (hs * (4 if type_ == 0 else 2))
            assert tiles.value == sum(-(-min(max(int(x), 0), cap) // keys) for x in lens) * kv * -(-(heads // kv) // 8)
            assert joined.value <= blocks
            most = max(most, joined.value)
    assert most > 0 or blocks == 1


def test_rules_of_tensors_that_do_not_hold_their_rows(bmb):
    """A call may read rows to their end, whatever the lengths are: the fronts of rows are taken, their backs, whose last one ends
    outside the memory, are not, nor are rows that lie on one another, other types and elements that lie apart."""
    import torch
    i, f = torch.zeros(3, 20, dtype=torch.int32), torch.zeros(3, 20)
    one = dict(history_lens=torch.zeros(3, dtype=torch.int32))
    assert bmb.LogitRules.of(history=i[:, :7], **one).history_stride == 20
    assert bmb.LogitRules.of(history=i[:2, 13:], **one).history_stride == 20
    assert bmb.LogitRules.of(history=i[2:, 13:], **one).history_stride == 7
    assert bmb.LogitRules.of(history=torch.zeros(3, 0, dtype=torch.int32), **one).history_stride == 0
    assert bmb.LogitRules.of(bias_ids=i[:, :5], bias=f[:, 2:7][:2], bias_lens=one["history_lens"]).bias_stride == 20
    for bad in (dict(history=i[:, 1:]), dict(history=i[:1].expand(3, 20)), dict(history=i.t()), dict(history=i[0]), dict(history=i.long()), dict(allowed=i[:, 19:]),
                dict(allowed=f), dict(bias_ids=i, bias=torch.zeros(3, 5)), dict(bias=f.double()), dict(bias=f[:, 3:]), dict(repetition=f[:, 0]),
                dict(frequency=i[0]), dict(presence=f[0].half()), dict(history_lens=i[:, 0]), dict(prompt_lens=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            bmb.LogitRules.of(**bad)


@pytest.mark.parametrize("at,value", [(0, None), (1, 0), (2, 0), (2, -2), (3, 0), (3, 4), (4, 96), (5, 3), (6, 0), (7, 0), (7, 513), (7, (1 << 31) - 1)])
def test_schedule_check_refuses(bmb, at, value):
    lens = (C.c_int * 2)(5, 300)
    args = [C.addressof(lens), 2, 6, 2, 64, 0, 1000, 148, None, None]
    assert bmb.lib().bmb_paged_attention_schedule_check(*args) == 0
    args[at] = value
    assert bmb.lib().bmb_paged_attention_schedule_check(*args) == bmb.E_ARG


@pytest.mark.parametrize("n", [(1 << 31) - 1023, (1 << 31) - 1])
def test_more_requests_than_stretches_can_count_are_refused(bmb, n):
    """Requests are taken in stretches of up to 1024, the first one behind the last of which is an int too."""
    assert bmb.lib().bmb_pages_assign(*[P] * 11, n, 8, 16, 32, 64, None) == bmb.E_LIMIT
    assert bmb.lib().bmb_pages_release(*[P] * 7, n, 8, 16, 32, None) == bmb.E_LIMIT
