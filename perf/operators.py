"""The operators of a serving step, as they are timed: a step of a program that answers several requests at once from one model.

  assign   bmb_pages_assign: pages of the cache's pool handed to requests by their lengths, and the slot of every new token
  release  bmb_pages_release: the pages of requests that have ended go back to the pool
  write    bmb_paged_kv_write: keys and values of new tokens, as they lie in the rows of a qkv product, into their slots
  attend   bmb_paged_attention: attention of one new token of each request over its pages
  adjust   bmb_logits_adjust: penalties for repeated tokens, biases and a mask of allowed tokens on rows of logits

prepare() makes what a serving program holds before the call; run() is one pass, in plain torch or, where `own` is true, through
the library's entry points; exact() the same from the definitions in 64 bits; work() the bytes and operations a pass cannot do without.
"""
import importlib
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
GOLDEN = 0.6180339887498949


def package():
    return importlib.import_module("bare-metal-bard_b200")


# ---- the cases --------------------------------------------------------------------------------------------------

def assign(n, page, max_pages, longest, new_share, new_longest, room):
    """n requests of up to `longest` cached tokens; `new_share` of them are prompts of up to new_longest tokens, the others add
    one; room: the part of the pages asked for that the pool has (under 1: some requests have to wait)."""
    return {"op": "assign", "n": n, "page": page, "max_pages": max_pages, "longest": longest, "new_share": new_share,
            "new_longest": new_longest, "room": room}


def release(n, page, longest, share):
    return {"op": "release", "n": n, "page": page, "longest": longest, "share": share}


def write(type_, tokens, heads, kv_heads, hs, page, padded):
    return {"op": "write", "type": type_, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "hs": hs, "page": page, "padded": padded}


def attend(type_, n, heads, kv_heads, hs, page, shortest, longest, empty=0):
    return {"op": "attend", "type": type_, "n": n, "heads": heads, "kv_heads": kv_heads, "hs": hs, "page": page, "shortest": shortest,
            "longest": longest, "empty": empty}


def adjust(n, V, Vp, history, biases, mask):
    return {"op": "adjust", "n": n, "V": V, "Vp": Vp, "history": history, "biases": biases, "mask": mask}


def listed():
    return [
        # One text of the character model (6 heads of 64, context 256) at its last position: launches and latency are its time.
        dict(attend("fp32", 1, 6, 6, 64, 16, 256, 256), name="attend_fp32_1x256_h6x64"),
        # The 124M configuration (12 heads of 64, context 1024) answering 64 requests of all lengths from a 16-bit cache.
        dict(attend("bf16", 64, 12, 12, 64, 16, 1, 1024), name="attend_bf16_64x1024_h12x64"),
        # Few requests with long contexts and query heads that share keys: the largest, a pass over 0.6 GB of cache.
        dict(attend("fp16", 8, 32, 8, 128, 64, 2049, 32768), name="attend_fp16_8x32768_h32_8x128"),
        # A cache in the activations' own type, odd lengths, and requests that have nothing yet.
        dict(attend("fp32", 37, 16, 4, 128, 24, 5, 2777, empty=2), name="attend_fp32_37x2777_h16_4x128"),
        # The keys and values of one step of 64 requests, some of the padded batch's rows unused.
        dict(write("bf16", 64, 12, 12, 64, 16, 5), name="write_bf16_64_h12x64"),
        # Prompts: 8 x 1024 tokens, the benchmark configuration's batch, into a cache of the activations' type.
        dict(write("fp32", 8192, 12, 12, 64, 16, 0), name="write_fp32_8192_h12x64"),
        # Every request adds its one token; about one in 16 begins a page.
        dict(assign(64, 16, 64, 1023, 0.0, 1, 1.5), name="assign_64_step"),
        # A step that admits prompts of up to 1024 tokens beside running requests, with pages for nine tenths of what is asked.
        dict(assign(128, 16, 128, 1000, 0.5, 1000, 0.9), name="assign_128_prompts"),
        # Some of 64 requests have ended.
        dict(release(64, 16, 1024, 0.25), name="release_64"),
        # Long contexts in small pages: 100 thousand pages come back.
        dict(release(250, 16, 16384, 0.8), name="release_250_long"),
        # One text: the logits of one position, penalties from its own 300 tokens.
        dict(adjust(1, 50257, 50304, 300, 0, False), name="adjust_1x50257"),
        # A batch with everything: long histories, biases, a grammar's mask that in one row allows nothing.
        dict(adjust(256, 50257, 50304, 1024, 64, True), name="adjust_256x50257_all"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "assign", "release", "adjust"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    if op == "attend":
        type_, hs, kv = rng.choice(sorted(TYPES)), rng.choice([32, 64, 128]), rng.choice([1, 2, 3, 4, 6, 8, 12])
        group = rng.choice([1, 1, 2, 3, 4, 5, 8, 12, 16])
        row = kv * hs * 2 * SIZE[type_]                                # bytes of a token
        longest = _log(rng, 1, min(60000, 200_000_000 // row))
        n = _log(rng, 1, max(1, min(256, 300_000_000 // (row * longest))))
        return attend(type_, n, kv * group, kv, hs, page, _log(rng, 1, longest), longest, rng.choice([0, 0, n // 7]))
    if op == "write":
        kv, hs = rng.choice([1, 2, 4, 6, 8, 12]), rng.choice([32, 64, 128])
        tokens = _log(rng, 1, 8000)
        return write(rng.choice(sorted(TYPES)), tokens, kv * rng.choice([1, 1, 2, 4]), kv, hs, page, rng.choice([0, tokens // 9]))
    if op == "assign":
        longest, new = _log(rng, 1, 3000), _log(rng, 1, 1000)
        return assign(_log(rng, 1, 500), page, -(-(longest + new) // page) + rng.choice([0, 0, -1, 7]) or 1, longest, rng.choice([0.0, 0.1, 0.5]),
                      new, rng.choice([0.0, 0.5, 1.0, 2.0]))
    if op == "release":
        return release(_log(rng, 1, 500), page, _log(rng, 1, 8000), rng.choice([0.05, 0.3, 0.7, 1.0]))
    V = rng.choice([65, 257, 1000, 32000, 50257, _log(rng, 50, 130000)])
    return adjust(_log(rng, 1, max(1, 12_000_000 // V if V > 50000 else 200)), V, -(-V // 128) * 128 + rng.choice([0, 0, 1]), _log(rng, 1, 4000),
                  rng.choice([0, 0, 3, 300]), rng.random() < 0.5)


# ---- what the program holds -----------------------------------------------------------------------------------------

def spread(n, lo, hi, shift=0):
    """n lengths from lo to hi, the same for every seed: what a pass has to do depends on them."""
    return [lo + int((hi - lo + 1) * ((i * GOLDEN + shift * 0.37 + 0.5) % 1.0)) for i in range(n)] if n > 1 else [hi]


def attend_lengths(c):
    lens = spread(c["n"], c["shortest"], c["longest"])
    for i in range(c["empty"]):
        lens[(i * 5 + 1) % c["n"]] = 0
    return lens


def assign_lengths(c):
    n = c["n"]
    lens, new = spread(n, 0, c["longest"]), spread(n, 1, c["new_longest"], 1)
    for i in range(n):
        prompt = (i * GOLDEN * 7) % 1.0 < c["new_share"]
        if prompt:
            lens[i] = 0 if i % 3 else lens[i]                         # (every third goes on with a prompt that was begun)
        else:
            new[i] = 0 if i % 11 == 10 else 1                          # (some have nothing in this step)
    return lens, new


def assign_asked(c):
    lens, new = assign_lengths(c)
    p = c["page"]
    return sum(-(-(a + b) // p) - -(-a // p) for a, b in zip(lens, new))


def release_lengths(c):
    lens = spread(c["n"], 1, c["longest"])
    return lens, [1 if (i * GOLDEN * 3) % 1.0 < c["share"] else 0 for i in range(c["n"])]


def slots_of(c):
    return c["tokens"] + 3 * c["page"]


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    order = lambda n: torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    empty = lambda *shape, dtype=torch.int32: torch.empty(*shape, dtype=dtype, device="cuda")
    s = {"case": c, "bmb": package() if own else None}
    op = c["op"]
    if op == "attend":
        lens, p, kv, hs = attend_lengths(c), c["page"], c["kv_heads"], c["hs"]
        counts = [-(-x // p) for x in lens]
        pages, width = sum(counts) + 3, max(max(counts), 1)
        # pages of one request lie anywhere in the pool; entries behind a request's last page are not pages
        ids, at = order(pages), 0
        tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
        for i, k in enumerate(counts):
            tables[i, :k] = ids[at:at + k]
            at += k
        # keys of a trained model have some directions that all of them share
        k = normal(pages, p, kv, hs).add_(normal(kv, hs)).to(TYPES[c["type"]])
        v = normal(pages, p, kv, hs).to(TYPES[c["type"]])
        # the queries lie in the rows of a qkv product
        qkv = normal(len(lens), (c["heads"] + 2 * kv) * hs)
        s.update(k=k, v=v, tables=tables, lens=ints(lens), qkv=qkv, out=empty(len(lens), c["heads"] * hs, dtype=torch.float32),
                 lse=empty(len(lens), c["heads"], dtype=torch.float32), scale=hs ** -0.5)
        if own:
            bmb = s["bmb"]
            s["cache"] = bmb.KvCache.of(k, v)
            s["workspace"] = empty(bmb.paged_attention_workspace(c["heads"], kv, hs), dtype=torch.uint8)
    elif op == "write":
        p, kv, hs, T = c["page"], c["kv_heads"], c["hs"], c["tokens"]
        pages = -(-slots_of(c) // p)
        k, v = (normal(pages, p, kv, hs).to(TYPES[c["type"]]) for _ in range(2))
        slots = order(pages * p)[:T].clone()
        if c["padded"]:
            slots[T - c["padded"]:] = -1
        s.update(k=k, v=v, slots=slots, qkv=normal(T, (c["heads"] + 2 * kv) * hs))
        if own:
            s["cache"] = s["bmb"].KvCache.of(k, v)
    elif op == "assign":
        lens, new = assign_lengths(c)
        n, p = c["n"], c["page"]
        free = int(c["room"] * assign_asked(c))
        held = sum(min(-(-x // p), c["max_pages"]) for x in lens)
        pages = held + free + 5
        ids = order(pages)
        tables = torch.full((n, c["max_pages"]), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, x in enumerate(lens):
            k = min(-(-x // p), c["max_pages"])
            tables[i, :k] = ids[at:at + k]
            at += k
        stack = torch.zeros(pages, dtype=torch.int32, device="cuda")
        stack[:free] = ids[at:at + free]
        T = sum(new) + 7                                               # (a batch is padded to a size of its own)
        s.update(tables=tables, lens=ints(lens), new=ints(new), stack=stack, free=ints([free]), tokens=T, pages=pages, lens_out=empty(n),
                 slots=empty(T), positions=empty(T), owners=empty(T), starts=empty(n + 1), free_out=empty(1))
    elif op == "release":
        lens, done = release_lengths(c)
        n, p = c["n"], c["page"]
        counts = [-(-x // p) for x in lens]
        pages = sum(counts) + 11
        ids = order(pages)
        tables = torch.full((n, max(counts)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, k in enumerate(counts):
            tables[i, :k] = ids[at:at + k]
            at += k
        stack = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        stack[:pages - at] = ids[at:]
        s.update(tables=tables, lens=ints(lens), done=ints(done), stack=stack, free=ints([pages - at]), pages=pages, lens_out=empty(n), free_out=empty(1))
    else:
        n, V, Vp, H, nb = c["n"], c["V"], c["Vp"], c["history"], c["biases"]
        uniform = lambda lo, hi, *shape: lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")
        # a text repeats some tokens often: ranks drawn so that few have most of the mass
        history = (V * uniform(0, 1, n, H) ** 4).to(torch.int32).clamp_(max=V - 1)
        lens = ints(spread(n, (H + 1) // 2, H))
        s.update(logits=normal(n, Vp) * 4, history=history, lens=lens, prompts=(lens * 0.4).to(torch.int32),
                 repetition=uniform(0.8, 1.5, n), frequency=uniform(-0.2, 0.8, n), presence=uniform(-0.2, 0.8, n), out=normal(n, Vp))
        if nb:
            s.update(bias_ids=(V * uniform(0, 1, n, nb)).to(torch.int32).clamp_(max=V - 1), bias=normal(n, nb) * 5, bias_lens=ints(spread(n, 0, nb)))
        if c["mask"]:
            words = torch.randint(-2 ** 31, 2 ** 31, (n, -(-V // 32)), generator=g, device="cuda", dtype=torch.int64)
            words &= torch.randint(-2 ** 31, 2 ** 31, words.shape, generator=g, device="cuda", dtype=torch.int64)
            words[n // 2] = 0
            s.update(mask=words.to(torch.int32))
        if own:
            s["rules"] = s["bmb"].LogitRules.of(history=history, history_lens=lens, prompt_lens=s["prompts"], repetition=s["repetition"],
                                                frequency=s["frequency"], presence=s["presence"], bias_ids=s.get("bias_ids"), bias=s.get("bias"),
                                                bias_lens=s.get("bias_lens"), allowed=s.get("mask"))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    return (run_own if own else run_plain)(s)


def run_own(s):
    c, bmb, op = s["case"], s["bmb"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "attend":
        n = len(s["lens"])
        bmb.call("bmb_paged_attention", s["out"], s["lse"], s["qkv"], s["cache"], s["tables"], s["lens"], n, c["heads"], s["qkv"].stride(0),
                 s["out"].stride(0), s["tables"].stride(0), s["scale"], s["workspace"], s["workspace"].numel(), stream)
        return s["out"], s["lse"]
    if op == "write":
        qkv, at, kv, hs = s["qkv"], c["heads"] * c["hs"], c["kv_heads"], c["hs"]
        bmb.call("bmb_paged_kv_write", s["cache"], qkv[:, at:], qkv[:, at + kv * hs:], qkv.stride(0), s["slots"], c["tokens"], stream)
        return s["k"], s["v"]
    if op == "assign":
        bmb.call("bmb_pages_assign", s["tables"], s["lens_out"], s["slots"], s["positions"], s["owners"], s["starts"], s["free_out"], s["lens"],
                 s["new"], s["stack"], s["free"], c["n"], c["max_pages"], c["page"], s["pages"], s["tokens"], stream)
        return s["tables"], s["lens_out"], s["slots"], s["positions"], s["owners"], s["starts"], s["free_out"]
    if op == "release":
        bmb.call("bmb_pages_release", s["stack"], s["free_out"], s["lens_out"], s["free"], s["lens"], s["tables"], s["done"], c["n"],
                 s["tables"].stride(0), c["page"], s["pages"], stream)
        return s["stack"], s["free_out"], s["lens_out"]
    bmb.call("bmb_logits_adjust", s["out"], s["logits"], c["n"], c["V"], c["Vp"], s["rules"], stream)
    return s["out"]


def run_plain(s):
    c = s["case"]
    return PLAIN[c["op"]](s, c)


def attend_plain(s, c):
    n, kv, hs, p = c["n"], c["kv_heads"], c["hs"], c["page"]
    group = c["heads"] // kv
    tables = s["tables"].clamp(min=0).long()
    keys, values = (x[tables].reshape(n, -1, kv, hs).float() for x in (s["k"], s["v"]))
    q = s["qkv"][:, :c["heads"] * hs].reshape(n, kv, group, hs)
    scores = torch.matmul(q, keys.permute(0, 2, 3, 1)) * s["scale"]
    inside = torch.arange(keys.shape[1], device="cuda") < s["lens"][:, None]
    scores = torch.where(inside[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    values = torch.where(inside[:, :, None, None], values, 0.0)
    out = torch.matmul(weights, values.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return out.reshape(n, -1), (top + torch.log(total)).reshape(n, -1)


def write_plain(s, c):
    at, kv, hs = c["heads"] * c["hs"], c["kv_heads"], c["hs"]
    used = s["slots"] >= 0
    rows = s["slots"][used].long()
    for cache, begin in ((s["k"], at), (s["v"], at + kv * hs)):
        cache.view(-1, kv * hs)[rows] = s["qkv"][used, begin:begin + kv * hs].to(cache.dtype)
    return s["k"], s["v"]


def assign_plain(s, c):
    p, width, T, pages = c["page"], c["max_pages"], s["tokens"], s["pages"]
    lens, new = s["lens"].clamp(min=0).long(), s["new"].clamp(min=0).long()
    free = s["free"].clamp(0, pages).long()
    ends = torch.cumsum(new, 0)
    begins = ends - new
    have, want = (lens + p - 1) // p, (lens + new + p - 1) // p
    fits = (want <= width) & (ends <= T)
    need = torch.where(fits, want - have, 0)
    taken = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (taken <= free))
    need = torch.where(served, need, 0)
    # pages from the top of the stack, in the order of requests
    column = torch.arange(width, device="cuda")
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    place = free - 1 - (taken[:, None] - need[:, None] + column - have[:, None])
    tables = torch.where(fresh, s["stack"][place.clamp(0, pages - 1)], s["tables"])
    lens_out = torch.where(served, lens + new, lens)
    t = torch.arange(T, device="cuda")
    owner = torch.searchsorted(ends, t, right=True)
    inside = owner < len(lens)
    owner = owner.clamp(max=len(lens) - 1)
    position = lens[owner] + t - begins[owner]
    page = tables[owner, (position // p).clamp(max=width - 1)].long()
    usable = inside & served[owner] & (page >= 0) & (page < pages)
    slots = torch.where(usable, page * p + position % p, -1)
    starts = torch.cat([begins, ends[-1:]]).clamp(max=T)
    i32 = lambda x: x.to(torch.int32)
    return (tables, i32(lens_out), i32(slots), i32(torch.where(inside, position, 0)), i32(torch.where(inside, owner, -1)), i32(starts),
            i32(free - need.sum()))


def release_plain(s, c):
    p, pages = c["page"], s["pages"]
    free, lens = s["free"].clamp(0, pages).long(), s["lens"].clamp(min=0).long()
    ends = s["done"] != 0
    held = (torch.arange(s["tables"].shape[1], device="cuda") < ((lens + p - 1) // p)[:, None]) & ends[:, None]
    held &= (s["tables"] >= 0) & (s["tables"] < pages)
    back = s["tables"][held]
    stack = s["stack"].clone()
    at = free + torch.arange(len(back), device="cuda")
    inside = at < pages
    stack[at[inside]] = back[inside]
    return stack, (free + len(back)).clamp(max=pages).to(torch.int32), torch.where(ends, 0, lens).to(torch.int32)


def adjust_plain(s, c):
    n, V, H = c["n"], c["V"], c["history"]
    x = s["logits"][:, :V]
    column = torch.arange(H, device="cuda")
    inside = column < s["lens"][:, None]
    drawn = inside & (column >= s["prompts"][:, None])
    tokens = s["history"].long()
    seen = torch.zeros(n, V, device="cuda").scatter_add_(1, tokens, inside.float()) > 0
    count = torch.zeros(n, V, device="cuda").scatter_add_(1, tokens, drawn.float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if c["biases"]:
        entry = torch.arange(c["biases"], device="cuda")
        rank = torch.where(entry < s["bias_lens"][:, None], entry + 1, 0)
        last = torch.zeros(n, V, dtype=torch.int64, device="cuda").scatter_reduce_(1, s["bias_ids"].long(), rank, "amax")
        x = torch.where(last > 0, x + s["bias"].gather(1, (last - 1).clamp(min=0)), x)
    if c["mask"]:
        v = torch.arange(V, device="cuda")
        x = torch.where((s["mask"][:, v // 32] >> (v % 32)) & 1 != 0, x, -math.inf)
    out = s["out"].clone()                                             # columns behind the vocabulary stay as they were
    out[:, :V] = x
    return out


PLAIN = {"attend": attend_plain, "write": write_plain, "assign": assign_plain, "release": release_plain, "adjust": adjust_plain}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(c, seed):
    op = c["op"]
    if op in ("assign", "release"):
        return None                                                    # whole numbers
    s = prepare(c, seed)
    if op == "attend":
        kv, hs, p = c["kv_heads"], c["hs"], c["page"]
        group = c["heads"] // kv
        outs = torch.zeros(c["n"], c["heads"], hs, dtype=torch.float64, device="cuda")
        lses = torch.full((c["n"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
        for i, L in enumerate(attend_lengths(c)):
            if L == 0:
                continue
            used = s["tables"][i, :-(-L // p)].long()
            for h in range(kv):
                k, v = (x[used, :, h].reshape(-1, hs)[:L].double() for x in (s["k"], s["v"]))
                q = s["qkv"][i, h * group * hs:(h + 1) * group * hs].reshape(group, hs).double()
                score = (q @ k.T) * s["scale"]
                lse = torch.logsumexp(score, 1)
                lses[i, h * group:(h + 1) * group] = lse
                outs[i, h * group:(h + 1) * group] = torch.exp(score - lse[:, None]) @ v
        return outs.reshape(c["n"], -1), lses
    if op == "write":
        at, kv, hs = c["heads"] * c["hs"], c["kv_heads"], c["hs"]
        got = [s["k"].double().reshape(-1, kv * hs), s["v"].double().reshape(-1, kv * hs)]
        T = c["tokens"] - c["padded"]
        for j in range(2):
            got[j][s["slots"][:T].long()] = s["qkv"][:T, at + j * kv * hs:at + (j + 1) * kv * hs].double()
        return [x.reshape(s["k"].shape) for x in got]
    n, V = c["n"], c["V"]
    out = s["out"].double()
    for i in range(n):
        x = s["logits"][i, :V].double()
        text = s["history"][i, :int(s["lens"][i])].long()
        seen = torch.unique(text)
        r = s["repetition"][i].double()
        x[seen] = torch.where(x[seen] > 0, x[seen] / r, x[seen] * r)
        drawn, times = torch.unique(text[int(s["prompts"][i]):], return_counts=True)
        x[drawn] -= s["frequency"][i].double() * times + s["presence"][i].double()
        if c["biases"]:
            ids, values = s["bias_ids"][i].tolist(), s["bias"][i].tolist()
            last = dict(zip(ids[:int(s["bias_lens"][i])], values))
            if last:
                x[torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if c["mask"]:
            bits = (s["mask"][i][:, None] >> torch.arange(32, device="cuda")) & 1
            x[bits.reshape(-1)[:V] == 0] = -math.inf
        out[i, :V] = x
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(c):
    op = c["op"]
    if op == "attend":
        tokens, q = sum(attend_lengths(c)), c["n"] * c["heads"] * c["hs"]
        return {"bytes": tokens * c["kv_heads"] * c["hs"] * 2 * SIZE[c["type"]] + 8 * q + 4 * c["n"] * c["heads"],
                "flops": 4 * tokens * c["heads"] * c["hs"]}
    if op == "write":
        return {"bytes": (c["tokens"] - c["padded"]) * c["kv_heads"] * c["hs"] * 2 * (4 + SIZE[c["type"]]) + 4 * c["tokens"], "flops": 0}
    if op == "assign":
        new = assign_lengths(c)[1]
        fresh = int(min(1.0, c["room"]) * assign_asked(c))
        return {"bytes": 4 * (4 * c["n"] + 2 * fresh + 3 * sum(new)), "flops": 0}
    if op == "release":
        lens, done = release_lengths(c)
        return {"bytes": 4 * (3 * c["n"] + 2 * sum(-(-x // c["page"]) for x, d in zip(lens, done) if d)), "flops": 0}
    rows = c["n"] * c["V"]
    return {"bytes": 8 * rows + (rows // 8 if c["mask"] else 0) + 3 * c["n"] * c["history"] + 6 * c["n"] * c["biases"], "flops": 2 * rows}
