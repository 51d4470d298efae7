"""Plain forms of the serving operators (paged cache, attention over it, adjusted logits), written from their definitions in
bmb.h: loops over requests in Python integers, and sums in 64 bits."""
import numpy as np


def assign(tables, lens, new, free_pages, free_count, page_size, pages, max_tokens):
    """(tables, lens_out, slots, positions, owners, starts, free_left) after bmb_pages_assign."""
    tables = tables.copy()
    n, max_pages = tables.shape
    free = min(max(int(free_count), 0), pages)
    lens_out, starts = [], []
    slots, positions, owners = (np.full(max_tokens, x, np.int64) for x in (-1, 0, -1))
    begin, taken, left = 0, 0, free
    for i in range(n):
        L, A = max(int(lens[i]), 0), max(int(new[i]), 0)
        starts.append(min(begin, max_tokens))
        have, want = -(-L // page_size), -(-(L + A) // page_size)
        fits = want <= max_pages and begin + A <= max_tokens
        if fits:
            taken += want - have
        served = fits and (want == have or taken <= free)
        if served:
            for k in range(have, want):
                left -= 1
                tables[i, k] = free_pages[left]
        lens_out.append(L + A if served else L)
        for j in range(min(A, max_tokens - begin) if begin < max_tokens else 0):
            t, pos = begin + j, L + j
            positions[t], owners[t] = min(pos, 2 ** 31 - 1), i
            if served:
                page = int(tables[i, pos // page_size])
                if 0 <= page < pages:
                    slots[t] = page * page_size + pos % page_size
        begin += A
    starts.append(min(begin, max_tokens))
    return tables, np.array(lens_out, np.int64), slots, positions, owners, np.array(starts), left


def release(free_pages, free_count, lens, tables, done, page_size, pages):
    """(free_pages, free_out, lens_out) after bmb_pages_release."""
    stack, free = free_pages.copy(), min(max(int(free_count), 0), pages)
    out = []
    for i in range(len(lens)):
        L = max(int(lens[i]), 0)
        if done[i]:
            for page in tables[i, :-(-L // page_size)]:
                if 0 <= page < pages and free < pages:
                    stack[free] = page
                    free += 1
        out.append(0 if done[i] else L)
    return stack, free, np.array(out, np.int64)


def attention(torch, q, k, v, tables, lens, scale):
    """q [n, heads, hs], k and v [pages, page, kv heads, hs] (any strides), in 64 bits on their device: outputs, lse, and for each
    output what it is made of: the largest sum |q k| scale of a token that counts, the largest |v|, and how many count."""
    n, heads, hs = q.shape
    pages, page, kv = k.shape[:3]
    group = heads // kv
    out = torch.zeros(n, heads, hs, dtype=torch.float64, device=q.device)
    lse = torch.full((n, heads), -float("inf"), dtype=torch.float64, device=q.device)
    size, top, count = (torch.zeros(n, heads, dtype=torch.float64, device=q.device) for _ in range(3))
    for i in range(n):
        held = [(int(p), min(page, lens[i] - j * page)) for j, p in enumerate(tables[i]) if lens[i] > j * page]
        rows = [(p, used) for p, used in held if 0 <= p < pages]
        if not rows:
            continue
        for h in range(kv):
            ks, vs = (torch.cat([x[p, :used, h] for p, used in rows]).double() for x in (k, v))
            mine = slice(h * group, (h + 1) * group)
            s = q[i, mine].double() @ ks.T * scale
            lse[i, mine] = torch.logsumexp(s, 1)
            out[i, mine] = torch.exp(s - lse[i, mine, None]) @ vs
            size[i, mine] = (q[i, mine].double().abs() @ ks.abs().T).amax(1) * abs(scale)
            top[i, mine] = vs.abs().max()
            count[i, mine] = len(ks)
    return out, lse, size, top, count


def attention_bounds(hs, size, top, count):
    """How far fp32 arithmetic may be from 64 bits, from its roundings (u = 2^-24 each).  A score is a sum of hs products in chains
    of at most hs / 4 + 8 roundings (steps of the matrix unit, which cuts off: two units each; pieces of operands; the joining of
    lanes), so it is off by d = (hs / 4 + 8) u sum|q k| scale at most.  A weight exp(s - m) is then off by 2 d of itself, and each output
    by 2 d max|v|; the exponential and its argument, the sums over tokens (at most count / 16 roundings a chain), the joining of
    parts and the division add (count / 16 + 48) u max|v|."""
    u = 2.0 ** -24
    d = (hs / 4 + 8) * u * size
    rest = (count / 16 + 48) * u
    return (2 * d + rest) * top, d + rest


def adjust(logits, V, history=None, lens=None, prompts=None, rep=None, freq=None, pres=None, bias_ids=None, bias=None, bias_lens=None, allowed=None):
    """Rows of fp32 logits after bmb_logits_adjust, every step rounded to fp32."""
    f = np.float32
    out = logits.copy()
    with np.errstate(all="ignore"):
        for i in range(len(out)):
            if history is not None:
                text = [int(t) for t in history[i][:max(min(int(lens[i]), history.shape[1]), 0)]]
                drawn = {}
                for t in text[max(int(prompts[i]), 0) if prompts is not None else 0:]:
                    drawn[t] = drawn.get(t, 0) + 1
                for t in set(text):
                    if not 0 <= t < V:
                        continue
                    x = out[i, t]
                    if rep is not None:
                        x = f(x / f(rep[i])) if x > 0 else f(x * f(rep[i]))
                    if t in drawn:
                        if freq is not None:
                            x = f(x - f(f(freq[i]) * f(drawn[t])))
                        if pres is not None:
                            x = f(x - f(pres[i]))
                    out[i, t] = x
            if bias_ids is not None:
                last = {}
                for j in range(max(min(int(bias_lens[i]), bias_ids.shape[1]), 0)):
                    if 0 <= bias_ids[i, j] < V:
                        last[int(bias_ids[i, j])] = bias[i, j]
                for t, b in last.items():
                    out[i, t] = f(out[i, t] + f(b))
            if allowed is not None:
                v = np.arange(V)
                out[i, :V][(allowed[i][v // 32] >> (v % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return out
