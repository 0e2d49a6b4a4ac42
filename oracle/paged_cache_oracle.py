"""Plain statements of the paged 8-bit KV cache operators: request by request, in 64 bits, on any device."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def plan_ref(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size):
    """Returns (slots, cu, lens, count, table, stack) as lists, by walking the requests and moving single pages."""
    lens, new = [int(x) for x in context_lens], [int(x) for x in new_lens]
    table, stack = [list(map(int, r)) for r in block_table.tolist()], [int(x) for x in free_blocks]
    width, capacity = len(table[0]), len(stack)
    pages = lambda n: -(-n // block_size)
    held = stack[:int(free_count)]
    for b, n in enumerate(new):
        if n < 0:
            held += table[b][:min(pages(max(lens[b], 0)), width)]
    slots, cu, out_lens, needed, available = [-1] * num_tokens, [0], [], 0, len(held)
    for b, n in enumerate(new):
        begin = cu[-1]
        cu.append(begin + max(n, 0))
        if n < 0:
            out_lens.append(0)
            continue
        L = lens[b]
        if L < 0 or L + n > width * block_size or cu[-1] > num_tokens:
            out_lens.append(L)
            continue
        need = pages(L + n) - pages(L)
        needed += need
        if need > 0 and needed > available:
            out_lens.append(L)
            continue
        for j in range(pages(L), pages(L + n)):
            table[b][j] = held.pop()
        for i in range(n):
            page = table[b][(L + i) // block_size]
            if 0 <= page < capacity:
                slots[begin + i] = page * block_size + (L + i) % block_size
        out_lens.append(L + n)
    left = min(len(held), capacity)             # (pages that return to a full stack are lost)
    for i in range(int(free_count), left):      # what lies above the old top is written; popped places stay
        stack[i] = held[i]
    return slots, cu, out_lens, left, table, stack


def round_codes(x, dtype):
    """64-bit values in units of their scale -> the nearest code, ties to even, as 64-bit values."""
    if dtype == torch.int8:
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
    exponent = torch.floor(torch.log2(x.abs().clamp(2.0 ** -40, 2.0 ** 40))).clamp(-6, 8)
    step = torch.exp2(exponent - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def scale_for(amax, dtype):
    """The smallest power of two s >= 2^-126 with amax <= s * largest code."""
    powers = torch.tensor([2.0 ** i for i in range(-126, 128)], dtype=torch.float64, device=amax.device)
    return powers[torch.searchsorted(powers * LARGEST[dtype], amax)]


def append_ref(x, cache, scales, slots):
    """(codes, scales) in 64 bits after the tokens x (tokens, heads, dim) went to their slots."""
    codes, unit = cache.double(), scales.double().clone()
    blocks, bs = cache.shape[:2]
    slots = [int(s) for s in slots]
    page = [s // bs if 0 <= s < blocks * bs else -1 for s in slots]
    t = 0
    while t < len(slots):
        if page[t] < 0:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and page[t + n] == page[t]:
            n += 1
        o, p = slots[t] % bs, page[t]
        assert slots[t:t + n] == list(range(slots[t], slots[t] + n))
        rows = x[t:t + n].double()
        finite = torch.where(torch.isfinite(rows), rows, torch.zeros_like(rows))
        s = scale_for(finite.abs().amax(dim=(0, 2)).contiguous(), cache.dtype)
        if o:
            s = torch.maximum(s, unit[p])
            codes[p, :o] = round_codes(codes[p, :o] * (unit[p] / s)[None, :, None], cache.dtype)
        codes[p, o:o + n] = round_codes(rows / s[None, :, None], cache.dtype)
        unit[p] = s
        t += n
    return codes, unit


def decode8_ref(q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, softmax_scale=None):
    """(out, bound) in 64 bits, both (batch, heads_q, dim). `bound` is what a kernel may be off before it rounds its
    output, by arithmetic:
      * p times value scale rounded to fp16 in front of the product with V, relative to a power of two: 2^-11 of each
        p |v|, and for those below fp16's normal range 2^-25 of that unit. The unit is at most 2^-10 of the row's largest
        p * scale, or 2^-110 of the largest p times the largest scale where that is more;
      * fp32 sums of dim products in the scores: at most (dim / 16 + 8) roundings or truncations of 2^-23 relative to
        sum |q k|, which the exponential turns into that relative error of p, once in the sum and once in its norm;
      * 2^-18 for the exponential and the fp32 sums over tokens (relative to sum p |v|), over at most 2^14 tokens a
        running sum of 16-token products."""
    B, Hq, D = q.shape
    blocks, bs, Hk, _ = k_cache.shape
    group, scale = Hq // Hk, 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = min(max(int(context_lens[b]), 0), block_table.shape[1] * bs)
        ks, vs, units, codes = [], [], [], []
        for j in range(-(-n // bs)):
            page, m = int(block_table[b, j]), min(bs, n - j * bs)
            if 0 <= page < blocks:
                ks.append(k_cache[page, :m].double() * k_scales[page].double()[None, :, None])
                codes.append(v_cache[page, :m].double())
                units.append(v_scales[page].double()[None].expand(m, Hk))
        if not ks:
            continue
        k, code, unit = torch.cat(ks), torch.cat(codes), torch.cat(units)
        v = code * unit[:, :, None]
        for h in range(Hk):
            rows = slice(h * group, (h + 1) * group)
            qh = q[b, rows].double()
            s = qh @ k[:, h].T * scale
            p = torch.softmax(s, dim=-1)
            out[b, rows] = p @ v[:, h]
            weighted = p @ v[:, h].abs()
            sums = (qh.abs() @ k[:, h].abs().T * abs(scale)).amax(-1, keepdim=True)
            relative = 2.0 ** -11 + 2 * (D / 16 + 8) * 2.0 ** -23 * sums + 2.0 ** -18
            top = 1.0 / torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)   # p of the largest score
            most = unit[:, h].abs().max() * top
            step = 2.0 ** -10 * torch.maximum((p * unit[:, h].abs()).amax(-1, keepdim=True), 2.0 ** -100 * most)
            bound[b, rows] = relative * weighted + 2.0 ** -25 * step * code[:, h].abs().sum(0)
    return out, bound
