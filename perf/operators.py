"""The operators of the paged 8-bit KV cache and the work they are measured on.

Three operators that a server runs one after the other in every step:

  plan     `paged_kv_plan`: pages for the tokens of this step from a stack of free pages, block-table entries, the slot
           of every new token; pages of finished requests go back to the stack.
  append   `paged_kv_append`: new keys and values are rounded to 8 bits (e4m3 or int8) into the pages of a cache that
           holds one power-of-two scale for each page and head.
  decode   `flash_attention_decode_paged_8bit`: one query token for each request against that cache.

`run` computes them in elementary torch operations where `own` is false and through the framework where it is true.
"""
import os
import sys

import torch

own = False

_E4M3_MAX, _INT8_MAX = 448.0, 127.0
_MIN_EXP = -126          # the smallest scale is 2^-126: a page of zeros has it


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------
def _plan(name, batch, lens, new, num_tokens_pad, bs, release, width):
    return {"name": name, "op": "plan", "batch": batch, "min_len": lens[0], "max_len": lens[1], "min_new": new[0],
            "max_new": new[1], "pad": num_tokens_pad, "block_size": bs, "release_every": release, "max_blocks": width}


def _append(name, batch, lens, new, heads, dim, bs, dtype, cache, pad):
    return {"name": name, "op": "append", "batch": batch, "min_len": lens[0], "max_len": lens[1], "min_new": new[0],
            "max_new": new[1], "heads_kv": heads, "head_dim": dim, "block_size": bs, "dtype": dtype, "cache": cache,
            "pad": pad}


def _decode(name, batch, lens, heads_q, heads_kv, dim, bs, dtype, cache):
    return {"name": name, "op": "decode", "batch": batch, "min_len": lens[0], "max_len": lens[1], "heads_q": heads_q,
            "heads_kv": heads_kv, "head_dim": dim, "block_size": bs, "dtype": dtype, "cache": cache}


def listed():
    return [
        # one decode step of a running batch: a token for each request, a new page for one request in sixteen
        _plan("plan step 64", 64, (1, 16000), (1, 1), 0, 16, 0, 1024),
        # a step that mixes chunks of prompts with running requests, some of which end; the packed batch is padded
        _plan("plan mixed 256", 256, (0, 6000), (1, 511), 77, 16, 7, 512),
        # the smallest decode step: four requests, 8 KV heads of 128 (the paged benchmark's cache)
        _append("append step 4", 4, (100, 5001), (1, 1), 8, 128, 16, "float16", "float8_e4m3fn", 0),
        # a large decode step: most pages are partly filled, and the new token outgrows the scale of some
        _append("append step 128", 128, (1, 4000), (1, 1), 8, 128, 64, "bfloat16", "int8", 0),
        # four prompts of 2048 tokens
        _append("append prompts 4x2048", 4, (0, 0), (2048, 2048), 8, 128, 16, "bfloat16", "float8_e4m3fn", 0),
        # a mixed step: ragged chunks of prompts beside running requests, narrow heads, padding behind the last token
        _append("append mixed 64", 64, (0, 2111), (1, 1021), 16, 64, 32, "float16", "int8", 53),
        # the shortest context of the paged benchmark, where latency is everything
        _decode("decode 1x8/8x256", 1, (256, 256), 8, 8, 128, 16, "float16", "float8_e4m3fn"),
        # one long conversation
        _decode("decode 1x32/8x4096", 1, (4096, 4096), 32, 8, 128, 16, "bfloat16", "float8_e4m3fn"),
        # the paged benchmark's batch with full and with ragged contexts
        _decode("decode 4x32/8x16384", 4, (16384, 16384), 32, 8, 128, 16, "float16", "int8"),
        _decode("decode 4x32/8 ragged", 4, (3218, 15003), 32, 8, 128, 16, "bfloat16", "float8_e4m3fn"),
        # a server's batch: many ragged contexts, larger pages
        _decode("decode 64x32/8 ragged", 64, (1, 16381), 32, 8, 128, 64, "bfloat16", "float8_e4m3fn"),
        # few narrow KV heads under wide groups, odd lengths
        _decode("decode 33x32/2x64 ragged", 33, (7, 8001), 32, 2, 64, 32, "float16", "int8"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "decode", "decode", "decode"])
    bs = rng.choice([8, 16, 32, 64, 128])
    if op == "plan":
        batch = _log_int(rng, 1, 300)
        new = _log_int(rng, 1, 500)
        longest = _log_int(rng, 1, 16000)
        width = -(-(longest + new) // bs) + rng.randint(0, 3)
        return {"op": op, "batch": batch, "min_len": 0, "max_len": longest, "min_new": 1, "max_new": new,
                "pad": rng.randint(0, 100), "block_size": bs, "release_every": rng.choice([0, 3, 10]),
                "max_blocks": width}
    dtype = rng.choice(["float16", "bfloat16"])
    cache = rng.choice(["float8_e4m3fn", "int8"])
    heads_kv = rng.choice([1, 2, 3, 4, 8, 16])
    dim = rng.choice([64, 128, 128, 256])
    if op == "append":
        room = 64 * 511 * 16 * 64       # values of the largest listed append
        batch = _log_int(rng, 1, 128)
        new = _log_int(rng, 1, max(1, min(4096, room // (batch * heads_kv * dim))))
        pool = room // (batch * heads_kv * dim)
        return {"op": op, "batch": batch, "min_len": 0, "max_len": _log_int(rng, 1, max(1, min(8000, pool))),
                "min_new": 1, "max_new": new, "heads_kv": heads_kv, "head_dim": dim, "block_size": bs, "dtype": dtype,
                "cache": cache, "pad": rng.randint(0, 60)}
    room = 64 * 8191 * 8 * 128          # values of the keys of the largest listed batch
    batch = _log_int(rng, 1, 128)
    longest = _log_int(rng, 1, max(1, min(32000, room // (batch * heads_kv * dim))))
    group = rng.choice([1, 2, 4, 5, 8, 16])
    return {"op": op, "batch": batch, "min_len": rng.choice([1, longest, max(1, longest // 3)]), "max_len": longest,
            "heads_q": heads_kv * group, "heads_kv": heads_kv, "head_dim": dim, "block_size": bs, "dtype": dtype,
            "cache": cache}


def _spread(n, lo, hi):
    """n lengths from lo to hi, both among them: the same for every seed (which only orders them)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _cdiv(a, b):
    return -(-a // b)


def work(case):
    lens = _spread(case["batch"], case["min_len"], case["max_len"])
    bs = case["block_size"]
    if case["op"] == "plan":
        new = _spread(case["batch"], case["min_new"], case["max_new"])
        tokens = sum(new) + case["pad"]
        pages = sum(_cdiv(a + b, bs) - _cdiv(a, bs) for a, b in zip(lens, new))
        if case["release_every"]:
            pages -= pages // case["release_every"]
        # lengths in and out, offsets, a stack entry read and a table entry written for each page, a slot for each token
        return {"bytes": 16 * case["batch"] + 8 * pages + 8 * tokens, "flops": 0}
    row = case["heads_kv"] * case["head_dim"]
    if case["op"] == "append":
        new = _spread(case["batch"], case["min_new"], case["max_new"])
        pages = sum(_cdiv(b, bs) for b in new)
        # 16-bit keys and values read, 8-bit ones written, a slot for each token, two scales for each page and head
        return {"bytes": sum(new) * (row * 6 + 8) + 8 * case["pad"] + pages * case["heads_kv"] * 8, "flops": 4 * sum(new) * row}
    pages, tokens = sum(_cdiv(n, bs) for n in lens), sum(lens)
    # keys and values of 8 bits, two scales for each page and head, the table, the queries and the outputs
    return {"bytes": 2 * tokens * row + pages * (8 * case["heads_kv"] + 4) + 4 * case["batch"]
            + 4 * case["batch"] * case["heads_q"] * case["head_dim"],
            "flops": 4 * tokens * case["heads_q"] * case["head_dim"]}


# ---------------------------------------------------------------------------------------------------
# 8-bit values under power-of-two scales
# ---------------------------------------------------------------------------------------------------
def _scale_for(amax, cache):
    """The smallest power of two s >= 2^-126 with amax <= s * (largest code); fp32 in, fp32 out, exact."""
    top = 0.875 if cache == "float8_e4m3fn" else 127.0 / 128.0    # the largest code's significand in [1/2, 1)
    top_exp = 9 if cache == "float8_e4m3fn" else 7
    m, e = torch.frexp(amax)
    e = e - top_exp + (m > top).to(e.dtype)
    e = torch.where(amax > 0, e, torch.full_like(e, _MIN_EXP)).clamp_min(_MIN_EXP)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x, cache):
    """fp32 values in units of their scale, rounded to the nearest 8-bit code (ties to even)."""
    if cache == "int8":
        return x.round().clamp(-_INT8_MAX, _INT8_MAX).to(torch.int8)
    return x.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _bytes_of(t):
    """The cache as bytes, for indexing and copies that keep bits."""
    return t.view(torch.uint8)


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ordered(values, g):
    v = torch.tensor(values, dtype=torch.int32, device="cuda")
    return v[torch.randperm(len(values), generator=g, device="cuda")].contiguous()


def _tables(lens, width, num_blocks, bs, g):
    """A block table of random pages that covers `lens` (int32 tensor), and the ids that are left over."""
    have = torch.div(lens + (bs - 1), bs, rounding_mode="floor").long()
    ids = torch.randperm(num_blocks, generator=g, device="cuda").int()
    before = have.cumsum(0) - have
    col = torch.arange(width, device="cuda")
    at = (before[:, None] + col[None]).clamp_max(num_blocks - 1)
    table = torch.where(col[None] < have[:, None], ids[at], torch.full_like(ids[:1], -1)).contiguous()
    return table, ids


def _values(g, dtype, *shape):
    """Keys or values as a projection gives them: channels of different size, and tokens that stand out."""
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    channel = torch.exp(0.7 * torch.randn(*shape[-2:], generator=g, device="cuda"))
    token = torch.exp(0.4 * torch.randn(*shape[:-2], 1, 1, generator=g, device="cuda"))
    return x.mul_(channel).mul_(token).to(dtype)


def _cache(g, num_blocks, bs, heads, dim, cache):
    """A filled cache and its scales."""
    x = _values(g, torch.float32, num_blocks, bs, heads, dim)
    scales = _scale_for(x.abs().amax(dim=(1, 3)), cache)
    return _codes(x.div_(scales[:, None, :, None]), cache), scales


def prepare(case, seed):
    g = _generator(seed)
    bs, batch = case["block_size"], case["batch"]
    lens = _ordered(_spread(batch, case["min_len"], case["max_len"]), g)
    if case["op"] == "decode":
        dtype = getattr(torch, case["dtype"])
        width = _cdiv(case["max_len"], bs)
        num_blocks = sum(_cdiv(n, bs) for n in _spread(batch, case["min_len"], case["max_len"])) + 3
        table, _ = _tables(lens, width, num_blocks, bs, g)
        k, ks = _cache(g, num_blocks, bs, case["heads_kv"], case["head_dim"], case["cache"])
        v, vs = _cache(g, num_blocks, bs, case["heads_kv"], case["head_dim"], case["cache"])
        q = torch.randn(batch, case["heads_q"], case["head_dim"], generator=g, device="cuda").to(dtype)
        return {"case": case, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table, "lens": lens}
    new_list = _spread(batch, case["min_new"], case["max_new"])
    new = _ordered(new_list, g)
    tokens = sum(new_list) + case["pad"]
    most = sum(_cdiv(a, bs) for a in _spread(batch, case["min_len"], case["max_len"])) + sum(_cdiv(n, bs) for n in new_list)
    num_blocks = most + 5
    if case["op"] == "plan":
        table, ids = _tables(lens, case["max_blocks"], num_blocks, bs, g)
        used = torch.div(lens + (bs - 1), bs, rounding_mode="floor").sum()
        free_count = (num_blocks - used).to(torch.int32).reshape(1)
        # the stack of free pages: the ids that no request holds, at its bottom
        at = torch.arange(num_blocks, device="cuda")
        free = torch.where(at < free_count, ids[(at + used) % num_blocks], torch.full_like(ids, -1)).contiguous()
        if case["release_every"]:
            new = torch.where(torch.arange(batch, device="cuda") % case["release_every"] == case["release_every"] - 1,
                              torch.full_like(new, -1), new).contiguous()
        return {"case": case, "lens": lens, "new": new, "table": table, "free": free, "count": free_count,
                "tokens": tokens}
    # append: pages for old and new tokens, a slot for each new one
    dtype = getattr(torch, case["dtype"])
    width = _cdiv(case["max_len"] + case["max_new"], bs) + 1
    table, _ = _tables(lens + new, width, num_blocks, bs, g)
    k, ks = _cache(g, num_blocks, bs, case["heads_kv"], case["head_dim"], case["cache"])
    v, vs = _cache(g, num_blocks, bs, case["heads_kv"], case["head_dim"], case["cache"])
    cu = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    cu[1:] = new.cumsum(0)
    t = torch.arange(tokens, device="cuda")
    b = (torch.searchsorted(cu, t.int(), right=True) - 1).clamp_max(batch - 1)
    pos = lens[b] + (t - cu[b])
    slots = table[b, torch.div(pos, bs, rounding_mode="floor").clamp_max(width - 1)].long() * bs + pos % bs
    slots = torch.where(t < cu[-1], slots, torch.full_like(slots, -1)).contiguous()
    key = _values(g, dtype, tokens, case["heads_kv"], case["head_dim"])
    value = _values(g, dtype, tokens, case["heads_kv"], case["head_dim"])
    return {"case": case, "key": key, "value": value, "k": k, "v": v, "ks": ks, "vs": vs, "slots": slots, "cu": cu}


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------
def _framework():
    """The package, from its folder in this repository."""
    if "fa_b200" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "flash-attention-rdna3_b200"))
    import fa_b200

    return fa_b200


def run(state):
    case = state["case"]
    if case["op"] == "plan":
        if own:
            slots, cu, lens, count = _framework().paged_kv_plan(
                state["lens"], state["new"], state["table"], state["free"], state["count"], state["tokens"],
                case["block_size"])
        else:
            slots, cu, lens, count = _plan_plain(state)
        return {"slots": slots, "cu": cu, "lens": lens, "count": count, "table": state["table"], "free": state["free"]}
    if case["op"] == "append":
        if own:
            _framework().paged_kv_append(state["key"], state["value"], state["k"], state["v"], state["ks"], state["vs"],
                                         state["slots"])
        else:
            _append_plain(state["key"], state["k"], state["ks"], state["slots"], state["cu"], case)
            _append_plain(state["value"], state["v"], state["vs"], state["slots"], state["cu"], case)
        return {"k": state["k"], "v": state["v"], "ks": state["ks"], "vs": state["vs"]}
    if own:
        return _framework().flash_attention_decode_paged_8bit(
            state["q"], state["k"], state["v"], state["ks"], state["vs"], state["table"], state["lens"])
    return _decode_plain(state)


def _plan_plain(state):
    case, lens, new = state["case"], state["lens"].long(), state["new"].long()
    table, free, count = state["table"], state["free"], state["count"].long()
    bs, width, capacity = case["block_size"], state["table"].shape[1], state["free"].numel()
    ending = new < 0
    fresh = new.clamp_min(0)
    cu = torch.cat((torch.zeros_like(fresh[:1]), fresh.cumsum(0)))
    have = torch.div(lens + (bs - 1), bs, rounding_mode="floor")
    back = torch.where(ending, have.clamp_max(width), torch.zeros_like(have))      # pages that return
    back_end = back.cumsum(0)
    available = count + back_end[-1]
    fits = ~ending & (lens + fresh <= width * bs) & (cu[1:] <= state["tokens"])
    need = torch.where(fits, torch.div(lens + fresh + (bs - 1), bs, rounding_mode="floor") - have, torch.zeros_like(have))
    need_end = need.cumsum(0)
    served = fits & ((need == 0) | (need_end <= available))
    taken = torch.where(served, need, torch.zeros_like(need)).sum()

    def entry(place):
        """What the stack holds at `place` once the pages of ending requests lie on top of it."""
        k = (place - count).clamp_min(0)
        b = torch.searchsorted(back_end, k.contiguous(), right=True).clamp_max(back_end.numel() - 1)
        col = (k - (back_end[b] - back[b])).clamp(0, width - 1)
        return torch.where(place < count, free[place.clamp(0, capacity - 1)], table[b, col])

    # block-table entries of the new pages, popped from the top of the stack in the order of the requests
    col = torch.arange(width, device=table.device)
    index = col[None] - have[:, None]
    ids = entry(available - 1 - (need_end - need)[:, None] - index)
    mine = served[:, None] & (index >= 0) & (index < need[:, None])
    at = torch.arange(capacity, device=table.device)
    left = available - taken
    pushed = torch.where((at >= count) & (at < left), entry(at), free)
    table.copy_(torch.where(mine, ids, table))
    free.copy_(pushed)
    # the slot of every token
    t = torch.arange(state["tokens"], device=table.device)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp_max(new.numel() - 1)
    pos = lens[b] + t - cu[b]
    page = table[b, torch.div(pos, bs, rounding_mode="floor").clamp(0, width - 1)].long()
    ok = (t < cu[-1]) & served[b] & (page >= 0) & (page < capacity)
    slots = torch.where(ok, page * bs + pos % bs, torch.full_like(pos, -1))
    after = torch.where(ending, torch.zeros_like(lens), torch.where(served, lens + fresh, lens))
    return slots, cu.int(), after.int(), left.int().reshape(1)


def _append_plain(x, cache, scales, slots, cu, case):
    bs, kind, pages = case["block_size"], case["cache"], scales.shape[0]
    heads, dim = x.shape[1], x.shape[2]
    codes = _bytes_of(cache)
    known = slots >= 0
    page = torch.where(known, torch.div(slots, bs, rounding_mode="floor"), torch.full_like(slots, pages))
    # the largest magnitude that each page receives (one more row takes what has no slot)
    amax = torch.zeros(pages + 1, heads, dtype=torch.float32, device=x.device)
    amax.scatter_reduce_(0, page[:, None].expand(-1, heads), x.float().abs().amax(-1), "amax")
    wanted = _scale_for(amax[:pages], kind)
    # a request's first page may hold older tokens: its scale never shrinks, and they are rounded again if it grows
    first = slots[cu[:-1].long()]
    offset, shared = first % bs, torch.div(first, bs, rounding_mode="floor")
    old = scales[shared]
    new = torch.where((offset > 0)[:, None], torch.maximum(old, wanted[shared]), wanted[shared])
    held = cache[shared].float() * (old / new)[:, None, :, None]
    keep = torch.arange(bs, device=x.device)[None] < offset[:, None]
    codes[shared] = torch.where(keep[:, :, None, None], _bytes_of(_codes(held, kind)), codes[shared])
    touched = torch.zeros(pages + 1, dtype=torch.bool, device=x.device)
    touched[page] = True
    wanted[shared] = new
    scales.copy_(torch.where(touched[:pages, None], wanted, scales))
    # the new tokens
    unit = scales[page.clamp_max(pages - 1)][:, :, None]
    fresh = _bytes_of(_codes(x.float() / unit, kind))
    flat = codes.view(pages * bs, heads, dim)
    last = torch.where(known, slots, first[-1:])
    flat[last] = torch.where(known[:, None, None], fresh, fresh[cu[-2:-1].long()])


def _decode_plain(state):
    q, table, lens = state["q"].float(), state["table"], state["lens"]
    batch, heads_q, dim = q.shape
    pages, bs, heads, _ = state["k"].shape
    width = table.shape[1]
    at = table.clamp(0, pages - 1).long()
    pos = torch.arange(width * bs, device=q.device)
    seen = (pos[None] < lens[:, None]) & (table >= 0).repeat_interleave(bs, 1)

    def rows(cache, scales):
        x = cache.view(torch.int8)[at].view(cache.dtype).float()
        x.mul_(scales[at][:, :, None, :, None])
        return x.view(batch, width * bs, heads, dim).permute(0, 2, 1, 3)

    q = q.view(batch, heads, heads_q // heads, dim)
    s = torch.matmul(q, rows(state["k"], state["ks"]).transpose(2, 3)) * dim ** -0.5
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, rows(state["v"], state["vs"])) / p.sum(-1, keepdim=True)
    return o.view(batch, heads_q, dim).to(state["q"].dtype)


# ---------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------
def _rounded64(x, kind):
    """64-bit values in units of their scale, to the nearest code."""
    if kind == "int8":
        return x.round().clamp(-127, 127)
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6)
    step = torch.exp2(exponent - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def exact(case, seed):
    if case["op"] == "plan":
        return None              # whole numbers only
    state = prepare(case, seed)
    bs = case["block_size"]
    if case["op"] == "decode":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads_q"] // case["heads_kv"]
        for b, n in enumerate(state["lens"].tolist()):
            ids = state["table"][b, :_cdiv(n, bs)].long()
            k, v = (torch.cat([(state[c][i:i + 1].double() * state[s][i].double()[None, None, :, None]).flatten(0, 1)
                               for i in ids.tolist()])[:n] if len(ids) < 4 else
                    (state[c].view(torch.uint8)[ids].view(state[c].dtype).double()
                     * state[s][ids].double()[:, None, :, None]).flatten(0, 1)[:n] for c, s in (("k", "ks"), ("v", "vs")))
            for h in range(case["heads_kv"]):
                q = state["q"][b, h * group:(h + 1) * group].double()
                p = torch.softmax(q @ k[:, h].T / case["head_dim"] ** 0.5, dim=-1)
                out[b, h * group:(h + 1) * group] = p @ v[:, h]
        return out
    largest = 127.0 if case["cache"] == "int8" else 448.0
    powers = torch.tensor([2.0 ** i for i in range(_MIN_EXP, 128)], dtype=torch.float64, device="cuda")
    cu, slots = state["cu"].tolist(), state["slots"]
    got = {}
    for x, c, s in (("key", "k", "ks"), ("value", "v", "vs")):
        codes, scales = state[c].double(), state[s].double()
        for b in range(case["batch"]):
            mine = slots[cu[b]:cu[b + 1]]
            o, n = int(mine[0]) % bs, len(mine)
            pages = _cdiv(o + n, bs)
            data = torch.zeros(pages * bs, *codes.shape[2:], dtype=torch.float64, device="cuda")
            data[o:o + n] = state[x][cu[b]:cu[b + 1]].double()
            data = data.view(pages, bs, *codes.shape[2:])
            ids = torch.div(mine[[max(0, j * bs - o) for j in range(pages)]], bs, rounding_mode="floor")
            amax = data.abs().amax(dim=(1, 3))
            unit = powers[torch.searchsorted(powers * largest, amax)]    # the smallest with amax <= power * largest
            if o:
                unit[0] = torch.maximum(unit[0], scales[ids[0]])
            fresh = _rounded64(data / unit[:, None, :, None], case["cache"])
            fresh[0, :o] = _rounded64(codes[ids[0], :o] * (scales[ids[0]] / unit[0])[None, :, None], case["cache"])
            place = torch.arange(pages * bs, device="cuda").view(pages, bs)
            codes[ids] = torch.where((place < o + n)[:, :, None, None], fresh, codes[ids])
            scales[ids] = unit
        got[c], got[s] = codes, scales
    return {"k": got["k"], "v": got["v"], "ks": got["ks"], "vs": got["vs"]}
