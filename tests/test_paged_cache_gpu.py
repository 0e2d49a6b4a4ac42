"""The paged 8-bit KV cache on the GPU: planning, appending and decoding against the oracle, and the three together."""
import pytest
import torch

import fa_b200
from fa_b200 import paged_cache
from oracle import paged_cache_oracle as oracle

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
CACHES = [E4M3, torch.int8]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def bytes_equal(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------------------
def random_plan(seed, batch, bs, width, max_new, spare, ends=0.2, pad=3):
    g = gen(seed)
    cap = width * bs
    lens = [int(x) for x in torch.randint(0, cap + 1, (batch,), generator=g)]
    new = [int(x) for x in torch.randint(0, max_new + 1, (batch,), generator=g)]
    new = [-int(e) if e else n for n, e in zip(new, (torch.rand(batch, generator=g) < ends).int())]
    held = [-(-n // bs) for n in lens]
    blocks = sum(held) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    table = torch.full((batch, width), -1, dtype=torch.int32)
    for b, n in enumerate(held):
        for j in range(n):
            table[b, j] = ids.pop()
    stack = torch.full((blocks,), -1, dtype=torch.int32)
    stack[:len(ids)] = ints(ids, "cpu")
    return ints(lens), ints(new), table.cuda(), stack.cuda(), ints([len(ids)]), sum(max(n, 0) for n in new) + pad


def check_plan(args, bs, inplace=False):
    lens, new, table, stack, count, tokens = args
    want = oracle.plan_ref(lens.tolist(), new.tolist(), table.cpu(), stack.cpu(), int(count), tokens, bs)
    before = lens.clone(), count.clone()
    got = fa_b200.paged_kv_plan(lens, new, table, stack, count, tokens, bs, inplace=inplace)
    for name, a, b in zip(("slots", "cu", "lens", "count", "table", "stack"),
                          (got[0], got[1], got[2], got[3][0], table, stack), want):
        assert a.tolist() == b, name
    if inplace:
        assert got[2] is lens and got[3] is count
    else:
        assert torch.equal(lens, before[0]) and torch.equal(count, before[1])
    return got


@pytest.mark.parametrize("batch, bs, width, max_new, spare", [
    (1, 16, 4, 1, 2), (3, 1, 9, 4, 20), (17, 16, 12, 40, 60), (64, 16, 128, 1, 9), (33, 64, 8, 300, 200),
    (512, 8, 30, 9, 500), (513, 16, 20, 30, 1000), (1500, 32, 6, 20, 1500), (40, 256, 3, 700, 100)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan(batch, bs, width, max_new, spare, inplace):
    check_plan(random_plan(batch + bs, batch, bs, width, max_new, spare), bs, inplace)


def test_plan_is_repeatable_with_lengths_kept():
    args = random_plan(5, 50, 16, 20, 60, 90)
    first = check_plan(args, 16)
    table, stack = args[2].clone(), args[3].clone()
    second = fa_b200.paged_kv_plan(*args, 16)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    assert torch.equal(table, args[2]) and torch.equal(stack, args[3])


def test_plan_when_pages_run_out_and_rows_are_full():
    for spare in (0, 1, 5, 17):
        check_plan(random_plan(spare, 40, 16, 10, 70, spare, ends=0.05), 16)


def test_plan_with_fewer_slots_than_tokens():
    lens, new, table, stack, count, tokens = random_plan(3, 30, 16, 20, 50, 200)
    for n in (0, 1, tokens // 2):
        check_plan((lens, new, table.clone(), stack.clone(), count, n), 16)


def test_plan_everything_ends_and_nothing_is_there():
    args = random_plan(8, 20, 16, 6, 5, 3)
    check_plan((args[0], torch.full_like(args[1], -1), *args[2:5], 4), 16)
    check_plan((torch.zeros_like(args[0]), torch.zeros_like(args[1]), torch.full_like(args[2], -1), args[3],
                ints([0]), 0), 16)


def test_plan_strange_values():
    """Negative and too large lengths, ids outside the pool, a count outside the stack: no slot, nothing written outside."""
    lens, new, table, stack, count, tokens = random_plan(11, 12, 16, 8, 40, 60, ends=0.0)
    lens[3], lens[5] = -7, 10 ** 9
    stack[:] = torch.where(torch.arange(stack.numel(), device="cuda") % 3 == 0, stack + 10 ** 6, stack)
    check_plan((lens, new, table, stack, count, tokens), 16)
    lens, new, table, stack, count, tokens = random_plan(12, 12, 16, 8, 40, 60, ends=0.3)
    fa_b200.paged_kv_plan(lens, new, table, stack, ints([10 ** 9]), tokens, 16)
    fa_b200.paged_kv_plan(lens, new, table, stack, ints([-5]), tokens, 16)
    torch.cuda.synchronize()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("given, meant", [(10 ** 9, None), (-5, 0), (2 ** 31 - 1, None), (-2 ** 31, 0)])
@pytest.mark.parametrize("ends", [0.0, 0.3, 1.0])
def test_plan_counts_outside_the_stack(given, meant, ends, inplace):
    """A count outside the stack is taken for a full or an empty one; neither the table nor the stack is written outside."""
    lens, new, table, stack, _, tokens = random_plan(12, 40, 16, 8, 40, 60, ends=ends)
    meant = stack.numel() if meant is None else meant
    want = oracle.plan_ref(lens.tolist(), new.tolist(), table.cpu(), stack.cpu(), meant, tokens, 16)
    wide, long = torch.full((44, 14), -9, dtype=torch.int32, device="cuda"), ints([-9] * (stack.numel() + 512))
    t, s = wide[2:42, 3:11], long[256:-256]
    t.copy_(table)
    s.copy_(stack)
    got = fa_b200.paged_kv_plan(lens, new, t, s, ints([given]), tokens, 16, inplace=inplace)
    for name, a, b in zip(("slots", "cu", "lens", "count", "table", "stack"), (*got[:3], got[3][0], t, s), want):
        assert a.tolist() == b, name
    t.fill_(-9)
    s.fill_(-9)
    assert (wide == -9).all() and (long == -9).all()


@pytest.mark.parametrize("inplace", [False, True])
def test_plan_of_the_largest_stack(inplace):
    """A stack of 2^31 - 1 places that is full but for ten: pages come back up to its last place, and a step that pops
    from there. (Only the top of the stack is looked at; the pool behind it need not exist for planning.)"""
    places = 2 ** 31 - 1
    stack = torch.empty(places, dtype=torch.int32, device="cuda")
    stack[-60:] = torch.arange(60, dtype=torch.int32, device="cuda")
    table = torch.full((600, 4), -1, dtype=torch.int32, device="cuda")
    table[5, :4], table[400, :2] = ints([2 ** 31 - 2, 7, 8, 9]), ints([1000, 11])
    lens, new = torch.zeros(2, 600, dtype=torch.int32, device="cuda")
    lens[5], lens[400], new[5], new[400] = 60, 20, -1, -1
    new[500], new[501] = 40, 17                 # three pages and two, popped from the ones that have just come back
    count = ints([places - 10])
    slots, cu, after, left = fa_b200.paged_kv_plan(lens, new, table, stack, count, 57, 16, inplace=inplace)
    assert int(left) == places - 10 + 6 - 5
    assert table[500].tolist() == [11, 1000, 9, -1] and table[501].tolist() == [8, 7, -1, -1]
    assert stack[-10:].tolist() == [2 ** 31 - 2] + list(range(51, 60))
    assert slots[:16].tolist() == list(range(176, 192)) and slots[-1] == 7 * 16
    assert after.nonzero().flatten().tolist() == [500, 501]


def test_plans_of_large_batches_from_two_threads():
    """C callers hold no lock: plans of different batches, both above what shared memory a kernel has unasked, are launched
    side by side, and none takes from another what it needs."""
    import ctypes
    import threading

    from fa_b200 import _lib

    lib, wrong = _lib.load(), []

    def caller(batch):
        torch.cuda.set_device(0)
        lens, new = torch.zeros(2, batch, dtype=torch.int32, device="cuda")
        table = torch.zeros(batch, 2, dtype=torch.int32, device="cuda")
        stack, count = torch.zeros(4, dtype=torch.int32, device="cuda"), ints([4])
        cu, lens_out = torch.empty(batch + 1, dtype=torch.int32, device="cuda"), torch.empty_like(lens)
        count_out = torch.empty_like(count)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        p = _lib.PagedPlanParams(batch, 2, 4, 16, 0, lens.data_ptr(), 1, new.data_ptr(), 1, table.data_ptr(), 2,
                                 stack.data_ptr(), count.data_ptr(), None, cu.data_ptr(), lens_out.data_ptr(),
                                 count_out.data_ptr())
        for _ in range(1500):
            rc = lib.fa_paged_plan(ctypes.byref(p), ctypes.c_void_p(stream.cuda_stream))
            if rc:
                wrong.append(rc)
        stream.synchronize()

    threads = [threading.Thread(target=caller, args=(n,)) for n in (8192, 2500, 8000, 3000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_plan_strided_inputs():
    lens, new, table, stack, count, tokens = random_plan(21, 25, 16, 9, 30, 60)
    wide = torch.full((25, 31), -9, dtype=torch.int32, device="cuda")
    wide[:, 4:13] = table
    lens2, new2 = torch.stack((lens, lens), 1)[:, 0], torch.stack((new, new, new), 1)[:, 1]
    check_plan((lens2, new2, wide[:, 4:13], stack, count, tokens), 16)
    assert (wide[:, :4] == -9).all() and (wide[:, 13:] == -9).all()


# ---------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------
def filled_cache(seed, blocks, bs, heads, dim, dtype):
    """Codes over the whole range under scales of different size (what lies in pages before a step)."""
    g = gen(seed)
    x = torch.randn(blocks, bs, heads, dim, generator=g)
    scales = torch.exp2(torch.randint(-6, 2, (blocks, heads), generator=g).float())
    if dtype == torch.int8:
        codes = (x * 40).round().clamp(-127, 127).to(torch.int8)
    else:
        codes = (x * 60).clamp(-448, 448).to(E4M3)
    return codes.cuda(), scales.cuda()


def runs_to_slots(runs, bs):
    """runs: (page, first offset, tokens); page None: tokens without a slot."""
    slots = []
    for page, o, n in runs:
        slots += [-1] * n if page is None else [page * bs + o + i for i in range(n)]
    return torch.tensor(slots, dtype=torch.int64, device="cuda")


def random_runs(seed, blocks, bs, requests, longest):
    """Requests whose first page may be half full, over a random permutation of pages."""
    g = gen(seed)
    pages = torch.randperm(blocks, generator=g).tolist()
    runs = []
    for _ in range(requests):
        o, n = int(torch.randint(0, bs, (1,), generator=g)), int(torch.randint(1, longest + 1, (1,), generator=g))
        while n > 0 and pages:
            m = min(n, bs - o)
            runs.append((pages.pop(), o, m))
            n, o = n - m, 0
        if int(torch.randint(0, 4, (1,), generator=g)) == 0:
            runs.append((None, 0, 2))
    return runs


def check_append(key, value, k, v, ks, vs, slots):
    want = [oracle.append_ref(x, c, s, slots.tolist()) for x, c, s in ((key, k, ks), (value, v, vs))]
    fa_b200.paged_kv_append(key, value, k, v, ks, vs, slots)
    for c, s, (codes, scales) in ((k, ks, want[0]), (v, vs, want[1])):
        assert torch.equal(s.double(), scales)
        assert torch.equal(torch.nan_to_num(c.double(), nan=1e9), torch.nan_to_num(codes, nan=1e9))


def inputs(seed, tokens, heads, dim, dtype):
    g = gen(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp(2 * torch.randn(tokens, heads, 1, generator=g))
    return x.to(dtype).cuda()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, dim, bs, requests, longest", [
    (8, 128, 16, 5, 1), (8, 128, 16, 7, 60), (2, 64, 32, 6, 100), (3, 256, 8, 5, 30), (1, 16, 64, 6, 150),
    (5, 32, 128, 4, 300), (1, 128, 256, 3, 600), (16, 64, 1, 9, 4), (4, 256, 64, 40, 1), (2, 128, 2, 11, 9),
    (1, 64, 16, 2, 1)])
def test_append(cache, dtype, heads, dim, bs, requests, longest):
    blocks = requests * (longest // bs + 2) + 2
    runs = random_runs(heads * dim + bs, blocks, bs, requests, longest)
    slots = runs_to_slots(runs, bs)
    k, ks = filled_cache(1, blocks, bs, heads, dim, cache)
    v, vs = filled_cache(2, blocks, bs, heads, dim, cache)
    n = slots.numel()
    check_append(inputs(3, n, heads, dim, dtype), inputs(4, n, heads, dim, dtype), k, v, ks, vs, slots)


@pytest.mark.parametrize("cache", CACHES)
def test_append_many_tokens(cache):
    """Enough tokens that a CTA starts the runs of several tokens, with runs across the CTAs' ranges."""
    blocks, bs, heads, dim = 700, 32, 8, 64
    runs = random_runs(9, blocks, bs, 60, 700)
    slots = runs_to_slots(runs, bs)
    assert slots.numel() > 8000
    k, ks = filled_cache(1, blocks, bs, heads, dim, cache)
    v, vs = filled_cache(2, blocks, bs, heads, dim, cache)
    n = slots.numel()
    check_append(inputs(3, n, heads, dim, torch.bfloat16), inputs(4, n, heads, dim, torch.bfloat16), k, v, ks, vs, slots)


@pytest.mark.parametrize("cache", CACHES)
def test_append_one_token_at_a_time(cache):
    """A page that fills token by token: its scale only grows, and every growth rounds the older tokens again."""
    bs, heads, dim = 16, 2, 64
    k, ks = filled_cache(1, 3, bs, heads, dim, cache)
    v, vs = filled_cache(2, 3, bs, heads, dim, cache)
    for i in range(2 * bs):
        x = inputs(i, 1, heads, dim, torch.float16) * (1.3 ** (i % bs))
        check_append(x, -x, k, v, ks, vs, torch.tensor([(1 + i // bs) * bs + i % bs], device="cuda"))
        if i % bs:
            assert (ks[1 + i // bs] >= grown).all()
        grown = ks[1 + i // bs].clone()


@pytest.mark.parametrize("cache", CACHES)
def test_append_special_values(cache):
    """Infinities, NaN, zeros, subnormals and the largest numbers; scales that the caller made are no powers of two."""
    bs, heads, dim = 16, 2, 64
    for dtype in (torch.float16, torch.bfloat16):
        k, ks = filled_cache(1, 5, bs, heads, dim, cache)
        v, vs = filled_cache(2, 5, bs, heads, dim, cache)
        ks.mul_(1.37)
        x = inputs(7, 4 * bs, heads, dim, dtype)
        x[3, 0, 5], x[4, 1, 0], x[5, 1, 63] = float("inf"), float("-inf"), float("nan")
        x[16:32] = 0
        x[33:36] = torch.finfo(dtype).max
        x[48:] = torch.finfo(dtype).smallest_normal / 8
        slots = runs_to_slots([(0, 3, 13), (1, 0, 16), (2, 7, 9), (3, 0, 16)], bs)
        check_append(x[:54], x[:54].flip(0).contiguous(), k, v, ks, vs, slots)


def test_append_a_run_that_is_all_non_finite():
    k, ks = filled_cache(1, 2, 16, 1, 64, E4M3)
    v, vs = filled_cache(2, 2, 16, 1, 64, E4M3)
    x = torch.full((3, 1, 64), float("inf"), dtype=torch.bfloat16, device="cuda")
    x[1] = float("nan")
    check_append(x, -x, k, v, ks, vs, torch.tensor([16, 17, 18], device="cuda"))
    assert (ks[1] == 2.0 ** -126).all()


@pytest.mark.parametrize("cache", CACHES)
def test_append_strided(cache):
    """Keys and values as slices of a fused projection; caches with padded rows, interleaved K and V and head-major pages."""
    bs, heads, dim, blocks, n = 16, 4, 64, 6, 40
    qkv = inputs(3, n, 3 * heads, dim, torch.float16)
    odd = inputs(4, n, heads, dim + 1, torch.float16)[..., 1:]        # rows on odd addresses: copied
    slots = torch.stack((runs_to_slots([(4, 5, 11), (None, 0, 1), (2, 0, 16), (0, 0, 12)], bs),) * 2, 1)[:, 0]
    a, s = filled_cache(1, blocks, bs, heads, 2 * dim, cache)
    scales = torch.stack((s, s * 2), 2)
    check_append(qkv[:, heads:2 * heads], qkv[:, 2 * heads:], a[..., :dim], a[..., dim:], scales[..., 0], scales[..., 1],
                 slots)
    b, s = filled_cache(2, blocks, heads, bs, dim, cache)
    b = b.transpose(1, 2)
    c = filled_cache(3, 2 * blocks, bs, heads, dim, cache)[0]
    check_append(odd, qkv[:, :heads], b, c[::2], scales[..., 1], torch.ones(heads, blocks, device="cuda").T, slots)


def test_append_skips_slots_outside_and_leaves_other_pages():
    bs, heads, dim, blocks = 16, 2, 64, 5
    k, ks = filled_cache(1, blocks, bs, heads, dim, E4M3)
    v, vs = filled_cache(2, blocks, bs, heads, dim, E4M3)
    slots = torch.tensor([-1, 80, 2 ** 40, -2 ** 40, 33, 34, 79], dtype=torch.int64, device="cuda")
    x = inputs(3, 7, heads, dim, torch.bfloat16)
    check_append(x, x + 1, k, v, ks, vs, slots)
    kept = [t.clone() for t in (k, v, ks, vs)]
    fa_b200.paged_kv_append(x, x, k, v, ks, vs, torch.full((7,), -1, dtype=torch.int64, device="cuda"))
    fa_b200.paged_kv_append(x[:0], x[:0], k, v, ks, vs, slots[:0])
    for t, u in zip((k, v, ks, vs), kept):
        assert bytes_equal(t, u)


@pytest.mark.parametrize("slots", [[5, 5], [6, 5], [3, 7], list(range(8, 16)) + [15] * 40])
def test_append_reports_slots_out_of_order(slots):
    k, ks = filled_cache(1, 3, 16, 2, 64, E4M3)
    v, vs = filled_cache(2, 3, 16, 2, 64, E4M3)
    x = inputs(3, len(slots), 2, 64, torch.float16)
    other = [t[1:].clone() for t in (k, v, ks, vs)]
    fa_b200.paged_kv_append(x, x, k, v, ks, vs, torch.tensor(slots, device="cuda"))
    with pytest.raises(RuntimeError, match="repeat or do not rise"):
        fa_b200.check_status()
    fa_b200.check_status()                      # reported once
    for t, u in zip((k, v, ks, vs), other):
        assert bytes_equal(t[1:].contiguous(), u)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, dim, bs, runs", [
    # few tokens of many heads: one warp for runs of up to four times what it holds
    (8, 128, 64, [(3, 0, 64), (0, 5, 59), (6, 0, 64), (None, 0, 2), (2, 60, 4), (1, 0, 7)]),
    (16, 256, 32, [(3, 0, 32), (0, 9, 23), (4, 0, 25), (1, 31, 1), (2, 0, 32)]),
    # several warps a run
    (2, 128, 256, [(1, 3, 253), (0, 0, 200), (None, 0, 1), (3, 255, 1), (2, 0, 16), (4, 100, 17)]),
    (1, 16, 1024, [(0, 0, 600), (1, 1000, 24), (2, 0, 1024), (4, 7, 3)])])
def test_append_runs_longer_than_the_registers_and_special_values(cache, dtype, heads, dim, bs, runs):
    """Infinities, NaN, zeros, the smallest and the largest numbers in runs that a warp reads twice and in runs that several
    warps share, over pages whose scales are no powers of two."""
    slots = runs_to_slots(runs, bs)
    n = slots.numel()
    for special in (False, True):
        k, ks = filled_cache(1, 7, bs, heads, dim, cache)
        v, vs = filled_cache(2, 7, bs, heads, dim, cache)
        x, y = inputs(3, n, heads, dim, dtype), inputs(4, n, heads, dim, dtype)
        if special:
            ks.mul_(1.37)
            vs[::2].mul_(2.0 ** 9)
            x[n // 3, 0, 5], x[n // 2, -1, 0], x[n - 1, 0, dim - 1] = float("inf"), float("-inf"), float("nan")
            x[runs[0][2] - 1, -1, 3] = float("nan")
            y[:runs[0][2]] = 0
            y[n // 2:] *= 2.0 ** -10
            y[-3:-1] = torch.finfo(dtype).max
        check_append(x, y, k, v, ks, vs, slots)


@pytest.mark.parametrize("dim, bs", [(64, 16), (128, 256)])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_rounds_once_under_any_scale(cache, dtype, dim, bs):
    """Quotients and products within 2^-25 of a tie between two codes, on either side: rounded to fp32 first they would be
    ties. Scales 1.37 * 2^i, 2^i (1 + 2^-22), 2^i (2 - 2^-22); every code as an older one, and new values next to every tie."""
    half = bs // 2
    for n, scale in enumerate(m * 2.0 ** i for i in (-70, -2, 0, 9) for m in (1.37, 1 + 2.0 ** -22, 2 - 2.0 ** -22)):
        if cache == torch.int8:
            codes = torch.arange(bs * dim) % 255 - 127
            mids = torch.arange(half * dim) % 254 - 126.5
        else:
            codes = torch.arange(bs * dim) % 254
            codes = torch.where(codes < 127, codes, codes + 1).to(torch.uint8).view(E4M3)
            finite = torch.arange(127, dtype=torch.uint8).view(E4M3).float()
            mids = torch.cat(((finite[1:] + finite[:-1]) / 2, -(finite[1:] + finite[:-1]) / 2))
            mids = mids[torch.arange(half * dim) % len(mids)]
        k = codes.to(torch.int8).view(1, bs, 1, dim).cuda() if cache == torch.int8 else codes.view(1, bs, 1, dim).cuda()
        ks = torch.full((1, 1), scale, dtype=torch.float32, device="cuda")
        x = (mids.double() * ks.item()).view(half, 1, dim).to(dtype).cuda()       # stays under the page's scale
        slots = torch.arange(half, bs, device="cuda")
        if torch.isfinite(x).all() and x.abs().max() > 0:
            check_append(x, -x, k.clone(), k.clone(), ks.clone(), ks.clone(), slots)
        # and one value that makes the scale grow by 2, 4, 8; where the old one was negative, the new one may be smaller
        for grow in (1.2, 3.0, 7.0, -0.01, -0.6, -3.0):
            if grow < 0 and n % 3:
                continue
            x = torch.zeros(1, 1, dim, dtype=dtype, device="cuda")
            x[0, 0, 0] = grow * oracle.LARGEST[cache] * ks.item()
            if x[0, 0, 0].isfinite():
                old = ks if grow > 0 else -ks
                check_append(x, -x, k.clone(), k.clone(), old.clone(), old.clone(), slots[:1])


@pytest.mark.parametrize("slots", [[5, 5], [6, 5], [3, 7], list(range(8, 16)) + [15] * 40, [9] * 400])
@pytest.mark.parametrize("dim, bs", [(128, 256), (64, 1024)])
def test_append_reports_slots_out_of_order_in_large_pages(slots, dim, bs):
    k, ks = filled_cache(1, 3, bs, 2, dim, E4M3)
    v, vs = filled_cache(2, 3, bs, 2, dim, E4M3)
    x = inputs(3, len(slots), 2, dim, torch.float16)
    other = [t[1:].clone() for t in (k, v, ks, vs)]
    fa_b200.paged_kv_append(x, x, k, v, ks, vs, torch.tensor(slots, device="cuda"))
    with pytest.raises(RuntimeError, match="repeat or do not rise"):
        fa_b200.check_status()
    fa_b200.check_status()
    for t, u in zip((k, v, ks, vs), other):
        assert bytes_equal(t[1:].contiguous(), u)


@pytest.mark.parametrize("slots", [[5, -1, 6, 17, 33], [5, 20, 6], [20, 5, 33, 4], list(range(16)) + [-1] * 300 + [3, 17]])
@pytest.mark.parametrize("bs, dim", [(16, 64), (16, 256), (256, 128)])
def test_append_leaves_other_pages_alone_when_tokens_of_one_lie_apart(slots, bs, dim):
    """Nothing is promised for page 0, and nothing else is touched."""
    slots = [s if s < 16 else s // 16 * bs + s % 16 for s in slots]
    x = inputs(3, len(slots), 2, dim, torch.float16)
    k, ks = filled_cache(1, 4, bs, 2, dim, E4M3)
    v, vs = filled_cache(2, 4, bs, 2, dim, torch.int8)[0].view(E4M3), ks * 2
    # the tokens of the other pages, by themselves
    others = [i for i, s in enumerate(slots) if s >= bs]
    want = [oracle.append_ref(y[others], c, s, [slots[i] for i in others]) for y, c, s in ((x, k, ks), (-x, v, vs))]
    fa_b200.paged_kv_append(x, -x, k, v, ks, vs, torch.tensor(slots, device="cuda"))
    for c, s, (codes, scales) in ((k, ks, want[0]), (v, vs, want[1])):
        assert torch.equal(s[1:].double(), scales[1:])
        assert torch.equal(torch.nan_to_num(c[1:].double(), nan=1e9), torch.nan_to_num(codes[1:], nan=1e9))


# ---------------------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------------------
def decode_case(seed, lens, heads_q, heads_kv, dim, bs, dtype, cache, spare=2):
    g = gen(seed)
    batch, width = len(lens), max(1, max(-(-n // bs) for n in lens))
    blocks = sum(-(-n // bs) for n in lens) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    table = torch.full((batch, width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(-(-n // bs)):
            table[b, j] = ids.pop()
    k, ks = filled_cache(seed + 1, blocks, bs, heads_kv, dim, cache)
    v, vs = filled_cache(seed + 2, blocks, bs, heads_kv, dim, cache)
    ks.mul_(0.02)
    q = torch.randn(batch, heads_q, dim, generator=g).to(dtype).cuda()
    return [q, k, v, ks, vs, table.cuda(), ints(lens)]


def check_decode(args, **kw):
    got = fa_b200.flash_attention_decode_paged_8bit(*args, **kw)
    want, bound = oracle.decode8_ref(*args, **kw)
    assert got.dtype == args[0].dtype and got.shape == args[0].shape
    half_step = torch.finfo(got.dtype).eps / 2
    # the result's own rounding (below the normal range: half of the smallest step), on top of what the kernel may be off
    allowed = bound * (1 + half_step) + want.abs() * half_step + torch.finfo(got.dtype).smallest_normal * half_step
    excess = (got.double() - want).abs() - allowed
    assert torch.isfinite(got).all()
    assert (excess <= 0).all(), f"off by {(excess + allowed).max():.3e}, {(excess).max():.3e} more than allowed"
    return got


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens, heads_q, heads_kv, dim, bs", [
    ([1], 1, 1, 64, 16), ([256], 8, 8, 128, 16), ([1000, 3], 32, 8, 128, 16), ([77, 0, 300], 4, 2, 64, 8),
    ([129, 128, 127], 16, 1, 128, 32), ([513], 10, 2, 256, 64), ([40, 900], 24, 8, 16, 16), ([65, 31], 15, 3, 32, 4),
    ([700, 1, 64], 32, 2, 64, 1), ([333], 12, 12, 128, 128), ([50, 2000], 20, 4, 128, 256), ([257], 33, 1, 256, 16),
    ([5, 6, 7, 8], 64, 4, 128, 2), ([1500], 40, 1, 128, 16), ([90, 91], 48, 16, 64, 16), ([333, 70], 6, 3, 64, 32),
    ([500, 129], 12, 2, 64, 2), ([260, 7], 8, 4, 64, 4), ([300, 5], 4, 2, 128, 64), ([300, 1], 3, 1, 256, 256),
    ([200, 130], 4, 1, 32, 128), ([77], 2, 2, 16, 1)])
def test_decode(cache, dtype, lens, heads_q, heads_kv, dim, bs):
    check_decode(decode_case(len(lens) * 7 + dim, lens, heads_q, heads_kv, dim, bs, dtype, cache))


@pytest.mark.parametrize("lens", [[1], [16384], [20000, 17], [3218, 15003, 6237, 12772], list(range(0, 2400, 17)),
                                  [31] * 300, [0] * 5, [4000] + [1] * 200])
def test_decode_lengths(lens):
    """Few long contexts, many short ones, and mixtures: every way in which the work is split and joined."""
    check_decode(decode_case(3, lens, 16, 4, 64, 16, torch.float16, E4M3))
    check_decode(decode_case(4, lens, 8, 1, 128, 16, torch.bfloat16, torch.int8))


def test_decode_batch_of_thousands():
    g = gen(1)
    lens = torch.randint(0, 40, (1700,), generator=g).tolist()
    check_decode(decode_case(5, lens, 4, 2, 64, 16, torch.float16, E4M3))


@pytest.mark.parametrize("cache", CACHES)
def test_decode_never_reads_behind_the_context_or_bad_pages(cache):
    """NaN behind every context, in pages that no request holds and in their scales; ids out of range; lengths that
    exceed the table or are negative."""
    args = decode_case(6, [37, 160, 5, 48], 8, 2, 128, 16, torch.float16, cache)
    q, k, v, ks, vs, table, lens = args
    used = {int(p) for p in table.flatten().tolist() if p >= 0}
    for t in (k, v):
        raw = t.view(torch.uint8)
        for p in range(t.shape[0]):
            if p not in used:
                raw[p] = 0x7f
        for b, n in enumerate(lens.tolist()):
            if n % 16:
                raw[int(table[b, n // 16]), n % 16:] = 0x7f
    for s in (ks, vs):
        for p in range(k.shape[0]):
            if p not in used:
                s[p] = float("nan")
    check_decode(args)
    table[0, 1], table[1, 0], table[2, 0] = -1, k.shape[0], 10 ** 9
    check_decode(args)
    lens[1], lens[3] = 10 ** 9, -4
    got = check_decode(args)
    assert (got[2] == 0).all() and (got[3] == 0).all()


def test_decode_scales_of_every_size():
    """Value scales from 2^-126 to 2^100 between pages, zero scales, and scores that grow along the context."""
    args = decode_case(7, [400, 250], 8, 2, 64, 16, torch.bfloat16, E4M3)
    g = gen(2)
    args[4].copy_(torch.exp2(torch.randint(-126, 101, args[4].shape, generator=g).float()))
    check_decode(args)
    args[4].zero_()
    assert (fa_b200.flash_attention_decode_paged_8bit(*args) == 0).all()
    args = decode_case(8, [600], 4, 1, 128, 16, torch.float16, torch.int8)
    ramp = torch.linspace(0.1, 60, 38, device="cuda")
    for j, p in enumerate(args[5][0].tolist()):
        args[3][p] = ramp[j] * 0.01
    check_decode(args)


@pytest.mark.parametrize("heads_q, heads_kv, dim", [(8, 2, 64), (32, 2, 64), (16, 8, 128), (12, 1, 128), (5, 1, 256)])
@pytest.mark.parametrize("first", [True, False])
def test_decode_large_value_scales_under_small_probabilities(heads_q, heads_kv, dim, first):
    """Values many powers of two larger than the others, in pages that the softmax leaves next to nothing of: the answer
    is that of the others. The large ones come in front of them or behind, and one row in two has them on top instead."""
    args = decode_case(12, [300, 5000, 64], heads_q, heads_kv, dim, 16, torch.bfloat16, E4M3)
    q, k, v, ks, vs, table, lens = args
    ks.fill_(2.0 ** -6)
    k.copy_((torch.randn(k.shape, generator=gen(4)) * 0.1).to(E4M3))
    q.copy_(torch.randn(q.shape, generator=gen(5)) * 0.1)
    q[:, :, 0] = 64.0
    q[:, 1::2, 0] = -64.0
    k[..., 0] = 448.0                           # the score's largest part: 448 q0 ks for pages of the one kind
    for b, n in enumerate(lens.tolist()):
        pages = table[b, :(n + 15) // 16].tolist()
        for j, page in enumerate(pages):
            if (j < len(pages) // 2) == first:
                k[page, :, :, 0] = -448.0
                vs[page] *= 2.0 ** (20 + 9 * (j % 7))
    scale = 40 / (448 * 64 * 2.0 ** -6)         # scores of +-40: probabilities e^-80, 2^-115, of the other kind
    check_decode(args, softmax_scale=scale)
    check_decode(args, softmax_scale=scale / 5)
    check_decode(args, softmax_scale=0.0)


@pytest.mark.parametrize("heads_q, heads_kv, dim", [(8, 2, 64), (32, 2, 64), (16, 8, 128), (5, 1, 256), (12, 3, 32)])
@pytest.mark.parametrize("lens", [[40, 3], [700, 9000], [30000], [300] * 50])
@pytest.mark.parametrize("cache", CACHES)
def test_decode_values_near_the_largest_numbers(heads_q, heads_kv, dim, lens, cache):
    """Values up to 2^117 under scores that rise above what the softmax started from: every sum that is kept in between
    stays in fp32's range."""
    args = decode_case(32, lens, heads_q, heads_kv, dim, 16, torch.bfloat16, cache)
    args[1].copy_((args[1].float() / 4).to(cache))
    args[4].copy_(torch.exp2(torch.randint(85, 111 if cache == torch.int8 else 109, args[4].shape, generator=gen(6)).float()))
    for b in range(len(lens)):                  # keys that grow along the context
        pages = args[5][b][args[5][b] >= 0].long()
        args[3][pages] *= torch.linspace(0.1, 4, len(pages), device="cuda")[:, None]
    largest = (args[2].double().abs().amax((1, 3)) * args[4].double()).max()
    assert 2.0 ** 105 < largest <= 2.0 ** 117   # (short contexts meet few of the large scales)
    check_decode(args)


def scored_case(seed, scores, heads_q, heads_kv, dim, dtype, cache):
    """One request whose token t scores scores[t] in the base-2 exponent (whole numbers from -64 to 63), in every head."""
    args = decode_case(seed, [len(scores)], heads_q, heads_kv, dim, 16, dtype, cache)
    q, k, v, ks, vs, table, lens = args
    q.zero_()
    q[:, :, :3] = 1.0
    k.view(torch.uint8).zero_()                 # (zero in both types)
    high, low = scores // 8 * 4, scores % 8     # high + high + low, each an e4m3 and an int8 value
    for t, page in enumerate(table[0].tolist()):
        at = slice(16 * t, 16 * t + 16)
        n = len(scores[at])
        for d, part in ((0, high), (1, high), (2, low)):
            k[page, :n, :, d] = part[at, None].expand(n, heads_kv).to(k.device).float().to(cache)
    ks.fill_(1.0)
    vs.fill_(1.0)
    return args, 0.6931471805599453             # softmax scale ln 2: q . k counts powers of two


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads_q, heads_kv, dim", [(8, 2, 64), (32, 2, 64), (32, 8, 128), (16, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("outlier", [1.0, 64.0, 2.0 ** 40])
@pytest.mark.parametrize("first", [0, 16000])
def test_decode_many_small_probabilities_beside_a_large_one(cache, heads_q, heads_kv, dim, outlier, first):
    """A token with next to all of the probability and zeros for values, 16383 others of 2^-20 each that make up the
    answer, and beside the first a page of larger scale and no probability to speak of (2^-60)."""
    scores = torch.full((16384,), 0)
    scores[first], scores[16:32] = 20, -40
    args, scale = scored_case(30, scores, heads_q, heads_kv, dim, torch.float16, cache)
    v, vs, table = args[2], args[4], args[5][0].tolist()
    v.copy_(v.float().abs().to(cache))
    v.view(torch.uint8)[table[first // 16], first % 16] = 0
    vs[table[1]] = outlier
    got = check_decode(args, softmax_scale=scale)
    assert (got > 0.1).all()


@pytest.mark.parametrize("heads_q, heads_kv, dim", [(8, 2, 64), (32, 2, 64), (32, 8, 128), (16, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("rise", [3, 5, 9, 11])
def test_decode_scores_that_rise_from_page_to_page(heads_q, heads_kv, dim, rise):
    """Scores that climb and fall by `rise` from page to page, below and above what moves the softmax reference, under
    scales that move the other way or the same way: the weights leave the range of what they are rounded to on both sides."""
    page = torch.arange(30 * 11) % 30
    climb = (torch.where(page < 15, page, 29 - page) * rise).clamp(max=120)
    for sign in (-1, 0, 1):
        args, scale = scored_case(31, (climb - 60).repeat_interleave(16), heads_q, heads_kv, dim, torch.bfloat16, E4M3)
        for j, p in enumerate(args[5][0].tolist()):
            args[4][p] = 2.0 ** (sign * int(climb[j]) / 2)
        check_decode(args, softmax_scale=scale)


@pytest.mark.parametrize("cache, power", [(E4M3, 108), (torch.int8, 110)])
@pytest.mark.parametrize("heads_q, heads_kv, dim, tokens", [(32, 8, 128, 16384), (8, 8, 256, 9000), (32, 2, 64, 100000)])
def test_decode_large_values_under_scores_above_the_reference(cache, power, heads_q, heads_kv, dim, tokens):
    """Tiles whose scores pass the ones before them by 2^9, just under what moves the softmax reference, over values of one
    sign up to 2^117: what a part of the context hands in is 2^9 times some hundred such values."""
    scores = 9 * (torch.arange(tokens) // 256 % 3 > 0)
    args, scale = scored_case(33, scores, heads_q, heads_kv, dim, torch.bfloat16, cache)
    args[2].copy_(args[2].float().abs().to(cache))
    args[4].fill_(2.0 ** power)
    assert check_decode(args, softmax_scale=scale).min() > 2.0 ** (power + 3)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-6])
def test_decode_softmax_scales(scale):
    check_decode(decode_case(9, [200, 31], 8, 2, 128, 16, torch.bfloat16, E4M3), softmax_scale=scale)


def test_decode_queries_of_every_size():
    for factor in (1e-30, 1e-4, 1e20):
        args = decode_case(10, [200, 31], 8, 2, 128, 16, torch.bfloat16, E4M3)
        args[0] *= factor
        args[3] /= factor
        check_decode(args)


def test_decode_nan_stays_in_its_row():
    args = decode_case(11, [100, 100], 8, 2, 64, 16, torch.float16, E4M3)
    clean = fa_b200.flash_attention_decode_paged_8bit(*args)
    args[0][0, 3, 7] = float("nan")
    got = fa_b200.flash_attention_decode_paged_8bit(*args)
    assert torch.isnan(got[0, 3]).all()
    rest = torch.ones(2, 8, dtype=torch.bool)
    rest[0, 3] = False
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache", CACHES)
def test_decode_strided(cache, dim):
    """Every layout against the oracle; at 128 dimensions all of them take the same way, bit for bit (at 64 neighbouring
    heads are read in pairs, heads that are not neighbours one by one, and the sums are split differently)."""
    args = decode_case(12, [100, 333], 8, 4, dim, 16, torch.float16, cache)
    q, k, v, ks, vs, table, lens = args
    both = torch.cat((k.view(torch.uint8), v.view(torch.uint8)), -1).view(cache)          # K and V side by side
    major = v.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(cache)   # head-major pages
    qkv = torch.cat((q, q, q), 1)
    want = check_decode(args)
    scales = torch.stack((ks, vs), 2)
    for kk, vv in ((both[..., :dim], both[..., dim:]), (k, major), (both[..., :dim], major)):
        got = check_decode([qkv[:, 8:16], kk, vv, scales[..., 0], scales[..., 1], table.T.contiguous().T,
                            torch.stack((lens, lens), 1)[:, 1]])
        assert dim == 64 or torch.equal(got, want)
    odd = torch.zeros(2, 8, dim + 1, dtype=q.dtype, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(fa_b200.flash_attention_decode_paged_8bit(odd, *args[1:]), want)


def test_contiguous_rows_off_a_16_byte_boundary():
    """Queries, keys and values that are contiguous but begin 2 or 8 bytes into memory are copied, not refused."""
    args = decode_case(12, [100, 333], 8, 4, 64, 16, torch.bfloat16, E4M3)
    want = check_decode(args)
    x = inputs(3, 5, 4, 64, torch.bfloat16)
    slots = torch.arange(16, 21, device="cuda")
    caches = [[t.clone() for t in args[1:5]] for _ in range(2)]
    fa_b200.paged_kv_append(x, -x, *caches[0], slots)
    for skip in (1, 4):
        def shifted(t):
            out = torch.empty(t.numel() + skip, dtype=t.dtype, device="cuda")[skip:].view(t.shape)
            assert out.is_contiguous() and out.data_ptr() % 16
            return out.copy_(t)

        assert torch.equal(fa_b200.flash_attention_decode_paged_8bit(shifted(args[0]), *args[1:]), want)
        fa_b200.paged_kv_append(shifted(x), shifted(-x), *caches[1], slots)
        assert all(bytes_equal(a, b) for a, b in zip(*caches))
    with pytest.raises(RuntimeError, match="16-byte"):      # caches are never copied
        k = torch.empty(args[1].numel() + 8, dtype=torch.uint8, device="cuda")[8:].view(E4M3).view(args[1].shape)
        fa_b200.flash_attention_decode_paged_8bit(args[0], k, *args[2:])


def test_decode_one_page_for_many_requests():
    """A prefix that requests share: the same page in several rows, and twice in one."""
    args = decode_case(13, [64, 64, 64], 8, 2, 128, 16, torch.float16, E4M3)
    args[5][1, :3] = args[5][0, :3]
    args[5][2, 1] = args[5][2, 0]
    check_decode(args)


def test_decode_results_do_not_change_between_calls():
    args = decode_case(14, [5000, 3, 700], 32, 8, 128, 16, torch.bfloat16, E4M3)
    first = fa_b200.flash_attention_decode_paged_8bit(*args)
    for _ in range(5):
        assert torch.equal(fa_b200.flash_attention_decode_paged_8bit(*args), first)


def test_decode_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes, whose last pages hold the context."""
    bs, heads, dim = 16, 8, 128
    blocks = 2 ** 32 // (bs * heads * dim) + 40
    small = decode_case(15, [300], 16, heads, dim, bs, torch.float16, torch.int8)
    pages = small[1].shape[0]
    k, v = (torch.zeros(blocks, bs, heads, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(blocks, heads, device="cuda") for _ in range(2))
    for big, little in zip((k, v, ks, vs), small[1:5]):
        big[-pages:] = little
    far = torch.where(small[5] >= 0, small[5] + (blocks - pages), small[5])
    got = fa_b200.flash_attention_decode_paged_8bit(small[0], k, v, ks, vs, far, small[6])
    assert torch.equal(got, fa_b200.flash_attention_decode_paged_8bit(*small))
    x = inputs(1, 5, heads, dim, torch.float16)
    slots = torch.arange((blocks - 1) * bs + 3, (blocks - 1) * bs + 8, device="cuda")
    tail = [t[-1:].clone() for t in (k, v, ks, vs)]
    fa_b200.paged_kv_append(x, -x, k, v, ks, vs, slots)
    fa_b200.paged_kv_append(x, -x, *tail, slots - (blocks - 1) * bs)
    for big, little in zip((k, v, ks, vs), tail):
        assert bytes_equal(big[-1:].contiguous(), little)


@pytest.mark.parametrize("heads_kv, dim, last", [(1, 16, 16), (1, 16, 1), (2, 64, 9)])
def test_decode_contexts_up_to_the_last_32_bit_length(heads_kv, dim, last):
    """2^27 - 1 rows of the table that all name one page, and a request of ordinary length behind: the answer is that of
    the one page (the last row holds `last` tokens, which at 2^-27 of the sum do not show). The longest running sums are
    2^31 / 148 / 256 units long with up to four additions a unit, each off by 2^-24 in the sum of the probabilities and by
    2^-23 in that of the products: together 4.1 % of sum p |v| at most. The values are positive, so that shows zeros and
    whatever lay in the output's memory before."""
    drift = 4 * 1.5 * 2.0 ** -23 * 2.0 ** 31 / 148 / 256
    args = decode_case(40, [16, 77], 4 * heads_kv, heads_kv, dim, 16, torch.bfloat16, torch.int8)
    q, k, v, ks, vs, table, lens = args
    v.copy_(v.float().abs().clamp(min=1).to(torch.int8))
    want, _ = oracle.decode8_ref(*args)
    width = 2 ** 27 - 1
    far = table[:1, :1].expand(1, width)
    lens[0] = (width - 1) * 16 + last
    got = fa_b200.flash_attention_decode_paged_8bit(q[:1], k, v, ks, vs, far, lens[:1])
    assert ((got.double() - want[:1]).abs() <= (drift + 2.0 ** -7) * want[:1]).all()
    # in a batch: a request of ordinary length in front and one behind (all rows of the table name their first page)
    ends, page = torch.tensor([1, 0, 1], device="cuda"), torch.stack((table[1, 0], table[0, 0], table[1, 0]))
    want = oracle.decode8_ref(q[ends], k, v, ks, vs, page[:, None], ints([13, 16, 16]))[0]
    got = fa_b200.flash_attention_decode_paged_8bit(q[ends], k, v, ks, vs, page[:, None].expand(3, width),
                                                    torch.stack((lens[0] * 0 + 13, lens[0], lens[0] * 0 + 1600)))
    assert ((got.double() - want).abs() <= (drift + 2.0 ** -7) * want).all()


# ---------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------
def packed(seed, new, pad, heads, dim, dtype):
    return inputs(seed, sum(max(n, 0) for n in new) + pad, heads, dim, dtype)


STEPS = [[40, 0, 7, 0], [1, 33, 1, 0], [1, 1, 1, 2], [-1, 1, 1, 1], [50, 1, -1, 1], [1, 1, 90, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("cache", CACHES)
def test_a_server_s_steps(cache):
    """Prompts, steps, ends and new requests in the same rows, two layers: every step against the oracle's own state."""
    heads, group, dim, bs, blocks = 2, 4, 64, 16, 24
    c = fa_b200.PagedKVCache8(2, blocks, bs, heads, dim, 4, 8, dtype=cache)
    for i, new in enumerate(STEPS):
        pad = i % 3
        state = oracle.plan_ref(c.context_lens.tolist(), new, c.block_table.cpu(), c.free_blocks.cpu(),
                                int(c.free_count), sum(max(n, 0) for n in new) + pad, bs)
        slots, cu = c.plan(ints(new), len(state[0]))
        assert slots.tolist() == state[0] and cu.tolist() == state[1]
        assert c.context_lens.tolist() == state[2] and int(c.free_count) == state[3]
        for layer in range(2):
            key, value = (packed(10 * i + j + 2 * layer, new, pad, heads, dim, torch.bfloat16) for j in range(2))
            want = [oracle.append_ref(x, y[layer], s[layer], slots.tolist())
                    for x, y, s in ((key, c.k_cache, c.k_scales), (value, c.v_cache, c.v_scales))]
            c.append(layer, key, value, slots)
            assert torch.equal(c.k_cache[layer].double(), want[0][0]) and torch.equal(c.v_scales[layer].double(), want[1][1])
            q = inputs(100 + i, 4, heads * group, dim, torch.bfloat16)
            got = c.decode(layer, q)
            ref, bound = oracle.decode8_ref(q, c.k_cache[layer], c.v_cache[layer], c.k_scales[layer], c.v_scales[layer],
                                            c.block_table, c.context_lens)
            assert ((got.double() - ref).abs() <= bound * 1.004 + ref.abs() * 2.0 ** -8 + 1e-30).all()


def test_the_8_bit_cache_stays_near_the_exact_one():
    """What rounding costs: attention over the cache against attention over the 16-bit keys and values. An e4m3 code is
    off by 2^-4 of its value at most, so values alone move a row by at most 2^-4 of sum p |v|, and a score by at most
    2^-4 of sum |q k|; with q of size 0.05 that is under 0.3 here and the whole under 2^-4 + (e^0.6 - 1)."""
    heads, dim, n = 2, 64, 500
    c = fa_b200.PagedKVCache8(1, 40, 16, heads, dim, 1, 40)
    slots, _ = c.plan(ints([n]), n)
    key, value = inputs(1, n, heads, dim, torch.float16).clamp(-3, 3), inputs(2, n, heads, dim, torch.float16).clamp(-3, 3)
    c.append(0, key, value, slots)
    q = (torch.randn(1, 8, dim, generator=gen(3)) * 0.05).half().cuda()
    got = c.decode(0, q, softmax_scale=1.0).double()
    k, v = (x.double().repeat_interleave(4, 1) for x in (key, value))
    sums = torch.einsum("hd,nhd->hn", q[0].double().abs(), k.abs()).max()
    assert sums / 16 < 0.6
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0].double(), k), -1)
    want, weight = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
    assert ((got[0] - want).abs() <= (2.0 ** -4 + 2 * (torch.exp(sums / 16) - 1)) * weight).all()


def test_steps_captured_in_a_graph():
    """A decode step as a CUDA graph: replays continue from the state that the step before left."""
    heads, dim, bs = 2, 64, 16
    live, ref = (fa_b200.PagedKVCache8(1, 30, bs, heads, dim, 3, 10) for _ in range(2))
    start = ints([20, 3, 0])
    x = inputs(1, 23, heads, dim, torch.float16)
    for c in (live, ref):
        slots, _ = c.plan(start, 23)
        c.append(0, x, -x, slots)
    new, key, q = ints([1, 1, 1]), inputs(2, 3, heads, dim, torch.float16), inputs(3, 3, 8, dim, torch.float16)

    def step(c, key, q):
        slots, _ = c.plan(new, 3)
        c.append(0, key, key, slots)
        return c.decode(0, q)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fa_b200.PagedKVCache8(1, 30, bs, heads, dim, 3, 10), key, q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(live, key, q)
    for i in range(20):
        key.copy_(inputs(50 + i, 3, heads, dim, torch.float16) * (1 + i))
        graph.replay()
        want = step(ref, key, q)
        assert torch.equal(out, want), i
    assert torch.equal(live.block_table, ref.block_table) and live.context_lens.tolist() == [40, 23, 20]
    assert bytes_equal(live.k_cache, ref.k_cache) and torch.equal(live.k_scales, ref.k_scales)


FIRST_CALLS_CAPTURED = """
import sys
sys.path[:0] = {path!r}
import torch, fa_b200
g = torch.Generator().manual_seed(1)
key, value, q = (torch.randn(2, n, 64, generator=g).half().cuda() for n in (2, 2, 8))
x = [fa_b200.PagedKVCache8(1, 30, 16, 2, 64, 2, 10) for _ in range(2)]
new = torch.ones(2, dtype=torch.int32, device="cuda")
junk = torch.full((1 << 22,), 0x55, dtype=torch.uint8, device="cuda")      # what the allocator hands out next is not zero
del junk

def step(c):
    slots, _ = c.plan(new, 2)
    c.append(0, key, value, slots)
    return c.decode(0, q)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step(x[0])
fa_b200.check_status()                      # nothing has run yet, and nothing is reported
for _ in range(3):
    graph.replay()
    assert torch.equal(out, step(x[1]))
fa_b200.check_status()
# a report of another call is not wiped out by a replay
caches = [t[0] for t in (x[1].k_cache, x[1].v_cache, x[1].k_scales, x[1].v_scales)]
fa_b200.paged_kv_append(key, value, *caches, torch.tensor([5, 5], device="cuda"))
graph.replay()
try:
    fa_b200.check_status()
except RuntimeError as e:
    assert "repeat" in str(e), e
    print("reported")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", FIRST_CALLS_CAPTURED.format(path=[p for p in sys.path if p])],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout[-500:] + r.stderr[-1500:]


def test_two_streams_at_once():
    a = decode_case(16, [9000, 50], 32, 8, 128, 16, torch.float16, E4M3)
    b = decode_case(17, [400] * 40, 32, 8, 128, 16, torch.float16, E4M3)
    want = [fa_b200.flash_attention_decode_paged_8bit(*x) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fa_b200.flash_attention_decode_paged_8bit(*(a, b)[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_ops_under_fake_tensors_and_opcheck():
    d = decode_case(18, [40, 70], 8, 2, 64, 16, torch.float16, E4M3)
    torch.library.opcheck(paged_cache._decode8_op, (*d, 0.125), test_utils="test_faketensor")
    tests = ("test_schema", "test_faketensor")        # the schema check multiplies, which torch cannot do in e4m3
    d = decode_case(18, [40, 70], 8, 2, 64, 16, torch.float16, torch.int8)
    torch.library.opcheck(paged_cache._decode8_op, (*d, 0.125), test_utils=tests)
    k, ks = filled_cache(1, 4, 16, 2, 64, torch.int8)
    v, vs = filled_cache(2, 4, 16, 2, 64, torch.int8)
    x = inputs(3, 4, 2, 64, torch.float16)
    slots = torch.arange(4, device="cuda")
    torch.library.opcheck(paged_cache._append_op, (x, x.clone(), k, v, ks, vs, slots), test_utils=tests)
    torch.library.opcheck(paged_cache._plan_op, (*random_plan(1, 5, 16, 8, 20, 30), 16), test_utils=tests)


def test_compiled_step_equals_the_eager_one():
    d = decode_case(19, [40, 70], 8, 2, 64, 16, torch.float16, E4M3)
    fn = torch.compile(lambda *t: fa_b200.flash_attention_decode_paged_8bit(*t) * 2, backend="aot_eager", fullgraph=True)
    assert torch.equal(fn(*d), fa_b200.flash_attention_decode_paged_8bit(*d) * 2)


def test_inference_only():
    d = decode_case(20, [40], 8, 2, 64, 16, torch.float16, E4M3)
    d[0].requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference-only"):
        fa_b200.flash_attention_decode_paged_8bit(*d)
    with torch.no_grad():
        fa_b200.flash_attention_decode_paged_8bit(*d)


@pytest.mark.parametrize("index", range(5))
def test_inference_only_for_caches_and_scales(index):
    d = decode_case(20, [40], 8, 2, 64, 16, torch.float16, E4M3)
    x = inputs(3, 4, 2, 64, torch.float16)
    slots = torch.arange(4, device="cuda")
    fa_b200.flash_attention_decode_paged_8bit(*d)        # (the compiled binding takes over behind the first call)
    fa_b200.paged_kv_append(x, x, *d[1:5], slots)
    before = [t.clone() for t in d[1:5]]
    d[index].requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference-only"):
        fa_b200.flash_attention_decode_paged_8bit(*d)
    if index > 0:
        with pytest.raises(RuntimeError, match="inference-only"):
            fa_b200.paged_kv_append(x * 2, x, *d[1:5], slots)
        assert all(bytes_equal(a.detach(), b) for a, b in zip(d[1:5], before))
    with torch.no_grad():
        fa_b200.flash_attention_decode_paged_8bit(*d)
        fa_b200.paged_kv_append(x, x, *d[1:5], slots)


def test_captured_behind_copies_and_joined_streams():
    """The kernels start early behind whatever precedes them: a copy, a fill, a kernel of another stream, in a graph and
    outside, never before it has written what they read."""
    args = decode_case(21, [700, 90, 1], 8, 2, 64, 16, torch.float16, E4M3)
    sources = [[t.clone() for t in decode_case(s, [700, 90, 1], 8, 2, 64, 16, torch.float16, E4M3)] for s in (22, 23)]
    plan = random_plan(31, 40, 16, 20, 60, 90)
    side = torch.cuda.Stream()

    def step(src):
        for t, u in zip(args[:5], src):                       # copies, then fills, right in front
            t.copy_(u)
        out = fa_b200.flash_attention_decode_paged_8bit(*args)
        args[0].zero_()
        zero = fa_b200.flash_attention_decode_paged_8bit(*args)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            args[0].copy_(src[0])
            other = fa_b200.flash_attention_decode_paged_8bit(*args)
            slots = fa_b200.paged_kv_plan(*plan, 16)[0]
        here.wait_stream(side)
        last = fa_b200.flash_attention_decode_paged_8bit(*args)
        x = args[1][0].float().half()
        fa_b200.paged_kv_append(x, -x, args[1], args[2], args[3], args[4], torch.arange(16, 32, device="cuda"))
        after = fa_b200.flash_attention_decode_paged_8bit(*args)
        return out, zero, other, last, after, slots

    want = []
    for src in sources:
        torch.cuda.synchronize()
        want.append([t.clone() for t in step(src)])
        torch.cuda.synchronize()
        full = [*src[:5], args[5], args[6]]
        assert torch.equal(want[-1][0], fa_b200.flash_attention_decode_paged_8bit(*full))
        assert torch.equal(want[-1][2], want[-1][0]) and torch.equal(want[-1][3], want[-1][0])
    live = [t.clone() for t in sources[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(live)
    for _ in range(5):
        for src, ref in zip(sources, want):
            for t, u in zip(live, src):
                t.copy_(u)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


@pytest.mark.parametrize("causal", [False, True])
def test_append_right_behind_a_backward(monkeypatch, causal):
    """The recomputing dQ kernel of 16384 queries over 128 keys ends long before the dK/dV kernel that it was let loose
    beside, which reads the queries to its end: an append that overwrites them comes after both."""
    from fa_b200 import interface

    monkeypatch.setattr(interface, "DS_WORKSPACE_LIMIT_BYTES", 0)
    heads, sq, dim = 4, 16384, 128
    g = gen(1)
    q0, k, v, dout = (torch.randn(1, heads, n, dim, generator=g).half().cuda() for n in (sq, 128, 128, sq))
    x = torch.randn(sq, 8, dim, generator=g).half().cuda()
    slots = torch.arange(sq, device="cuda")
    other = torch.empty(sq // 16, 16, 8, dim, dtype=torch.int8, device="cuda")
    scales = torch.ones(2, sq // 16, 8, device="cuda")
    got = []
    for append in (False, True, True, True):
        q = q0.clone()
        over = q.view(torch.int8).view(sq // 16, 16, 8, dim)     # the queries' memory as a cache of 8-bit pages
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = fa_b200.flash_attention(*leaves, causal=causal)
        grads = torch.autograd.grad(out, leaves, dout)
        if append:
            fa_b200.paged_kv_append(x, x, over, other, *scales, slots)
            torch.cuda.synchronize()
            assert not torch.equal(q, q0)
        got.append(grads)
    for grads in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(grads, got[0]))


@pytest.mark.parametrize("skip", [0, 4])
def test_decode_lost_wait_sets_the_status_word(skip):
    """The loading warp leaves a unit out, so that bounded waits run out on both sides; the kernel ends by itself, what it
    could not read counts as nothing, and the next call is right."""
    from fa_b200 import _lib

    args = decode_case(24, [30000], 32, 8, 128, 16, torch.float16, E4M3)
    check_decode(args)
    fa_b200.check_status()
    _lib.load().fa_test_decode_fault(1 << 12, skip)
    got = fa_b200.flash_attention_decode_paged_8bit(*args)
    with pytest.raises(RuntimeError, match="wait timeout"):
        fa_b200.check_status()
    assert torch.isfinite(got).all()
    check_decode(args)
    fa_b200.check_status()


def test_plan_of_the_largest_batches():
    check_plan(random_plan(41, 8192, 16, 24, 40, 60000), 16)
    args = random_plan(42, 300, 16, 400, 3000, 40000, ends=0.1, pad=5000)
    assert args[5] > 350000
    check_plan(args, 16)
    check_plan(random_plan(43, 300, 16, 400, 3000, 40000, ends=0.1), 16, inplace=True)


def test_plan_of_the_largest_batch_in_place():
    check_plan(random_plan(41, 8192, 16, 24, 40, 60000), 16, inplace=True)
    args = random_plan(44, 8192, 64, 24, 1, 8000, ends=0.1)
    for _ in range(3):                          # steps that go on from one another
        check_plan(args, 64, inplace=True)


@pytest.mark.parametrize("cache", CACHES)
def test_pages_of_a_thousand_tokens(cache):
    """Runs that are longer than what a CTA looks at, and boxes that are a part of a page."""
    bs, heads, dim = 1024, 2, 64
    k, ks = filled_cache(1, 5, bs, heads, dim, cache)
    v, vs = filled_cache(2, 5, bs, heads, dim, cache)
    slots = runs_to_slots([(3, 100, 924), (0, 0, 1024), (None, 0, 1), (4, 0, 333), (2, 1023, 1)], bs)
    n = slots.numel()
    check_append(inputs(3, n, heads, dim, torch.float16), inputs(4, n, heads, dim, torch.bfloat16).half(), k, v, ks, vs, slots)
    check_decode(decode_case(25, [2500, 1024, 1025, 3], 8, 2, 64, 1024, torch.bfloat16, cache))
    check_decode(decode_case(26, [1500, 77], 4, 1, 256, 512, torch.float16, cache))


def test_decode_one_kv_head_under_many_query_heads():
    check_decode(decode_case(27, [600, 90], 128, 1, 128, 16, torch.bfloat16, E4M3))
    check_decode(decode_case(28, [300], 71, 1, 256, 32, torch.float16, torch.int8))


def test_a_compiled_step_of_all_three():
    """plan, append and decode inside one compiled function, with the state that they change in place."""
    heads, dim, bs = 2, 64, 16

    def step(lens, new, table, free, count, key, value, k, v, ks, vs, q):
        slots, cu, lens, count = fa_b200.paged_kv_plan(lens, new, table, free, count, 40, bs)
        fa_b200.paged_kv_append(key, value, k, v, ks, vs, slots)
        return fa_b200.flash_attention_decode_paged_8bit(q, k, v, ks, vs, table, lens), slots, cu, lens, count

    def state():
        k, ks = filled_cache(1, 12, bs, heads, dim, torch.int8)
        v, vs = filled_cache(2, 12, bs, heads, dim, torch.int8)
        x = inputs(3, 40, heads, dim, torch.float16)
        return [ints([0, 0]), ints([30, 7]), torch.full((2, 5), -1, dtype=torch.int32, device="cuda"),
                torch.arange(12, dtype=torch.int32, device="cuda"), ints([12]), x, -x, k, v, ks, vs,
                inputs(4, 2 * 8, 1, dim, torch.float16).view(2, 8, dim)]

    a, b = state(), state()
    want, got = step(*a), torch.compile(step, backend="aot_eager", fullgraph=True)(*b)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
