"""The paged 8-bit cache on the GPU: the plan and the append exactly, the attention against 64
bits, and a run of them together as a server makes it."""

import math

import numpy as np
import pytest
import torch

import plain64
import tk_b200

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def ints(x, kind=torch.int32):
    return torch.tensor(np.asarray(x), dtype=kind, device="cuda")


# ---- plan ---------------------------------------------------------------------------------

def check_plan(cached, new, page, width, n_pages, n_free, max_tokens, seed=0, in_place=False, holes=False, capacity=None):
    g = np.random.default_rng(seed)
    order = g.permutation(n_pages).astype(np.int32)
    table = np.full((len(cached), width), -1, np.int32)
    at = 0
    for r, c in enumerate(cached):
        n = min(-(-max(c, 0) // page), width)
        table[r, :n] = order[at:at + n]
        at += n
    if holes:
        for r in range(0, len(cached), 3):
            table[r] = -5
    free = order[at:].copy()
    want_table = table.copy()
    lens, seq, starts, slots, left = plain64.plan(cached, new, page, want_table, free, n_free, max_tokens)
    d_cached, d_new, d_table, d_free, d_n = ints(cached), ints(new), ints(table).reshape(len(cached), width), ints(free), ints([n_free])
    kw = dict(lens_out=d_cached, n_free_out=d_n) if in_place is True else dict(lens_out=d_cached) if in_place == "lens" else {}
    got = tk_b200.kv_plan(d_cached, d_new, d_table, d_free, d_n, page_size=page, max_tokens=max_tokens, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(d_table.cpu().numpy(), want_table)
    for a, b, name in zip(got, (lens, seq, starts, slots, [left]), ("lens", "seq_lens", "starts", "slots", "n_free")):
        assert a.cpu().tolist() == list(b), name
    assert np.array_equal(d_free.cpu().numpy(), free)
    if not in_place:
        assert d_cached.cpu().tolist() == list(cached) and d_n.item() == n_free


@pytest.mark.parametrize("in_place", [False, True, "lens"])
@pytest.mark.parametrize("requests,page,longest,prompt", [(1, 16, 1, 1), (1, 1, 40, 7), (5, 7, 100, 30), (64, 32, 4096, 1),
                                                          (1024, 16, 300, 5), (1025, 16, 100, 1), (2500, 128, 1000, 40), (37, 64, 9, 1000)])
def test_plan(requests, page, longest, prompt, in_place):
    """One CTA and many, one kernel and two (in place), one group of requests and several."""
    g = np.random.default_rng(requests)
    cached = g.integers(0, longest, requests).tolist()
    new = g.integers(0, prompt + 1, requests).tolist()
    width = -(-(longest + prompt) // page)
    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3
    free = pages - sum(-(-c // page) for c in cached)
    check_plan(cached, new, page, width, pages, free, sum(new) + 11, in_place=in_place)


def test_plan_runs_out():
    """Too few pages, slots or row places, requests that need no page, negative lengths, holes."""
    cached = [0, 15, 16, 3, 0, -4, 64, 60, 31, 0]
    new = [20, 1, 1, 0, 40, 3, 1, 4, -2, 2]
    for n_free in (-3, 0, 1, 2, 3, 5, 6, 7, 50):
        for max_tokens in (0, 1, 21, 30, 72, 200):
            check_plan(cached, new, 16, 4, 60, n_free, max_tokens, seed=n_free + 9)
    check_plan(cached, new, 16, 4, 60, 20, 200, holes=True)
    check_plan(cached, new, 16, 4, 60, 10 ** 6, 200)  # more than the list holds: what it holds
    # many CTAs, and a second group of requests after the pages ran out
    g = np.random.default_rng(3)
    cached, new = g.integers(0, 50, 2300).tolist(), g.integers(0, 60, 2300).tolist()
    for n_free in (0, 700, 3000):
        for in_place in (False, True):
            check_plan(cached, new, 16, 6, 9000, n_free, 40000, in_place=in_place)


def test_plan_of_nothing():
    """No requests: the slots stand for nothing, the free pages stay."""
    n_free, starts, free = ints([5]), ints([9]), ints([1, 2, 3])
    slots = torch.full((7,), 3, dtype=torch.int64, device="cuda")
    room = ints([0] * 8)  # for the arrays that have no element
    at = [room.data_ptr() + 4 * i for i in range(5)]
    code = tk_b200.lib().tk_kv_plan(at[0], at[1], 0, 16, at[2], 4, free.data_ptr(), 3, n_free.data_ptr(), at[3], at[4], starts.data_ptr(),
                                    slots.data_ptr(), 7, n_free.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert code == 0 and starts.item() == 0 and n_free.item() == 3 and slots.tolist() == [-1] * 7


# ---- append -------------------------------------------------------------------------------

def new_cache(pages, heads, page, dim, seed, odd_scales=False):
    g = torch.Generator().manual_seed(seed)
    cache = torch.randint(0, 256, (pages, heads, page, dim), generator=g, dtype=torch.uint8)
    cache[(cache & 0x7f) == 0x7f] = 0x30  # no NaN unless a test wants them
    scale = 2.0 ** torch.randint(-6, 3, (pages, heads), generator=g).float()
    if odd_scales:
        scale = scale * (1 + torch.rand(pages, heads, generator=g))
    return cache.cuda(), scale.cuda()


def check_append(k, v, slots, caches, page):
    k_cache, v_cache, k_scale, v_scale = caches
    want = []
    for x, c, s in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        values, scales = plain64.cache_values(c), s.cpu().double().numpy()
        plain64.append(x.cpu().double().numpy(), slots, values, scales, page)
        want.append((values, scales))
    tk_b200.kv_append(k, v, ints(slots, torch.int64), k_cache, v_cache, k_scale, v_scale)
    torch.cuda.synchronize()
    for (values, scales), c, s in zip(want, (k_cache, v_cache), (k_scale, v_scale)):
        assert np.array_equal(s.cpu().double().numpy(), scales)
        assert np.array_equal(plain64.cache_values(c), values, equal_nan=True)


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("odd", [False, True])
def test_append(page, dim, kind, odd):
    """Runs from the first place of a page and from the middle, over page ends, of one token and of
    many; skipped tokens; scales that grow; the rest of the cache untouched."""
    heads, pages = 3, 12
    g = np.random.default_rng(page + dim)
    slots = []
    slots += list(range(2 * page + 5, 2 * page + 6))            # one token into a page that holds 5
    slots += [-1, pages * page, -9, 10 ** 12]                    # nowhere
    slots += list(range(4 * page + page - 2, 6 * page + 3))      # over two page ends
    slots += list(range(9 * page, 10 * page))                    # a whole page
    slots += list(range(0, 1)) + list(range(7 * page + 1, 7 * page + 1 + page // 2))
    n = len(slots)
    size = torch.from_numpy(2.0 ** g.integers(-8, 9, (n, 1, 1)))
    k = (torch.from_numpy(g.standard_normal((n, heads, dim))) * size).to(kind).cuda()
    v = (torch.from_numpy(g.standard_normal((n, heads, dim))) * size).to(kind).cuda()
    caches = new_cache(pages, heads, page, dim, 1, odd), new_cache(pages, heads, page, dim, 2, odd)
    check_append(k, v, slots, (caches[0][0], caches[1][0], caches[0][1], caches[1][1]), page)


@pytest.mark.parametrize("n", [1, 1024, 1025, 9000])
def test_append_sizes(n):
    """Each number of tokens per CTA, with pages that begin and end anywhere in its share."""
    page, dim, heads = 32, 64, 1
    pages = n // page + 60
    g = np.random.default_rng(n)
    slots, s, left = [], 3, n
    while left > 0:
        take = min(left, int(g.choice([1, 2, 31, 32, 40, 100])))
        slots += range(s, s + take)
        left -= take
        s += take
        s = min(-(-s // page) * page + int(g.integers(0, 3)), s + 10 ** 6) if g.random() < 0.3 and len(slots) < n - 200 else s
    assert max(slots) < pages * page * 2
    pages = max(slots) // page + 1
    # a page continued after a gap is named in one stretch only
    k = torch.from_numpy(g.standard_normal((n, heads, dim))).half().cuda()
    v = torch.from_numpy(g.standard_normal((n, heads, dim)) * 3).half().cuda()
    a, b = new_cache(pages, heads, page, dim, 3), new_cache(pages, heads, page, dim, 4)
    check_append(k, v, slots, (a[0], b[0], a[1], b[1]), page)


def test_append_unusual_values():
    """Zeros, the smallest and largest values, infinities and NaN, largest values of the format."""
    page, dim, heads = 16, 64, 2
    for kind in (F16, BF16):
        k = torch.zeros(8, heads, dim, dtype=kind)
        k[1, 0, 3] = torch.finfo(kind).max
        k[1, 1, 4] = torch.finfo(kind).smallest_normal / 4
        k[2, 0] = float("inf")
        k[2, 0, 1] = -float("inf")
        k[3, 0, 7] = float("nan")
        k[4] = 448.0
        k[5] = 449.0 if kind == F16 else 450.0
        k[6] = -1.75 * 2.0 ** -9
        k[7, :, ::2] = 1e-3
        slots = [0, page + 3, 2 * page, 3 * page, 4 * page, 5 * page, 6 * page + 2, 7 * page + 15]
        a, b = new_cache(8, heads, page, dim, 5), new_cache(8, heads, page, dim, 6)
        check_append(k.cuda(), k.flip(0).contiguous().cuda(), slots, (a[0], b[0], a[1], b[1]), page)


def test_append_strided_and_twice():
    """Slices of a fused projection; and the same call again changes nothing."""
    page, dim, heads, n = 32, 128, 2, 50
    g = torch.Generator().manual_seed(8)
    x = torch.randn(n, 6 * dim, generator=g).half().cuda()
    k, v = x[:, 2 * dim:4 * dim].view(n, heads, dim), x[:, 4 * dim:].view(n, heads, dim)
    slots = list(range(40, 90))
    a, b = new_cache(4, heads, page, dim, 7), new_cache(4, heads, page, dim, 8)
    caches = (a[0], b[0], a[1], b[1])
    check_append(k, v, slots, caches, page)
    before = [t.clone() for t in caches]
    tk_b200.kv_append(k, v, ints(slots, torch.int64), *caches)
    assert all(torch.equal(x, y) for x, y in zip(before, caches))


# ---- attention over the cache ---------------------------------------------------------------

def paged_case(lens, news, heads, kv_heads, page, dim, kind, *, cap=0.0, slopes=None, scale=None, hint=None, spread=1.5, seed=0,
               odd_scales=False, garbage=False, bad=None, padding=0):
    """Random caches; every output row within its bound, rows behind the last token as they were."""
    g = np.random.default_rng(seed)
    width = max(-(-max(x, 1) // page) for x in lens) + 1
    counts = [-(-x // page) for x in lens]
    pages = sum(counts) + 2
    order = g.permutation(pages).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
    k_cache, k_scale = new_cache(pages, kv_heads, page, dim, seed + 1, odd_scales)
    v_cache, v_scale = new_cache(pages, kv_heads, page, dim, seed + 2, odd_scales)
    k_scale *= 2.0 ** -5
    if garbage:  # NaN bytes in every place that holds no token
        for c in (k_cache, v_cache):
            for r, x in enumerate(lens):
                if x % page:
                    c[int(table[r, x // page]), :, x % page:] = 0x7f
    if bad is not None:
        r, col, value = bad
        table[r, col] = value
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    n = int(starts[-1])
    q = torch.from_numpy(g.standard_normal((n + padding, heads, dim)) * spread).to(kind).cuda()
    out = torch.full_like(q, 5.0)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    tk_b200.attention_paged(q, k_cache, v_cache, k_scale, v_scale, ints(table), ints(lens), ints(starts), scale=scale, softcap=cap,
                            alibi_slopes=None if slopes is None else torch.tensor(slopes, dtype=torch.float32).cuda(),
                            max_query_len=max(news + [1]), max_seq_len=max(lens) if hint is None else hint, out=out)
    torch.cuda.synchronize()
    assert torch.all(out[n:] == 5.0)
    kv, vv = plain64.cache_values(k_cache), plain64.cache_values(v_cache)
    ks, vs = k_scale.cpu().double().numpy(), v_scale.cpu().double().numpy()
    o64, q64 = out.cpu().double().numpy(), q.cpu().double().numpy()
    assert np.isfinite(o64).all()
    for r, (x, m) in enumerate(zip(lens, news)):
        pos = np.arange(x - m, x)
        key = np.arange(x)
        owner = table[r, key // page]
        there = (owner >= 0) & (owner < pages)
        own = np.where(there, owner, 0)
        allowed = (key[None] <= pos[:, None]) & there[None]
        for h in range(heads):
            gk = h * kv_heads // heads
            kk = kv[own, gk, key % page] * ks[own, gk][:, None]
            vw = np.where(there[:, None], vv[own, gk, key % page] * vs[own, gk][:, None], 0.0)
            kk = np.where(there[:, None], kk, 0.0)
            want, bound = plain64.attend(q64[starts[r]:starts[r + 1], h], kk, vw, allowed, pos, scale=scale, cap=cap,
                                         slope=0.0 if slopes is None else slopes[h], half_p=2.0 ** -11, half_out=plain64.HALF[kind])
            err = np.abs(o64[starts[r]:starts[r + 1], h] - want)
            assert np.all(err <= bound), (r, h, float((err / bound).max()))
            assert np.all(o64[starts[r]:starts[r + 1], h][~allowed.any(1)] == 0)
    return q, out


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (12, 1), (6, 2)])
def test_paged_single_tokens(heads, kv_heads, page, dim, kind):
    paged_case([1, 15, 16, 17, 63, 64, 65, 200, 513], [1] * 9, heads, kv_heads, page, dim, kind, seed=page + dim + heads)


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (14, 2), (40, 1)])
def test_paged_several_tokens(heads, kv_heads, kind):
    """Causal among the new tokens; row tiles of 8 and 16, the last ones partly filled; prompts whole."""
    paged_case([5, 40, 100, 130, 7], [5, 1, 3, 9, 7], heads, kv_heads, 16, 64, kind, seed=heads)
    paged_case([33, 300], [2, 1], heads, kv_heads, 32, 128, kind, seed=heads + 1)


@pytest.mark.parametrize("cap,slopes", [(30.0, False), (0.0, True), (5.0, True)])
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_score_changes(dim, cap, slopes):
    s = [2.0 ** -(1 + i) for i in range(8)] if slopes else None
    paged_case([1, 129, 400], [1, 1, 1], 8, 4, 16, dim, F16, cap=cap, slopes=s, spread=4.0, seed=3)
    paged_case([30, 129, 400], [3, 4, 1], 8, 2, 32, dim, BF16, cap=cap, slopes=s, spread=4.0, seed=4)


def test_paged_long_and_hints():
    """Contexts cut into chunks; whatever max_seq_len says, the result is right."""
    for hint in (0, 1, 1000, 5000, 9001, 60000):
        paged_case([9001, 1, 4500, 64], [1, 1, 2, 1], 8, 2, 64, 128, F16, hint=hint, seed=11)
    paged_case([3000, 2999], [1, 1], 4, 4, 16, 64, BF16, seed=12)


def test_paged_what_is_not_there():
    """Requests without tokens, without queries, more queries than tokens; packed rows behind the last."""
    paged_case([0, 20, 0, 33, 2], [1, 0, 0, 1, 5], 4, 2, 16, 64, F16, padding=3, seed=13)
    paged_case([0], [1], 4, 2, 16, 128, F16, hint=100000, seed=14)


def test_paged_bytes_behind_the_last_token():
    paged_case([1, 17, 100, 260], [1, 2, 1, 1], 8, 2, 32, 128, F16, garbage=True, seed=15)
    paged_case([1, 17, 100, 260], [1, 2, 1, 1], 8, 2, 128, 64, BF16, garbage=True, seed=16)


@pytest.mark.parametrize("value", [-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1])
def test_paged_bad_pages(value):
    """Pages outside the cache are as if their tokens were not there, in the middle and as the only ones."""
    paged_case([200, 60], [1, 1], 4, 2, 32, 64, F16, bad=(0, 2, value), seed=17)
    paged_case([20, 60], [1, 1], 4, 2, 32, 64, F16, bad=(0, 0, value), seed=18)


def test_paged_scales():
    """Scales of any value, negative and zero softmax scale, a bfloat16 query far from 1."""
    paged_case([100, 333], [1, 1], 8, 2, 16, 128, F16, odd_scales=True, seed=19)
    for scale in (-0.1, 0.0):
        paged_case([100, 333], [1, 1], 8, 2, 16, 64, F16, scale=scale, seed=20)
    paged_case([100, 333], [1, 1], 8, 2, 16, 64, BF16, spread=1e20, scale=1e-21, seed=21)
    paged_case([100, 333], [1, 1], 8, 2, 16, 64, BF16, spread=1e-20, scale=1e19, seed=22)


def test_paged_strides():
    """Queries out of a fused projection, outputs into a wider buffer."""
    heads, dim, page = 4, 64, 16
    q, out = paged_case([50, 70], [1, 1], heads, 2, page, dim, F16, seed=23)
    fused = torch.zeros(2, 3 * heads * dim, dtype=F16, device="cuda")
    fused[:, heads * dim:2 * heads * dim] = q.reshape(2, -1)
    g = np.random.default_rng(23)
    pages = 11
    order = g.permutation(pages).astype(np.int32)
    table = np.full((2, 6), -1, np.int32)
    table[0, :4], table[1, :5] = order[:4], order[4:9]  # as paged_case lays them out
    k_cache, k_scale = new_cache(pages, 2, page, dim, 24)
    v_cache, v_scale = new_cache(pages, 2, page, dim, 25)
    wide = torch.full((2, 2 * heads * dim), 3.0, dtype=F16, device="cuda")
    tk_b200.attention_paged(fused[:, heads * dim:2 * heads * dim].view(2, heads, dim), k_cache, v_cache, k_scale * 2.0 ** -5, v_scale,
                            ints(table), ints([50, 70]), ints([0, 1, 2]), scale=0.125, max_seq_len=70,
                            out=wide[:, :heads * dim].view(2, heads, dim))
    assert torch.equal(wide[:, :heads * dim].reshape(2, heads, dim), out) and torch.all(wide[:, heads * dim:] == 3.0)


def test_far_places():
    """A cache of more than 2^32 bytes and places x heads x dim: the last pages are read and written."""
    heads, page, dim = 8, 128, 128
    pages = (1 << 32) // (heads * page * dim) + 40
    k_cache = torch.zeros(pages, heads, page, dim, dtype=torch.uint8, device="cuda")
    v_cache = torch.zeros_like(k_cache)
    scale = [torch.zeros(pages, heads, device="cuda") for _ in range(2)]
    g = np.random.default_rng(1)
    k, v = (torch.from_numpy(g.standard_normal((200, heads, dim))).half().cuda() for _ in range(2))
    table = ints([[pages - 1, pages - 3]])
    slots = [(pages - 1) * page + i for i in range(128)] + [(pages - 3) * page + i for i in range(72)]
    tk_b200.kv_append(k, v, ints(slots, torch.int64), k_cache, v_cache, *scale)
    q = torch.from_numpy(g.standard_normal((1, heads, dim))).half().cuda()
    out = tk_b200.attention_paged(q, k_cache, v_cache, *scale, table, ints([200]), ints([0, 1]), scale=0.09, max_seq_len=200)
    near = [t[[pages - 3, pages - 1]].clone() for t in (k_cache, v_cache, *scale)]
    again = tk_b200.attention_paged(q, *near, ints([[1, 0]]), ints([200]), ints([0, 1]), scale=0.09, max_seq_len=200)
    assert torch.equal(out, again)
    assert torch.count_nonzero(k_cache[:pages - 3]).item() == 0


def test_streams_and_graphs_paged():
    """Another stream; two captured graphs whose chunk scratch must not be shared, replayed at once."""
    heads, kv_heads, page, dim = 8, 2, 32, 128
    calls, wants = [], []
    for i in range(2):
        g = np.random.default_rng(i)
        k_cache, k_scale = new_cache(300, kv_heads, page, dim, 30 + i)
        v_cache, v_scale = new_cache(300, kv_heads, page, dim, 40 + i)
        table = ints(g.permutation(300).reshape(2, 150))
        q = torch.from_numpy(g.standard_normal((2, heads, dim))).half().cuda()
        args = (q, k_cache, v_cache, k_scale * 2.0 ** -5, v_scale, table, ints([4700, 3000]), ints([0, 1, 2]))
        calls.append(args)
        wants.append(tk_b200.attention_paged(*args, scale=0.09, max_seq_len=4700))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = tk_b200.attention_paged(*calls[0], scale=0.09, max_seq_len=4700, stream=side)
    side.synchronize()
    assert torch.equal(got, wants[0])
    graphs, outs = [], []
    for args in calls:
        out = torch.empty_like(args[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tk_b200.attention_paged(*args, scale=0.09, max_seq_len=4700, out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))


# ---- together -------------------------------------------------------------------------------

class Server:
    """Plan, append and attention of one layer over a state that moves on in place."""

    def __init__(self, requests, page, pages, width, heads, kv_heads, dim):
        self.page, self.heads, self.kv_heads, self.dim = page, heads, kv_heads, dim
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.n_free = ints([pages])
        self.k_cache, self.v_cache = (torch.randint(0, 256, (pages, kv_heads, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2))
        self.k_scale, self.v_scale = (torch.full((pages, kv_heads), float("nan"), device="cuda") for _ in range(2))

    def step(self, q, k, v, new, max_query_len):
        _, seq, starts, slots, _ = tk_b200.kv_plan(self.lens, new, self.table, self.free, self.n_free, page_size=self.page,
                                                   max_tokens=q.shape[0], lens_out=self.lens, n_free_out=self.n_free)
        tk_b200.kv_append(k, v, slots, self.k_cache, self.v_cache, self.k_scale, self.v_scale)
        return tk_b200.attention_paged(q, self.k_cache, self.v_cache, self.k_scale, self.v_scale, self.table, seq, starts, scale=0.125,
                                       max_query_len=max_query_len)


def test_serving():
    """Prompts, then eager and captured decode steps: the outputs follow the dequantised cache
    exactly as the plain attention does, and the cache follows the unquantised tokens to 8 bits; one
    request is refused for want of pages and gets zeros."""
    heads, kv_heads, dim, page, width = 4, 2, 64, 16, 16
    prompts = [37, 5, 64, 18]
    server = Server(4, page, 14, width, heads, kv_heads, dim)
    g = torch.Generator().manual_seed(3)
    seen = [[[], []] for _ in prompts]  # K and V of each request

    def tokens(n):
        return [torch.randn(n, h, dim, generator=g).half().cuda() for h in (heads, kv_heads, kv_heads)]

    def check(q, k, v, out, new, taken):
        first = 0
        lens = server.lens.tolist()
        table = server.table.cpu().numpy()
        kc, vc = plain64.cache_values(server.k_cache), plain64.cache_values(server.v_cache)
        ks, vs = server.k_scale.cpu().double().numpy(), server.v_scale.cpu().double().numpy()
        for r, n in enumerate(new):
            rows = slice(first, first + n)
            first += n
            if not taken[r]:
                assert torch.all(out[rows] == 0)
                continue
            seen[r][0].append(k[rows].cpu())
            seen[r][1].append(v[rows].cpu())
            assert lens[r] == sum(len(x) for x in seen[r][0])
            key = np.arange(lens[r])
            own = table[r, key // page]
            pos = np.arange(lens[r] - n, lens[r])
            for h in range(heads):
                kk = kc[own, h // 2, key % page] * ks[own, h // 2][:, None]
                vv = vc[own, h // 2, key % page] * vs[own, h // 2][:, None]
                want, bound = plain64.attend(q[rows, h].cpu().double().numpy(), kk, vv, key[None] <= pos[:, None], pos, scale=0.125, cap=0.0,
                                             slope=0.0, half_p=2.0 ** -11, half_out=2.0 ** -11)
                assert np.all(np.abs(out[rows, h].cpu().double().numpy() - want) <= bound)
                # half a step of e4m3 for each rounding a token may have met, and of the last step
                k0 = torch.cat(seen[r][0])[:, h // 2].double().numpy()
                assert np.all(np.abs(kk - k0) <= 2.0 ** -4 * np.abs(k0) + ks[own, h // 2][:, None] * 2.0 ** -9)

    q, k, v = tokens(sum(prompts))
    out = server.step(q, k, v, ints(prompts), max(prompts))
    check(q, k, v, out, prompts, [True] * 4)
    # 3 + 1 + 4 + 2 pages are used, 4 are left; now 20 tokens for request 2 need 2 of them.
    q, k, v = tokens(23)
    new = [1, 1, 20, 1]
    out = server.step(q, k, v, ints(new), 20)
    check(q, k, v, out, new, [True] * 4)
    assert server.n_free.item() == 2
    q, k, v = tokens(51)
    new = [1, 1, 48, 1]  # 3 pages: refused
    out = server.step(q, k, v, ints(new), 48)
    check(q, k, v, out, new, [True, True, False, True])
    assert server.n_free.item() == 2

    # Decode steps from one captured graph.
    q, k, v = tokens(4)
    new = ints([1, 1, 1, 1])
    saved = [t.clone() for t in (server.lens, server.table, server.n_free, server.k_cache, server.v_cache, server.k_scale, server.v_scale)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        server.step(q, k, v, new, 1)
    torch.cuda.current_stream().wait_stream(side)
    for t, x in zip((server.lens, server.table, server.n_free, server.k_cache, server.v_cache, server.k_scale, server.v_scale), saved):
        t.copy_(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = server.step(q, k, v, new, 1)
    for _ in range(6):
        for t, x in zip((q, k, v), tokens(4)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        check(q, k, v, out, [1] * 4, [True] * 4)
    assert tk_b200.device_status() == 0


def test_prompt_attention_and_cache_agree():
    """A prompt through attention_masked on the unquantised tokens, and through the cache: they
    differ by the cache's rounding only (half a step of e4m3 in V, and in K as it moves the scores)."""
    heads, kv_heads, dim, n = 8, 2, 128, 300
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(n, h, dim, generator=g).half().cuda() for h in (heads, kv_heads, kv_heads))
    server = Server(1, 64, 8, 8, heads, kv_heads, dim)
    paged = server.step(q, k, v, ints([n]), n)
    key = np.arange(n)
    own = server.table.cpu().numpy()[0, key // 64]
    back = []
    for c, s in ((server.k_cache, server.k_scale), (server.v_cache, server.v_scale)):
        x = plain64.cache_values(c)[own, :, key % 64] * s.cpu().double().numpy()[own][:, :, None]
        back.append(torch.from_numpy(x).half().cuda())  # 4 significant bits: exact
    direct = tk_b200.attention_masked(q.transpose(0, 1)[None], back[0].transpose(0, 1)[None], back[1].transpose(0, 1)[None], scale=0.125,
                                      causal=True)[0].transpose(0, 1)
    for h in range(heads):
        want, bound = plain64.attend(q[:, h].cpu().double().numpy(), back[0][:, h // 4].cpu().double().numpy(),
                                     back[1][:, h // 4].cpu().double().numpy(), key[None] <= key[:, None], key, scale=0.125, cap=0.0, slope=0.0,
                                     half_p=2.0 ** -11, half_out=2.0 ** -11)
        for got in (paged, direct):
            assert np.all(np.abs(got[:, h].cpu().double().numpy() - want) <= bound)
