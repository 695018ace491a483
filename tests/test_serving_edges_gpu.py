"""Calls that the documentation of the prompt and serving operators allows and that ordinary sizes and
values do not make, against 64 bits."""

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


def rows_of(q, k, v, allowed, *, scale, cap, half_p, half_out, far=None, slope=0.0):
    """(out, bound) of one head as plain64.attend gives them, but with the error of a capped score following
    the score: tanh is a contraction, so the raw score's error stays as it is, and the capped one is off
    by 2^-20 of itself at most (argument, polynomial or exponential and reciprocal, product)."""
    d, m = q.shape[1], k.shape[0]
    x = q @ k.T * scale
    off = (d + 8) * 2.0 ** -23 * (np.abs(q) @ np.abs(k).T * abs(scale))
    if cap:
        x = cap * np.tanh(x / cap)
        off = off + np.abs(x) * 2.0 ** -20
    if slope:
        x = x - slope * far
        off = off + slope * far * 2.0 ** -22
    off = off + np.abs(x) * 2.0 ** -22 + 2.0 ** -21  # to log2 units, minus the reference point, 2^x
    x = np.where(allowed, x, -np.inf)
    some = allowed.any(1)
    top = np.where(some, x.max(1, initial=-np.inf), 0.0)
    w = np.where(allowed, np.exp(np.where(allowed, x - top[:, None], 0.0)), 0.0)
    p = w / np.where(some, w.sum(1), 1.0)[:, None]
    out = p @ v
    worst = np.where(allowed & (p > 1e-12), off, 0.0).max(1, initial=0.0)
    rel = 2.2 * worst + half_p + (m + 64) * 2.0 ** -23
    bound = p @ np.abs(v) * rel[:, None] + np.abs(v).sum(0)[None] * 2.0 ** -32
    return out, bound + half_out * (np.abs(out) + bound) + 2.0 ** -25


class Paged:
    """Requests over a cache with given K and V values (held exactly), in pages of random order."""

    def __init__(self, lens, heads, kv_heads, page, dim, seed=0, v_scales=None, width=None):
        g = np.random.default_rng(seed)
        self.lens, self.heads, self.kv_heads, self.page, self.dim = lens, heads, kv_heads, page, dim
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + 2
        order = g.permutation(pages).astype(np.int32)
        self.table = np.full((len(lens), width or max(counts + [1])), -1, np.int32)
        at = 0
        for r, c in enumerate(counts):
            self.table[r, :c] = order[at:at + c]
            at += c
        gen = torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.randn(pages, kv_heads, page, dim, generator=gen).to(torch.float8_e4m3fn) for _ in range(2))
        self.k_scale = torch.ones(pages, kv_heads)
        self.v_scale = torch.ones(pages, kv_heads) if v_scales is None else v_scales(g, pages, kv_heads, self.table)

    def values(self, r, h):
        """float64 K and V of request r for query head h."""
        key = np.arange(self.lens[r])
        own, g = self.table[r, key // self.page], h * self.kv_heads // self.heads
        return tuple(c.float().double().numpy()[own, g, key % self.page] * s.double().numpy()[own, g][:, None]
                     for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))

    def call(self, q, news, *, scale, cap=0.0, slopes=None, most=None, hint=None, out=None):
        starts = np.concatenate([[0], np.cumsum(news)])
        return tk_b200.attention_paged(q, self.k.cuda(), self.v.cuda(), self.k_scale.cuda(), self.v_scale.cuda(), ints(self.table),
                                       ints(self.lens), ints(starts), scale=scale, softcap=cap, alibi_slopes=slopes,
                                       max_query_len=max(news) if most is None else most, max_seq_len=hint, out=out)

    def held(self, q, news, out, *, scale, cap=0.0, keys=None, rows=None):
        """Each row within its bound; only `keys` of a request, if given, may carry weight; only the first `rows`."""
        o64, q64 = out.cpu().double().numpy(), q.cpu().double().numpy()
        first = 0
        for r, n in enumerate(news):
            pos = np.arange(self.lens[r] - n, self.lens[r])[:rows]
            key = np.arange(self.lens[r])
            allowed = key[None] <= pos[:, None]
            at = slice(first, first + len(pos))
            first += n
            for h in range(self.heads):
                k, v = self.values(r, h)
                pick = np.ones(len(key), bool) if keys is None else keys(r)
                want, bound = rows_of(q64[at, h], k[pick], v[pick], allowed[:, pick], scale=scale, cap=cap, half_p=2.0 ** -11,
                                      half_out=plain64.HALF[q.dtype])
                err = np.abs(o64[at, h] - want)
                assert np.all(err <= bound), (r, h, float((err / bound).max()))


def queries(n, heads, dim, kind, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, dim, generator=gen) * spread).to(kind)


# ---- caps of any size over the cache -----------------------------------------------------------

@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [1e-5, 0.7, 30.0, 1e3, 1e4, 1e6, 1e7, 1e9, 1e25, 1e30])
def test_paged_softcap_of_any_size(cap, dim, kind):
    """A cap far above the scores changes nothing, one far below them leaves their signs; the last head's
    scores are large beside the others', in the same tile of rows."""
    c = Paged([1, 70, 1300], 4, 1, 16, dim, seed=1)
    q = queries(4, 4, dim, kind, 2, 4.0)
    q[:, 3] *= min(cap, 4000.0)
    q = q.cuda()
    for hint in (70, 1300, 100000):
        out = c.call(q, [1, 2, 1], scale=0.09, cap=cap, hint=hint)
        c.held(q, [1, 2, 1], out, scale=0.09, cap=cap)


@pytest.mark.parametrize("cap", [1e7, 1e30])
def test_paged_softcap_with_slopes(cap):
    """As without a cap, slopes applied."""
    slopes = torch.tensor([0.5, 0.25], device="cuda")
    c = Paged([300], 2, 1, 32, 128, seed=3)
    q = queries(1, 2, 128, F16, 4, 4.0).cuda()
    out = c.call(q, [1], scale=0.09, cap=cap, slopes=slopes).cpu().double().numpy()
    far = 299.0 - np.arange(300)[None]
    for h in range(2):
        k, v = c.values(0, h)
        want, bound = rows_of(q[:, h].cpu().double().numpy(), k, v, np.ones((1, 300), bool), scale=0.09, cap=cap, half_p=2.0 ** -11,
                              half_out=2.0 ** -11, far=far, slope=float(slopes[h]))
        assert np.all(np.abs(out[:, h] - want) <= bound)


# ---- NaN over the cache ------------------------------------------------------------------------

SPLITS = [1, 700, 9001, 100000]  # one chunk, a cluster, scratch: what max_seq_len makes of the same context


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("hint", SPLITS)
def test_paged_nan_query(hint, cap, dim, kind):
    """A query row with a NaN is NaN, in the rows beside it nothing changes; a row that sees no key is 0 all the same."""
    c = Paged([17, 2500, 1], 4, 2, 16, dim, seed=5, width=700)
    q = queries(4, 4, dim, kind, 6)
    bad = q.clone()
    bad[0, 1, 5] = float("nan")
    bad[2, 0] = float("nan")  # one of two queries of the second request
    bad[3, 3, 0] = float("nan")
    out = c.call(bad.cuda(), [1, 2, 1], scale=0.1, cap=cap, hint=hint)
    hit = bad.isnan().any(-1).cuda()
    assert out[hit].isnan().all()
    clean = torch.where(hit[..., None], 0.0, out)
    fine = torch.where(hit.cpu()[..., None], 0.0, q)
    o64 = clean.cpu().double().numpy()
    assert np.isfinite(o64).all()
    first = 0
    for r, n in enumerate([1, 2, 1]):
        pos = np.arange(c.lens[r] - n, c.lens[r])
        for h in range(4):
            k, v = c.values(r, h)
            want, bound = rows_of(fine[first:first + n, h].double().numpy(), k, v, np.arange(c.lens[r])[None] <= pos[:, None], scale=0.1,
                                  cap=cap, half_p=2.0 ** -11, half_out=plain64.HALF[kind])
            ok = ~hit[first:first + n, h].cpu().numpy()
            assert np.all(np.abs(o64[first:first + n, h] - want)[ok] <= bound[ok]), (r, h)
        first += n
    c.lens = [0, 2500, 0]  # two requests without a token, their queries NaN or not
    out = c.call(bad.cuda(), [1, 2, 1], scale=0.1, cap=cap, hint=hint)
    assert torch.count_nonzero(out[[0, 3]]) == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("hint", SPLITS)
@pytest.mark.parametrize("length,key", [(1, 0), (17, 16), (17, 3), (65, 64), (2500, 0), (2500, 1040), (2500, 2499), (2500, 2498)])
def test_paged_nan_key(length, key, hint, cap, dim):
    """A NaN K token: rows that see it are NaN wherever it stands; an earlier one of the new tokens is as without it."""
    c = Paged([length], 4, 2, 16, dim, seed=7, width=700)
    n = min(length, 2)
    q = queries(n, 4, dim, F16, 8).cuda()
    where = int(c.table[0, key // 16]), key % 16
    fine = c.k.clone()
    c.k.view(torch.uint8)[where[0], 0, where[1], 9] = 0x7f  # for query heads 0 and 1
    out = c.call(q, [n], scale=0.1, cap=cap, hint=hint)
    c.k = fine
    sees = torch.arange(length - n, length) >= key
    assert out[sees.cuda()][:, :2].isnan().all()
    clean = out.clone()
    clean[sees.cuda(), :2] = c.call(q, [n], scale=0.1, cap=cap, hint=hint)[sees.cuda(), :2]
    c.held(q, [n], clean, scale=0.1, cap=cap)


# ---- rows past max_query_len ---------------------------------------------------------------------

@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (3, 1), (12, 2), (7, 1)])
@pytest.mark.parametrize("hint", [1, 700, 9001, 100000])
@pytest.mark.parametrize("most", [0, 1, 2, 3])
def test_paged_rows_past_the_most(most, hint, heads, kv_heads, kind):
    """Query tokens past max_query_len are left as they were; those before it stand where they stand."""
    news = [1, 5, 3, 4]
    c = Paged([40, 2600, 3, 900], heads, kv_heads, 16, 64, seed=9, width=700)
    q = queries(sum(news), heads, 64, kind, 10).cuda()
    out = torch.full_like(q, 7.0)
    c.call(q, news, scale=0.125, most=most, hint=hint, out=out)
    whole = c.call(q, news, scale=0.125, hint=hint)
    first = 0
    for n in news:
        assert torch.all(out[first + min(n, most):first + n] == 7.0)
        whole[first:first + min(n, most)] = out[first:first + min(n, most)]
        first += n
    c.held(q, news, whole, scale=0.125)


# ---- scales of V -----------------------------------------------------------------------------------

def two_scales(ratio, negative=False):
    def make(g, pages, kv_heads, table):
        s = torch.from_numpy(2.0 ** g.uniform(-1, 1, (pages, kv_heads))).float()
        for row in table:
            s[torch.from_numpy(row[::2][row[::2] >= 0].astype(np.int64))] *= ratio
        if negative:
            s = s * torch.from_numpy(g.choice([-1.0, 1.0], (pages, kv_heads))).float()
        return s
    return make


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 24, 2.0 ** 40, 2.0 ** 55, 2.0 ** -40])
@pytest.mark.parametrize("hint", [1, 700, 9001, 100000])
def test_paged_small_scales_with_all_the_weight(hint, ratio, page, dim):
    """Pages of large and small V scales in turn, and the weight on the small ones: the scores of the others
    are 60 and more below. What those add is below 2^-86 * 2^55 of a small page's values, nothing in bfloat16."""
    lens = [page * 2, 100, 3000]
    c = Paged(lens, 4, 2, page, dim, seed=11, v_scales=two_scales(ratio))
    small = 0 if ratio < 1 else 1  # which pages of two in turn
    ramp = torch.linspace(1.0, 2.0, dim)
    for r, row in enumerate(c.table):
        for col, own in enumerate(row[:-(-lens[r] // page)]):
            noise = 1 + 0.125 * torch.rand(c.kv_heads, page, dim, generator=torch.Generator().manual_seed(int(own)))
            c.k[int(own)] = ((1.0 if col % 2 == small else -1.0) * noise * ramp).to(torch.float8_e4m3fn)
    q = (ramp * (1 + 0.1 * torch.rand(3, 4, dim, generator=torch.Generator().manual_seed(12)))).to(BF16).cuda()
    # q.k is 7/3 dim at least (the mean square of the ramp); 30 on each side of 0.
    scale = 30.0 / (7 / 3 * dim)
    out = c.call(q, [1, 1, 1], scale=scale, hint=hint)
    c.held(q, [1, 1, 1], out, scale=scale, keys=lambda r: np.arange(lens[r]) // page % 2 == small)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ratio", [1.0, 2.0 ** 9])
@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
def test_paged_negative_scales(kind, ratio, dim):
    """A scale is a factor like another: pages of negative ones among the others, and alone."""
    c = Paged([5, 90, 1400], 4, 2, 16, dim, seed=13, v_scales=two_scales(ratio, negative=True))
    c.k_scale = c.k_scale * torch.from_numpy(np.random.default_rng(14).choice([-1.0, 1.0], tuple(c.k_scale.shape))).float()
    q = queries(3, 4, dim, kind, 15).cuda()
    for hint in (1, 1400, 50000):
        c.held(q, [1, 1, 1], c.call(q, [1, 1, 1], scale=0.1, hint=hint), scale=0.1)
    c.v_scale = -c.v_scale.abs()
    c.held(q, [1, 1, 1], c.call(q, [1, 1, 1], scale=0.1), scale=0.1)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("zero", [0.0, 2.0 ** -100])
def test_paged_pages_of_zeros(zero, dim):
    """Pages whose V are zeros carry the append's least scale (or 0): among others, first, last, and alone."""
    c = Paged([16, 64, 900], 4, 2, 16, dim, seed=16)
    for row in c.table:
        for own in row[::3]:
            if own >= 0:
                c.v.view(torch.uint8)[int(own)] = 0
                c.v_scale[int(own)] = zero
    q = queries(3, 4, dim, F16, 17).cuda()
    for hint in (1, 900, 50000):
        out = c.call(q, [1, 1, 1], scale=0.1, hint=hint)
        assert torch.count_nonzero(out[0]) == 0
        c.held(q, [1, 1, 1], out, scale=0.1)


# ---- capped scores of very different rows ------------------------------------------------------------

@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("slopes", [False, True], ids=["plain", "slopes"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [30.0, 200.0, 1e3, 1e4, 1e5, 1e6, 1e7])
def test_masked_softcap_beside_large_rows(cap, dim, slopes, kind):
    """Rows with scores of a few, beside rows of the same 32 whose scores are far beyond the cap."""
    n, h = 300, 2
    if kind == F16 and cap > 1e6:
        pytest.skip("queries that large are not binary16")
    gen = torch.Generator().manual_seed(20)
    small = 2.0 ** -9
    size = torch.where(torch.arange(n) % 3 == 1, small * cap, small)
    q = (torch.randn(1, h, n, dim, generator=gen) * size[:, None]).to(kind).cuda()
    k, v = (torch.randn(1, 1, n, dim, generator=gen).to(kind).cuda() for _ in range(2))
    scale = 3.0 / (small * math.sqrt(dim))
    s = torch.tensor([0.5, 0.125]) if slopes else None
    out = tk_b200.attention_masked(q, k, v, scale=scale, causal=True, softcap=cap, alibi_slopes=None if s is None else s.cuda())
    pos = np.arange(n)
    for j in range(h):
        want, bound = rows_of(q[0, j].cpu().double().numpy(), k[0, 0].cpu().double().numpy(), v[0, 0].cpu().double().numpy(),
                              pos[None] <= pos[:, None], scale=scale, cap=cap, half_p=plain64.HALF[kind], half_out=plain64.HALF[kind],
                              far=np.abs(pos[:, None] - pos[None]), slope=0.0 if s is None else float(s[j]))
        err = np.abs(out[0, j].cpu().double().numpy() - want)
        assert np.all(err <= bound), (j, float((err / bound).max()))
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("cap", [300.0, 1e9, 1e25, 1e30])
@pytest.mark.parametrize("scale", [1e-6, 1e-12, 1e-20, 1e-30, 1e-37])
def test_masked_small_scale_under_a_large_cap(scale, cap):
    """Large values and a small scale: the scores are a few, scale / softcap is below what FP32 holds."""
    gen = torch.Generator().manual_seed(21)
    size = math.sqrt(3.0 / (scale * 8.0))
    q, k = (torch.randn(1, 1, 200, 64, generator=gen).mul(size).to(BF16).cuda() for _ in range(2))
    v = torch.randn(1, 1, 200, 64, generator=gen).to(BF16).cuda()
    pos = np.arange(200)
    for s in (None, torch.tensor([0.25])):
        out = tk_b200.attention_masked(q, k, v, scale=scale, causal=True, softcap=cap, alibi_slopes=None if s is None else s.cuda())
        want, bound = rows_of(q[0, 0].cpu().double().numpy(), k[0, 0].cpu().double().numpy(), v[0, 0].cpu().double().numpy(),
                              pos[None] <= pos[:, None], scale=float(np.float32(scale)), cap=cap, half_p=2.0 ** -8, half_out=2.0 ** -8,
                              far=np.abs(pos[:, None] - pos[None]), slope=0.0 if s is None else 0.25)
        assert np.all(np.abs(out[0, 0].cpu().double().numpy() - want) <= bound)


# ---- an idle step ----------------------------------------------------------------------------------

@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("max_tokens", [0, 7, 9000])
def test_plan_of_no_requests(max_tokens, in_place):
    """The helper's call with empty tensors: the slots stand for nothing, the free pages stay; and the rest of the step."""
    none, table, n_free = ints([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([3])
    out = dict(lens_out=none, n_free_out=n_free) if in_place else {}
    lens, seq, starts, slots, left = tk_b200.kv_plan(none, ints([]), table, ints([4, 5, 6]), n_free, page_size=16, max_tokens=max_tokens, **out)
    assert lens.numel() == 0 and seq.numel() == 0 and starts.tolist() == [0] and left.tolist() == [3]
    assert slots.tolist() == [-1] * max_tokens
    cache, scale = torch.zeros(9, 2, 16, 64, dtype=torch.uint8, device="cuda"), torch.ones(9, 2, device="cuda")
    x = torch.ones(max_tokens, 2, 64, dtype=F16, device="cuda")
    tk_b200.kv_append(x, x, slots, cache, cache.clone(), scale, scale.clone())
    assert torch.count_nonzero(cache) == 0 and torch.all(scale == 1)
    q = torch.ones(max_tokens, 4, 64, dtype=F16, device="cuda")
    keep = torch.full_like(q, 3.0)
    assert torch.all(tk_b200.attention_paged(q, cache, cache, scale, scale, table, seq, starts, scale=0.1, out=keep) == 3.0)


# ---- autograd ------------------------------------------------------------------------------------

def attention_calls():
    """(call, tensors by name) of both attentions; any float tensor may be replaced."""
    gen = torch.Generator().manual_seed(30)
    q, k, v = (torch.randn(1, h, 40, 64, generator=gen).half().cuda() for h in (4, 2, 2))
    slopes = torch.rand(4, generator=gen).cuda()
    masked = dict(q=q, k=k, v=v, slopes=slopes)
    c = Paged([40], 4, 2, 16, 64, seed=31)
    paged = dict(q=queries(1, 4, 64, F16, 32).cuda(), ks=c.k_scale.cuda(), vs=c.v_scale.cuda(), slopes=slopes)
    kc, vc = c.k.cuda(), c.v.cuda()
    table, lens, starts = ints(c.table), ints([40]), ints([0, 1])

    def call_masked(q, k, v, slopes, out=None):
        return tk_b200.attention_masked(q, k, v, scale=0.1, causal=True, alibi_slopes=slopes, out=out)

    def call_paged(q, ks, vs, slopes, out=None):
        return tk_b200.attention_paged(q, kc, vc, ks, vs, table, lens, starts, scale=0.1, alibi_slopes=slopes, out=out)

    return [(call_masked, masked), (call_paged, paged)]


@pytest.mark.parametrize("which", [0, 1], ids=["masked", "paged"])
def test_backward_raises(which):
    """There is no gradient: an output of inputs that require one says so in backward, and is right otherwise."""
    call, given = attention_calls()[which]
    want = call(**given)
    assert not want.requires_grad
    for name in given:
        leaf = given[name].clone().requires_grad_()
        for x in (leaf, leaf * 1):
            args = {**given, name: x}
            out = call(**args)
            assert torch.equal(out, want) and out.requires_grad
            with pytest.raises(RuntimeError, match="not implemented"):
                out.float().sum().backward()
            assert leaf.grad is None
            with torch.no_grad():
                assert not call(**args).requires_grad
            with pytest.raises(ValueError, match="out"):
                call(**args, out=torch.empty_like(want))
            with torch.no_grad():
                out = torch.empty_like(want)
                call(**args, out=out)
                assert torch.equal(out, want)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(given[name], torch.ones_like(given[name]))
            with pytest.raises(ValueError, match="forward-mode"):
                call(**{**given, name: dual})
    with torch.inference_mode():
        inner = {k: v.clone() for k, v in given.items()}
        assert torch.equal(call(**inner), want)
        out = torch.empty_like(want)
    call(**inner, out=out)  # inference tensors have no version
    assert torch.equal(out, want)


def test_written_tensors_have_new_versions():
    """What a call writes in place counts as changed: a backward pass that saved it before raises."""
    for call, given in attention_calls():
        out = torch.empty_like(given["q"])
        version = out._version
        call(**given, out=out)
        assert out._version > version
        weight = torch.ones_like(out, requires_grad=True)
        loss = (out * weight).float().sum()
        call(**given, out=out)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        with pytest.raises(ValueError, match="out"):
            call(**given, out=torch.empty_like(out).requires_grad_())
    lens, new, table, free, n_free = ints([3]), ints([4]), ints([[0, -1]]), ints([1, 2]), ints([2])
    slots = torch.empty(4, dtype=torch.int64, device="cuda")
    before = [t._version for t in (lens, table, n_free, slots, new, free)]
    tk_b200.kv_plan(lens, new, table, free, n_free, page_size=4, max_tokens=4, lens_out=lens, n_free_out=n_free, slots=slots)
    after = [t._version for t in (lens, table, n_free, slots, new, free)]
    assert all(a > b for a, b in zip(after[:4], before[:4])) and after[4:] == before[4:]
    cache, scales = [torch.zeros(3, 2, 16, 64, dtype=torch.uint8, device="cuda") for _ in range(2)], [torch.ones(3, 2, device="cuda") for _ in range(2)]
    x = torch.ones(4, 2, 64, dtype=F16, device="cuda")
    before = [t._version for t in cache + scales]
    tk_b200.kv_append(x, x, slots, *cache, *scales)
    assert all(t._version > b for t, b in zip(cache + scales, before))
    tk_b200.kv_append(x.clone().requires_grad_(), x, slots, *cache, *scales)  # 8 bits carry no gradient
    for i in range(2):
        bad = list(scales)
        bad[i] = scales[i].clone().requires_grad_()
        with pytest.raises(ValueError, match="_scale"):
            tk_b200.kv_append(x, x, slots, *cache, *bad)


# ---- stream handles --------------------------------------------------------------------------------

def test_stream_handles():
    """A call on handle 0 runs on the default stream, on another stream's handle on that one."""
    call, given = attention_calls()[0]
    args = (given["q"], given["k"], given["v"])
    want = tk_b200.attention_masked(*args, scale=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for handle, stream in ((0, torch.cuda.default_stream()), (side.cuda_stream, side)):
        with tk_b200._on(handle, given["q"]):
            assert torch.cuda.current_stream().cuda_stream == stream.cuda_stream == handle
        out = tk_b200.attention_masked(*args, scale=0.1, stream=handle)
        stream.synchronize()
        assert torch.equal(out, want)


# ---- large caps under masks -------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("cap", [300.0, 1e6])
@pytest.mark.parametrize("mask", ["documents", "documents_causal", "prefix", "few_keys", "nan_key"])
def test_masked_large_caps_under_masks(mask, cap, dim, kind):
    """Caps above 256: padding that holds NaN, a prefix, rows before the first key, a NaN key; rows of a few beside large ones."""
    n, h = 400, 2
    gen = torch.Generator().manual_seed(40)
    size = torch.where(torch.arange(n) % 3 == 1, 0.01 * cap if cap < 1e4 else 3000.0, 2.0)
    q = (torch.randn(1, h, n, dim, generator=gen) * size[:, None]).to(kind)
    m = 150 if mask == "few_keys" else n
    k, v = (torch.randn(1, 1, m, dim, generator=gen).to(kind) for _ in range(2))
    scale, slopes = 1 / math.sqrt(dim), torch.tensor([0.5, 0.0625])
    pos, key = np.arange(n) + m - n, np.arange(m)
    allowed = key[None] <= pos[:, None] if mask != "documents" else np.ones((n, m), bool)
    kw, clean = dict(causal=mask != "documents"), [x.double().numpy() for x in (q, k, v)]
    if mask.startswith("documents"):
        ids = np.searchsorted([3, 100, 131, 260, 390], key, side="right").astype(np.int32)
        ids[100:131], ids[200:250] = -1, -5
        allowed = allowed & np.array([[a <= j < b for j in key] for a, b in plain64.runs_of(ids)])
        kw["doc_ids"] = ints(ids[None])
        pad = torch.from_numpy(ids < 0)
        for x in (q, k, v):
            x[:, :, pad] = float("nan")
        clean = [np.where((ids < 0)[None, None, :, None], 0.0, x) for x in clean]
    if mask == "prefix":
        allowed = allowed | (key < 170)[None]
        kw["prefix_lens"] = ints([170])
    if mask == "nan_key":
        k[:, :, 333] = float("nan")
    for s in (None, slopes):
        out = tk_b200.attention_masked(q.cuda(), k.cuda(), v.cuda(), scale=scale, softcap=cap, alibi_slopes=None if s is None else s.cuda(), **kw)
        o64 = out.cpu().double().numpy()
        rows = n
        if mask == "nan_key":
            assert out[:, :, 333:].isnan().all()
            rows = 333
        for j in range(h):
            want, bound = rows_of(clean[0][0, j][:rows], clean[1][0, 0], clean[2][0, 0], allowed[:rows], scale=scale, cap=cap,
                                  half_p=plain64.HALF[kind], half_out=plain64.HALF[kind], far=np.abs(pos[:rows, None] - key[None]),
                                  slope=0.0 if s is None else float(s[j]))
            err = np.abs(o64[0, j][:rows] - want)
            assert np.all(err <= bound), (j, float((err / bound).max()))
            assert np.all(o64[0, j][:rows][~allowed[:rows].any(1)] == 0)
    assert tk_b200.device_status() == 0


# ---- rescaled pages ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens", [1, 1500], ids=["warp", "cta"])
def test_append_rescales_with_one_rounding(tokens, dim):
    """14 * 2.7142856 / 4 = 9.4999996 is nearer to 9 than to 10; FP32 holds it as 9.5, a tie that goes to 10. All bytes, and
    scales that bring their products next to the ties of the format."""
    page, heads = 16, 2
    every = torch.arange(256, dtype=torch.uint8)
    every[(every & 0x7f) == 0x7f] = 0
    factors = [np.float32(t / v) for v in (14.0, 13.0, 11.0, 9.0, 15.0, 7.0) for t in (9.5, 8.5, 10.5, 4.75, 5.25)]
    factors = [f for f in factors if 0.5 < f < 1] + [np.nextafter(f, np.float32(s)) for f in factors if 0.5 < f < 1 for s in (0, 1)]
    pages = max(len(factors), -(-tokens // page)) + 1
    k_cache = every.repeat(pages * heads * page * dim // 256).view(pages, heads, page, dim).clone().cuda()
    k_scale = torch.ones(pages, heads)
    for p, f in enumerate(factors):
        k_scale[p] = 4.0 * float(f)  # from there to 4
    k_scale = k_scale.cuda()
    v_cache, v_scale = k_cache.clone(), k_scale.clone()
    slots = [p * page + 3 for p in range(len(factors))]
    slots += [-1] * max(0, tokens - len(slots))
    x = torch.full((len(slots), heads, dim), 1500.0, dtype=F16).cuda()  # needs a scale of 4
    values, scales = plain64.cache_values(k_cache), k_scale.cpu().double().numpy()
    plain64.append(x.cpu().double().numpy(), slots, values, scales, page)
    tk_b200.kv_append(x, x, ints(slots, torch.int64), k_cache, v_cache, k_scale, v_scale)
    for c, s in ((k_cache, k_scale), (v_cache, v_scale)):
        assert np.array_equal(s.cpu().double().numpy(), scales)
        assert np.array_equal(plain64.cache_values(c), values)
