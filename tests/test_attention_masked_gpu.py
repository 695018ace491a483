"""Attention under masks and score changes on the GPU, against 64 bits."""

import math

import numpy as np
import pytest
import torch

import plain64
import tk_b200

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(b, h, s, d, kind, seed, spread=1.0, tokens_first=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((b, s, h, d) if tokens_first else (b, h, s, d), generator=g) * spread).to(kind).cuda()
    return x.transpose(1, 2) if tokens_first else x


def held(q, k, v, out, *, scale, causal=False, cap=0.0, slopes=None, ids=None, prefix=None, heads=None, rows=None):
    """Every output element within its bound (for some heads and rows only, if given)."""
    half = plain64.HALF[q.dtype]
    q64, k64, v64, o64 = (t.detach().cpu().double().numpy() for t in (q, k, v, out))
    b, h, sq, _ = q64.shape
    group = h // k64.shape[1]
    skv = k64.shape[2]
    assert np.isfinite(o64).all()
    for i in range(b):
        allowed = plain64.intervals(sq, skv, causal, None if ids is None else ids[i], None if prefix is None else prefix[i])
        pos = np.arange(sq) + skv - sq
        pick = np.arange(sq) if rows is None else rows
        kk, vv = k64[i], v64[i]
        if ids is not None:  # padding may hold anything
            pad = np.array(ids[i]) < 0
            kk, vv = np.where(pad[None, :, None], 0.0, kk), np.where(pad[None, :, None], 0.0, vv)
        for j in range(h) if heads is None else heads:
            qq = np.where(np.isfinite(q64[i, j]), q64[i, j], 0.0)
            want, bound = plain64.attend(qq[pick], kk[j // group], vv[j // group], allowed[pick], pos[pick], scale=scale, cap=cap,
                                         slope=0.0 if slopes is None else float(slopes[j]), half_p=half, half_out=half)
            err = np.abs(o64[i, j][pick] - want)
            assert np.all(err <= bound), (i, j, float((err - bound).max()), float((err / bound).max()))
            assert np.all(o64[i, j][pick][~allowed[pick].any(1)] == 0)


def documents(b, s, seed, pad=True):
    """Runs of random lengths, ids that come back, padding runs among them."""
    g = np.random.default_rng(seed)
    out = np.zeros((b, s), np.int32)
    for i in range(b):
        at = 0
        while at < s:
            n = int(g.choice([1, 3, 40, 128, 200]))
            out[i, at:at + n] = -1 if pad and g.random() < 0.25 else int(g.integers(0, 3))
            at += n
    return out


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 64), (2, 3, 1, 1, 300, 128), (1, 2, 2, 7, 7, 16), (1, 2, 1, 129, 129, 32),
                                   (1, 4, 2, 300, 300, 64), (2, 2, 1, 257, 640, 128), (1, 1, 1, 515, 515, 128),
                                   (1, 2, 2, 300, 140, 64)], ids=lambda s: "x".join(map(str, s)))
def test_shapes(shape, causal, kind):
    """(batch, query heads, key heads, rows, keys, head_dim); the last has rows before the first key."""
    b, h, hkv, sq, skv, d = shape
    q, k, v = make(b, h, sq, d, kind, 1), make(b, hkv, skv, d, kind, 2), make(b, hkv, skv, d, kind, 3)
    out = tk_b200.attention_masked(q, k, v, scale=1 / math.sqrt(d), causal=causal)
    held(q, k, v, out, scale=1 / math.sqrt(d), causal=causal)
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("cap,spread", [(50.0, 6.0), (2.0, 8.0), (30.0, 200.0), (1e4, 1.0)])
def test_softcap(cap, spread, kind):
    """Scores well inside the cap, around it, and far beyond it on both sides."""
    q, k, v = make(1, 4, 300, 128, kind, 4, spread), make(1, 2, 300, 128, kind, 5), make(1, 2, 300, 128, kind, 6)
    out = tk_b200.attention_masked(q, k, v, scale=0.09, causal=True, softcap=cap)
    held(q, k, v, out, scale=0.09, causal=True, cap=cap)


@pytest.mark.parametrize("cap,scale", [(1e7, 0.09), (1e25, 0.09), (1e30, 1e-3), (300.0, 1e-9), (1e-5, 0.09), (5.0, 1e4), (2.0, -0.09), (2.0, 0.0)])
def test_softcap_of_any_size(cap, scale):
    """A cap far above the scores changes nothing; one far below them leaves their signs."""
    q, k, v = make(1, 2, 300, 64, F16, 60, 4.0), make(1, 2, 300, 64, F16, 61), make(1, 2, 300, 64, F16, 62)
    out = tk_b200.attention_masked(q, k, v, scale=scale, causal=True, softcap=cap)
    held(q, k, v, out, scale=scale, causal=True, cap=0.0 if cap > 1e6 else cap)
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("spread", [1.0, 12.0, 60.0])
def test_softcap_of_mixed_rows(spread, d):
    """Rows and keys of very different sizes: small and large scores change places along a row."""
    q, k, v = make(1, 2, 600, d, BF16, 63), make(1, 1, 900, d, BF16, 64), make(1, 1, 900, d, BF16, 65)
    size = torch.ones(900, device="cuda")
    size[130:140] = spread
    size[600:610] = spread
    k, q = k * size[:, None].to(BF16), q * torch.linspace(0, 4, 600, device="cuda")[:, None].to(BF16)
    out = tk_b200.attention_masked(q, k, v, scale=0.1, causal=True, softcap=6.0)
    held(q, k, v, out, scale=0.1, causal=True, cap=6.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [50.0, 0.7])
def test_softcap_under_masks(cap, d):
    """Documents with padding that holds NaN, a prefix, and rows before the first key."""
    s = 400
    ids = documents(1, s, 70)
    ids[0, 100:240] = -1
    q, k, v = make(1, 4, s, d, F16, 71, 3.0), make(1, 2, s, d, F16, 72), make(1, 2, s, d, F16, 73)
    for causal in (False, True):
        held(q, k, v, tk_b200.attention_masked(q, k, v, scale=0.1, causal=causal, softcap=cap, doc_ids=torch.from_numpy(ids).cuda()),
             scale=0.1, causal=causal, cap=cap, ids=ids)
    prefix = [130]
    held(q, k, v, tk_b200.attention_masked(q, k, v, scale=0.1, causal=True, softcap=cap, prefix_lens=torch.tensor(prefix, dtype=torch.int32).cuda()),
         scale=0.1, causal=True, cap=cap, prefix=prefix)
    few = k[:, :, :150], v[:, :, :150]
    held(q, *few, tk_b200.attention_masked(q, *few, scale=0.1, causal=True, softcap=cap), scale=0.1, causal=True, cap=cap)
    pad = torch.from_numpy(ids[0] < 0).cuda()
    for t in (q, k, v):
        t[:, :, pad] = float("nan")
    held(q, k, v, tk_b200.attention_masked(q, k, v, scale=0.1, causal=True, softcap=cap, doc_ids=torch.from_numpy(ids).cuda()),
         scale=0.1, causal=True, cap=cap, ids=ids)


@pytest.mark.parametrize("cap", [0.0, 50.0, 0.5])
@pytest.mark.parametrize("key", [38, 135, 299])
def test_nan_key(key, cap):
    """A NaN key: rows that see it are NaN, those before it are as without it."""
    q, k, v = make(1, 2, 300, 64, F16, 66, 3.0), make(1, 2, 300, 64, F16, 67), make(1, 2, 300, 64, F16, 68)
    bad = k.clone()
    bad[:, :, key] = float("nan")
    out = tk_b200.attention_masked(q, bad, v, scale=0.125, causal=True, softcap=cap)
    assert out[:, :, key:].isnan().all()
    held(q[:, :, :key], k[:, :, :key], v[:, :, :key], out[:, :, :key], scale=0.125, causal=True, cap=cap)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("causal", [False, True])
def test_slopes(causal, cap):
    h = 6
    slopes = torch.tensor([2.0 ** -i for i in range(h)])
    q, k, v = make(1, h, 270, 64, F16, 7, 2.0), make(1, 3, 400, 64, F16, 8), make(1, 3, 400, 64, F16, 9)
    out = tk_b200.attention_masked(q, k, v, scale=0.125, causal=causal, softcap=cap, alibi_slopes=slopes.cuda())
    held(q, k, v, out, scale=0.125, causal=causal, cap=cap, slopes=slopes)


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("s,d", [(1, 64), (128, 64), (300, 128), (777, 64), (1300, 128)])
def test_documents(s, d, causal, kind):
    ids = documents(2, s, s + d)
    q, k, v = make(2, 2, s, d, kind, 10), make(2, 1, s, d, kind, 11), make(2, 1, s, d, kind, 12)
    out = tk_b200.attention_masked(q, k, v, scale=1 / math.sqrt(d), causal=causal, doc_ids=torch.from_numpy(ids).cuda())
    held(q, k, v, out, scale=1 / math.sqrt(d), causal=causal, ids=ids)
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("layout", ["all_padding", "first_tiles", "whole_tile_between", "edges", "one_document", "all_single"])
def test_document_layouts(layout):
    """Tiles that see nothing, items of which one tile sees nothing, runs that end on tile edges."""
    s = 900
    ids = np.zeros((1, s), np.int32)
    if layout == "all_padding":
        ids[:] = -7
    elif layout == "first_tiles":
        ids[0, :300] = -1
    elif layout == "whole_tile_between":
        ids[0, 100:600] = -1
        ids[0, 700:] = 5
    elif layout == "edges":
        ids[0] = np.arange(s) // 128
    elif layout == "all_single":
        ids[0] = np.arange(s)
    for causal in (False, True):
        q, k, v = make(1, 2, s, 64, F16, 13), make(1, 2, s, 64, F16, 14), make(1, 2, s, 64, F16, 15)
        out = torch.full_like(q, float("nan"))
        tk_b200.attention_masked(q, k, v, scale=0.125, causal=causal, doc_ids=torch.from_numpy(ids).cuda(), out=out)
        held(q, k, v, out, scale=0.125, causal=causal, ids=ids)
        if layout == "all_single":
            assert torch.equal(out, v)
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
def test_many_items_without_keys(kind):
    """One CTA after another meets runs of items that see nothing: 96 heads of 8 query pairs, most of
    them padding, so that each takes several, in either size of the pipeline."""
    s = 2048
    ids = np.full((1, s), -1, np.int32)
    ids[0, 130:200] = 1
    ids[0, 1900:1930] = 2
    for d in (64, 128):
        q, k, v = make(1, 96, s, d, kind, 70), make(1, 96, s, d, kind, 71), make(1, 96, s, d, kind, 72)
        for causal in (False, True):
            out = torch.full_like(q, float("nan"))
            tk_b200.attention_masked(q, k, v, scale=0.1, causal=causal, doc_ids=torch.from_numpy(ids).cuda(), out=out)
            held(q, k, v, out, scale=0.1, causal=causal, ids=ids, heads=range(0, 96, 19))
            assert torch.count_nonzero(out[:, :, 200:1900]) == 0 and torch.count_nonzero(out[:, :, :130]) == 0
    assert tk_b200.device_status() == 0


@pytest.mark.parametrize("kind", [F16, BF16], ids=["f16", "bf16"])
def test_padding_may_hold_anything(kind):
    """NaN and infinities in Q, K and V at padding positions reach no other row."""
    s, d = 500, 128
    ids = documents(1, s, 99)
    ids[0, 90:200] = -3
    q, k, v = make(1, 2, s, d, kind, 16), make(1, 2, s, d, kind, 17), make(1, 2, s, d, kind, 18)
    pad = torch.from_numpy(ids[0] < 0).cuda()
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan"))):
        t[:, :, pad] = bad
    v[:, :, 95] = float("-inf")
    for causal in (False, True):
        out = tk_b200.attention_masked(q, k, v, scale=0.1, causal=causal, doc_ids=torch.from_numpy(ids).cuda())
        held(q, k, v, out, scale=0.1, causal=causal, ids=ids)


@pytest.mark.parametrize("sq,skv", [(300, 300), (129, 700), (513, 513)])
def test_prefix(sq, skv):
    prefix = [0, 1, 150, skv, skv + 99]
    b = len(prefix)
    q, k, v = make(b, 2, sq, 64, BF16, 19), make(b, 1, skv, 64, BF16, 20), make(b, 1, skv, 64, BF16, 21)
    out = tk_b200.attention_masked(q, k, v, scale=0.125, causal=True, prefix_lens=torch.tensor(prefix, dtype=torch.int32).cuda())
    held(q, k, v, out, scale=0.125, causal=True, prefix=prefix)


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_non_positive_scale(scale):
    q, k, v = make(1, 2, 300, 64, F16, 22), make(1, 2, 300, 64, F16, 23), make(1, 2, 300, 64, F16, 24)
    for causal in (False, True):
        out = tk_b200.attention_masked(q, k, v, scale=scale, causal=causal)
        held(q, k, v, out, scale=scale, causal=causal)


def test_far_smaller_scores_after_a_masked_block():
    """A row's first key block is all masked (another document) and its own scores are far
    below 0: the reference point must come from the keys it sees."""
    s, d = 384, 64
    ids = np.zeros((1, s), np.int32)
    ids[0, 200:] = 1
    q, k, v = make(1, 1, s, d, F16, 25), make(1, 1, s, d, F16, 26), make(1, 1, s, d, F16, 27)
    q[:, :, 200:] = 8.0
    k[:, :, 200:] = -8.0 + 0.01 * k[:, :, 200:]
    out = tk_b200.attention_masked(q, k, v, scale=0.125, doc_ids=torch.from_numpy(ids).cuda())
    held(q, k, v, out, scale=0.125, ids=ids)


@pytest.mark.parametrize("case", ["tokens_first", "fused", "odd_strides", "misaligned", "out_gaps"])
def test_layouts(case):
    b, h, hkv, s, d = 2, 4, 2, 200, 64
    kind = F16
    scale = 0.125
    if case == "tokens_first":
        q, k, v = (make(b, n, s, d, kind, i, tokens_first=True) for i, n in ((28, h), (29, hkv), (30, hkv)))
        out = tk_b200.attention_masked(q, k, v, scale=scale, causal=True)
        assert out.stride() == q.stride()
    elif case == "fused":
        x = make(b, h + 2 * hkv, s, d, kind, 31, tokens_first=True)
        q, k, v = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
        out = tk_b200.attention_masked(q, k, v, scale=scale, causal=True)
    elif case == "odd_strides":
        q, k, v = (make(b, n, s, d + 3, kind, i)[..., :d] for i, n in ((32, h), (33, hkv), (34, hkv)))
        out = torch.empty(b, h, s, d + 1, dtype=kind, device="cuda")[..., :d]
        tk_b200.attention_masked(q, k, v, scale=scale, causal=True, out=out)
    elif case == "misaligned":
        def shifted(t):
            buf = torch.empty(t.numel() + 1, dtype=kind, device="cuda")
            buf[1:] = t.reshape(-1)
            return buf[1:].view(t.shape)
        q, k, v = (shifted(make(b, n, s, d, kind, i)) for i, n in ((35, h), (36, hkv), (37, hkv)))
        out = shifted(torch.zeros_like(q))
        tk_b200.attention_masked(q, k, v, scale=scale, causal=True, out=out)
    else:
        q, k, v = make(b, h, s, d, kind, 38), make(b, hkv, s, d, kind, 39), make(b, hkv, s, d, kind, 40)
        whole = torch.full((b, h, s, 2 * d), 7.0, dtype=kind, device="cuda")
        out = whole[..., :d]
        tk_b200.attention_masked(q, k, v, scale=scale, causal=True, out=out)
        assert torch.all(whole[..., d:] == 7.0)
    held(q, k, v, out, scale=scale, causal=True)


def test_more_items_than_sms():
    """320 items: CTAs take several, from the shared counter (zeroed by a memset without documents,
    by the documents' pass with them)."""
    q, k, v = make(1, 160, 300, 64, F16, 41), make(1, 40, 300, 64, F16, 42), make(1, 40, 300, 64, F16, 43)
    out = tk_b200.attention_masked(q, k, v, scale=0.125, causal=True)
    held(q, k, v, out, scale=0.125, causal=True, heads=range(0, 160, 13))
    ids = documents(1, 300, 4)
    out = tk_b200.attention_masked(q, k, v, scale=0.125, doc_ids=torch.from_numpy(ids).cuda())
    held(q, k, v, out, scale=0.125, ids=ids, heads=range(0, 160, 13))
    assert tk_b200.device_status() == 0


def test_long_documents():
    """20000 positions: the documents' pass takes several steps, runs cross them."""
    s = 20000
    g = np.random.default_rng(5)
    cuts = np.sort(g.integers(0, s, 9))
    ids = np.searchsorted(cuts, np.arange(s), side="right").astype(np.int32)[None]
    ids[0, 8000:8400] = -1
    q, k, v = make(1, 1, s, 64, F16, 44), make(1, 1, s, 64, F16, 45), make(1, 1, s, 64, F16, 46)
    rows = np.unique(np.concatenate([g.integers(0, s, 60), [0, 8191, 8192, 16383, 16384, s - 1], cuts, np.maximum(cuts - 1, 0)]))
    for causal in (False, True):
        out = tk_b200.attention_masked(q, k, v, scale=0.125, causal=causal, doc_ids=torch.from_numpy(ids).cuda())
        o64 = out[0, 0].cpu().double().numpy()
        for r in rows:
            if ids[0, r] < 0:
                assert np.all(o64[r] == 0)
                continue
            a, e = r, r + 1
            while a > 0 and ids[0, a - 1] == ids[0, r]:
                a -= 1
            while e < s and ids[0, e] == ids[0, r]:
                e += 1
            e = min(e, r + 1) if causal else e
            want, bound = plain64.attend(q[0, 0, r:r + 1].cpu().double().numpy(), k[0, 0, a:e].cpu().double().numpy(),
                                         v[0, 0, a:e].cpu().double().numpy(), np.ones((1, e - a), bool), np.array([0]), scale=0.125,
                                         cap=0.0, slope=0.0, half_p=2.0 ** -11, half_out=2.0 ** -11)
            assert np.all(np.abs(o64[r] - want[0]) <= bound[0]), r


def test_streams_and_graphs():
    """On another stream; captured twice, with the two graphs replayed on two streams at once
    and with new contents in the same buffers."""
    s, d = 700, 64
    ids = torch.from_numpy(documents(1, s, 6)).cuda()
    sets = [[make(1, 160, s, d, F16, 50 + 3 * i + n) for n in range(3)] for i in range(2)]
    want = [tk_b200.attention_masked(*x, scale=0.1, causal=True, doc_ids=ids) for x in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = tk_b200.attention_masked(*sets[0], scale=0.1, causal=True, doc_ids=ids, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs = [], []
    for x in sets:
        out = torch.empty_like(x[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tk_b200.attention_masked(*x, scale=0.1, causal=True, doc_ids=ids, out=out)
        graphs.append(g)
        outs.append(out)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    sets[0][2].mul_(2)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], tk_b200.attention_masked(*sets[0], scale=0.1, causal=True, doc_ids=ids))
    assert tk_b200.device_status() == 0


def test_agrees_with_the_plain_entry_point():
    """Without masks or changes the result is that of tk_attention_forward_f16, to 16 bits."""
    q, k, v = make(2, 3, 640, 128, F16, 60), make(2, 3, 640, 128, F16, 61), make(2, 3, 640, 128, F16, 62)
    for causal in (False, True):
        a = tk_b200.attention(q, k, v, scale=0.09, causal=causal)
        held(q, k, v, a.half(), scale=0.09, causal=causal)
        held(q, k, v, tk_b200.attention_masked(q, k, v, scale=0.09, causal=causal), scale=0.09, causal=causal)
