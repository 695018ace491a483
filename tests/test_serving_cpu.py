"""Refusals of the prompt and serving operators: no GPU is touched by a call that is refused."""

import ctypes as C
import math

import pytest
import torch

import plain64
import tk_b200

INVALID = tk_b200.CUDA_ERROR_INVALID_VALUE
MB = 1 << 20  # addresses that are never dereferenced, megabytes apart


def masked(**over):
    a = dict(q=MB, k=2 * MB, v=3 * MB, out=4 * MB, strides=None, batch=1, heads=4, heads_kv=2, sq=64, skv=64, d=64, scale=0.125, cap=0.0,
             slopes=None, ids=None, prefix=None, causal=1)
    a.update(over)
    st = None if a["strides"] is None else C.cast((C.c_int64 * 12)(*a["strides"]), C.c_void_p)
    codes = {fn(a["q"], a["k"], a["v"], a["out"], st, a["batch"], a["heads"], a["heads_kv"], a["sq"], a["skv"], a["d"], a["scale"], a["cap"],
                a["slopes"], a["ids"], a["prefix"], a["causal"], None)
             for fn in (tk_b200.lib().tk_attention_masked_f16, tk_b200.lib().tk_attention_masked_bf16)}
    assert len(codes) == 1
    return codes.pop()


GOOD = [16384, 4096, 64, 8192, 4096, 64, 8192, 4096, 64, 16384, 4096, 64]


@pytest.mark.parametrize("over", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(batch=0), dict(heads=0), dict(heads_kv=0), dict(heads=5), dict(sq=0),
    dict(skv=0), dict(d=48), dict(d=256), dict(scale=math.nan), dict(scale=math.inf), dict(scale=-3e38), dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf), dict(cap=1e-9),
    dict(cap=3e38), dict(causal=2), dict(ids=5 * MB, prefix=6 * MB), dict(ids=5 * MB, skv=65), dict(prefix=5 * MB, causal=0), dict(out=MB), dict(out=2 * MB + 64),
    dict(ids=4 * MB + 4), dict(ids=5 * MB, batch=65536, heads=2), dict(prefix=4 * MB), dict(slopes=4 * MB), dict(batch=2 ** 31 - 1, heads=4), dict(sq=2 ** 31 - 1, skv=2 ** 31 - 1),
    dict(strides=GOOD[:2] + [0] + GOOD[3:]), dict(strides=GOOD[:4] + [-64] + GOOD[5:]), dict(strides=GOOD[:11] + [32]),
    dict(strides=GOOD[:10] + [64, 64]), dict(strides=GOOD[:9] + [4096, 4096, 64], batch=2), dict(strides=[2 ** 62] + GOOD[1:], batch=3),
], ids=lambda d: ",".join(f"{k}" for k in d))
def test_masked_refusals(over):
    assert masked(**over) == INVALID


def plan(**over):
    a = dict(cached=MB, new=2 * MB, r=8, page=16, table=3 * MB, width=10, free=4 * MB, cap=100, n_free=5 * MB, lens=6 * MB, seq=7 * MB,
             starts=8 * MB, slots=9 * MB, tokens=64, left=10 * MB)
    a.update(over)
    return tk_b200.lib().tk_kv_plan(a["cached"], a["new"], a["r"], a["page"], a["table"], a["width"], a["free"], a["cap"], a["n_free"],
                                    a["lens"], a["seq"], a["starts"], a["slots"], a["tokens"], a["left"], None)


@pytest.mark.parametrize("over", [
    dict(cached=None), dict(new=None), dict(table=None), dict(free=None), dict(n_free=None), dict(lens=None), dict(seq=None), dict(starts=None),
    dict(slots=None), dict(left=None), dict(r=-1), dict(page=0), dict(width=0), dict(cap=-1), dict(tokens=-1), dict(lens=MB + 4), dict(seq=MB),
    dict(lens=2 * MB), dict(left=5 * MB + 2), dict(slots=4 * MB), dict(table=2 * MB), dict(starts=7 * MB + 16), dict(slots=8 * MB + 8),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_plan_refusals(over):
    assert plan(**over) == INVALID


def append(**over):
    a = dict(k=MB, v=2 * MB, ks=256, vs=256, slots=3 * MB, n=10, heads=2, dim=128, kc=4 * MB, vc=5 * MB, ksc=6 * MB, vsc=7 * MB, pages=10,
             page=32)
    a.update(over)
    codes = {fn(a["k"], a["v"], a["ks"], a["vs"], a["slots"], a["n"], a["heads"], a["dim"], a["kc"], a["vc"], a["ksc"], a["vsc"], a["pages"],
                a["page"], None) for fn in (tk_b200.lib().tk_kv_append_e4m3_f16, tk_b200.lib().tk_kv_append_e4m3_bf16)}
    assert len(codes) == 1
    return codes.pop()


@pytest.mark.parametrize("over", [
    dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(ksc=None), dict(vsc=None), dict(n=-1), dict(heads=0),
    dict(heads=65536, ks=2 ** 24, vs=2 ** 24), dict(dim=96), dict(pages=0), dict(page=48), dict(page=8), dict(ks=255), dict(ks=248), dict(vs=260),
    dict(k=MB + 8), dict(v=2 * MB + 2), dict(kc=4 * MB + 8), dict(ksc=6 * MB + 2), dict(slots=3 * MB + 4), dict(vc=4 * MB), dict(ksc=4 * MB),
    dict(k=4 * MB + 64), dict(slots=5 * MB), dict(vsc=6 * MB + 16),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_append_refusals(over):
    assert append(**over) == INVALID


def paged(**over):
    a = dict(q=MB, qs=512, out=2 * MB, os=512, n=4, kc=3 * MB, vc=4 * MB, ksc=5 * MB, vsc=6 * MB, pages=10, page=32, table=7 * MB, width=4,
             lens=8 * MB, starts=9 * MB, r=3, heads=4, heads_kv=2, dim=128, mq=1, ms=100, scale=0.1, cap=0.0, slopes=None)
    a.update(over)
    codes = {fn(a["q"], a["qs"], a["out"], a["os"], a["n"], a["kc"], a["vc"], a["ksc"], a["vsc"], a["pages"], a["page"], a["table"], a["width"],
                a["lens"], a["starts"], a["r"], a["heads"], a["heads_kv"], a["dim"], a["mq"], a["ms"], a["scale"], a["cap"], a["slopes"], None)
             for fn in (tk_b200.lib().tk_attention_paged_e4m3_f16, tk_b200.lib().tk_attention_paged_e4m3_bf16)}
    assert len(codes) == 1
    return codes.pop()


@pytest.mark.parametrize("over", [
    dict(q=None), dict(out=None), dict(kc=None), dict(vc=None), dict(ksc=None), dict(vsc=None), dict(table=None), dict(lens=None),
    dict(starts=None), dict(n=-1), dict(pages=0), dict(width=0), dict(r=-1), dict(heads=0), dict(heads_kv=0), dict(heads=5), dict(dim=32),
    dict(page=8), dict(page=256), dict(mq=-1), dict(ms=-1), dict(scale=math.nan), dict(scale=-math.inf), dict(cap=-0.5), dict(cap=math.inf), dict(cap=1e-30),
    dict(width=2 ** 26),
    dict(qs=504), dict(os=516), dict(q=MB + 2), dict(out=2 * MB + 8), dict(kc=3 * MB + 16), dict(out=MB), dict(out=3 * MB), dict(out=4 * MB),
    dict(out=5 * MB), dict(out=7 * MB), dict(out=8 * MB), dict(out=9 * MB), dict(slopes=2 * MB), dict(mq=2 ** 31 - 1),
], ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_paged_refusals(over):
    assert paged(**over) == INVALID


def test_accepted_arguments_reach_the_device_check():
    """The calls that the refusals above are variations of are valid."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for code in (masked(), masked(strides=GOOD), plan(), plan(lens=MB, left=5 * MB), append(), paged()):
        assert code not in (0, INVALID)


def test_helpers_refuse_what_does_not_fit():
    h = torch.float16
    q = torch.zeros(1, 4, 8, 64, dtype=h)
    k = torch.zeros(1, 2, 8, 64, dtype=h)
    call = tk_b200.attention_masked
    for args, kw in [((q, k, k), {}), ((q.float(), k, k), {}), ((q, k, k.bfloat16()), {}), ((q, k[..., :32], k[..., :32]), {}),
                     ((q, k, torch.zeros(1, 2, 9, 64, dtype=h)), {}), ((q.transpose(2, 3), k, k), {}),
                     ((q, k, k), dict(doc_ids=torch.zeros(1, 8))), ((q, k, k), dict(alibi_slopes=torch.zeros(3))),
                     ((q, k, k), dict(prefix_lens=torch.zeros(2, dtype=torch.int32))), ((q, k, k), dict(out=q.to("meta")))]:
        with pytest.raises(ValueError):
            call(*args, scale=1.0, **kw)
    i = torch.int32
    with pytest.raises(ValueError):  # on the CPU
        tk_b200.kv_plan(torch.zeros(2, dtype=i), torch.zeros(2, dtype=i), torch.zeros(2, 4, dtype=i), torch.zeros(5, dtype=i),
                        torch.zeros(1, dtype=i), page_size=16, max_tokens=4)
    with pytest.raises(ValueError):
        tk_b200.kv_plan(torch.zeros(2, dtype=i), torch.zeros(3, dtype=i), torch.zeros(2, 4, dtype=i), torch.zeros(5, dtype=i),
                        torch.zeros(1, dtype=i), page_size=16, max_tokens=4)
    cache, scale = torch.zeros(3, 2, 16, 64, dtype=torch.uint8), torch.zeros(3, 2)
    t = torch.zeros(5, 2, 64, dtype=h)
    slots = torch.zeros(5, dtype=torch.int64)
    for args in [(t, t, slots, cache, cache, scale, scale), (t, t, slots.int(), cache, cache, scale, scale), (t, t[:4], slots, cache, cache, scale, scale),
                 (t, t, slots, cache.float(), cache, scale, scale), (t, t, slots, cache, cache[:2], scale, scale),
                 (t, t, slots, cache, cache, scale[:2], scale), (t.transpose(0, 1), t, slots, cache, cache, scale, scale)]:
        with pytest.raises(ValueError):
            tk_b200.kv_append(*args)
    lens, starts, table = torch.zeros(3, dtype=i), torch.zeros(4, dtype=i), torch.zeros(3, 4, dtype=i)
    for args in [(t, cache, cache, scale, scale, table, lens, starts), (t, cache, cache, scale, scale, table, lens, lens),
                 (t, cache, cache, scale, scale, table.long(), lens, starts), (t[:, :, :32], cache, cache, scale, scale, table, lens, starts)]:
        with pytest.raises(ValueError):
            tk_b200.attention_paged(*args, scale=1.0)


def test_plain_e4m3():
    """The tests' own rounding against torch's conversion, over all ties and the subnormals."""
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    every = every[torch.isfinite(every)].unique().double()
    between = torch.cat([every, (every[1:] + every[:-1]) / 2, (every[1:] * 3 + every[:-1]) / 4])
    want = between.float().to(torch.float8_e4m3fn).double().numpy()
    assert (plain64.e4m3(between.numpy()) == want).all()
