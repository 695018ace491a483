"""More refusals of the prompt and serving operators, on the CPU: no GPU is touched by a call that is refused."""

import pytest
import torch

import tk_b200

from test_serving_cpu import INVALID, MB, append, masked, paged, plan

# Pointers off their element's alignment: a kernel would fault on them.
MISALIGNED = (
    [(masked, {k: n * MB + 1}) for k, n in (("q", 1), ("k", 2), ("v", 3), ("out", 4))]
    + [(masked, over) for over in (dict(slopes=5 * MB + 2), dict(ids=5 * MB + 1), dict(prefix=5 * MB + 2))]
    + [(plan, {k: n * MB + off}) for k, n in (("cached", 1), ("new", 2), ("table", 3), ("free", 4), ("n_free", 5), ("lens", 6), ("seq", 7),
                                             ("starts", 8), ("left", 10)) for off in (1, 2)]
    + [(plan, dict(slots=9 * MB + 4))]
    + [(append, dict(ksc=6 * MB + 1)), (append, dict(vsc=7 * MB + 2)), (append, dict(slots=3 * MB + 4))]
    + [(paged, {k: n * MB + 2}) for k, n in (("ksc", 5), ("vsc", 6), ("table", 7), ("lens", 8), ("starts", 9), ("slopes", 10))]
)


@pytest.mark.parametrize("call,over", MISALIGNED, ids=[f"{c.__name__}-{k}+{v % MB}" for c, o in MISALIGNED for k, v in o.items()])
def test_misaligned_pointers(call, over):
    assert call(**over) == INVALID


def test_aligned_pointers_are_not_refused():
    """The same calls with the pointers on their element's alignment, and no more."""
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    good = [masked(q=MB + 2, k=2 * MB + 2, v=3 * MB + 2, out=4 * MB + 2, slopes=5 * MB + 4), masked(ids=5 * MB + 4), masked(prefix=5 * MB + 4),
            plan(cached=MB + 4, new=2 * MB + 4, table=3 * MB + 4, free=4 * MB + 4, n_free=5 * MB + 4, lens=6 * MB + 4, seq=7 * MB + 4,
                 starts=8 * MB + 4, slots=9 * MB + 8, left=10 * MB + 4),
            append(ksc=6 * MB + 4, vsc=7 * MB + 4, slots=3 * MB + 8),
            paged(ksc=5 * MB + 4, vsc=6 * MB + 4, table=7 * MB + 4, lens=8 * MB + 4, starts=9 * MB + 4, slopes=10 * MB + 4)]
    assert INVALID not in good


# scale / softcap below FP32's normal range would lose the scores' bits or all of them.
@pytest.mark.parametrize("scale,cap", [(1e-38, 1.0), (-1e-38, 30.0), (1e-45, 1e-6), (2e-36, 256.0)])
def test_scale_far_below_the_cap(scale, cap):
    assert masked(scale=scale, cap=cap) == INVALID


@pytest.mark.parametrize("scale,cap", [(0.0, 30.0), (1e-35, 30.0), (1e-37, 1.0), (1e-38, 0.0), (1e-38, 257.0), (1e-45, 1e30)])
def test_scale_above_that_is_not_refused(scale, cap):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert masked(scale=scale, cap=cap) != INVALID


OTHER_BYTES = [torch.int8, torch.bool, torch.float8_e5m2, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz]


@pytest.mark.parametrize("kinds", [(t, t) for t in OTHER_BYTES] + [(torch.uint8, t) for t in OTHER_BYTES],
                         ids=lambda p: "-".join(str(t).split(".")[1] for t in p))
def test_helpers_refuse_caches_of_other_bytes(kinds):
    """Bytes of another format would be read as e4m3. (All on the CPU: right types are refused for that.)"""
    k, v = (torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(t) for t in kinds)
    scale = torch.zeros(3, 2)
    x = torch.zeros(5, 2, 64, dtype=torch.float16)
    i = torch.int32
    with pytest.raises(ValueError, match="_cache"):
        tk_b200.kv_append(x, x, torch.zeros(5, dtype=torch.int64), k, v, scale, scale)
    with pytest.raises(ValueError, match="_cache"):
        tk_b200.attention_paged(x, k, v, scale, scale, torch.zeros(3, 4, dtype=i), torch.zeros(3, dtype=i), torch.zeros(4, dtype=i), scale=1.0)


@pytest.mark.parametrize("k_kind", [torch.uint8, torch.float8_e4m3fn], ids=["uint8", "e4m3fn"])
@pytest.mark.parametrize("v_kind", [torch.uint8, torch.float8_e4m3fn], ids=["uint8", "e4m3fn"])
def test_helpers_take_e4m3_bytes(v_kind, k_kind):
    k, v = (torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(t) for t in (k_kind, v_kind))
    scale = torch.zeros(3, 2)
    x = torch.zeros(5, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA device"):  # all that is left to refuse
        tk_b200.kv_append(x, x, torch.zeros(5, dtype=torch.int64), k, v, scale, scale)


def test_plan_of_no_requests_takes_null():
    """Arrays without an element may be null; the others may not."""
    empty = dict(r=0, cached=None, new=None, table=None, lens=None, seq=None)
    for over in (dict(n_free=None), dict(starts=None), dict(left=None), dict(slots=None), dict(free=None), dict(width=0), dict(left=8 * MB)):
        assert plan(**{**empty, **over}) == INVALID
    if not torch.cuda.is_available():
        assert plan(**empty) != INVALID and plan(**empty, free=None, cap=0, slots=None, tokens=0) != INVALID


@pytest.mark.parametrize("cap", [1e-50, 1e-46, -1e-50])
def test_helpers_refuse_caps_that_are_no_float(cap):
    """A cap that is 0 only in 32 bits is not 'none': refused, as the entry points refuse others below 1e-6."""
    q = torch.zeros(1, 2, 8, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="softcap"):
        tk_b200.attention_masked(q, q, q, scale=1.0, softcap=cap)
    cache, scale = torch.zeros(3, 2, 16, 64, dtype=torch.uint8), torch.ones(3, 2)
    i = torch.int32
    with pytest.raises(ValueError, match="softcap"):
        tk_b200.attention_paged(torch.zeros(5, 2, 64, dtype=torch.float16), cache, cache, scale, scale, torch.zeros(3, 4, dtype=i),
                                torch.zeros(3, dtype=i), torch.zeros(4, dtype=i), scale=1.0, softcap=cap)


class Handles:
    """Stands in for torch.cuda: which stream a handle becomes."""

    class Stream:
        def __init__(self, name, device):
            self.name, self.device = name, device

    def __init__(self, monkeypatch):
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: self.Stream("default", device))
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: self.Stream(handle, device))
        monkeypatch.setattr(torch.cuda, "stream", lambda stream: stream)


class OnCuda:
    device = torch.device("cuda:0")


@pytest.mark.parametrize("handle,want", [(0, "default"), (1, "default"), (0x7f00, 0x7f00)])
def test_stream_handles(handle, want, monkeypatch):
    """0 and 1 are handles of the default stream, for which ExternalStream makes a stream of its own."""
    Handles(monkeypatch)
    stream = tk_b200._on(handle, OnCuda)
    assert stream.name == want and stream.device == OnCuda.device


def test_stream_handle_of_the_thread(monkeypatch):
    """The per-thread default stream has no counterpart among torch's."""
    Handles(monkeypatch)
    with pytest.raises(ValueError, match="stream"):
        tk_b200._on(2, OnCuda)
