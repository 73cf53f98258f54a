"""Paged key/value cache: what the entry points refuse, on the CPU, before any CUDA call."""

import ctypes

import pytest
import torch

from chitudiffusion_b200 import _lib, ops

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def lib():
    from chitudiffusion_b200 import build

    build.build()
    return _lib.load()


def _args(**change):
    """A valid call on CPU tensors (which is refused last of all), with some of it changed."""
    page = change.pop("page", 16)
    a = dict(
        k=torch.zeros(5, 2, 128, dtype=BF16), v=torch.zeros(5, 2, 128, dtype=BF16),
        k_cache=torch.zeros(4, page, 2, 128, dtype=E4M3), v_cache=torch.zeros(4, page, 2, 128, dtype=E4M3),
        block_table=torch.zeros(2, 3, dtype=torch.int32), kv_lens=torch.tensor([3, 2], dtype=torch.int32),
        cu_seqlens=torch.tensor([0, 3, 5], dtype=torch.int32), k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2))
    a.update(change)
    return a


def _append(**change):
    return ops.kv_cache_append(**_args(**change))


def _attend(**change):
    a = _args(**{k: v for k, v in change.items() if k in _args()or k == "page"})
    extra = {k: v for k, v in change.items() if k not in a and k != "page"}
    q = extra.pop("q", torch.zeros(5, 4, 128, dtype=BF16))
    a.pop("k"), a.pop("v")
    return ops.attn_fwd_cache(q, **a, **extra)


TABLE = torch.zeros(64, 64, 2)
X, Y = torch.zeros(5, 2, 128), torch.zeros(5, 2, 128)

CACHE_REFUSALS = [
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=E4M3), v_cache=torch.zeros(4, 16, 2, 64, dtype=E4M3)), NotImplementedError, "head_dim"),
    (dict(page=48), NotImplementedError, "page_size"),
    (dict(page=8), NotImplementedError, "page_size"),
    (dict(page=512), NotImplementedError, "page_size"),
    (dict(v_cache=torch.zeros(3, 16, 2, 128, dtype=E4M3)), ValueError, "one shape"),
    (dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float8_e5m2), v_cache=torch.zeros(4, 16, 2, 128, dtype=torch.float8_e5m2)),
     NotImplementedError, "pages hold"),
    (dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=FP16), v_cache=torch.zeros(4, 16, 2, 128, dtype=FP16), k_scale=None, v_scale=None),
     NotImplementedError, "pages hold"),
    (dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=BF16), v_cache=torch.zeros(4, 16, 2, 128, dtype=BF16)), ValueError, "no scales"),
    (dict(k_scale=None), ValueError, "k_scale and v_scale"),
    (dict(v_scale=torch.ones(4, 3)), ValueError, "k_scale and v_scale"),
    (dict(v_scale=torch.ones(4, 2, dtype=FP16)), ValueError, "k_scale and v_scale"),
    (dict(k_cache=torch.zeros(4, 16, 2, 256, dtype=E4M3)[..., ::2]), ValueError, "contiguous"),
    (dict(k_cache=torch.zeros(4, 16, 2, 136, dtype=E4M3)[..., :128]), ValueError, "16-byte aligned"),
    (dict(k_cache=torch.zeros(1, 16, 2, 128, dtype=E4M3).expand(4, 16, 2, 128)), ValueError, "16-byte aligned"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError, "block_table"),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "kv_lens"),
    (dict(kv_lens=torch.zeros(2, dtype=torch.int64)), ValueError, "kv_lens"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), ValueError, "cu_seqlens"),
    (dict(cu_seqlens=torch.zeros(3)), ValueError, "cu_seqlens"),
]


@pytest.mark.parametrize("call", [_append, _attend])
@pytest.mark.parametrize("change,error,text", CACHE_REFUSALS)
def test_a_cache_that_does_not_fit_is_refused(call, change, error, text):
    with pytest.raises(error, match=text):
        call(**change)


@pytest.mark.parametrize("change,error,text", [
    (dict(k=torch.zeros(5, 256, dtype=BF16)), ValueError, "packed tokens"),
    (dict(k=torch.zeros(5, 2, 64, dtype=BF16)), ValueError, "packed tokens"),
    (dict(k=torch.zeros(5, 2, 128)), NotImplementedError, "bf16 or fp16"),
    (dict(v=torch.zeros(4, 2, 128, dtype=BF16)), ValueError, "shape mismatch"),
    (dict(v=torch.zeros(5, 2, 128, dtype=FP16)), ValueError, "shape mismatch"),
    (dict(k=torch.zeros(5, 3, 128, dtype=BF16), v=torch.zeros(5, 3, 128, dtype=BF16)), ValueError, "heads"),
    (dict(q=torch.zeros(4, 4, 128, dtype=BF16), rope_table=TABLE), ValueError, "k's tokens"),
    (dict(q=torch.zeros(5, 4, 128, dtype=FP16), rope_table=TABLE), ValueError, "k's tokens"),
    (dict(q=torch.zeros(5, 4, 128, dtype=BF16)), ValueError, "rope_table"),
    (dict(positions=torch.zeros(5, dtype=torch.int32)), ValueError, "rope_table"),
    (dict(rope_table=TABLE.double()), ValueError, "rope_table"),
    (dict(rope_table=torch.zeros(64, 72, 2)), ValueError, "turns 144"),
    (dict(rope_table=torch.zeros(64, 12, 2)), NotImplementedError, "multiple of 16"),
    (dict(rope_table=TABLE, positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(rope_table=TABLE, positions=torch.zeros(5)), ValueError, "positions"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
def test_append_refusals(change, error, text):
    with pytest.raises(error, match=text):
        _append(**change)


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(5, 512, dtype=BF16)), ValueError, "packed tokens"),
    (dict(q=torch.zeros(5, 4, 128)), NotImplementedError, "bf16 or fp16"),
    (dict(q=torch.zeros(5, 3, 128, dtype=BF16)), ValueError, "query heads"),
    (dict(q=torch.zeros(5, 0, 128, dtype=BF16)), ValueError, "query heads"),
    (dict(softmax_scale=0.0), ValueError, "softmax_scale"),
    (dict(softmax_scale=-1.0), ValueError, "softmax_scale"),
    (dict(softmax_scale=float("nan")), ValueError, "softmax_scale"),
    (dict(softmax_scale=float("inf")), ValueError, "softmax_scale"),
    (dict(out=torch.zeros(5, 4, 128, dtype=FP16)), ValueError, "out must be"),
    (dict(out=torch.zeros(5, 8, 128, dtype=BF16)[:, ::2]), ValueError, "out must be"),
    (dict(), RuntimeError, "CUDA tensors only"),
])
def test_attention_refusals(change, error, text):
    with pytest.raises(error, match=text):
        _attend(**change)


@pytest.mark.parametrize("x,change,error,text", [
    (torch.zeros(5, 256), dict(), ValueError, r"\[T, H, D\]"),
    (torch.zeros(5, 2, 128, dtype=torch.float64), dict(), ValueError, "bf16"),
    (torch.zeros(5, 2, 72), dict(), NotImplementedError, "head_dim"),
    (torch.zeros(5, 2, 528), dict(), NotImplementedError, "head_dim"),
    (torch.zeros(5, 2, 64), dict(), ValueError, "turns 128"),
    (torch.zeros(5, 2, 128), dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (torch.zeros(5, 2, 128), dict(positions=torch.zeros(5, dtype=torch.int16)), ValueError, "positions"),
    (torch.zeros(5, 2, 128), dict(rope_table=TABLE[:, :, 0]), ValueError, "rope_table"),
    (torch.zeros(5, 2, 128), dict(rope_table=TABLE[:, ::2]), ValueError, "rope_table"),
    ([torch.zeros(5, 2, 128), torch.zeros(4, 2, 128)], dict(), ValueError, "share"),
    ([torch.zeros(5, 2, 128), torch.zeros(5, 2, 128, dtype=BF16)], dict(), ValueError, "share"),
    ([torch.zeros(5, 2, 128)] * 4, dict(), ValueError, "one to three"),
    ([torch.zeros(5, 2, 128)] * 2, dict(out=[torch.zeros(5, 2, 128)]), ValueError, "as many outputs"),
    (torch.zeros(5, 2, 128), dict(out=torch.zeros(5, 2, 128, dtype=BF16)), ValueError, "out must"),
    (torch.zeros(5, 2, 128), dict(out=torch.zeros(5, 2, 130)[..., :128]), ValueError, "16-byte aligned"),
    ([X, torch.zeros(5, 2, 128)], dict(out=[Y, Y]), ValueError, "its own input"),
    ([X, Y], dict(out=[Y, X]), ValueError, "its own input"),
    ([X, X], dict(out=[X, X]), ValueError, "its own input"),
    (X, dict(out=X.view(2, 5, 128).transpose(0, 1)), ValueError, "its own input"),
    ([X, Y], dict(out=[X, Y]), RuntimeError, "CUDA tensors only"),
    (torch.zeros(5, 2, 128), dict(), RuntimeError, "CUDA tensors only"),
])
def test_rotary_refusals(x, change, error, text):
    a = dict(positions=torch.zeros(5, dtype=torch.int32), rope_table=TABLE)
    a.update(change)
    with pytest.raises(error, match=text):
        ops.rotary(x, **a)


def _descriptor(**change):
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    f = dict(k=p, v=p, ks=p, vs=p, kst=(4096, 256, 128), vst=(4096, 256, 128), kss=(2, 1), vss=(2, 1), table=p, lens=p, cu=p, stride=3,
             batch=2, width=3, pages=4, page=16, heads=2, format=1)
    f.update(change)
    return _lib.KV_CACHE.pack(f["k"], f["v"], f["ks"], f["vs"], *f["kst"], *f["vst"], *f["kss"], *f["vss"], f["table"], f["lens"], f["cu"],
                              f["stride"], f["batch"], f["width"], f["pages"], f["page"], f["heads"], f["format"]), buf, p


@pytest.mark.parametrize("change,code,text", [
    (dict(k=0), -1, b"null"), (dict(lens=0), -1, b"null"), (dict(vs=0), -1, b"scale"), (dict(format=7), -2, b"e4m3"),
    (dict(page=20), -2, b"page_size"), (dict(width=(1 << 26) + 1), -2, b"2^30"), (dict(pages=0), -1, b"page count"), (dict(width=0), -1, b"table"), (dict(batch=-1), -1, b"batch"),
    (dict(kst=(4096, 256, 8)), -1, b"stride"), (dict(vst=(0, 256, 128)), -1, b"stride"), (dict(vst=(4096, -256, 128)), -1, b"stride"),
])
def test_the_c_entries_check_the_descriptor_before_any_cuda_call(lib, change, code, text):
    desc, buf, p = _descriptor(**change)
    st = _lib._I64x2(256, 128)
    rc = lib.chitu_b200_attn_fwd_cache(desc, p, st, p, None, 4, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None)
    assert rc == code and text in lib.chitu_b200_last_error()
    rc = lib.chitu_b200_kv_append(desc, p, p, None, st, st, None, None, 0, 5, 0, 1, None, 0, None, 0, 0, 0, None)
    assert rc == code and text in lib.chitu_b200_last_error()


def test_the_c_entries_check_what_comes_with_it(lib):
    desc, buf, p = _descriptor()
    st, odd = _lib._I64x2(256, 128), _lib._I64x2(256, 124)
    attend = lib.chitu_b200_attn_fwd_cache
    assert attend(None, p, st, p, None, 4, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, None, st, p, None, 4, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, p, odd, p, None, 4, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, p, st, p + 8, None, 4, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, p, st, p, None, 3, 5, 1.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, p, st, p, None, 4, 5, 0.0, 0, 0, 1, 1, p, 1 << 40, None, None) == -1
    assert attend(desc, p, st, p, None, 4, 5, 1.0, 0, 2, 1, 1, p, 1 << 40, None, None) == -2
    assert attend(desc, p, st, p, None, 4, 5, 1.0, 0, 0, 1, 1, p, 16, None, None) == -1 and b"workspace" in lib.chitu_b200_last_error()
    assert attend(desc, p, st, p, None, 4, 5, 1.0, 0, 0, 1, 1, None, 0, None, None) == -1
    append = lib.chitu_b200_kv_append
    assert append(desc, p, None, None, st, st, None, None, 0, 5, 0, 1, None, 0, None, 0, 0, 0, None) == -1
    assert append(desc, p, p, None, odd, st, None, None, 0, 5, 0, 1, None, 0, None, 0, 0, 0, None) == -1
    assert append(desc, p, p, p, st, st, st, None, 4, 5, 0, 1, None, 0, p, 8, 128, 0, None) == -1
    assert append(desc, p, p, None, st, st, None, None, 0, 5, 2, 1, None, 0, None, 0, 0, 0, None) == -2
    assert append(desc, p, p, None, st, st, None, None, 0, 5, 0, 1, None, 0, p, 8, 24, 0, None) == -2
    assert append(desc, p, p, None, st, st, None, None, 0, 5, 0, 1, None, 0, p, 8, 144, 0, None) == -1
    rotary = lib.chitu_b200_rotary
    one, heads = _lib.ptr_array([p]), (ctypes.c_int * 1)(2)
    assert rotary(one, one, st, st, heads, 1, 5, 128, 128, 0, None, 0, p, 8, 0, None) == -1
    assert rotary(one, one, st, st, heads, 4, 5, 128, 128, 0, p, 0, p, 8, 0, None) == -2
    assert rotary(one, one, st, st, heads, 1, 5, 120, 112, 0, p, 0, p, 8, 0, None) == -2
    assert rotary(one, one, st, st, heads, 1, 5, 64, 128, 0, p, 0, p, 8, 0, None) == -1
    assert rotary(one, one, odd, st, heads, 1, 5, 128, 128, 0, p, 0, p, 8, 0, None) == -1
    assert rotary(one, one, st, st, heads, 1, 5, 128, 128, 3, p, 0, p, 8, 0, None) == -2


# ------------------------------------------------------------------------------------------------ tables, bookkeeping
@pytest.mark.parametrize("rot", [16, 64, 128])
def test_scaled_rope_tables(rot):
    from chitudiffusion_b200.pre_attention import axis_rope_table, scaled_rope_table

    plain = scaled_rope_table(rot, 300)
    assert torch.equal(plain, axis_rope_table(torch.arange(300)[:, None], [rot]))
    assert torch.equal(scaled_rope_table(rot, 300, scaling="linear", factor=4.0)[::4], plain[:75])
    # "base": the fastest pair as without, the slowest as with "linear"
    base, linear = (scaled_rope_table(rot, 300, scaling=s, factor=4.0) for s in ("base", "linear"))
    assert torch.equal(base[:, 0], plain[:, 0])
    assert (base[:, -1] - linear[:, -1]).abs().max() <= 1e-6
    # "by_parts": turns within 4096 positions decide, cos and sin share the gain
    parts = scaled_rope_table(rot, 300, scaling="by_parts", factor=4.0, original_len=4096).double()
    gain = 0.1 * torch.log(torch.tensor(4.0, dtype=torch.float64)) + 1.0
    assert (parts.square().sum(-1).sqrt() - gain).abs().max() <= 1e-6
    turns = 4096 / (2 * torch.pi) * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    fast, slow = turns > 32 * 10000.0 ** (2 / rot), turns < 10000.0 ** (-2 / rot)  # (the blend begins and ends at whole pairs)
    assert (parts[:, fast] / gain - plain[:, fast]).abs().max() <= 1e-6
    if slow.any():
        assert (parts[:, slow] / gain - linear[:, slow]).abs().max() <= 1e-6
    for bad in (dict(scaling="cubic"), dict(factor=0.5)):
        with pytest.raises(ValueError):
            scaled_rope_table(rot, 300, **bad)


class _Calls:
    """The operators' calls, in the place of the operators."""

    def __init__(self, monkeypatch):
        self.seen = []
        monkeypatch.setattr(ops, "kv_cache_append", lambda k, v, **a: self._note("append", k, a, a.get("q")))
        monkeypatch.setattr(ops, "attn_fwd_cache", lambda q, **a: self._note("attend", q, a, (q, torch.zeros(q.shape[1], q.shape[0]) if a["return_lse"] else None)))

    def _note(self, what, x, a, result):
        self.seen.append((what, tuple(x.shape), a["kv_lens"].tolist(), a["cu_seqlens"].tolist(), a["block_table"].clone(), a))
        return result


def test_paged_cache_bookkeeping(monkeypatch):
    from chitudiffusion_b200 import PagedKVCache

    calls = _Calls(monkeypatch)
    cache = PagedKVCache(2, 3, 100, page_size=16, num_pages=8, device="cpu")
    assert cache.tensors["k_cache"].shape == (8, 16, 3, 128) and cache.tensors["k_cache"].dtype == E4M3 and cache.free_pages == 8

    def tokens(*shape):
        return torch.zeros(*shape, 3, 128, dtype=BF16)

    q = torch.zeros(2, 5, 6, 128, dtype=BF16)
    assert cache.append(tokens(2, 5), tokens(2, 5), q=q, rope_table=TABLE).shape == q.shape
    assert calls.seen[-1][2:4] == ([5, 5], [0, 5, 10]) and calls.seen[-1][5]["max_new"] == 5 and cache.free_pages == 6
    out, lse = cache.attend(q, causal=True, return_lse=True)
    assert out.shape == q.shape and lse.shape == (2, 6, 5) and calls.seen[-1][1] == (10, 6, 128)
    cache.append(tokens(40), tokens(40), [33, 2])
    assert cache.lens == [38, 7] and calls.seen[-1][2:4] == ([38, 7], [0, 33, 35]) and cache.free_pages == 4
    used = calls.seen[-1][4]
    assert (used >= 0).sum().item() == 4 and used[used >= 0].unique().numel() == 4
    cache.attend(torch.zeros(3, 3, 128, dtype=BF16), q_lens=[1, 2])
    assert calls.seen[-1][3] == [0, 1, 3] and calls.seen[-1][5]["max_kv"] == 38
    # an output that would be copied to be written is refused
    cache.attend(q, out=torch.zeros_like(q))
    assert calls.seen[-1][5]["out"].shape == (10, 6, 128)
    for wrong in (torch.zeros(5, 2, 6, 128, dtype=BF16).transpose(0, 1), torch.zeros(10, 6, 128, dtype=BF16)):
        with pytest.raises(ValueError, match="contiguous"):
            cache.attend(q, out=wrong)
    # no page left: refused, nothing changes
    with pytest.raises(RuntimeError, match="free"):
        cache.append(tokens(90), tokens(90), [0, 90])
    with pytest.raises(ValueError, match="at most"):
        cache.append(tokens(63), tokens(63), [63, 0])
    assert cache.lens == [38, 7] and cache.free_pages == 4
    # what is forgotten is free again
    cache.truncate(0, 17)
    assert cache.lens == [17, 7] and cache.free_pages == 5 and cache.tensors["kv_lens"].tolist() == [17, 7]
    cache.truncate(1)
    assert cache.free_pages == 6
    # a call that the operator refuses appends nothing
    def refuse(*a, **k):
        raise ValueError("no")

    monkeypatch.setattr(ops, "kv_cache_append", refuse)
    with pytest.raises(ValueError, match="no"):
        cache.append(tokens(2, 30), tokens(2, 30))
    assert cache.lens == [17, 0] and cache.free_pages == 6 and cache.tensors["kv_lens"].tolist() == [17, 0]
    for bad in (lambda: cache.append(tokens(3, 1), tokens(3, 1)), lambda: cache.append(tokens(5), tokens(5)),
                lambda: cache.append(tokens(5), tokens(5), [3, 3]), lambda: cache.attend(q[:1]), lambda: cache.truncate(2),
                lambda: cache.truncate(0, 18), lambda: PagedKVCache(0, 1, 1, device="cpu")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        PagedKVCache(1, 1, 1, page_size=48, device="cpu")
    with pytest.raises(NotImplementedError):
        PagedKVCache(1, 1, 1, dtype=torch.float32, device="cpu")
