"""Paged key/value cache without a GPU: bookkeeping of calls that fail, ranks of the cross-step cache, tables, launch hints."""

import math

import pytest
import torch

import oracle
from chitudiffusion_b200 import PagedKVCache, ops
from chitudiffusion_b200.image_cp import B200ImageContextParallel

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------ the cross-step cache
class _Backend:
    impl = "torch_sdpa"

    def __call__(self, q, k, v, *_, softmax_scale=None, return_attn_probs=False, **__):
        out, lse = oracle.sdpa_fp32(q, k, v, softmax_scale, return_lse=True)
        return out.to(q.dtype), (lse if return_attn_probs else None), None


class _Group:
    """A rank of a group whose other ranks' rows are drawn."""

    def __init__(self, world, rank, others=None):
        self.group_size, self.rank_in_group, self.others = world, rank, others

    def all_gather_sequence(self, t):
        rows = [] if self.others is None else self.others(t)
        return torch.cat(rows[:self.rank_in_group] + [t] + rows[self.rank_in_group:], 1)


def _schedule(monkeypatch, group, eight):
    for name, value in (("CHITU_CP_KV_CACHE", "1"), ("CHITU_CP_KV_CACHE_WARMUP", "0"), ("CHITU_CP_KV_CACHE_INTERVAL", "2"),
                        ("CHITU_CP_KV_CACHE_TAIL", "0"), ("CHITU_B200_KV_CACHE_FP8", "1" if eight else "0")):
        monkeypatch.setenv(name, value)
    cp = B200ImageContextParallel(_Backend(), mode="agkv")
    cp.enable(group)
    return cp


def test_image_cache_of_a_group_of_one(monkeypatch):
    """A group without other ranks has nothing to keep in pages: fresh and stale steps are those of the 16-bit cache."""
    gen = torch.Generator().manual_seed(1)
    calls = [[torch.randn(2, rows, 2, 128, generator=gen) for rows in (3, 3, 3, 10, 10, 10)] for _ in range(4)]
    outs = []
    for eight in (False, True):
        cp = _schedule(monkeypatch, _Group(1, 0), eight)
        outs.append([])
        for step, args in enumerate(calls):
            cp.begin_forward(step, 100)
            outs[-1] += cp.attention(*args)
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and len(outs[1]) == 8
    txt_q, txt_k, txt_v, img_q, img_k, img_v = calls[1]  # a stale step: the fresh shard is all there is
    want = oracle.sdpa_fp32(torch.cat([txt_q, img_q], 1), torch.cat([txt_k, img_k], 1), torch.cat([txt_v, img_v], 1))
    assert (torch.cat(outs[1][2:4], 1) - want).abs().max() < 2e-6


def test_a_layer_whose_refill_fails_is_not_attended_to(monkeypatch):
    """The pages of a layer are filled again in place: where that ends half way the layer has no cache, and the next step gathers."""
    appended = []

    def append(k, v, **_):
        appended.append(k.shape[0])
        if len(appended) == 4:
            raise RuntimeError("no memory left")

    monkeypatch.setattr(ops, "kv_cache_append", append)
    gen = torch.Generator().manual_seed(1)
    gathered = []

    def others(t):
        gathered.append([torch.randn(t.shape, generator=gen) for _ in range(2)])
        return gathered[-1]

    group = _Group(3, 1, others)
    cp = _schedule(monkeypatch, group, True)
    cp._attn_agkv_stale_fp8 = lambda *a: pytest.fail("stale pages were attended to")
    args = [torch.randn(1, rows, 2, 128, generator=gen) for rows in (3, 3, 3, 10, 10, 10)]
    cp.begin_forward(0, 100)
    cp.attention(*args)
    cp.begin_forward(2, 100)
    with pytest.raises(RuntimeError, match="memory"):
        cp.attention(*args)
    cp.begin_forward(3, 100)  # stale by its number
    _, got = cp.attention(*args)
    assert appended == [10] * 6 and len(gathered) == 6
    (k0, k2), (v0, v2) = gathered[-2:]
    k, v = (torch.cat([a, own, b, text], 1) for a, own, b, text in ((k0, args[4], k2, args[1]), (v0, args[5], v2, args[2])))
    assert (got - oracle.sdpa_fp32(args[3], k, v)).abs().max() < 2e-6


# ------------------------------------------------------------------------------------------------ the class's bookkeeping
def test_a_table_names_no_page_behind_what_a_sequence_holds(monkeypatch):
    """Pages given back may be another sequence's: a length that the caller advances itself past its pages finds none there."""
    monkeypatch.setattr(ops, "kv_cache_append", lambda k, v, **a: None)
    cache = PagedKVCache(2, 1, 100, page_size=16, num_pages=6, device="cpu")
    tokens = torch.zeros(80, 1, 128, dtype=BF16)
    cache.append(tokens, tokens, [60, 5])
    cache.truncate(0, 16)
    cache.append(tokens, tokens, [0, 60])
    table = cache.tensors["block_table"]
    assert table.ge(0).sum(1).tolist() == [1, 5] and table[table >= 0].unique().numel() == 6
    cache.truncate(1)
    assert table.ge(0).sum(1).tolist() == [1, 0]


@pytest.mark.parametrize("error", [ValueError, TypeError, AttributeError, MemoryError, KeyboardInterrupt])
def test_a_call_that_fails_appends_nothing(monkeypatch, error):
    """Whatever ends an append: lengths, pages, table and offsets are those of before, for the next call and for the operators."""
    held = []
    monkeypatch.setattr(ops, "kv_cache_append", lambda k, v, **a: held.append(k.shape[0]))
    monkeypatch.setattr(ops, "attn_fwd_cache", lambda q, **a: (a["cu_seqlens"].clone(), None))
    cache = PagedKVCache(2, 1, 100, page_size=16, num_pages=9, device="cpu")
    tokens = [torch.zeros(n, 1, 128, dtype=BF16) for n in (0, 9, 20, 40)]
    cache.append(tokens[2], tokens[2], [17, 3])

    def state():
        return {n: None if t is None else t.clone() for n, t in cache.tensors.items() if not n.endswith("_cache")}, cache.lens, cache.free_pages

    def same(a, b):
        return a[1:] == b[1:] and all(torch.equal(a[0][n], b[0][n]) for n in a[0])

    before = state()

    def fail(*_, **__):
        raise error("no")

    with monkeypatch.context() as m:
        m.setattr(ops, "kv_cache_append", fail)
        for k, new in ((tokens[3], [8, 32]), (tokens[2].view(2, 10, 1, 128), None), (tokens[2], [17, 3]), (tokens[0], [0, 0])):
            with pytest.raises(error):
                cache.append(k, k, new)
            assert same(state(), before)
    # arguments that are no tensors fail on their own
    for bad in (lambda: cache.append(tokens[3], None, [8, 32]), lambda: cache.append(tokens[3], tokens[3], [8, 32], q=[1.0])):
        with pytest.raises((TypeError, AttributeError)):
            bad()
        assert same(state(), before)
    # queries of the last append that went through, then one more of it
    assert cache.attend(tokens[2])[0].tolist() == [0, 17, 20]
    cache.append(tokens[1], tokens[1], [9, 0])
    assert cache.lens == [26, 3] and cache.free_pages == 6 and cache.tensors["cu_seqlens"].tolist() == [0, 9, 9]
    assert cache.tensors["block_table"].ge(0).sum(1).tolist() == [2, 1] and held == [20, 9]


# ------------------------------------------------------------------------------------------------ launch hints
@pytest.mark.parametrize("tokens,batch,few", [
    (64, 64, True), (1, 1, True), (4, 1, True), (5, 1, False), (66, 64, True), (67, 64, True), (68, 64, False), (40, 64, True),
    (2699, 700, False),  # a prompt of 2000 tokens among 699 single ones
    (128, 64, False), (256, 64, False), (19200, 64, False)])
def test_an_append_without_a_hint_is_sized_for_the_longest_that_its_tokens_allow(tokens, batch, few):
    """The form for single tokens walks a sequence's tokens one after the other: it is taken where, with a token at least of every sequence, none can
    bring more than four.  Otherwise the other form, for no fewer tokens than the average."""
    expected = ops._expected_new(tokens, batch)
    assert (expected <= ops._APPEND_FEW) is few
    assert expected >= 1 and (few or expected == max(ops._APPEND_FEW + 1, -(-tokens // batch)))


# ------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("rot,factor,original_len,fast,slow", [(128, 4.0, 4096, 32.0, 1.0), (64, 8.0, 2048, 32.0, 1.0), (96, 1.0, 4096, 32.0, 1.0),
                                                               (128, 16.0, 8192, 20.0, 0.5), (16, 2.0, 100, 8.0, 1.0)])
def test_rope_table_by_parts_blends_by_turns(rot, factor, original_len, fast, slow):
    """A pair that makes r turns within the original length keeps the share (r - slow) / (fast - slow) of its angle, none below, all above."""
    from chitudiffusion_b200.pre_attention import scaled_rope_table

    table = scaled_rope_table(rot, 50, theta=10000.0, scaling="by_parts", factor=factor, original_len=original_len, beta_fast=fast, beta_slow=slow)
    gain = 0.1 * math.log(factor) + 1.0
    blended = 0
    for j in range(rot // 2):
        angle = 10000.0 ** (-2 * j / rot)
        turns = original_len * angle / (2 * math.pi)
        keep = 0.0 if turns < slow else 1.0 if turns > fast else (turns - slow) / (fast - slow)
        blended += 0.0 < keep < 1.0
        angle = keep * angle + (1.0 - keep) * angle / factor
        for p in (0, 1, 7, 49):
            # (fp32 entries: half a step of a value of at most 2)
            assert abs(table[p, j, 0].item() - gain * math.cos(p * angle)) <= 2.0 ** -23
            assert abs(table[p, j, 1].item() - gain * math.sin(p * angle)) <= 2.0 ** -23
    assert blended
    with pytest.raises(ValueError, match="beta_fast"):
        scaled_rope_table(rot, 50, scaling="by_parts", factor=factor, beta_fast=1.0, beta_slow=1.0)


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("scale", [torch.ones(1, 2).expand(4, 2), torch.ones(4, 1).expand(4, 2), torch.ones(1).expand(4, 2)])
def test_an_append_refuses_scales_that_share_memory(which, scale):
    """One scale for several pages or heads can be read, but an append would write it for each of them."""
    a = dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=E4M3), v_cache=torch.zeros(4, 16, 2, 128, dtype=E4M3),
             block_table=torch.zeros(1, 3, dtype=torch.int32), kv_lens=torch.tensor([5], dtype=torch.int32),
             cu_seqlens=torch.tensor([0, 5], dtype=torch.int32), k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2))
    a[which] = scale
    k = torch.zeros(5, 2, 128, dtype=BF16)
    with pytest.raises(ValueError, match="of its own"):
        ops.kv_cache_append(k, k, **a)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):  # (which is looked at last)
        ops.attn_fwd_cache(k, **a)


# ------------------------------------------------------------------------------------------------ scratch
def test_cache_attention_never_uses_the_key_split_buffer(monkeypatch):
    """That buffer's address may be part of a caller's captured graph, which is replayed on any stream beside eager calls."""
    cpu = torch.device("cpu")
    capturing = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: type("S", (), {"cuda_stream": 11})())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    for name, value in (("_stream_ptr", lambda dev: 11), ("_device_key", lambda dev: 0), ("_on", lambda dev: ops._NO_GUARD), ("_workspaces", {}),
                        ("_retired_workspaces", []), ("_cut_scratches", {})):
        monkeypatch.setattr(ops, name, value)
    held = ops.splitkv_workspace(cpu, 50 << 20)  # as a captured call's workspace=
    eager = ops._cache_scratch(cpu, 3 << 20)
    assert eager.data_ptr() != held.data_ptr() and not eager[:ops.SPLIT_HEADER_BYTES].any()
    assert ops._cache_scratch(cpu, 3 << 20) is eager
    larger = ops._cache_scratch(cpu, 45 << 20)
    assert larger.numel() >= 45 << 20 and larger.data_ptr() != held.data_ptr() and not larger[:ops.SPLIT_HEADER_BYTES].any()
    assert ops._cache_scratch(cpu, 3 << 20) is larger
    capturing.append(True)
    own = [ops._cache_scratch(cpu, 3 << 20) for _ in range(2)]
    assert len({t.data_ptr() for t in own + [held, larger]}) == 4 and not own[0][:ops.SPLIT_HEADER_BYTES].any()
