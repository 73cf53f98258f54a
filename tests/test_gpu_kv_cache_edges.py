"""Paged key/value cache on the GPU: rows and scales at the ends of their range, strides other than the plain ones, the class
without waits, what a call counts.

Tolerances as in test_gpu_kv_cache.py unless a test says otherwise.
"""

import math

import pytest
import torch

import _kv_cache_model as model
from test_gpu_kv_cache import _attention_close, _equal

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _ops():
    from chitudiffusion_b200 import ops

    return ops


# ------------------------------------------------------------------------------------------------ queries of nothing
@pytest.mark.parametrize("key_scale", [0.0, 2.0 ** -126, 2.0 ** -22, 2.0 ** -7])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n", [3, 40, 300])  # few rows; one tile of a block; blocks of two, and the diagonal in several
@pytest.mark.parametrize("causal", [True, False])
def test_zero_and_tiny_query_rows(n, dtype, key_scale, causal):
    """A zero query weighs all visible keys alike, whatever the keys' scale is: the mean of the values, and log(their number)."""
    gen = torch.Generator().manual_seed(n)
    heads, group, page, lens = 2, 2, 32, [430, n]
    (kc, ks), (vc, vs) = (model.make_cache(gen, 26, page, heads, dtype, True) for _ in range(2))
    table = model.make_tables(gen, lens, page, 26)
    ks[table[0, 3:].long()] = key_scale  # of some pages only: others have ordinary ones
    ks[table[1].clamp(min=0).long()] = key_scale
    q = torch.randn(2 * n, heads * group, 128, generator=gen).to(dtype)
    q[::2] = 0.0
    q[1, 0], q[1, 1] = torch.finfo(dtype).tiny, -torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    lens_t, cu = torch.tensor(lens, dtype=torch.int32), torch.tensor([0, n, 2 * n], dtype=torch.int32)
    ref = model.attend(q, kc, vc, ks, vs, table, lens_t, cu, 128 ** -0.5, causal)
    out, lse = _ops().attn_fwd_cache(*[t.cuda() for t in (q, kc, vc, table, lens_t, cu)], k_scale=ks.cuda(), v_scale=vs.cuda(), causal=causal,
                                     return_lse=True, max_q=n)
    _attention_close(out, lse, ref, dtype, True)
    seen = torch.cat([torch.arange(length - n, length) + 1 if causal else torch.full((n,), length) for length in lens])
    assert (lse.cpu().double()[:, ::2] - seen[::2].double().log()).abs().max() <= 1.4e-4


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n", [7, 40, 300])
def test_tokens_of_nothing_appended_and_attended_to(n, dtype):
    """Zeros through append and attention, as padding or a first run on empty inputs gives them; values are ordinary in between."""
    ops, heads, group, page = _ops(), 2, 2, 64
    gen = torch.Generator().manual_seed(n)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 12, page, heads, dtype, True) for _ in range(2))
    dev = [t.cuda() for t in (kc, vc, ks, vs)]
    table, rope = torch.randperm(12, generator=gen).int()[None], model.rope_table(128, 700)
    zeros = torch.zeros(n, heads, 128, dtype=dtype)
    v = torch.randn(n, heads, 128, generator=gen).to(dtype)
    v[: n // 2] = 0.0
    q, cu = torch.zeros(n, heads * group, 128, dtype=dtype), torch.tensor([0, n], dtype=torch.int32)
    for step in (1, 2):
        lens = torch.tensor([step * n], dtype=torch.int32)
        turned = ops.kv_cache_append(zeros.cuda(), v.cuda(), dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3],
                                     rope_table=rope.cuda(), q=q.cuda())
        for x, c, s in ((zeros.float(), kc, ks), (v.float(), vc, vs)):
            model.append(x, c, s, table, lens, cu)
        for got, want in zip(dev, (kc, vc, ks, vs)):
            assert torch.equal(got.float().cpu(), want.float())  # (values: a rotated zero may have either sign)
        for causal in (True, False):
            ref = model.attend(q, kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, causal)
            out, lse = ops.attn_fwd_cache(turned, dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3],
                                          causal=causal, return_lse=True)
            _attention_close(out, lse, ref, dtype, True)


# ------------------------------------------------------------------------------------------------ scales of values
@pytest.mark.parametrize("exponents", [(-126,), (-104,), (-100, -96), (-99, -126, -80), (-60, -30), (-8, 90), (110,)])
@pytest.mark.parametrize("n", [1, 40])
def test_value_scales_of_any_exponent(n, exponents):
    """Values as small as a bf16 can be, and as large: scales that the append gives them.

    A probability is held in fp16 with the value's scale in its exponent; scales below 2^-82 are below the largest by as much as they
    are smaller, and fp16 ends in steps of 2^-24, half of which is a probability's error, against a largest one of at
    least 2^(7 - x) for scales of 2^(-82 - x): 2^(x - 32) of the largest weight for every key, or all of it where that is more than 1."""
    gen = torch.Generator().manual_seed(n)
    heads, group, page, length = 2, 4, 32, 300
    (kc, ks), (vc, vs) = (model.make_cache(gen, 10, page, heads, BF16, True) for _ in range(2))
    for p in range(10):
        vs[p] = 2.0 ** exponents[p % len(exponents)]
    table, lens = torch.randperm(10, generator=gen).int()[None], torch.tensor([length], dtype=torch.int32)
    q, cu = torch.randn(n, heads * group, 128, generator=gen).to(BF16), torch.tensor([0, n], dtype=torch.int32)
    out, lse = _ops().attn_fwd_cache(*[t.cuda() for t in (q, kc, vc, table, lens, cu)], k_scale=ks.cuda(), v_scale=vs.cuda(), return_lse=True,
                                     max_q=n)
    want, want_lse, mag = model.attend(q, kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, False)
    assert ((lse.double().cpu() - want_lse).abs() <= 1.4e-4 + 1e-6 * want_lse.abs()).all()
    below = max(0, -82 - max(exponents))
    v, _ = model.gathered(vc, vs, table[0], length)
    steps = min(1.0, 2.0 ** (below - 32)) * v.abs().sum(0).repeat_interleave(group, 0)[None]
    # (a bf16 ends in steps of 2^-133)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * 1.4e-4) * 1.01 * mag + steps + 2.0 ** -133
    got = out.double().cpu()
    assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


@pytest.mark.parametrize("n", [1, 40])
def test_many_keys_without_values(n):
    """Values of zero have the smallest scale: their weights' sum stays finite over long sequences, and so does the log-sum-exp.

    All keys after a sequence's first page score the same, 5 above the first page's (below the 2^8 at which a running maximum moves)."""
    heads, page, batch, length = 8, 256, 40, 30000
    pages = 1 + -(-length // page)
    kc = torch.zeros(pages, page, heads, 128)
    q = torch.zeros(n * batch, heads, 128, dtype=FP16)
    q[..., 0] = 1.0
    kc[1:, :, :, 0] = 5.0
    kc, vc = kc.to(E4M3).cuda(), torch.zeros(pages, page, heads, 128, dtype=E4M3, device="cuda")
    ks, vs = torch.ones(pages, heads, device="cuda"), torch.full((pages, heads), 2.0 ** -126, device="cuda")
    table = torch.arange(pages - 1, dtype=torch.int32).clamp(min=0)[None].repeat(batch, 1)
    lens, cu = torch.full((batch,), length, dtype=torch.int32), n * torch.arange(batch + 1, dtype=torch.int32)
    out, lse = _ops().attn_fwd_cache(q.cuda(), kc, vc, table.cuda(), lens.cuda(), cu.cuda(), k_scale=ks, v_scale=vs, softmax_scale=1.0,
                                     return_lse=True, max_q=n)
    want = math.log(page + (length - page) * math.exp(5.0))
    assert (out == 0).all()
    assert ((lse - want).abs() <= 1.4e-4).all(), lse.min().item()


# ------------------------------------------------------------------------------------------------ the class's host path
class _NoWaits:
    """Operations that make the host wait for the GPU raise."""

    def __enter__(self):
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")

    def __exit__(self, *exc):
        torch.cuda.set_sync_debug_mode("default")
        return False


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_the_class_does_not_wait_for_the_gpu(dtype):
    """Appends that begin pages, of equal and differing lengths, queries of other lengths than the append's, truncation: the host runs
    ahead of all of it, and every result is, bit for bit, that of the operators called one by one on tables of their own."""
    from chitudiffusion_b200 import PagedKVCache

    ops = _ops()
    gen = torch.Generator(device="cuda").manual_seed(2)
    heads, group, B, page, width = 2, 2, 3, 16, 13
    cache = PagedKVCache(B, heads, 200, page_size=page, dtype=dtype, device="cuda")
    calls = [[40, 3, 17], [16, 16, 16], [1, 1, 1], [0, 30, 2], [1, 1, 1]]
    draws = [[torch.randn(sum(new), h, 128, generator=gen, device="cuda").to(BF16) for h in (heads, heads, heads * group)] for new in calls]
    other = torch.randn(B, 5, heads * group, 128, generator=gen, device="cuda").to(BF16)
    busy = torch.randn(4096, 4096, generator=gen, device="cuda")
    cache.append(*draws[0][:2], calls[0])  # (what the first call allocates is not at issue)
    cache.attend(draws[0][2])
    cache.attend(other)
    busy = busy @ busy * 1e-4
    for b in range(B):
        cache.truncate(b)
    outs = []
    with _NoWaits():
        for _ in range(40):
            busy = busy @ busy * 1e-4
        for new, (k, v, q) in zip(calls, draws):
            if len(set(new)) == 1:
                cache.append(*(t.view(B, new[0], heads, 128) for t in (k, v)))
            else:
                cache.append(k, v, new)
            outs.append([cache.attend(q, causal=True)[0], cache.attend(other)[0], cache.attend(q, q_lens=new[::-1])[0]])
        cache.truncate(1, 20)
        outs.append([cache.attend(other)[0]])

    table = torch.arange(B * width, dtype=torch.int32, device="cuda").view(B, width)
    pools = [torch.empty(B * width, heads, page, 128, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2)]
    scales = [torch.ones(B * width, heads, device="cuda") if dtype == E4M3 else None for _ in range(2)]
    lens = [0] * B

    def tensors(new):
        cu = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
        return dict(k_cache=pools[0], v_cache=pools[1], block_table=table, kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                    cu_seqlens=cu, k_scale=scales[0], v_scale=scales[1])

    def attend(q, new, causal=False):
        return ops.attn_fwd_cache(q, **tensors(new), causal=causal, max_q=max(new), max_kv=max(lens))[0]

    for new, (k, v, q), got in zip(calls, draws, outs):
        lens = [a + n for a, n in zip(lens, new)]
        ops.kv_cache_append(k, v, **tensors(new), max_new=max(new))
        want = [attend(q, new, True), attend(other.flatten(0, 1), [5] * B), attend(q, new[::-1])]
        for x, y in zip(got, want):
            assert torch.equal(x.flatten(0, -3), y)
    lens[1] = 20
    assert torch.equal(outs[-1][0].flatten(0, 1), attend(other.flatten(0, 1), [5] * B))
    assert cache.lens == lens and cache.tensors["kv_lens"].tolist() == lens


@pytest.mark.parametrize("rank", [0, 1])
def test_a_stale_step_over_8_bit_pages_does_not_wait_for_the_gpu(monkeypatch, rank):
    from chitudiffusion_b200 import B200AttnBackend
    from chitudiffusion_b200.image_cp import B200ImageContextParallel

    cp, draw = _image_cp(monkeypatch, B200ImageContextParallel(B200AttnBackend("b200"), mode="agkv"), 3, rank, 40)
    inputs = [[draw(6)] * 3 + [draw(40) for _ in range(3)] for _ in range(6)]
    for step in range(4):
        cp.begin_forward(step, 100)
        if step < 2:
            cp.attention(*inputs[step])
        else:  # (what the first fresh and the first stale call allocate is not at issue)
            with _NoWaits():
                cp.attention(*inputs[step])


# ------------------------------------------------------------------------------------------------ the cross-step cache's ranks
def _image_cp(monkeypatch, cp, world, rank, n, B=2, H=2):
    """`cp` as rank `rank` of `world` with shards of `n` rows and 8-bit pages, every second step stale, and what draws its inputs; the other
    ranks' rows of a step are drawn when they are gathered and kept in `cp.far`."""
    gen = torch.Generator(device="cuda").manual_seed(10 * world + rank)

    def draw(rows):
        return torch.randn(B, rows, H, 128, generator=gen, device="cuda").to(BF16)

    class Group:
        group_size, rank_in_group = world, rank

        def all_gather_sequence(self, t):
            others = [draw(n) for _ in range(world - 1)]
            cp.far = (cp.far + [others])[-2:]
            return torch.cat(others[:rank] + [t] + others[rank:], 1)

    cp.far = []
    cp._kvcache_enabled = cp._kvcache_fp8 = True
    cp._kvcache_warmup, cp._kvcache_interval, cp._kvcache_tail = 0, 2, 0
    cp.enable(Group())
    return cp, draw


@pytest.mark.parametrize("n", [150, 128, 37])
@pytest.mark.parametrize("world,rank", [(1, 0), (2, 0), (2, 1), (3, 0), (3, 1), (3, 2)])
def test_image_cache_in_8_bits_on_every_rank(monkeypatch, world, rank, n):
    """Fresh and stale steps of a rank that has others on one side of it, on both sides (pages that two appends share), or none.

    Tolerance as in test_image_cache_of_other_ranks_in_8_bits, against attention over the kept rows as their codes say; those
    are the gathered rows to half a step of e4m3 (2^-4), twice where a page's earlier codes move to a larger scale."""
    from chitudiffusion_b200 import B200AttnBackend
    from chitudiffusion_b200.image_cp import B200ImageContextParallel
    from test_gpu_kv_cache import SCORE, _dense, _held

    cp, draw = _image_cp(monkeypatch, B200ImageContextParallel(B200AttnBackend("b200"), mode="agkv"), world, rank, n)
    for step in range(4):
        cp.begin_forward(step, 100)
        tq, tk, tv, iq, ik, iv = (draw(rows) for rows in (20, 20, 20, n, n, n))
        gathered = len(cp.far)
        txt, img = cp.attention(tq, tk, tv, iq, ik, iv)
        for b in range(2):
            keys = [torch.cat([t[b] for t in others] + [ik[b][:0]]).cpu() for others in cp.far]
            if step % 2 and world > 1:
                kept = _held(cp._kvcache[("cond", 0)], b)
                for exact, got in zip(keys, kept):
                    exact = exact.double()
                    assert ((got - exact).abs() <= 2 * 2 ** -4 * exact.abs() + 2 ** -9 * 2.0 ** -6).all()
                keys = kept
            k, v = (torch.cat([x.double(), own[b].cpu().double(), t[b].cpu().double()]) for x, own, t in zip(keys, (ik, iv), (tk, tv)))
            want, _, mag = _dense(torch.cat([iq[b], tq[b]]).cpu(), k, v)
            got = torch.cat([img[b], txt[b]]).double().cpu()
            tol = 2 ** -8 * want.abs() + 1.02 * (2 ** -7 + 2 * SCORE) * mag + 1e-6
            assert ((got - want).abs() <= tol).all(), (step, ((got - want).abs() / tol).max().item())
        assert world == 1 or step % 2 == 0 or len(cp.far) == gathered  # a stale step gathers nothing


# ------------------------------------------------------------------------------------------------ what a call counts
def _kernels(call):
    """Kernels of this library that a captured `call` launches."""
    from cuda.bindings import driver

    def done(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS
        return result[1] if len(result) == 2 else result[1:]

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    names = []
    for node in done(driver.cuGraphGetNodes(raw, done(driver.cuGraphGetNodes(raw))[1]))[0]:
        if done(driver.cuGraphNodeGetType(node)) == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            params = done(driver.cuGraphKernelNodeGetParams(node))
            names.append(done(driver.cuFuncGetName(params.func)) if int(params.func) else done(driver.cuKernelGetName(params.kern)))
    return sum(b"chitu" in name for name in names)


@pytest.mark.parametrize("n", [1, 5, 9, 40, 130])
@pytest.mark.parametrize("group,page,eight", [(4, 64, True), (4, 256, True), (4, 256, False), (130, 32, True)])
def test_launch_count_is_the_number_of_kernels(n, group, page, eight):
    """The two attention kernels, the one that joins pieces, the append for few and for many tokens, and its form in two launches."""
    ops = _ops()
    gen = torch.Generator().manual_seed(1)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 4, page, 1, BF16, eight) for _ in range(2))
    cache = [t.cuda() for t in (kc, vc, torch.arange(4, dtype=torch.int32)[None], torch.tensor([n + 3], dtype=torch.int32),
                                torch.tensor([0, n], dtype=torch.int32))]
    scales = dict(k_scale=ks.cuda(), v_scale=vs.cuda()) if eight else {}
    k = torch.zeros(n, 1, 128, dtype=BF16, device="cuda")
    q, rope = torch.zeros(n, group, 128, dtype=BF16, device="cuda"), model.rope_table(64, 200).cuda()
    positions = torch.arange(n, device="cuda")
    calls = (lambda: ops.kv_cache_append(k, k, *cache, **scales, rope_table=rope, q=q),
             lambda: ops.kv_cache_append(k, k, *cache, **scales, max_new=n),
             lambda: ops.kv_cache_append(k, k, *cache, **scales, rope_table=rope, q=q, max_new=1),
             lambda: ops.attn_fwd_cache(q, *cache, **scales), lambda: ops.attn_fwd_cache(q, *cache, **scales, max_q=1),
             lambda: ops.attn_fwd_cache(q, *cache, **scales, max_q=1000),
             lambda: ops.rotary([q, k], positions, rope))
    for call in calls:
        call()
        before = ops.launch_count
        call()
        counted = ops.launch_count - before
        assert counted == _kernels(call), calls.index(call)


# ------------------------------------------------------------------------------------------------ strides
def _strided(t, kind):
    """`t [pages, page, H, 128]` or `[pages, H]` with other strides: every second page of a larger pool, tokens or heads outermost."""
    if t is None:
        return None
    if kind == "every other":
        wide = torch.empty((2 * t.shape[0],) + t.shape[1:], dtype=t.dtype, device="cuda")
        view = wide[::2]
    elif kind == "padded rows":
        wide = torch.empty(t.shape[:-1] + (t.shape[-1] + 32,), dtype=t.dtype, device="cuda")
        view = wide[..., :t.shape[-1]]
    elif kind == "transposed":
        view = torch.empty([t.shape[i] for i in (range(t.dim() - 2, -1, -1) if t.dim() == 4 else (1, 0))] + ([t.shape[3]] if t.dim() == 4 else []),
                           dtype=t.dtype, device="cuda")
        view = view.permute(2, 1, 0, 3) if t.dim() == 4 else view.t()
    else:
        view = torch.empty(t.shape, dtype=t.dtype, device="cuda")
    assert view.shape == t.shape
    view.view(torch.uint8).copy_(t.contiguous().view(torch.uint8)) if t.dtype == E4M3 else view.copy_(t)
    return view


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("n", [1, 3, 70, 300])
@pytest.mark.parametrize("forms", [("plain", "every other"), ("padded rows", "transposed"), ("transposed", "plain"), ("every other", "padded rows")])
def test_projections_pools_and_scales_of_any_strides(n, forms, eight):
    """k, v and q as parts of one projection, key and value pools of two different layouts, scales that are not contiguous, through append and
    attention."""
    ops = _ops()
    heads, group, page, old = 2, 4, 32, [5, 130]
    gen = torch.Generator().manual_seed(n)
    lens = [n + o for o in old]
    pages = sum(-(-length // page) for length in lens) + 1
    (kc, ks), (vc, vs) = (model.make_cache(gen, pages, page, heads, BF16, eight) for _ in range(2))
    table = model.make_tables(gen, lens, page, pages)
    lens, cu = torch.tensor(lens, dtype=torch.int32), torch.tensor([0, n, 2 * n], dtype=torch.int32)
    rope = model.rope_table(128, 500)
    packed = torch.randn(2 * n, heads * (group + 2), 128, generator=gen).to(BF16)
    parts = packed.split([heads * group, heads, heads], 1)
    q, k, v = packed.cuda().split([heads * group, heads, heads], 1)
    dev = [_strided(t, forms[i]) for t, i in ((kc, 0), (vc, 1), (ks, 1), (vs, 0))]
    turned = ops.kv_cache_append(k, v, dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3], rope_table=rope.cuda(), q=q)
    pos = torch.cat([torch.arange(length - n, length) for length in lens.tolist()])
    for x, c, s in ((model.rotate(parts[1], pos, rope, True), kc, ks), (parts[2].float(), vc, vs)):
        model.append(x, c, s, table, lens, cu)
    for got, want in zip(dev, (kc, vc, ks, vs)):
        if want is not None:
            _equal(got, want)
    _equal(turned, model.rotate(parts[0], pos, rope, True).to(BF16))
    for causal in (True, False):
        out, lse = ops.attn_fwd_cache(q, dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3], causal=causal,
                                      return_lse=True)
        _attention_close(out, lse, model.attend(parts[0], kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, causal), BF16, eight)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("n,group", [(1, 4), (40, 4), (300, 2), (1, 100), (5, 128), (7, 43), (1, 129), (3, 200), (40, 130)])
def test_outputs_off_the_32_byte_grid_and_many_heads_of_a_key_head(n, group, eight):
    ops = _ops()
    heads, page, lens = 2, 64, [n + 200, n]
    gen = torch.Generator().manual_seed(group)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 14, page, heads, BF16, eight) for _ in range(2))
    table, lens = model.make_tables(gen, lens, page, 14), torch.tensor(lens, dtype=torch.int32)
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32)
    q = torch.randn(2 * n, heads * group, 128, generator=gen).to(BF16)
    room = torch.full((q.numel() + 24,), 7.0, dtype=BF16, device="cuda")
    out = room[8:-16].view(q.shape)
    assert out.data_ptr() % 32 == 16
    for causal in (True, False):
        ref = model.attend(q, kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, causal)
        got, lse = ops.attn_fwd_cache(*[t.cuda() for t in (q, kc, vc, table, lens, cu)], k_scale=None if ks is None else ks.cuda(),
                                      v_scale=None if vs is None else vs.cuda(), causal=causal, return_lse=True, out=out)
        assert got is out
        _attention_close(out, lse, ref, BF16, eight)
        assert (room[:8] == 7.0).all() and (room[-16:] == 7.0).all()


# ------------------------------------------------------------------------------------------------ many sequences
@pytest.mark.parametrize("eight", [True, False])
def test_thousands_of_sequences(eight):
    """A padded batch of 3000: some bring nothing, some hold nothing, pages of a common beginning are shared by all."""
    ops, heads, group, page, B = _ops(), 1, 2, 16, 3000
    gen = torch.Generator().manual_seed(5)
    new = torch.randint(0, 4, (B,), generator=gen)
    new[7], new[100:400] = 150, 0
    lens = (new + torch.randint(0, 60, (B,), generator=gen)).int()
    lens[::9] = new[::9].int()
    lens[100:250] = 0
    (kc, ks), (vc, vs) = (model.make_cache(gen, 2000, page, heads, BF16, eight) for _ in range(2))
    table = torch.randint(0, 2000, (B, int(lens.max()) // page + 1), generator=gen).int()
    table[:, :2] = torch.tensor([3, 1999], dtype=torch.int32)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).int()
    q = torch.randn(int(cu[-1]), heads * group, 128, generator=gen).to(BF16)
    ref = model.attend(q, kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, True)
    dev = [t.cuda() for t in (q, kc, vc, table, lens, cu)]
    for hint in (1, 150, None):  # the kernel for few rows, the one for chunks
        out, lse = ops.attn_fwd_cache(*dev, k_scale=None if ks is None else ks.cuda(), v_scale=None if vs is None else vs.cuda(), causal=True,
                                      return_lse=True, max_q=hint)
        _attention_close(out, lse, ref, BF16, eight)
    # the same batch appended, a page for each of its own
    table = torch.arange(B * table.shape[1], dtype=torch.int32).view(B, -1)
    own = [model.make_cache(gen, table.numel(), page, heads, BF16, eight) for _ in range(2)]
    k, v = (torch.randn(q.shape[0], heads, 128, generator=gen).to(BF16) for _ in range(2))
    devs = [[t if t is None else t.cuda() for t in pair] for pair in own]
    args = (k.cuda(), v.cuda(), devs[0][0], devs[1][0], table.cuda(), dev[4], dev[5])
    for hint in (None, 1):  # (again: what a call leaves, the same call leaves again)
        ops.kv_cache_append(*args, k_scale=devs[0][1], v_scale=devs[1][1], max_new=hint)
        if hint is None:
            for (c, s), x in zip(own, (k, v)):
                model.append(x.float(), c, s, table, lens, cu)
        for pair, got in zip(own, devs):
            for a, b in zip(pair, got):
                if a is not None:
                    _equal(b, a)


def test_the_class_reports_a_wait_that_ran_out():
    """A status that a kernel has left is raised by the next attend, as by the other entries of the product path; the scratch is replaced."""
    from chitudiffusion_b200 import PagedKVCache, _lib

    ops = _ops()
    dev = torch.device("cuda", torch.cuda.current_device())
    cache = PagedKVCache(1, 2, 200, device=dev)
    k, q = torch.randn(1, 50, 2, 128, device=dev).to(BF16), torch.randn(1, 50, 4, 128, device=dev).to(BF16)
    cache.append(k, k)
    want = cache.attend(q)[0]
    torch.cuda.synchronize()
    try:
        ops.status_word(dev).fill_(3)
        with pytest.raises(_lib.ChituB200Error, match="softmax"):
            cache.attend(q)
        assert not any(used[0] == dev.index for used in [*ops._workspaces, *ops._cut_scratches])
        assert torch.equal(cache.attend(q)[0], want)
    finally:
        ops.status_word(dev).zero_()


def test_dense_and_cache_attention_in_turn_on_one_stream():
    """Query blocks cut for an even end, blocks of a cache that runs' borders cut, and few rows share a stream's scratch."""
    ops = _ops()
    gen = torch.Generator(device="cuda").manual_seed(3)
    S, H, page = 2400, 16, 64
    assert ops._balanced_workspace_bytes(torch.cuda.current_device(), 1, S, S, H) > 0  # (this call is cut)
    q, k, v = (torch.randn(1, S, H, 128, generator=gen, device="cuda").to(BF16) for _ in range(3))
    pools = [torch.randn(80, page, 2, 128, generator=gen, device="cuda").to(BF16) for _ in range(2)]
    table = torch.randperm(80, generator=gen, device="cuda").int()[None]
    lens = torch.tensor([5000], dtype=torch.int32, device="cuda")
    calls = [lambda: ops.attn_fwd(q, k, v, return_lse=True)]
    for n in (1, 700):
        x, cu = torch.randn(n, 16, 128, generator=gen, device="cuda").to(BF16), torch.tensor([0, n], dtype=torch.int32, device="cuda")
        calls.append(lambda x=x, cu=cu, n=n: ops.attn_fwd_cache(x, *pools, table, lens, cu, causal=True, return_lse=True, max_q=n))
    wants = []
    for call in calls:  # each by itself, in scratch of its own
        with torch.cuda.stream(torch.cuda.Stream()):
            wants.append(call())
            torch.cuda.synchronize()
    for _ in range(5):
        for i in (0, 1, 0, 2, 1, 2):
            for got, want in zip(calls[i](), wants[i]):
                assert torch.equal(got, want)
