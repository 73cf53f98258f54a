"""Rotary positions, the paged cache's append and attention over it, on the GPU against plain models.

Tolerances, fixed before the first run:
* rotary and append are the model's own fp32 operations, rounded one by one: equal bit for bit (16-bit values, codes and scales).
* attention: the result's own rounding is half a step, eps(q's type) / 2 of the value.  Probabilities are rounded to fp16
  (8-bit pages, fp16 inputs: 2^-11) or bf16 (2^-8) before they meet the values, which moves the result by at most that times
  softmax |v|.  A score is a sum of 128 products in fp32, off by at most 128 * 2^-24 of the sum of their sizes (below 16
  here: 1.3e-4), 2^x and the factors by 1e-6 more; twice that times softmax |v|.  The log-sum-exp moves by as much as a score.
"""

import math

import pytest
import torch

import _kv_cache_model as model

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
SCORE = 1.4e-4


def _ops():
    from chitudiffusion_b200 import ops

    return ops


def _equal(got, ref):
    got = got.cpu()
    assert got.dtype == ref.dtype and got.shape == ref.shape
    if ref.dtype == E4M3:
        got, ref = got.contiguous().view(torch.uint8), ref.contiguous().view(torch.uint8)
    off = int((got != ref).sum())
    assert off == 0, f"{off} of {ref.numel()} values differ"


def _attention_close(out, lse, ref, dtype, eight):
    want, want_lse, mag = ref
    probability = torch.finfo(FP16 if eight or dtype == FP16 else BF16).eps / 2
    got = out.double().cpu()
    assert torch.isfinite(got).all()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (probability + 2 * SCORE) * 1.01 * mag + 1e-7
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()
    if lse is not None:
        got = lse.double().cpu()
        none = want_lse == -math.inf
        assert torch.equal(got == -math.inf, none)
        assert ((got - want_lse).abs()[~none] <= SCORE + 1e-6 * want_lse.abs()[~none]).all(), (got - want_lse).abs()[~none].max().item()


# ------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 128, 128), (7, 5, 64, 64), (33, 3, 80, 32), (130, 12, 128, 96), (3, 2, 256, 16), (9, 1, 512, 512),
                                       (2111, 3, 16, 16)])
def test_rotary(T, H, D, rot, interleaved, dtype):
    gen = torch.Generator().manual_seed(T + D)
    q, k = (torch.randn(T, h, D, generator=gen).to(dtype) for h in (2 * H, H))
    table = model.rope_table(rot, 200)
    positions = torch.randint(-3, 210, (T,), generator=gen)  # some outside the table
    refs = [model.rotate(t, positions, table, interleaved).to(dtype) for t in (q, k)]
    for pos in (positions.cuda(), positions.int().cuda()):
        for got, ref in zip(_ops().rotary([q.cuda(), k.cuda()], pos, table.cuda(), interleaved=interleaved), refs):
            _equal(got, ref)


def test_rotary_strides_and_outputs():
    ops = _ops()
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(37, 4 + 2 + 2, 128, generator=gen).to(BF16)
    table, positions = model.rope_table(64, 512), torch.arange(100, 137)
    dev = qkv.cuda()
    parts = [dev[:, :4], dev[:, 4:6]]  # views of a packed projection
    refs = [model.rotate(t.cpu(), positions, table, False).to(BF16) for t in parts]
    for got, ref in zip(ops.rotary(parts, positions.cuda(), table.cuda(), interleaved=False), refs):
        _equal(got, ref)
    # in place, in the packed tensor: the values keep what they were
    same = ops.rotary(parts, positions.cuda(), table.cuda(), interleaved=False, out=parts)
    assert same[0] is parts[0]
    for got, ref in zip(parts, refs):
        _equal(got, ref)
    _equal(dev[:, 6:], qkv[:, 6:])
    # [B, S, H, D], channels that are not contiguous, an address off the 16-byte grid
    x = torch.randn(2, 9, 3, 128, generator=gen)
    ref = model.rotate(x.flatten(0, 1), torch.arange(18), table, True).view(x.shape)
    _equal(ops.rotary(x.cuda(), torch.arange(18).view(2, 9).cuda(), table.cuda()), ref)
    _equal(ops.rotary(x.transpose(-1, -2).contiguous().cuda().transpose(-1, -2), torch.arange(18).cuda(), table.cuda()), ref)
    flat = torch.zeros(x.numel() + 1).cuda()
    flat[1:] = x.flatten().cuda()
    _equal(ops.rotary(flat[1:].view(x.shape), torch.arange(18).cuda(), table.cuda()), ref)
    assert ops.rotary(x[:, :0].cuda(), torch.zeros(0, dtype=torch.int32).cuda(), table.cuda()).shape == (2, 0, 3, 128)


# ------------------------------------------------------------------------------------------------------------- append
def _append_case(page, new, old, heads, heads_q, dtype, eight, heads_first, rot, interleaved, explicit, seed=0, pages=None, spoil=None):
    gen = torch.Generator().manual_seed(seed + page)
    lens = [n + o for n, o in zip(new, old)]
    pages = sum(-(-n // page) for n in lens) + 2 if pages is None else pages
    table = model.make_tables(gen, lens, page, pages)
    if spoil is not None:
        spoil(table)
    T, behind = sum(new), 3  # rows that belong to no sequence
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    lens = torch.tensor(lens, dtype=torch.int32)
    k, v, q = (torch.randn(T + behind, h, 128, generator=gen) for h in (heads, heads, heads_q))
    if new and new[0] > 2:  # something larger, nothing at all, something tiny
        k[0], v[1], k[2] = 40 * k[0], 0.0, 1e-5 * k[2]
    k, v, q = (t.to(dtype) for t in (k, v, q))
    caches = [model.make_cache(gen, pages, page, heads, dtype, eight, heads_first) for _ in range(2)]
    rope = model.rope_table(rot, 500)
    hints = [max(new + [1]), 1, 1000, None]  # whatever the launch is sized for
    seq_pos = torch.cat([torch.arange(int(lens[b]) - n, int(lens[b])) for b, n in enumerate(new)] + [torch.zeros(behind, dtype=torch.long)])
    positions = torch.randint(-2, 505, (T + behind,), generator=gen) if explicit else None
    turn = seq_pos if positions is None else positions
    put = lambda c: c.transpose(1, 2).contiguous().cuda().transpose(1, 2) if heads_first else c.contiguous().cuda()  # noqa: E731
    devs = [[(put(c), None if s is None else s.cuda()) for c, s in caches] for _ in hints]
    got_qs = [_ops().kv_cache_append(
        k.cuda(), v.cuda(), dev[0][0], dev[1][0], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[0][1], v_scale=dev[1][1],
        positions=None if positions is None else positions.cuda(), rope_table=rope.cuda(), interleaved=interleaved, q=q.cuda(), max_new=hint)
        for hint, dev in zip(hints, devs)]
    for (c, s), x in zip(caches, (model.rotate(k, turn, rope, interleaved), v.float())):
        model.append(x, c, s, table, lens, cu)
    for dev, got_q in zip(devs, got_qs):
        for (c, s), (gc, gs) in zip(caches, dev):
            _equal(gc, c)
            if s is not None:
                _equal(gs, s)
        _equal(got_q[:T], model.rotate(q, turn, rope, interleaved).to(dtype)[:T])


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new,old", [([1], [0]), ([1, 1, 1, 1], [0, 5, 15, 16]), ([4, 3, 0, 2], [15, 62, 9, 254]), ([3, 0, 70, 17], [14, 9, 63, 0]),
                                     ([300], [130]), ([5, 600, 1, 33], [0, 1, 2, 300])])
def test_append(page, new, old, eight):
    _append_case(page, new, old, 3, 5, BF16, eight, True, 128, False, False)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("dtype,heads_first,rot,interleaved,explicit", [
    (FP16, False, 128, True, False), (BF16, False, 32, True, True), (FP16, True, 96, False, True), (BF16, True, 16, True, False)])
def test_append_forms(dtype, heads_first, rot, interleaved, explicit, eight):
    _append_case(32, [5, 40, 1], [30, 3, 64], 4, 4, dtype, eight, heads_first, rot, interleaved, explicit)


@pytest.mark.parametrize("eight", [True, False])
def test_append_into_pages_that_do_not_exist(eight):
    """Page numbers outside the pool, positions behind the table's end and before the sequence's begin: nothing is written."""
    def spoil(table):
        table[0, 1], table[1, 0], table[2, 1] = -5, 1000, 2 ** 31 - 1

    _append_case(16, [40, 3, 20], [3, 2, 9], 2, 2, BF16, eight, True, 128, False, False, spoil=spoil)
    for n in (40, 3):  # the length counts fewer tokens than come, or none
        _append_case(16, [n], [-2], 2, 2, BF16, eight, True, 128, False, True)
        _append_case(16, [n, 5], [-n, 7], 2, 2, BF16, eight, True, 128, False, True)


def test_append_without_rotation_and_twice():
    """The same call twice leaves what one leaves; a larger value later raises the page's scale and rescales what is there."""
    ops = _ops()
    gen = torch.Generator().manual_seed(5)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 3, 16, 2, BF16, True) for _ in range(2))
    table, cu = torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    dev = [t.cuda() for t in (kc, vc, ks, vs)]
    for n, grow in ((4, 1.0), (8, 300.0), (12, 1.0), (16, 0.0), (20, 2.0)):
        k, v = (grow * torch.randn(4, 2, 128, generator=gen).to(BF16) for _ in range(2))
        lens = torch.tensor([n], dtype=torch.int32)
        for _ in range(2):
            assert ops.kv_cache_append(k.cuda(), v.cuda(), dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3]) is None
        for x, c, s in ((k, kc, ks), (v, vc, vs)):
            model.append(x.float(), c, s, table, lens, cu)
        for got, ref in zip(dev, (kc, vc, ks, vs)):
            _equal(got, ref)


def test_append_of_values_at_the_ends_of_the_range():
    """Infinities saturate, nothing at all has the smallest scale, the largest and smallest finite values keep theirs."""
    ops = _ops()
    k = torch.zeros(4, 1, 128, dtype=BF16)
    k[0, 0, 0], k[1, 0, 0], k[1, 0, 1], k[2, 0, 0] = 3.3e38, math.inf, 1.0, 1e-38
    v = torch.full((4, 1, 128), 448.0, dtype=BF16)
    v[:, :, 1] = -1.75 * 2 ** -3
    # 3.3e38 is 1.94 * 2^127, above 1.75 * 2^127 = 448 * 2^119
    for row, want in ((0, 2.0 ** 120), (1, 2.0 ** 120), (2, 2.0 ** -126), (3, 2.0 ** -126)):
        kc, vc = (torch.zeros(1, 16, 1, 128, dtype=E4M3).cuda() for _ in range(2))
        ks, vs = torch.zeros(1, 1).cuda(), torch.zeros(1, 1).cuda()
        one = torch.tensor([1], dtype=torch.int32).cuda()
        ops.kv_cache_append(k[row:row + 1].cuda(), v[row:row + 1].cuda(), kc, vc, torch.zeros(1, 1, dtype=torch.int32).cuda(), one,
                            torch.tensor([0, 1], dtype=torch.int32).cuda(), k_scale=ks, v_scale=vs)
        assert ks.item() == want and vs.item() == 1.0
        assert torch.equal(vc[0, 0, 0].float().cpu(), v[row, 0].float().to(E4M3).float())
        assert torch.isfinite(kc.float()).all()


# ---------------------------------------------------------------------------------------------------------- attention
def _attend_case(page, new, lens, heads, group, dtype, eight, causal, heads_first=True, seed=0, scale=None, spoil=None, **hints):
    gen = torch.Generator().manual_seed(seed + page + group)
    pages = sum(-(-max(n, 0) // page) for n in lens) + 2
    table = model.make_tables(gen, lens, page, pages)
    (kc, ks), (vc, vs) = (model.make_cache(gen, pages, page, heads, dtype, eight, heads_first) for _ in range(2))
    # what no sequence owns: not a number, wherever it is
    owned = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for at in range(-(-max(n, 0) // page)):
            owned[table[b, at], :n - at * page] = True
    for c in (kc, vc):
        raw = c.view(torch.uint8) if eight else c
        raw[~owned] = 0x7f if eight else math.nan
    if ks is not None:
        dead = ~owned.any(1)
        ks[dead], vs[dead] = math.nan, math.inf
    if spoil is not None:
        spoil(table, ks, vs)
    T, behind = sum(new), 2
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    q = (0.7 * torch.randn(T + behind, heads * group, 128, generator=gen)).to(dtype)
    ref = model.attend(q[:T], kc, vc, ks, vs, table, lens_t, cu, 128 ** -0.5 if scale is None else scale, causal)
    put = lambda c: c.transpose(1, 2).contiguous().cuda().transpose(1, 2) if heads_first else c.contiguous().cuda()  # noqa: E731
    out = torch.full(q.shape, 7.0, dtype=dtype).cuda()
    dev = dict(k_scale=None if ks is None else ks.cuda(), v_scale=None if vs is None else vs.cuda(), softmax_scale=scale, causal=causal)
    args = (q.cuda(), put(kc), put(vc), table.cuda(), lens_t.cuda(), cu.cuda())
    got, lse = _ops().attn_fwd_cache(*args, **dev, return_lse=True, out=out, **hints)
    assert got is out and (out[T:] == 7.0).all()  # rows behind the last sequence
    _attention_close(out[:T], lse[:, :T], ref, dtype, eight)
    plain, none = _ops().attn_fwd_cache(*args, **dev, **hints)
    assert none is None and torch.equal(plain[:T], out[:T])  # and the same again, bit for bit
    return args, dev, ref


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 8])
def test_attention_of_single_tokens(page, group, dtype, eight):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 513, 1000]
    _attend_case(page, [1] * len(lens), lens, 3, group, dtype, eight, True, max_q=1)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,new,lens,heads,group", [
    (16, [1, 0, 3, 0], [0, 5, 2, 0], 2, 4),        # no keys, no queries, more queries than keys
    (32, [2, 5, 1], [70, 333, 64], 2, 8),          # a few tokens each: rows of more than one tile of 16
    (64, [17, 1, 40], [17, 300, 129], 1, 3),       # a first prompt, a step and a chunk in one call
    (128, [130], [700], 2, 1),
    (64, [257, 3], [257, 900], 2, 2),
    (16, [1], [2500], 1, 16),
    (16, [2], [100], 1, 33),
    (64, [300], [64], 1, 4),                       # mostly queries that see nothing
])
def test_attention_of_chunks(page, new, lens, heads, group, causal, eight):
    _attend_case(page, new, lens, heads, group, BF16, eight, causal)
    _attend_case(page, new, lens, heads, group, FP16, eight, causal, heads_first=False, max_q=max(new), max_kv=max(lens + [1]))


@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 100000), (100000, 1), (100000, 100000)])
@pytest.mark.parametrize("eight", [True, False])
def test_hints_do_not_change_what_is_right(max_q, max_kv, eight):
    _attend_case(64, [1, 70, 1, 9], [300, 400, 20, 1300], 2, 4, BF16, eight, True, max_q=max_q, max_kv=max_kv)


@pytest.mark.parametrize("new", [[1, 1], [40, 200]])
@pytest.mark.parametrize("eight", [True, False])
def test_pages_that_do_not_exist_are_not_attended_to(new, eight):
    def spoil(table, ks, vs):
        table[0, 1], table[0, 3], table[1, 0] = -1, 10 ** 6, -2 ** 31

    _attend_case(32, new, [150, 90], 2, 4, BF16, eight, False, spoil=spoil)

    def none(table, ks, vs):
        table[:] = -1

    _attend_case(32, new, [150, 90], 2, 4, BF16, eight, True, spoil=none)


@pytest.mark.parametrize("new", [[1, 1, 1], [1, 150, 3]])
def test_scales_from_zero_to_the_largest(new):
    """Scales are not only the append's powers of two: any size, neighbours of very different ones, zeros."""
    def spoil(table, ks, vs):
        gen = torch.Generator().manual_seed(1)
        ks *= 0.5 + torch.rand(ks.shape, generator=gen)
        vs *= torch.exp2(-12 * torch.rand(vs.shape, generator=gen))
        ks[table[0, 0]], vs[table[1, 1]] = 0.0, 0.0

    _attend_case(16, new, [200, 500, 33], 2, 4, BF16, True, True, spoil=spoil)


@pytest.mark.parametrize("new,eight", [([1], True), ([1], False), ([33], True), ([33], False)])
def test_scores_far_apart(new, eight):
    """A scale that makes softmax pick single keys, and one that makes it an average."""
    for scale in (4.0, 1e-4):
        gen = torch.Generator().manual_seed(9)
        q = torch.randn(sum(new), 4, 128, generator=gen).to(BF16)
        kc, ks = model.make_cache(gen, 40, 16, 2, BF16, eight)
        vc, vs = model.make_cache(gen, 40, 16, 2, BF16, eight)
        table, lens = torch.randperm(40, generator=gen).int()[None], torch.tensor([600], dtype=torch.int32)
        cu = torch.tensor([0, sum(new)], dtype=torch.int32)
        want, want_lse, mag = model.attend(q, kc, vc, ks, vs, table, lens, cu, scale, False)
        out, lse = _ops().attn_fwd_cache(*[t.cuda() for t in (q, kc, vc, table, lens, cu)], k_scale=ks if ks is None else ks.cuda(),
                                         v_scale=vs if vs is None else vs.cuda(), softmax_scale=scale, return_lse=True)
        # scores up to 4 * 128 * 3: a sum of products of that size, and its factor, in fp32
        score = 128 * 2.0 ** -24 * max(1.0, scale * 128) * 2
        probability = 2.0 ** -11 if eight else 2.0 ** -8
        tol = 2.0 ** -8 * want.abs() + 1.01 * (probability + 2 * score) * mag + 1e-7
        assert ((out.double().cpu() - want).abs() <= tol).all()
        assert ((lse.double().cpu() - want_lse).abs() <= score + 1e-6 * want_lse.abs()).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 9]])
@pytest.mark.parametrize("eight", [True, False])
def test_a_query_that_is_not_a_number_and_lengths_below_zero(new, eight):
    """NaN in one query stays in its row; a negative length holds no keys, for neither operator."""
    lens, T = [200, -5, 77], sum(new)
    args, dev, ref = _attend_case(32, new, lens, 2, 4, BF16, eight, False)
    q = args[0].clone()
    q[0, 3, 7] = math.nan
    out, lse = _ops().attn_fwd_cache(q, *args[1:], **dev, return_lse=True)
    assert out[0, 3].isnan().all() and lse[3, 0].isnan()
    keep = torch.ones(T, 8, dtype=torch.bool)
    keep[0, 3] = False
    plain, plain_lse = _ops().attn_fwd_cache(*args, **dev, return_lse=True)
    assert torch.equal(out[:T].cpu()[keep], plain[:T].cpu()[keep]) and torch.equal(lse[:, :T].cpu()[keep.T], plain_lse[:, :T].cpu()[keep.T])
    k = torch.randn(T, 2, 128).to(BF16).cuda()
    caches = [args[1].clone(), args[2].clone()]
    scales = [None if s is None else s.clone() for s in (dev["k_scale"], dev["v_scale"])]
    for length in (0, -2 ** 31):
        _ops().kv_cache_append(k, k, *caches, args[3], torch.full((3,), length, dtype=torch.int32).cuda(), args[5], k_scale=scales[0], v_scale=scales[1])
    for got, was in zip(caches + scales, (args[1], args[2], dev["k_scale"], dev["v_scale"])):
        if was is not None:
            raw = torch.uint8 if got.element_size() == 1 else torch.int16 if got.element_size() == 2 else torch.int32
            assert torch.equal(got.contiguous().view(raw), was.contiguous().view(raw))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("new,lens,causal", [([1, 1], [70001, 33333], True), ([64], [20000], True), ([300, 5], [9000, 4000], False)])
def test_long_caches(new, lens, causal, eight):
    """Against fp64 on the GPU, page by page in the pool's own order."""
    ops = _ops()
    gen = torch.Generator(device="cuda").manual_seed(4)
    page, heads, group = 64, 2, 4
    pages = sum(-(-n // page) for n in lens)
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(pages, page, heads, 128, generator=gen, device="cuda")
        if eight:
            s = torch.exp2(torch.randint(-9, -6, (pages, heads), generator=gen, device="cuda").float())
            pools.append((x / s[:, None, :, None]).clamp(-448, 448).to(E4M3))
            scales.append(s)
        else:
            pools.append(x.to(BF16))
            scales.append(None)
    width = max(-(-n // page) for n in lens)
    order, table, at = torch.randperm(pages, generator=gen, device="cuda").int(), torch.zeros(len(lens), width, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(lens):
        table[b, :-(-n // page)] = order[at:at + -(-n // page)]
        at += -(-n // page)
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    q = torch.randn(sum(new), heads * group, 128, generator=gen, device="cuda").to(BF16)
    out, lse = ops.attn_fwd_cache(q, *pools, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu, k_scale=scales[0], v_scale=scales[1],
                                  causal=causal, return_lse=True)
    want, mag = torch.empty(2, *q.shape, dtype=torch.float64, device="cuda")
    want_lse = torch.empty(lse.shape, dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(zip(new, lens)):
        rows, ids = slice(int(cu[b]), int(cu[b]) + n), table[b, :-(-length // page)].long()
        for h in range(heads):
            k, v = (p[ids][:, :, h].double() * (1.0 if s is None else s[ids, h].double()[:, None, None]) for p, s in zip(pools, scales))
            k, v = k.reshape(-1, 128)[:length], v.reshape(-1, 128)[:length]
            for g in range(h * group, (h + 1) * group):
                s = q[rows, g].double() @ k.T * 128 ** -0.5
                if causal:
                    s = s.masked_fill(torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None], -math.inf)
                w = torch.softmax(s, -1)
                want[rows, g], mag[rows, g], want_lse[g, rows] = w @ v, w @ v.abs(), torch.logsumexp(s, -1)
    _attention_close(out, lse, (want.cpu(), want_lse.cpu(), mag.cpu()), BF16, eight)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes, its last page in use."""
    ops = _ops()
    pages, page, heads = 16500, 256, 8  # 4.3 GB of codes, keys and values one pool
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    pool = torch.zeros(pages, page, heads, 128, dtype=torch.uint8, device="cuda").view(E4M3)
    scale = torch.ones(pages, heads, device="cuda")
    gen = torch.Generator().manual_seed(2)
    kv, table = torch.randn(300, heads, 128, generator=gen).to(BF16), torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    lens, cu = torch.tensor([300], dtype=torch.int32), torch.tensor([0, 300], dtype=torch.int32)
    ops.kv_cache_append(kv.cuda(), kv.cuda(), pool, pool, table.cuda(), lens.cuda(), cu.cuda(), k_scale=scale, v_scale=scale)
    small, small_scale = torch.zeros(2, page, heads, 128, dtype=E4M3), torch.ones(2, heads)
    model.append(kv.float(), small, small_scale, torch.tensor([[1, 0]]), lens, cu)
    _equal(pool[pages - 2:], small)
    for n in (1, 40):
        q, cu = torch.randn(n, heads, 128, generator=gen).to(BF16), torch.tensor([0, n], dtype=torch.int32)
        ref = model.attend(q, small, small, small_scale, small_scale, torch.tensor([[1, 0]]), lens, cu, 128 ** -0.5, True)
        out, lse = ops.attn_fwd_cache(q.cuda(), pool, pool, table.cuda(), lens.cuda(), cu.cuda(), k_scale=scale, v_scale=scale, causal=True,
                                      return_lse=True)
        _attention_close(out, lse, ref, BF16, True)


# --------------------------------------------------------------------------------------------- streams, graphs, together
@pytest.mark.parametrize("new", [[1] * 6, [70, 1, 200]])
def test_two_streams_at_once(new):
    ops = _ops()
    lens = [700 + 13 * b for b in range(len(new))]
    (args, dev, ref), (args2, dev2, ref2) = (_attend_case(64, new, lens, 2, 4, BF16, True, True, seed=s) for s in (1, 2))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (a, d) in enumerate(((args, dev), (args2, dev2))):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.attn_fwd_cache(*a, **d)[0])
    torch.cuda.synchronize()
    T = sum(new)
    for got, r in zip(outs, (ref, ref2)):
        _attention_close(got[0][:T], None, r, BF16, True)
        for o in got[1:]:
            assert torch.equal(o[:T], got[0][:T])


@pytest.mark.parametrize("n", [1, 9])
def test_two_captured_graphs_and_eager_calls_between(n):
    """A captured step of n tokens is replayed with lengths that grow in place, beside another graph and eager calls of the
    same stream."""
    ops = _ops()
    gen = torch.Generator().manual_seed(8)
    heads, group, page, B = 2, 4, 16, 3
    table = torch.randperm(B * 8, generator=gen).int().view(B, 8)
    rope = model.rope_table(128, 200)
    cu = n * torch.arange(B + 1, dtype=torch.int32)
    dev_table, dev_cu, dev_rope = table.cuda(), cu.cuda(), rope.cuda()
    graphs = []
    for i in range(2):
        caches = [model.make_cache(gen, B * 8, page, heads, BF16, True) for _ in range(2)]
        lens = torch.tensor([20, 37, 64], dtype=torch.int32)
        s = dict(k=torch.zeros(B * n, heads, 128, dtype=BF16).cuda(), v=torch.zeros(B * n, heads, 128, dtype=BF16).cuda(),
                 q=torch.zeros(B * n, heads * group, 128, dtype=BF16).cuda(), lens=lens.cuda(), caches=caches,
                 dev=[(c.cuda(), sc.cuda()) for c, sc in caches], host_lens=lens)

        def step(s=s):
            s["lens"] += n
            (kc, ks), (vc, vs) = s["dev"]
            qr = ops.kv_cache_append(s["k"], s["v"], kc, vc, dev_table, s["lens"], dev_cu, k_scale=ks, v_scale=vs, rope_table=dev_rope, q=s["q"])
            return ops.attn_fwd_cache(qr, kc, vc, dev_table, s["lens"], dev_cu, k_scale=ks, v_scale=vs, causal=True, return_lse=True)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s["out"], s["lse"] = step()
        graphs.append((graph, s, step))
    for turn in range(6):
        for i, (graph, s, step) in enumerate(graphs):
            k, v = (torch.randn(B * n, heads, 128, generator=gen).to(BF16) for _ in range(2))
            q = torch.randn(B * n, heads * group, 128, generator=gen).to(BF16)
            for name, t in (("k", k), ("v", v), ("q", q)):
                s[name].copy_(t)
            if (turn + i) % 3 == 2:
                out, lse = step()
            else:
                graph.replay()
                out, lse = s["out"], s["lse"]
            s["host_lens"] = s["host_lens"] + n
            pos = (s["host_lens"].long()[:, None] + torch.arange(-n, 0)).flatten()
            for (c, sc), x in zip(s["caches"], (model.rotate(k, pos, rope, True), v.float())):
                model.append(x, c, sc, table, s["host_lens"], cu)
            for (c, sc), (gc, gs) in zip(s["caches"], s["dev"]):
                _equal(gc, c)
                _equal(gs, sc)
            (kc, ks), (vc, vs) = s["caches"]
            ref = model.attend(model.rotate(q, pos, rope, True).to(BF16), kc, vc, ks, vs, table, s["host_lens"], cu, 128 ** -0.5, True)
            _attention_close(out, lse, ref, BF16, True)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_prompt_chunks_and_steps_together(eight, dtype):
    """Sequences of differing lengths: a prompt, a second chunk, single tokens - each call appends, then attends."""
    ops = _ops()
    gen = torch.Generator().manual_seed(6)
    heads, group, page = 2, 4, 32
    rope = model.rope_table(64, 400)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 24, page, heads, dtype, eight) for _ in range(2))
    dev = [None if t is None else t.cuda() for t in (kc, vc, ks, vs)]
    table = torch.randperm(24, generator=gen).int().view(3, 8)
    lens = torch.zeros(3, dtype=torch.int32)
    for new in ([100, 7, 31], [33, 0, 2], [1, 1, 1], [1, 1, 0], [60, 1, 1]):
        T = sum(new)
        cu = torch.tensor([0, new[0], new[0] + new[1], T], dtype=torch.int32)
        lens = lens + torch.tensor(new, dtype=torch.int32)
        k, v, q = (torch.randn(T, h, 128, generator=gen).to(dtype) for h in (heads, heads, heads * group))
        pos = torch.cat([torch.arange(int(lens[b]) - n, int(lens[b])) for b, n in enumerate(new)])
        qr = ops.kv_cache_append(k.cuda(), v.cuda(), dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3],
                                 rope_table=rope.cuda(), interleaved=False, q=q.cuda())
        for x, c, s in ((model.rotate(k, pos, rope, False), kc, ks), (v.float(), vc, vs)):
            model.append(x, c, s, table, lens, cu)
        _equal(dev[0], kc)
        _equal(dev[1], vc)
        _equal(qr, model.rotate(q, pos, rope, False).to(dtype))
        out, lse = ops.attn_fwd_cache(qr, dev[0], dev[1], table.cuda(), lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3], causal=True,
                                      return_lse=True)
        ref = model.attend(qr.cpu(), kc, vc, ks, vs, table, lens, cu, 128 ** -0.5, True)
        _attention_close(out, lse, ref, dtype, eight)


def test_an_empty_call_and_a_table_wider_than_the_sequences():
    ops = _ops()
    gen = torch.Generator().manual_seed(7)
    (kc, ks), (vc, vs) = (model.make_cache(gen, 4, 16, 2, BF16, True) for _ in range(2))
    dev = [t.cuda() for t in (kc, vc, ks, vs)]
    z = torch.zeros(2, dtype=torch.int32).cuda()
    cu = torch.zeros(3, dtype=torch.int32).cuda()
    none = torch.zeros(0, 2, 128, dtype=BF16).cuda()
    ops.kv_cache_append(none, none, dev[0], dev[1], torch.zeros(2, 4, dtype=torch.int32).cuda(), z, cu, k_scale=dev[2], v_scale=dev[3])
    out, lse = ops.attn_fwd_cache(none, dev[0], dev[1], torch.zeros(2, 4, dtype=torch.int32).cuda(), z, cu, k_scale=dev[2], v_scale=dev[3],
                                  return_lse=True)
    assert out.shape == (0, 2, 128) and lse.shape == (2, 0)
    _equal(dev[0], kc)
    # a row of a wider table, lengths behind what it can hold
    wide = torch.full((2, 9), -1, dtype=torch.int32)
    wide[:, :2] = torch.tensor([[0, 1], [2, 3]])
    lens, cu = torch.tensor([25, 900], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    q = torch.randn(2, 4, 128, generator=gen).to(BF16)
    view = wide.cuda()[:, :2]
    ref = model.attend(q, kc, vc, ks, vs, wide[:, :2], lens, cu, 128 ** -0.5, False)
    out, lse = ops.attn_fwd_cache(q.cuda(), dev[0], dev[1], view, lens.cuda(), cu.cuda(), k_scale=dev[2], v_scale=dev[3], return_lse=True)
    _attention_close(out, lse, ref, BF16, True)


# ------------------------------------------------------------------------------------------------ the class and its users
def _held(cache, sequence):
    """fp64 keys and values [length, H, 128] that a PagedKVCache holds of a sequence."""
    t = {k: None if v is None else v.cpu() for k, v in cache.tensors.items()}
    n = cache.lens[sequence]
    return tuple(model.gathered(t[x + "_cache"], t[x + "_scale"], t["block_table"][sequence], n)[0] for x in "kv")


def _dense(q, k, v, causal_from=None):
    """fp64 attention of q [S, Hq, 128] over k, v [n, H, 128]: (out, lse [Hq, S], softmax |v|)."""
    group = q.shape[1] // k.shape[1]
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.double(), k) * 128 ** -0.5
    if causal_from is not None:
        s = s.masked_fill(torch.arange(k.shape[0]) > (causal_from + torch.arange(q.shape[0]))[:, None], -math.inf)
    w = torch.softmax(s, -1)
    return torch.einsum("hqk,khd->qhd", w, v), torch.logsumexp(s, -1), torch.einsum("hqk,khd->qhd", w, v.abs())


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_paged_cache_and_backend_frame_by_frame(dtype):
    """Frames of a clip one after the other, two samples, then single tokens of one of them: as the class is used."""
    from chitudiffusion_b200 import B200AttnBackend, PagedKVCache

    gen = torch.Generator().manual_seed(12)
    heads, group, frame = 2, 2, 90
    rope = model.rope_table(128, 400)
    cache = PagedKVCache(2, heads, 400, page_size=32, dtype=dtype, device="cuda")
    backend = B200AttnBackend("b200")
    for step in range(3):
        k, v = (torch.randn(2, frame, heads, 128, generator=gen).to(BF16) for _ in range(2))
        q = torch.randn(2, frame, heads * group, 128, generator=gen).to(BF16)
        turned = cache.append(k.cuda(), v.cuda(), q=q.cuda(), rope_table=rope.cuda())
        pos = torch.arange(step * frame, (step + 1) * frame).repeat(2)
        _equal(turned, model.rotate(q.flatten(0, 1), pos, rope, True).to(BF16).view(q.shape))
        out, lse, none = backend.attend_cache(turned, cache, return_attn_probs=True)
        assert none is None and out.shape == q.shape and lse.shape == (2, heads * group, frame)
        for b in range(2):
            want = _dense(turned[b].cpu(), *_held(cache, b))
            _attention_close(out[b], lse[b], want, BF16, dtype == E4M3)
    cache.truncate(1, 75)
    k, v = (torch.randn(3, heads, 128, generator=gen).to(BF16) for _ in range(2))
    q = torch.randn(3, heads * group, 128, generator=gen).to(BF16)
    cache.append(k.cuda(), v.cuda(), [0, 3])
    out, lse = cache.attend(q.cuda(), causal=True, return_lse=True)
    assert cache.lens == [270, 78]
    _attention_close(out, lse, _dense(q, *_held(cache, 1), causal_from=75), BF16, dtype == E4M3)
    with pytest.raises(NotImplementedError):
        B200AttnBackend("b200_q8").attend_cache(q.cuda(), cache)


def test_image_cache_of_other_ranks_in_8_bits(monkeypatch):
    """The cross-step K/V cache in 8-bit pages, one rank of two: fresh steps as without it, stale ones attend to the kept pages and to
    this rank's fresh shard.

    Tolerance: the two partial results are rounded to bf16 (2^-8 of softmax |v| at most), their probabilities too (2^-8),
    the merged result once more (2^-8 of itself); scores as everywhere."""
    from chitudiffusion_b200 import B200AttnBackend
    from chitudiffusion_b200.image_cp import B200ImageContextParallel

    for name, value in (("CHITU_CP_KV_CACHE", "1"), ("CHITU_CP_KV_CACHE_WARMUP", "0"), ("CHITU_CP_KV_CACHE_INTERVAL", "2"),
                        ("CHITU_CP_KV_CACHE_TAIL", "0"), ("CHITU_B200_KV_CACHE_FP8", "1")):
        monkeypatch.setenv(name, value)
    gen = torch.Generator().manual_seed(3)
    B, n, text, H = 2, 150, 20, 2

    def draw(rows):
        return torch.randn(B, rows, H, 128, generator=gen).to(BF16)

    class Group:
        group_size, rank_in_group = 2, 1

        def all_gather_sequence(self, t):
            return torch.cat([others.pop(0), t], 1)

    cp = B200ImageContextParallel(B200AttnBackend("b200"), mode="agkv")
    cp.enable(Group())
    far = None
    for step in range(4):
        cp.begin_forward(step, 100)
        others = [draw(n).cuda() for _ in range(2)]
        if step % 2 == 0:
            far = [t.cpu().double() for t in others]
        tq, tk, tv, iq, ik, iv = draw(text), draw(text), draw(text), draw(n), draw(n), draw(n)
        txt, img = cp.attention(*[t.cuda() for t in (tq, tk, tv, iq, ik, iv)])
        assert len(others) == (0 if step % 2 == 0 else 2)  # a stale step gathers nothing
        for b in range(B):
            keys = far
            if step % 2:  # the kept rows as their codes say
                cache = cp._kvcache[("cond", 0)]
                keys = [t[None].expand(B, -1, -1, -1) for t in _held(cache, b)]
                for exact, kept in zip(far, keys):
                    assert ((kept[b] - exact[b]).abs() <= 2 ** -4 * exact[b].abs() + 2 ** -9 * 2.0 ** -6).all()
            k, v = (torch.cat([far_rows[b], own[b].double(), t[b].double()]) for far_rows, own, t in zip(keys, (ik, iv), (tk, tv)))
            want, _, mag = _dense(torch.cat([iq[b], tq[b]]), k, v)
            got = torch.cat([img[b], txt[b]]).double().cpu()
            tol = 2 ** -8 * want.abs() + 1.02 * (2 ** -7 + 2 * SCORE) * mag + 1e-6
            assert ((got - want).abs() <= tol).all(), (step, ((got - want).abs() / tol).max().item())
