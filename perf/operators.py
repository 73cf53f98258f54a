"""The operators of a paged key/value cache: rotary positions, appending, attention over what the cache holds.

``listed()`` gives the cases, ``draw()`` more of the same ranges, ``prepare`` / ``run`` one pass of a case - in plain torch
operations, or through the framework's entry points where ``own`` is true - and ``exact`` what it comes to in 64 bits.

A cache is a pool of pages of ``page`` tokens, ``[pages, page, heads, 128]``, a table of page numbers per sequence, and a length
per sequence that counts the tokens of the current call.  In 8 bits it holds e4m3 codes with one fp32 scale for each page and head.
Tokens of several sequences are packed one after the other, ``cu_seqlens`` says where each begins.
"""

from __future__ import annotations

import math

import torch

own = False

_E4M3_MAX = 448.0
_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # eight sequences in their generation loop, one token each: a launch and little else
        dict(name="rotary-step-8", op="rotary", tokens=8, heads_q=32, heads_kv=8, head_dim=128, rot=128, interleaved=False,
             dtype="bf16", table=32768, stretch=1.0),
        # part of a narrow head, a stretched table, an odd number of tokens
        dict(name="rotary-partial-4099", op="rotary", tokens=4099, heads_q=16, heads_kv=2, head_dim=80, rot=32, interleaved=True,
             dtype="fp16", table=131072, stretch=8.0),
        # the tokens of a whole 480p clip of 21 latent frames, 12 heads, adjacent pairs
        dict(name="rotary-clip-32760", op="rotary", tokens=32760, heads_q=12, heads_kv=12, head_dim=128, rot=128, interleaved=True,
             dtype="bf16", table=32768, stretch=1.0),
        # 64 sequences, one token each, into pages that are partly full
        dict(name="append-step-64", op="append", batch=64, new_lo=1, new_hi=1, old_lo=37, old_hi=2011, heads_q=32, heads_kv=8, rot=128,
             interleaved=False, dtype="bf16", cache="e4m3", page=64, heads_first=True, stretch=1.0),
        # prompts of differing lengths behind what each sequence already holds
        dict(name="append-prompts-8bit", op="append", batch=12, new_lo=61, new_hi=2603, old_lo=0, old_hi=1500, heads_q=32, heads_kv=8,
             rot=128, interleaved=False, dtype="bf16", cache="e4m3", page=64, heads_first=True, stretch=4.0),
        # three latent frames of a 480p clip, 12 heads, 16-bit pages with tokens outermost
        dict(name="append-frames-16bit", op="append", batch=1, new_lo=4680, new_hi=4680, old_lo=9360, old_hi=9360, heads_q=12, heads_kv=12,
             rot=128, interleaved=True, dtype="bf16", cache="16bit", page=128, heads_first=False, stretch=1.0),
        # one token of one short sequence: latency
        dict(name="attend-step-1", op="attend", batch=1, new_lo=1, new_hi=1, old_lo=1023, old_hi=1023, heads_q=32, heads_kv=8,
             causal=True, dtype="bf16", cache="e4m3", page=64, heads_first=True, lse=False),
        # 64 sequences of very different lengths, one token each
        dict(name="attend-step-64", op="attend", batch=64, new_lo=1, new_hi=1, old_lo=3, old_hi=16300, heads_q=32, heads_kv=8,
             causal=True, dtype="bf16", cache="e4m3", page=64, heads_first=True, lse=False),
        # two long documents in small pages, the log-sum-exp wanted for a merge
        dict(name="attend-step-long", op="attend", batch=2, new_lo=1, new_hi=1, old_lo=120011, old_hi=131070, heads_q=40, heads_kv=8,
             causal=True, dtype="fp16", cache="e4m3", page=16, heads_first=True, lse=True),
        # 16-bit pages, a key head for every query head
        dict(name="attend-step-16bit", op="attend", batch=16, new_lo=1, new_hi=1, old_lo=500, old_hi=8191, heads_q=16, heads_kv=16,
             causal=False, dtype="bf16", cache="16bit", page=32, heads_first=False, lse=False),
        # a prompt taken in chunks: 512 tokens each of four sequences behind what they hold
        dict(name="attend-chunks-causal", op="attend", batch=4, new_lo=389, new_hi=512, old_lo=700, old_hi=7600, heads_q=32, heads_kv=8,
             causal=True, dtype="bf16", cache="e4m3", page=64, heads_first=True, lse=False),
        # three latent frames of a 480p clip attend to all 21, 12 heads
        dict(name="attend-frames-32760", op="attend", batch=1, new_lo=4680, new_hi=4680, old_lo=28080, old_hi=28080, heads_q=12,
             heads_kv=12, causal=False, dtype="bf16", cache="e4m3", page=128, heads_first=True, lse=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads_kv = rng.choice([1, 2, 3, 4, 8, 10, 12])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
        heads = heads_kv * rng.choice([1, 2, 4])
        most = (32760 * 24 * 128) // ((heads + heads_kv) * head_dim)
        return dict(op=op, tokens=min(_log_int(rng, 1, 32760), most), heads_q=heads, heads_kv=heads_kv, head_dim=head_dim,
                    rot=rng.choice([r for r in (16, 32, 48, 64, 96, 128, 256) if r <= head_dim]), interleaved=rng.random() < 0.5,
                    dtype=dtype, table=rng.choice([4096, 32768, 131072]), stretch=rng.choice([1.0, 1.0, 4.0, 8.0]))
    page = rng.choice([16, 32, 64, 128, 256])
    cache = rng.choice(["e4m3", "e4m3", "16bit"])
    shared = dict(heads_kv=heads_kv, dtype=dtype, cache=cache, page=page, heads_first=rng.random() < 0.7)
    if op == "append":
        batch = _log_int(rng, 1, 64)
        heads_q = heads_kv * rng.choice([1, 2, 4])
        new_hi = _log_int(rng, 1, max(1, min(4680, 8_000_000 // (batch * (heads_q + 2 * heads_kv) * 128))))
        old_hi = _log_int(rng, 1, 4000)
        return dict(op=op, batch=batch, new_lo=rng.randint(1, new_hi), new_hi=new_hi, old_lo=rng.randint(0, old_hi), old_hi=old_hi,
                    heads_q=heads_q, rot=rng.choice([32, 64, 128, 128]), interleaved=rng.random() < 0.5,
                    stretch=rng.choice([1.0, 4.0]), **shared)
    batch = _log_int(rng, 1, 64)
    group = rng.choice([1, 2, 4, 5, 8])
    if rng.random() < 0.5:  # a token, or a few, each
        new_hi = rng.choice([1, 1, 1, 2, 3, 5])
        most = min(131070, 1_000_000_000 // (batch * heads_kv * (256 if cache == "e4m3" else 512)))
    else:  # chunks
        new_hi = _log_int(rng, 8, 2048)
        rows = 1_500_000_000 // (heads_kv * group * new_hi)  # keys of all sequences together
        batch = min(batch, 12, max(1, rows // (2 * new_hi)))
        most = min(32000, rows // batch - new_hi)
    old_hi = _log_int(rng, min(4, max(1, most)), max(4, most))
    return dict(op=op, batch=batch, new_lo=rng.randint(1, new_hi), new_hi=new_hi, old_lo=rng.randint(0, old_hi), old_hi=old_hi,
                heads_q=heads_kv * group, causal=rng.random() < 0.6, lse=rng.random() < 0.5, **shared)


def _ragged(batch, lo, hi, turn):
    """Lengths between lo and hi, both met, the same ones for the case whatever the seed."""
    if batch == 1:
        return [hi]
    return [hi if b == 0 else lo if b == 1 else lo + int((hi - lo + 1) * ((b * 0.6180339887498949 + turn) % 1.0)) for b in range(batch)]


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence."""
    new = _ragged(case["batch"], case["new_lo"], case["new_hi"], 0.11)
    old = _ragged(case["batch"], case["old_lo"], case["old_hi"], 0.53)
    return new, [n + o for n, o in zip(new, old)]


def _visible(case):
    """Key rows that the queries attend to, summed over queries."""
    new, lens = _lengths(case)
    if not case["causal"]:
        return sum(n * l for n, l in zip(new, lens))
    return sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(new, lens))


def work(case):
    es = 2
    if case["op"] == "rotary":
        n = case["tokens"] * (case["heads_q"] + case["heads_kv"])
        return {"bytes": 2 * es * n * case["head_dim"] + case["tokens"] * (8 + 4 * case["rot"]), "flops": 3 * n * case["rot"]}
    new, lens = _lengths(case)
    tokens, hq, hk = sum(new), case["heads_q"], case["heads_kv"]
    cs = 1 if case["cache"] == "e4m3" else es
    if case["op"] == "append":
        return {"bytes": 2 * tokens * hk * 128 * (es + cs) + 2 * tokens * hq * 128 * es + tokens * 4 * case["rot"],
                "flops": 3 * tokens * (hq + hk) * case["rot"]}
    scales = 8 * hk * sum(-(-l // case["page"]) for l in lens) if cs == 1 else 0
    out = tokens * hq * 128 * es + (4 * tokens * hq if case["lse"] else 0)
    return {"bytes": 2 * sum(lens) * hk * 128 * cs + scales + tokens * hq * 128 * es + out, "flops": 4 * 128 * hq * _visible(case)}


# ----------------------------------------------------------------------------------------------------------- inputs
def _angles(rot, stretch, rows, device):
    """Angles of positions 0 .. rows - 1 in 64 bits, positions divided by `stretch`."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    return torch.arange(rows, dtype=torch.float64, device=device)[:, None] / stretch * inv


def _table(rot, stretch, rows, device):
    a = _angles(rot, stretch, rows, device)
    return torch.stack([a.cos(), a.sin()], -1).float()


def _activations(gen, *shape, dtype):
    """Normal values whose channels differ in size, as projections give them."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x *= 0.5 + torch.rand(shape[-1], generator=gen, device="cuda")
    return x.to(dtype)


def _pool(case, gen, pages):
    """A cache pool with something everywhere, and its scales; `[pages, page, heads, 128]` in either order in memory."""
    hk, page = case["heads_kv"], case["page"]
    shape = (pages, hk, page, 128) if case["heads_first"] else (pages, page, hk, 128)
    if case["cache"] == "16bit":
        pool, scale = torch.empty(shape, dtype=_DTYPE[case["dtype"]], device="cuda").normal_(generator=gen), None
    else:
        scale = torch.exp2(torch.randint(-9, -6, (pages, hk), generator=gen, device="cuda").float())
        pool = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
        step = max(1, (1 << 27) // pool[0].numel())
        for at in range(0, pages, step):  # in pieces: the values are four times the codes
            some = torch.randn((min(step, pages - at),) + shape[1:], generator=gen, device="cuda")
            s = scale[at:at + step]
            some /= s[:, :, None, None] if case["heads_first"] else s[:, None, :, None]
            pool[at:at + step] = some.clamp_(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    return pool.transpose(1, 2) if case["heads_first"] else pool, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "rotary":
        t, d = case["tokens"], case["head_dim"]
        s["q"] = _activations(gen, t, case["heads_q"], d, dtype=dtype)
        s["k"] = _activations(gen, t, case["heads_kv"], d, dtype=dtype)
        first = torch.randint(0, max(1, case["table"] - t), (1,), generator=gen, device="cuda")
        s["positions"] = (first + torch.arange(t, device="cuda")).clamp_(max=case["table"] - 1).int()
        s["rope_table"] = _table(case["rot"], case["stretch"], case["table"], "cuda")
        return s
    new, lens = _lengths(case)
    page, tokens = case["page"], sum(new)
    width = max(-(-l // page) for l in lens)
    used = [-(-l // page) for l in lens]
    pages = sum(used) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    counts = torch.tensor(used, device="cuda")
    rank = torch.arange(width, device="cuda")[None, :]
    start = (counts.cumsum(0) - counts)[:, None]
    s["block_table"] = torch.where(rank < counts[:, None], order[(start + rank).clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cu_seqlens"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"] = max(new), max(lens)
    s["k_cache"], s["k_scale"] = _pool(case, gen, pages)
    s["v_cache"], s["v_scale"] = _pool(case, gen, pages)
    s["q"] = _activations(gen, tokens, case["heads_q"], 128, dtype=dtype)
    if case["op"] == "append":
        s["k"] = _activations(gen, tokens, case["heads_kv"], 128, dtype=dtype)
        s["v"] = _activations(gen, tokens, case["heads_kv"], 128, dtype=dtype)
        s["rope_table"] = _table(case["rot"], case["stretch"], max(lens), "cuda")
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, interleaved):
    """fp32 rotation of the first channels of `x [T, H, D]` by per-token factors `[T, rot / 2]`, each operation rounded by itself."""
    half = cos.shape[1]
    x, c, s = x.float(), cos[:, None, :], sin[:, None, :]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :half], head[..., half:])
    y = (a * c - b * s, a * s + b * c)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _plain_rotary(s):
    f = s["rope_table"][s["positions"].long()]
    inter = s["case"]["interleaved"]
    return {n: _rotate(s[n], f[..., 0], f[..., 1], inter).to(s[n].dtype) for n in ("q", "k")}


def _places(s):
    """Per packed token: its sequence and its position there."""
    cu, lens = s["cu_seqlens"].long(), s["kv_lens"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.bucketize(t, cu[1:], right=True)
    return seq, t - cu[seq] + lens[seq] - (cu[seq + 1] - cu[seq])


def _power_of_two_scale(amax):
    """The smallest power of two that brings `amax` to at most 448 (of nothing: the smallest normal one)."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.where(m > 0.875, e - 8, e - 9)).clamp(min=2.0 ** -126)


def _store_8bit(x, cache, scale, s, seq, pos):
    """Codes of `x` (fp32) into the pages, the pages' scales raised where that takes, their earlier codes brought to the new scale."""
    page, lens, cu = s["case"]["page"], s["kv_lens"].long(), s["cu_seqlens"].long()
    at = s["block_table"].long()[seq, pos // page]
    need = torch.zeros_like(scale).index_reduce_(0, at, x.abs().amax(-1), "amax")
    first = lens - (cu[1:] - cu[:-1])
    begun = s["block_table"].long().gather(1, (first // page).clamp(max=s["block_table"].shape[1] - 1)[:, None])[:, 0]
    held = (first % page > 0) & (cu[1:] > cu[:-1])  # sequences whose first page holds earlier tokens
    kept = torch.zeros_like(scale).index_add_(0, begun, scale[begun] * held[:, None])
    touched = torch.zeros_like(scale[:, 0]).index_fill_(0, at, 1.0)[:, None] > 0
    grown = torch.where(touched, torch.maximum(_power_of_two_scale(need), kept), scale)
    codes = cache[begun]
    old = torch.arange(page, device="cuda")[None, :] < (first % page)[:, None]
    again = (codes.float() * (scale / grown)[begun][:, None, :, None]).to(cache.dtype)
    raw = cache.view(torch.uint8)
    keep = (old & held[:, None])[:, :, None, None]
    raw[begun] = torch.where(keep, again.view(torch.uint8), codes.view(torch.uint8))
    raw[at, pos % page] = (x / grown[at][..., None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(cache.dtype).view(torch.uint8)
    scale.copy_(grown)


def _plain_append(s):
    seq, pos = _places(s)
    f = s["rope_table"][pos]
    inter, page = s["case"]["interleaved"], s["case"]["page"]
    q = _rotate(s["q"], f[..., 0], f[..., 1], inter).to(s["q"].dtype)
    k, v = _rotate(s["k"], f[..., 0], f[..., 1], inter), s["v"].float()
    if s["k_scale"] is None:
        at = s["block_table"].long()[seq, pos // page]
        s["k_cache"][at, pos % page] = k.to(s["k_cache"].dtype)
        s["v_cache"][at, pos % page] = v.to(s["v_cache"].dtype)
    else:
        _store_8bit(k, s["k_cache"], s["k_scale"], s, seq, pos)
        _store_8bit(v, s["v_cache"], s["v_scale"], s, seq, pos)
    return q


def _gathered(cache, scale, table):
    """`[B, heads, keys, 128]` fp32 of the pages of every sequence."""
    x = cache[table].float()
    if scale is not None:
        x *= scale[table][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


def _plain_attend(s):
    case, table = s["case"], s["block_table"].long()
    hk, group = case["heads_kv"], case["heads_q"] // case["heads_kv"]
    cu, lens = s["cu_seqlens"].long(), s["kv_lens"].long()
    n, rows, batch = s["q"].shape[0], s["max_q"], lens.shape[0]
    i = torch.arange(rows, device="cuda")
    there = (cu[:-1, None] + i).clamp(max=n - 1)
    q = s["q"].float()[there].view(batch, rows, hk, group, 128).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * rows, 128)
    scores = q @ _gathered(s["k_cache"], s["k_scale"], table).transpose(-1, -2)
    scores *= 128 ** -0.5
    j = torch.arange(scores.shape[-1], device="cuda")
    last = lens[:, None].expand(batch, rows)
    if case["causal"]:
        last = (lens - (cu[1:] - cu[:-1]))[:, None] + i + 1
    hidden = j >= torch.minimum(last, lens[:, None])[..., None]
    scores.view(batch, hk, group, rows, -1).masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    v = _gathered(s["v_cache"], s["v_scale"], table)
    out = scores @ v.masked_fill_((j >= lens[:, None])[:, None, :, None], 0.0) / total.clamp(min=1e-30)
    seq, _ = _places(s)
    t = torch.arange(n, device="cuda") - cu[seq]
    out = out.view(batch, hk, group, rows, 128)[seq, :, :, t].reshape(n, hk * group, 128).to(s["q"].dtype)
    if not case["lse"]:
        return out, None
    lse = (top + total.log()).view(batch, hk, group, rows)[seq, :, :, t].reshape(n, hk * group)
    return out, lse.t().contiguous()


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if own:
            from chitudiffusion_b200 import ops

            q, k = ops.rotary([state["q"], state["k"]], state["positions"], state["rope_table"], interleaved=case["interleaved"])
            return {"q": q, "k": k}
        return _plain_rotary(state)
    cache = (state["k_cache"], state["v_cache"], state["block_table"], state["kv_lens"], state["cu_seqlens"])
    if case["op"] == "append":
        if own:
            from chitudiffusion_b200 import ops

            q = ops.kv_cache_append(state["k"], state["v"], *cache, k_scale=state["k_scale"], v_scale=state["v_scale"],
                                    rope_table=state["rope_table"], interleaved=case["interleaved"], q=state["q"], max_new=state["max_q"])
        else:
            q = _plain_append(state)
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    if own:
        from chitudiffusion_b200 import ops

        out, lse = ops.attn_fwd_cache(state["q"], *cache, k_scale=state["k_scale"], v_scale=state["v_scale"], causal=case["causal"],
                                      return_lse=case["lse"], max_q=state["max_q"], max_kv=state["max_kv"])
    else:
        out, lse = _plain_attend(state)
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------------------ 64 bits, by definition
def _turn(x, angle, interleaved):
    """Rotation of `x [..., H, D]` as multiplication by e^{i angle}, in 64 bits."""
    half = angle.shape[-1]
    x = x.double()
    y = x.clone()
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous())
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous())
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    if interleaved:
        y[..., :2 * half] = torch.view_as_real(z).flatten(-2)
    else:
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _to_e4m3(x):
    """The nearest e4m3 value of each `x` (64 bits, at most 448 in size), ties to the even one."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_append(s):
    case, page = s["case"], s["case"]["page"]
    new, lens = _lengths(case)
    table = s["block_table"].tolist()
    held = {n: s[n].double() for n in ("k_cache", "v_cache")}
    scales = {n: None if s[n] is None else s[n].double() for n in ("k_scale", "v_scale")}
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    angle = _angles(case["rot"], case["stretch"], max(lens), "cuda")
    t = 0
    for b, n in enumerate(new):
        first = lens[b] - n
        mine = slice(t, t + n)
        t += n
        q[mine] = _turn(s["q"][mine], angle[first:lens[b]], case["interleaved"])
        rows = {"k": _turn(s["k"][mine], angle[first:lens[b]], case["interleaved"]), "v": s["v"][mine].double()}
        for p in range(first // page, -(-lens[b] // page)):
            lo, hi = max(first, p * page), min(lens[b], (p + 1) * page)
            for name, x in rows.items():
                part, cache = x[lo - first:hi - first], held[name + "_cache"][table[b][p]]
                if case["cache"] == "e4m3":
                    scale = scales[name + "_scale"][table[b][p]]
                    big = torch.exp2(torch.ceil(torch.log2(part.abs().amax((0, 2)) / _E4M3_MAX)))
                    if lo > p * page:
                        big = torch.maximum(big, scale)
                        cache[:lo - p * page] = _to_e4m3(cache[:lo - p * page] * (scale / big)[:, None])
                    scale.copy_(big)
                    part = _to_e4m3(part / big[:, None])
                cache[lo - p * page:hi - p * page] = part
    return {"q": q, **held, **scales}


def _exact_attend(s):
    case = s["case"]
    new, lens = _lengths(case)
    hk, group, page = case["heads_kv"], case["heads_q"] // case["heads_kv"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(case["heads_q"], s["q"].shape[0], dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, l) in enumerate(zip(new, lens)):
        pages = s["block_table"][b, :-(-l // page)].long()
        for h in range(hk):
            kv = []
            for name in ("k", "v"):
                x = s[name + "_cache"][pages][:, :, h].double()
                if case["cache"] == "e4m3":
                    x = x * s[name + "_scale"][pages, h].double()[:, None, None]
                kv.append(x.reshape(-1, 128)[:l])
            for g in range(h * group, (h + 1) * group):
                score = s["q"][t:t + n, g].double() @ kv[0].T / math.sqrt(128.0)
                if case["causal"]:
                    score = score.masked_fill(torch.arange(l, device="cuda") > torch.arange(l - n, l, device="cuda")[:, None], -math.inf)
                lse[g, t:t + n] = torch.logsumexp(score, -1)
                out[t:t + n, g] = torch.softmax(score, -1) @ kv[1]
        t += n
    return {"out": out, "lse": lse if case["lse"] else None}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        angle = _angles(case["rot"], case["stretch"], case["table"], "cuda")[s["positions"].long()]
        return {n: _turn(s[n], angle, case["interleaved"]) for n in ("q", "k")}
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
