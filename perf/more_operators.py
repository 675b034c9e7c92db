"""An attention layer's step over images and long contexts: positions with several axes, and a cache held in 4 bits.

  rope    per-head RMSNorm of queries and keys and the partial split-half rotation, each pair's angle from one of the axes
          (time, height, width) of its token's position, in place (attn_qk_norm_mrope_rows)
  store   fresh keys and values quantized into a paged cache of 4-bit codes, and the touched pages read back as the values
          they stand for (kv4_store_rows, kv4_read_rows)
  attn    attention of the step's rows over that cache, single tokens and prompts, with the output gate (attn_kv4_rows)

Head layouts are the ones of the library's attention layer (16 query and 2 KV heads of 256, 64 rotary dims) and generic ones
beside it. The cache, per page and KV head, with tokens t and dims d (NG = dim / 64 groups of keys):

  k        uint8 [page, dim / 2]: a token's row is words of 8 dims; word (lk, g, h) = lk * 2 NG + 2 g + h, lk < 4, g < NG, h < 2,
           holds dims 64 g + 16 lk + 8 h + 0..7; of a word's dims, 2 i lies in nibble i and 2 i + 1 in nibble 4 + i
  v        uint8 [page / 8, dim, 4]: a word of 8 tokens of one dim, token 2 i in nibble i, token 2 i + 1 in nibble 4 + i
  k_scale  bfloat16 [page / 8, NG, 8], k_min bfloat16 [page, NG]; v_scale, v_min bfloat16 [page]

A value is min + scale * code. Of a group (keys: 64 dims of a token; values: a token's dims) min is its smallest value rounded
down to bfloat16, scale the smallest bfloat16 of at least (largest - min) / 15 and 2^-100, a code rne((x - min) / scale).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False
DEV = "cuda"
F32, F64, I32, BF16 = torch.float32, torch.float64, torch.int32, torch.bfloat16
FLOOR = 2.0 ** -100   # smallest scale
THETA, EPS = 1e7, 1e-6


def _ops():
    path = str(Path.cwd() / "qwen-3.5-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from qwen35_hip import ops
    return ops


# ---------------------------------------------------------------- which cases
# name of a head layout: query heads, KV heads, head dim, pairs of each axis
LAYOUTS = {"16/2x256": (16, 2, 256, (11, 11, 10)), "24/8x128": (24, 8, 128, (24, 20, 20)), "12/12x64": (12, 12, 64, (16, 8, 8))}


def _layout(name):
    q_heads, heads, dim, sections = LAYOUTS[name]
    return {"layout": name, "q_heads": q_heads, "heads": heads, "dim": dim}


def listed():
    main, wide = _layout("16/2x256"), _layout("24/8x128")
    return [
        # one token of a chat; a picture with a question; a video's chunk in a layout whose heads are rotated whole
        {"name": "rope_1", "kind": "rope", "rows": 1, "interleaved": True, **main},
        {"name": "rope_1333", "kind": "rope", "rows": 1333, "interleaved": True, **main},
        {"name": "rope_7000_wide", "kind": "rope", "rows": 7000, "interleaved": False, **wide},
        # one fresh token of each of 64 requests; a document's chunk behind a prefix that ends inside a page
        {"name": "store_64", "kind": "store", "requests": 64, "fresh": 1, "cached": 700, "page": 64, **main},
        {"name": "store_2100", "kind": "store", "requests": 1, "fresh": 2100, "cached": 333, "page": 64, **main},
        # a short question's next token; a chat late in a very long context; a batch of chats of ragged lengths in small
        # pages; the same in another head layout
        {"name": "attn_1x300", "kind": "attn", "requests": 1, "fresh": 1, "prompt": 0, "cached": 300, "page": 64, **main},
        {"name": "attn_1x200000", "kind": "attn", "requests": 1, "fresh": 1, "prompt": 0, "cached": 200000, "page": 64, **main},
        {"name": "attn_90x2500", "kind": "attn", "requests": 90, "fresh": 1, "prompt": 0, "cached": 2500, "page": 16, **main},
        {"name": "attn_40x6000_wide", "kind": "attn", "requests": 40, "fresh": 1, "prompt": 0, "cached": 6000, "page": 32,
         **wide},
        # a prompt's chunk among decoding requests; a picture's rows behind a long prefix; a long document in one step
        {"name": "attn_mixed_777", "kind": "attn", "requests": 20, "fresh": 1, "prompt": 777, "cached": 1500, "page": 64,
         **main},
        {"name": "attn_prompt_5000", "kind": "attn", "requests": 1, "fresh": 0, "prompt": 5000, "cached": 0, "page": 64,
         **main},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "store", "attn", "attn", "attn"])
    heads = _layout(rng.choice(["16/2x256", "16/2x256", "24/8x128", "12/12x64"]))
    if kind == "rope":
        return {"kind": kind, "rows": _log_int(rng, 1, 7000), "interleaved": rng.random() < 0.6, **heads}
    page = rng.choice([16, 32, 64, 64, 128])
    base = {"kind": kind, "page": page, **heads}
    if kind == "store":
        if rng.random() < 0.5:
            return {**base, "requests": _log_int(rng, 1, 200), "fresh": rng.randint(1, 3), "cached": _log_int(rng, 1, 900)}
        return {**base, "requests": rng.randint(1, 3), "fresh": _log_int(rng, 5, 700), "cached": _log_int(rng, 1, 900)}
    form = rng.choice(["long", "batch", "batch", "mixed", "prompt"])
    if form == "long":
        return {**base, "requests": rng.randint(1, 3), "fresh": rng.randint(1, 3), "prompt": 0,
                "cached": _log_int(rng, 100, 60000)}
    if form == "batch":
        return {**base, "requests": _log_int(rng, 4, 100), "fresh": 1, "prompt": 0, "cached": _log_int(rng, 30, 2500)}
    if form == "mixed":
        return {**base, "requests": rng.randint(2, 25), "fresh": 1, "prompt": _log_int(rng, 20, 900),
                "cached": _log_int(rng, 30, 2000)}
    return {**base, "requests": 1, "fresh": 0, "prompt": _log_int(rng, 20, 4500), "cached": rng.choice([0, 0, 401])}


# ---------------------------------------------------------------- inputs
class _Host:
    """Lengths and permutations on the host, from one seed."""

    def __init__(self, seed):
        self.h = torch.Generator()
        self.h.manual_seed(int(seed) * 1000003 + 7777)

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.h).tolist()

    def perm(self, n):
        return torch.randperm(n, generator=self.h).to(I32)


class _Rng:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 1000003 + 7777)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEV)


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(case, host):
    """(cached, fresh) of each request: ragged lengths that go by the case, in an order that goes by the seed."""
    n, fixed = case["requests"], _Host(0)
    cached = fixed.ints(case["cached"] // 3, case["cached"] + 1, n)   # from a third of the longest up
    cached[n // 2] = case["cached"]
    fresh = [case["fresh"]] * n
    if case.get("prompt"):
        fresh[n // 3] = case["prompt"]
    order = host.perm(n).tolist()
    return [cached[i] for i in order], [fresh[i] for i in order]


def _tables(host, lens, page):
    """Block table [requests, widest] of shuffled pages that hold `lens` tokens each, and the number of pages."""
    need = [_pages(t, page) for t in lens]
    ids = host.perm(sum(need) + 3)
    table = torch.zeros(len(lens), max(max(need), 1), dtype=I32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = ids[at:at + k]
        at += k
    return table, sum(need) + 3


def _i32(values):
    return torch.tensor(values, dtype=I32, device=DEV)


def _slots(table, lo, hi, page):
    """Slots of tokens lo[b] .. hi[b] - 1 of each request, on the host."""
    out = []
    for b, (a, e) in enumerate(zip(lo, hi)):
        t = torch.arange(a, e)
        out.append(table[b][t // page].long() * page + t % page)
    return torch.cat(out).to(I32)


def _positions(rows, host):
    """[3, rows]: a text's tokens, a picture's rows and columns behind it, text again; somewhere in a long context."""
    before = rows // 5
    start = host.ints(0, 40000, 1)[0]
    side = max(int(math.sqrt(rows * 0.7)), 1)
    t = torch.arange(rows)
    cell = (t - before).clamp(min=0)
    image = (t >= before) & (cell < side * side)
    after = t - side * side + side
    pos = torch.stack([torch.where(image, before + 0 * t, torch.where(t < before, t, after)),
                       torch.where(image, before + cell // side, torch.where(t < before, t, after)),
                       torch.where(image, before + cell % side, torch.where(t < before, t, after))])
    return (pos + start).to(I32).to(DEV)


def _spread(r, dim):
    """Sizes of a head's channels: within a factor of four, a few larger ones."""
    s = torch.exp2(2.0 * r.uniform(dim) - 1.0)
    return torch.where(r.uniform(dim) < 0.03, 4.0 * s, s)


# ---------------------------------------------------------------- codes and their layout
def _up_bf16(x):
    """The smallest bfloat16 that is at least x (float64, positive)."""
    y = x.to(F32)
    bits = y.view(I32)
    up = (((bits + 0xffff) >> 16) << 16).view(F32)
    return torch.where(up.double() < x, ((up.view(I32) >> 16) + 1 << 16).view(F32), up)


def _down_bf16(x):
    """The largest bfloat16 that is at most x (float32)."""
    bits = x.view(I32)
    toward_zero = bits & -65536
    return torch.where((x < 0) & (bits != toward_zero), toward_zero + 65536, toward_zero).view(F32)


def _quantize(x):
    """x [..., n] -> codes uint8 [..., n], scale and min float32 [...] of each group of n."""
    low = _down_bf16(x.amin(dim=-1))
    span = x.amax(dim=-1).double() - low.double()
    scale = _up_bf16((span / 15.0).clamp(min=FLOOR))
    codes = torch.round((x.double() - low.double()[..., None]) / scale.double()[..., None]).clamp(0, 15)
    return codes.to(torch.uint8), scale, low


def _pack_words(codes):
    """[..., 8] codes -> [..., 4] bytes: the even ones in nibbles 0..3, the odd ones in nibbles 4..7."""
    even, odd = codes[..., 0::2], codes[..., 1::2]
    return torch.cat([even[..., 0::2] | (even[..., 1::2] << 4), odd[..., 0::2] | (odd[..., 1::2] << 4)], dim=-1)


def _unpack_words(b):
    """[..., 4] bytes -> [..., 8] codes."""
    n = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)   # nibbles in order
    return torch.stack([n[..., :4], n[..., 4:]], dim=-1).flatten(-2)


def _pack_keys(codes):
    """[..., token, dim] -> [..., token, dim / 2]."""
    d = codes.shape[-1]
    w = _pack_words(codes.unflatten(-1, (d // 64, 4, 2, 8)))           # [..., g, lk, h, 4]
    return w.movedim(-4, -3).flatten(-4)


def _unpack_keys(k):
    d = 2 * k.shape[-1]
    w = k.unflatten(-1, (4, d // 64, 2, 4)).movedim(-4, -3)            # [..., g, lk, h, 4]
    return _unpack_words(w).flatten(-4)


def _pack_values(codes):
    """[..., token, dim] -> [..., token / 8, dim, 4]."""
    return _pack_words(codes.unflatten(-2, (codes.shape[-2] // 8, 8)).transpose(-1, -2))


def _unpack_values(v):
    return _unpack_words(v).transpose(-1, -2).flatten(-3, -2)


def _pack_cache(k, v):
    """Keys and values [pages, heads, page, dim] as a cache."""
    kc, ks, km = _quantize(k.unflatten(-1, (k.shape[-1] // 64, 64)))
    vc, vs, vm = _quantize(v)
    return {"k": _pack_keys(kc.flatten(-2)).contiguous(), "v": _pack_values(vc).contiguous(),
            "k_scale": ks.unflatten(2, (-1, 8)).transpose(-1, -2).to(BF16).contiguous(), "k_min": km.to(BF16).contiguous(),
            "v_scale": vs.to(BF16).contiguous(), "v_min": vm.to(BF16).contiguous()}


def _keys_of(s, ids):
    """Values of pages `ids`, float32 [pages, heads, page, dim]."""
    codes = _unpack_keys(s["k"][ids]).float()
    scale = s["k_scale"][ids].float().transpose(-1, -2).flatten(2, 3)                      # [pages, heads, page, group]
    codes = codes.unflatten(-1, (scale.shape[-1], 64))
    return (s["k_min"][ids].float()[..., None] + scale[..., None] * codes).flatten(-2)


def _values_of(s, ids):
    codes = _unpack_values(s["v"][ids]).float()
    return s["v_min"][ids].float()[..., None] + s["v_scale"][ids].float()[..., None] * codes


def _filled_cache(r, pages, heads, dim, page):
    """Normal keys and values, whose sizes vary from channel to channel and from token to token."""
    parts, step = [], max(1, (1 << 25) // (heads * dim * page))
    spread = _spread(r, dim)
    for at in range(0, pages, step):
        n = min(step, pages - at)
        size = 0.5 + r.uniform(n, heads, page, 1)
        parts.append(_pack_cache(spread * size * r.normal(n, heads, page, dim),
                                 (1.5 - 0.5 * size) * r.normal(n, heads, page, dim)))
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def prepare(case, seed):
    r, kind, host = _Rng(seed), case["kind"], _Host(seed)
    s = {k: v for k, v in case.items() if k != "name"}
    q_heads, heads, dim, s["sections"] = LAYOUTS[case["layout"]]
    if kind == "rope":
        rows = case["rows"]
        s["q"], s["k"] = r.normal(rows, q_heads, dim), 2.0 * r.normal(rows, heads, dim)
        s["qw"], s["kw"] = _spread(r, dim), _spread(r, dim)
        s["pos"] = _positions(rows, host)
        return s
    cached, fresh = _lengths(case, host)
    page = case["page"]
    total = [c + n for c, n in zip(cached, fresh)]
    rows = sum(fresh)
    table, pages = _tables(host, total, page)
    s.update(_filled_cache(r, pages, heads, dim, page), table=table.to(DEV), len=_i32(total),
             start=_i32([0] + torch.tensor(fresh).cumsum(0).tolist()))
    if kind == "store":
        s["slots"] = _slots(table, cached, total, page).to(DEV)
        s["read"] = _slots(table, [c // page * page for c in cached], total, page).to(DEV)
        s["new_k"] = _spread(r, dim) * r.normal(rows, heads, dim)
        s["new_v"] = r.normal(rows, heads, dim)
        return s
    s["q"] = r.normal(rows, q_heads, dim)
    s["gate"] = r.normal(rows, q_heads, dim)
    s["host_lens"] = list(zip(fresh, total))
    if own:
        need = _ops().attn_kv4_workspace_bytes(rows, len(fresh), q_heads, heads, dim)
        s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------- the plain forms
def _axis_of_pairs(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out, a = list(sections), [], 0
    while len(out) < sum(sections):
        if left[a % len(left)]:
            left[a % len(left)] -= 1
            out.append(a % len(left))
        a += 1
    return out


def _rope_plain(s):
    half = sum(s["sections"])
    axis = torch.tensor(_axis_of_pairs(s["sections"], s["interleaved"]), device=DEV)
    i = torch.arange(half, device=DEV, dtype=F64)
    angle = s["pos"].double()[axis].T * torch.exp(i * (-math.log(THETA) / half))       # [rows, half]
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x * (1.0 / torch.sqrt((x * x).mean(dim=2, keepdim=True) + EPS)) * w
        a, b = y[:, :, :half], y[:, :, half:2 * half]
        x.copy_(torch.cat([a * c - b * sn, b * c + a * sn, y[:, :, 2 * half:]], dim=2))
    return {"q": s["q"], "k": s["k"]}


def _store_plain(s):
    page = s["page"]
    slots = s["slots"].long()
    ids, where = torch.unique(slots // page, return_inverse=True)
    off = slots % page
    kc, ks, km = _quantize(s["new_k"].unflatten(-1, (s["dim"] // 64, 64)))
    vc, vs, vm = _quantize(s["new_v"])
    codes = _unpack_keys(s["k"][ids])
    codes[where, :, off] = kc.flatten(-2)
    s["k"][ids] = _pack_keys(codes)
    codes = _unpack_values(s["v"][ids])
    codes[where, :, off] = vc
    s["v"][ids] = _pack_values(codes)
    s["k_scale"][slots // page, :, off // 8, :, off % 8] = ks.to(BF16)
    s["k_min"][slots // page, :, off] = km.to(BF16)
    s["v_scale"][slots // page, :, off] = vs.to(BF16)
    s["v_min"][slots // page, :, off] = vm.to(BF16)
    ids, where = torch.unique(s["read"].long() // page, return_inverse=True)
    off = s["read"].long() % page
    return {"k": _keys_of(s, ids)[where, :, off], "v": _values_of(s, ids)[where, :, off]}


def _attn_plain(s):
    heads, dim, page, group = s["heads"], s["dim"], s["page"], s["q_heads"] // s["heads"]
    out = torch.empty_like(s["q"])
    at = 0
    for b, (n, total) in enumerate(s["host_lens"]):
        ids = s["table"][b, :_pages(total, page)].long()
        k = _keys_of(s, ids).transpose(0, 1).reshape(heads, -1, dim)[:, :total]
        v = _values_of(s, ids).transpose(0, 1).reshape(heads, -1, dim)[:, :total]
        q = s["q"][at:at + n].view(n, heads, group, dim).permute(1, 0, 2, 3).reshape(heads, n * group, dim)
        score = torch.bmm(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(dim))
        if n > 1:
            pos = torch.arange(total - n, total, device=DEV).repeat_interleave(group)
            score.masked_fill_(torch.arange(total, device=DEV) > pos[:, None], -math.inf)
        p = torch.exp(score - score.amax(dim=2, keepdim=True))
        o = torch.bmm(p, v.contiguous()) / p.sum(dim=2, keepdim=True)
        out[at:at + n] = o.view(heads, n, group, dim).permute(1, 0, 2, 3).reshape(n, heads * group, dim)
        at += n
    return out * (1.0 / (1.0 + torch.exp(-s["gate"])))


# ---------------------------------------------------------------- the framework's calls
def _run_own(s):
    ops, kind = _ops(), s["kind"]
    if kind == "rope":
        ops.attn_qk_norm_mrope_rows(s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["sections"],
                                    interleaved=s["interleaved"], theta=THETA, eps=EPS)
        return {"q": s["q"], "k": s["k"]}
    cache = ops.Kv4Cache(s["k"], s["v"], s["k_scale"], s["k_min"], s["v_scale"], s["v_min"])
    if kind == "store":
        ops.kv4_store_rows(s["new_k"], s["new_v"], s["slots"], cache)
        k, v = ops.kv4_read_rows(cache, s["read"])
        return {"k": k, "v": v}
    return ops.attn_kv4_rows(s["q"], cache, s["table"], s["start"], s["len"], gate=s["gate"], workspace=s["ws"])


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _rope_plain, "store": _store_plain, "attn": _attn_plain}[state["kind"]](state)


# ---------------------------------------------------------------- the work
def work(case):
    q_heads, heads, dim, sections = LAYOUTS[case["layout"]]
    if case["kind"] == "rope":   # each element read and written once, the positions and the weights read
        rows = case["rows"]
        return {"bytes": 8 * rows * (q_heads + heads) * dim + 12 * rows + 8 * dim,
                "flops": rows * (q_heads + heads) * (4 * dim + 6 * sum(sections))}
    cached, fresh = _lengths(case, _Host(1))
    rows, total, page = sum(fresh), sum(cached) + sum(fresh), case["page"]
    token = dim + 4 * (dim // 64) + 4   # bytes of a token's keys and values and what scales them
    if case["kind"] == "store":   # fresh rows read, their codes written; codes of the touched pages read, values written
        back = sum(c % page for c in cached) + rows
        return {"bytes": heads * (8 * dim * rows + token * rows + token * back + 8 * dim * back) + 4 * (rows + back),
                "flops": 8 * rows * heads * dim}
    keys = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, fresh))
    return {"bytes": token * heads * total + 12 * rows * q_heads * dim, "flops": 4 * q_heads * dim * keys}


# ---------------------------------------------------------------- 64-bit references
def _exact_rope(s):
    half, rows = sum(s["sections"]), s["pos"].shape[1]
    left, turn = dict(enumerate(s["sections"])), 0
    angle = torch.empty(rows, half, dtype=F64, device=DEV)
    for i in range(half):
        if s["interleaved"]:   # the axes take turns; one whose pairs are used up is passed over
            while not left[turn % 3]:
                turn += 1
            axis = turn % 3
            turn += 1
        else:
            axis = min(a for a in left if left[a])
        left[axis] -= 1
        angle[:, i] = s["pos"][axis].double() / math.pow(THETA, i / half)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        y = x * torch.rsqrt((x ** 2).sum(dim=2, keepdim=True) / s["dim"] + EPS) * s[name + "w"].double()
        z = torch.complex(y[:, :, :half].contiguous(), y[:, :, half:2 * half].contiguous()) * turn
        y[:, :, :half], y[:, :, half:2 * half] = z.real, z.imag
        out[name] = y
    return out



def _exact_key_rows(s, pid, off, h):
    """Keys of slots (pid, off) of one head, from the layout's formulas: float64 [slots, dim]."""
    dim, groups = s["dim"], s["dim"] // 64
    d = torch.arange(dim, device=DEV)
    word = (d % 64) // 16 * 2 * groups + 2 * (d // 64) + (d % 16) // 8
    nib = (d % 8) // 2 + 4 * (d % 2)
    byte = s["k"][pid, h, off][:, 4 * word + nib // 2].long()
    code = (byte >> (4 * (nib % 2))) & 15
    scale = s["k_scale"][pid, h, off // 8][torch.arange(pid.numel(), device=DEV), :, off % 8].double()
    low = s["k_min"][pid, h, off].double()
    return low[:, d // 64] + scale[:, d // 64] * code.double()


def _exact_value_rows(s, pid, off, h):
    j = off % 8
    nib = (j // 2 + 4 * (j % 2))
    word = s["v"][pid, h, off // 8]                                    # [slots, dim, 4]
    byte = word[torch.arange(pid.numel(), device=DEV), :, nib // 2].long()
    code = (byte >> (4 * (nib % 2))[:, None]) & 15
    return s["v_min"][pid, h, off].double()[:, None] + s["v_scale"][pid, h, off].double()[:, None] * code.double()


def _exact_attn(s):
    dim, page, group = s["dim"], s["page"], s["q_heads"] // s["heads"]
    out = torch.empty(s["q"].shape, dtype=F64, device=DEV)
    at = 0
    for b, (n, total) in enumerate(s["host_lens"]):
        t = torch.arange(total, device=DEV)
        pid, off = s["table"][b][t // page].long(), t % page
        hidden = t[None, :] > torch.arange(total - n, total, device=DEV)[:, None] if n > 1 else None
        for g in range(s["heads"]):
            k, v = _exact_key_rows(s, pid, off, g), _exact_value_rows(s, pid, off, g)
            for h in range(g * group, (g + 1) * group):
                score = s["q"][at:at + n, h].double() @ k.T / math.sqrt(dim)
                if hidden is not None:
                    score = score.masked_fill(hidden, -math.inf)
                out[at:at + n, h] = torch.softmax(score, dim=1) @ v
        at += n
    return out * torch.sigmoid(s["gate"].double())


def _exact_group(x):
    """The values that x [..., n] is held as, in 64 bits, from numbers and their neighbours."""
    lo, hi = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True).double()
    m = lo.to(BF16)
    m = torch.where(m.double() > lo.double(), torch.nextafter(m, torch.full_like(m, -math.inf)), m)
    want = (hi - m.double()) / 15.0
    sc = want.to(BF16)
    sc = torch.where(sc.double() < want, torch.nextafter(sc, torch.full_like(sc, math.inf)), sc)
    sc = torch.maximum(sc, torch.full_like(sc, FLOOR)).double()
    return m.double() + sc * torch.round((x.double() - m.double()) / sc).clamp(0, 15)


def _exact_store(s):
    page, rows = s["page"], {slot: i for i, slot in enumerate(s["slots"].tolist())}
    read = s["read"].tolist()
    pid, off = s["read"].long() // page, s["read"].long() % page
    k = torch.stack([_exact_key_rows(s, pid, off, h) for h in range(s["heads"])], dim=1)
    v = torch.stack([_exact_value_rows(s, pid, off, h) for h in range(s["heads"])], dim=1)
    fresh = [(i, rows[slot]) for i, slot in enumerate(read) if slot in rows]
    to, of = torch.tensor([i for i, _ in fresh], device=DEV), torch.tensor([j for _, j in fresh], device=DEV)
    k[to] = torch.cat([_exact_group(s["new_k"][of][:, :, g:g + 64]) for g in range(0, s["dim"], 64)], dim=2)
    v[to] = _exact_group(s["new_v"][of])
    return {"k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "attn": _exact_attn}[case["kind"]](s)
