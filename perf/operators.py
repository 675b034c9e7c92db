"""The batch operators whose speed counts: one step of several requests through an attention and a MoE layer.

  plan    block tables and slots of a step, from the requests' lengths (kv8_plan)
  store   fresh keys and values into a paged cache of 8-bit codes with a scale per page and head, and the touched pages
          read back as the values they stand for (kv8_store_rows, kv8_read_rows)
  attn    attention of the step's rows over that cache, with the output gate (attn_kv8_rows)
  moe     the routed experts of the step's tokens: (token, pick) pairs grouped by expert, gate and up products with
          SwiGLU, down products, weighted sum (moe_group_rows, moe_experts_rows)

Head layouts, widths and expert counts are the ones of the library's layer classes (16 query and 2 KV heads of 256; 256
experts, 8 picked, 512 wide, model width 2048) and generic ones beside them. The cache: codes int8, keys
[page, head, token, dim], values [page, head, token / 8, dim, 8], scales float32 [page, head].
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False
DEV = "cuda"
F32, F64, I32 = torch.float32, torch.float64, torch.int32
BLOCK = {"Q4_K": 144, "Q6_K": 210}
FLOOR = 2.0 ** -100   # smallest scale of a page


def _ops():
    path = str(Path.cwd() / "qwen-3.5-cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from qwen35_hip import ops
    return ops


# ---------------------------------------------------------------- which cases
def listed():
    return [
        # a small server's decode step, and a large one's with prompts joining: the step's page bookkeeping
        {"name": "plan_8", "kind": "plan", "requests": 8, "longest": 900, "prompts": 0, "page": 64},
        {"name": "plan_500", "kind": "plan", "requests": 500, "longest": 9000, "prompts": 20, "page": 64},
        # one fresh token of each of 64 requests; a document's chunk
        {"name": "store_64", "kind": "store", "requests": 64, "fresh": 1, "cached": 700, "heads": 2, "dim": 256,
         "page": 64},
        {"name": "store_2100", "kind": "store", "requests": 1, "fresh": 2100, "cached": 333, "heads": 2, "dim": 256,
         "page": 64},
        # one chat late in a long context; a batch of chats of ragged lengths, small pages; a prompt's chunk behind a
        # cached prefix; a long document in one step
        {"name": "attn_1x30000", "kind": "attn", "requests": 1, "fresh": 1, "prompt": 0, "cached": 30000, "q_heads": 16,
         "heads": 2, "dim": 256, "page": 64},
        {"name": "attn_90x2500", "kind": "attn", "requests": 90, "fresh": 1, "prompt": 0, "cached": 2500, "q_heads": 16,
         "heads": 2, "dim": 256, "page": 16},
        {"name": "attn_mixed_777", "kind": "attn", "requests": 20, "fresh": 1, "prompt": 777, "cached": 1500,
         "q_heads": 16, "heads": 2, "dim": 256, "page": 64},
        {"name": "attn_prompt_5000", "kind": "attn", "requests": 1, "fresh": 0, "prompt": 5000, "cached": 0,
         "q_heads": 16, "heads": 2, "dim": 256, "page": 64},
        # the experts of a few decoding requests, a question, a page with Q6_K weights, a document
        {"name": "moe_5", "kind": "moe", "rows": 5, "experts": 256, "top": 8, "inter": 512, "width": 2048,
         "wtype": "Q4_K"},
        {"name": "moe_77", "kind": "moe", "rows": 77, "experts": 256, "top": 8, "inter": 512, "width": 2048,
         "wtype": "Q4_K"},
        {"name": "moe_777_q6", "kind": "moe", "rows": 777, "experts": 256, "top": 8, "inter": 512, "width": 2048,
         "wtype": "Q6_K"},
        {"name": "moe_4096", "kind": "moe", "rows": 4096, "experts": 256, "top": 8, "inter": 512, "width": 2048,
         "wtype": "Q4_K"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attn", "attn", "attn", "moe", "moe"])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "plan":
        n = _log_int(rng, 1, 500)
        return {"kind": kind, "requests": n, "longest": _log_int(rng, 20, 9000), "prompts": rng.randint(0, 1 + n // 25),
                "page": page}
    q_heads, heads, dim = rng.choice([(16, 2, 256), (16, 2, 256), (16, 4, 128), (24, 8, 128), (12, 12, 64)])
    if kind == "store":
        if rng.random() < 0.5:
            return {"kind": kind, "requests": _log_int(rng, 1, 200), "fresh": rng.randint(1, 3),
                    "cached": _log_int(rng, 1, 900), "heads": heads, "dim": dim, "page": page}
        return {"kind": kind, "requests": rng.randint(1, 3), "fresh": _log_int(rng, 5, 700),
                "cached": _log_int(rng, 1, 900), "heads": heads, "dim": dim, "page": page}
    if kind == "attn":
        form = rng.choice(["long", "batch", "batch", "mixed", "prompt"])
        base = {"kind": kind, "q_heads": q_heads, "heads": heads, "dim": dim, "page": page}
        if form == "long":
            return {**base, "requests": rng.randint(1, 3), "fresh": rng.randint(1, 3), "prompt": 0,
                    "cached": _log_int(rng, 100, 30000)}
        if form == "batch":
            return {**base, "requests": _log_int(rng, 4, 100), "fresh": 1, "prompt": 0, "cached": _log_int(rng, 30, 2500)}
        if form == "mixed":
            return {**base, "requests": rng.randint(2, 25), "fresh": 1, "prompt": _log_int(rng, 20, 900),
                    "cached": _log_int(rng, 30, 2000)}
        return {**base, "requests": 1, "fresh": 0, "prompt": _log_int(rng, 20, 4500), "cached": rng.choice([0, 0, 401])}
    return {"kind": kind, "rows": _log_int(rng, 1, 4000), "experts": rng.choice([256, 256, 60]), "top": rng.choice([8, 8, 4]),
            "inter": 512, "width": 2048, "wtype": rng.choice(["Q4_K", "Q4_K", "Q6_K"])}


# ---------------------------------------------------------------- inputs
class _Host:
    """Lengths and permutations on the host, from one seed."""

    def __init__(self, seed):
        self.h = torch.Generator()
        self.h.manual_seed(int(seed) * 1000003 + 54321)

    def ints(self, lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=self.h).tolist()

    def perm(self, n):
        return torch.randperm(n, generator=self.h).to(I32)


class _Rng:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 1000003 + 54321)

    def normal(self, *shape, sigma=1.0):
        return sigma * torch.randn(shape, generator=self.g, device=DEV)

    def ints(self, lo, hi, *shape, dtype=I32):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=dtype)

    def weight(self, wtype, n):
        """n elements of a quantized tensor as a file holds it, values spread around zero by about 0.02."""
        nb = n // 256
        b = self.ints(0, 256, nb, BLOCK[wtype], dtype=torch.uint8)
        spread = 0.7 + 0.6 * torch.rand((nb,), generator=self.g, device=DEV)
        if wtype == "Q6_K":   # (d sc) (q - 32), scales of either sign
            b[:, 192:208] = (self.ints(32, 128, nb, 16) * (1 - 2 * self.ints(0, 2, nb, 16))).to(torch.int8).view(torch.uint8)
            b[:, 208:210] = (spread * (0.02 / 1530.0)).to(torch.float16).view(torch.uint8).view(nb, 2)
            return b.view(-1)
        # (d sc) q - dmin m with m near sc and dmin = 7.5 d: the middle of 0..15 is near zero
        sc = self.ints(24, 64, nb, 8, dtype=torch.uint8)
        mn = (sc.to(torch.int16) + self.ints(-4, 5, nb, 8, dtype=torch.int16)).clamp_(0, 63).to(torch.uint8)
        b[:, 4:8] = sc[:, :4] | ((sc[:, 4:] >> 4) << 6)
        b[:, 8:12] = mn[:, :4] | ((mn[:, 4:] >> 4) << 6)
        b[:, 12:16] = (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)
        d = spread * (0.02 / 209.0)
        b[:, 0:2] = d.to(torch.float16).view(torch.uint8).view(nb, 2)
        b[:, 2:4] = (7.5 * d).to(torch.float16).view(torch.uint8).view(nb, 2)
        return b.view(-1)


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(case, host):
    """(cached, fresh) of each request: ragged lengths that go by the case, in an order that goes by the seed."""
    n, fixed = case["requests"], _Host(0)
    if case["kind"] == "plan":
        cached = fixed.ints(0, case["longest"] + 1, n)
        fresh = [1] * n
        for i in fixed.ints(0, n, case["prompts"]):
            fresh[i] = 1 + fixed.ints(0, 512, 1)[0]
    else:   # from a third of the longest up
        cached = fixed.ints(case["cached"] // 3, case["cached"] + 1, n)
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


def _filled_cache(r, pages, heads, dim, page):
    """A cache of quantized normal keys and values, whose sizes vary from page to page."""
    def codes(shape, amax_dims):
        x = torch.randn(shape, generator=r.g, device=DEV)
        x *= 0.5 + torch.rand((shape[0], shape[1]) + (1,) * (len(shape) - 2), generator=r.g, device=DEV)
        s = x.abs().amax(dim=amax_dims) / 127.0
        x /= s.view(shape[0], shape[1], *([1] * (len(shape) - 2)))
        return x.round_().to(torch.int8), s
    k, ks = codes((pages, heads, page, dim), (2, 3))
    v, vs = codes((pages, heads, page // 8, dim, 8), (2, 3, 4))
    return {"k": k, "v": v, "ks": ks, "vs": vs}


def prepare(case, seed):
    r, kind = _Rng(seed), case["kind"]
    s = {"kind": kind, **{k: v for k, v in case.items() if k != "name"}}
    if kind == "moe":
        rows, e, top, inter, width = (case[k] for k in ("rows", "experts", "top", "inter", "width"))
        s["x"] = r.normal(rows, width)
        logits = r.normal(rows, e) + 0.5 * r.normal(e)   # some experts are picked more often
        w, idx = torch.topk(logits, top, dim=1)
        s["idx"], s["w"] = idx.to(I32).contiguous(), torch.softmax(w, dim=1).contiguous()
        for name in ("gate", "up", "down"):
            s[name] = r.weight(case["wtype"], e * inter * width)
        if own:
            need = _ops().moe_experts_rows_workspace_bytes(rows, top, e, width, inter)
            s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        return s
    host = _Host(seed)
    cached, fresh = _lengths(case, host)
    page = case["page"]
    total = [c + n for c, n in zip(cached, fresh)]
    rows = sum(fresh)
    if kind == "plan":
        table, _ = _tables(host, cached, page)
        wide = torch.zeros(len(cached), _pages(case["longest"] + 512, page), dtype=I32)
        wide[:, :table.shape[1]] = table
        s.update(rows=rows + 7, table=wide.to(DEV), cached=_i32(cached), fresh=_i32(fresh),   # a padded batch
                 free=(host.perm(6000) + 100000).to(DEV), head=_i32([17]))
        return s
    table, pages = _tables(host, total, page)
    s.update(_filled_cache(r, pages, case["heads"], case["dim"], page), table=table.to(DEV),
             start=_i32([0] + torch.tensor(fresh).cumsum(0).tolist()), len=_i32(total), rows=rows)
    if kind == "store":
        s["slots"] = _slots(table, cached, total, page).to(DEV)
        s["read"] = _slots(table, [c // page * page for c in cached], total, page).to(DEV)
        s["new_k"] = r.normal(rows, case["heads"], case["dim"], sigma=1.2)
        s["new_v"] = r.normal(rows, case["heads"], case["dim"], sigma=1.2)
        return s
    s["q"] = r.normal(rows, case["q_heads"], case["dim"])
    s["gate"] = r.normal(rows, case["q_heads"], case["dim"])
    s["host_lens"] = list(zip(fresh, total))
    if own:
        need = _ops().attn_kv8_workspace_bytes(rows, len(fresh), case["q_heads"], case["heads"], case["dim"])
        s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------- the plain forms
def _plan_plain(s):
    page, table, head = s["page"], s["table"], s["head"]
    c, n = s["cached"].long(), s["fresh"].long()
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), n.cumsum(0)])
    first = (c + page - 1) // page
    room = (c + n <= page * table.shape[1]) & (start[1:] <= s["rows"])
    need = torch.where((n > 0) & room, (c + n + page - 1) // page - first, torch.zeros_like(n))
    upto = need.cumsum(0)
    fits = room & ((need == 0) | (upto <= s["free"].numel() - head))
    j = torch.arange(table.shape[1], device=DEV)
    fresh_page = fits[:, None] & (j >= first[:, None]) & (j < (first + need)[:, None])
    take = (head + (upto - need)[:, None] + j - first[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh_page, s["free"][take], table))
    row = torch.arange(s["rows"], device=DEV)
    b = (torch.searchsorted(start, row, right=True) - 1).clamp(0, c.numel() - 1)
    real = row < start[-1]
    pos = torch.where(real, c[b] + row - start[b], torch.zeros_like(row))
    slot = table[b, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    slot = torch.where(real & fits[b], slot, torch.full_like(slot, -1))
    kv_len = torch.where(fits, c + n, torch.zeros_like(c))
    used = head + torch.where(fits & (need > 0), upto, torch.zeros_like(upto)).amax()
    return {"table": table, "start": start.to(I32), "len": kv_len.to(I32), "slots": slot.to(I32), "pos": pos.to(I32),
            "head": used.to(I32)}


def _store_one(codes, scales, x, slots, page):
    """codes [pages, heads, page, dim] and scales updated with rows x [rows, heads, dim] at `slots`."""
    slots = slots.long()
    pid, off = slots // page, slots % page
    touched, inv = torch.unique(pid, return_inverse=True)
    heads = x.shape[1]
    amax = torch.zeros(touched.numel(), heads, device=DEV)
    amax.scatter_reduce_(0, inv[:, None].expand(-1, heads), x.abs().amax(dim=2), "amax")
    first = torch.full((touched.numel(),), page, dtype=torch.int64, device=DEV).scatter_reduce_(0, inv, off, "amin")
    old = torch.where((first == 0)[:, None], torch.zeros((), device=DEV), scales[touched])
    new = torch.maximum(torch.maximum(old, (amax.double() / 127.0).float()), torch.full((), FLOOR, device=DEV))
    ratio = (old.double() / new.double()).float().double()
    kept = torch.round(codes[touched].double() * ratio[:, :, None, None])
    codes[touched] = kept.to(torch.int8)
    scales[touched] = new
    codes[pid, :, off] = torch.round(x.double() / new[inv].double()[:, :, None]).clamp(-127, 127).to(torch.int8)


def _values_by_token(v):
    """[page, head, token / 8, dim, 8] -> [page, head, token, dim]."""
    return v.transpose(3, 4).reshape(v.shape[0], v.shape[1], v.shape[2] * 8, v.shape[3])


def _store_plain(s):
    page = s["page"]
    v = _values_by_token(s["v"]).clone(memory_format=torch.contiguous_format)
    _store_one(s["k"], s["ks"], s["new_k"], s["slots"], page)
    _store_one(v, s["vs"], s["new_v"], s["slots"], page)
    s["v"].copy_(v.view(v.shape[0], v.shape[1], page // 8, 8, v.shape[3]).transpose(3, 4))
    pid, off = s["read"].long() // page, s["read"].long() % page
    return {"k": s["k"][pid, :, off].float() * s["ks"][pid][:, :, None],
            "v": v[pid, :, off].float() * s["vs"][pid][:, :, None], "k_scale": s["ks"], "v_scale": s["vs"]}


def _attn_plain(s):
    heads, dim, page, group = s["heads"], s["dim"], s["page"], s["q_heads"] // s["heads"]
    out = torch.empty_like(s["q"])
    at = 0
    for b, (n, total) in enumerate(s["host_lens"]):
        ids = s["table"][b, :_pages(total, page)].long()
        k = (s["k"][ids].float() * s["ks"][ids][:, :, None, None]).transpose(0, 1).reshape(heads, -1, dim)[:, :total]
        v = _values_by_token(s["v"][ids]).float() * s["vs"][ids][:, :, None, None]
        v = v.transpose(0, 1).reshape(heads, -1, dim)[:, :total]
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


def _half(b, dt):
    return b.contiguous().view(torch.float16).to(dt)


def _dequant(raw, wtype, dt):
    """Blocks (uint8 [n, block bytes]) -> [n, 256] values."""
    n = raw.shape[0]
    if wtype == "Q4_K":
        d, dmin = _half(raw[:, 0:2], dt), _half(raw[:, 2:4], dt)
        a, m, t = raw[:, 4:8], raw[:, 8:12], raw[:, 12:16]
        sc = torch.cat([a & 63, (t & 15) | ((a >> 6) << 4)], 1)
        mn = torch.cat([m & 63, (t >> 4) | ((m >> 6) << 4)], 1)
        q = raw[:, 16:].view(n, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 2).view(n, 8, 32)
        return ((d * sc.to(dt))[:, :, None] * q.to(dt) - (dmin * mn.to(dt))[:, :, None]).view(n, 256)
    ql, qh = raw[:, :128].view(n, 2, 2, 32), raw[:, 128:192].view(n, 2, 1, 32)
    low = torch.cat([ql & 15, ql >> 4], 2)                                        # [n, half, quarter, 32]
    high = torch.cat([(qh >> (2 * i)) & 3 for i in range(4)], 2)
    q = (low | (high << 4)).to(dt) - 32.0
    sc = _half(raw[:, 208:210], dt) * raw[:, 192:208].contiguous().view(torch.int8).to(dt)   # [n, half x quarter x 2]
    return (sc[:, :, None] * q.reshape(n, 16, 16)).view(n, 256)


def _expert(raw, wtype, e, m, k, dt):
    nb = m * k // 256
    return _dequant(raw.view(-1, BLOCK[wtype])[e * nb:(e + 1) * nb], wtype, dt).view(m, k)


def _moe_plain(s):
    e, top, inter, width, wt = s["experts"], s["top"], s["inter"], s["width"], s["wtype"]
    pairs = s["idx"].view(-1)
    order = torch.sort(pairs, stable=True).indices
    starts = torch.searchsorted(pairs[order].contiguous(), torch.arange(e + 1, device=DEV, dtype=I32))
    y = torch.empty(pairs.numel(), width, device=DEV)
    at = starts.tolist()
    for i in range(e):
        if at[i] == at[i + 1]:
            continue
        p = order[at[i]:at[i + 1]]
        x = s["x"][p // top]
        g = x @ _expert(s["gate"], wt, i, inter, width, F32).T
        u = x @ _expert(s["up"], wt, i, inter, width, F32).T
        h = g / (1.0 + torch.exp(-g)) * u
        y[p] = h @ _expert(s["down"], wt, i, width, inter, F32).T
    out = (y.view(-1, top, width) * s["w"][:, :, None]).sum(dim=1)
    return {"order": order.to(I32), "starts": starts.to(I32), "out": out}


# ---------------------------------------------------------------- the framework's calls
def _run_own(s):
    ops, kind = _ops(), s["kind"]
    if kind == "plan":
        start, kv_len, slots, pos, head = ops.kv8_plan(s["cached"], s["fresh"], s["table"], s["free"], s["head"],
                                                       s["page"], s["rows"])
        return {"table": s["table"], "start": start, "len": kv_len, "slots": slots, "pos": pos, "head": head}
    if kind == "moe":
        order, starts = ops.moe_group_rows(s["idx"], s["experts"])
        out = ops.moe_experts_rows(s["gate"], s["up"], s["wtype"], s["down"], s["wtype"], s["experts"], order, starts,
                                   s["w"], s["x"], s["inter"], workspace=s["ws"])
        return {"order": order, "starts": starts, "out": out}
    cache = ops.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if kind == "store":
        ops.kv8_store_rows(s["new_k"], s["new_v"], s["slots"], cache)
        k, v = ops.kv8_read_rows(cache, s["read"])
        return {"k": k, "v": v, "k_scale": s["ks"], "v_scale": s["vs"]}
    return ops.attn_kv8_rows(s["q"], cache, s["table"], s["start"], s["len"], gate=s["gate"], workspace=s["ws"])


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan_plain, "store": _store_plain, "attn": _attn_plain, "moe": _moe_plain}[state["kind"]](state)


# ---------------------------------------------------------------- the work
def work(case):
    kind = case["kind"]
    if kind == "moe":
        rows, e, top, inter, width = (case[k] for k in ("rows", "experts", "top", "inter", "width"))
        pairs = rows * top
        g = torch.Generator().manual_seed(1)   # experts that a routing of this kind touches
        logits = torch.randn(rows, e, generator=g) + 0.5 * torch.randn(e, generator=g)
        touched = torch.unique(torch.topk(logits, top, dim=1).indices).numel()
        block = BLOCK[case["wtype"]] / 256
        return {"bytes": int(touched * 3 * inter * width * block + 4 * (2 * rows * width + 3 * pairs)),
                "flops": 6 * pairs * inter * width}
    cached, fresh = _lengths(case, _Host(1))
    rows, total, page = sum(fresh), sum(cached) + sum(fresh), case["page"]
    if kind == "plan":
        pages = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, fresh))
        return {"bytes": 4 * (4 * len(cached) + 2 * (rows + 7) + 2 * pages + rows), "flops": 4 * rows}
    heads, dim = case["heads"], case["dim"]
    if kind == "store":   # fresh rows read, codes of the touched pages' kept and fresh tokens written, read back once
        kept = sum(c % page for c in cached)
        return {"bytes": 2 * heads * dim * (4 * rows + 2 * kept + rows + 4 * (kept + rows)), "flops": 4 * rows * heads * dim}
    q_heads = case["q_heads"]
    keys = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, fresh))
    return {"bytes": 2 * heads * dim * total + 12 * rows * q_heads * dim, "flops": 4 * q_heads * dim * keys}


# ---------------------------------------------------------------- 64-bit references
def _exact_plan(s):
    page, table = s["page"], s["table"].tolist()
    cached, fresh, free = s["cached"].tolist(), s["fresh"].tolist(), s["free"].tolist()
    head = s["head"].item()
    start, lens, slots, pos, wanted, used = [0], [], [], [], head, head
    for b, (c, n) in enumerate(zip(cached, fresh)):
        have = -(-c // page)
        room = c + n <= page * len(table[b]) and start[-1] + n <= s["rows"]
        need = -(-(c + n) // page) - have if n and room else 0
        wanted += need
        good = room and (need == 0 or wanted <= len(free))
        if good and need:
            table[b][have:have + need] = free[wanted - need:wanted]
            used = wanted
        lens.append(c + n if good else 0)
        start.append(start[-1] + n)
        for t in range(c, c + n):
            pos.append(t)
            slots.append(table[b][t // page] * page + t % page if good else -1)
    pad = s["rows"] - len(pos)
    return {"table": _i32(table), "start": _i32(start), "len": _i32(lens), "slots": _i32(slots + [-1] * pad),
            "pos": _i32(pos + [0] * pad), "head": _i32([used])}


def _exact_quantized(codes, scales, x, slots, read, page):
    """The values of slots `read`, and the scales, after rows x went to `slots` (runs of one page are neighbours)."""
    codes, scales, x = codes.double().cpu(), scales.double().cpu(), x.double().cpu()
    slots = slots.tolist()
    i = 0
    while i < len(slots):
        p, o = divmod(slots[i], page)
        j = i
        while j < len(slots) and slots[j] // page == p:
            j += 1
        xs = x[i:j].transpose(0, 1)                                       # [heads, run, dim]
        old = scales[p] if o else torch.zeros_like(scales[p])
        top = (xs.abs().amax(dim=(1, 2)) / 127).float().double()
        new = torch.stack([old, top, torch.full_like(old, FLOOR)]).amax(0)
        ratio = (old / new).float().double()
        codes[p, :, :o] = torch.round(codes[p, :, :o] * ratio[:, None, None])
        codes[p, :, o:o + j - i] = torch.round(xs / new[:, None, None]).clamp(-127, 127)
        scales[p] = new
        i = j
    r = read.long().cpu()
    values = codes[r // page, :, r % page] * scales[r // page][:, :, None]
    return values.to(DEV), scales.to(DEV)


def _exact_attn(s):
    dim, page, group = s["dim"], s["page"], s["q_heads"] // s["heads"]
    outs, at = [], 0
    for b, (n, total) in enumerate(s["host_lens"]):
        t = torch.arange(total, device=DEV)
        pid, off = s["table"][b][t // page].long(), t % page
        q = s["q"][at:at + n].double()
        o = torch.empty_like(q)
        hidden = t[None, :] > torch.arange(total - n, total, device=DEV)[:, None]
        for h in range(s["q_heads"]):
            g = h // group
            k = s["k"][pid, g, off].double() * s["ks"][pid, g].double()[:, None]
            v = s["v"][pid, g, off // 8, :, off % 8].double() * s["vs"][pid, g].double()[:, None]
            score = (q[:, h] @ k.T / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(score, dim=1) @ v
        outs.append(o)
        at += n
    return torch.cat(outs) * torch.sigmoid(s["gate"].double())


def _exact_weights(raw, wtype, m, k):
    """All of a block tensor's values in 64 bits, element by element of a block from its formula."""
    b = raw.view(-1, BLOCK[wtype]).long()
    i = torch.arange(256, device=DEV)

    def fp16(lo):
        return raw.view(-1, BLOCK[wtype])[:, lo:lo + 2].contiguous().view(torch.float16).double()
    if wtype == "Q4_K":
        g = i // 32
        low = g < 4
        sc = torch.where(low, b[:, 4 + g % 4] & 63, (b[:, 12 + g % 4] & 15) + 16 * (b[:, 4 + g % 4] >> 6))
        mn = torch.where(low, b[:, 8 + g % 4] & 63, (b[:, 12 + g % 4] >> 4) + 16 * (b[:, 8 + g % 4] >> 6))
        q = (b[:, 16 + 32 * (i // 64) + i % 32] >> (4 * (i // 32 % 2))) & 15
        return (fp16(0) * sc * q - fp16(2) * mn).view(m, k)
    half, quarter, col = i // 128, i % 128 // 32, i % 32
    lo = (b[:, 64 * half + 32 * (quarter % 2) + col] >> (4 * (quarter // 2))) & 15
    hi = (b[:, 128 + 32 * half + col] >> (2 * quarter)) & 3
    sc = b[:, 192 + i // 16]
    sc = torch.where(sc > 127, sc - 256, sc)
    return (fp16(208) * sc * (lo + 16 * hi - 32)).view(m, k)


def _exact_moe(s):
    e, top, inter, width, wt = s["experts"], s["top"], s["inter"], s["width"], s["wtype"]
    ids = s["idx"].view(-1).tolist()
    groups = [[] for _ in range(e)]
    for p, i in enumerate(ids):
        groups[i].append(p)
    step = inter * width // 256 * BLOCK[wt]
    out = torch.zeros(len(ids) // top, width, dtype=F64, device=DEV)
    scale = s["w"].view(-1).double()
    for i, members in enumerate(groups):
        if not members:
            continue
        p = torch.tensor(members, device=DEV)
        x = s["x"][p // top].double()
        part = slice(i * step, (i + 1) * step)
        gate = torch.nn.functional.silu(x @ _exact_weights(s["gate"][part], wt, inter, width).T)
        h = gate * (x @ _exact_weights(s["up"][part], wt, inter, width).T)
        out.index_add_(0, p // top, scale[p, None] * (h @ _exact_weights(s["down"][part], wt, width, inter).T))
    starts = [0]
    for members in groups:
        starts.append(starts[-1] + len(members))
    return {"order": _i32([p for members in groups for p in members]), "starts": _i32(starts), "out": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(s)
    if case["kind"] == "store":
        v = s["v"].permute(0, 1, 2, 4, 3).reshape(s["k"].shape)
        k_rows, k_scale = _exact_quantized(s["k"], s["ks"], s["new_k"], s["slots"], s["read"], case["page"])
        v_rows, v_scale = _exact_quantized(v, s["vs"], s["new_v"], s["slots"], s["read"], case["page"])
        return {"k": k_rows, "v": v_rows, "k_scale": k_scale, "v_scale": v_scale}
    return _exact_attn(s) if case["kind"] == "attn" else _exact_moe(s)
