"""Cases of the grouped-query operators: prompt attention, and the 8-bit cache
with a scale for each block of tokens and head (append, decode, attention
weights, eviction).

``run`` computes each operator in its plain form, or, where ``own`` is true,
through the package's public entry points.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
FP8_MAX = 448.0
PACKAGE = "deepseek-v4-flash-sm120_b200"


def _api():
    path = os.path.join(os.getcwd(), PACKAGE)
    if path not in sys.path:
        sys.path.insert(0, path)
    import deepseek_v4_kernel
    return deepseek_v4_kernel


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one long prompt of a grouped-query model
        dict(name="prompt 16384", op="prompt", b=1, shortest=16384, longest=16384, mix=0, h=32, hkv=8, dqk=128,
             dv=128, dtype="bfloat16"),
        # a prefill batch of mixed requests, one-token ones among them
        dict(name="prompts packed", op="prompt", b=24, shortest=1, longest=4099, mix=3, h=64, hkv=8, dqk=128,
             dv=128, dtype="float16"),
        # latent attention's prompt with its heads expanded: 128 + 64 position columns, a KV head each
        dict(name="prompts 192/128", op="prompt", b=2, shortest=1500, longest=2600, mix=1, h=128, hkv=128, dqk=192,
             dv=128, dtype="bfloat16"),
        # one decode step's tokens of a large batch
        dict(name="append step", op="append", b=256, shortest=1, longest=1, mix=5, older=1000, hkv=8, d=128, page=64,
             dtype="bfloat16"),
        # a prefill batch's tokens, some of them behind a prefix that is in the cache already
        dict(name="append prompts", op="append", b=16, shortest=60, longest=4100, mix=6, older=700, hkv=8, d=128,
             page=64, dtype="bfloat16"),
        # one user, a short chat: latency
        dict(name="decode one", op="decode", b=1, shortest=4096, longest=4096, mix=0, sq=1, h=32, hkv=8, d=128,
             page=64, dtype="bfloat16"),
        # an ordinary serving batch with ragged contexts
        dict(name="decode batch", op="decode", b=32, shortest=1000, longest=32768, mix=8, sq=1, h=64, hkv=8, d=128,
             page=64, dtype="bfloat16"),
        # draft verification over long contexts
        dict(name="decode draft long", op="decode", b=16, shortest=120000, longest=131072, mix=9, sq=2, h=64, hkv=8,
             d=128, page=256, dtype="bfloat16"),
        # a decode step's weights, for the running sum that eviction goes by
        dict(name="weights step", op="weights", b=32, shortest=500, longest=16384, mix=10, sq=1, h=64, hkv=8, d=64,
             page=32, dtype="float16"),
        # the weights of a prompt's last queries, the window that eviction after a prompt goes by
        dict(name="weights window", op="weights", b=4, shortest=20000, longest=32768, mix=11, sq=32, h=32, hkv=8,
             d=128, page=128, dtype="bfloat16"),
        # one sequence over its budget
        dict(name="evict one", op="evict", b=1, shortest=8192, longest=8192, mix=0, hkv=8, d=128, page=16,
             budget=2048, recent=256),
        # a batch after its prompts, some of them within the budget
        dict(name="evict batch", op="evict", b=32, shortest=3900, longest=32768, mix=13, hkv=8, d=128, page=64,
             budget=4096, recent=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "append", "decode", "weights", "evict"])
    mix = rng.randrange(1 << 20)
    dtype = rng.choice(["bfloat16", "float16"])
    hkv = rng.choice([1, 2, 3, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 6, 7, 8, 12])
    if op == "prompt":
        longest = _log(rng, 5, 8192)
        b = max(1, min(_log(rng, 1, 64), 16384 // longest))
        dqk, dv = rng.choice([(64, 64), (128, 128), (192, 128)])
        return dict(op=op, b=b, shortest=rng.randint(1, longest), longest=longest, mix=mix, h=hkv * min(group, 4),
                    hkv=hkv, dqk=dqk, dv=dv, dtype=dtype)
    d = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        longest = _log(rng, 1, 4096)
        b = max(1, min(_log(rng, 1, 300), 32768 // longest))
        return dict(op=op, b=b, shortest=rng.randint(1, longest), longest=longest, mix=mix,
                    older=_log(rng, 1, 2000), hkv=min(hkv, 8), d=d, page=page, dtype=dtype)
    if op == "evict":
        longest = _log(rng, 40, 32768)
        b = max(1, min(_log(rng, 1, 64), 524288 // longest))
        budget = rng.randint(max(2, longest // 8), max(3, longest // 2))
        return dict(op=op, b=b, shortest=rng.randint(1, longest), longest=longest, mix=mix, hkv=min(hkv, 8), d=d,
                    page=page, budget=budget, recent=rng.randint(0, budget // 2))
    longest = _log(rng, 33, 100000)
    tokens = 1 << 20 if op == "decode" else 1 << 18
    b = max(1, min(_log(rng, 1, 128), tokens // longest))
    sq = rng.choice([1, 1, 2, 3, 4]) if op == "decode" else rng.choice([1, 1, 5, 16])
    return dict(op=op, b=b, shortest=rng.randint(sq, longest), longest=longest, mix=mix, sq=sq,
                h=min(hkv, 8) * group, hkv=min(hkv, 8), d=d, page=page, dtype=dtype)


def _lens(case):
    """The sequences' lengths: spread over their logarithm, the longest one among them."""
    r = random.Random(case["mix"])
    lens = [_log(r, case["shortest"], case["longest"]) for _ in range(case["b"])]
    lens[r.randrange(case["b"])] = case["longest"]
    return lens


def _older(case):
    """Tokens that are in the cache before an append: every third sequence starts afresh."""
    r = random.Random(case["mix"] + 1)
    return [0 if i % 3 == 2 else r.randint(0, case["older"]) for i in range(case["b"])]


def _total(lens):
    return [0] + [sum(lens[:i + 1]) for i in range(len(lens))]


def work(case):
    lens = _lens(case)
    n, b = sum(lens), case["b"]
    if case["op"] == "prompt":
        h, hkv, dqk, dv = case["h"], case["hkv"], case["dqk"], case["dv"]
        pairs = sum(x * (x + 1) // 2 for x in lens)
        return dict(bytes=n * (h * (dqk + dv) * 2 + hkv * (dqk + dv) * 2 + h * 4) + 4 * (b + 1),
                    flops=2 * pairs * h * (dqk + dv))
    hkv, d, page = case["hkv"], case["d"], case["page"]
    pages = sum(-(-x // page) for x in lens)
    if case["op"] == "append":
        pages = sum(-(-(o + x) // page) - o // page for o, x in zip(_older(case), lens))
        return dict(bytes=2 * n * hkv * d * 3 + 2 * pages * hkv * 4 + pages * 4 + 8 * b, flops=2 * n * hkv * d * 2)
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lens)
        return dict(bytes=n * hkv * 4 + kept * hkv * (4 * d + 8) + pages * (4 + 8 * hkv), flops=2 * kept * hkv * d)
    h, sq = case["h"], case["sq"]
    if case["op"] == "decode":
        return dict(bytes=n * hkv * 2 * d + pages * (4 + 8 * hkv) + b * sq * h * (4 * d + 4),
                    flops=4 * n * sq * h * d)
    return dict(bytes=n * hkv * (d + 4) + pages * (4 + 4 * hkv) + b * sq * h * (2 * d + 4), flops=2 * n * sq * h * d)


# ------------------------------------------------------------------ their inputs
def _table(lens, page, g, spare=0):
    """Block table [b, pages of the longest + 1] of randomly placed pages (0 where a sequence has none), and the
    number of pages."""
    counts = torch.tensor([-(-x // page) for x in lens])
    width = int(counts.max()) + 1
    used = torch.arange(width)[None] < counts[:, None]
    total = int(counts.sum())
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    table[used] = torch.randperm(total, generator=g).int() + spare
    return table.to(DEV), total


def _cache(blocks, page, hkv, d, g):
    """A filled cache: each head has a magnitude of its own, each block a scale of two's power."""
    kv, scales = [], []
    for _ in range(2):
        size = torch.exp2(torch.randint(-1, 2, (1, hkv), generator=g, device=DEV).float())
        scale = size * torch.exp2(torch.randint(-8, -5, (blocks, hkv), generator=g, device=DEV).float())
        c = torch.empty(blocks, page, hkv, d, dtype=torch.float8_e4m3fn, device=DEV)
        step = max(1, (1 << 27) // (page * hkv * d))
        for i in range(0, blocks, step):
            x = torch.randn(min(step, blocks - i), page, hkv, d, generator=g, device=DEV)
            c[i:i + step] = (x * 80).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
        kv.append(c)
        scales.append(scale)
    return kv[0], kv[1], scales[0], scales[1]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    lens = _lens(case)
    s = dict(case=case, lens=lens)
    if case["op"] == "prompt":
        dtype = getattr(torch, case["dtype"])
        n, h, hkv, dqk, dv = sum(lens), case["h"], case["hkv"], case["dqk"], case["dv"]
        # one projection's output, of which q, k and v are parts
        x = torch.randn(n, h * dqk + hkv * (dqk + dv), generator=g, device=DEV).to(dtype)
        q, k, v = x.split([h * dqk, hkv * dqk, hkv * dv], dim=1)
        s.update(q=q.unflatten(1, (h, dqk)), k=k.unflatten(1, (hkv, dqk)), v=v.unflatten(1, (hkv, dv)),
                 cu=torch.tensor(_total(lens), dtype=torch.int32, device=DEV), scale=dqk ** -0.5)
        return s
    hkv, d, page = case["hkv"], case["d"], case["page"]
    if case["op"] == "append":
        dtype = getattr(torch, case["dtype"])
        older = _older(case)
        ctx = [o + x for o, x in zip(older, lens)]
        s["table"], blocks = _table(ctx, page, gc)
        s["kc"], s["vc"], s["ks"], s["vs"] = _cache(blocks, page, hkv, d, g)
        size = torch.exp(torch.randn(sum(lens), 1, 1, generator=g, device=DEV) * 0.5)
        s["k"] = (torch.randn(sum(lens), hkv, d, generator=g, device=DEV) * size).to(dtype)
        s["v"] = (torch.randn(sum(lens), hkv, d, generator=g, device=DEV) * size).to(dtype)
        s["cu"] = torch.tensor(_total(lens), dtype=torch.int32, device=DEV)
        s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        return s
    s["ctx"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if case["op"] == "evict":
        budget = case["budget"]
        new_lens = [min(x, budget) for x in lens]
        new, blocks = _table(new_lens, page, gc)
        s["table"], more = _table(lens, page, gc, spare=blocks)
        s["new"], s["blocks"] = new, blocks
        s["kc"], s["vc"], s["ks"], s["vs"] = _cache(blocks + more, page, hkv, d, g)
        # a few positions draw most of the weight; some were never looked at and tie at zero
        w = torch.randn(case["b"], hkv, max(lens), generator=g, device=DEV).mul_(2).exp_()
        s["w"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.3, torch.zeros_like(w), w)
        return s
    dtype = getattr(torch, case["dtype"])
    s["table"], blocks = _table(lens, page, gc)
    s["kc"], s["vc"], s["ks"], s["vs"] = _cache(blocks, page, hkv, d, g)
    s["q"] = torch.randn(case["b"], case["sq"], case["h"], d, generator=g, device=DEV).to(dtype)
    s["scale"] = d ** -0.5
    if case["op"] == "weights":
        s["lse"] = torch.logsumexp(_scores(s), dim=-1)
    return s


# ------------------------------------------------------------------ the plain forms
def _prompt(s):
    """Softmax attention of each packed sequence, some rows at a time so that the scores fit."""
    q, k, v, cu = s["q"], s["k"], s["v"], _total(s["lens"])
    h, hkv = q.shape[1], k.shape[1]
    out = torch.empty(q.shape[0], h, v.shape[2], dtype=q.dtype, device=DEV)
    lse = torch.empty(q.shape[0], h, device=DEV)
    for lo, hi in zip(cu[:-1], cu[1:]):
        kt = k[lo:hi].float().permute(1, 2, 0)[:, None]
        vt = v[lo:hi].float().transpose(0, 1)[:, None]
        rows = max(128, (1 << 30) // (h * (hi - lo)))
        for a in range(lo, hi, rows):
            e = min(hi, a + rows)
            qt = q[a:e].float().permute(1, 0, 2).reshape(hkv, h // hkv, e - a, -1)
            x = (qt @ kt) * s["scale"]
            ahead = torch.arange(hi - lo, device=DEV)[None] > torch.arange(a - lo, e - lo, device=DEV)[:, None]
            x.masked_fill_(ahead, -math.inf)
            m = x.amax(-1, keepdim=True)
            x = x.sub_(m).exp_()
            total = x.sum(-1, keepdim=True)
            o = (x @ vt) / total
            out[a:e] = o.reshape(h, e - a, -1).transpose(0, 1).to(q.dtype)
            lse[a:e] = (m + total.log()).reshape(h, e - a).T
    return out, lse


def _held(cache, scale, table):
    """The values [b, h_kv, length, d] that a table's pages stand for."""
    x = cache.view(torch.uint8)[table.long()].view(torch.float8_e4m3fn).float() * scale[table.long()][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2)


def _scores(s):
    """Scaled scores [b, h_q, s_q, length], -inf where a query sees nothing."""
    q = s["q"].float()
    b, sq, h, d = q.shape
    k = _held(s["kc"], s["ks"], s["table"])
    hkv, length = k.shape[1], k.shape[2]
    qt = q.permute(0, 2, 1, 3).reshape(b, hkv, (h // hkv) * sq, d)
    x = ((qt @ k.transpose(2, 3)) * s["scale"]).view(b, h, sq, length)
    end = s["ctx"][:, None] - sq + 1 + torch.arange(sq, device=DEV)[None]
    return x.masked_fill_(torch.arange(length, device=DEV) >= end[:, None, :, None], -math.inf)


def _decode(s):
    x = _scores(s)
    b, h, sq, length = x.shape
    v = _held(s["vc"], s["vs"], s["table"])
    hkv = v.shape[1]
    m = x.amax(-1, keepdim=True)
    x = (x - m).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(b, hkv, (h // hkv) * sq, length) @ v).view(b, h, sq, -1) / total
    return o.transpose(1, 2).to(s["q"].dtype), (m + total.log()).squeeze(-1)


def _weights(s):
    x = (_scores(s) - s["lse"][..., None]).exp_()
    b, h, sq, length = x.shape
    return x.view(b, s["kc"].shape[2], -1, length).sum(2)[..., :max(s["lens"])]


def _exponent(amax):
    """The smallest e >= -100 with amax <= 448 * 2^e."""
    m, x = torch.frexp(amax)
    return (x - 9 + (m > 0.875).int()).masked_fill(amax == 0, -100).clamp_min(-100)


def _append_one(x, cache, scale, s):
    case = s["case"]
    page = case["page"]
    n = s["cu"][1:] - s["cu"][:-1]
    first = s["ctx"] - n
    seq = torch.repeat_interleave(torch.arange(case["b"], device=DEV), n.long(), output_size=x.shape[0])
    pos = torch.arange(x.shape[0], device=DEV) - s["cu"][seq] + first[seq]
    block = s["table"][seq, pos // page].long()
    x = x.float()
    need = torch.zeros_like(scale).index_reduce_(0, block, x.abs().amax(-1), "amax")
    need = torch.exp2(_exponent(need).float())
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV).index_fill_(0, block, True)
    # the pages that held tokens before keep the larger scale, and their rows the values they stand for
    begun = s["table"][torch.arange(case["b"], device=DEV), first // page].long()
    kept = torch.zeros_like(touched).index_fill_(0, begun[first % page > 0], True)[:, None]
    new = torch.where(touched[:, None], torch.where(kept, torch.maximum(need, scale), need), scale)
    old_rows = torch.arange(page, device=DEV)[None] < (first % page)[:, None]
    ratio = (scale / new)[begun]
    rows = cache.view(torch.uint8)[begun]
    moved = (rows.view(torch.float8_e4m3fn).float() * ratio[:, None, :, None]).to(torch.float8_e4m3fn)
    rows = torch.where(old_rows[..., None, None], moved.view(torch.uint8), rows)
    at = old_rows.nonzero(as_tuple=True)
    cache.view(torch.uint8)[begun[at[0]], at[1]] = rows[at]
    scale.copy_(new)
    y = (x / new[block][..., None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[block, pos % page] = y.view(torch.uint8)


def _append(s):
    _append_one(s["k"], s["kc"], s["ks"], s)
    _append_one(s["v"], s["vc"], s["vs"], s)


def _evict(s):
    case = s["case"]
    b, hkv, page, budget, recent = case["b"], case["hkv"], case["page"], case["budget"], case["recent"]
    w, ctx = s["w"], s["ctx"].long()[:, None, None]
    width = w.shape[2]
    pos = torch.arange(width, device=DEV)
    key = w.masked_fill(pos >= ctx - recent, math.inf).masked_fill(pos >= ctx, -math.inf)
    if width < budget:
        key = torch.nn.functional.pad(key, (0, budget - width), value=-math.inf)
    kept = key.sort(dim=-1, descending=True, stable=True)[1][..., :budget]
    new_lens = s["ctx"].clamp_max(budget)
    there = torch.arange(budget, device=DEV) < new_lens[:, None, None]
    kept = torch.where(there, kept, torch.full_like(kept, 1 << 40)).sort(dim=-1)[0]
    kept = torch.where(there, kept, torch.full_like(kept, -1))
    new_w = torch.where(there, w.gather(2, kept.clamp(0, width - 1)), torch.zeros((), device=DEV))
    seq = torch.arange(b, device=DEV)[:, None, None]
    head = torch.arange(hkv, device=DEV)[None, :, None].expand(b, hkv, budget)
    source = s["table"][seq, kept.clamp_min(0) // page].long()
    j = torch.arange(budget, device=DEV).expand(b, hkv, budget)
    dest = s["new"][seq, (j // page).clamp_max(s["new"].shape[1] - 1)].long()
    at = there.expand(b, hkv, budget)
    source, dest, head, off, j = source[at], dest[at], head[at], (kept % page)[at], (j % page)[at]
    for cache, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        old = scale[source, head]
        flat = scale.view(-1)
        top = torch.zeros_like(flat).index_reduce_(0, dest * hkv + head, old, "amax")
        new = top[dest * hkv + head]
        y = cache.view(torch.uint8)[source, off, head].view(torch.float8_e4m3fn).float() * (old / new)[:, None]
        cache.view(torch.uint8)[dest, j, head] = y.to(torch.float8_e4m3fn).view(torch.uint8)
        scale[dest, head] = new
    return kept.int(), new_w, new_lens


def run(state):
    s, op = state, state["case"]["op"]
    if op == "prompt":
        if own:
            return _api().gqa_prefill_fwd(s["q"], s["k"], s["v"], s["cu"], sm_scale=s["scale"])
        return _prompt(s)
    if op == "append":
        if own:
            _api().gqa_cache_append(s["k"], s["v"], s["cu"], s["ctx"], s["table"], s["kc"], s["vc"], s["ks"], s["vs"])
        else:
            _append(s)
        return s["kc"], s["vc"], s["ks"], s["vs"]
    if op == "decode":
        if own:
            return _api().gqa_decode_fwd(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["ctx"],
                                         sm_scale=s["scale"])
        return _decode(s)
    if op == "weights":
        if own:
            return _api().gqa_attention_weights(s["q"], s["lse"], s["kc"], s["ks"], s["table"], s["ctx"],
                                                sm_scale=s["scale"], max_context=max(s["lens"]))
        return _weights(s)
    if own:
        kept, new_w, new_lens = _api().gqa_cache_evict(s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["ctx"],
                                                       s["w"], s["case"]["budget"], s["case"]["recent"], s["new"])
    else:
        kept, new_w, new_lens = _evict(s)
    n = s["blocks"]
    return kept, new_w, new_lens, s["kc"][:n], s["vc"][:n], s["ks"][:n], s["vs"][:n]


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_rows(q, k, v, scale, first):
    """Attention of one KV head's queries [rows, g, d] over keys [n, d]: row r sees the keys up to first + r."""
    x = torch.einsum("rgd,nd->grn", q.double(), k.double()) * scale
    sees = torch.arange(k.shape[0], device=DEV)[None] <= first + torch.arange(q.shape[0], device=DEV)[:, None]
    x = torch.where(sees, x, torch.full((), -math.inf, dtype=torch.float64, device=DEV))
    lse = torch.logsumexp(x, dim=-1)
    o = None
    if v is not None:
        o = torch.einsum("grn,nd->rgd", torch.softmax(x, dim=-1), v.double())
    return x, o, lse


def _exact_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hkv = q.shape[1], k.shape[1]
    g = h // hkv
    out = torch.empty(q.shape[0], h, v.shape[2], dtype=torch.float64, device=DEV)
    lse = torch.empty(q.shape[0], h, dtype=torch.float64, device=DEV)
    lo = 0
    for n in s["lens"]:
        rows = max(64, (1 << 28) // (n * g))
        for kh in range(hkv):
            for a in range(0, n, rows):
                e = min(n, a + rows)
                _, o, l = _exact_rows(q[lo + a:lo + e, kh * g:(kh + 1) * g], k[lo:lo + e, kh], v[lo:lo + e, kh],
                                      s["scale"], a)
                out[lo + a:lo + e, kh * g:(kh + 1) * g] = o
                lse[lo + a:lo + e, kh * g:(kh + 1) * g] = l.T
        lo += n
    return out, lse


def _exact_held(cache, scale, table, n, kh):
    pages = table[:-(-n // cache.shape[1])].long()
    x = cache[:, :, kh].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * scale[pages, kh].double()[:, None, None]
    return x.reshape(-1, cache.shape[3])[:n]


def _exact_cached(s, with_v):
    """Per sequence and KV head: (sequence, head, scores [g, s_q, n], out, lse)."""
    q, hkv, sq = s["q"], s["kc"].shape[2], s["case"]["sq"]
    g = q.shape[2] // hkv
    for i, n in enumerate(s["lens"]):
        for kh in range(hkv):
            k = _exact_held(s["kc"], s["ks"], s["table"][i], n, kh)
            v = _exact_held(s["vc"], s["vs"], s["table"][i], n, kh) if with_v else None
            yield (i, kh) + _exact_rows(q[i, :, kh * g:(kh + 1) * g], k, v, s["scale"], n - sq)


def _exact_decode(s):
    b, sq, h, d = s["q"].shape
    g = h // s["kc"].shape[2]
    out = torch.empty(b, sq, h, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(b, h, sq, dtype=torch.float64, device=DEV)
    for i, kh, _, o, l in _exact_cached(s, True):
        out[i, :, kh * g:(kh + 1) * g] = o
        lse[i, kh * g:(kh + 1) * g] = l
    return out, lse


def _exact_weights(s):
    g = s["case"]["h"] // s["case"]["hkv"]
    w = torch.zeros(s["case"]["b"], s["case"]["hkv"], max(s["lens"]), dtype=torch.float64, device=DEV)
    for i, kh, x, _, _ in _exact_cached(s, False):
        p = torch.exp(x - s["lse"][i, kh * g:(kh + 1) * g].double()[..., None])
        w[i, kh, :x.shape[2]] = p.sum((0, 1))
    return w


def _e4m3(x):
    """The nearest e4m3 value, ties to even, of a number within +-448."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    case, out = s["case"], []
    page, ctx = case["page"], s["ctx"].tolist()
    cu = _total(s["lens"])
    for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        c, sc = cache.double(), scale.double()
        for i, table in enumerate(s["table"].tolist()):
            pos = ctx[i] - (cu[i + 1] - cu[i])
            t = cu[i]
            while t < cu[i + 1]:
                p, off = table[pos // page], pos % page
                n = min(page - off, cu[i + 1] - t)
                new = x[t:t + n].double()
                need = new.abs().amax((0, 2)) / FP8_MAX
                e = torch.ceil(torch.log2(need.clamp_min(2.0 ** -100)))
                e = torch.where(torch.exp2(e - 1) >= need, e - 1, e).clamp_min(-100.0)
                size = torch.exp2(e)
                if off:
                    size = torch.maximum(size, sc[p])
                    c[p, :off] = _e4m3(c[p, :off] * (sc[p] / size)[None, :, None])
                sc[p] = size
                c[p, off:off + n] = _e4m3((new / size[None, :, None]).clamp(-FP8_MAX, FP8_MAX))
                t, pos = t + n, pos + n
        out.append((c, sc))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_evict(s):
    case = s["case"]
    b, hkv, page, budget, recent = case["b"], case["hkv"], case["page"], case["budget"], case["recent"]
    kept = torch.full((b, hkv, budget), -1, dtype=torch.int32, device=DEV)
    new_w = torch.zeros(b, hkv, budget, dtype=torch.float64, device=DEV)
    n = s["blocks"]
    caches = [c[:n].double() for c in (s["kc"], s["vc"])]
    scales = [c[:n].double() for c in (s["ks"], s["vs"])]
    for i, length in enumerate(s["lens"]):
        m = min(length, budget)
        old = max(0, length - recent)
        w = s["w"][i, :, :length]
        if length > budget:
            # the lightest of the older positions go, the highest position first where weights tie
            order = torch.argsort(w[:, :old].flip(1), dim=1, stable=True)
            gone = torch.zeros(hkv, length, dtype=torch.bool, device=DEV)
            gone.scatter_(1, old - 1 - order[:, :length - budget], True)
            pos = (~gone).nonzero()[:, 1].view(hkv, m)
        else:
            pos = torch.arange(length, device=DEV).expand(hkv, length)
        kept[i, :, :m] = pos.int()
        new_w[i, :, :m] = w.gather(1, pos).double()
        head = torch.arange(hkv, device=DEV)[:, None]
        for cache, scale, c, sc in ((s["kc"], s["ks"], caches[0], scales[0]), (s["vc"], s["vs"], caches[1], scales[1])):
            source = s["table"][i].long()[pos // page]
            size = scale[source, head].double()
            x = cache.view(torch.uint8)[source, pos % page, head].view(torch.float8_e4m3fn).double()
            pad = -m % page
            size = torch.nn.functional.pad(size, (0, pad)).view(hkv, -1, page)
            x = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(hkv, -1, page, x.shape[-1])
            top = size.amax(-1)
            y = _e4m3(x * (size / top[..., None])[..., None])
            pages = s["new"][i, :top.shape[1]].long()
            sc[pages] = top.T
            whole = m // page
            c[pages[:whole]] = y[:, :whole].permute(1, 2, 0, 3)
            if pad:
                c[pages[whole], :m - whole * page] = y[:, whole, :m - whole * page].transpose(0, 1)
    return kept, new_w, s["ctx"].clamp_max(budget), caches[0], caches[1], scales[0], scales[1]


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "append": _exact_append, "decode": _exact_decode, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](s)
